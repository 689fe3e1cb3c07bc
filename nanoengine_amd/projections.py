"""From a layer's hidden states to the inputs of the DSA step and from its output back, on one GPU.

What surrounds ``DsaDecodeStep`` in a layer (the projections of DeepseekV2Attention.forward,
dlengine/runtime/models/deepseek_v2/deepseek_v2.py:1860-2018), with MLA in its absorbed form:

    h     = norm(hidden + residual), fp8                          rms_norm_quant (bf16 too, for the gate)
    c     = h W_a          [query latent | kv latent | rotated key | indexer key]   fp8_gemm
    q     = norm(c_q) W_q  heads of [nope | 64 rotated]           rms_norm_quant, fp8_gemm
    q_mla = [q_nope W_uk | rope(q_rot)],  kv = [norm(c_kv) | rope(k_rot)]           rope, one launch for both
    indexer query and gate -> indexer_q_prologue, its key -> indexer_k_transform_store, kv -> mla_kv_store

and, behind the step, attention = quant(o W_uv) W_o (act_quant, fp8_gemm). Weights are fp8 with a scale per
128 x 128 block, quantised once when the layer is made. The two products per head (W_uk, W_uv) are plain batched
bf16 products of the library. Every call allocates its results from torch's allocator; captured in a HIP graph they
come from the graph's pool.
"""
from __future__ import annotations

import torch

from . import ops

ROT = ops.MLA_D_QK - ops.MLA_D_V          # rotated dims of a head: 64
KV_RANK = ops.MLA_D_V                     # 512
IDX_HEADS = 64


def quantize_weight(weight: torch.Tensor, scale_dtype: torch.dtype = torch.float8_e8m0fnu):
    """[N, K] -> (codes [N, K] float8_e4m3fn, scales [ceil(N / 128), ceil(K / 128)]): a scale per 128 x 128 block, by
    the rule of ``ops.act_quant`` (max(amax, 2^-40) / 448, or the power of two above; a NaN counts for no scale)."""
    if scale_dtype not in (torch.float32, torch.float8_e8m0fnu):
        raise ValueError(f"scale_dtype must be float32 or float8_e8m0fnu, got {scale_dtype}")
    (N, K), B = weight.shape, ops.FP8_BLOCK
    full = torch.nn.functional.pad(weight.float(), (0, -K % B, 0, -N % B)).view(-(-N // B), B, -(-K // B), B)
    top = full.abs().masked_fill(full.isnan(), 0.0).amax(dim=(1, 3)).clamp_min(2.0 ** -40)
    scale = top / torch.full_like(top, 448.0)  # (by a number, torch multiplies with its rounded inverse on the GPU)
    if scale_dtype is torch.float8_e8m0fnu:
        bits = scale.view(torch.int32)  # positive: the exponent, one more where a fraction is left
        byte = ((bits >> 23) + ((bits & 0x7FFFFF) != 0).to(torch.int32)).clamp_max(254)
        stored, scale = byte.to(torch.uint8).view(scale_dtype), (byte << 23).view(torch.float32)
    else:
        stored = scale
    codes = (full / scale[:, None, :, None]).to(torch.float8_e4m3fn)
    return codes.view(full.shape[0] * B, -1)[:N, :K].contiguous(), stored


class Fp8Linear:
    """x @ weight.T with the weight in fp8 by blocks of 128 x 128."""

    def __init__(self, weight: torch.Tensor, scale_dtype: torch.dtype = torch.float8_e8m0fnu):
        if weight.shape[1] % 16:
            raise ValueError(f"fp8 products take a depth that is a multiple of 16, got {list(weight.shape)}")
        self.codes, self.scales = quantize_weight(weight, scale_dtype)

    def __call__(self, codes: torch.Tensor, scales: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        return ops.fp8_gemm(codes, scales, self.codes, self.scales, out=out)


class MlaProjections:
    """The projections of one layer. Weights [out, in] bf16 or float32 on the GPU:

    norm [D]; a [q_rank + 512 + 64 + 128, D] (query latent, kv latent, rotated key, indexer key); q_norm [q_rank];
    kv_norm [512]; q [H * (nope + 64), q_rank]; k_up [H, nope, 512]; v_up [H, 512, v]; o [D, H * v];
    idx_q [64 * 128, q_rank]; idx_gate [64, D]; idx_norm, idx_bias [128]. D, q_rank and H * v are multiples of 16.
    ``cos_sin_cache``: ``rotary.cos_sin_cache``.
    ``interleaved`` says whether the pairs of the MLA's rotated dims (the tails of q's heads and the shared key) lie beside each
    other or in halves, ``indexer_interleaved`` the same of the indexer's (the heads' first 64 dims and its key's): as the
    MLA's unless given. ``sm_scale`` of the attention is the step's own argument."""

    def __init__(self, *, norm, a, q_norm, kv_norm, q, k_up, v_up, o, idx_q, idx_gate, idx_norm, idx_bias,
                 cos_sin_cache: torch.Tensor, eps: float = 1e-6, interleaved: bool = True,
                 scale_dtype: torch.dtype = torch.float8_e8m0fnu, indexer_interleaved: bool | None = None):
        self.heads, self.nope = k_up.shape[0], k_up.shape[1]
        self.q_rank, self.eps, self.interleaved, self.scale_dtype = q_norm.shape[0], eps, interleaved, scale_dtype
        self.indexer_interleaved = interleaved if indexer_interleaved is None else indexer_interleaved
        D = norm.shape[0]
        want = {"a": (a, (self.q_rank + KV_RANK + ROT + ops.INDEXER_HEAD_DIM, D)), "kv_norm": (kv_norm, (KV_RANK,)),
                "q": (q, (self.heads * (self.nope + ROT), self.q_rank)), "k_up": (k_up, (self.heads, self.nope, KV_RANK)),
                "v_up": (v_up, (self.heads, KV_RANK, v_up.shape[-1])), "o": (o, (D, self.heads * v_up.shape[-1])),
                "idx_q": (idx_q, (IDX_HEADS * ops.INDEXER_HEAD_DIM, self.q_rank)), "idx_gate": (idx_gate, (IDX_HEADS, D))}
        for name, (t, shape) in want.items():
            if tuple(t.shape) != shape:
                raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
        bf16 = torch.bfloat16
        self.norm, self.q_norm, self.kv_norm = norm.contiguous(), q_norm.contiguous(), kv_norm.contiguous()
        self.a, self.q, self.o, self.idx_q = (Fp8Linear(w, scale_dtype) for w in (a, q, o, idx_q))
        self.k_up, self.v_up = k_up.to(bf16).contiguous(), v_up.to(bf16).contiguous()
        self.idx_gate = idx_gate.to(bf16).contiguous()
        self.idx_norm, self.idx_bias = idx_norm.float().contiguous(), idx_bias.float().contiguous()
        self.cos_sin_cache = ops._rope_cache(cos_sin_cache)

    def inputs(self, hidden: torch.Tensor, residual: torch.Tensor | None, positions: torch.Tensor,
               slot_mapping: torch.Tensor, kv_cache: torch.Tensor, indexer_cache: torch.Tensor, page_size: int = 64):
        """hidden [T, D] bf16 of one layer's tokens. Writes their rows of both caches at ``slot_mapping`` (-1: none) and
        returns (q_idx [T, 64, 128] fp8, weights [T, 64] f32, q_mla [T, H, 576] bf16, residual): the step's arguments
        and the residual stream, which is ``residual`` itself, updated, or ``hidden`` where there is none yet. Arguments
        that do not fit are refused before it is updated."""
        T, rank, H = hidden.shape[0], self.q_rank, self.heads
        q_idx = torch.empty(T, IDX_HEADS, ops.INDEXER_HEAD_DIM, dtype=torch.float8_e4m3fn, device=hidden.device)
        weights = torch.empty(T, IDX_HEADS, dtype=torch.float32, device=hidden.device)
        q_mla = torch.empty(T, H, ops.MLA_D_QK, dtype=torch.bfloat16, device=hidden.device)
        stream = hidden if residual is None else residual
        if T == 0:
            return q_idx, weights, q_mla, stream
        ops._positions(positions, T)
        ops._slots(slot_mapping, T)
        ops.mla_kv_geometry(kv_cache)
        ops._key_pages(indexer_cache, page_size, ops.INDEXER_ROW_BYTES)
        ops._gpu(hidden, positions, slot_mapping, kv_cache, indexer_cache)
        h = torch.empty_like(hidden)
        coded = ops.rms_norm_quant(hidden, self.norm, self.eps, out=h, residual=residual, residual_out=residual,
                                   scale_dtype=self.scale_dtype)
        c = self.a(*coded)
        c_q = ops.rms_norm_quant(c[:, :rank], self.q_norm, self.eps, scale_dtype=self.scale_dtype)
        kv = c.new_empty(T, ops.MLA_D_QK)
        ops.rms_norm(c[:, rank:rank + KV_RANK], self.kv_norm, self.eps, out=kv[:, :KV_RANK])
        q = self.q(*c_q).view(T, H, self.nope + ROT)
        q_mla[..., :KV_RANK] = torch.bmm(q[..., :self.nope].transpose(0, 1), self.k_up).transpose(0, 1)
        at = rank + KV_RANK
        ops.rope(q[..., self.nope:], positions, self.cos_sin_cache, out=q_mla[..., KV_RANK:],
                 k=c[:, at:at + ROT].unsqueeze(1), k_out=kv[:, KV_RANK:].unsqueeze(1), interleaved=self.interleaved)
        ops.mla_kv_store(kv, kv_cache, slot_mapping)
        ops.indexer_k_transform_store(c[:, at + ROT:], self.idx_norm, self.idx_bias, self.eps, positions,
                                      self.cos_sin_cache, indexer_cache, slot_mapping, page_size,
                                      self.indexer_interleaved)
        ops.indexer_q_prologue(self.idx_q(*c_q).view(T, IDX_HEADS, ops.INDEXER_HEAD_DIM), h @ self.idx_gate.t(),
                               IDX_HEADS ** -0.5 * ops.INDEXER_HEAD_DIM ** -0.5, self.cos_sin_cache, positions, q_idx,
                               weights, self.indexer_interleaved)
        return q_idx, weights, q_mla, stream

    def output(self, o: torch.Tensor) -> torch.Tensor:
        """The step's attention output [T, H, 512] bf16 -> [T, D] bf16."""
        v = torch.bmm(o.transpose(0, 1), self.v_up).transpose(0, 1).flatten(1)
        return self.o(*ops.act_quant(v, scale_dtype=self.scale_dtype))
