"""Performance cases of what surrounds the DSA attention in a layer: the norms, the 8-bit products and the rotary
positions that lead from hidden states to the indexer's and the attention's queries and keys, and back.

A layer adds its input to the residual stream, normalises it and rounds it to fp8 with a scale per 128 elements
(``norm``), takes it through 8-bit projections whose weights have a scale per 128 x 128 block (``gemm``), normalises
the latent queries and keys (``norm`` again, over rows inside wider ones), turns the positional part of each head
(``rope``), attends, and rounds the attention's output for the output projection (``quant``).

Scales are float32 (largest magnitude / 448) or a power of two held as its exponent (torch.float8_e8m0fnu).
"""
from __future__ import annotations

import math
import random

import torch

own = False  # False: the operators' plain forms; True: the framework's kernels

DEV = "cuda"
EPS = 1e-6
BLOCK = 128
FP8 = torch.float8_e4m3fn
E8M0 = torch.float8_e8m0fnu
BF16 = torch.bfloat16


def listed():
    return [
        # four interactive requests, one token each: the layer's first norm, whose result goes into 8-bit products
        {"name": "norm_b4", "kind": "norm", "tokens": 4, "dim": 8192, "row": 8192, "residual": True, "keep": False,
         "fp8": True, "scale": "e8m0"},
        # the latent keys of a ragged prefill: 512 dims inside the 576-wide rows of the down projection's output
        {"name": "norm_latent_1000", "kind": "norm", "tokens": 1000, "dim": 512, "row": 576, "residual": False,
         "keep": True, "fp8": False, "scale": "none"},
        # the benchmark's prefill chunk: residual stream, bf16 for the head weights' product and fp8 for the others
        {"name": "norm_8k", "kind": "norm", "tokens": 8192, "dim": 8192, "row": 8192, "residual": True, "keep": True,
         "fp8": True, "scale": "f32"},
        # the benchmark's decode batch: the attention's output before the output projection
        {"name": "quant_b128", "kind": "quant", "tokens": 128, "dim": 16384, "scale": "f32"},
        # an odd number of tokens, rows that end inside a block
        {"name": "quant_5001", "kind": "quant", "tokens": 5001, "dim": 1600, "scale": "e8m0"},
        # one interactive request: the indexer's queries (64 heads of 128) from the latent ones
        {"name": "gemm_b1", "kind": "gemm", "tokens": 1, "n": 8192, "k": 1536, "scale": "e8m0"},
        # the benchmark's decode batch: all heads' queries (128 heads of 192)
        {"name": "gemm_b128", "kind": "gemm", "tokens": 128, "n": 24576, "k": 1536, "scale": "f32"},
        # a mixed batch through the down projection (latent queries and the 576-wide keys)
        {"name": "gemm_333_down", "kind": "gemm", "tokens": 333, "n": 2112, "k": 8192, "scale": "e8m0"},
        # the benchmark's prefill chunk through the output projection
        {"name": "gemm_8k_out", "kind": "gemm", "tokens": 8192, "n": 8192, "k": 16384, "scale": "e8m0"},
        # four interactive requests: the positional part of every head's query and of the shared key
        {"name": "rope_b4", "kind": "rope", "tokens": 4, "heads": 128, "head": 192, "rot": 64, "pairs": True,
         "out_pairs": True, "wide": True, "table": 131072},
        # one rank of an eight-way tensor-parallel group, half layout, an odd batch
        {"name": "rope_257_tp8", "kind": "rope", "tokens": 257, "heads": 16, "head": 192, "rot": 64, "pairs": False,
         "out_pairs": False, "wide": False, "table": 32768},
        # the benchmark's prefill chunk, pairs in, halves out
        {"name": "rope_8k", "kind": "rope", "tokens": 8192, "heads": 128, "head": 192, "rot": 64, "pairs": True,
         "out_pairs": False, "wide": True, "table": 131072},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "quant", "gemm", "gemm", "gemm", "rope", "rope"])
    if kind == "norm":
        dim = rng.choice([512, 1536, 2048, 4096, 5120, 8192, 1000, 16 * rng.randint(4, 512)])
        fp8 = rng.random() < 0.6
        return {"kind": kind, "tokens": _log(rng, 1, 8192), "dim": dim, "row": dim + rng.choice([0, 0, 64, 8]),
                "residual": rng.random() < 0.5, "keep": not fp8 or rng.random() < 0.5, "fp8": fp8,
                "scale": rng.choice(["f32", "e8m0"]) if fp8 else "none"}
    if kind == "quant":
        return {"kind": kind, "tokens": _log(rng, 1, 8192), "dim": rng.choice([128, 1536, 4096, 8192, 8 * rng.randint(8, 1024)]),
                "scale": rng.choice(["f32", "e8m0"])}
    if kind == "gemm":
        n, k = rng.choice([576, 2112, 4096, 8192, rng.randint(64, 8192)]), rng.choice([512, 1536, 2048, 8192, 16 * rng.randint(8, 512)])
        return {"kind": kind, "tokens": _log(rng, 1, 8192), "n": n, "k": k, "scale": rng.choice(["f32", "e8m0", "e8m0"])}
    pairs = rng.random() < 0.6
    rot = rng.choice([64, 64, 32, 128])
    return {"kind": kind, "tokens": _log(rng, 1, 8192), "heads": rng.choice([1, 8, 16, 64, 96]),
            "head": rot + rng.choice([0, 64, 128]), "rot": rot, "pairs": pairs, "out_pairs": pairs and rng.random() < 0.5,
            "wide": rng.random() < 0.5, "table": rng.choice([4096, 32768, 131072])}


def _ceil(a, b):
    return -(-a // b)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rnd(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _hidden(gen, tokens, dim):
    """Activations: channels of different size, a few of them far larger than the others."""
    channel = torch.exp(0.4 * _rnd(gen, dim))
    channel[torch.randint(0, dim, (max(1, dim // 1000),), generator=gen, device=DEV)] *= 30.0
    return (_rnd(gen, tokens, dim) * channel).to(BF16)


def _scales(kind, *shape):
    return torch.empty(*shape, dtype=torch.float32 if kind == "f32" else E8M0, device=DEV)


def prepare(case, seed):
    return globals()["_prepare_" + case["kind"]](case, seed)


def _prepare_norm(case, seed):
    gen, T, D = _gen(seed), case["tokens"], case["dim"]
    st = {"kind": "norm", "x": _hidden(gen, T, case["row"])[:, :D], "weight": (1.0 + 0.2 * _rnd(gen, D)).to(BF16),
          "residual": None, "sum": None, "out": None, "codes": None, "scales": None}
    if case["residual"]:
        st["residual"] = (2.0 * _rnd(gen, T, D)).to(BF16)
        st["sum"] = torch.empty(T, D, dtype=BF16, device=DEV)
    if case["keep"]:
        st["out"] = torch.empty(T, D, dtype=BF16, device=DEV)
    if case["fp8"]:
        st["codes"] = torch.empty(T, D, dtype=FP8, device=DEV)
        st["scales"] = _scales(case["scale"], T, _ceil(D, BLOCK))
    return st


def _prepare_quant(case, seed):
    gen, T, D = _gen(seed), case["tokens"], case["dim"]
    return {"kind": "quant", "x": _hidden(gen, T, D), "codes": torch.empty(T, D, dtype=FP8, device=DEV),
            "scales": _scales(case["scale"], T, _ceil(D, BLOCK))}


def _prepare_gemm(case, seed):
    gen, T, N, K = _gen(seed), case["tokens"], case["n"], case["k"]
    a, sa = _to_fp8(_hidden(gen, T, K).float(), case["scale"])
    w = _rnd(gen, N, K) * (K ** -0.5) * torch.exp(0.3 * _rnd(gen, N, 1))
    # a weight's scale is one number per 128 x 128 block
    full = torch.nn.functional.pad(w, (0, -K % BLOCK, 0, -N % BLOCK)).view(_ceil(N, BLOCK), BLOCK, _ceil(K, BLOCK), BLOCK)
    sb, held = _scale_of(full.abs().amax(dim=(1, 3)), case["scale"])
    b = (full / sb[:, None, :, None]).view(full.shape[0] * BLOCK, -1)[:N, :K].to(FP8)
    return {"kind": "gemm", "a": a, "sa": sa, "b": b.contiguous(), "sb": held,
            "out": torch.empty(T, N, dtype=BF16, device=DEV)}


def _prepare_rope(case, seed):
    gen, T, H, R = _gen(seed), case["tokens"], case["heads"], case["rot"]
    # angles of far positions need 64 bits; slow dims are interpolated by 8 for long contexts, fast ones are not
    i = torch.arange(R // 2, dtype=torch.float64, device=DEV)
    freq = 10000.0 ** (-2.0 * i / R)
    slow = ((i - R / 8) / (R / 4)).clamp(0.0, 1.0)
    angle = torch.arange(case["table"], dtype=torch.float64, device=DEV)[:, None] * (freq * (1.0 - slow) + freq / 8.0 * slow)
    positions = torch.randint(0, case["table"], (T,), generator=gen, device=DEV)
    return {"kind": "rope", "table": torch.cat([angle.cos(), angle.sin()], dim=1).float(), "pairs": case["pairs"],
            "out_pairs": case["out_pairs"], "positions": positions if case["wide"] else positions.to(torch.int32),
            # the positional part lies behind the others of each head, and behind the latent key
            "q": _rnd(gen, T, H, case["head"]).to(BF16)[..., case["head"] - R:],
            "k": _rnd(gen, T, 512 + R).to(BF16)[:, None, 512:],
            "q_out": torch.empty(T, H, 512 + R, dtype=BF16, device=DEV)[..., 512:],
            "k_out": torch.empty(T, 1, 512 + R, dtype=BF16, device=DEV)[..., 512:]}


# ------------------------------------------------------------------ one pass
def run(state):
    return globals()["_run_" + state["kind"]](state)


def _scale_of(amax, kind):
    """Scales of blocks with these largest magnitudes, as float32 and as they are held."""
    s = amax.clamp(min=2.0 ** -40) / 448.0
    if kind == "f32":
        return s, s
    m, e = torch.frexp(s)  # s = m * 2^e, m in [0.5, 1): the smallest power of two that is not below it
    byte = e + 127 - (m == 0.5).to(e.dtype)
    held = byte.to(torch.uint8).view(E8M0)
    return _values(held), held


def _values(scales):
    """The float32 numbers that scales stand for (an exponent's bits: exp2 is not exact on every device)."""
    return scales if scales.dtype == torch.float32 else (scales.view(torch.uint8).to(torch.int32) << 23).view(torch.float32)


def _to_fp8(y, kind):
    """[T, D] float32 -> fp8 codes [T, D] and scales [T, ceil(D / 128)]."""
    T, D = y.shape
    blocks = torch.nn.functional.pad(y, (0, -D % BLOCK)).view(T, -1, BLOCK)
    s, held = _scale_of(blocks.abs().amax(dim=-1), kind)
    return (blocks / s[..., None]).view(T, -1)[:, :D].to(FP8).contiguous(), held


def _kind(scales):
    return "f32" if scales.dtype == torch.float32 else "e8m0"


def _run_norm(st):
    if own:
        from nanoengine_amd import ops
        if st["codes"] is None:
            ops.rms_norm(st["x"], st["weight"], EPS, out=st["out"], residual=st["residual"], residual_out=st["sum"])
        else:
            ops.rms_norm_quant(st["x"], st["weight"], EPS, st["codes"], st["scales"], out=st["out"],
                               residual=st["residual"], residual_out=st["sum"])
        return [st[k] for k in ("sum", "out", "codes", "scales")]
    h = st["x"].float()
    if st["residual"] is not None:
        st["sum"].copy_(h + st["residual"].float())
        h = st["sum"].float()
    y = h * torch.rsqrt((h * h).mean(dim=-1, keepdim=True) + EPS) * st["weight"].float()
    if st["out"] is not None:
        st["out"].copy_(y)
    if st["codes"] is None:
        return [st["sum"], st["out"], None, None]
    return [st["sum"], st["out"], *_to_fp8(y, _kind(st["scales"]))]


def _run_quant(st):
    if own:
        from nanoengine_amd import ops
        return ops.act_quant(st["x"], st["codes"], st["scales"])
    return _to_fp8(st["x"].float(), _kind(st["scales"]))


def _run_gemm(st):
    if own:
        from nanoengine_amd import ops
        return ops.fp8_gemm(st["a"], st["sa"], st["b"], st["sb"], out=st["out"])
    (T, K), N = st["a"].shape, st["b"].shape[0]
    a = st["a"].float() * _values(st["sa"]).repeat_interleave(BLOCK, dim=1)[:, :K]
    sb = _values(st["sb"]).repeat_interleave(BLOCK, dim=1)[:, :K]
    return (a @ (st["b"].float() * sb.repeat_interleave(BLOCK, dim=0)[:N]).T).to(BF16)


def _run_rope(st):
    if own:
        from nanoengine_amd import ops
        return ops.rope(st["q"], st["positions"], st["table"], out=st["q_out"], k=st["k"], k_out=st["k_out"],
                        interleaved=st["pairs"], out_interleaved=st["out_pairs"])
    cos, sin = st["table"][st["positions"].long()][:, None].chunk(2, dim=-1)
    for x, out in ((st["q"], st["q_out"]), (st["k"], st["k_out"])):
        x = x.float()
        a, b = (x[..., 0::2], x[..., 1::2]) if st["pairs"] else x.chunk(2, dim=-1)
        u, v = a * cos - b * sin, b * cos + a * sin
        out.copy_(torch.stack([u, v], dim=-1).flatten(-2) if st["out_pairs"] else torch.cat([u, v], dim=-1))
    return st["q_out"], st["k_out"]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind, T = case["kind"], case["tokens"]
    if kind in ("norm", "quant"):
        D = case["dim"]
        coded = D + _ceil(D, BLOCK) * (4 if case["scale"] == "f32" else 1)
        if kind == "quant":
            return {"bytes": T * (2 * D + coded), "flops": 3 * T * D}
        row = 2 * D * (1 + 2 * case["residual"] + case["keep"]) + coded * case["fp8"]
        return {"bytes": T * row + 2 * D, "flops": T * D * (4 + case["residual"] + 3 * case["fp8"])}
    if kind == "gemm":
        N, K, word = case["n"], case["k"], 4 if case["scale"] == "f32" else 1
        return {"bytes": (T + N) * K + (T + _ceil(N, BLOCK)) * _ceil(K, BLOCK) * word + 2 * T * N, "flops": 2 * T * N * K}
    R = case["rot"]
    return {"bytes": T * (case["heads"] + 1) * R * 4 + T * (8 if case["wide"] else 4) + min(T, case["table"]) * R * 4,
            "flops": 3 * T * (case["heads"] + 1) * R}


# ------------------------------------------------------------------ 64 bits
def _coded64(y, scale):
    """y / scale and scale of each block of 128, with no rounding to fp8."""
    T, D = y.shape
    n = _ceil(D, BLOCK)
    top = torch.zeros(T, n, dtype=torch.float64, device=y.device)
    top.scatter_reduce_(1, (torch.arange(D, device=y.device) // BLOCK).expand(T, D), y.abs(), "amax")
    s = top.clamp(min=2.0 ** -40) / 448.0
    if scale == "e8m0":  # the power of two below it, doubled unless it is that one
        whole = (s.view(torch.int64) >> 52 << 52).view(torch.float64)
        s = torch.where(whole == s, s, 2.0 * whole)
    return y / s[:, torch.arange(D, device=y.device) // BLOCK], s


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "quant":
        return _coded64(st["x"].double(), case["scale"])
    if kind == "norm":
        h, total = st["x"].double(), None
        if case["residual"]:
            total = h + st["residual"].double()
            h = total.to(BF16).double()  # the norm is that of the residual stream as it is kept
        y = h / torch.sqrt(h.square().sum(dim=1) / case["dim"] + EPS)[:, None] * st["weight"].double()
        codes, scales = _coded64(y, case["scale"]) if case["fp8"] else (None, None)
        return [total, y if case["keep"] else None, codes, scales]
    if kind == "gemm":
        out = torch.zeros(case["tokens"], case["n"], dtype=torch.float64, device=DEV)
        rows = torch.arange(case["n"], device=DEV) // BLOCK
        sa, sb = (s.double() if s.dtype == torch.float32 else
                  ((s.view(torch.uint8).long() + (1023 - 127)) << 52).view(torch.float64) for s in (st["sa"], st["sb"]))
        for at in range(_ceil(case["k"], BLOCK)):  # block by block: products of codes, then both scales
            cut = slice(at * BLOCK, (at + 1) * BLOCK)
            out += (st["a"][:, cut].double() @ st["b"][:, cut].double().T) * sa[:, at, None] * sb[rows, at]
        return out
    turn = torch.complex(*(t.double() for t in st["table"][st["positions"].long()].chunk(2, dim=1)))[:, None]
    outs = []
    for x in (st["q"].double(), st["k"].double()):
        half = case["rot"] // 2
        z = torch.view_as_complex(x.unflatten(-1, (half, 2)).contiguous()) if case["pairs"] else torch.complex(
            x[..., :half].contiguous(), x[..., half:].contiguous())
        z = torch.view_as_real(z * turn)
        outs.append(z.flatten(-2) if case["out_pairs"] else z.transpose(-1, -2).flatten(-2))
    return outs
