"""The layout of the indexer's rotated dims is one thing for its queries and its keys: pairs beside each other or in halves, apart from
the layout of the MLA's heads. Contexts past 2048 tokens, so that the step has to choose."""
import math

import numpy as np
import pytest
import torch

import oracle as O
from nanoengine_amd import indexer_transform, ops, projections, rotary, synth
from nanoengine_amd.pipeline import DsaDecodeStep

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
D, RANK, H, NOPE, V, CTX = 512, 256, 16, 64, 64, 8192
LENS = [4096, 3001]   # tokens in the caches before the step
SCALE = 128 ** -0.5


def u16(t):
    return t.contiguous().cpu().view(torch.int16).numpy().view(np.uint16)


@pytest.mark.parametrize("T", [1, 17, 200])
@pytest.mark.parametrize("interleaved", [True, False])
def test_key_layouts_bit_exact(cuda, T, interleaved):
    rng = np.random.default_rng(T)
    key = torch.from_numpy((2 * rng.standard_normal((T, 128)) + 0.3).astype(np.float32)).to(BF)
    w, b = rng.standard_normal(128).astype(np.float32), 0.1 * rng.standard_normal(128).astype(np.float32)
    cs, pos, slots = O.rope_cos_sin_cache(4096), rng.integers(0, 4096, T), rng.permutation(256)[:T].astype(np.int64)
    args = [torch.from_numpy(t).to(cuda) for t in (w, b, pos, cs, slots)]
    codes, sf = O.indexer_k_transform(u16(key), w, b, 1e-6, cs, pos, interleaved)
    want = O.pack_indexer_cache(codes, sf, slots, 4)
    for call in (ops.indexer_k_transform_store, indexer_transform.indexer_k_transform_store_fp8):
        cache = torch.zeros(4, 64 * 132, dtype=torch.uint8, device=cuda)
        call(key.to(cuda), args[0], args[1], 1e-6, args[2], args[3], cache, args[4], 64, rope_interleaved=interleaved)
        assert np.array_equal(cache.cpu().numpy(), want)


def make_weights(cuda):
    g = torch.Generator(device=cuda).manual_seed(3)

    def w(*shape):
        return torch.randn(*shape, generator=g, device=cuda) * shape[-1] ** -0.5

    # keys of the indexer live in the rotated dims alone: no score without the right angles
    only = (torch.arange(128, device=cuda) < 64).float()
    return dict(norm=1 + 0.1 * torch.randn(D, generator=g, device=cuda), a=w(RANK + 512 + 64 + 128, D),
                q_norm=(1 + 0.1 * torch.randn(RANK, generator=g, device=cuda)).to(BF), kv_norm=torch.ones(512, device=cuda),
                q=w(H * (NOPE + 64), RANK), k_up=w(H, NOPE, 512).to(BF),
                v_up=(torch.randn(H, 512, V, generator=g, device=cuda) * 512 ** -0.5).to(BF), o=w(D, H * V),
                idx_q=w(64 * 128, RANK), idx_gate=w(64, D), idx_norm=only, idx_bias=torch.zeros(128, device=cuda))


def plain(W, table, x, seq, pos, mla_pairs, idx_pairs, chosen):
    """In float64, for the last token of each sequence: (the indexer's scores of its whole context, the layer's output over the
    positions `chosen`)."""
    W = {k: v.double() for k, v in W.items()}

    def norm(x, w):
        return x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w

    def turn(x, at, pairs):
        c, s = (t[:, None] for t in table.double()[at].chunk(2, dim=-1))
        p, q = (x[..., 0::2], x[..., 1::2]) if pairs else x.chunk(2, dim=-1)
        return torch.cat([p * c - q * s, q * c + p * s], dim=-1)

    h = norm(x.double(), W["norm"])
    c = h @ W["a"].t()
    kv, k_rot = norm(c[:, RANK:RANK + 512], W["kv_norm"]), turn(c[:, None, RANK + 512:RANK + 576], pos, mla_pairs)[:, 0]
    idx = c[:, RANK + 576:]
    idx = (idx - idx.mean(1, keepdim=True)) / torch.sqrt(idx.var(1, keepdim=True, unbiased=False) + 1e-6) * W["idx_norm"]
    idx = torch.cat([turn(idx[:, None, :64], pos, idx_pairs)[:, 0], idx[:, 64:]], dim=1)
    n = len(LENS)
    c_q, at = norm(c[-n:, :RANK], W["q_norm"]), pos[-n:]
    q = (c_q @ W["q"].t()).view(n, H, NOPE + 64)
    q_rot = turn(q[..., NOPE:], at, mla_pairs)
    i_q = (c_q @ W["idx_q"].t()).view(n, 64, 128)
    i_q = torch.cat([turn(i_q[..., :64], at, idx_pairs), i_q[..., 64:]], dim=-1)
    gate = h[-n:] @ W["idx_gate"].t()
    scores, outs = [], []
    for b in range(n):
        mine = torch.nonzero(seq == b)[:, 0]
        mine = mine[torch.argsort(pos[mine])]
        scores.append(gate[b] @ (i_q[b] @ idx[mine].t()).clamp_min(0))
        keep = mine[chosen[b]]
        k = (kv[keep] @ W["k_up"].reshape(H * NOPE, 512).t()).view(-1, H, NOPE)
        s = torch.stack([k[:, i] @ q[b, i, :NOPE] + k_rot[keep] @ q_rot[b, i] for i in range(H)]) * SCALE
        o = s.softmax(-1) @ kv[keep]
        outs.append(torch.cat([o[i] @ W["v_up"][i] for i in range(H)]) @ W["o"].t())
    return scores, torch.stack(outs)


@pytest.mark.parametrize("mla_pairs,idx_pairs", [(True, True), (False, False), (True, False), (False, True)])
def test_layer_chooses_by_the_right_angles(cuda, monkeypatch, mla_pairs, idx_pairs):
    W = make_weights(cuda)
    table = rotary.cos_sin_cache(CTX, 64, device=cuda)
    kw = {} if idx_pairs == mla_pairs else {"indexer_interleaved": idx_pairs}  # one flag says both unless the other is given
    layer = projections.MlaProjections(**W, cos_sin_cache=table, interleaved=mla_pairs, **kw)
    n = len(LENS)
    tables, pages = synth.make_block_tables([x + 1 for x in LENS], torch.Generator().manual_seed(1), cuda)
    kv = torch.zeros(pages, 64, 1, 656, dtype=torch.uint8, device=cuda)
    cache = torch.zeros(pages, synth.IDX_PAGE_BYTES, dtype=torch.uint8, device=cuda)
    pos = torch.cat([torch.arange(x) for x in LENS] + [torch.tensor(LENS)]).to(cuda)
    seq = torch.cat([torch.full((x,), b) for b, x in enumerate(LENS)] + [torch.arange(n)]).to(cuda)
    slots = tables.long()[seq, pos // 64] * 64 + pos % 64
    x = torch.randn(len(pos), D, generator=torch.Generator(device=cuda).manual_seed(2), device=cuda).to(BF)

    keys, queries = [], []

    def record_key(key, *args, _fn=ops.indexer_k_transform_store, **kw):
        keys.append(key.clone())
        return _fn(key, *args, **kw)

    def record_query(query, gate, *args, _fn=ops.indexer_q_prologue, **kw):
        queries.append((query.clone(), gate.clone()))
        return _fn(query, gate, *args, **kw)

    monkeypatch.setattr(ops, "indexer_k_transform_store", record_key)
    monkeypatch.setattr(ops, "indexer_q_prologue", record_query)
    old = slice(0, len(pos) - n)
    layer.inputs(x[old], None, pos[old], slots[old], kv, cache)
    q_idx, weights, q_mla, _ = layer.inputs(x[-n:], None, pos[-n:], slots[-n:], kv, cache)
    monkeypatch.undo()
    step = DsaDecodeStep(n, 1, 64 * tables.shape[1], num_heads=H, device=cuda)
    o, _, logical, _ = step(q_idx.view(torch.uint8), weights, cache, (pos[-n:] + 1).int(), tables, tables, q_mla, kv, SCALE)
    out = layer.output(o)

    # the indexer's inputs, bit for bit from what the projections gave
    cs = table.cpu().numpy()
    want_q, want_w = O.indexer_q_prologue(u16(queries[1][0]), u16(queries[1][1]), 64 ** -0.5 * 128 ** -0.5, cs,
                                          pos[-n:].cpu().numpy(), idx_pairs)
    assert np.array_equal(q_idx.view(torch.uint8).cpu().numpy(), want_q)
    assert np.array_equal(weights.cpu().numpy().view(np.uint32), want_w.view(np.uint32))
    only = W["idx_norm"].cpu().numpy()
    codes, sf = O.indexer_k_transform(u16(torch.cat(keys)), only, 0 * only, 1e-6, cs, pos.cpu().numpy(), idx_pairs)
    assert np.array_equal(cache.cpu().numpy(), O.pack_indexer_cache(codes, sf, slots.cpu().numpy(), pages))

    # What is chosen, against the scores without any rounding. Eight fp8 roundings lie between the hidden states and a product of
    # query and key (hidden and a, twice; the latent query, idx_q, the query's and the key's codes), each of 2^-4 at most: off by
    # e = sqrt(8) 2^-4 of the product's spread in the mean square. Of half of the products ReLU keeps the error whole and
    # of their spread sqrt(1 / 2 - 1 / (2 pi)): e sqrt(0.5 / 0.341). Two normal scores that differ so part the contexts
    # at their median (elsewhere less) differently in atan(e) / pi of the tokens: 0.067. By angles of other pairs it is one half.
    e = 8 ** 0.5 * 2.0 ** -4 * (0.5 / (0.5 - 0.5 / math.pi)) ** 0.5
    chosen = [torch.sort(row.long())[0] for row in logical]
    scores, want = plain(W, table, x, seq, pos, mla_pairs, idx_pairs, chosen)
    for got, s in zip(chosen, scores):
        assert got[0] >= 0 and got.unique().numel() == 2048
        best = torch.zeros_like(s, dtype=torch.bool)
        best[s.topk(2048)[1]] = True
        share = 1 - best[got].float().mean().item()
        print(f"layout {mla_pairs} {idx_pairs}: {share:.3f} of {s.numel()} chosen differently", flush=True)
        assert share <= math.atan(e) / math.pi
    # and the layer over those keys: four roundings of 2^-4 on either side of its products, one after another
    off = (out.double() - want).norm() / want.norm()
    print(f"layer off by {off.item():.3f}", flush=True)
    assert off <= 4 * 2 ** 0.5 * 2.0 ** -4
