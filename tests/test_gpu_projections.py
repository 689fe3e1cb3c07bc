"""The operators around the attention in a run, as a layer uses them: hidden states -> caches and the step's inputs ->
the DSA step -> the layer's output. Every call of a run is held to its 64-bit restatement with its own bounds, the run as a
whole to the layer without any rounding, and a captured run to an eager one."""
import pytest
import torch

from nanoengine_amd import deep_gemm, ops, projections, rotary, synth
from nanoengine_amd.pipeline import DsaDecodeStep
from oracle import around_oracle as A

pytestmark = pytest.mark.gpu
BF, F32, E8M0 = torch.bfloat16, torch.float32, torch.float8_e8m0fnu
D, RANK, H, NOPE, V, CTX = 1024, 384, 32, 128, 128, 4096
LENS = [37, 200, 65]          # tokens in the caches before the step
SCALE = 192 ** -0.5


def make_layer(cuda, scale_dtype, interleaved=True):
    g = torch.Generator(device=cuda).manual_seed(3)

    def w(*shape):
        return torch.randn(*shape, generator=g, device=cuda) * shape[-1] ** -0.5

    weights = dict(norm=1 + 0.1 * torch.randn(D, generator=g, device=cuda), a=w(RANK + 512 + 64 + 128, D),
                   q_norm=(1 + 0.1 * torch.randn(RANK, generator=g, device=cuda)).to(BF),
                   kv_norm=1 + 0.1 * torch.randn(512, generator=g, device=cuda), q=w(H * (NOPE + 64), RANK),
                   k_up=w(H, NOPE, 512).to(BF), v_up=(torch.randn(H, 512, V, generator=g, device=cuda) * 512 ** -0.5).to(BF),
                   o=w(D, H * V), idx_q=w(64 * 128, RANK), idx_gate=w(64, D), idx_norm=torch.ones(128, device=cuda),
                   idx_bias=torch.zeros(128, device=cuda))
    table = rotary.cos_sin_cache(CTX, 64, factor=4.0, original_max_position=1024, attention_factor=1.0, device=cuda)
    return projections.MlaProjections(**weights, cos_sin_cache=table, scale_dtype=scale_dtype, interleaved=interleaved), weights


class Batch:
    """Tokens of three sequences: the caches' (all in one call) and one more each."""

    def __init__(self, cuda):
        self.tables, pages = synth.make_block_tables([n + 1 for n in LENS], torch.Generator().manual_seed(1), cuda)
        self.kv = torch.zeros(pages, 65, 1, 656, dtype=torch.uint8, device=cuda)[:, :64]
        self.idx = torch.zeros(pages, synth.IDX_PAGE_BYTES, dtype=torch.uint8, device=cuda)
        g = torch.Generator(device=cuda).manual_seed(2)
        self.before = torch.cat([torch.arange(n) for n in LENS]).to(cuda)
        self.seq = torch.cat([torch.full((n,), b) for b, n in enumerate(LENS)]).to(cuda)
        self.now = torch.tensor(LENS, device=cuda)
        self.x0 = torch.randn(sum(LENS), D, generator=g, device=cuda).to(BF)
        self.x1, self.r1 = (torch.randn(3, D, generator=g, device=cuda).to(BF) for _ in range(2))

    def slots(self, seq, pos):
        return self.tables.long()[seq, pos // 64] * 64 + pos % 64


def run(layer, step, b, residual):
    """The step of one layer for a token of each sequence."""
    own = torch.arange(3, device=b.now.device)
    q_idx, w, q, residual = layer.inputs(b.x1, residual, b.now, b.slots(own, b.now), b.kv, b.idx)
    o = step(q_idx.view(torch.uint8), w, b.idx, (b.now + 1).int(), b.tables, b.tables, q, b.kv, SCALE)[0]
    return layer.output(o), q, residual


def plain(weights, table, b, pairs):
    """The same without any rounding: float64, every token of a context attended to."""
    W = {k: v.double() for k, v in weights.items()}

    def norm(x, w):
        return x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w

    def turn(x, pos):
        c, s = (t[:, None] for t in table.double()[pos].chunk(2, dim=-1))
        p, q = (x[..., 0::2], x[..., 1::2]) if pairs else x.chunk(2, dim=-1)
        return torch.cat([p * c - q * s, q * c + p * s], dim=-1)  # (the same order for queries and keys)

    x = torch.cat([b.x0, b.x1]).double()
    x[sum(LENS):] += b.r1.double()
    pos, seq = torch.cat([b.before, b.now]), torch.cat([b.seq, torch.arange(3, device=b.seq.device)])
    c = norm(x, W["norm"]) @ W["a"].t()
    kv = norm(c[:, RANK:RANK + 512], W["kv_norm"])
    k_rot = turn(c[:, None, RANK + 512:RANK + 576], pos)[:, 0]
    q = (norm(c[:, :RANK], W["q_norm"]) @ W["q"].t()).view(-1, H, NOPE + 64)[-3:]
    q_rot = turn(q[..., NOPE:], pos[-3:])
    outs = []
    for i in range(3):
        mine = seq == i
        k = (kv[mine] @ W["k_up"].reshape(H * NOPE, 512).t()).view(-1, H, NOPE)  # not absorbed
        score = torch.stack([k[:, h] @ q[i, h, :NOPE] + k_rot[mine] @ q_rot[i, h] for h in range(H)]) * SCALE
        o = score.softmax(-1) @ kv[mine]
        outs.append(torch.cat([o[h] @ W["v_up"][h] for h in range(H)]) @ W["o"].t())
    return torch.stack(outs)


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("kind", [F32, E8M0])
def test_layer(cuda, monkeypatch, kind, interleaved):
    layer, weights = make_layer(cuda, kind, interleaved)
    b = Batch(cuda)
    step = DsaDecodeStep(3, 1, 64 * b.tables.shape[1], num_heads=H, device=cuda)
    first = layer.inputs(b.x0, None, b.before, b.slots(b.seq, b.before), b.kv, b.idx)
    assert first[3] is b.x0

    seen = []
    for name in ("rms_norm", "rms_norm_quant", "act_quant", "fp8_gemm", "rope"):
        def record(*args, _fn=getattr(ops, name), _name=name, **kw):
            kept = [t.clone() if isinstance(t, torch.Tensor) else t for t in args]
            kept_kw = {k: t.clone() if isinstance(t, torch.Tensor) else t for k, t in kw.items()}
            seen.append((_name, kept, kept_kw, kw, _fn(*args, **kw)))
            return seen[-1][-1]
        monkeypatch.setattr(ops, name, record)
    residual = b.r1.clone()
    out, q, stream = run(layer, step, b, residual)
    monkeypatch.undo()
    assert stream is residual and torch.equal(residual, (b.x1.float() + b.r1.float()).to(BF))

    assert [s[0] for s in seen] == ["rms_norm_quant", "fp8_gemm", "rms_norm_quant", "rms_norm", "fp8_gemm", "rope", "fp8_gemm",
                                    "act_quant", "fp8_gemm"]
    for name, args, kw, live, got in seen:
        if name.startswith("rms"):
            h, y = A.rms_norm(args[0], args[1], args[2], kw.get("residual"))
            rel = A.norm_rel(args[0].shape[1])
            if name == "rms_norm_quant":
                A.check_coded(*got, y, rel)
            if "out" in kw:
                assert A.within_bf16(live["out"], y, rel * y.abs())
        elif name == "act_quant":
            A.check_coded(*got, args[0].double(), 0.0)
        elif name == "fp8_gemm":
            want, err = A.gemm(*args[:4])
            assert A.within_bf16(got, want, err)
        else:
            for x, y in zip((args[0], kw["k"]), got):
                assert A.within_bf16(y, *A.rope(x, args[2], args[1], interleaved, interleaved))

    # The whole: with independent weights a rounding of relative size e on either side of a product leaves its result
    # off by e in the mean square, sqrt(2) 2^-4 for both at most. Four follow one another (a, then q or the keys in the
    # cache, the values in the cache, o), each on top of the ones before. A wrong wire is off by the size of the result.
    want = plain(weights, layer.cos_sin_cache, b, interleaved)
    off = (out.double() - want).norm() / want.norm()
    print(f"layer {kind} off by {off.item():.3f}", flush=True)
    assert off <= 4 * 2 ** 0.5 * 2.0 ** -4


def test_layer_captured(cuda):
    layer, _ = make_layer(cuda, E8M0)
    b = Batch(cuda)
    step = DsaDecodeStep(3, 1, 64 * b.tables.shape[1], num_heads=H, device=cuda)
    layer.inputs(b.x0, None, b.before, b.slots(b.seq, b.before), b.kv, b.idx)
    s, residual = torch.cuda.Stream(), b.r1.clone()
    eager = [t.clone() for t in run(layer, step, b, residual)]
    kv, idx = b.kv.clone(), b.idx.clone()
    torch.cuda.synchronize()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run(layer, step, b, residual)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs = run(layer, step, b, residual)
    torch.cuda.synchronize()
    x1 = b.x1.clone()
    for turn in range(4):
        for t in outs[:2]:
            t.zero_()
        # eager work of the same operators between the replays, and in odd turns other inputs
        b.x1.copy_(x1 if turn % 2 == 0 else x1.flip(0))
        residual.copy_(b.r1)
        other = [t.clone() for t in run(layer, step, b, b.r1.clone())]
        b.kv.copy_(kv)
        b.idx.copy_(idx)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, other if turn % 2 else eager):
            assert torch.equal(got, want), turn
    assert not torch.equal(other[0], eager[0])


@pytest.mark.parametrize("rows", [20, 40])
def test_two_streams_at_once(cuda, rows):
    """Products on two streams at once; of 40 rows in parts of K, each with a workspace from its own stream's pool."""
    g = torch.Generator(device=cuda).manual_seed(5)
    a, sa = ops.act_quant(torch.randn(rows, 8192, generator=g, device=cuda).to(BF))
    ws = [projections.Fp8Linear(torch.randn(300, 8192, generator=g, device=cuda)) for _ in range(2)]
    assert (ops.fp8_gemm_workspace_bytes(rows, 300, 8192) > 0) == (rows > 32)
    want = [w(a, sa) for w in ws]
    for w, o in zip(ws, want):
        assert A.within_bf16(o, *A.gemm(a, sa, w.codes, w.scales))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ws[i](a, sa))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_split_product_captured(cuda):
    """A product in parts of K, whose workspace comes from the graph's pool: replays between eager calls of the same, with
    inputs that change under the graph."""
    g = torch.Generator(device=cuda).manual_seed(8)
    xs = [torch.randn(100, 8192, generator=g, device=cuda).to(BF) for _ in range(2)]
    w = projections.Fp8Linear(torch.randn(300, 8192, generator=g, device=cuda))
    assert ops.fp8_gemm_workspace_bytes(100, 300, 8192) > 0
    want = [w(*ops.act_quant(x)) for x in xs]
    x, out = xs[0].clone(), torch.empty(100, 300, dtype=BF, device=cuda)
    codes, scales = ops.act_quant(x)
    torch.cuda.synchronize()
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        w(*ops.act_quant(x, codes, scales), out=out)
        with torch.cuda.graph(graph, stream=s):
            w(*ops.act_quant(x, codes, scales), out=out)
    torch.cuda.synchronize()
    for turn in range(4):
        x.copy_(xs[turn % 2])
        out.zero_()
        other = w(*ops.act_quant(xs[1 - turn % 2]))
        graph.replay()
        assert torch.equal(w(*ops.act_quant(xs[1 - turn % 2])), want[1 - turn % 2])
        torch.cuda.synchronize()
        assert torch.equal(out, want[turn % 2]) and torch.equal(other, want[1 - turn % 2])


def test_no_tokens(cuda):
    layer, _ = make_layer(cuda, E8M0)
    b = Batch(cuda)
    none = torch.empty(0, dtype=torch.int64, device=cuda)
    before = b.kv.clone()
    q_idx, w, q, _ = layer.inputs(b.x0[:0], None, none, none, b.kv, b.idx)
    assert q_idx.shape == (0, 64, 128) and w.shape == (0, 64) and q.shape == (0, H, 576)
    assert layer.output(torch.empty(0, H, 512, dtype=BF, device=cuda)).shape == (0, D) and torch.equal(b.kv, before)


def test_padded_tokens_write_nothing(cuda):
    """Rows of a padded batch (slot -1, any position, NaN in the hidden states) leave the caches and the other rows alone."""
    layer, _ = make_layer(cuda, E8M0)
    b, c = Batch(cuda), Batch(cuda)
    pos, slots = b.before[:5], b.slots(b.seq, b.before)[:5]
    want = layer.inputs(b.x0[:5], None, pos, slots, b.kv, b.idx)
    x = torch.cat([b.x0[:5], torch.full((3, D), float("nan"), dtype=BF, device=cuda)])
    pad = torch.tensor([-1, 7 * CTX, 0], device=cuda)
    got = layer.inputs(x, None, torch.cat([pos, pad]), torch.cat([slots, torch.full_like(pad, -1)]), c.kv, c.idx)
    for w, g in zip(want[:3], got[:3]):
        assert torch.equal(w.view(torch.uint8), g[:5].view(torch.uint8))
    assert torch.equal(b.kv, c.kv) and torch.equal(b.idx, c.idx)


def test_fp8_gemm_nt(cuda):
    g = torch.Generator(device=cuda).manual_seed(6)
    for kind, dtype in ((F32, BF), (E8M0, F32)):
        a, sa = ops.act_quant(torch.randn(33, 400, generator=g, device=cuda).to(BF), scale_dtype=kind)
        w = projections.Fp8Linear(torch.randn(200, 400, generator=g, device=cuda), kind)
        d = torch.empty(33, 200, dtype=dtype, device=cuda)
        assert deep_gemm.fp8_gemm_nt((a, sa.t().contiguous().t()), (w.codes, w.scales), d) is None
        assert torch.equal(d, ops.fp8_gemm(a, sa, w.codes, w.scales, out_dtype=dtype))


@pytest.mark.parametrize("kind", ["f32", "e8m0"])
def test_weight_rule_is_that_of_activations(cuda, kind):
    w = torch.randn(300, 401, generator=torch.Generator(device=cuda).manual_seed(7), device=cuda)
    w[0, :128], w[128:256, 128:256] = 0, 0
    w[256:, 256:384] = 448.0
    codes, scales = projections.quantize_weight(w, F32 if kind == "f32" else E8M0)
    want = A.quantise_weight(w, kind)
    got_s, want_s = A.scale_values(scales), A.scale_values(want[1])
    # one division and its rounding against the exact quotient's
    assert torch.all((got_s - want_s).abs() <= (2 * A.EPS32 if kind == "f32" else 0) * want_s)
    full = got_s.repeat_interleave(128, 0)[:300].repeat_interleave(128, 1)[:, :401]
    tol = torch.maximum(A.HALF_FP8 * w.double().abs() * (1 + 3 * A.EPS32), 2.0 ** -10 * full) + 3 * A.EPS32 * w.double().abs()
    assert torch.all((codes.double() * full - w.double()).abs() <= tol)
