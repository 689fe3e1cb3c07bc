"""The steps around the attention on the GPU, each against its 64-bit restatement: norms with a residual and an fp8
output, the fp8 rounding alone, block-scaled fp8 products, rotary positions."""
import pytest
import torch

from nanoengine_amd import ops
from oracle import around_oracle as A

pytestmark = pytest.mark.gpu
BF, FP8, E8M0, F32 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.float32
KINDS = {"f32": F32, "e8m0": E8M0}


def gen(device, seed=0):
    return torch.Generator(device=device).manual_seed(seed)


def rnd(g, *shape):
    return torch.randn(*shape, generator=g, device=g.device)


def activations(g, rows, dim, width=None):
    """Channels of very different size, in rows that may be wider."""
    x = rnd(g, rows, width or dim) * torch.exp(1.5 * rnd(g, width or dim))
    return x.to(BF)[:, :dim]


# ------------------------------------------------------------------ norm
@pytest.mark.parametrize("rows,dim,width", [(1, 1, 1), (1, 8, 8), (3, 127, 127), (5, 128, 136), (9, 512, 576), (6, 513, 600),
                                            (2, 1536, 2112), (3, 2048, 2048), (2, 2056, 2056), (3, 4095, 4096),
                                            (2, 8192, 8192), (2, 8200, 8200), (1, 16384, 16384), (2, 16392, 16400),
                                            (1, 32768, 32768), (1, 32765, 32765), (1000, 1600, 1600)])
@pytest.mark.parametrize("kind", ["f32", "e8m0"])
def test_norm_sizes(cuda, rows, dim, width, kind):
    print(f"norm {rows} {dim} {width} {kind}", flush=True)
    g = gen(cuda, dim)
    x, res = activations(g, rows, dim, width), activations(g, rows, dim)
    for weight in ((1 + 0.3 * rnd(g, dim)).to(BF), 1 + 0.3 * rnd(g, dim)):
        want_sum, y = A.rms_norm(x, weight, 1e-6, res)
        total, out = torch.empty(rows, dim, dtype=BF, device=cuda), torch.empty(rows, dim, dtype=BF, device=cuda)
        codes, scales = ops.rms_norm_quant(x, weight, 1e-6, out=out, residual=res, residual_out=total,
                                           scale_dtype=KINDS[kind])
        assert torch.equal(total, want_sum)
        assert A.within_bf16(out, y, A.norm_rel(dim) * y.abs())
        A.check_coded(codes, scales, y, A.norm_rel(dim))
        # each output by itself is the same
        assert torch.equal(ops.rms_norm(x, weight, 1e-6, residual=res), out)
        c2, s2 = ops.rms_norm_quant(x, weight, 1e-6, residual=res, scale_dtype=KINDS[kind])
        assert torch.equal(c2.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(s2.view(torch.uint8), scales.view(torch.uint8))
        _, y = A.rms_norm(x, weight, 1e-6)
        assert A.within_bf16(ops.rms_norm(x, weight, 1e-6), y, A.norm_rel(dim) * y.abs())


def test_norm_in_place_and_empty(cuda):
    g = gen(cuda, 1)
    for dim in (512, 515):
        x, res, w = activations(g, 7, dim), activations(g, 7, dim), torch.ones(dim, dtype=BF, device=cuda)
        want_sum, _ = A.rms_norm(x, w, 1e-5, res)
        want = ops.rms_norm(x, w, 1e-5, residual=res)
        kept = res.clone()
        assert torch.equal(ops.rms_norm(x, w, 1e-5, residual=kept, residual_out=kept), want) and torch.equal(kept, want_sum)
        y, s = x.clone(), res.clone()
        ops.rms_norm(y, w, 1e-5, out=y, residual=s, residual_out=s)
        assert torch.equal(y, want) and torch.equal(s, want_sum)
        z = x.clone()
        out = ops.rms_norm(z, w, 1e-5, residual=res, residual_out=z)  # the sum in x's place
        assert torch.equal(out, want) and torch.equal(z, want_sum)
    assert ops.rms_norm(x[:0], w, 1e-5).shape == (0, dim)
    assert ops.act_quant(x[:0])[0].shape == (0, dim)


def test_norm_special_values(cuda):
    x = torch.ones(6, 256, dtype=BF, device=cuda)
    x[0] = 0
    x[1, 130] = float("nan")
    x[2, 3] = float("inf")
    x[3] = 1e-30
    x[4, :128] = 2.0 ** -126
    w = torch.ones(256, dtype=BF, device=cuda)
    out = ops.rms_norm(x, w, 0.0)
    assert out[0].isnan().all()             # 0 / 0 without an eps, as the formula has it
    out = ops.rms_norm(x, w, 1e-6)
    assert torch.all(out[0] == 0) and out[1].isnan().all()
    assert out[2, 3].isnan() and torch.all(out[2, torch.arange(256, device=cuda) != 3] == 0)  # inf / inf, 1 / inf
    _, y = A.rms_norm(x[3:], w, 1e-6)
    assert A.within_bf16(out[3:], y, 2 ** -18 * y.abs())
    for kind in KINDS.values():
        codes, scales = ops.rms_norm_quant(x, w, 1e-6, scale_dtype=kind)
        assert torch.all(codes[0].float() == 0) and codes[1].float().isnan().all()
        s = A.scale_values(scales[0])
        assert torch.all(torch.isfinite(s) & (s > 0))


# ------------------------------------------------------------------ rounding alone
@pytest.mark.parametrize("rows,dim,width", [(1, 1, 1), (2, 7, 9), (1, 128, 128), (3, 129, 129), (5, 1600, 1600), (333, 264, 272),
                                            (2, 16384, 16384), (17, 40000, 40000), (4097, 128, 128)])
@pytest.mark.parametrize("kind", ["f32", "e8m0"])
def test_quant_sizes(cuda, rows, dim, width, kind):
    print(f"quant {rows} {dim} {kind}", flush=True)
    x = activations(gen(cuda, dim), rows, dim, width)
    codes, scales = ops.act_quant(x, scale_dtype=KINDS[kind])
    A.check_coded(codes, scales, x.double(), 0.0)
    if kind == "e8m0":  # no rounding on the way: the same scales, and the nearest codes
        want = A.exact_scales(A.blocks(x.double().abs()).amax(dim=-1), "e8m0")
        assert torch.equal(A.scale_values(scales), want)
        near = (x.double() / want.repeat_interleave(128, dim=1)[:, :dim]).float().to(FP8)
        assert torch.equal(codes.view(torch.uint8), near.view(torch.uint8))


def test_quant_strided_outputs(cuda):
    g = gen(cuda, 3)
    x = activations(g, 9, 384)
    want, ws = ops.act_quant(x)
    codes = torch.full((9, 400), 0x55, dtype=torch.uint8, device=cuda)
    scales = torch.full((9, 5), 0x55, dtype=torch.uint8, device=cuda)
    ops.act_quant(x, codes[:, :384], scales[:, :3])
    assert torch.equal(codes[:, :384], want.view(torch.uint8)) and torch.all(codes[:, 384:] == 0x55)
    assert torch.equal(scales[:, :3], ws.view(torch.uint8)) and torch.all(scales[:, 3:] == 0x55)
    ops.act_quant(x, codes[:, 3:387], scales[:, 1:4])  # codes at odd addresses
    assert torch.equal(codes[:, 3:387], want.view(torch.uint8)) and torch.equal(scales[:, 1:4], ws.view(torch.uint8))


@pytest.mark.parametrize("top", [0.0, 2.0 ** -41, 2.0 ** -40, 448.0, 449.0, 3.3895e38, float("inf")])
def test_quant_extremes(cuda, top):
    x = torch.zeros(1, 128, dtype=BF, device=cuda)
    x[0, 7], x[0, 8] = top, -1e-38
    x[0, 9] = float("nan")
    for kind, dtype in KINDS.items():
        codes, scales = ops.act_quant(x, scale_dtype=dtype)
        c = codes.float()
        assert c[0, 9].isnan() and torch.all(c[0, 10:] == 0) and c[0, 8] == 0
        if top == float("inf"):
            assert c[0, 7].isnan()
            assert scales.float().isinf() if kind == "f32" else scales.view(torch.uint8) == 254
        else:
            y = x.double()
            y[0, 9] = 0
            codes.view(torch.uint8)[0, 9] = 0
            A.check_coded(codes, scales, y, 0.0)


# ------------------------------------------------------------------ products
def product(g, M, N, K, kind, out_dtype=BF):
    a, sa = A.quantise_rows(rnd(g, M, K) * torch.exp(rnd(g, 1, K)), kind)
    b, sb = A.quantise_weight(rnd(g, N, K) * torch.exp(0.5 * rnd(g, N, 1)), kind)
    return a, sa, b, sb


def check_product(out, a, sa, b, sb):
    want, err = A.gemm(a, sa, b, sb)
    if out.dtype == BF:
        assert A.within_bf16(out, want, err), ((out.double() - want).abs() / (err + A.HALF_BF16 * want.abs())).max()
    else:
        assert torch.all((out.double() - want).abs() <= err)


@pytest.mark.parametrize("M,N,K", [(1, 1, 16), (1, 64, 128), (2, 130, 144), (7, 257, 1536), (16, 512, 2048), (17, 576, 4096), (31, 200, 272),
                                   (33, 2112, 1536), (64, 128, 4096), (65, 300, 1040), (100, 1000, 2048),
                                   (128, 4096, 512), (130, 129, 1168), (333, 777, 640), (600, 4100, 256)])
@pytest.mark.parametrize("kind", ["f32", "e8m0"])
def test_gemm_sizes(cuda, M, N, K, kind):
    print(f"gemm {M} {N} {K} {kind}", flush=True)
    ops_ = product(gen(cuda, M), M, N, K, kind)
    check_product(ops.fp8_gemm(*ops_), *ops_)
    check_product(ops.fp8_gemm(*ops_, out_dtype=F32), *ops_)


@pytest.mark.parametrize("M,N,K", [(4096, 4096, 256), (4100, 4090, 400), (4096, 4100, 16), (4100, 4104, 144)])
@pytest.mark.parametrize("kind", ["f32", "e8m0"])
def test_gemm_large(cuda, M, N, K, kind):
    """Enough tiles for the widest form, whole and ragged: rows from every part against the exact sums."""
    print(f"gemm large {M} {N} {K} {kind}", flush=True)
    a, sa, b, sb = product(gen(cuda, 5), M, N, K, kind)
    out = ops.fp8_gemm(a, sa, b, sb)
    rows = torch.cat([torch.arange(0, M, 37, device=cuda), torch.arange(M - 40, M, device=cuda)])
    check_product(out[rows], a[rows], sa[rows], b, sb)


@pytest.mark.parametrize("M,N,K", [(33, 129, 16528), (1000, 1000, 8336), (130, 8200, 8848), (65, 8200, 16528), (257, 16400, 8336),
                                   (1030, 2100, 8336), (1000, 520, 1168), (2050, 2100, 1168), (500, 8200, 8848),
                                   (2050, 4100, 8336)])
@pytest.mark.parametrize("kind", ["f32", "e8m0"])
def test_gemm_long(cuda, M, N, K, kind):
    """More blocks of K than a wave's register of weight scales and the chunks of activation scales hold, a short
    last one, whole and in parts, in every tile there is."""
    print(f"gemm long {M} {N} {K} {kind}", flush=True)
    a, sa, b, sb = product(gen(cuda, K), M, N, K, kind)
    out = ops.fp8_gemm(a, sa, b, sb)
    rows = torch.cat([torch.arange(0, M, 37, device=cuda), torch.arange(M - 33, M, device=cuda)])
    check_product(out[rows], a[rows], sa[rows], b, sb)


@pytest.mark.parametrize("M,N,K", [(32, 8200, 1536), (3, 2112, 1168), (1, 31, 1008), (32, 33, 400), (5, 24576, 128), (9, 100, 96),
                                   (1, 8192, 8192), (20, 4100, 3600), (32, 2112, 8208), (2, 576, 16400), (1, 64, 16384),
                                   (31, 576, 16144), (33, 129, 16), (64, 2100, 1536), (40, 8200, 3600), (63, 4100, 8080),
                                   (50, 8100, 400), (64, 300, 4096), (64, 8192, 8192), (65, 300, 1536)])
@pytest.mark.parametrize("kind", ["f32", "e8m0"])
def test_gemm_few_rows(cuda, M, N, K, kind):
    """Few rows, on both sides of the choice between waves over K and tiles; an odd result in between others."""
    print(f"gemm few {M} {N} {K} {kind}", flush=True)
    ops_ = product(gen(cuda, M + K), M, N, K, kind)
    want = ops.fp8_gemm(*ops_)
    check_product(want, *ops_)
    check_product(ops.fp8_gemm(*ops_, out_dtype=F32), *ops_)
    wide = torch.full((M + 2, N + 3), 3.0, dtype=BF, device=cuda)
    assert torch.equal(ops.fp8_gemm(*ops_, out=wide[1:M + 1, 1:N + 1]), want)
    wide[1:M + 1, 1:N + 1] = 3.0
    assert torch.all(wide == 3.0)


@pytest.mark.parametrize("K", [128, 1152])
@pytest.mark.parametrize("kind", ["f32", "e8m0"])
def test_gemm_far_rows(cuda, K, kind):
    """Rows whose offsets pass 32 bits, in the operands (2^23 bytes apart, the most) and in the result."""
    print(f"gemm far {K} {kind}", flush=True)
    M, N = 600, 40
    a, sa, b, sb = product(gen(cuda, 9), M, N, K, kind)
    want = ops.fp8_gemm(a, sa, b, sb)
    check_product(want, a, sa, b, sb)
    far = torch.empty(M << 23, dtype=torch.uint8, device=cuda).as_strided((M, K), (1 << 23, 1))
    far.copy_(a.view(torch.uint8))
    out = torch.empty((M << 22) + N, dtype=BF, device=cuda).as_strided((M, N), (1 << 22, 1))
    assert torch.equal(ops.fp8_gemm(far, sa, b, sb, out=out), want)
    # the weights' rows too: the product the other way round, with the activations' scales of the weights' rows
    b2, sb2 = ops.act_quant(torch.randn(M, K, device=cuda, generator=gen(cuda, 10)).to(BF), scale_dtype=sb.dtype)
    want = ops.fp8_gemm(b, sb.expand(N, -1).contiguous(), b2, sb2[:5].contiguous())
    far.copy_(b2.view(torch.uint8))
    assert torch.equal(ops.fp8_gemm(b, sb.expand(N, -1).contiguous(), far, sb2[:5].contiguous()), want)


def test_far_rows_of_norm_and_rope(cuda):
    """Rows 2^31 elements apart."""
    g = gen(cuda, 12)
    base = torch.empty((2 << 31) + 1024, dtype=BF, device=cuda)
    x = base.as_strided((3, 1000), (1 << 31, 1))
    near = rnd(g, 3, 1000).to(BF)
    x.copy_(near)
    w = rnd(g, 1000).to(BF)
    want = ops.rms_norm(near, w, 1e-6)
    assert torch.equal(ops.rms_norm(x, w, 1e-6), want)
    for got, exp in zip(ops.act_quant(x), ops.act_quant(near)):
        assert torch.equal(got.view(torch.uint8), exp.view(torch.uint8))
    t, pos = table(cuda, 50, 64), torch.tensor([0, 7, 49], device=cuda)
    q = base.as_strided((3, 5, 64), (1 << 31, 96, 1))
    close = q.contiguous()
    want = ops.rope(close, pos, t, out=torch.empty_like(close))
    assert torch.equal(ops.rope(q, pos, t), want) and torch.equal(q, want)
    assert torch.equal(ops.rms_norm(near, w, 1e-6, out=x), ops.rms_norm(near, w, 1e-6)) and x.stride(0) == 1 << 31


def test_gemm_strides_and_neighbours(cuda):
    """Rows inside wider ones, outputs inside wider ones: what lies beside them stays."""
    g = gen(cuda, 6)
    for M, N, K, kind in ((5, 200, 272, "e8m0"), (130, 333, 1152, "f32"), (7, 203, 272, "f32"), (45, 203, 1040, "e8m0")):
        a, sa, b, sb = product(g, M, N, K, kind)
        want = ops.fp8_gemm(a, sa, b, sb)

        def inside(t, extra, at):
            u8 = t.dtype in (FP8, E8M0)
            w = torch.full((t.shape[0], t.shape[1] + extra), 0x7f if u8 else float("nan"), device=cuda,
                           dtype=torch.uint8 if u8 else t.dtype)
            w[:, at:at + t.shape[1]] = t.view(torch.uint8) if u8 else t
            return w[:, at:at + t.shape[1]].view(t.dtype)
        wide = torch.full((M + 2, N + 7), 3.0, dtype=BF, device=cuda)
        got = ops.fp8_gemm(inside(a, 48, 16), inside(sa, 3, 1), inside(b, 32, 32), inside(sb, 2, 1), out=wide[1:M + 1, 3:N + 3])
        assert torch.equal(got, want)
        wide[1:M + 1, 3:N + 3] = 3.0
        assert torch.all(wide == 3.0)


def test_gemm_nan_stays_in_its_row_and_column(cuda):
    g = gen(cuda, 7)
    for M, N, K, kind in ((40, 300, 400, "e8m0"), (200, 300, 1040, "f32"), (20, 300, 400, "f32"), (20, 300, 8208, "e8m0")):
        a, sa, b, sb = product(g, M, N, K, kind)
        a.view(torch.uint8)[M - 3, K - 1] = 0x7f
        b.view(torch.uint8)[N - 2, 5] = 0xff
        out = ops.fp8_gemm(a, sa, b, sb)
        bad = out.isnan()
        want = torch.zeros_like(bad)
        want[M - 3], want[:, N - 2] = True, True
        assert torch.equal(bad, want)
        if kind == "e8m0":
            sa.view(torch.uint8)[1, 2] = 255
        else:
            sa[1, 2] = float("nan")
        want[1] = True
        assert torch.equal(ops.fp8_gemm(a, sa, b, sb).isnan(), want)


@pytest.mark.parametrize("kind", ["f32", "e8m0"])
def test_gemm_workspace(cuda, kind):
    """What a workspace held does not matter, nor that calls of several shapes share it; one that does not fit is not used."""
    need = []
    ops_ = [product(gen(cuda, 9 + i), M, N, 8192, kind) for i, (M, N) in enumerate(((100, 300), (40, 576), (70, 129)))]
    for a, sa, b, sb in ops_:
        need.append(ops.fp8_gemm_workspace_bytes(a.shape[0], b.shape[0], a.shape[1], sa.dtype))
    assert min(need) > 0
    want = [ops.fp8_gemm(*o) for o in ops_]
    check_product(want[0], *ops_[0])
    shared = torch.full((max(need) + 32,), 0xff, dtype=torch.uint8, device=cuda)
    for _ in range(2):
        for o, w in zip(ops_, want):
            assert torch.equal(ops.fp8_gemm(*o, workspace=shared), w)
    edge = shared[:max(need)]
    shared[max(need):] = 0x55
    for o, w in zip(ops_, want):
        assert torch.equal(ops.fp8_gemm(*o, workspace=edge), w)
    assert torch.all(shared[max(need):] == 0x55)
    shared.fill_(7)
    for bad in (shared[:min(need) - 1], shared[8:], torch.empty(max(need), dtype=torch.uint8)):
        assert torch.equal(ops.fp8_gemm(*ops_[0], workspace=bad), want[0])
    assert torch.all(shared == 7)


@pytest.mark.parametrize("kind", ["f32", "e8m0"])
def test_gemm_nan_in_the_widest_tile(cuda, kind):
    M, N, K = 4100, 4090, 400
    a, sa, b, sb = product(gen(cuda, 21), M, N, K, kind)
    a.view(torch.uint8)[M - 3, K - 1] = 0x7f
    b.view(torch.uint8)[N - 2, 5] = 0xff
    if kind == "e8m0":
        sa.view(torch.uint8)[300, 2] = 255
    else:
        sa[300, 2] = float("nan")
    bad = ops.fp8_gemm(a, sa, b, sb).isnan()
    want = torch.zeros_like(bad)
    want[M - 3], want[300], want[:, N - 2] = True, True, True
    assert torch.equal(bad, want)


def test_gemm_empty(cuda):
    a, sa, b, sb = product(gen(cuda, 8), 3, 5, 256, "e8m0")
    assert ops.fp8_gemm(a[:0], sa[:0], b, sb).shape == (0, 5)
    assert ops.fp8_gemm(a, sa, b[:0], sb[:0]).shape == (3, 0)


# ------------------------------------------------------------------ rotary positions
def table(device, rows, rot, seed=0):
    ang = torch.rand(rows, rot // 2, generator=gen(device, seed), device=device, dtype=torch.float64) * 6.3
    return torch.cat([ang.cos(), ang.sin()], dim=1).float()


@pytest.mark.parametrize("T,H,rot,head", [(1, 1, 2, 2), (3, 5, 6, 10), (4, 128, 64, 192), (257, 16, 64, 192), (33, 7, 96, 96), (9, 3, 128, 136),
                                          (2, 2, 512, 512), (5, 2, 510, 511), (1000, 1, 64, 576), (300, 40, 32, 64)])
@pytest.mark.parametrize("pairs,out_pairs", [(True, True), (True, False), (False, True), (False, False)])
def test_rope_sizes(cuda, T, H, rot, head, pairs, out_pairs):
    print(f"rope {T} {H} {rot} {pairs} {out_pairs}", flush=True)
    g = gen(cuda, T + rot)
    q_all, k_all = rnd(g, T, H, head).to(BF), rnd(g, T, 2, head + 8).to(BF)
    q, k = q_all[..., head - rot:], k_all[..., head + 8 - rot:]
    t = table(cuda, 50, rot)
    pos = torch.randint(-3, 60, (T,), generator=g, device=cuda)  # some are outside the table
    kept = q_all.clone(), k_all.clone()
    wants = [A.rope(x, t, pos, pairs, out_pairs) for x in (q, k)]
    outs = ops.rope(q, pos, t, out=torch.empty_like(q), k=k, k_out=torch.empty(T, 2, rot + 1, dtype=BF, device=cuda)[..., 1:],
                    interleaved=pairs, out_interleaved=out_pairs)
    for got, (want, err) in zip(outs, wants):
        assert A.within_bf16(got, want, err)
    assert torch.equal(q_all, kept[0]) and torch.equal(k_all, kept[1])
    # in place, and int32 positions: the same, and the rest of each head as it was
    ops.rope(q, pos.to(torch.int32), t, k=k, interleaved=pairs, out_interleaved=out_pairs)
    assert torch.equal(q, outs[0]) and torch.equal(k, outs[1])
    assert torch.equal(q_all[..., :head - rot], kept[0][..., :head - rot])
    assert torch.equal(k_all[..., :head + 8 - rot], kept[1][..., :head + 8 - rot])
    q1 = ops.rope(kept[0][..., head - rot:].contiguous(), pos, t, interleaved=pairs, out_interleaved=out_pairs)
    assert torch.equal(q1, outs[0])


def test_rope_many_heads_a_lane(cuda):
    """Enough tokens for several heads a lane, and a count of heads that these do not divide."""
    for T, H, rot in ((8200, 7, 64), (4099, 17, 64), (8200, 9, 40), (40000, 3, 30), (20000, 1, 128)):
        print(f"rope many {T} {H} {rot}", flush=True)
        g = gen(cuda, T)
        q, k = rnd(g, T, H, rot).to(BF), rnd(g, T, 1, rot + 8).to(BF)[..., 8:]
        t, pos = table(cuda, 5000, rot), torch.randint(0, 5000, (T,), generator=g, device=cuda)
        wants = [A.rope(x, t, pos, True, False) for x in (q, k)]
        for got, (want, err) in zip(ops.rope(q, pos, t, k=k, interleaved=True, out_interleaved=False), wants):
            assert A.within_bf16(got, want, err)


def test_rope_heads_outside(cuda):
    """Heads outside tokens in memory (a view [T, H, rot] of [H, T, rot]), in place and not."""
    g = gen(cuda, 4)
    x = rnd(g, 6, 33, 64).to(BF)
    q, t, pos = x.transpose(0, 1), table(cuda, 64, 64), torch.arange(33, device=cuda)
    want, err = A.rope(q, t, pos, True, True)
    assert A.within_bf16(ops.rope(q, pos, t, out=torch.empty_like(q)), want, err)
    assert A.within_bf16(ops.rope(q, pos, t), want, err)


def test_rope_refuses_shared_outputs(cuda):
    q, t, pos = torch.zeros(4, 1, 64, dtype=BF, device=cuda), table(cuda, 8, 64), torch.arange(4, device=cuda)
    with pytest.raises(ValueError, match="overlap"):
        ops.rope(q.expand(4, 3, 64), pos, t)
    with pytest.raises(ValueError, match="overlap"):
        ops.rope(q.clone(), pos, t, out=q[:1].expand(4, 1, 64))
    # read alike, they are fine
    got = ops.rope(q.expand(4, 3, 64), pos, t, out=torch.empty(4, 3, 64, dtype=BF, device=cuda))
    assert torch.all(got == 0)


def test_rope_empty(cuda):
    t = table(cuda, 4, 64)
    q = torch.zeros(0, 3, 64, dtype=BF, device=cuda)
    assert ops.rope(q, torch.zeros(0, dtype=torch.int64, device=cuda), t).shape == (0, 3, 64)
    q, k = torch.zeros(2, 0, 64, dtype=BF, device=cuda), torch.ones(2, 1, 64, dtype=BF, device=cuda)
    ops.rope(q, torch.zeros(2, dtype=torch.int64, device=cuda), t, k=k)
    want, err = A.rope(torch.ones(2, 1, 64, dtype=BF, device=cuda), t, torch.zeros(2, device=cuda), True, True)
    assert A.within_bf16(k, want, err)
