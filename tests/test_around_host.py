"""The steps around the attention without a GPU: refusals of the entry points and of their adapters, and the oracle's
format against known answers."""
import ctypes

import pytest
import torch

from nanoengine_amd import _lib, deep_gemm, ops, projections
from oracle import around_oracle as A

ONE = ctypes.c_void_p(16)   # a non-null, aligned address that is never dereferenced
ODD = ctypes.c_void_p(17)
TWO = ctypes.c_void_p(18)
P = None
BF, FP8, E8M0, F32 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.float32
KINDS = {"f32": F32, "e8m0": E8M0}


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        from nanoengine_amd import build
        build.build()
    return _lib.load()


def _bad(lib, name, args, changes):
    """Every change of one argument gives its status, and a message."""
    fn = getattr(lib, name)
    for at, value, status in changes:
        a = list(args)
        a[at] = value
        assert fn(*a) == status, (name, at, value, lib.dsa_last_error())
        if status:
            assert lib.dsa_last_error()


def test_norm_refusals(lib):
    f = ctypes.c_float
    args = [ONE, 256, ONE, 256, ONE, 256, ONE, 0, f(1e-6), 4, 256, ONE, 256, ONE, 256, ONE, 2, 0, P]
    _bad(lib, "dsa_rms_norm", args,
         [(0, P, 1), (6, P, 1), (0, ODD, 1), (6, ODD, 1), (1, 255, 1), (2, P, 1), (2, ODD, 1), (3, 255, 1), (4, ODD, 1), (5, 255, 1),
          (8, f(-1), 1), (8, f(float("nan")), 1), (8, f(float("inf")), 1), (9, -1, 1), (9, 2 ** 31, 1), (9, 0, 0), (10, 0, 1),
          (10, 32769, 2), (11, ODD, 1), (12, 255, 1), (13, P, 1), (14, 255, 1), (15, P, 1), (15, TWO, 1), (16, 1, 1), (17, 2, 1),
          (17, -1, 1)])
    a = list(args)
    a[11] = a[13] = a[15] = P  # no output at all
    assert lib.dsa_rms_norm(*a) == 1
    a = list(args)
    a[6], a[7] = TWO, 1        # f32 weights at an odd address
    assert lib.dsa_rms_norm(*a) == 1


def test_quant_refusals(lib):
    _bad(lib, "dsa_act_quant", [ONE, 256, 4, 256, ONE, 256, ONE, 2, 0, P],
         [(0, P, 1), (0, ODD, 1), (1, 255, 1), (2, -1, 1), (2, 2 ** 31, 1), (2, 0, 0), (3, 0, 1), (4, P, 1), (5, 255, 1), (6, P, 1),
          (6, TWO, 1), (7, 1, 1), (8, 2, 1)])


def test_gemm_refusals(lib):
    args = [ONE, 256, ONE, 2, ONE, 256, ONE, 2, 0, 4, 300, 256, ONE, 300, 0, P, 0, P]
    _bad(lib, "dsa_fp8_gemm", args,
         [(0, P, 1), (0, TWO, 1), (1, 240, 1), (1, 264, 1), (2, P, 1), (2, TWO, 1), (3, 1, 1), (4, P, 1), (4, TWO, 1), (5, 240, 1),
          (5, 264, 1), (6, P, 1), (6, TWO, 1), (7, 1, 1), (8, 2, 1), (9, -1, 1), (9, 0, 0), (10, -1, 1), (10, 0, 0), (11, 0, 1),
          (11, 200, 2), (12, P, 1), (12, ODD, 1), (13, 299, 1)])
    far = 2 ** 23 + 16
    _bad(lib, "dsa_fp8_gemm", args, [(1, far, 2), (5, far, 2), (1, 2 ** 40, 2)])
    assert lib.dsa_fp8_gemm_workspace_bytes(0, 8, 8, 0) == 0 and lib.dsa_fp8_gemm_workspace_bytes(8, 8, -1, 0) == 0
    assert lib.dsa_fp8_gemm_workspace_bytes(8, 8, 8192, 2) == 0


def test_gemm_refuses_a_workspace_too_small_or_unaligned(lib):
    m, n, k = 100, 256, 8192  # few tiles of many blocks: split over K
    need = lib.dsa_fp8_gemm_workspace_bytes(m, n, k, 0)
    assert need > 0
    args = [ONE, k, ONE, 64, ONE, k, ONE, 64, 0, m, n, k, ONE, n, 0, ONE, need, P]
    _bad(lib, "dsa_fp8_gemm", args, [(15, P, 4), (16, need - 1, 4), (15, ctypes.c_void_p(24), 1)])


def test_rope_refusals(lib):
    args = [ONE, 640, 64, 10, ONE, 640, 64, ONE, 64, 64, 1, ONE, 64, 64, 4, 64, ONE, 100, ONE, 0, 1, 1, P]
    _bad(lib, "dsa_rope", args,
         [(0, P, 1), (0, ODD, 1), (3, -1, 1), (4, P, 1), (4, ODD, 1), (7, P, 1), (7, ODD, 1), (10, -1, 1), (11, P, 1), (11, ODD, 1),
          (14, -1, 1), (14, 2 ** 31, 1), (14, 0, 0), (15, 63, 1), (15, 0, 1), (15, 514, 2), (16, P, 1), (16, TWO, 1), (17, 0, 1),
          (18, P, 1), (18, TWO, 1)])
    # output rows that share elements: of heads, of tokens, of the key; and more heads than an index holds
    _bad(lib, "dsa_rope", args, [(6, 0, 1), (6, 63, 1), (5, 0, 1), (5, 639, 1), (12, 0, 1), (12, 63, 1), (14, 2 ** 28, 2)])
    a = list(args)
    a[18], a[19] = ctypes.c_void_p(20), 1  # int64 positions at a 4-byte address
    assert lib.dsa_rope(*a) == 1
    a = list(args)
    a[3] = a[10] = 0                       # no heads
    assert lib.dsa_rope(*a) == 0


# ------------------------------------------------------------------ adapters
def test_adapters_refuse_bad_tensors():
    x, w = torch.zeros(3, 256, dtype=BF), torch.zeros(256, dtype=BF)
    for kw, match in (({"x": x.float()}, "x must be"), ({"x": x[0]}, "x must be"), ({"x": x.t()}, "x must be"), ({"weight": w[:255]}, "weight"),
                      ({"weight": w.half()}, "weight"), ({"residual": x[:2]}, "residual"), ({"residual_out": x}, "needs a residual"),
                      ({"residual": x, "residual_out": x.float()}, "residual_out"), ({"out": x[:, :255]}, "out must be"),
                      ({}, "GPU only")):
        with pytest.raises(RuntimeError, match=match):
            ops.rms_norm(**{**dict(x=x, weight=w, eps=1e-6), **kw})
    codes, scales = torch.zeros(3, 256, dtype=FP8), torch.zeros(3, 2, dtype=F32)
    for kw, match in (({"codes": codes[:2]}, "codes"), ({"codes": codes.float()}, "codes"), ({"scales": scales[:, :1]}, "scales"),
                      ({"scales": scales.double()}, "scales"), ({"scales": scales.t().contiguous().t()}, "scales"), ({"x": x[0]}, "x must be"),
                      ({}, "GPU only")):
        with pytest.raises(RuntimeError, match=match):
            ops.act_quant(**{**dict(x=x, codes=codes, scales=scales), **kw})
        with pytest.raises(RuntimeError, match=match):
            ops.rms_norm_quant(**{**dict(x=x, weight=w, eps=1e-6, codes=codes, scales=scales), **kw})
    a, sa = torch.zeros(3, 272, dtype=FP8), torch.zeros(3, 3, dtype=E8M0)
    b, sb = torch.zeros(200, 272, dtype=FP8), torch.zeros(2, 3, dtype=E8M0)
    for kw, match in (({"a": a.float()}, "a must be"), ({"b": b[:, :256]}, "share K"), ({"a_scale": sa[:, :2]}, "a_scale"),
                      ({"b_scale": sb[:1]}, "b_scale"), ({"a_scale": torch.zeros(3, 3)}, "both"), ({"b_scale": sb.to(F32).double()}, "both"),
                      ({"b": b.t().contiguous().t()}, "b must be"), ({}, "GPU only")):
        with pytest.raises(RuntimeError, match=match):
            ops.fp8_gemm(**{**dict(a=a, a_scale=sa, b=b, b_scale=sb), **kw})
    q, t, pos = torch.zeros(3, 4, 64, dtype=BF), torch.zeros(9, 64), torch.zeros(3, dtype=torch.int32)
    for kw, match in (({"q": q.float()}, "q must be"), ({"q": q[0]}, "q must be"), ({"q": q.transpose(1, 2)}, "q must be"), ({"positions": pos[:2]}, "positions"),
                      ({"positions": pos.float()}, "positions"), ({"cos_sin_cache": t[:, :32]}, "cos_sin_cache"),
                      ({"cos_sin_cache": t.double()}, "cos_sin_cache"), ({"out": q[:, :3]}, "out must be"), ({"k": q[:2]}, "k must be"),
                      ({"k": q[..., :32]}, "k must be"), ({"k_out": q}, "needs k"), ({"k": q[:, :1], "k_out": q}, "k_out"), ({}, "GPU only")):
        with pytest.raises(RuntimeError, match=match):
            ops.rope(**{**dict(q=q, positions=pos, cos_sin_cache=t), **kw})


def test_layer_refuses_weights_that_do_not_fit():
    D, rank, H, nope, v = 256, 128, 2, 64, 32
    shapes = dict(norm=(D,), a=(rank + 704, D), q_norm=(rank,), kv_norm=(512,), q=(H * (nope + 64), rank), k_up=(H, nope, 512),
                  v_up=(H, 512, v), o=(D, H * v), idx_q=(8192, rank), idx_gate=(64, D), idx_norm=(128,), idx_bias=(128,))
    good = {k: torch.zeros(s) for k, s in shapes.items()}
    layer = projections.MlaProjections(**good, cos_sin_cache=torch.zeros(8, 64))
    assert layer.q.codes.shape == (H * (nope + 64), rank) and layer.a.scales.shape == (7, 2)
    for name in ("a", "kv_norm", "q", "k_up", "v_up", "o", "idx_q", "idx_gate"):
        with pytest.raises(ValueError, match="must be"):
            projections.MlaProjections(**{**good, name: good[name][..., 1:]}, cos_sin_cache=torch.zeros(8, 64))
    with pytest.raises(ValueError, match="scale_dtype"):
        projections.quantize_weight(good["a"], torch.float16)
    x, s = torch.zeros(3, 256, dtype=FP8), torch.zeros(3, 2)
    with pytest.raises(RuntimeError, match="share K"):
        deep_gemm.fp8_gemm_nt((x, s), (x[:, :128], s[:1, :1]), torch.zeros(3, 3))


@pytest.mark.parametrize("kind", ["f32", "e8m0"])
def test_weights_are_rounded_by_the_rule_of_activations(kind):
    w = torch.randn(200, 300, generator=torch.Generator().manual_seed(0))
    w[:128, 128:256] = 0
    codes, scales = projections.quantize_weight(w, KINDS[kind])
    want = A.scale_values(A.quantise_weight(w, kind)[1])
    assert torch.all((A.scale_values(scales) - want).abs() <= (2 * A.EPS32 if kind == "f32" else 0) * want)
    full = A.scale_values(scales).repeat_interleave(128, 0)[:200].repeat_interleave(128, 1)[:, :300]
    tol = torch.maximum(A.HALF_FP8 * w.double().abs(), 2.0 ** -10 * full) * (1 + 3 * A.EPS32) + 3 * A.EPS32 * w.double().abs()
    assert torch.all((codes.double() * full - w.double()).abs() <= tol)


# ------------------------------------------------------------------ the oracle's format
@pytest.mark.parametrize("amax,byte", [(0.0, 79), (448.0, 127), (449.0, 128), (224.0, 126), (2.0 ** -40, 79), (2.0 ** -38, 81), (2.0 ** 127, 246)])
def test_power_of_two_scale(amax, byte):
    x = torch.zeros(1, 128, dtype=torch.float64)
    x[0, 5] = -amax
    assert A.quantise_rows(x, "e8m0")[1].view(torch.uint8).item() == byte
    assert A.scale_values(A.quantise_rows(x, "e8m0")[1]).item() == 2.0 ** (byte - 127)


def test_weight_blocks_and_their_product():
    w = torch.zeros(130, 144)
    w[0, 0], w[129, 143] = 448.0, 896.0
    codes, scales = A.quantise_weight(w, "f32")
    assert scales[0, 0] == 1 and scales[1, 1] == 2 and codes[129, 143].float() == 448 and codes[0, 0].float() == 448
    a, sa = A.quantise_rows(torch.eye(144)[[0, 143]], "f32")
    out, err = A.gemm(a, sa, codes, scales)
    assert abs(out[0, 0] - 448) < 1e-4 and abs(out[1, 129] - 896) < 1e-4 and torch.count_nonzero(out) == 2


def test_rope_quarter_turn():
    t = torch.tensor([[0.0, 1.0, 1.0, 0.0]])  # pair 0 turns by 90 degrees, pair 1 not at all
    x = torch.tensor([[[1.0, 2.0, 3.0, 4.0]]])
    pos = torch.tensor([5])                   # past the table: its last row
    assert A.rope(x, t, pos, True, True)[0].tolist() == [[[-2, 1, 3, 4]]]
    assert A.rope(x, t, pos, True, False)[0].tolist() == [[[-2, 3, 1, 4]]]
    assert A.rope(x, t, pos, False, False)[0].tolist() == [[[-3, 2, 1, 4]]]
    assert A.rope(x, t, pos, False, True)[0].tolist() == [[[-3, 1, 2, 4]]]
