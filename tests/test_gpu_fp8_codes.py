"""fp8 codes of activations and weights are e4m3(x / s) for the scale that is stored with them, byte for byte, also where x / s
lies on a tie or within a step of 2^-24 of one."""
import pytest
import torch

from nanoengine_amd import ops, projections

pytestmark = pytest.mark.gpu
BF, FP8, E8M0, F32 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.float32


def quotient_codes(x, scales):
    """e4m3 of x / s as bytes: one rounded division in float32 on the CPU."""
    s = scales.cpu()
    s = s if s.dtype == F32 else (s.view(torch.uint8).to(torch.int32) << 23).view(F32)
    return (x.float().cpu() / s.repeat_interleave(128, dim=1)[:, :x.shape[1]]).to(FP8).view(torch.uint8)


# bf16 elements of a block whose largest one is a whole multiple of a few steps meet ties often
@pytest.mark.parametrize("rows,dim", [(2048, 384), (515, 1600), (300, 131)])
@pytest.mark.parametrize("scale_dtype", [F32, E8M0])
def test_codes_are_those_of_the_quotient(cuda, rows, dim, scale_dtype):
    g = torch.Generator(device=cuda).manual_seed(dim)
    x = (torch.randn(rows, dim, generator=g, device=cuda) * torch.exp(1.5 * torch.randn(dim, generator=g, device=cuda))).to(BF)
    codes, scales = ops.act_quant(x, scale_dtype=scale_dtype)
    assert torch.equal(codes.view(torch.uint8).cpu(), quotient_codes(x, scales))


@pytest.mark.parametrize("scale_dtype", [F32, E8M0])
def test_codes_of_the_norm(cuda, scale_dtype):
    """Rows of ones with either sign and no eps: the mean square is 1, and y is the weight with the row's signs."""
    g = torch.Generator(device=cuda).manual_seed(4)
    x = torch.where(torch.rand(64, 8192, generator=g, device=cuda) < 0.5, -1.0, 1.0).to(BF)
    weight = torch.randn(8192, generator=g, device=cuda).to(BF)
    for w in (weight, weight.float()):
        codes, scales = ops.rms_norm_quant(x, w, 0.0, scale_dtype=scale_dtype)
        assert torch.equal(codes.view(torch.uint8).cpu(), quotient_codes(x.float() * w.float(), scales))
    # a layer's weights are rounded by the same rule
    tall = (x * weight).float()[:, :1000]
    codes, scales = projections.quantize_weight(tall, scale_dtype)
    assert torch.equal(codes.view(torch.uint8).cpu(), quotient_codes(tall, scales.repeat_interleave(128, dim=0)[:64]))


def test_scales_are_the_rounded_quotient(cuda):
    """float32 scales of activations and of weights: max(amax, 2^-40) / 448 rounded once, on whichever device."""
    g = torch.Generator(device=cuda).manual_seed(9)
    x = torch.randn(512, 1600, generator=g, device=cuda).to(BF)
    blocks = torch.nn.functional.pad(x.double().abs().cpu(), (0, 64)).view(512, 13, 128)
    want = (blocks.amax(-1).clamp_min(2.0 ** -40) / 448).float()
    assert torch.equal(ops.act_quant(x, scale_dtype=F32)[1].cpu(), want)
    want = blocks.view(4, 128, 13, 128).amax((1, 3)).clamp_min(2.0 ** -40)
    for w in (x, x.cpu()):
        assert torch.equal(projections.quantize_weight(w, F32)[1].cpu(), (want / 448).float())


@pytest.mark.parametrize("scale_dtype", [F32, E8M0])
def test_signs_of_zeros(cuda, scale_dtype):
    """Zeros, and what is rounded to zero, keep their sign, as a quotient does; over an infinite scale too."""
    x = torch.zeros(3, 128, dtype=BF, device=cuda)
    x[:, 1], x[:, 2], x[:, 3], x[:, 4] = -0.0, -1e-30, 1e-30, -3.0
    x[1, 5] = 1e30
    x[2, 6] = float("inf")
    codes, scales = ops.act_quant(x, scale_dtype=scale_dtype)
    got, want = codes.view(torch.uint8).cpu(), quotient_codes(x, scales)
    got[2, 6] = want[2, 6] = 0  # (NaN; its sign is free)
    assert torch.equal(got, want)
