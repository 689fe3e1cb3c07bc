"""Weights that are no numbers, rounded by the rule of the activations: a NaN is its own code and nobody else's."""
import pytest
import torch

from nanoengine_amd import projections

E8M0, F32 = torch.float8_e8m0fnu, torch.float32


@pytest.mark.parametrize("scale_dtype", [F32, E8M0])
def test_nan_leaves_its_block_alone(scale_dtype):
    w = torch.randn(200, 300, generator=torch.Generator().manual_seed(0))
    want, scales = projections.quantize_weight(w, scale_dtype)
    # where no block's largest one is
    at = [(0, 0), (127, 130), (199, 299)]
    w2 = w.clone()
    for r, c in at:
        block = w[r // 128 * 128:r // 128 * 128 + 128, c // 128 * 128:c // 128 * 128 + 128].abs()
        assert w[r, c].abs() < block.max()
        w2[r, c] = float("nan")
    got, got_scales = projections.quantize_weight(w2, scale_dtype)
    assert torch.equal(got_scales.view(torch.uint8), scales.view(torch.uint8))
    bad = got.float().isnan()
    assert bad.sum() == len(at) and all(bad[r, c] for r, c in at)
    assert torch.equal(got.view(torch.uint8)[~bad], want.view(torch.uint8)[~bad])


@pytest.mark.parametrize("scale_dtype", [F32, E8M0])
def test_infinity_and_blocks_of_nan(scale_dtype):
    w = torch.ones(130, 256)
    w[0, 0], w[128:, 128:] = float("-inf"), float("nan")
    codes, scales = projections.quantize_weight(w, scale_dtype)
    c, s = codes.float(), scales.float()
    assert c[0, 0].isnan() and torch.all(c[:128, :128].flatten()[1:] == 0) and c[128:, 128:].isnan().all()
    assert s[0, 0] == (float("inf") if scale_dtype == F32 else 2.0 ** 127)
    # nothing but NaN: the scale of zeros
    assert s[1, 1] == (torch.tensor(2.0 ** -40) / 448 if scale_dtype == F32 else 2.0 ** -48)
