"""The table of cosines and sines: plain and scaled frequencies, and what is refused."""
import math

import pytest
import torch

from nanoengine_amd import rotary


def test_plain_table():
    t = rotary.cos_sin_cache(70000, 64, base=10000.0, device="cpu")
    assert t.shape == (70000, 64) and t.dtype == torch.float32
    for pos in (0, 1, 65535, 65536, 69999):  # both sides of the rows that are made at a time
        for p in (0, 1, 17, 31):
            angle = pos * 10000.0 ** (-2 * p / 64)
            # half a step of float32, and float64's own error of an angle of 70000
            tol = 2.0 ** -25 + 1e-10
            assert abs(t[pos, p].item() - math.cos(angle)) <= tol and abs(t[pos, 32 + p].item() - math.sin(angle)) <= tol


def test_scaled_frequencies():
    plain = rotary.inverse_frequencies(64, 10000.0)
    slow = rotary.inverse_frequencies(64, 10000.0, factor=40.0, original_max_position=4096)
    turns = 4096 * plain / (2 * math.pi)
    ratio = slow / plain
    # (the bounds are whole pairs: a pair beyond them is kept, or slowed, in full)
    assert torch.all(ratio[turns > 32 * 10000.0 ** (2 / 64)] == 1)
    assert torch.allclose(ratio[turns < 10000.0 ** (-2 / 64)], torch.tensor(1 / 40, dtype=torch.float64), rtol=1e-12)
    # (the ratio of two rounded float64 values)
    assert torch.all(ratio[1:] <= ratio[:-1] * (1 + 2.0 ** -50)) and ratio[0] == 1 and 1 / 40 < ratio[15] < 1
    # pair(32) = 10.4 and pair(1) = 22.5: the blend goes from pair 10 to 23
    keep = 1 - (15 - 10) / 13
    assert abs(ratio[15].item() - (keep + (1 - keep) / 40)) < 1e-12
    assert torch.equal(rotary.inverse_frequencies(64, 10000.0, factor=1.0, original_max_position=4096), plain)


def test_scaled_table():
    freq = rotary.inverse_frequencies(32, 5000.0, factor=8.0, original_max_position=1024)
    angle = torch.outer(torch.arange(50, dtype=torch.float64), freq)
    kw = dict(factor=8.0, original_max_position=1024, device="cpu")
    by_default = rotary.cos_sin_cache(50, 32, 5000.0, **kw)
    want = torch.cat([angle.cos(), angle.sin()], dim=1)
    assert torch.equal(by_default, (want * (0.1 * math.log(8.0) + 1.0)).float())
    assert torch.equal(rotary.cos_sin_cache(50, 32, 5000.0, attention_factor=1.0, **kw), want.float())


@pytest.mark.parametrize("kw", [dict(rot_dim=7), dict(rot_dim=0), dict(base=1.0), dict(factor=0.5), dict(factor=2.0),
                                dict(factor=2.0, original_max_position=0), dict(beta_fast=1.0, beta_slow=1.0),
                                dict(max_position=0)])
def test_refusals(kw):
    with pytest.raises(ValueError):
        rotary.cos_sin_cache(**{"max_position": 8, "rot_dim": 64, "device": "cpu", **kw})
