"""Sparse MLA decode where keys score -inf for some heads and +inf for others (an infinite rope value).

A key at -inf weighs nothing: the head's result is that of its other keys, also where the kernel meets the
infinite ones first and has no finite score yet. A score of +inf makes the head's outputs NaN."""
import pytest
import torch

from nanoengine_amd import ops, synth
from oracle import fp4_oracle as F

pytestmark = pytest.mark.gpu
SCALE = 192 ** -0.5
ROWS = 40 * 64


def _query(T, H, g, device):
    """Heads' first rope element: negative for the even ones, positive for the odd ones."""
    q = torch.randn(T, H, 576, generator=g, device=device)
    sign = torch.where(torch.arange(H, device=device) % 2 == 0, -1.0, 1.0)
    q[..., 512] = (q[..., 512].abs() + 0.1) * sign
    return q.to(torch.bfloat16)


def _fp4_cache(g, device, infinite):
    rows = F.mla_rows(torch.randn(ROWS, 576, generator=g, device=device).to(torch.bfloat16))
    values = F.mla_values(rows)
    rows[infinite, 272], rows[infinite, 273] = 0x80, 0x7f   # bf16 +inf
    return rows.view(40, 64, 1, 400), values


def _batch(H, group):
    """The largest unsplit batch of head groups of 16 (0) or 32 (1), one past it (2)."""
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    return (cus // -(-H // 16), cus // -(-H // 32), cus // -(-H // 32) + 1)[group]


@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("first", [64, 32, 16])
@pytest.mark.parametrize("H,group", [(128, 0), (128, 1), (128, 2), (16, 2), (32, 2)])
def test_4bit_keys_at_minus_infinity_come_first(cuda, H, group, first, splits):
    """The first 64, 32 or 16 keys (a block, a score wave's keys of the wide and of the narrow form)."""
    T = _batch(H, group)
    print(f"mla fp4 infinite T={T} H={H} first={first} splits={splits}", flush=True)
    g = torch.Generator(device=cuda).manual_seed(first + H + group)
    infinite = torch.arange(100, device=cuda)
    cache, values = _fp4_cache(g, cuda, infinite)
    q = _query(T, H, g, cuda)
    idx = torch.randint(100, ROWS, (T, 256), generator=g, device=cuda)
    idx[:, :first] = torch.randint(0, 100, (T, first), generator=g, device=cuda)
    idx[1::3, 40:50] = -1                                   # some rows with masked keys beside
    idx[2::5, 128:] = 7                                     # a second part with nothing but infinite keys
    o, lse = ops.sparse_mla_decode_fp4(q, cache, idx.to(torch.int32), SCALE, num_splits=splits)
    torch.cuda.synchronize()
    assert torch.all(torch.isnan(o[:, 1::2])) and not torch.any(torch.isfinite(lse[:, 1::2]))
    for t in range(T):
        at = idx[t][idx[t] >= 100]
        eo, el, ot, lt = F.attend(q[t, 0::2], values[at], SCALE)
        assert torch.all((o[t, 0::2].double() - eo).abs() <= ot + 1e-30), t
        assert torch.all((lse[t, 0::2].double() - el).abs() <= lt), t


@pytest.mark.parametrize("H", [16, 32, 64])
def test_4bit_nothing_but_minus_infinity(cuda, H):
    g = torch.Generator(device=cuda).manual_seed(H)
    cache, _ = _fp4_cache(g, cuda, torch.arange(ROWS, device=cuda))
    idx = torch.randint(0, ROWS, (3, 128), generator=g, device=cuda).to(torch.int32)
    o, lse = ops.sparse_mla_decode_fp4(_query(3, H, g, cuda), cache, idx, SCALE)
    torch.cuda.synchronize()
    assert torch.all(o[:, 0::2] == 0) and torch.all(torch.isneginf(lse[:, 0::2]))
    assert torch.all(torch.isnan(o[:, 1::2]))


@pytest.mark.parametrize("H", [16, 64])
def test_fp8_keys_at_minus_infinity_come_first(cuda, H):
    """The fp8 kernel's running sum is the same one: the result is that of the call without those keys. (It keeps
    keys far below the largest at 2^-30 of it, 64 keys here: 2^-24 of the sum; outputs round to bf16.)"""
    g = torch.Generator(device=cuda).manual_seed(H)
    cache = synth.make_mla_cache(40, seed=1, device=cuda)
    flat = cache.view(torch.uint8)
    flat[0, :, 0, 528], flat[0, :, 0, 529] = 0x80, 0x7f     # the first block's keys
    q = _query(3, H, g, cuda)
    idx = torch.randint(64, ROWS, (3, 256), generator=g, device=cuda)
    idx[:, :64] = torch.arange(64, device=cuda)
    o, lse = ops.sparse_mla_decode(q, cache, idx.to(torch.int32), SCALE)
    idx[:, :64] = -1
    want, want_lse = ops.sparse_mla_decode(q, cache, idx.to(torch.int32), SCALE)
    torch.cuda.synchronize()
    even = slice(0, None, 2)
    near = want[:, even].float()
    assert torch.all((o[:, even].float() - near).abs() <= 2.0 ** -7 * near.abs() + 2.0 ** -20 * near.abs().amax())
    assert torch.all((lse[:, even] - want_lse[:, even]).abs() <= 2.0 ** -20 * want_lse[:, even].abs().clamp(min=1))
