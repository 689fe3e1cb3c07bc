"""4-bit sparse MLA decode past one round of CUs, where unsplit items come before split ones, and the order of a
row's slots."""
import pytest
import torch

from nanoengine_amd import ops
from oracle import fp4_oracle as F

pytestmark = pytest.mark.gpu
SCALE = 192 ** -0.5


def _cache(seed, device):
    g = torch.Generator(device=device).manual_seed(seed)
    rows = F.mla_rows(torch.randn(40 * 64, 576, generator=g, device=device).to(torch.bfloat16))
    return rows.view(40, 64, 1, 400), F.mla_values(rows), g


def _check(o, lse, q, values, idx):
    at = idx.long()
    eo, el, ot, lt = F.attend(q, values[at[at >= 0]], SCALE)
    assert torch.all((o.double() - eo).abs() <= ot + 1e-30)
    assert torch.all((lse.double() == el) | ((lse.double() - el).abs() <= lt))
    return ot, lt


# On 256 CUs: 300 items, 44 of them split five ways (32 blocks, uneven); 258 items, both of the last token's split eight
# ways; 258 items of three head groups, so that the last token's first group is whole and the others are split.
@pytest.mark.parametrize("T,H", [(150, 128), (129, 80), (86, 176)])
@pytest.mark.parametrize("last", ["plain", "nan", "empty", "parts"])
def test_whole_items_before_split_ones(cuda, T, H, last):
    print(f"mla fp4 mixed T={T} H={H} last={last}", flush=True)
    cache, values, g = _cache(T, cuda)
    q = torch.randn(T, H, 576, generator=g, device=cuda).to(torch.bfloat16)
    idx = torch.randint(0, 2559, (T, 2048), generator=g, device=cuda)
    idx[3::7, ::3] = -1
    idx[T // 2] = -1
    if last == "nan":
        idx[T - 1, 1700] = 2559
        cache[39, 63, 0, 256 + 9] = 255
    elif last == "empty":
        idx[T - 1] = -1
    elif last == "parts":                           # only some of its parts have keys
        idx[T - 1, :512] = -1
        idx[T - 1, 1000:] = -1
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        assert ops.sparse_mla_past_one_round(T, H) and ops.sparse_mla_num_splits(T, H, 2048) > 1
    outs = torch.full((T + 2, H, 512), 7.0, dtype=torch.bfloat16, device=cuda)
    lses = torch.full((T + 2, H), 7.0, device=cuda)
    o, lse = ops.sparse_mla_decode_fp4(q, cache, idx.to(torch.int32), SCALE, out=outs[1:-1], lse=lses[1:-1])
    torch.cuda.synchronize()
    assert torch.all(outs[::T + 1] == 7) and torch.all(lses[::T + 1] == 7)
    if last == "nan":
        assert torch.all(torch.isnan(o[T - 1])) and torch.all(torch.isnan(lse[T - 1]))
    for t in range(T - 1 if last == "nan" else T):
        _check(o[t], lse[t], q[t], values, idx[t])


@pytest.mark.parametrize("T,H", [(2, 16), (2, 128), (150, 64)])
def test_order_of_the_slots_changes_only_rounding(cuda, T, H):
    """The same slots, some of them twice and some masked, in two orders: both within their bound of the exact
    result, and so within twice that of each other."""
    cache, values, g = _cache(31, cuda)
    q = torch.randn(T, H, 576, generator=g, device=cuda).to(torch.bfloat16)
    idx = torch.randint(0, 300, (T, 512), generator=g, device=cuda)
    idx[:, ::5] = -1
    order = torch.rand(T, 512, generator=g, device=cuda).argsort(dim=1)
    other = idx.gather(1, order)
    a, la = ops.sparse_mla_decode_fp4(q, cache, idx.to(torch.int32), SCALE)
    b, lb = ops.sparse_mla_decode_fp4(q, cache, other.to(torch.int32), SCALE)
    torch.cuda.synchronize()
    for t in range(T):
        ot, lt = _check(a[t], la[t], q[t], values, idx[t])
        _check(b[t], lb[t], q[t], values, other[t])
        assert torch.all((a[t].double() - b[t].double()).abs() <= 2 * ot + 1e-30)
        assert torch.all((la[t].double() - lb[t].double()).abs() <= 2 * lt)
