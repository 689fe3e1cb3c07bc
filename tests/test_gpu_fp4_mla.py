"""Sparse MLA decode over the 4-bit cache on the GPU, against float64 with the oracle's bounds."""
import pytest
import torch

from nanoengine_amd import ops
from oracle import fp4_oracle as F

pytestmark = pytest.mark.gpu
SCALE = 192 ** -0.5


def _cache(blocks, seed, device, block_size=64, pad=1, spread=0.0):
    """[blocks, block_size, 1, 400] view (rows of quantised normal values, channels of different size) and its values."""
    g = torch.Generator(device=device).manual_seed(seed)
    kv = torch.randn(blocks * block_size, 576, generator=g, device=device)
    kv = kv * torch.exp(spread * torch.randn(576, generator=g, device=device))
    rows = F.mla_rows(kv.to(torch.bfloat16))
    buf = torch.full((blocks, block_size + pad, 1, 400), 0xff, dtype=torch.uint8, device=device)
    buf[:, :block_size, 0] = rows.view(blocks, block_size, 400)
    return buf[:, :block_size], F.mla_values(rows)


def _query(T, H, seed, device):
    return torch.randn(T, H, 576, generator=torch.Generator(device=device).manual_seed(seed + 1),
                       device=device).to(torch.bfloat16)


def _indices(T, K, total, seed, device, invalid=0.0):
    g = torch.Generator().manual_seed(seed)
    idx = torch.stack([torch.randperm(max(total, K), generator=g)[:K] for _ in range(T)])
    idx[torch.rand(T, K, generator=g) < invalid] = -1
    return idx.to(torch.int32).to(device)


def _check(o, lse, q, values, idx, scale):
    for t in range(q.shape[0]):
        at = idx[t].long()
        at = at[(at >= 0) & (at < values.shape[0])]
        eo, el, ot, lt = F.attend(q[t], values[at], scale)
        assert torch.all((o[t].double() - eo).abs() <= ot + 1e-30), (t, (o[t].double() - eo).abs().max())
        if at.numel() == 0:
            assert torch.all(o[t] == 0) and torch.all(torch.isneginf(lse[t]))
        else:
            assert torch.all((lse[t].double() - el).abs() <= lt), (t, (lse[t].double() - el).abs().max())


@pytest.mark.parametrize("T,H,K,invalid", [(1, 16, 64, 0.0), (3, 32, 192, 0.3), (2, 48, 320, 0.1), (5, 64, 512, 0.0),
                                           (2, 80, 2048, 0.5), (3, 128, 2048, 0.0), (9, 128, 576, 0.05),
                                           (130, 128, 64, 0.2), (300, 16, 512, 0.1)])
def test_matches_float64(cuda, T, H, K, invalid):
    print(f"mla fp4 T={T} H={H} K={K}", flush=True)
    cache, values = _cache(40, T * 1000 + K, cuda)
    q, idx = _query(T, H, T, cuda), _indices(T, K, 40 * 64, K, cuda, invalid)
    o, lse = ops.sparse_mla_decode_fp4(q, cache, idx, SCALE)
    torch.cuda.synchronize()
    _check(o, lse, q, values, idx, SCALE)


@pytest.mark.parametrize("splits", [1, 2, 4, 8, 32])
def test_split_counts(cuda, splits):
    cache, values = _cache(40, 3, cuda)
    q, idx = _query(2, 128, 3, cuda), _indices(2, 2048, 2560, 3, cuda, 0.02)
    idx[1, 64:] = -1                                # every split but the first has no key
    o, lse = ops.sparse_mla_decode_fp4(q, cache, idx, SCALE, num_splits=splits)
    torch.cuda.synchronize()
    _check(o, lse, q, values, idx, SCALE)


def test_rows_without_keys_and_short_rows(cuda):
    cache, values = _cache(40, 4, cuda)
    q, idx = _query(6, 64, 4, cuda), _indices(6, 512, 2560, 4, cuda)
    idx[0] = -1                                     # nothing
    idx[1, 1:] = -1                                 # one key, the first
    idx[2, :511] = -1                               # one key, the last
    idx[3, :32] = -1                                # no key in the first half of the first block
    idx[4, 40:] = 10 ** 6                           # stale slots past the cache
    idx[5, ::2] = -5
    for splits in (1, 2, 8):
        o, lse = ops.sparse_mla_decode_fp4(q, cache, idx, SCALE, num_splits=splits)
        torch.cuda.synchronize()
        _check(o, lse, q, values, idx, SCALE)


@pytest.mark.parametrize("scale", [1.0, 0.0, 1e-4])
@pytest.mark.parametrize("order", ["random", "rising", "falling"])
def test_far_apart_scores(cuda, scale, order):
    """A softmax scale of 1 spreads the scores over hundreds of powers of two; in rising order every block moves
    the running maximum, in falling order (interleaved by halves of a block) the second half stays far below."""
    cache, values = _cache(40, 5, cuda, spread=0.5)
    q, idx = _query(2, 64, 5, cuda), _indices(2, 1024, 2560, 5, cuda)
    if order != "random":
        s = (values[idx.long()] @ q[:, 0].double()[..., None]).squeeze(-1)
        by = s.argsort(dim=1, descending=order == "falling")
        if order == "falling":
            a, b = by[:, :512].view(2, 16, 32), by[:, 512:].flip(1).view(2, 16, 32)
            by = torch.stack([a, b], dim=2).view(2, 1024)
        idx = idx.gather(1, by)
    o, lse = ops.sparse_mla_decode_fp4(q, cache, idx, scale)
    torch.cuda.synchronize()
    _check(o, lse, q, values, idx, scale)


@pytest.mark.parametrize("block_size,pad", [(64, 0), (48, 1), (1, 0), (256, 3)])
def test_cache_geometries(cuda, block_size, pad):
    blocks = 4096 // block_size + 1
    cache, values = _cache(blocks, 6, cuda, block_size, pad)
    q, idx = _query(3, 32, 6, cuda), _indices(3, 256, blocks * block_size, 6, cuda)
    o, lse = ops.sparse_mla_decode_fp4(q, cache, idx, SCALE)
    torch.cuda.synchronize()
    _check(o, lse, q, values, idx, SCALE)


def test_strided_query_indices_and_given_outputs(cuda):
    cache, values = _cache(40, 7, cuda)
    q = _query(4, 128, 7, cuda).view(4, 2, 64, 576)[:, 1]                       # 64 of 128 heads
    idx = torch.nn.functional.pad(_indices(4, 512, 2560, 7, cuda), (3, 5), value=1)[:, 3:515]
    o = torch.empty(4, 64, 512, dtype=torch.bfloat16, device=cuda)
    lse = torch.empty(4, 64, device=cuda)
    got = ops.sparse_mla_decode_fp4(q, cache, idx, SCALE, out=o, lse=lse)
    torch.cuda.synchronize()
    assert got[0] is o and got[1] is lse
    _check(o, lse, q, values, idx, SCALE)


def test_scale_bytes_far_apart(cuda):
    """Rows whose blocks differ by up to 2^40 in size, and rows of zeros."""
    g = torch.Generator(device=cuda).manual_seed(8)
    kv = torch.randn(2560, 576, generator=g, device=cuda)
    kv[:, :512] *= torch.exp2(torch.randint(-20, 6, (2560, 16), generator=g, device=cuda).float()).repeat_interleave(32, 1)
    kv[::7, :512] = 0
    rows = F.mla_rows(kv.to(torch.bfloat16))
    q, idx = _query(3, 64, 8, cuda), _indices(3, 512, 2560, 8, cuda)
    o, lse = ops.sparse_mla_decode_fp4(q, rows.view(40, 64, 400), idx, 0.002)
    torch.cuda.synchronize()
    _check(o, lse, q, F.mla_values(rows), idx, 0.002)


def test_nan_rows(cuda):
    """A NaN in a selected row makes its token's outputs NaN; in a row that no token selects, or behind a skipped
    index, it does nothing."""
    cache, values = _cache(40, 9, cuda)
    idx = torch.stack([torch.arange(0, 256), torch.arange(1000, 1256), torch.arange(0, 256)]).to(torch.int32).to(cuda)
    idx[2, 17] = -1
    cache[0, 17, 0, 256 + 3] = 255                  # slot 17: selected by token 0 only
    cache[30, 1, 0, 256 + 3] = 255                  # by none
    q = _query(3, 128, 9, cuda)
    for splits in (1, 4):
        o, lse = ops.sparse_mla_decode_fp4(q, cache, idx, SCALE, num_splits=splits)
        torch.cuda.synchronize()
        assert torch.all(torch.isnan(o[0])) and torch.all(torch.isnan(lse[0]))
        _check(o[1:], lse[1:], q[1:], values, idx[1:], SCALE)


@pytest.mark.parametrize("H", [16, 32, 128])
def test_repeated_and_unordered_slots(cuda, H):
    """A slot listed twice counts twice; the order of a row's slots changes nothing but rounding."""
    cache, values = _cache(40, 10, cuda)
    q = _query(2, H, 10, cuda)
    idx = torch.randint(0, 300, (2, 512), device=cuda).to(torch.int32)
    o, lse = ops.sparse_mla_decode_fp4(q, cache, idx, SCALE)
    torch.cuda.synchronize()
    _check(o, lse, q, values, idx, SCALE)


def test_cache_past_4_gib(cuda):
    """Rows behind 2^32 bytes of cache are written, read back and attended over."""
    blocks = 2 ** 32 // (65 * 400) + 70
    cache = torch.zeros(blocks, 65, 1, 400, dtype=torch.uint8, device=cuda)[:, :64]
    slots = torch.cat([torch.arange(96), torch.arange(blocks * 64 - 160, blocks * 64)]).to(cuda)
    kv = torch.randn(256, 576, device=cuda).to(torch.bfloat16)
    ops.mla_kv_store_fp4(kv, cache, slots)
    assert torch.equal(cache[blocks - 2, 5, 0], F.mla_rows(kv[96 + 160 - 128 + 5:][:1])[0])
    values = F.mla_values(F.mla_rows(kv))
    assert torch.equal(ops.mla_kv_load_fp4(cache, slots).double(), values)
    q = _query(2, 64, 11, cuda)
    at = torch.stack([torch.randperm(256, device=cuda), torch.randperm(256, device=cuda)])
    o, lse = ops.sparse_mla_decode_fp4(q, cache, slots[at].to(torch.int32), SCALE)
    torch.cuda.synchronize()
    _check(o, lse, q, values, at, SCALE)


def test_workspace_of_the_caller(cuda):
    """A caller's workspace is used as it is, a small or unaligned one replaced; outputs of one token from a
    larger tensor."""
    cache, values = _cache(40, 12, cuda)
    q, idx = _query(3, 128, 12, cuda)[1:2], _indices(1, 2048, 2560, 12, cuda)
    need = ops.sparse_mla_workspace_bytes(1, 128, 8)
    for ws in (torch.empty(need, dtype=torch.uint8, device=cuda), torch.empty(need + 5, dtype=torch.uint8, device=cuda)[5:],
               torch.empty(64, dtype=torch.uint8, device=cuda)):
        o, lse = ops.sparse_mla_decode_fp4(q, cache, idx, SCALE, num_splits=8, workspace=ws)
        torch.cuda.synchronize()
        _check(o, lse, q, values, idx, SCALE)


def _group_batch(H, group):
    """The largest batch that is taken, unsplit, in head groups of 16 (group 0) or 32 (1); one in groups of 64 (2)."""
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    return (cus // -(-H // 16), cus // -(-H // 32), cus // -(-H // 32) + 1)[group]


@pytest.mark.parametrize("group", [0, 1, 2])
@pytest.mark.parametrize("H", [128, 112, 48])
def test_masks_in_every_head_group(cuda, group, H):
    """The rows of the mask and NaN tests at both ends of a batch of either head group, no output outside
    the batch touched."""
    T = _group_batch(H, group)
    print(f"mla fp4 head groups T={T} H={H}", flush=True)
    cache, values = _cache(40, 13, cuda)
    q, idx = _query(T, H, 13, cuda), _indices(T, 512, 2559, 13, cuda)
    for at in (0, T - 7):
        idx[at] = -1                                # nothing
        idx[at + 1, 1:] = -1                        # one key, the first
        idx[at + 2, :511] = -1                      # one key, the last
        idx[at + 3, :32] = -1                       # no key in the first half of the first block
        idx[at + 4, 40:] = 10 ** 6                  # stale slots past the cache
        idx[at + 5, ::2] = -5
        idx[at + 6, 77] = 2559
    cache[39, 63, 0, 256 + 15] = 255                # slot 2559: a NaN row, selected by tokens 6 and T - 1
    outs = torch.full((T + 2, H, 512), 7.0, dtype=torch.bfloat16, device=cuda)
    lses = torch.full((T + 2, H), 7.0, device=cuda)
    for splits in (1, 2):
        o, lse = ops.sparse_mla_decode_fp4(q, cache, idx, SCALE, out=outs[1:-1], lse=lses[1:-1], num_splits=splits)
        torch.cuda.synchronize()
        assert torch.all(outs[::T + 1] == 7) and torch.all(lses[::T + 1] == 7)
        for t in (6, T - 1):
            assert torch.all(torch.isnan(o[t])) and torch.all(torch.isnan(lse[t]))
        rest = [t for t in range(T) if t not in (6, T - 1)]
        _check(o[rest], lse[rest], q[rest], values, idx[rest], SCALE)


@pytest.mark.parametrize("group", [0, 1, 2])
@pytest.mark.parametrize("order", ["rising", "falling"])
def test_far_apart_scores_in_every_head_group(cuda, group, order):
    T, H, K = _group_batch(128, group), 128, 512
    cache, values = _cache(40, 14, cuda, spread=0.5)
    q, idx = _query(T, H, 14, cuda), _indices(T, K, 2560, 14, cuda)
    s = (values[idx.long()] @ q[:, 0].double()[..., None]).squeeze(-1)
    by = s.argsort(dim=1, descending=order == "falling")
    if order == "falling":
        by = torch.stack([by[:, :K // 2].view(T, -1, 32), by[:, K // 2:].flip(1).view(T, -1, 32)], dim=2).view(T, K)
    idx = idx.gather(1, by)
    o, lse = ops.sparse_mla_decode_fp4(q, cache, idx, 1.0, num_splits=1)
    torch.cuda.synchronize()
    _check(o, lse, q, values, idx, 1.0)


@pytest.mark.parametrize("group", [0, 1, 2])
def test_scale_bytes_in_every_head_group(cuda, group):
    g = torch.Generator(device=cuda).manual_seed(15)
    kv = torch.randn(2560, 576, generator=g, device=cuda)
    kv[:, :512] *= torch.exp2(torch.randint(-20, 6, (2560, 16), generator=g, device=cuda).float()).repeat_interleave(32, 1)
    kv[::7, :512] = 0
    rows = F.mla_rows(kv.to(torch.bfloat16))
    T = _group_batch(128, group)
    q, idx = _query(T, 128, 15, cuda), _indices(T, 512, 2560, 15, cuda, 0.05)
    o, lse = ops.sparse_mla_decode_fp4(q, rows.view(40, 64, 400), idx, 0.002, num_splits=1)
    torch.cuda.synchronize()
    _check(o, lse, q, F.mla_values(rows), idx, 0.002)
