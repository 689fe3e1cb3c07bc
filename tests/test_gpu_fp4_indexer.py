"""Indexer logits over the 4-bit pages on the GPU, against float64 with the oracle's bound."""
import pytest
import torch

from nanoengine_amd import ops
from oracle import fp4_oracle as F

pytestmark = pytest.mark.gpu


def _case(lens, n, seed, device, spare=2, exps=0):
    """Queries, head weights, pages in a shuffled pool, tables, and the pool's values [pages * 64, 128]."""
    g = torch.Generator(device=device).manual_seed(seed)
    B = len(lens)
    need = [-(-L // 64) for L in lens]
    M = max(max(need), 1) + spare
    pool = torch.randperm(sum(need) + 3, generator=g, device=device).to(torch.int32)
    bt = torch.full((B, M), -1, dtype=torch.int32, device=device)
    at = 0
    for b, p in enumerate(need):
        bt[b, :p] = pool[at:at + p]
        at += p
    k = torch.randn(pool.numel() * 64, 128, generator=g, device=device)
    if exps:
        k = k * torch.exp2(torch.randint(-exps, exps, (k.shape[0], 4), generator=g, device=device).float()
                           ).repeat_interleave(32, dim=1)
    cache = F.key_pages(k.to(torch.bfloat16))
    q = (torch.randn(B, n, 64, 128, generator=g, device=device) * 60).to(torch.float8_e4m3fn)
    w = torch.randn(B * n, 64, generator=g, device=device) * 0.01
    ctx = torch.tensor(lens, device=device)[:, None] - torch.arange(n - 1, -1, -1, device=device)
    return q, w, cache, bt, ctx.clamp(min=0).to(torch.int32), F.key_values(cache)


def _keys(values, bt_row, L):
    t = torch.arange(L, device=values.device)
    return values[bt_row.long()[t // 64] * 64 + t % 64]


def _check(got, q, w, bt, ctx, values, max_len):
    B, n = ctx.shape
    for b in range(B):
        for j in range(n):
            L, r = min(int(ctx[b, j]), max_len), b * n + j
            want, tol = F.logits_row(q[b, j].float(), w[r], _keys(values, bt[b], L))
            assert torch.all((got[r, :L].double() - want).abs() <= tol), (r, L)
            assert torch.all(torch.isneginf(got[r, L:max_len]))


@pytest.mark.parametrize("lens,n", [([1], 1), ([64], 2), ([63, 65, 0, 128], 1), ([1, 2, 700], 2), ([5000] * 3, 1),
                                    ([20000, 17, 3001, 1], 2), ([200] * 70, 1), ([131], 1)])
def test_matches_float64(cuda, lens, n):
    print(f"index fp4 lens={lens[:4]} n={n}", flush=True)
    q, w, cache, bt, ctx, values = _case(lens, n, len(lens) * 7 + n, cuda)
    max_len = max(max(lens), 1)
    got = ops.indexer_logits_fp4(q, cache, w, ctx, bt, max_len)
    torch.cuda.synchronize()
    assert got.shape == (len(lens) * n, max_len)
    _check(got, q, w, bt, ctx, values, max_len)


@pytest.mark.parametrize("clean", [True, False])
def test_padding_and_row_strides(cuda, clean):
    """A wider output: with clean_logits -inf to max_context_len, else to the end of the last page; never behind."""
    q, w, cache, bt, ctx, values = _case([70, 500, 1], 2, 3, cuda, spare=6)
    max_len = 701
    store = torch.full((6, 900), 5.0, device=cuda)
    got = ops.indexer_logits_fp4(q, cache, w, ctx, bt, max_len, out=store[:, :max_len], clean_logits=clean)
    torch.cuda.synchronize()
    assert torch.all(store[:, max_len:] == 5)
    if clean:
        _check(got, q, w, bt, ctx, values, max_len)
    else:
        for r, L in enumerate(ctx.view(-1).tolist()):
            longest = int(ctx[r // 2].max())
            end = min(-(-longest // 64) * 64, max_len)
            _check(got[r:r + 1, :end], q[r // 2, r % 2][None, None], w[r:r + 1], bt[r // 2][None], ctx.view(-1, 1)[r:r + 1],
                   values, end)
            assert torch.all(got[r, end:] == 5)


def test_lengths_past_max_context_len(cuda):
    q, w, cache, bt, ctx, values = _case([400, 130], 1, 4, cuda)
    got = ops.indexer_logits_fp4(q, cache, w, ctx, bt, 200)
    torch.cuda.synchronize()
    _check(got, q, w, bt, ctx, values, 200)


def test_bad_pages_score_minus_infinity(cuda):
    q, w, cache, bt, ctx, values = _case([300, 300], 1, 5, cuda)
    ref = ops.indexer_logits_fp4(q, cache, w, ctx, bt, 300)
    bt[0, 1], bt[0, 3], bt[1, 4] = -1, cache.shape[0], 10 ** 9
    got = ops.indexer_logits_fp4(q, cache, w, ctx, bt, 300)
    torch.cuda.synchronize()
    bad = torch.zeros(2, 300, dtype=torch.bool, device=cuda)
    bad[0, 64:128] = bad[0, 192:256] = bad[1, 256:] = True
    assert torch.all(torch.isneginf(got[bad])) and torch.equal(got[~bad], ref[~bad])


def test_blocks_of_different_size_and_nan_keys(cuda):
    q, w, cache, bt, ctx, values = _case([900], 2, 6, cuda, exps=12)
    got = ops.indexer_logits_fp4(q, cache, w, ctx, bt, 900)
    torch.cuda.synchronize()
    _check(got, q, w, bt, ctx, values, 900)
    page = int(bt[0, 2])
    cache[page, 64 * 64 + 4 * 5 + 1] = 255          # key 133's second block
    again = ops.indexer_logits_fp4(q, cache, w, ctx, bt, 900)
    torch.cuda.synchronize()
    assert torch.all(torch.isnan(again[:, 133]))
    keep = torch.arange(900, device=cuda) != 133
    assert torch.equal(again[:, keep], got[:, keep])


def test_cache_past_4_gib(cuda):
    """Pages behind 2^32 bytes of cache are written, read back and scored."""
    pages = 2 ** 32 // (64 * 68) + 40
    cache = torch.zeros(pages, 64 * 68, dtype=torch.uint8, device=cuda)
    slots = torch.arange(pages * 64 - 300, pages * 64, device=cuda)
    key = torch.randn(300, 128, device=cuda).to(torch.bfloat16)
    ops.indexer_k_store_fp4(key, cache, slots, 64)
    values = F.fp4_values(*F.fp4_quantize(key.float()))
    keys, s = ops.indexer_k_load_fp4(cache, slots, 64)
    assert torch.equal(keys.double() * s.double()[:, None], values)
    bt = torch.arange(pages - 4, pages, device=cuda, dtype=torch.int32)[None]
    q = (torch.randn(1, 1, 64, 128, device=cuda) * 60).to(torch.float8_e4m3fn)
    w = torch.randn(1, 64, device=cuda)
    got = ops.indexer_logits_fp4(q, cache, w, torch.tensor([[256]], device=cuda), bt, 256)
    torch.cuda.synchronize()
    want, tol = F.logits_row(q[0, 0].float(), w[0], values[300 - 256:])
    assert torch.all((got[0].double() - want).abs() <= tol)


@pytest.mark.parametrize("n", [1, 2])
def test_more_entries_than_a_launch_takes(cuda, n):
    """Past 4096 entries the batch goes in several launches; one table row serves every entry (row stride 0)."""
    B = 4097 + 4096
    q1, w1, cache, bt, _, values = _case([130], n, 8, cuda)
    g = torch.Generator().manual_seed(8)
    ctx = torch.randint(0, 131, (B, n), generator=g).to(torch.int32).to(cuda)
    q = q1.view(torch.uint8).expand(B, n, 64, 128).contiguous()
    got = ops.indexer_logits_fp4(q, cache, w1.repeat(B, 1), ctx, bt.expand(B, -1), 130)
    torch.cuda.synchronize()
    for j in range(n):
        want, tol = F.logits_row(q1[0, j].float(), w1[j], _keys(values, bt[0], 130))
        rows, L = got[j::n], ctx[:, j:j + 1]
        inside = torch.arange(130, device=cuda)[None] < L
        assert torch.all(((rows.double() - want).abs() <= tol) | ~inside)
        assert torch.all(torch.isneginf(rows) | inside)


def test_negative_lengths_and_wide_tables(cuda):
    q, w, cache, bt, ctx, values = _case([200, 64, 129], 1, 9, cuda, spare=40)
    ctx[1] = -5
    got = ops.indexer_logits_fp4(q, cache, w, ctx.view(-1), bt, bt.shape[1] * 64)
    torch.cuda.synchronize()
    _check(got, q, w, bt, ctx.clamp(min=0), values, bt.shape[1] * 64)
