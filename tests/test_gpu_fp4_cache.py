"""Writers and readers of the 4-bit caches on the GPU, byte for byte against the oracle."""
import pytest
import torch

from nanoengine_amd import ops
from oracle import fp4_oracle as F

pytestmark = pytest.mark.gpu


def _rows(n, width, seed, device):
    """bf16 rows of very different size, with zeros, the largest and the smallest values."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, width, generator=g) * torch.exp2(torch.randint(-30, 30, (n, width // 32), generator=g)
                                                        .float()).repeat_interleave(32, dim=1)
    x[0, :32] = 0
    x[0, 32:64] = torch.linspace(-7, 7, 32)
    x[-1, 0], x[-1, 33], x[-1, 70], x[-1, 96:128] = 3.3895e38, float("inf"), -3.3e38, 1e-38
    return x.to(torch.bfloat16).to(device)


def _slots(n, total, seed, dtype, device):
    """Distinct slots, some negative and some past the cache."""
    g = torch.Generator().manual_seed(seed)
    s = torch.randperm(total, generator=g)[:n]
    if n > 4:
        s[1], s[3] = -1, total + 5
        s[4] = -9
    return s.to(dtype).to(device)


def _kept(slots, total):
    ok = (slots >= 0) & (slots < total)
    return ok, slots[ok].long()


@pytest.mark.parametrize("n,slot_dtype,block_size", [(1, torch.int64, 64), (5, torch.int32, 64), (67, torch.int64, 48),
                                                     (300, torch.int32, 1)])
def test_mla_store_and_load(cuda, n, slot_dtype, block_size):
    print(f"mla store n={n} block={block_size}", flush=True)
    blocks = 2 * n // block_size + 3
    kv = _rows(n, 576, n, cuda)
    padded = torch.full((blocks, block_size + 1, 1, 400), 7, dtype=torch.uint8, device=cuda)
    cache = padded[:, :block_size]
    slots = _slots(n, blocks * block_size, n, slot_dtype, cuda)
    ops.mla_kv_store_fp4(kv, cache, slots)
    ok, at = _kept(slots, blocks * block_size)
    flat = cache.reshape(-1, 400)
    want = torch.full_like(flat, 7)
    want[at] = F.mla_rows(kv)[ok]
    assert torch.equal(flat, want)                  # written rows, and no other byte
    assert torch.all(padded[:, block_size] == 7)
    back = ops.mla_kv_load_fp4(cache, slots)
    exact = torch.zeros(n, 576, dtype=torch.float64, device=cuda)
    exact[ok] = F.mla_values(want[at])
    assert torch.equal(back.double(), exact) and torch.all(back[~ok] == 0)


@pytest.mark.parametrize("n,slot_dtype,page_size", [(1, torch.int32, 64), (5, torch.int64, 64), (35, torch.int32, 16),
                                                    (1001, torch.int64, 64)])
def test_index_store_and_load(cuda, n, slot_dtype, page_size):
    print(f"index store n={n} page={page_size}", flush=True)
    pages = 2 * n // page_size + 3
    key = _rows(n, 128, n + 1, cuda)
    cache = torch.full((pages, page_size * 68), 7, dtype=torch.uint8, device=cuda)
    slots = _slots(n, pages * page_size, n, slot_dtype, cuda)
    ops.indexer_k_store_fp4(key, cache, slots, page_size)
    ok, at = _kept(slots, pages * page_size)
    codes, scales = F.fp4_quantize(key.float())
    want = torch.full_like(cache, 7)
    wc, ws = want[:, :page_size * 64].unflatten(1, (page_size, 64)), want[:, page_size * 64:].unflatten(1, (page_size, 4))
    wc[at // page_size, at % page_size] = codes[ok]
    ws[at // page_size, at % page_size] = scales[ok]
    assert torch.equal(cache, want)
    keys, s = ops.indexer_k_load_fp4(cache, slots, page_size)
    v = F.fp4_values(codes, scales)
    # the scale is a power of two under the key's largest block's, the key is the value over it, rounded to e4m3
    top = scales.double().amax(dim=1)
    want_s = torch.where(ok, torch.exp2(torch.clamp(top, min=7) - 133), 2.0 ** -126)
    assert torch.equal(s.double(), want_s)
    want_k = torch.where(ok[:, None], (v / want_s[:, None]).float(), 0.0).to(torch.float8_e4m3fn)
    assert torch.equal(keys.float(), want_k.float())


def test_strided_rows_and_outputs(cuda):
    wide = torch.randn(9, 2, 640, device=cuda).to(torch.bfloat16)
    kv = wide[:, 1, 64:]                            # rows 1280 apart, 128 bytes in
    cache = torch.zeros(3, 16, 400, dtype=torch.uint8, device=cuda)
    slots = torch.arange(20, 29, device=cuda)
    ops.mla_kv_store_fp4(kv, cache, slots)
    assert torch.equal(cache.view(-1, 400)[20:29], F.mla_rows(kv.contiguous()))
    out = torch.full((9, 600), 3.0, dtype=torch.bfloat16, device=cuda)
    ops.mla_kv_load_fp4(cache, slots, out=out[:, :576])
    assert torch.equal(out[:, :576].double(), F.mla_values(cache.view(-1, 400)[20:29])) and torch.all(out[:, 576:] == 3)
    key = wide[:, 0, 128:256]
    pages = torch.zeros(1, 64 * 68, dtype=torch.uint8, device=cuda)
    ops.indexer_k_store_fp4(key, pages, slots, 64)
    assert torch.equal(pages.view(-1)[20 * 64:29 * 64].view(9, 64), F.fp4_quantize(key.float())[0])


def test_nan_blocks(cuda):
    kv = torch.randn(2, 576, device=cuda).to(torch.bfloat16)
    kv[0, 40] = float("nan")
    kv[1, 575] = float("nan")                       # the rope is bf16: kept as it is
    cache = torch.zeros(1, 64, 400, dtype=torch.uint8, device=cuda)
    slots = torch.tensor([3, 5], device=cuda)
    ops.mla_kv_store_fp4(kv, cache, slots)
    back = ops.mla_kv_load_fp4(cache, slots)
    nan = torch.isnan(back)
    assert torch.all(nan[0, 32:64]) and nan[0].sum() == 32 and nan[1].nonzero().tolist() == [[575]]
    assert torch.equal(cache[0, 3, :256], F.mla_rows(kv)[0, :256])
    key = torch.ones(1, 128, device=cuda, dtype=torch.bfloat16)
    key[0, 64] = float("nan")
    pages = torch.zeros(1, 64 * 68, dtype=torch.uint8, device=cuda)
    ops.indexer_k_store_fp4(key, pages, slots[:1], 64)
    keys, s = ops.indexer_k_load_fp4(pages, slots[:1], 64)
    assert s.item() == 2.0 ** (-2 - 6)              # from the finite blocks: 1 = 4 * 2^-2
    v = keys.float()[0] * s
    assert torch.all(torch.isnan(v[64:96])) and torch.all(v[:64] == 1) and torch.all(v[96:] == 1)


def test_empty_calls(cuda):
    cache = torch.zeros(2, 64, 400, dtype=torch.uint8, device=cuda)
    pages = torch.zeros(2, 64 * 68, dtype=torch.uint8, device=cuda)
    none = torch.zeros(0, dtype=torch.int64, device=cuda)
    ops.mla_kv_store_fp4(torch.zeros(0, 576, dtype=torch.bfloat16, device=cuda), cache, none)
    ops.indexer_k_store_fp4(torch.zeros(0, 128, dtype=torch.bfloat16, device=cuda), pages, none, 64)
    assert ops.mla_kv_load_fp4(cache, none).shape == (0, 576)
    assert ops.indexer_k_load_fp4(pages, none, 64)[0].shape == (0, 128)
    torch.cuda.synchronize()
    assert not cache.any() and not pages.any()
