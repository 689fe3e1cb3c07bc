"""The 4-bit caches and batch tables without a GPU: the oracle's format against known
answers, and the refusals of the entry points."""
import ctypes

import pytest
import torch

from nanoengine_amd import _lib, ops
from oracle import fp4_oracle as F

ONE = ctypes.c_void_p(16)   # a non-null, aligned address that is never dereferenced
ODD = ctypes.c_void_p(18)
P = None


# ------------------------------------------------------------------ format
def test_codes_of_a_unit_block():
    x = torch.zeros(1, 32)
    x[0, :16] = torch.tensor([6, -6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, 0.26, 4.9, 5.1, -1.5, 3, -0.0])
    codes, scale = F.fp4_quantize(x)
    assert scale.tolist() == [[127]]
    want = [7, 15, 0, 2, 2, 4, 4, 6, 6, 8, 1, 6, 7, 11, 5, 8] + [0] * 16
    assert codes[0].tolist() == [want[2 * i] | want[2 * i + 1] << 4 for i in range(16)]


@pytest.mark.parametrize("amax,byte", [(0.0, 87), (6.0, 127), (6.0625, 128), (3.0, 126), (3.015625, 127),
                                       (2.0 ** -45, 87), (3.3895e38, 252), (float("inf"), 252)])
def test_scale_byte(amax, byte):
    x = torch.zeros(1, 32)
    x[0, 5] = -torch.tensor(amax).to(torch.bfloat16).float()
    assert F.fp4_quantize(x)[1].item() == byte


def test_round_trip_is_within_half_a_step():
    x = torch.randn(64, 128, generator=torch.Generator().manual_seed(0)) * torch.logspace(-3, 3, 64)[:, None]
    codes, scale = F.fp4_quantize(x)
    k = torch.exp2(scale.double() - 127).repeat_interleave(32, dim=1)
    err = (F.fp4_values(codes, scale) - x.double()).abs()
    # the widest half step of the grid is 1 (between 4 and 6); relative to the value, half a mantissa bit
    assert torch.all(err <= torch.maximum(0.25 * k, x.double().abs() * 0.25))
    assert torch.all(err <= k)


def test_nan_blocks_have_zero_codes():
    x = torch.ones(1, 64)
    x[0, 40] = float("nan")
    codes, scale = F.fp4_quantize(x)
    assert scale.tolist() == [[125, 255]] and torch.all(codes[0, 16:] == 0)
    v = F.fp4_values(codes, scale)
    assert torch.all(v[0, :32] == 1) and torch.all(torch.isnan(v[0, 32:]))


def test_row_sizes():
    assert (ops.MLA_FP4_ROW_BYTES, ops.INDEXER_FP4_ROW_BYTES) == (F.MLA_ROW, F.KEY_BYTES)
    assert F.mla_rows(torch.ones(3, 576, dtype=torch.bfloat16)).shape == (3, 400)
    assert F.key_pages(torch.ones(128, 128)).shape == (2, 4352)


def test_tables_known_answer():
    t, slots, pos, seq, cu_q, cu_k, st = F.batch_tables([3, 0, 8], [2, 5, 1], [[7, 0, 0], [0, 0, 0], [5, 6, 0]], 4, 10,
                                                        free=[9, 8, 4, 2], head=0)
    assert t == [[7, 9, 0], [8, 4, 0], [5, 6, 2]]
    assert slots == [31, 36, 32, 33, 34, 35, 16, 8, -1, -1]
    assert pos == [3, 4, 0, 1, 2, 3, 4, 8, 0, 0] and seq[:8] == [4, 5, 1, 2, 3, 4, 5, 9]
    assert cu_q == [0, 2, 7, 8] and cu_k == [0, 5, 10, 19] and st == [0, 8, 4, 9]


# ------------------------------------------------------------------ refusals of the C entry points
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


def test_writer_and_reader_refusals(lib):
    _bad(lib, "dsa_mla_kv_store_fp4", [ONE, 576, ONE, 0, 4, ONE, 64 * 400, 64, 8, P],
         [(0, P, 1), (2, P, 1), (5, P, 1), (0, ODD, 1), (5, ODD, 1), (1, 577, 1), (6, 64 * 400 - 16, 1),
          (6, 64 * 400 + 8, 1), (7, 0, 1), (8, -1, 1), (4, -1, 1), (4, 0, 0)])
    _bad(lib, "dsa_mla_kv_load_fp4", [ONE, 64 * 400, 64, 8, ONE, 0, 4, ONE, 576, P],
         [(0, P, 1), (4, P, 1), (7, P, 1), (7, ODD, 1), (8, 568, 1), (8, 580, 1), (1, 100, 1), (2, 0, 1), (6, 0, 0)])
    _bad(lib, "dsa_indexer_k_store_fp4", [ONE, 128, ONE, 0, 4, ONE, 64, 8, P],
         [(0, P, 1), (2, P, 1), (5, P, 1), (0, ODD, 1), (5, ODD, 1), (1, 132, 1), (6, 0, 1), (7, -1, 1), (4, 0, 0)])
    _bad(lib, "dsa_indexer_k_load_fp4", [ONE, 64, 8, ONE, 0, 4, ONE, ONE, P],
         [(0, P, 1), (3, P, 1), (6, P, 1), (7, P, 1), (6, ODD, 1), (1, 0, 1), (2, -1, 1), (5, -1, 1), (5, 0, 0)])


def test_attention_and_logits_refusals(lib):
    f = ctypes.c_float(0.1)
    args = [ONE, 128 * 576, 576, ONE, 64 * 400, 64, 8, ONE, 2048, 2, 128, 2048, f, ONE, ONE, 1, P, 0, P]
    _bad(lib, "dsa_sparse_mla_decode_fp4", args,
         [(0, P, 1), (3, P, 1), (7, P, 1), (13, P, 1), (0, ODD, 1), (3, ODD, 1), (13, ODD, 1), (1, 4, 1), (2, 580, 1),
          (4, 64 * 400 - 16, 1), (4, 64 * 400 + 8, 1), (5, 0, 1), (6, -1, 1), (9, -1, 2), (10, 24, 2), (10, 0, 2),
          (11, 100, 2), (11, 0, 2), (9, 0, 0), (12, ctypes.c_float(-1), 1), (12, ctypes.c_float(float("nan")), 1),
          (12, ctypes.c_float(float("inf")), 1), (16, ODD, 1), (15, 4, 4)])
    args = [ONE, ONE, 8, ONE, ONE, ONE, 4, 2, 1, 64, 128, 64, 256, ONE, 256, 1, P]
    _bad(lib, "dsa_indexer_logits_fp4", args,
         [(0, P, 1), (1, P, 1), (3, P, 1), (4, P, 1), (5, P, 1), (13, P, 1), (0, ODD, 1), (1, ODD, 1), (2, -1, 1),
          (7, -1, 1), (8, 3, 2), (8, 0, 2), (9, 32, 2), (10, 64, 2), (11, 128, 2), (12, -1, 1), (14, 255, 1), (7, 0, 0),
          (12, 0, 0)])


def test_tables_refusals(lib):
    args = [ONE, ONE, 2, ONE, 4, 4, 64, ONE, 8, P, ONE, 0, P, 0, P, 10, P, P, 0, ONE, P]
    _bad(lib, "dsa_batch_tables", args,
         [(0, P, 1), (1, P, 1), (3, P, 1), (10, P, 1), (19, P, 1), (2, -1, 1), (2, 8193, 2), (4, 3, 1), (5, -1, 1),
          (6, 0, 1), (8, -1, 1), (15, -1, 1), (8, 2 ** 31, 2), (15, 2 ** 31, 2)])


# ------------------------------------------------------------------ refusals of the tensor adapters
def test_adapters_refuse_bad_tensors():
    bf, u8 = torch.bfloat16, torch.uint8
    cache = torch.zeros(4, 65, 1, 400, dtype=u8)[:, :64]
    assert ops.mla_fp4_geometry(cache) == (65 * 400, 64)
    pages = torch.zeros(4, 64 * 68, dtype=u8)
    kv, key, slots = torch.zeros(3, 576, dtype=bf), torch.zeros(3, 128, dtype=bf), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="400"):
        ops.mla_kv_store_fp4(kv, torch.zeros(4, 64, 1, 656, dtype=u8), slots)
    with pytest.raises(RuntimeError, match="apart"):
        ops.mla_kv_store_fp4(kv, torch.zeros(4, 64, 2, 400, dtype=u8)[:, :, :1], slots)
    with pytest.raises(RuntimeError, match="kv must be"):
        ops.mla_kv_store_fp4(kv.float(), cache, slots)
    with pytest.raises(RuntimeError, match="slot_mapping"):
        ops.mla_kv_store_fp4(kv, cache, slots[:2])
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.mla_kv_store_fp4(kv, cache, slots)
    with pytest.raises(RuntimeError, match="slot_mapping"):
        ops.mla_kv_load_fp4(cache, slots.float())
    with pytest.raises(RuntimeError, match="pages of page_size"):
        ops.indexer_k_store_fp4(key, torch.zeros(4, 64 * 132 + 1, dtype=u8), slots, 64)
    with pytest.raises(RuntimeError, match="pages of page_size"):
        ops.indexer_k_load_fp4(pages, slots, 0)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.indexer_k_load_fp4(pages, slots, 64)
    q = torch.zeros(2, 16, 576, dtype=bf)
    idx = torch.zeros(2, 64, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="q must be"):
        ops.sparse_mla_decode_fp4(q.float(), cache, idx, 1.0)
    with pytest.raises(RuntimeError, match="indices"):
        ops.sparse_mla_decode_fp4(q, cache, idx.long(), 1.0)
    with pytest.raises(RuntimeError, match="400"):
        ops.sparse_mla_decode_fp4(q, torch.zeros(4, 64, 1, 656, dtype=u8), idx, 1.0)
    qi, w = torch.zeros(2, 1, 64, 128, dtype=u8), torch.zeros(2, 64)
    lens, bt = torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="too narrow"):
        ops.indexer_logits_fp4(qi, pages, w, lens, bt, 129)
    with pytest.raises(RuntimeError, match="weights"):
        ops.indexer_logits_fp4(qi, pages, w[:1], lens, bt, 128)
    with pytest.raises(RuntimeError, match="context_lens"):
        ops.indexer_logits_fp4(qi, pages, w, lens[:1], bt, 128)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.indexer_logits_fp4(qi, pages, w, lens, bt, 128)


def test_tables_adapter_refuses_bad_tensors():
    i32 = torch.int32
    lens, bt = torch.zeros(2, dtype=i32), torch.zeros(2, 3, dtype=i32)
    slots, status = torch.zeros(5, dtype=i32), torch.zeros(4, dtype=torch.int64)
    for kw, match in (({"cached_lens": lens.long()}, "cached_lens"), ({"new_lens": lens[:1]}, "new_lens"),
                      ({"block_tables": bt[:1]}, "block_tables"), ({"block_tables": bt[:1].expand(2, 3)}, "overlap"),
                      ({"slot_mapping": slots.float()}, "slot_mapping"), ({"status": status[:3]}, "status"),
                      ({"positions": slots[:4]}, "positions"), ({"seq_lens": slots.long()}, "seq_lens"),
                      ({"cu_seqlens_q": slots}, "cu_seqlens_q"), ({"free_blocks": bt}, "free_blocks"),
                      ({"free_head": lens}, "free_head"), ({}, "GPU only"),
                      ({"cu_seqlens_q": slots[:3], "cu_seqlens_k": slots[:3].long()}, "share one dtype")):
        args = dict(cached_lens=lens, new_lens=lens, block_tables=bt, page_size=64, slot_mapping=slots, status=status)
        with pytest.raises(RuntimeError, match=match):
            ops.batch_tables(**{**args, **kw})
    with pytest.raises(ValueError, match="page_size"):
        ops.batch_tables(lens, lens, bt, 0, slots, status)


# ------------------------------------------------------------------ the classes around them
def test_cache_class_checks():
    from nanoengine_amd import indexer
    c = indexer.IndexerCacheFp4(2, 16, 64, device="cpu")
    assert c.bytes_per_token == 68 and c.get_buffer(1).shape == (16, 64 * 68) and len(c.buffers) == 2
    with pytest.raises(ValueError, match="128-dim"):
        indexer.IndexerCacheFp4(1, 4, 64, 64, device="cpu")
    with pytest.raises(ValueError, match="uint8"):
        indexer.IndexerCacheFp4(1, 4, 64, device="cpu", buffer=torch.zeros(1, 4, 64 * 132, dtype=torch.uint8))


def test_step_refuses_an_unknown_format():
    from nanoengine_amd.pipeline import DsaDecodeStep
    with pytest.raises(ValueError, match="indexer_format"):
        DsaDecodeStep(1, 1, 64, device="cpu", indexer_format="int4")


def test_batch_tables_report_their_faults():
    from nanoengine_amd.batch_tables import BatchTables
    t = BatchTables(3, 5, 4, device="cpu")
    t.status.copy_(torch.tensor([0, 5, 2, 77]))
    assert t.check() == (5, 2, 77)
    t.status[0] = 2 | 8
    with pytest.raises(RuntimeError, match="more pages than its block table; more new tokens than rows"):
        t.check()
    with pytest.raises(ValueError, match="cannot hold 2 tokens of 3"):
        t.context_fields(2)
    t.seq_lens.copy_(torch.tensor([9, 4, 0, 0, 0]))
    fields = t.context_fields()
    assert fields["context_lens"].tolist() == [[9, 4, 0]] and fields["block_tables"].shape == (1, 3, 4)
    with pytest.raises(RuntimeError, match="GPU only"):
        t.plan(torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
