"""The indexer key writers and readers refuse pages of the other format, whatever the number of pages.

Both formats are uint8 pages. 33 pages of 64 4-bit keys are as many bytes as 17 fp8 pages: taken as those, an
fp8 writer would write slots of the last 4-bit pages past the end. All of this is refused before anything is launched,
so the tensors are on the CPU."""
import pytest
import torch

from nanoengine_amd import indexer, indexer_transform, ops

BF, U8 = torch.bfloat16, torch.uint8


def _slots(n):
    return torch.arange(n, dtype=torch.int64)


def _store(cache, page_size=64):
    ops.indexer_k_store(torch.zeros(3, 128, dtype=BF), cache, _slots(3), page_size)


def _transform(call, cache, page_size=64):
    call(torch.zeros(3, 128, dtype=BF), torch.ones(128), torch.zeros(128), 1e-6, _slots(3), torch.zeros(8, 64), cache,
         _slots(3), page_size)


def _store_fp4(cache, page_size=64):
    ops.indexer_k_store_fp4(torch.zeros(3, 128, dtype=BF), cache, _slots(3), page_size)


def _load_fp4(cache, page_size=64):
    ops.indexer_k_load_fp4(cache, _slots(3), page_size)


FP8 = [_store, lambda c, p=64: _transform(ops.indexer_k_transform_store, c, p),
       lambda c, p=64: _transform(indexer_transform.indexer_k_transform_store_fp8, c, p)]
FP4 = [_store_fp4, _load_fp4]


@pytest.mark.parametrize("call", FP8)
@pytest.mark.parametrize("shape", [(33, 64 * 68), (66, 64 * 68), (1, 33, 64 * 68), (33, 64, 68), (33, 64, 1, 68)])
def test_fp8_writers_refuse_4bit_pages(call, shape):
    with pytest.raises(RuntimeError, match=r"pages of page_size\*132"):
        call(torch.zeros(shape, dtype=U8))


@pytest.mark.parametrize("call", FP8)
def test_fp8_writers_refuse_4bit_pages_of_another_size(call):
    with pytest.raises(RuntimeError, match=r"pages of page_size\*132"):
        call(torch.zeros(33, 64 * 68, dtype=U8), 16)


@pytest.mark.parametrize("call", FP4)
@pytest.mark.parametrize("shape", [(17, 64 * 132), (34, 64 * 132), (17, 64, 132), (17, 64, 1, 132)])
def test_4bit_writer_and_reader_refuse_fp8_pages(call, shape):
    with pytest.raises(RuntimeError, match=r"pages of page_size\*68"):
        call(torch.zeros(shape, dtype=U8))


def test_a_4bit_cache_is_not_stored_to_as_fp8():
    """The layer buffer of an IndexerCacheFp4 with 33 pages, given to the fp8 writers."""
    layer = indexer.IndexerCacheFp4(1, 33, 64, device="cpu").get_buffer(0)
    for call in FP8:
        with pytest.raises(RuntimeError, match="pages of page_size"):
            call(layer)


@pytest.mark.parametrize("calls,row", [(FP8, 132), (FP4, 68)])
def test_the_formats_own_shapes_are_taken(calls, row):
    """Pages, several layers of them, keys or flat bytes: past the width check, which leaves the device's."""
    for shape in ((33, 64 * row), (2, 33, 64 * row), (33, 64, row), (33, 64, 1, row), (33 * 64 * row,), (0, 64 * row)):
        for call in calls:
            with pytest.raises(RuntimeError, match="GPU only"):
                call(torch.zeros(shape, dtype=U8))


@pytest.mark.parametrize("call", FP8 + FP4)
def test_a_cache_without_dimensions_is_refused(call):
    with pytest.raises(RuntimeError, match="pages of page_size"):
        call(torch.zeros((), dtype=U8))
