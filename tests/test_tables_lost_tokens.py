"""BatchTables.check reports new tokens that got no cache slot where the status bits are clean."""
import pytest
import torch

from nanoengine_amd.batch_tables import BatchTables

I32, I64 = torch.int32, torch.int64


def _filled(slots, lens, faults=0, dtype=I64):
    t = BatchTables(2, len(slots), 4, device="cpu", slot_dtype=dtype)
    t.slot_mapping.copy_(torch.tensor(slots))
    t.seq_lens.copy_(torch.tensor(lens))
    t.status.copy_(torch.tensor([faults, sum(n > 0 for n in lens), 1, max(lens)]))
    return t


def test_a_token_without_a_slot_is_a_fault():
    assert _filled([70, 3, -1, -1], [7, 4, 0, 0]).check() == (2, 1, 7)      # padded rows have length 0
    with pytest.raises(RuntimeError, match="1 new tokens have no cache slot .* passes int64"):
        _filled([70, -1, -1, -1], [7, 4, 0, 0]).check()
    with pytest.raises(RuntimeError, match="2 new tokens have no cache slot .* passes int32"):
        _filled([-1, -1, 5, -1], [7, 4, 3, 0], dtype=I32).check()
    with pytest.raises(RuntimeError, match="the free list is too short$"):  # which is why they have none
        _filled([70, -1, -1, -1], [7, 4, 0, 0], faults=4).check()


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["table", "free", "int32"])
def test_plans_that_lose_tokens(cuda, where):
    t = BatchTables(3, 8, 4, page_size=16, device=cuda, slot_dtype=I32 if where == "int32" else I64)
    t.block_tables[:, 0] = torch.tensor([5, 6, 7], dtype=I32)
    cached = torch.tensor([3, 15, 0], dtype=I32, device=cuda)
    new = torch.tensor([2, 3, 0], dtype=I32, device=cuda)
    free = torch.tensor([9, 8], dtype=I32, device=cuda)
    t.plan(cached, new, free)
    assert t.check() == (5, 1, 18) and t.slot_mapping.tolist() == [83, 84, 111, 144, 145, -1, -1, -1]
    if where == "table":
        t.block_tables[0, 0] = -1
    elif where == "free":
        free[0] = -4
    else:
        t.block_tables[0, 0] = 2 ** 27
    t.plan(cached, new, free)
    assert t.status[0] == 0
    with pytest.raises(RuntimeError, match="2 new tokens have no cache slot"):
        t.check()
