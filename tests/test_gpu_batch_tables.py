"""Block tables and slot maps on the GPU, equal to the oracle's integers."""
import random

import pytest
import torch

from nanoengine_amd import ops
from oracle import fp4_oracle as F

pytestmark = pytest.mark.gpu
I32, I64 = torch.int32, torch.int64


def _call(cuda, cached, new, tables, page, rows, free=None, head=None, wide=I64, cu=I32, extra=5):
    """The operator's outputs as the oracle gives them; the tables lie inside wider rows."""
    dev = lambda v, t=I32: torch.tensor(v, dtype=t, device=cuda)  # noqa: E731
    B, M = len(cached), len(tables[0]) if tables else 3
    store = torch.full((B, M + extra), -77, dtype=I32, device=cuda)
    bt = store[:, :M]
    if B:
        bt.copy_(dev(tables))
    empty = lambda n, t: torch.full((n,), -55, dtype=t, device=cuda)  # noqa: E731
    slots, pos, seq = empty(rows, wide), empty(rows, wide), empty(rows, I32)
    cu_q, cu_k, status = empty(B + 1, cu), empty(B + 1, cu), empty(4, I64)
    ops.batch_tables(dev(cached).reshape(B), dev(new).reshape(B), bt, page, slots, status,
                     free_blocks=None if free is None else dev(free).reshape(len(free)),
                     free_head=None if head is None else dev([head]),
                     positions=pos, seq_lens=seq, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k)
    torch.cuda.synchronize()
    assert torch.all(store[:, M:] == -77)
    return [bt.tolist(), slots.tolist(), pos.tolist(), seq.tolist(), cu_q.tolist(), cu_k.tolist(), status.tolist()]


def _batch(r, B, page, most_cached, most_new, spare=2):
    cached = [r.choice([0, r.randint(0, most_cached), page * r.randint(0, most_cached // page)]) for _ in range(B)]
    new = [r.choice([0, 1, r.randint(0, most_new)]) for _ in range(B)]
    width = max(-(-(c + n) // page) for c, n in zip(cached, new)) + spare
    ids = list(range(1, 1 + B * width + 100))
    r.shuffle(ids)
    tables = [[ids.pop() if p < -(-c // page) else 0 for p in range(width)] for c in cached]
    return cached, new, tables, ids


@pytest.mark.parametrize("seed,B,page,most_cached,most_new,pad", [
    (0, 1, 64, 5000, 1, 0), (1, 4, 64, 4000, 2, 3), (2, 33, 16, 300, 40, 0), (3, 129, 7, 100, 30, 1),
    (4, 300, 64, 900, 2, 1500), (5, 5, 64, 70000, 9000, 0), (6, 1000, 1, 5, 9, 2), (7, 64, 100000, 90000, 300, 0)])
@pytest.mark.parametrize("wide", [I32, I64])
def test_matches_oracle(cuda, seed, B, page, most_cached, most_new, pad, wide):
    print(f"tables seed={seed} B={B} page={page}", flush=True)
    r = random.Random(seed)
    cached, new, tables, free = _batch(r, B, page, most_cached, most_new)
    rows, head = sum(new) + pad, r.randint(0, 20)
    got = _call(cuda, cached, new, tables, page, rows, free, head, wide, cu=wide)
    assert got == list(map(list, F.batch_tables(cached, new, tables, page, rows, free, head)))
    assert got[6][0] == 0


def test_tables_filled_by_the_caller(cuda):
    r = random.Random(9)
    cached, new, tables, ids = _batch(r, 20, 16, 200, 30)
    full = [[x or ids.pop() for x in row] for row in tables]
    got = _call(cuda, cached, new, full, 16, sum(new))
    assert got == list(map(list, F.batch_tables(cached, new, full, 16, sum(new)))) and got[6][2] == 0
    assert got[0] == full


def test_largest_batch(cuda):
    r = random.Random(10)
    B = 8192
    cached, new = [r.randint(0, 200) for _ in range(B)], [r.choice([0, 1, 1, 2]) for _ in range(B)]
    tables = [[r.randint(0, 99999) for _ in range(5)] for _ in range(B)]
    free = list(range(100000, 100000 + B))
    got = _call(cuda, cached, new, tables, 64, sum(new) + 7, free, 0)
    assert got == list(map(list, F.batch_tables(cached, new, tables, 64, sum(new) + 7, free, 0)))


@pytest.mark.parametrize("name", ["negative", "overflow", "narrow", "free", "head", "rows", "bad_block", "no_free"])
def test_faults_are_reported_and_stay_in_bounds(cuda, name):
    """Each fault gives its bit and slots of -1 where a token has no block; nothing else is written."""
    r = random.Random(11)
    cached, new, tables, free = _batch(r, 12, 16, 100, 40, spare=0)
    cached[3], new[3] = 5, 37                       # this request opens two pages
    tables[3] = ([9] + [0] * 30)[:max(3, len(tables[0]))]
    width = max(len(t) for t in tables)
    tables = [t + [0] * (width - len(t)) for t in tables]
    rows, head, bit = sum(new), 0, 0
    if name == "negative":
        cached[5], new[7], bit = -1, -3, 1
        rows = sum(max(n, 0) for n in new)
    elif name == "overflow":
        cached[5], new[5], bit = 2 ** 31 - 2, 5, 1
    elif name == "narrow":
        tables, bit = [t[:2] for t in tables], 2
    elif name == "free":
        free, bit = free[:3], 4
    elif name == "no_free":
        free, bit = [], 4
    elif name == "head":
        head, bit = -2, 4
    elif name == "rows":
        rows, bit = rows - 20, 8
    else:
        tables[3][0] = -1
    got = _call(cuda, cached, new, tables, 16, rows, free, head)
    assert got == list(map(list, F.batch_tables(cached, new, tables, 16, rows, free, head)))
    assert got[6][0] == bit


def test_values_past_32_bits(cuda):
    """A block whose slots pass int32, and a key total that does."""
    big = 2 ** 26
    got = _call(cuda, [63], [3], [[big - 1, 5 * big]], 64, 4, wide=I64)
    assert got[1] == [(big - 1) * 64 + 63, 5 * big * 64, 5 * big * 64 + 1, -1]
    got = _call(cuda, [63], [3], [[big // 2 - 1, big]], 64, 4, wide=I32)
    assert got[1] == [(big // 2 - 1) * 64 + 63, -1, -1, -1] and got[6][0] == 0
    lens = [2 ** 31 - 10] * 3
    got = _call(cuda, lens, [0, 1, 0], [[1]] * 3, 2 ** 30, 1, cu=I64)
    assert got[5] == [0, 2 ** 31 - 10, 2 ** 32 - 19, 3 * 2 ** 31 - 29] and got[6][0] == 2 and got[1] == [-1]
    got = _call(cuda, lens, [0, 1, 0], [[1]] * 3, 2 ** 30, 1, cu=I32)
    assert got[5] == [0, 2 ** 31 - 10, 2 ** 31 - 1, 2 ** 31 - 1] and got[6][0] == 2 | 16 and got[4] == [0, 0, 1, 1]


def test_empty_batches(cuda):
    assert _call(cuda, [], [], [], 64, 3, [5], 0)[1:] == [[-1] * 3, [0] * 3, [0] * 3, [0], [0], [0, 0, 0, 0]]
    assert _call(cuda, [3, 64], [0, 0], [[4, 0], [5, 0]], 64, 0, [5], 0) == \
        [[[4, 0], [5, 0]], [], [], [], [0, 0, 0], [0, 3, 67], [0, 0, 0, 64]]


def test_steps_in_a_graph(cuda):
    """Decode steps replayed from one captured call, the lengths and the free list's head moving on the device."""
    B, page = 5, 4
    cached = torch.tensor([0, 3, 4, 9, 15], dtype=I32, device=cuda)
    new = torch.tensor([2, 2, 2, 2, 2], dtype=I32, device=cuda)
    bt = torch.zeros(B, 12, dtype=I32, device=cuda)
    for b, n in enumerate([0, 1, 1, 3, 4]):
        bt[b, :n] = torch.arange(n, device=cuda, dtype=I32) + 200 + 10 * b
    free, head = torch.randperm(80, device=cuda).to(I32), torch.zeros(1, dtype=I32, device=cuda)
    slots, status = torch.zeros(B * 2 + 3, dtype=I64, device=cuda), torch.zeros(4, dtype=I64, device=cuda)

    def step():
        ops.batch_tables(cached, new, bt, page, slots, status, free_blocks=free, free_head=head)
        cached.add_(new)
        head.add_(status[2:3].to(I32))

    keep = [t.clone() for t in (cached, bt, head)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    for t, k in zip((cached, bt, head), keep):
        t.copy_(k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    tables, lens, at = bt.tolist(), cached.tolist(), 0
    for _ in range(6):
        graph.replay()
        tables, want, _, _, _, _, st = F.batch_tables(lens, [2] * B, tables, page, B * 2 + 3, free.tolist(), at)
        torch.cuda.synchronize()
        assert bt.tolist() == tables and slots.tolist() == want and status.tolist() == st
        lens, at = [n + 2 for n in lens], at + st[2]
