"""The 4-bit caches as a serving step uses them: tables from lengths, the new tokens written, keys scored and
selected, the selected rows attended; prefill over what was written; captured and on several streams."""
import pytest
import torch

from nanoengine_amd import deep_gemm, flash_mla, indexer, mla_backend, ops
from nanoengine_amd.batch_tables import BatchTables
from nanoengine_amd.pipeline import DsaDecodeStep
from oracle import fp4_oracle as F

pytestmark = pytest.mark.gpu
SCALE = 192 ** -0.5
BF, I32 = torch.bfloat16, torch.int32


class Server:
    """Both caches, the tables and the free list of a small engine."""

    def __init__(self, device, B, blocks, n, heads, max_ctx, seed=0):
        self.g = torch.Generator(device=device).manual_seed(seed)
        self.dev, self.B, self.n, self.heads, self.blocks = device, B, n, heads, blocks
        self.mla = torch.zeros(blocks, 65, 1, 400, dtype=torch.uint8, device=device)[:, :64]
        self.keys = indexer.IndexerCacheFp4(1, blocks, 64, device=device)
        self.tables = BatchTables(B, 4096, max_ctx // 64, device=device)
        self.free = torch.randperm(blocks, generator=self.g, device=device).to(I32)
        self.head = torch.zeros(1, dtype=I32, device=device)
        self.lens = torch.zeros(B, dtype=I32, device=device)
        self.step = DsaDecodeStep(B, n, max_ctx, num_heads=heads, index_topk=512, device=device, indexer_format="fp4")
        # what was written, by slot
        self.rows = torch.zeros(blocks * 64, 576, dtype=BF, device=device)
        self.key_rows = torch.zeros(blocks * 64, 128, dtype=BF, device=device)

    def rnd(self, *shape):
        return torch.randn(*shape, generator=self.g, device=self.dev).to(BF)

    def write(self, new):
        """Plan and store `new` tokens of each request; returns the number of rows."""
        total = sum(new)
        self.tables.plan(self.lens, torch.tensor(new, dtype=I32, device=self.dev), self.free, self.head)
        assert self.tables.check()[0] == total
        self.head += self.tables.status[2:3].to(I32)
        self.lens += torch.tensor(new, dtype=I32, device=self.dev)
        kv, key = self.rnd(total, 576), self.rnd(total, 128)
        slots = self.tables.slot_mapping[:total]
        ops.mla_kv_store_fp4(kv, self.mla, self.tables.slot_mapping)
        self.keys.store_key(0, key, self.tables.slot_mapping)
        self.rows[slots], self.key_rows[slots] = kv, key
        return total

    def query(self):
        q = (torch.randn(self.B * self.n, 64, 128, generator=self.g, device=self.dev) * 60).to(torch.float8_e4m3fn)
        w = torch.randn(self.B * self.n, 64, generator=self.g, device=self.dev) * 0.01
        return q, w, self.rnd(self.B * self.n, self.heads, 576)

    def decode(self, q, w, qm):
        bt, seq = self.tables.block_tables, self.tables.seq_lens[: self.B * self.n]
        pt = bt if self.n == 1 else bt.repeat_interleave(self.n, dim=0)
        return self.step(q, w, self.keys.get_buffer(0), seq, bt, pt, qm, self.mla, SCALE)

    def check(self, q, w, qm, o, lse, logical, physical):
        seq = self.tables.seq_lens[: self.B * self.n].tolist()
        bt = self.tables.block_tables.long()
        values = F.mla_values(F.mla_rows(self.rows))
        keys = F.fp4_values(*F.fp4_quantize(self.key_rows.float()))
        for r, L in enumerate(seq):
            t = torch.arange(L, device=self.dev)
            slots = bt[r // self.n][t // 64] * 64 + t % 64
            want, tol = F.logits_row(q[r].float(), w[r], keys[slots])
            picked = logical[r][logical[r] >= 0].long()
            assert picked.numel() == min(L, 512) and torch.equal(physical[r][:picked.numel()].long(), slots[picked])
            left = torch.ones(L, dtype=torch.bool, device=self.dev)
            left[picked] = False
            if left.any():  # no key left behind is better than one taken by more than both scores' rounding
                assert (want[left] - tol[left]).max() <= (want[picked] + tol[picked]).min()
            eo, el, ot, lt = F.attend(qm[r], values[slots[picked]], SCALE)
            assert torch.all((o[r].double() - eo).abs() <= ot + 1e-30)
            assert torch.all((lse[r].double() == el) | ((lse[r].double() - el).abs() <= lt))


@pytest.mark.parametrize("n,heads", [(1, 16), (2, 64)])
def test_serving_steps(cuda, n, heads):
    B = 5
    s = Server(cuda, B, 160, n, heads, 4096, seed=n)
    print(f"fp4 serving n={n}", flush=True)
    s.write([700, 64, 1, 1300, 2])
    for _ in range(3):
        s.write([n] * B)
        q, w, qm = s.query()
        out = s.decode(q, w, qm)
        torch.cuda.synchronize()
        s.check(q, w, qm, *out)


def test_padded_batch(cuda):
    """Requests without new tokens pad the batch behind the others: their rows come out empty, and nothing of theirs is written."""
    s = Server(cuda, 5, 160, 1, 32, 2048, seed=6)
    s.write([300, 64, 700, 0, 0])
    caches = s.mla.clone(), s.keys.buffer.clone()
    s.write([1, 1, 1, 0, 0])
    slots = s.tables.slot_mapping[:3]
    same = torch.ones(160 * 64, dtype=torch.bool, device=cuda)
    same[slots] = False
    assert torch.equal(s.mla.reshape(-1, 400)[same], caches[0].reshape(-1, 400)[same])
    assert s.tables.slot_mapping[3:].eq(-1).all() and s.tables.seq_lens[:5].tolist() == [301, 65, 701, 0, 0]
    q, w, qm = s.query()
    out = s.decode(q, w, qm)
    torch.cuda.synchronize()
    s.check(q, w, qm, *out)
    assert torch.all(out[0][3:] == 0) and torch.all(torch.isneginf(out[1][3:])) and torch.all(out[3][3:] == -1)


def test_prefill_over_what_was_written(cuda):
    """Reading the 4-bit caches back gives the operands of the fp8 prefill scorer and of the bf16 prefill attention."""
    s = Server(cuda, 2, 64, 1, 64, 2048, seed=3)
    s.write([900, 300])
    # the slots of every cached token: tables that are full already, all tokens "new"
    whole = BatchTables(2, 1200, 32, device=cuda)
    whole.block_tables.copy_(s.tables.block_tables)
    whole.plan(torch.zeros(2, dtype=I32, device=cuda), s.lens)
    assert whole.check() == (1200, 0, 900)
    slots = whole.slot_mapping
    rows = ops.mla_kv_load_fp4(s.mla, slots)
    assert torch.equal(rows.double(), F.mla_values(F.mla_rows(s.rows[slots])))
    q = s.rnd(40, 64, 576)
    idx = torch.stack([torch.randperm(1200, generator=s.g, device=cuda)[:128] for _ in range(40)]).to(I32)
    o, _, lse = flash_mla.flash_mla_sparse_fwd(q, rows[:, None], idx[:, None], SCALE)
    keys, scales = s.keys.load_key_fp8(0, slots)
    qi = (torch.randn(40, 64, 128, generator=s.g, device=cuda) * 60).to(torch.float8_e4m3fn)
    w = torch.randn(40, 64, generator=s.g, device=cuda) * 0.01
    ks = torch.tensor([0] * 20 + [900] * 20, dtype=I32, device=cuda)
    ke = torch.tensor([900] * 20 + [1200] * 20, dtype=I32, device=cuda)
    logits = deep_gemm.fp8_mqa_logits(qi, (keys, scales), w, ks, ke)
    torch.cuda.synchronize()
    exact = F.fp4_values(*F.fp4_quantize(s.key_rows[slots].float()))
    for t in range(40):
        eo, el, ot, lt = F.attend(q[t], rows[idx[t].long()].double(), SCALE)
        assert torch.all((o[t].double() - eo).abs() <= ot + 1e-30) and torch.all((lse[t].double() - el).abs() <= lt)
        a, b = int(ks[t]), int(ke[t])
        want, _ = F.logits_row(qi[t].float(), w[t], exact[a:b])
        # the keys are exact; the scorer's fp8 products keep 13 bits below the largest of each 64-term sum
        mass = (w[t].abs().double()[:, None] * (qi[t].double().abs() @ exact[a:b].abs().T)).sum(dim=0)
        assert torch.all((logits[t, a:b].double() - want).abs() <= 2.0 ** -11 * mass)


def test_backend_stores_and_decodes(cuda):
    B, H, K, blocks = 3, 128, 256, 8
    layer = mla_backend.create_mla(hardware_backend="mi355x", num_heads=H, head_dim=576, scale=SCALE,
                                   num_kv_heads=1, v_head_dim=512, nsa_index_topk=K)
    layer.k_cache = torch.zeros(blocks, 65, 1, 400, dtype=torch.uint8, device=cuda)[:, :64]
    g = torch.Generator(device=cuda).manual_seed(4)
    hist = torch.randn(blocks * 64, 576, generator=g, device=cuda).to(BF)
    ops.mla_kv_store_fp4(hist, layer.k_cache, torch.arange(blocks * 64, device=cuda))
    tables = BatchTables(B, B, 4, device=cuda)
    tables.block_tables.copy_(torch.tensor([[1, 2, 0, 0], [3, 0, 0, 0], [5, 6, 7, 0]]))
    lens = torch.tensor([70, 10, 150], dtype=I32, device=cuda)
    tables.plan(lens, torch.ones_like(lens))
    mla_backend.set_batch_context(**tables.context_fields())
    try:
        k, q = torch.randn(B, 1, 576, generator=g, device=cuda).to(BF), torch.randn(B, H, 576, generator=g, device=cuda).to(BF)
        idx = torch.stack([torch.randperm(blocks * 64, generator=g, device=cuda)[:K] for _ in range(B)]).to(I32)
        idx[:, 0] = tables.slot_mapping.to(I32)
        o = layer.forward(q, k, None, idx)
        warm = layer.forward(q, None, None)         # no indices: every one -1, as in capture warm-up
    finally:
        mla_backend.reset_batch_context()
    torch.cuda.synchronize()
    assert tables.slot_mapping.tolist() == [2 * 64 + 6, 3 * 64 + 10, 7 * 64 + 22]
    hist[tables.slot_mapping] = k[:, 0]
    values = F.mla_values(F.mla_rows(hist))
    assert torch.all(warm == 0)
    for t in range(B):
        eo, _, ot, _ = F.attend(q[t], values[idx[t].long()], SCALE)
        assert torch.all((o[t].double() - eo).abs() <= ot + 1e-30)


def test_decode_topk_with_more_query_tokens(cuda):
    """Three query tokens a request are scored position by position, into a given buffer or a new one."""
    s = Server(cuda, 2, 64, 1, 16, 2048, seed=5)
    s.write([900, 700])
    q = (torch.randn(6, 64, 128, generator=s.g, device=cuda) * 60).to(torch.float8_e4m3fn)
    w = torch.randn(6, 64, generator=s.g, device=cuda) * 0.01
    bt = s.tables.block_tables[:, :16]
    args = (q, w, s.keys.get_buffer(0), s.lens, bt, 512)
    got = indexer.indexer_decode_topk(*args, translate_topk=True, topk_page_size=64)
    again = indexer.indexer_decode_topk(*args, logits_out=torch.empty(6, 1024, device=cuda))
    torch.cuda.synchronize()
    assert torch.equal(got[0], again)
    for r in range(6):
        L = int(s.lens[r // 3]) - 2 + r % 3
        one = ops.indexer_logits_fp4(q[r][None, None], s.keys.get_buffer(0), w[r:r + 1], torch.tensor([L], device=cuda),
                                     bt[r // 3][None], L)
        want = one[0].topk(512).indices.sort().values
        assert torch.equal(got[0][r].long(), want)


@pytest.mark.parametrize("n", [1, 2])
def test_captured_step(cuda, n):
    """Plan, stores, scoring, selection and attention captured once and replayed over changing inputs, with eager
    work between, equal what the same calls give eagerly."""
    B, H = 4, 64
    a, b = (Server(cuda, B, 120, n, H, 2048, seed=7) for _ in range(2))
    for s in (a, b):
        s.write([500, 63, 1, 1000])
    new = torch.full((B,), n, dtype=I32, device=cuda)
    ins = [torch.empty(B * n, *shape, dtype=t, device=cuda) for shape, t in
           (((576,), BF), ((128,), BF), ((64, 128), torch.float8_e4m3fn), ((64,), torch.float32), ((H, 576), BF))]

    def step(s, kv, key, q, w, qm):
        s.tables.plan(s.lens, new, s.free, s.head)
        ops.mla_kv_store_fp4(kv, s.mla, s.tables.slot_mapping[: B * n])
        s.keys.store_key(0, key, s.tables.slot_mapping[: B * n])
        out = s.decode(q, w, qm)
        s.lens.add_(new)
        s.head.add_(s.tables.status[2:3].to(I32))
        return out

    def fill(seed):
        g = torch.Generator(device=cuda).manual_seed(seed)
        for t in ins:
            t.copy_((torch.randn(t.shape, generator=g, device=cuda) * (60 if t.dtype == torch.float8_e4m3fn else 1)).to(t.dtype))

    fill(1)
    state = [t.clone() for t in (a.lens, a.head, a.mla, a.keys.buffer, a.tables.block_tables)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step(a, *ins)                               # warm-up
        for t, k in zip((a.lens, a.head, a.mla, a.keys.buffer, a.tables.block_tables), state):
            t.copy_(k)
        with torch.cuda.graph(graph, stream=side):
            outs = step(a, *ins)
    torch.cuda.current_stream().wait_stream(side)
    for r in range(4):
        fill(10 + r)
        graph.replay()
        want = step(b, *ins)
        torch.cuda.synchronize()
        for x, y in zip(outs, want):
            assert torch.equal(x, y)
        assert torch.equal(a.tables.block_tables, b.tables.block_tables) and torch.equal(a.mla, b.mla)
        assert torch.equal(a.keys.buffer, b.keys.buffer) and torch.equal(a.lens, b.lens)


def test_two_streams(cuda):
    """Independent calls on two streams at once give what they give alone."""
    g = torch.Generator(device=cuda).manual_seed(9)
    rows = F.mla_rows(torch.randn(40 * 64, 576, generator=g, device=cuda).to(BF)).view(40, 64, 400)
    pages = F.key_pages(torch.randn(40 * 64, 128, generator=g, device=cuda))
    bt = torch.randperm(40, generator=g, device=cuda).to(I32).view(1, 40).repeat(8, 1)
    lens = torch.full((8, 1), 2500, dtype=I32, device=cuda)

    def call(seed):
        g2 = torch.Generator(device=cuda).manual_seed(seed)
        q = torch.randn(8, 64, 576, generator=g2, device=cuda).to(BF)
        idx = torch.randint(0, 2560, (8, 1024), generator=g2, device=cuda).to(I32)
        qi = (torch.randn(8, 1, 64, 128, generator=g2, device=cuda) * 60).to(torch.float8_e4m3fn)
        w = torch.randn(8, 64, generator=g2, device=cuda)
        return lambda: [*ops.sparse_mla_decode_fp4(q, rows, idx, SCALE), ops.indexer_logits_fp4(qi, pages, w, lens, bt, 2500)]

    calls = [call(1), call(2)]
    alone = [[t.clone() for t in c()] for c in calls]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for st, c in zip(streams, calls):
            with torch.cuda.stream(st):
                got.append(c())
        torch.cuda.synchronize()
        for x, y in zip(got, alone):
            assert all(torch.equal(p, q) for p, q in zip(x, y))
