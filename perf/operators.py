"""Performance cases of the 4-bit caches of the DSA path and of the tables that address them.

A serving engine first extends the block tables of its running requests and maps
the step's new tokens to cache slots (``tables``), writes the new tokens' MLA
rows and indexer keys into the 4-bit caches (``mla_store``, ``index_store``; the
rows are read back as prefill over a cached prefix does), scores a request's
keys with the lightning indexer (``index_logits``) and attends over the selected
rows (``mla_decode``).

Both caches hold e2m1 codes with one power-of-two scale per 32 elements:
  element 2i in the low nibble of byte i; value = code * 2^(scale byte - 127);
  MLA row (400 B): 256 B of codes (512 dims), 16 scale bytes, 64 bf16 rope values;
  indexer page of 64 keys (4352 B): 64 x 64 B of codes (128 dims), then 64 x 4 scale bytes.
"""
from __future__ import annotations

import math
import random

import torch

own = False  # False: the operators' plain forms; True: the framework's kernels

PAGE = 64
SCALE = 192 ** -0.5
DEV = "cuda"
MLA_ROW, MLA_CODES, MLA_SCALES = 400, 256, 16
KEY_CODES, KEY_SCALES = 64, 4
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # four interactive requests, one new token each: the call's latency
        {"name": "tables_b4", "kind": "tables", "batch": 4, "new": "decode", "next_n": 1, "hi": 4096, "page": 64,
         "pad": 0, "wide": True},
        # the benchmark's speculative verify batch: two tokens a request, padded to a captured batch size
        {"name": "tables_b64_verify", "kind": "tables", "batch": 64, "new": "decode", "next_n": 2, "hi": 131072,
         "page": 64, "pad": 128, "wide": False},
        # a large prefill batch of ragged prompts over cached prefixes
        {"name": "tables_prefill_128k", "kind": "tables", "batch": 96, "new": "prefill", "tokens": 131072, "hi": 32768,
         "page": 64, "pad": 1000, "wide": True},
        # the new tokens of the benchmark's decode batch, each into a page of its own
        {"name": "mla_store_128", "kind": "mla_store", "tokens": 128},
        # the benchmark's prefill chunk
        {"name": "mla_store_8k", "kind": "mla_store", "tokens": 8192},
        # a small interactive batch of short chats: launches and latency
        {"name": "mla_b4_short", "kind": "mla_decode", "batch": 4, "next_n": 1, "heads": 128, "topk": 2048,
         "lo": 1024, "hi": 4096},
        # one rank of an eight-way tensor-parallel group, a mixed batch, some of it shorter than the selection
        {"name": "mla_b90_tp8", "kind": "mla_decode", "batch": 90, "next_n": 1, "heads": 16, "topk": 2048,
         "lo": 300, "hi": 32768},
        # the benchmark's decode batch: 128 long contexts, all heads
        {"name": "mla_b128_64k", "kind": "mla_decode", "batch": 128, "next_n": 1, "heads": 128, "topk": 2048,
         "lo": 65536, "hi": 65536},
        # an odd number of new indexer keys of a small running batch
        {"name": "index_store_33", "kind": "index_store", "tokens": 33},
        # the keys of the benchmark's prefill chunk
        {"name": "index_store_8k", "kind": "index_store", "tokens": 8192},
        # a speculative verify batch of ragged contexts, two query tokens each
        {"name": "index_b33_verify", "kind": "index_logits", "batch": 33, "next_n": 2, "lo": 1000, "hi": 20000},
        # the benchmark's decode batch: every key of 128 contexts of 64K
        {"name": "index_b128_64k", "kind": "index_logits", "batch": 128, "next_n": 1, "lo": 65536, "hi": 65536},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "mla_store", "mla_decode", "mla_decode", "index_store", "index_logits", "index_logits"])
    if kind == "tables":
        case = {"kind": kind, "batch": _log(rng, 1, 1024), "hi": _log(rng, 64, 131072), "page": rng.choice([16, 64, 64, 128]),
                "pad": rng.choice([0, 1, 77, 512]), "wide": rng.random() < 0.5}
        if rng.random() < 0.5:
            return {**case, "new": "decode", "next_n": rng.choice([1, 1, 2, 4])}
        return {**case, "new": "prefill", "tokens": _log(rng, 16, 131072)}
    if kind in ("mla_store", "index_store"):
        return {"kind": kind, "tokens": _log(rng, 1, 8192)}
    n = rng.choice([1, 1, 1, 2])
    if kind == "mla_decode":
        batch = _log(rng, 1, 128 // n)
        hi = _log(rng, 64, 65536)
        return {"kind": kind, "batch": batch, "next_n": n, "heads": rng.choice([16, 32, 48, 64, 128, 128]),
                "topk": rng.choice([2048, 2048, 2048, 512]), "lo": _log(rng, n, hi), "hi": hi}
    hi = _log(rng, 64, 131072)
    return {"kind": kind, "batch": _log(rng, 1, max(1, min(128, (1 << 22) // (n * hi)))), "next_n": n,
            "lo": _log(rng, n, hi), "hi": hi}


# ------------------------------------------------------------------ sizes of a case
def _lens(case):
    """Context lengths of the batch after its last token: from the case alone."""
    r = random.Random("%(kind)s %(batch)d %(hi)d" % case)
    lo, hi = max(case.get("lo", 1), case.get("next_n", 1)), max(case["hi"], case.get("next_n", 1))
    return [r.randint(lo, hi) for _ in range(case["batch"])]


def _row_lens(case):
    """One length per query token."""
    n = case["next_n"]
    return [max(L - (n - 1 - j), 1) for L in _lens(case) for j in range(n)]


def _requests(case):
    """(cached tokens, new tokens) of each request of a `tables` case; some requests of a batch have no cached ones."""
    r = random.Random("requests %(batch)d %(hi)d" % case)
    cached = [0 if r.random() < 0.15 else r.randint(1, case["hi"]) for _ in range(case["batch"])]
    if case["new"] == "decode":
        return cached, [case["next_n"]] * case["batch"]
    cuts = sorted(r.randint(0, case["tokens"]) for _ in range(case["batch"] - 1))
    return cached, [b - a for a, b in zip([0] + cuts, cuts + [case["tokens"]])]


def _ceil(a, b):
    return -(-a // b)


# ------------------------------------------------------------------ the format
def _quantise(x):
    """[..., 32k] float32 -> (codes uint8 [..., 16k] packed, scale bytes uint8 [..., k])."""
    blocks = x.float().unflatten(-1, (-1, 32))
    amax = blocks.abs().amax(dim=-1).clamp(min=2.0 ** -60)
    m, e = torch.frexp(amax)  # amax = m * 2^e, m in [0.5, 1): amax <= 6 * 2^k where k = e - 3 + (m > 0.75)
    k = (e - 3 + (m > 0.75).to(e.dtype)).clamp(-40, 125)
    y = torch.ldexp(blocks, -k[..., None])
    mag = y.abs()
    # round to nearest, ties to the even code
    code = ((mag > 0.25).to(torch.uint8) + (mag >= 0.75) + (mag > 1.25) + (mag >= 1.75) + (mag > 2.5) + (mag >= 3.5)
            + (mag > 5.0)).to(torch.uint8)
    code = (code | (torch.signbit(y).to(torch.uint8) << 3)).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (k + 127).to(torch.uint8)


def _values(codes, scales):
    """Packed codes [..., n] and scale bytes [..., n / 16] -> float32 [..., 2n]."""
    grid = torch.tensor(GRID + tuple(-g for g in GRID), device=codes.device)
    v = grid[torch.stack([codes & 15, codes >> 4], dim=-1).to(torch.int32)]
    return (v.flatten(-2).unflatten(-1, (-1, 32)) * torch.exp2(scales.float() - 127.0)[..., None]).flatten(-2)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def prepare(case, seed):
    return globals()["_prepare_" + case["kind"]](case, seed)


def _prepare_tables(case, seed):
    gen, P = _gen(seed), case["page"]
    cached, new = _requests(case)
    old = [_ceil(c, P) for c in cached]
    need = [_ceil(c + n, P) - o for c, n, o in zip(cached, new, old)]
    ids = torch.randperm(sum(old) + sum(need) + 50, generator=gen, device=DEV).to(torch.int32)
    width = max(o + n for o, n in zip(old, need)) + 3
    col = torch.arange(width, device=DEV)[None]
    held = torch.tensor(old, device=DEV)[:, None]
    first = held.cumsum(0) - held
    tables = torch.where(col < held, ids[(first + col).clamp(max=ids.numel() - 1)], 0).to(torch.int32)
    # a free list of which the first few blocks went to an earlier step
    free = ids[sum(old):]
    rows, wide = sum(new) + case["pad"], torch.int64 if case["wide"] else torch.int32
    empty = lambda n, t: torch.empty(n, dtype=t, device=DEV)  # noqa: E731
    return {"kind": "tables", "page": P, "cached": torch.tensor(cached, dtype=torch.int32, device=DEV),
            "new": torch.tensor(new, dtype=torch.int32, device=DEV), "tables": tables, "free": free,
            "head": torch.tensor([seed % 40], dtype=torch.int32, device=DEV), "slots": empty(rows, wide),
            "positions": empty(rows, wide), "seq_lens": empty(rows, torch.int32),
            "cu_q": empty(case["batch"] + 1, torch.int32), "cu_k": empty(case["batch"] + 1, torch.int32),
            "status": empty(4, torch.int64)}


def _token_slots(T, gen):
    """Slots of T new tokens: a decode batch's in pages of their own, a prefill chunk's page by page."""
    pages = T + 7 if T <= 512 else _ceil(T, PAGE) + 7
    order = torch.randperm(pages, generator=gen, device=DEV)
    i = torch.arange(T, device=DEV)
    if T <= 512:
        return pages, order[:T] * PAGE + torch.randint(0, PAGE, (T,), generator=gen, device=DEV)
    return pages, order[i // PAGE] * PAGE + i % PAGE


def _prepare_mla_store(case, seed):
    gen, T = _gen(seed), case["tokens"]
    pages, slots = _token_slots(T, gen)
    # the compressed keys differ by channel, as learned weights leave them
    channel = torch.exp(0.5 * torch.randn(576, generator=gen, device=DEV))
    kv = (torch.randn(T, 576, generator=gen, device=DEV) * channel).to(torch.bfloat16)
    cache = torch.zeros(pages, PAGE + 1, 1, MLA_ROW, dtype=torch.uint8, device=DEV)
    return {"kind": "mla_store", "kv": kv, "cache": cache[:, :PAGE], "slots": slots}


def _prepare_index_store(case, seed):
    gen, T = _gen(seed), case["tokens"]
    pages, slots = _token_slots(T, gen)
    # the indexer rotates its keys with a Hadamard product: close to normal in every dim
    key = torch.randn(T, 128, generator=gen, device=DEV).to(torch.bfloat16)
    cache = torch.zeros(pages, PAGE * (KEY_CODES + KEY_SCALES), dtype=torch.uint8, device=DEV)
    return {"kind": "index_store", "key": key, "cache": cache, "slots": slots}


def _pages(case, gen):
    """Block tables [B, M] of the case's contexts over a shuffled pool, and the pool's size."""
    pages = torch.tensor([_ceil(L, PAGE) for L in _lens(case)], device=DEV)[:, None]
    total, width = int(pages.sum()), int(pages.max())
    pool = torch.randperm(total, generator=gen, device=DEV).to(torch.int32)
    col = torch.arange(width, device=DEV)[None]
    at = (pages.cumsum(0) - pages + col).clamp(max=total - 1)
    return torch.where(col < pages, pool[at], 0).to(torch.int32), total


def _picks(lens, k, gen):
    """[rows, k] distinct ascending positions below each row's length, -1 padded where it is shorter than k."""
    n = torch.tensor(lens, device=DEV, dtype=torch.float64)[:, None]
    i = torch.arange(k, device=DEV, dtype=torch.float64)[None]
    lo, hi = torch.floor(i * n / k), torch.floor((i + 1) * n / k)
    u = torch.rand(len(lens), k, generator=gen, device=DEV)
    spread = lo + torch.floor((hi - lo) * u).clamp(max=hi - lo - 1)
    return torch.where(n > k, spread, torch.where(i < n, i, torch.full_like(i, -1))).long()


def _prepare_mla_decode(case, seed):
    gen = _gen(seed)
    B, n, H = case["batch"], case["next_n"], case["heads"]
    tables, total = _pages(case, gen)
    # rows drawn from a pool of quantised ones
    kv = torch.randn(1 << 15, 576, generator=gen, device=DEV).to(torch.bfloat16)
    codes, scales = _quantise(kv[:, :512].float())
    pool = torch.cat([codes, scales, kv[:, 512:].contiguous().view(torch.uint8)], dim=1)
    cache = torch.zeros(total, PAGE + 1, 1, MLA_ROW, dtype=torch.uint8, device=DEV)
    cache[:, :PAGE, 0] = pool[torch.randint(0, 1 << 15, (total, PAGE), generator=gen, device=DEV)]
    pos = _picks(_row_lens(case), case["topk"], gen)
    slot = tables.repeat_interleave(n, dim=0).long().gather(1, pos.clamp(min=0) // PAGE) * PAGE + pos % PAGE
    return {"kind": "mla_decode", "cache": cache[:, :PAGE], "indices": torch.where(pos >= 0, slot, -1).to(torch.int32),
            "q": torch.randn(B * n, H, 576, generator=gen, device=DEV).to(torch.bfloat16)}


def _prepare_index_logits(case, seed):
    gen = _gen(seed)
    B, n = case["batch"], case["next_n"]
    tables, total = _pages(case, gen)
    codes, scales = _quantise(torch.randn(1 << 15, 128, generator=gen, device=DEV).to(torch.bfloat16).float())
    pool = torch.cat([codes.view(-1, PAGE * KEY_CODES), scales.reshape(-1, PAGE * KEY_SCALES)], dim=1)
    cache = pool[torch.randint(0, pool.shape[0], (total,), generator=gen, device=DEV)]
    # queries in fp8 with one power-of-two scale a row, which the head weights carry
    q = torch.randn(B * n, 64, 128, generator=gen, device=DEV).to(torch.bfloat16).float()
    sf = torch.exp2(torch.ceil(torch.log2(q.abs().amax(dim=-1).clamp(min=1e-4) / 448.0)))
    w = torch.randn(B * n, 64, generator=gen, device=DEV) * (64 ** -0.5) * (128 ** -0.5)
    return {"kind": "index_logits", "q": (q / sf[..., None]).to(torch.float8_e4m3fn).view(B, n, 64, 128),
            "weights": (w * sf).contiguous(), "cache": cache.contiguous(), "tables": tables,
            "lens": torch.tensor(_row_lens(case), dtype=torch.int32, device=DEV).view(B, n),
            "max_len": max(_lens(case))}


# ------------------------------------------------------------------ one pass
def run(state):
    return globals()["_run_" + state["kind"]](state)


def _run_tables(st):
    if own:
        from nanoengine_amd import ops
        ops.batch_tables(st["cached"], st["new"], st["tables"], st["page"], st["slots"], st["status"],
                         free_blocks=st["free"], free_head=st["head"], positions=st["positions"],
                         seq_lens=st["seq_lens"], cu_seqlens_q=st["cu_q"], cu_seqlens_k=st["cu_k"])
    else:
        c, n, P, tables = st["cached"].long(), st["new"].long(), st["page"], st["tables"]
        old = (c + P - 1) // P
        need = (c + n + P - 1) // P - old
        first = st["head"].long() + need.cumsum(0) - need
        st["cu_q"].copy_(torch.nn.functional.pad(n.cumsum(0), (1, 0)))
        st["cu_k"].copy_(torch.nn.functional.pad((c + n).cumsum(0), (1, 0)))
        col = torch.arange(tables.shape[1], device=DEV)[None]
        step = col - old[:, None]
        taken = st["free"][(first[:, None] + step).clamp(0, st["free"].numel() - 1)]
        tables.copy_(torch.where((step >= 0) & (step < need[:, None]), taken, tables))
        t = torch.arange(st["slots"].numel(), device=DEV)
        ends = n.cumsum(0)
        b = torch.searchsorted(ends, t, right=True).clamp(max=n.numel() - 1)
        pos = c[b] + t - (ends - n)[b]
        inside = t < ends[-1]
        block = tables[b, (pos // P).clamp(max=tables.shape[1] - 1)].long()
        st["slots"].copy_(torch.where(inside, block * P + pos % P, -1))
        st["positions"].copy_(torch.where(inside, pos, 0))
        st["seq_lens"].copy_(torch.where(inside, pos + 1, 0))
        st["status"].copy_(torch.stack([torch.zeros_like(ends[-1]), ends[-1], need.sum(), (c + n).max()]))
    return [st[k] for k in ("tables", "slots", "positions", "seq_lens", "cu_q", "cu_k", "status")]


def _run_mla_store(st):
    if own:
        from nanoengine_amd import ops
        ops.mla_kv_store_fp4(st["kv"], st["cache"], st["slots"])
        return ops.mla_kv_load_fp4(st["cache"], st["slots"])
    codes, scales = _quantise(st["kv"][:, :512].float())
    row = torch.cat([codes, scales, st["kv"][:, 512:].contiguous().view(torch.uint8)], dim=1)
    at, off = st["slots"] // PAGE, st["slots"] % PAGE
    st["cache"][at, off, 0] = row
    back = st["cache"][at, off, 0]
    nope = _values(back[:, :MLA_CODES], back[:, MLA_CODES:MLA_CODES + MLA_SCALES])
    rope = back[:, MLA_CODES + MLA_SCALES:].contiguous().view(torch.bfloat16)
    return torch.cat([nope.to(torch.bfloat16), rope], dim=1)


def _run_index_store(st):
    if own:
        from nanoengine_amd import ops
        ops.indexer_k_store_fp4(st["key"], st["cache"], st["slots"], PAGE)
        return ops.indexer_k_load_fp4(st["cache"], st["slots"], PAGE)
    codes, scales = _quantise(st["key"].float())
    at, off = st["slots"] // PAGE, st["slots"] % PAGE
    code_part = st["cache"][:, :PAGE * KEY_CODES].unflatten(1, (PAGE, KEY_CODES))
    scale_part = st["cache"][:, PAGE * KEY_CODES:].unflatten(1, (PAGE, KEY_SCALES))
    code_part[at, off] = codes
    scale_part[at, off] = scales
    # fp8 keys with one scale a key: the largest of its four block scales takes the codes to 6 * 2^6 at most
    s = torch.exp2(scale_part[at, off].float().amax(dim=1) - 127.0 - 6.0)
    return (_values(code_part[at, off], scale_part[at, off]) / s[:, None]).to(torch.float8_e4m3fn), s


def _run_mla_decode(st):
    if own:
        from nanoengine_amd import ops
        return ops.sparse_mla_decode_fp4(st["q"], st["cache"], st["indices"], SCALE)
    idx = st["indices"].long()
    rows = st["cache"][idx.clamp(min=0) // PAGE, idx.clamp(min=0) % PAGE, 0]
    nope = _values(rows[..., :MLA_CODES], rows[..., MLA_CODES:MLA_CODES + MLA_SCALES])
    rope = rows[..., MLA_CODES + MLA_SCALES:].contiguous().view(torch.bfloat16).float()
    s = torch.bmm(st["q"].float(), torch.cat([nope, rope], dim=-1).transpose(1, 2).contiguous()) * SCALE
    s = s.masked_fill((idx < 0)[:, None], -math.inf)
    m = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - m)
    total = p.sum(dim=-1, keepdim=True)
    return torch.bmm(p / total, nope).to(torch.bfloat16), (m + total.log()).squeeze(-1)


def _run_index_logits(st):
    if own:
        from nanoengine_amd import ops
        return ops.indexer_logits_fp4(st["q"], st["cache"], st["weights"], st["lens"], st["tables"], st["max_len"])
    B, n = st["lens"].shape
    pages = st["cache"][st["tables"].long()]
    codes = pages[..., :PAGE * KEY_CODES].reshape(B, -1, KEY_CODES)[:, :st["max_len"]]
    scales = pages[..., PAGE * KEY_CODES:].reshape(B, -1, KEY_SCALES)[:, :st["max_len"]]
    q = st["q"].float().view(B, n * 64, 128)
    s = torch.bmm(q, _values(codes, scales).transpose(1, 2).contiguous()).clamp_(min=0)
    logits = (s * st["weights"].view(B, n * 64, 1)).view(B * n, 64, -1).sum(dim=1)
    at = torch.arange(st["max_len"], device=DEV)[None]
    return logits.masked_fill(at >= st["lens"].view(-1, 1), -math.inf)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "tables":
        cached, new = _requests(case)
        P, word = case["page"], 8 if case["wide"] else 4
        pages = sum(_ceil(c + n, P) - _ceil(c, P) for c, n in zip(cached, new))
        return {"bytes": 16 * len(new) + 12 * pages + (sum(new) + case["pad"]) * (2 * word + 4) + 48, "flops": 0}
    if kind == "mla_store":  # written, then read back
        return {"bytes": case["tokens"] * (1152 + 8 + 400 + 8 + 1152), "flops": case["tokens"] * 512 * 4}
    if kind == "index_store":
        return {"bytes": case["tokens"] * (256 + 8 + 68 + 8 + 132), "flops": case["tokens"] * 128 * 4}
    rows = _row_lens(case)
    if kind == "mla_decode":
        keys, H = sum(min(L, case["topk"]) for L in rows), case["heads"]
        return {"bytes": keys * 400 + len(rows) * (case["topk"] * 4 + H * (1152 + 1024 + 4)),
                "flops": 2 * H * 1088 * keys}
    lens = _lens(case)
    return {"bytes": sum(lens) * 68 + sum(_ceil(L, PAGE) for L in lens) * 4 + len(rows) * (64 * 132 + 4 * max(lens)),
            "flops": 2 * 64 * 128 * sum(rows)}


# ------------------------------------------------------------------ 64 bits
def _grid64(nibble):
    """The number that a 4-bit code stands for: sign, two exponent bits, one mantissa bit."""
    sign, e, m = 1.0 - 2.0 * (nibble >> 3).double(), (nibble >> 1) & 3, (nibble & 1).double()
    return sign * torch.where(e == 0, 0.5 * m, (1.0 + 0.5 * m) * torch.exp2(e.double() - 1.0))


def _rows64(raw, dims):
    """dims / 2 code bytes and dims / 32 scale bytes a row -> the row's values."""
    codes, scales = raw[..., :dims // 2].int(), raw[..., dims // 2:dims // 2 + dims // 32].double()
    v = torch.empty(*raw.shape[:-1], dims, dtype=torch.float64, device=raw.device)
    v[..., 0::2], v[..., 1::2] = _grid64(codes & 15), _grid64(codes >> 4)
    return v * torch.exp2(scales - 127.0).repeat_interleave(32, dim=-1)


def _nearest64(x):
    """Each block of 32 on its scaled grid: the nearest value, of two equally near the one with the even code."""
    x = x.double()
    b = x.view(x.shape[0], -1, 32)
    k = torch.ceil(torch.log2(b.abs().amax(dim=-1, keepdim=True).clamp(min=2.0 ** -100) / 6.0)).clamp(-40, 125)
    y = b / torch.exp2(k)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    d = (y.abs()[..., None] - grid).abs()
    odd = torch.arange(8, device=x.device) % 2
    near = torch.where(d == d.amin(dim=-1, keepdim=True), odd, 2).argmin(dim=-1)
    return (grid[near] * y.sign() * torch.exp2(k)).view(x.shape), k.squeeze(-1)


def exact(case, seed):
    kind = case["kind"]
    if kind == "tables":
        return None  # whole numbers
    st = prepare(case, seed)
    if kind == "mla_store":
        kv = st["kv"].double()
        return torch.cat([_nearest64(kv[:, :512])[0], kv[:, 512:]], dim=1)
    if kind == "index_store":
        v, k = _nearest64(st["key"])
        s = torch.exp2(k.amax(dim=1) - 6.0)
        return v / s[:, None], s
    if kind == "mla_decode":
        outs, lses = [], []
        for q, idx in zip(st["q"].double(), st["indices"].long()):
            idx = idx[idx >= 0]
            raw = st["cache"][idx // PAGE, idx % PAGE, 0]
            k = torch.cat([_rows64(raw, 512), raw[:, 272:].contiguous().view(torch.bfloat16).double()], dim=1)
            s = SCALE * (q @ k.T)
            outs.append(torch.softmax(s, dim=1) @ k[:, :512])
            lses.append(torch.logsumexp(s, dim=1))
        return torch.stack(outs), torch.stack(lses)
    B, n = st["lens"].shape
    out = torch.full((B * n, st["max_len"]), -math.inf, dtype=torch.float64, device=DEV)
    for b in range(B):
        raw = st["cache"][st["tables"][b].long()]
        raw = torch.cat([raw[:, :4096].reshape(-1, 64), raw[:, 4096:].reshape(-1, 4)], dim=1)
        for j in range(n):
            L = int(st["lens"][b, j])
            dots = (st["q"][b, j].double() @ _rows64(raw[:L], 128).T).clamp(min=0)
            out[b * n + j, :L] = (st["weights"][b * n + j].double()[:, None] * dots).sum(dim=0)
    return out
