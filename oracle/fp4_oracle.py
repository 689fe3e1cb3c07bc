"""64-bit restatements of the 4-bit caches and of the tables that address them.

Written from the definitions, in torch float64 so that they run on either
device: the e2m1 block format, the two cache layouts, sparse attention and
indexer logits over them, each with the bound of its kernel's rounding, and the
batch tables in plain Python integers.
"""
from __future__ import annotations

import torch

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MIN_EXP, MAX_EXP, NAN_BYTE = -40, 125, 255
MLA_ROW, KEY_BYTES = 400, 68


def fp4_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """[N, 32k] -> (packed codes uint8 [N, 16k], scale bytes uint8 [N, k])."""
    b = x.double().reshape(x.shape[0], -1, 32)
    nan = torch.isnan(b).any(dim=-1)
    mag = torch.nan_to_num(b.abs(), nan=0.0, posinf=2.0 ** 130)
    top = mag.amax(dim=-1)
    # the smallest k in [-40, 125] with amax <= 6 * 2^k, by comparison with every candidate
    ks = torch.arange(MIN_EXP, MAX_EXP + 1, device=x.device)
    fits = top[..., None] <= 6.0 * torch.exp2(ks.double())
    k = torch.where(fits.any(dim=-1), MIN_EXP + fits.int().argmax(dim=-1), MAX_EXP)
    y = mag / torch.exp2(k.double())[..., None]
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    d = (y[..., None] - grid).abs()
    odd = torch.arange(8, device=x.device) % 2
    code = torch.where(d == d.amin(dim=-1, keepdim=True), odd, 2).argmin(dim=-1)
    code = code + 8 * torch.signbit(b).long()
    code = torch.where(nan[..., None], 0, code).reshape(x.shape[0], -1)
    byte = torch.where(nan, NAN_BYTE, k + 127)
    return (code[:, 0::2] | (code[:, 1::2] << 4)).to(torch.uint8), byte.to(torch.uint8)


def fp4_values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """Packed codes [..., n] and scale bytes [..., n/16] -> float64 [..., 2n]."""
    grid = torch.tensor(GRID + tuple(-g for g in GRID), dtype=torch.float64, device=codes.device)
    c = codes.long()
    v = torch.stack([grid[c & 15], grid[c >> 4]], dim=-1).flatten(-2)
    s = torch.where(scales == NAN_BYTE, float("nan"), torch.exp2(scales.double() - 127.0))
    return v * s.repeat_interleave(32, dim=-1)


# ------------------------------------------------------------------ cache layouts
def mla_rows(kv: torch.Tensor) -> torch.Tensor:
    """[N, 576] bf16 -> [N, 400] uint8 rows."""
    codes, scales = fp4_quantize(kv[:, :512].float())
    return torch.cat([codes, scales, kv[:, 512:].contiguous().view(torch.uint8).view(-1, 128)], dim=1)


def mla_values(rows: torch.Tensor) -> torch.Tensor:
    """[N, 400] uint8 rows -> [N, 576] float64."""
    rope = rows[:, 272:].contiguous().view(torch.bfloat16).double().view(-1, 64)
    return torch.cat([fp4_values(rows[:, :256], rows[:, 256:272]), rope], dim=1)


def key_pages(keys: torch.Tensor, page_size: int = 64) -> torch.Tensor:
    """[pages * page_size, 128] -> [pages, page_size * 68] uint8."""
    codes, scales = fp4_quantize(keys.float())
    return torch.cat([codes.view(-1, page_size * 64), scales.view(-1, page_size * 4)], dim=1)


def key_values(pages: torch.Tensor, page_size: int = 64) -> torch.Tensor:
    """[pages, page_size * 68] uint8 -> [pages * page_size, 128] float64."""
    return fp4_values(pages[:, :page_size * 64].reshape(-1, 64), pages[:, page_size * 64:].reshape(-1, 4))


# ------------------------------------------------------------------ attention
def attend(q: torch.Tensor, keys: torch.Tensor, scale: float):
    """One token: q [H, 576], its valid keys [n, 576] float64 -> (o [H, 512], lse [H], o_tol, lse_tol).

    The bounds: a score's product terms are exact, their f32 sum of 576 is off by at
    most 576 roundings of the running sum, each below 2^-23 (truncation) of sum |q k|;
    scaling, the exponential's argument and the logarithm add a few roundings of |s|
    and of 1. A probability is rounded to bf16 (2^-8) and carries its score's error
    twice (numerator and sum); the output is rounded to bf16 once more."""
    q = q.double()
    if keys.shape[0] == 0:
        z = torch.zeros(q.shape[0], 512, dtype=torch.float64, device=q.device)
        return z, torch.full_like(z[:, 0], float("-inf")), z, z[:, 0]
    s = scale * (q @ keys.T)
    p = torch.softmax(s, dim=1)
    o = p @ keys[:, :512]
    lse = torch.logsumexp(s, dim=1)
    mass = scale * (q.abs() @ keys.abs().T)
    ds = (576 * mass.amax(dim=1) + 8 * s.abs().amax(dim=1) + 16) * 2.0 ** -23
    spread = p @ keys[:, :512].abs()
    n32 = keys.shape[0] * 2.0 ** -23  # f32 sums over the keys
    o_tol = spread * (2.0 ** -8 + 2 * ds[:, None] + 2 * n32 + 2.0 ** -20) * 1.01 + o.abs() * 2.0 ** -8
    return o, lse, o_tol, ds + n32 + 2.0 ** -20


def logits_row(q: torch.Tensor, w: torch.Tensor, keys: torch.Tensor):
    """q [64, 128], w [64], keys [n, 128] float64 -> (logits [n], tol [n]): exact products, a f32 sum of
    128 (2^-23 of sum |q k| a step), then a f32 sum of 64 weighted heads."""
    q, w = q.double(), w.double()
    dot = q @ keys.T
    mass = q.abs() @ keys.abs().T
    logit = (w[:, None] * dot.clamp(min=0)).sum(dim=0)
    tol = (w.abs()[:, None] * mass * (128 + 66) * 2.0 ** -23).sum(dim=0)
    return logit, tol


# ------------------------------------------------------------------ tables
def batch_tables(cached, new, tables, page, rows, free=None, head=0):
    """Lists of ints in, lists of ints out: (tables, slots, positions, seq_lens, cu_q, cu_k, status). ``tables``:
    a list of rows. Faulty requests are taken as empty; fault bits as the C header lists them."""
    tables = [list(r) for r in tables]
    width = len(tables[0]) if tables else 0
    fault, taken, longest = 0, 0, 0
    slots, positions, cu_q, cu_k, wanted = [], [], [0], [0], []
    for b, (c, n) in enumerate(zip(cached, new)):
        if c < 0 or n < 0 or c + n >= 2 ** 31:
            fault, c, n = fault | 1, 0, 0
        old, total = -(-c // page), -(-(c + n) // page)
        if n > 0 and total > width:
            fault |= 2
        for j in range(n):
            pos, r = c + j, len(slots)
            pg = pos // page
            block = -1
            if pg < width:
                if free is None or pg < old:
                    block = tables[b][pg]
                else:
                    at = head + taken + pg - old
                    if 0 <= at < len(free):
                        block = free[at]
                        if r < rows:
                            tables[b][pg] = block
            slots.append(block * page + pos % page if block >= 0 else -1)
            positions.append(pos)
        if free is not None:
            taken += total - old
        longest = max(longest, c + n)
        cu_q.append(cu_q[-1] + n)
        cu_k.append(cu_k[-1] + c + n)
    if free is not None and taken and (head < 0 or head + taken > len(free)):
        fault |= 4
    total = len(slots)
    if total > rows:
        fault |= 8
    pad = max(0, rows - total)
    seq = [p + 1 for p in positions]
    return (tables, slots[:rows] + [-1] * pad, positions[:rows] + [0] * pad, seq[:rows] + [0] * pad, cu_q, cu_k,
            [fault, total, taken, longest])
