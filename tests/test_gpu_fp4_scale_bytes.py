"""Scale bytes that the writers never store (theirs are 87 to 252 and 255) are read as the format defines them.

value = code * 2^(byte - 127). Up to byte 252 that is a bf16 number for every code, subnormal ones among them;
at 253 and 254 the codes of 4 and more, and of 2 and more, pass bf16's range and read as infinities."""
import pytest
import torch

from nanoengine_amd import ops
from oracle import fp4_oracle as F

pytestmark = pytest.mark.gpu
BYTES = [0, 1, 2, 3, 60, 86, 127, 251, 252, 253, 254, 255]


def _codes(device):
    """16 bytes: every code twice."""
    c = torch.arange(16, dtype=torch.uint8, device=device)
    return (c[0::2] | (c[1::2] << 4)).repeat(2)


def test_mla_rows(cuda):
    rows = torch.zeros(len(BYTES), 400, dtype=torch.uint8, device=cuda)
    rows[:, :256] = _codes(cuda).repeat(16)
    rows[:, 256:272] = torch.tensor(BYTES, dtype=torch.uint8, device=cuda)[:, None]
    back = ops.mla_kv_load_fp4(rows[None], torch.arange(len(BYTES), device=cuda))
    want = F.mla_values(rows)
    torch.cuda.synchronize()
    for i, byte in enumerate(BYTES):
        nope = back[i, :512].double()
        if byte == 255:
            assert torch.all(torch.isnan(nope))
        elif byte <= 252:
            assert torch.equal(nope, want[i, :512]), byte
        else:
            past = want[i, :512].abs() >= 2.0 ** 128
            assert past.any() and torch.equal(nope[~past], want[i, :512][~past])
            assert torch.equal(nope[past], want[i, :512][past].sign() * float("inf"))


def test_indexer_keys(cuda):
    """Key and scale are exact for every byte: the pair holds what a bf16 number would not."""
    pages = torch.zeros(1, 64 * 68, dtype=torch.uint8, device=cuda)
    n = len(BYTES)
    pages[0, :n * 64] = _codes(cuda).repeat(4 * n)
    pages[0, 64 * 64:64 * 64 + 4 * n] = torch.tensor(BYTES, dtype=torch.uint8, device=cuda).repeat_interleave(4)
    keys, scales = ops.indexer_k_load_fp4(pages, torch.arange(n, device=cuda), 64)
    torch.cuda.synchronize()
    got, want = keys.double() * scales.double()[:, None], F.key_values(pages)[:n]
    assert torch.equal(got[:-1], want[:-1]) and torch.all(torch.isnan(got[-1]))


@pytest.mark.parametrize("n", [1, 2])
def test_logits_of_subnormal_keys(cuda, n):
    """Keys of bytes 0 to 3. The products are f32 numbers near its smallest normal one, below which a sum may drop
    what it is given: 2^-126 a product and a weighted head at most."""
    g = torch.Generator(device=cuda).manual_seed(n)
    pages = torch.randint(0, 256, (3, 64 * 68), generator=g, device=cuda).to(torch.uint8)
    pages[:, 64 * 64:] = torch.randint(0, 4, (3, 256), generator=g, device=cuda).to(torch.uint8)
    q = (torch.randn(1, n, 64, 128, generator=g, device=cuda) * 60).to(torch.float8_e4m3fn)
    w = torch.randn(n, 64, generator=g, device=cuda)
    lens = torch.tensor([[192 - n + 1 + j for j in range(n)]], dtype=torch.int32, device=cuda)
    got = ops.indexer_logits_fp4(q, pages, w, lens, torch.tensor([[1, 2, 0]], dtype=torch.int32, device=cuda), 192)
    torch.cuda.synchronize()
    values = F.key_values(pages[[1, 2, 0]])
    for j in range(n):
        L = int(lens[0, j])
        want, tol = F.logits_row(q[0, j].float(), w[j], values[:L])
        drop = (w[j].abs().double().sum() * 128 + 64) * 2.0 ** -126
        assert torch.any(want.abs() > tol + drop)       # (keys taken as zeros would be seen)
        assert torch.all((got[j, :L].double() - want).abs() <= tol + drop)
