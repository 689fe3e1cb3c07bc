"""Sparse MLA prefill where the first keys score -inf for some heads and +inf for others (an infinite rope value):
a key at -inf weighs nothing, and the head's result is that of its other keys."""
import pytest
import torch

from nanoengine_amd import ops

pytestmark = pytest.mark.gpu
SCALE = 192 ** -0.5


@pytest.mark.parametrize("H", [16, 64, 128])
@pytest.mark.parametrize("first", [32, 64])
def test_keys_at_minus_infinity_come_first(cuda, H, first):
    print(f"mla prefill infinite H={H} first={first}", flush=True)
    g = torch.Generator(device=cuda).manual_seed(H + first)
    T, N = 5, 1500
    kv = torch.randn(N, 576, generator=g, device=cuda).to(torch.bfloat16)
    kv[:100, 512] = float("inf")
    q = torch.randn(T, H, 576, generator=g, device=cuda)
    q[..., 512] = (q[..., 512].abs() + 0.1) * torch.where(torch.arange(H, device=cuda) % 2 == 0, -1.0, 1.0)
    q = q.to(torch.bfloat16)
    idx = torch.randint(100, N, (T, 256), generator=g, device=cuda)
    idx[:, :first] = torch.randint(0, 100, (T, first), generator=g, device=cuda)
    idx[1, 3:70] = -1
    idx[2] = torch.randint(0, 100, (256,), generator=g, device=cuda)   # nothing else
    o, mx, lse = ops.sparse_mla_prefill(q, kv, idx.to(torch.int32), SCALE)
    torch.cuda.synchronize()
    assert torch.all(torch.isnan(o[:, 1::2]))
    assert torch.all(o[2, 0::2] == 0) and torch.all(torch.isneginf(lse[2, 0::2])) and torch.all(torch.isneginf(mx[2, 0::2]))
    for t in (0, 1, 3, 4):
        at = idx[t][idx[t] >= 100]
        keys, qd = kv[at].double(), q[t, 0::2].double()
        s = SCALE * (qd @ keys.T)
        p = torch.softmax(s, dim=1)
        # scores: f32 sums of 576 exact products, 2^-23 of sum |q k| a step, and a few roundings of the score; a
        # probability is rounded to bf16 (2^-8) and carries its score's error twice, the output rounded to bf16 (2^-8)
        ds = (576 * SCALE * (qd.abs() @ keys.abs().T).amax(dim=1) + 8 * s.abs().amax(dim=1) + 16) * 2.0 ** -23
        spread, eo = p @ keys[:, :512].abs(), p @ keys[:, :512]
        tol = spread * (2.0 ** -8 + 2 * ds[:, None] + 2.0 ** -14) * 1.01 + eo.abs() * 2.0 ** -8
        assert torch.all((o[t, 0::2].double() - eo).abs() <= tol), t
        assert torch.all((lse[t, 0::2].double() - torch.logsumexp(s, dim=1)).abs() <= ds + 2.0 ** -14)
        assert torch.all((mx[t, 0::2].double() - s.amax(dim=1)).abs() <= ds)
