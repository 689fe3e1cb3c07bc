"""context_fields of a padded batch: requests without new tokens keep a length of 0 for every query token."""
import pytest
import torch

from nanoengine_amd import indexer, ops
from nanoengine_amd.batch_tables import BatchTables
from nanoengine_amd.pipeline import DsaDecodeStep
from oracle import fp4_oracle as F

I32 = torch.int32


@pytest.mark.parametrize("n,lens,want", [(1, [9, 4, 0], [[9], [4], [0]]), (2, [8, 9, 3, 4, 0, 0], [[8, 9], [3, 4], [0, 0]]),
                                         (4, [1, 2, 3, 4, 6, 7, 8, 9, 0, 0, 0, 0], [[1, 2, 3, 4], [6, 7, 8, 9], [0] * 4])])
def test_lengths_expand_to_zero_for_padding(n, lens, want):
    t = BatchTables(3, 3 * n + 2, 4, device="cpu")
    t.seq_lens[:3 * n].copy_(torch.tensor(lens))
    fields = t.context_fields(n)
    assert indexer._expand_decode_context_lens(fields["context_lens"][0], n).tolist() == want
    assert fields["num_tokens_per_seq"] == n and fields["block_tables"].shape == (1, 3, 4)


@pytest.mark.parametrize("n", [1, 2])
def test_step_takes_lengths_of_either_form(n):
    step = DsaDecodeStep.__new__(DsaDecodeStep)     # (expand_lens needs no device)
    step.next_n = n
    per_token = torch.tensor([[7, 8], [1, 2], [0, 0]], dtype=I32)[:, 2 - n:]
    assert step.expand_lens(per_token).tolist() == per_token.reshape(-1).tolist()
    assert step.expand_lens(torch.tensor([8, 1])).tolist() == ([8, 1] if n == 1 else [7, 8, 1, 1])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 3])
@pytest.mark.parametrize("fp4", [True, False])
def test_padding_requests_select_nothing(cuda, n, fp4):
    """Through the tables and the decode selection, over caches of either format."""
    print(f"padded context n={n} fp4={fp4}", flush=True)
    B, blocks = 5, 64
    g = torch.Generator(device=cuda).manual_seed(n)
    tables = BatchTables(B, B * n, 32, device=cuda)
    tables.block_tables.copy_(torch.randperm(blocks, generator=g, device=cuda)[:32].to(I32))  # pages others left behind
    cached = torch.tensor([700, 64 - n, 1300, 0, 0], dtype=I32, device=cuda)
    new = torch.tensor([n, n, n, 0, 0], dtype=I32, device=cuda)
    tables.plan(cached, new)
    fields = tables.context_fields(n)
    keys = torch.randn(blocks * 64, 128, generator=g, device=cuda).to(torch.bfloat16)
    cache = torch.zeros(blocks, 64 * (68 if fp4 else 132), dtype=torch.uint8, device=cuda)
    (ops.indexer_k_store_fp4 if fp4 else ops.indexer_k_store)(keys, cache, torch.arange(blocks * 64, device=cuda), 64)
    q = (torch.randn(B * n, 64, 128, generator=g, device=cuda) * 60).to(torch.float8_e4m3fn)
    w = torch.randn(B * n, 64, generator=g, device=cuda).abs() * 0.01
    logical, physical = indexer.indexer_decode_topk(q, w, cache, fields["context_lens"][0], fields["block_tables"][0], 512,
                                                    translate_topk=True, topk_page_size=64)
    torch.cuda.synchronize()
    assert torch.all(logical[3 * n:] == -1) and torch.all(physical[3 * n:] == -1)
    values = F.key_values(cache) if fp4 else None
    for r in range(3 * n):
        L = int(cached[r // n]) + r % n + 1
        picked = logical[r][logical[r] >= 0].long()
        assert picked.numel() == min(L, 512)
        at = tables.block_tables[r // n].long()[picked // 64] * 64 + picked % 64
        assert torch.equal(physical[r][:picked.numel()].long(), at)
        if fp4:
            t = torch.arange(L, device=cuda)
            slots = tables.block_tables[r // n].long()[t // 64] * 64 + t % 64
            want, tol = F.logits_row(q[r].float(), w[r], values[slots])
            left = torch.ones(L, dtype=torch.bool, device=cuda)
            left[picked] = False
            if left.any():
                assert (want[left] - tol[left]).max() <= (want[picked] + tol[picked]).min()
