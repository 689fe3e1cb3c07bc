"""Block tables and slot maps of a running batch, built on the device from its requests' lengths.

The reference's scheduler builds them on the host and ships them with every step
(BatchContext's ``block_tables`` and ``slot_mapping``, dlengine/runtime/context/batch.py:10-80).
Here one launch extends the block tables, maps the new tokens to cache slots and
forms the ragged offsets, so that a step whose lengths live on the device (a
captured graph, a speculative decode) needs no host round trip.
"""
from __future__ import annotations

import torch

from . import ops

_FAULTS = {1: "a request's length is negative or passes int32", 2: "a request has more pages than its block table",
           4: "the free list is too short", 8: "more new tokens than rows", 16: "a prefix sum does not fit int32"}


class BatchTables:
    """The tables of up to ``batch`` requests and ``num_rows`` new tokens a step, in
    buffers of their own (allocated once, as a captured graph wants them):
    ``block_tables`` [batch, table_width], ``slot_mapping`` / ``positions`` /
    ``seq_lens`` [num_rows], ``cu_seqlens_q`` / ``cu_seqlens_k`` [batch + 1], ``status`` [4]."""

    def __init__(self, batch: int, num_rows: int, table_width: int, page_size: int = 64, device="cuda",
                 slot_dtype: torch.dtype = torch.int64):
        self.batch, self.num_rows, self.page_size = batch, num_rows, page_size
        dev = torch.device(device)
        i32 = torch.int32
        self.block_tables = torch.zeros(batch, table_width, dtype=i32, device=dev)
        self.slot_mapping = torch.full((num_rows,), -1, dtype=slot_dtype, device=dev)
        self.positions = torch.zeros(num_rows, dtype=slot_dtype, device=dev)
        self.seq_lens = torch.zeros(num_rows, dtype=i32, device=dev)
        self.cu_seqlens_q = torch.zeros(batch + 1, dtype=i32, device=dev)
        self.cu_seqlens_k = torch.zeros(batch + 1, dtype=i32, device=dev)
        self.status = torch.zeros(4, dtype=torch.int64, device=dev)

    def plan(self, cached_lens: torch.Tensor, new_lens: torch.Tensor, free_blocks: torch.Tensor | None = None,
             free_head: torch.Tensor | None = None) -> "BatchTables":
        """Fill the buffers for requests of ``cached_lens`` cached and ``new_lens`` new tokens (int32 [batch]),
        taking the blocks of newly opened pages from ``free_blocks`` (see ``ops.batch_tables``). Launches
        only; ``check`` reports what went wrong."""
        ops.batch_tables(cached_lens, new_lens, self.block_tables, self.page_size, self.slot_mapping, self.status,
                         free_blocks=free_blocks, free_head=free_head, positions=self.positions,
                         seq_lens=self.seq_lens, cu_seqlens_q=self.cu_seqlens_q, cu_seqlens_k=self.cu_seqlens_k)
        return self

    def check(self) -> tuple[int, int, int]:
        """Read the last plan's status (synchronises): (new tokens, blocks taken, longest request), or
        RuntimeError naming its faults. A new token without a cache slot is one too: it counts in the lengths,
        but its row is not written."""
        lost = ((self.slot_mapping < 0) & (self.seq_lens > 0)).sum()
        faults, tokens, taken, longest, lost = torch.cat([self.status, lost.view(1)]).tolist()
        what = [m for bit, m in _FAULTS.items() if faults & bit]
        if lost and not what:
            what.append(f"{lost} new tokens have no cache slot (a negative block number, or a slot that passes "
                        f"{str(self.slot_mapping.dtype).replace('torch.', '')})")
        if what:
            raise RuntimeError("batch tables: " + "; ".join(what))
        return tokens, taken, longest

    def context_fields(self, num_tokens_per_seq: int = 1) -> dict:
        """The fields of ``mla_backend.BatchContext`` for a decode step of ``num_tokens_per_seq`` new tokens a
        request: tables, slot mapping and lengths. ``context_lens`` is [1, batch] for one new token, each request's
        length after the step, and [1, batch, num_tokens_per_seq] for more, each query token's own. Requests that
        pad the batch have no new tokens and come last; their lengths are 0. (A final length alone would not do
        for several tokens: its expansion to one length a token starts at 1.)"""
        n = num_tokens_per_seq
        if self.num_rows < self.batch * n:
            raise ValueError(f"{self.num_rows} rows cannot hold {n} tokens of {self.batch} requests")
        lens = self.seq_lens[: self.batch * n]
        return {"is_prefill": False, "context_lens": (lens if n == 1 else lens.view(self.batch, n)).unsqueeze(0),
                "block_tables": self.block_tables.unsqueeze(0), "slot_mapping": self.slot_mapping,
                "num_tokens_per_seq": n}
