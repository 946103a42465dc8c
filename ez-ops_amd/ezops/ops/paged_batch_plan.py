"""Batch plan of a ragged serving step over a paged cache, from request lengths.

No reference counterpart (the reference's cache is one contiguous tensor,
ezops/ops/attn_decode.py:60-61): this op makes, on the GPU and in one launch,
what the paged ops of this package take.  Sequence ``b`` brings ``q_lens[b]``
new tokens on top of ``past_lens[b]`` cached rows; the new tokens of all
sequences lie back to back in ``num_tokens`` rows (fewer may be used: a batch
padded to a captured size).  The result:

    cu_seqlens [B + 1]    first row of every sequence, then the rows used
    kv_lens [B]           past + new tokens (at most max_pages * page_size)
    positions [T]         position of every row, -1 behind the last token
    slot_mapping [T]      int64 cache slot page * page_size + offset, -1 where
                          there is none (no token, no page, no room)
    free_span [3]         (head behind the pages taken, tail, pages needed)

and ``block_table [B, max_pages]`` gets, in place, the pages that the new
tokens begin: taken in order from ``free_pages`` between head and tail
(``free_span``), sequence 0's first.  Entries of cached pages are read and kept,
entries behind the last page are left alone.  A list that ends too early, or an
id outside the pool, gives entries and slots of -1; ``free_span[2] >
tail - head`` says so.  ``free_span`` (the input) is not changed, so the same
inputs give the same plan; the next step is called with the result's.
"""

from typing import NamedTuple

import torch

from ..registry import get_kernel
from .base_op import Op, default_device
from .utils.roofline import RooflineResult


class PagedBatchPlan(NamedTuple):
    cu_seqlens: torch.Tensor    # [B + 1] int32
    kv_lens: torch.Tensor       # [B] int32
    positions: torch.Tensor     # [T] int32
    slot_mapping: torch.Tensor  # [T] int64
    free_span: torch.Tensor     # [3] int32: head behind the pages taken, tail, pages needed


class PagedBatchPlanOp(Op):
    _params_desc = {
        "batch": "Sequences in the step (at most 4096)",
        "num_tokens": "Rows for new tokens, all sequences together",
        "page_size": "Cache rows per page (power of two >= 32)",
        "max_pages": "Block-table width (pages per sequence)",
        "num_pages": "Pages in the shared pool",
        "num_free": "Length of the free list (default num_pages)",
    }
    _atol = 0
    _rtol = 0

    def __init__(self, batch: int, num_tokens: int, page_size: int, max_pages: int, num_pages: int,
                 num_free: int | None = None, backend: str = "ref"):
        if not 1 <= batch <= 4096:
            raise ValueError(f"batch ({batch}) must be in [1, 4096]")
        if not 1 <= num_tokens < 1 << 30:
            raise ValueError(f"num_tokens ({num_tokens}) must be in [1, 2^30)")
        if not 32 <= page_size <= 1 << 20 or page_size & (page_size - 1):
            raise ValueError(f"page_size ({page_size}) must be a power of two in [32, 2^20]")
        if max_pages < 1 or max_pages * page_size > 1 << 30:
            raise ValueError(f"max_pages ({max_pages}) must be >= 1 and max_pages * page_size at most 2^30")
        if not 1 <= num_pages < 1 << 31:
            raise ValueError(f"num_pages ({num_pages}) must be in [1, 2^31)")
        num_free = num_pages if num_free is None else num_free
        if not 0 <= num_free < 1 << 30:
            raise ValueError(f"num_free ({num_free}) must be in [0, 2^30)")
        self.batch, self.num_tokens, self.page_size, self.max_pages = batch, num_tokens, page_size, max_pages
        self.num_pages, self.num_free = num_pages, num_free
        self._backend = backend
        if backend != "ref":
            self._kernel = get_kernel("paged_batch_plan", backend)(batch, num_tokens, page_size, max_pages, num_pages,
                                                                   num_free)
        else:
            self._kernel = self._ref_forward

    def forward(self, q_lens, past_lens, block_table, free_pages, free_span, out=None) -> PagedBatchPlan:
        """``free_span`` [2] or more (a result's [3] serves); ``past_lens`` None = 0; ``out``: a plan to write into."""
        return self._kernel(q_lens, past_lens, block_table, free_pages, free_span, out)

    def alloc(self, device=None) -> PagedBatchPlan:
        """Buffers for ``out``: static ones for a captured step."""
        dev = default_device(device)
        i32 = dict(dtype=torch.int32, device=dev)
        return PagedBatchPlan(torch.empty(self.batch + 1, **i32), torch.empty(self.batch, **i32),
                              torch.empty(self.num_tokens, **i32),
                              torch.empty(self.num_tokens, dtype=torch.int64, device=dev), torch.empty(3, **i32))

    def gen_data(self, device=None):
        """Random lengths that fit rows, table and pool; cached pages and the free list partition the pool."""
        dev = default_device(device)
        B, P, M = self.batch, self.page_size, self.max_pages
        each = max(1, min(self.num_pages // B, M))  # pages a sequence may hold in the end
        new = torch.randint(0, max(1, min(self.num_tokens // B, each * P)) + 1, (B,))
        past = (torch.rand(B) * (each * P - new + 1).clamp(min=1)).long()
        have = (past + P - 1) // P
        order = torch.randperm(self.num_pages)
        table = torch.full((B, M), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(have.tolist()):
            table[b, :n] = order[at:at + n]
            at += n
        free = torch.zeros(self.num_free, dtype=torch.int32)
        rest = order[at:at + self.num_free]
        free[:rest.numel()] = rest.to(torch.int32)
        span = torch.tensor([0, rest.numel()], dtype=torch.int32)
        return tuple(x.to(torch.int32).to(dev) for x in (new, past, table, free, span))

    def get_roofline(self) -> RooflineResult:
        b = 4 * (2 * self.batch + 2 + 2 * self.batch + 1 + 3) + 12 * self.num_tokens
        return RooflineResult(0, b, b)

    def check(self, actual, expected) -> bool:
        return all(a.dtype == e.dtype and torch.equal(a, e) for a, e in zip(actual, expected, strict=True))

    def _ref_forward(self, q_lens, past_lens, block_table, free_pages, free_span, out=None):
        """Token by token, as an allocator on the host would do it."""
        B, T, P, M = self.batch, self.num_tokens, self.page_size, self.max_pages
        dev = block_table.device
        new = [max(0, n) for n in q_lens.tolist()]
        past = [min(max(0, n), M * P) for n in (past_lens.tolist() if past_lens is not None else [0] * B)]
        table, free = block_table.tolist(), free_pages.tolist()
        head, tail = free_span.tolist()[:2]
        last = min(tail, self.num_free) if head >= 0 else head
        ok = lambda i: 0 <= i < self.num_pages  # noqa: E731
        cu, kv, pos, slots, needed = [0], [], [], [], 0
        for b in range(B):
            n = min(new[b], T - cu[-1])
            for p in range(past[b], past[b] + n):
                j = p // P
                pos.append(p)
                if p >= M * P:
                    slots.append(-1)
                    continue
                if p % P == 0:
                    i = free[head + needed] if head + needed < last else -1
                    table[b][j] = i if ok(i) else -1
                    needed += 1
                slots.append(table[b][j] * P + p % P if ok(table[b][j]) else -1)
            cu.append(cu[-1] + n)
            kv.append(min(past[b] + n, M * P))
        pad = [-1] * (T - len(pos))
        span = [head + min(needed, max(last - head, 0)), tail, needed]
        block_table.copy_(torch.tensor(table, dtype=torch.int32))
        got = PagedBatchPlan(*(torch.tensor(x, dtype=torch.int32, device=dev) for x in (cu, kv, pos + pad)),
                             torch.tensor(slots + pad, dtype=torch.int64, device=dev),
                             torch.tensor(span, dtype=torch.int32, device=dev))
        if out is None:
            return got
        for o, g in zip(out, got):
            o.copy_(g)
        return out
