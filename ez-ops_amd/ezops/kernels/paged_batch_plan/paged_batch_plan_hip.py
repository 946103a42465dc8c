"""HIP batch plan (block table, slot map, positions, offsets from request lengths); no reference counterpart
(the reference's cache is contiguous, ezops/ops/attn_decode.py:60-61)."""

import torch

from ... import _hip
from ...registry import register_kernel
from ..base_kernel import BaseKernel


@register_kernel("paged_batch_plan", "hip", family="ragged")
class PagedBatchPlanHipKernel(BaseKernel):
    def __init__(self, batch: int, num_tokens: int, page_size: int, max_pages: int, num_pages: int, num_free: int):
        self.B, self.T, self.P, self.M, self.NP, self.NF = batch, num_tokens, page_size, max_pages, num_pages, num_free
        i32, i64 = torch.int32, torch.int64
        self._in = (("q_lens", (batch,), i32), ("block_table", (batch, max_pages), i32), ("free_pages", (num_free,), i32))
        self._past = (("past_lens", (batch,), i32),)
        self._out = (("out.cu_seqlens", (batch + 1,), i32), ("out.kv_lens", (batch,), i32),
                     ("out.positions", (num_tokens,), i32), ("out.slot_mapping", (num_tokens,), i64),
                     ("out.free_span", (3,), i32))

    def __call__(self, q_lens, past_lens, block_table, free_pages, free_span, out=None):
        given = out is not None
        if given:
            cu, kv, positions, slots, span = out
            dev = _hip.one_gpu(q_lens, past_lens, block_table, free_pages, free_span, cu, kv, positions, slots, span)
            _hip.check_all(self._out, cu, kv, positions, slots, span)
        else:
            dev = _hip.one_gpu(q_lens, past_lens, block_table, free_pages, free_span)
        _hip.check_all(self._in, q_lens, block_table, free_pages)
        if past_lens is not None:
            _hip.check_all(self._past, past_lens)
        if free_span.dtype is not torch.int32 or free_span.dim() != 1 or free_span.shape[0] < 2 or free_span.stride(0) != 1:
            raise ValueError("free_span: expected a contiguous int32 tensor of two or more (head, tail), got shape "
                             f"{tuple(free_span.shape)}, {free_span.dtype}")
        if not given:
            from ...ops.paged_batch_plan import PagedBatchPlan

            cu, kv, positions, slots, span = out = PagedBatchPlan(
                *(torch.empty(shape, dtype=dtype, device=dev) for _, shape, dtype in self._out))
        _hip.call_on(dev, "ezops_paged_batch_plan", q_lens.data_ptr(), None if past_lens is None else past_lens.data_ptr(),
                     block_table.data_ptr(), free_pages.data_ptr(), free_span.data_ptr(), cu.data_ptr(), kv.data_ptr(),
                     positions.data_ptr(), slots.data_ptr(), span.data_ptr(), self.B, self.T, self.P, self.M, self.NP,
                     self.NF)
        return out
