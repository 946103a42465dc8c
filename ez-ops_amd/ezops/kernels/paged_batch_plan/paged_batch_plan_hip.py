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

    def __call__(self, q_lens, past_lens, block_table, free_pages, free_span, out=None):
        from ...ops.paged_batch_plan import PagedBatchPlan

        dev = _hip.require_gpu(q_lens, past_lens, block_table, free_pages, free_span)
        i32, B, T = torch.int32, self.B, self.T
        _hip.check(q_lens, "q_lens", (B,), i32)
        if past_lens is not None:
            _hip.check(past_lens, "past_lens", (B,), i32)
        _hip.check(block_table, "block_table", (B, self.M), i32)
        _hip.check(free_pages, "free_pages", (self.NF,), i32)
        if free_span.dim() != 1 or free_span.numel() < 2:
            raise ValueError(f"free_span: expected (head, tail), got shape {tuple(free_span.shape)}")
        _hip.check(free_span, "free_span", tuple(free_span.shape), i32)
        if out is None:
            out = PagedBatchPlan(torch.empty(B + 1, dtype=i32, device=dev), torch.empty(B, dtype=i32, device=dev),
                                 torch.empty(T, dtype=i32, device=dev), torch.empty(T, dtype=torch.int64, device=dev),
                                 torch.empty(3, dtype=i32, device=dev))
        else:
            if _hip.require_gpu(*out) != dev:
                raise RuntimeError(f"out is not on {dev}")
            _hip.check(out.cu_seqlens, "out.cu_seqlens", (B + 1,), i32)
            _hip.check(out.kv_lens, "out.kv_lens", (B,), i32)
            _hip.check(out.positions, "out.positions", (T,), i32)
            _hip.check(out.slot_mapping, "out.slot_mapping", (T,), torch.int64)
            _hip.check(out.free_span, "out.free_span", (3,), i32)
        _hip.call_on(dev, "ezops_paged_batch_plan", q_lens.data_ptr(), _hip.ptr(past_lens), block_table.data_ptr(),
                     free_pages.data_ptr(), free_span.data_ptr(), out.cu_seqlens.data_ptr(), out.kv_lens.data_ptr(),
                     out.positions.data_ptr(), out.slot_mapping.data_ptr(), out.free_span.data_ptr(), B, T, self.P,
                     self.M, self.NP, self.NF)
        return out
