"""HIP attention over the 8-bit KV cache (single tokens, packed prompts); no reference counterpart (its attention reads
a contiguous bf16 cache, ezops/ops/attn_decode.py:9-67)."""

import operator

import torch

from ... import _hip
from ...registry import register_kernel
from ..base_kernel import BaseKernel
from ..kv_cache_quant.kv_cache_quant_hip import TYPE_CODES, aligned, pool_specs, rows16


class _QuantAttnKernel(BaseKernel):
    def _setup(self, rows, batch, num_heads, num_kv_heads, head_dim, page_size, max_pages, num_pages, cache_dtype, block_size,
               scale):
        self.B, self.H, self.Hkv, self.D = batch, num_heads, num_kv_heads, head_dim
        self.scale, self.S = scale, max_pages * page_size
        self._q = (rows, num_heads, head_dim)
        self._specs = pool_specs(num_pages, num_kv_heads, page_size, head_dim, block_size, cache_dtype) + (
            ("block_table", (batch, max_pages), torch.int32),)
        self._out = (("out", self._q, torch.bfloat16),)
        self._type = TYPE_CODES[cache_dtype]
        self._pool = (num_pages, page_size, max_pages, block_size)
        self._ws_bytes: dict = {}  # by the library, per bound on the lengths

    def _out_of(self, out, dev):
        if out is None:
            return torch.empty(self._q, dtype=torch.bfloat16, device=dev)
        _hip.check_all(self._out, out)
        aligned(out, "out")
        return out

    def _workspace(self, dev, max_kv_len, name, *shape):
        n = operator.index(max_kv_len if 0 < max_kv_len < self.S else self.S)
        step = 1 << max(7, n.bit_length() - 4)
        bound = -(-n // step) * step  # a size is enough for smaller bounds: a few of them serve all
        n = self._ws_bytes.get(bound)
        if n is None:
            n = self._ws_bytes[bound] = _hip.size(name, *shape, bound)
        # from torch's allocator at every call: stream-ordered, and a captured graph keeps its own
        return (torch.empty(n, dtype=torch.uint8, device=dev) if n else None), n


@register_kernel("quant_paged_attn_decode", "hip", family="kv8")
class QuantPagedAttnDecodeHipKernel(_QuantAttnKernel):
    def __init__(self, batch: int, num_heads: int, num_kv_heads: int, head_dim: int, page_size: int, max_pages: int,
                 num_pages: int, *, cache_dtype: torch.dtype, block_size: int, scale: float):
        self._setup(batch, batch, num_heads, num_kv_heads, head_dim, page_size, max_pages, num_pages, cache_dtype, block_size,
                    scale)
        self._specs += (("kv_lens", (batch,), torch.int32),)

    def __call__(self, q, K_cache, V_cache, K_scale, V_scale, block_table, kv_lens, max_kv_len: int = 0, *, out=None):
        if max_kv_len < 0:
            raise ValueError(f"max_kv_len ({max_kv_len}) must be >= 0")
        dev = _hip.one_gpu(q, K_cache, V_cache, K_scale, V_scale, block_table, kv_lens, out)
        q_rs = rows16(q, "q", self._q)
        _hip.check_all(self._specs, K_cache, V_cache, K_scale, V_scale, block_table, kv_lens)
        out = self._out_of(out, dev)
        ws, n = self._workspace(dev, max_kv_len, "ezops_quant_paged_attn_decode_workspace_size", self.B, self.H, self.Hkv,
                                self.D)
        _hip.call_on(dev, "ezops_quant_paged_attn_decode_bf16", q.data_ptr(), q_rs, K_cache.data_ptr(), V_cache.data_ptr(),
                     K_scale.data_ptr(), V_scale.data_ptr(), self._type, block_table.data_ptr(), kv_lens.data_ptr(),
                     out.data_ptr(), self.B, self.H, self.Hkv, self.D, *self._pool, max_kv_len, self.scale, _hip.ptr(ws), n)
        return out


@register_kernel("quant_prefill_attn", "hip", family="kv8")
class QuantPrefillAttnHipKernel(_QuantAttnKernel):
    def __init__(self, batch: int, num_tokens: int, num_heads: int, num_kv_heads: int, head_dim: int, page_size: int,
                 max_pages: int, num_pages: int, *, cache_dtype: torch.dtype, block_size: int, scale: float):
        self._setup(num_tokens, batch, num_heads, num_kv_heads, head_dim, page_size, max_pages, num_pages, cache_dtype,
                    block_size, scale)
        self.T = num_tokens
        self._specs += (("cu_seqlens", (batch + 1,), torch.int32),)
        self._past = (("past_lens", (batch,), torch.int32),)

    def __call__(self, q, K_cache, V_cache, K_scale, V_scale, block_table, cu_seqlens, past_lens=None, *,
                 max_kv_len: int = 0, out=None):
        if max_kv_len < 0:
            raise ValueError(f"max_kv_len ({max_kv_len}) must be >= 0")
        dev = _hip.one_gpu(q, K_cache, V_cache, K_scale, V_scale, block_table, cu_seqlens, past_lens, out)
        q_rs = rows16(q, "q", self._q)
        _hip.check_all(self._specs, K_cache, V_cache, K_scale, V_scale, block_table, cu_seqlens)
        if past_lens is not None:
            _hip.check_all(self._past, past_lens)
        out = self._out_of(out, dev)
        ws, n = self._workspace(dev, max_kv_len, "ezops_quant_prefill_attn_workspace_size", self.B, self.T, self.H, self.Hkv,
                                self.D)
        _hip.call_on(dev, "ezops_quant_prefill_attn_bf16", q.data_ptr(), q_rs, K_cache.data_ptr(), V_cache.data_ptr(),
                     K_scale.data_ptr(), V_scale.data_ptr(), self._type, block_table.data_ptr(), cu_seqlens.data_ptr(),
                     _hip.ptr(past_lens), out.data_ptr(), self.B, self.T, self.H, self.Hkv, self.D, *self._pool, max_kv_len,
                     self.scale, _hip.ptr(ws), n)
        return out
