"""HIP cache rows into 8 bits and back; no reference counterpart (its cache is bf16, ezops/ops/attn_decode.py:60-61)."""

import torch

from ... import _hip
from ...registry import register_kernel
from ..base_kernel import BaseKernel

TYPE_CODES = {torch.int8: 0, torch.float8_e4m3fn: 1}


def pool_specs(num_pages, num_kv_heads, page_size, head_dim, block_size, cache_dtype):
    """(name, shape, dtype) of K_cache, V_cache, K_scale and V_scale."""
    codes, scales = (num_pages, num_kv_heads, page_size, head_dim), (num_pages, num_kv_heads, page_size // block_size)
    return (("K_cache", codes, cache_dtype), ("V_cache", codes, cache_dtype), ("K_scale", scales, torch.uint8),
            ("V_scale", scales, torch.uint8))


def aligned(t, name):
    if t.data_ptr() % 16:
        raise ValueError(f"{name}: must begin at a multiple of 16 bytes")


def rows16(t, name, shape):
    """Row stride of a bf16 operand; the kernels read it 16 bytes at a time."""
    rs = _hip.check_rows(t, name, shape, torch.bfloat16)
    if rs % 8 or t.data_ptr() % 16:
        raise ValueError(f"{name}: rows must begin at multiples of 16 bytes")
    return rs


class _CacheRowsKernel(BaseKernel):
    def __init__(self, num_tokens: int, num_kv_heads: int, head_dim: int, page_size: int, num_pages: int, *,
                 cache_dtype: torch.dtype, block_size: int):
        self.T, self.Hkv, self.D = num_tokens, num_kv_heads, head_dim
        self._kv = (num_tokens, num_kv_heads, head_dim)
        self._specs = pool_specs(num_pages, num_kv_heads, page_size, head_dim, block_size, cache_dtype) + (
            ("slot_mapping", (num_tokens,), torch.int64),)
        self._out = (("k_out", self._kv, torch.bfloat16), ("v_out", self._kv, torch.bfloat16))
        self._pool = (TYPE_CODES[cache_dtype], num_pages, page_size, block_size)


@register_kernel("kv_cache_quant", "hip", family="kv8")
class KvCacheQuantHipKernel(_CacheRowsKernel):
    def __call__(self, k, v, K_cache, V_cache, K_scale, V_scale, slot_mapping):
        dev = _hip.one_gpu(k, v, K_cache, V_cache, K_scale, V_scale, slot_mapping)
        k_rs, v_rs = rows16(k, "k", self._kv), rows16(v, "v", self._kv)
        _hip.check_all(self._specs, K_cache, V_cache, K_scale, V_scale, slot_mapping)
        _hip.call_on(dev, "ezops_kv_cache_quant_bf16", k.data_ptr(), k_rs, v.data_ptr(), v_rs, slot_mapping.data_ptr(),
                     K_cache.data_ptr(), V_cache.data_ptr(), K_scale.data_ptr(), V_scale.data_ptr(), *self._pool, self.T,
                     self.Hkv, self.D)
        return K_cache, V_cache, K_scale, V_scale


@register_kernel("kv_cache_dequant", "hip", family="kv8")
class KvCacheDequantHipKernel(_CacheRowsKernel):
    def __call__(self, K_cache, V_cache, K_scale, V_scale, slot_mapping, *, k_out=None, v_out=None):
        dev = _hip.one_gpu(K_cache, V_cache, K_scale, V_scale, slot_mapping, k_out, v_out)
        _hip.check_all(self._specs, K_cache, V_cache, K_scale, V_scale, slot_mapping)
        if k_out is None:
            k_out = torch.empty(self._kv, dtype=torch.bfloat16, device=dev)
        if v_out is None:
            v_out = torch.empty(self._kv, dtype=torch.bfloat16, device=dev)
        _hip.check_all(self._out, k_out, v_out)
        aligned(k_out, "k_out")
        aligned(v_out, "v_out")
        _hip.call_on(dev, "ezops_kv_cache_dequant_bf16", K_cache.data_ptr(), V_cache.data_ptr(), K_scale.data_ptr(),
                     V_scale.data_ptr(), slot_mapping.data_ptr(), *self._pool, k_out.data_ptr(), v_out.data_ptr(), self.T,
                     self.Hkv, self.D)
        return k_out, v_out
