"""HIP QK norm + rotary positions with several axes + paged cache write
(extends ezops/kernels/fused_qk_norm_rope/*, which turn one token per sequence by one position)."""

import ctypes

import torch

from ... import _hip
from ...registry import register_kernel
from ..base_kernel import BaseKernel


@register_kernel("qk_norm_mrope", "hip", family="ragged")
class QkNormMropeHipKernel(BaseKernel):
    def __init__(self, num_tokens: int, num_heads: int, num_kv_heads: int, head_dim: int, max_position: int, sections, *,
                 interleaved: bool = False, norm: bool = True, page_size: int | None = None, num_pages: int | None = None,
                 eps: float = 1e-6):
        self.T, self.H, self.Hkv, self.D, self.S = num_tokens, num_heads, num_kv_heads, head_dim, max_position
        self.A, self.interleaved, self.norm, self.eps = len(sections), int(interleaved), int(norm), eps
        self._sections = (ctypes.c_int64 * self.A)(*sections)
        self.P, self.NP = page_size, num_pages
        T, H, Hkv, D, S, bf = num_tokens, num_heads, num_kv_heads, head_dim, max_position, torch.bfloat16
        self._q, self._kv = (T, H, D), (T, Hkv, D)
        self._positions = (("positions", (self.A, T), torch.int32),)
        self._tables = {d: (("cos", (S, D), d), ("sin", (S, D), d)) for d in (bf, torch.float32)}
        self._qw, self._kw = (("q_norm_w", (D,), bf),), (("k_norm_w", (D,), bf),)
        pool = (num_pages, Hkv, page_size, D)
        self._cache = (("K_cache", pool, bf), ("V_cache", pool, bf), ("slot_mapping", (T,), torch.int64))
        self._q_out, self._k_out = (("q_out", (T, H, D), bf),), (("k_out", (T, Hkv, D), bf),)

    def __call__(self, q, k, v, q_norm_w, k_norm_w, cos, sin, positions, K_cache=None, V_cache=None, slot_mapping=None, *,
                 q_out=None, k_out=None):
        paged = self.P is not None
        if paged != (K_cache is not None) or paged != (V_cache is not None) or paged != (slot_mapping is not None):
            raise ValueError("K_cache, V_cache and slot_mapping are required with a paged cache and only then")
        if v is None and paged:
            raise ValueError("v is required with a cache")
        if not self.norm and (q_norm_w is not None or k_norm_w is not None):
            raise ValueError("norm weights given to an op without norm")
        dev = _hip.one_gpu(q, k, v, q_norm_w, k_norm_w, cos, sin, positions, K_cache, V_cache, slot_mapping, q_out, k_out)
        bf = torch.bfloat16
        q_rs = _hip.check_rows(q, "q", self._q, bf)
        k_rs = _hip.check_rows(k, "k", self._kv, bf)
        if q_norm_w is not None:
            _hip.check_all(self._qw, q_norm_w)
        if k_norm_w is not None:
            _hip.check_all(self._kw, k_norm_w)
        tables = self._tables.get(cos.dtype)
        if tables is None:
            raise ValueError(f"cos: expected bfloat16 or float32, got {cos.dtype}")
        _hip.check_all(tables, cos, sin)
        _hip.check_all(self._positions, positions)
        if paged:
            v_rs = _hip.check_rows(v, "v", self._kv, bf)
            _hip.check_all(self._cache, K_cache, V_cache, slot_mapping)
            cache = (slot_mapping.data_ptr(), K_cache.data_ptr(), V_cache.data_ptr(), self.NP, self.P)
            v_ptr = v.data_ptr()
        else:
            v_rs, v_ptr, cache = 0, None, (None, None, None, 0, 0)
        if q_out is None:
            q_out = torch.empty(self._q, dtype=bf, device=dev)
        else:
            _hip.check_all(self._q_out, q_out)
        if k_out is not None:
            _hip.check_all(self._k_out, k_out)
        elif not paged:
            k_out = torch.empty(self._kv, dtype=bf, device=dev)
        _hip.call_on(dev, "ezops_qk_norm_mrope_bf16", q.data_ptr(), q_rs, k.data_ptr(), k_rs, v_ptr, v_rs,
                     _hip.ptr(q_norm_w), _hip.ptr(k_norm_w), self.norm, cos.data_ptr(), sin.data_ptr(),
                     cos.dtype is torch.float32, positions.data_ptr(), self.A, self._sections, self.interleaved, *cache,
                     q_out.data_ptr(), _hip.ptr(k_out), self.T, self.H, self.Hkv, self.D, self.S, self.eps)
        return q_out, k_out
