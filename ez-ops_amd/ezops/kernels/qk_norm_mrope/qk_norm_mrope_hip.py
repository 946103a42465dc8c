"""HIP QK norm + rotary positions with several axes + paged cache write
(extends ezops/kernels/fused_qk_norm_rope/*, which turn one token per sequence by one position)."""

import ctypes

import torch

from ... import _hip
from ...registry import register_kernel
from ..base_kernel import BaseKernel

_TABLES = (torch.bfloat16, torch.float32)


@register_kernel("qk_norm_mrope", "hip", family="ragged")
class QkNormMropeHipKernel(BaseKernel):
    def __init__(self, num_tokens: int, num_heads: int, num_kv_heads: int, head_dim: int, max_position: int, sections, *,
                 interleaved: bool = False, norm: bool = True, page_size: int | None = None, num_pages: int | None = None,
                 eps: float = 1e-6):
        self.T, self.H, self.Hkv, self.D, self.S = num_tokens, num_heads, num_kv_heads, head_dim, max_position
        self.A, self.interleaved, self.norm, self.eps = len(sections), int(interleaved), int(norm), eps
        self._sections = (ctypes.c_int64 * self.A)(*sections)
        self.P, self.NP = page_size, num_pages

    def __call__(self, q, k, v, q_norm_w, k_norm_w, cos, sin, positions, K_cache=None, V_cache=None, slot_mapping=None, *,
                 q_out=None, k_out=None):
        T, H, Hkv, D, S = self.T, self.H, self.Hkv, self.D, self.S
        paged = self.P is not None
        if paged != (K_cache is not None) or paged != (V_cache is not None) or paged != (slot_mapping is not None):
            raise ValueError("K_cache, V_cache and slot_mapping are required with a paged cache and only then")
        if v is None and paged:
            raise ValueError("v is required with a cache")
        if not self.norm and (q_norm_w is not None or k_norm_w is not None):
            raise ValueError("norm weights given to an op without norm")
        dev = _hip.require_gpu(q, k, v, q_norm_w, k_norm_w, cos, sin, positions, K_cache, V_cache, slot_mapping, q_out,
                               k_out)
        bf = torch.bfloat16
        q_rs = _hip.check_rows(q, "q", (T, H, D), bf)
        k_rs = _hip.check_rows(k, "k", (T, Hkv, D), bf)
        v_rs = _hip.check_rows(v, "v", (T, Hkv, D), bf) if paged else 0
        if q_norm_w is not None:
            _hip.check(q_norm_w, "q_norm_w", (D,), bf)
        if k_norm_w is not None:
            _hip.check(k_norm_w, "k_norm_w", (D,), bf)
        table = cos.dtype
        if table not in _TABLES:
            raise ValueError(f"cos: expected bfloat16 or float32, got {table}")
        _hip.check(cos, "cos", (S, D), table)
        _hip.check(sin, "sin", (S, D), table)
        _hip.check(positions, "positions", (self.A, T), torch.int32)
        if paged:
            pool = (self.NP, Hkv, self.P, D)
            _hip.check(K_cache, "K_cache", pool, bf)
            _hip.check(V_cache, "V_cache", pool, bf)
            _hip.check(slot_mapping, "slot_mapping", (T,), torch.int64)
        if q_out is None:
            q_out = torch.empty(T, H, D, dtype=bf, device=dev)
        else:
            _hip.check(q_out, "q_out", (T, H, D), bf)
        if k_out is not None:
            _hip.check(k_out, "k_out", (T, Hkv, D), bf)
        elif not paged:
            k_out = torch.empty(T, Hkv, D, dtype=bf, device=dev)
        _hip.call_on(dev, "ezops_qk_norm_mrope_bf16", q.data_ptr(), q_rs, k.data_ptr(), k_rs,
                     v.data_ptr() if paged else None, v_rs, _hip.ptr(q_norm_w), _hip.ptr(k_norm_w), self.norm,
                     cos.data_ptr(), sin.data_ptr(), int(table is torch.float32), positions.data_ptr(), self.A,
                     self._sections, self.interleaved, _hip.ptr(slot_mapping), _hip.ptr(K_cache), _hip.ptr(V_cache),
                     self.NP or 0, self.P or 0, q_out.data_ptr(), _hip.ptr(k_out), T, H, Hkv, D, S, self.eps)
        return q_out, k_out
