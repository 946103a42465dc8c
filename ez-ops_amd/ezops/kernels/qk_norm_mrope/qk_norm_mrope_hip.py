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
        self._q, self._kv = (num_tokens, num_heads, head_dim), (num_tokens, num_kv_heads, head_dim)
        self._specs: dict = {}  # what a call has to check, by what it passes

    def _spec(self, table, has_qw, has_kw, has_q_out, has_k_out):
        """(name, shape, dtype) of every tensor of a call that has to be contiguous, in the order __call__ lists them."""
        if table not in (torch.bfloat16, torch.float32):
            raise ValueError(f"cos: expected bfloat16 or float32, got {table}")
        bf, D = torch.bfloat16, self.D
        pool = (self.NP, self.Hkv, self.P, D)
        spec = [("cos", (self.S, D), table), ("sin", (self.S, D), table), ("positions", (self.A, self.T), torch.int32)]
        if self.P is not None:
            spec += [("K_cache", pool, bf), ("V_cache", pool, bf), ("slot_mapping", (self.T,), torch.int64)]
        spec += [("q_norm_w", (D,), bf)] * has_qw + [("k_norm_w", (D,), bf)] * has_kw
        return tuple(spec + [("q_out", self._q, bf)] * has_q_out + [("k_out", self._kv, bf)] * has_k_out)

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
        table = cos.dtype
        key = (table, q_norm_w is not None, k_norm_w is not None, q_out is not None, k_out is not None)
        spec = self._specs.get(key)
        if spec is None:
            spec = self._specs[key] = self._spec(*key)
        given = [t for t in (q_norm_w, k_norm_w, q_out, k_out) if t is not None]
        if paged:
            v_rs, v_ptr = _hip.check_rows(v, "v", self._kv, bf), v.data_ptr()
            _hip.check_all(spec, cos, sin, positions, K_cache, V_cache, slot_mapping, *given)
            cache = (slot_mapping.data_ptr(), K_cache.data_ptr(), V_cache.data_ptr(), self.NP, self.P)
        else:
            _hip.check_all(spec, cos, sin, positions, *given)
            v_rs, v_ptr, cache = 0, None, (None, None, None, 0, 0)
        if q_out is None:
            q_out = torch.empty(self._q, dtype=bf, device=dev)
        if k_out is None and not paged:
            k_out = torch.empty(self._kv, dtype=bf, device=dev)
        _hip.call_on(dev, "ezops_qk_norm_mrope_bf16", q.data_ptr(), q_rs, k.data_ptr(), k_rs, v_ptr, v_rs,
                     None if q_norm_w is None else q_norm_w.data_ptr(), None if k_norm_w is None else k_norm_w.data_ptr(),
                     self.norm, cos.data_ptr(), sin.data_ptr(), table is torch.float32, positions.data_ptr(), self.A,
                     self._sections, self.interleaved, *cache, q_out.data_ptr(),
                     None if k_out is None else k_out.data_ptr(), self.T, self.H, self.Hkv, self.D, self.S, self.eps)
        return q_out, k_out
