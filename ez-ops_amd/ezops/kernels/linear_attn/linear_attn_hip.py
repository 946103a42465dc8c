"""HIP linear attention with a decay per head (packed prompts, single tokens); no reference counterpart
(its attention is softmax over a cache, ezops/ops/attn_decode.py:9-67)."""

import torch

from ... import _hip
from ...registry import register_kernel
from ..base_kernel import BaseKernel


def _rows(t, name, shape):
    """Row stride of a bf16 operand; the kernels read it 16 bytes at a time."""
    rs = _hip.check_rows(t, name, shape, torch.bfloat16)
    if rs % 8 or t.data_ptr() % 16:
        raise ValueError(f"{name}: rows must begin at multiples of 16 bytes")
    return rs


def _pool(t, shape):
    _hip.check(t, "state", shape, torch.float32)
    if t.data_ptr() % 16:
        raise ValueError("state: must begin at a multiple of 16 bytes")


def _out(out, shape, dev):
    if out is None:
        return torch.empty(shape, dtype=torch.bfloat16, device=dev)
    _hip.check(out, "out", shape, torch.bfloat16)
    if out.data_ptr() % 16:
        raise ValueError("out: must begin at a multiple of 16 bytes")
    return out


@register_kernel("linear_attn_prefill", "hip", family="ragged")
class LinearAttnPrefillHipKernel(BaseKernel):
    def __init__(self, batch: int, num_tokens: int, num_heads: int, num_kv_heads: int, head_dim: int, *,
                 num_slots: int | None = None, scale: float):
        self.B, self.T, self.H, self.Hkv, self.D = batch, num_tokens, num_heads, num_kv_heads, head_dim
        self.num_slots, self.scale = num_slots, scale
        self._ws_bytes: dict = {}  # by the library, per max_q_len

    def __call__(self, q, k, v, log_decay, cu_seqlens, state=None, state_slots=None, past_lens=None, *, max_q_len: int = 0,
                 out=None):
        B, T, H, Hkv, D = self.B, self.T, self.H, self.Hkv, self.D
        if (state is not None) != (self.num_slots is not None):
            raise ValueError("state is required with num_slots and only then")
        if state is None and state_slots is not None:
            raise ValueError("state_slots given without a state")
        if max_q_len < 0:
            raise ValueError(f"max_q_len ({max_q_len}) must be >= 0")
        dev = _hip.require_gpu(q, k, v, log_decay, cu_seqlens, state, state_slots, past_lens, out)
        q_rs, k_rs, v_rs = _rows(q, "q", (T, H, D)), _rows(k, "k", (T, Hkv, D)), _rows(v, "v", (T, Hkv, D))
        _hip.check(log_decay, "log_decay", (Hkv,), torch.float32)
        _hip.check(cu_seqlens, "cu_seqlens", (B + 1,), torch.int32)
        if state is not None:
            _pool(state, (self.num_slots, Hkv, D, D))
        if state_slots is not None:
            _hip.check(state_slots, "state_slots", (B,), torch.int32)
        if past_lens is not None:
            _hip.check(past_lens, "past_lens", (B,), torch.int32)
        out = _out(out, (T, H, D), dev)
        n = self._ws_bytes.get(max_q_len)
        if n is None:
            n = _hip.size("ezops_linear_attn_prefill_workspace_size", B, T, H, Hkv, D, max_q_len)
            self._ws_bytes[max_q_len] = n
        # from torch's allocator at every call: stream-ordered, and a captured graph keeps its own
        ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
        _hip.call_on(dev, "ezops_linear_attn_prefill_bf16", q.data_ptr(), q_rs, k.data_ptr(), k_rs, v.data_ptr(), v_rs,
                     log_decay.data_ptr(), cu_seqlens.data_ptr(), _hip.ptr(past_lens), _hip.ptr(state),
                     _hip.ptr(state_slots), self.num_slots or 0, out.data_ptr(), B, T, H, Hkv, D, max_q_len, self.scale,
                     _hip.ptr(ws), n)
        return out


@register_kernel("linear_attn_decode", "hip", family="ragged")
class LinearAttnDecodeHipKernel(BaseKernel):
    def __init__(self, batch: int, num_heads: int, num_kv_heads: int, head_dim: int, num_slots: int, *, scale: float):
        self.B, self.H, self.Hkv, self.D, self.num_slots, self.scale = (batch, num_heads, num_kv_heads, head_dim,
                                                                        num_slots, scale)

    def __call__(self, q, k, v, log_decay, state, state_slots=None, *, out=None):
        B, H, Hkv, D = self.B, self.H, self.Hkv, self.D
        dev = _hip.require_gpu(q, k, v, log_decay, state, state_slots, out)
        q_rs, k_rs, v_rs = _rows(q, "q", (B, H, D)), _rows(k, "k", (B, Hkv, D)), _rows(v, "v", (B, Hkv, D))
        _hip.check(log_decay, "log_decay", (Hkv,), torch.float32)
        _pool(state, (self.num_slots, Hkv, D, D))
        if state_slots is not None:
            _hip.check(state_slots, "state_slots", (B,), torch.int32)
        out = _out(out, (B, H, D), dev)
        _hip.call_on(dev, "ezops_linear_attn_decode_bf16", q.data_ptr(), q_rs, k.data_ptr(), k_rs, v.data_ptr(), v_rs,
                     log_decay.data_ptr(), state.data_ptr(), _hip.ptr(state_slots), self.num_slots, out.data_ptr(), B, H,
                     Hkv, D, self.scale)
        return out
