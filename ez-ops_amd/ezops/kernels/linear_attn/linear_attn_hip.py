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


def _aligned(t, name):
    if t.data_ptr() % 16:
        raise ValueError(f"{name}: must begin at a multiple of 16 bytes")


@register_kernel("linear_attn_prefill", "hip", family="ragged")
class LinearAttnPrefillHipKernel(BaseKernel):
    def __init__(self, batch: int, num_tokens: int, num_heads: int, num_kv_heads: int, head_dim: int, *,
                 num_slots: int | None = None, scale: float):
        self.B, self.T, self.H, self.Hkv, self.D = batch, num_tokens, num_heads, num_kv_heads, head_dim
        self.num_slots, self.scale = num_slots, scale
        i32, f32 = torch.int32, torch.float32
        self._q, self._kv = (num_tokens, num_heads, head_dim), (num_tokens, num_kv_heads, head_dim)
        self._in = (("log_decay", (num_kv_heads,), f32), ("cu_seqlens", (batch + 1,), i32))
        self._state = (("state", (num_slots, num_kv_heads, head_dim, head_dim), f32),)
        self._slots, self._past = (("state_slots", (batch,), i32),), (("past_lens", (batch,), i32),)
        self._out = (("out", self._q, torch.bfloat16),)
        self._ws_bytes: dict = {}  # by the library, per max_q_len

    def __call__(self, q, k, v, log_decay, cu_seqlens, state=None, state_slots=None, past_lens=None, *, max_q_len: int = 0,
                 out=None):
        if (state is not None) != (self.num_slots is not None):
            raise ValueError("state is required with num_slots and only then")
        if state is None and state_slots is not None:
            raise ValueError("state_slots given without a state")
        if max_q_len < 0:
            raise ValueError(f"max_q_len ({max_q_len}) must be >= 0")
        dev = _hip.one_gpu(q, k, v, log_decay, cu_seqlens, state, state_slots, past_lens, out)
        q_rs, k_rs, v_rs = _rows(q, "q", self._q), _rows(k, "k", self._kv), _rows(v, "v", self._kv)
        _hip.check_all(self._in, log_decay, cu_seqlens)
        if state is not None:
            _hip.check_all(self._state, state)
            _aligned(state, "state")
        if state_slots is not None:
            _hip.check_all(self._slots, state_slots)
        if past_lens is not None:
            _hip.check_all(self._past, past_lens)
        if out is None:
            out = torch.empty(self._q, dtype=torch.bfloat16, device=dev)
        else:
            _hip.check_all(self._out, out)
            _aligned(out, "out")
        n = self._ws_bytes.get(max_q_len)
        if n is None:
            n = _hip.size("ezops_linear_attn_prefill_workspace_size", self.B, self.T, self.H, self.Hkv, self.D, max_q_len)
            if len(self._ws_bytes) >= 1024:
                self._ws_bytes.clear()
            self._ws_bytes[max_q_len] = n
        # from torch's allocator at every call: stream-ordered, and a captured graph keeps its own
        ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
        _hip.call_on(dev, "ezops_linear_attn_prefill_bf16", q.data_ptr(), q_rs, k.data_ptr(), k_rs, v.data_ptr(), v_rs,
                     log_decay.data_ptr(), cu_seqlens.data_ptr(), _hip.ptr(past_lens), _hip.ptr(state),
                     _hip.ptr(state_slots), self.num_slots or 0, out.data_ptr(), self.B, self.T, self.H, self.Hkv, self.D,
                     max_q_len, self.scale, _hip.ptr(ws), n)
        return out


@register_kernel("linear_attn_decode", "hip", family="ragged")
class LinearAttnDecodeHipKernel(BaseKernel):
    def __init__(self, batch: int, num_heads: int, num_kv_heads: int, head_dim: int, num_slots: int, *, scale: float):
        self.B, self.H, self.Hkv, self.D, self.num_slots, self.scale = (batch, num_heads, num_kv_heads, head_dim,
                                                                        num_slots, scale)
        self._q, self._kv = (batch, num_heads, head_dim), (batch, num_kv_heads, head_dim)
        self._in = (("log_decay", (num_kv_heads,), torch.float32),
                    ("state", (num_slots, num_kv_heads, head_dim, head_dim), torch.float32))
        self._slots = (("state_slots", (batch,), torch.int32),)
        self._out = (("out", self._q, torch.bfloat16),)

    def __call__(self, q, k, v, log_decay, state, state_slots=None, *, out=None):
        dev = _hip.one_gpu(q, k, v, log_decay, state, state_slots, out)
        q_rs, k_rs, v_rs = _rows(q, "q", self._q), _rows(k, "k", self._kv), _rows(v, "v", self._kv)
        _hip.check_all(self._in, log_decay, state)
        _aligned(state, "state")
        if state_slots is not None:
            _hip.check_all(self._slots, state_slots)
        if out is None:
            out = torch.empty(self._q, dtype=torch.bfloat16, device=dev)
        else:
            _hip.check_all(self._out, out)
            _aligned(out, "out")
        _hip.call_on(dev, "ezops_linear_attn_decode_bf16", q.data_ptr(), q_rs, k.data_ptr(), k_rs, v.data_ptr(), v_rs,
                     log_decay.data_ptr(), state.data_ptr(), _hip.ptr(state_slots), self.num_slots, out.data_ptr(),
                     self.B, self.H, self.Hkv, self.D, self.scale)
        return out
