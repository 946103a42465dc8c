"""Linear attention with a decay per head: packed ragged prompts, and one token per sequence.

No reference counterpart (its attention is softmax over a cache,
ezops/ops/attn_decode.py:9-67); these ops stand beside PrefillAttnOp and
AttnDecodeOp for layers whose past is a state of fixed size.  Per kv head, with
``lambda = exp(log_decay)`` (log_decay <= 0, -inf = no memory):

    S_t = lambda S_{t-1} + k_t v_t^T        S [D, D] fp32
    o_t = scale * q_t^T S_t

and query head ``h`` reads the state of kv head ``h // (H / Hkv)``.  States live in
a pool ``state [num_slots, Hkv, D, D]``; sequence ``b`` owns slot
``state_slots[b]`` (None: slot ``b``), updated in place.  A sequence whose slot is
outside the pool (-1: a padded row of the batch), or that an earlier sequence of
the batch with tokens holds already, is left out whole: its rows of ``out`` and
every state stay as they were.  In a prompt a token whose k or v is not finite leaves its own
sequence's outputs undefined from the first token of its 64-token chunk on; other
sequences are not touched.  States and the products ``q . k`` of a prompt have to stay
below 2^127: past that a query's own outputs are undefined (a product), or the own
sequence's outputs from there on (a state), also where the recurrence gives an infinity.
"""

import ctypes

import torch

from ..registry import get_kernel
from .base_op import Op, default_device, randn
from .utils.roofline import RooflineResult

GROUPS = (1, 2, 4, 8, 16)


def usable_slots(state_slots, lens: list[int], num_slots: int) -> list[int]:
    """The slot of every sequence, -1 where it has none (outside the pool, or held by an earlier sequence with tokens)."""
    slots = list(range(len(lens))) if state_slots is None else state_slots.tolist()
    held, out = set(), []
    for s, n in zip(slots, lens):
        out.append(s if 0 <= s < num_slots and s not in held else -1)
        if n > 0:
            held.add(s)
    return out


def _check_heads(num_heads, num_kv_heads, head_dim):
    if num_kv_heads < 1 or not 1 <= num_heads <= 4096 or num_heads % num_kv_heads:
        raise ValueError(f"num_heads ({num_heads}) must be divisible by num_kv_heads ({num_kv_heads}) and at most 4096")
    if num_heads // num_kv_heads not in GROUPS:
        raise ValueError(f"GQA group size {num_heads}/{num_kv_heads} not supported (1, 2, 4, 8 or 16)")
    if head_dim not in (64, 128):
        raise ValueError(f"head_dim ({head_dim}) must be 64 or 128")


def _scale(scale, head_dim):
    if scale is None:
        return head_dim ** -0.5
    if not 0 < ctypes.c_float(scale).value < float("inf"):
        raise ValueError(f"scale ({scale}) must be positive and in the range of fp32")
    return float(scale)


def _decays(num_kv_heads, device):
    """ln of the decays, from exp(-1/2) to exp(-1/256) per token."""
    if torch.device(device).type == "meta":
        return torch.empty(num_kv_heads, dtype=torch.float32, device="meta")
    return -torch.exp2(-1 - 7 * torch.arange(num_kv_heads, dtype=torch.float32) / max(1, num_kv_heads - 1)).to(device)


class LinearAttnPrefillOp(Op):
    _params_desc = {
        "batch": "Sequences in the chunk",
        "num_tokens": "Rows of packed tokens (fewer may be used)",
        "num_heads": "Query heads",
        "num_kv_heads": "KV heads (one state each)",
        "head_dim": "Dimension per head (64 or 128)",
        "num_slots": "State slots in the pool (None: no states, every sequence starts from zero)",
        "scale": "Factor on the outputs (default head_dim ** -0.5)",
    }
    _atol = 1e-2
    _rtol = 1e-2

    def __init__(self, batch: int, num_tokens: int, num_heads: int, num_kv_heads: int, head_dim: int, backend: str = "ref",
                 *, num_slots: int | None = None, scale: float | None = None):
        _check_heads(num_heads, num_kv_heads, head_dim)
        if not 1 <= batch <= 65536 or not 1 <= num_tokens < 1 << 30:
            raise ValueError("batch must be in [1, 65536] and num_tokens in [1, 2^30)")
        if num_slots is not None and not 1 <= num_slots < 1 << 31:
            raise ValueError(f"num_slots ({num_slots}) must be in [1, 2^31)")
        self.batch, self.num_tokens, self.num_heads, self.num_kv_heads = batch, num_tokens, num_heads, num_kv_heads
        self.head_dim, self.num_slots, self.scale = head_dim, num_slots, _scale(scale, head_dim)
        self._backend = backend
        if backend != "ref":
            self._kernel = get_kernel("linear_attn_prefill", backend)(
                batch, num_tokens, num_heads, num_kv_heads, head_dim, num_slots=num_slots, scale=self.scale)
        else:
            self._kernel = self._ref_forward

    def forward(self, q, k, v, log_decay, cu_seqlens, state=None, state_slots=None, past_lens=None, *, max_q_len: int = 0,
                out=None):
        """q [T, H, D], k / v [T, Hkv, D] (tokens may lie apart), log_decay [Hkv] fp32; sequence ``b`` owns rows
        cu_seqlens[b] .. cu_seqlens[b+1]-1.  It continues from its state if past_lens[b] > 0 and starts from zero
        otherwise (past_lens None: all do); one without tokens leaves its state alone.  max_q_len: the caller's bound
        on the new tokens of a sequence (0 = num_tokens; longer ones are cut off there).  Returns out [T, H, D]; rows
        of no sequence are not written."""
        return self._kernel(q, k, v, log_decay, cu_seqlens, state, state_slots, past_lens, max_q_len=max_q_len, out=out)

    def gen_data(self, device=None):
        """The rows shared out evenly to fresh sequences."""
        dev = default_device(device)
        bf = dict(dtype=torch.bfloat16, device=dev)
        B, T, H, Hkv, D = self.batch, self.num_tokens, self.num_heads, self.num_kv_heads, self.head_dim
        q, k, v = randn(T, H, D, **bf), randn(T, Hkv, D, **bf), randn(T, Hkv, D, **bf)
        cu = torch.tensor([T * b // B for b in range(B + 1)], dtype=torch.int32, device=dev)
        if self.num_slots is None:
            return q, k, v, _decays(Hkv, dev), cu
        return q, k, v, _decays(Hkv, dev), cu, randn(self.num_slots, Hkv, D, D, dtype=torch.float32, device=dev)

    def get_roofline(self) -> RooflineResult:
        T, H, Hkv, D = self.num_tokens, self.num_heads, self.num_kv_heads, self.head_dim
        b = 4 * T * (H + Hkv) * D + 4 * (self.batch + 1 + Hkv)
        b += 4 * self.batch * Hkv * D * D if self.num_slots is not None else 0
        return RooflineResult(T * (3 * Hkv + 2 * H) * D * D, b, b)

    def _ref_forward(self, q, k, v, log_decay, cu_seqlens, state=None, state_slots=None, past_lens=None, *,
                     max_q_len: int = 0, out=None):
        """The recurrence, token by token."""
        B, T, H, Hkv, D = self.batch, self.num_tokens, self.num_heads, self.num_kv_heads, self.head_dim
        out = torch.empty(T, H, D, dtype=q.dtype, device=q.device) if out is None else out
        lam = torch.exp(log_decay.float())[:, None, None]
        cu = [min(max(0, x), T) for x in cu_seqlens.tolist()]
        lens = [min(e - s, max_q_len or T) for s, e in zip(cu, cu[1:])]
        slots = usable_slots(state_slots, lens, self.num_slots) if state is not None else [-1] * B
        past = past_lens.tolist() if past_lens is not None else [0] * B
        for b in range(B):
            n = lens[b]
            if n <= 0 or (state is not None and slots[b] < 0):
                continue
            keep = state is not None and past[b] > 0
            S = state[slots[b]].clone() if keep else torch.zeros(Hkv, D, D, device=q.device)
            for t in range(cu[b], cu[b] + n):
                S = lam * S + k[t].float()[:, :, None] * v[t].float()[:, None, :]
                o = q[t].float().reshape(Hkv, H // Hkv, D) @ S
                out[t] = (o * self.scale).reshape(H, D).to(out.dtype)
            if state is not None:
                state[slots[b]] = S
        return out


class LinearAttnDecodeOp(Op):
    _params_desc = {
        "batch": "Sequences (one token each)",
        "num_heads": "Query heads",
        "num_kv_heads": "KV heads (one state each)",
        "head_dim": "Dimension per head (64 or 128)",
        "num_slots": "State slots in the pool",
        "scale": "Factor on the outputs (default head_dim ** -0.5)",
    }
    _atol = 1e-2
    _rtol = 1e-2

    def __init__(self, batch: int, num_heads: int, num_kv_heads: int, head_dim: int, num_slots: int, backend: str = "ref", *,
                 scale: float | None = None):
        _check_heads(num_heads, num_kv_heads, head_dim)
        if not 1 <= batch <= 65536:
            raise ValueError(f"batch ({batch}) must be in [1, 65536]")
        if not 1 <= num_slots < 1 << 31:
            raise ValueError(f"num_slots ({num_slots}) must be in [1, 2^31)")
        self.batch, self.num_heads, self.num_kv_heads, self.head_dim = batch, num_heads, num_kv_heads, head_dim
        self.num_slots, self.scale = num_slots, _scale(scale, head_dim)
        self._backend = backend
        if backend != "ref":
            self._kernel = get_kernel("linear_attn_decode", backend)(batch, num_heads, num_kv_heads, head_dim, num_slots,
                                                                     scale=self.scale)
        else:
            self._kernel = self._ref_forward

    def forward(self, q, k, v, log_decay, state, state_slots=None, *, out=None):
        """q [B, H, D], k / v [B, Hkv, D] (rows may lie apart), log_decay [Hkv] fp32, state [num_slots, Hkv, D, D] fp32,
        updated in place.  Returns out [B, H, D]; rows of sequences without a slot are not written."""
        return self._kernel(q, k, v, log_decay, state, state_slots, out=out)

    def gen_data(self, device=None):
        dev = default_device(device)
        bf = dict(dtype=torch.bfloat16, device=dev)
        B, H, Hkv, D = self.batch, self.num_heads, self.num_kv_heads, self.head_dim
        data = [randn(B, H, D, **bf), randn(B, Hkv, D, **bf), randn(B, Hkv, D, **bf), _decays(Hkv, dev),
                randn(self.num_slots, Hkv, D, D, dtype=torch.float32, device=dev)]
        if dev.type == "meta":
            data.append(torch.empty(B, dtype=torch.int32, device=dev))
        else:
            slots = torch.full((B,), -1, dtype=torch.int32)
            n = min(B, self.num_slots)
            slots[:n] = torch.randperm(self.num_slots)[:n].to(torch.int32)
            data.append(slots.to(dev))
        return tuple(data)

    def get_roofline(self) -> RooflineResult:
        B, H, Hkv, D = self.batch, self.num_heads, self.num_kv_heads, self.head_dim
        b = B * (8 * Hkv * D * D + 4 * (H + Hkv) * D + 4)
        return RooflineResult(B * (3 * Hkv + 2 * H) * D * D, b, b)

    def _ref_forward(self, q, k, v, log_decay, state, state_slots=None, *, out=None):
        B, H, Hkv, D = self.batch, self.num_heads, self.num_kv_heads, self.head_dim
        out = torch.empty(B, H, D, dtype=q.dtype, device=q.device) if out is None else out
        lam = torch.exp(log_decay.float())[:, None, None]
        for b, s in enumerate(usable_slots(state_slots, [1] * B, self.num_slots)):
            if s < 0:
                continue
            S = lam * state[s] + k[b].float()[:, :, None] * v[b].float()[:, None, :]
            state[s] = S
            out[b] = ((q[b].float().reshape(Hkv, H // Hkv, D) @ S) * self.scale).reshape(H, D).to(out.dtype)
        return out
