"""Per-head QK RMSNorm + rotary positions with several axes + paged cache write.

Extension of FusedQkNormRopeOp (reference: ezops/ops/fused_qk_norm_rope.py:7-169)
to packed tokens whose position has up to four coordinates: time, height and
width of an image or video patch; text has the same position on every axis.
For token ``t`` and every head

    y = x * rsqrt(mean(x^2) + eps) * w                      (``norm``)
    o[i], o[i + D/2] = y[i] c - y[i + D/2] s, y[i + D/2] c + y[i] s
    c, s = cos[p, i], sin[p, i]  with  p = positions[axis(i), t],  i < D/2

in fp32 with one bf16 rounding.  ``sections`` gives each axis its number of
pairs (their sum is D/2): consecutive runs of pairs, or with ``interleaved``
pair ``i`` belongs to axis ``i % A`` while that axis has pairs left and to axis 0
after that.  ``cos`` / ``sin`` are HF tables ``[max_position, D]`` (both halves
equal; the first is read), bf16 or fp32.  Column ``i`` belongs to pair ``i`` whatever
its axis, so where each axis has the same frequencies ``f`` (vision encoders: rows
and columns of the patches) the table repeats them: with two axes of ``n`` pairs
``angles = arange(max_position)[:, None] * f.repeat(2)``, ``cos =
angles.cos().repeat(1, 2)``; one run of D/2 frequencies is the text decoders' form.

With a paged cache (``page_size``, ``num_pages``) token ``t`` goes to slot
``slot_mapping[t]`` (int64, page * page_size + offset, as PagedBatchPlanOp makes
it): k rotated, v as it is; slots outside the pool are skipped.  Two tokens of a
call must not share a slot.  A token with a position outside
``[0, max_position)`` on any axis (the plan's -1 behind the last token) is left
out whole: its rows of q_out and k_out stay as they were.
"""

import torch

from ..registry import get_kernel
from .base_op import Op, default_device, randn
from .fused_qk_norm_rope import head_rmsnorm_f32, rope_half_f32, rope_tables
from .utils.roofline import RooflineResult


def axis_of_pair(half: int, sections, interleaved: bool) -> list[int]:
    """The axis of every pair i < D/2."""
    A = len(sections)
    if interleaved:
        return [i % A if i < A * sections[i % A] else 0 for i in range(half)]
    return [a for a, n in enumerate(sections) for _ in range(n)]


class QkNormMropeOp(Op):
    _params_desc = {
        "num_tokens": "Rows of packed tokens",
        "num_heads": "Query heads",
        "num_kv_heads": "KV heads",
        "head_dim": "Dimension per head (even, at most 512)",
        "max_position": "Rows of the cos/sin tables",
        "sections": "Rotary pairs per position axis (1 to 4 axes, adding up to head_dim / 2)",
        "interleaved": "Pairs dealt to the axes in turn, not in runs",
        "norm": "RMSNorm of the q and k heads before the rotation",
        "page_size": "Cache rows per page (None: no cache, k is returned)",
        "num_pages": "Pages in the cache pools",
    }
    _atol = 1e-2
    _rtol = 1e-2

    rms_eps = 1e-6
    rope_theta = 1e6

    def __init__(self, num_tokens: int, num_heads: int, num_kv_heads: int, head_dim: int, max_position: int, sections,
                 backend: str = "ref", *, interleaved: bool = False, norm: bool = True, page_size: int | None = None,
                 num_pages: int | None = None):
        sections = tuple(int(s) for s in sections)
        if not 1 <= num_tokens < 1 << 30 or not 1 <= max_position < 1 << 31:
            raise ValueError("num_tokens must be in [1, 2^30) and max_position in [1, 2^31)")
        if num_kv_heads < 1 or not 1 <= num_heads <= 4096 or num_heads % num_kv_heads:
            raise ValueError(f"num_heads ({num_heads}) must be divisible by num_kv_heads ({num_kv_heads}) and at most 4096")
        if not 2 <= head_dim <= 512 or head_dim % 2:
            raise ValueError(f"head_dim ({head_dim}) must be even and at most 512")
        if not 1 <= len(sections) <= 4 or min(sections) < 0 or sum(sections) != head_dim // 2:
            raise ValueError(f"sections {sections} must be 1 to 4 counts that add up to head_dim / 2 = {head_dim // 2}")
        A = len(sections)
        if interleaved and any(s and A * (s - 1) + a >= head_dim // 2 for a, s in enumerate(sections) if a):
            raise ValueError(f"sections {sections}: an interleaved section has more pairs than turns")
        if (page_size is None) != (num_pages is None):
            raise ValueError("page_size and num_pages go together")
        if page_size is not None and (not 32 <= page_size <= 1 << 20 or page_size & (page_size - 1)):
            raise ValueError(f"page_size ({page_size}) must be a power of two in [32, 2^20]")
        if num_pages is not None and not 1 <= num_pages < 1 << 31:
            raise ValueError(f"num_pages ({num_pages}) must be in [1, 2^31)")
        self.num_tokens, self.num_heads, self.num_kv_heads, self.head_dim = num_tokens, num_heads, num_kv_heads, head_dim
        self.max_position, self.sections, self.interleaved, self.norm = max_position, sections, interleaved, norm
        self.page_size, self.num_pages = page_size, num_pages
        self._backend = backend
        if backend != "ref":
            self._kernel = get_kernel("qk_norm_mrope", backend)(
                num_tokens, num_heads, num_kv_heads, head_dim, max_position, sections, interleaved=interleaved, norm=norm,
                page_size=page_size, num_pages=num_pages, eps=self.rms_eps)
        else:
            self._kernel = self._ref_forward

    def forward(self, q, k, v, q_norm_w, k_norm_w, cos, sin, positions, K_cache=None, V_cache=None, slot_mapping=None, *,
                q_out=None, k_out=None):
        """q [T, H, D], k / v [T, Hkv, D] (tokens may lie apart: slices of a packed projection); norm weights [D] or
        None (unit); positions [axes, T] int32.  Returns (q_out, k_out); with a cache k_out is None unless passed in.
        v may be None without a cache; q_out may be q itself, k_out k, where those are contiguous."""
        return self._kernel(q, k, v, q_norm_w, k_norm_w, cos, sin, positions, K_cache, V_cache, slot_mapping,
                            q_out=q_out, k_out=k_out)

    def gen_data(self, device=None):
        dev = default_device(device)
        bf = dict(dtype=torch.bfloat16, device=dev)
        T, H, Hkv, D, S = self.num_tokens, self.num_heads, self.num_kv_heads, self.head_dim, self.max_position
        q, k, v = randn(T, H, D, **bf), randn(T, Hkv, D, **bf), randn(T, Hkv, D, **bf)
        qw = randn(D, scale=0.1, mean=1.0, **bf) if self.norm else None
        kw = randn(D, scale=0.1, mean=1.0, **bf) if self.norm else None
        A = len(self.sections)
        if dev.type == "meta":
            cos, sin = torch.empty(S, D, **bf), torch.empty(S, D, **bf)
            pos = torch.empty(A, T, dtype=torch.int32, device=dev)
        else:
            cos, sin = rope_tables(S, D, self.rope_theta, dev)
            pos = torch.randint(0, S, (A, T), dtype=torch.int32).to(dev)
        if self.page_size is None:
            return q, k, v, qw, kw, cos, sin, pos
        shape = (self.num_pages, Hkv, self.page_size, D)
        if dev.type == "meta":
            slots = torch.empty(T, dtype=torch.int64, device=dev)
        else:
            rows = self.num_pages * self.page_size
            slots = torch.full((T,), -1, dtype=torch.int64)
            n = min(T, rows)
            slots[:n] = torch.randperm(rows)[:n]
            slots = slots.to(dev)
        return q, k, v, qw, kw, cos, sin, pos, randn(*shape, **bf), randn(*shape, **bf), slots

    def get_roofline(self) -> RooflineResult:
        T, H, Hkv, D = self.num_tokens, self.num_heads, self.num_kv_heads, self.head_dim
        heads = 2 * H + (4 if self.page_size else 2) * Hkv
        b = 2 * T * heads * D + T * (4 * len(self.sections) + (8 if self.page_size else 0)) + 2 * min(T, self.max_position) * D
        return RooflineResult(T * (H + Hkv) * D * (7 if self.norm else 3), b, b)

    def check(self, actual, expected) -> bool:
        pairs = [(a, e) for a, e in zip(actual, expected, strict=True) if e is not None]
        return all(a.shape == e.shape and torch.allclose(a, e, atol=self._atol, rtol=self._rtol) for a, e in pairs)

    def _ref_forward(self, q, k, v, q_norm_w, k_norm_w, cos, sin, positions, K_cache=None, V_cache=None,
                     slot_mapping=None, *, q_out=None, k_out=None):
        half = self.head_dim // 2
        pos = positions.long()
        live = ((pos >= 0) & (pos < self.max_position)).all(0)
        axis = torch.tensor(axis_of_pair(half, self.sections, self.interleaved), device=q.device)
        rows = torch.where(live, pos, 0)[axis].t()  # [T, D/2]
        pair = torch.arange(half, device=q.device)
        c = cos[rows, pair].float().repeat(1, 2)[:, None]
        s = sin[rows, pair].float().repeat(1, 2)[:, None]
        unit = torch.ones(self.head_dim, device=q.device)

        def turned(x, w):
            xf = head_rmsnorm_f32(x, unit if w is None else w, self.rms_eps) if self.norm else x.float()
            return rope_half_f32(xf, c, s)

        qr, kr = turned(q, q_norm_w), turned(k, k_norm_w)
        on = live[:, None, None]
        q_out = qr if q_out is None else q_out.copy_(torch.where(on, qr, q_out))
        if k_out is not None:
            k_out.copy_(torch.where(on, kr, k_out))
        elif K_cache is None:
            k_out = kr
        if K_cache is not None:
            ok = live & (slot_mapping >= 0) & (slot_mapping < self.num_pages * self.page_size)
            slot = slot_mapping[ok]
            page, row = slot // self.page_size, slot % self.page_size
            K_cache[page, :, row] = kr[ok]
            V_cache[page, :, row] = v[ok]
        return q_out, k_out
