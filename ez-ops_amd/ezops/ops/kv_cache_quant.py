"""A paged KV cache held in 8 bits: rows quantised as they are written, and read back.

No reference counterpart (the reference's cache is one contiguous bf16 tensor,
ezops/ops/attn_decode.py:60-61); these ops stand beside the cache write of
QkNormMropeOp for caches that QuantPagedAttnDecodeOp and QuantPrefillAttnOp read.

Codes live in pools ``K_cache`` / ``V_cache`` ``[num_pages, Hkv, page_size, D]``,
``int8`` or ``float8_e4m3fn``; ``K_scale`` / ``V_scale``
``[num_pages, Hkv, page_size / block_size]`` (uint8) hold one exponent for each block of
``block_size`` rows of a page and kv head: a row stands for ``code * 2^(e - 127)``, all
NaN where e = 255 (the encoding of ``torch.float8_e8m0fnu``; an exponent outside [67, 187]
is read as the nearer of the two).  With TOP = 127 (int8) or
448 (e4m3)

    need = least e with max|x| <= TOP * 2^(e - 127) over the rows a block gets in a call, in [67, 187]
    e    = need where the call writes the block's first row, else max(need, e as it was)
    code = round(x * 2^(127 - e)), to nearest even, saturating

and where e grows the rows that the block held before become
``round(code * 2^(e_old - e))``.  The scales are powers of two so that every factor here
is exact: the values read back are exact in bf16, an int8 row stays within one step of
its block's present scale however often the block grew, and e4m3 codes only lose bits
that leave their range.

Token ``t`` goes to slot ``slot_mapping[t]`` (int64, page * page_size + offset, as
PagedBatchPlanOp makes it); slots outside the pool are skipped.  The tokens that a block
gets in one call have to be one run, consecutive tokens in consecutive slots (as a plan
has them), and nothing is kept of rows of that block behind the last of them; a block whose
tokens are not (a row or a token left out between them, another order), or a slot used
twice, is left with undefined rows and scale, other blocks are not touched.  Values of magnitude 2^67 and more saturate and such below 2^-61 become
zero.  A k or v that is not finite is a NaN code (0x7f) of its own in an e4m3 cache; int8 has no
such code, and its block reads as NaN until its first row is written again.
"""

import torch

from ..registry import get_kernel
from .base_op import Op, default_device, randn
from .utils.roofline import RooflineResult

DTYPES = (torch.int8, torch.float8_e4m3fn)
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
LOW_EXP, HIGH_EXP, NAN_EXP = 127 - 60, 127 + 60, 255


def check_cache(page_size, num_pages, block_size, cache_dtype, head_dim):
    if cache_dtype not in DTYPES:
        raise ValueError(f"cache_dtype ({cache_dtype}) must be torch.int8 or torch.float8_e4m3fn")
    if not 32 <= page_size <= 1 << 20 or page_size & (page_size - 1):
        raise ValueError(f"page_size ({page_size}) must be a power of two in [32, 2^20]")
    if not 16 <= block_size <= min(256, page_size) or block_size & (block_size - 1):
        raise ValueError(f"block_size ({block_size}) must be a power of two in [16, 256], at most page_size ({page_size})")
    if not 1 <= num_pages < 1 << 31:
        raise ValueError(f"num_pages ({num_pages}) must be in [1, 2^31)")
    if head_dim not in (64, 128):
        raise ValueError(f"head_dim ({head_dim}) must be 64 or 128")


def check_rows(num_tokens, num_kv_heads):
    if not 1 <= num_tokens < 1 << 30:
        raise ValueError(f"num_tokens ({num_tokens}) must be in [1, 2^30)")
    if not 1 <= num_kv_heads <= 4096:
        raise ValueError(f"num_kv_heads ({num_kv_heads}) must be in [1, 4096]")


def alloc_pools(num_pages, num_kv_heads, page_size, head_dim, block_size, cache_dtype, device=None):
    """(K_cache, V_cache, K_scale, V_scale), zeros."""
    dev = default_device(device)
    codes, scales = (num_pages, num_kv_heads, page_size, head_dim), (num_pages, num_kv_heads, page_size // block_size)
    make = lambda shape, dtype: torch.zeros(shape, dtype=torch.uint8, device=dev).view(dtype)  # noqa: E731
    return make(codes, cache_dtype), make(codes, cache_dtype), make(scales, torch.uint8), make(scales, torch.uint8)


def read_exp(e):
    """Exponents as they are read: 255 as it is, others within [67, 187]."""
    e = e.to(torch.int32)
    return torch.where(e == NAN_EXP, e, e.clamp(LOW_EXP, HIGH_EXP))


def exp2_of(e):
    """2^(e - 127) in fp32, from the bits; 255 is NaN."""
    e = e.to(torch.int32)
    return torch.where(e == NAN_EXP, torch.nan, (e.clamp(1, 254) << 23).view(torch.float32))


def needed_exponent(amax, cache_dtype):
    """Least e with amax <= TOP 2^(e - 127), within the range of scales (amax finite)."""
    m, x = torch.frexp(amax)
    tm, tx = torch.frexp(torch.tensor(TOP[cache_dtype]))
    e = 127 + x - int(tx) + (m > float(tm)).to(x.dtype)
    return torch.where(amax > 0, e, LOW_EXP).clamp(LOW_EXP, HIGH_EXP).to(torch.int32)


def to_codes(y, cache_dtype):
    """Rows in units of their scale, rounded: bytes."""
    top = TOP[cache_dtype]
    if cache_dtype == torch.int8:
        return y.nan_to_num(0.0, top, -top).clamp(-top, top).round().to(torch.int8).view(torch.uint8)
    y = torch.where(y.isfinite(), y.clamp(-top, top), torch.nan)
    return y.to(torch.float8_e4m3fn).view(torch.uint8)


def read_rows(cache, scale, slots, block_size):
    """Rows of valid slots in fp32, [n, Hkv, D]."""
    P = cache.shape[2]
    page, row = slots // P, slots % P
    codes = cache.view(torch.uint8)[page, :, row].view(cache.dtype).float()
    return codes * exp2_of(read_exp(scale[page, :, row // block_size]))[..., None]


def random_cache(num_pages, num_kv_heads, page_size, head_dim, block_size, cache_dtype, device):
    """(K_cache, V_cache, K_scale, V_scale) of normal rows, every block quantised as a whole."""
    if torch.device(device).type == "meta":
        return alloc_pools(num_pages, num_kv_heads, page_size, head_dim, block_size, cache_dtype, device)
    codes, scales = [], []
    for _ in range(2):
        x = torch.randn(num_pages, num_kv_heads, page_size // block_size, block_size * head_dim)
        e = needed_exponent(x.abs().amax(-1), cache_dtype)
        c = to_codes(x * exp2_of(254 - e)[..., None], cache_dtype)
        codes.append(c.reshape(num_pages, num_kv_heads, page_size, head_dim).to(device).view(cache_dtype))
        scales.append(e.to(torch.uint8).to(device))
    return codes[0], codes[1], scales[0], scales[1]


class _CacheRowsOp(Op):
    _params_desc = {
        "num_tokens": "Rows of packed tokens",
        "num_kv_heads": "KV heads",
        "head_dim": "Dimension per head (64 or 128)",
        "page_size": "Cache rows per page (power of two >= 32)",
        "num_pages": "Pages in the cache pools",
        "cache_dtype": "torch.int8 or torch.float8_e4m3fn",
        "block_size": "Rows of a page that share a scale (power of two in [16, 256])",
    }
    _name = ""

    def __init__(self, num_tokens: int, num_kv_heads: int, head_dim: int, page_size: int, num_pages: int,
                 backend: str = "ref", *, cache_dtype: torch.dtype = torch.int8, block_size: int = 32):
        check_rows(num_tokens, num_kv_heads)
        check_cache(page_size, num_pages, block_size, cache_dtype, head_dim)
        self.num_tokens, self.num_kv_heads, self.head_dim = num_tokens, num_kv_heads, head_dim
        self.page_size, self.num_pages, self.cache_dtype, self.block_size = page_size, num_pages, cache_dtype, block_size
        self._backend = backend
        if backend != "ref":
            self._kernel = get_kernel(self._name, backend)(num_tokens, num_kv_heads, head_dim, page_size, num_pages,
                                                           cache_dtype=cache_dtype, block_size=block_size)
        else:
            self._kernel = self._ref_forward

    def alloc(self, device=None):
        """Pools of zeros: (K_cache, V_cache, K_scale, V_scale)."""
        return alloc_pools(self.num_pages, self.num_kv_heads, self.page_size, self.head_dim, self.block_size,
                           self.cache_dtype, device)

    def _random_cache(self, dev):
        return random_cache(self.num_pages, self.num_kv_heads, self.page_size, self.head_dim, self.block_size,
                            self.cache_dtype, dev)

    def _slots(self, dev):
        """The first num_tokens rows of the pool, page by page; -1 behind its end."""
        t = torch.arange(self.num_tokens, dtype=torch.int64)
        return torch.where(t < self.num_pages * self.page_size, t, -1).to(dev)

    def get_roofline(self) -> RooflineResult:
        T, row = self.num_tokens, self.num_kv_heads * self.head_dim
        b = T * (6 * row + 8) + 2 * -(-T // self.block_size) * self.num_kv_heads
        return RooflineResult(0, b, b)

    def _live(self, slot_mapping):
        return (slot_mapping >= 0) & (slot_mapping < self.num_pages * self.page_size)


class KvCacheQuantOp(_CacheRowsOp):
    _name = "kv_cache_quant"
    _atol = 0
    _rtol = 0

    def forward(self, k, v, K_cache, V_cache, K_scale, V_scale, slot_mapping):
        """k / v [T, Hkv, D] bf16 (tokens may lie apart: slices of a packed projection), slot_mapping [T] int64.  Writes
        the pools in place and returns them."""
        return self._kernel(k, v, K_cache, V_cache, K_scale, V_scale, slot_mapping)

    def gen_data(self, device=None):
        dev = default_device(device)
        bf = dict(dtype=torch.bfloat16, device=dev)
        shape = (self.num_tokens, self.num_kv_heads, self.head_dim)
        return randn(*shape, **bf), randn(*shape, **bf), *self._random_cache(dev), self._slots(dev)

    def check(self, actual, expected) -> bool:
        return all(torch.equal(a.view(torch.uint8), e.view(torch.uint8)) for a, e in zip(actual, expected, strict=True))

    def _ref_forward(self, k, v, K_cache, V_cache, K_scale, V_scale, slot_mapping):
        """Run by run."""
        P, blk, T = self.page_size, self.block_size, self.num_tokens
        slots, live = slot_mapping.tolist(), self._live(slot_mapping).tolist()
        t = 0
        while t < T:
            n = 1
            if live[t]:
                page, row = slots[t] // P, slots[t] % P
                off = row % blk
                while n < blk - off and t + n < T and slots[t + n] == slots[t] + n:
                    n += 1
                for x, cache, scale in ((k, K_cache, K_scale), (v, V_cache, V_scale)):
                    self._write(x[t:t + n].float(), cache.view(torch.uint8)[page, :, row - off:row - off + blk],
                                scale[page, :, row // blk], off)
            t += n
        return K_cache, V_cache, K_scale, V_scale

    def _write(self, x, rows, scale, off):
        """x [n, Hkv, D] into rows [Hkv, block, D] (bytes) from ``off`` on, scale [Hkv]."""
        n, dt = x.shape[0], self.cache_dtype
        finite = x.isfinite()
        e = needed_exponent(torch.where(finite, x.abs(), 0.0).amax((0, 2)), dt)
        if dt == torch.int8:
            e = torch.where(finite.all(2).all(0), e, NAN_EXP)
        old = read_exp(scale) if off else torch.zeros_like(e)
        e = torch.maximum(e, old)
        if off:
            held = rows[:, :off].view(dt).float()
            factor = torch.where(e == NAN_EXP, 0.0, exp2_of(127 + old - e))
            turned = to_codes(held * factor[:, None, None], dt)
            rows[:, :off] = torch.where((e > old)[:, None, None], turned, rows[:, :off])
        y = x * torch.where(e == NAN_EXP, 0.0, exp2_of(254 - e))[None, :, None]
        if dt == torch.int8:
            y = torch.where((e == NAN_EXP)[None, :, None], 0.0, y)
        rows[:, off:off + n] = to_codes(y, dt).transpose(0, 1)
        scale.copy_(e.to(torch.uint8))


class KvCacheDequantOp(_CacheRowsOp):
    _name = "kv_cache_dequant"
    _atol = 0
    _rtol = 0

    def forward(self, K_cache, V_cache, K_scale, V_scale, slot_mapping, *, k_out=None, v_out=None):
        """Rows of slots slot_mapping [T] (any order, any slot more than once) in bf16: (k_out, v_out) [T, Hkv, D].  Rows
        of slots outside the pool are not written."""
        return self._kernel(K_cache, V_cache, K_scale, V_scale, slot_mapping, k_out=k_out, v_out=v_out)

    def gen_data(self, device=None):
        dev = default_device(device)
        return *self._random_cache(dev), self._slots(dev)

    def check(self, actual, expected) -> bool:
        return all(torch.equal(a, e) for a, e in zip(actual, expected, strict=True))

    def _ref_forward(self, K_cache, V_cache, K_scale, V_scale, slot_mapping, *, k_out=None, v_out=None):
        live = self._live(slot_mapping)
        got = []
        for out, cache, scale in ((k_out, K_cache, K_scale), (v_out, V_cache, V_scale)):
            if out is None:
                out = torch.empty(self.num_tokens, self.num_kv_heads, self.head_dim, dtype=torch.bfloat16,
                                  device=cache.device)
            out[live] = read_rows(cache, scale, slot_mapping[live], self.block_size).to(torch.bfloat16)
            got.append(out)
        return tuple(got)
