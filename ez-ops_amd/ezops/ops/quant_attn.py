"""GQA attention over a paged KV cache held in 8 bits: one token per sequence, and packed prompts.

No reference counterpart (its attention reads a contiguous bf16 cache,
ezops/ops/attn_decode.py:9-67); these ops are PagedAttnDecodeOp and PrefillAttnOp over
the pools of KvCacheQuantOp: codes ``[num_pages, Hkv, page_size, D]`` (int8 or e4m3) with
an exponent for each block of ``block_size`` rows and kv head.  With k_j and v_j the rows
that the codes stand for

    o = sum_j softmax_j(scale * q . k_j) v_j

over the rows that a query sees: the first ``kv_lens[b]`` of its sequence (decode), or
rows ``0 .. past_lens[b] + i`` for the sequence's new token ``i`` (prefill; the new tokens
are in the cache already).  Query head ``h`` reads kv head ``h // (H / Hkv)``;
``block_table [B, max_pages]`` (int32) maps logical pages to pool pages.  Ids of pages that
hold visible rows must lie in the pool (others are read as a page of it); codes and scales
of rows that no query sees may hold anything.  The scale is any positive
number of fp32.  Products of q with a row's codes have to stay below 2^128, and so do scores
and, unless all of a row's codes are 0, ``1.45 * scale * 2^(e - 127)`` of its block; past that the
query's own output is undefined.
"""

import operator

import torch

from ..registry import get_kernel
from .base_op import Op, default_device, randn
from .kv_cache_quant import check_cache, exp2_of, random_cache, read_exp
from .linear_attn import GROUPS, _scale
from .utils.roofline import RooflineResult


def cache_rows(cache, scale, table, block_size):
    """Rows of the pages of ``table`` [n] in fp32: [Hkv, n * page_size, D]."""
    x = cache.view(torch.uint8)[table].view(cache.dtype).float()
    x = x * exp2_of(read_exp(scale[table])).repeat_interleave(block_size, -1)[..., None]
    return x.transpose(0, 1).flatten(1, 2)


MAX_ROWS = 1 << 30  # of a block table


def bound(max_kv_len):
    """A caller's bound on the lengths as the kernels take it; 0 for none."""
    n = operator.index(max_kv_len)
    if n < 0:
        raise ValueError(f"max_kv_len ({max_kv_len}) must be >= 0")
    return min(n, MAX_ROWS)


class _QuantAttnOp(Op):
    _atol = 1e-2
    _rtol = 1e-2
    _name = ""

    def _setup(self, batch, rows, num_heads, num_kv_heads, head_dim, page_size, max_pages, num_pages, backend, cache_dtype,
               block_size, scale, *args):
        if not 1 <= batch <= 65536:
            raise ValueError(f"batch ({batch}) must be in [1, 65536]")
        if not 1 <= rows < 1 << 30:
            raise ValueError(f"num_tokens ({rows}) must be in [1, 2^30)")
        if num_kv_heads < 1 or not 1 <= num_heads <= 4096 or num_heads % num_kv_heads:
            raise ValueError(f"num_heads ({num_heads}) must be divisible by num_kv_heads ({num_kv_heads}) and at most 4096")
        if num_heads // num_kv_heads not in GROUPS:
            raise ValueError(f"GQA group size {num_heads}/{num_kv_heads} not supported (1, 2, 4, 8 or 16)")
        if max_pages < 1 or max_pages * page_size > MAX_ROWS:
            raise ValueError(f"max_pages ({max_pages}) must be >= 1 and max_pages * page_size at most 2^30")
        num_pages = batch * max_pages if num_pages is None else num_pages
        check_cache(page_size, num_pages, block_size, cache_dtype, head_dim)
        self.batch, self.num_heads, self.num_kv_heads, self.head_dim = batch, num_heads, num_kv_heads, head_dim
        self.page_size, self.max_pages, self.num_pages = page_size, max_pages, num_pages
        self.cache_dtype, self.block_size, self.scale = cache_dtype, block_size, _scale(scale, head_dim)
        self._rows = rows
        self._backend = backend
        if backend != "ref":
            self._kernel = get_kernel(self._name, backend)(
                *args, num_heads, num_kv_heads, head_dim, page_size, max_pages, num_pages, cache_dtype=cache_dtype,
                block_size=block_size, scale=self.scale)
        else:
            self._kernel = self._ref_forward

    def _gen(self, device):
        """(device, q, the pools, a block table of distinct pages where there are enough)."""
        dev = default_device(device)
        q = randn(self._rows, self.num_heads, self.head_dim, dtype=torch.bfloat16, device=dev)
        pools = random_cache(self.num_pages, self.num_kv_heads, self.page_size, self.head_dim, self.block_size,
                             self.cache_dtype, dev)
        n = self.batch * self.max_pages
        ids = torch.randperm(self.num_pages)[:n] if self.num_pages >= n else torch.randint(0, self.num_pages, (n,))
        return dev, q, pools, ids.reshape(self.batch, self.max_pages).to(torch.int32).to(dev)

    def _row_bytes(self, rows):
        """Codes and scales of ``rows`` cached tokens."""
        return rows * 2 * self.num_kv_heads * self.head_dim + 2 * self.num_kv_heads * -(-rows // self.block_size)

    def _attend(self, q, K, V, Ks, Vs, table, past):
        """q [n, H, D] of one sequence, query i over rows 0 .. past + i."""
        n, H, D = q.shape
        Hkv, L = self.num_kv_heads, past + n
        ids = table[:-(-L // self.page_size)].long().clamp(0, self.num_pages - 1)
        k, v = (cache_rows(c, s, ids, self.block_size)[:, None, :L] for c, s in ((K, Ks), (V, Vs)))
        x = q.float().reshape(n, Hkv, H // Hkv, D).permute(1, 2, 0, 3) @ k.transpose(-1, -2) * self.scale
        hidden = torch.arange(L, device=q.device) > past + torch.arange(n, device=q.device)[:, None]
        w = torch.softmax(x.masked_fill(hidden, -torch.inf), dim=-1)
        return (w @ v).permute(2, 0, 1, 3).reshape(n, H, D).to(torch.bfloat16)


class QuantPagedAttnDecodeOp(_QuantAttnOp):
    _params_desc = {
        "batch": "Sequences (one token each)",
        "num_heads": "Query heads",
        "num_kv_heads": "KV heads",
        "head_dim": "Dimension per head (64 or 128)",
        "page_size": "Cache rows per page (power of two >= 32)",
        "max_pages": "Block-table width (pages per sequence)",
        "num_pages": "Pages in the shared pools (default batch * max_pages)",
        "cache_dtype": "torch.int8 or torch.float8_e4m3fn",
        "block_size": "Rows of a page that share a scale (power of two in [16, 256])",
        "scale": "Factor on the scores (default head_dim ** -0.5)",
    }
    _name = "quant_paged_attn_decode"

    def __init__(self, batch: int, num_heads: int, num_kv_heads: int, head_dim: int, page_size: int, max_pages: int,
                 num_pages: int | None = None, backend: str = "ref", *, cache_dtype: torch.dtype = torch.int8,
                 block_size: int = 32, scale: float | None = None):
        self._setup(batch, batch, num_heads, num_kv_heads, head_dim, page_size, max_pages, num_pages, backend, cache_dtype,
                    block_size, scale, batch)

    def forward(self, q, K_cache, V_cache, K_scale, V_scale, block_table, kv_lens, max_kv_len: int = 0, *, out=None):
        """q [B, H, D] (rows may lie apart), kv_lens [B] int32 -> out [B, H, D]; a sequence of no rows gets zeros.
        max_kv_len: the caller's bound on the lengths (0 = max_pages * page_size), which plans the work; longer ones are
        cut off there."""
        return self._kernel(q, K_cache, V_cache, K_scale, V_scale, block_table, kv_lens, bound(max_kv_len), out=out)

    def gen_data(self, device=None):
        dev, q, pools, table = self._gen(device)
        lens = torch.randint(1, self.max_pages * self.page_size + 1, (self.batch,), dtype=torch.int32).to(dev)
        return q, *pools, table, lens

    def get_roofline(self) -> RooflineResult:
        """At full lengths."""
        rows = self.max_pages * self.page_size
        b = self.batch * (self._row_bytes(rows) + 4 * self.num_heads * self.head_dim + 4 * self.max_pages + 4)
        return RooflineResult(4 * self.batch * rows * self.num_heads * self.head_dim, b, b)

    def _ref_forward(self, q, K_cache, V_cache, K_scale, V_scale, block_table, kv_lens, max_kv_len: int = 0, *, out=None):
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out is None else out
        cap = min(max_kv_len or MAX_ROWS, self.max_pages * self.page_size)
        for b, n in enumerate(kv_lens.tolist()):
            n = min(max(n, 0), cap)
            out[b] = self._attend(q[b:b + 1], K_cache, V_cache, K_scale, V_scale, block_table[b], n - 1)[0] if n else 0
        return out


class QuantPrefillAttnOp(_QuantAttnOp):
    _params_desc = {
        "batch": "Sequences in the chunk",
        "num_tokens": "Rows of packed tokens (fewer may be used)",
        **{k: v for k, v in QuantPagedAttnDecodeOp._params_desc.items() if k != "batch"},
    }
    _name = "quant_prefill_attn"

    def __init__(self, batch: int, num_tokens: int, num_heads: int, num_kv_heads: int, head_dim: int, page_size: int,
                 max_pages: int, num_pages: int | None = None, backend: str = "ref", *,
                 cache_dtype: torch.dtype = torch.int8, block_size: int = 32, scale: float | None = None):
        self.num_tokens = num_tokens
        self._setup(batch, num_tokens, num_heads, num_kv_heads, head_dim, page_size, max_pages, num_pages, backend,
                    cache_dtype, block_size, scale, batch, num_tokens)

    def forward(self, q, K_cache, V_cache, K_scale, V_scale, block_table, cu_seqlens, past_lens=None, *,
                max_kv_len: int = 0, out=None):
        """q [T, H, D] (tokens may lie apart); sequence ``b`` owns rows cu_seqlens[b] .. cu_seqlens[b+1]-1 (int32, not
        decreasing), its token ``i`` stands at cache row past_lens[b] + i (past_lens None: 0).  Returns out [T, H, D];
        rows of no sequence, and of tokens at or past max_pages * page_size, are not written.  max_kv_len: the caller's
        bound on past + new tokens of a sequence (0 = none), which plans the work; tokens past it are not written
        either."""
        return self._kernel(q, K_cache, V_cache, K_scale, V_scale, block_table, cu_seqlens, past_lens,
                            max_kv_len=bound(max_kv_len), out=out)

    def gen_data(self, device=None):
        """The rows shared out evenly, each sequence on a few cached rows where there is room."""
        dev, q, pools, table = self._gen(device)
        cu = [self.num_tokens * b // self.batch for b in range(self.batch + 1)]
        room = self.max_pages * self.page_size
        past = [max(0, min(room - (e - s), (37 * b) % room)) for b, (s, e) in enumerate(zip(cu, cu[1:]))]
        i32 = dict(dtype=torch.int32, device=dev)
        return q, *pools, table, torch.tensor(cu, **i32), torch.tensor(past, **i32)

    def get_roofline(self) -> RooflineResult:
        """Of a fresh prompt a sequence, the rows shared out evenly."""
        B, T, H, D = self.batch, self.num_tokens, self.num_heads, self.head_dim
        n = min(T // B, self.max_pages * self.page_size)
        b = B * (self._row_bytes(n) + 4 * n * H * D + 4 * -(-n // self.page_size) + 8)
        return RooflineResult(2 * B * n * (n + 1) * H * D, b, b)

    def _ref_forward(self, q, K_cache, V_cache, K_scale, V_scale, block_table, cu_seqlens, past_lens=None, *,
                     max_kv_len: int = 0, out=None):
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out is None else out
        cap = min(max_kv_len or MAX_ROWS, self.max_pages * self.page_size)
        cu = [min(max(0, x), self.num_tokens) for x in cu_seqlens.tolist()]
        past = past_lens.tolist() if past_lens is not None else [0] * self.batch
        for b, (s, e) in enumerate(zip(cu, cu[1:])):
            p = min(max(past[b], 0), cap)
            n = min(e - s, cap - p)
            if n > 0:
                out[s:s + n] = self._attend(q[s:s + n], K_cache, V_cache, K_scale, V_scale, block_table[b], p)
        return out
