"""Timed cases of the 8-bit KV cache: inputs, one pass, its work and its result in 64 bits.

Four ops over page pools whose rows are held in 8 bits (``int8`` or ``e4m3``) with a power-of-two scale for each block of
tokens and kv head:

  store    new tokens' k and v quantised into their slots, and the rows of the blocks they touch read back
           (``KvCacheQuantOp``, ``KvCacheDequantOp``)
  load     cached rows read back to bf16 (``KvCacheDequantOp``)
  decode   attention of one token per sequence over its cached rows (``QuantPagedAttnDecodeOp``)
  prefill  causal attention of packed prompts and chunks over the rows cached up to each token (``QuantPrefillAttnOp``)

A case is a dict of plain values with an ``op`` key; ragged lengths come from the case's ``lens_seed``, so they are part
of the case, the tensors' values from the seed that ``prepare`` is given.  With ``own`` false ``run`` computes an op from
elementary torch operations, with ``own`` true it calls the package's op.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

BF, F32, F64, I32, I64, U8 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.int64, torch.uint8
TYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}
LOW, HIGH = 127 - 60, 127 + 60  # scales lie in 2^-60 .. 2^60
DEV = "cuda"
_PKG = str(Path(__file__).resolve().parent.parent / "ez-ops_amd")


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one decode step of 64 conversations: a token each into blocks begun before (latency)
        dict(name="store_decode_b64", op="store", cache="int8", seqs=64, new_min=1, new_max=1, past_min=100,
             past_max=4000, pad=0, kv_heads=8, head_dim=128, page=64, block=32, packed=True, lens_seed=21),
        # chunks of a mixed step on cached prefixes, single tokens and idle rows among them, a padded batch
        dict(name="store_mixed_37", op="store", cache="e4m3", seqs=37, new_min=0, new_max=190, past_min=0,
             past_max=3000, pad=77, kv_heads=8, head_dim=128, page=64, block=16, packed=True, lens_seed=22),
        # a long fresh prompt of the 8B layer
        dict(name="store_prompt_t16384", op="store", cache="int8", seqs=1, new_min=16384, new_max=16384, past_min=0,
             past_max=0, pad=0, kv_heads=8, head_dim=128, page=128, block=64, packed=True, lens_seed=23),
        # a short cached prefix handed to another worker (latency)
        dict(name="load_t333", op="load", cache="e4m3", seqs=1, new_min=0, new_max=0, past_min=333, past_max=333, pad=0,
             kv_heads=8, head_dim=128, page=32, block=32, packed=True, lens_seed=24),
        # the caches of three conversations read back
        dict(name="load_t40000", op="load", cache="int8", seqs=3, new_min=0, new_max=0, past_min=10000, past_max=16000,
             pad=5, kv_heads=8, head_dim=128, page=64, block=32, packed=True, lens_seed=25),
        # one token of a single conversation (latency)
        dict(name="decode_b1", op="decode", cache="e4m3", seqs=1, kv_min=2000, kv_max=2000, heads=32, kv_heads=8,
             head_dim=128, page=64, max_pages=64, block=32, lens_seed=26),
        # a ragged batch of the small layer, a few rows of it idle
        dict(name="decode_b48_ragged", op="decode", cache="int8", seqs=48, kv_min=0, kv_max=4096, heads=16, kv_heads=8,
             head_dim=128, page=64, max_pages=64, block=16, lens_seed=27),
        # long conversations of the 8B layer
        dict(name="decode_b32_s16384", op="decode", cache="e4m3", seqs=32, kv_min=16000, kv_max=16384, heads=32,
             kv_heads=8, head_dim=128, page=128, max_pages=128, block=64, lens_seed=28),
        # a short question on a cached document (latency)
        dict(name="prefill_t70_on_3000", op="prefill", cache="int8", seqs=1, new_min=70, new_max=70, past_min=3000,
             past_max=3000, pad=0, heads=32, kv_heads=8, head_dim=128, page=64, max_pages=64, block=32, packed=True,
             lens_seed=29),
        # chunks and single tokens of a mixed step on cached prefixes, heads of 64 dims
        dict(name="prefill_mixed_9", op="prefill", cache="e4m3", seqs=9, new_min=1, new_max=700, past_min=0,
             past_max=2500, pad=33, heads=16, kv_heads=2, head_dim=64, page=32, max_pages=128, block=32, packed=False,
             lens_seed=30),
        # a fresh prompt of the 8B layer
        dict(name="prefill_t4096", op="prefill", cache="int8", seqs=1, new_min=4096, new_max=4096, past_min=0,
             past_max=0, pad=0, heads=32, kv_heads=8, head_dim=128, page=64, max_pages=64, block=64, packed=True,
             lens_seed=31),
        # a chunk of a very long prompt of the 8B layer
        dict(name="prefill_t2048_on_30000", op="prefill", cache="e4m3", seqs=1, new_min=2048, new_max=2048,
             past_min=30000, past_max=30000, pad=0, heads=32, kv_heads=8, head_dim=128, page=128, max_pages=256,
             block=32, packed=True, lens_seed=32),
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], uniform in its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["store", "store", "load", "decode", "decode", "decode", "prefill", "prefill", "prefill"])
    seed = rng.randrange(1 << 20)
    page = rng.choice([32, 64, 128, 256])
    kv, D = rng.choice([1, 2, 4, 8, 8, 16]), rng.choice([64, 128, 128])
    c = dict(op=op, cache=rng.choice(["int8", "e4m3"]), kv_heads=kv, head_dim=D, page=page,
             block=rng.choice([b for b in (16, 32, 64, 128, 256) if b <= page]), lens_seed=seed)
    if op in ("store", "load"):
        seqs = _log(rng, 1, 128)
        each = max(1, (1 << 24) // (kv * D * seqs))  # tokens a sequence may bring
        if op == "load":
            n = _log(rng, 1, min(each, 40000))
            return dict(c, seqs=seqs, new_min=0, new_max=0, past_min=rng.choice([n, n // 2 + 1]), past_max=n,
                        pad=rng.choice([0, 5]), packed=True)
        n = _log(rng, 1, min(each, 16384))
        past = _log(rng, 1, 4000)
        return dict(c, seqs=seqs, new_min=rng.choice([0, n // 2, n]), new_max=n, past_min=0,
                    past_max=rng.choice([0, past, past]), pad=rng.choice([0, 9]), packed=rng.random() < 0.7)
    g = rng.choice([1, 2, 4, 4, 8, 16] if op == "decode" else [1, 2, 4, 4, 8])
    c.update(heads=kv * g, seqs=_log(rng, 1, 100 if op == "decode" else 16))
    if op == "decode":
        cap = min(30000, (1 << 28) // (kv * D * c["seqs"]), (1 << 29) // (kv * g * D * c["seqs"]) * 4)
        n = _log(rng, 1, max(1, cap))
        return dict(c, kv_min=rng.choice([0, n // 2, n]), kv_max=n, max_pages=-(-n // page) + rng.choice([0, 3]))
    n = _log(rng, 1, max(1, min(4096, (1 << 24) // (kv * g * D * c["seqs"]))))
    past = _log(rng, 1, max(1, min(20000, (1 << 33) // (kv * g * D * c["seqs"] * n))))
    return dict(c, new_min=rng.choice([0, 1, n]), new_max=n, past_min=0, past_max=rng.choice([0, past, past]),
                pad=rng.choice([0, 9]), max_pages=-(-(n + past) // page) + rng.choice([0, 2]), packed=rng.random() < 0.7)


# ---------------------------------------------------------------- inputs
def _lens(c):
    """(new tokens, rows cached before them) of every sequence."""
    r = random.Random(c["lens_seed"])
    if c["op"] == "decode":
        kv = [r.randint(c["kv_min"], c["kv_max"]) for _ in range(c["seqs"])]
        kv[0] = c["kv_max"]
        return [min(1, n) for n in kv], [max(0, n - 1) for n in kv]
    new = [r.randint(c["new_min"], c["new_max"]) for _ in range(c["seqs"])]
    if not sum(new):
        new[0] = c["new_max"]
    return new, [r.randint(c["past_min"], c["past_max"]) for _ in range(c["seqs"])]


def _ints(v, dtype=I32):
    return torch.tensor(v, dtype=dtype, device=DEV)


def _pow2(e):
    """2^(e - 127) in fp32, from its bits."""
    return (e.to(I32).clamp(0, 254) << 23).view(F32)


def _exponent(amax, cache):
    """The least e with amax <= TOP 2^(e - 127), within the range of scales."""
    m, x = torch.frexp(amax)
    tm, tx = math.frexp(TOP[cache])
    e = 127 + x - tx + (m > tm).to(x.dtype)
    return torch.where(amax > 0, e, LOW).clamp(LOW, HIGH).to(I32)


def _codes(y, cache):
    """Rows in units of their scale, rounded to codes: bytes."""
    y = y.clamp(-TOP[cache], TOP[cache])
    return (y.round().to(torch.int8) if cache == "int8" else y.to(torch.float8_e4m3fn)).view(U8)


def _pools(c, pages, g):
    """Pools whose blocks are quantised as they stand: rows of k with a few strong channels, rows of v."""
    Hkv, D, P, blk = c["kv_heads"], c["head_dim"], c["page"], c["block"]
    got = []
    for kind in "kv":
        amp = torch.exp(0.4 * torch.randn(Hkv, 1, D, generator=g, device=DEV))
        if kind == "k":
            amp[:, :, ::37] *= 4
        codes = torch.empty(pages, Hkv, P, D, dtype=U8, device=DEV)
        scale = torch.empty(pages, Hkv, P // blk, dtype=U8, device=DEV)
        step = max(1, (1 << 27) // (Hkv * P * D))
        for at in range(0, pages, step):
            x = torch.randn(codes[at:at + step].shape, generator=g, device=DEV) * amp
            e = _exponent(x.reshape(-1, Hkv, P // blk, blk * D).abs().amax(-1), c["cache"])
            codes[at:at + step] = _codes(x * _pow2(254 - e).repeat_interleave(blk, 2)[..., None], c["cache"])
            scale[at:at + step] = e.to(U8)
        got += [codes.view(TYPES[c["cache"]]), scale]
    return got


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    P, blk, Hkv, D = c["page"], c["block"], c["kv_heads"], c["head_dim"]
    new, past = _lens(c)
    need = [-(-(p + n) // P) for n, p in zip(new, past)]
    width = c.get("max_pages") or max(1, *need)
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEV).tolist()
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    K, Ks, V, Vs = _pools(c, pages, g)
    s = dict(c=c, K=K, Ks=Ks, V=V, Vs=Vs, pages=pages, new=new, past=past, table=_ints(table))
    if c["op"] == "decode":
        s["q"] = torch.randn(c["seqs"], c["heads"], D, generator=g, device=DEV).to(BF)
        s["kv_lens"], s["longest"] = _ints([n + p for n, p in zip(new, past)]), max(n + p for n, p in zip(new, past))
        return s
    T = sum(new) + c["pad"]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    if c["op"] == "prefill":
        H = c["heads"]
        x = torch.randn(T, H + 2 * Hkv if c["packed"] else H, D, generator=g, device=DEV).to(BF)
        s.update(q=x[:, :H], cu=_ints(cu), past_lens=_ints(past), longest=max(n + p for n, p in zip(new, past)),
                 out=torch.zeros(T, H, D, dtype=BF, device=DEV))
        return s
    slot = lambda b, r: table[b][r // P] * P + r % P  # noqa: E731
    if c["op"] == "store":
        slots = [slot(b, p + i) for b, (n, p) in enumerate(zip(new, past)) for i in range(n)]
        back = [slot(b, r) for b, (n, p) in enumerate(zip(new, past)) if n for r in range(p // blk * blk, p + n)]
        x = torch.randn(T, 2 * Hkv, D, generator=g, device=DEV) * torch.exp(0.7 * torch.randn(T, 1, 1, generator=g, device=DEV))
        k, v = x.to(BF)[:, :Hkv], x.to(BF)[:, Hkv:]
        s.update(k=k if c["packed"] else k.contiguous(), v=v if c["packed"] else v.contiguous(),
                 slots=_ints(slots + [-1] * c["pad"], I64))
        # the blocks that the call touches: the block of every token, the first row that each block gets
        blocks = [x // blk for x in slots]
        seen = {}
        for x in slots:
            seen.setdefault(x // blk, (len(seen), x % blk))
        s.update(touched=_ints(list(seen), I64), block_of=_ints([seen[x][0] for x in blocks], I64),
                 first=_ints([f for _, f in seen.values()], I64), live=sum(new))
    else:
        back = [slot(b, r) for b, p in enumerate(past) for r in range(p)] + [-1] * c["pad"]
    s.update(back=_ints(back, I64), k_out=torch.zeros(len(back), Hkv, D, dtype=BF, device=DEV),
             v_out=torch.zeros(len(back), Hkv, D, dtype=BF, device=DEV))
    return s


# ---------------------------------------------------------------- the package's ops
def _ops(s):
    """The case's ops, which a program makes once and keeps."""
    if "ops" not in s:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        import ezops

        c = s["c"]
        how = dict(backend="hip", cache_dtype=TYPES[c["cache"]], block_size=c["block"])
        if c["op"] in ("store", "load"):
            pool = (c["kv_heads"], c["head_dim"], c["page"], s["pages"])
            s["ops"] = [ezops.KvCacheDequantOp(s["back"].numel(), *pool, **how)]
            if c["op"] == "store":
                s["ops"].append(ezops.KvCacheQuantOp(s["slots"].numel(), *pool, **how))
        else:
            shape = (c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["max_pages"], s["pages"])
            if c["op"] == "decode":
                s["ops"] = [ezops.QuantPagedAttnDecodeOp(c["seqs"], *shape, **how)]
            else:
                s["ops"] = [ezops.QuantPrefillAttnOp(c["seqs"], s["q"].shape[0], *shape, **how)]
    return s["ops"]


# ---------------------------------------------------------------- one pass
def run(s):
    op = s["c"]["op"]
    pools = (s["K"], s["V"], s["Ks"], s["Vs"])
    if op in ("store", "load"):
        if own:
            ops = _ops(s)
            if op == "store":
                ops[1](s["k"], s["v"], *pools, s["slots"])
            ops[0](*pools, s["back"], k_out=s["k_out"], v_out=s["v_out"])
        else:
            if op == "store":
                _write(s, s["K"], s["Ks"], s["k"])
                _write(s, s["V"], s["Vs"], s["v"])
            _read(s, s["K"], s["Ks"], s["k_out"])
            _read(s, s["V"], s["Vs"], s["v_out"])
        return [s["k_out"], s["v_out"]]
    if op == "decode":
        if own:
            return _ops(s)[0](s["q"], *pools, s["table"], s["kv_lens"], s["longest"])
        return _decode(s)
    if own:
        return _ops(s)[0](s["q"], *pools, s["table"], s["cu"], s["past_lens"], max_kv_len=s["longest"], out=s["out"])
    return _prefill(s)


def _write(s, pool, scale, x):
    c = s["c"]
    blk, P, Hkv, D = c["block"], c["page"], c["kv_heads"], c["head_dim"]
    n, of, first = s["live"], s["block_of"], s["first"][:, None]
    x = x[:n].float()
    page, j = s["touched"] // (P // blk), s["touched"] % (P // blk)
    top = torch.zeros(page.numel(), Hkv, device=DEV)
    top.scatter_reduce_(0, of[:, None].expand(n, Hkv), x.abs().amax(-1), "amax")
    old = torch.where(first > 0, scale[page, :, j].to(I32), 0)
    e = torch.maximum(_exponent(top, c["cache"]), old)
    scale[page, :, j] = e.to(U8)
    # rows that a block held before, in units of its new scale
    rows = pool.view(U8).view(-1, Hkv, P // blk, blk, D)
    held = rows[page, :, j]
    turned = _codes(held.view(pool.dtype).float() * _pow2(127 + old - e)[..., None, None], c["cache"])
    keep = (torch.arange(blk, device=DEV) < first)[:, None, :, None]
    rows[page, :, j] = torch.where(keep, turned, held)
    slot = s["slots"][:n]
    pool.view(U8)[slot // P, :, slot % P] = _codes(x * _pow2(254 - e)[of][..., None], c["cache"])


def _read(s, pool, scale, out):
    c = s["c"]
    n = s["back"].numel() - (c["pad"] if c["op"] == "load" else 0)
    slot = s["back"][:n]
    page, row = slot // c["page"], slot % c["page"]
    x = pool.view(U8)[page, :, row].view(pool.dtype).float() * _pow2(scale[page, :, row // c["block"]])[..., None]
    out[:n] = x.to(BF)


def _rows(s, pool, scale, table):
    """[..., pages] table -> its rows in fp32, [..., Hkv, pages * P, D]."""
    c = s["c"]
    x = pool.view(U8)[table].view(pool.dtype).float() * _pow2(scale[table]).repeat_interleave(c["block"], -1)[..., None]
    return x.transpose(-4, -3).flatten(-3, -2)


def _decode(s):
    c = s["c"]
    B, H, Hkv, D = c["seqs"], c["heads"], c["kv_heads"], c["head_dim"]
    table = s["table"][:, :max(1, -(-s["longest"] // c["page"]))].clamp(min=0).long()
    k, v = _rows(s, s["K"], s["Ks"], table), _rows(s, s["V"], s["Vs"], table)
    p = s["q"].float().reshape(B, Hkv, H // Hkv, D) @ k.transpose(-1, -2).contiguous() * D ** -0.5
    p = p.masked_fill(torch.arange(k.shape[2], device=DEV) >= s["kv_lens"][:, None, None, None], -torch.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True).clamp(min=-1e30))
    out = p @ v / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return out.reshape(B, H, D).to(BF)


def _prefill(s):
    c = s["c"]
    H, Hkv, D, P = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    at = 0
    for b, (n, past) in enumerate(zip(s["new"], s["past"])):
        if n:
            L = past + n
            table = s["table"][b, :-(-L // P)].long()
            k, v = (_rows(s, *x, table)[:, :L].contiguous() for x in ((s["K"], s["Ks"]), (s["V"], s["Vs"])))
            q = s["q"][at:at + n].float().reshape(n, Hkv, H // Hkv, D).permute(1, 2, 0, 3).reshape(Hkv, -1, D)
            p = q @ k.transpose(-1, -2).contiguous() * D ** -0.5
            hidden = torch.arange(L, device=DEV) > past + torch.arange(n, device=DEV)[:, None]
            p = p.reshape(Hkv, H // Hkv, n, L).masked_fill_(hidden, -torch.inf)
            p = p.sub_(p.amax(-1, keepdim=True)).exp_()
            o = (p.reshape(Hkv, -1, L) @ v).reshape(H, n, D) / p.sum(-1).reshape(H, n, 1)
            s["out"][at:at + n] = o.transpose(0, 1).to(BF)
        at += n
    return s["out"]


# ---------------------------------------------------------------- its work
def work(case):
    c = case
    new, past = _lens(c)
    Hkv, D, blk = c["kv_heads"], c["head_dim"], c["block"]
    row = 2 * Hkv * D  # codes of a token's k and v
    scales = lambda r: 2 * Hkv * (-(-r // blk))  # noqa: E731  (of r rows in a run)
    if c["op"] in ("store", "load"):
        if c["op"] == "load":
            back = sum(past)
            return {"bytes": back * (row + 2 * row + 8) + sum(scales(p) for p in past), "flops": 0}
        runs = [p % blk + n for n, p in zip(new, past) if n]
        back, T = sum(runs), sum(new)
        # bf16 rows in, their codes and scales out; then codes and scales in, bf16 rows out
        return {"bytes": T * (2 * row + row + 8) + back * (row + 2 * row + 8) + 2 * sum(scales(r) for r in runs), "flops": 0}
    H = c["heads"]
    kv = [n + p if n else 0 for n, p in zip(new, past)]
    pairs = sum(kv) if c["op"] == "decode" else sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past))
    tables = sum(4 * -(-n // c["page"]) + 8 for n in kv)
    return {"bytes": sum(n * row + scales(n) for n in kv) + 4 * sum(new) * H * D + tables, "flops": 4 * pairs * H * D}


# ---------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(dict(case), seed)
    return {"store": _exact_rows, "load": _exact_rows, "decode": _exact_attn, "prefill": _exact_attn}[s["c"]["op"]](s)


def _two(e):
    """2^e in 64 bits, from its bits."""
    return (e.to(I64) + 1023 << 52).view(F64)


def _above(x):
    """The least e with x <= 2^e (x > 0): an estimate, put right by comparisons."""
    e = torch.ceil(torch.log2(x)).clamp(-1000, 1000)
    e = e + (x > _two(e))
    return torch.where(x <= _two(e - 1), e - 1, e)


def _held(s, name, b, lo, hi):
    """Rows lo .. hi - 1 of a sequence as the pool holds them, one by one: [rows, Hkv, D]."""
    c, pool, scale = s["c"], s[name], s[name + "s"]
    r = torch.arange(lo, hi, device=DEV)
    page = s["table"][b].long()[r // c["page"]]
    x = pool.view(U8)[page, :, r % c["page"]].view(pool.dtype).to(F32).double()
    return x * _two(scale[page, :, r % c["page"] // c["block"]].to(I64) - 127)[..., None]


def _rounded(x, e, cache):
    """Values nearest to x among those that codes of scale 2^e stand for, ties to even."""
    y = x / _two(e)
    step = torch.ones_like(y)
    if cache == "e4m3":  # four significant bits, down to 2^-9: |y| in [2^(n-1), 2^n) has steps of 2^(n-4)
        size = y.abs().clamp(min=2.0 ** -6)
        n = _above(size)
        step = _two(n + (size == _two(n)) - 4)
    return ((y / step).round() * step).clamp(-TOP[cache], TOP[cache]) * _two(e)


def _exact_rows(s):
    """Sequence by sequence, the rows in blocks."""
    c = s["c"]
    blk, Hkv, D = c["block"], c["kv_heads"], c["head_dim"]
    got = []
    for name in "KV":
        out = s[name.lower() + "_out"].double()
        row = at = 0
        for b, (n, past) in enumerate(zip(s["new"], s["past"])):
            if c["op"] == "load":
                out[at:at + past] = _held(s, name, b, 0, past)
                at += past
                continue
            if not n:
                continue
            lo = past // blk * blk
            count = -(-(past + n - lo) // blk)
            x = torch.zeros(count * blk, Hkv, D, dtype=F64, device=DEV)
            x[past - lo:past - lo + n] = s[name.lower()][row:row + n].double()
            most = x.reshape(count, blk, Hkv, D).abs().amax((1, 3))
            # TOP is 127/128 of 2^7 or 7/8 of 2^9: the quotient is a power of two only where it is exact
            e = _above((most / TOP[c["cache"]]).clamp(min=2.0 ** -100)).clamp(LOW - 127, HIGH - 127)
            if past > lo:  # a block begun before: its scale does not fall, its rows are rounded again
                page = int(s["table"][b, lo // c["page"]])
                e[0] = torch.maximum(e[0], s[name + "s"][page, :, lo % c["page"] // blk].double() - 127)
                x[:past - lo] = _held(s, name, b, lo, past)
            x = _rounded(x.reshape(count, blk, Hkv, D), e[:, None, :, None], c["cache"]).reshape(-1, Hkv, D)
            out[at:at + past + n - lo] = x[:past + n - lo]
            at += past + n - lo
            row += n
        got.append(out)
    return got


def _exact_attn(s):
    """Sequence by sequence and kv head by kv head, a few hundred queries at a time."""
    c = s["c"]
    H, Hkv, D = c["heads"], c["kv_heads"], c["head_dim"]
    G = H // Hkv
    out = torch.zeros(s["q"].shape, dtype=F64, device=DEV)
    at = 0
    for b, (n, past) in enumerate(zip(s["new"], s["past"])):
        at = b if c["op"] == "decode" else at
        if n:
            k, v = (_held(s, x, b, 0, past + n).transpose(0, 1).contiguous() for x in "KV")
            for h in range(Hkv):
                for i in range(0, n, 512):
                    m = min(512, n - i)
                    q = s["q"][at + i:at + i + m, h * G:(h + 1) * G].double().reshape(m * G, D)
                    x = (q @ k[h].t().contiguous()).reshape(m, G, -1) / math.sqrt(D)
                    far = torch.arange(past + n, device=DEV) > past + i + torch.arange(m, device=DEV)[:, None]
                    w = torch.softmax(x.masked_fill(far[:, None], -torch.inf), -1).reshape(m * G, -1)
                    out[at + i:at + i + m, h * G:(h + 1) * G] = (w @ v[h]).reshape(m, G, D)
        at += n
    return out
