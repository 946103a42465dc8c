"""Timed cases of the ragged-batch serving ops: inputs, one pass, its work and its result in 64 bits.

Four ops of one serving step over a ragged batch:

  plan            block table, slot map, positions and offsets from request lengths (``PagedBatchPlanOp``)
  mrope           QK norm, rotary positions with several axes, cache write by slot (``QkNormMropeOp``)
  linattn         linear attention with a decay per head over packed prompts (``LinearAttnPrefillOp``)
  linattn_decode  its recurrent form for one token per sequence (``LinearAttnDecodeOp``)

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

BF, F32, F64, I32, I64 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.int64
DEV = "cuda"
EPS = 1e-6
THETA = 1e6
_PKG = str(Path(__file__).resolve().parent.parent / "ez-ops_amd")


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one decode step of 64 conversations: a token each, a page now and then (latency)
        dict(name="plan_decode_b64", op="plan", batch=64, rows=64, new_min=1, new_max=1, past_min=1024, past_max=16000,
             page=64, max_pages=256, lens_seed=11),
        # a large mixed step: prompts, chunks on cached prefixes, single tokens and idle rows, padded to a fixed row count
        dict(name="plan_mixed_b512", op="plan", batch=512, rows=32768, new_min=0, new_max=120, past_min=0, past_max=4000,
             page=32, max_pages=160, lens_seed=12),
        # one decode step of 16 multimodal conversations
        dict(name="mrope_decode_t16", op="mrope", rows=16, live=16, heads=32, kv_heads=8, head_dim=128, axes=3, s0=24,
             s1=20, s2=20, interleaved=True, norm=True, page=64, span=16384, table="bf16", packed=True),
        # a prompt of text and one image for the small vision-language layer, odd length, padded rows behind it
        dict(name="mrope_prompt_t4097", op="mrope", rows=4160, live=4097, heads=16, kv_heads=8, head_dim=128, axes=3,
             s0=16, s1=24, s2=24, interleaved=False, norm=True, page=64, span=16384, table="bf16", packed=True),
        # the patches of an image in a vision encoder: height and width, no norm, no cache, 80 dims a head
        dict(name="mrope_vision_t9999", op="mrope", rows=9999, live=9999, heads=16, kv_heads=16, head_dim=80, axes=2,
             s0=20, s1=20, s2=0, interleaved=False, norm=False, page=0, span=1024, table="f32", packed=True),
        # a long prompt of the 8B layer
        dict(name="mrope_prompt_t16384", op="mrope", rows=16384, live=16384, heads=32, kv_heads=8, head_dim=128, axes=3,
             s0=24, s1=20, s2=20, interleaved=True, norm=True, page=128, span=32768, table="bf16", packed=True),
        # a short fresh prompt (latency)
        dict(name="linattn_prompt_t70", op="linattn", seqs=1, rows=70, new_min=70, new_max=70, cont=0, heads=16,
             kv_heads=8, head_dim=128, packed=False, lens_seed=13),
        # short ragged prompts, half of them continued from a stored state
        dict(name="linattn_ragged_6", op="linattn", seqs=6, rows=1024, new_min=17, new_max=260, cont=50, heads=32,
             kv_heads=8, head_dim=128, packed=True, lens_seed=14),
        # one fresh prompt of the 8B layer's heads
        dict(name="linattn_prompt_t4096", op="linattn", seqs=1, rows=4096, new_min=4096, new_max=4096, cont=0, heads=32,
             kv_heads=8, head_dim=128, packed=True, lens_seed=15),
        # two long prompts, a state for every head, one of them continued
        dict(name="linattn_prompts_t32768", op="linattn", seqs=2, rows=32768, new_min=16384, new_max=16384, cont=50,
             heads=32, kv_heads=32, head_dim=128, packed=False, lens_seed=16),
        # one token of a single conversation (latency)
        dict(name="linattn_decode_b1", op="linattn_decode", batch=1, live=1, heads=32, kv_heads=8, head_dim=128),
        # one token of 200 conversations in a batch padded to 256, a state for every head
        dict(name="linattn_decode_b256", op="linattn_decode", batch=256, live=200, heads=32, kv_heads=32, head_dim=128),
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], uniform in its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["plan", "plan", "mrope", "mrope", "mrope", "linattn", "linattn", "linattn", "linattn_decode",
                     "linattn_decode"])
    seed = rng.randrange(1 << 20)
    if op == "plan":
        batch = _log(rng, 1, 1024)
        new_max = _log(rng, 1, max(1, 65536 // batch))
        page = rng.choice([32, 64, 128, 256])
        past_max = _log(rng, 16, 16384)
        return dict(op=op, batch=batch, rows=batch * new_max + rng.choice([0, 0, 7]), new_min=rng.choice([0, 1, new_max]),
                    new_max=new_max, past_min=rng.choice([0, past_max // 2]), past_max=past_max, page=page,
                    max_pages=-(-(past_max + new_max) // page), lens_seed=seed)
    if op == "mrope":
        D = rng.choice([64, 80, 96, 128, 128, 128, 256])
        kv, g = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 2, 4, 8])
        live = _log(rng, 1, max(1, min(20000, (1 << 26) // (kv * (g + 2) * D))))
        axes, half = rng.choice([1, 2, 3, 3]), D // 2
        inter = axes > 1 and rng.random() < 0.5
        if inter:  # every axis takes at most its share of the turns
            s1 = rng.randint(1, half // axes)
            s2 = rng.randint(1, half // axes) if axes == 3 else 0
        else:
            s1 = rng.randint(0, half // 2) if axes > 1 else 0
            s2 = rng.randint(0, half - s1) if axes == 3 else 0
        return dict(op=op, rows=live + rng.choice([0, 0, 5]), live=live, heads=kv * g, kv_heads=kv, head_dim=D, axes=axes,
                    s0=half - s1 - s2, s1=s1, s2=s2, interleaved=inter, norm=rng.random() < 0.7,
                    page=rng.choice([0, 32, 64, 256]), span=_log(rng, 256, 32768), table=rng.choice(["bf16", "bf16", "f32"]),
                    packed=rng.random() < 0.7)
    kv, g, D = rng.choice([1, 2, 4, 8, 16, 32]), rng.choice([1, 1, 2, 4, 8]), rng.choice([64, 128, 128])
    if op == "linattn":
        seqs = rng.choice([1, 1, 2, 3, 8, 24])
        cap = max(1, min(20000, (1 << 26) // (kv * (g + 1) * D)) // seqs)
        new_max = _log(rng, 1, cap)
        new_min = rng.choice([0, new_max // 2, new_max])
        return dict(op=op, seqs=seqs, rows=seqs * new_max + rng.choice([0, 0, 9]), new_min=new_min, new_max=new_max,
                    cont=rng.choice([0, 50, 100]), heads=kv * g, kv_heads=kv, head_dim=D, packed=rng.random() < 0.5,
                    lens_seed=seed)
    batch = _log(rng, 1, max(1, min(512, (1 << 27) // (kv * D * D))))
    return dict(op=op, batch=batch, live=batch if rng.random() < 0.5 else max(1, batch - batch // 5), heads=kv * g,
                kv_heads=kv, head_dim=D)


# ---------------------------------------------------------------- inputs
def _lens(c):
    """(new tokens, cached rows) of every sequence."""
    r = random.Random(c["lens_seed"])
    if c["op"] == "plan":
        return ([r.randint(c["new_min"], c["new_max"]) for _ in range(c["batch"])],
                [r.randint(c["past_min"], c["past_max"]) for _ in range(c["batch"])])
    new = [r.randint(c["new_min"], c["new_max"]) for _ in range(c["seqs"])]
    if not sum(new):
        new[0] = c["new_max"]
    return new, [r.randint(1, 5000) if (i + 1) * c["cont"] // 100 > i * c["cont"] // 100 else 0 for i in range(c["seqs"])]


def _sections(c):
    return tuple(c["s%d" % a] for a in range(c["axes"]))


def _ints(v, dtype=I32):
    return torch.tensor(v, dtype=dtype, device=DEV)


def _qkv(g, rows, heads, kv_heads, D, packed):
    """q, k, v of ``rows`` tokens: views into one projection's output (packed) or tensors of their own."""
    x = torch.randn(rows, heads + 2 * kv_heads, D, generator=g, device=DEV).to(BF)
    q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    return (q, k, v) if packed else (q.contiguous(), k.contiguous(), v.contiguous())


def _package():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import ezops

    return ezops


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    return {"plan": _prepare_plan, "mrope": _prepare_mrope, "linattn": _prepare_linattn,
            "linattn_decode": _prepare_linattn_decode}[c["op"]](c, g)


def _prepare_plan(c, g):
    """A pool in which the cached pages of all sequences lie in random order; the rest of it is free, in another."""
    B, P, M = c["batch"], c["page"], c["max_pages"]
    new, past = _lens(c)
    have = [-(-p // P) for p in past]
    need = [-(-(p + n) // P) for p, n in zip(past, new)]
    used, wanted = sum(have), sum(need) - sum(have)
    pool = used + wanted + 17
    order = torch.randperm(pool, generator=g, device=DEV).to(I32)
    table = torch.full((B, M), -1, dtype=I32, device=DEV)
    live = torch.arange(M, device=DEV)[None, :] < _ints(have, I64)[:, None]
    table[live] = order[:used]
    free = order[used:].contiguous()
    s = dict(c=c, q_lens=_ints(new), past_lens=_ints(past), table=table, free=free, span=_ints([3, free.numel()]), pool=pool)
    if own:
        s["op"] = _package().PagedBatchPlanOp(B, c["rows"], P, M, pool, free.numel(), backend="hip")
        s["out"] = s["op"].alloc(DEV)
    return s


def _grid_positions(c):
    """[axes, rows] positions: text, then an image (one time step, rows by columns), then text; -1 behind the last token."""
    n, span, A = c["live"], c["span"], c["axes"]
    if n <= 64:  # single tokens of many conversations: far and near
        r = random.Random(n)
        base = torch.tensor([r.randrange(span) for _ in range(n)])
        p = torch.stack([base, *[(base * 3 // 4 + 1).clamp(max=span - 1)] * (A - 1)]) if A > 1 else base[None]
    else:
        i, text = torch.arange(n), n // 4
        w = max(1, int(math.isqrt(n // 2)))
        img = n // 2
        k = i - text
        inside = (k >= 0) & (k < img)
        after = text + w + (i - text - img)
        axes = [torch.full_like(i, text), text + k // w, text + k % w]
        pick = axes[-A:] if A < 3 else axes
        p = torch.stack([torch.where(inside, a, torch.where(k < 0, i, after)) for a in pick]) % span
    out = torch.full((A, c["rows"]), -1, dtype=torch.int64)
    out[:, :n] = p
    return out.to(I32).to(DEV)


def _prepare_mrope(c, g):
    T, H, Hkv, D, S = c["rows"], c["heads"], c["kv_heads"], c["head_dim"], c["span"]
    q, k, v = _qkv(g, T, H, Hkv, D, c["packed"])
    inv = THETA ** (-torch.arange(0, D, 2, dtype=F64, device=DEV) / D)
    ang = torch.arange(S, dtype=F64, device=DEV)[:, None] * inv
    dt = BF if c["table"] == "bf16" else F32
    s = dict(c=c, q=q, k=k, v=v, cos=ang.cos().repeat(1, 2).to(dt), sin=ang.sin().repeat(1, 2).to(dt),
             positions=_grid_positions(c), qw=None, kw=None, K=None, V=None, slots=None,
             q_out=torch.zeros(T, H, D, dtype=BF, device=DEV), k_out=None)
    if c["norm"]:
        s["qw"] = (1 + 0.1 * torch.randn(D, generator=g, device=DEV)).to(BF)
        s["kw"] = (1 + 0.1 * torch.randn(D, generator=g, device=DEV)).to(BF)
    pages = 0
    if c["page"]:
        P = c["page"]
        pages = -(-T // P) + 3
        s["K"] = torch.randn(pages, Hkv, P, D, generator=g, device=DEV).to(BF)
        s["V"] = torch.randn(pages, Hkv, P, D, generator=g, device=DEV).to(BF)
        order = torch.randperm(pages, generator=g, device=DEV)
        i = torch.arange(T, device=DEV)
        slots = order[i // P] * P + i % P
        s["slots"] = torch.where(i < c["live"], slots, -1)
    else:
        s["k_out"] = torch.zeros(T, Hkv, D, dtype=BF, device=DEV)
    if own:
        s["op"] = _package().QkNormMropeOp(T, H, Hkv, D, S, _sections(c), backend="hip", interleaved=c["interleaved"],
                                           norm=c["norm"], page_size=c["page"] or None, num_pages=pages or None)
    return s


def _decay(c):
    """ln of the decay of every head: from about exp(-1/256) a token up to exp(-1/2), slower heads last."""
    n = c["kv_heads"]
    return -torch.exp2(-1 - 7 * torch.arange(n, dtype=F32, device=DEV) / max(1, n - 1))


def _prepare_linattn(c, g):
    B, T, H, Hkv, D = c["seqs"], c["rows"], c["heads"], c["kv_heads"], c["head_dim"]
    new, past = _lens(c)
    q, k, v = _qkv(g, T, H, Hkv, D, c["packed"])
    for x in (q, k):  # the usual feature map of such layers
        x.copy_(torch.nn.functional.silu(x.float()).to(BF))
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    slots = torch.randperm(B + 2, generator=g, device=DEV)[:B].to(I32)
    s = dict(c=c, q=q, k=k, v=v, g=_decay(c), cu=_ints(cu), past=_ints(past), slots=slots, longest=max(new),
             state=torch.randn(B + 2, Hkv, D, D, generator=g, device=DEV), out=torch.zeros(T, H, D, dtype=BF, device=DEV))
    if own:
        s["op"] = _package().LinearAttnPrefillOp(B, T, H, Hkv, D, backend="hip", num_slots=B + 2)
    return s


def _prepare_linattn_decode(c, g):
    B, H, Hkv, D = c["batch"], c["heads"], c["kv_heads"], c["head_dim"]
    q, k, v = _qkv(g, B, H, Hkv, D, True)
    for x in (q, k):
        x.copy_(torch.nn.functional.silu(x.float()).to(BF))
    n = c["live"] + 3
    slots = torch.full((B,), -1, dtype=I32, device=DEV)
    slots[:c["live"]] = torch.randperm(n, generator=g, device=DEV)[:c["live"]].to(I32)
    s = dict(c=c, q=q, k=k, v=v, g=_decay(c), slots=slots, state=torch.randn(n, Hkv, D, D, generator=g, device=DEV),
             out=torch.zeros(B, H, D, dtype=BF, device=DEV))
    if own:
        s["op"] = _package().LinearAttnDecodeOp(B, H, Hkv, D, n, backend="hip")
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    return {"plan": _run_plan, "mrope": _run_mrope, "linattn": _run_linattn,
            "linattn_decode": _run_linattn_decode}[s["c"]["op"]](s)


def _run_plan(s):
    if own:
        p = s["op"](s["q_lens"], s["past_lens"], s["table"], s["free"], s["span"], out=s["out"])
        return [s["table"], *p]
    c, table, free = s["c"], s["table"], s["free"]
    P, T, M = c["page"], c["rows"], c["max_pages"]
    new, past = s["q_lens"].long(), s["past_lens"].long()
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)]).clamp(max=T)
    kv = (past + cu.diff()).clamp(max=M * P)
    have, need = (past + P - 1) // P, (kv + P - 1) // P
    taken = (need - have).cumsum(0)
    first = taken - (need - have)
    head, tail = s["span"][0].long(), s["span"][1].long()
    j = torch.arange(M, device=DEV)
    at = head + first[:, None] + j - have[:, None]
    got = torch.where(at < tail, free[at.clamp(0, free.numel() - 1)], -1)
    table.copy_(torch.where((j >= have[:, None]) & (j < need[:, None]), got, table))
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(cu[1:], t, right=True).clamp(max=c["batch"] - 1)
    pos = past[b] + t - cu[b]
    page = table[b, (pos // P).clamp(max=M - 1)].long()
    live = t < cu[-1]
    slot = torch.where(live & (page >= 0) & (pos < M * P), page * P + pos % P, -1)
    wanted = taken[-1]
    span = torch.stack([head + torch.minimum(wanted, tail - head), tail, wanted])
    return [table, cu.to(I32), kv.to(I32), torch.where(live, pos, -1).to(I32), slot, span.to(I32)]


def _axis_of_pair(c):
    i, A, sec = torch.arange(c["head_dim"] // 2, device=DEV), c["axes"], _sections(c)
    if c["interleaved"]:
        a = i % A
        return torch.where(i < A * _ints(sec, I64)[a], a, 0)
    return torch.searchsorted(_ints(sec, I64).cumsum(0), i, right=True)


def _run_mrope(s):
    c = s["c"]
    if own:
        s["op"](s["q"], s["k"], s["v"], s["qw"], s["kw"], s["cos"], s["sin"], s["positions"], s["K"], s["V"], s["slots"],
                q_out=s["q_out"], k_out=s["k_out"])
    else:
        half = c["head_dim"] // 2
        pos = s["positions"].long()
        live = (pos >= 0).all(0)
        pair = torch.arange(half, device=DEV)
        rows = pos.clamp(min=0)[_axis_of_pair(c)].t()
        cos, sin = s["cos"].float()[rows, pair][:, None], s["sin"].float()[rows, pair][:, None]

        def turned(x, w):
            x = x.float()
            if c["norm"]:
                x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
            a, b = x[..., :half], x[..., half:]
            return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(BF)

        s["q_out"].copy_(torch.where(live[:, None, None], turned(s["q"], s["qw"]), s["q_out"]))
        k = turned(s["k"], s["kw"])
        if c["page"]:
            slots = s["slots"][live]
            page, row = slots // c["page"], slots % c["page"]
            s["K"][page, :, row] = k[live]
            s["V"][page, :, row] = s["v"][live]
        else:
            s["k_out"].copy_(torch.where(live[:, None, None], k, s["k_out"]))
    return [s["q_out"], s["K"], s["V"]] if c["page"] else [s["q_out"], s["k_out"]]


def _run_linattn(s):
    c = s["c"]
    if own:
        s["op"](s["q"], s["k"], s["v"], s["g"], s["cu"], s["state"], s["slots"], s["past"], max_q_len=s["longest"],
                out=s["out"])
        return [s["out"], s["state"]]
    B, H, Hkv, D, C = c["seqs"], c["heads"], c["kv_heads"], c["head_dim"], 64
    G, n = H // Hkv, -(-s["longest"] // C)
    cu, g = s["cu"].long(), s["g"].double()
    new = cu.diff()
    i = torch.arange(n * C, device=DEV)
    live = i < new[:, None]
    row = torch.where(live, cu[:-1, None] + i, 0)

    def cut(x):  # [B, n C, h, D] -> [B, h, n, C, D], zeros behind the last token
        x = torch.where(live[:, :, None, None], x[row].float(), 0.0)
        return x.reshape(B, n, C, -1, D).permute(0, 3, 1, 2, 4).contiguous()

    q, k, v = cut(s["q"]).reshape(B, Hkv, G, n, C, D), cut(s["k"]), cut(s["v"])
    slots = s["slots"].long()
    start = torch.where((s["past"] > 0)[:, None, None, None], s["state"][slots], 0.0)
    r = torch.arange(C, device=DEV)
    back = (r[:, None] - r).clamp(min=0)
    decay = torch.where(r[:, None] >= r, torch.exp(g[:, None, None] * back), 0.0).float()
    out = (q @ k[:, :, None].transpose(-1, -2).contiguous() * decay[:, None, None]) @ v[:, :, None]
    # the state at the start of every chunk: what the chunks before it add, and the first state
    kw = k * torch.exp(g[:, None] * (C - 1 - r)).float()[:, None, :, None]
    adds = kw.transpose(-1, -2).contiguous() @ v
    m = torch.arange(n, device=DEV)
    gap = (m[:, None] - 1 - m).clamp(min=0)
    carry = torch.where(m[:, None] > m, torch.exp(g[:, None, None] * (C * gap)), 0.0).float()
    states = (carry @ adds.reshape(B, Hkv, n, D * D)).reshape(B, Hkv, n, D, D)
    states = states + torch.exp(g[:, None] * (C * m)).float()[:, :, None, None] * start[:, :, None]
    out = out + torch.exp(g[:, None] * (r + 1)).float()[:, None, None, :, None] * (q @ states[:, :, None])
    out = (out * D ** -0.5).reshape(B, H, n * C, D).transpose(1, 2).to(BF)
    s["out"][row[live]] = out[live]
    # the state behind the last token
    ago = (new[:, None] - 1 - i).clamp(min=0)
    w = torch.where(live[:, None], torch.exp(g[:, None] * ago[:, None]), 0.0).float()
    kw = k.reshape(B, Hkv, n * C, D) * w[..., None]
    last = kw.transpose(-1, -2).contiguous() @ v.reshape(B, Hkv, n * C, D)
    last = last + torch.exp(g * new[:, None]).float()[:, :, None, None] * start
    s["state"][slots] = torch.where((new > 0)[:, None, None, None], last, s["state"][slots])
    return [s["out"], s["state"]]


def _run_linattn_decode(s):
    c = s["c"]
    if own:
        s["op"](s["q"], s["k"], s["v"], s["g"], s["state"], s["slots"], out=s["out"])
        return [s["out"], s["state"]]
    B, Hkv, D = c["batch"], c["kv_heads"], c["head_dim"]
    live = s["slots"] >= 0
    slots = s["slots"][live].long()
    q, k, v = s["q"][live].float(), s["k"][live].float(), s["v"][live].float()
    state = torch.exp(s["g"])[:, None, None] * s["state"][slots] + k[..., :, None] * v[..., None, :]
    s["state"][slots] = state
    out = q.reshape(-1, Hkv, c["heads"] // Hkv, D) @ state * D ** -0.5
    s["out"][live] = out.reshape(-1, c["heads"], D).to(BF)
    return [s["out"], s["state"]]


# ---------------------------------------------------------------- its work
def work(case):
    c = case
    if c["op"] == "plan":
        new, past = _lens(c)
        P, T = c["page"], sum(new)
        fresh = sum(-(-(p + n) // P) + -p // P for p, n in zip(past, new))
        read = 8 * c["batch"] + 4 * fresh + 4 * sum(p % P > 0 and n > 0 for p, n in zip(past, new)) + 8
        return {"bytes": read + 4 * fresh + 4 * (2 * c["batch"] + 1) + 12 * c["rows"] + 12, "flops": 0}
    H, Hkv, D = c["heads"], c["kv_heads"], c["head_dim"]
    if c["op"] == "mrope":
        heads = 2 * H + (4 if c["page"] else 2) * Hkv  # q and k in and out, v into the cache
        rows = min(c["span"], c["live"])
        extra = c["live"] * (4 * c["axes"] + (8 if c["page"] else 0)) + rows * D * (2 if c["table"] == "bf16" else 4)
        return {"bytes": 2 * c["live"] * heads * D + extra, "flops": c["live"] * (H + Hkv) * D * (7 if c["norm"] else 3)}
    if c["op"] == "linattn_decode":
        return {"bytes": c["live"] * (2 * Hkv * D * D * 4 + (2 * H + 2 * Hkv) * D * 2),
                "flops": c["live"] * (3 * Hkv + 2 * H) * D * D}
    new, past = _lens(c)
    T = sum(new)
    states = sum((n > 0) + (n > 0 and p > 0) for n, p in zip(new, past))
    # the recurrence: a state update a kv head, a product with the state a query head
    return {"bytes": 2 * T * (2 * H + 2 * Hkv) * D + 4 * states * Hkv * D * D, "flops": T * (3 * Hkv + 2 * H) * D * D}


# ---------------------------------------------------------------- in 64 bits
def exact(case, seed):
    c = dict(case)
    s = prepare(c, seed)
    return {"plan": _exact_plan, "mrope": _exact_mrope, "linattn": _exact_linattn,
            "linattn_decode": _exact_linattn_decode}[c["op"]](s)


def _exact_plan(s):
    """Request by request, as an allocator on the host does it."""
    c = s["c"]
    P, T = c["page"], c["rows"]
    new, past = _lens(c)
    table, free = s["table"].tolist(), s["free"].tolist()
    head, tail = s["span"].tolist()
    cu, kv, pos, slots, wanted = [0], [], [], [], 0
    for b, (n, p) in enumerate(zip(new, past)):
        for t in range(p, p + n):
            if t % P == 0:
                table[b][t // P] = free[head + wanted]
                wanted += 1
            pos.append(t)
            slots.append(table[b][t // P] * P + t % P)
        cu.append(cu[-1] + n)
        kv.append(p + n)
    pad = [-1] * (T - len(pos))
    return [_ints(table), _ints(cu), _ints(kv), _ints(pos + pad), _ints(slots + pad, I64), _ints([head + wanted, tail, wanted])]


def _exact_mrope(s):
    """Pairs as complex numbers, turned by cos + i sin."""
    c = s["c"]
    D, n, A, sec = c["head_dim"], c["live"], c["axes"], _sections(c)
    half = D // 2
    axis = []
    for i in range(half):
        if c["interleaved"]:
            axis.append(i % A if i < A * sec[i % A] else 0)
        else:
            axis.append(next(a for a in range(A) if i < sum(sec[:a + 1])))
    turn = torch.empty(n, half, dtype=torch.complex128, device=DEV)
    for i, a in enumerate(axis):
        p = s["positions"][a, :n].long()
        turn[:, i] = torch.complex(s["cos"][p, i].double(), s["sin"][p, i].double())

    def turned(x, w):
        x = x[:n].double()
        if c["norm"]:
            x = x / (x.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
        z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn[:, None]
        return torch.cat([z.real, z.imag], -1)

    q_out = s["q_out"].double()
    q_out[:n] = turned(s["q"], s["qw"])
    k = turned(s["k"], s["kw"])
    if not c["page"]:
        k_out = s["k_out"].double()
        k_out[:n] = k
        return [q_out, k_out]
    P, got = c["page"], []
    for pool, x in ((s["K"], k), (s["V"], s["v"][:n].double())):
        flat = pool.double().transpose(1, 2).reshape(-1, c["kv_heads"], D)  # [slot, head, dim]
        flat[s["slots"][:n]] = x
        got.append(flat.reshape(-1, P, c["kv_heads"], D).transpose(1, 2))
    return [q_out, *got]


def _exact_linattn(s):
    """Sequence by sequence, 100 tokens at a time from the state before them."""
    c = s["c"]
    H, Hkv, D = c["heads"], c["kv_heads"], c["head_dim"]
    G = H // Hkv
    out, pool = s["out"].double(), s["state"].double()
    cu, past, slots = s["cu"].tolist(), s["past"].tolist(), s["slots"].tolist()
    lam = torch.exp(s["g"].double())
    for b in range(c["seqs"]):
        if cu[b + 1] == cu[b]:
            continue
        S = pool[slots[b]].clone() if past[b] > 0 else torch.zeros(Hkv, D, D, dtype=F64, device=DEV)
        for t in range(cu[b], cu[b + 1], 100):
            e = min(t + 100, cu[b + 1])
            n = e - t
            i = torch.arange(n, device=DEV)
            q, k, v = (x[t:e].double().transpose(0, 1).contiguous() for x in (s["q"], s["k"], s["v"]))
            q = q.reshape(Hkv, G * n, D)
            w = lam[:, None, None] ** (i[:, None] - i).clamp(min=0) * (i[:, None] >= i)
            a = (q @ k.transpose(1, 2).contiguous()).reshape(Hkv, G, n, n) * w[:, None]
            o = (a @ v[:, None]).reshape(Hkv, G, n, D)
            o += lam[:, None, None, None] ** (i + 1)[:, None] * (q @ S).reshape(Hkv, G, n, D)
            out[t:e] = (o / math.sqrt(D)).reshape(H, n, D).transpose(0, 1)
            S = lam[:, None, None] ** n * S + (k * lam[:, None, None] ** (n - 1 - i)[:, None]).transpose(1, 2).contiguous() @ v
        pool[slots[b]] = S
    return [out, pool]


def _exact_linattn_decode(s):
    """Row by row."""
    c = s["c"]
    G = c["heads"] // c["kv_heads"]
    out, pool = s["out"].double(), s["state"].double()
    lam = torch.exp(s["g"].double())[:, None, None]
    for b, at in enumerate(s["slots"].tolist()):
        if at < 0:
            continue
        pool[at] = pool[at] * lam + s["k"][b].double()[:, :, None] * s["v"][b].double()[:, None, :]
        q = s["q"][b].double().reshape(c["kv_heads"], G, 1, c["head_dim"])
        out[b] = (q @ pool[at][:, None]).reshape(c["heads"], c["head_dim"]) / math.sqrt(c["head_dim"])
    return [out, pool]
