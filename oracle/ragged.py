"""Plain 64-bit restatements of the ragged-batch ops (numpy, from their definitions; no reference counterpart)."""

from __future__ import annotations

import numpy as np


def batch_plan(q_lens, past_lens, block_table, free_pages, free_span, T, P, num_pages):
    """Request by request.  -> (block_table, cu_seqlens, kv_lens, positions, slots, span)."""
    table = np.array(block_table, dtype=np.int64)
    B, M = table.shape
    head, tail = int(free_span[0]), int(free_span[1])
    last = min(tail, len(free_pages))
    cu, kv, pos, slots, needed = [0], [], np.full(T, -1), np.full(T, -1), 0
    for b in range(B):
        past = min(max(int(past_lens[b]) if past_lens is not None else 0, 0), M * P)
        n = min(max(int(q_lens[b]), 0), T - cu[-1])
        for i in range(n):
            p, t = past + i, cu[-1] + i
            pos[t] = p
            if p >= M * P:
                continue
            if p % P == 0:  # a page begins
                page = int(free_pages[head + needed]) if 0 <= head and head + needed < last else -1
                table[b, p // P] = page if 0 <= page < num_pages else -1
                needed += 1
            page = table[b, p // P]
            if 0 <= page < num_pages:
                slots[t] = page * P + p % P
        cu.append(cu[-1] + n)
        kv.append(min(past + n, M * P))
    avail = max(last - head, 0) if head >= 0 else 0
    return table, np.array(cu), np.array(kv), pos, slots, np.array([head + min(needed, avail), tail, needed])


def pair_axes(half, sections, interleaved):
    A, out = len(sections), []
    for i in range(half):
        if interleaved:
            a = i % A
            out.append(a if i // A < sections[a] else 0)
        else:
            a, left = 0, i
            while left >= sections[a]:
                left -= sections[a]
                a += 1
            out.append(a)
    return out


def qk_norm_mrope(x, w, cos, sin, positions, sections, interleaved, norm, eps=1e-6):
    """x [T, heads, D] -> rotated heads in 64 bits, as complex numbers turned by cos + i sin; rows with a position
    outside the table are NaN."""
    x = np.asarray(x, dtype=np.float64)
    T, _, D = x.shape
    half = D // 2
    if norm:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps)
        if w is not None:
            x = x * np.asarray(w, dtype=np.float64)
    z = x[..., :half] + 1j * x[..., half:]
    out = np.full_like(x, np.nan)
    axes = pair_axes(half, sections, interleaved)
    for t in range(T):
        p = [int(v) for v in positions[:, t]]
        if any(v < 0 or v >= cos.shape[0] for v in p):
            continue
        turn = np.array([cos[p[a], i] + 1j * sin[p[a], i] for i, a in enumerate(axes)])
        y = z[t] * turn
        out[t] = np.concatenate([y.real, y.imag], -1)
    return out


def linear_attn(q, k, v, lam, S, scale):
    """The recurrence of one sequence: q [n, H, D], k / v [n, Hkv, D], lam [Hkv], S [Hkv, D, D] -> (out [n, H, D], S)."""
    q, k, v, S = (np.asarray(x, dtype=np.float64) for x in (q, k, v, S))
    n, H, D = q.shape
    Hkv = k.shape[1]
    out = np.empty((n, H, D))
    for t in range(n):
        S = np.asarray(lam, dtype=np.float64)[:, None, None] * S + k[t][:, :, None] * v[t][:, None, :]
        out[t] = scale * (q[t].reshape(Hkv, H // Hkv, D) @ S).reshape(H, D)
    return out, S
