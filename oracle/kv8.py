"""Plain 64-bit restatement of the 8-bit KV cache and the attention over it (numpy, from their definitions; no
reference counterpart).  Codes are bytes, exponents whole numbers; a row is ``value(code) * 2^(e - 127)``."""

from __future__ import annotations

import math

import numpy as np

TOP = {"int8": 127.0, "e4m3": 448.0}


def _e4m3_values():
    """Value of every byte: sign, 4 exponent bits (bias 7), 3 fraction bits; 0x7f and 0xff are NaN."""
    out = np.empty(256)
    for c in range(256):
        e, f = (c >> 3) & 15, c & 7
        v = math.nan if c & 127 == 127 else (f / 8 * 2.0 ** -6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7))
        out[c] = -v if c & 128 else v
    return out


VALUES = {"int8": np.arange(256, dtype=np.uint8).view(np.int8).astype(np.float64), "e4m3": _e4m3_values()}


def need(amax, kind):
    """Least exponent whose scale holds amax, by trying."""
    e = 67
    while e < 187 and amax > TOP[kind] * 2.0 ** (e - 127):
        e += 1
    return e


def encode(y, kind):
    """Bytes of values in units of their scale: the nearest code, ties to the even one, saturating; not finite: NaN
    (e4m3) or 0 (int8)."""
    y = np.asarray(y, dtype=np.float64)
    if kind == "int8":
        q = np.rint(np.clip(np.where(np.isfinite(y), y, 0), -127, 127))
        return q.astype(np.int8).view(np.uint8)
    pos = VALUES["e4m3"][:127]
    a = np.minimum(np.abs(np.where(np.isfinite(y), y, 0)), 448.0)
    hi = np.minimum(np.searchsorted(pos, a), 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - pos[lo], pos[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi).astype(np.uint8)
    code = code | (np.signbit(y).astype(np.uint8) << 7)
    return np.where(np.isfinite(y), code, 127).astype(np.uint8)


def clamped(e):
    """An exponent as it is read: 255, or within [67, 187]."""
    return 255 if e == 255 else min(max(int(e), 67), 187)


def decode(codes, e, kind):
    return VALUES[kind][codes] * (math.nan if e == 255 else 2.0 ** (clamped(e) - 127))


def write(x, cache, scale, slots, block, kind):
    """x [T, Hkv, D] into cache [pages, Hkv, P, D] (bytes) and scale [pages, Hkv, P / block], in place, run by run."""
    pages, Hkv, P, D = cache.shape
    t, T = 0, len(slots)
    while t < T:
        n, s = 1, int(slots[t])
        if 0 <= s < pages * P:
            page, row = divmod(s, P)
            off = row % block
            while off + n < block and t + n < T and slots[t + n] == s + n:
                n += 1
            for h in range(Hkv):
                new = np.asarray(x[t:t + n, h], dtype=np.float64)
                fine = np.isfinite(new)
                e = need(np.abs(np.where(fine, new, 0)).max(), kind)
                if kind == "int8" and not fine.all():
                    e = 255
                old = clamped(scale[page, h, row // block]) if off else 0
                e = max(e, old)
                first = row - off
                if off and e > old:
                    held = VALUES[kind][cache[page, h, first:row]]
                    f = 0.0 if e == 255 else 2.0 ** (old - e)
                    cache[page, h, first:row] = encode(held * f, kind)
                y = new * (0.0 if e == 255 else 2.0 ** (127 - e)) if e != 255 or kind == "e4m3" else np.zeros_like(new)
                cache[page, h, row:row + n] = encode(y, kind)
                scale[page, h, row // block] = e
        t += n


def rows(cache, scale, table, L, block, kind):
    """The first L rows of a sequence: [L, Hkv, D]."""
    P = cache.shape[2]
    out = np.empty((L, cache.shape[1], cache.shape[3]))
    for r in range(L):
        page, row = int(table[r // P]), r % P
        for h in range(cache.shape[1]):
            out[r, h] = decode(cache[page, h, row], scale[page, h, row // block], kind)
    return out


def attend(q, k, v, past, scale):
    """q [n, H, D] of one sequence, k / v [past + n, Hkv, D]; query i sees rows 0 .. past + i.
    -> (out, sum of |weights * v|, the largest sum of |q k| scale a query meets) [n, H, D], [n, H, D], [n, H]."""
    n, H, D = q.shape
    G = H // k.shape[1]
    out, mag, most = np.zeros((n, H, D)), np.zeros((n, H, D)), np.zeros((n, H))
    for h in range(H):
        kh, vh = k[:, h // G], v[:, h // G]
        s = q[:, h] @ kh.T * scale
        a = np.abs(q[:, h]) @ np.abs(kh).T * scale
        seen = np.arange(len(k))[None, :] <= past + np.arange(n)[:, None]
        s = np.where(seen, s, -np.inf)
        w = np.exp(s - s.max(1, keepdims=True))
        w /= w.sum(1, keepdims=True)
        out[:, h], mag[:, h], most[:, h] = w @ vh, w @ np.abs(vh), np.where(seen, a, 0).max(1)
    return out, mag, most
