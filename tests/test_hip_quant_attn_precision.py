"""Attention over the 8-bit KV cache on the GPU: weights of 16 significant bits in the single-token op, and exponents from one
end to the other beside each other, against ``oracle.kv8`` in 64 bits.

With A = sum_j w_j |v_j| and S = the largest scale * sum_d |q_d k_jd| that a query meets: products of q and codes are exact in
fp32, a score sums D of them (2^-23 each, the matrix cores may truncate) and is scaled and shifted (the factor, the product
and the sum, 2^-24 of at most 2 S log2 e + 60 + 60 log2 units each, the exponents of v being within 60), and raised (2^-22):
a weight is off by a relative

    d = (D + 8) 2^-23 S + 2^-17 + 2^-22

and its sum by another d, L terms of it by 2^-23 each, L of the weighted rows twice that (two products a row).

  single tokens   a weight in two bf16 parts is off by 2^-8 of 2^-8:  2^-8 |o| + (2^-16 + 2 d + (3 L + 64) 2^-23) A
  prompts         a weight is rounded to bf16, and the sum takes the rounded one:
                                                              2^-8 |o| + (2 2^-8 + 2 d + (3 L + 64) 2^-23) A

(2^-8 |o| the rounding of the result).
"""

import numpy as np
import pytest
import torch

from ezops import QuantPagedAttnDecodeOp, QuantPrefillAttnOp
from oracle import kv8
from test_hip_quant_attn import KINDS, Cache, n64

DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)
gpu = pytest.mark.gpu


def tolerance(want, mag, most, D, L, weights):
    d = (D + 8) * 2.0 ** -23 * most[..., None] + 2.0 ** -17 + 2.0 ** -22
    return 2.0 ** -8 * np.abs(want) + (weights + 2 * d + (3 * L + 64) * 2.0 ** -23) * mag + 1e-30


TWO_PARTS, ONE_PART = 2.0 ** -16, 2 * 2.0 ** -8


def bf16(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(torch.bfloat16).double().numpy()


def one_part(q, k, v, scale):
    """One token's result with weights of one bf16 part, and everything else exact but the result's rounding."""
    H, G = q.shape[0], q.shape[0] // k.shape[1]
    out = np.empty(q.shape)
    for h in range(H):
        s = k[:, h // G] @ q[h] * scale
        w = np.exp(s - s.max())
        out[h] = bf16(w) @ v[:, h // G] / w.sum()
    return bf16(out)


FEW = [2, 3, 5, 9, 17, 33]  # rows, where roundings of weights do not average out


def test_the_tolerance_sees_weights_of_one_part():
    """Shown on the CPU: results with half the weight's bits are outside at every one of these lengths."""
    g = np.random.RandomState(31)
    for D in (64, 128):
        for L in FEW:
            q, k, v = bf16(g.randn(8, D) * 0.5), g.randn(L, 2, D), bf16(g.randn(L, 2, D))
            want, mag, most = kv8.attend(q[None], k, v, L - 1, D ** -0.5)
            tol = tolerance(want, mag, most, D, L, TWO_PARTS)[0]
            assert (np.abs(one_part(q, k, v, D ** -0.5) - want[0]) > tol).any(), (D, L)
            assert (np.abs(bf16(want[0]) - want[0]) <= tol).all()


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("G,Hkv,D", [(4, 2, 128), (1, 3, 64), (16, 1, 128), (8, 2, 64), (2, 2, 128)])
def test_decode_weights(kind, G, Hkv, D):
    """Few rows, and some hundreds whose chunks are joined."""
    for lens in (FEW, [300, 513, 40]):
        c = Cache(kind, lens, Hkv, D, 64, 32, 40 + G, spread=0.0)
        q = c.q(len(lens), G * Hkv, 0.5)
        out = n64(QuantPagedAttnDecodeOp(len(lens), G * Hkv, Hkv, D, 64, c.M, c.pages, **c.how)(
            q, *c.pools, c.t, torch.tensor(lens, **I32)))
        for b, n in enumerate(lens):
            want, mag, most = c.want(q[b:b + 1], b, n - 1, D ** -0.5)
            tol = tolerance(want, mag, most, D, n, TWO_PARTS)[0]
            assert (np.abs(out[b] - want[0]) <= tol).all(), (b, n, float((np.abs(out[b] - want[0]) / tol).max()))


CHUNK = 20
SHORT, LONG = [20, 21, 63, 77, 128], [20, 47, 129, 700, 1500]  # no joins; joins of up to a dozen parts


def extreme(kind, lens, D, block, k_exps, v_exps, seed, spread=0.0):
    """A cache whose blocks of rows, one after the other, take these exponents; None leaves one as it was written."""
    c = Cache(kind, lens, 2, D, 64, block, seed, spread=spread)
    for s, exps in ((2, k_exps), (3, v_exps)):
        for b, n in enumerate(lens):
            for i, r in enumerate(range(0, n, block)):
                e = exps[i % len(exps)]
                if e is not None:
                    c.np[s][int(c.table[b, r // 64]), :, r % 64 // block] = e
        c.pools[s].copy_(torch.from_numpy(c.np[s]))
    c.held = [[kv8.rows(c.np[x], c.np[s], c.table[b].numpy(), n, block, kind) for x, s in ((0, 2), (1, 3))]
              for b, n in enumerate(lens)]
    return c


def both(c, scale, size=1.0, bound=0):
    B, D, H = len(c.lens), c.D, 8
    how = dict(c.how, scale=scale)
    q = c.q(CHUNK * B, H, size)
    last = q[CHUNK - 1::CHUNK].contiguous()
    one = QuantPagedAttnDecodeOp(B, H, 2, D, 64, c.M, c.pages, **how)(last, *c.pools, c.t, torch.tensor(c.lens, **I32), bound)
    many = QuantPrefillAttnOp(B, CHUNK * B, H, 2, D, 64, c.M, c.pages, **how)(
        q, *c.pools, c.t, torch.arange(0, CHUNK * B + 1, CHUNK, **I32), torch.tensor([n - CHUNK for n in c.lens], **I32),
        max_kv_len=bound)
    for b, n in enumerate(c.lens):
        want, mag, most = kv8.attend(n64(q[CHUNK * b:CHUNK * (b + 1)]), *c.held[b], n - CHUNK, scale)
        dt, pt = tolerance(want, mag, most, D, n, TWO_PARTS)[-1], tolerance(want, mag, most, D, n, ONE_PART)
        for what, got, w, t in (("single", n64(one[b]), want[-1], dt), ("chunk", n64(many[CHUNK * b:CHUNK * (b + 1)]), want, pt)):
            assert np.isfinite(got).all(), (what, b, n)
            assert (np.abs(got - w) <= t).all(), (what, b, n, float((np.abs(got - w) / t).max()))


V_EXPS = {"least beside ordinary": [67, None], "far apart": [None, 127 + 55, 127 - 55], "both ends": [67, 187, None, 120],
          "no write makes": [0, 254, None, 66, 188], "all least": [67], "all largest": [187]}


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D,block", [(64, 16), (128, 16), (128, 64)])
@pytest.mark.parametrize("v_exps", V_EXPS)
def test_exponents_of_v(kind, D, block, v_exps):
    for lens in (SHORT, LONG):
        both(extreme(kind, lens, D, block, [None], V_EXPS[v_exps], 51), D ** -0.5, 0.5, max(lens))


# Exponents of K, the factor on the scores and the size of q: scores of ordinary size where the exponent is largest.
K_EXPS = {"least beside ordinary": ([67, None], 2.0 ** -4, 0.5), "far apart": ([None, 127 + 48, 127 - 55], 2.0 ** -58, 0.5),
          "both ends": ([67, 187, None, 120], 2.0 ** -70, 0.5), "no write makes": ([0, 254, None, 66, 188], 2.0 ** -70, 0.5),
          "all least": ([67], 2.0 ** 50, 0.5), "all largest": ([187], 2.0 ** -70, 0.5)}


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D,block", [(64, 32), (128, 16)])
@pytest.mark.parametrize("k_exps", K_EXPS)
def test_exponents_of_k(kind, D, block, k_exps):
    exps, scale, size = K_EXPS[k_exps]
    for lens in (SHORT, LONG):
        both(extreme(kind, lens, D, block, exps, V_EXPS["both ends"], 52), scale, size, max(lens))


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_zeros_beside_ordinary_rows(kind):
    """Blocks as a write of zeros leaves them, in K and V, at the front, in the middle and last."""
    for lens in (SHORT, LONG):
        c = extreme(kind, lens, 128, 16, [67, None, None], [None, 67, None], 53)
        for x, s in ((0, 2), (1, 3)):
            codes, e = c.np[x].reshape(c.pages, 2, 4, 16, 128), c.np[s]
            codes[e == 67] = 0
            c.pools[x].view(torch.uint8).copy_(torch.from_numpy(c.np[x]))
        c.held = [[kv8.rows(c.np[x], c.np[s], c.table[b].numpy(), n, 16, kind) for x, s in ((0, 2), (1, 3))]
                  for b, n in enumerate(lens)]
        both(c, 128 ** -0.5, 0.5, max(lens))
