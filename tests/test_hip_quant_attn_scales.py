"""Attention over the 8-bit KV cache at the ends of the scales: factors on the scores that fp32 holds only as a subnormal
number, or not at all, beside masked rows, whose weight is 0 whatever the factor is.

Against ``oracle.kv8`` in 64 bits, within ``test_hip_quant_attn.tolerance``.  What that does not count: the factor
c = scale log2(e) 2^(e - 127) is off by less than 2^-148 where it is below 2^-126, and a sum q . codes stays below 2^128, so
a score is off by 2^-20 in the exponent of its weight at most, which is added here as 2 * 2^-20 A.
"""

import ctypes

import numpy as np
import pytest
import torch

from ezops import QuantPagedAttnDecodeOp, QuantPrefillAttnOp
from oracle import kv8
from test_hip_quant_attn import KINDS, Cache, n64, tolerance

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)


def both(c, H, scale, size):
    """Single tokens and chunks of 40 rows against the cache's lengths."""
    scale = ctypes.c_float(scale).value
    lens, B = c.lens, len(c.lens)
    how = dict(c.how, scale=scale)
    q = c.q(40 * B, H, size)
    last = q[39::40].contiguous()
    one = QuantPagedAttnDecodeOp(B, H, c.Hkv, c.D, c.P, c.M, c.pages, **how)(last, *c.pools, c.t, torch.tensor(lens, **I32))
    many = QuantPrefillAttnOp(B, 40 * B, H, c.Hkv, c.D, c.P, c.M, c.pages, **how)(
        q, *c.pools, c.t, torch.arange(0, 40 * B + 1, 40, **I32), torch.tensor([n - 40 for n in lens], **I32))
    for b, n in enumerate(lens):
        x = q[40 * b:40 * b + 40]
        want, mag, most = kv8.attend(n64(x), *c.held[b], n - 40, scale)
        tol = tolerance(want, mag, most, c.D) + 2 * 2.0 ** -20 * mag
        for what, got, w, t in (("decode", one[b], want[-1], tol[-1]), ("prefill", many[40 * b:40 * b + 40], want, tol)):
            got = n64(got)
            assert np.isfinite(got).all(), (what, b, n)
            assert (np.abs(got - w) <= t).all(), (what, b, n, float((np.abs(got - w) / t).max()))


LENS = [40, 41, 63, 77, 129, 1500]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scale,size", [(1e-30, 1.0), (1e-38, 1.0), (1e-40, 1.0), (1.4e-45, 1.0), (1e-40, 1e34), (2.0 ** -120, 2.0 ** 110)])
def test_tiny_scales(kind, D, scale, size):
    both(Cache(kind, LENS, 2, D, 64, 32, 21), 8, scale, size)


def zero_keys(c, first, last):
    """Rows [first, last) of K of every sequence, whole blocks, as a write of zeros leaves them."""
    for b, n in enumerate(c.lens):
        for r in range(first, min(last, n), c.block):
            page, row = int(c.table[b, r // c.P]), r % c.P
            c.np[0][page, :, row:row + c.block] = 0
            c.np[2][page, :, row // c.block] = 67
            c.held[b][0][r:r + c.block] = 0
    c.pools[0].view(torch.uint8).copy_(torch.from_numpy(c.np[0]))
    c.pools[2].copy_(torch.from_numpy(c.np[2]))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale", [None, 1e-27, 1e-30])
def test_blocks_of_zeros(kind, scale):
    """K rows of zeros, whose scale is the least there is, in front of and behind ordinary ones."""
    c = Cache(kind, LENS, 2, 128, 64, 16, 22)
    zero_keys(c, 32, 80)
    both(c, 8, scale or 128 ** -0.5, 1.0)


@pytest.mark.parametrize("kind", KINDS)
def test_large_factors(kind):
    """A factor past fp32 on rows of zeros: their scores are 0, as those of all other rows."""
    c = Cache(kind, LENS, 2, 128, 64, 16, 23)
    zero_keys(c, 0, max(LENS))
    c.np[2][c.np[2] == 67] = 187
    c.pools[2].copy_(torch.from_numpy(c.np[2]))
    both(c, 8, 1e30, 1.0)
