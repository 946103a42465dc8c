"""What holds the states of the linear attention to fp32: the weighted values as three bf16 parts, and lambda^n S as
S + (lambda^n - 1) S.  On the CPU an emulation of both forms and of the cheaper ones they stand in for shows that the
bounds tell them apart; on the GPU the kernels meet the bounds.

Bounds, as norms over a state relative to its own (r = 2^-24 / sqrt(3) = 3.4e-8: the rms of one rounding to fp32; terms
have random signs, so independent errors of the terms add up as the terms do):

  one prompt of up to 257 tokens, 3e-7.  Per term two powers, 0.3 units of 2^-23 each at the rms, and two products:
  7e-8.  The sum: 12 steps a chunk (four of 16 tokens, three parts), each rounded at the size the sum has by then: 8.4e-8
  a chunk, with the decays here (lambda^64 <= 0.88) twice that after many: 1.7e-7.  Together 1.9e-7, half as much again.
  Two parts leave 2^-18 / 6 = 6.4e-7 of each term.

  n tokens one by one at lambda ~ 1 from a state, 4 r sqrt(n m): m roundings of the whole state a step (one in the
  recurrent form, S + y; four in the chunked form: lambda S and the three parts) at a size that it has all along; 4 is
  the margin.  lambda rounded to fp32 is off by d up to 2^-25 at every step in the same direction: d n of the start
  state is lost or kept too long, with the decays here above 0.8 * 2^-25 n.
"""

import numpy as np
import pytest
import torch

from ezops import LinearAttnDecodeOp, LinearAttnPrefillOp

R = 2.0 ** -24 / 3 ** 0.5
PROMPT = 3e-7
F32 = np.float32


def _drift_bound(n, m):
    return 4 * R * (n * m) ** 0.5


def _decays_off(count):
    """Decays between 1e-4 and 2e-4 whose lambda lies furthest from fp32 numbers."""
    g = -np.linspace(1e-4, 2e-4, 4001).astype(F32)
    lam = np.exp(g.astype(np.float64))
    off = np.abs(lam.astype(F32).astype(np.float64) - lam)
    best = np.sort(g[np.argsort(off)[-count:]])
    lam = np.exp(best.astype(np.float64))
    assert (np.abs(lam.astype(F32) - lam) > 0.8 * 2.0 ** -25).all()
    return best


def _bf16(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(torch.bfloat16).float().numpy()


def _inputs(T, D, seed):
    g = torch.Generator().manual_seed(seed)
    k, v = torch.randn(T, D, generator=g), torch.randn(T, D, generator=g)
    return _bf16(torch.nn.functional.silu(k).numpy()), _bf16(v.numpy())


def _chunk_emulated(k, v, g, parts):
    """The chunked sums of one head: fp32 weights, `parts` bf16 parts of the weighted values, 16 tokens a rounding."""
    T, D = k.shape
    S, g2 = np.zeros((D, D), F32), F32(g) * F32(1.4426950408889634)
    pad = -T % 64
    k, v = np.concatenate([np.zeros((pad, D), F32), k]), np.concatenate([np.zeros((pad, D), F32), v])
    for c in range(0, T + pad, 64):
        S = S + F32(np.expm1(F32(g) * F32(64))) * S
        for s in range(4):
            t = slice(c + 16 * s, c + 16 * s + 16)
            w = np.exp2(g2 * np.arange(15, -1, -1, dtype=F32)) * np.exp2(g2 * F32(48 - 16 * s))
            rest = (v[t] * w[:, None].astype(F32)).astype(F32)
            split = []
            for _ in range(parts):
                split.append(_bf16(rest))
                rest = rest - split[-1]
            for p in reversed(split):
                S = (S.astype(np.float64) + k[t].T.astype(np.float64) @ p).astype(F32)
    return S


def _exact(k, v, g, S=None):
    S = np.zeros((k.shape[1],) * 2) if S is None else S.astype(np.float64)
    lam = np.exp(np.float64(g))
    for t in range(len(k)):
        S = lam * S + np.outer(k[t].astype(np.float64), v[t])
    return S


def _off(got, want):
    return np.linalg.norm(got - want) / np.linalg.norm(want)


@pytest.mark.parametrize("T", [64, 257])
def test_two_parts_would_fail(T):
    k, v = _inputs(T, 64, T)
    for g in (-0.5, -0.02, -0.002):
        want = _exact(k, v, F32(g))
        assert _off(_chunk_emulated(k, v, g, 3), want) < PROMPT
        assert _off(_chunk_emulated(k, v, g, 2), want) > PROMPT


def test_a_rounded_decay_would_fail():
    n, D = 3000, 16
    k, v = _inputs(n, D, 1)
    S0 = (100 * np.random.RandomState(1).randn(D, D)).astype(F32)
    for g in _decays_off(4):
        want = _exact(k, v, g, S0)
        S, plain = S0.copy(), S0.copy()
        m, lam = F32(np.expm1(np.float64(g))), F32(np.exp(np.float64(g)))
        for t in range(n):
            x = np.outer(k[t], v[t])
            S = S + (m * S + x)
            plain = lam * plain + x
        assert _off(S, want) < _drift_bound(n, 1)
        assert _off(plain, want) > _drift_bound(n, 4)


def _gpu(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to("cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 16, 64, 65, 128, 257])
def test_states_of_prompts(T, D):
    """With and without segments (a length bound of 257 or not), fresh and continued."""
    H = 4
    g = np.array([-0.5, -0.02, -0.01, -0.002], F32)
    kv = [_inputs(T, D, 10 * T + h) for h in range(H)]
    k, v = (_gpu(np.stack([x[i] for x in kv], 1)).to(torch.bfloat16) for i in (0, 1))
    i32 = dict(dtype=torch.int32, device="cuda")
    start = np.random.RandomState(T).randn(H, D, D).astype(F32)
    for past in (0, 5):
        for pad in (0, 900):
            op = LinearAttnPrefillOp(1, T + pad, H, H, D, backend="hip", num_slots=1)
            rows = [torch.cat([x, x.new_zeros(pad, H, D)]) for x in (k, k, v)]
            S = _gpu(start[None])
            op(*rows, _gpu(g), torch.tensor([0, T], **i32), S, None, torch.tensor([past], **i32))
            got = S[0].double().cpu().numpy()
            for h in range(H):
                want = _exact(*kv[h], g[h], start[h] if past else None)
                assert _off(got[h], want) < PROMPT, (past, pad, h, _off(got[h], want))


@pytest.mark.gpu
@pytest.mark.parametrize("form,n,m", [("single tokens", 4096, 1), ("prompts of one token", 2048, 4)])
def test_states_do_not_drift(form, n, m):
    H, D = 4, 64
    g = _decays_off(H)
    kv = [_inputs(n, D, 7 + h) for h in range(H)]
    k, v = (_gpu(np.stack([x[i] for x in kv], 1)).to(torch.bfloat16) for i in (0, 1))
    start = (100 * np.random.RandomState(2).randn(H, D, D)).astype(F32)
    S, want, gd, out = _gpu(start[None]), _gpu(start).double(), _gpu(g), torch.empty(1, H, D, dtype=torch.bfloat16, device="cuda")
    lam = torch.exp(gd.double())[:, None, None]
    i32 = dict(dtype=torch.int32, device="cuda")
    if m == 1:
        op = LinearAttnDecodeOp(1, H, H, D, 1, backend="hip")
        step = lambda t: op(k[t:t + 1], k[t:t + 1], v[t:t + 1], gd, S, out=out)  # noqa: E731
    else:
        op = LinearAttnPrefillOp(1, 1, H, H, D, backend="hip", num_slots=1)
        cu, past = torch.tensor([0, 1], **i32), torch.ones(1, **i32)
        step = lambda t: op(k[t:t + 1], k[t:t + 1], v[t:t + 1], gd, cu, S, None, past, out=out)  # noqa: E731
    for t in range(n):
        step(t)
        want = lam * want + k[t].double()[:, :, None] * v[t].double()[:, None, :]
    for h in range(H):
        off = float((S[0, h].double() - want[h]).norm() / want[h].norm())
        assert off < _drift_bound(n, m), (h, off)
