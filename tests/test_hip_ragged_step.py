"""The ragged-batch ops together, as a serving step uses them: plan, QK norm + rotation + cache write through the plan's
slots, paged attention of this package over the planned block table, and linear attention over the planned offsets; a
prompt step of several requests, then decode steps, the latter also through replays of one graph.

Expected values: the 64-bit restatements on contiguous per-request caches.  Tolerances: q, k and v of a layer are bf16
inputs of the attention, so the oracle takes the rotated heads rounded to bf16 as well; a rotated value at a rounding
border may fall on the other side (one bf16 step, 2^-7 of it), which moves a score by at most D max|q||k| 2^-7 / sqrt(D)
and is far below the attention ops' own 1e-2 at these values; linear attention: 2^-8 of the value and 2^-6 of the sum of
absolute terms for the same step.
"""

import numpy as np
import pytest
import torch

from ezops import (LinearAttnDecodeOp, LinearAttnPrefillOp, PagedAttnDecodeOp, PagedBatchPlanOp, QkNormMropeOp, _hip)
from ezops.ops.fused_qk_norm_rope import rope_tables
from oracle import ragged

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)
H, HKV, D, P, M = 8, 2, 128, 32, 8
SEC = (24, 20, 20)
S = 400


def n(x):
    return x.detach().double().cpu().numpy()


def bf(x):
    return n(torch.from_numpy(x).to(torch.bfloat16))


class Requests:
    """Requests on the GPU side (paged cache, block table, free list, states) and on the oracle's (plain lists)."""

    def __init__(self, B, seed):
        g = torch.Generator().manual_seed(seed)
        self.B, self.g = B, g
        self.pool = B * M + 5
        order = torch.randperm(self.pool, generator=g).to(torch.int32)
        self.free, self.span = order.to(DEV), torch.tensor([0, self.pool], **I32)
        self.table = torch.full((B, M), -1, **I32)
        nan = torch.full((self.pool, HKV, P, D), float("nan"), dtype=torch.bfloat16, device=DEV)
        self.K, self.V = nan, nan.clone()
        self.state = torch.full((B + 1, HKV, D, D), float("nan"), device=DEV)
        self.slots = torch.randperm(B + 1, generator=g)[:B].to(**I32)
        self.past = torch.zeros(B, **I32)
        self.decay = torch.tensor([-0.4, -0.01], device=DEV)
        self.cos, self.sin = rope_tables(S, D, 1e6, DEV)
        self.qw, self.kw = ((1 + 0.1 * torch.randn(D, generator=g)).to(torch.bfloat16).to(DEV) for _ in range(2))
        self.o_k, self.o_v = [np.zeros((0, HKV, D))] * B, [np.zeros((0, HKV, D))] * B
        self.o_S = [np.zeros((HKV, D, D)) for _ in range(B)]

    def tokens(self, T):
        return torch.randn(T, H + 2 * HKV, D, generator=self.g).to(torch.bfloat16).to(DEV)

    def expect(self, x, pos, lens):
        """Advance the oracle's requests by the tokens x; -> per request (rotated q, outputs of linear attention, tol)."""
        q, k, v = n(x[:, :H]), n(x[:, H:H + HKV]), n(x[:, H + HKV:])
        ax = dict(sections=SEC, interleaved=True, norm=True)
        cos, sin = n(self.cos), n(self.sin)
        q = bf(ragged.qk_norm_mrope(q, n(self.qw), cos, sin, pos, **ax))
        k = bf(ragged.qk_norm_mrope(k, n(self.kw), cos, sin, pos, **ax))
        lam, out, at = np.exp(n(self.decay)), [], 0
        for b, m in enumerate(lens):
            r = slice(at, at + m)
            at += m
            o, ao = np.zeros((0, H, D)), np.zeros((0, H, D))
            if m:
                ao, _ = ragged.linear_attn(np.abs(q[r]), np.abs(k[r]), np.abs(v[r]), lam, np.abs(self.o_S[b]), D ** -0.5)
                o, self.o_S[b] = ragged.linear_attn(q[r], k[r], v[r], lam, self.o_S[b], D ** -0.5)
            self.o_k[b] = np.concatenate([self.o_k[b], k[r]])
            self.o_v[b] = np.concatenate([self.o_v[b], v[r]])
            out.append((q[r], o, 2.0 ** -8 * np.abs(o) * 1.01 + 2.0 ** -6 * ao))
        return out

    def attn(self, b, q, upto):
        """Softmax attention of one query [H, D] over the request's first `upto` rows."""
        k, v = self.o_k[b][:upto], self.o_v[b][:upto]
        out = np.empty((H, D))
        for h in range(H):
            s = k[:, h // (H // HKV)] @ q[h] * D ** -0.5
            p = np.exp(s - s.max())
            out[h] = p @ v[:, h // (H // HKV)] / p.sum()
        return out


def _positions(plan, rows):
    """Text and image tokens: three axes from the plan's positions, apart from each other in the middle of a request."""
    p = plan.positions
    img = (p >= 5) & (p < 30)
    return torch.stack([p, torch.where(img, 5 + (p - 5) // 5, p), torch.where(img, 5 + (p - 5) % 5, p)])


def _prompt_step(rq, lens, T):
    q_lens = torch.tensor(lens, **I32)
    plan = PagedBatchPlanOp(rq.B, T, P, M, rq.pool, backend="hip")(q_lens, rq.past, rq.table, rq.free, rq.span)
    x = rq.tokens(T)
    q, k, v = x[:, :H], x[:, H:H + HKV], x[:, H + HKV:]
    mrope = QkNormMropeOp(T, H, HKV, D, S, SEC, backend="hip", interleaved=True, page_size=P, num_pages=rq.pool)
    pos = _positions(plan, T)
    k_out = torch.zeros(T, HKV, D, dtype=torch.bfloat16, device=DEV)
    qr, kr = mrope(q, k, v, rq.qw, rq.kw, rq.cos, rq.sin, pos, rq.K, rq.V, plan.slot_mapping, k_out=k_out)
    # softmax attention of this package over the pages, offsets and lengths from the plan
    attn = torch.zeros(T, H, D, dtype=torch.bfloat16, device=DEV)
    _hip.call("ezops_prefill_attn_bf16", qr.data_ptr(), rq.K.data_ptr(), rq.V.data_ptr(), attn.data_ptr(),
              plan.cu_seqlens.data_ptr(), rq.past.data_ptr(), rq.B, T, H, HKV, M * P, D, max(lens), rq.table.data_ptr(),
              rq.pool, P, 0.0, _hip.stream())
    lin = LinearAttnPrefillOp(rq.B, T, H, HKV, D, backend="hip", num_slots=rq.B + 1)(
        qr, kr, v, rq.decay, plan.cu_seqlens, rq.state, rq.slots, rq.past, max_q_len=max(lens))
    past = rq.past.tolist()
    want = rq.expect(x[:sum(lens)], pos[:, :sum(lens)].cpu().numpy(), lens)
    at = 0
    for b, (m, (wq, wl, tol)) in enumerate(zip(lens, want)):
        if m:
            assert (np.abs(n(lin[at:at + m]) - wl) <= tol).all(), b
        for i in {0, m // 2, m - 1} if m else ():
            np.testing.assert_allclose(n(attn[at + i]), rq.attn(b, wq[i], past[b] + i + 1), rtol=1e-2, atol=2e-2)
        at += m
    rq.past, rq.span = plan.kv_lens, plan.free_span
    return plan


def test_prompts_chunks_and_decode_steps():
    rq = Requests(4, 1)
    assert _prompt_step(rq, [40, 1, 0, 100], 150).kv_lens.tolist() == [40, 1, 0, 100]
    plan = _prompt_step(rq, [30, 64, 7, 0], 101)  # a second chunk on cached prefixes, a first prompt, an idle request
    assert plan.kv_lens.tolist() == [70, 65, 7, 100]
    head, tail, needed = plan.free_span.tolist()
    assert needed == 1 + 2 + 1 and head == 2 + 1 + 0 + 4 + needed and tail == rq.pool
    # decode steps: eager, then replays of one graph that carries plan, cache and states on by itself
    B = rq.B
    op = PagedBatchPlanOp(B, B, P, M, rq.pool, backend="hip")
    mrope = QkNormMropeOp(B, H, HKV, D, S, SEC, backend="hip", interleaved=True, page_size=P, num_pages=rq.pool)
    dec = PagedAttnDecodeOp(B, H, HKV, D, P, M, rq.pool, backend="hip")
    lin = LinearAttnDecodeOp(B, H, HKV, D, B + 1, backend="hip")
    x, ones, out, past, span = rq.tokens(B), torch.ones(B, **I32), op.alloc(DEV), rq.past.clone(), rq.span[:2].clone()
    k_out = torch.zeros(B, HKV, D, dtype=torch.bfloat16, device=DEV)

    def step():
        plan = op(ones, past, rq.table, rq.free, span, out=out)
        qr, kr = mrope(x[:, :H], x[:, H:H + HKV], x[:, H + HKV:], rq.qw, rq.kw, rq.cos, rq.sin,
                       torch.stack([plan.positions] * 3), rq.K, rq.V, plan.slot_mapping, k_out=k_out)
        a = dec(qr.unsqueeze(2), rq.K, rq.V, rq.table, plan.kv_lens)
        o = lin(qr, kr, x[:, H + HKV:], rq.decay, rq.state, rq.slots)
        past.copy_(plan.kv_lens)
        span.copy_(plan.free_span[:2])
        return a, o

    def check(a, o):
        pos = np.stack([[len(k) for k in rq.o_k]] * 3)
        for b, (wq, wl, tol) in enumerate(rq.expect(x, pos, [1] * B)):
            assert (np.abs(n(o[b:b + 1]) - wl) <= tol).all(), b
            np.testing.assert_allclose(n(a[b, :, 0]), rq.attn(b, wq[0], len(rq.o_k[b])), rtol=1e-2, atol=2e-2)

    check(*step())
    keep = [t.clone() for t in (past, span, rq.table, rq.K, rq.V, rq.state)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, o = step()
    for t, k in zip((past, span, rq.table, rq.K, rq.V, rq.state), keep):
        assert torch.equal(t.nan_to_num(9.0) if t.is_floating_point() else t, k.nan_to_num(9.0) if k.is_floating_point() else k)
    for _ in range(40):  # past the end of a page
        x.copy_(rq.tokens(B))
        graph.replay()
        check(a, o)
    assert past.tolist() == [111, 106, 48, 141]
    for b in range(B):
        np.testing.assert_allclose(n(rq.state[rq.slots[b]]), rq.o_S[b], rtol=2e-2, atol=2e-2 * np.abs(rq.o_S[b]).max())


def test_padded_batch_and_exhausted_pool():
    """Idle rows (no tokens, no state slot) and a free list that ends: what has a place is right, the rest is left out."""
    rq = Requests(3, 2)
    rq.span[1] = 2  # two pages in all
    rq.slots[1] = -1
    lens, T = [33, 20, 0], 64
    plan = PagedBatchPlanOp(3, T, P, M, rq.pool, backend="hip")(torch.tensor(lens, **I32), None, rq.table, rq.free, rq.span)
    assert plan.free_span.tolist() == [2, 2, 3]
    assert (plan.slot_mapping[:33] >= 0).all() and (plan.slot_mapping[33:] == -1).all()
    x = rq.tokens(T)
    q_out = torch.full((T, H, D), 3.0, dtype=torch.bfloat16, device=DEV)
    mrope = QkNormMropeOp(T, H, HKV, D, S, SEC, backend="hip", interleaved=True, page_size=P, num_pages=rq.pool)
    pos = torch.stack([plan.positions] * 3)
    mrope(x[:, :H], x[:, H:H + HKV], x[:, H + HKV:], rq.qw, rq.kw, rq.cos, rq.sin, pos, rq.K, rq.V, plan.slot_mapping,
          q_out=q_out)
    assert bool((q_out[53:] == 3).all()) and bool(torch.isfinite(q_out[:53].float()).all())
    written = torch.isfinite(rq.K.float()).all(-1).sum().item()
    assert written == 33 * HKV
    out = torch.full((T, H, D), 3.0, dtype=torch.bfloat16, device=DEV)
    before = rq.state.clone()
    LinearAttnPrefillOp(3, T, H, HKV, D, backend="hip", num_slots=4)(q_out, x[:, H:H + HKV], x[:, H + HKV:], rq.decay,
                                                                     plan.cu_seqlens, rq.state, rq.slots, out=out)
    assert bool((out[33:] == 3).all()) and bool(torch.isfinite(out[:33].float()).all())
    touched = [s for s in range(4) if torch.isfinite(rq.state[s]).all()]
    assert touched == [int(rq.slots[0])] and torch.isnan(before).all()
