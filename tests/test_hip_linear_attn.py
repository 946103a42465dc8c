"""HIP linear attention (packed prompts, single tokens) against the recurrence in 64 bits.

Tolerances, element by element.  With A the same recurrence over absolute values (|q|, |k|, |v|, |S0|):
  out    one bf16 rounding, 2^-8 |o|, plus 2^-14 A: probabilities and states enter the matrix products as two bf16 parts
         (2^-16 of each term), powers of the decay and fp32 sums of at most 192 terms a chunk add 192 * 2^-24 < 2^-16 each,
         the carried state 2^-22 a chunk (at most 64 chunks here: 2^-16); three halves of 2^-14 in all, rounded up.
  state  2^-15 A: the decay-weighted values enter as three parts (2^-24), sums and carries as above.
Powers exp(n g) are off by |n g| 2^-23 of themselves, at most 2^-23 / e * 2 of the terms they weigh.
"""

import numpy as np
import pytest
import torch

from ezops import LinearAttnDecodeOp, LinearAttnPrefillOp
from oracle import ragged

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF = float("inf")


def n(x):
    return x.detach().double().cpu().numpy()


def _inputs(T, H, Hkv, D, seed, packed=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H + 2 * Hkv, D, generator=g)
    x[:, :H + Hkv] = torch.nn.functional.silu(x[:, :H + Hkv])
    x = x.to(torch.bfloat16).to(DEV)
    q, k, v = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
    return (q, k, v) if packed else (q.contiguous(), k.contiguous(), v.contiguous())


def _decay(Hkv):
    return -torch.exp2(-1 - 7 * torch.arange(Hkv, dtype=torch.float32, device=DEV) / max(1, Hkv - 1))


def _expect(q, k, v, g, S0, scale):
    """(out, state, their tolerances) of one sequence."""
    lam = np.exp(n(g))
    o, S = ragged.linear_attn(n(q), n(k), n(v), lam, S0, scale)
    ao, aS = ragged.linear_attn(np.abs(n(q)), np.abs(n(k)), np.abs(n(v)), lam, np.abs(S0), scale)
    return o, S, 2.0 ** -8 * np.abs(o) * (1 + 2.0 ** -8) + 2.0 ** -14 * ao, 2.0 ** -15 * aS


def _close(got, want, tol, what):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(np.abs(got - want)[bad].max()), np.argwhere(bad)[:3].tolist())


def _prefill(lens, past, H, Hkv, D, *, slots=None, pool=None, pad=0, seed=0, g=None, max_q_len=None, packed=True, state=True,
             scale=None, poison=True):
    B, T = len(lens), sum(lens) + pad
    q, k, v = _inputs(max(T, 1), H, Hkv, D, seed, packed)
    T = q.shape[0]
    g = _decay(Hkv) if g is None else g
    pool = B + 2 if pool is None else pool
    slots = list(range(B))[::-1] if slots is None else slots
    cu = np.concatenate([[0], np.cumsum(lens)])
    if poison:  # rows of no sequence
        for x in (q, k, v):
            x[cu[-1]:] = float("nan")
    op = LinearAttnPrefillOp(B, T, H, Hkv, D, backend="hip", num_slots=pool if state else None, scale=scale)
    i32 = dict(dtype=torch.int32, device=DEV)
    S = torch.randn(pool, Hkv, D, D, generator=torch.Generator().manual_seed(seed + 1)).to(DEV)
    if poison:  # states that are not read: unused slots, slots of fresh sequences
        used = {s for s, p in zip(slots, past) if p > 0}
        for s in range(pool):
            if s not in used:
                S[s] = float("nan")
    before = S.clone()
    out = torch.full((T, H, D), 7.0, dtype=torch.bfloat16, device=DEV)
    args = [q, k, v, g, torch.tensor(cu, **i32)]
    if state:
        args += [S, torch.tensor(slots, **i32), torch.tensor(past, **i32)]
    mq = max(lens) if max_q_len is None else max_q_len
    got = op(*args, max_q_len=mq, out=out)
    assert got is out
    scale = D ** -0.5 if scale is None else scale
    touched = set()
    for b, m in enumerate(lens):
        m = min(m, mq) if mq else m
        rows = slice(int(cu[b]), int(cu[b]) + m)
        end = slice(rows.stop, int(cu[b + 1]))
        assert bool((out[end] == 7).all())
        if state and (not 0 <= slots[b] < pool or slots[b] in slots[:b]):
            assert bool((out[rows] == 7).all()), b
            continue
        if m == 0:
            continue
        S0 = n(before[slots[b]]) if state and past[b] > 0 else np.zeros((Hkv, D, D))
        o, S1, to, ts = _expect(q[rows], k[rows], v[rows], g, S0, scale)
        _close(n(out[rows]), o, to, f"out of sequence {b}")
        if state:
            touched.add(slots[b])
            _close(n(S[slots[b]]), S1, ts, f"state of sequence {b}")
    assert bool((out[int(cu[-1]):] == 7).all())
    for s in range(pool):
        if s not in touched:
            assert torch.equal(S[s].view(torch.int32), before[s].view(torch.int32)), s
    if state:  # the same call again from the same states: the same bits
        first, last = out.clone(), S.clone()
        S.copy_(before)
        op(*args, max_q_len=mq, out=out)
        assert torch.equal(first, out) and torch.equal(last.view(torch.int32), S.view(torch.int32))


@pytest.mark.parametrize("m", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 257])
def test_lengths(m):
    _prefill([m], [0], 4, 2, 128, seed=m)
    _prefill([m], [5], 2, 2, 64, seed=m, packed=False)


@pytest.mark.parametrize("H,Hkv,D", [(1, 1, 128), (2, 1, 64), (16, 1, 128), (8, 1, 64), (32, 8, 128), (8, 8, 128), (16, 8, 64),
                                     (3, 3, 128)])
def test_heads(H, Hkv, D):
    _prefill([70, 0, 1, 130], [0, 3, 9, 0], H, Hkv, D, seed=H, pad=5)


@pytest.mark.parametrize("D", [64, 128])
def test_ragged_padded_and_left_out(D):
    """Empty sequences, slots outside the pool, a slot held by an earlier sequence, NaN in every row, state and slot that
    the call has no business with."""
    _prefill([0, 65, 64, 0, 90, 3, 100, 1], [1, 0, 7, 0, 2, 0, 4, 8], 4, 2, D, slots=[5, 1, 6, 2, -1, 1, 9, 0], pool=9,
             pad=40, seed=2)
    _prefill([40, 33], [0, 0], 4, 2, D, slots=[2, 2], pool=3, seed=3)


def test_neighbours_do_not_leak():
    """A sequence of NaN and infinities between two others, all within one tile."""
    H, Hkv, D = 4, 2, 128
    q, k, v = _inputs(60, H, Hkv, D, 8)
    for x in (q, k, v):
        x[20:40] = float("nan")
        x[25:30] = INF
    cu = torch.tensor([0, 20, 40, 60], dtype=torch.int32, device=DEV)
    op = LinearAttnPrefillOp(3, 60, H, Hkv, D, backend="hip", num_slots=3)
    S = torch.zeros(3, Hkv, D, D, device=DEV)
    out = op(q, k, v, _decay(Hkv), cu, S)
    for b, r in ((0, slice(0, 20)), (2, slice(40, 60))):
        o, S1, to, ts = _expect(q[r], k[r], v[r], _decay(Hkv), np.zeros((Hkv, D, D)), D ** -0.5)
        _close(n(out[r]), o, to, b)
        _close(n(S[b]), S1, ts, b)


@pytest.mark.parametrize("g", [[-INF, 0.0], [-1e-6, -80.0], [-200.0, -0.01], [-1e30, -3e-39]])
def test_decays(g):
    """No memory, no forgetting, and both ends between them."""
    t = torch.tensor(g, dtype=torch.float32, device=DEV)
    _prefill([150, 70], [0, 4], 4, 2, 128, g=t, seed=6)
    _prefill([150, 70], [0, 4], 2, 2, 64, g=t, seed=7)


def test_no_state_and_scale():
    _prefill([100, 0, 65], [0, 0, 0], 4, 2, 128, state=False, seed=1)
    _prefill([100], [0], 4, 2, 128, scale=1.0, seed=1)


@pytest.mark.parametrize("mq", [0, 1, 64, 100])
def test_length_bound(mq):
    """0: no bound known; sequences longer than the bound are cut off there."""
    _prefill([100, 30, 150], [0, 3, 0], 4, 2, 64, max_q_len=mq, seed=4, pad=3)


@pytest.mark.parametrize("H,Hkv,D,lens", [(2, 1, 128, [1500]), (4, 2, 128, [700, 0, 900]), (1, 1, 64, [2500]),
                                          (2, 2, 64, [300] * 5)])
def test_long_sequences(H, Hkv, D, lens):
    """Long ones, which are worked on in pieces; bounds known and not known."""
    past = [(i % 2) * 3 for i in range(len(lens))]
    _prefill(lens, past, H, Hkv, D, seed=5, pad=9)
    _prefill(lens, past, H, Hkv, D, seed=5, max_q_len=0)


@pytest.mark.parametrize("H,Hkv,D,lens", [(32, 2, 128, [701, 1, 340]), (16, 16, 128, [130, 2000]), (32, 4, 64, [1500, 3, 650])])
def test_many_segments(H, Hkv, D, lens):
    """Many segments and heads: short first chunks, states taken on, rows behind the last sequence."""
    _prefill(lens, [4 * (i % 2) for i in range(len(lens))], H, Hkv, D, seed=31, pad=7)


@pytest.mark.parametrize("D", [64, 128])
def test_more_sequences_than_threads(D):
    """Sequences are found by a block of 128 or 256 threads: 300 short ones, some empty, some continued, a slot twice."""
    r = np.random.RandomState(3)
    lens = r.choice([0, 1, 2, 5, 70], 300, p=[0.2, 0.4, 0.2, 0.18, 0.02]).tolist()
    slots = r.permutation(303)[:300].tolist()
    slots[290] = slots[4]
    _prefill(lens, r.choice([0, 3], 300).tolist(), 2, 1, D, slots=slots, pool=303, seed=9, pad=11)


@pytest.mark.parametrize("H,lens,past", [(8, [64], [3]), (16, [100, 300], [7, 0]), (4, [130, 0, 64, 5], [1, 1, 1, 1])])
def test_shared_query_heads_of_few_blocks(H, lens, past):
    """The query heads of a kv head in several blocks, all of which start from the stored state that one replaces."""
    for known in (None, 0):
        _prefill(lens, past, H, 1, 128, seed=21, max_q_len=known)
        _prefill(lens, [0] * len(lens), H, 1, 64, seed=22, max_q_len=known)


def test_chunks_equal_the_whole():
    """A prompt in two calls through the state gives what one call gives (within the sum of both tolerances)."""
    H, Hkv, D, T = 4, 2, 128, 300
    q, k, v = _inputs(T, H, Hkv, D, 11)
    g, i32 = _decay(Hkv), dict(dtype=torch.int32, device=DEV)
    S1, S2 = torch.zeros(1, Hkv, D, D, device=DEV), torch.full((1, Hkv, D, D), float("nan"), device=DEV)
    whole = LinearAttnPrefillOp(1, T, H, Hkv, D, backend="hip", num_slots=1)(q, k, v, g, torch.tensor([0, T], **i32), S1)
    parts = []
    for a, b in ((0, 130), (130, 300)):
        op = LinearAttnPrefillOp(1, b - a, H, Hkv, D, backend="hip", num_slots=1)
        parts.append(op(q[a:b], k[a:b], v[a:b], g, torch.tensor([0, b - a], **i32), S2, None, torch.tensor([a], **i32)))
    o, S, to, ts = _expect(q, k, v, g, np.zeros((Hkv, D, D)), D ** -0.5)
    _close(n(torch.cat(parts)), n(whole), 2 * to, "out")
    _close(n(S2[0]), n(S1[0]), 2 * ts, "state")


def test_bad_offsets_stay_in_bounds():
    """Offsets outside the rows are clamped: the sequences with good ones get their results, nothing else breaks."""
    H, Hkv, D, T = 2, 2, 64, 100
    q, k, v = _inputs(T, H, Hkv, D, 12)
    i32 = dict(dtype=torch.int32, device=DEV)
    op = LinearAttnPrefillOp(2, T, H, Hkv, D, backend="hip", num_slots=2)
    for cu in ([0, 40, 1 << 30], [-7, 40, 100]):
        S = torch.zeros(2, Hkv, D, D, device=DEV)
        out = op(q, k, v, _decay(Hkv), torch.tensor(cu, **i32), S)
        for b, r in ((0, slice(0, 40)), (1, slice(40, 100))):
            o, S1, to, ts = _expect(q[r], k[r], v[r], _decay(Hkv), np.zeros((Hkv, D, D)), D ** -0.5)
            _close(n(out[r]), o, to, b)


def test_first_sequence_behind_the_first_row():
    """Rows in front of the first sequence are of no sequence; one long enough to be cut into segments."""
    H, Hkv, D, T = 4, 2, 128, 900
    q, k, v = _inputs(T, H, Hkv, D, 14)
    for x in (q, k, v):
        x[:130] = float("nan")
    S = torch.full((2, Hkv, D, D), float("nan"), device=DEV)
    out = torch.full((T, H, D), 7.0, dtype=torch.bfloat16, device=DEV)
    cu = torch.tensor([130, 170, 880], dtype=torch.int32, device=DEV)
    LinearAttnPrefillOp(2, T, H, Hkv, D, backend="hip", num_slots=2)(q, k, v, _decay(Hkv), cu, S, out=out)
    assert bool((out[:130] == 7).all()) and bool((out[880:] == 7).all())
    for b, r in ((0, slice(130, 170)), (1, slice(170, 880))):
        o, S1, to, ts = _expect(q[r], k[r], v[r], _decay(Hkv), np.zeros((Hkv, D, D)), D ** -0.5)
        _close(n(out[r]), o, to, b)
        _close(n(S[b]), S1, ts, b)


def test_rows_of_one_token_with_any_stride():
    """A single row's stride does not matter."""
    H, Hkv, D = 4, 2, 64
    x = torch.randn(3, (H + 2 * Hkv) * D + 3, device=DEV).bfloat16()
    row = x[:1, :(H + 2 * Hkv) * D].unflatten(1, (H + 2 * Hkv, D))
    q, k, v = row[:, :H], row[:, H:H + Hkv], row[:, H + Hkv:]
    S = torch.randn(1, Hkv, D, D, device=DEV)
    want = S.clone()
    op = LinearAttnDecodeOp(1, H, Hkv, D, 1, backend="hip")
    a = op(q, k, v, _decay(Hkv), S)
    b = op(q.contiguous(), k.contiguous(), v.contiguous(), _decay(Hkv), want)
    assert torch.equal(a, b) and torch.equal(S, want)


def test_prefill_on_another_stream_and_in_two_graphs():
    H, Hkv, D, T = 8, 2, 128, 1100
    q, k, v = _inputs(T, H, Hkv, D, 13)
    g, cu = _decay(Hkv), torch.tensor([0, 400, 1100], dtype=torch.int32, device=DEV)
    past = torch.tensor([0, 2], dtype=torch.int32, device=DEV)
    op = LinearAttnPrefillOp(2, T, H, Hkv, D, backend="hip", num_slots=2)
    S0 = torch.randn(2, Hkv, D, D, device=DEV)
    S = S0.clone()
    want = op(q, k, v, g, cu, S, None, past).clone()
    end = S.clone()
    graphs, outs, states = [], [], []
    for _ in range(2):
        st, out = S0.clone(), torch.zeros_like(want)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            op(q, k, v, g, cu, st, None, past, out=out)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(st, end)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            op(q, k, v, g, cu, st, None, past, out=out)
        graphs.append(graph), outs.append(out), states.append(st)
    for i in range(3):  # the two graphs at once, on two streams
        for st, out in zip(states, outs):
            st.copy_(S0)
            out.zero_()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for st, out in zip(states, outs):
            assert torch.equal(out, want) and torch.equal(st, end), i


@pytest.mark.parametrize("B,H,Hkv,D,slots", [
    (1, 1, 1, 64, None), (1, 32, 8, 128, None), (5, 16, 1, 128, [4, -1, 0, 9, 4]), (3, 8, 8, 64, [2, 1, 0]),
    (70, 4, 2, 128, None), (9, 8, 4, 64, [3, 3, -5, 8, 1, 0, 1, 7, 1 << 30]), (300, 2, 2, 64, "all"), (2, 4, 1, 128, None),
])
def test_decode(B, H, Hkv, D, slots):
    """One step: the state is off by at most 8 fp32 roundings of its terms, the output by D + 16 more and one to bf16."""
    q, k, v = _inputs(B, H, Hkv, D, B)
    pool = 9 if isinstance(slots, list) else B + 3
    if slots == "all":
        perm = np.random.RandomState(1).permutation(pool)[:B].tolist()
        perm[200] = perm[7]
        slots = perm
    g = _decay(Hkv)
    g[0] = -INF if B == 5 else g[0]
    op = LinearAttnDecodeOp(B, H, Hkv, D, pool, backend="hip")
    S = torch.randn(pool, Hkv, D, D, device=DEV)
    t = None if slots is None else torch.tensor(slots, dtype=torch.int32, device=DEV)
    at = list(range(B)) if slots is None else slots
    before = S.clone()
    out = torch.full((B, H, D), 7.0, dtype=torch.bfloat16, device=DEV)
    assert op(q, k, v, g, S, t, out=out) is out
    lam, touched = np.exp(n(g)), set()
    for b, s in enumerate(at):
        if not 0 <= s < pool or s in at[:b]:
            assert bool((out[b] == 7).all())
            continue
        touched.add(s)
        o, S1 = ragged.linear_attn(n(q[b:b + 1]), n(k[b:b + 1]), n(v[b:b + 1]), lam, n(before[s]), D ** -0.5)
        ao, aS = ragged.linear_attn(*(np.abs(n(x[b:b + 1])) for x in (q, k, v)), lam, np.abs(n(before[s])), D ** -0.5)
        _close(n(S[s]), S1, 8 * 2.0 ** -24 * aS, f"state {b}")
        _close(n(out[b]), o[0], 2.0 ** -8 * np.abs(o[0]) * (1 + 2.0 ** -8) + (D + 24) * 2.0 ** -24 * ao[0], f"out {b}")
    for s in range(pool):
        if s not in touched:
            assert torch.equal(S[s], before[s])


def test_decode_state_past_32_bits():
    """A pool of 6 GiB, the last slot."""
    Hkv, D = 8, 128
    pool = (6 << 30) // (Hkv * D * D * 4)
    q, k, v = _inputs(1, Hkv, Hkv, D, 1)
    S = torch.zeros(pool, Hkv, D, D, device=DEV)
    at = torch.tensor([pool - 1], dtype=torch.int32, device=DEV)
    LinearAttnDecodeOp(1, Hkv, Hkv, D, pool, backend="hip")(q, k, v, _decay(Hkv), S, at)
    assert torch.equal(S[-1], k[0].float()[:, :, None] * v[0].float()[:, None, :])
    LinearAttnPrefillOp(1, 1, Hkv, Hkv, D, backend="hip", num_slots=pool)(q, k, v, _decay(Hkv), torch.tensor(
        [0, 1], dtype=torch.int32, device=DEV), S, at, torch.tensor([0], dtype=torch.int32, device=DEV))
    assert torch.allclose(S[-1], k[0].float()[:, :, None] * v[0].float()[:, None, :], rtol=2 ** -20)
    assert not bool(S[:-1].any())


def test_decode_continues_prefill_in_a_graph():
    """A prompt, then tokens one by one through replays of one graph, against the whole in one call."""
    H, Hkv, D, T, P = 4, 2, 128, 90, 70
    q, k, v = _inputs(T, H, Hkv, D, 17)
    g, i32 = _decay(Hkv), dict(dtype=torch.int32, device=DEV)
    slots = torch.tensor([2], **i32)
    S = torch.full((3, Hkv, D, D), float("nan"), device=DEV)
    first = LinearAttnPrefillOp(1, P, H, Hkv, D, backend="hip", num_slots=3)(q[:P], k[:P], v[:P], g, torch.tensor(
        [0, P], **i32), S, slots)
    op = LinearAttnDecodeOp(1, H, Hkv, D, 3, backend="hip")
    b = [x[:1].clone() for x in (q, k, v)]
    out = torch.zeros(1, H, D, dtype=torch.bfloat16, device=DEV)
    keep = S.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op(*b, g, S, slots, out=out)
    S.copy_(keep)
    rows = [first]
    for t in range(P, T):
        for dst, src in zip(b, (q, k, v)):
            dst.copy_(src[t:t + 1])
        graph.replay()
        rows.append(out.clone())
    o, S1, to, ts = _expect(q, k, v, g, np.zeros((Hkv, D, D)), D ** -0.5)
    _close(n(torch.cat(rows)), o, to, "out")
    _close(n(S[2]), S1, ts, "state")


def test_argument_checks():
    H, Hkv, D = 4, 2, 64
    q, k, v = _inputs(8, H, Hkv, D, 0)
    cu = torch.tensor([0, 8], dtype=torch.int32, device=DEV)
    S = torch.zeros(2, Hkv, D, D, device=DEV)
    op = LinearAttnPrefillOp(1, 8, H, Hkv, D, backend="hip", num_slots=2)
    good = [q, k, v, _decay(Hkv), cu, S]
    odd = torch.zeros(8 * H * D + 1, dtype=torch.bfloat16, device=DEV)[1:].view(8, H, D)
    for i, bad in ((0, odd), (0, q.float()), (1, k[:7]), (2, v.transpose(1, 2)), (3, _decay(Hkv).double()), (4, cu.long()),
                   (5, S[:1]), (5, S.bfloat16()), (5, None), (0, q[:1].expand(8, H, D))):
        args = list(good)
        args[i] = bad
        with pytest.raises(ValueError):
            op(*args)
    with pytest.raises(ValueError, match="max_q_len"):
        op(*good, max_q_len=-1)
    with pytest.raises(ValueError, match="out"):
        op(*good, out=torch.empty(8, H, D, device=DEV))
    with pytest.raises(ValueError, match="without a state"):
        LinearAttnPrefillOp(1, 8, H, Hkv, D, backend="hip")(*good[:5], None, torch.zeros(1, dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError, match="GPU tensors"):
        op(q.cpu(), *good[1:])
    dec = LinearAttnDecodeOp(8, H, Hkv, D, 8, backend="hip")
    S8 = torch.zeros(8, Hkv, D, D, device=DEV)
    for args in ((q, k, v, _decay(Hkv), S), (odd, k, v, _decay(Hkv), S8),
                 (q, k, v, _decay(Hkv), S8, torch.zeros(8, dtype=torch.int64, device=DEV))):
        with pytest.raises(ValueError):
            dec(*args)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("mq", [0, 400])
def test_bad_offsets_of_long_sequences_stay_in_bounds(D, mq):
    """Ends far below zero, and offsets that decrease, in calls whose sequences are cut into segments (with a workspace):
    the good sequence gets its result, the bad one nothing, and the rows and states around the tensors stay as they were."""
    H, Hkv, T, guard = 2, 2, 1100, 1200
    qg, kg, vg = _inputs(T + guard, H, Hkv, D, 40)
    for x in (qg, kg, vg):
        x[T:] = float("nan")
    q, k, v = qg[:T], kg[:T], vg[:T]
    i32, lo = dict(dtype=torch.int32, device=DEV), -(1 << 31)
    op = LinearAttnPrefillOp(2, T, H, Hkv, D, backend="hip", num_slots=2)
    for end in (-1, lo, lo + 40, lo + 701, 3):
        pool = torch.full((4, Hkv, D, D), 7.0, device=DEV)
        rows = torch.full((T + guard, H, D), 7.0, dtype=torch.bfloat16, device=DEV)
        S, out = pool[1:3], rows[:T]
        S[0] = torch.randn(Hkv, D, D, generator=torch.Generator().manual_seed(3)).to(DEV)
        first = n(S[0])
        op(q, k, v, _decay(Hkv), torch.tensor([0, 700, end], **i32), S, None, torch.tensor([5, 9], **i32), max_q_len=mq, out=out)
        m = mq or 700
        o, S1, to, ts = _expect(q[:m], k[:m], v[:m], _decay(Hkv), first, D ** -0.5)
        _close(n(out[:m]), o, to, end)
        _close(n(S[0]), S1, ts, end)
        assert bool((rows[m:] == 7).all()) and bool((pool[[0, 2, 3]] == 7).all()), end


@pytest.mark.parametrize("H,Hkv,D,lens", [
    (16, 16, 64, [1] * 30 + [700] + [1] * 20 + [0, 64, 65, 1, 300]),     # more slots by number than by row
    (32, 8, 64, [1] * 45 + [200, 1, 64, 0, 130]),                         # heads in groups, one block a kv head
    (2, 2, 128, [1100, 1, 64, 900, 3]),                                   # few sequences
    (8, 2, 128, [300, 1, 64, 70, 1]),                                     # heads shared out: copies of all states
])
def test_mixed_steps(H, Hkv, D, lens):
    """Chunks of long prompts beside single tokens and idle rows, all continued or every other one: what is not cut into
    segments goes from its state to its state."""
    B = len(lens)
    order = np.random.RandomState(B).permutation(B + 2)[:B].tolist()
    for past in ([3] * B, [i % 2 for i in range(B)]):
        for mq in (None, 0):
            _prefill(lens, past, H, Hkv, D, slots=order, seed=41, pad=6, max_q_len=mq)


def test_workspace_of_a_mixed_step():
    """2048 tokens of one prompt beside 256 single tokens, 32 states of 128 x 128 each: a call takes less than 128 MiB."""
    B, T, H, D = 257, 2304, 32, 128
    q, k, v = _inputs(T, H, H, D, 5)
    i32 = dict(dtype=torch.int32, device=DEV)
    S = torch.zeros(B, H, D, D, device=DEV)
    cu, past = torch.tensor([0, *range(2048, T + 1)], **i32), torch.ones(B, **i32)
    op = LinearAttnPrefillOp(B, T, H, H, D, backend="hip", num_slots=B)
    out = torch.empty(T, H, D, dtype=torch.bfloat16, device=DEV)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    op(q, k, v, _decay(H), cu, S, None, past, max_q_len=2048, out=out)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < 128 << 20


@pytest.mark.parametrize("H,D", [(8, 128), (16, 64)])
def test_shared_query_heads_that_continue(H, D):
    """One kv head's query heads in several blocks (more than a segment of tokens, few blocks), all of which start from
    the stored state that one of them replaces: 65 tokens are the fewest."""
    for lens in ([65], [66, 0, 64, 1], [130]):
        _prefill(lens, [3] * len(lens), H, 1, D, seed=51)
        _prefill(lens, [3 * (i % 2) for i in range(len(lens))], H, 1, D, seed=52, max_q_len=0)


@pytest.mark.parametrize("H,D", [(8, 128), (16, 128), (8, 64), (16, 64)])
def test_shared_query_heads_of_one_segment(H, D):
    """The same without a workspace, which is where past_lens is None: every block starts from zero, one leaves the state;
    and without states."""
    T = 64
    q, k, v = _inputs(T, H, 1, D, 53)
    cu, g = torch.tensor([0, 40, T], dtype=torch.int32, device=DEV), _decay(1)
    for slots in (None, torch.tensor([2, 0], dtype=torch.int32, device=DEV)):
        S = torch.full((3, 1, D, D), float("nan"), device=DEV)
        out = LinearAttnPrefillOp(2, T, H, 1, D, backend="hip", num_slots=3)(q, k, v, g, cu, S, slots, max_q_len=T)
        for b, r in ((0, slice(0, 40)), (1, slice(40, T))):
            o, S1, to, ts = _expect(q[r], k[r], v[r], g, np.zeros((1, D, D)), D ** -0.5)
            _close(n(out[r]), o, to, b)
            _close(n(S[b if slots is None else int(slots[b])]), S1, ts, b)
    _prefill([40, 24], [0, 0], H, 1, D, state=False, seed=54, max_q_len=T)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("mq", [0, 200, 64])
def test_idle_rows_hold_no_slot(D, mq):
    """Sequences without tokens that carry the slot of a later one (a default of 0) do not silence it; those with tokens
    still keep a later one out.  With segments and without."""
    H, Hkv = 4, 2
    lens, slots, past = [0, 65, 0, 40, 200, 3, 0, 5], [0, 0, 1, 1, 2, 2, 3, 3], [2, 1, 0, 0, 4, 4, 9, 9]
    T, B = sum(lens), len(lens)
    cu = np.concatenate([[0], np.cumsum(lens)])
    i32 = dict(dtype=torch.int32, device=DEV)
    q, k, v = _inputs(T, H, Hkv, D, 61)
    S = torch.randn(4, Hkv, D, D, generator=torch.Generator().manual_seed(6)).to(DEV)
    before, out = S.clone(), torch.full((T, H, D), 7.0, dtype=torch.bfloat16, device=DEV)
    LinearAttnPrefillOp(B, T, H, Hkv, D, backend="hip", num_slots=4)(
        q, k, v, _decay(Hkv), torch.tensor(cu, **i32), S, torch.tensor(slots, **i32), torch.tensor(past, **i32), max_q_len=mq,
        out=out)
    for b in (1, 3, 4, 7):
        m = min(lens[b], mq) if mq else lens[b]
        r = slice(int(cu[b]), int(cu[b]) + m)
        S0 = n(before[slots[b]]) if past[b] else np.zeros((Hkv, D, D))
        o, S1, to, ts = _expect(q[r], k[r], v[r], _decay(Hkv), S0, D ** -0.5)
        _close(n(out[r]), o, to, b)
        _close(n(S[slots[b]]), S1, ts, b)
    assert bool((out[cu[5]:cu[6]] == 7).all())


@pytest.mark.parametrize("H,D", [(4, 128), (2, 64)])
def test_overflow_stays_in_its_query_and_sequence(H, D):
    """Finite inputs whose products leave the range (states and powers enter the products in bf16 parts, whose remainder
    of an infinity is NaN): a query that overflows with its keys leaves other queries and the states alone, a state past
    the range other sequences; states of up to 2^126 give the recurrence's outputs."""
    Hkv, lens = 2, [70, 40, 30]
    T, g, i32 = sum(lens), _decay(Hkv), dict(dtype=torch.int32, device=DEV)
    q, k, v = _inputs(T, H, Hkv, D, 71, packed=False)
    q[20], q[75] = 3e38, -3e38  # with keys of the size of 1: past 2^128
    cu, past = [0, 70, 110, 140], torch.tensor([1, 0, 2], **i32)
    S = torch.randn(3, Hkv, D, D, generator=torch.Generator().manual_seed(7)).to(DEV)
    S[2, 1] = 3.4e38  # rounds to infinity in bf16
    before = S.clone()
    out = LinearAttnPrefillOp(3, T, H, Hkv, D, backend="hip", num_slots=3)(q, k, v, g, torch.tensor(cu, **i32), S, None, past)
    for b, bad in ((0, 20), (1, 5)):
        r = slice(cu[b], cu[b + 1])
        x = q[r].clone()
        x[bad] = 0
        o, S1, to, ts = _expect(x, k[r], v[r], g, n(before[b]) if b == 0 else np.zeros((Hkv, D, D)), D ** -0.5)
        keep = np.arange(lens[b]) != bad
        _close(n(out[r])[keep], o[keep], to[keep], b)
        _close(n(S[b]), S1, ts, b)
    r, G = slice(110, 140), H // Hkv  # the head whose state is in range
    o, S1, to, ts = _expect(q[r, :G], k[r, :1], v[r, :1], g[:1], n(before[2, :1]), D ** -0.5)
    _close(n(out[r, :G]), o, to, 2)
    _close(n(S[2, :1]), S1, ts, 2)
    # large, but in range
    S = torch.randn(1, Hkv, D, D, generator=torch.Generator().manual_seed(8)).clamp(-4, 4).to(DEV) * 2.0 ** 124
    x, first = q[:64] * 2.0 ** -20, n(S[0])
    x[20] = 0
    out = LinearAttnPrefillOp(1, 64, H, Hkv, D, backend="hip", num_slots=1)(x, k[:64], v[:64], g, torch.tensor([0, 64], **i32), S,
                                                                        None, past[:1])
    o, S1, to, ts = _expect(x, k[:64], v[:64], g, first, D ** -0.5)
    _close(n(out), o, to, "large")
    _close(n(S[0]), S1, ts, "large")


def test_largest_batch():
    """65536 sequences: a long prompt first (so that all kernels run), then fresh single tokens, one slot held already;
    and 65536 single tokens of the recurrent form."""
    B, D, L = 65536, 64, 300
    T = B - 1 + L
    q, k, v = _inputs(T, 1, 1, D, 81)
    i32, g = dict(dtype=torch.int32, device=DEV), _decay(1)
    cu = torch.cat([torch.zeros(1, **i32), torch.arange(L, T + 1, **i32)])
    slots = torch.arange(B, **i32)
    slots[-1] = 5
    S = torch.full((B, 1, D, D), 7.0, device=DEV)
    out = torch.full((T, 1, D), 7.0, dtype=torch.bfloat16, device=DEV)
    LinearAttnPrefillOp(B, T, 1, 1, D, backend="hip", num_slots=B)(q, k, v, g, cu, S, slots, out=out)
    o, S1, to, ts = _expect(q[:L], k[:L], v[:L], g, np.zeros((1, D, D)), D ** -0.5)
    _close(n(out[:L]), o, to, "long")
    _close(n(S[0]), S1, ts, "long")
    x, y, z = (t[L:-1, 0].double() for t in (q, k, v))
    want, most = (x * y).sum(-1, keepdim=True) * z * D ** -0.5, (x * y).abs().sum(-1, keepdim=True) * z.abs() * D ** -0.5
    assert bool(((out[L:-1, 0].double() - want).abs() <= 2.0 ** -8 * want.abs() * 1.01 + 2.0 ** -14 * most).all())
    assert bool(((S[1:-1, 0] - k[L:-1, 0].float()[:, :, None] * v[L:-1, 0].float()[:, None]).abs() <= 2.0 ** -15 * S[1:-1, 0].abs()).all())
    assert bool((out[-1] == 7).all()) and bool((S[-1] == 7).all())
    start = S.clone()
    q, k, v = (t[L - 1:] for t in (q, k, v))
    got = LinearAttnDecodeOp(B, 1, 1, D, B, backend="hip")(q, k, v, g, S, out=torch.empty_like(out[L - 1:]))
    lam, b = torch.exp(g.double())[0], torch.tensor([0, 1, 77, 40000, B - 1], device=DEV)
    S1 = lam * start[b, 0].double() + k[b, 0].double()[:, :, None] * v[b, 0].double()[:, None]
    aS = lam * start[b, 0].double().abs() + (k[b, 0].double()[:, :, None] * v[b, 0].double()[:, None]).abs()
    assert bool(((S[b, 0].double() - S1).abs() <= 8 * 2.0 ** -24 * aS).all())
    o, ao = ((x[:, :, None] * s).sum(1) * D ** -0.5 for x, s in ((q[b, 0].double(), S1), (q[b, 0].double().abs(), aS)))
    assert bool(((got[b, 0].double() - o).abs() <= 2.0 ** -8 * o.abs() * 1.01 + (D + 24) * 2.0 ** -24 * ao).all())
