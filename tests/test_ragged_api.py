"""The ragged-batch ops on the CPU: registry family, argument checks of the ops and of the C entries (before any device
call), and the torch ``ref`` backends against the 64-bit restatements in ``oracle.ragged``."""

import ctypes

import numpy as np
import pytest
import torch

from ezops import (LinearAttnDecodeOp, LinearAttnPrefillOp, PagedBatchPlanOp, QkNormMropeOp, _hip, get_kernel,
                   list_backends, list_ops, register_kernel)
from ezops.ops.qk_norm_mrope import axis_of_pair
from oracle import ragged

RAGGED = ["linear_attn_decode", "linear_attn_prefill", "paged_batch_plan", "qk_norm_mrope"]


def test_registry_family():
    assert list_ops("ragged") == RAGGED
    assert list_ops(None) == sorted(list_ops() + RAGGED)
    for op in RAGGED:
        assert list_backends(op) == ["hip"] and get_kernel(op, "hip").op_name == op
    with pytest.raises(ValueError, match="family"):
        register_kernel("qk_norm_mrope", "other")(type("K", (), {}))
    assert list_backends("qk_norm_mrope") == ["hip"]


def _raises(text, cls, *args, **kw):
    for backend in ("ref", "hip"):
        with pytest.raises(ValueError, match=text):
            cls(*args, backend=backend, **kw)


def test_constructor_refusals():
    for args, text in [((0, 8, 64, 4, 16), "batch"), ((4097, 8, 64, 4, 16), "batch"), ((1, 0, 64, 4, 16), "num_tokens"),
                       ((1, 1 << 30, 64, 4, 16), "num_tokens"), ((1, 8, 16, 4, 16), "page_size"),
                       ((1, 8, 48, 4, 16), "page_size"), ((1, 8, 64, 0, 16), "max_pages"),
                       ((1, 8, 64, 1 << 25, 16), "max_pages"), ((1, 8, 64, 4, 0), "num_pages"),
                       ((1, 8, 64, 4, 16, -1), "num_free")]:
        _raises(text, PagedBatchPlanOp, *args)
    for args, kw, text in [
            ((0, 4, 2, 64, 16, (32,)), {}, "num_tokens"), ((1, 4, 3, 64, 16, (32,)), {}, "divisible"),
            ((1, 4, 0, 64, 16, (32,)), {}, "divisible"), ((1, 4, 2, 63, 16, (31,)), {}, "head_dim"),
            ((1, 4, 2, 514, 16, (257,)), {}, "head_dim"), ((1, 4, 2, 64, 16, (16, 15)), {}, "sections"),
            ((1, 4, 2, 64, 16, (33, -1)), {}, "sections"), ((1, 4, 2, 64, 16, (8, 8, 8, 4, 4)), {}, "sections"),
            ((1, 4, 2, 64, 16, ()), {}, "sections"), ((1, 4, 2, 64, 16, (8, 12, 12)), dict(interleaved=True), "interleaved"),
            ((1, 4, 2, 64, 16, (32,)), dict(page_size=64), "go together"),
            ((1, 4, 2, 64, 16, (32,)), dict(page_size=48, num_pages=4), "page_size"),
            ((1, 4, 2, 64, 16, (32,)), dict(page_size=64, num_pages=0), "num_pages")]:
        _raises(text, QkNormMropeOp, *args, **kw)
    for args, kw, text in [((0, 8, 4, 2, 64), {}, "batch"), ((1, 0, 4, 2, 64), {}, "num_tokens"),
                           ((1, 8, 4, 3, 64), {}, "divisible"), ((1, 8, 6, 2, 64), {}, "group size"),
                           ((1, 8, 4, 2, 96), {}, "head_dim"), ((1, 8, 4, 2, 64), dict(num_slots=0), "num_slots"),
                           ((1, 8, 4, 2, 64), dict(scale=0.0), "scale"),
                           ((1, 8, 4, 2, 64), dict(scale=float("nan")), "scale")]:
        _raises(text, LinearAttnPrefillOp, *args, **kw)
    for args, text in [((0, 4, 2, 64, 8), "batch"), ((1, 32, 1, 64, 8), "group size"), ((1, 4, 2, 80, 8), "head_dim"),
                       ((1, 4, 2, 64, 0), "num_slots")]:
        _raises(text, LinearAttnDecodeOp, *args)


def test_c_entries_reject_bad_arguments():
    """Before any device call: the dummy addresses are never touched."""
    lib, d, e = _hip.lib(), 4096, 8192
    err = lib.ezops_hip_last_error

    def plan(B=2, T=8, P=64, M=4, NP=16, NF=16, span=d, out=e, q=d, free=d):
        return lib.ezops_paged_batch_plan(q, None, d, free, span, d, d, d, d, out, B, T, P, M, NP, NF, None)

    for kw, text in [(dict(q=None), b"null"), (dict(free=None), b"free_pages"), (dict(out=d), b"free_span_out"),
                     (dict(B=0), b"batch"), (dict(B=4097), b"batch"), (dict(T=0), b"rows"), (dict(T=1 << 30), b"rows"),
                     (dict(P=16), b"page_size"), (dict(P=96), b"page_size"), (dict(M=0), b"max_pages"),
                     (dict(M=1 << 25), b"max_pages"), (dict(NP=0), b"num_pages"), (dict(NF=-1), b"num_free")]:
        assert plan(**kw) == _hip.EINVAL and text in err(), (kw, err())

    def mrope(T=4, H=4, Hkv=2, D=64, S=16, sec=(12, 10, 10), inter=0, P=64, NP=4, qs=256, ks=128, vs=128, q=d, v=d, K=d,
              V=d, slots=d, k_out=None):
        s = (ctypes.c_int64 * len(sec))(*sec)
        return lib.ezops_qk_norm_mrope_bf16(q, qs, d, ks, v, vs, None, None, 1, d, d, 0, d, len(sec), s, inter, slots, K, V,
                                            NP, P, d, k_out, T, H, Hkv, D, S, 1e-6, None)

    for kw, text in [(dict(q=None), b"null"), (dict(T=0), b"tokens"), (dict(S=0), b"table rows"), (dict(Hkv=3), b"divisible"),
                     (dict(Hkv=0), b"divisible"), (dict(D=63), b"head_dim"), (dict(D=514), b"head_dim"),
                     (dict(qs=255), b"strides"), (dict(ks=100), b"strides"), (dict(vs=100), b"strides"),
                     (dict(sec=(12, 10)), b"add up"), (dict(sec=(42, -10)), b"sections"),
                     (dict(sec=(10, 11, 11), inter=1), b"turns"), (dict(sec=(8, 8, 8, 4, 4)), b"axes"),
                     (dict(V=None), b"go together"), (dict(v=None), b"slot_mapping"), (dict(slots=None), b"slot_mapping"),
                     (dict(P=48), b"page_size"), (dict(NP=0), b"page_size"), (dict(K=None, V=None), b"k_out")]:
        assert mrope(**kw) == _hip.EINVAL and text in err(), (kw, err())

    def prefill(B=2, T=64, H=4, Hkv=2, D=64, q=d, qs=256, ks=128, cu=d, state=d, slots=8, mq=0, out=d, ws=None, nb=0):
        return lib.ezops_linear_attn_prefill_bf16(q, qs, d, ks, d, 128, d, cu, None, state, None, slots, out, B, T, H, Hkv, D,
                                                  mq, 0.0, ws, nb, None)

    for kw, text in [(dict(q=None), b"null"), (dict(cu=None), b"null"), (dict(B=0), b"batch"), (dict(T=0), b"tokens"),
                     (dict(H=6, qs=384), b"group size"), (dict(Hkv=3), b"divisible"), (dict(D=96, qs=384, ks=192), b"head_dim"),
                     (dict(qs=252), b"strides"), (dict(qs=260), b"16-byte"), (dict(q=d + 2), b"16-byte"),
                     (dict(state=d + 4), b"16-byte"), (dict(out=d + 8), b"16-byte"), (dict(slots=0), b"num_slots"),
                     (dict(mq=-1), b"max_q_len")]:
        assert prefill(**kw) == _hip.EINVAL and text in err(), (kw, err())

    def decode(B=2, H=4, Hkv=2, D=64, q=d, qs=256, state=d, slots=8):
        return lib.ezops_linear_attn_decode_bf16(q, qs, d, 128, d, 128, d, state, None, slots, d, B, H, Hkv, D, 0.0, None)

    for kw, text in [(dict(state=None), b"null"), (dict(q=None), b"null"), (dict(B=0), b"batch"), (dict(H=6, qs=384), b"group"),
                     (dict(D=32), b"head_dim"), (dict(q=d + 2), b"16-byte"), (dict(slots=0), b"num_slots")]:
        assert decode(**kw) == _hip.EINVAL and text in err(), (kw, err())


def test_prefill_workspace_is_checked_before_any_launch():
    lib, d = _hip.lib(), 4096
    need = lib.ezops_linear_attn_prefill_workspace_size(1, 1 << 16, 8, 8, 128, 0)
    if need == 0:
        pytest.skip("this shape needs no workspace")
    args = [d, 1024, d, 1024, d, 1024, d, d, None, None, None, 0, d, 1, 1 << 16, 8, 8, 128, 0, 0.0]
    for ws, n in ((None, need), (d, need - 1), (d + 4, need)):
        assert lib.ezops_linear_attn_prefill_bf16(*args, ws, n, None) == _hip.EINVAL
        assert b"workspace" in lib.ezops_hip_last_error()


def test_c_entries_reject_overlaps():
    """An output in an input's place, wholly or by an element, where another block may still read it."""
    lib, err = _hip.lib(), _hip.lib().ezops_hip_last_error
    at = lambda i: (i + 1) << 24  # noqa: E731  addresses far apart, never touched
    B, T = 2, 8
    good = [at(i) for i in range(10)]  # q_lens past table free span | cu kv positions slots span_out

    def plan(p):
        return lib.ezops_paged_batch_plan(*p, B, T, 64, 4, 16, 16, None)

    for i, j, off in [(6, 1, 0), (6, 0, 4), (5, 0, 4), (9, 4, 0), (9, 4, 4), (7, 3, 60), (2, 0, 4), (8, 1, -60)]:
        p = list(good)
        p[i] = p[j] + off
        assert plan(p) == _hip.EINVAL and (b"overlaps" in err() or b"free_span_out" in err()), (i, j, off, err())

    sec = (ctypes.c_int64 * 1)(32)

    def mrope(q=at(0), qs=256, k=at(1), ks=128, v=at(2), q_out=at(3), k_out=None):
        return lib.ezops_qk_norm_mrope_bf16(q, qs, k, ks, v, 128, None, None, 1, at(5), at(5), 0, at(6), 1, sec, 0, at(7),
                                            at(8), at(9), 4, 64, q_out, k_out, 4, 4, 2, 64, 16, 1e-6, None)

    for kw in (dict(q_out=at(0) + 16), dict(q_out=at(0), qs=512), dict(q_out=at(1)), dict(q_out=at(2) + 64),
               dict(k_out=at(0)), dict(k_out=at(1) - 16), dict(k_out=at(2)), dict(k_out=at(3) + 256),
               dict(k_out=at(1), ks=256)):
        assert mrope(**kw) == _hip.EINVAL and b"overlap" in err(), (kw, err())
    for out in (at(0), at(1) + 128, at(2) - 16):
        rc = lib.ezops_linear_attn_prefill_bf16(at(0), 256, at(1), 128, at(2), 128, at(3), at(4), None, None, None, 0, out, 1,
                                                8, 4, 2, 64, 0, 0.0, None, 0, None)
        assert rc == _hip.EINVAL and b"overlap" in err(), err()
        rc = lib.ezops_linear_attn_decode_bf16(at(0), 256, at(1), 128, at(2), 128, at(3), at(5), None, 8, out, 2, 4, 2, 64,
                                               0.0, None)
        assert rc == _hip.EINVAL and b"overlap" in err(), err()


def test_c_entries_reject_overlaps_of_caches_states_and_outputs():
    lib, err = _hip.lib(), _hip.lib().ezops_hip_last_error
    at = lambda i: (i + 1) << 24  # noqa: E731  addresses far apart, never touched
    good = [at(i) for i in range(10)]  # q_lens past table free span | cu kv positions slots span_out
    for i, j, off in [(5, 6, 0), (6, 5, 8), (7, 8, 60), (9, 5, 8), (2, 7, -124), (8, 2, 124)]:
        p = list(good)
        p[i] = p[j] + off
        rc = lib.ezops_paged_batch_plan(*p, 2, 8, 64, 16, 16, 16, None)
        assert rc == _hip.EINVAL and b"two outputs overlap" in err(), (i, j, off, err())

    sec = (ctypes.c_int64 * 1)(32)
    pool = 4 * 2 * 64 * 64 * 2
    for kc, vc in [(at(0), at(9)), (at(1) - pool + 2, at(9)), (at(8), at(2) + 16), (at(8), at(3)), (at(4) + 64, at(9)),
                   (at(8), at(8)), (at(8), at(8) + pool - 16)]:
        rc = lib.ezops_qk_norm_mrope_bf16(at(0), 256, at(1), 128, at(2), 128, None, None, 1, at(5), at(5), 0, at(6), 1, sec,
                                          0, at(7), kc, vc, 4, 64, at(3), at(4), 4, 4, 2, 64, 16, 1e-6, None)
        assert rc == _hip.EINVAL and b"overlap" in err(), (kc, vc, err())

    states = 8 * 2 * 64 * 64 * 4
    for state in (at(0), at(1) + 1024, at(2) - states + 16, at(6)):
        rc = lib.ezops_linear_attn_prefill_bf16(at(0), 256, at(1), 128, at(2), 128, at(3), at(4), None, state, None, 8, at(6),
                                                1, 8, 4, 2, 64, 0, 0.0, None, 0, None)
        assert rc == _hip.EINVAL and b"state must not overlap" in err(), err()
        rc = lib.ezops_linear_attn_decode_bf16(at(0), 256, at(1), 128, at(2), 128, at(3), state, None, 8, at(6), 8, 4, 2, 64,
                                               0.0, None)
        assert rc == _hip.EINVAL and b"state must not overlap" in err(), err()


def test_c_entries_reject_launches_past_the_grid():
    """65536 sequences of 256 heads would take 2^32 threads along one axis."""
    lib, err = _hip.lib(), _hip.lib().ezops_hip_last_error
    at = lambda i: (i + 1) << 40  # noqa: E731  addresses far apart, never touched
    rs = 256 * 64
    rc = lib.ezops_linear_attn_decode_bf16(at(0), rs, at(1), rs, at(2), rs, at(3), at(5), None, 8, at(6), 65536, 256, 256, 64,
                                           0.0, None)
    assert rc == _hip.EINVAL and b"one launch" in err(), err()
    need = lib.ezops_linear_attn_prefill_workspace_size(65536, 65536, 256, 256, 64, 64)
    rc = lib.ezops_linear_attn_prefill_bf16(at(0), rs, at(1), rs, at(2), rs, at(3), at(4), None, None, None, 0, at(6), 65536,
                                            65536, 256, 256, 64, 64, 0.0, at(7), need, None)
    assert rc == _hip.EINVAL and b"one launch" in err(), err()


def test_calls_make_the_tensors_device_current(monkeypatch):
    """``call_on`` with another device current: the call runs inside a switch to the tensors' device, on its stream."""
    seen, current = [], [1]

    class Switch:
        def __init__(self, device):
            self.to = device.index

        def __enter__(self):
            current[0], self.back = self.to, current[0]

        def __exit__(self, *exc):
            current[0] = self.back

    monkeypatch.setattr(torch.cuda, "device", Switch)
    monkeypatch.setattr(_hip, "_current_device", lambda: current[0])
    monkeypatch.setattr(_hip, "_raw_stream", lambda index: 100 + index)
    monkeypatch.setattr(_hip, "_entries", (None, {}))
    monkeypatch.setattr(_hip, "_fn", lambda name: lambda *a: seen.append((name, a, current[0])) or 0)
    _hip.call_on(torch.device("cuda", 0), "f", 7)
    _hip.call_on(torch.device("cuda", 1), "g")
    assert seen == [("f", (7, 100), 0), ("g", (101,), 1)] and current == [1]
    monkeypatch.setattr(_hip, "_fn", lambda name: lambda *a: -22)
    for index in (0, 1):
        with pytest.raises(RuntimeError, match="h failed"):
            _hip.call_on(torch.device("cuda", index), "h")
    assert current == [1]


def _np(t):
    return t.detach().double().numpy()


@pytest.mark.parametrize("q,past,T,P,M,NP,head,tail", [
    ([3, 0, 70, 1], [0, 5, 63, 64], 80, 32, 8, 20, 0, 20),   # empty sequence, a page that ends exactly, padded rows
    ([40, 40], [0, 0], 64, 32, 8, 10, 2, 9),                 # more tokens than rows: the second is cut off
    ([100, 1], [0, 0], 128, 32, 2, 10, 0, 9),                # past the table's width
    ([100, 9], [3, 0], 128, 32, 8, 10, 1, 3),                # the free list ends
    ([5, 5], [-4, 31], 10, 32, 1, 4, 0, 4),                  # negative length, a single page
    ([5], [0], 16, 32, 1, 4, -1, 4),                         # bad span
])
def test_ref_plan(q, past, T, P, M, NP, head, tail):
    g = torch.Generator().manual_seed(1)
    B = len(q)
    table = torch.randint(-2, NP + 2, (B, M), generator=g, dtype=torch.int32)
    free = torch.randint(-1, NP + 1, (9,), generator=g, dtype=torch.int32)
    op = PagedBatchPlanOp(B, T, P, M, NP, 9)
    want = ragged.batch_plan(q, past, table.numpy(), free.numpy(), [head, tail], T, P, NP)
    i32 = dict(dtype=torch.int32)
    got = op(torch.tensor(q, **i32), torch.tensor(past, **i32), table, free, torch.tensor([head, tail], **i32))
    for g_, w in zip((table, *got), want):
        np.testing.assert_array_equal(g_.numpy(), w)


def test_plan_gen_data_is_a_whole_plan():
    for B, T, P, M, NP in ((1, 5, 32, 4, 9), (7, 300, 32, 12, 50), (64, 64, 64, 16, 700)):
        torch.manual_seed(B)
        op = PagedBatchPlanOp(B, T, P, M, NP)
        data = op.gen_data("cpu")
        p = op(*data)
        head, tail, needed = p.free_span.tolist()
        assert head == needed <= tail
        live = p.positions >= 0
        assert int(live.sum()) == int(data[0].sum()) and bool((p.slot_mapping[live] >= 0).all())
        assert p.slot_mapping[live].unique().numel() == int(live.sum())


def test_axis_of_pair():
    assert axis_of_pair(8, (2, 3, 3), False) == [0, 0, 1, 1, 1, 2, 2, 2]
    assert axis_of_pair(8, (4, 2, 2), True) == [0, 1, 2, 0, 1, 2, 0, 0]
    for half, sec in ((64, (24, 20, 20)), (32, (30, 1, 1)), (40, (20, 20)), (64, (64,)), (64, (16, 16, 16, 16))):
        for inter in (False, True):
            axes = axis_of_pair(half, sec, inter)
            assert axes == ragged.pair_axes(half, sec, inter)
            assert [axes.count(a) for a in range(len(sec))] == list(sec)


@pytest.mark.parametrize("D,sec,inter,norm,page", [(128, (24, 20, 20), True, True, 32), (80, (20, 20), False, False, None),
                                                   (64, (32,), False, True, 64), (6, (1, 0, 2), False, True, None)])
def test_ref_mrope(D, sec, inter, norm, page):
    torch.manual_seed(2)
    op = QkNormMropeOp(9, 4, 2, D, 50, sec, interleaved=inter, norm=norm, page_size=page, num_pages=2 if page else None)
    data = list(op.gen_data("cpu"))
    data[7][0, 3] = -1
    data[7][-1, 5] = 50
    if page:
        data[10][1] = 2 * page
        before = data[8].clone()
    q_out, k_out = op(*data)
    axes = dict(sections=sec, interleaved=inter, norm=norm)
    for x, w, got in ((data[0], data[3], q_out), (data[1], data[4], k_out)):
        want = ragged.qk_norm_mrope(_np(x), None if w is None else _np(w), _np(data[5]), _np(data[6]), data[7].numpy(), **axes)
        live = ~np.isnan(want[:, 0, 0])
        assert list(np.where(~live)[0]) == [3, 5]
        if got is not None:
            np.testing.assert_allclose(_np(got)[live], want[live], rtol=2 ** -8, atol=1e-5)
    if page:
        for t in (0, 2, 4, 6, 7, 8):
            s = int(data[10][t])
            np.testing.assert_allclose(_np(data[8])[s // page, :, s % page], want[t], rtol=2 ** -8, atol=1e-5)
            assert torch.equal(data[9][s // page, :, s % page], data[2][t])
        for t in (3, 5):  # bad positions write nothing
            s = int(data[10][t])
            assert torch.equal(data[8][s // page, :, s % page], before[s // page, :, s % page])


def test_ref_linear_attn():
    """Prefill against the recurrence in 64 bits, and the same tokens one by one through the decode op."""
    torch.manual_seed(3)
    B, T, H, Hkv, D = 4, 24, 4, 2, 64
    op = LinearAttnPrefillOp(B, T, H, Hkv, D, num_slots=5)
    q, k, v, g, _, state = op.gen_data("cpu")
    cu = torch.tensor([0, 7, 7, 17, 20], dtype=torch.int32)
    slots = torch.tensor([3, 0, 3, 4], dtype=torch.int32)  # the third holds the first's slot: left out
    past = torch.tensor([0, 2, 5, 9], dtype=torch.int32)
    first = state.clone()
    out = torch.full((T, H, D), 7.0, dtype=torch.bfloat16)
    op(q, k, v, g, cu, state, slots, past, out=out)
    lam = np.exp(_np(g))
    step_state = first.clone()
    for b, n in ((0, 7), (3, 3)):
        t = int(cu[b])
        S0 = _np(first[slots[b]]) if past[b] > 0 else np.zeros((Hkv, D, D))
        want, S = ragged.linear_attn(_np(q[t:t + n]), _np(k[t:t + n]), _np(v[t:t + n]), lam, S0, D ** -0.5)
        np.testing.assert_allclose(_np(out[t:t + n]), want, rtol=2 ** -8, atol=1e-4)
        np.testing.assert_allclose(_np(state[slots[b]]), S, rtol=1e-5, atol=1e-5)
        one = LinearAttnDecodeOp(1, H, Hkv, D, 5)
        if not past[b]:
            step_state[slots[b]] = 0
        for i in range(t, t + n):
            o = one(q[i:i + 1], k[i:i + 1], v[i:i + 1], g, step_state, slots[b:b + 1])
            assert torch.allclose(o[0].float(), out[i].float(), rtol=2 ** -7, atol=1e-4)
        assert torch.allclose(step_state[slots[b]], state[slots[b]], rtol=1e-5, atol=1e-5)
    for s in (0, 1, 2):
        assert torch.equal(state[s], first[s])
    assert bool((out[7:17] == 7).all()) and bool((out[20:] == 7).all())


def test_rooflines():
    assert QkNormMropeOp(10, 4, 2, 64, 100, (32,)).get_roofline().bytes == 2 * 10 * 12 * 64 + 40 + 2 * 10 * 64
    assert LinearAttnDecodeOp(3, 4, 2, 64, 8).get_roofline().bytes == 3 * (8 * 2 * 64 * 64 + 4 * 6 * 64 + 4)
    assert PagedBatchPlanOp(3, 10, 64, 4, 8).get_roofline().flops == 0
    assert LinearAttnPrefillOp(1, 10, 4, 2, 64).get_roofline().flops == 10 * (6 + 8) * 64 * 64


def test_ref_idle_rows_hold_no_slot():
    """Sequences without tokens that carry the slot of a later one (a default of 0) do not silence it."""
    torch.manual_seed(4)
    H, Hkv, D = 2, 1, 64
    op = LinearAttnPrefillOp(5, 9, H, Hkv, D, num_slots=2)
    q, k, v, g, _, state = op.gen_data("cpu")
    i32 = dict(dtype=torch.int32)
    cu, slots, past = torch.tensor([0, 0, 4, 4, 7, 9], **i32), torch.tensor([0, 0, 1, 1, 0], **i32), torch.tensor([3, 2, 0, 0, 1], **i32)
    first = state.clone()
    out = torch.full((9, H, D), 7.0, dtype=torch.bfloat16)
    op(q, k, v, g, cu, state, slots, past, out=out)
    lam = np.exp(_np(g))
    for b, r, S0 in ((1, slice(0, 4), _np(first[0])), (3, slice(4, 7), np.zeros((Hkv, D, D)))):
        want, S = ragged.linear_attn(_np(q[r]), _np(k[r]), _np(v[r]), lam, S0, D ** -0.5)
        np.testing.assert_allclose(_np(out[r]), want, rtol=2 ** -8, atol=1e-4)
        np.testing.assert_allclose(_np(state[slots[b]]), S, rtol=1e-5, atol=1e-5)
    assert bool((out[7:] == 7).all())  # the last one's slot is held by one with tokens


def test_scales_that_fp32_does_not_hold_are_refused():
    """The kernels take the scale in fp32, where 0 selects the default: one that rounds to 0 or to infinity is no scale."""
    for scale in (1e-50, 1e39, float("inf"), -1.0):
        for args in ((LinearAttnPrefillOp, 1, 8, 4, 2, 64), (LinearAttnDecodeOp, 1, 4, 2, 64, 3)):
            for backend in ("ref", "hip"):
                with pytest.raises(ValueError, match="scale"):
                    args[0](*args[1:], backend=backend, scale=scale)
    lib, err = _hip.lib(), _hip.lib().ezops_hip_last_error
    at = lambda i: (i + 1) << 24  # noqa: E731  addresses far apart, never touched
    for scale in (float("nan"), float("inf")):
        rc = lib.ezops_linear_attn_prefill_bf16(at(0), 256, at(1), 128, at(2), 128, at(3), at(4), None, None, None, 0, at(6), 1,
                                                8, 4, 2, 64, 0, scale, None, 0, None)
        assert rc == _hip.EINVAL and b"scale" in err(), err()
        rc = lib.ezops_linear_attn_decode_bf16(at(0), 256, at(1), 128, at(2), 128, at(3), at(5), None, 8, at(6), 2, 4, 2, 64,
                                               scale, None)
        assert rc == _hip.EINVAL and b"scale" in err(), err()


def test_c_entries_reject_outputs_over_small_inputs():
    """Tables, positions, slots, weights, offsets and decays are read by blocks that run after others have written."""
    lib, err = _hip.lib(), _hip.lib().ezops_hip_last_error
    at = lambda i: (i + 1) << 24  # noqa: E731  addresses far apart, never touched
    sec = (ctypes.c_int64 * 2)(20, 12)
    T, H, Hkv, D, S = 4, 4, 2, 64, 16
    pool = 4 * 2 * 64 * 64 * 2
    good = dict(qw=at(10), kw=at(11), cos=at(5), sin=at(12), pos=at(6), slots=at(7), K=at(8), V=at(9), q_out=at(3), k_out=at(4))

    def mrope(f32=0, **kw):
        a = {**good, **kw}
        return lib.ezops_qk_norm_mrope_bf16(at(0), 256, at(1), 128, at(2), 128, a["qw"], a["kw"], 1, a["cos"], a["sin"], f32,
                                            a["pos"], 2, sec, 0, a["slots"], a["K"], a["V"], 4, 64, a["q_out"], a["k_out"], T,
                                            H, Hkv, D, S, 1e-6, None)

    size = dict(qw=2 * D, kw=2 * D, cos=2 * S * D, sin=2 * S * D, pos=2 * 4 * T, slots=8 * T)
    for out, n in (("q_out", T * H * D * 2), ("k_out", T * Hkv * D * 2), ("K", pool), ("V", pool)):
        for x, m in size.items():
            for off in (0, m - 2, 2 - n):  # its start, its last element, the output's last element on its first
                assert mrope(**{out: good[x] + off}) == _hip.EINVAL and b"overlap" in err(), (out, x, off, err())
    assert mrope(f32=1, q_out=at(5) + 4 * S * D - 4) == _hip.EINVAL and b"overlap" in err(), err()

    B, T, states = 2, 200, 8 * 2 * 64 * 64 * 4
    need = lib.ezops_linear_attn_prefill_workspace_size(B, T, 4, 2, 64, 0)
    assert need > 0
    rows = dict(g=4 * 2, cu=4 * (B + 1), past=4 * B, slots=4 * B)
    base = dict(g=at(3), cu=at(4), past=at(5), slots=at(6), state=at(7), out=at(9), ws=at(10))

    def prefill(**kw):
        a = {**base, **kw}
        return lib.ezops_linear_attn_prefill_bf16(at(0), 256, at(1), 128, at(2), 128, a["g"], a["cu"], a["past"], a["state"],
                                                  a["slots"], 8, a["out"], B, T, 4, 2, 64, 0, 0.0, a["ws"], need, None)

    def decode(**kw):
        a = {**base, **kw}
        return lib.ezops_linear_attn_decode_bf16(at(0), 256, at(1), 128, at(2), 128, a["g"], a["state"], a["slots"], 8,
                                                 a["out"], B, 4, 2, 64, 0.0, None)

    for x, m in rows.items():
        for out, n in (("out", T * 4 * 64 * 2), ("state", states), ("ws", need)):
            for addr in (base[x] & ~15, base[x] - n + 16):
                assert prefill(**{out: addr}) == _hip.EINVAL and b"overlap" in err(), (out, x, err())
        if x in ("g", "slots"):
            for out in ("out", "state"):
                assert decode(**{out: base[x]}) == _hip.EINVAL and b"overlap" in err(), (out, x, err())
    for x, n in ((at(0), 256 * 2 * T), (at(1), 128 * 2 * T), (at(2), 128 * 2 * T), (at(7), states), (at(9), 4 * 64 * 2 * T)):
        for addr in (x, x + n - 16, x - need + 16):
            assert prefill(ws=addr) == _hip.EINVAL and b"overlap" in err(), (x, err())


def test_ref_mrope_repeated_frequencies():
    """A vision encoder's rotation, the same frequencies for rows and for columns, with the table that the op's docstring
    gives: pair i of the section of either axis turns by position * f[i]."""
    torch.manual_seed(6)
    T, H, D, S, n = 12, 2, 72, 30, 18
    f = 1e4 ** (-torch.arange(n, dtype=torch.float64) / n)
    angles = torch.arange(S)[:, None] * f.repeat(2)  # sections (18, 18): each begins with f[0] again
    cos, sin = (x.repeat(1, 2).float() for x in (angles.cos(), angles.sin()))
    op = QkNormMropeOp(T, H, H, D, S, (n, n), norm=False)
    q, k = (torch.randn(T, H, D).to(torch.bfloat16) for _ in range(2))
    pos = torch.stack([torch.arange(T) // 4 * 7, torch.arange(T) % 4 + 3]).to(torch.int32)
    got, _ = op(q, k, None, None, None, cos, sin, pos)
    turn = torch.cat([pos[0, :, None] * f, pos[1, :, None] * f], 1)[:, None]
    a, b = q.double()[..., :D // 2], q.double()[..., D // 2:]
    want = torch.cat([a * turn.cos() - b * turn.sin(), b * turn.cos() + a * turn.sin()], -1)
    np.testing.assert_allclose(_np(got), want.numpy(), rtol=2 ** -8, atol=1e-5)
