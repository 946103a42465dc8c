"""HIP QK norm + multi-axis rotation + slot write against the 64-bit restatement.

Tolerance, element by element: one bf16 rounding is at most 2^-8 of the value; before it, the fp32 pipeline has the sum of
squares (at most 16 products a lane and 6 additions across lanes: 2^-24 each, halved by the root), rsqrt, two products of
the norm, two of the rotation and a sum: under 32 steps of 2^-24 on |y1 c| + |y2 s| <= sqrt(y1^2 + y2^2) * sqrt(2).
"""

import numpy as np
import pytest
import torch

from ezops import FusedQkNormRopeOp, QkNormMropeOp
from oracle import ragged

pytestmark = pytest.mark.gpu
DEV = "cuda"


def n(x):
    return None if x is None else x.detach().double().cpu().numpy()


def _close(got, want, x, w, norm):
    """got bf16, want 64-bit; x the input heads (for the amplitude of the pairs)."""
    y = x
    if norm:
        y = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + 1e-6) * (1 if w is None else w)
    half = x.shape[-1] // 2
    amp = np.sqrt(y[..., :half] ** 2 + y[..., half:] ** 2)
    tol = 2.0 ** -8 * np.abs(want) * (1 + 2.0 ** -8) + 2.0 ** -19 * 1.5 * np.concatenate([amp, amp], -1) + 1e-38
    bad = np.abs(got - want) > tol
    assert not bad.any(), (int(bad.sum()), np.abs(got - want)[bad].max())


def _data(op, seed, packed=False, table=torch.bfloat16):
    torch.manual_seed(seed)
    d = list(op.gen_data(DEV))
    T, H, Hkv, D = op.num_tokens, op.num_heads, op.num_kv_heads, op.head_dim
    if packed:
        x = torch.cat(d[:3], 1).contiguous()
        d[:3] = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
    if table is torch.float32:
        inv = op.rope_theta ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
        ang = torch.arange(op.max_position, dtype=torch.float64)[:, None] * inv
        d[5], d[6] = ang.cos().repeat(1, 2).float().to(DEV), ang.sin().repeat(1, 2).float().to(DEV)
    return d


def _run(op, d, q_out=None, k_out=None):
    """One call and its check: rotated q and k, v and k in their slots, everything else as it was."""
    K0, V0 = (n(d[8]), n(d[9])) if op.page_size else (None, None)
    q, k, v, qw, kw, cos, sin = (n(x) for x in d[:7])
    q0, k0 = n(q_out), n(k_out)
    got_q, got_k = op(*d, q_out=q_out, k_out=k_out)
    ax = dict(sections=op.sections, interleaved=op.interleaved, norm=op.norm)
    pos = d[7].cpu().numpy()
    want_q = ragged.qk_norm_mrope(q, qw, cos, sin, pos, **ax)
    want_k = ragged.qk_norm_mrope(k, kw, cos, sin, pos, **ax)
    live = ~np.isnan(want_q[:, 0, 0])
    _close(n(got_q)[live], want_q[live], q[live], qw, op.norm)
    if q0 is not None:
        np.testing.assert_array_equal(n(got_q)[~live], q0[~live])
    if got_k is not None:
        _close(n(got_k)[live], want_k[live], k[live], kw, op.norm)
        if k0 is not None:
            np.testing.assert_array_equal(n(got_k)[~live], k0[~live])
    if op.page_size:
        P, slots = op.page_size, d[10].cpu().numpy()
        K, V = n(d[8]), n(d[9])
        ok = live & (slots >= 0) & (slots < op.num_pages * P)
        pg, row = slots[ok] // P, slots[ok] % P
        _close(K[pg, :, row], want_k[ok], k[ok], kw, op.norm)
        np.testing.assert_array_equal(V[pg, :, row], v[ok])
        K[pg, :, row], V[pg, :, row] = K0[pg, :, row], V0[pg, :, row]
        np.testing.assert_array_equal(K, K0)
        np.testing.assert_array_equal(V, V0)
    return got_q, got_k


@pytest.mark.parametrize("T,H,Hkv,D,sec,inter,norm,page,table,packed", [
    (1, 32, 8, 128, (24, 20, 20), True, True, 64, torch.bfloat16, True),
    (17, 16, 8, 128, (16, 24, 24), False, True, 32, torch.bfloat16, False),
    (67, 32, 8, 128, (24, 20, 20), True, True, None, torch.float32, True),
    (300, 16, 16, 80, (20, 20), False, False, None, torch.float32, True),
    (33, 4, 4, 96, (16, 16, 16), True, True, 256, torch.bfloat16, True),
    (5, 3, 1, 64, (32,), False, True, 32, torch.float32, False),
    (9, 8, 1, 256, (32, 32, 32, 32), True, True, 32, torch.bfloat16, True),
    (9, 8, 2, 256, (0, 100, 28, 0), False, False, 64, torch.bfloat16, False),
    (11, 2, 2, 72, (12, 12, 12), True, True, None, torch.bfloat16, True),   # pairs in no multiple of 8
    (7, 2, 1, 6, (1, 0, 2), False, True, 32, torch.bfloat16, True),
    (3, 4, 2, 512, (128, 64, 64), False, True, 32, torch.float32, True),
    (5, 6, 2, 16, (8,), False, True, 32, torch.bfloat16, True),
    (5, 5, 5, 32, (6, 5, 5), True, True, 32, torch.bfloat16, False),
    (130, 64, 8, 128, (64,), False, True, 32, torch.bfloat16, True),
    (21, 4, 2, 2, (1,), False, True, 32, torch.bfloat16, True),
    (4100, 16, 8, 128, (24, 20, 20), True, True, 128, torch.bfloat16, True),
])
def test_against_64_bits(T, H, Hkv, D, sec, inter, norm, page, table, packed):
    pages = -(-T // page) + 2 if page else None
    op = QkNormMropeOp(T, H, Hkv, D, 97, sec, backend="hip", interleaved=inter, norm=norm, page_size=page, num_pages=pages)
    d = _data(op, T, packed, table)
    if T > 4:  # bad positions on any axis, the ends of the table, slots outside the pool
        d[7][0, 1], d[7][-1, 2], d[7][:, 0], d[7][:, 3] = -1, 97, 0, 96
        if page:
            d[10][0], d[10][4] = -1, pages * page
    q_out = torch.full((T, H, D), 7.0, dtype=torch.bfloat16, device=DEV)
    k_out = torch.full((T, Hkv, D), 5.0, dtype=torch.bfloat16, device=DEV) if T % 2 else None
    a = _run(op, d, q_out, k_out)
    b = op(*d)  # fresh outputs: the same bits where something is written
    live = (d[7] >= 0).all(0) & (d[7] < 97).all(0)
    assert torch.equal(a[0][live], b[0][live])


@pytest.mark.parametrize("T,H,Hkv,D,sec,page,table", [
    # bytes of the heads read and written: 8, 32 and 64 MB change how they are accessed, T * heads the heads a group
    (511, 16, 8, 128, (24, 20, 20), 64, torch.bfloat16),    # 7.98 MB
    (513, 16, 8, 128, (24, 20, 20), 64, torch.bfloat16),    # 8.02 MB
    (2047, 16, 8, 128, (24, 20, 20), 32, torch.bfloat16),   # one head a group, then four
    (2051, 15, 5, 128, (64,), None, torch.float32),
    (1025, 8, 4, 256, (64, 32, 32), 64, torch.bfloat16),
    (819, 16, 16, 80, (20, 20), None, torch.float32),       # 7.998 MB
    (821, 16, 16, 80, (20, 20), None, torch.float32),
    (2049, 16, 16, 80, (20, 20), None, torch.bfloat16),
    (3277, 16, 16, 80, (20, 20), None, torch.float32),      # 32.002 MB
    (3001, 32, 8, 64, (16, 8, 8), 64, torch.bfloat16),
    (5500, 32, 8, 64, (32,), 64, torch.bfloat16),           # 64.5 MB
    (2741, 16, 16, 48, (8, 8, 8), 32, torch.bfloat16),
    (901, 16, 4, 144, (24, 24, 24), 32, torch.bfloat16),
    (1301, 8, 4, 272, (136,), 32, torch.bfloat16),
])
def test_large_against_64_bits(T, H, Hkv, D, sec, page, table):
    pages = -(-T // page) + 1 if page else None
    op = QkNormMropeOp(T, H, Hkv, D, 211, sec, backend="hip", interleaved=len(sec) > 1, page_size=page, num_pages=pages)
    d = _data(op, T, True, table)
    d[7][0, T // 2], d[7][-1, T - 2] = -1, 211
    q_out = torch.full((T, H, D), 7.0, dtype=torch.bfloat16, device=DEV)
    k_out = torch.full((T, Hkv, D), 5.0, dtype=torch.bfloat16, device=DEV)
    _run(op, d, q_out, k_out)


def test_unit_weights_and_extremes():
    """No weights = unit; zeros, the largest and the smallest values, infinities and NaN stay in their own head."""
    T, H, Hkv, D = 6, 4, 2, 128
    op = QkNormMropeOp(T, H, Hkv, D, 50, (24, 20, 20), backend="hip")
    d = _data(op, 3)
    d[3] = d[4] = None
    d[0][0] = 0
    d[0][1] *= 1e-18
    d[0][2] *= 1e17
    _run(op, d)
    clean = op(*d)[0]
    d[0][4, 1, 5], d[0][4, 2, 9] = float("nan"), float("inf")
    got = op(*d)[0]
    assert torch.isnan(got[4, 1]).all() and torch.isnan(got[4, 2]).any()
    keep = torch.ones(T, H, dtype=torch.bool, device=DEV)
    keep[4, 1:3] = False
    assert torch.equal(got[keep], clean[keep])


def test_in_place_and_equal_to_one_axis_op():
    """q_out = q, k_out = k; with the same position on all axes the result is FusedQkNormRopeOp's up to one rounding
    (the sums of squares are added in another order)."""
    B, H, Hkv, D, S = 5, 8, 2, 128, 64
    one = FusedQkNormRopeOp(B, H, D, S, [3, 0, 63, 17, 40], backend="hip", num_kv_heads=Hkv)
    torch.manual_seed(5)
    q, k, v, qw, kw, cos, sin, K, V = one.gen_data(DEV)
    q1, k1 = one(q, k, v, qw, kw, cos, sin, K, V)
    op = QkNormMropeOp(B, H, Hkv, D, S, (24, 20, 20), backend="hip", interleaved=True)
    pos = torch.tensor([[3, 0, 63, 17, 40]] * 3, dtype=torch.int32, device=DEV)
    q2, k2 = op(q, k, None, qw, kw, cos, sin, pos)
    assert torch.allclose(q1.float(), q2.float(), rtol=2 ** -7, atol=1e-5)
    assert torch.allclose(k1.float(), k2.float(), rtol=2 ** -7, atol=1e-5)
    qc, kc = q.clone(), k.clone()
    q3, k3 = op(qc, kc, None, qw, kw, cos, sin, pos, q_out=qc, k_out=kc)
    assert q3 is qc and torch.equal(q3, q2) and torch.equal(k3, k2)


@pytest.mark.parametrize("off", [1, 4, 8])
def test_unaligned_operands(off):
    """Operands that begin at any element (4: 8 bytes, 1: 2 bytes) and tokens at odd distances."""
    T, H, Hkv, D = 13, 4, 2, 64
    op = QkNormMropeOp(T, H, Hkv, D, 40, (12, 10, 10), backend="hip", page_size=32, num_pages=2)
    d = _data(op, 9)
    x = torch.zeros(T, (H + 2 * Hkv) * D + off, dtype=torch.bfloat16, device=DEV)
    views, at = [], off
    for src in d[:3]:
        w = src.shape[1] * D
        view = x[:, at:at + w].unflatten(1, (src.shape[1], D))
        view.copy_(src)
        views.append(view)
        at += w
    d[:3] = views
    for i in (3, 4, 5, 6):  # weights and tables too
        flat = torch.zeros(d[i].numel() + off, dtype=d[i].dtype, device=DEV)
        flat[off:] = d[i].reshape(-1)
        d[i] = flat[off:].view(d[i].shape)
    q_out = torch.zeros(T * H * D + off, dtype=torch.bfloat16, device=DEV)[off:].view(T, H, D)
    k_out = torch.zeros(T * Hkv * D + off, dtype=torch.bfloat16, device=DEV)[off:].view(T, Hkv, D)
    _run(op, d, q_out, k_out)
    pool = torch.randn(2 * Hkv * 32 * D + off, device=DEV).bfloat16()[off:].view(2, Hkv, 32, D)
    d[8] = pool
    _run(op, d, q_out, k_out)


def test_cache_offsets_past_32_bits():
    """A pool of 5 GiB: slots on its last page."""
    Hkv, D, P = 8, 128, 256
    pages = (5 << 30) // (Hkv * D * P * 2)
    op = QkNormMropeOp(3, 8, Hkv, D, 40, (24, 20, 20), backend="hip", page_size=P, num_pages=pages)
    small = QkNormMropeOp(3, 8, Hkv, D, 40, (24, 20, 20), backend="hip", page_size=P, num_pages=1)
    d = _data(small, 1)
    want = op_in = None
    small(*d)
    K = torch.zeros(pages, Hkv, P, D, dtype=torch.bfloat16, device=DEV)
    V = torch.zeros_like(K)
    slots = d[10] + (pages - 1) * P
    op(*d[:8], K, V, slots)
    rows = d[10]
    assert torch.equal(K[-1][:, rows], d[8][0][:, rows]) and torch.equal(V[-1][:, rows], d[9][0][:, rows])
    assert not bool(K[:-1].any()) and not bool(V[:-1].any())


def test_other_stream_and_graph():
    op = QkNormMropeOp(70, 8, 2, 128, 200, (24, 20, 20), backend="hip", page_size=32, num_pages=4)
    d = _data(op, 4)
    want = op(*d)[0].clone()
    K, V = d[8].clone(), d[9].clone()
    q_out = torch.zeros_like(want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    d[8].zero_()
    with torch.cuda.stream(s):
        s.wait_stream(torch.cuda.default_stream())
        op(*d, q_out=q_out)
    torch.cuda.synchronize()
    assert torch.equal(q_out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op(*d, q_out=q_out)
    for i in range(3):
        fresh = torch.randn_like(d[0])
        d[0].copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q_out, op(*d)[0]), i


def test_argument_checks():
    op = QkNormMropeOp(4, 4, 2, 64, 16, (12, 10, 10), backend="hip", page_size=32, num_pages=2)
    d = _data(op, 0)
    for i, bad in ((0, d[0].float()), (0, d[0][:3]), (1, d[1].transpose(0, 1).contiguous().transpose(0, 1)),
                   (2, None), (3, d[3].float()), (5, d[5].half()), (6, d[6].float()), (7, d[7].long()), (8, d[8][:1]),
                   (10, d[10].int()), (10, None), (8, None), (0, d[0][:1].expand(4, 4, 64))):
        args = list(d)
        args[i] = bad
        with pytest.raises(ValueError):
            op(*args)
    with pytest.raises(ValueError, match="q_out"):
        op(*d, q_out=torch.empty(4, 4, 64, device=DEV))
    with pytest.raises(ValueError, match="without norm"):
        QkNormMropeOp(4, 4, 2, 64, 16, (32,), backend="hip", norm=False)(*d[:7], d[7][:1].contiguous())
    with pytest.raises(RuntimeError, match="GPU tensors"):
        op(d[0].cpu(), *d[1:])
