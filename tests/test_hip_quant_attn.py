"""Attention over the 8-bit KV cache on the GPU, against ``oracle.kv8`` in 64 bits.

Tolerance of an output o = sum_j w_j v_j, with A = sum_j w_j |v_j| and S = the largest scale * sum_d |q_d k_jd| that the
query meets (log2 e of it in the exponent's units): a score is a fp32 sum of D exact products, off by at most
D 2^-24 S, then scaled and shifted in fp32 (three roundings of a value of at most 2 S log2 e) and raised (a relative 2^-22),
so a weight is off by a relative d = (D + 8) 2^-23 S + 2^-22, and once more through the sum; a weight is rounded to bf16
(2^-8 of it) for the product with v, while the sum takes the rounded or the exact ones (2^-8 of A again); the sums of the
products add D-independent fp32 roundings, 2^-24 for each of the up to 2^13 terms of a partial sum at most; the result is
rounded to bf16 (2^-8).  In all 2^-8 |o| + (2 * 2^-8 + 2 d + 2^-11) A.
"""

import numpy as np
import pytest
import torch

from ezops import KvCacheQuantOp, QuantPagedAttnDecodeOp, QuantPrefillAttnOp
from oracle import kv8

pytestmark = pytest.mark.gpu
DEV = "cuda"
KINDS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def n64(x):
    return x.detach().double().cpu().numpy()


def raw(x):
    return x.view(torch.uint8).cpu().numpy()


def tolerance(want, mag, most, D):
    d = (D + 8) * 2.0 ** -23 * most[..., None] + 2.0 ** -22
    return 2.0 ** -8 * np.abs(want) + (2 * 2.0 ** -8 + 2 * d + 2.0 ** -11) * mag + 1e-30


class Cache:
    """Pools whose unused rows and scales are NaN, and the tables of sequences with given numbers of rows."""

    def __init__(self, kind, lens, Hkv, D, P, block, seed, spread=2.0, spare=3, extra=1):
        g = torch.Generator().manual_seed(seed)
        self.g, self.kind, self.lens, self.block, self.P, self.Hkv, self.D = g, kind, lens, block, P, Hkv, D
        need = [-(-x // P) for x in lens]
        self.M, self.pages = max(1, *need) + extra, sum(need) + spare
        order = torch.randperm(self.pages, generator=g).tolist()
        self.table = torch.full((len(lens), self.M), -1, dtype=torch.int32)
        self.table[:, -1] = 1 << 30  # never a page
        slots = []
        for b, n in enumerate(lens):
            ids = [order.pop() for _ in range(need[b])]
            self.table[b, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
            slots += [ids[r // P] * P + r % P for r in range(n)]
        codes = (self.pages, Hkv, P, D)
        self.np = [np.full(codes, 127, np.uint8), np.full(codes, 127, np.uint8),
                   np.full((self.pages, Hkv, P // block), 255, np.uint8), np.full((self.pages, Hkv, P // block), 255, np.uint8)]
        for c, s in ((0, 2), (1, 3)):
            x = torch.randn(len(slots), Hkv, D, generator=g) * torch.exp2(spread * torch.randn(len(slots), 1, 1, generator=g)).clamp(max=8)
            kv8.write(n64(x), self.np[c], self.np[s], slots, block, kind)
        dt = KINDS[kind]
        self.pools = [torch.from_numpy(p).to(DEV).view(dt if p.ndim == 4 else torch.uint8) for p in self.np]
        self.held = []
        for b, n in enumerate(lens):
            at = np.arange(n)
            page = self.table[b].numpy()[at // P]
            kv = []
            for c, s in ((0, 2), (1, 3)):
                e = self.np[s][page, :, at % P // block].astype(float)
                kv.append(kv8.VALUES[kind][self.np[c][page, :, at % P]] * 2.0 ** (e - 127)[..., None])
            self.held.append(kv)
        self.t = self.table.to(DEV)
        self.how = dict(backend="hip", cache_dtype=dt, block_size=block)

    def q(self, T, H, size=1.0, packed=0):
        x = (torch.randn(T, H + packed, self.D, generator=self.g) * size).to(torch.bfloat16).to(DEV)
        return x[:, packed:]

    def want(self, q, b, past, scale):
        n = q.shape[0]
        return kv8.attend(n64(q), self.held[b][0][:past + n], self.held[b][1][:past + n], past, scale)

    def near(self, got, q, b, past, scale, what):
        want, mag, most = self.want(q, b, past, scale)
        err = np.abs(n64(got) - want) / tolerance(want, mag, most, self.D)
        assert np.isfinite(n64(got)).all() and err.max() <= 1, (what, float(err.max()))


EDGES = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 257]


def decode(c, H, lens=None, mx=0, scale=None, packed=0, size=1.0):
    lens = c.lens if lens is None else lens
    q = c.q(len(lens), H, size, packed)
    op = QuantPagedAttnDecodeOp(len(lens), H, c.Hkv, c.D, c.P, c.M, c.pages, **c.how, scale=scale)
    out = op(q, *c.pools, c.t, torch.tensor(lens, dtype=torch.int32, device=DEV), mx)
    for b, n in enumerate(lens):
        n = min(n, mx or c.M * c.P)
        if n <= 0:
            assert not out[b].any(), b
        else:
            c.near(out[b:b + 1], q[b:b + 1], b, n - 1, scale or c.D ** -0.5, (b, n))
    return op, q, out


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("G,Hkv,D,P,block", [(4, 8, 128, 64, 32), (1, 3, 64, 32, 16), (2, 2, 128, 32, 32), (8, 1, 64, 128, 128),
                                             (16, 2, 128, 256, 256), (4, 2, 64, 64, 64), (16, 1, 64, 32, 16), (1, 4, 128, 128, 16),
                                             (8, 2, 128, 64, 16), (2, 5, 64, 32, 32)])
def test_decode_lengths(kind, G, Hkv, D, P, block):
    decode(Cache(kind, EDGES, Hkv, D, P, block, G + P), G * Hkv, packed=3 if D == 64 else 0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens,Hkv,G,D", [([5000], 8, 4, 128), ([3000, 1, 0, 2999], 2, 8, 128), ([1500] * 3, 1, 16, 64), ([2049], 1, 1, 128),
                                          ([4097, 70], 4, 2, 64)])
def test_decode_long(kind, lens, Hkv, G, D):
    """Long sequences of few heads, whose rows are shared out over blocks."""
    c = Cache(kind, lens, Hkv, D, 64, 32, sum(lens))
    decode(c, G * Hkv)
    decode(c, G * Hkv, mx=max(lens))
    decode(c, G * Hkv, mx=max(1, max(lens) // 3))


@pytest.mark.parametrize("kind", KINDS)
def test_decode_many_sequences(kind):
    lens = [(7 * i) % 90 for i in range(150)]
    decode(Cache(kind, lens, 2, 128, 32, 16, 1), 8)


def test_decode_more_sequences_than_are_summed():
    """300 (several steps of the scan, shared out by rows) and 1100 sequences (whole), a long one among short ones."""
    for B, long in ((300, 9000), (1100, 3000)):
        lens = [3 + i % 5 for i in range(B)]
        lens[B // 2], lens[7], lens[B - 1] = long, 0, 1
        decode(Cache("int8", lens, 1, 64, 32, 32, B), 2)


@pytest.mark.parametrize("kind", KINDS)
def test_decode_lengths_outside(kind):
    """Lengths below zero and above what the table or the bound holds."""
    c = Cache(kind, [64, 64, 128, 20], 2, 64, 32, 16, 2, extra=0)
    decode(c, 4, [-5, 10, 1 << 30, 3])
    decode(c, 4, [-(1 << 31), 64, (1 << 31) - 1, 20], mx=50)


@pytest.mark.parametrize("kind", KINDS)
def test_decode_sharp_and_flat_scores(kind):
    """Scores of hundreds (one row has all the weight), of nothing at all, and another scale."""
    c = Cache(kind, [300, 77, 130], 2, 128, 64, 32, 3, spread=0.0)
    decode(c, 8, size=64.0)
    decode(c, 8, size=2.0 ** -30)
    decode(c, 8, scale=1.0)


@pytest.mark.parametrize("kind", KINDS)
def test_decode_out_and_streams(kind):
    c = Cache(kind, [100, 513, 40], 2, 128, 64, 32, 4)
    op, q, out = decode(c, 8)
    lens = torch.tensor(c.lens, dtype=torch.int32, device=DEV)
    buf = torch.full_like(out, 7.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert op(q, *c.pools, c.t, lens, out=buf) is buf
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(buf, out) and torch.equal(op(q, *c.pools, c.t, lens), out)


@pytest.mark.parametrize("kind", KINDS)
def test_decode_nan_stays_in_its_sequence(kind):
    c = Cache(kind, [90, 90, 90], 2, 64, 32, 16, 5)
    op, q, out = decode(c, 4)
    pools = [p.clone() for p in c.pools]
    page = int(c.table[1, 1])
    if kind == "int8":
        pools[2][page, 1, 0] = 255
    else:
        pools[0].view(torch.uint8)[page, 1, 3, 5] = 127
    bad = op(q, *pools, c.t, torch.tensor(c.lens, dtype=torch.int32, device=DEV))
    assert torch.equal(bad[[0, 2]], out[[0, 2]]) and torch.equal(bad[1, :2], out[1, :2]) and bad[1, 2:].isnan().all()
    short = op(q, *pools, c.t, torch.tensor([90, 32, 90], dtype=torch.int32, device=DEV))
    assert short.isfinite().all()


def prefill(c, H, new, past, mx=0, scale=None, packed=0, lead=0, tail=0, with_past=True):
    T = lead + sum(new) + tail
    q = c.q(T, H, 1.0, packed)
    cu = [lead]
    for n in new:
        cu.append(cu[-1] + n)
    op = QuantPrefillAttnOp(len(new), T, H, c.Hkv, c.D, c.P, c.M, c.pages, **c.how, scale=scale)
    out = torch.full((T, H, c.D), 7.0, dtype=torch.bfloat16, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    args = (q, *c.pools, c.t, torch.tensor(cu, **i32), torch.tensor(past, **i32) if with_past else None)
    assert op(*args, max_kv_len=mx, out=out) is out
    written = torch.zeros(T, dtype=torch.bool)
    for b, (n, p) in enumerate(zip(new, past)):
        n = min(n, (min(mx, c.M * c.P) if mx else c.M * c.P) - p)
        if n > 0:
            r = slice(cu[b], cu[b] + n)
            written[r] = True
            c.near(out[r], q[r], b, p, scale or c.D ** -0.5, (b, n, p))
    assert (out[~written.to(DEV)] == 7).all()
    return op, args, out


NEW = [1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 0, 100, 129]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("G,Hkv,D,P,block", [(4, 2, 128, 64, 32), (1, 3, 64, 32, 16), (2, 2, 128, 32, 32), (8, 1, 64, 128, 128),
                                             (16, 1, 128, 256, 256), (4, 1, 64, 64, 64), (16, 1, 64, 32, 16), (1, 2, 128, 128, 16),
                                             (8, 1, 128, 64, 16), (2, 3, 64, 32, 32)])
def test_prefill_lengths(kind, G, Hkv, D, P, block):
    """Fresh prompts and chunks on cached rows, rows of no sequence before and behind them."""
    past = [(37 * i) % 150 for i in range(len(NEW))]
    lens = [n + p for n, p in zip(NEW, past)]
    c = Cache(kind, lens, Hkv, D, P, block, G + D)
    prefill(c, G * Hkv, NEW, past, packed=2 if P == 32 else 0, lead=3, tail=5)
    prefill(c, G * Hkv, NEW, [0] * len(NEW), with_past=False)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new,past,Hkv,G,D", [([300], [0], 2, 4, 128), ([260, 1, 0, 40], [30, 700, 9, 0], 1, 8, 64), ([20], [3000], 1, 4, 128),
                                              ([1], [2500], 2, 2, 64), ([129, 5], [1000, 2000], 1, 16, 128)])
def test_prefill_long(kind, new, past, Hkv, G, D):
    """Chunks on long prefixes, whose rows are shared out over blocks where the queries are few."""
    c = Cache(kind, [n + p for n, p in zip(new, past)], Hkv, D, 64, 32, sum(past))
    prefill(c, G * Hkv, new, past)
    prefill(c, G * Hkv, new, past, mx=max(n + p for n, p in zip(new, past)))


@pytest.mark.parametrize("kind", KINDS)
def test_prefill_past_the_cache(kind):
    """Tokens that stand at or behind the end of the table, or of the caller's bound, are left alone; so are their rows."""
    c = Cache(kind, [64, 64, 64], 2, 64, 32, 16, 6, extra=0)
    prefill(c, 4, [40, 10, 30], [50, 64, 34])
    prefill(c, 4, [40, 10, 30], [50, 20, 0], mx=25)
    prefill(c, 4, [3, 3, 3], [100, 1 << 30, 61])


@pytest.mark.parametrize("kind", KINDS)
def test_prefill_many_sequences(kind):
    new = [(5 * i) % 7 for i in range(200)]
    past = [(11 * i) % 60 for i in range(200)]
    prefill(Cache(kind, [n + p for n, p in zip(new, past)], 2, 64, 32, 32, 7), 4, new, past, tail=4)


@pytest.mark.parametrize("kind", KINDS)
def test_prefill_nan_of_later_rows_is_not_seen(kind):
    """A row that is not finite touches the queries at and behind its block's first row (int8) or itself (e4m3), of its
    head alone; queries before see nothing of it, in the same tile or not."""
    new, past, block = [90, 60], [10, 0], 16
    c = Cache(kind, [100, 60], 2, 128, 64, block, 8)
    op, args, out = prefill(c, 8, new, past)
    pools = [p.clone() for p in c.pools]
    row = 53
    page = int(c.table[0, 0])
    for which in (0, 1):  # k, then v
        mod = [p.clone() for p in c.pools]
        if kind == "int8":
            mod[2 + which][page, 1, row // block] = 255
            first = row // block * block
        else:
            mod[which].view(torch.uint8)[page, 1, row, 9] = 127
            first = row
        bad = op(args[0], *mod, *args[5:])
        q0 = first - past[0]
        assert torch.equal(bad[:q0], out[:q0]) and torch.equal(bad[90:], out[90:]) and torch.equal(bad[:, :4], out[:, :4])
        hit = bad[q0:90, 4:]
        assert (hit.isnan().all() if which == 0 or kind == "int8" else hit[..., 9].isnan().all())


def test_attention_past_32_bits():
    """Rows behind 2^32 codes of a pool."""
    Hkv, D, P, block = 8, 128, 128, 32
    pages = 33000
    kv = KvCacheQuantOp(200, Hkv, D, P, pages, backend="hip", block_size=block)
    pools = kv.alloc(DEV)
    assert pools[0].numel() > 1 << 32
    g = torch.Generator().manual_seed(9)
    x = torch.randn(200, 2 * Hkv, D, generator=g).to(torch.bfloat16).to(DEV)
    ids = [pages - 1, pages - 2]
    slots = torch.tensor([ids[r // P] * P + r % P for r in range(200)], device=DEV)
    kv(x[:, :Hkv], x[:, Hkv:], *pools, slots)
    small = [torch.stack([p[i] for i in ids]).view(torch.uint8).cpu().numpy() for p in pools]
    k, v = (kv8.rows(small[c], small[s], [0, 1], 200, block, "int8") for c, s in ((0, 2), (1, 3)))
    q = torch.randn(31, 16, D, generator=g).to(torch.bfloat16).to(DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    table = torch.tensor([ids], **i32)
    one = QuantPagedAttnDecodeOp(1, 16, Hkv, D, P, 2, pages, backend="hip", block_size=block)(
        q[-1:], *pools, table, torch.tensor([200], **i32))
    many = QuantPrefillAttnOp(1, 31, 16, Hkv, D, P, 2, pages, backend="hip", block_size=block)(
        q, *pools, table, torch.tensor([0, 31], **i32), torch.tensor([169], **i32))
    want, mag, most = kv8.attend(n64(q), k, v, 169, D ** -0.5)
    tol = tolerance(want, mag, most, D)
    assert (np.abs(n64(many) - want) <= tol).all() and (np.abs(n64(one) - want[-1:]) <= tol[-1:]).all()


@pytest.mark.parametrize("kind", KINDS)
def test_wide_tables(kind):
    """Tables for 2^16 and more rows a sequence that hold a few hundred: plans for what could be, work for what is."""
    c = Cache(kind, [300, 33, 700, 1], 2, 128, 64, 32, 12, extra=1020)
    decode(c, 8)
    prefill(c, 8, [20, 33, 1, 0], [280, 0, 699, 1])
    prefill(Cache(kind, [515], 1, 64, 64, 16, 13, extra=2000), 4, [70], [445])


def test_two_streams_at_once():
    """The same ops on two streams that run together: neither disturbs the other."""
    c = Cache("e4m3", [3000, 90, 1500], 2, 128, 64, 32, 14)
    i32 = dict(dtype=torch.int32, device=DEV)
    dec = QuantPagedAttnDecodeOp(3, 8, 2, 128, 64, c.M, c.pages, **c.how)
    pre = QuantPrefillAttnOp(3, 40, 8, 2, 128, 64, c.M, c.pages, **c.how)
    lens, cu, past = torch.tensor(c.lens, **i32), torch.tensor([0, 20, 37, 40], **i32), torch.tensor([2980, 73, 1497], **i32)
    qs = [(c.q(3, 8), c.q(40, 8)) for _ in range(2)]
    both = lambda q: (dec(q[0], *c.pools, c.t, lens), pre(q[1], *c.pools, c.t, cu, past))  # noqa: E731
    want = [both(q) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(both(qs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert torch.equal(out[0], want[i][0]) and torch.equal(out[1], want[i][1])


@pytest.mark.parametrize("kind", KINDS)
def test_captured_calls(kind):
    """Two graphs of both ops, replayed in turn with eager calls between: every replay equals the eager result."""
    c = Cache(kind, [700, 90, 33], 2, 128, 64, 32, 10)
    i32 = dict(dtype=torch.int32, device=DEV)
    dec = QuantPagedAttnDecodeOp(3, 8, 2, 128, 64, c.M, c.pages, **c.how)
    pre = QuantPrefillAttnOp(3, 40, 8, 2, 128, 64, c.M, c.pages, **c.how)
    lens, cu, past = torch.tensor(c.lens, **i32), torch.tensor([0, 20, 37, 40], **i32), torch.tensor([680, 73, 30], **i32)
    qd, qp = c.q(3, 8), c.q(40, 8)
    both = lambda: (dec(qd, *c.pools, c.t, lens), pre(qp, *c.pools, c.t, cu, past))  # noqa: E731
    eager = [x.clone() for x in both()]
    graphs = []
    for _ in range(2):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            both()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = both()
        graphs.append((g, out))
    keep = [x.clone() for x in (qd, qp)]
    for r in range(6):
        scale = 1.0 if r % 2 == 0 else 0.5
        qd.copy_(keep[0] * scale)
        qp.copy_(keep[1] * scale)
        g, out = graphs[r % 2 if r < 4 else 0]
        for x in out:
            x.fill_(float("nan"))
        g.replay()
        fresh = both()
        for a, e in zip(out, fresh):
            assert torch.equal(a, e), r
        if scale == 1.0:
            for a, e in zip(out, eager):
                assert torch.equal(a, e), r


def test_refusals_on_the_gpu():
    c = Cache("int8", [40, 20], 2, 64, 32, 32, 11)
    i32 = dict(dtype=torch.int32, device=DEV)
    op = QuantPagedAttnDecodeOp(2, 4, 2, 64, 32, c.M, c.pages, **c.how)
    q, lens = c.q(2, 4), torch.tensor([40, 20], **i32)
    for args in [(q[:1], *c.pools, c.t, lens), (q.float(), *c.pools, c.t, lens), (q, *c.pools, c.t.long(), lens),
                 (q, *c.pools, c.t[:, :1], lens), (q, *c.pools, c.t, lens.long()), (q, c.pools[0].float(), *c.pools[1:], c.t, lens),
                 (q, *c.pools, c.t, lens, -1)]:
        with pytest.raises(ValueError):
            op(*args)
    with pytest.raises(RuntimeError, match="GPU"):
        op(q, *c.pools, c.t.cpu(), lens)
    with pytest.raises(RuntimeError, match="overlap"):
        op(q, *c.pools, c.t, lens, out=q.contiguous() if not q.is_contiguous() else q)
    pre = QuantPrefillAttnOp(1, 5, 4, 2, 64, 32, c.M, c.pages, **c.how)
    q5, cu = c.q(5, 4), torch.tensor([0, 5], **i32)
    for args, kw in [((q5, *c.pools, c.t, cu), {}), ((q5, *c.pools, c.t[:1].contiguous(), cu[:1]), {}),
                     ((q5, *c.pools, c.t[:1].contiguous(), cu, lens), {}),
                     ((q5, *c.pools, c.t[:1].contiguous(), cu), dict(max_kv_len=-1))]:
        with pytest.raises(ValueError):
            pre(*args, **kw)
