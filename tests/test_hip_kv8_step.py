"""The ops over the 8-bit KV cache together, as a serving step uses them: plan, QK norm + rotation, quantised write through
the plan's slots, attention over the planned block table, read-back; a prompt step of several requests, a second chunk, then
decode steps, the latter also through replays of one graph.

Expected values: the pools byte by byte from ``oracle.kv8`` fed with the rotated k and the v that the cache was given; the
attention from those pools in 64 bits, within the tolerance that test_hip_quant_attn derives.
"""

import numpy as np
import pytest
import torch

from ezops import (KvCacheDequantOp, KvCacheQuantOp, PagedBatchPlanOp, QkNormMropeOp, QuantPagedAttnDecodeOp,
                   QuantPrefillAttnOp, profiling)
from ezops.ops.fused_qk_norm_rope import rope_tables
from oracle import kv8
from test_hip_quant_attn import tolerance

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)
KINDS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
H, HKV, D, P, M, S, SEC, BLOCK = 8, 2, 128, 32, 8, 400, (24, 20, 20), 16


def n64(x):
    return x.detach().double().cpu().numpy()


class Serving:
    """Pools and requests on the GPU, the same pools as bytes on the host."""

    def __init__(self, B, kind, seed):
        g = torch.Generator().manual_seed(seed)
        self.B, self.g, self.kind, self.how = B, g, kind, dict(backend="hip", cache_dtype=KINDS[kind], block_size=BLOCK)
        self.pool = B * M + 5
        self.free = torch.randperm(self.pool, generator=g).to(**I32)
        self.span, self.table, self.past = torch.tensor([0, self.pool], **I32), torch.full((B, M), -1, **I32), torch.zeros(B, **I32)
        self.np = [np.full((self.pool, HKV, P, D), 127, np.uint8), np.full((self.pool, HKV, P, D), 127, np.uint8),
                   np.full((self.pool, HKV, P // BLOCK), 255, np.uint8), np.full((self.pool, HKV, P // BLOCK), 255, np.uint8)]
        self.pools = [torch.from_numpy(p).to(DEV).view(KINDS[kind] if p.ndim == 4 else torch.uint8) for p in self.np]
        self.cos, self.sin = rope_tables(S, D, 1e6, DEV)
        self.w = [(1 + 0.1 * torch.randn(D, generator=g)).to(torch.bfloat16).to(DEV) for _ in range(2)]

    def tokens(self, T):
        return torch.randn(T, H + 2 * HKV, D, generator=self.g).to(torch.bfloat16).to(DEV)

    def rope(self, T):
        return QkNormMropeOp(T, H, HKV, D, S, SEC, backend="hip", interleaved=True)

    def written(self, k, v, slots):
        """The host's pools after the same write; the GPU's have to be equal."""
        for x, c, s in ((k, 0, 2), (v, 1, 3)):
            kv8.write(n64(x), self.np[c], self.np[s], slots.tolist(), BLOCK, self.kind)
        for p, w in zip(self.pools, self.np):
            np.testing.assert_array_equal(p.view(torch.uint8).cpu().numpy(), w)

    def attended(self, out, q, b, past, table):
        n = q.shape[0]
        k, v = (kv8.rows(self.np[c], self.np[s], table[b], past + n, BLOCK, self.kind) for c, s in ((0, 2), (1, 3)))
        want, mag, most = kv8.attend(n64(q), k, v, past, D ** -0.5)
        assert (np.abs(n64(out) - want) <= tolerance(want, mag, most, D)).all(), b


def prompt_step(sv, lens, T):
    plan = PagedBatchPlanOp(sv.B, T, P, M, sv.pool, backend="hip")(torch.tensor(lens, **I32), sv.past, sv.table, sv.free, sv.span)
    x = sv.tokens(T)
    v = x[:, H + HKV:]
    q, k = sv.rope(T)(x[:, :H], x[:, H:H + HKV], None, *sv.w, sv.cos, sv.sin, torch.stack([plan.positions] * 3),
                      q_out=torch.zeros(T, H, D, dtype=torch.bfloat16, device=DEV),
                      k_out=torch.zeros(T, HKV, D, dtype=torch.bfloat16, device=DEV))
    KvCacheQuantOp(T, HKV, D, P, sv.pool, **sv.how)(k, v, *sv.pools, plan.slot_mapping)
    out = torch.full((T, H, D), 7.0, dtype=torch.bfloat16, device=DEV)
    QuantPrefillAttnOp(sv.B, T, H, HKV, D, P, M, sv.pool, **sv.how)(q, *sv.pools, sv.table, plan.cu_seqlens, sv.past, out=out)
    back = KvCacheDequantOp(T, HKV, D, P, sv.pool, **sv.how)(*sv.pools, plan.slot_mapping)
    sv.written(k, v, plan.slot_mapping)
    table, past, at = sv.table.cpu().numpy(), sv.past.tolist(), 0
    for b, n in enumerate(lens):
        if n:
            sv.attended(out[at:at + n], q[at:at + n], b, past[b], table)
            for x, c, s in ((back[0], 0, 2), (back[1], 1, 3)):
                np.testing.assert_array_equal(n64(x[at:at + n]), kv8.rows(sv.np[c], sv.np[s], table[b], past[b] + n, BLOCK, sv.kind)[past[b]:])
        at += n
    assert (out[at:] == 7).all()
    sv.past, sv.span = plan.kv_lens, plan.free_span


@pytest.mark.parametrize("kind", KINDS)
def test_prompts_chunks_and_decode_steps(kind):
    sv = Serving(4, kind, 1)
    prompt_step(sv, [40, 1, 0, 100], 150)
    prompt_step(sv, [30, 64, 7, 0], 101)
    B = sv.B
    plan_op = PagedBatchPlanOp(B, B, P, M, sv.pool, backend="hip")
    rope, quant = sv.rope(B), KvCacheQuantOp(B, HKV, D, P, sv.pool, **sv.how)
    dec = QuantPagedAttnDecodeOp(B, H, HKV, D, P, M, sv.pool, **sv.how)
    x, ones, plan_out, past, span = sv.tokens(B), torch.ones(B, **I32), plan_op.alloc(DEV), sv.past.clone(), sv.span[:2].clone()

    def step():
        plan = plan_op(ones, past, sv.table, sv.free, span, out=plan_out)
        q, k = rope(x[:, :H], x[:, H:H + HKV], None, *sv.w, sv.cos, sv.sin, torch.stack([plan.positions] * 3))
        quant(k, x[:, H + HKV:], *sv.pools, plan.slot_mapping)
        out = dec(q, *sv.pools, sv.table, plan.kv_lens)
        past.copy_(plan.kv_lens)
        span.copy_(plan.free_span[:2])
        return q, k, out

    def check(q, k, out):
        sv.written(k, x[:, H + HKV:], plan_out.slot_mapping)
        table, lens = sv.table.cpu().numpy(), past.tolist()
        for b in range(B):
            sv.attended(out[b:b + 1], q[b:b + 1], b, lens[b] - 1, table)

    check(*step())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(40):  # past the end of a page
        x.copy_(sv.tokens(B) * (1.0 if i % 7 else 30.0))  # blocks that grow
        graph.replay()
        check(*got)
    assert past.tolist() == [111, 106, 48, 141]


def test_wave_records():
    """Records of the ops: each names its kernels, and results with the recorder are the same bits."""
    from test_hip_profiling import check_records

    torch.manual_seed(0)
    cases = [(KvCacheQuantOp(300, 2, 128, 64, 6, backend="hip"), {"kv_quant"}),
             (KvCacheDequantOp(300, 2, 64, 64, 6, backend="hip", cache_dtype=torch.float8_e4m3fn), {"kv_dequant"}),
             (QuantPagedAttnDecodeOp(3, 8, 2, 128, 64, 20, backend="hip"), {"quant_attn_decode", "quant_attn_combine"}),
             (QuantPagedAttnDecodeOp(2, 8, 2, 64, 64, 2, backend="hip"), {"quant_attn_decode"}),
             (QuantPrefillAttnOp(2, 300, 8, 2, 128, 64, 3, backend="hip"), {"quant_attn_prefill"}),
             (QuantPrefillAttnOp(1, 20, 8, 2, 64, 64, 60, backend="hip"), {"quant_attn_prefill", "quant_attn_combine"})]
    for op, names in cases:
        data = op.gen_data()
        kw = {}
        if isinstance(op, QuantPagedAttnDecodeOp) and op.max_pages == 2:
            kw = dict(max_kv_len=100)  # one block a sequence
        again = [x.clone() for x in data]
        want = op(*data, **kw)
        with profiling.WaveTrace() as tr:
            got = op(*again, **kw)
        for a, w in zip(got if isinstance(got, tuple) else [got], want if isinstance(want, tuple) else [want]):
            assert torch.equal(a.view(torch.uint8), w.view(torch.uint8)), type(op)
        check_records(tr.records, names)


@pytest.mark.parametrize("seed", range(24))
def test_drawn_shapes(seed):
    """Write in two calls, read-back and both attentions of one small batch of any shape."""
    r = np.random.RandomState(seed)
    kind = ["int8", "e4m3"][seed % 2]
    d, hkv, g = int(r.choice([64, 128])), int(r.choice([1, 2, 3, 5])), int(r.choice([1, 2, 4, 8, 16]))
    page = int(r.choice([32, 64, 128, 256]))
    block = int(r.choice([b for b in (16, 32, 64, 128, 256) if b <= page]))
    B = int(r.randint(1, 6))
    past, new = r.randint(0, 300, B) * r.randint(0, 2, B), r.randint(0, 90, B)
    new[0] += 1
    how = dict(backend="hip", cache_dtype=KINDS[kind], block_size=block)
    need = -(-(past + new) // page)
    pages, width = int(need.sum()) + 2, int(need.max()) + int(r.randint(0, 2))
    order, table = list(r.permutation(pages)), np.full((B, width), -1, np.int32)
    for b in range(B):
        table[b, :need[b]] = [order.pop() for _ in range(need[b])]
    slot = lambda b, i: int(table[b, i // page]) * page + i % page  # noqa: E731
    gen = torch.Generator().manual_seed(seed)
    pools = KvCacheQuantOp(1, hkv, d, page, pages, **how).alloc(DEV)
    host = [p.view(torch.uint8).cpu().numpy() for p in pools]
    for first in (True, False):
        slots = [slot(b, i) for b in range(B) for i in (range(past[b]) if first else range(past[b], past[b] + new[b]))]
        T = len(slots) + 1
        x = (torch.randn(T, 2 * hkv, d, generator=gen) * (1 + 3 * (not first))).to(torch.bfloat16).to(DEV)
        KvCacheQuantOp(T, hkv, d, page, pages, **how)(x[:, :hkv], x[:, hkv:], *pools, torch.tensor(slots + [-1], device=DEV))
        for c, s, y in ((0, 2, x[:, :hkv]), (1, 3, x[:, hkv:])):
            kv8.write(n64(y), host[c], host[s], slots + [-1], block, kind)
    for p, w in zip(pools, host):
        np.testing.assert_array_equal(p.view(torch.uint8).cpu().numpy(), w)
    T = int(new.sum())
    q = torch.randn(T, g * hkv, d, generator=gen).to(torch.bfloat16).to(DEV)
    cu = np.concatenate([[0], np.cumsum(new)])
    t, i32 = torch.from_numpy(table).to(DEV), dict(dtype=torch.int32, device=DEV)
    out = QuantPrefillAttnOp(B, T, g * hkv, hkv, d, page, width, pages, **how)(
        q, *pools, t, torch.tensor(cu, **i32), torch.tensor(past, **i32))
    last = q[torch.tensor(np.maximum(cu[1:] - 1, 0), device=DEV)]
    lens = np.where(new > 0, past + new, 0)
    one = QuantPagedAttnDecodeOp(B, g * hkv, hkv, d, page, width, pages, **how)(last, *pools, t, torch.tensor(lens, **i32))
    for b in range(B):
        n, p = int(new[b]), int(past[b])
        if not n:
            assert not one[b].any()
            continue
        k, v = (kv8.rows(host[c], host[s], table[b], p + n, block, kind) for c, s in ((0, 2), (1, 3)))
        want, mag, most = kv8.attend(n64(q[cu[b]:cu[b] + n]), k, v, p, d ** -0.5)
        tol = tolerance(want, mag, most, d)
        assert (np.abs(n64(out[cu[b]:cu[b] + n]) - want) <= tol).all(), b
        assert (np.abs(n64(one[b]) - want[-1]) <= tol[-1]).all(), b
