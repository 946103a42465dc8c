"""HIP batch plan against the restatement on the host: every output and the table exactly."""

import random

import numpy as np
import pytest
import torch

from ezops import PagedBatchPlanOp
from oracle import ragged

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)


def _check(q, past, T, P, M, NP, free, span, seed=0, with_past=True):
    B = len(q)
    g = torch.Generator().manual_seed(seed)
    table = torch.randint(0, NP, (B, M), generator=g, dtype=torch.int32)
    table[torch.rand(B, M, generator=g) < 0.05] = -1
    table[torch.rand(B, M, generator=g) < 0.05] = NP
    op = PagedBatchPlanOp(B, T, P, M, NP, len(free), backend="hip")
    want = ragged.batch_plan(q, past if with_past else None, table.numpy(), free, span, T, P, NP)
    dev_table = table.to(DEV)
    args = (torch.tensor(q, **I32), torch.tensor(past, **I32) if with_past else None, dev_table,
            torch.tensor(free, **I32), torch.tensor(span, **I32))
    for _ in range(2):  # the same inputs give the same plan
        got = op(*args)
        for name, a, w in zip(("table", *got._fields), (dev_table, *got), want):
            np.testing.assert_array_equal(a.cpu().numpy(), w, err_msg=name)
    assert args[4].tolist() == list(span)
    return op, args, got


@pytest.mark.parametrize("B", [1, 2, 63, 64, 65, 255, 256, 257, 1000, 4096])
def test_batch_sizes(B):
    r = random.Random(B)
    q = [r.choice([0, 1, 1, 2, 40, 70]) for _ in range(B)]
    past = [r.choice([0, 0, 1, 31, 32, 33, 300]) for _ in range(B)]
    free = [r.randrange(500) for _ in range(6 * B)]
    _check(q, past, sum(q) + r.choice([1, 300]), 32, 14, 500, free, [1, len(free)], seed=B)


@pytest.mark.parametrize("P,M", [(32, 1), (32, 700), (256, 40), (1 << 20, 1 << 10)])
def test_page_sizes(P, M):
    r = random.Random(P)
    cap = P * M
    q = [0, 1, P, 33, 1000, 2, 5]
    past = [cap, cap - 1, 0, max(0, cap - 20), r.randrange(min(cap, 9000)), 7 * P, (1 << 31) - 1]
    _check(q, past, sum(q), P, M, 1 << 22, [r.randrange(1 << 22) for _ in range(99)], [3, 99])


@pytest.mark.parametrize("span", [[0, 0], [0, 3], [5, 3], [-1, 9], [2, 1000], [9, 9], [20, 30], [(1 << 31) - 1, (1 << 31) - 1],
                                  [-(1 << 31), 5]])
def test_short_and_bad_free_lists(span):
    free = [4, -1, 7, 30, 2, 1 << 30, 5, 11, -(1 << 31)]
    _check([40, 1, 100, 0, 64], [0, 31, 5, 64, 32], 210, 32, 9, 30, free, span)


def test_no_free_list_and_no_past():
    _check([5, 0, 40], [0, 0, 0], 50, 32, 4, 8, [], [0, 0], with_past=False)
    _check([5, 0, 40], [0, 0, 0], 50, 32, 4, 8, [3, 1, 2, 0], [0, 4], with_past=False)


@pytest.mark.parametrize("q,T", [([100, 100, 100], 150), ([(1 << 31) - 1, 5, (1 << 31) - 1], 64), ([-5, 3, -(1 << 31), 4], 7),
                                 ([0, 0, 0], 3), ([70000, 3], 70001)])
def test_rows_run_out(q, T):
    _check(q, [3, 0, 64, 1][:len(q)], T, 64, 2000, 4000, list(range(1500)), [0, 1500])


def test_more_rows_than_one_pass_of_the_grid():
    T = 1024 * 256 + 777
    _check([T // 2, 17, T], [0, 100, 5], T, 256, 2000, 5000, list(range(4000)), [0, 4000])


def test_out_buffers_other_stream_and_graph():
    q, past = [3, 40, 0, 1], [30, 0, 9, 64]
    op, args, want = _check(q, past, 64, 32, 5, 40, list(range(20, 40)), [2, 20])
    out = op.alloc(DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = op(*args, out=out)
    torch.cuda.current_stream().wait_stream(s)
    assert got is out
    for a, w in zip(out, want):
        assert torch.equal(a, w)
    # a decode loop in one graph: the plan of step n takes the span that step n - 1 left
    torch.cuda.synchronize()
    span, past_t, table = args[4].clone(), args[1].clone(), args[2].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op(args[0], past_t, table, args[3], span, out=out)
        span.copy_(out.free_span[:2])
        past_t.copy_(out.kv_lens)
    e_span, e_past, e_table = [2, 20], list(past), args[2].cpu().numpy()
    for step in range(4):
        graph.replay()
        e = ragged.batch_plan(q, e_past, e_table, list(range(20, 40)), e_span, 64, 32, 40)
        e_table, e_past, e_span = e[0], e[2].tolist(), e[5][:2].tolist()
        torch.cuda.synchronize()
        for a, w in zip((table, *out), e):
            np.testing.assert_array_equal(a.cpu().numpy(), w, err_msg=f"replay {step}")


def test_argument_checks():
    op = PagedBatchPlanOp(2, 8, 32, 4, 9, backend="hip")
    data = list(op.gen_data(DEV))
    for i, bad in ((0, data[0].long()), (1, data[1][:1]), (2, data[2].t()), (3, data[3][:-1]), (4, data[4][:1]),
                   (4, data[4].long())):
        args = list(data)
        args[i] = bad
        with pytest.raises(ValueError):
            op(*args)
    with pytest.raises(ValueError, match="slot_mapping"):
        op(*data, out=op.alloc(DEV)._replace(slot_mapping=torch.empty(8, **I32)))
    with pytest.raises(RuntimeError, match="GPU tensors"):
        op(*data[:4], data[4].cpu())
    with pytest.raises(RuntimeError, match="free_span_out"):
        span = torch.tensor([0, 9, 0], **I32)
        op(*data[:4], span, out=op.alloc(DEV)._replace(free_span=span))
