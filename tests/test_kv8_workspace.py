"""Workspace sizes of attention over the 8-bit KV cache: what is enough for a bound on the lengths is enough for every
smaller one, and for a bound past the table too.  CPU only: the entries are called with no workspace, and name the size
that they need when they refuse (one query tile and at least 640 rows: the keys are always shared out)."""

import re

import numpy as np
import pytest
import torch

from ezops import QuantPagedAttnDecodeOp, QuantPrefillAttnOp, _hip

AT = [(i + 1) << 32 for i in range(10)]  # far apart, 16-byte aligned; nothing is read before the refusal


def needed(which, B, T, H, Hkv, D, pages, bound):
    lib = _hip.lib()
    head = (AT[0], H * D, AT[3], AT[4], AT[5], AT[6], 0, AT[7], AT[8])
    tail = (D, pages * B, 64, pages, 32, bound, 0.0, None, 0, None)
    if which == "decode":
        rc = lib.ezops_quant_paged_attn_decode_bf16(*head, AT[1], B, H, Hkv, *tail)
    else:
        rc = lib.ezops_quant_prefill_attn_bf16(*head, None, AT[1], B, T, H, Hkv, *tail)
    m = re.search(rb"workspace too small \(0 < (\d+)\)", lib.ezops_hip_last_error())
    assert rc == _hip.EINVAL and m, lib.ezops_hip_last_error()
    return int(m.group(1))


def size(which, B, T, H, Hkv, D, n):
    lib = _hip.lib()
    if which == "decode":
        return lib.ezops_quant_paged_attn_decode_workspace_size(B, H, Hkv, D, n)
    return lib.ezops_quant_prefill_attn_workspace_size(B, T, H, Hkv, D, n)


LENS = [640, 704, 705, 832, 1000, 1344, 1500, 2112, 2500, 2624, 3136, 3200, 3400, 3777, 4100, 5504, 6500, 7800, 8192, 20000,
        131072, 1 << 20, 1 << 27, 1 << 30]
SHAPES = [(1, 8, 32, 8, 128), (1, 70, 32, 8, 128), (2, 8, 4, 2, 64), (1, 512, 8, 1, 128), (1, 1, 16, 16, 64)]


@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_size_is_enough_for_every_smaller_bound(which, shape):
    sizes = [size(which, *shape, n) for n in LENS]
    assert sizes == sorted(sizes) and sizes[0] > 0
    for n, enough in zip(LENS, sizes):
        pages = -(-n // 64)
        assert needed(which, *shape, pages, n) <= enough, n
        if n < 1 << 30:
            assert needed(which, *shape, pages + 1, n) <= enough, n  # the bound cuts the table


@pytest.mark.parametrize("which", ["decode", "prefill"])
def test_bounds_past_the_table(which):
    """Sized with the bound itself, though the table holds fewer rows; and with bounds past any table."""
    for shape in SHAPES:
        assert needed(which, *shape, 49, 3200) <= size(which, *shape, 3200)
        most = size(which, *shape, 1 << 30)
        for n in ((1 << 30) + 1, 1 << 40, (1 << 63) - 1):
            assert size(which, *shape, n) == most
            assert needed(which, *shape, 49, n) <= most


def test_every_bound_of_a_range():
    for shape in SHAPES:
        last = {"decode": 0, "prefill": 0}
        for n in range(640, 6000, 7):
            for which in last:
                now = size(which, *shape, n)
                assert now >= last[which] and needed(which, *shape, 100, n) <= now, (shape, which, n)
                last[which] = now


def test_sizes_of_the_python_ops():
    """Workspaces that the ops allocate: enough for the call, for any bound, whole numbers of numpy among them."""
    for shape in SHAPES:
        B, T, H, Hkv, D = shape
        for pages in (12, 49, 100, 2000):
            ops = {"decode": QuantPagedAttnDecodeOp(B, H, Hkv, D, 64, pages, backend="hip"),
                   "prefill": QuantPrefillAttnOp(B, T, H, Hkv, D, 64, pages, backend="hip")}
            for bound in (0, 640, 700, 1597, 1641, 3200, 5555, 1 << 40, np.int64(2624), np.int32(705)):
                for which, op in ops.items():
                    k = op._kernel
                    name = {"decode": "ezops_quant_paged_attn_decode_workspace_size",
                            "prefill": "ezops_quant_prefill_attn_workspace_size"}[which]
                    ws, n = k._workspace(torch.device("cpu"), bound, name, *((B, H, Hkv, D) if which == "decode" else shape))
                    assert ws.numel() == n >= needed(which, *shape, pages, int(bound))
