"""Bounds on the lengths that the ops over the 8-bit KV cache are given: refused below zero by every backend, and whole
numbers of any size otherwise.  CPU only."""

import numpy as np
import pytest
import torch

from ezops import QuantPagedAttnDecodeOp, QuantPrefillAttnOp


def _ops(backend):
    yield QuantPagedAttnDecodeOp(2, 4, 2, 64, 32, 2, backend=backend)
    yield QuantPrefillAttnOp(2, 9, 4, 2, 64, 32, 2, backend=backend)


def _call(op, data, bound):
    out = torch.zeros_like(data[0])  # rows past a bound are left as they were
    return op(*data, max_kv_len=bound, out=out)


@pytest.mark.parametrize("backend", ["ref", "hip"])
def test_bounds_below_zero_are_refused(backend):
    for op in _ops(backend):
        data = op.gen_data("cpu")
        for bound in (-1, -(1 << 31), -(1 << 63), -(1 << 64) + 7):
            with pytest.raises(ValueError, match="max_kv_len"):
                _call(op, data, bound)
        for bound in (1.5, 40.0, "40", None):
            with pytest.raises(TypeError):
                _call(op, data, bound)


def test_large_bounds_are_none():
    for op in _ops("ref"):
        data = op.gen_data("cpu")
        want = _call(op, data, 0)
        for bound in (64, 1 << 31, 1 << 63, 1 << 64, (1 << 64) + 5, np.int64(1 << 40)):
            assert torch.equal(_call(op, data, bound), want), bound
        assert torch.equal(_call(op, data, np.int32(40)), _call(op, data, 40))


def test_the_kernels_get_bounds_as_they_were_given(monkeypatch):
    """A bound whose low 64 bits are another number reaches the entries as one past every table."""
    from ezops.kernels.quant_attn import quant_attn_hip

    got = []
    monkeypatch.setattr(quant_attn_hip._hip, "one_gpu", lambda first, *rest: first.device)
    monkeypatch.setattr(quant_attn_hip._hip, "call_on", lambda dev, name, *args: got.append(args))
    for op in _ops("hip"):
        data = op.gen_data("cpu")
        for bound in (0, 5, 1 << 40, (1 << 64) + 5, 1 << 63):
            got.clear()
            _call(op, data, bound)
            passed = got[0][-4]  # in front of the scale and the workspace
            assert passed == bound if bound < 1 << 30 else 1 << 30 <= passed < 1 << 63
