"""The ops over the 8-bit KV cache on the CPU: registry family, argument checks of the ops and of the C entries (before
any device call), and the torch ``ref`` backends against the 64-bit restatement in ``oracle.kv8``."""

import numpy as np
import pytest
import torch

from ezops import (KvCacheDequantOp, KvCacheQuantOp, QuantPagedAttnDecodeOp, QuantPrefillAttnOp, _hip, get_kernel,
                   list_backends, list_ops)
from oracle import kv8

KV8 = ["kv_cache_dequant", "kv_cache_quant", "quant_paged_attn_decode", "quant_prefill_attn"]
KINDS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def test_registry_family():
    assert list_ops("kv8") == KV8
    assert list_ops("all") == sorted(list_ops(None) + KV8)
    for op in KV8:
        assert list_backends(op) == ["hip"] and get_kernel(op, "hip").op_name == op


def _raises(text, cls, *args, **kw):
    for backend in ("ref", "hip"):
        with pytest.raises(ValueError, match=text):
            cls(*args, backend=backend, **kw)


def test_constructor_refusals():
    for cls in (KvCacheQuantOp, KvCacheDequantOp):
        for args, kw, text in [((0, 2, 64, 64, 4), {}, "num_tokens"), ((1 << 30, 2, 64, 64, 4), {}, "num_tokens"),
                               ((1, 0, 64, 64, 4), {}, "num_kv_heads"), ((1, 2, 96, 64, 4), {}, "head_dim"),
                               ((1, 2, 64, 48, 4), {}, "page_size"), ((1, 2, 64, 16, 4), {}, "page_size"),
                               ((1, 2, 64, 64, 0), {}, "num_pages"), ((1, 2, 64, 64, 4), dict(block_size=8), "block_size"),
                               ((1, 2, 64, 64, 4), dict(block_size=24), "block_size"),
                               ((1, 2, 64, 64, 4), dict(block_size=128), "block_size"),
                               ((1, 2, 64, 1024, 4), dict(block_size=512), "block_size"),
                               ((1, 2, 64, 64, 4), dict(cache_dtype=torch.uint8), "cache_dtype"),
                               ((1, 2, 64, 64, 4), dict(cache_dtype=torch.float8_e5m2), "cache_dtype")]:
            _raises(text, cls, *args, **kw)
    for args, kw, text in [((0, 4, 2, 64, 64, 4), {}, "batch"), ((65537, 4, 2, 64, 64, 4), {}, "batch"),
                           ((1, 4, 3, 64, 64, 4), {}, "divisible"), ((1, 6, 2, 64, 64, 4), {}, "group size"),
                           ((1, 4, 2, 80, 64, 4), {}, "head_dim"), ((1, 4, 2, 64, 40, 4), {}, "page_size"),
                           ((1, 4, 2, 64, 64, 0), dict(num_pages=1), "max_pages"), ((1, 4, 2, 64, 64, 0), {}, "max_pages"),
                           ((1, 4, 2, 64, 64, 1 << 25), {}, "max_pages"), ((1, 4, 2, 64, 64, 4, 0), {}, "num_pages"),
                           ((1, 4, 2, 64, 64, 4), dict(scale=0.0), "scale"),
                           ((1, 4, 2, 64, 64, 4), dict(block_size=128), "block_size"),
                           ((1, 4, 2, 64, 64, 4), dict(cache_dtype=torch.bfloat16), "cache_dtype")]:
        _raises(text, QuantPagedAttnDecodeOp, *args, **kw)
        _raises(text, QuantPrefillAttnOp, args[0], 8, *args[1:], **kw)
    _raises("num_tokens", QuantPrefillAttnOp, 1, 0, 4, 2, 64, 64, 4)


AT = [(i + 1) << 24 for i in range(12)]  # addresses far apart, never touched


def _quant(k=AT[0], ks=128, v=AT[1], vs=128, slots=AT[2], K=AT[3], V=AT[4], Ks=AT[5], Vs=AT[6], ty=0, NP=4, P=64, blk=32, T=8,
           Hkv=2, D=64):
    return _hip.lib().ezops_kv_cache_quant_bf16(k, ks, v, vs, slots, K, V, Ks, Vs, ty, NP, P, blk, T, Hkv, D, None)


def _dequant(K=AT[3], V=AT[4], Ks=AT[5], Vs=AT[6], slots=AT[2], ty=0, NP=4, P=64, blk=32, ko=AT[0], vo=AT[1], T=8, Hkv=2, D=64):
    return _hip.lib().ezops_kv_cache_dequant_bf16(K, V, Ks, Vs, slots, ty, NP, P, blk, ko, vo, T, Hkv, D, None)


def _decode(q=AT[0], qs=256, K=AT[3], V=AT[4], Ks=AT[5], Vs=AT[6], ty=0, table=AT[7], lens=AT[8], out=AT[1], B=2, H=4, Hkv=2,
            D=64, NP=4, P=64, M=2, blk=32, mx=0, scale=0.0, ws=AT[9], nb=1 << 24):
    return _hip.lib().ezops_quant_paged_attn_decode_bf16(q, qs, K, V, Ks, Vs, ty, table, lens, out, B, H, Hkv, D, NP, P, M, blk,
                                                         mx, scale, ws, nb, None)


def _prefill(q=AT[0], qs=256, K=AT[3], V=AT[4], Ks=AT[5], Vs=AT[6], ty=0, table=AT[7], lens=AT[8], past=None, out=AT[1], B=2,
             T=8, H=4, Hkv=2, D=64, NP=4, P=64, M=2, blk=32, mx=0, scale=0.0, ws=AT[9], nb=1 << 24):
    return _hip.lib().ezops_quant_prefill_attn_bf16(q, qs, K, V, Ks, Vs, ty, table, lens, past, out, B, T, H, Hkv, D, NP, P, M,
                                                    blk, mx, scale, ws, nb, None)


def _refused(fn, kw, *texts):
    err = _hip.lib().ezops_hip_last_error
    assert fn(**kw) == _hip.EINVAL and any(t in err() for t in texts), (fn.__name__, kw, err())


def test_c_entries_reject_bad_arguments():
    pools = [(dict(K=None), b"null"), (dict(V=None), b"null"), (dict(Ks=None), b"null"), (dict(Vs=None), b"null"),
             (dict(ty=2), b"cache type"), (dict(ty=-1), b"cache type"), (dict(NP=0), b"num_pages"),
             (dict(NP=1 << 31), b"num_pages"), (dict(P=48), b"page_size"), (dict(P=16), b"page_size"),
             (dict(P=1 << 21), b"page_size"), (dict(P=0), b"page_size"), (dict(blk=8), b"block_size"),
             (dict(blk=48), b"block_size"), (dict(blk=128), b"block_size"), (dict(blk=0), b"block_size"),
             (dict(blk=512, P=1024), b"block_size"), (dict(K=AT[3] + 8), b"16-byte"), (dict(V=AT[4] + 1), b"16-byte"),
             (dict(D=96), b"head_dim"), (dict(D=0), b"head_dim")]
    for kw, text in pools:
        for fn in (_quant, _dequant, _decode, _prefill):
            _refused(fn, dict(kw, **({"qs": 4 * kw["D"]} if fn in (_decode, _prefill) and kw.get("D") else {}),
                              **({"ks": 2 * kw["D"], "vs": 2 * kw["D"]} if fn is _quant and "D" in kw else {})), text)
    for kw, text in [(dict(k=None), b"null"), (dict(v=None), b"null"), (dict(slots=None), b"null"), (dict(T=0), b"tokens"),
                     (dict(T=1 << 30), b"tokens"), (dict(Hkv=0), b"num_kv_heads"), (dict(Hkv=4097), b"num_kv_heads"),
                     (dict(ks=120), b"strides"), (dict(vs=0), b"strides"), (dict(ks=132), b"16 bytes"),
                     (dict(k=AT[0] + 2), b"16 bytes"), (dict(v=AT[1] + 8), b"16 bytes")]:
        _refused(_quant, kw, text)
    for kw, text in [(dict(slots=None), b"null"), (dict(ko=None), b"null"), (dict(vo=None), b"null"), (dict(T=0), b"tokens"),
                     (dict(Hkv=0), b"num_kv_heads"), (dict(ko=AT[0] + 8), b"16-byte"), (dict(vo=AT[1] + 2), b"16-byte")]:
        _refused(_dequant, kw, text)
    for fn in (_decode, _prefill):
        for kw, text in [(dict(q=None), b"null"), (dict(out=None), b"null"), (dict(table=None), b"null"),
                         (dict(lens=None), b"null"), (dict(B=0), b"batch"), (dict(B=65537), b"batch"),
                         (dict(H=0), b"num_heads"), (dict(Hkv=3), b"divisible"), (dict(Hkv=0), b"divisible"),
                         (dict(H=6, qs=384), b"group size"), (dict(H=4097, Hkv=4097), b"num_heads"),
                         (dict(M=0), b"max_pages"), (dict(M=1 << 25), b"max_pages"), (dict(mx=-1), b"max_kv_len"),
                         (dict(qs=248), b"strides"), (dict(qs=260), b"16 bytes"), (dict(q=AT[0] + 2), b"16 bytes"),
                         (dict(out=AT[1] + 8), b"16 bytes"), (dict(scale=float("inf")), b"scale"),
                         (dict(scale=float("nan")), b"scale")]:
            _refused(fn, kw, text)
    _refused(_prefill, dict(T=0), b"tokens")
    _refused(_prefill, dict(T=1 << 30), b"tokens")


def test_sizes_are_checked_in_64_bits():
    """Heads and dims whose low 32 bits would pass, and pools whose size would wrap."""
    for fn in (_decode, _prefill):
        for kw, text in [(dict(Hkv=(1 << 32) + 2), b"divisible"), (dict(D=(1 << 32) + 64, qs=1 << 40), b"head_dim"),
                         (dict(H=(1 << 32) + 4, qs=1 << 40), b"num_heads"),
                         (dict(B=(1 << 32) + 1), b"batch")]:
            _refused(fn, kw, text)
    for fn in (_quant, _dequant):
        for kw, text in [(dict(Hkv=(1 << 32) + 2), b"num_kv_heads"), (dict(D=(1 << 32) + 64), b"head_dim"),
                         (dict(T=(1 << 32) + 1), b"tokens")]:
            _refused(fn, kw, text)
    for fn in (_quant, _dequant, _decode, _prefill):
        for kw in (dict(P=1 << 20, NP=(1 << 20) + 1), dict(P=(1 << 32) + 64), dict(blk=(1 << 32) + 32), dict(NP=(1 << 32) + 4)):
            _refused(fn, kw, b"page_size", b"block_size")


def test_workspaces_are_checked_before_any_launch():
    lib = _hip.lib()
    need = lib.ezops_quant_paged_attn_decode_workspace_size(2, 4, 2, 64, 128)
    assert need == 0 and lib.ezops_quant_paged_attn_decode_workspace_size(2, 4, 2, 64, 0) == 0
    need = lib.ezops_quant_paged_attn_decode_workspace_size(2, 4, 2, 64, 4096)
    assert 0 < need < 1 << 24
    for kw in (dict(ws=None), dict(nb=need - 1), dict(ws=AT[9] + 8), dict(ws=AT[1]), dict(ws=AT[3] + 64), dict(ws=AT[8])):
        _refused(_decode, dict(M=64, NP=200, **kw), b"workspace")
    # a bound on the lengths plans the work: what is enough for it may be too little without it
    short = lib.ezops_quant_paged_attn_decode_workspace_size(2, 4, 2, 64, 256)
    assert 0 < short < need
    _refused(_decode, dict(M=64, NP=200, nb=short), b"workspace too small")
    need = lib.ezops_quant_prefill_attn_workspace_size(2, 8, 4, 2, 64, 8192)
    assert need > 0 and lib.ezops_quant_prefill_attn_workspace_size(2, 8, 4, 2, 64, 64) == 0
    for kw in (dict(ws=None), dict(nb=need - 1), dict(ws=AT[9] + 8), dict(ws=AT[0] + 16), dict(ws=AT[7])):
        _refused(_prefill, dict(M=128, NP=300, **kw), b"workspace")
    # many sequences stay whole, so that the workspace does not grow with them
    for B in (1, 7, 64, 300, 1024):
        assert lib.ezops_quant_paged_attn_decode_workspace_size(B, 32, 8, 128, 1 << 20) <= (B + 96 + B // 2) * 32 * 520 + B * 64 + 1024
    assert lib.ezops_quant_paged_attn_decode_workspace_size(1025, 32, 8, 128, 1 << 20) == 0


def test_c_entries_reject_overlaps():
    pool, sc = 4 * 2 * 64 * 64, 4 * 2 * 2
    for kw in (dict(K=AT[0]), dict(V=AT[1] - pool + 16), dict(Ks=AT[2] + 8), dict(Vs=AT[0] + 256), dict(K=AT[2] - 16)):
        _refused(_quant, kw, b"overlaps an input")
    for kw in (dict(K=AT[4] + 16), dict(Ks=AT[3] + pool - 1), dict(Vs=AT[5] + sc - 1), dict(V=AT[6] - 16)):
        _refused(_quant, kw, b"caches and scales overlap")
    for kw in (dict(ko=AT[3]), dict(vo=AT[4] + pool - 16), dict(ko=AT[5]), dict(vo=AT[6] - 16), dict(ko=AT[2] + 48)):
        _refused(_dequant, kw, b"overlaps an input")
    _refused(_dequant, dict(vo=AT[0] + 16), b"outputs overlap")
    for fn in (_decode, _prefill):
        for kw in (dict(out=AT[0]), dict(out=AT[3] + 64), dict(out=AT[4] - 16), dict(out=AT[5]), dict(out=AT[6] - 16),
                   dict(out=AT[7]), dict(out=AT[8])):
            _refused(fn, kw, b"out overlaps an input")
    _refused(_prefill, dict(past=AT[1] + 16), b"out overlaps an input")


def _np(t):
    return t.detach().double().numpy()


def _bytes(t):
    return t.view(torch.uint8).numpy()


SPECIAL = [0.0, -0.0, 1.0, -127.0, 127.5, 448.0, -449.0, 464.0, 3e38, -1e-38, 2.0 ** -20, 1e-30]


def _tokens(g, n, Hkv, D, wide):
    x = torch.randn(n, Hkv, D, generator=g)
    if wide:
        x = x * torch.exp2(torch.randint(-12, 12, (n, 1, 1), generator=g).float())
        x.view(-1)[torch.randint(0, x.numel(), (7,), generator=g)] = torch.tensor(SPECIAL)[torch.randint(0, 12, (7,), generator=g)]
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("block,P", [(16, 32), (32, 32), (64, 64), (256, 256)])
def test_ref_quant(kind, block, P):
    """Several calls that fill sequences piece by piece against the oracle, and the read-back."""
    Hkv, D, pages = 2, 64, 5
    g = torch.Generator().manual_seed(block)
    pools = KvCacheQuantOp(1, Hkv, D, P, pages, cache_dtype=KINDS[kind], block_size=block).alloc("cpu")
    for p in pools:
        p.view(torch.uint8).random_(0, 255, generator=g)
    o = [_bytes(p).copy() for p in pools]
    at = 3
    for n in (1, 1, 5, 14, block, 2, 1, 40):
        n = min(n, 2 * P - at)
        slots = torch.tensor([(3 if (at + i) < P else 1) * P + (at + i) % P for i in range(n)] + [-1, pages * P, -P])
        at += n
        T = slots.numel()
        k, v = _tokens(g, T, Hkv, D, True), _tokens(g, T, Hkv, D, False)
        op = KvCacheQuantOp(T, Hkv, D, P, pages, cache_dtype=KINDS[kind], block_size=block)
        assert op(k, v, *pools, slots)[0] is pools[0]
        for x, c, s in ((k, 0, 2), (v, 1, 3)):
            kv8.write(_np(x), o[c], o[s], slots.tolist(), block, kind)
        for p, want in zip(pools, o):
            np.testing.assert_array_equal(_bytes(p), want)
    slots = torch.tensor([3 * P + 3, P - 1, -1, 3 * P + 3, pages * P])
    back = KvCacheDequantOp(5, Hkv, D, P, pages, cache_dtype=KINDS[kind], block_size=block)
    out = [torch.full((5, Hkv, D), 7.0, dtype=torch.bfloat16) for _ in range(2)]
    back(*pools, slots, k_out=out[0], v_out=out[1])
    for x, c, s in ((out[0], 0, 2), (out[1], 1, 3)):
        for i, slot in enumerate(slots.tolist()):
            for h in range(Hkv):
                if not 0 <= slot < pages * P:
                    assert (x[i, h] == 7).all()
                    continue
                page, row = divmod(slot, P)
                want = kv8.decode(o[c][page, h, row], o[s][page, h, row // block], kind)
                want = torch.tensor(want).to(torch.bfloat16)  # exact but for exponents that no write makes
                assert torch.equal(x[i, h].nan_to_num(5.0), want.nan_to_num(5.0))


@pytest.mark.parametrize("kind", KINDS)
def test_not_finite(kind):
    """A NaN code of its own (e4m3); the block's exponent, until its first row is written again (int8)."""
    Hkv, D, P, block = 2, 64, 32, 16
    op = KvCacheQuantOp(2, Hkv, D, P, 2, cache_dtype=KINDS[kind], block_size=block)
    pools = op.alloc("cpu")
    x = torch.ones(2, Hkv, D, dtype=torch.bfloat16)
    bad = x.clone()
    bad[1, 0, 3], bad[1, 0, 5] = float("nan"), float("-inf")
    o = [_bytes(p).copy() for p in pools]
    for tokens, slots in ((x, [0, 1]), (bad, [2, 3]), (x * 3, [4, 5]), (x, [0, 1])):
        op(tokens, tokens, *pools, torch.tensor(slots))
        for c, s in ((0, 2), (1, 3)):
            kv8.write(_np(tokens), o[c], o[s], slots, block, kind)
        for p, want in zip(pools, o):
            np.testing.assert_array_equal(_bytes(p), want)
        if slots == [4, 5]:
            k, _ = KvCacheDequantOp(6, Hkv, D, P, 2, cache_dtype=KINDS[kind], block_size=block)(*pools, torch.arange(6))
            nan = torch.zeros(6, Hkv, D, dtype=torch.bool)
            if kind == "int8":
                nan[:, 0] = True
            else:
                nan[3, 0, 3] = nan[3, 0, 5] = True
            assert torch.equal(k.isnan(), nan)
    assert int(pools[2][0, 0, 0]) < 255


@pytest.mark.parametrize("kind", KINDS)
def test_error_of_a_row_after_many_growths(kind):
    """A block grown token by token, each twice as large as the one before: int8 rows are within one step of the present
    scale; e4m3 rows within half a step of four bits and, below 2^-6 of a scale, of the smallest code, 2^-10, twice."""
    Hkv, D, P = 1, 64, 32
    op = KvCacheQuantOp(1, Hkv, D, P, 1, cache_dtype=KINDS[kind], block_size=32)
    pools = op.alloc("cpu")
    g = torch.Generator().manual_seed(3)
    x = (torch.rand(32, Hkv, D, generator=g) * 2 - 1) * torch.exp2(torch.arange(32) / 2)[:, None, None]
    x = x.to(torch.bfloat16)
    for t in range(32):
        op(x[t:t + 1], x[t:t + 1], *pools, torch.tensor([t]))
    k, _ = KvCacheDequantOp(32, Hkv, D, P, 1, cache_dtype=KINDS[kind], block_size=32)(*pools, torch.arange(32))
    step = 2.0 ** (int(pools[2][0, 0, 0]) - 127)
    err, a = (k.double() - x.double()).abs(), x.double().abs()
    assert (err <= (step if kind == "int8" else torch.maximum(a * 2.0 ** -4, torch.tensor(step * 2.0 ** -9)))).all()


def _case(kind, H, Hkv, D, P, block, M, seed):
    g = torch.Generator().manual_seed(seed)
    pages = 2 * M + 1
    pools = KvCacheQuantOp(1, Hkv, D, P, pages, cache_dtype=KINDS[kind], block_size=block).alloc("cpu")
    for c, s in ((0, 2), (1, 3)):
        kv8_x = torch.randn(pages * P, Hkv, D, generator=g)
        kv8.write(_np(kv8_x), _bytes(pools[c]), _bytes(pools[s]), range(pages * P), block, kind)
    return g, pools, torch.randperm(pages, generator=g)[:2 * M].reshape(2, M).to(torch.int32)


@pytest.mark.parametrize("kind", KINDS)
def test_ref_attention(kind):
    H, Hkv, D, P, block, M = 4, 2, 64, 32, 16, 2
    g, pools, table = _case(kind, H, Hkv, D, P, block, M, 5)
    held = [[kv8.rows(_bytes(pools[c]), _bytes(pools[s]), table[b], M * P, block, kind) for c, s in ((0, 2), (1, 3))]
            for b in range(2)]
    q = torch.randn(2, H, D, generator=g).to(torch.bfloat16)
    how = dict(cache_dtype=KINDS[kind], block_size=block)
    op = QuantPagedAttnDecodeOp(2, H, Hkv, D, P, M, 2 * M + 1, **how)
    for lens, mx in (([33, 0], 0), ([1, 64], 0), ([99, 50], 40)):
        out = op(q, *pools, table, torch.tensor(lens, dtype=torch.int32), mx)
        for b, n in enumerate(lens):
            n = min(n, mx or 64)
            want = kv8.attend(_np(q[b:b + 1]), held[b][0][:n], held[b][1][:n], n - 1, D ** -0.5)[0][0] if n else 0 * _np(q[b])
            np.testing.assert_allclose(_np(out[b]), want, rtol=2 ** -8, atol=1e-5)
    T = 30
    q = torch.randn(T, H, D, generator=g).to(torch.bfloat16)
    op = QuantPrefillAttnOp(2, T, H, Hkv, D, P, M, 2 * M + 1, **how, scale=0.2)
    cu, past = torch.tensor([2, 13, 28], dtype=torch.int32), torch.tensor([20, 55], dtype=torch.int32)
    out = torch.full((T, H, D), 7.0, dtype=torch.bfloat16)
    assert op(q, *pools, table, cu, past, out=out) is out
    written = list(range(2, 13)) + list(range(13, 22))  # 9 of the second's 15 tokens stand inside the cache
    for b, (s, n) in enumerate(((2, 11), (13, 9))):
        p = int(past[b])
        want = kv8.attend(_np(q[s:s + n]), held[b][0][:p + n], held[b][1][:p + n], p, 0.2)[0]
        np.testing.assert_allclose(_np(out[s:s + n]), want, rtol=2 ** -8, atol=1e-5)
    rest = [t for t in range(T) if t not in written]
    assert (out[rest] == 7).all()


def test_rooflines_and_gen_data():
    q = KvCacheQuantOp(100, 2, 64, 64, 3)
    assert q.get_roofline().bytes == 100 * (6 * 128 + 8) + 2 * 4 * 2
    out = q(*q.gen_data("cpu"))
    assert q.check(out, out)
    d = KvCacheDequantOp(100, 2, 64, 64, 1, cache_dtype=torch.float8_e4m3fn)
    k, v = d(*d.gen_data("cpu"))
    assert k.shape == (100, 2, 64) and (k[:64] != 0).any()
    a = QuantPagedAttnDecodeOp(2, 4, 2, 64, 32, 4, cache_dtype=torch.float8_e4m3fn)
    assert a.get_roofline().bytes == 2 * (128 * 2 * 128 + 2 * 2 * 4 + 4 * 4 * 64 + 4 * 4 + 4)
    assert a(*a.gen_data("cpu")).shape == (2, 4, 64)
    p = QuantPrefillAttnOp(3, 20, 4, 2, 64, 32, 4)
    assert p.get_roofline().flops == 2 * 3 * 6 * 7 * 4 * 64
    assert p(*p.gen_data("cpu")).isfinite().all()
