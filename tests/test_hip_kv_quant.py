"""Cache rows into 8 bits and back on the GPU, against ``oracle.kv8`` (codes, exponents and values: equal, byte by byte)."""

import numpy as np
import pytest
import torch

from ezops import KvCacheDequantOp, KvCacheQuantOp
from oracle import kv8

pytestmark = pytest.mark.gpu
DEV = "cuda"
KINDS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
SPECIAL = [0.0, -0.0, 1.0, -127.0, 127.5, 448.0, -449.0, 464.0, 3e38, -1e-38, 2.0 ** -20, 1e-30]


def n64(x):
    return x.detach().double().cpu().numpy()


def raw(x):
    return x.view(torch.uint8).cpu().numpy()


def tokens(g, T, Hkv, D, wide, packed=0):
    """k and v [T, Hkv, D], with ``packed`` as slices of rows of that many heads more."""
    x = torch.randn(T, 2 * Hkv + packed, D, generator=g)
    if wide:
        x = x * torch.exp2(torch.randint(-12, 12, (T, x.shape[1], 1), generator=g).float())
        x.view(-1)[torch.randint(0, x.numel(), (40,), generator=g)] = torch.tensor(SPECIAL)[torch.randint(0, 12, (40,), generator=g)]
    x = x.to(torch.bfloat16).to(DEV)
    k, v = x[:, packed:packed + Hkv], x[:, packed + Hkv:]
    return (k, v) if packed else (k.contiguous(), v.contiguous())


def junk_pools(g, op):
    pools = op.alloc(DEV)
    for p in pools:
        p.view(torch.uint8).copy_(torch.randint(0, 256, p.shape, generator=g, dtype=torch.uint8))
    return pools


def plan(lens, P, order):
    """Slots of new tokens: (new, past) of every sequence, pages from ``order``."""
    out = []
    for new, past in lens:
        pages = [order.pop() for _ in range(-(-(new + past) // P))]
        out += [pages[r // P] * P + r % P for r in range(past, past + new)]
    return out


LENS = {
    "single tokens": [(1, p) for p in (0, 1, 15, 16, 17, 31, 32, 63, 64, 65, 127, 128)],
    "prompts": [(1, 0), (2, 0), (15, 0), (16, 0), (17, 0), (33, 0), (64, 0), (65, 0), (257, 0), (300, 0)],
    "chunks": [(0, 5), (40, 3), (1, 31), (64, 30), (130, 200), (7, 9), (100, 1)],
}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("block,P,Hkv,D,packed", [(16, 32, 2, 64, 3), (32, 32, 8, 128, 32), (64, 64, 1, 128, 0), (128, 128, 3, 64, 0),
                                                  (256, 256, 2, 128, 1), (16, 256, 5, 128, 0), (32, 128, 2, 64, 0)])
def test_quant_matches_the_oracle(kind, lens, block, P, Hkv, D, packed):
    """Fresh blocks, blocks begun before (of random codes and exponents), slots outside the pool between the runs."""
    g = torch.Generator().manual_seed(P + block)
    lens = LENS[lens]
    pages = sum(-(-(a + b) // P) for a, b in lens) + 2
    slots = plan(lens, P, torch.randperm(pages, generator=g).tolist())
    half = sum(a for a, _ in lens[:len(lens) // 2])  # between two sequences: a block's tokens stay in one run
    for i, at in enumerate((len(slots), half, 0)):
        slots[at:at] = [-1, pages * P, -(1 << 40), 1 << 40][i:][:2]
    T = len(slots)
    op = KvCacheQuantOp(T, Hkv, D, P, pages, backend="hip", cache_dtype=KINDS[kind], block_size=block)
    pools = junk_pools(g, op)
    pools[2][:, :, ::2], pools[3][:, :, 1::2] = 125, 121  # exponents that writes make; the others are anything
    k, v = tokens(g, T, Hkv, D, True, packed)
    want = [raw(p).copy() for p in pools]
    for x, c, s in ((k, 0, 2), (v, 1, 3)):
        kv8.write(n64(x), want[c], want[s], slots, block, kind)
    got = op(k, v, *pools, torch.tensor(slots, device=DEV))
    for name, p, q, w in zip(("K", "V", "Ks", "Vs"), pools, got, want):
        assert p is q
        np.testing.assert_array_equal(raw(p), w, err_msg=name)


@pytest.mark.parametrize("kind", KINDS)
def test_not_finite(kind):
    Hkv, D, P, block = 3, 128, 64, 32
    g = torch.Generator().manual_seed(4)
    op = KvCacheQuantOp(40, Hkv, D, P, 3, backend="hip", cache_dtype=KINDS[kind], block_size=block)
    pools = op.alloc(DEV)
    want = [raw(p).copy() for p in pools]
    for first, bad in ((0, [(3, 0), (35, 1)]), (40, []), (70, [(0, 2)]), (0, [])):
        k, v = tokens(g, 40, Hkv, D, False)
        for t, h in bad:
            k[t, h, 7], v[t, h, 100] = float("nan"), -float("inf")
        slots = list(range(first, first + 40))
        for x, c, s in ((k, 0, 2), (v, 1, 3)):
            kv8.write(n64(x), want[c], want[s], slots, block, kind)
        op(k, v, *pools, torch.tensor(slots, device=DEV))
        for p, w in zip(pools, want):
            np.testing.assert_array_equal(raw(p), w)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("block", [16, 32, 64, 128, 256])
def test_every_block_and_head_size(kind, D, block):
    """Runs that begin, go on, fill and leave a block, single tokens between them, and values that are not finite."""
    Hkv, P = 2, 256
    g = torch.Generator().manual_seed(block + D)
    lens = [(block // 2 - 1, 0), (1, 3), (2 * block + 5, block - 7), (1, block - 1), (block, 0), (P - 1, 1), (3, 0), (0, 9)]
    slots = plan(lens, P, torch.randperm(20, generator=g).tolist())
    T = len(slots)
    op = KvCacheQuantOp(T, Hkv, D, P, 20, backend="hip", cache_dtype=KINDS[kind], block_size=block)
    pools = junk_pools(g, op)
    pools[2][:, :, ::2], pools[3][:, :, 1::2] = 125, 121
    want = [raw(p).copy() for p in pools]
    for bad in ((), (0, T // 3, T // 2, T - 1)):
        k, v = tokens(g, T, Hkv, D, False)
        for t in bad:
            k[t, 0, 7], v[t, 1, D - 1], v[t, 0, 0] = float("nan"), float("inf"), -float("inf")
        for x, c, s in ((k, 0, 2), (v, 1, 3)):
            kv8.write(n64(x), want[c], want[s], slots, block, kind)
        op(k, v, *pools, torch.tensor(slots, device=DEV))
        for name, p, w in zip(("K", "V", "Ks", "Vs"), pools, want):
            np.testing.assert_array_equal(raw(p), w, err_msg=name)


@pytest.mark.parametrize("kind", KINDS)
def test_growth_token_by_token(kind):
    """Blocks that grow at nearly every token, as decode steps do it."""
    B, Hkv, D, P, block = 7, 2, 128, 64, 64
    g = torch.Generator().manual_seed(5)
    op = KvCacheQuantOp(B, Hkv, D, P, B, backend="hip", cache_dtype=KINDS[kind], block_size=block)
    pools = op.alloc(DEV)
    want = [raw(p).copy() for p in pools]
    for t in range(48):
        k, v = tokens(g, B, Hkv, D, False)
        k, v = k * 1.4 ** t, v * 1.9 ** (t % 20)
        slots = [b * P + t for b in range(B)]
        for x, c, s in ((k, 0, 2), (v, 1, 3)):
            kv8.write(n64(x), want[c], want[s], slots, block, kind)
        op(k, v, *pools, torch.tensor(slots, device=DEV))
    for p, w in zip(pools, want):
        np.testing.assert_array_equal(raw(p), w)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("block,P,Hkv,D,T", [(16, 32, 2, 64, 1), (32, 64, 8, 128, 333), (256, 256, 1, 128, 70), (64, 128, 5, 64, 3001)])
def test_dequant_matches_the_oracle(kind, block, P, Hkv, D, T):
    """Any order, repeats, slots outside the pool; exponents from one end to the other."""
    g = torch.Generator().manual_seed(T)
    pages = 9
    op = KvCacheDequantOp(T, Hkv, D, P, pages, backend="hip", cache_dtype=KINDS[kind], block_size=block)
    pools = junk_pools(g, op)
    for s in pools[2:]:
        s.copy_(torch.randint(67, 189, s.shape, generator=g, dtype=torch.uint8))
        s[s == 188] = 255
    slots = torch.randint(0, pages * P, (T,), generator=g)
    if T > 9:
        slots[5], slots[9] = -1, pages * P
    out = [torch.full((T, Hkv, D), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    got = op(*pools, slots.to(DEV), k_out=out[0], v_out=out[1])
    fresh = op(*pools, slots.to(DEV))
    live = (slots >= 0) & (slots < pages * P)
    at = slots[live].numpy()
    for i, (c, s) in enumerate(((0, 2), (1, 3))):
        assert got[i] is out[i]
        assert (out[i][~live.to(DEV)] == 7).all()
        e = raw(pools[s])[at // P, :, at % P // block].astype(int)
        want = kv8.VALUES[kind][raw(pools[c])[at // P, :, at % P]] * np.where(e == 255, np.nan, 2.0 ** (e - 127.0))[..., None]
        np.testing.assert_array_equal(n64(out[i][live.to(DEV)]), want)  # codes times a power of two: exact in bf16
        np.testing.assert_array_equal(n64(fresh[i][live.to(DEV)]), want)


@pytest.mark.parametrize("kind", KINDS)
def test_slots_past_32_bits(kind):
    """Pools of 2.3e9 codes: the last rows of the last page."""
    Hkv, D, P, block = 8, 128, 128, 32
    pages = 17600
    op = KvCacheQuantOp(40, Hkv, D, P, pages, backend="hip", cache_dtype=KINDS[kind], block_size=block)
    pools = op.alloc(DEV)
    assert pools[0].numel() > 1 << 31
    g = torch.Generator().manual_seed(6)
    k, v = tokens(g, 40, Hkv, D, False)
    slots = torch.arange(pages * P - 40, pages * P)
    op(k, v, *pools, slots.to(DEV))
    small = [torch.zeros((1, *p.shape[1:]), dtype=torch.uint8).numpy() for p in pools]
    for x, c, s in ((k, 0, 2), (v, 1, 3)):
        kv8.write(n64(x), small[c], small[s], range(P - 40, P), block, kind)
    for p, w in zip(pools, small):
        np.testing.assert_array_equal(raw(p[-1:]), w)
        assert not p[:-1].view(torch.uint8)[::97].any()
    back = KvCacheDequantOp(40, Hkv, D, P, pages, backend="hip", cache_dtype=KINDS[kind], block_size=block)(*pools, slots.to(DEV))
    for x, c, s in ((back[0], 0, 2), (back[1], 1, 3)):
        want = kv8.rows(small[c], small[s], [0], P, block, kind)[P - 40:]
        np.testing.assert_array_equal(n64(x), want)


def test_other_blocks_stay_as_they_are_where_a_block_comes_twice():
    """Two runs of one block, and one slot twice: that block is undefined, nothing else moves."""
    Hkv, D, P, block = 2, 64, 32, 16
    g = torch.Generator().manual_seed(7)
    op = KvCacheQuantOp(6, Hkv, D, P, 3, backend="hip", block_size=block)
    pools = junk_pools(g, op)
    before = [raw(p).copy() for p in pools]
    k, v = tokens(g, 6, Hkv, D, False)
    op(k, v, *pools, torch.tensor([34, 35, 40, 41, 41, 36], device=DEV))  # page 1, its first block
    for p, b in zip(pools, before):
        now = raw(p)
        if p.dim() == 4:
            np.testing.assert_array_equal(now[[0, 2]], b[[0, 2]])
            np.testing.assert_array_equal(now[1, :, 16:], b[1, :, 16:])
        else:
            np.testing.assert_array_equal(now[[0, 2]], b[[0, 2]])
            np.testing.assert_array_equal(now[1, :, 1], b[1, :, 1])


def test_refusals_on_the_gpu():
    op = KvCacheQuantOp(4, 2, 64, 32, 3, backend="hip")
    k, v, *pools, slots = op.gen_data(DEV)
    bad = [(k[:3], v, *pools, slots), (k.float(), v, *pools, slots), (k, v[:, :1], *pools, slots),
           (k, v, pools[0].view(torch.uint8), *pools[1:], slots), (k, v, *pools[:2], pools[2].to(torch.int32), pools[3], slots),
           (k, v, *pools, slots.to(torch.int32)), (k.transpose(1, 2), v, *pools, slots), (k, v, *pools[:2], pools[2][:1], pools[3], slots),
           (k, v, pools[0].transpose(1, 2), *pools[1:], slots)]
    for args in bad:
        with pytest.raises(ValueError):
            op(*args)
    wide = torch.zeros(4, 2 * 64 + 4, dtype=torch.bfloat16, device=DEV)
    for x in (wide[:, 4:].unflatten(1, (2, 64)), wide[:, :128].unflatten(1, (2, 64))):
        with pytest.raises(ValueError, match="16 bytes"):
            op(x, v, *pools, slots)
    with pytest.raises(RuntimeError, match="GPU"):
        op(k.cpu(), v, *pools, slots)
    with pytest.raises(RuntimeError, match="overlap"):
        op(k, v, pools[0], pools[0], *pools[2:], slots)
    back = KvCacheDequantOp(4, 2, 64, 32, 3, backend="hip")
    out = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="overlap"):
        back(*pools, slots, k_out=out, v_out=out)
    with pytest.raises(ValueError):
        back(*pools, slots, k_out=out.float())
