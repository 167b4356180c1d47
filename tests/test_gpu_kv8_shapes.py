"""tree_attention_q8 in every launch shape that it has: head size x codes x column tiles a wave x waves that share a tile's
keys x key splits, for chains and trees, with and without the second segment, cached and past the caches.

Bar: that of tests/test_gpu_kv8_attn.py."""
import math

import numpy as np
import pytest
import torch

import kv8_ref as R
from versenext_amd import tree as VT

pytestmark = pytest.mark.gpu

I8, E4 = torch.int8, torch.float8_e4m3fn
SHAPES = [(d, ct, kw) for d in (64, 128) for ct in range(1, 256 // d + 1) for kw in (1, 2, 4, 8)]


def _close(o, ref, mag, what):
    half = 2.0 ** -8 if o.dtype == torch.bfloat16 else 2.0 ** -11
    err = (o.cpu().to(R.F64) - ref).abs()
    worst = (err / (2.0 ** -10 * mag + half * ref.abs() + 2.0 ** -25)).max().item()
    assert torch.isfinite(o).all() and worst <= 1.0, (what, worst)


def _attend(q, k, v, sees):
    """(out, mag) in 64 bits; q (H, N, d), k and v (Hkv, T, d), sees (N, T); zeros where a node sees nothing."""
    rep = q.shape[0] // k.shape[0]
    k, v = k.repeat_interleave(rep, 0), v.repeat_interleave(rep, 0)
    s = (q.to(R.F64) @ k.transpose(-1, -2) / math.sqrt(q.shape[-1])).masked_fill(~sees, -math.inf)
    p = torch.softmax(s, -1).nan_to_num(0.0)
    return p @ v, p @ v.abs()


def _sees(N, t, words, window):
    node = torch.arange(N)
    if words is None:
        bits, depth = torch.tril(torch.ones(N, N, dtype=torch.bool)), node
    else:
        bits = torch.tensor([[bool(w >> j & 1) for j in range(N)] for w in words])
        depth = bits.sum(1) - 1
    ok = torch.cat([torch.ones(N, t, dtype=torch.bool), bits], 1)
    place = torch.cat([torch.arange(t), t + depth])
    return ok & ((t + depth)[:, None] - place[None] < window) if window else ok


def _case(hip, d, dtype, H, Hkv, N, lens, words, window, G, shapes, seed):
    """One set of inputs through several (tiles, waves, splits)."""
    dev = hip.torch_device
    B, Tp = len(lens), max(lens)
    g = R.gen(seed)
    (kc, ks), (vc, vs) = (R.cache(g, B, Hkv, Tp + N, d, dtype) for _ in range(2))
    q = (torch.randn(B, H, N, d, generator=g) * 1.5).to(torch.bfloat16)
    k, v = R.values(kc, ks), R.values(vc, vs)
    seg2 = gates = None
    if G:
        seg2 = tuple(torch.randn(1, Hkv, G, d, generator=g).to(torch.bfloat16) for _ in range(2))
        gates = torch.tensor([0.7, -0.4])
    both = []
    for b, t in enumerate(lens):
        o, m = _attend(q[b], k[b, :, :t + N], v[b, :, :t + N], _sees(N, t, words, window))
        if G:
            o2, m2 = _attend(q[b], seg2[0][0].to(R.F64), seg2[1][0].to(R.F64), torch.ones(N, G, dtype=torch.bool))
            g0, g1 = gates.to(R.F64)
            o, m = g0 * o + g1 * o2, g0.abs() * m + g1.abs() * m2
        both.append((o, m))
    ref, mag = (torch.stack(x) for x in zip(*both))
    for b, t in enumerate(lens):       # NaN behind every sequence's last row
        for c, s in ((kc, ks), (vc, vs)):
            c[b, :, t + N:].view(torch.uint8).fill_(0x7F)
            s[b, :, t + N:] = math.nan
    args = [x.to(dev) for x in (q, kc, vc, ks, vs)]
    anc = None if words is None else np.array(words, dtype=np.uint64)
    for tiles, waves, splits in shapes:
        what = f"d={d} {dtype} N={N} window={window} G={G} tree={words is not None} tiles={tiles} waves={waves} splits={splits}"
        print(what, flush=True)
        o = hip.tree_attention_q8(*args, lens, anc=anc, window=window, seg2=seg2, gates=gates, max_len=Tp,
                                  out_dtype=torch.float16, force_tiles=tiles, force_waves=waves, force_splits=splits)
        _close(o, ref, mag, what)


def _splits(kw):
    return (1,) if kw < 4 else (1, 2, 32)


@pytest.mark.parametrize("dtype", [I8, E4], ids=["int8", "e4m3"])
@pytest.mark.parametrize("d,ct,kw", SHAPES)
def test_chain(hip, d, ct, kw, dtype):
    """More than one column group with an odd rest, and fewer columns than a tile."""
    shapes = [(ct, kw, s) for s in _splits(kw)]
    for N, lens in ((150, [300, 0]), (3, [37, 700])):
        for window, G in ((0, 0), (70, 0), (70, 37), (0, 5)):
            if not G or kw <= 4:
                _case(hip, d, dtype, 6, 2, N, lens, None, window, G, shapes, N + ct)


@pytest.mark.parametrize("dtype", [I8, E4], ids=["int8", "e4m3"])
@pytest.mark.parametrize("d,ct,kw", [s for s in SHAPES if s[2] >= 4])
def test_tree(hip, d, ct, kw, dtype):
    """A tree of 40 nodes and one of 7, four query heads a KV head; a node that sees the prefix alone."""
    shapes = [(ct, kw, s) for s in _splits(kw)]
    for tree, lens in (((4, 3, 2), [300, 0]), ((1, 2, 2), [33, 500])):
        words = [int(w) for w in VT.ancestor_words(VT.tree_from_branching(list(tree)))]
        words[-1] = 0
        for window, G in ((0, 0), (64, 0), (64, 37), (0, 5)):
            if not G or kw <= 4:
                _case(hip, d, dtype, 8, 2, len(words), lens, words, window, G, shapes, ct)


@pytest.mark.parametrize("dtype", [I8, E4], ids=["int8", "e4m3"])
@pytest.mark.parametrize("tree", [False, True], ids=["chain", "tree"])
@pytest.mark.parametrize("ct", [1, 2])
@pytest.mark.parametrize("d", [64, 128])
def test_past_the_caches(hip, d, ct, tree, dtype):
    """192 MiB of rows and more that one column group reads; every head and sequence shares one head's rows (strides of 0)."""
    dev = hip.torch_device
    rep, Hkv, Tp, G, B = 4, 8, 16001, 40, 16 if d == 64 else 8
    words = [int(w) for w in VT.ancestor_words(VT.tree_from_branching([2, 1]))] if tree else None
    N = len(words) if tree else 4 * ct - 1
    assert B * Hkv * Tp * 2 * d >= 192 << 20 and rep * N <= 16 * ct
    g = R.gen(d + ct)
    (kc, ks), (vc, vs) = (R.cache(g, 1, 1, Tp + N + 32, d, dtype) for _ in range(2))
    for c, s in ((kc, ks), (vc, vs)):
        c[:, :, Tp + N:].view(torch.uint8).fill_(0x7F)
        s[:, :, Tp + N:] = math.nan
    q = torch.randn(B, rep * Hkv, N, d, generator=g).to(torch.bfloat16)
    seg2 = tuple(torch.randn(1, Hkv, G, d, generator=g).to(torch.bfloat16) for _ in range(2))
    gates = torch.tensor([0.6, 0.5])
    lens = [Tp, 0, 15970] + [Tp - 17 * b for b in range(B - 3)]
    wide = [t.to(dev).expand(B, Hkv, *t.shape[2:]) for t in (kc, vc, ks, vs)]
    k, v = R.values(kc[0], ks[0]), R.values(vc[0], vs[0])
    want = {}
    for b in (0, 1, 2, B - 1):
        t = lens[b]
        for h in (0, Hkv - 1):
            at = slice(h * rep, (h + 1) * rep)
            a = _attend(q[b, at], k[:, :t + N], v[:, :t + N], _sees(N, t, words, 0))
            s = _attend(q[b, at], seg2[0][0, h:h + 1].to(R.F64), seg2[1][0, h:h + 1].to(R.F64),
                        torch.ones(N, G, dtype=torch.bool))
            want[b, at.start] = a, [0.6 * x + 0.5 * y for x, y in zip(a, s)]
    anc = np.array(words, dtype=np.uint64) if tree else None
    for waves, two in ((4, False), (8, False), (4, True)):
        for splits in (1, 4):
            what = f"d={d} {dtype} tree={tree} tiles={ct} waves={waves} splits={splits} seg2={two}"
            print(what, flush=True)
            o = hip.tree_attention_q8(q, *wide, lens, anc=anc, max_len=Tp, force_tiles=ct, force_waves=waves,
                                      force_splits=splits, seg2=seg2 if two else None, gates=gates if two else None)
            for (b, h), r in want.items():
                _close(o[b, h:h + rep], *r[two], what)


def test_the_plan_is_one_of_them(hip):
    """An unforced call gives the bits of the shape that it takes; forcing one field leaves the others to the plan."""
    dev = hip.torch_device
    g = R.gen(1)
    (kc, ks), (vc, vs) = (R.cache(g, 2, 2, 500, 64, I8) for _ in range(2))
    args = [t.to(dev) for t in (torch.randn(2, 4, 5, 64, generator=g).to(torch.bfloat16), kc, vc, ks, vs)]
    one = hip.tree_attention_q8(*args, [495, 100])
    every = [hip.tree_attention_q8(*args, [495, 100], force_tiles=1, force_waves=w, force_splits=s)
             for w in (1, 2, 4, 8) for s in _splits(w) + ((4, 8, 16) if w >= 4 else ())]
    assert any(torch.equal(one, o) for o in every)
    for kw in (dict(force_tiles=1), dict(force_waves=4), dict(force_splits=1), dict(force_splits=4), dict(force_tiles=4)):
        assert (hip.tree_attention_q8(*args, [495, 100], **kw) - one).abs().max() <= 2.0 ** -6 * one.abs().max()


def test_refusals(hip):
    dev = hip.torch_device
    kc = torch.zeros(1, 1, 9, 128, dtype=I8, device=dev)
    ks = torch.ones(1, 1, 9, device=dev)
    q = torch.zeros(1, 1, 1, 128, dtype=torch.bfloat16, device=dev)
    s2 = torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16, device=dev)
    for kw in (dict(force_tiles=3), dict(force_tiles=-1), dict(force_waves=3), dict(force_waves=16), dict(force_waves=-4),
               dict(force_splits=3), dict(force_splits=64), dict(force_splits=-1), dict(force_waves=2, force_splits=2),
               dict(force_waves=2, anc=[1]), dict(force_waves=8, seg2=(s2, s2), gates=[1.0, 1.0])):
        with pytest.raises(ValueError):
            hip.tree_attention_q8(q, kc, kc, ks, ks, [3], **kw)


@pytest.mark.parametrize("dtype", [I8, E4], ids=["int8", "e4m3"])
@pytest.mark.parametrize("d,H,Hkv,N,lens,tree,window,G", [
    (64, 40, 1, 3, [90, 0], None, 0, 0), (128, 33, 1, 1, [200, 31], None, 17, 3), (64, 34, 2, 70, [5, 64], None, 33, 40),
    (64, 24, 1, 0, [100, 3], (4, 3, 2), 40, 0), (128, 32, 2, 0, [64, 0], (2, 2, 2, 2), 30, 9)])
def test_many_query_heads_to_a_kv_head(hip, d, H, Hkv, N, lens, tree, window, G, dtype):
    """17 to 40 query heads a KV head, so a column tile holds one node or a part of one; trees with the smallest window."""
    words = [int(w) for w in VT.ancestor_words(VT.tree_from_branching(list(tree)))] if tree else None
    _case(hip, d, dtype, H, Hkv, len(words) if tree else N, lens, words, window, G,
          [(0, 0, 0), (1, 4, 1), (2, 4, 4)] + ([] if tree else [(1, 1, 1), (2, 2, 1)]), H)
