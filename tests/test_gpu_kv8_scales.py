"""tree_attention_q8 where the value rows' scales lie far apart, and where they are not finite.

Bar: that of tests/test_gpu_kv8_attn.py, whatever the scales: mag is the sum over the rows that a node sees, so a row that it
does not see may not cost it a bit."""
import math

import numpy as np
import pytest
import torch

import kv8_ref as R
from versenext_amd import tree as VT

pytestmark = pytest.mark.gpu

I8, E4 = torch.int8, torch.float8_e4m3fn


def _bar(o, ref, mag):
    half = 2.0 ** -8 if o.dtype == torch.bfloat16 else 2.0 ** -11
    err = (o.cpu().to(R.F64) - ref).abs()
    ok = err <= 2.0 ** -10 * mag + half * ref.abs() + 2.0 ** -25
    assert ok.all(), (err / (2.0 ** -10 * mag + half * ref.abs() + 2.0 ** -25)).amax((0, 1, 3))


def _call(hip, q, kc, vc, ks, vs, lens, words=None, window=0, **kw):
    anc = None if words is None else np.array(words, dtype=np.uint64)
    return hip.tree_attention_q8(q, *(t.to(hip.torch_device) for t in (kc, vc, ks, vs)), lens, anc=anc, window=window, **kw)


@pytest.mark.parametrize("dtype", [I8, E4], ids=["int8", "e4m3"])
@pytest.mark.parametrize("big", [2.0 ** 14, 2.0 ** 25, 2.0 ** 33, 2.0 ** 60, 1e37])
@pytest.mark.parametrize("d", [64, 128])
def test_large_scales_of_hidden_rows(hip, d, big, dtype):
    """A later row of the chain, a sibling of the tree, a row before the window: the nodes that do not see it keep their
    bits.  (Those that see it: 1e37 * |v| * 448 is past bf16, so they are compared below 2^60.)"""
    words = [int(w) for w in VT.ancestor_words(VT.tree_from_branching([2, 2]))]
    cases = [  # (nodes, prefix, words, window, the large row, who sees it)
        (4, 40, None, 0, 42, [2, 3]), (4, 0, None, 0, 3, [3]), (70, 10, None, 0, 15, range(5, 70)),
        (len(words), 40, words, 0, 41, [i for i, w in enumerate(words) if w >> 1 & 1]),
        (3, 100, None, 8, 93, [0]), (3, 100, None, 8, 85, []), (65, 33, None, 5, 60, range(27, 32)),
        (1, 500, None, 30, 468, []), (2, 700, None, 300, 402, [0])]
    for N, T, w, window, row, sees in cases:
        print(f"d={d} big={big} {dtype} N={N} T={T} window={window} row={row}", flush=True)
        g = R.gen(row)
        (kc, ks), (vc, vs) = (R.cache(g, 1, 2, T + N, d, dtype) for _ in range(2))
        q = torch.randn(1, 4, N, d, generator=g).to(torch.bfloat16)
        vs[:, :, row] *= big
        ref, mag = R.attention(q, R.values(kc, ks), R.values(vc, vs), [T], T, w, window)
        o = _call(hip, q, kc, vc, ks, vs, [T], w, window)
        blind = [i for i in range(N) if i not in set(sees)]
        _bar(o[:, :, blind], ref[:, :, blind], mag[:, :, blind])
        if big <= 2.0 ** 60:
            _bar(o, ref, mag)


@pytest.mark.parametrize("dtype", [I8, E4], ids=["int8", "e4m3"])
def test_a_large_row_of_no_weight(hip, dtype):
    """Rows with scales 2^20 to 2^60 times the others' whose scores are so low that they add nothing: the others decide,
    before and after them in the walk, with one and with several waves."""
    d = 64
    for N, T in ((1, 100), (5, 2000), (300, 20)):
        g = R.gen(N)
        (kc, ks), (vc, vs) = (R.cache(g, 1, 1, T + N, d, dtype) for _ in range(2))
        q = torch.randn(1, 2, N, d, generator=g).abs().to(torch.bfloat16)
        for row, e, s in ((3, 20, 30.0), (T // 2, 60, 8.0), (17, 35, 5.0)):
            kc[0, 0, row] = (-torch.ones(d)).to(dtype)          # score: -sum |q| s / 8, far below the others
            ks[0, 0, row] = s
            vs[0, 0, row] *= 2.0 ** e
        ref, mag = R.attention(q, R.values(kc, ks), R.values(vc, vs), [T], T)
        _bar(_call(hip, q, kc, vc, ks, vs, [T]), ref, mag)


@pytest.mark.parametrize("dtype", [I8, E4], ids=["int8", "e4m3"])
def test_scales_of_every_size(hip, dtype):
    """Scales from 2^-100 to 2^60, rows of zeros among them; negative scales."""
    d, T = 64, 600
    g = R.gen(77)
    for lo, hi in ((-100, -60), (-60, 0), (-12, 30), (0, 60)):
        (kc, ks), (vc, vs) = (R.cache(g, 2, 2, T, d, dtype) for _ in range(2))
        vs = vs * torch.exp2(torch.randint(lo, hi, vs.shape, generator=g).float())
        vs[torch.rand(vs.shape, generator=g) < 0.1] = 0.0
        vs *= torch.where(torch.rand(vs.shape, generator=g) < 0.3, -1.0, 1.0)
        q = torch.randn(2, 4, 3, d, generator=g).to(torch.bfloat16)
        ref, mag = R.attention(q, R.values(kc, ks), R.values(vc, vs), [T - 3, 70], T - 3)
        o = _call(hip, q, kc, vc, ks, vs, [T - 3, 70]).cpu().to(R.F64)
        # (bf16 holds what is left of 2^-100; no absolute term here)
        assert ((o - ref).abs() <= 2.0 ** -10 * mag + 2.0 ** -8 * ref.abs()).all()


@pytest.mark.parametrize("dtype", [I8, E4], ids=["int8", "e4m3"])
@pytest.mark.parametrize("N,T", [(1, 0), (2, 0), (1, 1500), (3, 40), (300, 0)])
def test_columns_of_nan(hip, N, T, dtype):
    """A node whose scores are all NaN gives NaN, not zeros: a query with a NaN, keys whose scales are NaN in every row (or
    in every row of one wave's share)."""
    d = 64
    g = R.gen(N + T)
    (kc, ks), (vc, vs) = (R.cache(g, 1, 2, T + N, d, dtype) for _ in range(2))
    q = torch.randn(1, 4, N, d, generator=g).to(torch.bfloat16)
    ref, mag = R.attention(q, R.values(kc, ks), R.values(vc, vs), [T], T)
    bad = q.clone()
    bad[0, 1, N // 2, 5] = math.nan
    o = _call(hip, bad, kc, vc, ks, vs, [T])
    assert o[0, 1, N // 2].isnan().all()
    keep = torch.ones(4, N, dtype=torch.bool)
    keep[1, N // 2] = False
    _bar(o[:, keep][None], ref[:, keep][None], mag[:, keep][None])
    for rows in (slice(0, T + N), slice(0, min(32, T + N))):
        k2 = ks.clone()
        k2[0, 0, rows] = math.nan
        o = _call(hip, q, kc, vc, k2, vs, [T])
        assert o[0, :2].isnan().all()
        _bar(o[:, 2:], ref[:, 2:], mag[:, 2:])
    # the second segment
    if N < 300:
        seg2 = torch.randn(1, 2, 70, d, generator=g).to(torch.bfloat16)
        seg2[0, 1, :32] = math.nan
        o = _call(hip, q, kc, vc, ks, vs, [T], seg2=(seg2, seg2.nan_to_num()), gates=[1.0, 0.5])
        assert o[0, 2:].isnan().all() and torch.isfinite(o[0, :2]).all()
