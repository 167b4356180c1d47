"""tree_attention_q8 (vnx_tree_attn_q8) against the 64-bit form.

Bar: |out - ref| <= 2^-10 mag + half a step of the output type, mag = sum over the terms of |gate| sum_j p_j |v_j|.  2^-11
of each term is the rounding of p_j sv_j to an fp16 operand; another 2^-11 covers the fp32 scores: sums of at most 128
exact products and three multiplies, 2^-22 of |q| |k| scale log2(e) (below 2^7 here) in the exponent, and the fp32 sums."""
import math

import numpy as np
import pytest
import torch

import kv8_ref as R
from versenext_amd import tree as VT

pytestmark = pytest.mark.gpu

I8, E4 = torch.int8, torch.float8_e4m3fn
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _close(o, ref, mag):
    err = (o.cpu().to(R.F64) - ref).abs()
    bar = 2.0 ** -10 * mag + HALF[o.dtype] * ref.abs() + 2.0 ** -25
    assert torch.isfinite(o.float()).all()
    worst = (err / bar.clamp_min(1e-30)).max().item()
    assert worst <= 1.0, worst


def _poison(kc, vc, ks, vs, ends):
    """What lies behind every sequence's last row: NaN codes and scales."""
    for b, e in enumerate(ends):
        for c, s in ((kc, ks), (vc, vs)):
            c[b, :, e:].view(torch.uint8).fill_(0x7F)
            s[b, :, e:] = math.nan


def _run(hip, B, H, Hkv, d, N, lens, dtype, cap=None, words=None, window=0, G=0, gb=1, out=torch.bfloat16, seed=0,
         max_len=None, scale=None):
    dev = hip.torch_device
    Tp = max(max(lens), 0) if max_len is None else max_len
    cap = Tp + N if cap is None else cap
    print(f"B={B} H={H} Hkv={Hkv} d={d} N={N} lens={lens} {dtype} cap={cap} window={window} G={G} {out}", flush=True)
    g = R.gen(seed)
    kc, ks = R.cache(g, B, Hkv, cap, d, dtype)
    vc, vs = R.cache(g, B, Hkv, cap, d, dtype)
    q = (torch.randn(B, H, N, d, generator=g) * 1.5).to(torch.bfloat16)
    seg2 = gates = None
    if G:
        seg2 = tuple(torch.randn(gb, Hkv, G, d, generator=g).to(torch.bfloat16) for _ in range(2))
        gates = torch.tensor([0.7, -0.4])
    ref, mag = R.attention(q, R.values(kc, ks), R.values(vc, vs), lens, Tp, words, window, scale, seg2, gates)
    _poison(kc, vc, ks, vs, [min(max(t, 0), Tp) + N for t in lens])
    anc = None if words is None else np.array(words, dtype=np.uint64)
    o = hip.tree_attention_q8(q, *(t.to(dev) for t in (kc, vc, ks, vs)), lens, anc=anc, window=window, seg2=seg2,
                              gates=gates, max_len=Tp if max_len is None else max_len, out_dtype=out, scale=scale)
    assert o.shape == (B, H, N, d) and o.dtype == out
    _close(o, ref, mag)


def _tree(*branching):
    return [int(w) for w in VT.ancestor_words(VT.tree_from_branching(list(branching)))]


# one key, one step short of / at / past 32, several waves, splits; one query head to a KV head up to five; columns one
# short of / at / past a tile of 16 and a group of 64
CHAINS = [
    dict(B=1, H=1, Hkv=1, d=64, N=1, lens=[0]),
    dict(B=1, H=2, Hkv=1, d=128, N=1, lens=[1]),
    dict(B=3, H=4, Hkv=2, d=64, N=1, lens=[30, 31, 32]),
    dict(B=2, H=8, Hkv=8, d=128, N=2, lens=[0, 700]),
    dict(B=2, H=6, Hkv=2, d=64, N=5, lens=[97, 128], G=37),
    dict(B=1, H=4, Hkv=1, d=64, N=4, lens=[1500]),
    dict(B=1, H=5, Hkv=1, d=128, N=7, lens=[1030], G=5),
    dict(B=1, H=2, Hkv=1, d=64, N=33, lens=[63]),
    dict(B=2, H=2, Hkv=2, d=64, N=65, lens=[0, 40]),
    dict(B=1, H=4, Hkv=2, d=128, N=80, lens=[17], G=128),
]


@pytest.mark.parametrize("dtype", [I8, E4], ids=["int8", "e4m3"])
@pytest.mark.parametrize("case", range(len(CHAINS)))
def test_chain(hip, case, dtype):
    _run(hip, dtype=dtype, out=torch.float16 if case % 2 else torch.bfloat16, seed=case, **CHAINS[case])


@pytest.mark.parametrize("dtype", [I8, E4], ids=["int8", "e4m3"])
@pytest.mark.parametrize("d,N,lens,window,G", [
    (64, 1, [200, 3], 1, 0), (64, 5, [150, 0], 7, 0), (128, 40, [90, 10], 33, 16), (64, 70, [100, 5], 16, 0),
    (128, 3, [600, 599], 512, 8), (64, 9, [1300, 40], 1024, 128)])
def test_window(hip, d, N, lens, window, G, dtype):
    _run(hip, 2, 4, 2, d, N, lens, dtype, window=window, G=G, gb=2)


@pytest.mark.parametrize("dtype", [I8, E4], ids=["int8", "e4m3"])
@pytest.mark.parametrize("d,tree,lens,window", [
    (64, (1,), [5, 0], 0), (64, (4, 3, 2), [70, 0], 0), (128, (2, 2, 2), [33, 1], 0), (64, (2, 2, 2, 2, 2), [129, 31], 0),
    (128, (8,), [400, 7], 64), (64, (1, 4, 2, 1), [90, 1100], 100)])
def test_tree(hip, d, tree, lens, window, dtype):
    words = _tree(*tree)
    _run(hip, 2, 4, 2, d, len(words), lens, dtype, words=words, window=window)


def test_tree_of_64_nodes(hip):
    words = [(1 << (i + 1)) - 1 for i in range(64)]
    _run(hip, 1, 2, 1, 64, 64, [50], I8, words=words)


def test_tree_per_sequence(hip):
    """A tree a batch row, on the host and on the device, the same results."""
    a, b = _tree(3, 2), [(1 << (i + 1)) - 1 for i in range(9)]
    _run(hip, 2, 4, 2, 64, 9, [20, 45], E4, words=[a, b])
    dev = hip.torch_device
    g = R.gen(2)
    kc, ks = (t.to(dev) for t in R.cache(g, 2, 2, 60, 64, I8))
    q = torch.randn(2, 4, 9, 64, generator=g).to(torch.bfloat16).to(dev)
    w = np.array([a, b], dtype=np.uint64)
    one = hip.tree_attention_q8(q, kc, kc, ks, ks, [20, 45], anc=w)
    two = hip.tree_attention_q8(q, kc, kc, ks, ks, [20, 45], anc=torch.from_numpy(w.view(np.int64)).to(dev))
    assert torch.equal(one, two)


def test_nodes_that_see_nothing(hip):
    """Empty words over an empty prefix: zeros, or the second segment alone."""
    words = [0, 2, 0, 10]
    for G in (0, 9):
        _run(hip, 2, 2, 1, 64, 4, [0, 3], I8, words=words, G=G)


def test_lens_outside_their_bound(hip):
    """lens past max_len are cut to it, negative ones to 0."""
    _run(hip, 3, 2, 1, 64, 3, [-5, 90, 60], I8, cap=64, max_len=60)


def test_hidden_rows_hold_nan(hip):
    """Tree rows with NaN scales reach only the nodes that see them."""
    dev = hip.torch_device
    words = _tree(2, 2)
    N, T, d = len(words), 40, 64
    g = R.gen(4)
    kc, ks = R.cache(g, 1, 1, T + N, d, I8)
    vc, vs = R.cache(g, 1, 1, T + N, d, I8)
    q = torch.randn(1, 2, N, d, generator=g).to(torch.bfloat16)
    ref, mag = R.attention(q, R.values(kc, ks), R.values(vc, vs), [T], T, words)
    ks[0, 0, T + 1] = math.nan
    vs[0, 0, T + 1] = math.inf
    o = hip.tree_attention_q8(q, *(t.to(dev) for t in (kc, vc, ks, vs)), [T], anc=np.array(words, dtype=np.uint64))
    sees = torch.tensor([(w >> 1) & 1 for w in words], dtype=torch.bool)
    assert o[0, :, sees].isnan().all() and sees.any()
    _close(o[:, :, ~sees], ref[:, :, ~sees], mag[:, :, ~sees])


def test_extreme_scores(hip):
    """Scores far below and above zero, equal scores, a scale other than 1 / sqrt(d)."""
    dev = hip.torch_device
    d, T = 64, 300
    g = R.gen(6)
    kc, ks = R.cache(g, 1, 1, T, d, I8)
    vc, vs = R.cache(g, 1, 1, T, d, I8)
    for mul, scale in ((1e-6, 0.125), (8.0, 1.0), (-8.0, 1.0), (0.0, 0.125)):
        q = (mul * kc[:, :, :2].float()).to(torch.bfloat16) / 16
        # 2^-22 of |q| |k| scale log2(e) in the exponent: at most 2^-22 * 64 * 127 * 64 * scale * max(ks) * 1.45
        slack = 2.0 ** -22 * float((q.abs().float().sum(-1).max() * 127 * ks.max()) * scale * 1.45) * 2
        # probabilities below 2^-126 of the largest are 0 in fp32: 300 keys of |v| < 2^10, under 2^-126 * 2^19 in all
        ref, mag = R.attention(q, R.values(kc, ks), R.values(vc, vs), [T - 2], T - 2, scale=scale)
        o = hip.tree_attention_q8(q, *(t.to(dev) for t in (kc, vc, ks, vs)), [T - 2], scale=scale).cpu().to(R.F64)
        assert ((o - ref).abs() <= (2.0 ** -8 * 1.02 + slack) * mag + 2.0 ** -8 * ref.abs() + 2.0 ** -107).all()


def test_strides_and_out(hip):
    """A (B, cap, Hkv, d) cache, queries and output in (B, N, H, d) order: the contiguous call's bits."""
    dev = hip.torch_device
    B, H, Hkv, d, N, cap = 2, 6, 2, 128, 5, 83
    g = R.gen(7)
    kc, ks = (t.to(dev) for t in R.cache(g, B, Hkv, cap, d, E4))
    vc, vs = (t.to(dev) for t in R.cache(g, B, Hkv, cap, d, E4))
    q = torch.randn(B, H, N, d, generator=g).to(torch.bfloat16).to(dev)
    one = hip.tree_attention_q8(q, kc, vc, ks, vs, [70, 78])

    def turned(t):
        u = t.view(torch.uint8).transpose(1, 2).contiguous().view(t.dtype)
        return u.transpose(1, 2)

    buf = torch.full((B, N + 1, H, d), 5.0, dtype=torch.bfloat16, device=dev)
    out = buf[:, :N].transpose(1, 2)
    wide = torch.zeros(B, Hkv, cap + 5, device=dev)
    ks2, vs2 = wide.clone()[:, :, 3:cap + 3], wide.clone()[:, :, 3:cap + 3]
    ks2.copy_(ks)
    vs2.copy_(vs)
    qt = q.transpose(1, 2).contiguous().transpose(1, 2)
    two = hip.tree_attention_q8(qt, turned(kc), turned(vc), ks2, vs2, [70, 78], out=out)
    assert two is out and torch.equal(one, two) and (buf[:, N] == 5.0).all()


@pytest.mark.parametrize("dtype", [I8, E4], ids=["int8", "e4m3"])
@pytest.mark.parametrize("d", [64, 128])
def test_long_and_large(hip, d, dtype):
    """Against fp32 on the GPU where the 64-bit loops would be slow: many tiles (a wave each), many splits."""
    dev = hip.torch_device
    for B, H, Hkv, N, T, window, G in ((4, 16, 8, 300, 100, 0, 0), (8, 16, 8, 260, 0, 64, 128), (1, 16, 8, 1, 9000, 0, 0),
                                       (3, 12, 4, 6, 5000, 0, 40), (2, 8, 8, 700, 1500, 1024, 0)):
        print(B, H, Hkv, d, N, T, window, G, flush=True)
        g = R.gen(N)
        (kc, ks), (vc, vs) = (R.cache(g, B, Hkv, T + N, d, dtype) for _ in range(2))
        kc, ks, vc, vs = (t.to(dev) for t in (kc, ks, vc, vs))
        q = torch.randn(B, H, N, d, generator=g).to(torch.bfloat16).to(dev)
        lens = [T - 31 * b % (T + 1) if T else 0 for b in range(B)]
        rep = H // Hkv
        k, v = (c.float().mul(s[..., None]).to(R.F64).repeat_interleave(rep, 1) for c, s in ((kc, ks), (vc, vs)))
        s = q.to(R.F64) @ k.transpose(-1, -2).contiguous() / math.sqrt(d)
        pos = torch.tensor(lens, device=dev).view(B, 1, 1, 1) + torch.arange(N, device=dev).view(1, 1, N, 1)
        dist = pos - torch.arange(T + N, device=dev)
        s = s.masked_fill((dist < 0) | (dist >= window if window else dist < 0), -math.inf)
        p = torch.softmax(s, -1)
        ref, mag = p @ v, p @ v.abs()
        seg2 = gates = None
        if G:
            seg2 = tuple(torch.randn(1, Hkv, G, d, generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
            gates = torch.tensor([0.3, 0.9], device=dev)
            k2, v2 = (t.to(R.F64).repeat_interleave(rep, 1).expand(B, H, G, d).contiguous() for t in seg2)
            p = torch.softmax(q.to(R.F64) @ k2.transpose(-1, -2).contiguous() / math.sqrt(d), -1)
            ref, mag = 0.3 * ref + 0.9 * (p @ v2), 0.3 * mag + 0.9 * (p @ v2.abs())
        o = hip.tree_attention_q8(q, kc, vc, ks, vs, lens, window=window, seg2=seg2, gates=gates, max_len=T)
        _close(o, ref.cpu(), mag.cpu())


def test_write_then_attend_in_a_graph(hip):
    """A decode step (write, attend over splits, read) captured and replayed as its inputs change, with eager work and
    synchronisations between the replays; two graphs of different sizes share the stream."""
    dev = hip.torch_device
    B, H, Hkv, d, cap = 2, 8, 4, 64, 2100
    g = R.gen(9)
    (kc0, ks0), (vc0, vs0) = (R.cache(g, B, Hkv, cap, d, I8) for _ in range(2))
    ang = torch.rand(cap, d // 2, generator=g) * 6.28
    cos, sin = (torch.cat([f(ang)] * 2, 1).to(dev) for f in (torch.cos, torch.sin))
    kc, vc, ks, vs = (t.to(dev) for t in (kc0, vc0, ks0, vs0))
    graphs = []
    side = torch.cuda.Stream(device=dev)
    for n, bound in ((1, 2000), (6, 2080)):
        x = torch.randn(B, n, (H + 2 * Hkv) * d, generator=g).to(torch.bfloat16).to(dev)
        lens = torch.tensor([1000, 30], dtype=torch.int32, device=dev)

        def step(x=x, lens=lens, n=n, bound=bound):
            q = hip.kv_write(x, kc, vc, lens, k_scale=ks, v_scale=vs, cos=cos, sin=sin)
            o = hip.tree_attention_q8(q, kc, vc, ks, vs, lens, max_len=bound)
            return [o, *hip.kv_read(kc, vc, ks, vs, start=lens, rows=n)]

        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize(dev)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            outs = step()
        graphs.append((gr, x, lens, step, outs))
    for r in range(4):
        for gr, x, lens, step, outs in graphs:
            x.copy_(torch.randn(x.shape, generator=g).to(torch.bfloat16))
            lens.copy_(torch.tensor([900 + 257 * r, 20 + r], dtype=torch.int32))
            gr.replay()
            torch.cuda.synchronize(dev)
            got = [t.clone() for t in outs]
            for a, b in zip(got, step()):
                assert torch.equal(a, b)


def test_shared_cache(hip):
    """One sequence's cache seen by several batch rows (batch stride 0): the results of copies."""
    dev = hip.torch_device
    g = R.gen(14)
    (kc, ks), (vc, vs) = (R.cache(g, 1, 2, 90, 64, E4) for _ in range(2))
    q = torch.randn(3, 4, 2, 64, generator=g).to(torch.bfloat16).to(dev)
    lens = torch.tensor([88, 3, 40], dtype=torch.int32, device=dev)
    kc, vc, ks, vs = (t.to(dev) for t in (kc, vc, ks, vs))
    wide = [t.expand(3, *t.shape[1:]) for t in (kc, vc, ks, vs)]
    one = hip.tree_attention_q8(q, *wide, lens)
    two = hip.tree_attention_q8(q, *(t.view(torch.uint8).contiguous().view(t.dtype) if t.element_size() == 1
                                     else t.contiguous() for t in wide), lens)
    assert torch.equal(one, two)
    for got, want in zip(hip.kv_read(*wide, start=lens, rows=2), hip.kv_read(*(t.clone() for t in wide), start=lens, rows=2)):
        assert torch.equal(got, want)


def test_ranges_of_row_scales(hip):
    """Rows whose scales lie a factor 2^12 apart (a sink with tiny values under the largest weight): the bar of the terms,
    plus the 2^-32 of the largest row that the running scale allows a term (n of them)."""
    dev = hip.torch_device
    d, T = 64, 700
    g = R.gen(15)
    (kc, ks), (vc, vs) = (R.cache(g, 1, 1, T, d, I8) for _ in range(2))
    vs = vs * torch.exp2(torch.randint(-12, 1, vs.shape, generator=g).float())
    vs[0, 0, 0] *= 2.0 ** -12
    q = (kc[:, :, :1].float() / 24).to(torch.bfloat16)         # the first row's key scores highest
    ref, mag = R.attention(q, R.values(kc, ks), R.values(vc, vs), [T - 1], T - 1)
    o = hip.tree_attention_q8(q, *(t.to(dev) for t in (kc, vc, ks, vs)), [T - 1]).cpu().to(R.F64)
    big = float(R.values(vc, vs).abs().max())
    assert ((o - ref).abs() <= 2.0 ** -10 * mag + 2.0 ** -8 * ref.abs() + T * 2.0 ** -32 * big).all()


def test_same_call_on_two_streams(hip):
    """Two streams at once, each with its own workspace: the results of one after the other."""
    dev = hip.torch_device
    g = R.gen(12)
    data = []
    for i in range(2):
        (kc, ks), (vc, vs) = (R.cache(g, 1, 4, 3000, 64, I8) for _ in range(2))
        q = torch.randn(1, 8, 3, 64, generator=g).to(torch.bfloat16)
        data.append([t.to(dev) for t in (q, kc, vc, ks, vs)] + [torch.tensor([2900], dtype=torch.int32, device=dev)])
    want = [hip.tree_attention_q8(*d) for d in data]
    torch.cuda.synchronize(dev)
    streams = [torch.cuda.Stream(device=dev) for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(hip.tree_attention_q8(*data[i]))
    torch.cuda.synchronize(dev)
    for w, many in zip(want, got):
        assert all(torch.equal(w, o) for o in many)


@pytest.mark.parametrize("dtype", [I8, E4], ids=["int8", "e4m3"])
@pytest.mark.parametrize("d,B,N,rep,window", [(64, 16, 3, 2, 0), (64, 16, 1, 4, 0), (128, 8, 5, 4, 0), (128, 8, 1, 1, 0),
                                              (64, 18, 2, 2, 15000)])
def test_rows_read_past_the_caches(hip, d, B, N, rep, window, dtype):
    """192 MiB of rows and more, which one column group reads: every head and sequence shares one head's rows (strides
    of 0), so the memory is small.  NaN behind the last row."""
    dev = hip.torch_device
    Hkv, Tp = 8, 16001
    assert B * Hkv * (window or Tp) * 2 * d >= 192 << 20
    g = R.gen(d + N)
    kc, ks = R.cache(g, 1, 1, Tp + N + 40, d, dtype)
    vc, vs = R.cache(g, 1, 1, Tp + N + 40, d, dtype)
    _poison(kc, vc, ks, vs, [Tp + N])
    q = (torch.randn(B, rep * Hkv, N, d, generator=g) * 1.5).to(torch.bfloat16)
    lens = [Tp, 0, 31, 32, 15970] + [Tp - 17 * b for b in range(B - 5)]
    print(f"d={d} B={B} N={N} rep={rep} window={window} {dtype}", flush=True)
    wide = [t.to(dev).expand(B, Hkv, *t.shape[2:]) for t in (kc, vc, ks, vs)]
    for _ in range(2):                      # one call behind the other: the same rows again
        o = hip.tree_attention_q8(q, *wide, lens, window=window, max_len=Tp)
    pick = [0, 1, 2, 3, 4, B - 1]           # sequences of the 64-bit form, two KV heads of each
    heads = list(range(rep)) + list(range((Hkv - 1) * rep, Hkv * rep))
    k, v = (R.values(c, s).expand(len(pick), 2, -1, -1) for c, s in ((kc, ks), (vc, vs)))
    ref, mag = R.attention(q[pick][:, heads], k, v, [lens[b] for b in pick], Tp, window=window)
    _close(o[pick][:, heads], ref, mag)
