"""The product of 8-bit rows with an INT8 weight (vnx_q8_linear) against 64 bits, every launch shape: the sums are exact, so
the tolerance is the roundings of what follows them (q8_ref.linear)."""
import pytest
import torch

import q8_ref as R
from versenext_amd import _lib

pytestmark = pytest.mark.gpu

SHAPES = range(0, 8)     # 0: the plan's choice
TILES = [0, 1, 2, 3, 4, 6, 7]      # those that take SwiGLU


def check(hip, shape, M, N, K, out=torch.bfloat16, bias=False, residual=None, swiglu=False, low=-127, fill=77, seed=0):
    g = R.gen(seed + 1000003 * M + 1009 * N + K)
    dev = hip.torch_device
    c, w = R.codes(g, M, K, low), R.codes(g, N, K, low)
    cs, ws = R.scales(g, M), R.scales(g, N)
    cols = N // 2 if swiglu else N
    b = torch.randn(N, generator=g) if bias else None
    r = torch.randn(M, cols, generator=g).to(residual) if residual else None
    ld = (K + 15) // 16 * 16 + 16
    got = hip.linear_q8(R.pitched(c, ld, fill, dev), cs.to(dev), R.pitched(w, ld + 32, -fill, dev), ws.to(dev),
                        bias=None if b is None else b.to(dev), residual=None if r is None else r.to(dev), swiglu=swiglu,
                        out_dtype=out, force_shape=shape)
    y, tol = R.linear(c, cs, w, ws, b, r, swiglu, out)
    assert got.shape == (M, cols) and got.dtype == out
    bad = R.off(got, y, tol).nonzero()
    assert bad.numel() == 0, (bad[:5].tolist(), len(bad))


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("M,N,K", [
    (1, 1, 1), (1, 7, 15), (2, 16, 16), (3, 33, 17), (1, 2048, 1024), (15, 100, 127), (16, 64, 128), (17, 65, 129),
    (31, 129, 64), (32, 1024, 4096), (33, 31, 1000), (63, 256, 63), (64, 130, 256), (65, 515, 255), (128, 128, 144),
    (129, 257, 400), (224, 1003, 1024), (255, 255, 192), (256, 512, 257), (300, 96, 2000), (513, 770, 320)])
def test_sizes(hip, shape, M, N, K):
    check(hip, shape, M, N, K)
    check(hip, shape, M, N, K, out=torch.float32, bias=True, residual=torch.float32, low=-128, seed=1)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("out", R.DTYPES)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("residual", [None, *R.DTYPES])
def test_epilogues(hip, shape, out, bias, residual):
    for M, N, K in ((5, 70, 200), (70, 301, 130), (260, 264, 96)):
        check(hip, shape, M, N, K, out, bias, residual)


@pytest.mark.parametrize("shape", TILES)
@pytest.mark.parametrize("out", R.DTYPES)
@pytest.mark.parametrize("bias", [False, True])
def test_swiglu(hip, shape, out, bias):
    for M, N, K in ((1, 2, 5), (4, 34, 100), (9, 512, 64), (40, 200, 128), (130, 1026, 272), (260, 130, 1024)):
        check(hip, shape, M, N, K, out, bias, swiglu=True)


@pytest.mark.parametrize("shape", SHAPES)
def test_largest_sums(hip, shape):
    """K of 131,071 with every product 2^14: the sum is 2^31 - 2^14, the last one below the sign."""
    dev = hip.torch_device
    K = 131071
    c, w = torch.full((2, K), -128, dtype=torch.int8), torch.full((3, K), -128, dtype=torch.int8)
    w[1], w[2, 1:] = 127, 0
    c, w = R.pitched(c, K + 1, 5, dev), R.pitched(w, K + 1, 5, dev)
    y = hip.linear_q8(c, torch.ones(2), w, torch.ones(3), out_dtype=torch.float32, force_shape=shape)
    assert y.cpu().tolist() == [[2147467264.0, float(torch.tensor(-128 * 127 * K, dtype=torch.float32)), 16384.0]] * 2


@pytest.mark.parametrize("shape", SHAPES)
def test_rows_without_a_scale(hip, shape):
    """A row of scale NaN is NaN, one of scale 0 is 0 (with the bias), a column's too; the others are as without them."""
    dev = hip.torch_device
    g = R.gen(4)
    c, w = R.codes(g, 70, 96), R.codes(g, 45, 96)
    cs, ws = R.scales(g, 70), R.scales(g, 45)
    want = hip.linear_q8(c.to(dev), cs, w.to(dev), ws, force_shape=shape)
    cs[3], cs[64], ws[2] = float("nan"), 0.0, float("nan")
    got = hip.linear_q8(c.to(dev), cs, w.to(dev), ws, force_shape=shape)
    assert got[3].isnan().all() and got[:, 2].isnan().all()
    keep = torch.ones(70, 45, dtype=torch.bool)
    keep[3], keep[:, 2], keep[64] = False, False, False
    assert torch.equal(got.cpu()[keep], want.cpu()[keep]) and got[64].cpu()[keep[0]].eq(0).all()


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("M,N", [(3, 33), (70, 131), (260, 260)])
def test_outputs_in_place(hip, shape, M, N):
    """Into rows of a wider tensor at an odd element, and over the residual: what lies beside them stays."""
    dev = hip.torch_device
    g = R.gen(M)
    c, w, cs, ws = R.codes(g, M, 80), R.codes(g, N, 80), R.scales(g, M), R.scales(g, N)
    for dtype in R.DTYPES:
        buf = torch.randn(M, N + 7, generator=g).to(dtype)
        d = buf.to(dev)
        y, tol = R.linear(c, cs, w, ws, residual=buf[:, 3:3 + N], out=dtype)
        view = d[:, 3:3 + N]
        got = hip.linear_q8(c.to(dev), cs, w.to(dev), ws, residual=view, out=view, force_shape=shape)
        assert got is view and not R.off(view, y, tol).any()
        assert torch.equal(d[:, :3].cpu(), buf[:, :3]) and torch.equal(d[:, 3 + N:].cpu(), buf[:, 3 + N:])


def test_more_dimensions_and_layouts(hip):
    """(..., K) codes; rows that are not on 16 bytes, transposed ones, scales as (N, 1): the same values."""
    dev = hip.torch_device
    g = R.gen(8)
    c, w, cs, ws = R.codes(g, 12, 50), R.codes(g, 40, 50), R.scales(g, 12), R.scales(g, 40)
    want = hip.linear_q8(R.pitched(c, 64, 0, dev), cs.to(dev), R.pitched(w, 64, 0, dev), ws.to(dev))
    for cc, ww, s in ((c, w, ws), (c.t().contiguous().t(), w.t().contiguous().t(), ws[:, None]),
                      (c.view(3, 4, 50), w, ws)):
        got = hip.linear_q8(cc.to(dev), cs.view(cc.shape[:-1]).to(dev), ww.to(dev), s.to(dev))
        assert got.shape == (*cc.shape[:-1], 40) and torch.equal(got.view(12, 40), want)
    assert torch.equal(hip.linear_q8(c.numpy(), cs.numpy(), w.numpy(), ws.numpy()), want)
    for M, N in ((0, 40), (12, 0)):
        assert hip.linear_q8(c[:M].to(dev), cs[:M], w[:N].to(dev), ws[:N]).shape == (M, N)


def test_shapes_agree_bit_for_bit(hip):
    """The sums are exact and what follows is in one order: every launch shape gives the same bits."""
    dev = hip.torch_device
    g = R.gen(11)
    c, w, cs, ws = R.codes(g, 100, 1000), R.codes(g, 302, 1000), R.scales(g, 100).to(dev), R.scales(g, 302).to(dev)
    c, w = R.pitched(c, 1008, 3, dev), R.pitched(w, 1008, 3, dev)
    b, r = torch.randn(302, generator=g).to(dev), torch.randn(100, 302, generator=g).to(dev)
    for kw in (dict(), dict(bias=b, residual=r), dict(bias=b, swiglu=True)):
        want = hip.linear_q8(c, cs, w, ws, out_dtype=torch.float32, force_shape=1, **kw)
        for shape in TILES if "swiglu" in kw else SHAPES:
            assert torch.equal(hip.linear_q8(c, cs, w, ws, out_dtype=torch.float32, force_shape=shape, **kw), want)


def test_refusals(hip):
    dev = hip.torch_device
    c, w = torch.ones(4, 32, dtype=torch.int8, device=dev), torch.ones(6, 32, dtype=torch.int8, device=dev)
    cs, ws = torch.ones(4, device=dev), torch.ones(6, device=dev)
    y = torch.zeros(4, 6, device=dev)
    for call in (lambda: hip.linear_q8(c.float(), cs, w, ws), lambda: hip.linear_q8(c, cs, w.float(), ws),
                 lambda: hip.linear_q8(c, cs, w[:, :31], ws), lambda: hip.linear_q8(c, cs, w[None], ws),
                 lambda: hip.linear_q8(c, cs[:3], w, ws), lambda: hip.linear_q8(c, cs, w, ws[:5]),
                 lambda: hip.linear_q8(c, cs, w, ws, bias=ws[:5]), lambda: hip.linear_q8(c, cs, w, ws, residual=y[:3]),
                 lambda: hip.linear_q8(c, cs, w, ws, residual=y, swiglu=True),
                 lambda: hip.linear_q8(c, cs, w[:5], ws[:5], swiglu=True),
                 lambda: hip.linear_q8(c, cs, w, ws, out_dtype=torch.int8),
                 lambda: hip.linear_q8(c, cs, w, ws, out=y[:3]), lambda: hip.linear_q8(c, cs, w, ws, out=y.cpu()),
                 lambda: hip.linear_q8(c, cs, w, ws, out=y.double()),
                 lambda: hip.linear_q8(c, cs, w, ws, out=torch.zeros(6, 4, device=dev).t()),
                 lambda: hip.linear_q8(c, cs, w, ws, out=torch.zeros(1, 6, device=dev).expand(4, 6)),
                 lambda: hip.linear_q8(c, cs, w, ws, force_shape=-1),
                 lambda: hip.linear_q8(c, cs, w, ws, force_shape=99),
                 lambda: hip.linear_q8(c, cs, w, ws, swiglu=True, force_shape=5)):
        with pytest.raises(ValueError):
            call()
    buf = torch.zeros(5 * 6, device=dev)                   # over rows of the residual that others still need
    with pytest.raises(ValueError):
        hip.linear_q8(c, cs, w, ws, residual=buf[:24].view(4, 6), out=buf[6:].view(4, 6))
    assert buf.eq(0).all()


def layer(hip, x, r, nw, up, down):
    codes, scale, s = hip.rmsnorm_q8(x, nw, residual=r)
    act = hip.linear_q8(codes, scale, *up, swiglu=True)
    codes, scale = hip.quantize_rows(act)
    return s, act, hip.linear_q8(codes, scale, *down, residual=s, out_dtype=torch.float32)


def layer_inputs(g, M, D, H):
    def weight(N, K):
        return R.quantize(torch.randn(N, K, generator=g) * K ** -0.5)
    return (torch.randn(M, D, generator=g), torch.randn(M, D, generator=g).bfloat16(), 1 + 0.1 * torch.randn(D, generator=g),
            weight(2 * H, D), weight(D, H))


@pytest.mark.parametrize("M,D,H", [(1, 64, 176), (7, 1024, 2752), (130, 192, 320)])
def test_a_layer(hip, M, D, H):
    """Norm, gate and up, codes, down: every step against the plain form of what it was given."""
    dev = hip.torch_device
    x, r, nw, up, down = layer_inputs(R.gen(M + D), M, D, H)
    put = lambda t: tuple(v.to(dev) for v in t)
    s, act, y = (t.cpu() for t in layer(hip, x.to(dev), r.to(dev), nw.to(dev), put(up), put(down)))
    c, s64, total = R.rmsnorm(x, nw, 1e-6, r)
    assert torch.equal(s, total)
    want, tol = R.linear(c, s64, *up, swiglu=True, out=torch.bfloat16)
    # the scale has 30 roundings of its own: in gate and up, 1 + |gate's| sensitivity < 2 + |g| <= 34
    assert ((act.double() - want).abs() <= tol + 34 * 30 * R.U * want.abs()).all()
    want, tol = R.linear(*R.quantize(act), *down, residual=s, out=torch.float32)
    assert ((y.double() - want).abs() <= tol).all()


def test_captured_and_replayed(hip):
    """The chain in a graph: replays on new inputs, eager calls and synchronizations between them, equal the eager result;
    two graphs share nothing."""
    dev = hip.torch_device
    sets = [layer_inputs(R.gen(s), M, 256, 384) for s, M in ((1, 33), (2, 200))]
    sets = [[v.to(dev) if isinstance(v, torch.Tensor) else tuple(t.to(dev) for t in v) for v in st] for st in sets]
    graphs = []
    st = torch.cuda.Stream(device=dev)
    st.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(st):
        for a in sets:
            layer(hip, *a)
    torch.cuda.synchronize()
    for a in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = layer(hip, *a)
        graphs.append((g, out))
    for k in range(4):
        for a in sets:
            a[0].normal_()
        want = [layer(hip, *a) for a in sets]
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (_, out), w in zip(graphs, want):
            assert all(torch.equal(p, q) for p, q in zip(out, w))


def test_split_captured_and_replayed(hip):
    """Two graphs of products whose k is split (each with partial sums of its own), replayed at once on two streams with
    eager calls between, equal the eager result."""
    dev = hip.torch_device
    g = R.gen(21)
    sets, graphs = [], []
    for M, N, K, force, swiglu in ((200, 500, 16000, 0, False), (70, 260, 8192, 6, True)):
        sets.append((R.codes(g, M, K).to(dev), R.scales(g, M).to(dev), R.codes(g, N, K).to(dev), R.scales(g, N).to(dev),
                     None, None, swiglu, torch.float32, None, force))
        p = _lib.pack_q8_linear(*[0] * 7, K, K, 0, N, M, N, K, 0, _lib.VNX_F32, _lib.VNX_EPI_SWIGLU if swiglu else _lib.VNX_EPI_NONE,
                                force)
        assert hip._L.vnx_q8_linear_workspace(p) > 256       # two launches
    want = [hip.linear_q8(*a[:-1], force_shape=2) for a in sets]
    streams = [torch.cuda.Stream(device=dev) for _ in sets]
    for a, st in zip(sets, streams):
        st.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(st):
            hip.linear_q8(*a)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            out = hip.linear_q8(*a)
        graphs.append((gr, out))
    for k in range(4):
        for a in sets:
            a[1].uniform_(0.001, 0.1)
        want = [hip.linear_q8(*a[:-1], force_shape=2) for a in sets]
        for _, out in graphs:
            out.fill_(7.0)
        torch.cuda.synchronize()
        for (gr, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        eager = [hip.linear_q8(*a) for a in sets]
        torch.cuda.synchronize()
        for (_, out), e, w in zip(graphs, eager, want):
            assert torch.equal(out, w) and torch.equal(e, w)


def test_one_row_of_a_wide_tensor(hip, monkeypatch):
    """A single row has no pitch to refuse, however far its tensor's next one would be."""
    dev = hip.torch_device
    g = R.gen(3)
    wide = torch.zeros(1, (1 << 22) + 64, dtype=torch.int8, device=dev)
    c, w = R.codes(g, 1, 100).to(dev), R.codes(g, 5, 100).to(dev)
    wide[:, :100] = c
    cs, ws = R.scales(g, 1).to(dev), R.scales(g, 5).to(dev)
    for bind in (_lib.bind(), _lib.NoBind):
        monkeypatch.setattr(hip, "_bind", bind)
        want = hip.linear_q8(c, cs, w, ws)
        assert torch.equal(hip.linear_q8(wide[:, :100], cs, w, ws), want)
        assert torch.equal(hip.linear_q8(w, ws, wide[:, :100], cs), hip.linear_q8(w, ws, c, cs))
        assert torch.equal(hip.dequantize_rows(wide[:, :100], cs), hip.dequantize_rows(c, cs))


def test_streams(hip):
    """Two streams at once give what one gives."""
    dev = hip.torch_device
    a = [v.to(dev) if isinstance(v, torch.Tensor) else tuple(t.to(dev) for t in v)
         for v in layer_inputs(R.gen(5), 64, 512, 640)]
    want = layer(hip, *a)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=dev) for _ in range(2)]
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(layer(hip, *a))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(p, q) for p, q in zip(g, want))


def test_binding_and_general_path_agree(hip, monkeypatch):
    dev = hip.torch_device
    g = R.gen(9)
    c, w = (R.pitched(R.codes(g, n, 100), 112, 9, dev) for n in (21, 34))
    cs, ws, b = R.scales(g, 21).to(dev), R.scales(g, 34).to(dev), torch.randn(34, generator=g).to(dev)
    r = torch.randn(21, 34, generator=g).to(dev)
    got = []
    for bind in (_lib.bind(), _lib.NoBind):
        monkeypatch.setattr(hip, "_bind", bind)
        got.append([hip.linear_q8(c, cs, w, ws, bias=b, residual=r, out_dtype=torch.float16),
                    hip.linear_q8(c, cs, w, ws, swiglu=True), hip.linear_q8(c, cs, w, ws, residual=r, out=r.clone())])
    for p, q in zip(*got):
        assert torch.equal(p, q) and p.dtype == q.dtype
