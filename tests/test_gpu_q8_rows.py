"""Rows to 8-bit integers and back (vnx_q8_quantize, vnx_q8_rmsnorm, vnx_q8_dequantize) against the plain form: codes and
sums bit for bit, scales within the roundings of their steps."""
import pytest
import torch

import q8_ref as R

pytestmark = pytest.mark.gpu

# every launch shape and its border, rows that 8 does not divide, fewer than 8 values, more than a workgroup holds
WIDTHS = [1, 3, 7, 8, 9, 64, 511, 512, 513, 1000, 1024, 1025, 2047, 2048, 2056, 4096, 4101, 8192, 8200, 12288, 12289,
          16384, 16385, 32768, 32777, 70001]


def rows(seed, M, K, dtype):
    g = R.gen(seed)
    return (torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g))).to(dtype)


def scale_steps(K):
    """Roundings of a norm's scale: the sum of squares (at most 33 in a thread of 32 values, 6 in a wave, 15 over sixteen
    waves: 54; K / 256 + 16 where a thread walks the row), halved by the root; the mean, eps, the root, a / 127 and the
    quotient."""
    return (54 if 8 <= K <= 32768 else K / 256 + 16) / 2 + 6


@pytest.mark.parametrize("K", WIDTHS)
@pytest.mark.parametrize("dtype", R.DTYPES)
def test_quantize(hip, K, dtype):
    for M in (1, 5):
        x = rows(K + M, M, K, dtype)
        codes, scale = hip.quantize_rows(x.to(hip.torch_device))
        c, s = R.quantize(x)
        assert torch.equal(codes.cpu(), c) and torch.equal(scale.cpu(), s)
        assert codes.stride(0) % 16 == 0 or M == 1
        for out in R.DTYPES:
            v = hip.dequantize_rows(codes, scale, out_dtype=out)
            assert torch.equal(v.cpu(), (c.float() * s[:, None]).to(out))


@pytest.mark.parametrize("K", WIDTHS)
@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize("res", [None, *R.DTYPES])
def test_rmsnorm(hip, K, dtype, res):
    g = R.gen(K)
    dev = hip.torch_device
    for M in (1, 6):
        x = rows(2 * K + M, M, K, dtype)
        r = None if res is None else rows(3 * K + M, M, K, res)
        w = 1 + 0.3 * torch.randn(K, generator=g)
        c, s64, s = R.rmsnorm(x, w, 1e-6, r)
        xd, rd = x.to(dev), None if r is None else r.to(dev)
        codes, scale, total = hip.rmsnorm_q8(xd, w.to(dev), residual=rd)
        assert torch.equal(total.cpu(), s) and torch.equal(codes.cpu(), c)
        assert ((scale.cpu().double() - s64).abs() <= scale_steps(K) * R.U * s64).all()
        assert torch.equal(xd.cpu(), x)
        if r is None:
            assert total.data_ptr() == xd.data_ptr()
            continue
        # in place: over x, and over the residual where the types agree
        for over in [0] + [1] * (dtype == res):
            pair = [x.to(dev), r.to(dev)]
            again = hip.rmsnorm_q8(pair[0], w.to(dev), residual=pair[1], sum_out=pair[over])
            assert again[2] is pair[over] and torch.equal(pair[over].cpu(), s)
            assert torch.equal(again[0], codes) and torch.equal(again[1], scale)


@pytest.mark.parametrize("M", [0, 1, 3, 4, 5, 1023])
def test_many_rows(hip, M):
    x = rows(M, M, 200, torch.bfloat16)
    codes, scale = hip.quantize_rows(x.to(hip.torch_device))
    c, s = R.quantize(x)
    assert torch.equal(codes.cpu(), c) and torch.equal(scale.cpu(), s)
    assert hip.dequantize_rows(codes, scale).shape == (M, 200)
    codes, scale, _ = hip.rmsnorm_q8(x.to(hip.torch_device), torch.ones(200))
    assert torch.equal(codes.cpu(), R.rmsnorm(x, torch.ones(200), 1e-6)[0])


@pytest.mark.parametrize("K", [5, 96, 1030, 5000, 33000])
def test_rows_without_values(hip, K):
    """All zeros, below the smallest maximum, an infinity, a NaN: codes 0, scale 0 or NaN; the rows beside them as ever."""
    x = rows(K, 7, K, torch.float32)
    x[0] = 0
    x[1] = 2.0 ** -101
    x[2, K // 2] = float("inf")
    x[3, K - 1] = float("nan")
    x[4, 0] = -float("inf")
    x[5] = 2.0 ** -100 * torch.sign(x[5])
    dev = hip.torch_device
    c, s = R.quantize(x)
    codes, scale = hip.quantize_rows(x.to(dev))
    assert torch.equal(codes.cpu(), c) and torch.equal(scale.cpu().nan_to_num(-1.0), s.nan_to_num(-1.0))
    assert (c[:5] == 0).all() and (c[5].abs() == 127).all() and s[:2].eq(0).all() and s[2:5].isnan().all()
    w = torch.ones(K)
    c, s, _ = R.rmsnorm(x, w, 1e-6)
    codes, scale, _ = hip.rmsnorm_q8(x.to(dev), w.to(dev))
    assert torch.equal(codes.cpu(), c)
    assert ((scale.cpu().double().nan_to_num(-1.0) - s.nan_to_num(-1.0)).abs() <= scale_steps(K) * R.U * s.nan_to_num(1.0)).all()
    # squares that pass fp32's range: no scale, not one of zero
    big = torch.full((1, K), 1e25)
    assert hip.rmsnorm_q8(big.to(dev), w.to(dev))[1].isnan().all()


def test_eps_and_weights(hip):
    dev = hip.torch_device
    x = 1e-4 * rows(1, 4, 300, torch.float32)
    for eps in (0.0, 1e-6, 1.0):
        for w in (torch.ones(300), torch.linspace(-2, 3, 300), torch.zeros(300)):
            c, s, _ = R.rmsnorm(x, w, eps)
            codes, scale, _ = hip.rmsnorm_q8(x.to(dev), w.to(dev), eps=eps)
            assert torch.equal(codes.cpu(), c) and ((scale.cpu().double() - s).abs() <= 30 * R.U * s).all()
    zero = hip.rmsnorm_q8(torch.zeros(2, 300, device=dev), torch.ones(300, device=dev), eps=0.0)
    assert zero[0].eq(0).all() and zero[1].eq(0).all()


@pytest.mark.parametrize("off", [0, 1, 3])
def test_strides(hip, off):
    """Rows inside wider ones, at any element: what lies beside the outputs stays."""
    dev = hip.torch_device
    for dtype in R.DTYPES:
        big = rows(5, 9, 700, dtype)
        v = big[:, off:off + 603]
        bd = big.to(dev)
        vd = bd[:, off:off + 603]
        c, s = R.quantize(v)
        codes, scale = hip.quantize_rows(vd)
        assert torch.equal(codes.cpu(), c) and torch.equal(scale.cpu(), s)
        w = torch.ones(603)
        c, _, t = R.rmsnorm(v, w, 1e-6, v)
        total = hip.rmsnorm_q8(vd, w.to(dev), residual=vd.clone(), sum_out=vd)
        assert torch.equal(total[0].cpu(), c) and torch.equal(vd.cpu(), t)
        big[:, off:off + 603] = t
        assert torch.equal(bd.cpu(), big)
        # every other row, rows of a transposed matrix, more dimensions
        for make in (lambda t: t[::2], lambda t: t[:, :8].t(), lambda t: t[:8].view(2, 4, 700)[:, 1:3]):
            a, b = hip.quantize_rows(make(bd))
            c, s = R.quantize(make(big))
            assert a.shape == c.shape and torch.equal(a.cpu(), c) and torch.equal(b.cpu(), s)
            assert torch.equal(hip.dequantize_rows(a, b).cpu(), c.float() * s[..., None])


def test_binding_and_general_path_agree(hip, monkeypatch):
    from versenext_amd import _lib
    dev = hip.torch_device
    x, r, w = rows(1, 40, 777, torch.bfloat16).to(dev), rows(2, 40, 777, torch.float16).to(dev), torch.rand(777, device=dev)
    got = []
    for bind in (_lib.bind(), _lib.NoBind):
        monkeypatch.setattr(hip, "_bind", bind)
        codes, scale = hip.quantize_rows(x)
        got.append([codes, scale, hip.dequantize_rows(codes, scale, torch.float16), *hip.rmsnorm_q8(x, w, 1e-5, r)])
    for a, b in zip(*got):
        assert torch.equal(a, b) and a.stride() == b.stride() and a.dtype == b.dtype


def test_refusals(hip):
    dev = hip.torch_device
    x, w = torch.ones(4, 32, device=dev), torch.ones(32, device=dev)
    for call in (lambda: hip.quantize_rows(x.double()), lambda: hip.quantize_rows(x[:, :0]),
                 lambda: hip.quantize_rows(torch.tensor(1.0, device=dev)),
                 lambda: hip.dequantize_rows(x, w), lambda: hip.dequantize_rows(x.to(torch.int8), w),
                 lambda: hip.dequantize_rows(x.to(torch.int8), w[:4], torch.float64),
                 lambda: hip.rmsnorm_q8(x, w[:31]), lambda: hip.rmsnorm_q8(x, w, eps=-1.0),
                 lambda: hip.rmsnorm_q8(x, w, eps=float("nan")), lambda: hip.rmsnorm_q8(x, w, residual=x[:3]),
                 lambda: hip.rmsnorm_q8(x, w, residual=x, sum_out=x[:3]),
                 lambda: hip.rmsnorm_q8(x, w, residual=x, sum_out=x.bfloat16()),
                 lambda: hip.rmsnorm_q8(x, w, residual=x, sum_out=x.cpu()),
                 lambda: hip.rmsnorm_q8(x, w, residual=x, sum_out=x.t().contiguous().t()),
                 lambda: hip.rmsnorm_q8(x, w, residual=x, sum_out=torch.ones(1, 32, device=dev).expand(4, 32))):
        with pytest.raises(ValueError):
            call()
    # a sum over rows that other rows of x still need
    buf = torch.ones(5 * 32, device=dev)
    with pytest.raises(ValueError):
        hip.rmsnorm_q8(buf[:128].view(4, 32), w, residual=x, sum_out=buf[32:].view(4, 32))
    assert buf.eq(1).all()
    # (halves of one buffer's rows do not meet)
    two = torch.ones(4, 64, device=dev)
    assert hip.rmsnorm_q8(two[:, :32], w, residual=x, sum_out=two[:, 32:])[2].eq(2).all() and two[:, :32].eq(1).all()
