"""The argument checks of the products in 8-bit integers: bad calls are refused on the host, before anything is launched and
before any pointer is read; the binding leaves what is not on the GPU (no GPU needed)."""
import ctypes

import pytest
import torch

from versenext_amd import _lib

AT = 1 << 30     # an address that is never read
FAR = 1 << 46
OK, INVALID, UNSUPPORTED = 0, _lib.VNX_ERR_INVALID_ARG, _lib.VNX_ERR_UNSUPPORTED


def quantize(**over):
    a = dict(x=AT, dtype=_lib.VNX_BF16, ldx=64, M=4, K=64, codes=FAR, ldc=64, scale=FAR * 2, stream=None)
    return _lib.lib().vnx_q8_quantize(*(a | over).values())


def rmsnorm(**over):
    a = dict(x=AT, dtype=_lib.VNX_F32, ldx=64, res=2 * AT, res_dtype=_lib.VNX_BF16, ldr=64, w=3 * AT, eps=1e-6, M=4,
             K=64, sum=4 * AT, lds=64, codes=FAR, ldc=64, scale=2 * FAR, stream=None)
    return _lib.lib().vnx_q8_rmsnorm(*(a | over).values())


def dequantize(**over):
    a = dict(codes=AT, ldc=64, scale=2 * AT, M=4, K=64, out=FAR, out_dtype=_lib.VNX_F16, ldo=64, stream=None)
    return _lib.lib().vnx_q8_dequantize(*(a | over).values())


def linear(**over):
    a = _lib.Q8LinearArgs()
    for k, v in (dict(x=AT, x_scale=2 * AT, w=3 * AT, w_scale=4 * AT, bias=5 * AT, res=6 * AT, y=FAR, ldx=64, ldw=64,
                      ldr=32, ldy=32, M=4, N=32, K=64, res_dtype=_lib.VNX_BF16, y_dtype=_lib.VNX_F32) | over).items():
        setattr(a, k, v)
    return _lib.lib().vnx_q8_linear(ctypes.byref(a), None, 0, None)


BAD = [
    (quantize, INVALID, [dict(M=-1), dict(K=0), dict(ldx=63), dict(ldc=63), dict(x=None), dict(codes=None),
                         dict(scale=None), dict(x=AT + 1), dict(scale=FAR * 2 + 2), dict(codes=AT + 100)]),
    (quantize, UNSUPPORTED, [dict(dtype=_lib.VNX_I8), dict(dtype=9), dict(K=2 ** 31 - 9, ldx=2 ** 31, ldc=2 ** 31),
                             dict(M=2 ** 34)]),
    (rmsnorm, INVALID, [dict(M=-1), dict(K=0), dict(ldx=63), dict(ldr=63), dict(lds=63), dict(ldc=63), dict(x=None),
                        dict(w=None), dict(codes=None), dict(scale=None), dict(x=AT + 2), dict(res=AT * 2 + 1),
                        dict(w=3 * AT + 1), dict(sum=4 * AT + 2), dict(eps=-1.0), dict(eps=float("nan")),
                        dict(eps=float("inf")), dict(codes=AT), dict(codes=2 * AT + 5), dict(codes=4 * AT),
                        dict(sum=AT + 4), dict(sum=AT, lds=72), dict(sum=2 * AT), dict(sum=AT + 256)]),
    (rmsnorm, UNSUPPORTED, [dict(dtype=3), dict(res_dtype=4), dict(K=2 ** 31, ldx=2 ** 32, ldc=2 ** 32, ldr=2 ** 32,
                                                                   lds=2 ** 32)]),
    (dequantize, INVALID, [dict(M=-1), dict(K=0), dict(ldc=63), dict(ldo=63), dict(codes=None), dict(scale=None),
                           dict(out=None), dict(out=FAR + 1), dict(out=AT)]),
    (dequantize, UNSUPPORTED, [dict(out_dtype=3), dict(M=2 ** 34, K=2000, ldc=2000, ldo=2000)]),
    (linear, INVALID, [dict(M=-1), dict(N=-1), dict(K=0), dict(ldx=48), dict(ldw=48), dict(ldy=31), dict(ldr=31),
                       dict(epilogue=2), dict(epilogue=1), dict(epilogue=1, res=None, N=31), dict(x=None),
                       dict(x_scale=None), dict(w=None), dict(w_scale=None), dict(y=None), dict(y=FAR + 2),
                       dict(res=6 * AT + 1), dict(x_scale=2 * AT + 1), dict(w_scale=4 * AT + 2), dict(bias=5 * AT + 3),
                       dict(y=AT), dict(y=3 * AT + 64), dict(y=2 * AT), dict(y=4 * AT), dict(y=5 * AT),
                       dict(y=6 * AT), dict(res=FAR, res_dtype=0, ldr=40), dict(res=FAR + 4, res_dtype=0),
                       dict(res=FAR + 128, res_dtype=0)]),
    (linear, UNSUPPORTED, [dict(y_dtype=3), dict(res_dtype=4), dict(K=131072, ldx=131072, ldw=131072),
                           dict(M=2 ** 31 - 4), dict(N=2 ** 31 - 4, ldy=2 ** 31, ldr=2 ** 31), dict(x=AT + 8), dict(w=AT * 3 + 4),
                           dict(ldx=72), dict(ldw=65), dict(ldx=1 << 22), dict(ldw=1 << 22), dict(force_shape=-1),
                           dict(force_shape=99)]),
]


@pytest.mark.parametrize("call,status,over", [(c, s, o) for c, s, all_ in BAD for o in all_])
def test_refused(call, status, over):
    assert call(**over) == status


@pytest.mark.parametrize("call", [quantize, rmsnorm, dequantize, linear])
def test_no_rows(call):
    """An empty batch is a call without work: no pointer is read."""
    none = {k: None for k in ("x", "res", "w", "sum", "codes", "scale", "out", "bias", "y", "x_scale", "w_scale")}
    fields = {quantize: ("x", "codes", "scale"), rmsnorm: ("x", "res", "w", "sum", "codes", "scale"),
              dequantize: ("codes", "scale", "out"), linear: ("x", "res", "w", "bias", "y", "x_scale", "w_scale")}[call]
    assert call(M=0, **{k: none[k] for k in fields}) == OK


def test_null_block():
    assert _lib.lib().vnx_q8_linear(None, None, 0, None) == INVALID
    assert _lib.lib().vnx_q8_linear_workspace(None) == 256


def test_binding_leaves_calls_off_the_gpu():
    b = _lib.bind()
    x, s = torch.zeros(4, 32), torch.zeros(4)
    c = x.to(torch.int8)
    for n in (None, 1, x, c, x[0], x.double()):
        assert b.q8_quantize(0, 0, n) is None and b.q8_dequantize(0, 0, n, s, torch.float32) is None
        assert b.q8_rmsnorm(0, 0, n, s, 1e-6, None, None) is None
        assert b.q8_linear(0, 0, n, s, c, s, None, None, False, torch.float32, None) is None
    assert b.q8_quantize() is None and b.q8_linear(1, 2) is None and b.q8_rmsnorm(*range(7)) is None
    for bad in ((), (1, 2, 3, 4, 0), ("a", 1, 1, 1, 1)):
        with pytest.raises((TypeError, ValueError)):
            b.init_q8(*bad)


def test_workspace():
    """Sums that are split over k need one; what the sizes alone refuse needs none."""
    L, a = _lib.lib(), _lib.Q8LinearArgs()
    for k, v in dict(ldx=8192, ldw=8192, ldy=64, M=64, N=64, K=8192, y_dtype=_lib.VNX_F32, force_shape=6).items():
        setattr(a, k, v)
    need = L.vnx_q8_linear_workspace(ctypes.byref(a))
    assert need >= 2 * 64 * 64 * 4
    a.x, a.x_scale, a.w, a.w_scale, a.y = AT, 2 * AT, 3 * AT, 4 * AT, FAR
    for ws, n in ((None, need), (FAR * 2, need - 1), (FAR * 2 + 8, need)):
        assert L.vnx_q8_linear(ctypes.byref(a), ws, n, None) == _lib.VNX_ERR_WORKSPACE
    for over in (dict(M=0), dict(ldy=63), dict(force_shape=4), dict(K=0)):
        for k, v in over.items():
            old = getattr(a, k)
            setattr(a, k, v)
            assert L.vnx_q8_linear_workspace(ctypes.byref(a)) == 256
            setattr(a, k, old)
