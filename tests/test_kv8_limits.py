"""Sizes past what a launch or a product of sizes holds are refused on the host, before any pointer is read (no GPU needed)."""
import ctypes

import pytest

from versenext_amd import _lib

AT = 1 << 40     # an address that is never read
BIG = 2 ** 31 - 1


def _call(cls, f, *rest, **kw):
    a = cls()
    for k, v in kw.items():
        if isinstance(v, (list, tuple)):
            getattr(a, k)[:] = list(v)
        else:
            setattr(a, k, v)
    return f(ctypes.byref(a), *rest)


def _attn(**over):
    kw = dict(q=AT, k_cache=AT, v_cache=AT, k_scale=AT, v_scale=AT, lens=AT, out=AT, q_strides=[64, 64, 64],
              cache_strides=[64, 64, 64], scale_strides=[1, 1], out_strides=[1 << 34, 1 << 14, 64], cap=100, B=1, H=1, Hkv=1,
              Tp=0, N=1, d=64, kv_dtype=_lib.VNX_I8, out_dtype=_lib.VNX_BF16, scale=0.125)
    kw.update(over)
    return _call(_lib.AttnQ8Args, _lib.lib().vnx_tree_attn_q8, None, 0, None, **kw)


@pytest.mark.parametrize("over", [
    # B * Hkv * tiles * splits past 64 bits
    dict(B=1 << 30, H=1 << 30, Hkv=1 << 30), dict(B=1 << 28, H=1 << 29, Hkv=1 << 29, N=97),
    dict(B=BIG, H=BIG, Hkv=BIG),
    # 2^32 threads and more in a launch
    dict(B=1 << 21, H=8, Hkv=8), dict(B=1 << 20, H=32, Hkv=32), dict(B=1 << 21, H=8, Hkv=8, anc=AT),
])
def test_attn(over):
    assert _attn(**over) == _lib.VNX_ERR_UNSUPPORTED


@pytest.mark.parametrize("over", [dict(B=1 << 26, n=1), dict(B=1, n=1 << 26), dict(B=1 << 13, n=(1 << 13) + 1)])
def test_write(over):
    kw = dict(qkv=AT, ldq=48, lens=AT, q_out=AT, k_cache=AT, v_cache=2 * AT, k_scale=4 * AT, v_scale=5 * AT,
              cache_strides=[160, 160, 16], scale_strides=[10, 10], B=1, cap=10, n=1, H=1, Hkv=1, d=16,
              dtype=_lib.VNX_BF16, cache_dtype=_lib.VNX_I8)
    kw.update(over)
    assert _call(_lib.KvWriteArgs, _lib.lib().vnx_kv_write, None, **kw) == _lib.VNX_ERR_UNSUPPORTED


@pytest.mark.parametrize("d,rows", [(256, 1 << 27), (128, 1 << 28), (32, 1 << 30), (64, BIG)])
def test_read(d, rows):
    kw = dict(k_cache=AT, v_cache=AT, k_scale=AT, v_scale=AT, k_out=AT, v_out=1 << 45, cache_strides=[0, 0, d],
              scale_strides=[0, 0], out_strides=[0, 0, d], B=1, cap=rows, rows=rows, Hkv=1, d=d, cache_dtype=_lib.VNX_I8,
              out_dtype=_lib.VNX_BF16)
    assert _call(_lib.KvReadArgs, _lib.lib().vnx_kv_read, None, **kw) == _lib.VNX_ERR_UNSUPPORTED


def test_values_past_their_field():
    """An argument that its field does not hold is a ValueError, as other bad arguments."""
    for pack, cls in ((_lib.pack_kv_write, _lib.KvWriteArgs), (_lib.pack_kv_read, _lib.KvReadArgs),
                      (_lib.pack_attn_q8, _lib.AttnQ8Args)):
        n = sum(getattr(t, "_length_", 1) for _, t in cls._fields_)
        for bad in (1 << 70, "x", None):
            with pytest.raises(ValueError):
                pack(*[bad] * n)
