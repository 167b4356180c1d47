"""The argument checks of the 8-bit KV cache's entries: bad calls are refused on the host, before anything is launched and
before any pointer is read (no GPU needed)."""
import ctypes

import pytest

from versenext_amd import _lib

AT = 1 << 20     # an address that is never read


def _block(cls, **over):
    a = cls()
    for k, v in over.items():
        if isinstance(v, (list, tuple)):
            getattr(a, k)[:] = list(v)
        else:
            setattr(a, k, v)
    return a


def _write(**over):
    kw = dict(qkv=AT, ldq=32 * 64, lens=AT, cos_table=AT, sin_table=AT, table_rows=100, q_norm=AT, k_norm=AT, q_out=AT,
              k_cache=AT, v_cache=AT, k_scale=AT, v_scale=AT, cache_strides=[8 * 100 * 64, 100 * 64, 64],
              scale_strides=[800, 100], B=2, cap=100, n=3, H=16, Hkv=8, d=64, dtype=_lib.VNX_BF16,
              cache_dtype=_lib.VNX_I8, eps=1e-6)
    kw.update(over)
    return _lib.lib().vnx_kv_write(ctypes.byref(_block(_lib.KvWriteArgs, **kw)), None)


def _read(**over):
    kw = dict(k_cache=AT, v_cache=AT, k_scale=AT, v_scale=AT, start=AT, k_out=AT, v_out=AT,
              cache_strides=[8 * 100 * 64, 100 * 64, 64], scale_strides=[800, 100],
              out_strides=[8 * 100 * 64, 100 * 64, 64], B=2, cap=100, rows=100, Hkv=8, d=64, cache_dtype=_lib.VNX_I8,
              out_dtype=_lib.VNX_BF16)
    kw.update(over)
    return _lib.lib().vnx_kv_read(ctypes.byref(_block(_lib.KvReadArgs, **kw)), None)


def _attn(ws=None, **over):
    kw = dict(q=AT, k_cache=AT, v_cache=AT, k_scale=AT, v_scale=AT, lens=AT, out=AT, k_seg2=AT, v_seg2=AT, gates=AT,
              q_strides=[16 * 192, 192, 64], cache_strides=[8 * 100 * 64, 100 * 64, 64], scale_strides=[800, 100],
              out_strides=[16 * 192, 192, 64], seg2_strides=[0, 640, 64], cap=100, B=2, H=16, Hkv=8, Tp=97, N=3,
              d=64, T2=10, window=0, kv_dtype=_lib.VNX_I8, out_dtype=_lib.VNX_BF16, scale=0.125)
    kw.update(over)
    return _lib.lib().vnx_tree_attn_q8(ctypes.byref(_block(_lib.AttnQ8Args, **kw)), ws, 0, None)


INVALID, UNSUPPORTED = _lib.VNX_ERR_INVALID_ARG, _lib.VNX_ERR_UNSUPPORTED


@pytest.mark.parametrize("status,over", [
    (INVALID, dict(qkv=None)), (INVALID, dict(lens=None)), (INVALID, dict(q_out=None)), (INVALID, dict(k_cache=None)),
    (INVALID, dict(v_scale=None)), (INVALID, dict(sin_table=None)), (INVALID, dict(table_rows=0)),
    (INVALID, dict(eps=-1.0)), (INVALID, dict(eps=float("nan"))), (INVALID, dict(n=0)), (INVALID, dict(H=0)),
    (INVALID, dict(Hkv=0)), (INVALID, dict(B=-1)), (INVALID, dict(cap=0)), (INVALID, dict(ldq=32 * 64 - 8)),
    (INVALID, dict(cache_strides=[51200, 6400, 48])), (INVALID, dict(scale_strides=[-1, 100])),
    (INVALID, dict(cache_strides=[0, 6400, 64])), (INVALID, dict(cache_strides=[51200, 0, 64])),
    (INVALID, dict(scale_strides=[0, 100])), (INVALID, dict(scale_strides=[800, 0])),
    (UNSUPPORTED, dict(dtype=_lib.VNX_I8)), (UNSUPPORTED, dict(cache_dtype=_lib.VNX_F16)),
    (UNSUPPORTED, dict(cache_dtype=9)), (UNSUPPORTED, dict(d=48)), (UNSUPPORTED, dict(d=8)), (UNSUPPORTED, dict(d=512)),
    (UNSUPPORTED, dict(qkv=AT + 8)), (UNSUPPORTED, dict(ldq=32 * 64 + 4)), (UNSUPPORTED, dict(k_cache=AT + 8)),
    (UNSUPPORTED, dict(cache_strides=[51200, 6400, 72])), (UNSUPPORTED, dict(cache_strides=[-51200, 6400, 64])),
    (UNSUPPORTED, dict(cos_table=AT + 4)), (UNSUPPORTED, dict(q_norm=AT + 4)), (UNSUPPORTED, dict(k_scale=AT + 2)),
    (UNSUPPORTED, dict(lens=AT + 2)), (UNSUPPORTED, dict(B=1 << 26, n=4)), (UNSUPPORTED, dict(B=1 << 40, n=1 << 30)),
    (UNSUPPORTED, dict(H=2 ** 31 - 1, Hkv=2 ** 31 - 1, ldq=1 << 50)), (0, dict(B=0, qkv=None, lens=None)),
])
def test_write_refusals(status, over):
    assert _write(**over) == status


@pytest.mark.parametrize("status,over", [
    (INVALID, dict(k_cache=None)), (INVALID, dict(k_scale=None)), (INVALID, dict(v_out=None)), (INVALID, dict(rows=-1)),
    (INVALID, dict(Hkv=0)), (INVALID, dict(cap=0)), (INVALID, dict(out_strides=[51200, 6400, 32])),
    (INVALID, dict(scale_strides=[800, -1])), (UNSUPPORTED, dict(cache_dtype=_lib.VNX_F16)),
    (UNSUPPORTED, dict(out_dtype=_lib.VNX_I8)), (UNSUPPORTED, dict(d=80)), (UNSUPPORTED, dict(v_out=AT + 8)),
    (UNSUPPORTED, dict(out_strides=[51200, 6400, 68])), (UNSUPPORTED, dict(start=AT + 1)),
    (UNSUPPORTED, dict(B=1 << 30)), (0, dict(B=0, k_cache=None)), (0, dict(rows=0, k_out=None)),
])
def test_read_refusals(status, over):
    assert _read(**over) == status


@pytest.mark.parametrize("status,over", [
    (INVALID, dict(q=None)), (INVALID, dict(k_cache=None)), (INVALID, dict(v_scale=None)), (INVALID, dict(lens=None)),
    (INVALID, dict(out=None)), (INVALID, dict(k_seg2=None)), (INVALID, dict(gates=None)), (INVALID, dict(N=0)),
    (INVALID, dict(Tp=-1)), (INVALID, dict(Tp=98)), (INVALID, dict(H=15)), (INVALID, dict(Hkv=0)), (INVALID, dict(T2=-1)),
    (INVALID, dict(window=-1)), (INVALID, dict(scale=0.0)), (INVALID, dict(scale=float("inf"))),
    (INVALID, dict(scale=float("nan"))), (INVALID, dict(anc=AT, anc_batch_stride=-1)),
    (INVALID, dict(cache_strides=[51200, 6400, 48])), (INVALID, dict(scale_strides=[800, -4])),
    (UNSUPPORTED, dict(d=32)), (UNSUPPORTED, dict(kv_dtype=_lib.VNX_BF16)), (UNSUPPORTED, dict(out_dtype=_lib.VNX_F32)),
    (UNSUPPORTED, dict(anc=AT, N=65, Tp=30)), (UNSUPPORTED, dict(anc=AT, window=2)), (UNSUPPORTED, dict(anc=AT + 4)),
    (UNSUPPORTED, dict(q=AT + 8)), (UNSUPPORTED, dict(v_cache=AT + 8)), (UNSUPPORTED, dict(out=AT + 8)),
    (UNSUPPORTED, dict(q_strides=[4096 + 4, 192, 64])), (UNSUPPORTED, dict(out_strides=[4096, 196, 64])),
    (UNSUPPORTED, dict(cache_strides=[51200, 6400, 72])), (UNSUPPORTED, dict(seg2_strides=[0, 644, 64])),
    (UNSUPPORTED, dict(seg2_strides=[0, 640, 1 << 24])), (UNSUPPORTED, dict(cache_strides=[0, 0, 1 << 25])),
    (UNSUPPORTED, dict(cap=2 ** 31)), (UNSUPPORTED, dict(B=1 << 24, N=80, Tp=20)), (0, dict(B=0, q=None, lens=None)),
])
def test_attn_refusals(status, over):
    assert _attn(**over) == status


def test_packed_blocks_are_the_structures():
    """struct.pack gives the bytes of the ctypes structure with the same values."""
    for cls, pack in ((_lib.KvWriteArgs, _lib.pack_kv_write), (_lib.KvReadArgs, _lib.pack_kv_read),
                      (_lib.AttnQ8Args, _lib.pack_attn_q8)):
        vals, a, n = [], cls(), 3
        for name, t in cls._fields_:
            k = getattr(t, "_length_", 0)
            these = list(range(n, n + max(k, 1)))
            n += max(k, 1)
            vals += these
            if k:
                getattr(a, name)[:] = these
            else:
                setattr(a, name, these[0])
        assert pack(*vals) == bytes(a)


def test_workspace_query_of_refused_sizes():
    for over in (dict(d=32), dict(N=0), dict(H=3, Hkv=2)):
        kw = dict(B=1, H=2, Hkv=1, Tp=10, N=2, d=64, cap=100, kv_dtype=_lib.VNX_I8, out_dtype=_lib.VNX_BF16)
        kw.update(over)
        assert _lib.lib().vnx_tree_attn_q8_workspace(ctypes.byref(_block(_lib.AttnQ8Args, **kw))) == 256
    assert _lib.lib().vnx_tree_attn_q8_workspace(None) == 256
