"""Outputs of the 8-bit cache's entries that lie on one another are refused on the host, before any pointer is read (no
GPU needed): workgroups would write the same rows."""
import ctypes
import itertools

import pytest

from versenext_amd import _lib

AT = 1 << 30     # an address that is never read
INVALID = _lib.VNX_ERR_INVALID_ARG


def _call(cls, f, *rest, **kw):
    a = cls()
    for k, v in kw.items():
        if isinstance(v, (list, tuple)):
            getattr(a, k)[:] = list(v)
        else:
            setattr(a, k, v)
    return f(ctypes.byref(a), *rest)


def _write(**over):
    kw = dict(qkv=AT, ldq=32 * 64, lens=AT, q_out=AT, k_cache=AT, v_cache=2 * AT, k_scale=3 * AT, v_scale=4 * AT,
              cache_strides=[8 * 100 * 64, 100 * 64, 64], scale_strides=[800, 100], B=2, cap=100, n=3, H=16, Hkv=8, d=64,
              dtype=_lib.VNX_BF16, cache_dtype=_lib.VNX_I8)
    kw.update(over)
    return _call(_lib.KvWriteArgs, _lib.lib().vnx_kv_write, None, **kw)


def _read(**over):
    kw = dict(k_cache=AT, v_cache=AT, k_scale=AT, v_scale=AT, k_out=AT, v_out=2 * AT,
              cache_strides=[8 * 100 * 64, 100 * 64, 64], scale_strides=[800, 100], out_strides=[8 * 640, 640, 64], B=2,
              cap=100, rows=10, Hkv=8, d=64, cache_dtype=_lib.VNX_I8, out_dtype=_lib.VNX_BF16)
    kw.update(over)
    return _call(_lib.KvReadArgs, _lib.lib().vnx_kv_read, None, **kw)


def _attn(**over):
    kw = dict(q=AT, k_cache=AT, v_cache=AT, k_scale=AT, v_scale=AT, lens=AT, out=AT, q_strides=[16 * 192, 192, 64],
              cache_strides=[8 * 100 * 64, 100 * 64, 64], scale_strides=[800, 100], out_strides=[16 * 192, 192, 64],
              cap=100, B=2, H=16, Hkv=8, Tp=97, N=3, d=64, kv_dtype=_lib.VNX_I8, out_dtype=_lib.VNX_BF16, scale=0.125)
    kw.update(over)
    return _call(_lib.AttnQ8Args, _lib.lib().vnx_tree_attn_q8, None, 0, None, **kw)


@pytest.mark.parametrize("over", [
    dict(cache_strides=[8 * 100 * 64 - 16, 100 * 64, 64]), dict(cache_strides=[8 * 100 * 64, 100 * 64 - 64, 64]),
    dict(cache_strides=[6400, 6400, 64]), dict(cache_strides=[64, 128, 512]), dict(cache_strides=[1 << 20, 32, 80]),
    dict(scale_strides=[800, 99]), dict(scale_strides=[799, 100]), dict(scale_strides=[100, 100]),
    # keys and values on one another: the same tensor, rows shifted by a few bytes, by whole rows, heads and sequences
    dict(v_cache=AT), dict(v_cache=AT + 16), dict(v_cache=AT - 48), dict(v_cache=AT + 64 * 99), dict(v_cache=AT + 6400),
    dict(v_cache=AT - 51200 - 6400 * 7 - 64), dict(v_scale=3 * AT), dict(v_scale=3 * AT + 4 * 99), dict(v_scale=3 * AT - 3200),
    dict(cache_dtype=_lib.VNX_BF16, v_cache=AT + 2 * 51200),
    # codes 128 bytes apart, the values' between the keys' but for 16 bytes
    dict(cache_strides=[8 * 100 * 128, 100 * 128, 128], v_cache=AT + 48),
])
def test_write(over):
    assert _write(**over) == INVALID


@pytest.mark.parametrize("over", [
    dict(out_strides=[0, 640, 64]), dict(out_strides=[8 * 640, 0, 64]), dict(out_strides=[8 * 640, 632, 64]),
    dict(out_strides=[640, 640, 64]), dict(v_out=AT), dict(v_out=AT + 128), dict(v_out=AT + 2 * 5120),
])
def test_read(over):
    assert _read(**over) == INVALID


@pytest.mark.parametrize("over", [
    dict(out_strides=[0, 192, 64]), dict(out_strides=[16 * 192, 0, 64]), dict(out_strides=[16 * 192, 192, 0]),
    dict(out_strides=[16 * 192, 192, 56]), dict(out_strides=[16 * 192, 128, 64]), dict(out_strides=[192, 192, 64]),
])
def test_attn(over):
    assert _attn(**over) == INVALID


def test_layouts_that_stay():
    """The same strides with one sequence, head or row: a stride that is never taken may be anything.  Batch-major, row-major,
    interleaved keys and values.  (No GPU here: the launch itself fails, with another status.)"""
    import torch
    if torch.cuda.is_available():
        pytest.skip("would launch on addresses that do not exist")
    for over in (dict(), dict(B=1, cache_strides=[0, 6400, 64], scale_strides=[0, 100]),
                 dict(cache_strides=[100 * 8 * 64, 64, 8 * 64]),                                    # (B, cap, Hkv, d)
                 dict(cache_strides=[64, 2 * 64, 16 * 64], scale_strides=[100, 200]),               # (cap, Hkv, B, d)
                 dict(cache_strides=[8 * 100 * 128, 100 * 128, 128], v_cache=AT + 64),              # K and V a row
                 dict(cache_strides=[2 * 51200, 6400, 64], v_cache=AT + 51200),                     # K and V a sequence
                 dict(scale_strides=[1600, 200], v_scale=3 * AT + 400),
                 dict(cap=1, cache_strides=[8 * 64, 64, 1 << 20], scale_strides=[8, 1])):
        assert _write(**over) != INVALID, over
    for over in (dict(), dict(out_strides=[640 * 8, 64, 512]), dict(rows=1, out_strides=[512, 64, 64]),
                 dict(out_strides=[8 * 640 * 2, 640, 64], v_out=AT + 2 * 5120)):
        assert _read(**over) != INVALID, over
    for over in (dict(), dict(out_strides=[16 * 192, 64, 16 * 64]), dict(B=1, out_strides=[0, 192, 64])):
        assert _attn(**over) != INVALID, over


def test_small_layouts_against_every_index():
    """Every stride triple of small layouts, keys and values at every distance: accepted only where no element is written
    twice, and always where the dims nest and the two tensors do not meet."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("would launch on addresses that do not exist")
    B, Hkv, cap, d = 2, 2, 3, 16
    seen = [0, 0]
    for st in itertools.product((0, 16, 32, 48, 64, 96, 112), (0, 16, 32, 48, 96, 192), (16, 32, 64, 96)):
        rows = [b * st[0] + h * st[1] + r * st[2] for b in range(B) for h in range(Hkv) for r in range(cap)]
        clash = len({x // 16 for x in rows}) < len(rows)
        for delta in (0, 16, 32, 48, 80, 96, 144, 400):
            got = _write(B=B, Hkv=Hkv, cap=cap, d=d, H=2, n=1, ldq=96, cache_strides=list(st), scale_strides=[100, 10],
                         v_cache=AT + delta)
            meets = {x // 16 for x in rows} & {(x + delta) // 16 for x in rows}
            if clash or meets:
                assert got == INVALID, (st, delta)
            seen[got != INVALID] += 1
    assert min(seen) > 20
