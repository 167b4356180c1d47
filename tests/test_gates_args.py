"""Argument checks of the attention operators' gates without a second segment: refused on the host, before any pointer is
read (no GPU needed)."""
import ctypes

from versenext_amd import _lib

AT = 1 << 20     # an address that is never read


def test_q8_gates_on_four_bytes():
    a = _lib.AttnQ8Args()
    a.q = a.k_cache = a.v_cache = a.k_scale = a.v_scale = a.lens = a.out = AT
    a.q_strides[:] = a.out_strides[:] = [128, 64, 64]
    a.cache_strides[:] = [640, 640, 64]
    a.scale_strides[:] = [10, 10]
    a.cap, a.B, a.H, a.Hkv, a.Tp, a.N, a.d, a.scale = 10, 1, 2, 1, 4, 1, 64, 1.0
    a.kv_dtype, a.out_dtype, a.gates = _lib.VNX_I8, _lib.VNX_BF16, AT + 2
    assert _lib.lib().vnx_tree_attn_q8(ctypes.byref(a), None, 0, None) == _lib.VNX_ERR_UNSUPPORTED


def test_tree_and_chain_gates_on_four_bytes():
    for f32 in (0, 1):
        a = _lib.TreeAttnArgs()
        a.q = a.k_tree = a.v_tree = a.anc = a.out = AT
        a.B, a.H, a.Hkv, a.Tp, a.N, a.d, a.scale, a.f32_rows = 1, 2, 1, 0, 1, 16 if f32 else 64, 1.0, f32
        a.out_dtype, a.gates = _lib.VNX_F32, AT + 2
        assert _lib.lib().vnx_tree_attn(ctypes.byref(a), None, 0, None) == _lib.VNX_ERR_INVALID_ARG
    a = _lib.TreeAttnArgs()
    a.q = a.k_cache = a.v_cache = a.out = AT
    a.B, a.H, a.Hkv, a.Tp, a.N, a.d, a.scale, a.out_dtype, a.gates = 1, 2, 1, 0, 1, 64, 1.0, _lib.VNX_BF16, AT + 2
    assert _lib.lib().vnx_chain_attn(ctypes.byref(a), None) == _lib.VNX_ERR_INVALID_ARG
