"""The Python binding of the 8-bit KV cache's entries leaves every call that is not on the GPU as the kernels read it to
HipBackend's general path (None), without touching anything (no GPU needed)."""
import numpy as np
import pytest
import torch

from versenext_amd import _lib


def test_calls_off_the_gpu_are_left():
    b = _lib.bind()
    k = torch.zeros(1, 2, 8, 64, dtype=torch.int8)
    s = torch.zeros(1, 2, 8)
    x = torch.zeros(1, 1, 6 * 64)
    lens = torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16)
    for kc, ks in ((k, s), (k, None), (None, None), (k.numpy(), s), (k[0], s), (torch.zeros(0, 2, 8, 64), s)):
        assert b.kv_write(0, 0, kc, kc, ks, ks, x, lens, None, None, None, None, 1e-6) is None
        assert b.kv_read(0, 0, kc, kc, ks, ks, None, None, torch.float32) is None
        for anc in (None, np.ones(1, dtype=np.uint64), np.ones(1), [1], "x"):
            assert b.tree_attn_q8(0, 0, kc, kc, ks, ks, q, lens, anc, None, None, None, 0, None, torch.bfloat16,
                                  None) is None


def test_wrong_argument_counts_and_types_are_left():
    b = _lib.bind()
    assert b.kv_write() is None and b.kv_read(0, 0) is None and b.tree_attn_q8(*range(16)) is None
    k = torch.zeros(1, 2, 8, 64, dtype=torch.int8)
    s = torch.zeros(1, 2, 8)
    for dev, st in ((-1, 0), ("a", 0), (0, None), (2 ** 70, 0), (0, 1.5)):
        assert b.kv_read(dev, st, k, k, s, s, None, None, torch.float32) is None


def test_init_wants_addresses():
    b = _lib.bind()
    with pytest.raises(TypeError):
        b.init()
    with pytest.raises(ValueError):
        b.init(1, 2, 3, 0)
    with pytest.raises(TypeError):
        b.init("a", 1, 1, 1)
