"""The backend without the binding: the 8-bit cache's calls give the same bits."""
import pytest
import torch

import kv8_ref as R
from versenext_amd import _lib

pytestmark = pytest.mark.gpu


def test_general_path_alone(hip, monkeypatch):
    dev = hip.torch_device
    g = R.gen(3)
    x = torch.randn(2, 3, 8 * 64, generator=g).to(torch.bfloat16).to(dev)
    lens = torch.tensor([4, 11], dtype=torch.int32, device=dev)
    got = []
    for bind in (_lib.bind(), _lib.NoBind):
        monkeypatch.setattr(hip, "_bind", bind)
        (kc, ks), (vc, vs) = (R.cache(R.gen(s), 2, 2, 600, 64, torch.int8) for s in (1, 2))
        kc, vc, ks, vs = (t.to(dev) for t in (kc, vc, ks, vs))
        q = hip.kv_write(x, kc, vc, lens, ks, vs)
        got.append([q, kc, vc, ks, vs, *hip.kv_read(kc, vc, ks, vs, start=lens, rows=3),
                    hip.tree_attention_q8(q, kc, vc, ks, vs, lens, max_len=590)])
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_a_backend_without_it(hip, monkeypatch):
    def missing():
        raise RuntimeError("vnx binding not found")

    monkeypatch.setattr(_lib, "bind", missing)
    with pytest.warns(RuntimeWarning, match="not found"):
        b = type(hip)("rocm:0")
    assert b._bind is _lib.NoBind
    assert b.argmax(torch.tensor([[1.0, 3.0, 2.0]], device=b.torch_device)).item() == 1
