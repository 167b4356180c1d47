"""w8a8 models whose MoD layers no packed kernel takes: the 8-bit calls against the plain forms, the stream between them."""
import pytest
import torch

from test_gpu_q8_model import _cfg, _check, _spy, _weights
from versenext_amd import model as VM

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pattern", [("mod",), ("mod", "trisparse"), ("trisparse", "mod", "mod")])
@pytest.mark.parametrize("dim,heads,n", [(136, 2, 9), (136, 2, 70), (256, 4, 300)])
def test_forward(hip, dim, heads, n, pattern):
    cfg = _cfg(heads=heads, kv=heads // 2, dim=dim, pattern=pattern, V=301)
    m = VM.CometSparkGPU(cfg, _weights(cfg), hip, 2, n + 20, w8a8=True)
    rec = _spy(m, hip)
    dev = hip.torch_device
    lens = torch.zeros(2, dtype=torch.int32, device=dev)
    for k in (n, 1):
        tok = torch.randint(0, 301, (2, k), generator=torch.Generator().manual_seed(k)).to(dev)
        rec.calls.clear()
        h = m.forward(tok, lens)
        lens += k
        m.logits(h)
        assert torch.isfinite(h).all()
        want = [c for kind in pattern for c in ["rmsnorm_q8", "linear_q8", "quantize_rows", "linear_q8"]
                + (["rmsnorm_q8", "linear_q8", "quantize_rows", "linear_q8"] if kind == "trisparse" else [])]
        assert [c[0] for c in rec.calls] == want + ["quantize_rows", "linear_q8"]
        for c in rec.calls:
            _check(c)


def test_next_to_the_bf16_model(hip):
    """Routing may differ where two experts are close, so the bound is loose: 2 layers, 8-bit products in the attention
    alone (0.9% an operand, 1.3% a product, four of them: 5.2%), and as much again for a token in ten routed otherwise."""
    cfg = _cfg(heads=2, kv=1, dim=136, pattern=("mod", "trisparse"), V=301)
    W = _weights(cfg)
    a, b = (VM.CometSparkGPU(cfg, W, hip, 1, 60, w8a8=q) for q in (True, False))
    tok = torch.arange(50, device=hip.torch_device).view(1, 50)
    lens = torch.zeros(1, dtype=torch.int32, device=hip.torch_device)
    x, y = a.forward(tok, lens), b.forward(tok, lens)
    assert 0 < (x - y).norm() <= 0.104 * y.norm()
