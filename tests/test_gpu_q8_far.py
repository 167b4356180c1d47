"""8-bit calls whose tensors pass 2^31 bytes or elements: the last rows and columns have the bits of a call on them alone."""
import pytest
import torch

import q8_ref as R

pytestmark = pytest.mark.gpu

FAR = (1 << 31) // 4096 + 300        # rows of 4,096 bytes


def _codes(dev, rows, K):
    """Codes of a pattern that no two near rows share."""
    a = torch.arange(rows, device=dev, dtype=torch.int32)[:, None] * 37 + torch.arange(K, device=dev, dtype=torch.int32) * 11
    return (a % 251 - 125).to(torch.int8)


@pytest.mark.parametrize("which", ["x", "w", "y"])
def test_product(hip, which):
    dev, g = hip.torch_device, R.gen(1)
    if which == "y":                                      # 9,000 x 248,320 of y
        c, w = R.codes(g, 9000, 64).to(dev), R.codes(g, 248320, 64).to(dev)
    else:
        near, far = R.codes(g, 40, 4096).to(dev), torch.empty((FAR, 4096), dtype=torch.int8, device=dev)
        for r in range(0, FAR, 1 << 16):
            far[r:r + (1 << 16)] = _codes(dev, min(1 << 16, FAR - r), 4096)
        far[-300:] = R.codes(g, 300, 4096).to(dev)
        c, w = (far, near) if which == "x" else (near, far)
    s, ws = R.scales(g, c.shape[0]).to(dev), R.scales(g, w.shape[0]).to(dev)
    y = hip.linear_q8(c, s, w, ws)
    for rows, cols in ((slice(0, 33), slice(0, 65)), (slice(-33, None), slice(-65, None)), (slice(-300, -290), slice(0, 40))):
        want = hip.linear_q8(c[rows].contiguous(), s[rows], w[cols].contiguous(), ws[cols])
        assert torch.equal(y[rows, cols], want)
    del y, c, w
    torch.cuda.empty_cache()


def test_rows(hip):
    dev, g = hip.torch_device, R.gen(2)
    x = torch.empty((FAR, 4096), dtype=torch.bfloat16, device=dev)
    for r in range(0, FAR, 1 << 16):
        x[r:r + (1 << 16)] = _codes(dev, min(1 << 16, FAR - r), 4096).to(torch.bfloat16) / 7
    x[-50:] = torch.randn(50, 4096, generator=g).bfloat16().to(dev)
    w = torch.ones(4096, device=dev)
    last = x[-50:].clone()
    codes, scale = hip.quantize_rows(x)
    a, b = hip.quantize_rows(last)
    assert torch.equal(codes[-50:], a) and torch.equal(scale[-50:], b)
    assert torch.equal(hip.dequantize_rows(codes, scale, torch.bfloat16)[-50:], hip.dequantize_rows(a, b, torch.bfloat16))
    a, b, s = hip.rmsnorm_q8(last, w, residual=last)
    codes, scale, total = hip.rmsnorm_q8(x, w, residual=x, sum_out=x)
    assert torch.equal(codes[-50:], a) and torch.equal(scale[-50:], b) and torch.equal(x[-50:], s)
    del x, codes, scale, total
    torch.cuda.empty_cache()
