"""Outputs of the 8-bit calls in more dimensions: rows that cannot be written as they lie are a ValueError, empty ones a call
without work."""
import pytest
import torch

import q8_ref as R

pytestmark = pytest.mark.gpu


def _in(hip, *shape):
    g = R.gen(len(shape))
    return R.codes(g, 6, 32).view(*shape, 32).to(hip.torch_device), R.scales(g, 6).view(shape).to(hip.torch_device)


def test_product_into_more_dimensions(hip):
    dev, g = hip.torch_device, R.gen(3)
    c, s = _in(hip, 2, 3)
    w, ws = R.codes(g, 8, 32).to(dev), R.scales(g, 8).to(dev)
    want = hip.linear_q8(c, s, w, ws, out_dtype=torch.float32)
    wide = torch.full((2, 3, 20), 7.0, device=dev)
    out = wide[..., 4:12]                                  # (rows of one pitch: written in place)
    assert hip.linear_q8(c, s, w, ws, out=out) is out and torch.equal(out, want)
    assert wide[..., :4].eq(7).all() and wide[..., 12:].eq(7).all()
    for bad in (torch.zeros(2, 4, 8, device=dev)[:, :3],    # rows of two pitches
                torch.zeros(3, 2, 8, device=dev).transpose(0, 1), torch.zeros(2, 3, 16, device=dev)[..., ::2],
                torch.zeros(1, 3, 8, device=dev).expand(2, 3, 8)):
        with pytest.raises(ValueError):
            hip.linear_q8(c, s, w, ws, out=bad)
        assert bad.eq(0).all()
    none = torch.zeros(2, 3, 0, device=dev)
    assert hip.linear_q8(c, s, w[:0], ws[:0], out=none) is none
    assert hip.linear_q8(c[:0], s[:0], w, ws, out=wide[:0, :, :8]).shape == (0, 3, 8)


def test_sum_into_more_dimensions(hip):
    dev = hip.torch_device
    x = torch.randn(2, 3, 32, generator=R.gen(1)).to(dev)
    w = torch.ones(32, device=dev)
    want = hip.rmsnorm_q8(x, w, residual=x)
    out = torch.zeros(2, 3, 40, device=dev)[..., 4:36]
    got = hip.rmsnorm_q8(x, w, residual=x, sum_out=out)
    assert got[2] is out and all(torch.equal(a, b) for a, b in zip(got, want))
    for bad in (torch.zeros(2, 4, 32, device=dev)[:, :3], torch.zeros(3, 2, 32, device=dev).transpose(0, 1)):
        with pytest.raises(ValueError):
            hip.rmsnorm_q8(x, w, residual=x, sum_out=bad)
        assert bad.eq(0).all()
    assert hip.rmsnorm_q8(x[:0], w, residual=x[:0], sum_out=out[:0])[2].shape == (0, 3, 32)
