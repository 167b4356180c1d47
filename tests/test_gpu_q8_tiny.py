"""rmsnorm_q8 of rows whose squares fp32 cannot hold, with an eps of that size or none: the norm of such a row is as large as
any other's, and its scale is held to 64 bits."""
import pytest
import torch

import q8_ref as R
from test_gpu_q8_rows import scale_steps

pytestmark = pytest.mark.gpu

# every launch shape: a wave, workgroups of 4, 8 and 16 waves, and rows that are walked
WIDTHS = [5, 8, 96, 1030, 2047, 5000, 9001, 14000, 20001, 33000]


def check(hip, x, w, eps, residual=None):
    """The scale within the roundings of its steps: those of rmsnorm, and none for powers of two."""
    dev = hip.torch_device
    c, s, total = R.rmsnorm(x, w, eps, residual)
    codes, scale, got = hip.rmsnorm_q8(x.to(dev), w.to(dev), eps=eps, residual=None if residual is None else residual.to(dev))
    assert torch.equal(codes.cpu(), c) and torch.equal(got.cpu(), total)
    assert torch.isfinite(s).all()
    assert ((scale.cpu().double() - s).abs() <= scale_steps(x.shape[1]) * R.U * s).all(), (scale.cpu(), s)
    return s


@pytest.mark.parametrize("K", WIDTHS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tiny_rows(hip, K, dtype):
    """Rows from 2^-50 to 2^-95, where squares lose bits and then vanish, beside one of ordinary size and one of zeros."""
    g = R.gen(K)
    x = torch.randn(9, K, generator=g)
    x *= torch.tensor([1.0, 2.0 ** -50, 2.0 ** -55, 2.0 ** -60, 2.0 ** -66, 2.0 ** -74, 2.0 ** -80, 2.0 ** -95, 0.0])[:, None]
    x, w = x.to(dtype), 1 + 0.3 * torch.rand(K, generator=g)
    for eps in (0.0, 2.0 ** -149, 700 * 2.0 ** -149, 1e-37, 2.0 ** -110, 1e-30, 1e-6):
        s = check(hip, x, w, eps)
        if eps == 0.0:                # a norm of about 1: max|t| is between 0.3 and 8 times the root mean square
            assert ((s[:8] * 127 > 0.3) & (s[:8] * 127 < 8)).all() and s[8] == 0


@pytest.mark.parametrize("K", WIDTHS)
def test_residual_of_the_same_size(hip, K):
    g = R.gen(K)
    x, r = (torch.randn(4, K, generator=g) * 2.0 ** -70 for _ in range(2))
    check(hip, x, torch.ones(K), 0.0, r)
    check(hip, x.bfloat16(), torch.ones(K), 0.0, r.bfloat16())


@pytest.mark.parametrize("K", [5, 300, 4096, 33000])
def test_weights_that_lift_the_row(hip, K):
    """Subnormal values under large weights: codes are those of the products, the scale their maximum over the root."""
    g = R.gen(K)
    x = torch.randn(3, K, generator=g) * 2.0 ** -135
    for lift in (2.0 ** 40, 2.0 ** 100):
        check(hip, x, torch.full((K,), lift), 0.0)
    big = torch.ones(K)
    big[0] = 2.0 ** 120               # (one value carries the maximum: 2^-70 * 2^120)
    check(hip, torch.full((2, K), 2.0 ** -70), big, 0.0)


@pytest.mark.parametrize("K", WIDTHS)
@pytest.mark.parametrize("over", [0, 1])
def test_sum_in_place(hip, K, over):
    """The sum over x, or over the residual, of rows that are summed twice: the bits of the call that writes elsewhere."""
    g, dev = R.gen(K), hip.torch_device
    x, r = ((torch.randn(70, K, generator=g) * 2.0 ** -80).to(dev) for _ in range(2))
    x[::3] *= 2.0 ** 80
    w = torch.ones(K, device=dev)
    want = hip.rmsnorm_q8(x, w, eps=0.0, residual=r)
    pair = [x.clone(), r.clone()]
    got = hip.rmsnorm_q8(pair[0], w, eps=0.0, residual=pair[1], sum_out=pair[over])
    assert got[2] is pair[over] and all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.isfinite(got[1]).all() and (got[1] > 0).all()
