"""What 8 bits cost: kv_write and tree_attention_q8 against the 64-bit attention over the rows as they were before they were
quantised, within the error of the codes.

A value of a row with scale s is off by at most dv = s / 2 (int8) or max(2^-4 |v|, 2^-10 s) (e4m3), and 2^-22 |v| of the
scale's own arithmetic.  A score is off by at most D = scale sum |q| dk, so every probability by a factor within exp(+-2 D),
D the largest of the node's keys:
  |out - ref| <= (exp(2 D) - 1) sum p |v| + exp(2 D) sum p dv,
and on top the attention's own bar (2^-10 of the terms, half a step of the output type), on terms of up to |v| + dv."""
import math

import pytest
import torch

import kv8_ref as R

pytestmark = pytest.mark.gpu

I8, E4 = torch.int8, torch.float8_e4m3fn


def _off(x, dtype):
    """The largest error of a row's values."""
    s = x.abs().amax(-1, keepdim=True) / R.TOP[dtype]
    half = s / 2 if dtype == I8 else torch.maximum(2.0 ** -4 * x.abs(), 2.0 ** -10 * s)
    return half.expand_as(x) + 2.0 ** -22 * x.abs()


@pytest.mark.parametrize("dtype", [I8, E4], ids=["int8", "e4m3"])
@pytest.mark.parametrize("d,H,Hkv,T,n", [(64, 4, 2, 300, 5), (128, 8, 2, 40, 1), (64, 2, 2, 0, 90), (64, 16, 8, 1500, 7)])
def test_against_the_rows_before_the_codes(hip, d, H, Hkv, T, n, dtype):
    dev = hip.torch_device
    g = R.gen(T + n)
    cap = T + n
    x = torch.randn(1, cap, H + 2 * Hkv, d, generator=g) * torch.exp(0.4 * torch.randn(d, generator=g))
    x[:, :, :H] *= 0.3
    kc, vc = (torch.zeros(1, Hkv, cap, d, dtype=dtype, device=dev) for _ in range(2))
    ks, vs = (torch.zeros(1, Hkv, cap, device=dev) for _ in range(2))
    if T:
        hip.kv_write(x[:, :T].reshape(1, T, -1), kc, vc, [0], ks, vs)
    q = hip.kv_write(x[:, T:].reshape(1, n, -1), kc, vc, [T], ks, vs)
    o = hip.tree_attention_q8(q, kc, vc, ks, vs, [T]).cpu().to(R.F64)[0]
    k, v = (x[0, :, a:a + Hkv].to(R.F64).transpose(0, 1).repeat_interleave(H // Hkv, 0) for a in (H, H + Hkv))
    dk, dv = _off(k, dtype), _off(v, dtype)
    qf = q.cpu().to(R.F64)[0]
    hide = torch.arange(cap)[None] > T + torch.arange(n)[:, None]
    p = torch.softmax((qf @ k.transpose(-1, -2) / math.sqrt(d)).masked_fill(hide, -math.inf), -1)
    D = (qf.abs() @ dk.transpose(-1, -2) / math.sqrt(d)).masked_fill(hide, 0.0).amax(-1, keepdim=True)
    ref, mag, off = p @ v, p @ v.abs(), p @ dv
    grow = torch.exp(2 * D)
    code = (grow - 1) * mag + grow * off
    err = (o - ref).abs()
    assert (err <= code + 2.0 ** -10 * grow * (mag + off) + 2.0 ** -8 * (ref.abs() + code) + 2.0 ** -25).all()
    # in the norm the codes cost 0.01 (int8) and 0.03 (e4m3) of such inputs by the 64-bit forms alone
    assert (err.norm() / ref.norm()).item() <= (0.02 if dtype == I8 else 0.06)
