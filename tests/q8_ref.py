"""Plain forms of the products in 8-bit integers, on the CPU: the codes in the steps that define them (fp32), everything
else in 64 bits."""
import torch

F64, U = torch.float64, 2.0 ** -24
TINY = 2.0 ** -100
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def codes_of(t):
    """(codes, a) of fp32 rows t: rint(t * RN(127 / a)), a = max|t|; rows that have none are zeros."""
    a = t.abs().amax(-1)
    ok = torch.isfinite(a) & (a >= TINY)              # (amax carries a NaN)
    r = torch.where(ok, torch.full_like(a, 127.0) / torch.where(ok, a, torch.ones_like(a)), torch.zeros_like(a))
    c = torch.where(ok[..., None], torch.round(t * r[..., None]), torch.zeros_like(t))
    return c.to(torch.int8), a


def quantize(x):
    """(codes, scale) of rows of any type."""
    c, a = codes_of(x.float())
    s = torch.where(a >= TINY, a / torch.full_like(a, 127.0), torch.zeros_like(a))
    return c, torch.where(torch.isfinite(a), s, torch.full_like(a, float("nan")))


def rmsnorm(x, w, eps, residual=None):
    """(codes, scale in 64 bits, s)."""
    s = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    c, a = codes_of(s.float() * w)
    sc = (a / torch.full_like(a, 127.0)).to(F64) / torch.sqrt(s.to(F64).square().mean(-1) + eps)
    sc = torch.where(a >= TINY, sc, torch.zeros_like(sc))
    return c, torch.where(torch.isfinite(a), sc, torch.full_like(sc, float("nan"))), s


def linear(codes, scale, wq, w_scale, bias=None, residual=None, swiglu=False, out=torch.float32):
    """(y in 64 bits, how far the kernel's may be from it, elementwise).

    The kernel converts the exact sum to fp32, multiplies twice, adds the bias and the residual: half a step (2^-24)
    each of the value it rounds, and half a step of the output's type.  SwiGLU: |silu'| < 1.1, so it carries an error d of
    the gate into 1.1 d |u|; its own steps are an exp (the argument rounded twice to |g| 2^-24 each, 2 steps of its own),
    a sum, a quotient and a product: (8 + 4 |g|) 2^-24 covers them."""
    acc = codes.to(F64) @ wq.to(F64).t()
    v0 = acc * scale.to(F64)[:, None] * w_scale.to(F64).reshape(-1)
    y = v0
    err = 3 * U * v0.abs()
    if bias is not None:
        y = y + bias.to(F64)
        err = err + U * y.abs()
    if swiglu:
        h = y.shape[1] // 2
        g, u, eg, eu = y[:, :h], y[:, h:], err[:, :h], err[:, h:]
        sg = g * torch.sigmoid(g)
        y = sg * u
        err = 1.1 * eg * u.abs() + eu * sg.abs() + (8 + 4 * g.abs()) * U * y.abs() + 1.1 * eg * eu + 1e-37
    if residual is not None:
        y = y + residual.to(F64)
        err = err + U * y.abs()
    small = torch.finfo(out).smallest_normal
    # (the last step of a type ends half a step above its largest value: what lies behind rounds to infinity)
    top = torch.finfo(out).max * (1 + half_step(out))
    if out == torch.float16:
        assert not ((y.abs() - top).abs() <= 2 * err).any()
        y = torch.where(y.abs() > top, y.sign() * float("inf"), y)
    return y, err * 1.01 + half_step(out) * 1.01 * (y.abs().clamp(max=top) + err).clamp(min=small)


def off(got, y, tol):
    """Where a result is further from y than it may be; infinities are equal or wrong."""
    got = got.cpu().double()
    return ((got - y).abs() > tol) & (got != y) | got.isnan()


def codes(g, M, K, low=-127):
    return torch.randint(low, 128, (M, K), generator=g, dtype=torch.int8)


def pitched(c, ld, fill, device):
    """c on the device as rows `ld` apart, the bytes between them `fill`."""
    M, K = c.shape
    b = torch.full((M, ld), fill, dtype=torch.int8, device=device)
    b[:, :K] = c.to(device)
    return b[:, :K]


def scales(g, n):
    return torch.exp(torch.randn(n, generator=g)) * 0.01
