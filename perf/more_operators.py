"""Timed cases of products in 8-bit integers: the product, and what makes the codes that it reads.

Each case is a dict of plain values; its "kind" names the operator:

  norm    HipBackend.rmsnorm_q8: a residual added to the stream, the sum, and its RMS norm as codes and a scale a row;
          then HipBackend.dequantize_rows, the values that the codes stand for
  rows    HipBackend.quantize_rows, then HipBackend.dequantize_rows
  linear  HipBackend.linear_q8: codes and scales of M rows times an INT8 weight with a scale a row (quant.quantize_int8),
          with a bias, a residual or SwiGLU where the case has them
  ffn     the calls as a feed-forward layer makes them: rmsnorm_q8, linear_q8 of gate and up rows with SwiGLU (bfloat16
          out), quantize_rows, linear_q8

A row x is held as its codes and one 32-bit scale:
  a = max|x|, scale = a / 127, code = round(x * (127 / a))
(nearest, ties to even) and stands for code * scale.  A norm's codes come from t = s * w, s the sum in the stream's type,
and its scale is that of t over the root of mean(s^2) + EPS.

`own` false computes the plain form with elementary torch operations in 32 bits, each operator's result rounded once;
true makes the framework's calls.  Rows of 1,024, an FFN of 2,752 or 4,096 and the vocabulary of 248,320 are
CometSparkV05's and its draft's.
"""
from __future__ import annotations

import math

import torch

own = False

_DEV = torch.device("cuda:0")
_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6


def listed():
    return [
        # one user's token: the residual stream in 32 bits
        dict(name="norm_1x1024_f32", kind="norm", M=1, D=1024, x="f32", res="bf16"),
        # eight prompts of 1,024 tokens, rows of 4,096, the stream in 16 bits
        dict(name="norm_8192x4096_bf16", kind="norm", M=8192, D=4096, x="bf16", res="bf16"),
        # a decode batch's activations before the down product
        dict(name="rows_32x2752_bf16", kind="rows", M=32, K=2752, x="bf16"),
        # long rows in 32 bits whose codes do not fill their last 16 bytes
        dict(name="rows_4096x8200_f32", kind="rows", M=4096, K=8200, x="f32"),
        # one token through a q | k | v projection
        dict(name="linear_1x2048x1024", kind="linear", M=1, N=2048, K=1024, out="bf16", bias=False, res="", swiglu=False),
        # a verify round of one user with sizes that no tile divides
        dict(name="linear_7x1003x1000_bias_f16", kind="linear", M=7, N=1003, K=1000, out="f16", bias=True, res="",
             swiglu=False),
        # a decode batch's down product into the residual stream
        dict(name="linear_32x1024x4096_res_f32", kind="linear", M=32, N=1024, K=4096, out="f32", bias=False, res="f32",
             swiglu=False),
        # the LM head over 32 x 7 verified rows
        dict(name="linear_224x248320x1024", kind="linear", M=224, N=248320, K=1024, out="bf16", bias=False, res="",
             swiglu=False),
        # the prompts of four sequences through gate and up
        dict(name="linear_2048x5504x1024_swiglu", kind="linear", M=2048, N=5504, K=1024, out="bf16", bias=False, res="",
             swiglu=True),
        # a large product
        dict(name="linear_8192x8192x8192", kind="linear", M=8192, N=8192, K=8192, out="bf16", bias=False, res="",
             swiglu=False),
        # a verify round's feed-forward layer
        dict(name="ffn_224x1024x2752", kind="ffn", M=224, D=1024, H=2752, x="f32", res="bf16"),
        # a long prompt's feed-forward layer, a wider model
        dict(name="ffn_4096x4096x10944", kind="ffn", M=4096, D=4096, H=10944, x="bf16", res="bf16"),
    ]


# ---------------------------------------------------------------------------
# Drawn cases
# ---------------------------------------------------------------------------
def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A row's length: mostly a multiple of 64, as models have it, or any number."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.3 else max(64, n // 64 * 64)


def draw(rng):
    kind = rng.choice(["norm", "rows", "linear", "linear", "linear", "linear", "ffn"])
    x = rng.choice(["f32", "bf16", "bf16", "f16"])
    if kind == "norm":
        return dict(kind=kind, M=_log_int(rng, 1, 8192), D=_width(rng, 64, 4096), x=x, res=rng.choice(["", "bf16", x]))
    if kind == "rows":
        return dict(kind=kind, M=_log_int(rng, 1, 4096), K=_width(rng, 64, 8200), x=x)
    if kind == "ffn":
        M = _log_int(rng, 1, 4096)
        D = _log_int(rng, 4, 64) * 64
        return dict(kind=kind, M=M, D=D, H=_log_int(rng, 4, 171) * 64, x=rng.choice(["f32", "bf16"]), res="bf16")
    if rng.random() < 0.15:                                       # an LM head
        return dict(kind=kind, M=_log_int(rng, 1, 256), N=_log_int(rng, 32000, 248320), K=_log_int(rng, 8, 16) * 64,
                    out=rng.choice(["f32", "bf16"]), bias=False, res="", swiglu=False)
    step = rng.choice(["decode", "verify", "prompt"])
    M = _log_int(rng, 1, 64) if step == "decode" else _log_int(rng, 65, 512) if step == "verify" \
        else _log_int(rng, 513, 8192)
    swiglu = rng.random() < 0.25
    N = _width(rng, 64, 8192)
    return dict(kind=kind, M=M, N=N + N % 2 if swiglu else N, K=_width(rng, 64, 8192),
                out=rng.choice(["bf16", "bf16", "f16", "f32"]), bias=rng.random() < 0.3,
                res="" if swiglu else rng.choice(["", "", "f32", "bf16"]), swiglu=swiglu)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _rows(g, *shape):
    """Rows as layers give them: channels of different strength, rows of different strength."""
    return torch.randn(shape, generator=g, device=_DEV) * torch.exp(
        0.5 * torch.randn(shape[-1], generator=g, device=_DEV)) * torch.exp(
        0.5 * torch.randn((shape[0], 1), generator=g, device=_DEV))


def _quantise(x):
    """(codes, scales) of 32-bit rows."""
    a = x.abs().amax(-1, keepdim=True)
    codes = torch.round(x * torch.div(torch.full_like(a, 127.0), a)).to(torch.int8)
    return codes, torch.div(a, torch.full_like(a, 127.0)).squeeze(-1)


def _pitched(codes):
    """Codes as the framework holds them: rows on 16 bytes."""
    M, K = codes.shape
    buf = torch.zeros((M, -(-K // 16) * 16), dtype=torch.int8, device=_DEV)
    buf[:, :K] = codes
    return buf[:, :K]


def _weight(g, N, K):
    """An INT8 weight and its scales."""
    codes, scale = _quantise(torch.randn((N, K), generator=g, device=_DEV) / math.sqrt(K))
    return _pitched(codes), scale


def _prepare(case, seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(int(seed) * 1000003 + 17)
    kind, M = case["kind"], case["M"]
    if kind == "rows":
        return dict(x=_rows(g, M, case["K"]).to(_DT[case["x"]]))
    if kind == "linear":
        codes, scale = _quantise(_rows(g, M, case["K"]))
        wq, ws = _weight(g, case["N"], case["K"])
        return dict(codes=_pitched(codes), scale=scale, wq=wq, w_scale=ws,
                    bias=torch.randn(case["N"], generator=g, device=_DEV) if case["bias"] else None,
                    residual=_rows(g, M, case["N"]).to(_DT[case["res"]]) if case["res"] else None)
    D = case["D"]
    s = dict(x=_rows(g, M, D).to(_DT[case["x"]]),
             residual=_rows(g, M, D).to(_DT[case["res"]]) if case["res"] else None,
             weight=1.0 + 0.1 * torch.randn(D, generator=g, device=_DEV))
    if kind == "ffn":
        s["up"] = _weight(g, 2 * case["H"], D)
        s["down"] = _weight(g, D, case["H"])
    return s


def prepare(case, seed):
    return dict(case=case, x=_prepare(case, seed))


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------
_backend = None


def _hip():
    global _backend
    if _backend is None:
        from versenext_amd import get_backend
        _backend = get_backend("rocm:0")
    return _backend


def _run_own(case, x):
    hip = _hip()
    kind = case["kind"]
    if kind == "rows":
        codes, scale = hip.quantize_rows(x["x"])
        return hip.dequantize_rows(codes, scale, out_dtype=torch.bfloat16)
    if kind == "linear":
        return hip.linear_q8(x["codes"], x["scale"], x["wq"], x["w_scale"], bias=x["bias"], residual=x["residual"],
                             swiglu=case["swiglu"], out_dtype=_DT[case["out"]])
    codes, scale, s = hip.rmsnorm_q8(x["x"], x["weight"], eps=EPS, residual=x["residual"])
    if kind == "norm":
        return dict(sum=s, values=hip.dequantize_rows(codes, scale, out_dtype=torch.bfloat16))
    act = hip.linear_q8(codes, scale, *x["up"], swiglu=True, out_dtype=torch.bfloat16)
    codes, scale = hip.quantize_rows(act)
    return dict(sum=s, y=hip.linear_q8(codes, scale, *x["down"], out_dtype=torch.bfloat16))


# ---------------------------------------------------------------------------
# The plain form
# ---------------------------------------------------------------------------
def _plain_norm(x):
    """(codes, scales, sum)"""
    s = x["x"]
    if x["residual"] is not None:
        s = (s.to(torch.float32) + x["residual"].to(torch.float32)).to(s.dtype)
    v = s.to(torch.float32)
    codes, scale = _quantise(v * x["weight"])
    return codes, scale / torch.sqrt((v * v).mean(-1) + EPS), s


def _plain_linear(codes, scale, wq, w_scale, out, bias=None, residual=None, swiglu=False):
    y = torch.matmul(codes.to(torch.float32), wq.to(torch.float32).t()) * scale.unsqueeze(-1) * w_scale
    if bias is not None:
        y = y + bias
    if swiglu:
        gate, up = y.chunk(2, dim=-1)
        y = gate / (1.0 + torch.exp(-gate)) * up
    if residual is not None:
        y = y + residual.to(torch.float32)
    return y.to(out)


def _values(codes, scale):
    return (codes.to(torch.float32) * scale.unsqueeze(-1)).to(torch.bfloat16)


def run(state):
    case, x = state["case"], state["x"]
    if own:
        return _run_own(case, x)
    kind = case["kind"]
    if kind == "rows":
        return _values(*_quantise(x["x"].to(torch.float32)))
    if kind == "linear":
        return _plain_linear(x["codes"], x["scale"], x["wq"], x["w_scale"], _DT[case["out"]], x["bias"], x["residual"],
                             case["swiglu"])
    codes, scale, s = _plain_norm(x)
    if kind == "norm":
        return dict(sum=s, values=_values(codes, scale))
    act = _plain_linear(codes, scale, *x["up"], torch.bfloat16, swiglu=True)
    codes, scale = _quantise(act.to(torch.float32))
    return dict(sum=s, y=_plain_linear(codes, scale, *x["down"], torch.bfloat16))


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind, M = case["kind"], case["M"]
    if kind == "rows":
        # the rows in, codes and scales out and in again, the values out
        n = M * case["K"]
        return dict(bytes=n * (_SIZE[case["x"]] + 2 + 2) + 8 * M, flops=4 * n)
    if kind == "linear":
        N, K = case["N"], case["K"]
        cols = N // 2 if case["swiglu"] else N
        return dict(bytes=(M + N) * (K + 4) + M * cols * (_SIZE[case["out"]] + _SIZE.get(case["res"], 0))
                    + (4 * N if case["bias"] else 0), flops=2 * M * N * K)
    n, D = M * case["D"], case["D"]
    stream = n * (_SIZE[case["x"]] + (_SIZE[case["res"]] + _SIZE[case["x"]] if case["res"] else 0)) + 4 * D
    if kind == "norm":
        return dict(bytes=stream + n * (2 + 2) + 8 * M, flops=8 * n)
    H = case["H"]
    return dict(bytes=stream + 3 * D * H + 4 * (2 * H + D) + 2 * n, flops=6 * M * D * H + 8 * n)


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------
def _exact_rows(t):
    """What rows of 64-bit values stand for as codes and a scale: steps of max / 127."""
    step = t.abs().amax(-1, keepdim=True) / 127.0
    return torch.round(t / step) * step


def _exact_weight(wq, ws):
    return wq.to(torch.float64) * ws.to(torch.float64)[:, None]


def _exact_swiglu(y):
    h = y.shape[-1] // 2
    return y[:, :h] * torch.sigmoid(y[:, :h]) * y[:, h:]


def exact(case, seed):
    x = _prepare(case, seed)
    f = torch.float64
    kind = case["kind"]
    if kind == "rows":
        return _exact_rows(x["x"].to(f))
    if kind == "linear":
        y = _exact_weight(x["codes"], x["scale"]) @ _exact_weight(x["wq"], x["w_scale"]).t()
        if x["bias"] is not None:
            y += x["bias"].to(f)
        if case["swiglu"]:
            y = _exact_swiglu(y)
        if x["residual"] is not None:
            y += x["residual"].to(f)
        return y
    total = x["x"].to(f)
    if x["residual"] is not None:
        total = total + x["residual"].to(f)
    s = total.to(_DT[case["x"]]).to(f)                            # the stream holds the sum in its own type
    v = _exact_rows(s * x["weight"].to(f)) * torch.rsqrt(s.square().mean(-1, keepdim=True) + EPS)
    if kind == "norm":
        return dict(sum=total, values=v)
    act = _exact_swiglu(v @ _exact_weight(*x["up"]).t()).to(torch.bfloat16).to(f)
    return dict(sum=total, y=_exact_rows(act) @ _exact_weight(*x["down"]).t())
