"""Plain 64-bit forms of the 8-bit KV cache's operators (numpy-free torch on the CPU) and their inputs."""
import math

import torch

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
F64 = torch.float64


def gen(seed):
    return torch.Generator().manual_seed(seed)


def quantise(x, dtype):
    """(codes, scales) of fp32 rows by the format's definition, in fp32."""
    amax = x.abs().amax(-1)
    top = torch.full_like(amax, TOP[dtype])
    ok = amax >= 2.0 ** -100
    safe = torch.where(ok, amax, torch.ones_like(amax))
    y = torch.where(ok[..., None], x * (top / safe)[..., None], torch.zeros_like(x))
    bad = ~torch.isfinite(amax)
    y = torch.where(bad[..., None], torch.zeros_like(y), y)
    codes = torch.round(y).clamp(-127, 127).to(torch.int8) if dtype == torch.int8 \
        else y.clamp(-448, 448).to(torch.float8_e4m3fn)
    scale = torch.where(ok, safe / top, torch.zeros_like(amax))
    return codes, torch.where(bad, torch.full_like(scale, math.nan), scale)


def values(codes, scale):
    return codes.to(torch.float32).to(F64) * scale.to(F64)[..., None]


def cache(g, B, Hkv, cap, d, dtype):
    """Random codes and scales of a full cache."""
    x = torch.randn(B, Hkv, cap, d, generator=g) * torch.exp(0.4 * torch.randn(d, generator=g))
    return quantise(x, dtype)


def rotate(x, cos, sin):
    """x * cos + rotate_half(x) * sin; cos, sin broadcast over x."""
    h = x.shape[-1] // 2
    return torch.cat([x[..., :h] * cos[..., :h] - x[..., h:] * sin[..., :h],
                      x[..., h:] * cos[..., h:] + x[..., :h] * sin[..., h:]], -1)


def attention(q, k, v, lens, Tp, words=None, window=0, scale=None, seg2=None, gates=None):
    """(out, mag) (B, H, N, d) in 64 bits; k, v (B, Hkv, cap, d) values; mag = sum over the terms of |gate| sum_j p_j
    |v_j|.  words (N,) or (B, N) Python integers, None: a chain."""
    q = q.to(F64)
    B, H, N, d = q.shape
    rep = H // k.shape[1]
    c = scale if scale is not None else 1.0 / math.sqrt(d)
    g0, g1 = (1.0, 0.0) if gates is None else (float(gates[0]), float(gates[1]))
    out, mag = torch.zeros_like(q), torch.zeros_like(q)
    for b in range(B):
        t = min(max(int(lens[b]), 0), Tp)
        for i in range(N):
            if words is None:
                sees, pos = list(range(t + i + 1)), t + i
                at = sees
            else:
                w = int(words[b][i]) if isinstance(words[0], (list, tuple)) else int(words[i])
                row = words[b] if isinstance(words[0], (list, tuple)) else words
                nodes = [j for j in range(N) if (w >> j) & 1]
                sees = list(range(t)) + [t + j for j in nodes]
                pos = t + bin(w).count("1") - 1
                at = list(range(t)) + [t + bin(int(row[j])).count("1") - 1 for j in nodes]
            if window:
                sees = [s for s, a in zip(sees, at) if pos - a < window]
            for h in range(H):
                if sees:
                    kk, vv = k[b, h // rep, sees], v[b, h // rep, sees]
                    p = torch.softmax(kk @ q[b, h, i] * c, 0)
                    out[b, h, i] += g0 * (p @ vv)
                    mag[b, h, i] += abs(g0) * (p @ vv.abs())
                if seg2 is not None:
                    z = 0 if seg2[0].shape[0] == 1 else b
                    kk, vv = (x[z, h // rep].to(F64) for x in seg2)
                    p = torch.softmax(kk @ q[b, h, i] * c, 0)
                    out[b, h, i] += g1 * (p @ vv)
                    mag[b, h, i] += abs(g1) * (p @ vv.abs())
    return out, mag
