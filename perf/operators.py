"""Timed cases of the 8-bit KV cache: writing it, reading it back, attending over it.

Each case is a dict of plain values; its "kind" names the operator:

  write   HipBackend.kv_write, then HipBackend.kv_read of the rows it wrote: the q | k | v rows of a projection, their
          per-head norms (optional) and position rotation, the new rows quantised into the cache, and the values that
          the cache then stands for
  read    HipBackend.kv_read of a whole cache
  attn    HipBackend.tree_attention_q8: the new rows of every sequence (one token, a chain of drafts, a token tree, a
          prompt) over their cached rows, with a sliding window and gated global rows where the case has them

A row of a cache (one token of one KV head, d values x) is held as d codes and one 32-bit scale:
  int8   scale = max|x| / 127, code = round(x * (127 / max|x|))
  e4m3   scale = max|x| / 448, code = x * (448 / max|x|) rounded to e4m3
  bf16   the values rounded, no scale
and stands for code * scale.  Rounding is to nearest, ties to even.

`own` false computes the plain form with elementary torch operations in 32 bits, rounded once at the end; true makes the
framework's calls.  Heads of 64 with 16 over 8 KV heads, the window of 1,024 and 128 global rows are CometSparkV05's.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DEV = torch.device("cuda:0")
_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_TOP = {"int8": 127.0, "e4m3": 448.0}
EPS = 1e-6
THETA = 10000.0


def listed():
    return [
        # one user's chat: the new token of a plain decode step
        dict(name="write_b1_n1_int8", kind="write", B=1, n=1, H=16, Hkv=8, d=64, T=2000, src="bf16", cache="int8",
             norm=False),
        # a decode step of a full batch, rows from a quantized projection (32 bits), an odd length
        dict(name="write_b32_n1_e4m3_f32", kind="write", B=32, n=1, H=16, Hkv=8, d=64, T=1203, src="f32", cache="e4m3",
             norm=False),
        # four prompts into a 16-bit cache, queries and keys normed per head
        dict(name="write_b4_n512_bf16_norm", kind="write", B=4, n=512, H=16, Hkv=8, d=64, T=0, src="bf16",
             cache="bf16", norm=True),
        # a batch of long prompts, heads of 128
        dict(name="write_b16_n1024_int8_norm", kind="write", B=16, n=1024, H=32, Hkv=8, d=128, T=0, src="bf16",
             cache="int8", norm=True),
        # one user's cache handed on
        dict(name="read_b1_t2000_int8", kind="read", B=1, Hkv=8, d=64, T=2000, cache="int8"),
        # a batch's long caches
        dict(name="read_b16_t8192_e4m3", kind="read", B=16, Hkv=8, d=128, T=8192, cache="e4m3"),
        # one user, one token, a few thousand cached rows
        dict(name="attn_b1_n1_t4000_int8", kind="attn", B=1, n=1, H=16, Hkv=8, d=64, T=4000, cache="int8", tree="",
             window=0, G=0, out="f16"),
        # one verify round of 32 sequences, six drafts each, with the window and the global rows
        dict(name="attn_b32_n7_t617_int8", kind="attn", B=32, n=7, H=16, Hkv=8, d=64, T=617, cache="int8", tree="",
             window=1024, G=128, out="bf16"),
        # a (4, 3, 2) token tree over 2,048 cached rows
        dict(name="attn_b16_n40_t2048_e4m3", kind="attn", B=16, n=40, H=16, Hkv=8, d=64, T=2048, cache="e4m3",
             tree="4,3,2", window=0, G=0, out="bf16"),
        # a verify round over long contexts, heads of 128
        dict(name="attn_b8_n5_t16000_int8", kind="attn", B=8, n=5, H=32, Hkv=8, d=128, T=16000, cache="int8", tree="",
             window=0, G=0, out="bf16"),
        # the prompts of four sequences, with the window and the global rows
        dict(name="attn_b4_n512_t0_int8", kind="attn", B=4, n=512, H=16, Hkv=8, d=64, T=0, cache="int8", tree="",
             window=1024, G=128, out="bf16"),
        # the last piece of one long prompt
        dict(name="attn_b1_n2048_t8192_e4m3", kind="attn", B=1, n=2048, H=16, Hkv=8, d=64, T=8192, cache="e4m3",
             tree="", window=0, G=0, out="bf16"),
    ]


# ---------------------------------------------------------------------------
# Drawn cases
# ---------------------------------------------------------------------------
def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    return dict(zip(("H", "Hkv", "d"), rng.choice([(16, 8, 64), (16, 4, 64), (8, 8, 128), (32, 8, 128), (12, 4, 64)])))


def _parents(tree):
    """Parent indices of a token tree with these branching factors, breadth first."""
    parent, level = [], [-1]
    for b in (int(x) for x in tree.split(",")):
        nodes = []
        for p in level:
            for _ in range(b):
                nodes.append(len(parent))
                parent.append(p)
        level = nodes
    return parent


def draw(rng):
    kind = rng.choice(["write", "write", "read", "attn", "attn", "attn", "attn"])
    cache = rng.choice(["int8", "e4m3"])
    h = _heads(rng)
    if kind == "write":
        step = rng.choice(["decode", "verify", "prompt"])
        n = 1 if step == "decode" else rng.randint(2, 40) if step == "verify" else _log_int(rng, 41, 1500)
        return dict(kind=kind, B=_log_int(rng, 1, min(64, max(1, 8192 // n))), n=n, T=_log_int(rng, 1, 4000),
                    src=rng.choice(["bf16", "bf16", "f32", "f16"]), cache=rng.choice([cache, cache, "bf16"]),
                    norm=rng.random() < 0.4, **h)
    if kind == "read":
        T = _log_int(rng, 16, 16000)
        del h["H"]
        return dict(kind=kind, B=_log_int(rng, 1, max(1, min(32, 100000 // T))), T=T, cache=cache, **h)
    step = rng.choice(["token", "verify", "tree", "prompt"])
    out = rng.choice(["bf16", "bf16", "f16"])
    window, G = rng.choice([(0, 0), (0, 0), (1024, 128), (1024, 0), (0, 37)])
    tree = ""
    if step == "prompt":
        n = _log_int(rng, 65, 1500)
        T = rng.choice([0, _log_int(rng, 1, 6000)])
        B = _log_int(rng, 1, max(1, min(8, 4_000_000 // (n * (T + n)))))
    else:
        n = 1 if step == "token" else rng.randint(2, 9)
        if step == "tree":
            tree = rng.choice(["2", "4,3,2", "2,2,2", "4,1,1", "3,3", "1,4,2,1", "8", "2,2,2,2,2"])
            n = len(_parents(tree))
        T = _log_int(rng, 1, 16000)
        B = _log_int(rng, 1, max(1, min(64, 120000 // T)))
    return dict(kind=kind, B=B, n=n, T=T, cache=cache, tree=tree, window=window, G=G, out=out, **h)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _gen(seed, salt=0):
    g = torch.Generator(device=_DEV)
    g.manual_seed(int(seed) * 1000003 + salt)
    return g


def _lens(case):
    """Committed lengths: T for the first sequence, down to about 3 T / 4 for the others."""
    T = case["T"]
    return [T - (b * 37) % (T // 4 + 1) for b in range(case["B"])]


def _tables(rows, d):
    """(rows, d) cosine and sine of position * THETA^(-2 i / d), each half the same angles."""
    i = np.arange(d // 2, dtype=np.float64)
    ang = np.outer(np.arange(rows, dtype=np.float64), THETA ** (-2.0 * i / d))
    ang = np.concatenate([ang, ang], axis=1)
    return (torch.from_numpy(np.cos(ang).astype(np.float32)).to(_DEV),
            torch.from_numpy(np.sin(ang).astype(np.float32)).to(_DEV))


def _rows(g, *shape):
    """Rows as projections give them: channels of different strength."""
    return torch.randn(shape, generator=g, device=_DEV) * torch.exp(
        0.4 * torch.randn(shape[-1], generator=g, device=_DEV))


def _quantise(x, cache):
    """(codes, scales) of 32-bit rows (..., d); a bf16 cache has no scales."""
    if cache == "bf16":
        return x.to(torch.bfloat16), None
    top = _TOP[cache]
    amax = x.abs().amax(-1)
    safe = torch.where(amax > 0, amax, torch.ones_like(amax))
    y = x * torch.div(torch.full_like(safe, top), safe).unsqueeze(-1)
    codes = torch.round(y).clamp(-127, 127).to(torch.int8) if cache == "int8" \
        else y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return codes, torch.where(amax > 0, torch.div(safe, torch.full_like(safe, top)), torch.zeros_like(amax))


def _full_cache(case, g, rows):
    """(codes, scales) of a cache that holds `rows` rows of every sequence."""
    return _quantise(_rows(g, case["B"], case["Hkv"], rows, case["d"]), case["cache"])


def _prepare(case, seed):
    g = _gen(seed)
    B, Hkv, d = case["B"], case["Hkv"], case["d"]
    if case["kind"] == "read":
        kc, ks = _full_cache(case, g, case["T"])
        vc, vs = _full_cache(case, g, case["T"])
        return dict(k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs)
    H, n, T = case["H"], case["n"], case["T"]
    lens = torch.tensor(_lens(case), dtype=torch.int32, device=_DEV)
    if case["kind"] == "write":
        cap = T + n
        x = _rows(g, B, n, H + 2 * Hkv, d).reshape(B, n, -1).to(_DT[case["src"]])
        dt = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn, "bf16": torch.bfloat16}[case["cache"]]
        kc, vc = (torch.zeros((B, Hkv, cap, d), device=_DEV).to(dt) for _ in range(2))
        ks = vs = None
        if case["cache"] != "bf16":
            ks, vs = (torch.zeros((B, Hkv, cap), device=_DEV) for _ in range(2))
        cos, sin = _tables(cap, d)
        qn = kn = None
        if case["norm"]:
            qn, kn = (1.0 + 0.1 * torch.randn(d, generator=g, device=_DEV) for _ in range(2))
        return dict(qkv=x, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, lens=lens, cos=cos, sin=sin, q_norm=qn,
                    k_norm=kn)
    cap = T + n
    kc, ks = _full_cache(case, g, cap)
    vc, vs = _full_cache(case, g, cap)
    q = _rows(g, B, H, n, d).to(torch.bfloat16)
    parent = _parents(case["tree"]) if case["tree"] else None
    words = None
    if parent is not None:
        words = np.zeros(n, dtype=np.uint64)
        for i, p in enumerate(parent):
            words[i] = np.uint64(1 << i) | (words[p] if p >= 0 else np.uint64(0))
    seg2 = gates = None
    if case["G"]:
        seg2 = tuple(_rows(g, 1, Hkv, case["G"], d).to(torch.bfloat16) for _ in range(2))
        gates = torch.sigmoid(0.5 * torch.randn(2, generator=g, device=_DEV))
    return dict(q=q, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, lens=lens, anc=words, seg2=seg2, gates=gates)


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
    if case["kind"] == "read":
        return hip.kv_read(**x)
    if case["kind"] == "write":
        q = hip.kv_write(**x, eps=EPS)
        k, v = hip.kv_read(x["k_cache"], x["v_cache"], x["k_scale"], x["v_scale"], start=x["lens"], rows=case["n"])
        return dict(q=q, k=k, v=v)
    return hip.tree_attention_q8(**x, window=case["window"], max_len=case["T"], out_dtype=_DT[case["out"]])


# ---------------------------------------------------------------------------
# The plain form
# ---------------------------------------------------------------------------
def _values(codes, scale):
    x = codes.to(torch.float32)
    return x if scale is None else x * scale.unsqueeze(-1)


def _put(cache, b, pos, rows):
    """cache[b, :, pos[b, i]] = rows[b, i] (one-byte types by their bytes)."""
    if cache.element_size() == 1:
        cache, rows = cache.view(torch.uint8), rows.view(torch.uint8)
    cache[b, :, pos] = rows


def _take(cache, b, pos):
    if cache.element_size() == 1:
        return cache.view(torch.uint8)[b, :, pos].view(cache.dtype)
    return cache[b, :, pos]


def _plain_write(case, x):
    B, n, H, Hkv, d = (case[k] for k in ("B", "n", "H", "Hkv", "d"))
    q, k, v = x["qkv"].to(torch.float32).view(B, n, H + 2 * Hkv, d).split([H, Hkv, Hkv], dim=2)
    if case["norm"]:
        q = q / torch.sqrt((q * q).mean(-1, keepdim=True) + EPS) * x["q_norm"]
        k = k / torch.sqrt((k * k).mean(-1, keepdim=True) + EPS) * x["k_norm"]
    pos = x["lens"].long().view(B, 1) + torch.arange(n, device=_DEV)
    cos, sin = x["cos"][pos].unsqueeze(2), x["sin"][pos].unsqueeze(2)
    q, k = (t * cos + torch.cat([-t[..., d // 2:], t[..., :d // 2]], -1) * sin for t in (q, k))
    b = torch.arange(B, device=_DEV).view(B, 1)
    got = []
    for rows, cache, scale in ((k, x["k_cache"], x["k_scale"]), (v, x["v_cache"], x["v_scale"])):
        codes, s = _quantise(rows, case["cache"])
        _put(cache, b, pos, codes)
        if scale is not None:
            scale[b, :, pos] = s
        read = _values(_take(cache, b, pos), scale[b, :, pos] if scale is not None else None)
        got.append(read.transpose(1, 2).to(torch.bfloat16).contiguous())
    return dict(q=q.transpose(1, 2).to(torch.bfloat16).contiguous(), k=got[0], v=got[1])


def _seen(case, x, T):
    """(B, n, T) bool: which cached rows each new row sees."""
    B, n = case["B"], case["n"]
    lens = x["lens"].long().view(B, 1, 1)
    j = torch.arange(T, device=_DEV).view(1, 1, T)
    i = torch.arange(n, device=_DEV).view(1, n, 1)
    if x["anc"] is None:
        pos, sees = lens + i, j <= lens + i
    else:
        bits = torch.tensor([[(int(w) >> t) & 1 for t in range(n)] for w in x["anc"]], device=_DEV)   # (n, n)
        pos = lens + (bits.sum(1) - 1).view(1, n, 1)
        node = (j - lens).clamp(0, n - 1)                                                            # (B, 1, T)
        sees = (j < lens) | ((j < lens + n) & (bits[i.expand(B, n, T), node.expand(B, n, T)] > 0))
    if case["window"]:
        depth = torch.arange(n, device=_DEV) if x["anc"] is None else bits.sum(1) - 1
        at = torch.where(j < lens, j, lens + depth[(j - lens).clamp(0, n - 1)])
        sees = sees & (pos - at < case["window"])
    return sees


def _attend(q, k, v, sees, scale):
    """softmax over the seen keys, zeros where there is none: q (B, Hkv, rep, n, d), k and v (B or 1, Hkv, T, d)."""
    B, Hkv, rep, n, d = q.shape
    T = k.shape[2]
    k, v = (t.expand(B, Hkv, T, d).contiguous() for t in (k, v))
    s = torch.matmul(q.reshape(B, Hkv, rep * n, d), k.transpose(-1, -2).contiguous()).view(B, Hkv, rep, n, T) * scale
    if sees is not None:
        s = s.masked_fill(~sees.view(B, 1, 1, n, T), -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isfinite(m), m, torch.zeros_like(m)))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Hkv, rep * n, T), v).view(B, Hkv, rep, n, d)
    return torch.where(total > 0, o / total, torch.zeros_like(o))


def _plain_attn(case, x):
    B, n, H, Hkv, d = (case[k] for k in ("B", "n", "H", "Hkv", "d"))
    T = case["T"] + n
    q = x["q"].to(torch.float32).view(B, Hkv, H // Hkv, n, d)
    k, v = _values(x["k_cache"], x["k_scale"]), _values(x["v_cache"], x["v_scale"])
    scale = 1.0 / math.sqrt(d)
    o = _attend(q, k, v, _seen(case, x, T), scale)
    if case["G"]:
        g = _attend(q, x["seg2"][0].to(torch.float32), x["seg2"][1].to(torch.float32), None, scale)
        o = x["gates"][0] * o + x["gates"][1] * g
    return o.view(B, H, n, d).to(_DT[case["out"]])


def run(state):
    case, x = state["case"], state["x"]
    if own:
        return _run_own(case, x)
    if case["kind"] == "read":
        return tuple(_values(x[a], x[b]).to(torch.bfloat16)
                     for a, b in (("k_cache", "k_scale"), ("v_cache", "v_scale")))
    return _plain_write(case, x) if case["kind"] == "write" else _plain_attn(case, x)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    B, Hkv, d = case["B"], case["Hkv"], case["d"]
    row = 2 * d if case["cache"] == "bf16" else d + 4            # a row's codes and its scale
    if case["kind"] == "read":
        n = 2 * B * Hkv * case["T"]
        return dict(bytes=n * (row + 2 * d), flops=n * d)
    H, n = case["H"], case["n"]
    if case["kind"] == "write":
        size = 4 if case["src"] == "f32" else 2
        tok = B * n
        at = len({p for t in set(_lens(case)) for p in range(t, t + n)})
        # q | k | v in, q out, the cache's rows out and in again, their values out, the table rows
        return dict(bytes=tok * ((H + 2 * Hkv) * d * size + H * d * 2 + 2 * Hkv * (2 * row + 2 * d)) + at * d * 8,
                    flops=tok * (H + 2 * Hkv) * d * (8 if case["norm"] else 5))
    depth = None
    if case["tree"]:
        parent = _parents(case["tree"])
        depth = [0] * n
        for i, p in enumerate(parent):
            depth[i] = depth[p] + 1 if p >= 0 else 0
    W = case["window"] or 1 << 40
    pairs, rows = 0, 0
    for t in _lens(case):
        # keys a new row sees: itself, its ancestors or the rows before it, within the window
        at = depth if depth is not None else range(n)
        pairs += sum(min(t + a + 1, W) for a in at)
        rows += min(t + n, W - 1 + n)
    return dict(bytes=rows * 2 * Hkv * row + 2 * B * H * n * d * 2 + 2 * Hkv * case["G"] * d * 2,
                flops=4 * H * d * (pairs + B * n * case["G"]))


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------
def _exact_codes(x, cache):
    """What a row of 64-bit values stands for once it has been through the cache."""
    if cache == "bf16":
        return x
    top = _TOP[cache]
    s = x.abs().amax(-1, keepdim=True) / top
    y = torch.where(s > 0, x / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(x))
    if cache == "int8":
        return torch.round(y) * s
    # e4m3: steps of 2^(e - 3) from 2^e on, 2^-9 below 2^-6
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3.0)
    return torch.round(y / step) * step * s


def exact(case, seed):
    x = _prepare(case, seed)
    f = torch.float64
    if case["kind"] == "read":
        return tuple(x[a].to(torch.float32).to(f) * x[b].to(f)[..., None]
                     for a, b in (("k_cache", "k_scale"), ("v_cache", "v_scale")))
    B, n, H, Hkv, d = (case[k] for k in ("B", "n", "H", "Hkv", "d"))
    if case["kind"] == "write":
        t = x["qkv"].to(f).reshape(B, n, H + 2 * Hkv, d).permute(0, 2, 1, 3)
        q, k, v = t[:, :H], t[:, H:H + Hkv], t[:, H + Hkv:]
        if case["norm"]:
            q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * x["q_norm"].to(f)
            k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * x["k_norm"].to(f)
        at = torch.stack([torch.arange(s, s + n, device=_DEV) for s in _lens(case)])
        c, s = (x[w].to(f)[at][:, None] for w in ("cos", "sin"))
        h = d // 2
        lo, hi = slice(0, h), slice(h, d)

        def turn(y):
            return torch.cat([y[..., lo] * c[..., lo] - y[..., hi] * s[..., lo],
                              y[..., hi] * c[..., hi] + y[..., lo] * s[..., hi]], -1)

        return dict(q=turn(q), k=_exact_codes(turn(k), case["cache"]), v=_exact_codes(v, case["cache"]))
    out = torch.zeros((B, H, n, d), dtype=f, device=_DEV)
    up = None
    if case["tree"]:
        up = []
        for i, p in enumerate(_parents(case["tree"])):
            up.append((up[p] if p >= 0 else []) + [i])
    for b, t in enumerate(_lens(case)):
        ok = torch.ones((n, t + n), dtype=torch.bool, device=_DEV)
        place = torch.arange(t + n, device=_DEV)
        if up is None:
            ok = torch.tril(ok, diagonal=t)
            here = place[t:]
        else:
            ok[:, t:] = torch.tensor([[c in u for c in range(n)] for u in up], device=_DEV)
            here = torch.tensor([t + len(u) - 1 for u in up], device=_DEV)
            place = torch.cat([place[:t], here])
        if case["window"]:
            ok &= here[:, None] - place[None] < case["window"]
        for h in range(H):
            g = h // (H // Hkv)
            q = x["q"][b, h].to(f)
            k, v = (x[a][b, g, :t + n].to(torch.float32).to(f) * x[s][b, g, :t + n].to(f)[:, None]
                    for a, s in (("k_cache", "k_scale"), ("v_cache", "v_scale")))
            w = torch.softmax((q @ k.t().contiguous() / math.sqrt(d)).masked_fill(~ok, -math.inf), -1)
            y = w @ v
            if case["G"]:
                k2, v2 = (z[0, g].to(f) for z in x["seg2"])
                y = x["gates"][0].to(f) * y + x["gates"][1].to(f) * (
                    torch.softmax(q @ k2.t().contiguous() / math.sqrt(d), -1) @ v2)
            out[b, h] = y
    return out
