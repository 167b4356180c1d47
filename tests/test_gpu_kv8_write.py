"""kv_write and kv_read (vnx_kv_write, vnx_kv_read) against plain forms.

Codes, scales and bf16 rows without norms are compared bit for bit with the definition in 32 bits (the kernel rounds
every product and sum of the rotation as the formula is written).  With norms the row's 1 / sqrt(mean) may differ in its
last bits, so the values are held to the 64-bit form: half a code step (int8: scale / 2; e4m3: 2^-4 of the value or half
the smallest step, 2^-10 scale), plus 2^-20 of the rotated pair's magnitude for the fp32 arithmetic before it (fewer than
16 roundings of 2^-24), plus 2^-22 of the value for the scale's own division and product."""
import math

import pytest
import torch

import kv8_ref as R

pytestmark = pytest.mark.gpu

I8, E4 = torch.int8, torch.float8_e4m3fn


def _inputs(g, B, n, H, Hkv, d, src, rows):
    x = (torch.randn(B, n, H + 2 * Hkv, d, generator=g) * 3.0 ** torch.randn(B, n, H + 2 * Hkv, 1, generator=g))
    x = x.reshape(B, n, -1).to(src)
    ang = torch.rand(rows, d // 2, generator=g) * 6.28
    return x, torch.cat([torch.cos(ang)] * 2, 1), torch.cat([torch.sin(ang)] * 2, 1)


def _split(x, H, Hkv):
    B, n, w = x.shape
    t = x.view(B, n, H + 2 * Hkv, -1).transpose(1, 2)
    return t[:, :H], t[:, H:H + Hkv], t[:, H + Hkv:]


def _empty(B, Hkv, cap, d, dtype, dev):
    """A cache whose bytes are all 0x55 and its scales -7: what is not written stays so."""
    kc, vc = (torch.full((B, Hkv, cap, d * (2 if dtype == torch.bfloat16 else 1)), 0x55, dtype=torch.uint8,
                         device=dev).view(dtype) for _ in range(2))
    ks, vs = (torch.full((B, Hkv, cap), -7.0, device=dev) for _ in range(2))
    return kc, vc, ks, vs


CASES = [
    dict(B=1, n=1, H=16, Hkv=8, d=64, src=torch.bfloat16, cap=9, lens=[8]),
    dict(B=3, n=5, H=4, Hkv=2, d=128, src=torch.float32, cap=31, lens=[0, 7, 26]),
    dict(B=2, n=3, H=3, Hkv=1, d=16, src=torch.float16, cap=7, lens=[4, 1]),
    dict(B=2, n=7, H=5, Hkv=5, d=32, src=torch.bfloat16, cap=40, lens=[33, 0]),
    dict(B=1, n=130, H=2, Hkv=1, d=256, src=torch.bfloat16, cap=133, lens=[3]),
    dict(B=33, n=1, H=12, Hkv=4, d=64, src=torch.float32, cap=5, lens=[i % 5 for i in range(33)]),
    # positions before the cache, past it, and across its end
    dict(B=4, n=4, H=2, Hkv=2, d=64, src=torch.bfloat16, cap=10, lens=[-2, 8, 10, 2 ** 31 - 1]),
]


@pytest.mark.parametrize("dtype", [I8, E4, torch.bfloat16], ids=["int8", "e4m3", "bf16"])
@pytest.mark.parametrize("rope", [True, False], ids=["rope", "plain"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_write_bits(hip, case, rope, dtype):
    c = CASES[case]
    B, n, H, Hkv, d, cap = (c[k] for k in ("B", "n", "H", "Hkv", "d", "cap"))
    print(c, rope, dtype, flush=True)
    dev = hip.torch_device
    x, cos, sin = _inputs(R.gen(case), B, n, H, Hkv, d, c["src"], cap)
    kc, vc, ks, vs = _empty(B, Hkv, cap, d, dtype, dev)
    lens = torch.tensor(c["lens"], dtype=torch.int32)
    kw = dict(cos=cos, sin=sin) if rope else {}
    if dtype != torch.bfloat16:
        kw.update(k_scale=ks, v_scale=vs)
    want = [t.cpu().clone() for t in (kc.view(torch.uint8), vc.view(torch.uint8), ks, vs)]
    q = hip.kv_write(x, kc, vc, lens, **kw).cpu()
    qf, kf, vf = _split(x.float(), H, Hkv)
    for b in range(B):
        for i in range(n):
            pos = c["lens"][b] + i
            if not 0 <= pos < cap:
                assert (q[b, :, i] == 0).all()
                continue
            turn = (lambda t: R.rotate(t, cos[pos], sin[pos])) if rope else (lambda t: t)
            assert torch.equal(q[b, :, i], turn(qf[b, :, i]).to(torch.bfloat16))
            for at, rows in ((0, turn(kf[b, :, i])), (1, vf[b, :, i])):
                if dtype == torch.bfloat16:
                    want[at][b, :, pos] = rows.to(torch.bfloat16).contiguous().view(torch.uint8)
                else:
                    codes, s = R.quantise(rows, dtype)
                    want[at][b, :, pos] = codes.view(torch.uint8)
                    want[2 + at][b, :, pos] = s
    for got, w in zip((kc.view(torch.uint8), vc.view(torch.uint8), ks, vs), want):
        assert torch.equal(got.cpu(), w)


@pytest.mark.parametrize("dtype", [I8, E4, torch.bfloat16], ids=["int8", "e4m3", "bf16"])
@pytest.mark.parametrize("which", ["both", "q", "k"])
@pytest.mark.parametrize("d,src", [(64, torch.bfloat16), (128, torch.float32), (16, torch.float16)])
def test_write_norms(hip, d, src, which, dtype):
    B, n, H, Hkv, cap, eps = 2, 9, 6, 3, 20, 1e-5
    dev = hip.torch_device
    g = R.gen(d)
    x, cos, sin = _inputs(g, B, n, H, Hkv, d, src, cap)
    qn, kn = (1.0 + 0.3 * torch.randn(d, generator=g) for _ in range(2))
    qn, kn = qn if which != "k" else None, kn if which != "q" else None
    kc, vc, ks, vs = _empty(B, Hkv, cap, d, dtype, dev)
    lens = torch.tensor([11, 2], dtype=torch.int32)
    kw = {} if dtype == torch.bfloat16 else dict(k_scale=ks, v_scale=vs)
    q = hip.kv_write(x, kc, vc, lens, cos=cos, sin=sin, q_norm=qn, k_norm=kn, eps=eps, **kw).cpu().to(R.F64)
    qf, kf, vf = _split(x.to(R.F64), H, Hkv)

    def norm(t, w):
        return t if w is None else t / torch.sqrt(t.square().mean(-1, keepdim=True) + eps) * w.to(R.F64)

    at = torch.stack([torch.arange(int(s), int(s) + n) for s in lens])
    c, s = cos.to(R.F64)[at][:, None], sin.to(R.F64)[at][:, None]
    for got, t in ((q, norm(qf, qn)), (None, norm(kf, kn)), (None, vf)):
        is_v = t is vf
        h = d // 2
        pair = torch.cat([t[..., :h].abs() + t[..., h:].abs()] * 2, -1)      # the rotated pair's magnitude
        ref = t if is_v else R.rotate(t, c, s)
        fp = 2.0 ** -20 * pair
        if got is not None:
            assert ((got - ref).abs() <= 2.0 ** -8 * ref.abs() + fp).all()
            continue
        cache, scale = (vc, vs) if is_v else (kc, ks)
        rows = torch.stack([cache[b].cpu()[:, at[b]] for b in range(B)])
        if dtype == torch.bfloat16:
            val, half = rows.to(R.F64), 2.0 ** -8 * ref.abs()
        else:
            sc = torch.stack([scale[b].cpu()[:, at[b]] for b in range(B)]).to(R.F64)[..., None]
            val = rows.float().to(R.F64) * sc
            half = sc / 2 if dtype == I8 else torch.maximum(2.0 ** -4 * ref.abs(), 2.0 ** -10 * sc)
            half = half + 2.0 ** -22 * ref.abs()
        assert ((val - ref).abs() <= half + fp).all()


def test_write_odd_rows(hip):
    """Rows of zeros, of subnormal and of huge values, with an infinity and with a NaN."""
    dev = hip.torch_device
    d, Hkv = 64, 6
    g = R.gen(3)
    rows = torch.randn(Hkv, d, generator=g)
    rows[0] = 0.0
    rows[1] *= 1e-40
    rows[2] *= 1e37
    rows[3, 5] = math.inf
    rows[4, 63] = math.nan
    x = torch.cat([torch.zeros(1, d), rows, rows]).reshape(1, 1, -1)
    for dtype in (I8, E4):
        kc, vc, ks, vs = _empty(1, Hkv, 2, d, dtype, dev)
        hip.kv_write(x, kc, vc, [1], k_scale=ks, v_scale=vs)
        codes, s = R.quantise(rows, dtype)
        for cache, scale in ((kc, ks), (vc, vs)):
            assert torch.equal(cache[0, :, 1].view(torch.uint8).cpu(), codes.view(torch.uint8))
            assert torch.equal(scale[0, :, 1].cpu().nan_to_num(nan=-1.0), s.nan_to_num(nan=-1.0))
        k, v = hip.kv_read(kc, vc, ks, vs, start=[1], rows=1, out_dtype=torch.float32)
        want = R.values(codes, s).float()
        for t in (k, v):
            assert torch.equal(t[0, :, 0].cpu().nan_to_num(nan=-1.0), want.nan_to_num(nan=-1.0))
        assert k[0, 3].isnan().all() and k[0, 4].isnan().all() and (k[0, 0] == 0).all()


def test_write_strided(hip):
    """Rows inside a wider buffer, batch rows apart, and a (B, cap, Hkv, d) cache seen as (B, Hkv, cap, d)."""
    dev = hip.torch_device
    B, n, H, Hkv, d, cap = 2, 3, 4, 2, 64, 8
    g = R.gen(8)
    w = (H + 2 * Hkv) * d
    big = torch.randn(B, n + 2, w + 64, generator=g).to(torch.bfloat16).to(dev)
    lens = torch.tensor([5, 0], dtype=torch.int32, device=dev)
    for x in (big[:, 1:n + 1, 32:32 + w], big[:, :n, 1:w + 1], big[:, 0:1, :w], big[:1, :n, :w].expand(B, n, w)):
        flat = x.clone(memory_format=torch.contiguous_format)
        got = []
        for lay in (0, 1):
            if lay:
                kc, vc = (torch.zeros(B, cap, Hkv, d, dtype=I8, device=dev).permute(0, 2, 1, 3) for _ in range(2))
                ks, vs = (torch.zeros(B, Hkv + 1, cap + 3, device=dev)[:, 1:, 2:cap + 2] for _ in range(2))
            else:
                kc, vc = (torch.zeros(B, Hkv, cap, d, dtype=I8, device=dev) for _ in range(2))
                ks, vs = (torch.zeros(B, Hkv, cap, device=dev) for _ in range(2))
            q = hip.kv_write(x if lay else flat, kc, vc, lens, k_scale=ks, v_scale=vs)
            k, v = hip.kv_read(kc, vc, ks, vs)
            got.append([t.cpu() for t in (q, kc, vc, ks, vs, k, v)])
        for a, b in zip(*got):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [I8, E4], ids=["int8", "e4m3"])
@pytest.mark.parametrize("d", [16, 32, 64, 128, 256])
def test_read(hip, d, dtype):
    """code * scale rounded once, every type, ranges that leave the cache, every code."""
    dev = hip.torch_device
    B, Hkv, cap = 2, 3, 37
    g = R.gen(d)
    kc, ks = R.cache(g, B, Hkv, cap, d, dtype)
    vc, vs = R.cache(g, B, Hkv, cap, d, dtype)
    every = torch.arange(256, dtype=torch.int64).to(torch.uint8)
    every = every[(every & 0x7F) != 0x7F] if dtype == E4 else every
    flat = kc.view(torch.uint8).view(-1)
    flat[:every.numel()] = every
    dv = [t.to(dev) for t in (kc, vc, ks, vs)]
    for out in (torch.float32, torch.bfloat16, torch.float16):
        for start, rows in ((None, None), ([3, 30], 11), ([-4, 36], 6), ([0, 37], 1), ([5, 5], 0)):
            k, v = hip.kv_read(*dv, start=start, rows=rows, out_dtype=out)
            r = cap if rows is None else rows
            st = [0, 0] if start is None else start
            for got, c, s in ((k, kc, ks), (v, vc, vs)):
                assert got.shape == (B, Hkv, r, d) and got.dtype == out
                want = torch.zeros(B, Hkv, r, d)
                for b in range(B):
                    for i in range(r):
                        if 0 <= st[b] + i < cap:
                            want[b, :, i] = c[b, :, st[b] + i].float() * s[b, :, st[b] + i, None]
                assert torch.equal(got.cpu(), want.to(out))


def test_read_of_a_bf16_cache(hip):
    """The values themselves, in every type."""
    kc, vc = (torch.randn(2, 3, 21, 32, generator=R.gen(s)).to(torch.bfloat16) for s in (1, 2))
    for out in (torch.float32, torch.bfloat16, torch.float16):
        k, v = hip.kv_read(kc.to(hip.torch_device), vc.to(hip.torch_device), start=[2, 15], rows=8, out_dtype=out)
        for got, c in ((k, kc), (v, vc)):
            assert torch.equal(got[0].cpu(), c[0, :, 2:10].to(out))
            assert torch.equal(got[1, :, :6].cpu(), c[1, :, 15:].to(out)) and (got[1, :, 6:] == 0).all()


def test_rows_past_4_gib(hip):
    """A cache whose rows lie a MiB apart: byte offsets past 32 bits, written, read and attended over."""
    dev = hip.torch_device
    cap, d, pitch = 4104, 64, 1 << 20
    g = R.gen(1)
    kc, vc = (torch.empty((cap - 1) * pitch + d, dtype=I8, device=dev).as_strided((1, 1, cap, d),
                                                                                 (cap * pitch, cap * pitch, pitch, 1))
              for _ in range(2))
    ks, vs = (torch.zeros(1, 1, cap, device=dev) for _ in range(2))
    x = torch.randn(1, cap, 3, d, generator=g).reshape(1, cap, -1)
    q = hip.kv_write(x, kc, vc, [0], k_scale=ks, v_scale=vs)
    _, kf, vf = _split(x, 1, 1)
    k, v = hip.kv_read(kc, vc, ks, vs, out_dtype=torch.float32)
    kd, vd = (R.quantise(t, I8) for t in (kf, vf))
    assert torch.equal(k.cpu(), R.values(*kd).float()) and torch.equal(v.cpu(), R.values(*vd).float())
    o = hip.tree_attention_q8(q[:, :, -3:], kc, vc, ks, vs, [cap - 3]).cpu()
    ref, mag = R.attention(q[:, :, -3:].cpu(), R.values(*kd), R.values(*vd), [cap - 3], cap - 3)
    assert ((o.to(R.F64) - ref).abs() <= 2.0 ** -8 * (1.02 * mag + ref.abs())).all()


def test_binding_and_general_path_agree(hip):
    """The calls that the binding serves and the same calls through the general path (lengths as a list, scales' strides
    alike): the same bits.  What the binding leaves: strides and types that need a copy."""
    dev = hip.torch_device
    B, n, H, Hkv, d, cap = 2, 3, 4, 2, 64, 16
    g = R.gen(21)
    x = torch.randn(B, n, (H + 2 * Hkv) * d, generator=g).to(torch.bfloat16).to(dev)
    ang = torch.rand(cap, d // 2, generator=g) * 6.28
    cos, sin = (torch.cat([f(ang)] * 2, 1).to(dev) for f in (torch.cos, torch.sin))
    lens = torch.tensor([4, 11], dtype=torch.int32, device=dev)
    b, st = hip._bind, hip._stream()
    got = []
    for ln in (lens, [4, 11]):
        kc, vc = (torch.zeros(B, Hkv, cap, d, dtype=E4, device=dev) for _ in range(2))
        ks, vs = (torch.zeros(B, Hkv, cap, device=dev) for _ in range(2))
        q = hip.kv_write(x, kc, vc, ln, k_scale=ks, v_scale=vs, cos=cos, sin=sin)
        k, v = hip.kv_read(kc, vc, ks, vs, start=ln, rows=n)
        o = hip.tree_attention_q8(q, kc, vc, ks, vs, ln)
        got.append((q, kc.view(torch.uint8), vc.view(torch.uint8), ks, vs, k, v, o))
    for a, c in zip(*got):
        assert torch.equal(a, c)
    assert b.kv_write(0, st, kc, vc, ks, vs, x, lens, cos, sin, None, None, 1e-6) is not None
    for xx in (x.double(), x[:, :, :-32], x.expand(B, n, -1)[:1], x.transpose(1, 2)):
        assert b.kv_write(0, st, kc, vc, ks, vs, xx, lens, cos, sin, None, None, 1e-6) is None
    assert b.kv_write(0, st, kc, vc, ks, vs, x, lens.long(), cos, sin, None, None, 1e-6) is None
    assert b.kv_write(0, st, kc, vc, ks, vs, x, lens, cos, None, None, None, 1e-6) is None
    assert b.kv_write(1, st, kc, vc, ks, vs, x, lens, cos, sin, None, None, 1e-6) is None
    assert b.tree_attn_q8(0, st, kc, vc, ks, vs, q.float(), lens, None, None, None, None, 0, None, torch.bfloat16,
                          None) is None
    assert b.tree_attn_q8(0, st, kc, vc, ks, vs, q, lens, None, None, None, None, 0, cap, torch.bfloat16, None) is None
    assert b.tree_attn_q8(0, st, kc, vc, ks, vs, q, lens, None, -1.0, None, None, 0, None, torch.bfloat16,
                          None) == -1


def test_refusals(hip):
    """What neither path can serve raises ValueError and writes nothing."""
    dev = hip.torch_device
    B, n, H, Hkv, d, cap = 2, 3, 4, 2, 64, 16
    kc, vc, ks, vs = _empty(B, Hkv, cap, d, I8, dev)
    x = torch.zeros(B, n, (H + 2 * Hkv) * d, device=dev)
    q = torch.zeros(B, H, n, d, dtype=torch.bfloat16, device=dev)
    lens = [1, 2]
    cos = torch.zeros(cap, d, device=dev)
    before = [t.clone() for t in (kc, ks)]
    bad = [
        lambda: hip.kv_write(x[:, :, :-1], kc, vc, lens, ks, vs), lambda: hip.kv_write(x[:1], kc, vc, lens, ks, vs),
        lambda: hip.kv_write(x.long(), kc, vc, lens, ks, vs), lambda: hip.kv_write(x, kc, vc, [1], ks, vs),
        lambda: hip.kv_write(x, kc, vc, lens), lambda: hip.kv_write(x, kc.cpu(), vc, lens, ks, vs),
        lambda: hip.kv_write(x, kc, vc[:, :, :8], lens, ks, vs), lambda: hip.kv_write(x, kc, vc, lens, ks, vs, cos=cos),
        lambda: hip.kv_write(x, kc, vc, lens, ks, vs, cos=cos[:, :32], sin=cos[:, :32]),
        lambda: hip.kv_write(x, kc, vc, lens, ks, vs, q_norm=cos[0, :32]),
        lambda: hip.kv_write(x, kc, vc, lens, ks.double(), vs.double()), lambda: hip.kv_write(x, kc.short(), vc.short(), lens),
        lambda: hip.kv_write(x[:, :, :4 * d], kc, vc, lens, ks, vs),
        lambda: hip.kv_read(kc, vc, ks, vs, rows=-1), lambda: hip.kv_read(kc, vc, ks[:, :, :4], vs[:, :, :4]),
        lambda: hip.kv_read(kc, vc, ks, vs, out_dtype=torch.float64), lambda: hip.kv_read(kc, vc),
        lambda: hip.kv_read(kc[..., 1:], vc[..., 1:], ks, vs),
        lambda: hip.tree_attention_q8(q, kc, vc, ks, vs, lens, max_len=cap), lambda: hip.tree_attention_q8(q, kc, vc, ks, vs, [1]),
        lambda: hip.tree_attention_q8(q[..., :32], kc, vc, ks, vs, lens), lambda: hip.tree_attention_q8(q[:, :3], kc, vc, ks, vs, lens),
        lambda: hip.tree_attention_q8(q, kc, vc, ks, vs, lens, window=-1), lambda: hip.tree_attention_q8(q, kc, vc, ks, vs, lens, scale=0.0),
        lambda: hip.tree_attention_q8(q, kc, vc, ks, vs, lens, anc=[1, 3]),
        lambda: hip.tree_attention_q8(q, kc, vc, ks, vs, lens, anc=[1, 3, 7], window=2),
        lambda: hip.tree_attention_q8(q, kc, vc, ks, vs, lens, out_dtype=torch.float32),
        lambda: hip.tree_attention_q8(q, kc, vc, ks, vs, lens, out=q.float()), lambda: hip.tree_attention_q8(q, kc, vc, ks, vs, lens, out=q[:1]),
        lambda: hip.tree_attention_q8(q, kc, vc, ks, vs, lens, seg2=(q[:, :2], q[:, :2])),
        lambda: hip.tree_attention_q8(q, kc, vc, ks, vs, lens, seg2=(q[:, :2, :0], q[:, :2, :0]), gates=[1, 1]),
        lambda: hip.tree_attention_q8(q, kc.bfloat16(), vc.bfloat16(), None, None, lens),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            print("accepted:", i)
    torch.cuda.synchronize(dev)
    for t, w in zip((kc, ks), before):
        assert torch.equal(t, w)
    # empty batches and ranges are no errors
    assert hip.kv_read(kc, vc, ks, vs, rows=0)[0].shape == (B, Hkv, 0, d)
    assert hip.kv_read(kc[:0], vc[:0], ks[:0], vs[:0])[0].shape == (0, Hkv, cap, d)
    assert hip.kv_write(x[:0], kc[:0], vc[:0], [], ks[:0], vs[:0]).shape == (0, H, n, d)
    assert hip.tree_attention_q8(q[:0], kc[:0], vc[:0], ks[:0], vs[:0], []).shape == (0, H, n, d)
