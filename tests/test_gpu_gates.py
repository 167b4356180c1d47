"""gates[0] scales the first term of every attention operator whether or not a second segment stands beside it
(TriSparseAttention mixes its paths with sigmoid gates, packages/verse_nex/verse_nex/tri_sparse_attn.py:585-608; a layer
without global rows keeps gates[0] * path A).

Bars: those of tests/test_gpu_kv8_attn.py, tests/test_gpu_tree.py and tests/test_gpu_chain.py; the gate is one more fp32
product."""
import ctypes

import numpy as np
import pytest
import torch

import kv8_ref as R
from oracle import tree as OT
from versenext_amd import _lib
from versenext_amd import model as VM
from versenext_amd import tree as VT

pytestmark = pytest.mark.gpu

I8, E4 = torch.int8, torch.float8_e4m3fn
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 0.0}
GATES = [0.15, -0.6, 2.0]


def _close(o, ref, mag, term=2.0 ** -10):
    err = (o.cpu().to(R.F64) - ref).abs()
    assert (err <= term * mag + HALF[o.dtype] * ref.abs() + 2.0 ** -25).all()


# a split walk, several waves a tile, a wave a tile; heads of 128; a tree, a tree over split keys
Q8 = [dict(B=1, H=4, Hkv=2, d=64, N=1, lens=[1500]), dict(B=2, H=4, Hkv=2, d=64, N=5, lens=[40, 0]),
      dict(B=1, H=2, Hkv=1, d=64, N=300, lens=[33]), dict(B=1, H=8, Hkv=2, d=128, N=3, lens=[900]),
      dict(B=2, H=4, Hkv=2, d=128, lens=[50, 3], tree=(3, 2)), dict(B=1, H=2, Hkv=1, d=64, lens=[2000], tree=(2, 2))]


@pytest.mark.parametrize("dtype", [I8, E4], ids=["int8", "e4m3"])
@pytest.mark.parametrize("case", range(len(Q8)))
def test_q8_without_a_second_segment(hip, case, dtype):
    c = dict(Q8[case])
    tree = c.pop("tree", None)
    words = [int(w) for w in VT.ancestor_words(VT.tree_from_branching(list(tree)))] if tree else None
    B, H, Hkv, d, lens = (c[k] for k in ("B", "H", "Hkv", "d", "lens"))
    N, Tp = len(words) if tree else c["N"], max(lens)
    dev = hip.torch_device
    g = R.gen(case)
    (kc, ks), (vc, vs) = (R.cache(g, B, Hkv, Tp + N, d, dtype) for _ in range(2))
    q = torch.randn(B, H, N, d, generator=g).to(torch.bfloat16)
    ref, mag = R.attention(q, R.values(kc, ks), R.values(vc, vs), lens, Tp, words, gates=torch.tensor(GATES[:1] + [0.0]))
    kw = dict(anc=None if words is None else np.array(words, dtype=np.uint64), max_len=Tp)
    args = (q.to(dev), *(t.to(dev) for t in (kc, vc, ks, vs)), torch.tensor(lens, dtype=torch.int32, device=dev))
    plain = hip.tree_attention_q8(*args, **kw)
    # fp32 on the device (one value is enough), a list: the binding's call and the general one
    for gates in (torch.tensor(GATES, device=dev), torch.tensor(GATES[:1], device=dev), GATES[:1], GATES):
        o = hip.tree_attention_q8(*args, gates=gates, **kw)
        _close(o, ref, mag)
        assert not torch.equal(o, plain)


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("d", [64, 128])
def test_tree_attention_without_a_second_segment(hip, d, splits):
    dev = hip.torch_device
    rng = np.random.default_rng(d)
    bf = lambda *s: torch.from_numpy(rng.normal(0, 1, s)).to(torch.bfloat16)
    words = VT.ancestor_words(VT.tree_from_branching([2, 2]))
    B, H, Hkv, N, Tp = 2, 4, 2, len(words), 300
    q, kc, vc, kt, vt = bf(B, H, N, d), bf(B, Hkv, Tp, d), bf(B, Hkv, Tp, d), bf(B, Hkv, N, d), bf(B, Hkv, N, d)
    gates = np.asarray(GATES, np.float32)
    ref, mag = OT.tree_attention_paths(*(t.float().numpy() for t in (q, kc, vc, kt, vt)), words, tp=[300, 7], gates=gates)
    o = hip.tree_attention(*(t.to(dev) for t in (q, kc, vc, kt, vt)), words, tp=np.asarray([300, 7], np.int32),
                           gates=gates, force_splits=splits)
    _close(o, torch.from_numpy(ref), torch.from_numpy(mag), 2e-5)


def test_fp32_rows_without_a_second_segment(hip):
    dev = hip.torch_device
    rng = np.random.default_rng(5)
    f = lambda *s: torch.from_numpy(rng.normal(0, 1, s).astype(np.float32))
    q, kc, vc, kt, vt = f(2, 4, 3, 16), f(2, 2, 20, 16), f(2, 2, 20, 16), f(2, 2, 3, 16), f(2, 2, 3, 16)
    gates = np.asarray(GATES, np.float32)
    ref, mag = OT.tree_attention_paths(*(t.numpy() for t in (q, kc, vc, kt, vt)), None, tp=[20, 4], gates=gates)
    o = hip.tree_attention(*(t.to(dev) for t in (q, kc, vc, kt, vt)), None, tp=np.asarray([20, 4], np.int32), gates=gates,
                           fp32_rows=True, out_dtype=torch.float32)
    _close(o, torch.from_numpy(ref), torch.from_numpy(mag), 2e-5)


@pytest.mark.parametrize("d,N", [(64, 40), (128, 300)])
def test_chain_attention_without_a_second_segment(hip, d, N):
    dev = hip.torch_device
    g = R.gen(d)
    B, H, Hkv, Tp = 2, 4, 2, 50
    q, kc, vc = (torch.randn(s, generator=g).to(torch.bfloat16).to(dev) for s in
                 ((B, H, N, d), (B, Hkv, Tp + N, d), (B, Hkv, Tp + N, d)))
    out = torch.empty_like(q)
    gates = torch.tensor(GATES, device=dev)
    tp = torch.tensor([50, 9], dtype=torch.int32, device=dev)
    a = _lib.TreeAttnArgs()
    a.q, a.k_cache, a.v_cache, a.out = q.data_ptr(), kc.data_ptr(), vc.data_ptr(), out.data_ptr()
    a.q_strides[:] = a.out_strides[:] = list(q.stride()[:3])
    a.cache_strides[:] = list(kc.stride()[:3])
    a.B, a.H, a.Hkv, a.Tp, a.N, a.d, a.scale, a.out_dtype = B, H, Hkv, Tp, N, d, d ** -0.5, _lib.VNX_BF16
    a.tp_batch, a.gates = tp.data_ptr(), gates.data_ptr()
    _lib.check(hip._L.vnx_chain_attn(ctypes.byref(a), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    ref, mag = R.attention(q.cpu(), kc.cpu().to(R.F64), vc.cpu().to(R.F64), [50, 9], Tp, gates=gates.cpu())
    _close(out, ref, mag, 2e-5)


def _model(hip, d, kv_dtype, cap):
    cfg = VM.ModelConfig(vocab_size=64, dim=4 * d, n_layer=1, n_head=4, n_kv_head=2, layer_pattern=("trisparse",),
                         window_size=70, num_global_tokens=0, use_alibi=False, use_rope=True, num_dense_parts=2,
                         num_experts_per_part=2, top_k=1)
    w = VM.init_weights(cfg, seed=1)
    w = {k: torch.tensor([-1.7, 0.4, 0.0]) if k.endswith("gate_logits") else t for k, t in w.items()}
    return VM.CometSparkGPU(cfg, w, hip, 2, cap, kv_dtype=kv_dtype)


@pytest.mark.parametrize("kv", [I8, E4, None], ids=["int8", "e4m3", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
def test_model_without_global_rows(hip, d, kv):
    """Every attention path of such a layer, on the same cache: gates[0] times the windowed attention."""
    dev = hip.torch_device
    Tp, lens = 90, [90, 20]
    m = _model(hip, d, kv, Tp + 80)
    g = R.gen(3)
    if kv is None:
        for c in (m.kc[0], m.vc[0]):
            c.copy_(torch.randn(c.shape, generator=g))
        k, v = (c.cpu().to(R.F64) for c in (m.kc[0], m.vc[0]))
        paths = dict(tree=m._attn_kernel, chunks=m._attn_tree_chunks, chain=m._attn_chain)
    else:
        for c, s in ((m.kc[0], m.ks[0]), (m.vc[0], m.vs[0])):
            codes, sc = R.cache(g, *c.shape, kv)
            c.copy_(codes.to(dev))
            s.copy_(sc.to(dev))
        k, v = (R.values(c.cpu(), s.cpu()) for c, s in ((m.kc[0], m.ks[0]), (m.vc[0], m.vs[0])))
        paths = dict(q8=m._attn_q8)
    ln = torch.tensor(lens, dtype=torch.int32, device=dev)
    assert abs(float(m.layers[0].gates[0]) - 0.1545) < 1e-3
    for n in (1, 5, 75):
        q = torch.randn(2, 4, n, d, generator=g).to(torch.bfloat16)
        ref, mag = R.attention(q, k, v, lens, Tp, window=70, gates=m.layers[0].gates.cpu())
        for name, f in dict(paths, torch=m._attn_torch).items():
            if name == "tree" and n > 64:
                continue
            print(f"d={d} {kv} n={n} {name}", flush=True)
            o = f(q.to(dev), 0, ln, n, Tp)
            o = o if o.dim() == 4 else o.view(2, n, 4, d).transpose(1, 2)
            _close(o, ref, mag)


def test_refusals(hip):
    dev = hip.torch_device
    kc = torch.zeros(1, 1, 4, 64, dtype=I8, device=dev)
    ks = torch.ones(1, 1, 4, device=dev)
    q = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16, device=dev)
    s2 = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16, device=dev)
    for kw in (dict(gates=[]), dict(gates=torch.ones(0, device=dev)), dict(gates=[1.0], seg2=(s2, s2)),
               dict(gates=torch.ones(1, device=dev), seg2=(s2, s2)), dict(seg2=(s2, s2))):
        with pytest.raises(ValueError):
            hip.tree_attention_q8(q, kc, kc, ks, ks, [3], **kw)
        with pytest.raises(ValueError):
            hip.tree_attention(q, None, None, q, q, [1], **kw)
    with pytest.raises(ValueError):
        hip.tree_attention(q, None, None, q, q, [1], gates=[1.0, 1.0], alibi_slopes=[0.5])
