"""CometSparkGPU and SpecDecodeEngine with the cache in 8 bits.

Every kv_write and tree_attention_q8 call that a forward makes is recorded and held to the plain forms (tests/kv8_ref.py)
on the tensors it was given: the wiring (positions, window, global rows, gates, layouts) is what these tests are for."""
import numpy as np
import pytest
import torch

import kv8_ref as R
from versenext_amd import model as VM
from versenext_amd.e2e import SpecDecodeEngine

pytestmark = pytest.mark.gpu

I8, E4 = torch.int8, torch.float8_e4m3fn


def _cfg(heads=4, kv=2, dim=256, window=40, G=5, pattern=("mod", "trisparse"), alibi=False, V=512):
    return VM.ModelConfig(vocab_size=V, dim=dim, n_layer=len(pattern), n_head=heads, n_kv_head=kv, layer_pattern=pattern,
                          window_size=window, num_global_tokens=G, use_alibi=alibi, use_rope=True, num_dense_parts=2,
                          num_experts_per_part=2, top_k=1)


def _model(hip, cfg, B, cap, kv_dtype, int4=False, seed=3):
    w = VM.init_weights(cfg, seed=seed)
    g = torch.Generator().manual_seed(seed)
    w = {k: (t * 4 if k.endswith(("wq.weight", "wk.weight")) else torch.randn(3, generator=g) if k.endswith("gate_logits")
             else t) for k, t in w.items()}
    return VM.CometSparkGPU(cfg, w, hip, B, cap, int4=int4, kv_dtype=kv_dtype)


class _Recorder:
    """The backend, with the 8-bit cache's calls written down (arguments as they were before the call)."""

    def __init__(self, hip):
        self._hip, self.calls = hip, []

    def __getattr__(self, name):
        return getattr(self._hip, name)

    def kv_write(self, qkv, kc, vc, lens, ks, vs, **kw):
        q = self._hip.kv_write(qkv, kc, vc, lens, ks, vs, **kw)
        self.calls.append(("write", qkv.clone(), [t.clone() for t in (kc, vc, ks, vs)], lens.clone(), kw, q.clone()))
        return q

    def tree_attention_q8(self, q, kc, vc, ks, vs, lens, **kw):
        o = self._hip.tree_attention_q8(q, kc, vc, ks, vs, lens, **kw)
        self.calls.append(("attn", q.clone(), [t.clone() for t in (kc, vc, ks, vs)], lens.clone(), kw, o.clone()))
        return o


def _check(m, call, lens, n):
    what, x, cache, ln, kw, got = call
    cfg = m.cfg
    kc, vc, ks, vs = (t.cpu() for t in cache)
    assert ln.tolist() == lens
    if what == "write":
        B = len(lens)
        d, H, Hkv = cfg.head_dim, cfg.n_head, cfg.n_kv_head
        t = x.float().cpu().view(B, n, H + 2 * Hkv, d).transpose(1, 2)
        at = torch.stack([torch.arange(s, s + n) for s in lens])
        cos, sin = (z.cpu()[at][:, None] for z in (m.cos, m.sin))
        assert torch.equal(got.cpu(), R.rotate(t[:, :H], cos, sin).to(torch.bfloat16))
        for rows, c, s in ((R.rotate(t[:, H:H + Hkv], cos, sin), kc, ks), (t[:, H + Hkv:], vc, vs)):
            codes, sc = R.quantise(rows, c.dtype)
            for b in range(B):
                assert torch.equal(c[b][:, at[b]].view(torch.uint8), codes[b].view(torch.uint8))
                assert torch.equal(s[b][:, at[b]], sc[b])
        return
    assert kw["window"] == cfg.window_size and kw["max_len"] >= max(lens)
    end = max(lens) + n
    ref, mag = R.attention(x.cpu(), R.values(kc[:, :, :end], ks[:, :, :end]), R.values(vc[:, :, :end], vs[:, :, :end]),
                           lens, kw["max_len"], None, kw["window"], None, [t.cpu() for t in kw["seg2"]], kw["gates"].cpu())
    err = (got.cpu().to(R.F64) - ref).abs()
    half = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -11
    assert (err <= 2.0 ** -10 * mag + half * ref.abs() + 2.0 ** -25).all()   # P in 11 bits, the 64-bit form's own values


@pytest.mark.parametrize("kv", [I8, E4], ids=["int8", "e4m3"])
@pytest.mark.parametrize("int4", [False, True], ids=["bf16", "int4"])
@pytest.mark.parametrize("heads,kvh", [(4, 2), (2, 2)])
def test_forward_calls(hip, heads, kvh, int4, kv):
    """A ragged prompt, a verify chunk and single tokens: every write and attention of every layer."""
    pattern = ("trisparse", "trisparse") if int4 else ("mod", "trisparse")
    m = _model(hip, _cfg(heads, kvh, pattern=pattern), 2, 130, kv, int4=int4)
    m.hip = rec = _Recorder(hip)
    for L in m.layers:
        L.wqkv.hip = hip
    g = torch.Generator().manual_seed(1)
    lens = [0, 0]
    for n, step in ((70, [70, 33]), (5, [2, 5]), (1, [1, 1]), (1, [1, 0])):
        tok = torch.randint(0, 512, (2, n), generator=g).to(hip.torch_device)
        rec.calls.clear()
        h = m.forward(tok, torch.tensor(lens, dtype=torch.int32, device=hip.torch_device))
        assert h.shape == (2, n, 256) and torch.isfinite(h).all()
        assert [c[0] for c in rec.calls] == ["write", "attn"] * 2
        for c in rec.calls:
            _check(m, c, lens, n)
        lens = [a + b for a, b in zip(lens, step)]
    # the caller that needs the rows alone: both layers written, no attention after the last
    rec.calls.clear()
    assert m.forward(tok, torch.tensor(lens, dtype=torch.int32, device=hip.torch_device), cache_only=True) is None
    assert [c[0] for c in rec.calls] == ["write", "attn", "write"]


@pytest.mark.parametrize("kv", [I8, E4], ids=["int8", "e4m3"])
def test_kernel_and_read_back_paths(hip, kv):
    """The same forwards with vnx_tree_attn_q8 and with kv_read + PyTorch attention: both round the attention to bf16 once
    (2^-8) a layer, through two layers of a residual stream that carries more than it: 2^-6 in the norm."""
    cfg = _cfg()
    dev = hip.torch_device
    a, b = (_model(hip, cfg, 2, 100, kv) for _ in range(2))
    b.kernel_q8 = False
    g = torch.Generator().manual_seed(2)
    for n, lens in ((66, [0, 0]), (6, [60, 66])):
        tok = torch.randint(0, 512, (2, n), generator=g).to(dev)
        ln = torch.tensor(lens, dtype=torch.int32, device=dev)
        x, y = a.forward(tok, ln), b.forward(tok, ln)
        assert (x - y).norm() <= 2.0 ** -6 * y.norm()


@pytest.mark.parametrize("kv", [I8, E4], ids=["int8", "e4m3"])
def test_models_that_the_kernel_does_not_take(hip, kv):
    """Heads of 16 and ALiBi: the read-back path; a model without global rows."""
    dev = hip.torch_device
    tok = torch.arange(2 * 9, device=dev).view(2, 9)
    lens = torch.zeros(2, dtype=torch.int32, device=dev)
    for cfg in (_cfg(4, 2, 64), _cfg(2, 1, 128, alibi=True)):
        m = _model(hip, cfg, 2, 20, kv)
        assert not m.kernel_q8
        assert torch.isfinite(m.forward(tok, lens)).all()
        assert (m.ks[0][:, :, :9] > 0).all() and (m.ks[0][:, :, 9:] == 0).all()
    m = _model(hip, _cfg(2, 1, 128, G=0), 2, 20, kv)
    assert m.kernel_q8 and torch.isfinite(m.forward(tok, lens)).all()


def test_kv_dtype_refusals(hip):
    cfg = _cfg()
    w = VM.init_weights(cfg)
    for kw in (dict(kv_dtype=torch.float16), dict(kv_dtype=torch.int8, dtype=torch.float32)):
        with pytest.raises(ValueError):
            VM.CometSparkGPU(cfg, w, hip, 1, 16, **kw)
    odd = _cfg(2, 2, 96)
    with pytest.raises(ValueError):
        VM.CometSparkGPU(odd, VM.init_weights(odd), hip, 1, 16, kv_dtype=torch.int8)


@pytest.mark.parametrize("kv", [I8, E4], ids=["int8", "e4m3"])
def test_engine(hip, kv):
    """Speculative rounds with both caches in 8 bits, captured: each round's acceptance against the logits that it was
    given, the caches' lengths, a second run of the same prompts the same bits, and the first round against an eager one."""
    dev = hip.torch_device
    B, k, T0, new = 2, 3, 20, 24
    tc, dc = _cfg(), _cfg(pattern=("trisparse",))
    target, draft = _model(hip, tc, B, 80, kv), _model(hip, dc, B, 80, kv, int4=True)
    prompts = torch.randint(0, 512, (B, T0), generator=torch.Generator().manual_seed(4)).to(dev)
    eng = SpecDecodeEngine(target, draft, hip, k, 0.0, use_graph=True)
    one, st = eng.generate(prompts, new)
    assert one.shape == (B, new) and st.emitted == B * new and (one >= 0).all() and (one < 512).all()
    two, _ = eng.generate(prompts, new)
    assert torch.equal(one, two)
    eng.prefill(prompts, new)
    eng.step()
    torch.cuda.synchronize(dev)
    first = eng.pbuf.float().argmax(-1).cpu()
    toks, alen = eng.toks.cpu(), eng.last["accept_len"].cpu()
    lens = (eng.lens_t.cpu() - (T0 - 1)).tolist()
    for b in range(B):
        n = 0
        while n < k and toks[b, n + 1] == first[b, n]:
            n += 1
        assert alen[b] == n and lens[b] == n + 1
    # the same round eagerly: the launch shapes differ, the logits by bf16 roundings of the attention alone
    plain = SpecDecodeEngine(target, draft, hip, k, 0.0)
    plain.prefill(prompts, new)
    plain.step()
    assert (plain.pbuf[:, :1] - eng.pbuf[:, :1]).norm() <= 2.0 ** -6 * eng.pbuf[:, :1].norm()
