"""CometSparkGPU and SpecDecodeEngine with 8-bit products (w8a8), QuantizedLinear with 8-bit activations.

Every 8-bit call that a forward makes is recorded and held to the plain forms (tests/q8_ref.py) on the tensors it was given;
the wiring (which rows, which weights, residuals in place) is what these tests are for."""
import numpy as np
import pytest
import torch

import q8_ref as R
from versenext_amd import model as VM
from versenext_amd import quant as VQ
from versenext_amd.e2e import SpecDecodeEngine

pytestmark = pytest.mark.gpu


def _cfg(heads=4, kv=2, dim=256, window=40, G=5, pattern=("mod", "trisparse"), V=512, tied=True, **kw):
    return VM.ModelConfig(vocab_size=V, dim=dim, n_layer=len(pattern), n_head=heads, n_kv_head=kv, layer_pattern=pattern,
                          window_size=window, num_global_tokens=G, use_alibi=False, use_rope=True, num_dense_parts=2,
                          num_experts_per_part=2, top_k=1, tie_weights=tied, **kw)


def _weights(cfg, seed=3):
    return VM.init_weights(cfg, seed=seed)


class _Recorder:
    """The backend, with the 8-bit calls written down (arguments as they were before the call)."""

    def __init__(self, hip):
        self._hip, self.calls = hip, []

    def __getattr__(self, name):
        return getattr(self._hip, name)

    def _note(self, name, args, kw):
        keep = lambda t: t.detach().clone() if isinstance(t, torch.Tensor) else t
        before = [keep(t) for t in args], {k: keep(t) for k, t in kw.items()}
        out = getattr(self._hip, name)(*args, **kw)
        self.calls.append((name, *before, [keep(t) for t in (out if isinstance(out, tuple) else (out,))]))
        return out

    def quantize_rows(self, *a, **kw):
        return self._note("quantize_rows", a, kw)

    def rmsnorm_q8(self, *a, **kw):
        return self._note("rmsnorm_q8", a, kw)

    def linear_q8(self, *a, **kw):
        return self._note("linear_q8", a, kw)


def _check(call):
    name, a, kw, out = call
    cpu = lambda t: t.cpu() if isinstance(t, torch.Tensor) else t
    a, kw, out = [cpu(t) for t in a], {k: cpu(t) for k, t in kw.items()}, [cpu(t) for t in out]
    if name == "quantize_rows":
        c, s = R.quantize(a[0])
        assert torch.equal(out[0], c) and torch.equal(out[1], s)
    elif name == "rmsnorm_q8":
        x, w, eps = a
        c, s, total = R.rmsnorm(x, w, eps, kw.get("residual"))
        assert torch.equal(out[0], c) and torch.equal(out[2], total)
        assert ((out[1].double() - s).abs() <= 30 * R.U * s).all()
    else:
        y, tol = R.linear(*a, residual=kw.get("residual"), swiglu=kw.get("swiglu", False), out=out[0].dtype)
        assert not R.off(out[0], y, tol).any()


def _spy(m, hip):
    rec = _Recorder(hip)
    m.hip = rec
    for L in m.layers:
        for lin in (L.wqkv, L.proj, *(v for v in L.ffn.values() if isinstance(v, VM._Linear))):
            lin.hip = rec
    m.head.hip = rec
    return rec


@pytest.mark.parametrize("kv", [None, torch.int8], ids=["bf16", "int8"])
@pytest.mark.parametrize("pattern", [("trisparse", "trisparse"), ("mod", "trisparse")])
def test_forward_calls(hip, pattern, kv):
    """A ragged prompt, a verify chunk, single tokens, logits: every 8-bit call, and what the products were given."""
    cfg = _cfg(pattern=pattern)
    W = _weights(cfg)
    m = VM.CometSparkGPU(cfg, W, hip, 2, 130, kv_dtype=kv, w8a8=True)
    rec = _spy(m, hip)
    g = torch.Generator().manual_seed(1)
    lens = [0, 0]
    ffn = {"trisparse": ["rmsnorm_q8", "linear_q8", "quantize_rows", "linear_q8"], "mod": []}
    for n, step in ((70, [70, 33]), (5, [2, 5]), (1, [1, 1])):
        tok = torch.randint(0, 512, (2, n), generator=g).to(hip.torch_device)
        rec.calls.clear()
        h = m.forward(tok, torch.tensor(lens, dtype=torch.int32, device=hip.torch_device))
        assert h.shape == (2, n, 256) and torch.isfinite(h).all()
        want = [c for k in pattern for c in ["rmsnorm_q8", "linear_q8", "quantize_rows", "linear_q8"] + ffn[k]]
        assert [c[0] for c in rec.calls] == want
        for c in rec.calls:
            _check(c)
        # each norm's codes go into the product behind it; the residual stream runs through the layers
        for a, b in zip(rec.calls, rec.calls[1:]):
            if b[0] == "linear_q8":
                assert torch.equal(a[3][0], b[1][0]) and torch.equal(a[3][1], b[1][1])
        first = W["tok_emb.weight"].to(torch.bfloat16).float()[tok.cpu().view(-1)] * 16.0
        assert torch.equal(rec.calls[0][1][0].cpu(), first)
        q, s = VQ.quantize_int8(torch.cat([W[f"blocks.0.attn.{k}.weight"] for k in ("wq", "wk", "wv")]))
        assert torch.equal(rec.calls[1][1][2].cpu(), q) and torch.equal(rec.calls[1][1][3].cpu(), s.view(-1))
        if pattern[0] == "trisparse":                     # down's result is the next layer's norm's input
            assert torch.equal(rec.calls[7][3][0], rec.calls[8][1][0])
        rec.calls.clear()
        for out in (None, torch.empty(2, n, 512, dtype=torch.bfloat16, device=hip.torch_device),
                    torch.empty(2, n + 1, 512, device=hip.torch_device)[:, 1:] if n == 1 else None):
            lg = m.logits(h, out=out)
            assert lg.shape == (2, n, 512) and (out is None or lg is out)
        for c in rec.calls:
            _check(c)
        lens = [a + b for a, b in zip(lens, step)]


def test_next_to_the_bf16_model(hip):
    """Eight products of two layers, each of whose operands is off by at most half a step of max / 127 a value: with a
    maximum of four times the root mean square 4 / 127 / sqrt(12) = 0.9% of it, 1.3% a product; added up, 0.104."""
    cfg = _cfg(pattern=("trisparse", "trisparse"), tied=False)
    W = _weights(cfg)
    a = VM.CometSparkGPU(cfg, W, hip, 2, 100, w8a8=True)
    b = VM.CometSparkGPU(cfg, W, hip, 2, 100)
    assert a.head_w is None and a.layers[0].wqkv.q.dtype == torch.int8
    tok = torch.randint(0, 512, (2, 40), generator=torch.Generator().manual_seed(5)).to(hip.torch_device)
    lens = torch.zeros(2, dtype=torch.int32, device=hip.torch_device)
    x, y = a.forward(tok, lens), b.forward(tok, lens)
    assert 0 < (x - y).norm() <= 0.104 * y.norm()
    p, q = a.logits(x), b.logits(x)
    assert 0 < (p - q).norm() <= 0.02 * q.norm()          # one product, and the bf16 head's 2^-8 an operand
    # the global rows of INT8 key weights
    wk = VQ.quantize_int8(W["blocks.0.attn.wk.weight"])
    gk = W["blocks.0.attn.global_tokens.weight"].double() @ (wk[0].double() * wk[1].double()).t()
    got = a.layers[0].gk[0].permute(1, 0, 2).reshape(5, -1).double().cpu()
    assert ((got - gk).abs() <= 2.0 ** -8 * gk.abs() + 1e-4 * gk.abs().max()).all()


def test_odd_sizes(hip):
    """Rows that 16 does not divide."""
    cfg = _cfg(heads=2, kv=1, dim=136, pattern=("trisparse",), V=301, mlp_hidden=203)
    m = VM.CometSparkGPU(cfg, _weights(cfg), hip, 1, 30, w8a8=True)
    assert m.layers[0].ffn["down"].q.stride(0) == 208
    rec = _spy(m, hip)
    tok = torch.arange(9, device=hip.torch_device).view(1, 9)
    h = m.forward(tok, torch.zeros(1, dtype=torch.int32, device=hip.torch_device))
    m.logits(h)
    assert len(rec.calls) == 10
    for c in rec.calls:
        _check(c)


def test_refusals(hip):
    cfg = _cfg()
    W = _weights(cfg)
    for kw in (dict(w8a8=True, int4=True), dict(w8a8=True, dtype=torch.float32)):
        with pytest.raises(ValueError):
            VM.CometSparkGPU(cfg, W, hip, 1, 16, **kw)


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_engine(hip, temperature):
    """Speculative rounds of a w8a8 target, captured: a second run of the same prompts gives the same bits, and the rounds
    equal eager ones."""
    dev = hip.torch_device
    B, k, T0, new = 2, 3, 20, 24
    target = VM.CometSparkGPU(_cfg(), _weights(_cfg()), hip, B, 80, w8a8=True)
    dc = _cfg(pattern=("trisparse",))
    draft = VM.CometSparkGPU(dc, _weights(dc), hip, B, 80, w8a8=True)
    prompts = torch.randint(0, 512, (B, T0), generator=torch.Generator().manual_seed(4)).to(dev)
    got = []
    for graph in (True, True, False):
        eng = SpecDecodeEngine(target, draft, hip, k, temperature, use_graph=graph, seed=7)
        out, st = eng.generate(prompts, new, uniforms=lambda r: (torch.full((k, B), 0.3 + 0.01 * r),
                                                                 torch.full((B, k + 1), 0.6)))
        assert st.emitted == B * new and ((out >= 0) & (out < 512)).all()
        assert temperature == 0.0 or eng.logits_dtype == torch.bfloat16
        got.append(out)
    assert torch.equal(got[0], got[1])
    # (attention's launch shape goes by the bound of the lengths, so the eager rounds differ in its roundings)
    assert got[2].shape == got[0].shape


@pytest.mark.parametrize("N,K", [(300, 512), (77, 100)])
@pytest.mark.parametrize("bias", [False, True])
def test_quantized_linear(hip, N, K, bias):
    g = R.gen(N)
    w, x = torch.randn(N, K, generator=g), torch.randn(3, 5, K, generator=g)
    b = torch.randn(N, generator=g) if bias else None
    lin = VQ.QuantizedLinear(w, bias=b, qtype="int8", act_bits=8)
    q, s = VQ.quantize_int8(w)
    assert torch.equal(lin.wq.cpu(), q) and torch.equal(lin.dequantize().cpu(), q * s)
    for t in (x, x.bfloat16(), x.double(), x.numpy(), x.half().to(hip.torch_device)):
        rows = torch.as_tensor(t).cpu()
        rows = (rows.float() if rows.dtype == torch.float64 else rows).view(15, K)
        y, tol = R.linear(*R.quantize(rows), q, s.view(-1), b)
        got = lin(t)
        assert got.shape == (3, 5, N) and got.dtype == torch.float32 and not R.off(got.view(15, N), y, tol).any()
    with pytest.raises(ValueError):
        lin(x[..., :-1])


def test_quantized_linear_refusals(hip):
    w = torch.randn(16, 128)
    for kw in (dict(qtype="int4", act_bits=8), dict(act_bits=8), dict(qtype="int8", act_bits=4)):
        with pytest.raises(ValueError):
            VQ.QuantizedLinear(w, **kw)
    assert np.isfinite(VQ.QuantizedLinear(w, qtype="int8")(torch.randn(2, 128)).cpu().numpy()).all()
