"""Captured speculative rounds of w8a8 models against eager rounds of the same attention bounds: tokens, acceptances and
logits bit for bit, round after round, prompts changing under the graph."""
import pytest
import torch

from test_gpu_q8_model import _cfg, _weights
from versenext_amd import model as VM
from versenext_amd.e2e import SpecDecodeEngine

pytestmark = pytest.mark.gpu

B, K, NEW = 2, 3, 20


class _Eager(SpecDecodeEngine):
    """Eager rounds that size their attention calls as a captured round does."""

    def _round(self, tmax_t, tmax_d):
        super()._round(self.bound_t, self.bound_d)


def _models(hip, pattern, kv, same):
    """Target and draft; the same weights in both: drafts are accepted."""
    cfg = _cfg(pattern=pattern)
    dc = cfg if same else _cfg(pattern=("trisparse",))
    return [VM.CometSparkGPU(c, _weights(c), hip, B, 80, kv_dtype=kv, w8a8=True) for c in (cfg, dc)]


def _uniforms(r):
    g = torch.Generator().manual_seed(100 + r)
    return torch.rand(K, B, generator=g), torch.rand(B, K + 1, generator=g)


def _prompts(hip, n):
    g = torch.Generator().manual_seed(7)
    return [torch.randint(0, 512, (B, 20), generator=g).to(hip.torch_device) for _ in range(n)]


@pytest.mark.parametrize("temperature", [0.0, 0.8])
@pytest.mark.parametrize("kv", [None, torch.int8], ids=["bf16", "int8"])
@pytest.mark.parametrize("pattern,same", [(("trisparse", "trisparse"), True), (("mod", "trisparse"), False)])
def test_generate(hip, pattern, same, kv, temperature):
    target, draft = _models(hip, pattern, kv, same)
    graph = SpecDecodeEngine(target, draft, hip, K, temperature, use_graph=True, seed=7)
    for p in _prompts(hip, 3):
        out, st = graph.generate(p, NEW, uniforms=_uniforms)
        want, eager = _Eager(target, draft, hip, K, temperature, seed=7).generate(p, NEW, uniforms=_uniforms)
        assert torch.equal(out, want) and st.per_round_tokens == eager.per_round_tokens
        assert not same or temperature or st.accepted_drafts > 0
    assert graph.graph is not None


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_every_round(hip, temperature):
    """Two pairs of models of the same weights side by side: logits, acceptances and lengths after each round, eager work
    between the replays."""
    pair = [_models(hip, ("mod", "trisparse"), None, False) for _ in range(2)]
    engines = [SpecDecodeEngine(*pair[0], hip, K, temperature, use_graph=True), _Eager(*pair[1], hip, K, temperature)]
    p = _prompts(hip, 1)[0]
    for e in engines:
        e.prefill(p, NEW)
    engines[0]._capture()
    for r in range(5):
        infos = [e.step(_uniforms(r)) for e in engines]
        torch.cuda.synchronize()
        a, b = engines
        assert torch.equal(*infos) and torch.equal(a.toks, b.toks)
        assert torch.equal(a.pbuf, b.pbuf) and torch.equal(a.qbuf, b.qbuf)
        assert torch.equal(a.last["accept_len"], b.last["accept_len"]) and torch.equal(a.lens_t, b.lens_t)
        assert torch.equal(a.out, b.out)
