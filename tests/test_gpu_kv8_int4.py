"""INT4 models with the cache in 8 bits hold one copy of the q|k|v weights: the one in the order of the GEMVs that write
16-bit cache rows is not built, and the rest of the forward stays fused as it is with that copy."""
import pytest
import torch

from versenext_amd import model as VM

pytestmark = pytest.mark.gpu


def _model(hip, kv_dtype, hidden):
    cfg = VM.ModelConfig(vocab_size=256, dim=256, n_layer=2, n_head=4, n_kv_head=2, layer_pattern=("trisparse",) * 2,
                         window_size=64, num_global_tokens=3, use_alibi=False, use_rope=True, mlp_hidden=hidden)
    return VM.CometSparkGPU(cfg, VM.init_weights(cfg, seed=3), hip, 2, 40, int4=True, kv_dtype=kv_dtype)


# (704, the width's own: no multiple of INT4's groups of 128, so those products are not fused either way)
@pytest.mark.parametrize("hidden,fused", [(None, 0), (768, 3 * 2)])
@pytest.mark.parametrize("kv", [torch.int8, torch.float8_e4m3fn], ids=["int8", "e4m3"])
def test_one_copy(hip, kv, hidden, fused, monkeypatch):
    dev = hip.torch_device
    a, b = _model(hip, kv, hidden), _model(hip, kv, hidden)
    used = []
    for m in (a, b):
        for L in m.layers:
            assert L.wqkv.int4 and L.wqkv.wq_rope is None and not hasattr(L.wqkv, "sc_rope")
    for L in b.layers:                       # as if it were there: the same calls, the same bits
        L.wqkv.wq_rope, L.wqkv.sc_rope = L.wqkv.wq, L.wqkv.sc
    for L in a.layers:
        monkeypatch.setattr(L.proj, "gemv_residual", lambda *x, f=L.proj.gemv_residual: used.append(1) or f(*x))
    tok = torch.arange(2 * 9, device=dev).view(2, 9)
    lens = torch.zeros(2, dtype=torch.int32, device=dev)
    for n in (9, 1, 4):
        assert torch.equal(a.forward(tok[:, :n], lens), b.forward(tok[:, :n], lens))
        lens += n
    assert len(used) == fused                # two layers of three forwards
    assert _model(hip, None, hidden).layers[0].wqkv.wq_rope is not None
