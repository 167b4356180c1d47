"""CometSparkGPU.from_vn(w8a8=True): the codes, scales, global rows and results of the model of the same weights in memory."""
import numpy as np
import pytest
import torch

from test_gpu_vn import _draft_cfg, _nex_config
from tests.vn_fixture import write_vn
from versenext_amd import model as VM

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,chunk", [("safetensors", 1 << 20), ("npz", 300 << 10)])
def test_equals_the_model_in_memory(hip, tmp_path, fmt, chunk):
    cfg = _draft_cfg()
    W = VM.init_weights(cfg, seed=21)
    state = {k: v.numpy().astype(np.float32) for k, v in W.items()}
    state["head.weight"] = state["tok_emb.weight"]
    path = tmp_path / "m.vn"
    write_vn(path, state, _nex_config(cfg), fmt=fmt)
    a = VM.CometSparkGPU.from_vn(str(path), hip, batch=2, capacity=40, chunk_bytes=chunk, w8a8=True)
    b = VM.CometSparkGPU(cfg, W, hip, batch=2, capacity=40, w8a8=True)
    assert torch.equal(a.head.q, b.head.q) and torch.equal(a.head.qs, b.head.qs) and torch.equal(a.emb, b.emb)
    for x, y in zip(a.layers, b.layers):
        assert torch.equal(x.gk, y.gk) and torch.equal(x.gv, y.gv)
        for p, q in ((x.wqkv, y.wqkv), (x.proj, y.proj), (x.ffn["gu"], y.ffn["gu"]), (x.ffn["down"], y.ffn["down"])):
            assert torch.equal(p.q, q.q) and torch.equal(p.qs, q.qs)
    tok = torch.randint(0, cfg.vocab_size, (2, 9), generator=torch.Generator().manual_seed(1)).to(hip.torch_device)
    lens = torch.zeros(2, dtype=torch.int32, device=hip.torch_device)
    p, q = (m.logits(m.forward(tok, lens, 0)[:, -2:]) for m in (a, b))
    assert torch.isfinite(p).all() and torch.equal(p, q)
