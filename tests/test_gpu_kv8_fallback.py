"""Models with the cache in 8 bits whose attention no kernel takes (heads of 16 and 32, ALiBi): the values that the cache
stands for, the window, the global rows, ALiBi and the gates, against the 64-bit form.

Bar: fp32 scores and sums, 2e-5 of sum p |v|; with ALiBi 2^-13 (a bias of up to 1,000 rounded in the exponent)."""
import numpy as np
import pytest
import torch

import kv8_ref as R
from oracle import tree as OT
from versenext_amd import model as VM

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", [torch.int8, torch.float8_e4m3fn], ids=["int8", "e4m3"])
@pytest.mark.parametrize("d,alibi,G,lens", [(16, False, 5, [60, 3]), (32, False, 0, [0, 41]), (64, True, 5, [70, 9]),
                                            (64, True, 0, [1020, 200]), (128, True, 3, [30, 30]), (16, True, 4, [50, 0])])
def test_read_back_attention(hip, d, alibi, G, lens, kv):
    dev = hip.torch_device
    cfg = VM.ModelConfig(vocab_size=64, dim=4 * d, n_layer=1, n_head=4, n_kv_head=2, layer_pattern=("trisparse",),
                         window_size=40, num_global_tokens=G, use_alibi=alibi, use_rope=True, num_dense_parts=2,
                         num_experts_per_part=2, top_k=1)
    w = VM.init_weights(cfg, seed=1)
    w = {k: torch.tensor([-1.2, 0.4, 0.9]) if k.endswith("gate_logits") else t for k, t in w.items()}
    m = VM.CometSparkGPU(cfg, w, hip, 2, max(lens) + 20, kv_dtype=kv)
    assert not m.kernel_q8
    g = R.gen(d)
    for c, s in ((m.kc[0], m.ks[0]), (m.vc[0], m.vs[0])):
        codes, sc = R.cache(g, *c.shape, kv)
        c.copy_(codes.to(dev))
        s.copy_(sc.to(dev))
    k, v = (R.values(c.cpu(), s.cpu()).numpy() for c, s in ((m.kc[0], m.ks[0]), (m.vc[0], m.vs[0])))
    L = m.layers[0]
    seg2 = tuple(t.float().cpu().numpy() for t in (L.gk, L.gv)) if G else None
    slopes = m.slopes.cpu().numpy() if alibi else None
    ln = torch.tensor(lens, dtype=torch.int32, device=dev)
    for n in (1, 7):
        q = torch.randn(2, 4, n, d, generator=g).to(torch.bfloat16)
        o = m._attn_torch(q.to(dev), 0, ln, n, max(lens)).double().cpu().numpy()
        for b, t in enumerate(lens):
            at = slice(b, b + 1)
            ref, mag = OT.tree_attention_paths(q[at].float().numpy(), k[at, :, :t] if t else None, v[at, :, :t] if t else None,
                                               k[at, :, t:t + n], v[at, :, t:t + n], None, window=40, slopes=slopes,
                                               alibi_max=1024, seg2=seg2, gates=L.gates.cpu().numpy())
            err = np.abs(o[b] - ref[0])
            assert (err <= (2.0 ** -13 if alibi else 2e-5) * mag[0] + 1e-9).all(), (b, n, (err / mag[0]).max())
