"""What a tree's launch carries among its arguments (ancestor words, parents' rows, ranks), call after call: 8-bit and 16-bit
tree attention give the bits of the call whose words lie on the device, the greedy verify and the expansion what the tree's
definition says."""
import numpy as np
import pytest
import torch

import kv8_ref as R
from oracle import tree as OT
from versenext_amd import tree as VT

pytestmark = pytest.mark.gpu

CALLS = 12


def tree_of(N, seed):
    return np.concatenate([[-1], np.random.default_rng(seed).integers(-1, np.arange(1, N))]).astype(np.int32) if N > 1 \
        else np.array([-1], np.int32)


# one to sixteen nodes a tile (16 columns, or 32): query heads to a KV head 16, 4, 3 and 1
@pytest.mark.parametrize("tiles,waves", [(1, 4), (1, 8), (2, 4), (2, 8)])
@pytest.mark.parametrize("N,H,Hkv,d,window", [(1, 16, 1, 64, 0), (40, 8, 2, 128, 0), (64, 6, 2, 64, 70), (23, 2, 2, 128, 0),
                                              (64, 3, 3, 64, 0)])
def test_8bit_attention(hip, N, H, Hkv, d, window, tiles, waves):
    dev = hip.torch_device
    words = VT.ancestor_words(tree_of(N, N))
    words[-1] = 0
    g = R.gen(N + d)
    dtype = torch.float8_e4m3fn if N % 2 else torch.int8
    (kc, ks), (vc, vs) = (R.cache(g, 2, Hkv, 200 + N, d, dtype) for _ in range(2))
    q = torch.randn(2, H, N, d, generator=g).to(torch.bfloat16)
    args = [x.to(dev) for x in (q, kc, vc, ks, vs)]
    on_device = torch.from_numpy(np.asarray(words, np.uint64).view(np.int64)).to(dev)[None].repeat(2, 1).contiguous()
    for splits in (1, 8):
        kw = dict(max_len=200, window=window, force_tiles=tiles, force_waves=waves, force_splits=splits)
        want = hip.tree_attention_q8(*args, [200, 3], anc=on_device, **kw)
        for _ in range(CALLS):
            assert torch.equal(hip.tree_attention_q8(*args, [200, 3], anc=words, **kw), want)


@pytest.mark.parametrize("waves", [4, 5, 8, 9, 16])
@pytest.mark.parametrize("N,H,Hkv,d,Tp", [(1, 16, 8, 64, 640), (7, 16, 8, 64, 301), (40, 8, 2, 128, 300), (64, 4, 4, 64, 0),
                                          (64, 8, 1, 64, 1000)])
def test_16bit_attention(hip, N, H, Hkv, d, Tp, waves):
    dev = hip.torch_device
    words = VT.ancestor_words(tree_of(N, N))
    g = torch.Generator(device=dev).manual_seed(N + Tp)
    r = lambda *s: torch.randn(s, generator=g, device=dev).to(torch.bfloat16)
    kc, vc = (r(2, Hkv, Tp, d), r(2, Hkv, Tp, d)) if Tp else (None, None)
    args = (r(2, H, N, d), kc, vc, r(2, Hkv, N, d), r(2, Hkv, N, d))
    want = hip.tree_attention(*args, np.tile(words, (2, 1)), force_waves=waves)
    for _ in range(CALLS):
        assert torch.equal(hip.tree_attention(*args, words, force_waves=waves), want)


@pytest.mark.parametrize("N", [1, 6, 40, 64])
def test_greedy_and_expansion(hip, N):
    dev = hip.torch_device
    par, rng = tree_of(N, 3 * N), np.random.default_rng(N)
    B, V = 3, 997
    logits = rng.standard_normal((B, N + 1, V)).astype(np.float32)
    best = logits.argmax(-1)
    tokens = np.where(rng.random((B, N)) < 0.8, best[:, np.where(par < 0, 0, par + 1)], rng.integers(0, V, (B, N)))
    want = OT.tree_greedy(logits, tokens, par)           # (accept_len, best, out_ids, pred)
    width = want[2].shape[1]
    d, t = torch.from_numpy(logits).to(dev), torch.from_numpy(tokens.astype(np.int64)).to(dev)
    nodes = OT.expand_tree(logits, par)
    for _ in range(CALLS):
        alen, at, out, pred = (x.cpu().numpy() for x in hip.tree_greedy(d, t, par))
        for a, b in zip((alen, at, out[:, :width], pred), want):
            assert np.array_equal(a, b)
        assert (out[:, width:] == -1).all()
        assert np.array_equal(hip.expand_tree(d, par).cpu().numpy(), nodes)
