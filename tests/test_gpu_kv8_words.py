"""tree_attention_q8 with the ancestor words on the host (they travel among the kernel's arguments) gives, call after call,
the bits of the call with them on the device."""
import numpy as np
import pytest
import torch

import kv8_ref as R
from versenext_amd import tree as VT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn], ids=["int8", "e4m3"])
@pytest.mark.parametrize("d,splits", [(64, 1), (64, 32), (128, 1), (128, 2), (128, 32)])
def test_words_on_the_host(hip, d, splits, dtype):
    dev = hip.torch_device
    words = np.array([int(w) for w in VT.ancestor_words(VT.tree_from_branching([4, 3, 2]))], dtype=np.uint64)
    words[-1] = 0
    N, lens = len(words), [300, 0]
    g = R.gen(d + splits)
    caches = [R.cache(g, 2, 2, 300 + N, d, dtype) for _ in range(2)]
    q = (torch.randn(2, 8, N, d, generator=g) * 1.5).to(torch.bfloat16)
    args = [x.to(dev) for x in (q, caches[0][0], caches[1][0], caches[0][1], caches[1][1])]
    kw = dict(max_len=300, out_dtype=torch.float16, force_tiles=1, force_waves=4, force_splits=splits)
    on_device = torch.from_numpy(words.view(np.int64)).to(dev)[None].repeat(2, 1).contiguous()
    want = hip.tree_attention_q8(*args, lens, anc=on_device, **kw)
    for _ in range(24):
        assert torch.equal(hip.tree_attention_q8(*args, lens, anc=words, **kw), want)
