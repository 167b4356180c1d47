"""CometSparkGPU.from_vn with w8a8: what does not go together is refused before the file is opened (no GPU needed)."""
import pytest
import torch

from versenext_amd import model as VM


@pytest.mark.parametrize("kw", [dict(int4=True), dict(dtype=torch.float32), dict(dtype=torch.float16, int4=False)])
def test_refused_before_the_file(kw):
    with pytest.raises(ValueError, match="w8a8"):
        VM.CometSparkGPU.from_vn("/no/such/file.vn", None, 1, 16, w8a8=True, **kw)


def test_the_plain_call_opens_the_file():
    with pytest.raises(OSError):
        VM.CometSparkGPU.from_vn("/no/such/file.vn", None, 1, 16, w8a8=True)
