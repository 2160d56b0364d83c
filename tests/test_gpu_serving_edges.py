"""The serving operators on the GPU where they are easily wrong, beyond test_gpu_serving.py: each test holds a case
that one of the kernels or its host side once got wrong."""

import pytest
import torch

from exactattention_b200 import serving
from test_gpu_serving import DEV, attention_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [1, 40])
def test_tree_attention_out_off_a_16_byte_boundary_is_refused(new):
    """A contiguous slice of a larger buffer. Refused on the host: nothing is launched."""
    x = attention_inputs([90], [new], 8, 2, 128, 16, torch.bfloat16)
    want = serving.tree_attention(**x)
    buf = torch.zeros(want.numel() + 8, dtype=want.dtype, device=DEV)
    for off in (1, 2, 4, 7):
        with pytest.raises(ValueError, match="16-byte"):
            serving.tree_attention(**x, out=buf[off:off + want.numel()].view(want.shape))
    out = buf[8:].view(want.shape)
    assert serving.tree_attention(**x, out=out) is out and torch.equal(out, want)
    assert not bool(buf[:8].any())
