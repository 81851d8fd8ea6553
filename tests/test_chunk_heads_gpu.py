"""GPU tests of the chunk attention's refusals by head counts and scale, with the split count left to its rule."""

import pytest

from chunk_cases import ChunkBatch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads", [(300, 2), (18, 2), (10, 4), (2, 4)])
def test_unsupported_heads(cuda_device, heads):
    with pytest.raises(NotImplementedError, match="1 to 8, 16 or 32"):
        ChunkBatch([(1, 3, 4)], *heads, cuda_device).attend()


@pytest.mark.parametrize("scale", [0.0, -1.0, float("nan"), float("inf"), 1e39, 1e30, 1e-60])
def test_scales_out_of_range(cuda_device, scale):
    with pytest.raises(ValueError, match="softmax_scale"):
        ChunkBatch([(1, 3, 4)], 4, 2, cuda_device).attend(softmax_scale=scale)
