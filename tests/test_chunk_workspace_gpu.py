"""GPU tests of the chunk attention with a workspace that the caller sized: by the package's own names, nothing allocated."""

import pytest
import torch

from chunk_cases import ChunkBatch
from nvfp4_attn_kernel_b200.nvfp4_decode_kernel import chunk_split_heuristic, chunk_workspace_bytes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,bound", [([(40, 9, 4), (3, 0, 2)], 4), ([(40, 9, 4), (3, 0, 2)], 1000), ([(60, 0, 200)], 200)])
def test_the_rules_count_and_its_scratch(cuda_device, rows, bound):
    """`bound`: max_chunk_len, also one far above the tokens that there are."""
    batch = ChunkBatch(rows, 8, 2, cuda_device, seed=60)
    sms = torch.cuda.get_device_properties(cuda_device).multi_processor_count
    splits = chunk_split_heuristic(len(rows), batch.tokens, bound, 8, 2, batch.columns, sms=sms)
    need = chunk_workspace_bytes(batch.tokens, 8, splits)
    assert splits > 1 and need > 0
    space, out = torch.empty(need, dtype=torch.uint8, device=cuda_device), torch.empty_like(batch.query)
    kw = dict(max_chunk_len=bound, out=out, trusted_metadata=True)
    want = batch.attend(**kw).clone()
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    batch.attend(workspace=space, **kw)
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before
    assert torch.equal(out, want)
    with pytest.raises(ValueError, match="workspace"):
        batch.attend(workspace=space[:-1], **kw)
