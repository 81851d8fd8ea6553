"""GPU tests of append_kv_chunk's checked form on page tables whose new columns name sealed history."""

import pytest
import torch

from chunk_cases import ChunkBatch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("row,column", [(0, 0), (1, 0), (2, 1)])
def test_history_is_not_written_over(cuda_device, row, column):
    """The page that row 0 would seal next is one of its own, of a row with a chunk of its own, of a row without one."""
    batch = ChunkBatch([(1, 100, 60), (2, 7, 9), (2, 3, 0)], 2, 2, cuda_device, seed=41)
    batch.table[0, 1] = batch.table_host[row, column]
    before = batch.cache.clone(), batch.tail_key.clone()
    with pytest.raises(ValueError, match="are history"):
        batch.append()
    assert torch.equal(batch.cache, before[0]) and torch.equal(batch.tail_key.view(torch.int16), before[1].view(torch.int16))


def test_rows_that_share_their_history_append_beside_it(cuda_device):
    """Forked rows: the same sealed pages, new pages of their own; a column behind a row's last page may hold anything."""
    batch = ChunkBatch([(1, 100, 60), (1, 100, 60), (0, 5, 6)], 2, 2, cuda_device, seed=42)
    batch.table[1, 0] = batch.table_host[0, 0]
    batch.table[2, 0] = batch.table_host[0, 0]
    full, rest = batch.append()
    assert full.tolist() == [256, 256, 0] and rest.tolist() == [32, 32, 11]
