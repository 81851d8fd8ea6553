"""GPU tests of append_kv_chunk on rows that it cannot write: nothing of such a row changes, whichever page is missing."""

import pytest
import torch

import nvfp4_attn_kernel_b200._lib as L
from chunk_cases import ChunkBatch

pytestmark = pytest.mark.gpu

# row 0 has 100 tail tokens and three pages to seal, row 1 seals one, row 2 none
ROWS = [(1, 100, 300), (0, 20, 130), (2, 5, 6)]


@pytest.mark.parametrize("heads_kv", [1, 8])
@pytest.mark.parametrize("column,page", [(1, -1), (2, -5), (3, None), (3, 1 << 30), (1, -(1 << 31))])
def test_a_missing_page_keeps_the_whole_row(cuda_device, heads_kv, column, page):
    """An id below zero or past the cache, in the first, the second or the last column that the row would write: its pages,
    both tails and its lengths stay, the status bit is set, and the other rows are written as without it."""
    batch = ChunkBatch(ROWS, heads_kv, heads_kv, cuda_device, seed=40)
    whole = ChunkBatch(ROWS, heads_kv, heads_kv, cuda_device, seed=40)
    whole.append()
    before = [x.clone() for x in (batch.cache, batch.tail_key, batch.tail_value)]
    batch.table[0, column] = batch.cache.shape[0] if page is None else page
    with pytest.raises(ValueError, match="page id outside"):
        batch.append()
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    full, rest = batch.append(status=status, trusted_metadata=True)
    assert int(status) == L.STATUS_BAD_PAGE_ID
    assert full.tolist() == [128, 128, 256] and rest.tolist() == [100, 22, 11]
    mine, slot = batch.table_host[0, 1:4].long().to(cuda_device), int(batch.ids_host[0])
    want = [x.clone() for x in (whole.cache, whole.tail_key, whole.tail_value)]
    want[0][mine] = before[0][mine]
    for x, old in zip(want[1:], before[1:]):
        x[slot] = old[slot]
    assert torch.equal(batch.cache, want[0])
    assert torch.equal(batch.tail_key.view(torch.int16), want[1].view(torch.int16))
    assert torch.equal(batch.tail_value.view(torch.int16), want[2].view(torch.int16))
    # the page entered, the same call goes through
    batch.table[0, column] = batch.table_host[0, column]
    status.zero_()
    one = torch.tensor([0, 300, 300, 300], dtype=torch.int32, device=cuda_device)
    batch.starts, batch.seqused_fp4, batch.seqused_tail = one, full, rest
    full, rest = batch.append(status=status)
    assert int(status) == 0 and full.tolist() == [512, 128, 256] and rest.tolist() == [16, 22, 11]
    assert torch.equal(batch.cache, whole.cache)


@pytest.mark.parametrize("column", [0, 255, 256, 257])
def test_a_missing_page_among_more_than_a_block_has_threads(cuda_device, column):
    """258 pages of one chunk: the one that is missing may be any thread's first or second."""
    rows = [(0, 24, 33000), (1, 0, 5)]
    batch = ChunkBatch(rows, 1, 1, cuda_device, seed=43)
    before = [x.clone() for x in (batch.cache, batch.tail_key, batch.tail_value)]
    batch.table[0, column] = -1
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    full, rest = batch.append(status=status, trusted_metadata=True)
    assert int(status) == L.STATUS_BAD_PAGE_ID and full.tolist() == [0, 128] and rest.tolist() == [24, 5]
    assert torch.equal(batch.cache, before[0])
    slot = int(batch.ids_host[0])
    for now, old in zip((batch.tail_key, batch.tail_value), before[1:]):
        assert torch.equal(now[slot].view(torch.int16), old[slot].view(torch.int16))
    batch.table[0, column] = batch.table_host[0, column]
    full, rest = batch.append()
    assert full.tolist() == [258 * 128, 128] and rest.tolist() == [0, 5]
