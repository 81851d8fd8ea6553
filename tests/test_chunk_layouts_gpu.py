"""GPU tests of the chunk attention over layouts and batches that a server has: queries whose heads lie apart, page tables
far wider than any row, one-token rows with a long history beside a prompt's chunk."""

import numpy as np
import pytest
import torch

from chunk_cases import ChunkBatch
from test_chunk_gpu import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [[(2, 30, 40), (0, 0, 1)], [(1, 0, 200), (3, 128, 5)], [(0, 9, 3)]])
@pytest.mark.parametrize("layout", ["padded", "heads first", "every other token"])
def test_query_heads_apart(cuda_device, rows, layout):
    batch = ChunkBatch(rows, 8, 2, cuda_device, seed=70, shift=True, pad=2)
    dense = batch.query
    if layout == "padded":                 # 72 more channels after each head
        store = torch.full((batch.tokens, 8, 200), float("nan"), dtype=torch.bfloat16, device=cuda_device)
        batch.query = store[:, :, :128]
    elif layout == "heads first":          # [heads, tokens, 128]
        store = torch.full((8, batch.tokens + 1, 128), float("nan"), dtype=torch.bfloat16, device=cuda_device)
        batch.query = store[:, 1:].transpose(0, 1)
    else:                                  # every other token, heads far apart
        store = torch.full((8, 2 * batch.tokens, 128), float("nan"), dtype=torch.bfloat16, device=cuda_device)
        batch.query = store.transpose(0, 1)[1::2]
    batch.query.copy_(dense)
    assert batch.query.stride(1) != 128
    got = batch.attend()
    check(batch, got)
    live = int(batch.starts_host[-1])
    batch.query = dense
    assert torch.equal(got[:live], batch.attend()[:live])


def widen(batch, columns):
    """The same table in one of `columns` columns; what lies behind the rows' own is out of range."""
    table = torch.full((len(batch.rows), columns), -(1 << 31), dtype=torch.int32, device=batch.device)
    table[:, :batch.columns] = batch.table
    batch.table = table


@pytest.mark.parametrize("rows", [[(5, 30, 512)], [(16, 0, 4), (3, 77, 4), (0, 0, 1), (12, 128, 2)], [(2, 0, 256)] * 8])
def test_a_table_far_wider_than_its_rows(cuda_device, rows):
    """131072 tokens' worth of columns and the rule's own split count: more ranges than tiles, most of them empty."""
    batch = ChunkBatch(rows, 8, 2, cuda_device, seed=71, pad=1)
    lse = torch.full((batch.tokens, 8), 3.0, device=cuda_device)
    widen(batch, 1024)
    out = torch.full((batch.tokens, 8, 128), 3.0, dtype=torch.bfloat16, device=cuda_device)
    check(batch, batch.attend(lse=lse, out=out), lse)
    assert (out[-1] == 3.0).all() and (lse[-1] == 3.0).all()
    full, rest = batch.append()
    assert full.tolist() == [(f + (t + n) // 128) * 128 for f, t, n in rows]
    assert rest.tolist() == [(t + n) % 128 for _, t, n in rows]


@pytest.mark.parametrize("heads", [(8, 2), (5, 1)])
@pytest.mark.parametrize("splits", [None, 1, 6])
def test_one_token_rows_beside_a_prompts_chunk(cuda_device, heads, splits):
    rows = [(100, 60, 1), (3, 10, 400), (130, 0, 1), (0, 127, 1), (77, 128, 1), (4, 0, 0), (31, 1, 2)]
    batch = ChunkBatch(rows, *heads, cuda_device, seed=72, shift=True)
    lse = torch.empty(batch.tokens, heads[0], device=cuda_device)
    got = batch.attend(num_splits=splits, lse=lse)
    check(batch, got, lse)
    # and each row by itself, through the form for short chunks: within the two bounds of one another
    bounds = [b for _, _, b, _ in batch.plain()]
    for r in (0, 2, 4):
        a, n = batch.starts_host[r], rows[r][2]
        one = ChunkBatch([rows[r]], *heads, cuda_device, seed=1)
        one.views, one.tail_key, one.tail_value, one.shift = batch.views, batch.tail_key, batch.tail_value, batch.shift
        one.table, one.ids = batch.table[r:r + 1], batch.ids[r:r + 1]
        one.query, one.key, one.value = (x[a:a + n] for x in (batch.query, batch.key, batch.value))
        alone = one.attend(num_splits=1)
        distance = np.abs((alone.float() - got[a:a + n].float()).cpu().numpy())
        assert (distance <= 2 * bounds[r]).all()
