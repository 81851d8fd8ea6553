"""GPU tests of PagePool.compact over tables that hold pages whose count is zero."""

import pytest
import torch

import nvfp4_attn_kernel_b200._lib as L
from nvfp4_attn_kernel_b200.nvfp4_vllm.pages import PagePool

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("reserved", [0, 1])
@pytest.mark.parametrize("pages", [12, 2100])
@pytest.mark.parametrize("dead", ["below", "above"])
def test_an_unheld_page_is_taken_out_of_the_table(cuda_device, pages, dead, reserved):
    """Row 0's second entry names a page that nobody holds: a hole that another row's page moves into, or one past the
    live pages.  It becomes -1 and is flagged, so that no row reads what is not its own; everything else moves as it
    would."""
    high = pages - 1
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[[3, 4, high, high - 2]] = torch.tensor([1, 2, 1, 3], dtype=torch.int32)
    free = 2 if dead == "below" else high - 1
    table = torch.tensor([[3, free, 4], [high, 4, high - 2], [-7, -7, -7]], dtype=torch.int32)
    held = torch.tensor([3, 3, 0], dtype=torch.int32)
    blocks = [torch.arange(pages, dtype=torch.int32)[:, None].repeat(1, 4).view(torch.uint8).to(cuda_device)]
    pool = PagePool(blocks, refs=refs.to(cuda_device), reserved_pages=reserved)
    table_d = table.to(cuda_device)
    live = int(pool.compact(table_d, held.to(cuda_device)))
    alive = (refs > 0) | (torch.arange(pages) < reserved)
    assert live == int(alive.sum()) and int(pool.status) == L.STATUS_BAD_PAGE_ID
    holes = [p for p in range(live) if not alive[p]]
    movers = [p for p in range(live, pages) if alive[p]]
    new = {p: p for p in range(live) if alive[p]} | dict(zip(movers, holes))
    assert table_d.tolist() == [[new[3], -1, new[4]], [new[high], new[4], new[high - 2]], [-7, -7, -7]]
    content = blocks[0].view(torch.int32)[:, 0].tolist()
    assert all(content[to] == of for of, to in new.items())
    assert [int(pool.refs[to]) for to in new.values()] == [int(refs[of]) for of in new] and int(pool.refs.sum()) == 7
    # again: the -1 is flagged as any id outside the cache
    pool.status.zero_()
    before = table_d.clone()
    assert int(pool.compact(table_d, held.to(cuda_device))) == live
    assert torch.equal(table_d, before) and int(pool.status) == L.STATUS_BAD_PAGE_ID
