"""GPU tests of the page pool against plain Python."""

import numpy as np
import pytest
import torch

import nvfp4_attn_kernel_b200._lib as L
from nvfp4_attn_kernel_b200.nvfp4_vllm.pages import PagePool

pytestmark = pytest.mark.gpu


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def build(device, pages=40, block=48, layers=3, rows=6, columns=7, slots=8, heads=1, seed=0, reserved=1, tails=True):
    rng = np.random.default_rng(seed)
    blocks = [torch.from_numpy(rng.integers(0, 256, (pages, block), dtype=np.uint8)).to(device) for _ in range(layers)]
    free = list(rng.permutation(np.arange(reserved, pages)))
    table, held, refs = np.full((rows, columns), -1, np.int32), [], np.zeros(pages, np.int32)
    for r in range(rows):
        n = int(rng.integers(0, min(columns, len(free)) + 1))
        for c in range(n):
            table[r, c] = free.pop()
            refs[table[r, c]] = 1
        held.append(n)
    tail = [torch.from_numpy(rng.standard_normal((layers, slots, 128, heads, 128), dtype=np.float32)).to(torch.bfloat16).to(device)
            for _ in range(2)] if tails else [None, None]
    pool = PagePool(blocks, refs=ints(refs, device), tail_key=tail[0], tail_value=tail[1], reserved_pages=reserved)
    return pool, ints(table, device), ints(held, device), table, held, refs


def test_release_counts_down_and_lists_free_pages(cuda_device):
    pool, table, held, t, h, refs = build(cuda_device, seed=1)
    ids, count = pool.free_list()
    want = [p for p in range(1, 40) if refs[p] == 0]
    assert ids.tolist() == want + [-1] * (40 - len(want)) and int(count) == len(want)
    pool.release(ints([4, 1], cuda_device), table, held)
    for r in (4, 1):
        refs[t[r, :h[r]]] -= 1
        h[r] = 0
    assert pool.refs.tolist() == refs.tolist() and held.tolist() == h and int(pool.status) == 0
    # the same row twice, a row that does not exist, a row that holds nothing any more
    pool.release(ints([2, 2, 99, -1, 4], cuda_device), table, held)
    refs[t[2, :h[2]]] -= 1
    assert pool.refs.tolist() == refs.tolist() and int(pool.status) == L.STATUS_BAD_ROW
    # a page that nobody holds is not counted below zero
    pool.status.zero_()
    held[2] = max(1, h[2])
    table[2, 0] = pool.free_list()[0][0]
    before = pool.refs.clone()
    pool.release(ints([2], cuda_device), table, held)
    assert int(pool.refs.min()) == 0 and int(pool.status) == L.STATUS_BAD_PAGE_ID and int(before.min()) == 0
    pool.release(ints([], cuda_device), table, held)


@pytest.mark.parametrize("heads,seed", [(1, 2), (2, 3), (8, 4)])
def test_fork_shares_pages_and_copies_tails(cuda_device, heads, seed):
    pool, table, held, t, h, refs = build(cuda_device, pages=60, rows=9, slots=12, heads=heads, seed=seed)
    rng = np.random.default_rng(seed)
    slots = rng.permutation(12)[:9]
    # row 0 holds a block for its open page beyond the sealed ones
    fp4 = [max(0, n - (r == 0)) * 128 for r, n in enumerate(h)]
    used = [int(x) for x in rng.choice([0, 1, 77, 127, 128], 9)]
    used[0], used[3] = 128, 1
    targets, sources = [7, 2, 5], [0, 0, 3]
    pool.release(ints(targets, cuda_device), table, held)
    for r in targets:
        refs[t[r, :h[r]]] -= 1
    tails = [pool.tail_key.clone(), pool.tail_value.clone()]
    full_d, used_d = ints(fp4, cuda_device), ints(used, cuda_device)
    pool.fork(ints(sources, cuda_device), ints(targets, cuda_device), table, held, full_d, used_d, ints(slots, cuda_device))
    for s, d in zip(sources, targets):
        n = fp4[s] // 128
        t[d, :n] = t[s, :n]
        np.add.at(refs, t[s, :n], 1)
        h[d], fp4[d], used[d] = n, fp4[s], used[s]
        for x in tails:
            x[:, slots[d], :used[s]] = x[:, slots[s], :used[s]]
    assert table.tolist() == t.tolist() and held.tolist() == h and pool.refs.tolist() == refs.tolist()
    assert full_d.tolist() == fp4 and used_d.tolist() == used
    assert torch.equal(pool.tail_key, tails[0]) and torch.equal(pool.tail_value, tails[1]) and int(pool.status) == 0
    # a source whose sealed pages are more than it holds shares what it holds, and is flagged
    pool.release(ints([5], cuda_device), table, held)
    full_d[8] = (h[8] + 2) * 128
    pool.fork(ints([8], cuda_device), ints([5], cuda_device), table, held, full_d, used_d, ints(slots, cuda_device))
    assert int(pool.status) == L.STATUS_BAD_LENGTH and int(held[5]) == h[8] and int(full_d[5]) == h[8] * 128
    pool.status.zero_()
    # pairs that would depend on an order are skipped and flagged: a target twice, a target that is a source
    before = (table.clone(), pool.refs.clone(), pool.tail_key.clone())
    pool.fork(ints([0, 5, 99], cuda_device), ints([5, 5, 1], cuda_device), table, held, full_d, used_d, ints(slots, cuda_device))
    assert int(pool.status) == L.STATUS_BAD_ROW
    assert torch.equal(table, before[0]) and torch.equal(pool.refs, before[1]) and torch.equal(pool.tail_key, before[2])


@pytest.mark.parametrize("pages,live,seed", [(40, 20, 0), (1, 0, 1), (1, 1, 2), (2500, 1200, 3), (1024, 1023, 4), (1025, 1, 5),
                                             (64, 64, 6), (64, 0, 7)])
@pytest.mark.parametrize("reserved", [0, 1])
def test_compaction(cuda_device, pages, live, seed, reserved):
    rng = np.random.default_rng(seed)
    layers, rows, columns, block = 2, 5, 2 * live // 5 + 9, 16 * 1100 if pages < 100 else 16
    blocks = [torch.from_numpy(rng.integers(0, 256, (pages, block), dtype=np.uint8)).to(cuda_device) for _ in range(layers)]
    chosen = rng.permutation(np.arange(reserved, pages))[:live]
    refs, table, held = np.zeros(pages, np.int32), np.full((rows, columns), 1 << 29, np.int32), []
    for r in range(rows):
        mine = list(chosen[r::rows]) + (list(chosen[:min(3, live)]) if r == 4 else [])   # row 4 shares
        table[r, :len(mine)] = mine
        np.add.at(refs, np.array(mine, dtype=int), 1)
        held.append(len(mine))
    before = [b.cpu().numpy() for b in blocks]
    pool = PagePool(blocks, refs=ints(refs, cuda_device), reserved_pages=reserved)
    table_d = ints(table, cuda_device)
    count = int(pool.compact(table_d, ints(held, cuda_device)))
    alive = (refs > 0) | (np.arange(pages) < reserved)
    assert count == alive.sum()
    holes = [p for p in range(count) if not alive[p]]
    movers = [p for p in range(count, pages) if alive[p]]
    new = np.arange(pages)
    new[movers] = holes
    want_refs = np.zeros(pages, np.int32)
    want_refs[new[refs > 0]] = refs[refs > 0]
    assert pool.refs.tolist() == want_refs.tolist()
    for r in range(rows):
        table[r, :held[r]] = new[table[r, :held[r]]]
    assert table_d.tolist() == table.tolist()
    for b, old in zip(blocks, before):
        want = old.copy()
        want[holes] = old[movers]
        assert np.array_equal(b.cpu().numpy(), want)
    assert int(pool.status) == 0
    again = [b.clone() for b in blocks]
    assert int(pool.compact(table_d, ints(held, cuda_device))) == count       # nothing left to move
    assert all(torch.equal(a, b) for a, b in zip(again, blocks))


def test_copy_pages(cuda_device):
    pool, *_ = build(cuda_device, pages=30, block=16 * 1025, layers=3, rows=2, tails=False)
    before = [b.clone() for b in pool.blocks]
    pool.copy(ints([3, -1, 7, 3], cuda_device), ints([9, 4, 11, 29], cuda_device))
    for old, b in zip(before, pool.blocks):
        old[[9, 11, 29]] = old[[3, 7, 3]]
        assert torch.equal(old, b)
    with pytest.raises(ValueError, match="copied to once"):
        pool.copy(ints([1, 2], cuda_device), ints([3, 3], cuda_device))
    with pytest.raises(ValueError, match="copied to once"):
        pool.copy(ints([1, 3], cuda_device), ints([3, 4], cuda_device))
    with pytest.raises(ValueError, match="below 30"):
        pool.copy(ints([1], cuda_device), ints([30], cuda_device))
    pool.copy(ints([1], cuda_device), ints([30], cuda_device), trusted_metadata=True)      # flagged, nothing written
    assert int(pool.status) == L.STATUS_BAD_PAGE_ID
    assert all(torch.equal(old, b) for old, b in zip(before, pool.blocks))


def test_pool_refusals(cuda_device):
    pool, table, held, *_ = build(cuda_device)
    with pytest.raises(ValueError, match="same length"):
        pool.copy(ints([1], cuda_device), ints([2, 3], cuda_device))
    with pytest.raises(ValueError, match="row_to_slot"):
        pool.fork(ints([1], cuda_device), ints([2], cuda_device), table, held, held, held)
    with pytest.raises(ValueError, match="rows must"):
        pool.release(torch.zeros(1, dtype=torch.int64, device=cuda_device), table, held)
    with pytest.raises(ValueError, match="pages_held"):
        pool.release(ints([1], cuda_device), table, held[:2])
    with pytest.raises(ValueError, match="one shape"):
        PagePool([pool.blocks[0], pool.blocks[0][:5]])
    with pytest.raises(ValueError, match="multiple of 16"):
        PagePool([torch.zeros(3, 40, dtype=torch.uint8, device=cuda_device)])
    with pytest.raises(ValueError, match="at least one"):
        PagePool([])
    with pytest.raises(ValueError, match="go together"):
        PagePool(pool.blocks, tail_key=pool.tail_key)
    with pytest.raises(ValueError, match="refs"):
        PagePool(pool.blocks, refs=torch.zeros(3, dtype=torch.int32, device=cuda_device))


def test_fork_in_a_graph_and_on_another_stream(cuda_device):
    pool, table, held, t, h, refs = build(cuda_device, pages=60, rows=9, slots=12, seed=8)
    slots = ints(list(range(9)), cuda_device)
    fp4 = ints([n * 128 for n in h], cuda_device)
    used = ints([5] * 9, cuda_device)
    source, target = ints([0], cuda_device), ints([1], cuda_device)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        pool.release(target, table, held)
        pool.fork(source, target, table, held, fp4, used, slots)
    for s, d in ((0, 1), (3, 4), (0, 4)):
        source.fill_(s)
        target.fill_(d)
        graph.replay()
        torch.cuda.synchronize()
        refs[t[d, :h[d]]] -= 1
        t[d, :h[s]] = t[s, :h[s]]
        refs[t[s, :h[s]]] += 1
        h[d] = h[s]
        assert pool.refs.tolist() == refs.tolist() and held.tolist() == h
        assert torch.equal(pool.tail_key[:, d, :5], pool.tail_key[:, s, :5])
    assert int(pool.status) == 0
