"""GPU tests of PagePool.fork in a row of calls that depend on one another, over many pairs and long rows, and without tails."""

import numpy as np
import pytest
import torch

import nvfp4_attn_kernel_b200._lib as L
from nvfp4_attn_kernel_b200.nvfp4_vllm.pages import PagePool

pytestmark = pytest.mark.gpu


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


@pytest.mark.parametrize("captured", [False, True])
def test_forks_of_forks_in_one_stream(cuda_device, captured):
    """0 to 1, 1 to 2, ... with nothing in between, then 1 released and made again from the last: the calls' launches may
    overlap, their effects may not."""
    rows, layers, heads = 12, 8, 4
    g = torch.Generator().manual_seed(3)
    tails = [torch.randn(layers, rows, 128, heads, 128, generator=g).to(torch.bfloat16).to(cuda_device) for _ in range(2)]
    table = torch.full((rows, 4), -1, dtype=torch.int32, device=cuda_device)
    table[0] = ints([5, 1, 7, 3], cuda_device)
    refs = torch.zeros(9, dtype=torch.int32, device=cuda_device)
    refs[table[0].long()] = 1
    held, full, used = (ints([x] + [0] * (rows - 1), cuda_device) for x in (4, 512, 113))
    slots = torch.randperm(rows, generator=g).int().to(cuda_device)
    pool = PagePool([torch.zeros(9, 32, dtype=torch.uint8, device=cuda_device)], refs=refs, tail_key=tails[0], tail_value=tails[1])
    names = [ints([r], cuda_device) for r in range(rows)]
    want = [t[:, int(slots[0]), :113].clone() for t in tails]

    def steps():
        for r in range(rows - 1):
            pool.fork(names[r], names[r + 1], table, held, full, used, slots)
        pool.release(names[1], table, held)
        pool.fork(names[rows - 1], names[1], table, held, full, used, slots)

    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            steps()
        graph.replay()
    else:
        steps()
    torch.cuda.synchronize()
    assert int(pool.status) == 0 and held.tolist() == [4] * rows and full.tolist() == [512] * rows and used.tolist() == [113] * rows
    assert table.tolist() == [[5, 1, 7, 3]] * rows and refs[table[0].long()].tolist() == [rows] * 4 and int(refs.sum()) == 4 * rows
    for t, first in zip(tails, want):
        assert all(torch.equal(t[:, s, :113], first) for s in range(rows))


@pytest.mark.parametrize("tails", [True, False])
def test_many_pairs_and_long_rows(cuda_device, tails):
    """More pairs, and more pages a row, than a block has threads; every seventh pair names a page outside the cache last."""
    pairs, columns, pages = 300, 610, 5000
    rows = 20 + pairs
    rng = np.random.default_rng(5)
    table = np.full((rows, columns), -1, np.int32)
    held, used = np.zeros(rows, np.int32), np.zeros(rows, np.int32)
    held[:20], used[:20] = rng.integers(1, columns + 1, 20), rng.integers(0, 129, 20)
    held[3], used[3] = columns, 128
    for r in range(20):
        table[r, :held[r]] = rng.integers(0, pages, held[r])
    bad = [3, 9]
    for r in bad:
        table[r, held[r] - 1] = pages if r == 3 else -3
    refs = np.zeros(pages, np.int32)
    for r in range(20):
        ok = table[r, :held[r]]
        np.add.at(refs, ok[(ok >= 0) & (ok < pages)], 1)
    sources = rng.integers(0, 20, pairs)
    sources[::7] = np.where(np.arange(len(sources[::7])) % 2, 3, 9)
    targets = 20 + rng.permutation(pairs)
    tail = [torch.randn(1, rows, 128, 1, 128).to(torch.bfloat16).to(cuda_device) for _ in range(2)] if tails else [None, None]
    pool = PagePool([torch.zeros(pages, 16, dtype=torch.uint8, device=cuda_device)], refs=ints(refs, cuda_device), tail_key=tail[0],
                    tail_value=tail[1])
    before = [x.clone() for x in tail] if tails else []
    table_d, held_d, used_d = ints(table, cuda_device), ints(held, cuda_device), ints(used, cuda_device)
    full_d = ints(held * 128, cuda_device)
    slots = rng.permutation(rows).astype(np.int32)
    pool.fork(ints(sources, cuda_device), ints(targets, cuda_device), table_d, held_d, full_d, used_d,
              ints(slots, cuda_device) if tails else None)
    for s, d in zip(sources, targets):
        if s in bad:
            continue
        table[d, :held[s]] = table[s, :held[s]]
        np.add.at(refs, table[s, :held[s]], 1)
        held[d], used[d] = held[s], used[s]
        for x in before:
            x[:, slots[d], :used[s]] = x[:, slots[s], :used[s]]
    assert int(pool.status) == L.STATUS_BAD_PAGE_ID
    assert np.array_equal(table_d.cpu().numpy(), table) and np.array_equal(pool.refs.cpu().numpy(), refs)
    assert held_d.tolist() == held.tolist() and used_d.tolist() == used.tolist() and full_d.tolist() == (held * 128).tolist()
    assert all(torch.equal(x, y) for x, y in zip(tail if tails else [], before))
