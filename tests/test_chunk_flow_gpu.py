"""GPU tests of the chunk operators and the page pool together, as a server would run them."""

import numpy as np
import pytest
import torch

from chunk_cases import PAGE, ChunkBatch
from helpers import to_np
from nvfp4_attn_kernel_b200.nvfp4_decode_kernel import append_kv_chunk, fp4_chunk_attention
from nvfp4_attn_kernel_b200.nvfp4_vllm import layout
from nvfp4_attn_kernel_b200.nvfp4_vllm.runtime import LayerRuntime

pytestmark = pytest.mark.gpu


class Server:
    """Two layers over one page pool; rows are continued by chunks, forked and released."""

    def __init__(self, device, layers=2, rows=5, heads_q=8, heads_kv=2, pages=40, columns=8, seed=0):
        self.device, self.layers, self.rows, self.heads_q, self.heads_kv = device, layers, rows, heads_q, heads_kv
        self.gen = torch.Generator().manual_seed(seed)
        self.runtime = LayerRuntime(num_layers=layers, num_slots=rows, num_heads=heads_q, num_kv_heads=heads_kv,
                                    head_dim=128, device=device)
        self.caches = [torch.full((pages, layout.page_bytes(heads_kv)), 255, dtype=torch.uint8, device=device)
                       for _ in range(layers)]
        self.pool = self.runtime.page_pool(self.caches)
        self.table = torch.full((rows, columns), -1, dtype=torch.int32, device=device)
        self.held, self.full, self.used = (torch.zeros(rows, dtype=torch.int32, device=device) for _ in range(3))
        self.slots = torch.randperm(rows, generator=self.gen).int().to(device)

    def take(self, row, count):
        """Give ``row`` that many free pages (the host's part: here it reads the list back)."""
        ids, free = self.pool.free_list()
        assert int(free) >= count
        held = int(self.held[row])
        self.table[row, held:held + count] = ids[:count]
        self.pool.refs[ids[:count].long()] += 1
        self.held[row] += count

    def step(self, lengths, draw=None):
        """Continue every row by ``lengths[row]`` random tokens; returns each layer's outputs."""
        lengths = list(lengths)
        for r, n in enumerate(lengths):
            grown = (int(self.full[r]) + int(self.used[r]) + n) // PAGE - int(self.held[r])
            if n and grown > 0:
                self.take(r, grown)
        starts = torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device=self.device)
        outputs = []
        for layer in range(self.layers):
            if draw is None:
                x = [torch.randn(sum(lengths), h, 128, generator=self.gen).to(torch.bfloat16).to(self.device)
                     for h in (self.heads_q, self.heads_kv, self.heads_kv)]
            else:
                x = draw[layer]
            views = layout.carve(self.caches[layer], self.heads_kv, 128)
            kw = dict(max_chunk_len=max(lengths), residual_key_pages_bf16=self.runtime.tail_key[layer],
                      residual_value_pages_bf16=self.runtime.tail_value[layer], residual_page_ids=self.slots,
                      seqused_residual=self.used)
            outputs.append((x, fp4_chunk_attention(*x, *views, self.table, self.full, starts, **kw)))
            full, used = append_kv_chunk(*x[1:], *views, self.table, self.full, starts, **kw)
        self.full, self.used = full, used
        return outputs


def test_prefix_shared_by_forks_then_released_and_compacted(cuda_device):
    server = Server(cuda_device)
    pool = server.pool
    server.step([300, 0, 0, 0, 700])                      # two prompts
    server.step([33, 0, 0, 0, 1])
    assert server.full.tolist() == [256, 0, 0, 0, 640] and server.used.tolist() == [77, 0, 0, 0, 61]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_device)   # noqa: E731
    pool.fork(ints([0, 0, 4]), ints([1, 3, 2]), server.table, server.held, server.full, server.used, server.slots)
    assert server.held.tolist() == [2, 2, 5, 2, 5]
    shared = server.table[0, :2].long()
    assert pool.refs[shared].tolist() == [3, 3] and pool.refs[server.table[4, :5].long()].tolist() == [2] * 5
    # the forks and their sources get the same tokens: the same outputs, bit for bit (same lengths, same walk)
    n = 60
    same = []
    for _ in range(server.layers):
        per_head = lambda h: torch.randn(1, n, h, 128, generator=server.gen).to(torch.bfloat16).to(cuda_device)   # noqa: E731
        same.append([x.expand(5, -1, -1, -1).reshape(5 * n, x.shape[2], 128).contiguous()
                     for x in (per_head(8), per_head(2), per_head(2))])
    outputs = server.step([n] * 5, draw=same)
    for _, out in outputs:
        parts = out.view(5, n, 8, 128)
        assert torch.equal(parts[0], parts[1]) and torch.equal(parts[0], parts[3])
        assert torch.equal(parts[4], parts[2]) and not torch.equal(parts[0], parts[4])
    # (each has sealed a page of its own by now)
    assert len({int(server.table[r, 2]) for r in (0, 1, 3)}) == 3
    # release two rows, pack the pool: what the others attend to does not change by a bit
    pool.release(ints([0, 2]), server.table, server.held)
    server.full[[0, 2]] = 0
    server.used[[0, 2]] = 0
    probe = [[torch.randn(9, h, 128, generator=server.gen).to(torch.bfloat16).to(cuda_device) for h in (8, 2, 2)]
             for _ in range(server.layers)]

    def look():
        found = []
        for layer in range(server.layers):
            views = layout.carve(server.caches[layer], 2, 128)
            found.append(fp4_chunk_attention(
                *probe[layer], *views, server.table, server.full, ints([0, 0, 3, 3, 6, 9]), max_chunk_len=3,
                residual_key_pages_bf16=server.runtime.tail_key[layer],
                residual_value_pages_bf16=server.runtime.tail_value[layer], residual_page_ids=server.slots,
                seqused_residual=server.used))
        return found

    before, table = look(), server.table.clone()
    live = int(pool.compact(server.table, server.held))
    held = [server.table[r, :int(server.held[r])] for r in range(5)]
    assert live == 1 + len(torch.cat(held).unique()) and int(torch.cat(held).max()) < live
    assert not torch.equal(table, server.table)
    assert all(torch.equal(a, b) for a, b in zip(before, look()))
    assert int(pool.refs[live:].abs().sum()) == 0 and int(pool.status) == 0
    # and they go on
    server.step([0, 100, 0, 5, 128])
    assert int(pool.status) == 0


def test_two_streams_and_graphs_at_once(cuda_device):
    """Different batches on two streams at the same time, eager beside a replayed graph: each as alone."""
    a = ChunkBatch([(9, 40, 300), (2, 0, 70)], 8, 2, cuda_device, seed=31)
    b = ChunkBatch([(30, 5, 4), (3, 128, 2)], 16, 2, cuda_device, seed=32, shift=True)
    alone = [a.attend(trusted_metadata=True).clone(), b.attend(trusted_metadata=True, num_splits=5).clone()]
    out = torch.empty_like(alone[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.attend(trusted_metadata=True, num_splits=5, out=out)
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        with torch.cuda.stream(one):
            got.append(a.attend(trusted_metadata=True))
        with torch.cuda.stream(two):
            graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(g, alone[0]) for g in got)
    assert torch.equal(out, alone[1])


def test_long_cache_and_a_wide_batch(cuda_device):
    """Page addresses past 2^31 bytes, and more rows and tokens than one wave of CTAs."""
    from nvfp4_attn_kernel_b200.nvfp4_decode_kernel import _quantize

    heads, pages = 8, 20000                                # 20000 blocks of 147456 bytes: 2.9 GB
    cache = torch.zeros(pages, layout.page_bytes(heads), dtype=torch.uint8, device=cuda_device)
    views = layout.carve(cache, heads, 128)
    g = torch.Generator(device=cuda_device).manual_seed(1)
    used = torch.tensor([19999, 3, 15001, 7777], device=cuda_device)
    k, v = (torch.randn(4, PAGE, heads, 128, generator=g, device=cuda_device).to(torch.bfloat16) for _ in range(2))
    for view, new in zip(views, (*_quantize.quantize_key_pages(k), *_quantize.quantize_value_pages(v))):
        view.view(torch.uint8)[used] = new.view(torch.uint8)
    rows, n = 300, 3
    table = used.int()[torch.randint(0, 4, (rows, 4), generator=g, device=cuda_device)].contiguous()
    length = torch.randint(0, 5, (rows,), generator=g, device=cuda_device).int() * PAGE
    q, key, value = (torch.randn(rows * n, h, 128, generator=g, device=cuda_device).to(torch.bfloat16) for h in (16, heads, heads))
    starts = torch.arange(rows + 1, device=cuda_device).int() * n
    out = fp4_chunk_attention(q, key, value, *views, table, length, starts, max_chunk_len=n)
    # rows that walk the same pages in the same order through small copies of them
    small = torch.zeros(4, layout.page_bytes(heads), dtype=torch.uint8, device=cuda_device)
    small.copy_(cache[used])
    place = {int(p): i for i, p in enumerate(used)}
    table_small = torch.tensor([[place[p] for p in row] for row in table.tolist()], dtype=torch.int32, device=cuda_device)
    again = fp4_chunk_attention(q, key, value, *layout.carve(small, heads, 128), table_small, length, starts, max_chunk_len=n)
    assert torch.equal(out, again)
    want = torch.softmax(torch.tensor([0.0]), 0)           # one row by hand: token 0 of a row without history is its value
    first = int((length == 0).nonzero()[0])
    assert float(want) == 1.0 and torch.equal(out[first * n].view(heads, 2, 128)[:, 0], value[first * n])


@pytest.mark.parametrize("tokens,rows", [(0, 0), (0, 3), (5, 0)])
def test_nothing_to_do(cuda_device, tokens, rows):
    cache = torch.zeros(2, layout.page_bytes(2), dtype=torch.uint8, device=cuda_device)
    views = layout.carve(cache, 2, 128)
    x = [torch.zeros(tokens, h, 128, dtype=torch.bfloat16, device=cuda_device) for h in (4, 2, 2)]
    table = torch.zeros(rows, 1, dtype=torch.int32, device=cuda_device)
    zeros = torch.zeros(rows, dtype=torch.int32, device=cuda_device)
    starts = torch.zeros(rows + 1, dtype=torch.int32, device=cuda_device)
    out = torch.full((tokens, 4, 128), 2.0, dtype=torch.bfloat16, device=cuda_device)
    fp4_chunk_attention(*x, *views, table, zeros, starts, max_chunk_len=0, out=out)
    assert (out == 2.0).all()
    tail = torch.zeros(1, PAGE, 2, 128, dtype=torch.bfloat16, device=cuda_device)
    full, rest = append_kv_chunk(*x[1:], *views, table, zeros, starts, max_chunk_len=0, residual_key_pages_bf16=tail,
                                 residual_value_pages_bf16=tail.clone(), residual_page_ids=zeros, seqused_residual=zeros)
    assert full.tolist() == [0] * rows and rest.tolist() == [0] * rows
    assert (cache == 0).all()
