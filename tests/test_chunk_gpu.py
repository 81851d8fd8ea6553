"""GPU tests of the chunk operators against their plain form in 64 bits."""

import numpy as np
import pytest
import torch

import nvfp4_attn_kernel_b200._lib as L
import nvfp4_oracle as O
from chunk_cases import PAGE, ChunkBatch, blocks_of
from helpers import to_np

pytestmark = pytest.mark.gpu

# (full pages, tail tokens, chunk tokens) of every row
SINGLE = [(0, 0, 1)]
TINY = [(0, 0, 1), (1, 0, 1), (0, 1, 1), (2, 127, 3), (0, 128, 2), (3, 128, 0)]
EDGES = [(0, 0, 127), (1, 5, 128), (2, 64, 129), (0, 128, 131), (1, 0, 0), (0, 127, 1), (4, 1, 33)]
LONG = [(9, 77, 300), (0, 0, 517), (17, 0, 64), (3, 128, 5)]


def check(batch, out, lse=None):
    got = to_np(out).astype(np.float64)
    for r, (o, want_lse, bound, lse_bound) in enumerate(batch.plain()):
        a, n = batch.starts_host[r], batch.rows[r][2]
        error = np.abs(got[a:a + n] - o)
        assert np.isfinite(got[a:a + n]).all(), f"row {r}"
        assert (error <= bound).all(), f"row {r}: {(error / np.maximum(bound, 1e-30)).max():.2f} times the bound"
        if lse is not None and n:
            assert (np.abs(to_np(lse)[a:a + n] - want_lse) <= lse_bound).all(), f"row {r}"


@pytest.mark.parametrize("rows", [SINGLE, TINY, EDGES, LONG], ids=["single", "tiny", "edges", "long"])
@pytest.mark.parametrize("heads", [(8, 2), (4, 4), (10, 2)], ids=["4to1", "1to1", "5to1"])
def test_attention_matches_the_plain_form(cuda_device, rows, heads):
    batch = ChunkBatch(rows, *heads, cuda_device, seed=len(rows) + heads[0], shift=True, pad=3)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    out = torch.full((batch.tokens, heads[0], 128), 3.0, dtype=torch.bfloat16, device=cuda_device)
    lse = torch.full((batch.tokens, heads[0]), 3.0, device=cuda_device)
    result = batch.attend(out=out, lse=lse, status=status)
    assert result.data_ptr() == out.data_ptr()
    check(batch, out, lse)
    assert (out[-3:] == 3.0).all() and (lse[-3:] == 3.0).all()      # padding is left as it was
    assert int(status) == 0


@pytest.mark.parametrize("group", [2, 3, 6, 7, 8, 16, 32])
def test_attention_group_sizes(cuda_device, group):
    batch = ChunkBatch([(2, 30, 40), (0, 0, 9), (1, 128, 1)], group, 1, cuda_device, seed=group)
    check(batch, batch.attend())


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 40])
def test_attention_split_over_the_keys(cuda_device, splits):
    batch = ChunkBatch(LONG + [(0, 0, 1)], 8, 2, cuda_device, seed=11, shift=True, pad=2)
    out = torch.full((batch.tokens, 8, 128), 3.0, dtype=torch.bfloat16, device=cuda_device)
    lse = torch.full((batch.tokens, 8), 3.0, device=cuda_device)
    check(batch, batch.attend(out=out, lse=lse, num_splits=splits), lse)
    assert (out[-2:] == 3.0).all() and (lse[-2:] == 3.0).all()


@pytest.mark.parametrize("splits", [1, 2, 5])
@pytest.mark.parametrize("heads,lengths", [((8, 2), (15, 16, 17)), ((6, 2), (20, 21, 22)), ((8, 1), (7, 8, 9)),
                                           ((32, 1), (1, 2, 3)), ((4, 4), (63, 64, 65, 128))],
                         ids=["4to1", "3to1", "8to1", "32to1", "1to1"])
def test_attention_around_half_a_tile(cuda_device, heads, lengths, splits):
    """Just below, at and above 64 query rows of a KV head (up to there a tile holds each twice), over the chunk alone, a
    tail, pages, and both; split, the ranges are of one tile and less."""
    rows = [(f, t, n) for n in lengths for f, t in ((0, 0), (0, 5), (1, 0), (2, 128), (5, 9))]
    batch = ChunkBatch(rows, *heads, cuda_device, seed=31, shift=heads[1] == 2)
    lse = torch.empty(batch.tokens, heads[0], device=cuda_device)
    check(batch, batch.attend(num_splits=splits, lse=lse), lse)


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("chunk", [3, 70])
def test_attention_leaves_refused_pages_out(cuda_device, chunk, splits):
    """Ids outside the cache among 75 pages (the first, the last of 32, the first of the next 32, neighbours, the last):
    what a table without them gives, and a status bit."""
    batch = ChunkBatch([(75, 20, chunk), (40, 0, 1)], 8, 2, cuda_device, seed=32, shift=True)
    refused = [0, 31, 32, 40, 41, 42, 74]
    batch.table[0, refused] = torch.tensor([-1, 1 << 30, -5, 1 << 28, -1, batch.cache.shape[0], -1], dtype=torch.int32,
                                           device=cuda_device)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    out = batch.attend(num_splits=splits, status=status, trusted_metadata=True)
    assert int(status) == L.STATUS_BAD_PAGE_ID
    kept = [c for c in range(75) if c not in refused]
    batch.table_host[0, :len(kept)] = batch.table_host[0, kept].clone()
    batch.rows[0] = (len(kept), 20, chunk)
    check(batch, out)


def test_attention_of_strided_projections(cuda_device):
    batch = ChunkBatch(EDGES, 8, 2, cuda_device, seed=5, spread=True)
    wide = torch.zeros(batch.tokens, 8 * 128 + 256, dtype=torch.bfloat16, device=cuda_device)
    out = wide[:, :1024].unflatten(1, (8, 128))
    batch.attend(out=out)
    check(batch, out)
    assert (wide[:, 1024:] == 0).all()


def test_attention_without_a_tail_or_pages(cuda_device):
    batch = ChunkBatch([(0, 0, 200), (0, 0, 1)], 8, 2, cuda_device, seed=6)
    none = dict(residual_key_pages_bf16=None, residual_value_pages_bf16=None, residual_page_ids=None,
                seqused_residual=None)
    check(batch, batch.attend(**none))


@pytest.mark.parametrize("gain", [1e-3, 40.0, 3e4])
def test_attention_of_flat_and_peaked_scores(cuda_device, gain):
    batch = ChunkBatch([(3, 50, 140), (0, 128, 20)], 8, 2, cuda_device, seed=7, query_gain=gain)
    check(batch, batch.attend(num_splits=2))
    check(batch, batch.attend(num_splits=1))


def test_attention_of_infinite_and_tiny_queries(cuda_device):
    """A row whose query is not finite gives NaN in its own outputs and in no other's; a query of zeros averages."""
    batch = ChunkBatch([(1, 20, 6)], 4, 2, cuda_device, seed=8)
    batch.query[2, 1] = float("nan")
    batch.query[3, 0] = 0.0
    batch.query[4, 2] = 1e-30
    out = to_np(batch.attend())
    assert np.isnan(out[2, 1]).all()
    keep = np.ones(out.shape[:2], dtype=bool)
    keep[2, 1] = False
    assert np.isfinite(out[keep]).all()
    batch.query[2, 1] = 0.0
    want = batch.plain()[0]
    assert (np.abs(out - want[0])[keep] <= want[2][keep]).all()


def test_attention_is_deterministic_and_replayable(cuda_device):
    batch = ChunkBatch(EDGES, 8, 2, cuda_device, seed=9, shift=True)
    out = torch.empty(batch.tokens, 8, 128, dtype=torch.bfloat16, device=cuda_device)
    first = batch.attend(out=out, trusted_metadata=True, num_splits=3).clone()
    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        batch.attend(out=out, trusted_metadata=True, num_splits=3)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    # the lengths are read at replay: one row shorter, the padding behind it untouched
    cut = batch.starts.clone()
    cut[-1] -= 20
    batch.starts.copy_(cut)
    out.fill_(5.0)
    graph.replay()
    torch.cuda.synchronize()
    assert (out[-20:] == 5.0).all()
    # (a shorter row may be walked in another order, so its sums may round differently; the others have their bits)
    last = batch.starts_host[-2]
    assert torch.equal(out[:last], first[:last])
    batch.rows = batch.rows[:-1] + [(*batch.rows[-1][:2], batch.rows[-1][2] - 20)]
    check(batch, out)


def test_attention_flags_bad_metadata_and_stays_in_bounds(cuda_device):
    batch = ChunkBatch([(2, 10, 4), (1, 0, 3), (1, 3, 2)], 8, 2, cuda_device, seed=10)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    table = batch.table.clone()
    table[0, 1] = 1 << 30
    kw = dict(status=status, trusted_metadata=True)
    old = batch.table
    batch.table = table
    batch.attend(**kw)
    assert int(status) & L.STATUS_BAD_PAGE_ID
    batch.table = old
    status.zero_()
    batch.attend(residual_page_ids=torch.full_like(batch.ids, -7), **kw)
    assert int(status) & L.STATUS_BAD_TAIL_ID
    status.zero_()
    starts = batch.starts
    batch.starts = torch.tensor([0, 4, 2, 1 << 30], dtype=torch.int32, device=cuda_device)
    batch.attend(**kw)
    assert int(status) & L.STATUS_BAD_LENGTH
    batch.starts = starts
    for bad in ("seqused_fp4", "starts", "table"):
        keep = getattr(batch, bad)
        value = keep.clone()
        value[-1] = 1000
        setattr(batch, bad, value)
        with pytest.raises(ValueError):
            batch.attend()
        setattr(batch, bad, keep)


def test_attention_refusals(cuda_device):
    batch = ChunkBatch([(1, 3, 2)], 8, 2, cuda_device)
    with pytest.raises(NotImplementedError, match="1 to 8, 16 or 32"):
        nine = ChunkBatch([(1, 3, 2)], 18, 2, cuda_device)
        nine.attend()
    for change, words in (
        (dict(softmax_scale=0.0), "softmax_scale"), (dict(num_splits=0), "num_splits"),
        (dict(max_chunk_len=1), "longer than max_chunk_len"), (dict(residual_page_ids=None), "together"),
        (dict(key_shift=torch.zeros(2, 128, device=cuda_device)), "key_shift"),
        (dict(out=torch.empty(1, 8, 128, dtype=torch.bfloat16, device=cuda_device)), "out must"),
        (dict(lse=torch.empty(2, 8, dtype=torch.bfloat16, device=cuda_device)), "lse must"),
        (dict(status=torch.zeros(1, device=cuda_device)), "status"),
        (dict(num_splits=2, workspace=torch.empty(16, dtype=torch.uint8, device=cuda_device)), "workspace"),
        (dict(seqused_residual=batch.seqused_tail.long()), "seqused_residual"),
    ):
        with pytest.raises(ValueError, match=words):
            batch.attend(**change)
    batch.query = batch.query.float()
    with pytest.raises(ValueError, match="query"):
        batch.attend()


# -- append and read-back ------------------------------------------------------------------------


def streams(batch):
    """Every row's K and V stream (tail, then shifted chunk) in fp32, exact."""
    found = []
    for r, (_, t, n) in enumerate(batch.rows):
        a, slot = batch.starts_host[r], int(batch.ids_host[r])
        key = batch.key[a:a + n]
        if batch.shift is not None:
            key = key - batch.shift       # one BF16 subtract
        found.append((torch.cat([batch.tail_key[slot, :t], key]), torch.cat([batch.tail_value[slot, :t], batch.value[a:a + n]])))
    return found


@pytest.mark.parametrize("rows", [SINGLE, TINY, EDGES, LONG], ids=["single", "tiny", "edges", "long"])
@pytest.mark.parametrize("heads_kv,shift,spread", [(2, True, False), (1, False, True), (8, True, True)])
def test_append_writes_the_quantisers_bytes(cuda_device, rows, heads_kv, shift, spread):
    from nvfp4_attn_kernel_b200.nvfp4_decode_kernel import _quantize, dequantize_pages
    from nvfp4_attn_kernel_b200.nvfp4_vllm import layout

    batch = ChunkBatch(rows, heads_kv, heads_kv, cuda_device, seed=3, shift=shift, pad=2, spread=spread)
    want = streams(batch)
    cache, tails = batch.cache.clone(), (batch.tail_key.clone(), batch.tail_value.clone())
    for r, (f, t, n) in enumerate(rows):
        key, value = want[r]
        sealed = len(key) // PAGE
        if sealed:
            pages = lambda x: x[:sealed * PAGE].reshape(sealed, PAGE, heads_kv, 128).contiguous()   # noqa: E731
            kp, ks = _quantize.quantize_key_pages(pages(key))
            vp, vs = _quantize.quantize_value_pages(pages(value))
            ids = batch.table_host[r, f:f + sealed].long().to(cuda_device)
            for view, new in zip(layout.carve(cache, heads_kv, 128), (kp, ks, vp, vs)):
                view.view(torch.uint8)[ids] = new.view(torch.uint8)
        slot, rest = int(batch.ids_host[r]), len(key) % PAGE
        tails[0][slot, :rest], tails[1][slot, :rest] = key[sealed * PAGE:], value[sealed * PAGE:]
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    full, rest = batch.append(status=status)
    assert full.tolist() == [(f + (t + n) // PAGE) * PAGE for f, t, n in rows]
    assert rest.tolist() == [(t + n) % PAGE for _, t, n in rows]
    assert torch.equal(batch.cache, cache)          # the sealed pages, and not a byte of any other
    assert torch.equal(batch.tail_key.view(torch.int16), tails[0].view(torch.int16))
    assert torch.equal(batch.tail_value.view(torch.int16), tails[1].view(torch.int16))
    assert int(status) == 0
    written = torch.cat([batch.table_host[r, f:f + (t + n) // PAGE] for r, (f, t, n) in enumerate(rows)])
    k, v = dequantize_pages(*batch.views, written.to(cuda_device))
    want_k, want_v = batch.page_values()
    assert np.array_equal(to_np(k), want_k[written.tolist()].reshape(to_np(k).shape))
    assert np.array_equal(to_np(v), want_v[written.tolist()].reshape(to_np(v).shape))


def test_dequantize_every_code_and_scale(cuda_device):
    """All 256 byte values as packed nibbles and all 256 scale bytes (NaN scales give NaN), odd page lists."""
    from nvfp4_attn_kernel_b200.nvfp4_decode_kernel import dequantize_pages

    g = torch.Generator().manual_seed(1)
    cache, views = blocks_of(5, 3, 0, cuda_device)
    cache.copy_(torch.randint(0, 256, cache.shape, generator=g).to(torch.uint8))
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    ids = torch.tensor([4, 0, 4, -1, 2, 5], dtype=torch.int32, device=cuda_device)
    k, v = dequantize_pages(*views, ids, status=status)
    assert int(status) == L.STATUS_BAD_PAGE_ID
    with np.errstate(invalid="ignore"):
        from helpers import scale_bytes
        want = (O.dequantize_key_pages(to_np(views[0]), scale_bytes(views[1])),
                O.dequantize_value_pages(to_np(views[2]), scale_bytes(views[3])))
    for got, full in ((to_np(k), want[0]), (to_np(v), want[1])):
        full = full.reshape(5, PAGE, 3, 128)
        for i, page in enumerate(ids.tolist()):
            if 0 <= page < 5:
                assert np.array_equal(got[i], full[page], equal_nan=True)
            else:
                assert (got[i] == 0).all()
    empty = dequantize_pages(*views, ids[:0])
    assert empty[0].shape == (0, PAGE, 3, 128)


def test_append_keeps_rows_with_bad_metadata(cuda_device):
    rows = [(1, 100, 60), (0, 20, 30), (2, 128, 1)]
    for change, bit in (("table", L.STATUS_BAD_PAGE_ID), ("ids", L.STATUS_BAD_TAIL_ID), ("columns", L.STATUS_BAD_LENGTH),
                        ("tail", L.STATUS_BAD_LENGTH), ("starts", L.STATUS_BAD_LENGTH)):
        batch = ChunkBatch(rows, 2, 2, cuda_device, seed=4)
        status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
        kw = {}
        if change == "table":
            batch.table[0, 1] = -5
        elif change == "ids":
            batch.ids[0] = 99
        elif change == "columns":
            batch.table = batch.table[:, :1]
            batch.seqused_fp4[2] = 128       # its own page would be column 1
        elif change == "tail":
            batch.seqused_tail[0] = 129
        else:
            kw["max_chunk_len"] = 40
        cache, tail = batch.cache.clone(), batch.tail_key.clone()
        with pytest.raises(ValueError):
            batch.append(**kw)
        assert torch.equal(batch.cache, cache)
        full, rest = batch.append(status=status, trusted_metadata=True, **kw)
        assert int(status) & bit, change
        slot = int(batch.ids_host[0])
        if change != "table":
            assert torch.equal(batch.tail_key[slot].view(torch.int16), tail[slot].view(torch.int16))
            assert int(full[0]) == int(batch.seqused_fp4[0]) and int(rest[0]) == int(batch.seqused_tail[0])
        assert (int(full[1]), int(rest[1])) == (0, 50)        # the healthy row goes through


def test_append_refuses_shared_destinations(cuda_device):
    batch = ChunkBatch([(1, 100, 60), (0, 120, 30)], 2, 2, cuda_device, seed=4)
    batch.ids[1] = batch.ids[0]
    with pytest.raises(ValueError, match="one residual page"):
        batch.append()
    batch.ids.copy_(batch.ids_host)
    batch.table[1, 0] = batch.table[0, 1]
    with pytest.raises(ValueError, match="one page"):
        batch.append()
    batch.table.copy_(batch.table_host)
    with pytest.raises(ValueError, match="of their own"):
        batch.append(seqused_fp4_out=batch.seqused_fp4)


def test_chunks_of_a_prompt_equal_the_whole_prompt(cuda_device):
    """A prompt served in ragged chunks (attend, append, attend ...) against the 64-bit form over what the cache
    holds at each step; afterwards the cache has the bytes that one append of the whole prompt writes."""
    from nvfp4_attn_kernel_b200.nvfp4_decode_kernel import append_kv_chunk, fp4_chunk_attention

    cuts, heads_q, heads_kv = [0, 3, 130, 131, 387, 512, 700], 8, 2
    whole = ChunkBatch([(0, 0, 700)], heads_q, heads_kv, cuda_device, seed=21, shift=True)
    cache, views = blocks_of(whole.cache.shape[0], heads_kv, 255, cuda_device)
    tail_key, tail_value = torch.full_like(whole.tail_key, float("nan")), torch.full_like(whole.tail_value, float("nan"))
    full = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    used = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    for a, b in zip(cuts, cuts[1:]):
        step = ChunkBatch([(int(full) // PAGE, int(used), b - a)], heads_q, heads_kv, cuda_device, seed=1)
        step.views, step.table, step.table_host = views, whole.table, whole.table_host
        step.tail_key, step.tail_value, step.ids, step.ids_host = tail_key, tail_value, whole.ids, whole.ids_host
        step.query, step.key, step.value = whole.query[a:b], whole.key[a:b], whole.value[a:b]
        step.seqused_fp4, step.seqused_tail, step.shift = full, used, whole.shift
        check(step, step.attend())
        full, used = step.append()
    assert (int(full), int(used)) == (640, 60)
    whole.append()
    assert torch.equal(cache[whole.table[0, :5].long()], whole.cache[whole.table[0, :5].long()])
    slot = int(whole.ids_host[0])
    assert torch.equal(tail_key[slot, :60], whole.tail_key[slot, :60])
    assert torch.equal(tail_value[slot, :60], whole.tail_value[slot, :60])


def test_decode_continues_what_chunks_wrote(cuda_device):
    """After an append, fp4_decode of the next token agrees with the attention of a one-token chunk: the same cache
    through two operators (decode's own quantisation of query and probabilities sets the distance)."""
    from nvfp4_attn_kernel_b200.nvfp4_decode_kernel import fp4_decode

    batch = ChunkBatch([(2, 100, 200), (0, 0, 70)], 8, 2, cuda_device, seed=22, poison=False)
    full, used = batch.append()
    g = torch.Generator().manual_seed(5)
    token = lambda heads: torch.randn(2, heads, 128, generator=g).to(torch.bfloat16).to(cuda_device)   # noqa: E731
    query, key, value = token(8), token(2), token(2)
    step = ChunkBatch([(int(f) // PAGE, int(t), 1) for f, t in zip(full, used)], 8, 2, cuda_device, seed=1)
    step.views, step.table, step.table_host, step.shift = batch.views, batch.table, batch.table_host, None
    step.tail_key, step.tail_value, step.ids, step.ids_host = batch.tail_key, batch.tail_value, batch.ids, batch.ids_host
    step.query, step.key, step.value = query, key, value
    want = step.attend()
    check(step, want)
    got = fp4_decode(query, *batch.views, batch.table, full, residual_key_pages_bf16=batch.tail_key,
                     residual_value_pages_bf16=batch.tail_value, residual_page_ids=batch.ids,
                     seqused_residual=used + 1, append_key=key, append_value=value)
    # decode rounds query and probabilities to four bits: a fifth of the spread at worst, far less on average
    assert (got.float() - want.float()).abs().max() < 0.2 * want.float().abs().max()
