"""Chunks: several new tokens per row over the paged NVFP4 cache.

The reference serves whole prompts and single tokens only (``src/nvfp4_vllm/guards.py:30-116`` refuses
chunked prefill, prefix reuse and drafts); these operators have no counterpart in it.  They are for callers of the
operators: the vLLM backend of ``nvfp4_vllm`` keeps the reference's guards and does not call them.

A batch is ragged: row r's tokens are ``[chunk_start_loc[r], chunk_start_loc[r + 1])`` of the token tensors,
0 to ``max_chunk_len`` of them.  Its history is ``seqused_fp4[r]`` tokens in sealed pages (a multiple of
128) followed by ``seqused_residual[r]`` tokens (0 to 128) in BF16 residual page ``residual_page_ids[r]``.
A step that continues sequences is :func:`fp4_chunk_attention` in every layer, then
:func:`append_kv_chunk` with the same lengths.
"""

from __future__ import annotations

import functools
import math
import struct

import torch

from .. import _lib

PAGE_SIZE = 128
HEAD_DIM = 128

_GROUPS = (1, 2, 3, 4, 5, 6, 7, 8, 16, 32)      # query heads per KV head
_BF16, _I32 = torch.bfloat16, torch.int32
# the argument block of the C ABI (struct nvfp4_chunk_args), packed in one call: filling a ctypes structure field by field
# costs more than the checks
_BLOCK = struct.Struct("@" + "Pq" * 4 + "qPqiPPPqPP" + "PPPqqPiiiiP" + "PqqPqPifiPN" + "PP")


def _device_index(tensor: torch.Tensor, name: str) -> int:
    index = tensor.get_device()
    if index < 0:
        raise ValueError(f"{name} must be a CUDA tensor")
    return index


def _tokens(tensor: torch.Tensor, name: str, index: int) -> tuple[int, int, int]:
    """Rows, heads and token stride of a BF16 [tokens, heads, 128] tensor that is dense within a token."""
    if tensor.dtype is not _BF16 or tensor.ndim != 3 or tensor.get_device() != index:
        raise ValueError(f"{name} must be BF16 [tokens, heads, 128] on device {index}")
    tokens, heads, dim = tensor.shape
    token_stride, head_stride, unit = tensor.stride()
    if dim != HEAD_DIM:
        raise ValueError(f"{name} must be BF16 [tokens, heads, 128] on device {index}")
    if unit != 1 or (head_stride != HEAD_DIM and heads > 1):
        raise ValueError(f"{name} must be dense within a token")
    return tokens, heads, token_stride if tokens > 1 else heads * HEAD_DIM


def _index(tensor: torch.Tensor, name: str, length: int, index: int) -> int:
    """Address of a contiguous INT32 vector."""
    if tensor.dtype is not _I32 or tensor.get_device() != index or tensor.ndim != 1 or tensor.shape[0] != length or \
            not tensor.is_contiguous():
        raise ValueError(f"{name} must be contiguous INT32 of shape [{length}] on device {index}")
    return tensor.data_ptr()


def _page_regions(key_pages_fp4, key_scales, value_pages_fp4, value_scales, index):
    """Check the four page regions; their addresses and pitches, the page and the KV head count."""
    shape = key_pages_fp4.shape
    if len(shape) != 4 or shape[1] != PAGE_SIZE or shape[3] != HEAD_DIM // 2:
        raise ValueError("key_pages_fp4 must be packed FP4 with shape [pages, 128, heads_kv, 64]")
    pages, _, heads, _ = shape
    if value_pages_fp4.shape != (pages, heads, HEAD_DIM, 64):
        raise ValueError(f"value_pages_fp4 must have shape {(pages, heads, HEAD_DIM, 64)}")
    want = (pages, 32, 4, 1, 4, 2, heads)
    if key_scales.shape != want or value_scales.shape != want:
        raise ValueError(f"key_scales and value_scales must have shape {want}")
    k, ks, v, vs = key_pages_fp4.stride(), key_scales.stride(), value_pages_fp4.stride(), value_scales.stride()
    if k != (k[0], heads * 64, 64, 1) or v != (v[0], HEAD_DIM * 64, 64, 1):
        raise ValueError("key_pages_fp4 and value_pages_fp4 must be dense within a page")
    if ks != (ks[0], 16, 4, 1024, 1, 512, 1024) or vs != (vs[0], 16, 4, 1024, 1, 512, 1024):
        raise ValueError("key_scales and value_scales must use the quantisers' layout")
    if not (key_pages_fp4.get_device() == key_scales.get_device() == value_pages_fp4.get_device()
            == value_scales.get_device() == index and key_pages_fp4.itemsize == key_scales.itemsize
            == value_pages_fp4.itemsize == value_scales.itemsize == 1):
        raise ValueError(f"the page regions must hold bytes on device {index}")
    return (key_pages_fp4.data_ptr(), k[0], key_scales.data_ptr(), ks[0], value_pages_fp4.data_ptr(), v[0],
            value_scales.data_ptr(), vs[0]), pages, heads


def _shared(key, value, key_pages_fp4, key_scales, value_pages_fp4, value_scales, fp4_page_table, seqused_fp4,
            chunk_start_loc, max_chunk_len, residual, key_shift, status, index):
    """What the attention and the append share, checked: the first fields of the argument block, and rows, tokens,
    the chunk bound, KV heads, table columns, pages."""
    regions, pages, heads = _page_regions(key_pages_fp4, key_scales, value_pages_fp4, value_scales, index)
    tokens, key_heads, key_stride = _tokens(key, "key", index)
    value_tokens, value_heads, value_stride = _tokens(value, "value", index)
    if tokens != value_tokens or key_heads != heads or value_heads != heads:
        raise ValueError("key and value must have the same tokens, and the pages' heads")
    if fp4_page_table.dtype is not _I32 or fp4_page_table.ndim != 2 or fp4_page_table.get_device() != index:
        raise ValueError(f"fp4_page_table must be INT32 [rows, max_pages] on device {index}")
    rows, columns = fp4_page_table.shape
    row_stride, unit = fp4_page_table.stride()
    if unit != 1 and columns > 1:
        raise ValueError("fp4_page_table must be dense within a row")
    if type(max_chunk_len) is not int or max_chunk_len < 0:
        raise ValueError(f"max_chunk_len must be a non-negative int, got {max_chunk_len!r}")
    tail_key, tail_value, tail_ids, tail_used = residual
    if tail_key is None and tail_value is None and tail_ids is None and tail_used is None:
        tail = (0, 0, 0, 0, 0)
    else:
        if tail_key is None or tail_value is None or tail_ids is None or tail_used is None:
            raise ValueError("the four residual arguments must be provided together")
        shape = tail_key.shape
        for tensor in (tail_key, tail_value):
            if tensor.dtype is not _BF16 or tensor.get_device() != index or tensor.shape != shape or len(shape) != 4 or \
                    shape[1] != PAGE_SIZE or shape[2] != heads or shape[3] != HEAD_DIM or not tensor.is_contiguous():
                raise ValueError("residual_key_pages_bf16 and residual_value_pages_bf16 must be contiguous BF16 "
                                 f"[pages, 128, {heads}, 128] on device {index}")
        tail = (tail_key.data_ptr(), tail_value.data_ptr(), shape[0], _index(tail_ids, "residual_page_ids", rows, index),
                _index(tail_used, "seqused_residual", rows, index))
    shift = 0
    if key_shift is not None:
        if key_shift.dtype is not _BF16 or key_shift.get_device() != index or key_shift.shape != (heads, HEAD_DIM) or \
                not key_shift.is_contiguous():
            raise ValueError(f"key_shift must be contiguous BF16 [{heads}, 128] on device {index}")
        shift = key_shift.data_ptr()
    chunk = max_chunk_len if max_chunk_len < tokens else tokens
    fields = (*regions, pages, fp4_page_table.data_ptr(), row_stride if rows > 1 else columns, columns,
              _index(seqused_fp4, "seqused_fp4", rows, index), *tail,
              _index(chunk_start_loc, "chunk_start_loc", rows + 1, index), key.data_ptr(), value.data_ptr(), key_stride,
              value_stride, shift, rows, tokens, chunk, heads, 0 if status is None else _status(status, index))
    return fields, rows, tokens, chunk, heads, columns, pages


def _status(status: torch.Tensor, index: int) -> int:
    if status.element_size() != 4 or status.is_floating_point() or status.numel() < 1 or status.get_device() != index:
        raise ValueError(f"status must be one 32-bit integer on device {index}")
    return status.data_ptr()


def _check_metadata(table, seqused_fp4, starts, max_chunk_len, tokens, residual, num_pages, appending) -> None:
    """The checks that read device values back (skipped with ``trusted_metadata``)."""
    starts_h, full_h = starts.tolist(), seqused_fp4.tolist()
    if starts_h[0] < 0 or starts_h[-1] > tokens or any(b < a for a, b in zip(starts_h, starts_h[1:])):
        raise ValueError(f"chunk_start_loc must ascend within the {tokens} tokens, got {starts_h}")
    lengths = [b - a for a, b in zip(starts_h, starts_h[1:])]
    if lengths and max(lengths) > max_chunk_len:
        raise ValueError(f"a chunk of {max(lengths)} tokens is longer than max_chunk_len={max_chunk_len}")
    tails = [0] * len(full_h)
    if residual[3] is not None:
        tails, ids = residual[3].tolist(), residual[2].tolist()
        if any(not 0 <= t <= PAGE_SIZE for t in tails):
            raise ValueError("seqused_residual must be within [0, 128]")
        needed = [t > 0 or (appending and n > 0) for t, n in zip(tails, lengths)]
        pages = residual[0].shape[0]
        if any(need and not 0 <= i < pages for need, i in zip(needed, ids)):
            raise ValueError("residual_page_ids must be within the residual cache")
        used = [i for need, i in zip(needed, ids) if need]
        if appending and len(set(used)) != len(used):
            raise ValueError("two rows must not append to one residual page")
    table_h = table.tolist()
    written, history = [], set()
    for r, (full, t, n) in enumerate(zip(full_h, tails, lengths)):
        last = full // PAGE_SIZE
        if full < 0 or full % PAGE_SIZE:
            raise ValueError(f"seqused_fp4 must hold non-negative multiples of 128, got {full}")
        if appending:
            last += (t + n) // PAGE_SIZE
        if last > table.shape[1]:
            raise ValueError(f"row {r} needs {last} page-table columns, the table has {table.shape[1]}")
        if any(not 0 <= p < num_pages for p in table_h[r][:last]):
            raise ValueError(f"row {r} uses a page id outside [0, {num_pages})")
        if appending:
            written += table_h[r][full // PAGE_SIZE:last]
            history.update(table_h[r][:full // PAGE_SIZE])
    if len(set(written)) != len(written):
        raise ValueError("two chunks must not be appended to one page")
    if history.intersection(written):
        raise ValueError(f"pages {sorted(history.intersection(written))} are history: a chunk must not be appended to them")


@functools.lru_cache(maxsize=4096)      # of sizes alone
def chunk_split_heuristic(rows: int, tokens: int, max_chunk_len: int, heads_q: int, heads_kv: int, max_pages: int, *,
                          sms: int) -> int:
    """Ranges that each row's keys are cut into, by predicted makespan: what ``num_splits=None`` takes.  ``tokens``: rows of
    ``query``; ``max_pages``: columns of the page table; ``sms``: multiprocessors of the device.

    A CTA takes one KV head of one row and a block of query rows (one tile of 128 query rows, two where a chunk has
    more), one CTA per SM.  It costs about 10 us before and after its K/V tiles and 0.95 us a tile with one query tile,
    2.1 with two (measured: 32 rows x 4 tokens after 4096 tokens 87 us in two waves of 33 tiles, 512 tokens after 16384
    270 us); a split adds a launch of 3 us and its partial results' way through memory.  The table's width stands for
    the lengths, which the host does not know: hand a table as wide as the batch's longest row (``table[:, :columns]``, a
    view), or say ``num_splits``; a much wider one is cut as if its rows were that long (1 x 512 tokens of 32 / 8 heads
    and 1024 columns: 11 ranges, 93 MB of scratch).  Only counts that just fill a number of waves are tried; one that is
    not a twentieth faster than whole rows is not taken.  Over twelve shapes of 1 to 777 tokens after 0 to 32768, tables
    as wide as their longest row, the counts so found are within 2 % (geometric mean) of the fastest of 1 to 32.
    """
    if rows < 1 or tokens < 1 or max_chunk_len < 1 or sms < 1 or heads_kv < 1 or heads_q % heads_kv or \
            heads_q // heads_kv not in _GROUPS:
        return 1        # nothing to do, or a call that the library refuses
    max_chunk_len = min(max_chunk_len, tokens)
    tile = 128 // (heads_q // heads_kv)
    per, tile_us = (tile, 0.95) if max_chunk_len <= tile else (2 * tile, 2.1)
    ctas = min(rows * -(-max_chunk_len // per), tokens // per + rows) * heads_kv
    tiles = max_pages + -(-max_chunk_len // 128)
    best, best_us = 1, 0.95 * -(-ctas // sms) * (10.0 + tiles * tile_us)
    partial_us = tokens * heads_q * 1032 / 5e6
    for waves in (1, 2, 3, 5, 7):
        splits = min(waves * sms // ctas, 32, tiles)
        if splits > best:
            us = -(-ctas * splits // sms) * (10.0 + -(-tiles // splits) * tile_us) + 3.0 + splits * partial_us
            if us < best_us:
                best, best_us = splits, us
    return best


def fp4_chunk_attention(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    key_pages_fp4: torch.Tensor,
    key_scales: torch.Tensor,
    value_pages_fp4: torch.Tensor,
    value_scales: torch.Tensor,
    fp4_page_table: torch.Tensor,
    seqused_fp4: torch.Tensor,
    chunk_start_loc: torch.Tensor,
    *,
    max_chunk_len: int,
    residual_key_pages_bf16: torch.Tensor | None = None,
    residual_value_pages_bf16: torch.Tensor | None = None,
    residual_page_ids: torch.Tensor | None = None,
    seqused_residual: torch.Tensor | None = None,
    key_shift: torch.Tensor | None = None,
    softmax_scale: float | None = None,
    out: torch.Tensor | None = None,
    lse: torch.Tensor | None = None,
    num_splits: int | None = None,
    workspace: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
    trusted_metadata: bool = False,
) -> torch.Tensor:
    """Attention of a chunk of new tokens over each row's cache and, causally, over the chunk itself.

    Args:
        query: BF16 ``[tokens, heads_q, 128]`` (strides free, 16-byte aligned rows); ``heads_q / heads_kv`` is
            1 to 8, 16 or 32.
        key / value: BF16 ``[tokens, heads_kv, 128]``, the chunk's own, dense within a token.
        key_pages_fp4 .. value_scales / fp4_page_table / seqused_fp4: the sealed history, as in ``fp4_decode``.
        chunk_start_loc: INT32 ``[rows + 1]``; a row may bring no token.  Tokens behind the last row's are padding:
            nothing of them is read, and their rows of ``out`` and ``lse`` stay as they are.
        max_chunk_len: bound on a row's tokens (host value: it sizes the launch).
        residual_*: the BF16 partial page, as in ``fp4_decode``; the four go together.
        key_shift: BF16 ``[heads_kv, 128]``, the shift that the cached keys were stored with; it is subtracted from
            the chunk's keys, unrounded.
        out: optional BF16 ``[>= tokens, heads_q, 128]``, dense within a token.
        lse: optional contiguous FP32 ``[>= tokens, heads_q]``: natural-log sum of the exponentials of the scaled scores.
        num_splits: ranges that each row's keys are cut into (None: :func:`chunk_split_heuristic`, by the launch's shape);
            ``workspace``: their scratch, UINT8, ``chunk_workspace_bytes(tokens, heads_q, num_splits)`` long (None:
            allocated).  Calls, or captured graphs, that share one must not run at the same time.
        status: one 32-bit integer on the device, a sticky OR of the ``NVFP4_STATUS_*`` bits.
        trusted_metadata: skip every check that reads device values back.

    The chunk is read from ``key`` / ``value`` in BF16 whether or not it has been appended already; ``seqused_*``
    are the lengths before it.  Unlike ``fp4_decode`` the query and the probabilities are not quantised to four bits: over
    chunk and tail the probabilities are rounded to BF16 (2^-8 of each at most), over pages to FP16 (2^-11 of each, or
    2^-32 of the row's largest), and the BF16 query enters exactly, over pages down to 2^-17 of its row's largest
    magnitude.  Scores, maximum, sum and accumulators are fp32.  Against 64 bits the outputs are 0.0013 to 0.0021 off
    (2-norm over batches of 4 x 4 to 2 x 2048 tokens), the BF16 rounding of an exact result alone 0.0012 to 0.0017.
    A key that a token does not see does not reach it, whatever it holds; a chunk's value that is not finite also
    reaches the earlier tokens of its 128 (zero times it is NaN), as in a plain product with the probabilities.
    Returns ``out[:tokens]``, or a fresh tensor whose padding rows are undefined.
    """
    index = _device_index(query, "query")
    residual = (residual_key_pages_bf16, residual_value_pages_bf16, residual_page_ids, seqused_residual)
    fields, rows, tokens, chunk, heads, columns, pages = _shared(
        key, value, key_pages_fp4, key_scales, value_pages_fp4, value_scales, fp4_page_table, seqused_fp4,
        chunk_start_loc, max_chunk_len, residual, key_shift, status, index)
    if query.dtype is not _BF16 or query.ndim != 3 or query.shape[2] != HEAD_DIM or query.stride(2) != 1:
        raise ValueError("query must be BF16 [tokens, heads_q, 128] with unit channel stride")
    query_tokens, heads_q, _ = query.shape
    token_stride, head_stride, _ = query.stride()
    if query_tokens != tokens:
        raise ValueError(f"query has {query_tokens} tokens, key and value have {tokens}")
    if out is None:
        out = torch.empty(tokens, heads_q, HEAD_DIM, dtype=_BF16, device=query.device)
        out_tokens, out_stride = tokens, heads_q * HEAD_DIM
    else:
        out_tokens, out_heads, out_stride = _tokens(out, "out", index)
        if out_heads != heads_q or out_tokens < tokens:
            raise ValueError(f"out must have shape [at least {tokens}, {heads_q}, 128]")
    lse_address = 0
    if lse is not None:
        if lse.dtype is not torch.float32 or lse.get_device() != index or lse.ndim != 2 or lse.shape[0] < tokens or \
                lse.shape[1] != heads_q or not lse.is_contiguous():
            raise ValueError(f"lse must be contiguous FP32 of shape [at least {tokens}, {heads_q}] on device {index}")
        lse_address = lse.data_ptr()
    scale = HEAD_DIM ** -0.5 if softmax_scale is None else softmax_scale
    if not 0.0 < scale < math.inf:
        raise ValueError("softmax_scale must be finite and positive")
    if num_splits is None:
        num_splits = chunk_split_heuristic(rows, tokens, chunk, heads_q, heads, columns, sms=_sm_count(index))
    elif type(num_splits) is not int or not 1 <= num_splits <= 128:
        raise ValueError(f"num_splits must be 1 to 128, got {num_splits!r}")
    space, need = 0, 0
    if num_splits > 1:
        need = chunk_workspace_bytes(tokens, heads_q, num_splits)
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=query.device)
        elif workspace.dtype is not torch.uint8 or workspace.get_device() != index or not workspace.is_contiguous() or \
                workspace.numel() < need:
            raise ValueError(f"workspace must be contiguous UINT8 of at least {need} bytes on device {index}")
        space = workspace.data_ptr()
    if not trusted_metadata:
        _check_metadata(fp4_page_table, seqused_fp4, chunk_start_loc, max_chunk_len, tokens, residual, pages, False)
    block = _BLOCK.pack(*fields, query.data_ptr(), token_stride if tokens > 1 else heads_q * HEAD_DIM,
                        head_stride if heads_q > 1 else HEAD_DIM, out.data_ptr(), out_stride, lse_address, heads_q, scale,
                        num_splits, space, need, 0, 0)
    _launch(_lib.load().nvfp4_chunk_attention, index, block)
    return out if out_tokens == tokens else out[:tokens]


def append_kv_chunk(
    key: torch.Tensor,
    value: torch.Tensor,
    key_pages_fp4: torch.Tensor,
    key_scales: torch.Tensor,
    value_pages_fp4: torch.Tensor,
    value_scales: torch.Tensor,
    fp4_page_table: torch.Tensor,
    seqused_fp4: torch.Tensor,
    chunk_start_loc: torch.Tensor,
    *,
    max_chunk_len: int,
    residual_key_pages_bf16: torch.Tensor,
    residual_value_pages_bf16: torch.Tensor,
    residual_page_ids: torch.Tensor,
    seqused_residual: torch.Tensor,
    key_shift: torch.Tensor | None = None,
    seqused_fp4_out: torch.Tensor | None = None,
    seqused_residual_out: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
    trusted_metadata: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Write a chunk's K and V into pages and residual pages; returns the rows' lengths afterwards.

    Row r's residual tokens followed by its chunk (``key_shift`` subtracted with one BF16 subtract) are one stream:
    every full 128 tokens of it are quantised into the pages ``fp4_page_table[r, seqused_fp4[r] / 128 ...]``, byte for
    byte what ``quantize_key_tokens_into`` / ``quantize_value_tokens_into`` write, and what is left (0 to 127
    tokens) becomes the residual.  A full residual page (128 tokens) is sealed even by an empty chunk.  One launch.

    ``seqused_fp4_out`` / ``seqused_residual_out``: INT32 ``[rows]``, not the input tensors (None: allocated).
    A row whose metadata is out of range (lengths, residual page, any page that it would write), or whose table has no
    column left, keeps its pages, tail and lengths and is flagged in ``status``; with ``trusted_metadata=False`` such a
    batch is refused before anything is written, as is one that would write a page or a residual page twice, or a page of
    a row's sealed history.
    """
    index = _device_index(key, "key")
    residual = (residual_key_pages_bf16, residual_value_pages_bf16, residual_page_ids, seqused_residual)
    if residual_key_pages_bf16 is None:
        raise ValueError("append_kv_chunk needs the four residual arguments")
    fields, rows, tokens, _, _, _, pages = _shared(
        key, value, key_pages_fp4, key_scales, value_pages_fp4, value_scales, fp4_page_table, seqused_fp4,
        chunk_start_loc, max_chunk_len, residual, key_shift, status, index)
    if seqused_fp4_out is None or seqused_residual_out is None:
        full, rest = torch.empty(2, rows, dtype=_I32, device=key.device).unbind()
        seqused_fp4_out = full if seqused_fp4_out is None else seqused_fp4_out
        seqused_residual_out = rest if seqused_residual_out is None else seqused_residual_out
    after = (_index(seqused_fp4_out, "seqused_fp4_out", rows, index),
             _index(seqused_residual_out, "seqused_residual_out", rows, index))
    if not trusted_metadata:
        _check_metadata(fp4_page_table, seqused_fp4, chunk_start_loc, max_chunk_len, tokens, residual, pages, True)
    _launch(_lib.load().nvfp4_append_chunk, index, _BLOCK.pack(*fields, 0, 0, 0, 0, 0, 0, 0, 0.0, 0, 0, 0, *after))
    return seqused_fp4_out, seqused_residual_out


def dequantize_pages(
    key_pages_fp4: torch.Tensor,
    key_scales: torch.Tensor,
    value_pages_fp4: torch.Tensor,
    value_scales: torch.Tensor,
    page_ids: torch.Tensor,
    *,
    key_out: torch.Tensor | None = None,
    value_out: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Pages back to BF16: K and V ``[len(page_ids), 128, heads_kv, 128]``, exact (``e2m1 * e4m3`` has at most six
    significant bits).  Keys come back as they are cached, shifted ones shifted.  An id outside the cache gives
    zeros and sets a bit of ``status``.  One launch."""
    index = _device_index(key_pages_fp4, "key_pages_fp4")
    regions, pages, heads = _page_regions(key_pages_fp4, key_scales, value_pages_fp4, value_scales, index)
    if page_ids.ndim != 1:
        raise ValueError("page_ids must be contiguous 1-D INT32")
    count = page_ids.shape[0]
    ids = _index(page_ids, "page_ids", count, index)
    shape = (count, PAGE_SIZE, heads, HEAD_DIM)
    if key_out is None:
        key_out = torch.empty(shape, dtype=_BF16, device=page_ids.device)
    elif key_out.dtype is not _BF16 or key_out.get_device() != index or key_out.shape != shape or \
            not key_out.is_contiguous():
        raise ValueError(f"key_out must be contiguous BF16 {shape} on device {index}")
    if value_out is None:
        value_out = torch.empty(shape, dtype=_BF16, device=page_ids.device)
    elif value_out.dtype is not _BF16 or value_out.get_device() != index or value_out.shape != shape or \
            not value_out.is_contiguous():
        raise ValueError(f"value_out must be contiguous BF16 {shape} on device {index}")
    _launch(_lib.load().nvfp4_dequantize_pages, index, *regions, pages, ids, count, heads, key_out.data_ptr(),
            value_out.data_ptr(), None if status is None else _status(status, index))
    return key_out, value_out


def chunk_workspace_bytes(tokens: int, heads_q: int, num_splits: int) -> int:
    """Scratch of :func:`fp4_chunk_attention` (``nvfp4_chunk_attention_workspace_bytes``): an fp32 output row and its
    LSE per token, head and range."""
    return 0 if num_splits <= 1 else num_splits * tokens * heads_q * (HEAD_DIM + 1) * 4


_SM_COUNT: dict[int, int] = {}


def _sm_count(index: int) -> int:
    count = _SM_COUNT.get(index)
    if count is None:
        count = _SM_COUNT[index] = torch.cuda.get_device_properties(index).multi_processor_count
    return count


def _launch(call, index: int, *arguments) -> None:
    """A call of the library on the current stream of device ``index``."""
    if torch._C._cuda_getDevice() == index:
        code = call(*arguments, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            code = call(*arguments, torch._C._cuda_getCurrentRawStream(index))
    if code:
        _lib.check(code)
