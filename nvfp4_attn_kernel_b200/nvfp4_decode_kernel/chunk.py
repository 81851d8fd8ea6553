"""Chunks: several new tokens per row over the paged NVFP4 cache.

The reference serves whole prompts and single tokens only (``src/nvfp4_vllm/guards.py:30-116`` refuses
chunked prefill, prefix reuse and drafts); these operators have no counterpart in it.

A batch is ragged: row r's tokens are ``[chunk_start_loc[r], chunk_start_loc[r + 1])`` of the token tensors,
0 to ``max_chunk_len`` of them.  Its history is ``seqused_fp4[r]`` tokens in sealed pages (a multiple of
128) followed by ``seqused_residual[r]`` tokens (0 to 128) in BF16 residual page ``residual_page_ids[r]``.
A step that continues sequences is :func:`fp4_chunk_attention` in every layer, then
:func:`append_kv_chunk` with the same lengths.
"""

from __future__ import annotations

import math

import torch

from .. import _lib

PAGE_SIZE = 128
HEAD_DIM = 128


def _device_of(tensor: torch.Tensor, name: str) -> torch.device:
    if not tensor.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    return tensor.device


def _tokens(tensor: torch.Tensor, name: str, device: torch.device) -> tuple[int, int]:
    """Rows and heads of a BF16 [tokens, heads, 128] tensor that is dense within a token."""
    shape, stride = tensor.shape, tensor.stride()
    if tensor.dtype is not torch.bfloat16 or len(shape) != 3 or shape[2] != HEAD_DIM or tensor.device != device:
        raise ValueError(f"{name} must be BF16 [tokens, heads, 128] on {device}")
    if stride[2] != 1 or (shape[1] > 1 and stride[1] != HEAD_DIM):
        raise ValueError(f"{name} must be dense within a token")
    return shape[0], shape[1]


def _index(tensor: torch.Tensor, name: str, length: int, device: torch.device) -> int:
    if tensor.dtype is not torch.int32 or tensor.device != device or tensor.shape != (length,) or \
            (length > 1 and tensor.stride(0) != 1):
        raise ValueError(f"{name} must be contiguous INT32 of shape [{length}] on {device}")
    return tensor.data_ptr()


def _page_regions(args, key_pages_fp4, key_scales, value_pages_fp4, value_scales, device) -> int:
    """Check the four page regions and enter them in an argument block; returns the KV head count."""
    if key_pages_fp4.ndim != 4:
        raise ValueError("key_pages_fp4 must be packed FP4 with shape [pages, 128, heads_kv, 64]")
    pages, page, heads, half = key_pages_fp4.shape
    if page != PAGE_SIZE or half != HEAD_DIM // 2:
        raise ValueError("key_pages_fp4 must be packed FP4 with shape [pages, 128, heads_kv, 64]")
    want_scales = (pages, 32, 4, 1, 4, 2, heads)
    for name, tensor, shape, inner in (
        ("key_pages_fp4", key_pages_fp4, None, (heads * 64, 64, 1)),
        ("value_pages_fp4", value_pages_fp4, (pages, heads, HEAD_DIM, 64), (HEAD_DIM * 64, 64, 1)),
        ("key_scales", key_scales, want_scales, (16, 4, 1024, 1, 512, 1024)),
        ("value_scales", value_scales, want_scales, (16, 4, 1024, 1, 512, 1024)),
    ):
        if tensor.device != device or tensor.element_size() != 1:
            raise ValueError(f"{name} must hold bytes on {device}")
        if shape is not None and tensor.shape != shape:
            raise ValueError(f"{name} must have shape {shape}")
        if tensor.stride()[1:] != inner:
            raise ValueError(f"{name} must be dense within a page, in the quantisers' layout")
    args.k_packed, args.k_pitch = key_pages_fp4.data_ptr(), key_pages_fp4.stride(0)
    args.k_sf, args.k_sf_pitch = key_scales.data_ptr(), key_scales.stride(0)
    args.v_packed, args.v_pitch = value_pages_fp4.data_ptr(), value_pages_fp4.stride(0)
    args.v_sf, args.v_sf_pitch = value_scales.data_ptr(), value_scales.stride(0)
    args.num_pages, args.heads_kv = pages, heads
    return heads


def _fill(key, value, key_pages_fp4, key_scales, value_pages_fp4, value_scales, fp4_page_table, seqused_fp4,
          chunk_start_loc, max_chunk_len, residual, key_shift, status, device):
    """The argument block with everything the attention and the append share, checked."""
    args = _lib.ChunkArgs()
    heads = _page_regions(args, key_pages_fp4, key_scales, value_pages_fp4, value_scales, device)
    tokens, key_heads = _tokens(key, "key", device)
    if (tokens, key_heads) != _tokens(value, "value", device) or key_heads != heads:
        raise ValueError("key and value must have the same tokens, and the pages' heads")
    args.key, args.value = key.data_ptr(), value.data_ptr()
    width = heads * HEAD_DIM
    args.key_token_stride = key.stride(0) if tokens > 1 else width
    args.value_token_stride = value.stride(0) if tokens > 1 else width
    if fp4_page_table.dtype is not torch.int32 or fp4_page_table.ndim != 2 or fp4_page_table.device != device or \
            (fp4_page_table.shape[1] > 1 and fp4_page_table.stride(1) != 1):
        raise ValueError(f"fp4_page_table must be INT32 [rows, max_pages] on {device}, dense within a row")
    rows, columns = fp4_page_table.shape
    args.page_table, args.max_pages = fp4_page_table.data_ptr(), columns
    args.page_table_row_stride = fp4_page_table.stride(0) if rows > 1 else columns
    args.seqused_fp4 = _index(seqused_fp4, "seqused_fp4", rows, device)
    args.chunk_start = _index(chunk_start_loc, "chunk_start_loc", rows + 1, device)
    if not isinstance(max_chunk_len, int) or max_chunk_len < 0:
        raise ValueError(f"max_chunk_len must be a non-negative int, got {max_chunk_len!r}")
    args.rows, args.tokens, args.max_chunk = rows, tokens, min(max_chunk_len, tokens)
    tail_key, tail_value, tail_ids, tail_used = residual
    if any(item is not None for item in residual):
        if any(item is None for item in residual):
            raise ValueError("the four residual arguments must be provided together")
        for name, tensor in (("residual_key_pages_bf16", tail_key), ("residual_value_pages_bf16", tail_value)):
            if tensor.dtype is not torch.bfloat16 or tensor.device != device or tensor.ndim != 4 or \
                    tensor.shape[1:] != (PAGE_SIZE, heads, HEAD_DIM) or not tensor.is_contiguous():
                raise ValueError(f"{name} must be contiguous BF16 [pages, 128, {heads}, 128] on {device}")
        if tail_key.shape[0] != tail_value.shape[0]:
            raise ValueError("the residual caches must have the same pages")
        args.tail_key, args.tail_value, args.tail_pages = tail_key.data_ptr(), tail_value.data_ptr(), tail_key.shape[0]
        args.tail_ids = _index(tail_ids, "residual_page_ids", rows, device)
        args.seqused_tail = _index(tail_used, "seqused_residual", rows, device)
    if key_shift is not None:
        if key_shift.dtype is not torch.bfloat16 or key_shift.device != device or \
                key_shift.shape != (heads, HEAD_DIM) or not key_shift.is_contiguous():
            raise ValueError(f"key_shift must be contiguous BF16 [{heads}, 128] on {device}")
        args.key_shift = key_shift.data_ptr()
    if status is not None:
        args.status = _status(status, device)
    return args


def _status(status: torch.Tensor, device: torch.device) -> int:
    if status.element_size() != 4 or status.is_floating_point() or status.numel() < 1 or status.device != device:
        raise ValueError(f"status must be one 32-bit integer on {device}")
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
    written = []
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
    if len(set(written)) != len(written):
        raise ValueError("two chunks must not be appended to one page")


def chunk_split_heuristic(rows: int, tokens: int, max_chunk_len: int, heads_q: int, heads_kv: int, max_pages: int, *,
                          sms: int) -> int:
    """Ranges that each row's keys are cut into."""
    return 1


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
        num_splits: ranges that each row's keys are cut into (None: by the launch's shape);
            ``workspace``: their scratch, UINT8, ``chunk_workspace_bytes`` long (None: allocated).
        status: one 32-bit integer on the device, a sticky OR of the ``NVFP4_STATUS_*`` bits.
        trusted_metadata: skip every check that reads device values back.

    The chunk is read from ``key`` / ``value`` in BF16 whether or not it has been appended already; ``seqused_*``
    are the lengths before it.  Unlike ``fp4_decode`` the query and the probabilities are not quantised.
    Returns ``out[:tokens]``, or a fresh tensor whose padding rows are undefined.
    """
    device = _device_of(query, "query")
    args = _fill(key, value, key_pages_fp4, key_scales, value_pages_fp4, value_scales, fp4_page_table, seqused_fp4,
                 chunk_start_loc, max_chunk_len,
                 (residual_key_pages_bf16, residual_value_pages_bf16, residual_page_ids, seqused_residual), key_shift,
                 status, device)
    shape, stride = query.shape, query.stride()
    if query.dtype is not torch.bfloat16 or len(shape) != 3 or shape[2] != HEAD_DIM or stride[2] != 1:
        raise ValueError("query must be BF16 [tokens, heads_q, 128] with unit channel stride")
    tokens, heads_q = shape[0], shape[1]
    if tokens != args.tokens:
        raise ValueError(f"query has {tokens} tokens, key and value have {args.tokens}")
    args.query, args.heads_q = query.data_ptr(), heads_q
    args.q_token_stride = stride[0] if tokens > 1 else heads_q * HEAD_DIM
    args.q_head_stride = stride[1] if heads_q > 1 else HEAD_DIM
    if out is None:
        out = torch.empty(tokens, heads_q, HEAD_DIM, dtype=torch.bfloat16, device=device)
    else:
        out_tokens, out_heads = _tokens(out, "out", device)
        if out_heads != heads_q or out_tokens < tokens:
            raise ValueError(f"out must have shape [at least {tokens}, {heads_q}, 128]")
    args.out, args.out_token_stride = out.data_ptr(), out.stride(0) if out.shape[0] > 1 else heads_q * HEAD_DIM
    if lse is not None:
        if lse.dtype is not torch.float32 or lse.device != device or lse.ndim != 2 or lse.shape[0] < tokens or \
                lse.shape[1] != heads_q or not lse.is_contiguous():
            raise ValueError(f"lse must be contiguous FP32 of shape [at least {tokens}, {heads_q}] on {device}")
        args.lse = lse.data_ptr()
    scale = HEAD_DIM ** -0.5 if softmax_scale is None else softmax_scale
    if not math.isfinite(scale) or scale <= 0.0:
        raise ValueError("softmax_scale must be finite and positive")
    args.softmax_scale = scale
    if num_splits is None:
        num_splits = chunk_split_heuristic(args.rows, tokens, args.max_chunk, heads_q, args.heads_kv, args.max_pages,
                                           sms=_sm_count(device))
    elif not isinstance(num_splits, int) or not 1 <= num_splits <= 128:
        raise ValueError(f"num_splits must be 1 to 128, got {num_splits!r}")
    args.num_splits = num_splits
    need = chunk_workspace_bytes(tokens, heads_q, num_splits)
    if need:
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=device)
        elif workspace.dtype is not torch.uint8 or workspace.device != device or not workspace.is_contiguous() or \
                workspace.numel() < need:
            raise ValueError(f"workspace must be contiguous UINT8 of at least {need} bytes on {device}")
        args.workspace, args.workspace_bytes = workspace.data_ptr(), workspace.numel()
    if not trusted_metadata:
        _check_metadata(fp4_page_table, seqused_fp4, chunk_start_loc, max_chunk_len, tokens,
                        (residual_key_pages_bf16, residual_value_pages_bf16, residual_page_ids, seqused_residual),
                        args.num_pages, False)
    _launch("nvfp4_chunk_attention", args, device)
    return out[:tokens] if out.shape[0] != tokens else out


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
    A row whose metadata is out of range, or whose table has no column left, keeps its cache and lengths and is
    flagged in ``status``; with ``trusted_metadata=False`` such a batch is refused before anything is written.
    """
    device = _device_of(key, "key")
    residual = (residual_key_pages_bf16, residual_value_pages_bf16, residual_page_ids, seqused_residual)
    if any(item is None for item in residual):
        raise ValueError("append_kv_chunk needs the four residual arguments")
    args = _fill(key, value, key_pages_fp4, key_scales, value_pages_fp4, value_scales, fp4_page_table, seqused_fp4,
                 chunk_start_loc, max_chunk_len, residual, key_shift, status, device)
    rows = args.rows
    if seqused_fp4_out is None or seqused_residual_out is None:
        fresh = torch.empty(2, rows, dtype=torch.int32, device=device)
        seqused_fp4_out = fresh[0] if seqused_fp4_out is None else seqused_fp4_out
        seqused_residual_out = fresh[1] if seqused_residual_out is None else seqused_residual_out
    args.seqused_fp4_out = _index(seqused_fp4_out, "seqused_fp4_out", rows, device)
    args.seqused_tail_out = _index(seqused_residual_out, "seqused_residual_out", rows, device)
    if not trusted_metadata:
        _check_metadata(fp4_page_table, seqused_fp4, chunk_start_loc, max_chunk_len, args.tokens, residual,
                        args.num_pages, True)
    _launch("nvfp4_append_chunk", args, device)
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
    device = _device_of(key_pages_fp4, "key_pages_fp4")
    args = _lib.ChunkArgs()
    heads = _page_regions(args, key_pages_fp4, key_scales, value_pages_fp4, value_scales, device)
    if page_ids.ndim != 1:
        raise ValueError("page_ids must be contiguous 1-D INT32")
    count = page_ids.shape[0]
    ids = _index(page_ids, "page_ids", count, device)
    shape = (count, PAGE_SIZE, heads, HEAD_DIM)
    outs = []
    for name, tensor in (("key_out", key_out), ("value_out", value_out)):
        if tensor is None:
            tensor = torch.empty(shape, dtype=torch.bfloat16, device=device)
        elif tensor.dtype is not torch.bfloat16 or tensor.device != device or tensor.shape != shape or \
                not tensor.is_contiguous():
            raise ValueError(f"{name} must be contiguous BF16 {shape} on {device}")
        outs.append(tensor)
    flag = None if status is None else _status(status, device)
    call = _lib.load().nvfp4_dequantize_pages
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    block = (args.k_packed, args.k_pitch, args.k_sf, args.k_sf_pitch, args.v_packed, args.v_pitch, args.v_sf,
             args.v_sf_pitch, args.num_pages, ids, count, heads, outs[0].data_ptr(), outs[1].data_ptr(), flag, stream)
    if torch.cuda.current_device() == index:
        _lib.check(call(*block))
    else:
        with torch.cuda.device(index):
            _lib.check(call(*block))
    return outs[0], outs[1]


def chunk_workspace_bytes(tokens: int, heads_q: int, num_splits: int) -> int:
    """Scratch of :func:`fp4_chunk_attention` (``nvfp4_chunk_attention_workspace_bytes``): an fp32 output row and its
    LSE per token, head and range."""
    return 0 if num_splits <= 1 else num_splits * tokens * heads_q * (HEAD_DIM + 1) * 4


_SM_COUNT: dict[int, int] = {}


def _sm_count(device: torch.device) -> int:
    count = _SM_COUNT.get(device.index)
    if count is None:
        count = _SM_COUNT[device.index] = torch.cuda.get_device_properties(device).multi_processor_count
    return count


def _launch(name: str, args, device: torch.device) -> None:
    call = getattr(_lib.load(), name)
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch.cuda.current_device() == index:
        _lib.check(call(args, stream))
    else:
        with torch.cuda.device(index):
            _lib.check(call(args, stream))
