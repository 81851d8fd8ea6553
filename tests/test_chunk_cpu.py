"""CPU tests of the chunk and page-pool entry points: struct layout, sizes, refusals before any launch."""

import ctypes
import os
import re

import pytest

import nvfp4_attn_kernel_b200._lib as L

ROOT = os.path.dirname(os.path.dirname(__file__))
SOME = 1 << 20      # an aligned address that nothing reads: every call here is refused or has no work


def test_struct_mirror_matches_header_field_order():
    text = open(os.path.join(ROOT, "include", "nvfp4_b200.h")).read()
    body = text[text.index("typedef struct nvfp4_chunk_args {"):text.index("} nvfp4_chunk_args;")]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    assert re.findall(r"\b([a-z_0-9]+)\s*;", body) == [name for name, _ in L.ChunkArgs._fields_]


def test_packed_block_is_the_struct():
    from nvfp4_attn_kernel_b200.nvfp4_decode_kernel.chunk import _BLOCK

    assert _BLOCK.size == ctypes.sizeof(L.ChunkArgs)
    values = [i + 0.5 if kind is ctypes.c_float else i + 1 for i, (_, kind) in enumerate(L.ChunkArgs._fields_)]
    args = L.ChunkArgs.from_buffer_copy(_BLOCK.pack(*values))
    assert [getattr(args, name) for name, _ in L.ChunkArgs._fields_] == values


def test_workspace_sizes():
    from nvfp4_attn_kernel_b200.nvfp4_decode_kernel.chunk import chunk_workspace_bytes

    lib = L.load()
    for tokens, heads, splits in ((1, 1, 1), (7, 32, 2), (4096, 40, 16), (0, 8, 4), (300000, 128, 100)):
        assert lib.nvfp4_chunk_attention_workspace_bytes(tokens, heads, splits) == chunk_workspace_bytes(tokens, heads, splits)
    assert lib.nvfp4_pool_compact_workspace_bytes(1000) >= 3001 * 4


def arguments(**changes):
    args = L.ChunkArgs()
    for name in ("k_packed", "k_sf", "v_packed", "v_sf", "page_table", "seqused_fp4", "tail_key", "tail_value", "tail_ids",
                 "seqused_tail", "chunk_start", "key", "value", "query", "out"):
        setattr(args, name, SOME)
    args.seqused_fp4, args.seqused_tail = SOME + 16, SOME + 32
    args.k_pitch = args.v_pitch = 128 * 2 * 64
    args.k_sf_pitch = args.v_sf_pitch = 2 * 1024
    args.num_pages, args.max_pages, args.page_table_row_stride, args.tail_pages = 4, 2, 2, 3
    args.key_token_stride = args.value_token_stride = 256
    args.rows, args.tokens, args.max_chunk, args.heads_kv, args.heads_q = 2, 5, 4, 2, 8
    args.q_token_stride, args.q_head_stride, args.out_token_stride = 1024, 128, 1024
    args.softmax_scale, args.num_splits = 0.1, 1
    args.seqused_fp4_out, args.seqused_tail_out = SOME + 48, SOME + 64
    for name, value in changes.items():
        setattr(args, name, value)
    return args


@pytest.mark.parametrize("entry", ["nvfp4_chunk_attention", "nvfp4_append_chunk"])
@pytest.mark.parametrize("changes,words", [
    (dict(rows=-1), "negative"), (dict(tokens=-1), "negative"), (dict(rows=70000), "too many rows"),
    (dict(max_chunk=5 << 20), "max_chunk"),
    (dict(heads_kv=0), "heads_kv"), (dict(seqused_fp4=None), "lengths"), (dict(chunk_start=None), "lengths"),
    (dict(key=None), "key and value"), (dict(key=SOME + 2), "16-byte"), (dict(key_token_stride=128), "dense within a token"),
    (dict(value_token_stride=260), "16-byte"), (dict(key_shift=SOME + 4), "16-byte"), (dict(k_sf=None), "non-null"),
    (dict(page_table_row_stride=1), "page_table_row_stride"), (dict(k_pitch=100), "pitch"), (dict(v_sf_pitch=2056), "pitch"),
    (dict(v_packed=SOME + 8), "alignment"), (dict(tail_ids=None), "go together"), (dict(tail_key=SOME + 2), "tail pages"),
    (dict(num_pages=-1), "page counts"),
])
def test_shared_refusals(entry, changes, words):
    assert getattr(L.load(), entry)(ctypes.byref(arguments(**changes)), None) == L.ERR_INVALID
    assert words in L.last_error()


def test_attention_refusals():
    call = L.load().nvfp4_chunk_attention
    assert call(None, None) == L.ERR_INVALID
    for changes, words in ((dict(softmax_scale=0.0), "softmax_scale"), (dict(softmax_scale=float("inf")), "softmax_scale"),
                           (dict(softmax_scale=float("nan")), "softmax_scale"), (dict(num_splits=0), "num_splits"),
                           (dict(num_splits=129), "num_splits"), (dict(query=None), "query and out"),
                           (dict(out=SOME + 8), "alignment"), (dict(q_head_stride=129), "alignment"),
                           (dict(out_token_stride=128), "dense in a token"), (dict(num_splits=2), "workspace"),
                           (dict(num_splits=2, workspace=SOME, workspace_bytes=2 * 5 * 8 * 516 - 1), "workspace")):
        assert call(ctypes.byref(arguments(**changes)), None) == L.ERR_INVALID
        assert words in L.last_error()
    assert call(ctypes.byref(arguments(heads_q=18)), None) == L.ERR_UNSUPPORTED
    for empty in (dict(rows=0), dict(tokens=0), dict(max_chunk=0)):
        assert call(ctypes.byref(arguments(**empty)), None) == 0


def test_append_refusals():
    call = L.load().nvfp4_append_chunk
    assert call(None, None) == L.ERR_INVALID
    for changes, words in ((dict(tail_key=None, tail_value=None, tail_ids=None, seqused_tail=None), "needs the BF16 tail"),
                           (dict(seqused_fp4_out=None), "need buffers"), (dict(seqused_tail_out=SOME + 32), "of their own")):
        assert call(ctypes.byref(arguments(**changes)), None) == L.ERR_INVALID
        assert words in L.last_error()
    assert call(ctypes.byref(arguments(rows=0)), None) == 0


def test_dequantize_refusals():
    call = L.load().nvfp4_dequantize_pages
    good = [SOME, 16384, SOME, 2048, SOME, 16384, SOME, 2048, 4, SOME, 3, 2, SOME, SOME, None, None]
    for at, value, words in ((0, None, "null"), (1, 16368, "pitch"), (3, 2050, "pitch"), (6, SOME + 4, "alignment"), (8, -1, "negative"),
                             (10, -1, "negative"), (11, 0, "heads_kv"), (12, None, "null"), (13, SOME + 2, "alignment")):
        block = list(good)
        block[at] = value
        assert call(*block) == L.ERR_INVALID
        assert words in L.last_error()
    good[10] = 0
    assert call(*good) == 0


def test_pool_refusals():
    lib = L.load()
    assert lib.nvfp4_pool_release(SOME, -1, SOME, 4, 4, 2, SOME, SOME, 8, None, None) == L.ERR_INVALID
    assert lib.nvfp4_pool_release(SOME, 1, None, 4, 4, 2, SOME, SOME, 8, None, None) == L.ERR_INVALID
    assert lib.nvfp4_pool_release(SOME, 1, SOME, 3, 4, 2, SOME, SOME, 8, None, None) == L.ERR_INVALID
    assert lib.nvfp4_pool_release(None, 0, None, 0, 0, 0, None, None, 0, None, None) == 0
    fork = [SOME, SOME, 1, SOME, 4, 4, 2, SOME, SOME, SOME, SOME, SOME, 8, SOME, SOME, 65536 * 2, 16384, 2, 8, 1, None, None]
    for at, value in ((2, -1), (2, 70000), (3, None), (4, 3), (10, None), (13, None), (13, SOME + 2), (16, 16383), (16, 100),
                      (17, -1), (17, 2000), (19, 0)):
        block = list(fork)
        block[at] = value
        assert lib.nvfp4_pool_fork(*block) == L.ERR_INVALID, (at, value)
    fork[2] = 0
    assert lib.nvfp4_pool_fork(*fork) == 0
    assert lib.nvfp4_pool_free_list(None, 8, 0, SOME, SOME, None) == L.ERR_INVALID
    assert lib.nvfp4_pool_free_list(SOME, 8, -1, SOME, SOME, None) == L.ERR_INVALID
    assert lib.nvfp4_pool_copy(SOME, 1, 24, 8, SOME, SOME, 1, None, None) == L.ERR_INVALID
    assert lib.nvfp4_pool_copy(None, 1, 32, 8, SOME, SOME, 1, None, None) == L.ERR_INVALID
    assert lib.nvfp4_pool_copy(None, 1, 32, 8, None, None, 0, None, None) == 0
    compact = [SOME, 1, 32, 8, 0, SOME, SOME, 4, 4, 2, SOME, SOME, 25 * 4, SOME, None, None]
    for at, value in ((0, None), (1, 0), (2, 40), (3, 0), (4, -1), (5, None), (7, 3), (10, None), (11, None), (12, 24 * 4), (13, None)):
        block = list(compact)
        block[at] = value
        assert lib.nvfp4_pool_compact(*block) == L.ERR_INVALID, (at, value)


def test_operators_refuse_host_tensors():
    import torch

    from nvfp4_attn_kernel_b200.nvfp4_decode_kernel import append_kv_chunk, dequantize_pages, fp4_chunk_attention
    from nvfp4_attn_kernel_b200.nvfp4_vllm.pages import PagePool

    z = torch.zeros(2, 128, 2, 64, dtype=torch.uint8)
    with pytest.raises(ValueError, match="query must be a CUDA tensor"):
        fp4_chunk_attention(z, z, z, z, z, z, z, z, z, z, max_chunk_len=1)
    with pytest.raises(ValueError, match="key must be a CUDA tensor"):
        append_kv_chunk(z, z, z, z, z, z, z, z, z, max_chunk_len=1, residual_key_pages_bf16=z,
                        residual_value_pages_bf16=z, residual_page_ids=z, seqused_residual=z)
    with pytest.raises(ValueError, match="key_pages_fp4 must be a CUDA tensor"):
        dequantize_pages(z, z, z, z, z)
    with pytest.raises(ValueError, match="UINT8 CUDA"):
        PagePool([torch.zeros(4, 32, dtype=torch.uint8)])


@pytest.mark.parametrize("changes", [
    dict(seqused_fp4_out=SOME + 16 + 4), dict(seqused_fp4_out=SOME + 16 - 4), dict(seqused_tail_out=SOME + 48),
    dict(seqused_tail_out=SOME + 48 + 4), dict(seqused_tail_out=SOME + 32 + 4), dict(seqused_fp4_out=SOME + 8),
    dict(seqused_tail_out=SOME - 4)])
def test_append_refuses_overlapping_lengths(changes):
    """Lengths that are written over ones that are read (shifted by one entry, the other output, the chunk's starts,
    the residual ids), with two rows."""
    assert L.load().nvfp4_append_chunk(ctypes.byref(arguments(**changes)), None) == L.ERR_INVALID
    assert "of their own" in L.last_error()
