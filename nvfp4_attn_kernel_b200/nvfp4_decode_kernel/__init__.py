"""Operator API of the paged NVFP4 decode kernel (drop-in for ``nvfp4_decode_kernel``)."""

from .chunk import (append_kv_chunk, chunk_split_heuristic, chunk_workspace_bytes, dequantize_pages,
                    fp4_chunk_attention)
from .interface import RESIDUAL_ROW_TILE, KernelNotAvailableError, fp4_decode, host_io_step

__all__ = ["RESIDUAL_ROW_TILE", "KernelNotAvailableError", "fp4_decode", "host_io_step", "fp4_chunk_attention",
           "append_kv_chunk", "dequantize_pages", "chunk_split_heuristic", "chunk_workspace_bytes"]
