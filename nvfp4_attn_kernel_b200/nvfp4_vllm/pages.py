"""Pages that several rows share: reference counts, forks, releases, compaction, copies.

The reference has none of it (its cache gives every sequence pages of its own).  Sealed NVFP4 pages are never
written again, so a fork shares them by counting and copies the BF16 tail alone; nothing is copied on write.
Every method works on the device in one or two launches on the current stream and reads nothing back, except
:meth:`PagePool.copy` without ``trusted_metadata=True``, which checks its lists on the host first.
The vLLM backend gives every sequence pages of its own, as the reference does, and uses no pool.
"""

from __future__ import annotations

import torch

from .. import _lib

PAGE_SIZE = 128


class PagePool:
    """The physical pages of a model's cache and their reference counts.

    Args:
        blocks: every layer's block array, UINT8 ``[pages, block_bytes]``, contiguous, all of one shape (the arrays
            that ``layout.carve`` views as pages).
        refs: INT32 ``[pages]``, how many rows hold each page (None: zeros).
        tail_key / tail_value: BF16 ``[layers, slots, 128, heads_kv, 128]`` (``LayerRuntime.tail_key``), for forks.
        reserved_pages: the first pages that are never free and never moved (vLLM's null block: 1).
        status: one INT32 on the device, a sticky OR of ``NVFP4_STATUS_*`` bits (None: allocated, ``pool.status``).

    A row of ``page_table`` (INT32 ``[rows, columns]``) holds its first ``pages_held[row]`` entries.  Calls on one
    pool must be ordered (one stream): they share its counts and its scratch.
    """

    def __init__(self, blocks, *, refs: torch.Tensor | None = None, tail_key: torch.Tensor | None = None,
                 tail_value: torch.Tensor | None = None, reserved_pages: int = 0,
                 status: torch.Tensor | None = None) -> None:
        blocks = list(blocks)
        if not blocks:
            raise ValueError("a pool needs at least one layer's block array")
        device, shape = blocks[0].device, blocks[0].shape
        for layer in blocks:
            if not layer.is_cuda or layer.device != device or layer.dtype is not torch.uint8 or layer.ndim != 2 or \
                    layer.shape != shape or not layer.is_contiguous():
                raise ValueError("blocks must be contiguous UINT8 CUDA arrays [pages, bytes] of one shape and device")
            if layer.data_ptr() % 16:
                raise ValueError("block arrays must be 16-byte aligned")
        if shape[0] < 1 or shape[1] < 16 or shape[1] % 16:
            raise ValueError("a pool needs at least one page, and a block must be a multiple of 16 bytes")
        if not 0 <= reserved_pages <= shape[0]:
            raise ValueError(f"reserved_pages must be within [0, {shape[0]}]")
        if (tail_key is None) != (tail_value is None):
            raise ValueError("tail_key and tail_value go together")
        if tail_key is not None:
            for name, tail in (("tail_key", tail_key), ("tail_value", tail_value)):
                if tail.dtype is not torch.bfloat16 or tail.device != device or tail.ndim != 5 or \
                        tail.shape[2] != PAGE_SIZE or tail.shape[4] != 128 or not tail.is_contiguous() or \
                        tail.shape != tail_key.shape:
                    raise ValueError(f"{name} must be contiguous BF16 [layers, slots, 128, heads_kv, 128] on {device}")
        self.blocks, self.device, self._index = blocks, device, device.index
        self._lib = _lib.load()
        self.num_pages, self.block_bytes = int(shape[0]), int(shape[1])
        self.reserved_pages = reserved_pages
        self.refs = torch.zeros(self.num_pages, dtype=torch.int32, device=device) if refs is None else refs
        self._vector(self.refs, "refs", self.num_pages)
        self.tail_key, self.tail_value = tail_key, tail_value
        self.status = torch.zeros(1, dtype=torch.int32, device=device) if status is None else status
        self._vector(self.status, "status", 1)
        self._fork_tail = (None, None, 0, 0, 0, 0, 1) if tail_key is None else (
            tail_key.data_ptr(), tail_value.data_ptr(), tail_key.stride(0), tail_key.stride(1), tail_key.shape[0],
            tail_key.shape[1], tail_key.shape[3])
        self._bases = torch.tensor([b.data_ptr() for b in blocks], dtype=torch.int64, device=device)
        self._scratch = torch.empty(3 * self.num_pages + 1, dtype=torch.int32, device=device)
        if self._scratch.numel() * 4 < self._lib.nvfp4_pool_compact_workspace_bytes(self.num_pages):
            raise RuntimeError("the pool's scratch does not match the library's")

    # -- checks ------------------------------------------------------------------------------

    def _vector(self, tensor: torch.Tensor, name: str, length: int | None = None) -> int:
        if tensor.dtype is not torch.int32 or tensor.ndim != 1 or tensor.get_device() != self._index or \
                not tensor.is_contiguous() or (length is not None and tensor.shape[0] != length):
            want = "n" if length is None else length
            raise ValueError(f"{name} must be contiguous INT32 [{want}] on {self.device}")
        return tensor.data_ptr()

    def _table(self, page_table: torch.Tensor, pages_held: torch.Tensor) -> tuple[int, int, int, int, int]:
        if page_table.dtype is not torch.int32 or page_table.ndim != 2 or page_table.get_device() != self._index:
            raise ValueError(f"page_table must be INT32 [rows, columns] on {self.device}, dense within a row")
        rows, columns = page_table.shape
        row_stride, unit = page_table.stride()
        if (unit != 1 and columns > 1) or (row_stride < columns and rows > 1):
            raise ValueError(f"page_table must be INT32 [rows, columns] on {self.device}, dense within a row")
        return page_table.data_ptr(), row_stride, columns, rows, self._vector(pages_held, "pages_held", rows)

    def _call(self, call, *args) -> None:
        index = self._index
        if torch._C._cuda_getDevice() == index:
            code = call(*args, torch._C._cuda_getCurrentRawStream(index))
        else:
            with torch.cuda.device(index):
                code = call(*args, torch._C._cuda_getCurrentRawStream(index))
        if code:
            _lib.check(code)

    # -- operations --------------------------------------------------------------------------

    def release(self, rows: torch.Tensor, page_table: torch.Tensor, pages_held: torch.Tensor) -> None:
        """Give back what the rows of the list (INT32) hold; ``pages_held`` of them becomes 0.  A row named twice is
        released once; that, a row that does not exist and a page nobody holds set bits of ``status``."""
        table, stride, columns, count, held = self._table(page_table, pages_held)
        self._call(self._lib.nvfp4_pool_release, self._vector(rows, "rows"), rows.shape[0], table, stride, columns, count, held,
                   self.refs.data_ptr(), self.num_pages, self.status.data_ptr())

    def fork(self, sources: torch.Tensor, targets: torch.Tensor, page_table: torch.Tensor, pages_held: torch.Tensor,
             seqused_fp4: torch.Tensor, seqused_residual: torch.Tensor, row_to_slot: torch.Tensor | None = None) -> None:
        """Make row ``targets[i]`` a copy of row ``sources[i]`` (INT32 lists): its sealed pages shared, both lengths, and
        the tail tokens of every layer copied into slot ``row_to_slot[targets[i]]``.  A source may be named
        often.  A target must hold nothing (:meth:`release` it first), be named once and be no pair's source, and its
        slot must be no other named row's.  A pair that breaks one of these, or whose source has an unusable length,
        slot or page id, is skipped as a whole and sets a bit of ``status``.  Entries that the source holds
        beyond its sealed pages (a block for its open page) stay its own; a source that holds fewer pages than its
        length says gives those, without its tail, and sets a bit."""
        table, stride, columns, count, held = self._table(page_table, pages_held)
        if sources.shape != targets.shape:
            raise ValueError("sources and targets must have the same length")
        slots = None
        if self.tail_key is not None:
            if row_to_slot is None:
                raise ValueError("a pool with tails needs row_to_slot to fork")
            slots = self._vector(row_to_slot, "row_to_slot", count)
        self._call(self._lib.nvfp4_pool_fork, self._vector(sources, "sources"), self._vector(targets, "targets"),
                   sources.shape[0], table, stride, columns, count, held, self._vector(seqused_fp4, "seqused_fp4", count),
                   self._vector(seqused_residual, "seqused_residual", count), slots, self.refs.data_ptr(),
                   self.num_pages, *self._fork_tail, self.status.data_ptr())

    def compact(self, page_table: torch.Tensor, pages_held: torch.Tensor) -> torch.Tensor:
        """Move the live pages into the lowest ids, in every layer: with L of them, the k-th at or above L goes to the
        k-th free one below L.  Counts move along and the table's held entries are rewritten (one that names a page
        that nobody holds becomes -1 and sets a bit of ``status``); returns L (INT32 ``[1]`` on the device): pages
        from L on are free.  Every table that holds pages of the pool has to be the one given."""
        table, stride, columns, count, held = self._table(page_table, pages_held)
        live = torch.empty(1, dtype=torch.int32, device=self.device)
        self._call(self._lib.nvfp4_pool_compact, self._bases.data_ptr(), len(self.blocks), self.block_bytes, self.num_pages,
                   self.reserved_pages, self.refs.data_ptr(), table, stride, columns, count, held,
                   self._scratch.data_ptr(), self._scratch.numel() * 4, live.data_ptr(), self.status.data_ptr())
        return live

    def copy(self, source_pages: torch.Tensor, destination_pages: torch.Tensor, *,
             trusted_metadata: bool = False) -> None:
        """Copy page ``source_pages[i]`` over page ``destination_pages[i]`` in every layer (INT32 lists, -1 = nothing);
        counts stay.  No page may be in both lists or twice among the destinations (checked unless
        ``trusted_metadata``)."""
        if source_pages.shape != destination_pages.shape:
            raise ValueError("source_pages and destination_pages must have the same length")
        src = self._vector(source_pages, "source_pages")
        dst = self._vector(destination_pages, "destination_pages")
        if not trusted_metadata:
            pairs = [(s, d) for s, d in zip(source_pages.tolist(), destination_pages.tolist()) if s >= 0 and d >= 0]
            written = [d for _, d in pairs]
            if any(max(p) >= self.num_pages for p in pairs):
                raise ValueError(f"page ids must be below {self.num_pages}")
            if len(set(written)) != len(written) or set(written) & {s for s, _ in pairs}:
                raise ValueError("a page may be copied to once, and not from a page that is copied to")
        self._call(self._lib.nvfp4_pool_copy, self._bases.data_ptr(), len(self.blocks), self.block_bytes, self.num_pages, src,
                   dst, source_pages.shape[0], self.status.data_ptr())

    def free_list(self) -> tuple[torch.Tensor, torch.Tensor]:
        """The free pages, ascending, then -1 (INT32 ``[pages]``), and how many they are (INT32 ``[1]``)."""
        ids = torch.empty(self.num_pages, dtype=torch.int32, device=self.device)
        count = torch.empty(1, dtype=torch.int32, device=self.device)
        self._call(self._lib.nvfp4_pool_free_list, self.refs.data_ptr(), self.num_pages, self.reserved_pages, ids.data_ptr(),
                   count.data_ptr())
        return ids, count
