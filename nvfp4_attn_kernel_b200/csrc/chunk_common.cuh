// What the chunk kernels share: the cache they read and write, and the resolution of one row's
// share of it from device-resident metadata.
#pragma once

#include "nvfp4_common.cuh"
#include "nvfp4_kernels.h"
#include "../../include/nvfp4_b200.h"

namespace nvfp4 {

__device__ __forceinline__ void chunk_status(uint32_t* status, uint32_t bit) {
  if (status) atomicOr(status, bit);
}

// One row of a chunk call: `pages` sealed pages, `tail` tokens in tail page `tail_id`, `n` chunk
// tokens from `first` on.  Anything out of range is clamped and flagged, never made an address.
struct ChunkRow { int pages, tail, tail_id, first, n; uint32_t bad; };

__device__ __forceinline__ ChunkRow resolve_chunk_row(const ChunkCache& c, int row, bool report) {
  ChunkRow r;
  uint32_t bad = 0;
  const int fp4 = c.seqused_fp4[row];
  r.pages = fp4 < 0 ? 0 : fp4 >> 7;
  if (fp4 < 0 || (fp4 & 127) || r.pages > c.max_pages) {
    bad |= NVFP4_STATUS_BAD_LENGTH;
    r.pages = min(r.pages, c.max_pages);
  }
  r.tail = c.seqused_tail ? c.seqused_tail[row] : 0;
  r.tail_id = c.tail_ids ? c.tail_ids[row] : 0;
  if (r.tail < 0 || r.tail > kPage) {
    bad |= NVFP4_STATUS_BAD_LENGTH;
    r.tail = min(max(r.tail, 0), kPage);
  }
  if (r.tail > 0 && (r.tail_id < 0 || (int64_t)r.tail_id >= c.tail_pages)) {
    bad |= NVFP4_STATUS_BAD_TAIL_ID;
    r.tail = 0;
  }
  const int begin = c.chunk_start[row], end = c.chunk_start[row + 1];
  r.first = min(max(begin, 0), c.tokens);
  r.n = min(max(end, r.first), c.tokens) - r.first;
  if (begin != r.first || (int64_t)end - begin != r.n || r.n > c.max_chunk) {
    bad |= NVFP4_STATUS_BAD_LENGTH;
    r.n = min(r.n, c.max_chunk);
  }
  r.bad = bad;
  if (report && bad) chunk_status(c.status, bad);
  return r;
}

}  // namespace nvfp4
