// Writing a chunk of new tokens into the paged cache, and reading pages back.
//
// Row r's stream is its t tail tokens followed by its n chunk tokens.  Every full 128 tokens of
// the stream are quantised into a page (K in groups of 16 channels, V in groups of 16 tokens, the
// arithmetic of quantize_group16), what is left over becomes the new tail.  One CTA owns one head
// of one page column of one row, K or V, so nothing is shared between CTAs but the tail page: the
// first page is sealed from the old tail while the leftover overwrites it.  Both are therefore
// done by the same CTA, reads first, whenever both happen; else the leftover has a CTA of its own.
#include <cuda_fp16.h>

#include "chunk_common.cuh"

namespace nvfp4 {

namespace {

constexpr int kAppendThreads = 256;
// Word of channel pair `pair` of a token in the V tile: one word of padding a token, and four more per group of 16
// tokens, so that a warp that reads four pairs of a token of each group has every lane in a bank of its own.
__device__ __forceinline__ int tile_word(int tok, int pair) { return tok * 65 + (tok >> 4) * 4 + pair; }

struct AppendSmem {
  uint32_t tile[kPage * 65 + 7 * 4];             // V: [token][channel pairs]
  __align__(16) uint8_t scales[kSfBlockBytes];
};

// Channels [g*16, g*16 + 16) of stream token p of this head: from the tail below t, else from the chunk.
__device__ __forceinline__ const uint4* group_at(const ChunkCache& c, const ChunkRow& r, int head, bool is_value, int p, int g) {
  const uint16_t* src;
  if (p < r.tail) {
    src = (is_value ? c.tail_value : c.tail_key) + ((int64_t)r.tail_id * kPage + p) * c.heads_kv * kHeadDim;
  } else {
    const int64_t token = (int64_t)r.first + (p - r.tail);
    src = is_value ? c.value + token * c.value_stride : c.key + token * c.key_stride;
  }
  return reinterpret_cast<const uint4*>(src + head * kHeadDim + g * 16);
}

// The key shift's 16 channels of a group, as fp32.
__device__ __forceinline__ void load_shift(const ChunkCache& c, int head, int g, float (&m)[16]) {
  const uint4* at = reinterpret_cast<const uint4*>(c.key_shift + head * kHeadDim + g * 16);
  unpack_bf16x8(at[0], m);
  unpack_bf16x8(at[1], m + 8);
}

__device__ __forceinline__ uint4 pack_bf16x8(const float* x) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 d = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&d);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

constexpr int kItems = kPage * 8 / kAppendThreads;   // groups of a page and head per thread

__device__ __forceinline__ void seal_key(const ChunkCache& c, const ChunkRow& r, AppendSmem& sm, int head, int column,
                                         int64_t page) {
  uint8_t* packed = c.k_packed + page * c.k_pitch;
  const int g = threadIdx.x & 7, tok0 = threadIdx.x >> 3;     // a thread keeps its group of channels
  uint4 a[kItems], b[kItems];
#pragma unroll
  for (int k = 0; k < kItems; ++k) {      // every load of the thread first: the kernel lives on loads in flight
    const uint4* at = group_at(c, r, head, false, column * kPage + tok0 + k * (kAppendThreads / 8), g);
    a[k] = at[0];
    b[k] = at[1];
  }
  float shift[16];
  if (c.key_shift) load_shift(c, head, g, shift);
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int tok = tok0 + k * (kAppendThreads / 8);
    float x[16];
    unpack_bf16x8(a[k], x);
    unpack_bf16x8(b[k], x + 8);
    if (c.key_shift && column * kPage + tok >= r.tail) {      // one BF16 subtract per channel; the tail's are shifted
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = __bfloat162float(__float2bfloat16_rn(x[i] - shift[i]));
    }
    uint32_t lo, hi;
    uint8_t s;
    quantize_group16(x, lo, hi, s);
    *reinterpret_cast<uint2*>(packed + ((int64_t)tok * c.heads_kv + head) * 64 + g * 8) = make_uint2(lo, hi);
    sm.scales[sf_offset(tok, g)] = s;
  }
  __syncthreads();
  uint8_t* scales = c.k_sf + page * c.k_sf_pitch + head * kSfBlockBytes;
  if (threadIdx.x < kSfBlockBytes / 16)
    reinterpret_cast<uint4*>(scales)[threadIdx.x] = reinterpret_cast<const uint4*>(sm.scales)[threadIdx.x];
}

__device__ __forceinline__ void seal_value(const ChunkCache& c, const ChunkRow& r, AppendSmem& sm, int head, int column,
                                           int64_t page) {
  {
    const int g = threadIdx.x & 7, tok0 = threadIdx.x >> 3;
    uint4 a[kItems], b[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const uint4* at = group_at(c, r, head, true, column * kPage + tok0 + k * (kAppendThreads / 8), g);
      a[k] = at[0];
      b[k] = at[1];
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      uint32_t* dst = sm.tile + tile_word(tok0 + k * (kAppendThreads / 8), g * 8);
      dst[0] = a[k].x; dst[1] = a[k].y; dst[2] = a[k].z; dst[3] = a[k].w;
      dst[4] = b[k].x; dst[5] = b[k].y; dst[6] = b[k].z; dst[7] = b[k].w;
    }
  }
  __syncthreads();
  // a thread takes 16 tokens of two neighbouring channels; eight lanes store the 64 bytes of a channel
  uint8_t* packed = c.v_packed + page * c.v_pitch + (int64_t)head * kHeadDim * 64;
  const int g = threadIdx.x & 7;
#pragma unroll
  for (int k = 0; k < kItems / 2; ++k) {
    const int pair = (threadIdx.x >> 3) + k * (kAppendThreads / 8);
    float even[16], odd[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t w = sm.tile[tile_word(g * 16 + i, pair)];
      even[i] = __uint_as_float(w << 16);
      odd[i] = __uint_as_float(w & 0xFFFF0000u);
    }
    uint32_t lo, hi;
    uint8_t s;
    quantize_group16(even, lo, hi, s);
    *reinterpret_cast<uint2*>(packed + 2 * pair * 64 + g * 8) = make_uint2(lo, hi);
    sm.scales[sf_offset(2 * pair, g)] = s;
    quantize_group16(odd, lo, hi, s);
    *reinterpret_cast<uint2*>(packed + (2 * pair + 1) * 64 + g * 8) = make_uint2(lo, hi);
    sm.scales[sf_offset(2 * pair + 1, g)] = s;
  }
  __syncthreads();
  uint4* scales = reinterpret_cast<uint4*>(c.v_sf + page * c.v_sf_pitch + head * kSfBlockBytes);
  if (threadIdx.x < kSfBlockBytes / 16) scales[threadIdx.x] = reinterpret_cast<const uint4*>(sm.scales)[threadIdx.x];
}

// grid (heads_kv * 2, columns, rows).  512 bytes in and 144 out per token and head, bound by the loads in flight: 64
// registers, so four CTAs an SM: 8 rows x 2048 tokens of 8 heads 19.1 us (61 MB, 3.2 TB/s; 18.5 without the look at the
// row's pages); 80 registers and three CTAs 20.3 us, 48 and five (with spills) 22.4 us.  4 rows x 5 tokens: 2.6 us, a launch
// and loads that follow one another.
__global__ void __launch_bounds__(kAppendThreads, 4)
append_chunk_kernel(const ChunkCache c, int32_t* seqused_fp4_out, int32_t* seqused_tail_out) {
  __shared__ AppendSmem sm;
  const int row = blockIdx.z, column = blockIdx.y;
  const bool is_value = (int)blockIdx.x >= c.heads_kv;
  const int head = is_value ? blockIdx.x - c.heads_kv : blockIdx.x;
  const bool speaker = blockIdx.x == 0 && column == 0;
  const ChunkRow r = resolve_chunk_row(c, row, speaker && threadIdx.x == 0);
  const int total = r.tail + r.n;
  const int room = c.max_pages - r.pages;                 // table columns that are left
  const int sealed = min(total >> 7, room);
  const int rest = total - sealed * kPage;                // > 127 only when the table is full
  const bool full_table = rest >= kPage;
  if (column > sealed) return;                            // neither a page nor the leftover is this CTA's
  // A row with unusable metadata keeps what it has.  So every CTA of a row looks at every page that the row would write
  // (page ids are few beside a page's bytes) and all come to one verdict before any of them writes.
  const bool tail_ok = rest == 0 || (r.tail_id >= 0 && (int64_t)r.tail_id < c.tail_pages);
  const int32_t* pages = c.page_table + (int64_t)row * c.page_table_row_stride + r.pages;
  bool missing = false;
  for (int i = threadIdx.x; i < sealed; i += kAppendThreads) missing = missing || pages[i] < 0 || pages[i] >= c.num_pages;
  missing = __syncthreads_or(missing);
  const bool refused = r.bad || full_table || !tail_ok || missing;
  if (speaker && threadIdx.x == 0) {
    if (full_table) chunk_status(c.status, NVFP4_STATUS_BAD_LENGTH);
    if (!tail_ok) chunk_status(c.status, NVFP4_STATUS_BAD_TAIL_ID);
    if (missing) chunk_status(c.status, NVFP4_STATUS_BAD_PAGE_ID);
    seqused_fp4_out[row] = refused ? c.seqused_fp4[row] : (r.pages + sealed) * kPage;
    seqused_tail_out[row] = refused ? c.seqused_tail[row] : rest;
  }
  if (refused) return;
  if (column < sealed) {
    const int64_t page = pages[column];
    if (is_value) seal_value(c, r, sm, head, column, page);
    else seal_key(c, r, sm, head, column, page);
  }
  // the leftover: behind the first page's reads of the old tail when both happen, else on its own
  const int owner = r.tail > 0 && sealed > 0 ? 0 : sealed;
  if (column != owner || rest == 0) return;
  __syncthreads();
  const int begin = sealed ? 0 : r.tail;                  // tail positions [begin, rest) change
  uint16_t* tail = (is_value ? c.tail_value : c.tail_key) + ((int64_t)r.tail_id * kPage * c.heads_kv + head) * kHeadDim;
  for (int it = threadIdx.x; it < (rest - begin) * 8; it += kAppendThreads) {
    const int p = begin + (it >> 3), g = it & 7;
    const uint4* at = group_at(c, r, head, is_value, sealed * kPage + p, g);
    uint4 a = at[0], b = at[1];
    if (!is_value && c.key_shift) {      // (the leftover is the chunk's: what the tail keeps stays where it is)
      float x[16], m[16];
      unpack_bf16x8(a, x);
      unpack_bf16x8(b, x + 8);
      load_shift(c, head, g, m);
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] -= m[i];
      a = pack_bf16x8(x);
      b = pack_bf16x8(x + 8);
    }
    uint16_t* dst = tail + (int64_t)p * c.heads_kv * kHeadDim + g * 16;
    *reinterpret_cast<uint4*>(dst) = a;
    *reinterpret_cast<uint4*>(dst + 8) = b;
  }
}

// Eight nibbles times their scale (an FP16 pair of it) as BF16 pairs, in order: exact, since the product has at most
// six significant bits, which both formats hold.
__device__ __forceinline__ uint4 dequantize8(uint32_t nibbles, uint32_t scale2) {
  uint32_t h[4], r[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(nibbles));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&h[i]), *reinterpret_cast<const __half2*>(&scale2));
    const float2 f = __half22float2(v);
    const __nv_bfloat162 o = __floats2bfloat162_rn(f.x, f.y);
    r[i] = *reinterpret_cast<const uint32_t*>(&o);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}
__device__ __forceinline__ uint32_t scale_pair(uint8_t e4m3) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)(e4m3 * 0x0101)));
  return h;
}

constexpr int kOutWords = 68;   // a token's 64 channel pairs and four words of padding: 16-byte rows
// Word of channel pair `pair` of a token in the V tile.  Eight more words per 32 tokens: a warp stores eight pairs of
// four tokens that are 32 apart, each lane then in a bank of its own.
__device__ __forceinline__ int out_word(int tok, int pair) { return tok * kOutWords + (tok >> 5) * 8 + pair; }

// grid (pages, heads_kv * 2).  K rows are rows of the result: four bytes in, sixteen out per thread.  V is packed along the
// tokens: a thread takes 32 tokens of two neighbouring channels, and the page is turned in shared memory.  Bound by
// memory: 144 bytes in and 512 out per token and head; 256 pages of 8 heads 32 us (5.4 TB/s), 90
// pages just written 9.7 us (6.3 TB/s).
__global__ void __launch_bounds__(kAppendThreads)
dequantize_pages_kernel(const ChunkCache c, const int32_t* __restrict__ page_ids, uint16_t* __restrict__ key_out,
                        uint16_t* __restrict__ value_out) {
  __shared__ __align__(16) uint32_t tile[kPage * kOutWords + 3 * 8];
  const int item = blockIdx.x;
  const bool is_value = (int)blockIdx.y >= c.heads_kv;
  const int head = is_value ? blockIdx.y - c.heads_kv : blockIdx.y;
  const int64_t page = page_ids[item];
  const bool valid = page >= 0 && page < c.num_pages;
  if (!valid && blockIdx.y == 0 && threadIdx.x == 0) chunk_status(c.status, NVFP4_STATUS_BAD_PAGE_ID);
  uint16_t* out = (is_value ? value_out : key_out) + ((int64_t)item * kPage * c.heads_kv + head) * kHeadDim;
  const int64_t pitch = (int64_t)c.heads_kv * kHeadDim;
  const int part = threadIdx.x & 15;      // of a row of the result: eight channels
  if (!valid) {
    for (int tok = threadIdx.x >> 4; tok < kPage; tok += kAppendThreads / 16)
      *reinterpret_cast<uint4*>(out + tok * pitch + part * 8) = make_uint4(0, 0, 0, 0);
    return;
  }
  if (!is_value) {
    const uint8_t* packed = c.k_packed + page * c.k_pitch + head * 64 + part * 4;
    const uint8_t* scales = c.k_sf + page * c.k_sf_pitch + head * kSfBlockBytes;
    uint32_t n[8];
    uint8_t s[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int tok = (threadIdx.x >> 4) + k * (kAppendThreads / 16);
      n[k] = __ldg(reinterpret_cast<const uint32_t*>(packed + (int64_t)tok * c.heads_kv * 64));
      s[k] = __ldg(scales + sf_offset(tok, part >> 1));
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int tok = (threadIdx.x >> 4) + k * (kAppendThreads / 16);
      *reinterpret_cast<uint4*>(out + tok * pitch + part * 8) = dequantize8(n[k], scale_pair(s[k]));
    }
    return;
  }
  {
    const int piece = threadIdx.x & 3, pair = threadIdx.x >> 2;       // tokens 32 * piece ..., channels 2 * pair and the next
    const uint8_t* packed = c.v_packed + page * c.v_pitch + ((int64_t)head * kHeadDim + 2 * pair) * 64 + piece * 16;
    const uint8_t* scales = c.v_sf + page * c.v_sf_pitch + head * kSfBlockBytes;
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(packed)), b = __ldg(reinterpret_cast<const uint4*>(packed + 64));
    const uint32_t wa[4] = {a.x, a.y, a.z, a.w}, wb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const uint32_t sa = scale_pair(__ldg(scales + sf_offset(2 * pair, 2 * piece + g)));
      const uint32_t sb = scale_pair(__ldg(scales + sf_offset(2 * pair + 1, 2 * piece + g)));
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint4 x = dequantize8(wa[2 * g + half], sa), y = dequantize8(wb[2 * g + half], sb);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
        const int tok = piece * 32 + g * 16 + half * 8;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          tile[out_word(tok + 2 * i, pair)] = __byte_perm(xs[i], ys[i], 0x5410);
          tile[out_word(tok + 2 * i + 1, pair)] = __byte_perm(xs[i], ys[i], 0x7632);
        }
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int tok = (threadIdx.x >> 4) + k * (kAppendThreads / 16);
    *reinterpret_cast<uint4*>(out + tok * pitch + part * 8) = *reinterpret_cast<const uint4*>(tile + out_word(tok, part * 4));
  }
}

}  // namespace

cudaError_t launch_append_chunk(const ChunkCache& c, int32_t* seqused_fp4_out, int32_t* seqused_tail_out,
                                cudaStream_t stream) {
  // at most (128 + max_chunk) / 128 sealed pages, and a column for a leftover of its own
  const dim3 grid(2 * c.heads_kv, (kPage + c.max_chunk) / kPage + 1, c.rows);
  append_chunk_kernel<<<grid, kAppendThreads, 0, stream>>>(c, seqused_fp4_out, seqused_tail_out);
  return cudaGetLastError();
}

cudaError_t launch_dequantize_pages(const ChunkCache& c, const int32_t* page_ids, int count, void* key_out,
                                    void* value_out, cudaStream_t stream) {
  dequantize_pages_kernel<<<dim3(count, 2 * c.heads_kv), kAppendThreads, 0, stream>>>(
      c, page_ids, static_cast<uint16_t*>(key_out), static_cast<uint16_t*>(value_out));
  return cudaGetLastError();
}

}  // namespace nvfp4
