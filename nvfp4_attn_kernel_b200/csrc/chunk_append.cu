// Writing a chunk of new tokens into the paged cache, and reading pages back.
//
// Row r's stream is its t tail tokens followed by its n chunk tokens.  Every full 128 tokens of
// the stream are quantised into a page (K in groups of 16 channels, V in groups of 16 tokens, the
// arithmetic of quantize_group16), what is left over becomes the new tail.  One CTA owns one head
// of one page column of one row, K or V, so nothing is shared between CTAs but the tail page: the
// first page is sealed from the old tail while the leftover overwrites it.  Both are therefore
// done by the same CTA, reads first, whenever both happen; else the leftover has a CTA of its own.
#include "chunk_common.cuh"

namespace nvfp4 {

namespace {

constexpr int kAppendThreads = 256;
constexpr int kTileWords = 65;   // a token's 128 bf16 as 64 words, one word of padding

struct AppendSmem {
  uint32_t tile[kPage * kTileWords];             // V: [token][channel pairs]
  __align__(16) uint8_t packed[kHeadDim * 64];   // V: [channel][64 B]
  __align__(16) uint8_t scales[kSfBlockBytes];
};

// Channels [g*16, g*16 + 16) of stream token p of this head: from the tail below t, else from the
// chunk, shifted.
__device__ __forceinline__ void load_group(const ChunkCache& c, const ChunkRow& r, int head, bool is_value, int p, int g,
                                           uint4& a, uint4& b) {
  const uint16_t* src;
  if (p < r.tail) {
    src = (is_value ? c.tail_value : c.tail_key) +
          (((int64_t)r.tail_id * kPage + p) * c.heads_kv + head) * kHeadDim + g * 16;
    a = *reinterpret_cast<const uint4*>(src);
    b = *reinterpret_cast<const uint4*>(src + 8);
    return;
  }
  const int64_t token = (int64_t)r.first + (p - r.tail);
  src = (is_value ? c.value + token * c.value_stride : c.key + token * c.key_stride) + head * kHeadDim + g * 16;
  a = *reinterpret_cast<const uint4*>(src);
  b = *reinterpret_cast<const uint4*>(src + 8);
  if (!is_value && c.key_shift) {
    const uint16_t* m = c.key_shift + head * kHeadDim + g * 16;
    float x[16], y[16];
    unpack_bf16x8(a, x);
    unpack_bf16x8(b, x + 8);
    unpack_bf16x8(*reinterpret_cast<const uint4*>(m), y);
    unpack_bf16x8(*reinterpret_cast<const uint4*>(m + 8), y + 8);
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {   // one BF16 subtract per channel, as the page quantiser's shift
      const __nv_bfloat162 d = __floats2bfloat162_rn(x[2 * i] - y[2 * i], x[2 * i + 1] - y[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
    a = make_uint4(w[0], w[1], w[2], w[3]);
    b = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

__device__ __forceinline__ void seal_key(const ChunkCache& c, const ChunkRow& r, AppendSmem& sm, int head, int column,
                                         int64_t page) {
  uint8_t* packed = c.k_packed + page * c.k_pitch;
#pragma unroll
  for (int k = 0; k < kPage * 8 / kAppendThreads; ++k) {
    const int it = threadIdx.x + k * kAppendThreads;
    const int tok = it >> 3, g = it & 7;
    uint4 a, b;
    load_group(c, r, head, false, column * kPage + tok, g, a, b);
    float x[16];
    unpack_bf16x8(a, x);
    unpack_bf16x8(b, x + 8);
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
#pragma unroll
  for (int k = 0; k < kPage * 8 / kAppendThreads; ++k) {
    const int it = threadIdx.x + k * kAppendThreads;
    const int tok = it >> 3, g = it & 7;
    uint4 a, b;
    load_group(c, r, head, true, column * kPage + tok, g, a, b);
    uint32_t* dst = sm.tile + tok * kTileWords + g * 8;
    dst[0] = a.x; dst[1] = a.y; dst[2] = a.z; dst[3] = a.w;
    dst[4] = b.x; dst[5] = b.y; dst[6] = b.z; dst[7] = b.w;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kHeadDim * 8 / kAppendThreads; ++k) {
    const int it = threadIdx.x + k * kAppendThreads;
    const int g = it >> 7, d = it & 127;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t w = sm.tile[(g * 16 + i) * kTileWords + (d >> 1)];
      x[i] = (d & 1) ? __uint_as_float(w & 0xFFFF0000u) : __uint_as_float(w << 16);
    }
    uint32_t lo, hi;
    uint8_t s;
    quantize_group16(x, lo, hi, s);
    *reinterpret_cast<uint2*>(sm.packed + d * 64 + g * 8) = make_uint2(lo, hi);
    sm.scales[sf_offset(d, g)] = s;
  }
  __syncthreads();
  uint4* packed = reinterpret_cast<uint4*>(c.v_packed + page * c.v_pitch + (int64_t)head * kHeadDim * 64);
  uint4* scales = reinterpret_cast<uint4*>(c.v_sf + page * c.v_sf_pitch + head * kSfBlockBytes);
  for (int i = threadIdx.x; i < kHeadDim * 64 / 16; i += kAppendThreads)
    packed[i] = reinterpret_cast<const uint4*>(sm.packed)[i];
  if (threadIdx.x < kSfBlockBytes / 16) scales[threadIdx.x] = reinterpret_cast<const uint4*>(sm.scales)[threadIdx.x];
}

// grid (heads_kv * 2, columns, rows)
__global__ void __launch_bounds__(kAppendThreads)
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
  // a row with unusable metadata keeps what it has
  const bool tail_ok = rest == 0 || (r.tail_id >= 0 && (int64_t)r.tail_id < c.tail_pages);
  const bool refused = r.bad || full_table || !tail_ok;
  if (speaker && threadIdx.x == 0) {
    if (full_table) chunk_status(c.status, NVFP4_STATUS_BAD_LENGTH);
    if (!tail_ok) chunk_status(c.status, NVFP4_STATUS_BAD_TAIL_ID);
    seqused_fp4_out[row] = refused ? c.seqused_fp4[row] : (r.pages + sealed) * kPage;
    seqused_tail_out[row] = refused ? c.seqused_tail[row] : rest;
  }
  if (refused) return;
  if (column < sealed) {
    const int64_t page = c.page_table[(int64_t)row * c.page_table_row_stride + r.pages + column];
    if (page < 0 || page >= c.num_pages) {
      if (threadIdx.x == 0) chunk_status(c.status, NVFP4_STATUS_BAD_PAGE_ID);
    } else if (is_value) {
      seal_value(c, r, sm, head, column, page);
    } else {
      seal_key(c, r, sm, head, column, page);
    }
  }
  // the leftover: behind the first page's reads of the old tail when both happen, else on its own
  const int owner = r.tail > 0 && sealed > 0 ? 0 : sealed;
  if (column != owner || rest == 0) return;
  __syncthreads();
  const int begin = sealed ? 0 : r.tail;                  // tail positions [begin, rest) change
  uint16_t* tail = (is_value ? c.tail_value : c.tail_key) + ((int64_t)r.tail_id * kPage * c.heads_kv + head) * kHeadDim;
  for (int it = threadIdx.x; it < (rest - begin) * 8; it += kAppendThreads) {
    const int p = begin + (it >> 3), g = it & 7;
    uint4 a, b;
    load_group(c, r, head, is_value, sealed * kPage + p, g, a, b);
    uint16_t* dst = tail + (int64_t)p * c.heads_kv * kHeadDim + g * 16;
    *reinterpret_cast<uint4*>(dst) = a;
    *reinterpret_cast<uint4*>(dst + 8) = b;
  }
}

// 16 nibbles of one group times its scale, as BF16 (exact: at most six significant bits).
__device__ __forceinline__ void dequantize_group(uint2 nibbles, uint8_t scale, float (&x)[16]) {
  const float s = e4m3_to_f32(scale);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = e2m1_to_f32(nibbles.x >> (4 * i)) * s;
    x[8 + i] = e2m1_to_f32(nibbles.y >> (4 * i)) * s;
  }
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// grid (pages, heads_kv * 2)
__global__ void __launch_bounds__(kAppendThreads)
dequantize_pages_kernel(const ChunkCache c, const int32_t* __restrict__ page_ids, uint16_t* __restrict__ key_out,
                        uint16_t* __restrict__ value_out) {
  __shared__ uint32_t tile[kPage * kTileWords];
  const int item = blockIdx.x;
  const bool is_value = (int)blockIdx.y >= c.heads_kv;
  const int head = is_value ? blockIdx.y - c.heads_kv : blockIdx.y;
  const int64_t page = page_ids[item];
  const bool valid = page >= 0 && page < c.num_pages;
  if (!valid && blockIdx.y == 0 && threadIdx.x == 0) chunk_status(c.status, NVFP4_STATUS_BAD_PAGE_ID);
  const int64_t first = (int64_t)item * kPage;
  uint16_t* out = (is_value ? value_out : key_out) + (first * c.heads_kv + head) * kHeadDim;
  const int64_t pitch = (int64_t)c.heads_kv * kHeadDim;
  if (!is_value) {
#pragma unroll
    for (int k = 0; k < kPage * 8 / kAppendThreads; ++k) {
      const int it = threadIdx.x + k * kAppendThreads;
      const int tok = it >> 3, g = it & 7;
      uint4 a = make_uint4(0, 0, 0, 0), b = a;
      if (valid) {
        const uint2 n = *reinterpret_cast<const uint2*>(c.k_packed + page * c.k_pitch +
                                                        ((int64_t)tok * c.heads_kv + head) * 64 + g * 8);
        float x[16];
        dequantize_group(n, c.k_sf[page * c.k_sf_pitch + head * kSfBlockBytes + sf_offset(tok, g)], x);
        a = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
        b = make_uint4(pack_bf16(x[8], x[9]), pack_bf16(x[10], x[11]), pack_bf16(x[12], x[13]), pack_bf16(x[14], x[15]));
      }
      uint16_t* dst = out + tok * pitch + g * 16;
      *reinterpret_cast<uint4*>(dst) = a;
      *reinterpret_cast<uint4*>(dst + 8) = b;
    }
    return;
  }
  if (valid) {
    uint16_t* half = reinterpret_cast<uint16_t*>(tile);
#pragma unroll
    for (int k = 0; k < kHeadDim * 8 / kAppendThreads; ++k) {
      const int it = threadIdx.x + k * kAppendThreads;
      const int g = it >> 7, d = it & 127;
      const uint2 n = *reinterpret_cast<const uint2*>(c.v_packed + page * c.v_pitch +
                                                      ((int64_t)head * kHeadDim + d) * 64 + g * 8);
      float x[16];
      dequantize_group(n, c.v_sf[page * c.v_sf_pitch + head * kSfBlockBytes + sf_offset(d, g)], x);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        half[(g * 16 + i) * (2 * kTileWords) + d] = (uint16_t)(__float_as_uint(x[i]) >> 16);   // exact in BF16
    }
  }
  __syncthreads();
  for (int it = threadIdx.x; it < kPage * 16; it += kAppendThreads) {
    const int tok = it >> 4, q = it & 15;
    const uint32_t* src = tile + tok * kTileWords + q * 4;
    *reinterpret_cast<uint4*>(out + tok * pitch + q * 8) =
        valid ? make_uint4(src[0], src[1], src[2], src[3]) : make_uint4(0, 0, 0, 0);
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
