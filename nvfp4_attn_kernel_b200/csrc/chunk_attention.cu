// Attention of a chunk of new tokens over the paged cache and, causally, over the chunk itself.
//
// Token i of a row sees h history tokens (sealed NVFP4 pages, then the BF16 tail) and the chunk's
// tokens 0..i.  The G query heads of a KV head and the tokens of a chunk are packed into tiles of
// 128 query rows, so a K/V tile that has been read (and dequantised) once serves all of them.  A CTA
// takes one KV head of one row and two streams of work, S = Q K^T and O += P V on the tensor cores
// (tcgen05, kind::f16, fp32 accumulators in tensor memory: 512 columns, all of them), a softmax warpgroup each:
//   - two tiles of query rows over the same K/V tiles, when the chunk has more than one, or
//   - one tile of query rows whose K/V tiles the streams take in turns, joined at the end.
// While one stream computes its softmax the tensor cores work for the other.  Beside the two softmax warpgroups one
// makes K operands and one V operands (dequantising pages that a warp for each fetches with tensor copies, or
// copying BF16 rows), a warp per stream issues the products.  Waits are bounded; an expired one sets a status bit.
//
// Operands.  A page's e2m1 * e4m3 is exact in FP16 (six significant bits, 2^-10 to 2688), and FP16
// probabilities carry eleven bits (down to 2^-21 of the row's largest: kAboveLog2), so pages meet an FP16 query: a BF16
// query row whose largest magnitude is scaled to [1, 2) by a power of two is exact in FP16 down to 2^-17 of that (the
// last of its eight bits at 2^-24), and what is smaller is off by at most 2^-25 of it, which moves a score by at most 2^-25
// of the row's largest magnitude times the key's sum of magnitudes.  Tail and chunk are BF16 as they lie in memory and
// meet the BF16 query and BF16 probabilities.  The BF16 tiles come first; then each query tile is
// converted in place, once.
//
// Softmax.  A thread owns a query row: running maximum and sum in fp32, exponentials of the scaled
// scores relative to a maximum that is only replaced when a new one exceeds it by 2^8 (O and the sum are
// rescaled then).  A chunk token whose
// value is not finite makes earlier tokens of its 128-token tile not finite too (0 * inf in the product).
//
// Probabilities are rounded (BF16 over chunk and tail, FP16 over pages) and the sum they are divided by is of the unrounded
// ones.  Where most tiles are BF16 the outputs are then 0.0019 off the 64-bit result (2-norm, 7 rows of up to 777 tokens
// after up to 5000), of which 0.0016 are the BF16 result's own rounding.  Carrying 16 bits (what the first rounding took off
// in a second BF16 operand, P V twice) leaves 0.0016 and was slower: these rows 238 -> 253 us, 4 fresh prompts of 2048
// tokens 213 -> 263 us, 2 x 2048 tokens after 32768 2190 -> 2295 us; eight bits match the result's.
//
// What bounds it: long chunks, the chain scores -> softmax -> P V of the two streams: of about 3900 clocks per pair of
// tiles the products take 2048 and the exponentials 2048, side by side, and neither pipe is busy more than 57 % of the
// time; the rest is the softmax warpgroups' other instructions and their waits (with the softmax left out the products run
// at 1430 TFLOP/s).  1152 tokens of 32 / 8 heads over 16384 tokens: 276 us = 1161 TFLOP/s, 0.70 of a large library
// product's burst rate.  A CTA spends about 10 us before
// and after its tiles (query rows in, the first products, rows out).  Short chunks: 128-row products for a few live rows
// (1024 clocks a tile) and a tile's way through dequantisation, scores, softmax and P V, 1700 clocks a tile: 32 rows x 4
// tokens over 4096 tokens 85 us for 160 MB.
#include <cuda_fp16.h>

#include <atomic>

#include "chunk_common.cuh"
#include "sm100_device.cuh"

namespace nvfp4 {

namespace {

using namespace sm100;

constexpr int kThreads = 640;         // warpgroups: softmax of two streams, K operands, V operands, issuers and fetch
constexpr int kIssueWarp = 16;        // and 17: one per stream
constexpr int kFetchWarp = 18;        // page bytes of K; 19: of V
constexpr int kOperandBytes = 128 * 256;       // 128 rows of 128 16-bit elements: two 128-byte swizzled halves
constexpr int kHalfBytes = 128 * 128;
constexpr int kRawBytes = 8192 + 1024;         // a page's nibbles and scales for one head
// Probabilities are formed as 2^kAboveLog2 times those relative to the row's maximum, which is only replaced when a new one
// exceeds it by 2^kRescaleLog2: 2^15 at most, below FP16's 65504.  FP16 holds what is below 2^-14 in steps of 2^-24, so a
// key's probability is off by at most 2^-11 of itself or 2^-32 of the row's largest, whichever is more (formed as they are,
// without the 2^7, 2^-25: a long flat history beside one strong key then loses its share).  More of the range above
// the maximum and less before a replacement, 2^11 and 2^4, costs replacements: 512 tokens after 16384 186 us instead of 159.
constexpr float kAboveLog2 = 7.f, kRescaleLog2 = 8.f;
constexpr uint32_t kColS = 0, kColO = 256;     // tensor-memory columns of stream 0; stream 1: + 128
constexpr float kLn2 = 0.6931471805599453f;

// What a CTA works on.
struct Work {
  ChunkRow r;
  int group, tile_tokens;      // query heads per KV head; tokens in a tile of query rows
  int token0;                  // first chunk token of tile 0
  bool two;                    // two tiles of query rows; else one, the streams taking turns
  bool apart;                  // one tile of at most 64 rows: rows 0..63 are stream 0's, their copies 64..127 stream 1's
  int fresh, tail_tiles;       // K/V tiles: the chunk's, then the tail's (0 or 1), then the pages
  int begin, end;              // this split's range of them
  int bf16_tiles;              // of these, how many are BF16
  int steps;                   // softmax steps of both streams together
};

// QTILES query tiles in shared memory, RAW slots of page bytes in flight, RAWK of them for K.  (A ring per operand: a
// waiter on a slot's barrier has to have seen each of its phases, and loads do not land in the order of their issue.)
template <int QTILES, int RAW>
struct ChunkSmem {
  static constexpr int kQTiles = QTILES, kRaw = RAW, kRawK = (RAW + 1) / 2, kRawV = RAW - kRawK;
  uint8_t q[QTILES][kOperandBytes];
  uint8_t k[2][kOperandBytes];
  uint8_t v[2][kOperandBytes];
  uint8_t raw[RAW][kRawBytes];
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t q_ready[2], q_f16[2], s_full[2][2], p_ready[2][2], o_done[2], all_done;
  uint64_t raw_full[RAW], raw_empty[RAW];
  float join[2][2][128];     // [stream] maximum and sum, when the streams share a tile; first the row's exponent and shift
  int page_ok[2][8];         // whether K's, V's page of tile t was fetched (0: a refused id), at t % 8: K's fetch is at
                             // most seven tiles ahead of the softmax, V's five ahead of its operand
  uint32_t tmem_base;
  Work work;
  volatile int abort_flag;
};

__device__ __forceinline__ uint32_t swizzled(int row, int unit) {   // 16-byte unit 0..15 of a row
  return (uint32_t)((unit >> 3) * kHalfBytes + row * 128 + (((unit ^ row) & 7) << 4));
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  const uint32_t bytes = valid ? 16 : 0;     // 0: the destination is zero-filled
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// Descriptors of a 16-bit operand tile, 128-byte swizzle, eight-row groups 1024 bytes apart.  K-major:
// a row's 64 elements are contiguous (the leading offset is not used).  MN-major (V of BF16 tiles, rows
// are tokens): the leading offset leads to the next 64 channels.
__device__ __forceinline__ uint64_t desc_k_major(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(kHalfBytes >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// M = 128, fp32 accumulators; A and B both FP16 or both BF16
__device__ __forceinline__ uint32_t idesc(bool bf16, bool b_mn_major, uint32_t n) {
  const uint32_t f = bf16 ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

__device__ __forceinline__ bool elect_one() {
  uint32_t leader;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(leader));
  return leader != 0;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(id), "r"(accumulate)
      : "memory");
}

#define NVFP4_R8(a, i) "=r"(a[i]), "=r"(a[i + 1]), "=r"(a[i + 2]), "=r"(a[i + 3]), "=r"(a[i + 4]), "=r"(a[i + 5]), "=r"(a[i + 6]), "=r"(a[i + 7])
#define NVFP4_W8(a, i) "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3]), "r"(a[i + 4]), "r"(a[i + 5]), "r"(a[i + 6]), "r"(a[i + 7])

// 32 columns of this warp's 32 lanes; the caller waits (tmem_ld_wait)
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : NVFP4_R8(r, 0), NVFP4_R8(r, 8), NVFP4_R8(r, 16), NVFP4_R8(r, 24)
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      NVFP4_W8(r, 0), NVFP4_W8(r, 8), NVFP4_W8(r, 16), NVFP4_W8(r, 24)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr), NVFP4_W8(r, 0), NVFP4_W8(r, 8)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Four bytes of nibbles -> four FP16 pairs (nibble 2i in the low half of pair i).
__device__ __forceinline__ void e2m1x8_to_f16x8(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
  return h;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Tensor maps of the packed page regions.
struct ChunkMaps { CUtensorMap k, v; };

__device__ __forceinline__ int stream_steps(const Work& w, int stream) {
  return w.two ? w.end - w.begin : (w.end - w.begin + 1 - stream) >> 1;
}

// The biased exponent e of a query row's largest magnitude (BF16 bits without sign): the row times 2^(127 - e)
// lies within [1, 2).  Both powers of two are normal numbers: e from 1 (zero and subnormal rows) to 253 (the two
// largest binades end below 4 instead); rows that are not finite stay as they are.
__device__ __forceinline__ int row_exponent(uint32_t amax_bits) {
  const int e = amax_bits >> 7;
  return e == 255 ? 127 : min(max(e, 1), 253);
}
__device__ __forceinline__ float exponent_value(int biased) { return __uint_as_float((uint32_t)biased << 23); }
__device__ __forceinline__ uint32_t bf16x2_to_f16x2(uint32_t w, float factor) {
  const __half2 h = __floats2half2_rn(__uint_as_float(w << 16) * factor, __uint_as_float(w & 0xFFFF0000u) * factor);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint4 bf16x8_to_f16x8(const uint4& v, float f) {
  return make_uint4(bf16x2_to_f16x2(v.x, f), bf16x2_to_f16x2(v.y, f), bf16x2_to_f16x2(v.z, f), bf16x2_to_f16x2(v.w, f));
}

// -- producers -----------------------------------------------------------------------------------

template <class SM>
struct Producer {
  const ChunkAttention& a;
  SM& sm;
  const Work& w;
  int kvh, warp, lane;

  // 128 tokens of BF16 rows straight into an operand tile
  __device__ __forceinline__ void issue_bf16(int tile, bool is_v, uint32_t dst) {
    const ChunkCache& c = a.c;
    const uint16_t* src;
    int64_t stride;
    int valid;
    if (tile < w.fresh) {
      stride = is_v ? c.value_stride : c.key_stride;
      src = (is_v ? c.value : c.key) + ((int64_t)w.r.first + tile * 128) * stride + kvh * kHeadDim;
      valid = min(128, w.r.n - tile * 128);
    } else {
      stride = (int64_t)c.heads_kv * kHeadDim;
      src = (is_v ? c.tail_value : c.tail_key) + (int64_t)w.r.tail_id * kPage * stride + kvh * kHeadDim;
      valid = w.r.tail;
    }
    const int unit = lane & 15;
#pragma unroll 4
    for (int i = 0; i < 16; ++i) {
      const int tok = warp * 32 + i * 2 + (lane >> 4);
      const bool ok = tok < valid;
      cp_async16(dst + swizzled(tok, unit), src + (ok ? tok : 0) * stride + unit * 8, ok);
    }
  }

  // row warp * 32 + lane of a raw slot (the fetch's 64-byte swizzle undone), dequantised into an operand tile; a
  // refused page: zeros (its scores are masked)
  __device__ __forceinline__ void expand(const uint8_t* slot, uint8_t* dst, bool valid) {
    const int r = warp * 32 + lane;
    const uint8_t* scales = slot + 8192 + lane * 16 + warp * 4;
    const uint32_t s[2] = {*reinterpret_cast<const uint32_t*>(scales), *reinterpret_cast<const uint32_t*>(scales + 512)};
    uint4 n[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) n[p] = *reinterpret_cast<const uint4*>(slot + r * 64 + ((p ^ ((r >> 1) & 3)) << 4));
    if (!valid) {
#pragma unroll
      for (int p = 0; p < 16; ++p) *reinterpret_cast<uint4*>(dst + swizzled(r, p)) = make_uint4(0, 0, 0, 0);
      return;
    }
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const uint32_t two = e4m3x2_to_f16x2(s[p >> 1] >> ((p & 1) * 16));
      const uint32_t s0 = __byte_perm(two, two, 0x1010), s1 = __byte_perm(two, two, 0x3232);
      const uint32_t words[4] = {n[p].x, n[p].y, n[p].z, n[p].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t h[4];
        e2m1x8_to_f16x8(words[j], h);
        const uint32_t sc = j < 2 ? s0 : s1;
        *reinterpret_cast<uint4*>(dst + swizzled(r, p * 4 + j)) =
            make_uint4(hmul2(h[0], sc), hmul2(h[1], sc), hmul2(h[2], sc), hmul2(h[3], sc));
      }
    }
  }
};

// Page bytes into the raw slots of K, or of V: a warp each.  One tensor copy of the head's 128 x 64 bytes and one bulk
// copy of its scales a page; page ids are fetched 32 at a time.  (One warp for both took 1400 clocks a tile,
// longer than the tile's products: 18 rows x 30 tokens after 8192 tokens 94 us, with two 89 us.)
template <bool V, class SM>
__device__ __forceinline__ void fetch(const ChunkAttention& a, const ChunkMaps& maps, SM& sm, const Work& w, int row, int kvh,
                                      int lane) {
  constexpr uint32_t kAll = 0xffffffffu;
  constexpr int ring = V ? SM::kRawV : SM::kRawK, base = V ? SM::kRawK : 0;
  const ChunkCache& c = a.c;
  const int pages = w.end - w.begin - w.bf16_tiles;
  const int32_t* table = c.page_table + (int64_t)row * c.page_table_row_stride + w.begin + w.bf16_tiles - w.fresh - w.tail_tiles;
  int ids = 0, slot = 0, p = 0;
  uint32_t parity = 1;       // of the slot's last emptying
  for (; p < pages; ++p) {
    if (!(p & 31)) ids = p + lane < pages ? table[p + lane] : -1;
    const int64_t page = __shfl_sync(kAll, ids, p & 31);
    const bool ok = page >= 0 && page < c.num_pages;
    uint64_t* full = &sm.raw_full[base + slot];
    if (p >= ring && !__all_sync(kAll, mbar_wait(&sm.raw_empty[base + slot], parity, sm, c.status))) break;
    if (lane == 0) {
      sm.page_ok[V][(w.bf16_tiles + p) & 7] = ok;
      if (ok) {
        mbar_expect_tx(full, kRawBytes);
        const uint32_t dst = smem_u32(sm.raw[base + slot]);
        if (V) tma_load_4d(dst, &maps.v, full, 0, 0, kvh, (int)page);
        else tma_load_4d(dst, &maps.k, full, 0, kvh, 0, (int)page);
        bulk_load(dst + 8192, (V ? c.v_sf + page * c.v_sf_pitch : c.k_sf + page * c.k_sf_pitch) + kvh * kSfBlockBytes,
                  kSfBlockBytes, full);
      } else {
        if (!V) chunk_status(c.status, NVFP4_STATUS_BAD_PAGE_ID);
        mbar_arrive(full);
      }
    }
    __syncwarp();
    if (++slot == ring) {
      slot = 0;
      parity ^= 1;
    }
  }
  // nothing lands in shared memory after the CTA is gone, also after an expired wait: the last loads of each slot
  const unsigned long long t0 = global_ns();
  for (int q = max(0, p - ring); q < p; ++q)
    while (!mbar_try(&sm.raw_full[base + q % ring], (q / ring) & 1) && global_ns() - t0 < 200000000ull) {}
}

// One warpgroup makes the K operands, one the V operands.
template <class SM>
__device__ __forceinline__ void produce(const ChunkAttention& a, SM& sm, const Work& w, int kvh, int warp, int lane, bool is_v) {
  Producer<SM> p{a, sm, w, kvh, warp, lane};
  uint8_t (*stage)[kOperandBytes] = is_v ? sm.v : sm.k;
  uint64_t *full = is_v ? sm.v_full : sm.k_full, *empty = is_v ? sm.v_empty : sm.k_empty;
  const int tiles = w.end - w.begin, last = is_v ? SM::kRaw : SM::kRawK;
  int slot = is_v ? SM::kRawK : 0;
  uint32_t parity = 0;
  auto wait_empty = [&](int t) -> bool {       // the products of the tile before last are through
    return t < 2 || mbar_wait(&empty[t & 1], ((t >> 1) - 1) & 1, sm, a.c.status);
  };
  auto hand_over = [&](int t) {
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) mbar_arrive(&full[t & 1]);
  };
  // BF16 tiles: copied straight into an operand stage, the next one in flight while this one lands
  for (int t = 0; t <= w.bf16_tiles; ++t) {
    if (t < w.bf16_tiles) {
      if (!__all_sync(0xffffffffu, wait_empty(t))) goto out;
      p.issue_bf16(w.begin + t, is_v, smem_u32(stage[t & 1]));
    }
    cp_async_commit();
    if (t > 0) {
      cp_async_wait<1>();
      __syncwarp();
      hand_over(t - 1);
    }
  }
  for (int t = w.bf16_tiles; t < tiles; ++t) {      // pages: through this operand's ring of raw slots
    if (!__all_sync(0xffffffffu, mbar_wait(&sm.raw_full[slot], parity, sm, a.c.status) && wait_empty(t))) goto out;
    p.expand(sm.raw[slot], stage[t & 1], sm.page_ok[is_v][t & 7] != 0);
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.raw_empty[slot]);
    hand_over(t);
    if (++slot == last) {
      slot = is_v ? SM::kRawK : 0;
      parity ^= 1;
    }
  }
out:
  cp_async_wait<0>();
}

// -- issuers -------------------------------------------------------------------------------------

// One warp per stream.  A tile's 128 tokens go through tensor memory as two halves of 64 columns: scores of a
// half, its probabilities over the same columns, P V, scores of the next tile's half - so that the softmax
// always has one half to work on while the tensor cores turn the other around.  (The scores of the next tile may
// follow P V unawaited: the tensor core works off one thread's products in the order of their issue.)  With one issuer
// for both streams the products alone ran at 650 TFLOP/s, with two at 1430: issuing an instruction costs its thread
// about as long as the instruction runs.
template <class SM>
__device__ __forceinline__ void issue(const ChunkAttention& a, SM& sm, const Work& work, uint32_t tensor_memory, int stream) {
  constexpr uint32_t kAll = 0xffffffffu;
  uint32_t* status = a.c.status;
  const bool leader = elect_one();
  // (a value out of lane 0 is known to be the same in every lane, so that what follows from it can stay in uniform
  // registers, where the tensor instructions take their operands from)
  auto uniform = [](int v) { return __shfl_sync(kAll, v, 0); };
  const int s = uniform(stream), bf16_tiles = uniform(work.bf16_tiles), tiles = uniform(work.end - work.begin);
  const bool two = uniform(work.two);
  const uint32_t tmem = uniform((int)tensor_memory);
  const int qt = two ? s : 0, first = two ? 0 : s, stride = two ? 1 : 2;
  const uint64_t q_desc = desc_k_major(smem_u32(sm.q[SM::kQTiles > 1 ? qt : 0]));
  const uint32_t col_s = tmem + kColS + s * 128, col_o = tmem + kColO + s * 128;
  bool ready = mbar_wait(&sm.q_ready[qt], 0, sm, status), f16_seen = bf16_tiles == 0;
  auto scores = [&](int t, int half) -> bool {
    const bool bf16 = t < bf16_tiles;
    if (half == 0) {
      bool ok = mbar_wait(&sm.k_full[t & 1], (t >> 1) & 1, sm, status);
      if (!bf16 && !f16_seen) {
        ok = ok && mbar_wait(&sm.q_f16[qt], 0, sm, status);
        f16_seen = true;
      }
      if (!__all_sync(kAll, ok)) return false;
      tc_fence_after();
    }
    const uint64_t k_desc = desc_k_major(smem_u32(sm.k[t & 1]) + half * (kHalfBytes / 2));
    const uint32_t id = idesc(bf16, false, 64);
    if (leader) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint64_t at = ((i >> 2) * kHalfBytes + (i & 3) * 32) >> 4;
        mma_ss(col_s + half * 64, q_desc + at, k_desc + at, id, i > 0);
      }
      mma_commit(&sm.s_full[s][half]);
      if (half) mma_commit(&sm.k_empty[t & 1]);
    }
    __syncwarp();
    return true;
  };
  ready = __all_sync(kAll, ready);
  bool ok = ready && first < tiles && scores(first, 0) && scores(first, 1);
  for (int t = first, u = 0; t < tiles && ok; t += stride, ++u) {
    const bool bf16 = t < bf16_tiles;
    ok = mbar_wait(&sm.v_full[t & 1], (t >> 1) & 1, sm, status);
    const uint32_t v = smem_u32(sm.v[t & 1]);
    const uint32_t id = idesc(bf16, bf16, 128);
    const uint64_t v_desc = bf16 ? desc_mn_major(v) : desc_k_major(v);
    const uint32_t step16 = (bf16 ? 2048 : 32) >> 4, step64 = (bf16 ? 4 * 2048 : kHalfBytes) >> 4;
    for (int half = 0; half < 2; ++half) {
      ok = ok && mbar_wait(&sm.p_ready[s][half], u & 1, sm, status);
      if (!__all_sync(kAll, ok)) { ok = false; break; }
      tc_fence_after();
      if (leader) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          mma_ts(col_o, col_s + half * 64 + i * 8, v_desc + half * step64 + i * step16, id, u > 0 || half > 0 || i > 0);
        mma_commit(&sm.o_done[s]);
        if (half) mma_commit(&sm.v_empty[t & 1]);
      }
      __syncwarp();
      if (t + stride < tiles && !scores(t + stride, half)) { ok = false; break; }
    }
  }
  if (leader) mma_commit(&sm.all_done);
  __syncwarp();
}

// -- softmax -------------------------------------------------------------------------------------

// A thread's query row (tile row r).
struct QueryRow {
  int token, head;       // of the chunk; query head
  bool live;
};

__device__ __forceinline__ QueryRow query_row(const Work& w, int kvh, int tile, int r, bool apart = false) {
  QueryRow q;
  const int index = apart ? r & 63 : r, in_tile = index / w.group;
  q.token = w.token0 + tile * w.tile_tokens + in_tile;
  q.head = kvh * w.group + index - in_tile * w.group;
  q.live = in_tile < w.tile_tokens && q.token < w.r.n;
  return q;
}

// The row becomes FP16 in place, scaled so that its largest magnitude is in [1, 2); returns the exponent.
__device__ __forceinline__ int query_to_f16(uint8_t* tile, int r) {
  uint4 x[16];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    x[i] = *reinterpret_cast<const uint4*>(tile + swizzled(r, i));
    top = __vmaxu2(top, __vmaxu2(__vmaxu2(x[i].x & 0x7FFF7FFFu, x[i].y & 0x7FFF7FFFu),
                                 __vmaxu2(x[i].z & 0x7FFF7FFFu, x[i].w & 0x7FFF7FFFu)));
  }
  const int exponent = row_exponent(max(top & 0xFFFFu, top >> 16));
  const float f = exponent_value(254 - exponent);
#pragma unroll
  for (int i = 0; i < 16; ++i) *reinterpret_cast<uint4*>(tile + swizzled(r, i)) = bf16x8_to_f16x8(x[i], f);
  return exponent;
}

// Lays the warp's 32 rows out as an operand, in BF16, two whole rows of 256 bytes at a time.
__device__ __forceinline__ void load_query(const ChunkAttention& a, const Work& w, int r, const QueryRow& q, uint8_t* tile) {
  const int lane = r & 31;
  const uint16_t* src = a.query + (int64_t)(w.r.first + q.token) * a.q_token_stride + (int64_t)q.head * a.q_head_stride;
  const unsigned long long mine = q.live ? reinterpret_cast<unsigned long long>(src) : 0;
  const uint32_t dst = smem_u32(tile) + swizzled((r & ~31) + (lane >> 4), lane & 15);
#pragma unroll
  for (int i = 0; i < 16; ++i) {      // row 2 i + (lane >> 4), and its place in the swizzle
    const unsigned long long from = __shfl_sync(0xffffffffu, mine, i * 2 + (lane >> 4));
    cp_async16((dst ^ ((2 * i & 7) << 4)) + i * 256, from ? reinterpret_cast<const uint16_t*>(from) + (lane & 15) * 8 : a.query,
               from != 0);
  }
  cp_async_commit();
  cp_async_wait<0>();
}

__device__ __forceinline__ float dot_row(const uint8_t* tile, int r, const uint16_t* y) {
  float even = 0.f, odd = 0.f;
#pragma unroll 4
  for (int i = 0; i < 16; ++i) {
    float u[8], v[8];
    unpack_bf16x8(*reinterpret_cast<const uint4*>(tile + swizzled(r, i)), u);
    unpack_bf16x8(*reinterpret_cast<const uint4*>(y + i * 8), v);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      even += u[j] * v[j];
      odd += u[j + 1] * v[j + 1];
    }
  }
  return even + odd;
}

__device__ __forceinline__ uint32_t pack16(float lo, float hi, bool bf16) {
  uint32_t v;
  if (bf16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
  return v;
}

// Pairs of fp32 in one instruction.
__device__ __forceinline__ uint64_t pair(uint32_t lo, uint32_t hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
  return v;
}
__device__ __forceinline__ uint64_t pair(float v) { return pair(__float_as_uint(v), __float_as_uint(v)); }
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ float max3(float a, uint32_t b, uint32_t c) {
  float v;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(a), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
  return v;
}

struct RowState { float m, l; };    // reference of the row's exponentials (log2 units) and their sum

// Largest of 64 scores.
__device__ __forceinline__ float max64(const uint32_t* raw) {
  float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < 64; i += 8) {
#pragma unroll
    for (int j = 0; j < 4; ++j) top[j] = max3(top[j], raw[i + 2 * j], raw[i + 2 * j + 1]);
  }
  return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}

// 64 scores -> probabilities, packed over the first half of `raw` and stored; their sum is added to l.
template <bool BF16>
__device__ __forceinline__ void exp64(uint32_t* raw, float scale, float base, float& l, uint32_t col_p) {
  const uint64_t scale2 = pair(scale), minus_base = pair(-base);
  uint64_t sum[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    float x, y;
    unpair(fma2(pair(raw[2 * i], raw[2 * i + 1]), scale2, minus_base), x, y);
    x = ex2(x);
    y = ex2(y);
    sum[i & 3] = add2(sum[i & 3], pair(__float_as_uint(x), __float_as_uint(y)));
    raw[i] = pack16(x, y, BF16);
  }
  tmem_st32(col_p, raw);
  float x, y;
  unpair(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), x, y);
  l += x + y;
}

// Steps [first, last) of a stream, all over BF16 tiles or all over pages.  `scored` is called when the last step's scores
// are there, before their softmax.
template <bool BF16, class SM, class Scored>
__device__ __forceinline__ bool softmax_steps(const ChunkAttention& a, SM& sm, const Work& w, uint32_t col_s, uint32_t col_o, int stream,
                                              const QueryRow& q, float shift, bool warp_live, float scale, int first, int last, float& m, float& l,
                                              const Scored& scored) {
  uint32_t* status = a.c.status;
  constexpr uint32_t kAll = 0xffffffffu;
  const bool two = SM::kQTiles > 1 && w.two;
  for (int u = first; u < last; ++u) {
    const int t = two ? u : 2 * u + stream, tile = w.begin + t;
    const float offset = BF16 && tile < w.fresh ? shift * scale : 0.f;
    int limit = 128;
    if (BF16) limit = tile < w.fresh ? q.token - tile * 128 + 1 : w.r.tail;
#pragma unroll SM::kQTiles
    for (int half = 0; half < 2; ++half) {
      if (!__all_sync(kAll, mbar_wait(&sm.s_full[stream][half], u & 1, sm, status))) return false;
      tc_fence_after();
      if (BF16 && half == 1 && u == last - 1 && !scored()) return false;
      if (!BF16 && half == 0) limit = sm.page_ok[0][t & 7] ? 128 : 0;
      if (half) limit -= 64;
      if (warp_live) {
        const uint32_t col = col_s + half * 64;
        bool formed = false;
        if (!__any_sync(kAll, limit < 64)) {
          // The common half-step, on a path of its own (with the masks and the rescaling in line the compiler spends a
          // quarter more time on the rest): nothing masked, no maximum that has grown too far.
          uint32_t raw[64];
          tmem_ld32(col, raw);
          tmem_ld32(col + 32, raw + 32);
          tmem_ld_wait();
          // (at least, not above: a row that has only seen -inf has no reference yet)
          if (!__any_sync(kAll, max64(raw) * scale - offset >= m + (kAboveLog2 + kRescaleLog2))) {
            exp64<BF16>(raw, scale, m + offset, l, col);
            formed = true;
          }
        }
        if (!formed) {
          uint32_t raw[64];
          tmem_ld32(col, raw);
          tmem_ld32(col + 32, raw + 32);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 64; ++i) raw[i] = i < limit ? raw[i] : 0xFF800000u;
          const float best = max64(raw);
          const float now = best == -INFINITY ? -INFINITY : best * scale - offset;
          const bool grows = now > m + (kAboveLog2 + kRescaleLog2);
          if (__any_sync(kAll, grows)) {
            const float reference = now - kAboveLog2;
            const float alpha = grows ? ex2(m - reference) : 1.f;       // 0 from an empty row
            if (u > 0 || half > 0) {      // every product so far has to be in O: the last one is half-step 2 u + half - 1
              if (!__all_sync(kAll, mbar_wait(&sm.o_done[stream], (half + 1) & 1, sm, status))) return false;
              tc_fence_after();
#pragma unroll 1
              for (int i = 0; i < 8; ++i) {
                uint32_t o[16];
                tmem_ld16(col_o + i * 16, o);
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
                tmem_st16(col_o + i * 16, o);
              }
            }
            l *= alpha;
            if (grows) m = reference;
          }
          exp64<BF16>(raw, scale, (m == -INFINITY ? 0.f : m) + offset, l, col);
        }
        tmem_st_wait();
      }
      tc_fence_before();
      mbar_arrive(&sm.p_ready[stream][half]);
    }
  }
  return true;
}

template <class SM>
__device__ __forceinline__ bool softmax(const ChunkAttention& a, SM& sm, const Work& w, uint32_t tmem, int stream, int r,
                                        int kvh, RowState& state) {
  uint32_t* status = a.c.status;
  constexpr uint32_t kAll = 0xffffffffu;
  const bool two = SM::kQTiles > 1 && w.two;
  const int qt = two ? stream : 0;
  uint8_t* query = sm.q[SM::kQTiles > 1 ? qt : 0];
  const bool apart = SM::kQTiles == 1 && w.apart;
  const QueryRow q = query_row(w, kvh, qt, r, apart);
  // rows that no query has are left as they are: nobody reads what comes of them
  const bool warp_loads = __any_sync(kAll, q.live), warp_live = warp_loads && (!apart || r >> 6 == stream);
  const bool loads = two || stream == 0, shifted = a.c.key_shift && w.fresh > w.begin;
  int exponent = 127;
  float shift = 0.f;
  if (loads) {
    if (warp_loads) load_query(a, w, r, q, query);
    if (w.bf16_tiles) {
      fence_proxy_async();
      mbar_arrive(&sm.q_ready[qt]);
    }
    __syncwarp();
    if (warp_loads && shifted) shift = dot_row(query, r, a.c.key_shift + kvh * kHeadDim);
    if (w.bf16_tiles == 0) {
      if (warp_loads) exponent = query_to_f16(query, r);
      if (!two) sm.join[0][0][r] = __int_as_float(exponent);
      fence_proxy_async();
      mbar_arrive(&sm.q_ready[qt]);
      mbar_arrive(&sm.q_f16[qt]);
    }
  }
  if (!two && shifted) {
    if (stream == 0) sm.join[0][1][r] = shift;
    asm volatile("bar.sync 1, 256;" ::: "memory");
    shift = sm.join[0][1][r];
  }
  const uint32_t lanes = (uint32_t)(r & ~31) << 16;
  const uint32_t col_s = tmem + lanes + kColS + stream * 128, col_o = tmem + lanes + kColO + stream * 128;
  float m = -INFINITY, l = 0.f;
  // this stream's steps over BF16 tiles, then those over pages; a score in log2 units is the product with the BF16
  // query, or with the row's FP16 form, times a scale (never zero, so that a masked -inf stays -inf)
  const int steps = stream_steps(w, stream);
  const int bf16_steps = two ? w.bf16_tiles : (w.bf16_tiles + 1 - stream) >> 1;
  // The last BF16 tile's stream makes the rows FP16 as soon as its scores - and, where the streams share the query, the
  // other's last ones, whose next wait for what follows - are formed, so that those of the first page are under way while
  // it computes its softmax.
  const bool converts = w.bf16_tiles > 0 && w.bf16_tiles < w.end - w.begin && (two || stream == ((w.bf16_tiles - 1) & 1));
  const auto convert = [&] {
    if (!converts) return true;
    if (!two && w.bf16_tiles > 1 &&
        !__all_sync(kAll, mbar_wait(&sm.s_full[stream ^ 1][1], ((w.bf16_tiles - 2) >> 1) & 1, sm, status)))
      return false;
    if (warp_loads) exponent = query_to_f16(query, r);
    if (!two) sm.join[0][0][r] = __int_as_float(exponent);
    fence_proxy_async();
    mbar_arrive(&sm.q_f16[qt]);
    return true;
  };
  if (!softmax_steps<true>(a, sm, w, col_s, col_o, stream, q, shift, warp_live, a.scale_log2, 0, bf16_steps, m, l, convert))
    return false;
  if (!two && bf16_steps < steps) {      // by the other stream, perhaps
    if (!__all_sync(kAll, mbar_wait(&sm.q_f16[0], 0, sm, status))) return false;
    exponent = __float_as_int(sm.join[0][0][r]);
  }
  if (!softmax_steps<false>(a, sm, w, col_s, col_o, stream, q, shift, warp_live,
                            fmaxf(a.scale_log2 * exponent_value(exponent), 1.2e-38f), bf16_steps, steps, m, l,
                            [] { return true; }))
    return false;
  state.m = m;
  state.l = l;
  return true;
}

// Channels [begin, end) of a thread's row out, 32 at a time: o * w0 and, where the streams share a tile, the other
// stream's o (shared_o, [channel][row] from this row on) * w1.  PARTIAL: fp32, else BF16.  JOIN: stored directly (a tile
// has few live rows then, a half of the channels each); else rows go through shared memory, 256 bytes of each at a time,
// and a warp stores them as whole lines.
template <bool PARTIAL, bool JOIN>
__device__ __forceinline__ void store_rows(uint32_t col_o, int r, bool live, const float* shared_o, float w0, float w1,
                                           uint8_t* row, uint8_t* stage, int begin, int end) {
  constexpr uint32_t kAll = 0xffffffffu;
  constexpr int kBytes = PARTIAL ? 4 : 2, kPass = 256 / kBytes, kUnits = 2 * kBytes;
  const int lane = r & 31, unit = lane & 15, ahead = lane >> 4;
  const uint32_t at = swizzled((r & ~31) + ahead, unit);
#pragma unroll 1
  for (int c = begin; c < end; c += 32) {
    uint32_t o[32];
    __syncwarp();
    tmem_ld32(col_o + c, o);
    tmem_ld_wait();
    float x[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) x[j] = __uint_as_float(o[j]) * w0;
    if (JOIN) {
#pragma unroll
      for (int j = 0; j < 32; ++j) x[j] += shared_o[(c + j) * 128] * w1;
    }
    uint4 y[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const float* z = x + (PARTIAL ? 4 : 8) * u;
      if constexpr (PARTIAL) y[u] = make_uint4(__float_as_uint(z[0]), __float_as_uint(z[1]), __float_as_uint(z[2]), __float_as_uint(z[3]));
      else y[u] = make_uint4(pack16(z[0], z[1], true), pack16(z[2], z[3], true), pack16(z[4], z[5], true), pack16(z[6], z[7], true));
    }
    if (JOIN) {
      if (live) {
        uint4* dst = reinterpret_cast<uint4*>(row + c * kBytes);
#pragma unroll
        for (int u = 0; u < kUnits; ++u) dst[u] = y[u];
      }
      continue;
    }
    const int first = (c & (kPass - 1)) * kBytes >> 4;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) *reinterpret_cast<uint4*>(stage + swizzled(r, first + u)) = y[u];
    if ((c & (kPass - 1)) != kPass - 32) continue;
    __syncwarp();
    const unsigned long long to = live ? reinterpret_cast<unsigned long long>(row + (c + 32 - kPass) * kBytes) : 0;
#pragma unroll 8
    for (int i = 0; i < 16; ++i) {            // row 2 i + ahead, and its place in the swizzle
      uint4* dst = reinterpret_cast<uint4*>(__shfl_sync(kAll, to, 2 * i + ahead));
      if (dst) dst[unit] = *reinterpret_cast<const uint4*>(stage + ((at ^ (2 * i & 7) << 4) + i * 256));
    }
  }
}

// Rows out: divided by the sum, as BF16, or as a normalised fp32 partial with its log2-sum.
template <class SM>
__device__ __forceinline__ void finish(const ChunkAttention& a, SM& sm, const Work& w, uint32_t tmem, int stream, int r,
                                       int kvh, const RowState& state, int split, bool ok) {
  constexpr uint32_t kAll = 0xffffffffu;
  const bool two = SM::kQTiles > 1 && w.two;
  const bool apart = SM::kQTiles == 1 && w.apart;
  QueryRow q = query_row(w, kvh, two ? stream : 0, r, apart);
  if (apart && r >> 6 != stream) q.live = false;
  const int other = apart ? r ^ 64 : r;       // the same query in the other stream
  const bool join = !two && w.steps > 1;      // the other stream has a part of the same rows
  ok = __all_sync(kAll, ok && mbar_wait(&sm.all_done, 0, sm, a.c.status));
  tc_fence_after();
  const uint32_t lanes = (uint32_t)(r & ~31) << 16;
  const uint32_t col_o = tmem + lanes + kColO + stream * 128;
  const bool warp_live = __any_sync(kAll, q.live);
  float* shared_o = reinterpret_cast<float*>(sm.k);     // [channel][row]: every product has been formed
  if (join) {
    const int give = (stream ^ 1) * 64;
    if (ok && warp_live) {
#pragma unroll 1
      for (int i = give; i < give + 64; i += 32) {
        uint32_t o[32];
        tmem_ld32(col_o + i, o);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) shared_o[(i + j) * 128 + r] = __uint_as_float(o[j]);
      }
    }
    sm.join[stream][0][r] = state.m;
    sm.join[stream][1][r] = state.l;
    asm volatile("bar.sync 1, 256;" ::: "memory");
  }
  if (!ok || sm.abort_flag || !warp_live || (!two && !join && stream == 1)) return;
  float w0 = 1.f, w1 = 0.f, m = state.m, l = state.l;
  if (join) {
    const float m1 = sm.join[stream ^ 1][0][other];
    m = fmaxf(state.m, m1);
    w0 = state.m == -INFINITY ? 0.f : ex2(state.m - m);
    w1 = m1 == -INFINITY ? 0.f : ex2(m1 - m);
    l = state.l * w0 + sm.join[stream ^ 1][1][other] * w1;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  w0 *= inv;
  w1 *= inv;
  const int64_t token = (int64_t)w.r.first + q.token;
  const bool partial = a.num_splits > 1;
  const int64_t part = ((int64_t)split * a.c.tokens + token) * a.heads_q + q.head;
  uint8_t* row = partial ? reinterpret_cast<uint8_t*>(a.o_partial + part * kHeadDim)
                         : reinterpret_cast<uint8_t*>(a.out + token * a.out_token_stride + q.head * kHeadDim);
  const int begin = join ? stream * 64 : 0, end = join ? begin + 64 : kHeadDim;
  if (join) {
    if (partial) store_rows<true, true>(col_o, r, q.live, shared_o + other, w0, w1, row, nullptr, begin, end);
    else store_rows<false, true>(col_o, r, q.live, shared_o + other, w0, w1, row, nullptr, begin, end);
  } else {
    if (partial) store_rows<true, false>(col_o, r, q.live, nullptr, w0, 0.f, row, sm.v[stream], begin, end);
    else store_rows<false, false>(col_o, r, q.live, nullptr, w0, 0.f, row, sm.v[stream], begin, end);
  }
  if (q.live && begin == 0) {
    const float lse2 = l == 0.f ? -INFINITY : m + log2f(l);
    if (partial) a.lse_partial[part] = lse2;
    else if (a.lse) a.lse[token * a.heads_q + q.head] = lse2 * kLn2;
  }
}

// grid (query blocks * splits, heads_kv, rows)
template <int QTILES, int RAW>
__global__ void __launch_bounds__(kThreads, 1)
chunk_attention_kernel(const ChunkAttention a, const __grid_constant__ ChunkMaps maps, int query_blocks,
                       int group, int tile_tokens) {
  using SM = ChunkSmem<QTILES, RAW>;
  extern __shared__ uint8_t smem_raw[];
  SM& sm = *reinterpret_cast<SM*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int row = blockIdx.z, kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the barriers whose counts are known, while the row's lengths are on their way
  if (threadIdx.x == kFetchWarp * 32) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.k_full[i], 4);
      mbar_init(&sm.v_full[i], 4);
      mbar_init(&sm.s_full[i][0], 1);
      mbar_init(&sm.s_full[i][1], 1);
      mbar_init(&sm.p_ready[i][0], 128);
      mbar_init(&sm.p_ready[i][1], 128);
      mbar_init(&sm.o_done[i], 1);
      mbar_init(&sm.q_ready[i], 128);
      mbar_init(&sm.q_f16[i], 128);
    }
    mbar_init(&sm.all_done, 2);
    for (int i = 0; i < RAW; ++i) {
      mbar_init(&sm.raw_full[i], 1);
      mbar_init(&sm.raw_empty[i], 4);
    }
    sm.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // the blocks with the longest causal reach first
  const int split = a.num_splits == 1 ? 0 : blockIdx.x / query_blocks, block = query_blocks - 1 - (blockIdx.x - split * query_blocks);
  Work w;
  w.r = resolve_chunk_row(a.c, row, blockIdx.x == 0 && kvh == 0 && threadIdx.x == 0);
  w.group = group;
  w.tile_tokens = tile_tokens;
  w.token0 = block * QTILES * w.tile_tokens;
  if (w.token0 >= w.r.n) return;
  w.two = QTILES > 1 && w.token0 + w.tile_tokens < w.r.n;
  const int last_token = min(w.r.n, w.token0 + (w.two ? 2 : 1) * w.tile_tokens);
  w.fresh = (last_token + 127) >> 7;
  w.tail_tiles = w.r.tail > 0;
  const int tiles = w.fresh + w.tail_tiles + w.r.pages;
  const int per = a.num_splits == 1 ? tiles : (tiles + a.num_splits - 1) / a.num_splits;
  w.begin = min(split * per, tiles);
  w.end = min(w.begin + per, tiles);
  w.bf16_tiles = max(0, min(w.end, w.fresh + w.tail_tiles) - w.begin);
  w.steps = (w.two ? 2 : 1) * (w.end - w.begin);
  // (so that the streams' softmax warps are on different quarters of the SM: 32 rows x 4 tokens after 4096 tokens, 16
  // query rows a tile, 97 us with both streams on the same warps' rows, 87 us apart)
  w.apart = QTILES == 1 && w.steps > 1 && (w.r.n - w.token0) * group <= 64;
  const int stream = warp >> 2, r = threadIdx.x & 127;
  if (w.begin == w.end) {      // nothing in this range of the keys
    if (stream < (w.two ? 2 : 1)) {
      const QueryRow q = query_row(w, kvh, stream, r);
      if (q.live) a.lse_partial[((int64_t)split * a.c.tokens + w.r.first + q.token) * a.heads_q + q.head] = -INFINITY;
    }
    return;
  }
  if (threadIdx.x == 0) {
    sm.work = w;
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.k_empty[i], w.two ? 2 : 1);      // a tile serves both streams, or one
      mbar_init(&sm.v_empty[i], w.two ? 2 : 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kIssueWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sm.tmem_base))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  // registers: 640 threads at 96, shared out as 2 x 144 + 2 x 72 + 48 = 5 x 96
  if (stream < 2) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
    RowState state{-INFINITY, 0.f};
    const Work w = sm.work;
    const bool ok = softmax(a, sm, w, tmem, stream, r, kvh, state);
    finish(a, sm, w, tmem, stream, r, kvh, state, split, ok);
  } else if (stream < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    const Work w = sm.work;
    produce(a, sm, w, kvh, warp & 3, lane, stream == 3);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    const Work w = sm.work;
    if (warp < kIssueWarp + 2) {
      issue(a, sm, w, tmem, warp - kIssueWarp);
      // nothing of this CTA's is in flight when its tensor memory goes back, also after an expired wait
      const unsigned long long t0 = global_ns();
      while (!mbar_try(&sm.all_done, 0) && global_ns() - t0 < 200000000ull) {}
      __syncwarp();
    } else if (warp == kFetchWarp) {
      fetch<false>(a, maps, sm, w, row, kvh, lane);
    } else {
      fetch<true>(a, maps, sm, w, row, kvh, lane);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kIssueWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// Joins the splits of a row's tokens: one warp per (token, query head), a lane holds four channels.
constexpr int kMergeWarps = 8;
__global__ void __launch_bounds__(32 * kMergeWarps)
chunk_merge_kernel(const ChunkAttention a) {
  const int lane = threadIdx.x & 31;
  // (the launch itself is under way before the attention's last CTAs are gone, which release it by ending: 0.6 us of 18.9 at
  // 16 tokens after 2048)
  cudaGridDependencySynchronize();
  const ChunkRow r = resolve_chunk_row(a.c, blockIdx.y, false);
  const int64_t unit = (int64_t)blockIdx.x * kMergeWarps + (threadIdx.x >> 5);
  const int i = (int)(unit / a.heads_q), head = (int)(unit - (int64_t)i * a.heads_q);
  if (i >= r.n) return;
  const int64_t token = (int64_t)r.first + i;
  const int64_t at = token * a.heads_q + head, pitch = (int64_t)a.c.tokens * a.heads_q;
  float top = -INFINITY;
  for (int s = lane; s < a.num_splits; s += 32) top = fmaxf(top, a.lse_partial[s * pitch + at]);
  top = warp_max(top);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float total = 0.f;
  for (int s = 0; s < a.num_splits; ++s) {
    const float lse = a.lse_partial[s * pitch + at];
    if (lse == -INFINITY) continue;           // an empty range wrote no rows
    const float4 x = *reinterpret_cast<const float4*>(a.o_partial + (s * pitch + at) * kHeadDim + lane * 4);
    const float weight = ex2(lse - top);
    total += weight;
    o.x += weight * x.x; o.y += weight * x.y; o.z += weight * x.z; o.w += weight * x.w;
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  *reinterpret_cast<uint2*>(a.out + token * a.out_token_stride + head * kHeadDim + lane * 4) =
      make_uint2(pack16(o.x * inv, o.y * inv, true), pack16(o.z * inv, o.w * inv, true));
  if (a.lse && lane == 0) a.lse[at] = (top + log2f(total)) * kLn2;
}

template <int QTILES, int RAW>
cudaError_t launch(const ChunkAttention& a, cudaStream_t stream) {
  const int bytes = (int)sizeof(ChunkSmem<QTILES, RAW>) + 1024;
  static_assert(sizeof(ChunkSmem<QTILES, RAW>) + 1024 <= 232448, "shared memory of one CTA");
  // once per device (the attribute belongs to the function on it)
  static std::atomic<uint64_t> prepared{0};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (device & 63);
  if (device > 63 || !(prepared.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(chunk_attention_kernel<QTILES, RAW>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    prepared.fetch_or(bit, std::memory_order_release);
  }
  ChunkMaps maps{};
  if (a.c.max_pages > 0 && a.c.num_pages > 0) {
    e = encode_map(0, a.c.k_packed, a.c.k_pitch, a.c.num_pages, a.c.heads_kv, &maps.k);
    if (e == cudaSuccess) e = encode_map(1, a.c.v_packed, a.c.v_pitch, a.c.num_pages, a.c.heads_kv, &maps.v);
    if (e != cudaSuccess) return e;
  }
  const int group = a.heads_q / a.c.heads_kv, tile_tokens = 128 / group, tokens = tile_tokens * QTILES;
  const int blocks = (a.c.max_chunk + tokens - 1) / tokens;
  chunk_attention_kernel<QTILES, RAW><<<dim3(blocks * a.num_splits, a.c.heads_kv, a.c.rows), kThreads, bytes, stream>>>(
      a, maps, blocks, group, tile_tokens);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_chunk_attention(const ChunkAttention& a, cudaStream_t stream) {
  // one tile of query rows holds 128 / G tokens: longer chunks pair tiles, shorter ones leave the second tile's
  // shared memory to page bytes in flight
  const int tile_tokens = 128 / (a.heads_q / a.c.heads_kv);
  cudaError_t e = a.c.max_chunk > tile_tokens ? launch<2, 3>(a, stream) : launch<1, 7>(a, stream);
  if (e != cudaSuccess || a.num_splits == 1) return e;
  const int64_t units = (int64_t)a.c.max_chunk * a.heads_q;
  cudaLaunchAttribute serial{};
  serial.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  serial.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((unsigned)((units + kMergeWarps - 1) / kMergeWarps), a.c.rows);
  config.blockDim = dim3(32 * kMergeWarps);
  config.stream = stream;
  config.attrs = &serial;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, chunk_merge_kernel, a);
}

}  // namespace nvfp4
