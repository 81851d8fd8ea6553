// Attention of a chunk of new tokens over the paged cache and over the chunk itself (causal).
#include "chunk_common.cuh"

namespace nvfp4 {

namespace {

// One warp per (token, query head); a lane holds four channels.
__global__ void __launch_bounds__(128)
chunk_attention_kernel(const ChunkAttention a) {
  const ChunkCache& c = a.c;
  const int row = blockIdx.z, head = blockIdx.y, lane = threadIdx.x & 31;
  const ChunkRow r = resolve_chunk_row(c, row, blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0);
  const int i = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (i >= r.n) return;
  const int kvh = head / (a.heads_q / c.heads_kv);
  const uint16_t* qp = a.query + (int64_t)(r.first + i) * a.q_token_stride + (int64_t)head * a.q_head_stride + lane * 4;
  float q[4], o[4] = {0, 0, 0, 0};
  for (int j = 0; j < 4; ++j) q[j] = bf16_bits_to_f32(qp[j]) * a.scale_log2;
  float m = -INFINITY, l = 0.f;
  auto fold = [&](const float (&k)[4], const float (&v)[4]) {
    const float s = warp_sum(q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3]);
    const float top = fmaxf(m, s);
    const float keep = exp2f(m - top), p = exp2f(s - top);
    for (int j = 0; j < 4; ++j) o[j] = o[j] * keep + p * v[j];
    l = l * keep + p;
    m = top;
  };
  for (int pg = 0; pg < r.pages; ++pg) {
    const int64_t page = c.page_table[(int64_t)row * c.page_table_row_stride + pg];
    if (page < 0 || page >= c.num_pages) {
      if (lane == 0) chunk_status(c.status, NVFP4_STATUS_BAD_PAGE_ID);
      continue;
    }
    const uint8_t* ks = c.k_sf + page * c.k_sf_pitch + kvh * kSfBlockBytes;
    const uint8_t* vs = c.v_sf + page * c.v_sf_pitch + kvh * kSfBlockBytes;
    for (int t = 0; t < kPage; ++t) {
      const uint16_t n = *reinterpret_cast<const uint16_t*>(c.k_packed + page * c.k_pitch +
                                                            ((int64_t)t * c.heads_kv + kvh) * 64 + lane * 2);
      const float s = e4m3_to_f32(ks[sf_offset(t, lane >> 2)]);
      float k[4], v[4];
      for (int j = 0; j < 4; ++j) {
        k[j] = e2m1_to_f32(n >> (4 * j)) * s;
        const int ch = lane * 4 + j;
        const uint8_t b = c.v_packed[page * c.v_pitch + ((int64_t)kvh * kHeadDim + ch) * 64 + t / 2];
        v[j] = e2m1_to_f32(b >> (4 * (t & 1))) * e4m3_to_f32(vs[sf_offset(ch, t >> 4)]);
      }
      fold(k, v);
    }
  }
  for (int t = 0; t < r.tail + i + 1; ++t) {
    const bool old = t < r.tail;
    const int64_t tok = old ? (int64_t)r.tail_id * kPage + t : (int64_t)r.first + t - r.tail;
    const uint16_t* kp = old ? c.tail_key + (tok * c.heads_kv + kvh) * kHeadDim : c.key + tok * c.key_stride + kvh * kHeadDim;
    const uint16_t* vp = old ? c.tail_value + (tok * c.heads_kv + kvh) * kHeadDim : c.value + tok * c.value_stride + kvh * kHeadDim;
    float k[4], v[4];
    for (int j = 0; j < 4; ++j) {
      k[j] = bf16_bits_to_f32(kp[lane * 4 + j]);
      if (!old && c.key_shift) k[j] -= bf16_bits_to_f32(c.key_shift[kvh * kHeadDim + lane * 4 + j]);
      v[j] = bf16_bits_to_f32(vp[lane * 4 + j]);
    }
    fold(k, v);
  }
  uint16_t* out = a.out + (int64_t)(r.first + i) * a.out_token_stride + head * kHeadDim + lane * 4;
  for (int j = 0; j < 4; ++j) out[j] = __bfloat16_as_ushort(__float2bfloat16_rn(o[j] / l));
  if (a.lse && lane == 0) a.lse[(int64_t)(r.first + i) * a.heads_q + head] = (m + log2f(l)) * 0.6931471805599453f;
}

}  // namespace

cudaError_t launch_chunk_attention(const ChunkAttention& a, cudaStream_t stream) {
  chunk_attention_kernel<<<dim3((a.c.max_chunk + 3) / 4, a.heads_q, a.c.rows), 128, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace nvfp4
