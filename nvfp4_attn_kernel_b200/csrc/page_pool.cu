// The page pool: reference counts over the physical pages of a cache whose sealed pages several
// rows may share.  Sealed pages are never written again, so a fork shares them by counting and
// copies only the BF16 tail, each pair as a whole or not at all; a release counts down, and a page whose count is zero is free.
// Compaction moves the live pages into the lowest ids: with L live pages, the k-th live page at or
// above L goes to the k-th free id below L, so sources and destinations never meet, every page is
// moved by whoever gets to it, and the result does not depend on any order.
//
// Bound by memory where pages or tails move (a thread has four 16-byte loads in flight, eight CTAs an SM): forks of 40
// rows x 32 layers 108 us (6.7 TB/s read and written: several pairs of a source find its tail in the L2 cache, so a little
// above a plain copy's 6.5), a compaction of 1500 pages in 8 layers 140 us (5.4 TB/s).
// Small calls are two launches: three forks of one KV head 6.3 us with their release, a compaction of 300 pages in one
// layer 8 us.
#include "chunk_common.cuh"

namespace nvfp4 {

namespace {

constexpr int kCopyThreads = 256;
constexpr int kCopyVectors = 4;                                     // 16-byte loads in flight per thread
constexpr int kCopyBytes = kCopyThreads * kCopyVectors * 16;        // 16 KB a step
constexpr int kPlanThreads = 1024;

// bytes [begin, begin + kCopyBytes) of a run of `bytes` (a multiple of 16)
__device__ __forceinline__ void copy_step(uint8_t* dst, const uint8_t* src, int64_t begin, int64_t bytes) {
  uint4 v[kCopyVectors];
#pragma unroll
  for (int i = 0; i < kCopyVectors; ++i) {
    const int64_t at = begin + ((int64_t)i * kCopyThreads + threadIdx.x) * 16;
    if (at < bytes) v[i] = *reinterpret_cast<const uint4*>(src + at);
  }
#pragma unroll
  for (int i = 0; i < kCopyVectors; ++i) {
    const int64_t at = begin + ((int64_t)i * kCopyThreads + threadIdx.x) * 16;
    if (at < bytes) *reinterpret_cast<uint4*>(dst + at) = v[i];
  }
}

// Whether entry i of the list may act: its row exists and no earlier entry names it.
__device__ __forceinline__ bool first_of_its_row(const int32_t* list, int i, int rows) {
  const int row = list[i];
  bool ok = row >= 0 && row < rows;
  for (int j = threadIdx.x; j < i; j += blockDim.x) ok = ok && list[j] != row;
  return __syncthreads_and(ok);
}

// grid (list entries)
__global__ void __launch_bounds__(kCopyThreads)
pool_release_kernel(const int32_t* __restrict__ list, int count, const int32_t* __restrict__ page_table,
                    int64_t table_stride, int columns, int rows, int32_t* pages_held, int32_t* refs, int64_t num_pages,
                    uint32_t* status) {
  const int i = blockIdx.x;
  if (!first_of_its_row(list, i, rows)) {
    if (threadIdx.x == 0) chunk_status(status, NVFP4_STATUS_BAD_ROW);
    return;
  }
  const int row = list[i];
  const int raw = pages_held[row];
  const int held = min(max(raw, 0), columns);
  uint32_t bad = raw != held ? NVFP4_STATUS_BAD_LENGTH : 0;
  for (int c = threadIdx.x; c < held; c += blockDim.x) {
    const int64_t page = page_table[row * table_stride + c];
    if (page < 0 || page >= num_pages) {
      bad |= NVFP4_STATUS_BAD_PAGE_ID;
    } else if (atomicSub(refs + page, 1) <= 0) {      // nobody held it: put the count back
      atomicAdd(refs + page, 1);
      bad |= NVFP4_STATUS_BAD_PAGE_ID;
    }
  }
  if (bad) chunk_status(status, bad);
  __syncthreads();
  if (threadIdx.x == 0) pages_held[row] = 0;
}

// What a pair of a fork may do.  The whole block judges it, from nothing that this launch writes, so that every block of a
// pair comes to one verdict; `report`: the bits go into the status word.
struct ForkVerdict { bool ok; int source, target, pages, tail, from, to; };
__device__ __forceinline__ ForkVerdict judge_fork(const PoolFork& f, int i, bool report) {
  ForkVerdict v{};
  v.source = f.sources[i];
  v.target = f.targets[i];
  bool named = v.source >= 0 && v.source < f.rows && v.target >= 0 && v.target < f.rows;
  // a target named before, or one that is any pair's source, would make the result depend on order
  for (int j = threadIdx.x; j < f.count; j += blockDim.x)
    named = named && (j >= i || f.targets[j] != v.target) && f.sources[j] != v.target;
  if (!__syncthreads_and(named)) {
    if (report && threadIdx.x == 0) chunk_status(f.status, NVFP4_STATUS_BAD_ROW);
    return v;
  }
  uint32_t bad = 0;
  if (f.pages_held[v.target] != 0) bad |= NVFP4_STATUS_BAD_ROW;      // what it holds would be held by nobody
  const int held = f.pages_held[v.source], fp4 = f.seqused_fp4[v.source];
  v.tail = f.seqused_tail[v.source];
  if (held < 0 || held > f.columns || fp4 < 0 || fp4 % kPage || v.tail < 0 || v.tail > kPage) bad |= NVFP4_STATUS_BAD_LENGTH;
  v.pages = fp4 / kPage;
  const bool shortened = v.pages > held;      // what the source holds is shared, without the tail that would come later
  if (shortened) {
    v.pages = held;
    v.tail = 0;
    if (report && threadIdx.x == 0 && !bad) chunk_status(f.status, NVFP4_STATUS_BAD_LENGTH);
  }
  if (!bad && v.tail > 0 && f.layers > 0) {
    v.from = f.row_to_slot[v.source];
    v.to = f.row_to_slot[v.target];
    if (v.from < 0 || v.from >= f.slots || v.to < 0 || v.to >= f.slots || v.from == v.to) bad |= NVFP4_STATUS_BAD_TAIL_ID;
    for (int j = threadIdx.x; j < f.count; j += blockDim.x) {      // nor may another pair read or write the target's slot
      const int source = f.sources[j], target = f.targets[j];
      if (j != i && ((source >= 0 && source < f.rows && f.row_to_slot[source] == v.to) ||
                     (target >= 0 && target < f.rows && target != v.target && f.row_to_slot[target] == v.to)))
        bad |= NVFP4_STATUS_BAD_TAIL_ID;
    }
  }
  if (!bad) {
    for (int c = threadIdx.x; c < v.pages; c += blockDim.x) {
      const int page = f.page_table[v.source * f.page_table_stride + c];
      if (page < 0 || (int64_t)page >= f.num_pages) bad |= NVFP4_STATUS_BAD_PAGE_ID;
    }
  }
  if (report && bad) chunk_status(f.status, bad);
  v.ok = !__syncthreads_or(bad != 0);
  return v;
}

// The tails, in a launch before the rows' (which writes what the verdict reads).  grid (blocks, pairs): a block judges its
// pair once and takes every gridDim.x-th step of it.
__global__ void __launch_bounds__(kCopyThreads)
fork_tails_kernel(const PoolFork f) {
  cudaTriggerProgrammaticLaunchCompletion();      // the rows' launch may come and judge
  const ForkVerdict v = judge_fork(f, blockIdx.y, false);
  if (!v.ok) return;
  const int64_t bytes = (int64_t)v.tail * f.heads_kv * kHeadDim * 2;
  const int pieces = (int)((bytes + kCopyBytes - 1) / kCopyBytes);
  for (int step = blockIdx.x; step < 2 * f.layers * pieces; step += gridDim.x) {
    const int run = step / pieces, piece = step - run * pieces;
    uint16_t* base = (run & 1 ? f.tail_value : f.tail_key) + (run >> 1) * f.layer_stride;
    copy_step(reinterpret_cast<uint8_t*>(base + v.to * f.slot_stride),
              reinterpret_cast<const uint8_t*>(base + v.from * f.slot_stride), (int64_t)piece * kCopyBytes, bytes);
  }
}

// Tables, counts and lengths.  grid (pairs).  Judged while the tails are copied; written when every block of that launch
// is through, which has then judged for itself.
__global__ void __launch_bounds__(kCopyThreads)
fork_rows_kernel(const PoolFork f) {
  const ForkVerdict v = judge_fork(f, blockIdx.x, true);
  cudaGridDependencySynchronize();
  if (!v.ok) return;
  for (int c = threadIdx.x; c < v.pages; c += blockDim.x) {
    const int page = f.page_table[v.source * f.page_table_stride + c];
    f.page_table[v.target * f.page_table_stride + c] = page;
    atomicAdd(f.refs + page, 1);
  }
  if (threadIdx.x == 0) {
    f.pages_held[v.target] = v.pages;
    f.seqused_fp4[v.target] = v.pages * kPage;
    f.seqused_tail[v.target] = v.tail;
  }
}

// Inclusive scan of two counts over the block; totals in `sum`.
__device__ __forceinline__ int2 block_scan(int2 v, int2* warp_sums, int2& sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, v.x, o), b = __shfl_up_sync(0xffffffffu, v.y, o);
    if (lane >= o) { v.x += a; v.y += b; }
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int2 w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, w.x, o), b = __shfl_up_sync(0xffffffffu, w.y, o);
      if (lane >= o) { w.x += a; w.y += b; }
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  if (warp > 0) { v.x += warp_sums[warp - 1].x; v.y += warp_sums[warp - 1].y; }
  sum = warp_sums[31];
  __syncthreads();
  return v;
}

// One CTA.  holes [0, moves) and movers [0, moves): where the k-th moved page goes and comes from;
// map: the new id of every live page, -1 for the others; counts follow their pages.
__global__ void __launch_bounds__(kPlanThreads)
compact_plan_kernel(int32_t* refs, int64_t num_pages, int reserved, int32_t* map, int32_t* holes, int32_t* movers,
                    int32_t* moves, int32_t* live_count) {
  __shared__ int2 warp_sums[32];
  __shared__ int2 before;
  int mine = 0;
  for (int64_t p = threadIdx.x; p < num_pages; p += kPlanThreads) mine += refs[p] > 0 || p < reserved;
  int2 sum;
  block_scan(make_int2(mine, 0), warp_sums, sum);
  const int live = sum.x;
  if (threadIdx.x == 0) before = make_int2(0, 0);
  __syncthreads();
  for (int64_t base = 0; base < num_pages; base += kPlanThreads) {
    const int64_t p = base + threadIdx.x;
    const bool inside = p < num_pages;
    const bool alive = inside && (refs[p] > 0 || p < reserved);
    const bool hole = inside && !alive && p < live, mover = alive && p >= live;
    const int2 at = block_scan(make_int2(hole, mover), warp_sums, sum);
    const int2 first = before;
    if (hole) holes[first.x + at.x - 1] = (int)p;
    if (mover) movers[first.y + at.y - 1] = (int)p;
    else if (inside) map[p] = alive ? (int)p : -1;
    __syncthreads();
    if (threadIdx.x == 0) before = make_int2(first.x + sum.x, first.y + sum.y);
    __syncthreads();
  }
  const int n = before.y;      // as many movers as holes
  for (int k = threadIdx.x; k < n; k += kPlanThreads) {
    const int to = holes[k], from = movers[k];
    map[from] = to;
    refs[to] = refs[from];
    refs[from] = 0;
  }
  if (threadIdx.x == 0) {
    *moves = n;
    *live_count = live;
  }
}

__device__ __forceinline__ void copy_pages(const int64_t* __restrict__ bases, int layers, int64_t pitch, int64_t num_pages,
                                           const int32_t* __restrict__ src, const int32_t* __restrict__ dst, int count,
                                           int64_t block, int64_t blocks, uint32_t* status) {
  const int64_t steps = (pitch + kCopyBytes - 1) / kCopyBytes;
  const int64_t total = steps * layers * count;
  for (int64_t w = block; w < total; w += blocks) {
    const int64_t item = w / steps;
    const int k = (int)(item / layers), layer = (int)(item - (int64_t)k * layers);
    const int64_t from = src[k], to = dst[k];
    if (from < 0 || to < 0) continue;                  // -1: no copy
    if (from >= num_pages || to >= num_pages) {
      if (threadIdx.x == 0) chunk_status(status, NVFP4_STATUS_BAD_PAGE_ID);
      continue;
    }
    uint8_t* base = reinterpret_cast<uint8_t*>(bases[layer]);
    copy_step(base + to * pitch, base + from * pitch, (w - item * steps) * kCopyBytes, pitch);
  }
}

__global__ void __launch_bounds__(kCopyThreads)
pool_copy_kernel(const int64_t* __restrict__ bases, int layers, int64_t pitch, int64_t num_pages,
                 const int32_t* __restrict__ src, const int32_t* __restrict__ dst, int count, uint32_t* status) {
  copy_pages(bases, layers, pitch, num_pages, src, dst, count, blockIdx.x, gridDim.x, status);
}

// The first `rows` blocks rewrite a row of the table each, the others move pages.
__global__ void __launch_bounds__(kCopyThreads)
compact_move_kernel(const int64_t* __restrict__ bases, int layers, int64_t pitch, int64_t num_pages,
                    const int32_t* __restrict__ movers, const int32_t* __restrict__ holes, const int32_t* __restrict__ moves,
                    const int32_t* __restrict__ map, int32_t* page_table, int64_t table_stride, int columns, int rows,
                    const int32_t* __restrict__ pages_held, uint32_t* status) {
  if ((int)blockIdx.x < rows) {
    const int row = blockIdx.x;
    const int raw = pages_held[row];
    const int held = min(max(raw, 0), columns);
    uint32_t bad = raw != held ? NVFP4_STATUS_BAD_LENGTH : 0;
    for (int c = threadIdx.x; c < held; c += blockDim.x) {
      int32_t* entry = page_table + row * table_stride + c;
      const int64_t page = *entry;
      const int to = page < 0 || page >= num_pages ? -1 : map[page];
      if (to < 0) bad |= NVFP4_STATUS_BAD_PAGE_ID;
      if (page >= 0 && page < num_pages) *entry = to;      // -1 for a page that nobody counts: another row's may be there now
    }
    if (bad) chunk_status(status, bad);
    return;
  }
  copy_pages(bases, layers, pitch, num_pages, movers, holes, *moves, blockIdx.x - rows, gridDim.x - rows, status);
}

// One CTA: the ids whose count is zero, ascending, and how many they are.
__global__ void __launch_bounds__(kPlanThreads)
free_list_kernel(const int32_t* __restrict__ refs, int64_t num_pages, int reserved, int32_t* __restrict__ ids,
                 int32_t* __restrict__ count) {
  __shared__ int2 warp_sums[32];
  int first = 0;
  for (int64_t base = 0; base < num_pages; base += kPlanThreads) {
    const int64_t p = base + threadIdx.x;
    const bool vacant = p < num_pages && p >= reserved && refs[p] <= 0;
    int2 sum;
    const int2 at = block_scan(make_int2(vacant, 0), warp_sums, sum);
    if (vacant) ids[first + at.x - 1] = (int)p;
    first += sum.x;
  }
  for (int64_t p = first + threadIdx.x; p < num_pages; p += kPlanThreads) ids[p] = -1;
  if (threadIdx.x == 0) *count = first;
}

cudaError_t copy_grid(int64_t steps, unsigned* blocks) {
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int64_t most = 8ll * sms;      // resident CTAs of 256 threads per SM
  *blocks = (unsigned)(steps < most ? (steps < 1 ? 1 : steps) : most);
  return e;
}

}  // namespace

cudaError_t launch_pool_release(const int32_t* list, int count, const int32_t* page_table, int64_t page_table_stride,
                                int columns, int rows, int32_t* pages_held, int32_t* refs, int64_t num_pages,
                                uint32_t* status, cudaStream_t stream) {
  pool_release_kernel<<<count, kCopyThreads, 0, stream>>>(list, count, page_table, page_table_stride, columns, rows,
                                                          pages_held, refs, num_pages, status);
  return cudaGetLastError();
}

cudaError_t launch_pool_fork(const PoolFork& f, cudaStream_t stream) {
  cudaLaunchAttribute serial{};
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(f.count);
  config.blockDim = dim3(kCopyThreads);
  config.stream = stream;
  if (f.layers > 0) {
    // Blocks that fill the GPU four times over (a verdict costs a block about as much as a step): 40 rows x 32 layers of 8
    // heads 108 us, filled once 111, a block for every step 128.
    const int64_t steps = 2 * f.layers * (((int64_t)kPage * f.heads_kv * kHeadDim * 2 + kCopyBytes - 1) / kCopyBytes);
    unsigned fill;
    cudaError_t e = copy_grid(steps * f.count, &fill);
    if (e != cudaSuccess) return e;
    const int64_t share = (4ll * fill + f.count - 1) / f.count;
    fork_tails_kernel<<<dim3((unsigned)(share < steps ? share : steps), f.count), kCopyThreads, 0, stream>>>(f);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    serial.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    serial.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &serial;
    config.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&config, fork_rows_kernel, f);
}

cudaError_t launch_pool_free_list(const int32_t* refs, int64_t num_pages, int reserved, int32_t* ids, int32_t* count,
                                  cudaStream_t stream) {
  free_list_kernel<<<1, kPlanThreads, 0, stream>>>(refs, num_pages, reserved, ids, count);
  return cudaGetLastError();
}

cudaError_t launch_pool_copy(const int64_t* bases, int layers, int64_t pitch, int64_t num_pages, const int32_t* src,
                             const int32_t* dst, int count, uint32_t* status, cudaStream_t stream) {
  unsigned blocks;
  cudaError_t e = copy_grid((pitch + kCopyBytes - 1) / kCopyBytes * layers * count, &blocks);
  if (e != cudaSuccess) return e;
  pool_copy_kernel<<<blocks, kCopyThreads, 0, stream>>>(bases, layers, pitch, num_pages, src, dst, count, status);
  return cudaGetLastError();
}

cudaError_t launch_pool_compact(const int64_t* bases, int layers, int64_t pitch, int64_t num_pages, int reserved,
                                int32_t* refs, int32_t* page_table, int64_t page_table_stride, int columns, int rows,
                                const int32_t* pages_held, int32_t* workspace, int32_t* live_count, uint32_t* status,
                                cudaStream_t stream) {
  int32_t* map = workspace;
  int32_t* holes = map + num_pages;
  int32_t* movers = holes + num_pages;
  int32_t* moves = movers + num_pages;
  unsigned blocks;
  // at most half of the pages move
  cudaError_t e = copy_grid((pitch + kCopyBytes - 1) / kCopyBytes * layers * ((num_pages + 1) / 2), &blocks);
  if (e != cudaSuccess) return e;
  compact_plan_kernel<<<1, kPlanThreads, 0, stream>>>(refs, num_pages, reserved, map, holes, movers, moves, live_count);
  compact_move_kernel<<<blocks + rows, kCopyThreads, 0, stream>>>(bases, layers, pitch, num_pages, movers, holes, moves,
                                                                  map, page_table, page_table_stride, columns, rows,
                                                                  pages_held, status);
  return cudaGetLastError();
}

}  // namespace nvfp4
