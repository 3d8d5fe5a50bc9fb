// Grouping routed pairs by expert (see rows.cuh): a stable counting sort. Warps own contiguous
// ranges of pairs and a row of counters each, so the place of a pair is its segment's start + the
// pairs of its expert in earlier warps + those before it in its own warp.
//
// Up to kSmall pairs one block does it all (one launch: 4.8 us for 512 pairs of 256 experts).
// Beyond that up to kMostBlocks blocks of kBlockPairs or more pairs work side by side, in three
// launches with no workspace: the blocks' counts wait in `position`, whose own contents come
// last, from `order`.
#include "rows.cuh"

namespace ovvs {
namespace prim {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kSmall = 4096;
constexpr int kBlockPairs = 4096;  // and multiples of it
constexpr int kMostBlocks = 512;   // every block reads all blocks' counts
static_assert(kBlockPairs >= kRouteMaxExperts, "position holds a count per block and expert");

__device__ __forceinline__ int expert_of(const int* ids, int64_t i, int64_t end, int experts) {
  const int e = i < end ? __ldg(ids + i) : -1;
  return e >= 0 && e < experts ? e : -1;
}

// Exclusive running sum over the block's threads; *all gets the sum.
__device__ __forceinline__ int block_scan(int v, int* buf, int* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(~0u, s, o);
    if (lane >= o) s += y;
  }
  if (lane == 31) buf[warp] = s;
  __syncthreads();
  int t = buf[lane];  // kWarps == 32
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(~0u, t, o);
    if (lane >= o) t += y;
  }
  *all = __shfl_sync(~0u, t, 31);
  const int before = __shfl_sync(~0u, t, warp) - buf[warp];
  __syncthreads();
  return before + s - v;
}
static_assert(kWarps == 32, "one total a lane");

// counts[warp][expert] of the pairs [i0, i1) of each warp.
__device__ __forceinline__ void count_pairs(const int* ids, int64_t i0, int64_t i1, int experts,
                                            int* counts) {
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kWarps * experts; i += kThreads) counts[i] = 0;
  __syncthreads();
  int* own = counts + (threadIdx.x >> 5) * experts;
  for (int64_t i = i0 + lane; i < i1; i += 32) {
    const int e = expert_of(ids, i, i1, experts);
    if (e >= 0) atomicAdd(own + e, 1);
  }
  __syncthreads();
}

// Puts the pairs [i0, i1) of this warp in place; counts[warp][expert] is the next free place.
template <bool kPosition>
__device__ __forceinline__ void place_pairs(const int* ids, int64_t i0, int64_t i1, int experts,
                                            int* counts, int* order, int* position) {
  const int lane = threadIdx.x & 31;
  int* own = counts + (threadIdx.x >> 5) * experts;
  for (int64_t b = i0; b < i1; b += 32) {
    const int64_t i = b + lane;
    const int e = expert_of(ids, i, i1, experts);
    const unsigned same = __match_any_sync(~0u, e);
    int at = -1;
    if (e >= 0) at = own[e] + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (e >= 0 && lane == __ffs(same) - 1) own[e] += __popc(same);
    __syncwarp();
    if (i < i1) {
      if (kPosition) position[i] = at;
      if (at >= 0) order[at] = static_cast<int>(i);
    }
  }
}

__global__ void __launch_bounds__(kThreads)
route_plan_kernel(const int* ids, int64_t pairs, int experts, int align, int* offsets, int* order,
                  int64_t capacity, int* position) {
  extern __shared__ int counts[];  // [kWarps][experts]
  __shared__ int buf[kWarps];
  const int tid = threadIdx.x, warp = tid >> 5;
  const int64_t span = ((pairs + kWarps - 1) / kWarps + 31) / 32 * 32;
  const int64_t i0 = warp * span, i1 = i0 + span < pairs ? i0 + span : pairs;
  count_pairs(ids, i0, i1, experts, counts);
  int total = 0;
  if (tid < experts) {  // experts <= kThreads
#pragma unroll 8
    for (int w = 0; w < kWarps; ++w) total += counts[w * experts + tid];
  }
  const int padded = (total + align - 1) / align * align;
  int all;
  const int first = block_scan(padded, buf, &all);
  if (tid < experts) {
    offsets[tid] = first;
    if (tid == experts - 1) offsets[experts] = all;
    int next = first;
#pragma unroll 8
    for (int w = 0; w < kWarps; ++w) {
      const int c = counts[w * experts + tid];
      counts[w * experts + tid] = next;
      next += c;
    }
    for (int i = total; i < padded; ++i) order[first + i] = -1;
  }
  for (int64_t i = all + tid; i < capacity; i += kThreads) order[i] = -1;
  __syncthreads();
  place_pairs<true>(ids, i0, i1, experts, counts, order, position);
}

// Large plans, first: the pairs of each expert in every block of pairs, to table[block][expert].
__global__ void __launch_bounds__(kThreads)
plan_count_kernel(const int* ids, int64_t pairs, int64_t block_pairs, int experts, int* table) {
  extern __shared__ int counts[];  // [experts]
  for (int e = threadIdx.x; e < experts; e += kThreads) counts[e] = 0;
  __syncthreads();
  const int64_t b = blockIdx.x * block_pairs;
  const int64_t end = b + block_pairs < pairs ? b + block_pairs : pairs;
#pragma unroll 4
  for (int64_t i = b + threadIdx.x; i < end; i += kThreads) {
    const int e = expert_of(ids, i, end, experts);
    if (e >= 0) atomicAdd(counts + e, 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += kThreads)
    table[static_cast<int64_t>(blockIdx.x) * experts + e] = counts[e];
}

// Second: every block sums the table for itself (the whole of it, from L2), which gives the
// segments and where its own pairs start in them, and puts its pairs in order.
__global__ void __launch_bounds__(kThreads)
plan_order_kernel(const int* ids, int64_t pairs, int64_t block_pairs, int experts, int align,
                  const int* table, int* offsets, int* order, int64_t capacity) {
  extern __shared__ int counts[];  // [kWarps][experts]
  __shared__ int buf[kWarps];
  const int tid = threadIdx.x, warp = tid >> 5;
  const int blocks = gridDim.x, block = blockIdx.x;
  // `parts` threads an expert, each over every parts-th block: (pairs before this block, in all)
  int parts = 1;
  while (parts * 2 * experts <= kThreads) parts *= 2;
  const int e = tid / parts, part = tid % parts;
  int before = 0, total = 0;
  if (e < experts) {
#pragma unroll 8
    for (int b = part; b < blocks; b += parts) {
      const int c = __ldg(table + static_cast<int64_t>(b) * experts + e);
      total += c;
      before += b < block ? c : 0;
    }
  }
  // parts is a power of two, but may be more than a warp's lanes: joined in shared memory
  for (int i = tid; i < 2 * experts; i += kThreads) counts[i] = 0;
  __syncthreads();
  if (e < experts) {
    atomicAdd(&counts[e], total);
    atomicAdd(&counts[experts + e], before);
  }
  __syncthreads();
  total = tid < experts ? counts[tid] : 0;
  before = tid < experts ? counts[experts + tid] : 0;
  __syncthreads();
  const int padded = (total + align - 1) / align * align;
  int all;
  const int first = block_scan(padded, buf, &all);
  if (tid < experts) {
    if (block == 0) {
      offsets[tid] = first;
      if (tid == experts - 1) offsets[experts] = all;
    }
    if (tid % blocks == block)
      for (int i = total; i < padded; ++i) order[first + i] = -1;
  }
  for (int64_t i = all + static_cast<int64_t>(block) * kThreads + tid; i < capacity;
       i += static_cast<int64_t>(blocks) * kThreads)
    order[i] = -1;
  const int64_t span = block_pairs / kWarps;
  const int64_t i0 = block * block_pairs + warp * span;
  const int64_t i1 = i0 + span < pairs ? i0 + span : pairs;
  count_pairs(ids, i0, i1, experts, counts);
  if (tid < experts) {
    int next = first + before;
#pragma unroll 8
    for (int w = 0; w < kWarps; ++w) {
      const int c = counts[w * experts + tid];
      counts[w * experts + tid] = next;
      next += c;
    }
  }
  __syncthreads();
  place_pairs<false>(ids, i0, i1, experts, counts, order, nullptr);
}

// Third: position is the inverse of order; pairs without an expert have none.
__global__ void __launch_bounds__(256)
plan_position_kernel(const int* ids, int64_t pairs, int experts, const int* order,
                     int64_t capacity, int* position) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t s = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; s < capacity; s += step) {
    const int i = __ldg(order + s);
    if (i >= 0) position[i] = static_cast<int>(s);
    if (s < pairs && expert_of(ids, s, pairs, experts) < 0) position[s] = -1;
  }
}

}  // namespace

cudaError_t launch_route_plan(const int* ids, int64_t pairs, int experts, int align,
                              int* offsets, int* order, int64_t capacity, int* position,
                              cudaStream_t stream) {
  const int smem = kWarps * experts * static_cast<int>(sizeof(int));
  constexpr int kMost = kWarps * kRouteMaxExperts * static_cast<int>(sizeof(int));
  if (pairs <= kSmall) {
    static std::atomic<uint64_t> done;
    const cudaError_t e = allow_smem(route_plan_kernel, kMost, done);
    if (e != cudaSuccess) return e;
    route_plan_kernel<<<1, kThreads, smem, stream>>>(ids, pairs, experts, align, offsets, order,
                                                     capacity, position);
    return cudaGetLastError();
  }
  static std::atomic<uint64_t> done;
  const cudaError_t e = allow_smem(plan_order_kernel, kMost, done);
  if (e != cudaSuccess) return e;
  const int64_t units = (pairs + kBlockPairs - 1) / kBlockPairs;
  const int64_t block_pairs = (units + kMostBlocks - 1) / kMostBlocks * kBlockPairs;
  const unsigned blocks = static_cast<unsigned>((pairs + block_pairs - 1) / block_pairs);
  plan_count_kernel<<<blocks, kThreads, experts * sizeof(int), stream>>>(ids, pairs, block_pairs,
                                                                         experts, position);
  plan_order_kernel<<<blocks, kThreads, smem, stream>>>(ids, pairs, block_pairs, experts, align,
                                                        position, offsets, order, capacity);
  const int64_t sweep = (capacity + 255) / 256;
  plan_position_kernel<<<static_cast<unsigned>(sweep < 148 * 8 ? sweep : 148 * 8), 256, 0,
                         stream>>>(ids, pairs, experts, order, capacity, position);
  return cudaGetLastError();
}

}  // namespace prim
}  // namespace ovvs
