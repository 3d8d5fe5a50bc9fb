// Grouping routed pairs by expert (see rows.cuh): a stable counting sort. Warps own contiguous
// ranges of pairs and a row of counters each, so the place of a pair is its segment's start + the
// pairs of its expert in earlier warps + those before it in its own warp.
//
// What bounds it: latency. Up to kSmall pairs one block does it all in one launch (256 experts:
// 512 pairs 5.4 us, 4096 9; it would take 12 for 8192 and 18 for 16384). Beyond that up to
// kMostBlocks blocks of kBlockPairs or more pairs work side by side, in four launches with no
// workspace: the blocks' counts wait in `position` and the experts' in `offsets`, whose own
// contents come last. Each launch is set up while the one before it runs. 4096 pairs would take
// 11 us that way, 8192 to 131,072 take 12 to 14, 524,288 take 14.4 (17 without the early set-up).
// The order's writes are scattered, a sector each: 6 MB move, 1 us at HBM's rate.
#include "rows.cuh"

namespace ovvs {
namespace prim {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kSmall = 4096;
constexpr int kBlockPairs = 2048;  // and multiples of it
constexpr int kMostBlocks = 148;   // one an SM
static_assert(kBlockPairs >= kRouteMaxExperts, "position holds a count per block and expert");

// The launches of a large plan follow one another closely: each says at once that the next may
// be set up, and waits for the one before it to have finished before it reads what that wrote.
__device__ __forceinline__ void let_next_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void wait_for_last() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

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

// The lanes that hold the same e, for e in [-1, 2^bits): one vote a bit. (__match_any_sync takes
// longer the more values there are, some 60 cycles of the SM here.)
__device__ __forceinline__ unsigned same_expert(int e, int bits) {
  const unsigned there = __ballot_sync(~0u, e >= 0);
  unsigned same = e >= 0 ? there : ~there;
  for (int b = 0; b < bits; ++b) {
    const bool one = e >> b & 1;
    const unsigned ones = __ballot_sync(~0u, one);
    same &= one ? ones : ~ones;
  }
  return same;
}

// counts[warp][expert] of the pairs [i0, i1) of each warp.
__device__ __forceinline__ void count_pairs(const int* ids, int64_t i0, int64_t i1, int experts,
                                            int* counts) {
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kWarps * experts; i += kThreads) counts[i] = 0;
  __syncthreads();
  int* own = counts + (threadIdx.x >> 5) * experts;
#pragma unroll 4
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
  constexpr int kAhead = 4;  // rows of ids under way at once
  const int bits = 32 - __clz(experts - 1);
  for (int64_t b = i0; b < i1; b += 32 * kAhead) {
    int ahead[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) ahead[j] = expert_of(ids, b + j * 32 + lane, i1, experts);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (kPosition && b + j * 32 >= i1) break;  // a warp of a small plan has few
      const int64_t i = b + j * 32 + lane;
      const int e = ahead[j];
      const unsigned same = same_expert(e, bits);
      int at = -1;
      if (e >= 0) at = own[e] + __popc(same & ((1u << lane) - 1));
      __syncwarp();
      if (e >= 0 && lane == __ffs(same) - 1) own[e] = at + __popc(same);
      __syncwarp();
      if (i < i1) {
        if (kPosition) position[i] = at;
        if (at >= 0) order[at] = static_cast<int>(i);
      }
    }
  }
}

__global__ void __launch_bounds__(kThreads)
route_plan_kernel(const int* ids, int64_t pairs, int experts, int align, int* offsets, int* order,
                  int64_t capacity, int* position) {
  extern __shared__ int counts[];  // [kWarps][experts]
  __shared__ int buf[kWarps];
  int* pad = counts + kWarps * experts;  // [2][experts]: where padding starts and ends
  const int tid = threadIdx.x, warp = tid >> 5;
  const int64_t span = ((pairs + kWarps - 1) / kWarps + 31) / 32 * 32;
  const int64_t i0 = warp * span, i1 = i0 + span < pairs ? i0 + span : pairs;
  count_pairs(ids, i0, i1, experts, counts);
  int total = 0;
  if (tid < experts) {  // experts <= kThreads
#pragma unroll 8
    for (int w = 0; w < kWarps; ++w) total += counts[w * experts + tid];
  }
  const int padded = (total + (align - 1)) / align * align;
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
    pad[tid] = first + total;
    pad[experts + tid] = first + padded;
  }
  // places go up to 2^31 - 2, a thread's steps beyond
  const uint32_t places = static_cast<uint32_t>(capacity);
  for (uint32_t i = static_cast<uint32_t>(all) + tid; i < places; i += kThreads) order[i] = -1;
  __syncthreads();
  place_pairs<true>(ids, i0, i1, experts, counts, order, position);
  for (int x = warp; x < experts; x += kWarps) {  // a warp an expert
    const uint32_t end = pad[experts + x];
    for (uint32_t i = static_cast<uint32_t>(pad[x]) + (tid & 31); i < end; i += 32) order[i] = -1;
  }
}

// Large plans, first: the pairs of each expert in every block of pairs, to table[expert][block].
__global__ void __launch_bounds__(kThreads)
plan_count_kernel(const int* ids, int64_t pairs, int64_t block_pairs, int experts, int* table) {
  extern __shared__ int counts[];  // [experts]
  let_next_start();
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
    table[e * static_cast<int>(gridDim.x) + blockIdx.x] = counts[e];
}

// Second: a warp an expert; running sums over the blocks, in place, and the total.
__global__ void __launch_bounds__(kThreads)
plan_sum_kernel(int experts, int blocks, int* table, int* totals) {
  const int lane = threadIdx.x & 31;
  const int e = blockIdx.x * kWarps + (threadIdx.x >> 5);
  let_next_start();
  wait_for_last();
  if (e >= experts) return;
  int* row = table + e * blocks;
  constexpr int kPer = (kMostBlocks + 31) / 32;
  int c[kPer], run = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) c[j] = j * 32 + lane < blocks ? row[j * 32 + lane] : 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    if (j * 32 >= blocks) break;
    int s = c[j];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(~0u, s, o);
      if (lane >= o) s += y;
    }
    if (j * 32 + lane < blocks) row[j * 32 + lane] = run + s - c[j];
    run += __shfl_sync(~0u, s, 31);
  }
  if (lane == 0) totals[e] = run;
}

// Third: every block puts its pairs in order.
__global__ void __launch_bounds__(kThreads)
plan_order_kernel(const int* ids, int64_t pairs, int64_t block_pairs, int experts, int align,
                  const int* table, const int* totals, int* order, int64_t capacity) {
  extern __shared__ int counts[];  // [kWarps][experts]
  __shared__ int buf[kWarps];
  const int tid = threadIdx.x, warp = tid >> 5;
  const int blocks = gridDim.x, block = blockIdx.x;
  let_next_start();
  const int64_t span = block_pairs / kWarps;
  const int64_t i0 = block * block_pairs + warp * span;
  const int64_t i1 = i0 + span < pairs ? i0 + span : pairs;
  count_pairs(ids, i0, i1, experts, counts);
  int* pad = counts + kWarps * experts;  // [2][experts]: where padding starts and ends
  wait_for_last();
  const int total = tid < experts ? __ldcg(totals + tid) : 0;
  const int before = tid < experts ? __ldcg(table + tid * blocks + block) : 0;
  const int padded = (total + (align - 1)) / align * align;
  int all;
  const int first = block_scan(padded, buf, &all);
  if (tid < experts) {
    int next = first + before;
#pragma unroll 8
    for (int w = 0; w < kWarps; ++w) {
      const int c = counts[w * experts + tid];
      counts[w * experts + tid] = next;
      next += c;
    }
    pad[tid] = first + total;
    pad[experts + tid] = first + padded;
  }
  __syncthreads();
  place_pairs<false>(ids, i0, i1, experts, counts, order, nullptr);
  // four warps an expert's padding, so that a tile of 128 rows takes one write
  for (int x = block + tid / 128 * blocks; x < experts; x += blocks * (kThreads / 128)) {
    const uint32_t end = pad[experts + x];
    for (uint32_t i = static_cast<uint32_t>(pad[x]) + tid % 128; i < end; i += 128) order[i] = -1;
  }
  for (int64_t i = all + static_cast<int64_t>(block) * kThreads + tid; i < capacity;
       i += static_cast<int64_t>(blocks) * kThreads)
    order[i] = -1;
}

// Last: position is the inverse of order, pairs without an expert have none; the totals become
// the offsets.
__global__ void __launch_bounds__(kThreads)
plan_position_kernel(const int* ids, int64_t pairs, int experts, int align, const int* order,
                     int64_t capacity, int* position, int* offsets) {
  __shared__ int buf[kWarps];
  const int tid = threadIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  wait_for_last();
#pragma unroll 4
  for (int64_t s = static_cast<int64_t>(blockIdx.x) * kThreads + tid; s < capacity; s += step) {
    const int i = __ldcg(order + s);
    if (i >= 0) position[i] = static_cast<int>(s);
    if (s < pairs && expert_of(ids, s, pairs, experts) < 0) position[s] = -1;
  }
  if (blockIdx.x == 0) {
    const int total = tid < experts ? offsets[tid] : 0;
    int all;
    const int first = block_scan((total + (align - 1)) / align * align, buf, &all);
    if (tid < experts) offsets[tid] = first;
    if (tid == 0) offsets[experts] = all;
  }
}

}  // namespace

cudaError_t launch_route_plan(const int* ids, int64_t pairs, int experts, int align,
                              int* offsets, int* order, int64_t capacity, int* position,
                              cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(kWarps + 2) * experts * sizeof(int);
  constexpr int kMost = (kWarps + 2) * kRouteMaxExperts * static_cast<int>(sizeof(int));
  if (pairs <= kSmall) {
    static std::atomic<uint64_t> done;
    const cudaError_t e = allow_smem(route_plan_kernel, kMost, done);
    if (e != cudaSuccess) return e;
    return launch(route_plan_kernel, {1, kThreads, smem}, stream, ids, pairs,
                  experts, align, offsets, order, capacity, position);
  }
  static std::atomic<uint64_t> done;
  cudaError_t e = allow_smem(plan_order_kernel, kMost, done);
  if (e != cudaSuccess) return e;
  const int64_t units = (pairs + kBlockPairs - 1) / kBlockPairs;
  const int64_t block_pairs = (units + kMostBlocks - 1) / kMostBlocks * kBlockPairs;
  const unsigned blocks = static_cast<unsigned>((pairs + block_pairs - 1) / block_pairs);
  const int64_t sweep = (capacity + 2 * kThreads - 1) / (2 * kThreads);
  const unsigned sweep_blocks = static_cast<unsigned>(sweep < 296 ? sweep : 296);
  const unsigned sum_blocks = static_cast<unsigned>((experts + kWarps - 1) / kWarps);
  LaunchShape shape{blocks, kThreads, experts * sizeof(int)};
  e = launch(plan_count_kernel, shape, stream, ids, pairs, block_pairs, experts, position);
  if (e != cudaSuccess) return e;
  shape = {sum_blocks, kThreads, 0, 1, true};
  e = launch(plan_sum_kernel, shape, stream, experts, static_cast<int>(blocks), position, offsets);
  if (e != cudaSuccess) return e;
  // more than half of an SM's shared memory: its blocks are set up early, and two on one SM beside
  // idle ones would take longer (14.4 us for 524,288 pairs against 17.8)
  constexpr size_t kAlone = 116 * 1024;
  shape = {blocks, kThreads, smem > kAlone ? smem : kAlone, 1, true};
  e = launch(plan_order_kernel, shape, stream, ids, pairs, block_pairs, experts, align, position,
             offsets, order, capacity);
  if (e != cudaSuccess) return e;
  shape = {sweep_blocks, kThreads, 0, 1, true};
  return launch(plan_position_kernel, shape, stream, ids, pairs, experts, align, order, capacity,
                position, offsets);
}

}  // namespace prim
}  // namespace ovvs
