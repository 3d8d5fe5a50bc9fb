// Grouping routed pairs by expert (see rows.cuh): a stable counting sort in one block. Each warp
// owns a contiguous range of pairs and a row of counters, so the place of a pair is the segment's
// start + the pairs of its expert in earlier warps + those before it in its own warp.
#include "rows.cuh"

namespace ovvs {
namespace prim {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;

__global__ void __launch_bounds__(kThreads)
route_plan_kernel(const int* ids, int64_t pairs, int experts, int align, int* offsets, int* order,
                  int64_t capacity, int* position) {
  extern __shared__ int counts[];  // [kWarps][experts], then [experts] segment starts
  __shared__ int warp_total[kWarps];
  int* start = counts + kWarps * experts;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int i = tid; i < kWarps * experts; i += kThreads) counts[i] = 0;
  __syncthreads();
  const int64_t span = ((pairs + kWarps - 1) / kWarps + 31) / 32 * 32;
  const int64_t i0 = warp * span, i1 = i0 + span < pairs ? i0 + span : pairs;
  auto id_at = [&](int64_t i) {
    const int e = i < i1 ? ids[i] : -1;
    return e >= 0 && e < experts ? e : -1;
  };
  for (int64_t i = i0 + lane; i < i1; i += 32) {
    const int e = id_at(i);
    if (e >= 0) atomicAdd(&counts[warp * experts + e], 1);
  }
  __syncthreads();
  // totals per expert (experts <= kThreads), padded, and their exclusive scan
  int total = 0, padded = 0;
  if (tid < experts) {
    for (int w = 0; w < kWarps; ++w) {
      const int c = counts[w * experts + tid];
      counts[w * experts + tid] = total;
      total += c;
    }
    padded = (total + align - 1) / align * align;
  }
  int scan = padded;
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(~0u, scan, o);
    if (lane >= o) scan += y;
  }
  if (lane == 31) warp_total[warp] = scan;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += warp_total[w];
    all += warp_total[w];
  }
  const int first = before + scan - padded;
  if (tid < experts) {
    start[tid] = first;
    offsets[tid] = first;
    if (tid == experts - 1) offsets[experts] = all;
    for (int i = total; i < padded; ++i) order[first + i] = -1;
  }
  for (int64_t i = all + tid; i < capacity; i += kThreads) order[i] = -1;
  __syncthreads();
  for (int64_t b = i0; b < i1; b += 32) {
    const int64_t i = b + lane;
    const int e = id_at(i);
    const unsigned same = __match_any_sync(~0u, e);
    int at = -1;
    if (e >= 0) at = start[e] + counts[warp * experts + e] + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (e >= 0 && lane == __ffs(same) - 1) counts[warp * experts + e] += __popc(same);
    __syncwarp();
    if (i < i1) {
      position[i] = at;
      if (at >= 0) order[at] = static_cast<int>(i);
    }
  }
}

}  // namespace

cudaError_t launch_route_plan(const int* ids, int64_t pairs, int experts, int align,
                              int* offsets, int* order, int64_t capacity, int* position,
                              cudaStream_t stream) {
  const int smem = (kWarps + 1) * experts * static_cast<int>(sizeof(int));
  const cudaError_t e =
      cudaFuncSetAttribute(route_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  route_plan_kernel<<<1, kThreads, smem, stream>>>(ids, pairs, experts, align, offsets, order,
                                                   capacity, position);
  return cudaGetLastError();
}

}  // namespace prim
}  // namespace ovvs
