// Operators over rows of scores that already live in GPU memory: drawing from a row, routing
// tokens to experts with its gradient, and grouping the routed pairs by expert. They are the
// drawn and the trained counterparts of the top-k selection in dense.cuh and keep its order:
// larger scores first, equal ones (-0 == +0) by lower column.
//
// A score of -inf, and a NaN, is masked: it is never drawn or chosen and carries no weight or
// gradient. Any other value, the type's lowest among them, is an ordinary score.
//
// No operator uses global workspace, so calls on several streams, or several captured graphs,
// share nothing.
#pragma once

#include <atomic>
#include <cstdint>
#include <cuda_runtime.h>

namespace ovvs {
namespace prim {

// Opts a kernel in to `bytes` of dynamic shared memory on the current device, once per device:
// the attribute lasts, and setting it costs more than a launch.
template <class Kernel>
inline cudaError_t allow_smem(Kernel* kernel, int bytes, std::atomic<uint64_t>& done) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const uint64_t bit = device < 64 ? uint64_t{1} << device : 0;
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

// One launch; the status is its own. `cluster`: blocks a cluster; `follows`: it may be set up while
// the kernel before it on the stream still runs (and waits for that one itself).
struct LaunchShape {
  unsigned blocks;
  int threads;
  size_t smem = 0;
  unsigned cluster = 1;
  bool follows = false;
};
template <class... P, class... A>
cudaError_t launch(void (*kernel)(P...), const LaunchShape& shape, cudaStream_t stream,
                   A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(shape.blocks);
  cfg.blockDim = dim3(static_cast<unsigned>(shape.threads));
  cfg.dynamicSmemBytes = shape.smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2]{};
  if (shape.cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = shape.cluster;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (shape.follows) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  cfg.attrs = attr;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

// ovvsScoreType (ovvs_cuda.h).
enum ScoreType : int { kScoreF32 = 0, kScoreF16 = 1, kScoreBf16 = 16 };

struct SampleParams {
  const void* logits;        // [rows x cols], row stride ld elements
  int64_t rows, cols, ld;
  const float* temperature;  // [rows] each, or null: 1, off, off, off
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* uniforms;     // [rows x draws]
  int64_t draws;
  int64_t* ids;              // [rows x draws]
  float* probs;              // [rows x draws] or null
  int* kept;                 // [rows] or null
};
cudaError_t launch_sample_rows(const SampleParams& p, int type, cudaStream_t stream);

constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxK = 32;
constexpr int kRouteMaxGroups = 32;

struct RouteParams {
  const void* logits;  // [tokens x experts], row stride ld elements
  int64_t tokens, ld;
  int experts;
  const float* bias;   // [experts] or null
  bool sigmoid;        // else softmax
  int groups, topk_groups;
  bool group_top2;     // else the group's best
  int k;
  bool renormalize;
  float scale;
  int* ids;            // [tokens x k]
  float* weights;      // [tokens x k]
  float* scores;       // [tokens x experts] or null
};
cudaError_t launch_route_topk(const RouteParams& p, int type, cudaStream_t stream);

struct RouteBackwardParams {
  const void* logits;
  int64_t tokens, ld;
  int experts;
  const int* ids;         // [tokens x k]
  int k;
  bool sigmoid, renormalize;
  float scale;
  const float* dweights;  // [tokens x k]
  const float* dscores;   // [tokens x experts] or null
  void* dlogits;          // [tokens x experts], the logits' type, row stride ldd
  int64_t ldd;
};
cudaError_t launch_route_topk_backward(const RouteBackwardParams& p, int type,
                                       cudaStream_t stream);

// Stable counting sort of pairs by expert. offsets [experts + 1]; order [capacity], -1 where no
// pair stands; position [pairs], -1 for a pair whose id is outside [0, experts).
cudaError_t launch_route_plan(const int* ids, int64_t pairs, int experts, int align,
                              int* offsets, int* order, int64_t capacity, int* position,
                              cudaStream_t stream);

}  // namespace prim
}  // namespace ovvs
