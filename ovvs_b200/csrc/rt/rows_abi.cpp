// Entry points of the row operators (ovvs_cuda.h): argument checks, then one launch on the
// caller's stream. They take no lock and touch no workspace, so any number of threads may call
// them on one Resources at once, and they may be captured into graphs.
#include <cuda_runtime.h>

#include <cstdint>

#include "../prim/rows.cuh"
#include "ovvs/ovvs_cuda.h"
#include "overlap.hpp"
#include "runtime.hpp"

using ovvs::rt::Resources;
using ovvs::rt::clash;
using ovvs::rt::from_handle;
using ovvs::rt::Span;
using ovvs::rt::span_of;

namespace {

// Makes a Resources' device current for one call and gives the caller its own back.
class DeviceScope {
 public:
  ovvsStatus enter(const Resources& r) {
    OVVS_TRY(r.check_policy());
    if (!r.gpu_available) return OVVS_STATUS_DEVICE_UNAVAILABLE;
    OVVS_TRY_CUDA(cudaGetDevice(&before_));
    if (before_ == r.device) {
      before_ = -1;
      return OVVS_STATUS_SUCCESS;
    }
    OVVS_TRY_CUDA(cudaSetDevice(r.device));
    return OVVS_STATUS_SUCCESS;
  }
  ~DeviceScope() {
    if (before_ >= 0) cudaSetDevice(before_);
  }

 private:
  int before_ = -1;
};

// `shared`: an output lies where another or an input does. The kernels read and write in no order
// that a caller could rely on, and the plan's places come from counts of ids that must not change.
template <class F>
ovvsStatus launched(Resources& r, bool shared, F&& launch) {
  try {
    DeviceScope scope;
    OVVS_TRY(scope.enter(r));
    if (shared) return OVVS_STATUS_INVALID_ARGUMENT;
    const cudaError_t e = launch();
    if (e != cudaSuccess) {
      (void)cudaGetLastError();  // a refused launch is reported once, by this call
      return ovvs::rt::status_of(e);
    }
    r.last_device = OVVS_DEVICE_GPU;
    return OVVS_STATUS_SUCCESS;
  } catch (...) {
    return OVVS_STATUS_ERROR;
  }
}

size_t type_bytes(int32_t type) {
  return type == OVVS_SCORE_F32 ? 4 : type == OVVS_SCORE_F16 || type == OVVS_SCORE_BF16 ? 2 : 0;
}

bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

bool too_big(int64_t a, int64_t b) { return a > 0 && b > (INT64_MAX / 16) / a; }

// A [rows x cols] matrix of scores with row stride ld.
ovvsStatus check_matrix(const void* p, int32_t type, int64_t rows, int64_t cols, int64_t ld) {
  const size_t bytes = type_bytes(type);
  if (!p || bytes == 0 || rows <= 0 || cols <= 0 || ld < cols || !aligned(p, bytes))
    return OVVS_STATUS_INVALID_ARGUMENT;
  if (too_big(rows, ld) || rows > 0x7fffffLL * 16 || cols > 0x7fffffffLL)
    return OVVS_STATUS_SHAPE_MISMATCH;
  return OVVS_STATUS_SUCCESS;
}

bool known_score(int32_t score) {
  return score == OVVS_ROUTE_SOFTMAX || score == OVVS_ROUTE_SIGMOID;
}

}  // namespace

extern "C" {

ovvsStatus ovvsSampleRowsDevice(ovvsResources_t res, const void* d_logits, int32_t type,
                                int64_t rows, int64_t cols, int64_t ld,
                                const float* d_temperature, const int32_t* d_top_k,
                                const float* d_top_p, const float* d_min_p,
                                const float* d_uniforms, int64_t draws, int64_t* d_ids,
                                float* d_probs, int32_t* d_kept, void* stream) {
  if (!res || !d_uniforms || !d_ids || draws <= 0 || !aligned(d_ids, 8) ||
      !aligned(d_uniforms, 4) || !aligned(d_temperature, 4) || !aligned(d_top_k, 4) ||
      !aligned(d_top_p, 4) || !aligned(d_min_p, 4) || !aligned(d_probs, 4) || !aligned(d_kept, 4))
    return OVVS_STATUS_INVALID_ARGUMENT;
  OVVS_TRY(check_matrix(d_logits, type, rows, cols, ld));
  if (too_big(rows, draws)) return OVVS_STATUS_SHAPE_MISMATCH;
  ovvs::prim::SampleParams p{};
  p.logits = d_logits;
  p.rows = rows;
  p.cols = cols;
  p.ld = ld;
  p.temperature = d_temperature;
  p.top_k = d_top_k;
  p.top_p = d_top_p;
  p.min_p = d_min_p;
  p.uniforms = d_uniforms;
  p.draws = draws;
  p.ids = d_ids;
  p.probs = d_probs;
  p.kept = d_kept;
  const bool shared = clash(
      {span_of(d_ids, rows * draws, 8), span_of(d_probs, rows * draws, 4), span_of(d_kept, rows, 4)},
      {span_of(d_logits, rows, cols, ld, type_bytes(type)), span_of(d_uniforms, rows * draws, 4),
       span_of(d_temperature, rows, 4), span_of(d_top_k, rows, 4), span_of(d_top_p, rows, 4),
       span_of(d_min_p, rows, 4)});
  return launched(*from_handle(res), shared, [&] {
    return ovvs::prim::launch_sample_rows(p, type, static_cast<cudaStream_t>(stream));
  });
}

ovvsStatus ovvsRouteTopkDevice(ovvsResources_t res, const void* d_logits, int32_t type,
                               int64_t tokens, int64_t experts, int64_t ld, const float* d_bias,
                               int32_t score, int32_t groups, int32_t topk_groups,
                               int32_t group_rule, int32_t k, int32_t renormalize, float scale,
                               int32_t* d_ids, float* d_weights, float* d_scores, void* stream) {
  if (!res || !d_ids || !d_weights || !known_score(score) || k <= 0 || groups <= 0 ||
      topk_groups <= 0 || topk_groups > groups ||
      (group_rule != OVVS_ROUTE_GROUP_MAX && group_rule != OVVS_ROUTE_GROUP_TOP2) ||
      !aligned(d_bias, 4) || !aligned(d_ids, 4) || !aligned(d_weights, 4) || !aligned(d_scores, 4))
    return OVVS_STATUS_INVALID_ARGUMENT;
  OVVS_TRY(check_matrix(d_logits, type, tokens, experts, ld));
  if (experts % groups != 0) return OVVS_STATUS_INVALID_ARGUMENT;
  if (experts > ovvs::prim::kRouteMaxExperts || groups > ovvs::prim::kRouteMaxGroups ||
      k > ovvs::prim::kRouteMaxK || k > experts)
    return OVVS_STATUS_SHAPE_MISMATCH;
  ovvs::prim::RouteParams p{};
  p.logits = d_logits;
  p.tokens = tokens;
  p.ld = ld;
  p.experts = static_cast<int>(experts);
  p.bias = d_bias;
  p.sigmoid = score == OVVS_ROUTE_SIGMOID;
  p.groups = groups;
  p.topk_groups = topk_groups;
  p.group_top2 = group_rule == OVVS_ROUTE_GROUP_TOP2;
  p.k = k;
  p.renormalize = renormalize != 0;
  p.scale = scale;
  p.ids = d_ids;
  p.weights = d_weights;
  p.scores = d_scores;
  const bool shared = clash(
      {span_of(d_ids, tokens * k, 4), span_of(d_weights, tokens * k, 4),
       span_of(d_scores, tokens * experts, 4)},
      {span_of(d_logits, tokens, experts, ld, type_bytes(type)), span_of(d_bias, experts, 4)});
  return launched(*from_handle(res), shared, [&] {
    return ovvs::prim::launch_route_topk(p, type, static_cast<cudaStream_t>(stream));
  });
}

ovvsStatus ovvsRouteTopkBackwardDevice(ovvsResources_t res, const void* d_logits, int32_t type,
                                       int64_t tokens, int64_t experts, int64_t ld,
                                       const int32_t* d_ids, int32_t k, int32_t score,
                                       int32_t renormalize, float scale, const float* d_dweights,
                                       const float* d_dscores, void* d_dlogits, int64_t ldd,
                                       void* stream) {
  if (!res || !d_ids || !d_dweights || !known_score(score) || k <= 0 || !aligned(d_ids, 4) ||
      !aligned(d_dweights, 4) || !aligned(d_dscores, 4))
    return OVVS_STATUS_INVALID_ARGUMENT;
  OVVS_TRY(check_matrix(d_logits, type, tokens, experts, ld));
  OVVS_TRY(check_matrix(d_dlogits, type, tokens, experts, ldd));
  if (experts > ovvs::prim::kRouteMaxExperts || k > ovvs::prim::kRouteMaxK)
    return OVVS_STATUS_SHAPE_MISMATCH;
  ovvs::prim::RouteBackwardParams p{};
  p.logits = d_logits;
  p.tokens = tokens;
  p.ld = ld;
  p.experts = static_cast<int>(experts);
  p.ids = d_ids;
  p.k = k;
  p.sigmoid = score == OVVS_ROUTE_SIGMOID;
  p.renormalize = renormalize != 0;
  p.scale = scale;
  p.dweights = d_dweights;
  p.dscores = d_dscores;
  p.dlogits = d_dlogits;
  p.ldd = ldd;
  // the logits' own memory, row for row, is allowed
  const bool in_place = d_dlogits == d_logits && (ldd == ld || tokens == 1);
  const Span out = span_of(d_dlogits, tokens, experts, ldd, type_bytes(type));
  const bool shared = clash(
      {out}, {in_place ? Span{} : span_of(d_logits, tokens, experts, ld, type_bytes(type)),
              span_of(d_ids, tokens * k, 4), span_of(d_dweights, tokens * k, 4),
              span_of(d_dscores, tokens * experts, 4)});
  return launched(*from_handle(res), shared, [&] {
    return ovvs::prim::launch_route_topk_backward(p, type, static_cast<cudaStream_t>(stream));
  });
}

ovvsStatus ovvsRoutePlanDevice(ovvsResources_t res, const int32_t* d_ids, int64_t pairs,
                               int64_t experts, int32_t align, int32_t* d_offsets,
                               int32_t* d_order, int64_t capacity, int32_t* d_position,
                               void* stream) {
  if (!res || !d_ids || !d_offsets || !d_order || !d_position || pairs <= 0 || experts <= 0 ||
      align <= 0 || capacity <= 0 || !aligned(d_ids, 4) || !aligned(d_offsets, 4) ||
      !aligned(d_order, 4) || !aligned(d_position, 4))
    return OVVS_STATUS_INVALID_ARGUMENT;
  if (pairs > 0x7fffffffLL || capacity > 0x7fffffffLL || experts > ovvs::prim::kRouteMaxExperts)
    return OVVS_STATUS_SHAPE_MISMATCH;
  // every expert that has a pair may leave align - 1 places of its last tile empty
  if (capacity < pairs + (experts < pairs ? experts : pairs) * (int64_t{align} - 1))
    return OVVS_STATUS_SHAPE_MISMATCH;
  const bool shared = clash({span_of(d_offsets, experts + 1, 4), span_of(d_order, capacity, 4),
                             span_of(d_position, pairs, 4)},
                            {span_of(d_ids, pairs, 4)});
  return launched(*from_handle(res), shared, [&] {
    return ovvs::prim::launch_route_plan(d_ids, pairs, static_cast<int>(experts), align,
                                         d_offsets, d_order, capacity, d_position,
                                         static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
