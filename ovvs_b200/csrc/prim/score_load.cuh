// Scores of the three types the row operators take, as fp32 (every fp16 and bf16 value is one).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace ovvs {
namespace prim {

__device__ __forceinline__ float score_f32(float v) { return v; }
__device__ __forceinline__ float score_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float score_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// One rounding, to nearest even.
template <class T>
__device__ __forceinline__ T score_from(float v);
template <>
__device__ __forceinline__ float score_from<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half score_from<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 score_from<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

}  // namespace prim
}  // namespace ovvs
