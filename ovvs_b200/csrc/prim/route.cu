// Routing tokens to experts and its gradient (see rows.cuh).
//
// s = softmax(x) or sigmoid(x) over the experts of a token; the choice c is x itself without a
// bias and s + bias with one. With groups, only the experts of the topk_groups groups with the
// best group values (best c, or the sum of the two best) stand. The k experts with the largest c
// are chosen, equal ones by lower id, and weighted by scale * s, or by scale * s / (sum of the
// chosen s).
//
// Which expert is chosen is decided in 64 bits: two experts of one token may stand nearer than
// 32 bits tell apart.
#include "rows.cuh"

#include "score_load.cuh"

namespace ovvs {
namespace prim {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;

__device__ __forceinline__ bool better(double a, int i, double b, int j) {
  return a > b || (a == b && i < j);
}

// The best (value, id) of the warp, on every lane.
__device__ __forceinline__ void warp_best(double& v, int& id) {
  for (int o = 16; o; o >>= 1) {
    const double w = __shfl_xor_sync(~0u, v, o);
    const int j = __shfl_xor_sync(~0u, id, o);
    if (better(w, j, v, id)) {
      v = w;
      id = j;
    }
  }
}

__device__ __forceinline__ double warp_sum(double v) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  return v;
}

// -inf and NaN are masked.
__device__ __forceinline__ float masked(float v) { return v > -INFINITY ? v : -INFINITY; }

// One warp a token; choice and score of each expert in shared memory.
template <class T>
__global__ void __launch_bounds__(kThreads) route_kernel(RouteParams p) {
  extern __shared__ double smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double* choice = smem + static_cast<size_t>(warp) * 2 * p.experts;
  double* score = choice + p.experts;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  if (t >= p.tokens) return;
  const T* x = static_cast<const T*>(p.logits) + t * p.ld;
  const int n = p.experts;

  float m = -INFINITY;
  for (int e = lane; e < n; e += 32) m = fmaxf(m, masked(score_f32(x[e])));
  m = warp_max(m);
  double z = 0.0;
  for (int e = lane; e < n; e += 32) {
    const float v = masked(score_f32(x[e]));
    double s = 0.0;
    if (v > -INFINITY)
      s = p.sigmoid ? 1.0 / (1.0 + exp(-static_cast<double>(v)))
                    : (v == m ? 1.0 : exp(static_cast<double>(v) - m));
    score[e] = s;
    z += s;
  }
  z = warp_sum(z);
  for (int e = lane; e < n; e += 32) {
    const float v = masked(score_f32(x[e]));
    double s = score[e];
    if (!p.sigmoid && s > 0.0) s /= z;
    score[e] = s;
    double c = p.bias ? s + p.bias[e] : static_cast<double>(v);
    if (!(v > -INFINITY) || !(c > -INFINITY)) c = -INFINITY;
    choice[e] = c;
    if (p.scores) p.scores[t * n + e] = static_cast<float>(s);
  }
  __syncwarp();
  if (p.groups > 1) {
    const int per = n / p.groups;
    double g = -INFINITY;
    if (lane < p.groups) {
      double a = -INFINITY, b = -INFINITY;  // the two best
      for (int i = 0; i < per; ++i) {
        const int e = lane * per + i;
        double c = choice[e];
        if (p.group_top2 && !p.bias && c > -INFINITY) c = score[e];
        if (c > a) {
          b = a;
          a = c;
        } else if (c > b) {
          b = c;
        }
      }
      g = p.group_top2 && b > -INFINITY ? a + b : a;
    }
    unsigned open = 0;
    for (int i = 0; i < p.topk_groups; ++i) {
      double v = lane < p.groups && !(open >> lane & 1) ? g : -INFINITY;
      int id = v > -INFINITY ? lane : 32;
      warp_best(v, id);
      if (id < 32) open |= 1u << id;
    }
    for (int e = lane; e < n; e += 32)
      if (!(open >> (e / per) & 1)) choice[e] = -INFINITY;
    __syncwarp();
  }
  int mine = -1;  // lane i: the i-th expert
  for (int i = 0; i < p.k; ++i) {
    double v = -INFINITY;
    int id = n;
    for (int e = lane; e < n; e += 32) {
      if (choice[e] > v) {
        v = choice[e];
        id = e;
      }
    }
    warp_best(v, id);
    if (id < n && lane == (id & 31)) choice[id] = -INFINITY;
    if (lane == i && id < n) mine = id;
    __syncwarp();
  }
  // The ratio of the chosen scores from exponentials relative to the largest of them, so that it
  // holds where the scores themselves would vanish.
  const float v = mine >= 0 ? score_f32(x[mine]) : -INFINITY;
  const float top = warp_max(v);
  double w = 0.0;
  if (mine >= 0) {
    if (!p.renormalize) {
      w = score[mine];
    } else if (p.sigmoid) {
      const double base = fminf(top, 0.f);
      w = 1.0 / (exp(base) + (v == base ? 1.0 : exp(base - v)));
    } else {
      w = v == top ? 1.0 : exp(static_cast<double>(v) - top);
    }
  }
  if (p.renormalize) {
    const double total = warp_sum(w);
    w = total > 0.0 ? w / total : 0.0;
  }
  if (lane < p.k) {
    p.ids[t * p.k + lane] = mine;
    p.weights[t * p.k + lane] = static_cast<float>(w * p.scale);
  }
}

// dL/dx for L a function of the weights and, with dscores, of the scores. With p the chosen
// scores and S their sum: dL/dp_i = scale * dw_i, renormalised scale * (dw_i - sum_j w_j dw_j) / S
// (w before the scale); then ds = dscores + the chosen dp and dx = ds s (1 - s), or
// s (ds - sum ds s). Renormalised weights alone need no S: p_i / S is a ratio of exponentials
// relative to the largest chosen one.
template <class T>
__global__ void __launch_bounds__(kThreads) route_backward_kernel(RouteBackwardParams p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  if (t >= p.tokens) return;
  const T* x = static_cast<const T*>(p.logits) + t * p.ld;
  T* dx = static_cast<T*>(p.dlogits) + t * p.ldd;
  const float* dsc = p.dscores ? p.dscores + t * p.experts : nullptr;
  const int n = p.experts;

  int id = lane < p.k ? p.ids[t * p.k + lane] : -1;
  if (id >= n) id = -1;
  float v = id >= 0 ? masked(score_f32(x[id])) : -INFINITY;
  if (!(v > -INFINITY)) id = -1;
  const float dw = id >= 0 ? p.dweights[t * p.k + lane] * p.scale : 0.f;

  float m = -INFINITY, z = 1.f;
  if (!p.sigmoid) {
    for (int e = lane; e < n; e += 32) m = fmaxf(m, masked(score_f32(x[e])));
    m = warp_max(m);
    z = 0.f;
    for (int e = lane; e < n; e += 32) {
      const float y = masked(score_f32(x[e]));
      if (y > -INFINITY) z += y == m ? 1.f : expf(y - m);
    }
    z = warp_sum(z);
  }
  // own: the chosen experts' part of the gradient, where it stands alone (times 1 - s later for
  // the sigmoid); dense: what every expert's softmax gradient subtracts.
  float own = 0.f, dot = 0.f;
  if (p.renormalize) {
    const float top = warp_max(v);
    float r = 0.f;
    if (id >= 0) {
      if (p.sigmoid) {
        const float base = fminf(top, 0.f);
        r = 1.f / (expf(base) + (v == base ? 1.f : expf(base - v)));
      } else {
        r = v == top ? 1.f : expf(v - top);
      }
    }
    const float total = warp_sum(r);
    r = total > 0.f ? r / total : 0.f;
    own = r * (dw - warp_sum(r * dw));
  } else if (id >= 0) {
    const float s = p.sigmoid ? 1.f / (1.f + expf(-v)) : (v == m ? 1.f : expf(v - m)) / z;
    own = s * dw;
  }
  if (!p.sigmoid) {
    if (!p.renormalize) dot = warp_sum(own);
    if (dsc) {
      float d = 0.f;
      for (int e = lane; e < n; e += 32) {
        const float y = masked(score_f32(x[e]));
        if (y > -INFINITY) d += (y == m ? 1.f : expf(y - m)) / z * dsc[e];
      }
      dot += warp_sum(d);
    }
  }
  for (int e0 = 0; e0 < n; e0 += 32) {
    const int e = e0 + lane;
    float sum = 0.f;
    for (int i = 0; i < p.k; ++i) {
      const int at = __shfl_sync(~0u, id, i);
      const float part = __shfl_sync(~0u, own, i);
      if (at == e) sum += part;
    }
    if (e >= n) continue;
    const float y = masked(score_f32(x[e]));
    float g = 0.f;
    if (y > -INFINITY) {
      const float d = dsc ? dsc[e] : 0.f;
      if (p.sigmoid) {
        const float ex = expf(-fabsf(y));
        const float low = ex / (1.f + ex), high = 1.f / (1.f + ex);
        const float rest = y >= 0.f ? low : high;  // 1 - s
        g = sum * rest + d * low * high;
      } else {
        const float s = (y == m ? 1.f : expf(y - m)) / z;
        g = sum + s * (d - dot);
      }
    }
    dx[e] = score_from<T>(g);
  }
}

template <class T>
cudaError_t route(const RouteParams& p, cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(kWarps) * 2 * p.experts * sizeof(double);
  const cudaError_t e = cudaFuncSetAttribute(
      route_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  route_kernel<T><<<static_cast<unsigned>((p.tokens + kWarps - 1) / kWarps), kThreads, smem,
                    stream>>>(p);
  return cudaGetLastError();
}

template <class T>
cudaError_t route_backward(const RouteBackwardParams& p, cudaStream_t stream) {
  route_backward_kernel<T>
      <<<static_cast<unsigned>((p.tokens + kWarps - 1) / kWarps), kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_route_topk(const RouteParams& p, int type, cudaStream_t stream) {
  if (type == kScoreF32) return route<float>(p, stream);
  if (type == kScoreF16) return route<__half>(p, stream);
  return route<__nv_bfloat16>(p, stream);
}

cudaError_t launch_route_topk_backward(const RouteBackwardParams& p, int type,
                                       cudaStream_t stream) {
  if (type == kScoreF32) return route_backward<float>(p, stream);
  if (type == kScoreF16) return route_backward<__half>(p, stream);
  return route_backward<__nv_bfloat16>(p, stream);
}

}  // namespace prim
}  // namespace ovvs
