// Routing tokens to experts and its gradient (see rows.cuh).
//
// s = softmax(x) or sigmoid(x) over the experts of a token; the choice c is x itself without a
// bias and s + bias with one. With groups, only the experts of the topk_groups groups with the
// best group values (best c, or the sum of the two best) stand. The k experts with the largest c
// are chosen, equal ones by lower id, and weighted by scale * s, or by scale * s / (sum of the
// chosen s).
//
// Which expert is chosen is what 64 bits say: two experts of one token may stand nearer than 32
// bits tell apart. The fast way computes in 32 bits and knows how far it may be off (kDoubt): it
// decides alone where neighbours in the order stand further apart than that, orders the few
// doubtful experts by their 64-bit values where not, and hands a token whose groups are in doubt
// to the plain 64-bit way.
#include "rows.cuh"

#include "keys.cuh"
#include "score_load.cuh"

namespace ovvs {
namespace prim {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;

// How near two choices s + bias computed in 32 bits may stand before their order is in doubt,
// relative to the larger of 1 and their size, in units of 2^-24. A sigmoid is off by at most 4.3:
// the exponential's own 4, which s (1 - s) quarters, its rounded argument 1.2 |x| s (1 - s) < 0.3,
// one rounding of the denominator, two of the reciprocal. A softmax by at most 49: the same for
// its numerator, and its sum of up to 1024 terms. Adding the bias rounds half a unit. Both sides
// of a pair, and twice that to be safe; sums of two choices count twice again.
constexpr float kUnit = 5.9604645e-8f;
constexpr float kDoubtSigmoid = 24.f * kUnit;
constexpr float kDoubtSoftmax = 200.f * kUnit;

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

// Sum and maximum over groups of kLanes lanes.
template <int kLanes, class V>
__device__ __forceinline__ V lanes_sum(V v) {
#pragma unroll
  for (int o = kLanes / 2; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}
template <int kLanes>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = kLanes / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  return v;
}
template <int kLanes>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  if constexpr (kLanes == 32) {
    return __reduce_max_sync(~0u, v);
  } else {
#pragma unroll
    for (int o = kLanes / 2; o; o >>= 1) v = max(v, __shfl_xor_sync(~0u, v, o));
    return v;
  }
}

// -inf and NaN are masked.
__device__ __forceinline__ float masked(float v) { return v > -INFINITY ? v : -INFINITY; }

// Position in the order as an integer: larger is earlier, 0 cannot be chosen.
__device__ __forceinline__ uint32_t choice_key(float c) {
  return c > -INFINITY ? keys::order_bits(c) : 0u;
}

__device__ __forceinline__ float exp_fast(float x) {  // 2^-22 and the argument's rounding
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.44269504f));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {  // one unit
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float sigmoid_fast(float x) { return rcp_fast(1.f + exp_fast(-x)); }

// A chosen expert's score over a power of e common to the token's chosen ones, whose largest
// logit is `top`: their ratios hold where the scores themselves would vanish.
__device__ __forceinline__ float relative_score(float v, float top, bool sigmoid) {
  if (!sigmoid) return v == top ? 1.f : exp_fast(v - top);
  const float base = fminf(top, 0.f);
  return 1.f / (exp_fast(base) + (v == base ? 1.f : exp_fast(base - v)));
}

// The plain way: one warp takes the token, choice and score of each expert in shared memory
// (2 * experts doubles), everything in 64 bits. Scores are written only if asked for.
template <class T>
__device__ __noinline__ void route_token(const RouteParams& p, int64_t t, double* choice,
                                         bool write_scores) {
  const int lane = threadIdx.x & 31;
  double* score = choice + p.experts;
  const T* x = static_cast<const T*>(p.logits) + t * p.ld;
  const int n = p.experts;

  float m = -INFINITY;
  for (int e = lane; e < n; e += 32) m = fmaxf(m, masked(score_f32(x[e])));
  m = lanes_max<32>(m);
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
  z = lanes_sum<32>(z);
  for (int e = lane; e < n; e += 32) {
    const float v = masked(score_f32(x[e]));
    double s = score[e];
    if (!p.sigmoid && s > 0.0) s /= z;
    score[e] = s;
    double c = p.bias ? s + p.bias[e] : static_cast<double>(v);
    if (!(v > -INFINITY) || !(c > -INFINITY)) c = -INFINITY;
    choice[e] = c;
    if (write_scores) p.scores[t * n + e] = static_cast<float>(s);
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
  const float top = lanes_max<32>(v);
  double w = 0.0;
  if (mine >= 0) {
    if (!p.renormalize) {
      w = score[mine];
    } else if (p.sigmoid) {
      const double base = fminf(top, 0.f);
      w = 1.0 / (exp(base) + (v == base ? 1.0 : exp(base - static_cast<double>(v))));
    } else {
      w = v == top ? 1.0 : exp(static_cast<double>(v) - top);
    }
  }
  if (p.renormalize) {
    const double total = lanes_sum<32>(w);
    w = total > 0.0 ? w / total : 0.0;
  }
  if (lane < p.k) {
    p.ids[t * p.k + lane] = mine;
    p.weights[t * p.k + lane] = static_cast<float>(w * p.scale);
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads) route_plain_kernel(RouteParams p) {
  extern __shared__ double smem[];
  const int warp = threadIdx.x >> 5;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  if (t < p.tokens)
    route_token<T>(p, t, smem + static_cast<size_t>(warp) * 2 * p.experts, p.scores != nullptr);
}

// Loads or stores the kPer neighbours of a row from column e0 on; `whole` rows allow 16-byte
// (or, for fewer bytes, one) accesses.
template <class T, int kPer>
__device__ __forceinline__ void load_cells(const T* row, int e0, int n, bool whole,
                                           float (&v)[kPer], float other) {
  constexpr int kBytes = kPer * sizeof(T);
  if (whole) {
    if (e0 < n) {
      T raw[kPer];
      if constexpr (kBytes >= 16) {
#pragma unroll
        for (int i = 0; i < kBytes / 16; ++i)
          reinterpret_cast<uint4*>(raw)[i] = __ldg(reinterpret_cast<const uint4*>(row + e0) + i);
      }
#pragma unroll
      for (int i = 0; i < kPer; ++i) v[i] = score_f32(raw[i]);
      return;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = other;
    return;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) v[i] = e0 + i < n ? score_f32(row[e0 + i]) : other;
}
template <class T, int kPer>
__device__ __forceinline__ void store_cells(T* row, int e0, int n, bool whole,
                                            const float (&v)[kPer]) {
  constexpr int kBytes = kPer * sizeof(T);
  if (whole) {
    if (e0 >= n) return;
    T raw[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) raw[i] = score_from<T>(v[i]);
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i)
      reinterpret_cast<uint4*>(row + e0)[i] = reinterpret_cast<const uint4*>(raw)[i];
    return;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (e0 + i < n) row[e0 + i] = score_from<T>(v[i]);
}

// The fast way: kLanes lanes take a token, each kPer neighbouring experts in registers. Groups,
// where there are any, are whole lanes: group_lanes (a power of two) each.
template <class T, int kLanes, int kPer>
__global__ void __launch_bounds__(kThreads)
route_kernel(RouteParams p, int group_lanes, bool whole, bool whole_scores) {
  extern __shared__ double smem[];
  __shared__ int ids_of[kWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kTokens = 32 / kLanes;
  const int sub = lane % kLanes, n = p.experts, k = p.k;
  const int64_t t0 = (static_cast<int64_t>(blockIdx.x) * kWarps + warp) * kTokens;
  if (t0 >= p.tokens) return;
  const int64_t t = t0 + lane / kLanes;
  const bool live = t < p.tokens;
  const T* x = static_cast<const T*>(p.logits) + (live ? t : t0) * p.ld;
  const int e0 = sub * kPer;
  const unsigned mine = (kLanes == 32 ? ~0u : (1u << kLanes) - 1) << (lane / kLanes * kLanes);

  float v[kPer];
  load_cells<T, kPer>(x, e0, n, whole, v, -INFINITY);
#pragma unroll
  for (int i = 0; i < kPer; ++i) v[i] = masked(v[i]);
  const bool need_scores = p.bias || p.scores || (p.groups > 1 && p.group_top2);
  float m = 0.f, inv_z = 0.f;
  if (!p.sigmoid && (need_scores || !p.renormalize)) {
    m = v[0];
#pragma unroll
    for (int i = 1; i < kPer; ++i) m = fmaxf(m, v[i]);
    m = lanes_max<kLanes>(m);
    float z = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      z += v[i] > -INFINITY ? (v[i] == m ? 1.f : exp_fast(v[i] - m)) : 0.f;
    z = lanes_sum<kLanes>(z);
    inv_z = z > 0.f ? 1.f / z : 0.f;
  }
  auto score = [&](float y) {
    if (!(y > -INFINITY)) return 0.f;
    if (p.sigmoid) return sigmoid_fast(y);
    return (y == m ? 1.f : exp_fast(y - m)) * inv_z;
  };
  uint32_t key[kPer];
  if (need_scores) {
    float s[kPer], b[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) s[i] = score(v[i]);
    if (p.scores && live)
      store_cells<float, kPer>(p.scores + t * n, e0, n, whole_scores, s);
    if (p.bias) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) b[i] = e0 + i < n ? __ldg(p.bias + e0 + i) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      key[i] = v[i] > -INFINITY ? choice_key(p.bias ? s[i] + b[i] : v[i]) : 0u;
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) key[i] = choice_key(v[i]);
  }
  const float doubt = p.sigmoid ? kDoubtSigmoid : kDoubtSoftmax;
  auto near = [&](float a, float b) {
    return a - b <= doubt * fmaxf(1.f, fmaxf(fabsf(a), fabsf(b)));
  };
  bool plain = false;  // this token goes the plain way

  if (p.groups > 1) {
    // the group's value on its lanes: the best choice, or the sum of the two best
    uint32_t gkey;
    const bool sums = p.group_top2;
    {
      uint32_t best = 0, second = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        second = max(second, min(best, key[i]));
        best = max(best, key[i]);
      }
      for (int o = 1; o < group_lanes; o <<= 1) {
        const uint32_t b2 = __shfl_xor_sync(~0u, best, o), s2 = __shfl_xor_sync(~0u, second, o);
        second = max(min(best, b2), max(second, s2));
        best = max(best, b2);
      }
      if (sums && best) {
        auto value = [&](uint32_t key) {
          const float c = keys::order_value(key);
          return p.bias ? c : score(c);
        };
        gkey = choice_key(second ? value(best) + value(second) : value(best));
      } else {
        gkey = best;
      }
    }
    // stands: how many groups are better (equal ones: lower) is below topk_groups
    uint32_t left = gkey, last = 0;
    bool open = false;
    for (int i = 0; i < p.topk_groups; ++i) {
      const uint32_t big = lanes_max<kLanes>(left);
      const unsigned who = __ballot_sync(~0u, left == big && big) & mine;
      if (who && sub / group_lanes == (__ffs(who) - 1) % kLanes / group_lanes) {
        open = true;
        left = 0;
      }
      last = big;
    }
    if (sums || p.bias) {  // in doubt: the best group that fell, near the last that stands
      const uint32_t fell = lanes_max<kLanes>(left);
      const float a = keys::order_value(last), b = keys::order_value(fell);
      plain = last && fell && near(sums ? 0.5f * a : a, sums ? 0.5f * b : b);
    }
    if (!open) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) key[i] = 0;
    }
  }

  // The k best, one at a time (with a bias also the one after them), on lanes 0.. of the token:
  // slot j of lane s is number j * kLanes + s.
  constexpr int kSlots = 32 / kLanes;
  int id[kSlots];
  uint32_t at[kSlots];
#pragma unroll
  for (int j = 0; j < kSlots; ++j) {
    id[j] = -1;
    at[j] = 0;
  }
  uint32_t best = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) best = max(best, key[i]);
  int next_id = -1;
  uint32_t next_key = 0;
  const int rounds = p.bias ? k + 1 : k;
  for (int r = 0; r < rounds; ++r) {
    const uint32_t big = lanes_max<kLanes>(best);
    const unsigned who = __ballot_sync(~0u, best == big) & mine;
    const int from = __ffs(who) - 1;
    int e = 0;
    if (lane == from && big) {
      bool found = false;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const bool hit = !found && key[i] == big;
        found = found || hit;
        e = hit ? i : e;
        if (hit && r < k) key[i] = 0;
      }
      best = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) best = max(best, key[i]);
    }
    e = __shfl_sync(~0u, e, from) + from % kLanes * kPer;
    if (r < k) {
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        if (j * kLanes + sub == r && big) {
          id[j] = e;
          at[j] = big;
        }
      }
    } else if (big) {
      next_id = e;
      next_key = big;
    }
  }

  if (p.bias) {
    // Neighbours in the order that stand too near: settled if they are equal in logit and bias
    // (lower ids come first); the k-th and what is left have to be clear apart. Else 64 bits
    // decide.
    bool in_doubt = false;
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      const int r = j * kLanes + sub;
      int i2 = __shfl_down_sync(~0u, id[j], 1, kLanes);
      uint32_t k2 = __shfl_down_sync(~0u, at[j], 1, kLanes);
      const int i3 = j + 1 < kSlots ? __shfl_sync(~0u, id[j + 1 < kSlots ? j + 1 : j], 0, kLanes) : -1;
      const uint32_t k3 = j + 1 < kSlots ? __shfl_sync(~0u, at[j + 1 < kSlots ? j + 1 : j], 0, kLanes) : 0;
      if (sub == kLanes - 1) {
        i2 = i3;
        k2 = k3;
      }
      if (r == k - 1) {
        i2 = next_id;
        k2 = next_key;
      }
      if (r < k && at[j] && k2 && near(keys::order_value(at[j]), keys::order_value(k2))) {
        const float xa = score_f32(x[id[j]]), xb = score_f32(x[i2]);
        const bool settled = r < k - 1 && __ldg(p.bias + id[j]) == __ldg(p.bias + i2) &&
                             xa == xb && id[j] < i2;
        in_doubt = in_doubt || !settled;
      }
    }
    in_doubt = __ballot_sync(~0u, in_doubt) & mine;
    unsigned todo = __ballot_sync(~0u, in_doubt && live && !plain && sub == 0);
    while (todo) {  // one token at a time, by the whole warp
      const int lead = __ffs(todo) - 1, first = lead, slot0 = lead / kLanes;
      todo &= todo - 1;
      const T* xt = static_cast<const T*>(p.logits) + (t0 + slot0) * p.ld;
      const bool here = lane / kLanes == slot0;
      // candidates: the chosen, and what is left within reach of the last of them
      uint32_t cut = 0;
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        const uint32_t y = __shfl_sync(~0u, at[j], first + (k - 1) % kLanes);
        if (j == (k - 1) / kLanes) cut = y;
      }
      int count = 0;
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        const bool in = here && id[j] >= 0;
        const unsigned who = __ballot_sync(~0u, in);
        if (in) ids_of[warp][count + __popc(who & ((1u << lane) - 1))] = id[j];
        count += __popc(who);
      }
      if (cut) {
        const float least = keys::order_value(cut);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const bool in = here && key[i] && near(least, keys::order_value(key[i]));
          const unsigned who = __ballot_sync(~0u, in);
          const int place = count + __popc(who & ((1u << lane) - 1));
          if (in && place < 32) ids_of[warp][place] = e0 + i;
          count += __popc(who);
        }
      }
      if (count > 32) {
        if (here) plain = true;
        continue;
      }
      __syncwarp();
      double md = -INFINITY, z = 1.0;
      if (!p.sigmoid) {
        float mf = -INFINITY;
        for (int e = lane; e < n; e += 32) mf = fmaxf(mf, masked(score_f32(xt[e])));
        mf = lanes_max<32>(mf);
        md = mf;
        z = 0.0;
        for (int e = lane; e < n; e += 32) {
          const float y = masked(score_f32(xt[e]));
          if (y > -INFINITY) z += y == mf ? 1.0 : exp(static_cast<double>(y) - md);
        }
        z = lanes_sum<32>(z);
      }
      int e = n;
      double c = -INFINITY;
      if (lane < count) {
        e = ids_of[warp][lane];
        const float y = score_f32(xt[e]);
        const double s = p.sigmoid ? 1.0 / (1.0 + exp(-static_cast<double>(y)))
                                   : (y == md ? 1.0 : exp(static_cast<double>(y) - md)) / z;
        c = s + static_cast<double>(__ldg(p.bias + e));
      }
      int rank = 0;
      for (int l = 0; l < count; ++l) {
        const double cl = __shfl_sync(~0u, c, l);
        const int el = __shfl_sync(~0u, e, l);
        rank += better(cl, el, c, e);
      }
      __syncwarp();
      if (lane < count) ids_of[warp][rank] = e;
      __syncwarp();
      if (here) {
#pragma unroll
        for (int j = 0; j < kSlots; ++j) {
          const int r = j * kLanes + sub;
          if (r < k && r < count) id[j] = ids_of[warp][r];
        }
      }
      __syncwarp();
    }
  }

  // weights
  float y[kSlots], top = -INFINITY;
#pragma unroll
  for (int j = 0; j < kSlots; ++j) {
    y[j] = id[j] >= 0 ? score_f32(x[id[j]]) : -INFINITY;
    top = fmaxf(top, y[j]);
  }
  float w[kSlots], total = 0.f;
  if (p.renormalize) {
    top = lanes_max<kLanes>(top);
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      w[j] = id[j] >= 0 ? relative_score(y[j], top, p.sigmoid) : 0.f;
      total += w[j];
    }
    total = lanes_sum<kLanes>(total);
#pragma unroll
    for (int j = 0; j < kSlots; ++j) w[j] = total > 0.f ? w[j] / total : 0.f;
  } else {
#pragma unroll
    for (int j = 0; j < kSlots; ++j) w[j] = score(y[j]);
  }
  if (live && !plain) {
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      const int r = j * kLanes + sub;
      if (r < k) {
        p.ids[t * k + r] = id[j];
        p.weights[t * k + r] = w[j] * p.scale;
      }
    }
  }
  unsigned again = __ballot_sync(~0u, plain && live && sub == 0);
  while (again) {
    const int lead = __ffs(again) - 1;
    again &= again - 1;
    route_token<T>(p, t0 + lead / kLanes, smem + static_cast<size_t>(warp) * 2 * n, false);
    __syncwarp();
  }
}

// dL/dx for L a function of the weights and, with dscores, of the scores. With p the chosen
// scores and S their sum: dL/dp_i = scale * dw_i, renormalised scale * (dw_i - sum_j w_j dw_j) / S
// (w before the scale); then ds = dscores + the chosen dp and dx = ds s (1 - s), or
// s (ds - sum ds s). Renormalised weights alone need no S: p_i / S is a ratio of exponentials
// relative to the largest chosen one. Where only chosen experts have a gradient (no dscores, and
// sigmoids or renormalised weights), the other logits are not read at all.
template <class T, int kLanes, int kPer>
__global__ void __launch_bounds__(kThreads)
route_backward_kernel(RouteBackwardParams p, bool whole, bool whole_out, bool whole_scores) {
  extern __shared__ __align__(16) float rows[];  // a row of the chosen experts' parts for each token
  constexpr int kTokens = 32 / kLanes, kCells = kLanes * kPer;
  constexpr int kSlots = 32 / kLanes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane % kLanes, n = p.experts, k = p.k;
  const int64_t t0 = (static_cast<int64_t>(blockIdx.x) * kWarps + warp) * kTokens;
  if (t0 >= p.tokens) return;
  const bool live = t0 + lane / kLanes < p.tokens;
  const int64_t t = live ? t0 + lane / kLanes : t0;
  const T* x = static_cast<const T*>(p.logits) + t * p.ld;
  T* dx = static_cast<T*>(p.dlogits) + t * p.ldd;
  const int e0 = sub * kPer;
  float* part = rows + (warp * kTokens + lane / kLanes) * (kCells + 64);
  float* own_of = part + kCells;
  int* id_of = reinterpret_cast<int*>(own_of + 32);
  const bool dense = p.dscores || (!p.sigmoid && !p.renormalize);

  // the chosen: slot j of lane s is number j * kLanes + s
  int id[kSlots];
  float y[kSlots], dw[kSlots], top = -INFINITY;
#pragma unroll
  for (int j = 0; j < kSlots; ++j) {
    const int r = j * kLanes + sub;
    id[j] = r < k ? p.ids[t * k + r] : -1;
    if (id[j] >= n) id[j] = -1;
    y[j] = id[j] >= 0 ? masked(score_f32(x[id[j]])) : -INFINITY;
    if (!(y[j] > -INFINITY)) id[j] = -1;
    dw[j] = id[j] >= 0 ? p.dweights[t * k + r] * p.scale : 0.f;
    top = fmaxf(top, y[j]);
  }
  float v[kPer], d[kPer], m = 0.f, inv_z = 0.f;
  if (dense) {
    load_cells<T, kPer>(x, e0, n, whole, v, -INFINITY);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      v[i] = masked(v[i]);
      d[i] = 0.f;
    }
    if (p.dscores) {
      load_cells<float, kPer>(p.dscores + t * n, e0, n, whole_scores, d, 0.f);
#pragma unroll
      for (int i = 0; i < kPer; ++i) d[i] = v[i] > -INFINITY ? d[i] : 0.f;
    }
    if (!p.sigmoid) {
      m = v[0];
#pragma unroll
      for (int i = 1; i < kPer; ++i) m = fmaxf(m, v[i]);
      m = lanes_max<kLanes>(m);
      float z = 0.f;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        v[i] = v[i] > -INFINITY ? (v[i] == m ? 1.f : exp_fast(v[i] - m)) : 0.f;
        z += v[i];
      }
      z = lanes_sum<kLanes>(z);
      inv_z = z > 0.f ? 1.f / z : 0.f;
#pragma unroll
      for (int i = 0; i < kPer; ++i) v[i] *= inv_z;  // the scores from here on
    }
  }
  // own: the chosen experts' part of the gradient; dot: what every softmax gradient subtracts
  float own[kSlots], dot = 0.f;
  if (p.renormalize) {
    top = lanes_max<kLanes>(top);
    float total = 0.f, mean = 0.f;
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      own[j] = id[j] >= 0 ? relative_score(y[j], top, p.sigmoid) : 0.f;
      total += own[j];
    }
    total = lanes_sum<kLanes>(total);
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      own[j] = total > 0.f ? own[j] / total : 0.f;
      mean += own[j] * dw[j];
    }
    mean = lanes_sum<kLanes>(mean);
#pragma unroll
    for (int j = 0; j < kSlots; ++j) own[j] *= dw[j] - mean;
  } else {
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      const float s = p.sigmoid ? sigmoid_fast(y[j])
                                : (y[j] == m ? 1.f : exp_fast(y[j] - m)) * inv_z;
      own[j] = id[j] >= 0 ? s * dw[j] : 0.f;
      if (!p.sigmoid) dot += own[j];
    }
  }
  if (p.sigmoid) {
#pragma unroll
    for (int j = 0; j < kSlots; ++j)
      if (id[j] >= 0) own[j] *= sigmoid_fast(-y[j]);  // 1 - s
  } else if (dense) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) dot += v[i] * d[i];
    dot = lanes_sum<kLanes>(dot);
  }
  // the parts at their places, added in order where an expert stands twice
  float4* cells = reinterpret_cast<float4*>(part + e0);
#pragma unroll
  for (int i = 0; i < kPer / 4; ++i) cells[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int j = 0; j < kSlots; ++j) {
    own_of[j * kLanes + sub] = own[j];
    id_of[j * kLanes + sub] = id[j];
  }
  __syncwarp();
  if (sub == 0) {
    for (int r = 0; r < k; ++r)
      if (id_of[r] >= 0) part[id_of[r]] += own_of[r];
  }
  __syncwarp();
  float g[kPer];
#pragma unroll
  for (int i = 0; i < kPer / 4; ++i) {
    const float4 c = cells[i];
    g[4 * i] = c.x;
    g[4 * i + 1] = c.y;
    g[4 * i + 2] = c.z;
    g[4 * i + 3] = c.w;
  }
  if (dense) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (p.sigmoid) {
        const float ex = exp_fast(-fabsf(v[i])), q = rcp_fast(1.f + ex);
        if (v[i] > -INFINITY) g[i] += d[i] * ex * q * q;
      } else {
        g[i] += v[i] * (d[i] - dot);
      }
    }
  }
  if (live) store_cells<T, kPer>(dx, e0, n, whole_out, g);
}

bool lines_up(const void* p, int64_t stride_bytes, size_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride_bytes % static_cast<int64_t>(bytes) == 0;
}

template <class T, int kLanes, int kPer>
cudaError_t route_fast(const RouteParams& p, int group_lanes, cudaStream_t stream) {
  const bool whole = p.experts % kPer == 0 && lines_up(p.logits, p.ld * sizeof(T), 16);
  const bool whole_scores = p.experts % kPer == 0 &&
                            lines_up(p.scores, int64_t{p.experts} * sizeof(float), 16);
  // the plain way's room: only a token whose groups or many experts are in doubt needs it
  const size_t smem = p.bias || (p.groups > 1 && p.group_top2)
                          ? static_cast<size_t>(kWarps) * 2 * p.experts * sizeof(double) : 0;
  static std::atomic<uint64_t> done;
  const cudaError_t e = allow_smem(route_kernel<T, kLanes, kPer>, 64 * 1024, done);
  if (e != cudaSuccess) return e;
  constexpr int kTokens = kWarps * 32 / kLanes;
  route_kernel<T, kLanes, kPer>
      <<<static_cast<unsigned>((p.tokens + kTokens - 1) / kTokens), kThreads, smem, stream>>>(
          p, group_lanes, whole, whole_scores);
  return cudaGetLastError();
}

template <class T>
cudaError_t route(const RouteParams& p, cudaStream_t stream) {
  // Eight experts a lane, and as few lanes a token as hold them: four tokens of 64 experts share
  // a warp's instructions. Groups have to be whole lanes, a power of two of them.
  const int per = p.experts <= 256 ? 8 : p.experts <= 512 ? 16 : 32;
  const int size = p.experts / p.groups;
  const int lanes = size / per;
  if (p.groups == 1 || (size % per == 0 && (lanes & (lanes - 1)) == 0)) {
    const int group_lanes = p.groups == 1 ? 1 : lanes;
    if (p.experts <= 64) return route_fast<T, 8, 8>(p, group_lanes, stream);
    if (p.experts <= 128) return route_fast<T, 16, 8>(p, group_lanes, stream);
    if (p.experts <= 256) return route_fast<T, 32, 8>(p, group_lanes, stream);
    if (p.experts <= 512) return route_fast<T, 32, 16>(p, group_lanes, stream);
    return route_fast<T, 32, 32>(p, group_lanes, stream);
  }
  const size_t smem = static_cast<size_t>(kWarps) * 2 * p.experts * sizeof(double);
  static std::atomic<uint64_t> done;
  const cudaError_t e = allow_smem(route_plain_kernel<T>, 64 * 1024, done);
  if (e != cudaSuccess) return e;
  route_plain_kernel<T><<<static_cast<unsigned>((p.tokens + kWarps - 1) / kWarps), kThreads, smem,
                          stream>>>(p);
  return cudaGetLastError();
}

template <class T, int kLanes, int kPer>
cudaError_t route_backward_as(const RouteBackwardParams& p, cudaStream_t stream) {
  const bool cells = p.experts % kPer == 0;
  const bool whole = cells && lines_up(p.logits, p.ld * sizeof(T), 16);
  const bool whole_out = cells && lines_up(p.dlogits, p.ldd * sizeof(T), 16);
  const bool whole_scores = cells && lines_up(p.dscores, int64_t{p.experts} * sizeof(float), 16);
  constexpr int kTokens = kWarps * 32 / kLanes;
  constexpr size_t smem = static_cast<size_t>(kTokens) * (kLanes * kPer + 64) * sizeof(float);
  static_assert(smem <= 48 * 1024, "no opt-in needed");
  route_backward_kernel<T, kLanes, kPer>
      <<<static_cast<unsigned>((p.tokens + kTokens - 1) / kTokens), kThreads, smem, stream>>>(
          p, whole, whole_out, whole_scores);
  return cudaGetLastError();
}

template <class T>
cudaError_t route_backward(const RouteBackwardParams& p, cudaStream_t stream) {
  if (p.experts <= 64) return route_backward_as<T, 8, 8>(p, stream);
  if (p.experts <= 128) return route_backward_as<T, 16, 8>(p, stream);
  if (p.experts <= 256) return route_backward_as<T, 32, 8>(p, stream);
  if (p.experts <= 512) return route_backward_as<T, 32, 16>(p, stream);
  return route_backward_as<T, 32, 32>(p, stream);
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
