// Routing tokens to experts and its gradient (see rows.cuh).
//
// s = softmax(x) or sigmoid(x) over the experts of a token; the choice c is x itself without a
// bias and s + bias with one. With groups, only the experts of the topk_groups groups with the
// best group values (best c, or the sum of the two best) stand. The k experts with the largest c
// are chosen, equal ones by lower id, and weighted by scale * s, or by scale * s / (sum of the
// chosen s).
//
// Which expert is chosen is what 64 bits say: two experts of one token may stand nearer than 32
// bits tell apart. The fast way computes in 32 bits and knows how far it may be off: it decides
// alone where neighbours in the order stand further apart than that, orders the few doubtful
// experts by their 64-bit values where not, and hands a token whose groups are in doubt to the
// plain 64-bit way (which takes 70 us for the first case below, were it to do all of it; a bias
// of 6 for every expert, whose codes are all cut off, sends every token there by way of the fast
// one: 103 us).
//
// What bounds it: instructions. A token of 256 experts, sigmoids, bias, 4 of 8 groups by their two
// best, top-8, costs a warp 780; 16,384 of them as fp32 take 22.4 us, of which reading them is 3.
// 32,768 tokens of 64 experts, softmax, top-6, bf16, all scores written: 9.3 us (14 MB, 2.2 at
// HBM's rate). Their gradient 6.7 us (18 MB, 2.8); that of 10,007 tokens of the first kind, which
// reads no logits but the chosen ones', 5.8 us (11 MB moved). 16,384 tokens of 512 and 1,024
// experts, softmax, top-8, bf16: 15 and 24 us; 160 experts in 8 groups, the plain way: 52.
#include "rows.cuh"

#include "keys.cuh"
#include "score_load.cuh"

namespace ovvs {
namespace prim {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;

// In the fast way an expert's place in the order is one 32-bit integer, its value's code above
// and its id (lower ones larger) below, so that no two are equal and the best is one maximum;
// 0 cannot be chosen. A value's code is
// - without a bias the leading bits of the logit's order-preserving image: all of a 16-bit
//   type's, so that nothing is in doubt; fp32 logits with the same leading bits are;
// - with one, s + bias in units of 2^-20 (2^-19 for more than 256 experts) between -4 and 4; what
//   lies beyond counts as the end of the range, and is in doubt among itself.
// A sigmoid is off by at most 4.3 * 2^-24: the exponential's own 4, which s (1 - s) quarters, its
// rounded argument 1.2 |x| s (1 - s) < 0.3, one rounding of the denominator, two of the
// reciprocal. A softmax by at most 49 * 2^-24: the same for its numerator, and its sum of up to
// 1024 terms. Adding the bias rounds by up to 4 * 2^-24 and the code by half a unit: 1.1 units
// for a sigmoid, 3.9 for a softmax (0.6 and 2 of the coarser units, and one that is cut off).
// Codes of a pair no further apart than twice that, rounded up, are in doubt.
constexpr int kNearSigmoid = 3, kNearSoftmax = 9;

// A group's sum of two is not made of codes, of which one that is cut off says nothing of the sum,
// but of fp32 values s + b of any size. It is off by at most two scores' errors, half a step of
// each part and of itself: 8.6 or 98 + 2 (|a| + |b|) in units of 2^-24; the bounds below leave room
// for their own rounding. What stands has to be clear of what falls by both errors; sums beyond
// fp32 are infinite, and in doubt among one another, as the bound stays finite.
constexpr float kUnit = 1.f / (1 << 24);
constexpr float kOffSigmoid = 9.f * kUnit, kOffSoftmax = 99.f * kUnit;

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

// c in units of 2^-20 above -4: c + 12 lies in [8, 16), where a float's last bit is one unit. At
// least 2, so that a code without its last bit is not 0 either: with the id 0 that would mark what
// cannot be chosen.
__device__ __forceinline__ uint32_t fixed_code(float c) {
  return __float_as_uint(fminf(fmaxf(c + 12.f, 8.000002f), 15.999999f)) & 0x7fffffu;
}

// Order-preserving image of what is not a NaN; -0 comes before +0.
__device__ __forceinline__ uint32_t image(float v) {
  const int u = __float_as_int(v);
  return static_cast<uint32_t>(u ^ (u >> 31 | static_cast<int>(0x80000000u)));
}

// For the choice alone, whose error is counted above: 2^-22 and the argument's rounding, which
// grows with it.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float exp_fast(float x) { return exp2_fast(x * 1.44269504f); }
__device__ __forceinline__ float rcp_fast(float x) {  // one unit
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float sigmoid_fast(float x) { return rcp_fast(1.f + exp_fast(-x)); }

// e^x for x <= 0, for what is written: e^x = 2^t e^(x - t ln 2) with t near x / ln 2, and the second
// factor, which makes up for t's rounding, is 1 + its exponent. Off by the first factor's 4 units
// of 2^-24, one rounding, and 0.05 |x| for ln 2 as a float: 9 at most. Three instructions more than
// the above: 1 % of the first case below, 4 of a gradient with all scores; expf cost 8 to 14 in
// every place. 0 from -104 down and for a NaN.
__device__ __forceinline__ float exp_down(float x) {
  x = fmaxf(x, -104.f);
  const float t = x * 1.44269504f, y = exp2_fast(t);
  return fmaf(y, fmaf(t, -0.693147182f, x), y);
}
__device__ __forceinline__ float sigmoid(float x) {  // 18 units of 2^-24 of itself
  const float e = exp_down(-fabsf(x)), q = rcp_fast(1.f + e);
  return x < 0.f ? e * q : q;
}

// A chosen expert's score over a power of e common to the token's chosen ones, whose largest
// logit is `top`: their ratios hold where the scores themselves would vanish.
__device__ __forceinline__ float relative_score(float v, float top, bool sigmoid) {
  if (!sigmoid) return v == top ? 1.f : exp_down(v - top);
  const float base = fminf(top, 0.f);
  return rcp_fast(exp_down(base) + (v == base ? 1.f : expf(base - v)));
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
// (or, for fewer bytes, one) accesses. kConst: nothing that the kernel writes may lie there.
template <class T, int kPer, bool kConst = true>
__device__ __forceinline__ void load_cells(const T* row, int e0, int n, bool whole,
                                           float (&v)[kPer], float other) {
  constexpr int kBytes = kPer * sizeof(T);
  if (whole) {
    if (e0 < n) {
      T raw[kPer];
      if constexpr (kBytes >= 16) {
#pragma unroll
        for (int i = 0; i < kBytes / 16; ++i) {
          const uint4* from = reinterpret_cast<const uint4*>(row + e0) + i;
          reinterpret_cast<uint4*>(raw)[i] = kConst ? __ldg(from) : *from;
        }
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
template <class T, int kLanes, int kPer, bool kBias>
__global__ void __launch_bounds__(kThreads)
route_kernel(RouteParams p, int group_lanes, bool whole, bool whole_scores) {
  extern __shared__ double smem[];
  __shared__ int ids_of[kWarps][32];
  constexpr int kIdBits = kLanes * kPer <= 256 ? 8 : 10;
  constexpr uint32_t kIds = (1u << kIdBits) - 1;
  constexpr int kDrop = kIdBits == 8 ? 0 : 1;  // of a code's 23 bits
  constexpr int kTokens = 32 / kLanes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
  const bool sums = p.groups > 1 && p.group_top2;
  const bool need_scores = kBias || p.scores;
  const bool scores_out = p.scores || !p.renormalize;  // they are not for the choice alone
  float s[kPer], m = 0.f, inv_z = 0.f;
  if (!p.sigmoid && (need_scores || sums || !p.renormalize)) {
    m = v[0];  // a NaN is not the larger one
#pragma unroll
    for (int i = 1; i < kPer; ++i) m = fmaxf(m, v[i]);
    m = lanes_max<kLanes>(fmaxf(m, -INFINITY));
    if (scores_out) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) s[i] = v[i] == m ? 1.f : exp_down(v[i] - m);
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) s[i] = v[i] == m ? 1.f : exp_fast(v[i] - m);
    }
    float z = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      s[i] = v[i] > -INFINITY ? s[i] : 0.f;
      z += s[i];
    }
    z = lanes_sum<kLanes>(z);
    inv_z = z > 0.f ? rcp_fast(z) : 0.f;
  }
  uint32_t key[kPer];
  if (need_scores) {
    if (!p.sigmoid) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) s[i] *= inv_z;
    } else if (scores_out) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) s[i] = v[i] > -INFINITY ? sigmoid(v[i]) : 0.f;
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) s[i] = v[i] > -INFINITY ? sigmoid_fast(v[i]) : 0.f;
    }
    if (p.scores && live) store_cells<float, kPer>(p.scores + t * n, e0, n, whole_scores, s);
    if constexpr (kBias) {
      float b[kPer];
      load_cells<float, kPer>(p.bias, e0, n, whole_scores, b, 0.f);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const float c = s[i] + b[i];
        const bool can = v[i] > -INFINITY && c > -INFINITY;
        key[i] = can ? fixed_code(c) >> kDrop << kIdBits | (kIds - (e0 + i)) : 0u;
        v[i] = can ? c : -INFINITY;  // from here on
      }
    }
  }
  if constexpr (!kBias) {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      key[i] = v[i] > -INFINITY ? (keys::order_bits(v[i]) & ~kIds) | (kIds - (e0 + i)) : 0u;
  }
  constexpr bool kExact = !kBias && sizeof(T) == 2;
  const uint32_t reach = kBias ? (p.sigmoid ? kNearSigmoid : kNearSoftmax) : 0;
  // whether b, which comes after a in the order, may belong before it
  auto near = [&](uint32_t a, uint32_t b) {
    return !kExact && (a >> kIdBits) - (b >> kIdBits) <= reach;
  };
  bool plain = false;  // this token goes the plain way

  if (p.groups > 1) {
    const int group = sub / group_lanes;
    uint32_t value;  // the group's, on its lanes, made unique by its number
    float sum = 0.f, off = 0.f;
    if (!sums) {
      value = key[0];
#pragma unroll
      for (int i = 1; i < kPer; ++i) value = max(value, key[i]);
      for (int o = 1; o < group_lanes; o <<= 1)
        value = max(value, __shfl_xor_sync(~0u, value, o));
    } else {
      // the group's two best s + b, or its two best logits, whose scores make the sum
      float first = -INFINITY, second = -INFINITY;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const float y = kBias ? v[i] : masked(v[i]);
        second = fmaxf(second, fminf(first, y));
        first = fmaxf(first, y);
      }
      for (int o = 1; o < group_lanes; o <<= 1) {
        const float a = __shfl_xor_sync(~0u, first, o), b = __shfl_xor_sync(~0u, second, o);
        second = fmaxf(fminf(first, a), fmaxf(second, b));
        first = fmaxf(first, a);
      }
      const bool one = first > -INFINITY;
      if constexpr (kBias) {
        second = second > -INFINITY ? second : 0.f;
      } else {
        auto score = [&](float y) {
          const float c = p.sigmoid ? sigmoid_fast(y) : (y == m ? 1.f : exp_fast(y - m)) * inv_z;
          return y > -INFINITY ? c : 0.f;
        };
        first = score(first);
        second = score(second);
      }
      sum = first + second;
      off = fminf(fmaf(4.f * kUnit, fabsf(first) + fabsf(second),
                       p.sigmoid ? kOffSigmoid : kOffSoftmax), 3e38f);
      value = one ? (image(sum) & ~31u) | (31 - group) : 0;
    }
    uint32_t left = value, last = 0;
    for (int i = 0; i < p.topk_groups; ++i) {
      const uint32_t big = lanes_max<kLanes>(left);
      left = left == big ? 0 : left;
      last = big;
    }
    if (!sums) {
      const uint32_t fell = lanes_max<kLanes>(left);
      plain = last && fell && near(last, fell);
    } else {
      // the highest that a group that fell may be, and the lowest that one that stands may be
      const uint32_t high = lanes_max<kLanes>(left ? image(sum + off) : 0u);
      const uint32_t low = ~lanes_max<kLanes>(left == value ? 0u : ~image(sum - off));
      plain = high && low <= high;
    }
    if (left) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) key[i] = 0;
    }
  }

  // The k best, one at a time, and the one after them if it could be in doubt. Slot j of lane s
  // of the token holds number j * kLanes + s.
  constexpr int kSlots = 32 / kLanes;
  int id[kSlots];
  uint32_t at[kSlots], previous = 0;
#pragma unroll
  for (int j = 0; j < kSlots; ++j) {
    id[j] = -1;
    at[j] = 0;
  }
  bool doubt = false;
  uint32_t best = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) best = max(best, key[i]);
  const int wanted = kExact ? k : k + 1;
  bool listed = false;
  if constexpr (kLanes == 32) {
    // With a whole warp a token: the wanted-th largest of the lanes' bests bounds the wanted-th
    // key from below, and the few keys that reach it (13 on average for 9 of 256) are ranked
    // against one another, a lane each. Where more than a warp's lanes reach it they are taken
    // out one by one, as for smaller tokens.
    uint32_t left = best, bound = 0;
    for (int r = 0; r < wanted; ++r) {
      bound = __reduce_max_sync(~0u, left);
      left = left == bound ? 0 : left;
    }
    bound = max(bound, 1u);
    int count = 0;
    uint32_t* keys_of = reinterpret_cast<uint32_t*>(ids_of[warp]);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const bool in = key[i] >= bound;
      const unsigned who = __ballot_sync(~0u, in);
      const int place = count + __popc(who & ((1u << lane) - 1));
      if (in && place < 32) keys_of[place] = key[i];
      count += __popc(who);
    }
    listed = count <= 32;
    if (listed) {
      __syncwarp();
      const uint32_t own = lane < count ? keys_of[lane] : 0;
      int rank = 0;
      for (int l = 0; l < count; ++l) rank += keys_of[l] > own;
      __syncwarp();
      if (lane < count) keys_of[rank] = own;
      __syncwarp();
      const uint32_t big = lane < count ? keys_of[lane] : 0;
      const uint32_t after = __shfl_down_sync(~0u, big, 1);
      doubt = __any_sync(~0u, lane < 31 && lane < wanted - 1 && after && near(big, after));
      previous = __shfl_sync(~0u, big, min(wanted - 1, 31));
      if (wanted > 32) previous = 0;
      if (lane < k) {
        id[0] = big ? static_cast<int>(kIds - (big & kIds)) : -1;
        at[0] = big;
      }
      if (!kExact && doubt) {  // what is left, for the candidates below
        const uint32_t last = __shfl_sync(~0u, big, k - 1);
#pragma unroll
        for (int i = 0; i < kPer; ++i) key[i] = key[i] >= last ? 0 : key[i];
      }
    }
    __syncwarp();
  }
  if (!listed) {
#pragma unroll
    for (int j = 0; j < kSlots + 1; ++j) {
      if (j * kLanes >= wanted) break;
      for (int r = j * kLanes; r < min((j + 1) * kLanes, wanted); ++r) {
        const uint32_t big = lanes_max<kLanes>(best);
        doubt = doubt || (r && big && near(previous, big));
        previous = big;
        if (r == k) break;
        if (j < kSlots && sub == r - j * kLanes && big) {
          id[j < kSlots ? j : 0] = static_cast<int>(kIds - (big & kIds));
          at[j < kSlots ? j : 0] = big;
        }
        best = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          key[i] = key[i] == big ? 0 : key[i];
          best = max(best, key[i]);
        }
      }
    }
  }

  if (!kExact && __any_sync(~0u, doubt && live && !plain)) {
    // Neighbours in the order that stand too near: settled if they are equal in logit and bias
    // (lower ids come first); the k-th and what is left have to be clear apart. Else 64 bits
    // decide.
    const int next_id = static_cast<int>(kIds - (previous & kIds));
    bool open = false;
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      const int r = j * kLanes + sub;
      constexpr int kLast = kSlots - 1;
      int i2 = __shfl_down_sync(~0u, id[j], 1, kLanes);
      uint32_t k2 = __shfl_down_sync(~0u, at[j], 1, kLanes);
      const int i3 = __shfl_sync(~0u, id[j < kLast ? j + 1 : j], 0, kLanes);
      const uint32_t k3 = __shfl_sync(~0u, at[j < kLast ? j + 1 : j], 0, kLanes);
      if (sub == kLanes - 1) {
        i2 = j < kLast ? i3 : -1;
        k2 = j < kLast ? k3 : 0;
      }
      if (r == k - 1) {
        i2 = next_id;
        k2 = previous;
      }
      if (r < k && at[j] && k2 && near(at[j], k2)) {
        const bool equal = score_f32(x[id[j]]) == score_f32(x[i2]) &&
                           (!kBias || __ldg(p.bias + id[j]) == __ldg(p.bias + i2));
        open = open || !(r < k - 1 && equal);
      }
    }
    open = __ballot_sync(~0u, open) & mine;
    unsigned todo = __ballot_sync(~0u, open && live && !plain && sub == 0);
    while (todo) {  // one token at a time, by the whole warp
      const int first = __ffs(todo) - 1, slot0 = first / kLanes;
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
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const bool in = here && key[i] && near(cut, key[i]);
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
      if (kBias && !p.sigmoid) {
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
        c = score_f32(xt[e]);
        if constexpr (kBias) {
          const double s = p.sigmoid ? 1.0 / (1.0 + exp(-c)) : (c == md ? 1.0 : exp(c - md)) / z;
          c = s + static_cast<double>(__ldg(p.bias + e));
        }
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

  // weights; slots beyond k hold nothing
  float y[kSlots], top = -INFINITY;
#pragma unroll
  for (int j = 0; j < kSlots; ++j) {
    if (j * kLanes >= k) break;
    y[j] = id[j] >= 0 ? score_f32(x[id[j]]) : -INFINITY;
    top = fmaxf(top, y[j]);
  }
  float w[kSlots], total = 0.f, inv = 1.f;
  if (p.renormalize) {
    top = lanes_max<kLanes>(top);
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      if (j * kLanes >= k) break;
      w[j] = id[j] >= 0 ? relative_score(y[j], top, p.sigmoid) : 0.f;
      total += w[j];
    }
    total = lanes_sum<kLanes>(total);  // 0, or at least a half
    inv = total > 0.f ? rcp_fast(total) : 0.f;
  } else {
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      if (j * kLanes >= k) break;
      w[j] = p.sigmoid ? sigmoid(y[j]) : (y[j] == m ? 1.f : exp_down(y[j] - m)) * inv_z;
      w[j] = id[j] >= 0 ? w[j] : 0.f;
    }
  }
  if (live && !plain) {
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      const int r = j * kLanes + sub;
      if (r >= k) break;
      p.ids[t * k + r] = id[j];
      p.weights[t * k + r] = w[j] * inv * p.scale;
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

  // the chosen: slot j of lane s is number j * kLanes + s; slots beyond k hold nothing
  int id[kSlots];
  float y[kSlots], dw[kSlots], top = -INFINITY;
#pragma unroll
  for (int j = 0; j < kSlots; ++j) {
    id[j] = -1;
    y[j] = -INFINITY;
    dw[j] = 0.f;
    if (j * kLanes >= k) continue;
    const int r = j * kLanes + sub;
    if (r < k) id[j] = p.ids[t * k + r];
    if (id[j] >= n) id[j] = -1;
    if (id[j] >= 0) y[j] = masked(score_f32(x[id[j]]));
    if (!(y[j] > -INFINITY)) id[j] = -1;
    if (id[j] >= 0) dw[j] = p.dweights[t * k + r] * p.scale;
    top = fmaxf(top, y[j]);
  }
  float v[kPer], d[kPer], m = 0.f, inv_z = 0.f;
  if (dense) {
    load_cells<T, kPer, false>(x, e0, n, whole, v, -INFINITY);  // dlogits may be the logits
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
        v[i] = v[i] > -INFINITY ? (v[i] == m ? 1.f : exp_down(v[i] - m)) : 0.f;
        z += v[i];
      }
      z = lanes_sum<kLanes>(z);
      inv_z = z > 0.f ? rcp_fast(z) : 0.f;
#pragma unroll
      for (int i = 0; i < kPer; ++i) v[i] *= inv_z;  // the scores from here on
    }
  }
  // own: the chosen experts' part of the gradient; dot: what every softmax gradient subtracts
  float own[kSlots], dot = 0.f;
#pragma unroll
  for (int j = 0; j < kSlots; ++j) own[j] = 0.f;
  if (p.renormalize) {
    top = lanes_max<kLanes>(top);
    float total = 0.f, mean = 0.f;
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      if (j * kLanes >= k) break;
      own[j] = id[j] >= 0 ? relative_score(y[j], top, p.sigmoid) : 0.f;
      total += own[j];
    }
    total = lanes_sum<kLanes>(total);  // 0, or at least a half
    const float inv = total > 0.f ? rcp_fast(total) : 0.f;
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      own[j] *= inv;
      mean += own[j] * dw[j];
    }
    mean = lanes_sum<kLanes>(mean);
#pragma unroll
    for (int j = 0; j < kSlots; ++j) own[j] *= dw[j] - mean;
  } else {
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      if (j * kLanes >= k) break;
      const float s = p.sigmoid ? sigmoid(y[j])
                                : (y[j] == m ? 1.f : exp_down(y[j] - m)) * inv_z;
      own[j] = id[j] >= 0 ? s * dw[j] : 0.f;
      if (!p.sigmoid) dot += own[j];
    }
  }
  if (p.sigmoid) {
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      if (j * kLanes >= k) break;
      if (id[j] >= 0) own[j] *= sigmoid(-y[j]);  // 1 - s
    }
  } else if (dense) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) dot += v[i] * d[i];
    dot = lanes_sum<kLanes>(dot);
  }
  // The parts at their places. Each lane writes its own where no expert stands twice for a token
  // (which shows when every lane finds its own mark again); else one lane adds them in order.
  float4* cells = reinterpret_cast<float4*>(part + e0);
#pragma unroll
  for (int i = 0; i < kPer / 4; ++i) cells[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  __syncwarp();
  if (id[0] >= 0) part[id[0]] = __int_as_float(lane);
  __syncwarp();
  const bool alone = id[0] < 0 || __float_as_int(part[id[0]]) == lane;
  if (__all_sync(~0u, alone && k <= kLanes)) {
    if (id[0] >= 0) part[id[0]] = own[0];
  } else {
    if (id[0] >= 0) part[id[0]] = 0.f;
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
  if (dense && p.sigmoid) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float ex = exp_down(-fabsf(v[i])), q = rcp_fast(1.f + ex);
      g[i] += v[i] > -INFINITY ? d[i] * ex * q * q : 0.f;
    }
  } else if (dense) {  // 0 where the score is 0, whatever dot is
#pragma unroll
    for (int i = 0; i < kPer; ++i) g[i] += v[i] > 0.f ? v[i] * (d[i] - dot) : 0.f;
  }
  if (live) store_cells<T, kPer>(dx, e0, n, whole_out, g);
}

bool lines_up(const void* p, int64_t stride_bytes, size_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride_bytes % static_cast<int64_t>(bytes) == 0;
}

template <class T, int kLanes, int kPer>
cudaError_t route_fast(const RouteParams& p, int group_lanes, cudaStream_t stream) {
  const bool cells = p.experts % kPer == 0;
  const bool whole = cells && lines_up(p.logits, p.ld * sizeof(T), 16);
  const bool whole_scores =
      cells && lines_up(p.scores, int64_t{p.experts} * sizeof(float), 16) && lines_up(p.bias, 0, 16);
  // the plain way's room, for a token whose groups or whose many experts are in doubt
  const bool doubt = p.bias || sizeof(T) == 4 || (p.groups > 1 && p.group_top2);
  const size_t smem = doubt ? static_cast<size_t>(kWarps) * 2 * p.experts * sizeof(double) : 0;
  auto kernel = p.bias ? route_kernel<T, kLanes, kPer, true> : route_kernel<T, kLanes, kPer, false>;
  static std::atomic<uint64_t> done[2];
  const cudaError_t e = allow_smem(kernel, 64 * 1024, done[p.bias != nullptr]);
  if (e != cudaSuccess) return e;
  constexpr int kTokens = kWarps * 32 / kLanes;
  const LaunchShape shape{static_cast<unsigned>((p.tokens + kTokens - 1) / kTokens), kThreads, smem};
  return launch(kernel, shape, stream, p, group_lanes, whole, whole_scores);
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
  const LaunchShape shape{static_cast<unsigned>((p.tokens + kWarps - 1) / kWarps), kThreads, smem};
  return launch(route_plain_kernel<T>, shape, stream, p);
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
  const LaunchShape shape{static_cast<unsigned>((p.tokens + kTokens - 1) / kTokens), kThreads, smem};
  return launch(route_backward_kernel<T, kLanes, kPer>, shape, stream, p, whole, whole_out,
                whole_scores);
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
