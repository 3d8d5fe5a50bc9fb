// Drawing from rows of scores (see rows.cuh).
//
// Row x, temperature T, m = max x: weights w_j = exp((x_j - m) / T). Top-k, top-p and min-p each
// keep a prefix of the row in top-k order (larger first, equal ones by lower column), so what is
// kept is the shortest of the three and ends at one (score, column), the edge. The draw for a
// uniform u is the first column whose running sum of kept weights, in column order, is above u
// times their total.
//
// Where a running sum crosses u * total, or p * total, must not hang on rounding or on the order
// of an addition: neighbouring sums differ by one weight out of up to 2^31. So a weight is a
// 64-bit integer, w_j * 2^frac rounded once, and every sum is an exact integer sum whatever its
// order. frac = min(50, 62 - ceil(log2 cols)) leaves no sum above 2^63; weights below 2^-frac of
// the row's largest (2^-45 at 131,072 columns) count as zero.
//
// What bounds it: for top-k rows HBM and the latency of a dozen dependent steps, otherwise the
// weights. A weight good to 2^-51 costs twelve 64-bit operations, and the GPU does 64 of those a
// clock and SM: 25.6 million take 17 us, where reading them as fp16 takes 8.
//
// One cluster of blocks takes one row. Each block holds its columns in shared memory, so the row
// is read from HBM once and every later look at it costs shared memory only; what a block cannot
// hold it reads again. Two ways lead from there:
//   - top_k up to kDirectK, greedy rows, and rows of up to kList columns: the k-th largest of the
//     warps' best maxima bounds the k-th score from below and lets little more than k columns
//     pass. Those go to block 0, which orders and draws; the other blocks are done. In large
//     batches one block takes the row, holds nothing, finds the bound in a part of it and lists
//     what reaches it as it streams by. 1000 rows of 100,000 fp32, top-100, 64 draws: 103 us, the
//     400 MB at 3.9 TB/s (a block either loads or orders, four an SM: 592 of the 1000 rows are
//     under way at once); one row of 32,000: 8.8 us.
//   - anything else: the edge of top-p is bracketed by a histogram of the weights over
//     (m - x) / T, the few columns in the bracket are ordered by block 0, the weights above it
//     are summed exactly. The draw walks the columns of the warp whose range of running sums
//     holds it. 256 rows of 100,003 fp16, top-p 0.9, 11,000 columns kept: 162 us, 117 instructions
//     for every 32 columns at 54 % of the issue rate, the rest waits of the cluster.
// Where either meets more columns than its list holds (many equal or nearly equal scores), the
// edge is found by parts of the range of score bits. 64 rows of 131,072 equal scores, top-p:
// 401 us, against 81 for different ones.
#include "rows.cuh"

#include <cooperative_groups.h>

#include <type_traits>
#include <utility>

#include "keys.cuh"
#include "score_load.cuh"

namespace cg = cooperative_groups;

namespace ovvs {
namespace prim {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kList = 1024;     // columns block 0 can order
constexpr int kRankList = 256;  // up to here it counts instead of sorting
constexpr int kDirectK = 448;   // the largest top_k that the list serves
constexpr int kRound = 8;       // chunks a thread has in flight where one block takes the row
constexpr int kWanted = 520;    // columns it means to list
constexpr int kNoted = 16;      // chunks a thread can note there
constexpr int kBins = 2048;     // of the weight histogram
static_assert(kBins * sizeof(float) == kList * sizeof(uint64_t), "wts holds the histogram, pre its totals");

using u64 = unsigned long long;

// Top-k order as an integer: larger is earlier; 0 marks a masked score.
__device__ __forceinline__ uint32_t sort_key(float v) {
  return v > -INFINITY ? keys::order_bits(v) : 0u;
}

// (score, column) in top-k order as one integer: larger is earlier.
__device__ __forceinline__ u64 element(uint32_t key, uint32_t col) {
  return (static_cast<u64>(key) << 32) | static_cast<uint32_t>(~col);
}
__device__ __forceinline__ uint32_t element_col(u64 e) { return ~static_cast<uint32_t>(e); }
__device__ __forceinline__ uint32_t element_key(u64 e) { return static_cast<uint32_t>(e >> 32); }

// 2^(i / 16), i < 16: one entry per pair of shared-memory banks.
__constant__ double kSixteenths[16] = {
    1.0, 1.0442737824274138, 1.0905077326652577, 1.1387886347566916,
    1.189207115002721, 1.241857812073484, 1.2968395546510096, 1.3542555469368927,
    1.4142135623730951, 1.4768261459394993, 1.5422108254079407, 1.6104903319492543,
    1.681792830507429, 1.7562521603732995, 1.8340080864093424, 1.9152065613971474};

// Weights of one row. 2^(t / 16) = 2^(n >> 4) * 2^((n & 15) / 16) * 2^(f / 16) with n = round(t),
// the last factor by the polynomial of degree 6 through its values at the Chebyshev points of
// [-1/2, 1/2], which is 2^-56.8 off at most: twelve 64-bit operations a weight, where the power
// function takes some forty. With the table's rounding and the polynomial's own, p * scaled is off
// by 3 * 2^-53 of itself, under half a step of the finest grid, 2^-50. The result is rounded to an
// integer by adding 2^52.
struct Weigher {
  double m, rate;  // max; 16 log2(e) / T
  float cut;       // scores below it weigh 0
  bool top_inf;    // m is +inf: the columns that hold it weigh 1, the others 0
  int frac;
  const double* table;  // 2^(i / 16 + frac)

  __device__ __forceinline__ void set(float max, float t, int frac_bits, const double* tab) {
    frac = frac_bits;
    table = tab;
    top_inf = max == INFINITY;
    m = top_inf ? 0.0 : max;
    rate = 23.083120654223414 / static_cast<double>(t);
    const double low = m - static_cast<double>(t) * 0.6931471805599453 * (frac + 1);
    cut = fmaxf(__double2float_ru(low), -3.402823466e38f);
  }
  // For x >= cut where m is finite. Without a branch, so that several are under way at once.
  __device__ __forceinline__ u64 plain(float x) const {
    const double magic = 6755399441055744.0;  // 1.5 * 2^52
    const double d = static_cast<double>(x) - m;
    const double r = fma(d, rate, magic);
    const int n = __double2loint(r);
    const double f = fma(d, rate, magic - r);
    const double f2 = f * f;
    double p = fma(f2, 9.181354192172116e-12, fma(f, 1.2716120543851127e-09, 1.4676100321236697e-07));
    p = fma(f2, p, fma(f, 1.3550807776390032e-05, 0.0009383847928089877));
    p = fma(f2, p, fma(f, 0.04332169878499668, 1.0));
    const double s = table[n & 15];
    const double scaled = __hiloint2double(__double2hiint(s) + (n & ~15) * (1 << 16),
                                           __double2loint(s));
    const double w = fma(p, scaled, 4503599627370496.0);
    return static_cast<u64>(__double_as_longlong(w)) & ((u64{1} << 52) - 1);
  }
  __device__ __forceinline__ u64 operator()(float x) const {
    if (top_inf) return x == INFINITY ? u64{1} << frac : 0;
    return x >= cut ? plain(x) : 0;
  }
};

// 16 bytes of scores.
template <class T>
struct Chunk {
  static constexpr int kN = 16 / sizeof(T);
  static constexpr uint32_t kMasked =  // -inf
      sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00u : 0xff80u;
  static __device__ __forceinline__ uint32_t bits(float v) { return __float_as_uint(v); }
  static __device__ __forceinline__ uint32_t bits(__half v) { return __half_as_ushort(v); }
  static __device__ __forceinline__ uint32_t bits(__nv_bfloat16 v) {
    return __bfloat16_as_ushort(v);
  }
  static __device__ __forceinline__ uint4 masked() {
    const uint32_t w = sizeof(T) == 4 ? kMasked : kMasked << 16 | kMasked;
    return make_uint4(w, w, w, w);
  }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[kN]);
  // Largest of the chunk's scores that are not NaN; -inf without one.
  static __device__ __forceinline__ float largest(const uint4& v) {
    float m;
    if constexpr (sizeof(T) == 4) {
      m = fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)),
                fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
    } else {
      const Pair p = __hmax2(__hmax2(pair(v.x), pair(v.y)), __hmax2(pair(v.z), pair(v.w)));
      m = score_f32(__hmax(p.x, p.y));
    }
    return fmaxf(m, -INFINITY);
  }
  // Marks of the scores that reach a bound (kGroup chunks make a word): where bit b of it stands.
  using Pair = typename std::conditional<std::is_same<T, __half>::value, __half2,
                                         __nv_bfloat162>::type;
  using Bound = typename std::conditional<sizeof(T) == 4, float, Pair>::type;
  static constexpr int kGroup = 32 / kN;
  static __device__ __forceinline__ Pair pair(uint32_t w) {
    return *reinterpret_cast<const Pair*>(&w);
  }
  static __device__ __forceinline__ Bound bound(float x);  // the first value that is not below x
  static __device__ __forceinline__ uint32_t mark(const uint4& v, Bound b, int chunk) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4)
        bits |= __uint_as_float(w[i]) >= b ? 1u << (chunk * 4 + i) : 0u;
      else
        bits |= __hge2_mask(pair(w[i]), b) & 0x00010001u << (chunk * 4 + i);
    }
    return bits;
  }
  static __device__ __forceinline__ int chunk_of(int bit) { return (bit & (4 * kGroup - 1)) >> 2; }
  static __device__ __forceinline__ int cell_of(int bit) {
    return sizeof(T) == 4 ? bit & 3 : (bit & 3) * 2 + (bit >> 4);
  }
};
template <>
__device__ __forceinline__ float Chunk<float>::bound(float x) { return x; }
template <>
__device__ __forceinline__ __half2 Chunk<__half>::bound(float x) {
  return __half2half2(__float2half_ru(x));
}
template <>
__device__ __forceinline__ __nv_bfloat162 Chunk<__nv_bfloat16>::bound(float x) {
  return __bfloat162bfloat162(__float2bfloat16_ru(x));
}
template <>
__device__ __forceinline__ void Chunk<float>::unpack(const uint4& v, float (&x)[4]) {
  x[0] = __uint_as_float(v.x);
  x[1] = __uint_as_float(v.y);
  x[2] = __uint_as_float(v.z);
  x[3] = __uint_as_float(v.w);
}
template <>
__device__ __forceinline__ void Chunk<__half>::unpack(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = *reinterpret_cast<const __half2*>(&w[i]);
    x[2 * i] = __low2float(h);
    x[2 * i + 1] = __high2float(h);
  }
}
template <>
__device__ __forceinline__ void Chunk<__nv_bfloat16>::unpack(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

struct Shared {
  u64 list[kList];     // candidates (block 0)
  u64 wts[kList];      // their weights; the histogram before there are any
  u64 pre[kList];      // running sums; before them maxima, the histogram's totals, columns on
                       // their way to block 0
  u64 tot[kMaxCluster * kWarps];  // kept weight of every warp of the cluster
  u64 xch[2][kMaxCluster];        // cluster_sum
  u64 red[kWarps];
  double table[16];
  u64 edge;            // what block 0 found out
  u64 above;
  int state;
  unsigned list_n;
  unsigned staged;
  unsigned pick;
  unsigned bracket[2];
  unsigned first;
  int found;
  int cnt;
};
static_assert(sizeof(int) * kNoted * kThreads == 2 * sizeof(u64) * kList,
              "wts and pre hold the noted chunks");
static_assert(sizeof(uint32_t) * kMaxCluster * kThreads == sizeof(u64) * kList, "maxima fit");

template <class V, class Op>
__device__ __forceinline__ V warp_reduce(V v, Op op) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(~0u, v, o));
  return v;
}

struct Add {
  template <class V>
  __device__ __forceinline__ V operator()(V a, V b) const { return a + b; }
};

__device__ __forceinline__ u64 block_sum(u64 v, u64* red) {
  v = warp_reduce(v, Add());
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) v += red[w];
  return v;
}

// Exclusive running sum over the block's threads; *total gets the sum.
__device__ __forceinline__ u64 block_scan(u64 v, u64* red, u64* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(~0u, s, o);
    if (lane >= o) s += y;
  }
  __syncthreads();
  if (lane == 31) red[warp] = s;
  __syncthreads();
  u64 before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += red[w];
    all += red[w];
  }
  *total = all;
  return before + s - v;
}

// Descending bitonic sort of n (a power of two, at least 2) integers.
__device__ void sort_list(u64* a, int n) {
  for (int size = 2; size <= n; size <<= 1) {
    for (int stride = size >> 1; stride; stride >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < n / 2; i += kThreads) {
        const int lo = 2 * i - (i & (stride - 1)), hi = lo + stride;
        const u64 x = a[lo], y = a[hi];
        if ((x < y) == ((lo & size) == 0)) {
          a[lo] = y;
          a[hi] = x;
        }
      }
    }
  }
  __syncthreads();
}

// One warp: a bound that at least k of n keys reach, and, where the keys allow it, no more than
// slack others; the key of the type's lowest value, which every score reaches, when fewer than k
// are not 0. The keys, at most 32 * kPer, are held in registers, or for kPer = 0 read every time.
template <int kPer>
__device__ uint32_t kth_bound(const uint32_t* key, int n, int k, int slack) {
  const int lane = threadIdx.x & 31;
  uint32_t own[kPer ? kPer : 1];
  if constexpr (kPer != 0) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) own[i] = i * 32 + lane < n ? key[i * 32 + lane] : 0;
  }
  auto each = [&](auto&& f) {
    if constexpr (kPer != 0) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) f(own[i]);
    } else {
      for (int i = lane; i < n; i += 32) f(key[i]);
    }
  };
  uint32_t hi = 0, least = ~0u;
  int valid = 0;
  each([&](uint32_t y) {
    hi = max(hi, y);
    if (y) {
      least = min(least, y);
      ++valid;
    }
  });
  if (static_cast<int>(__reduce_add_sync(~0u, valid)) < k) return sort_key(-3.402823466e38f);
  hi = __reduce_max_sync(~0u, hi);
  uint32_t lo = __reduce_min_sync(~0u, least);
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo + 1) / 2;
    int c = 0;
    each([&](uint32_t y) { c += y >= mid; });
    c = __reduce_add_sync(~0u, c);
    if (c >= k) {
      lo = mid;
      if (c <= k + slack) break;
    } else {
      hi = mid - 1;
    }
  }
  return lo;
}

// The same for the n listed columns, by the whole block; lo is a bound that k of them reach.
__device__ uint32_t list_bound(Shared& sh, int n, int k, uint32_t lo) {
  uint32_t own[kList / kThreads], hi = 0;
#pragma unroll
  for (int i = 0; i < kList / kThreads; ++i) {
    const int at = i * kThreads + threadIdx.x;
    own[i] = at < n ? element_key(sh.list[at]) : 0;
    hi = max(hi, own[i]);
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto all = [&](unsigned v, u64* buf, auto op) {
    if (lane == 0) buf[warp] = v;
    __syncthreads();
    unsigned r = static_cast<unsigned>(buf[0]);
    for (int w = 1; w < kWarps; ++w) r = op(r, static_cast<unsigned>(buf[w]));
    return r;
  };
  hi = all(__reduce_max_sync(~0u, hi), sh.red, [](unsigned a, unsigned b) { return max(a, b); });
  for (int step = 0; lo < hi; ++step) {
    const uint32_t mid = lo + (hi - lo + 1) / 2;
    unsigned c = 0;
#pragma unroll
    for (int i = 0; i < kList / kThreads; ++i) c += own[i] >= mid;
    c = all(__reduce_add_sync(~0u, c), sh.tot + (step & 1) * kWarps, Add());
    if (c >= static_cast<unsigned>(k)) {
      lo = mid;
      if (c <= static_cast<unsigned>(k + (k >> 3))) break;
    } else {
      hi = mid - 1;
    }
  }
  return lo;
}

// Keeps those of the first n listed columns whose key reaches lo; returns how many.
__device__ unsigned keep_listed(Shared& sh, int n, uint32_t lo) {
  u64 own[kList / kThreads];
#pragma unroll
  for (int i = 0; i < kList / kThreads; ++i) {
    const int at = i * kThreads + threadIdx.x;
    own[i] = at < n ? sh.list[at] : 0;
  }
  __syncthreads();
  if (threadIdx.x == 0) sh.list_n = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kList / kThreads; ++i)
    if (element_key(own[i]) >= lo) sh.list[atomicAdd(&sh.list_n, 1u)] = own[i];
  __syncthreads();
  const unsigned kept = sh.list_n;
  __syncthreads();
  return kept;
}

// Scores from here on pass min-p; 0 where it is off.
__device__ __forceinline__ uint32_t min_p_key(float m, float t, float mp) {
  if (!(mp > 0.f)) return 0;
  const double edge = static_cast<double>(m) +
                      static_cast<double>(t) * log(fmin(static_cast<double>(mp), 1.0));
  return sort_key(__double2float_ru(edge));
}

// A row with every score masked.
__device__ void nothing(const SampleParams& p, int64_t row) {
  for (int64_t d = threadIdx.x; d < p.draws; d += kThreads) {
    p.ids[row * p.draws + d] = -1;
    if (p.probs) p.probs[row * p.draws + d] = 0.f;
  }
  if (threadIdx.x == 0 && p.kept) p.kept[row] = 0;
}

__device__ __forceinline__ u64 draw_target(float u, u64 z) {
  u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;
  return static_cast<u64>(static_cast<double>(u) * static_cast<double>(z));
}

// The weight that a top-p prefix has to reach.
__device__ __forceinline__ u64 top_p_target(float tp, u64 z) {
  const double want = ceil(static_cast<double>(fmaxf(tp, 0.f)) * static_cast<double>(z));
  const u64 t = want < 1.0 ? 1 : static_cast<u64>(want);
  return t < z ? t : z;
}

// Settings of one row.
struct Settings {
  float t, tp;
  int k;
  uint32_t mp_key;  // min-p: keys from here on stay (0: off)
};

// Block 0: orders the n listed columns, which hold every column that can be kept, and draws.
__device__ void finish_list(const SampleParams& p, int64_t row, int n, const Settings& o,
                            const Weigher& w, Shared& sh) {
  const int tid = threadIdx.x;
  const bool p_on = o.tp < 1.f;
  u64 z = 0;
  int nd = 0;  // columns with a weight to draw
  int kept = 0;
  if (n <= kRankList) {
    // `share` threads count what stands before a column: its rank, and the weight before it.
    const int share = n <= 32 ? 8 : n <= 64 ? 4 : n <= 128 ? 2 : 1;
    const int i = tid / share, part = tid % share;
    auto joined = [&](auto v) {
      for (int s = 1; s < share; s <<= 1) v += __shfl_xor_sync(~0u, v, s);
      return v;
    };
    const bool here = i < n, one = here && part == 0;
    const u64 e = here ? sh.list[i] : 0;
    const u64 own = here ? w(keys::order_value(element_key(e))) : 0;
    if (one) sh.wts[i] = own;
    __syncthreads();
    int rank = 0;
    u64 before = 0;
    const int loops = (tid & ~31) / share < n ? n : 0;  // not for a warp without a column
#pragma unroll 4
    for (int j = part; j < loops; j += share) {
      const bool less = sh.list[j] > e;
      rank += less;
      before += less ? sh.wts[j] : 0;
    }
    rank = joined(rank);
    before = joined(before);
    const int n1 = o.k > 0 && o.k < n ? o.k : n;
    bool keep = here && rank < n1 && element_key(e) >= o.mp_key;
    if (p_on) {
      const u64 z1 = block_sum(one && rank < n1 ? own : 0, sh.red);
      keep = keep && before < top_p_target(o.tp, z1);
    }
    kept = __syncthreads_count(keep && one);
    nd = __syncthreads_count(keep && one && own);
    z = block_sum(keep && one ? own : 0, sh.red);
    if (one) sh.wts[i] = keep ? own : 0;
    __syncthreads();
    int at = 0;
    before = 0;
#pragma unroll 4
    for (int j = part; j < loops; j += share) {
      const bool earlier = static_cast<uint32_t>(sh.list[j]) > static_cast<uint32_t>(e);
      const u64 wj = sh.wts[j];
      at += earlier && wj;
      before += earlier ? wj : 0;
    }
    at = joined(at);
    before = joined(before);
    __syncthreads();
    if (keep && one && own) {
      sh.list[at] = (e << 32) | static_cast<unsigned>(i);
      sh.pre[at] = before;
    }
    __syncthreads();
  } else {
    const int n2 = n <= 512 ? 512 : kList;
    for (int i = n + tid; i < n2; i += kThreads) sh.list[i] = 0;
    sort_list(sh.list, n2);
    const int per = n2 / kThreads, i0 = tid * per;
    u64 sum = 0;
    const int n1 = o.k > 0 && o.k < n ? o.k : n;
    for (int i = i0; i < i0 + per; ++i) {
      const u64 own = i < n1 ? w(keys::order_value(element_key(sh.list[i]))) : 0;
      sh.wts[i] = own;
      sum += own;
    }
    u64 z1;
    u64 before = block_scan(sum, sh.red, &z1);
    const u64 target = p_on ? top_p_target(o.tp, z1) : ~u64{0};
    u64 part = 0;
    int mine = 0, drawn = 0;
    for (int i = i0; i < i0 + per; ++i) {
      const u64 e = sh.list[i], own = sh.wts[i];
      const bool keep = i < n1 && element_key(e) >= o.mp_key && before < target;
      before += own;
      mine += keep;
      const bool draw = keep && own;
      drawn += draw;
      if (draw) part += own;
      sh.list[i] = draw ? (e << 32) | static_cast<unsigned>(i) : 0;
    }
    kept = static_cast<int>(block_sum(mine, sh.red));
    nd = static_cast<int>(block_sum(drawn, sh.red));
    z = block_sum(part, sh.red);
    sort_list(sh.list, n2);
    sum = 0;
    for (int i = i0; i < i0 + per && i < nd; ++i)
      sum += sh.wts[static_cast<uint32_t>(sh.list[i])];
    u64 all;
    before = block_scan(sum, sh.red, &all);
    for (int i = i0; i < i0 + per && i < nd; ++i) {
      sh.pre[i] = before;
      before += sh.wts[static_cast<uint32_t>(sh.list[i])];
    }
    __syncthreads();
  }
  if (tid == 0 && p.kept) p.kept[row] = kept;
  for (int64_t d = tid; d < p.draws; d += kThreads) {
    const u64 target = draw_target(p.uniforms[row * p.draws + d], z);
    int lo = 0, hi = nd - 1;  // the last column whose running sum does not pass the target
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (sh.pre[mid] <= target)
        lo = mid;
      else
        hi = mid - 1;
    }
    const u64 e = sh.list[lo];
    p.ids[row * p.draws + d] = element_col(e >> 32);
    if (p.probs)
      p.probs[row * p.draws + d] = static_cast<float>(
          static_cast<double>(sh.wts[static_cast<uint32_t>(e)]) / static_cast<double>(z));
  }
}

// kBlocks: blocks an SM can hold by their registers. Where one block takes a row, four of 64
// registers a thread, and kOneBlock of shared memory each. Their loads on the way stand in what
// shared memory leaves of the SM's 256 KB, so that this must be little: 1000 rows of 100,000 fp32,
// top-100, take 103 us with four blocks of 38 KB (92 KB left), 105 with 46, but 131 with 56 (28
// left). A fifth block, for 48 registers, spills and brings nothing: 107 us with 38 KB, 134 with
// 44; rows of that batch under top-p alone 905 us against 835.
// Where a cluster takes a row, the weights want the registers: four of 64 in a large batch (256
// rows of 100,003 fp16, top-p: 157 us, three of 80: 171), three of 80 in one that leaves the SMs
// room (64 rows of 131,072 fp32, mixed: 57 us against 62). How many stand on an SM
// is then often said by the part of the row that they hold: of that last case's blocks, 89 KB each,
// two, so that 37 of its 64 clusters run at once. Three or four that hold less of it and read the
// rest again take longer (67 us against 57).
constexpr int kOneBlock = 38 * 1024;
static_assert(4 * (kOneBlock + 1024) <= 164 * 1024, "four blocks, and 92 KB beside them");
static_assert(kOneBlock >= sizeof(Shared) + 4096, "and room to hold some chunks");
template <class T, int kBlocks>
__global__ void __launch_bounds__(kThreads, kBlocks)
sample_kernel(SampleParams p, int frac, int block_chunks, int resident) {
  using C = Chunk<T>;
  extern __shared__ __align__(16) unsigned char smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  uint4* held = reinterpret_cast<uint4*>(smem + (sizeof(Shared) + 15) / 16 * 16);
  cg::cluster_group cluster = cg::this_cluster();
  const int nb = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  const int64_t row = blockIdx.x / nb;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cols = static_cast<int>(p.cols);

  // The row as 16-byte chunks on the boundaries of memory: chunk g holds columns g * kN - head
  // and on. Each block, and in it each warp, takes a contiguous range of chunks.
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  const int head = static_cast<int>((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % C::kN);
  const uint4* base = reinterpret_cast<const uint4*>(x - head);
  const int chunks = static_cast<int>((int64_t{cols} + head + C::kN - 1) / C::kN);
  const int64_t b0 = int64_t{rank} * block_chunks;
  const int local = static_cast<int>(
      b0 < chunks ? (chunks - b0 < block_chunks ? chunks - b0 : block_chunks) : 0);
  const int warp_chunks = (block_chunks + kWarps - 1) / kWarps;
  const int c0 = warp * warp_chunks;
  const int c1 = c0 + warp_chunks < local ? c0 + warp_chunks : local;
  // chunks of this block that lie in the row whole
  const int whole0 = rank == 0 && head ? 1 : 0;
  const bool cut_end = b0 + local == chunks && (static_cast<unsigned>(cols) + head) % C::kN;
  const int whole = local - whole0 - (cut_end ? 1 : 0);
  const uint4* here = base + b0;
  auto cut = [&](int c) {  // a chunk at either end of the row: what lies outside is masked
    const int64_t col = (b0 + c) * C::kN - head;
    uint32_t bits[4] = {};
#pragma unroll
    for (int e = 0; e < C::kN; ++e) {
      const bool in = col + e >= 0 && col + e < cols;
      const uint32_t y = in ? C::bits(x[col + e]) : C::kMasked;
      bits[e * 4 / C::kN] |= y << (e * sizeof(T) * 8 % 32);
    }
    return make_uint4(bits[0], bits[1], bits[2], bits[3]);
  };
  auto fetch = [&](int c) {  // from global memory
    if (c - whole0 >= 0 && c - whole0 < whole) return __ldg(here + c);
    return cut(c);
  };
  // kRound chunks at once, `step` apart; those from `end` on are masked
  auto fetch_round = [&](uint4 (&v)[kRound], int c, int step, int end) {
    const int last = c + (kRound - 1) * step;
    if (__all_sync(~0u, c >= whole0 && last < whole0 + whole && last < end)) {
#pragma unroll
      for (int i = 0; i < kRound; ++i) v[i] = __ldg(here + c + i * step);
    } else {
#pragma unroll
      for (int i = 0; i < kRound; ++i)
        v[i] = c + i * step < end ? fetch(c + i * step) : C::masked();
    }
  };
  auto chunk_at = [&](int c) { return c < resident ? held[c] : fetch(c); };
  auto first_col = [&](int c) { return static_cast<int>((b0 + c) * C::kN - head); };

  const float t = p.temperature ? p.temperature[row] : 1.f;
  Settings o;
  o.t = t;
  o.tp = p.top_p ? p.top_p[row] : 1.f;
  o.k = p.top_k ? p.top_k[row] : 0;
  const float mp = p.min_p ? p.min_p[row] : 0.f;
  const bool greedy = !(t > 0.f);

  if (tid < 16) sh.table[tid] = ldexp(kSixteenths[tid], frac);
  if (tid == 0) {
    sh.list_n = 0;
    sh.staged = 0;
    sh.first = ~0u;
  }
  auto started = cluster.barrier_arrive();
  const bool small = cols <= kList;  // the list holds the row (and one block takes it)
  const bool direct = !greedy && (small || (o.k > 0 && o.k <= kDirectK));
  if (direct && nb == 1) {
    // One block for the row, nothing held. A look at every `skip`-th round of chunks, and the
    // last, gives a bound: the k-th of all threads' two best chunks. Then every column that
    // reaches it is listed, some k * skip of them; the rounds seen before come from L2.
    __syncthreads();
    uint32_t* maxima = reinterpret_cast<uint32_t*>(sh.pre);
    const int skip = small ? 1 : min(8, max(1, kWanted / o.k));
    const int rounds = (local + kRound * kThreads - 1) / (kRound * kThreads);
    uint4 v[kRound];
    auto load_round = [&](int r) {
      fetch_round(v, r * kRound * kThreads + tid, kThreads, local);
    };
    if (small) {
      if (tid == 0) sh.pick = sort_key(-3.402823466e38f);
    } else {
      float big = -INFINITY, second = -INFINITY;
      for (int r = 0; r < rounds; r = r + 1 < rounds ? min(r + skip, rounds - 1) : rounds) {
        load_round(r);
#pragma unroll
        for (int i = 0; i < kRound; ++i) {
          const float y = C::largest(v[i]);
          second = fmaxf(second, fminf(big, y));
          big = fmaxf(big, y);
        }
      }
      maxima[tid] = sort_key(big);
      maxima[kThreads + tid] = sort_key(second);
      __syncthreads();
      if (warp == 0) {
        const uint32_t found = kth_bound<2 * kThreads / 32>(maxima, 2 * kThreads, o.k, o.k >> 5);
        if (lane == 0) sh.pick = found;
      }
    }
    __syncthreads();
    const float bound = keys::order_value(sh.pick);
    // Each thread notes its chunks that reach the bound (some kWanted of all threads' together)
    // and lists their columns afterwards: the pass itself has no atomic and no vote.
    int* noted = reinterpret_cast<int*>(sh.wts) + tid;
    int count = 0;
    for (int r = 0; r < rounds; ++r) {
      load_round(r);
#pragma unroll
      for (int i = 0; i < kRound; ++i) {
        if (C::largest(v[i]) >= bound) {
          if (count < kNoted) noted[count * kThreads] = (r * kRound + i) * kThreads + tid;
          ++count;
        }
      }
    }
    const bool fits = !__syncthreads_or(count > kNoted);
    for (int i = 0; i < count && fits; ++i) {
      const int c = noted[i * kThreads];
      float y[C::kN];
      C::unpack(fetch(c), y);
#pragma unroll
      for (int e = 0; e < C::kN; ++e) {
        if (!(y[e] >= bound)) continue;
        const unsigned at = atomicAdd(&sh.list_n, 1u);
        if (at < kList)
          sh.list[at] = element(sort_key(y[e]), static_cast<uint32_t>(first_col(c) + e));
      }
    }
    __syncthreads();
    unsigned listed = sh.list_n;
    if (fits && listed <= kList) {
      if (o.k > 0 && o.k < kList && listed > static_cast<unsigned>(o.k + o.k / 4)) {
        const uint32_t lo = list_bound(sh, static_cast<int>(listed), o.k, sh.pick);
        listed = keep_listed(sh, static_cast<int>(listed), lo);
      }
      uint32_t best = 0;
      for (unsigned i = lane; i < listed; i += 32) best = max(best, element_key(sh.list[i]));
      best = __reduce_max_sync(~0u, best);
      if (best) {
        Weigher w;
        w.set(keys::order_value(best), t, frac, sh.table);
        o.mp_key = min_p_key(keys::order_value(best), t, mp);
        finish_list(p, row, static_cast<int>(listed), o, w, sh);
      } else {
        nothing(p, row);
      }
      return;
    }
    __syncthreads();
    if (tid == 0) sh.list_n = 0;
  }
  float own = -INFINITY;
  for (int c = c0; c < c1; c += 32 * kRound) {
    uint4 v[kRound];
    fetch_round(v, c + lane, 32, c1);
#pragma unroll
    for (int i = 0; i < kRound; ++i) {
      const int at = c + i * 32 + lane;
      if (at < c1 && at < resident) held[at] = v[i];
      own = fmaxf(own, C::largest(v[i]));
    }
  }

  // The `heads` largest of each warp's threads' maxima, on every block.
  uint32_t* maxima = reinterpret_cast<uint32_t*>(sh.pre);
  const uint32_t own_key = sort_key(own);
  const int heads = greedy || o.k <= 0 ? 1 : min(32, 1 + 2 * min(o.k, 2048) / (nb * kWarps));
  cluster.barrier_wait(std::move(started));  // every block runs: its shared memory may be written
  {
    uint32_t left = own_key;
    for (int i = 0; i < heads; ++i) {
      const uint32_t big = __reduce_max_sync(~0u, left);
      if (lane < nb)
        cluster.map_shared_rank(maxima, lane)[(rank * kWarps + warp) * heads + i] = big;
      const unsigned at = __ballot_sync(~0u, left == big);
      if (lane == __ffs(at) - 1) left = 0;
    }
  }
  cluster.sync();
  const int num_maxima = nb * kWarps * heads;
  uint32_t best = 0;  // a warp's first is its largest
  for (int i = lane; i < nb * kWarps; i += 32) best = max(best, maxima[i * heads]);
  best = __reduce_max_sync(~0u, best);
  if (best == 0) {  // every score is masked
    if (rank == 0) nothing(p, row);
    return;
  }
  const float m = keys::order_value(best);
  Shared* zero = cluster.map_shared_rank(&sh, 0);
  // Columns for block 0's list wait in this block's `pre` and go over together.
  auto stage = [&](float y, int col) {
    const unsigned at = atomicAdd(&sh.staged, 1u);
    if (at < kList) sh.pre[at] = element(sort_key(y), static_cast<uint32_t>(col));
  };
  auto hand_over = [&] {
    __syncthreads();
    const unsigned n = sh.staged;
    if (tid == 0 && n) sh.pick = atomicAdd(&zero->list_n, n);
    __syncthreads();
    for (unsigned i = tid; i < n && i < kList; i += kThreads)
      if (sh.pick + i < kList) zero->list[sh.pick + i] = sh.pre[i];
  };

  if (greedy) {  // the first column that holds the largest score
    unsigned first = ~0u;
    if (own_key == best) {
      for (int c = c0 + lane; c < c1 && first == ~0u; c += 32) {
        float v[C::kN];
        C::unpack(chunk_at(c), v);
#pragma unroll
        for (int e = C::kN - 1; e >= 0; --e)
          if (v[e] == m) first = static_cast<unsigned>(first_col(c) + e);
      }
      atomicMin(&zero->first, first);
    }
    cluster.sync();
    if (rank == 0) {
      for (int64_t d = tid; d < p.draws; d += kThreads) {
        p.ids[row * p.draws + d] = sh.first;
        if (p.probs) p.probs[row * p.draws + d] = 1.f;
      }
      if (tid == 0 && p.kept) p.kept[row] = 1;
    }
    return;
  }

  Weigher w;
  w.set(m, t, frac, sh.table);
  o.mp_key = min_p_key(m, t, mp);

  float bound = -3.402823466e38f;
  if (o.k > 0) {
    // A bound that at least k maxima reach, found by halving; every maximum is a score, so at
    // least k scores reach it too.
    if (warp == 0) {
      const uint32_t found = num_maxima <= 128 ? kth_bound<4>(maxima, num_maxima, o.k, o.k >> 3)
                                               : kth_bound<0>(maxima, num_maxima, o.k, o.k >> 4);
      if (lane == 0) sh.pick = found;
    }
    __syncthreads();
    bound = keys::order_value(sh.pick);
  }
  if (direct) {
    for (int c = c0 + lane; c < c1; c += 32) {
      const uint4 v = chunk_at(c);
      if (!(C::largest(v) >= bound)) continue;
      float y[C::kN];
      C::unpack(v, y);
#pragma unroll
      for (int e = 0; e < C::kN; ++e) {
        if (y[e] >= bound) stage(y[e], first_col(c) + e);
      }
    }
    hand_over();
    cluster.sync();
    const unsigned n = zero->list_n;
    if (n <= kList) {
      // block 0 stays until the others have read its count
      auto read = cluster.barrier_arrive();
      if (rank != 0) return;
      finish_list(p, row, static_cast<int>(n), o, w, sh);
      cluster.barrier_wait(std::move(read));
      return;
    }
  }

  // ---- the general way ----
  // Value of each column of this warp's range, in column order per lane.
  auto each = [&](auto&& f) {
    for (int c = c0 + lane; c < c1; c += 32) {
      float y[C::kN];
      C::unpack(chunk_at(c), y);
      const int col = first_col(c);
#pragma unroll
      for (int e = 0; e < C::kN; ++e) f(y[e], col + e);
    }
  };
  // Sum and number of the weights from `high` on, and rare(score, column) for the scores below it
  // from `low` on. Each lane marks them among 32 of its scores first and then takes its marked
  // ones, two at a time, so that a warp does not weigh every score for the few that need it.
  const bool all_held = block_chunks <= resident;
  auto sum_from = [&](float low, float high, u64* sum, int* number, auto&& rare) {
    const auto bound = C::bound(fmaxf(low, -3.402823466e38f));  // -inf: there is no column
    high = fmaxf(high, w.cut);
    for (int c = c0 + lane; c < c1; c += 32 * C::kGroup) {
      uint32_t marked = 0;
#pragma unroll
      for (int i = 0; i < C::kGroup; ++i)
        marked |= C::mark(c + i * 32 < c1 ? chunk_at(c + i * 32) : C::masked(), bound, i);
      auto score_at = [&](int bit) {
        const int at = c + C::chunk_of(bit) * 32, e = C::cell_of(bit);
        if (all_held || at < resident) return score_f32(reinterpret_cast<const T*>(held + at)[e]);
        return score_f32(x[first_col(at) + e]);
      };
      while (marked) {
        const int b0 = __ffs(marked) - 1;
        marked &= marked - 1;
        const int b1 = marked ? __ffs(marked) - 1 : -1;
        marked &= marked - 1;
        const float y0 = score_at(b0), y1 = b1 >= 0 ? score_at(b1) : -INFINITY;
        const u64 v0 = w.plain(y0), v1 = w.plain(y1);
        const bool in0 = y0 >= high, in1 = y1 >= high;
        *sum += (in0 ? v0 : 0) + (in1 ? v1 : 0);
        *number += in0 + in1;
        if (!in0) rare(y0, first_col(c + C::chunk_of(b0) * 32) + C::cell_of(b0));
        if (!in1 && b1 >= 0) rare(y1, first_col(c + C::chunk_of(b1) * 32) + C::cell_of(b1));
      }
    }
  };
  int turn = 0;
  auto cluster_sum = [&](u64 v) {
    v = block_sum(v, sh.red);
    turn ^= 1;
    if (tid < nb) cluster.map_shared_rank(&sh, tid)->xch[turn][rank] = v;
    cluster.sync();
    u64 s = 0;
    for (int b = 0; b < nb; ++b) s += sh.xch[turn][b];
    return s;
  };
  // Sum over the lanes of every warp, on every block.
  auto share_totals = [&](u64 s) {
    s = warp_reduce(s, Add());
    cluster.sync();
    if (lane < nb) cluster.map_shared_rank(&sh, lane)->tot[rank * kWarps + warp] = s;
    cluster.sync();
  };
  // then(column, value, i) for the column of this warp's range at which before + the running sum
  // of value passes lane i's target, for every lane i of todo.
  auto walk = [&](u64 before, u64 target, unsigned todo, auto&& value, auto&& then) {
    for (int c = c0; c < c1 && todo; c += 32) {
      float y[C::kN];
      u64 v[C::kN], sum = 0;
      C::unpack(c + lane < c1 ? chunk_at(c + lane) : C::masked(), y);
      const int col = first_col(c + lane);
#pragma unroll
      for (int e = 0; e < C::kN; ++e) {
        v[e] = value(y[e], col + e);
        sum += v[e];
      }
      u64 s = sum;
#pragma unroll
      for (int i = 1; i < 32; i <<= 1) {
        const u64 z = __shfl_up_sync(~0u, s, i);
        if (lane >= i) s += z;
      }
      s += before;
      before = __shfl_sync(~0u, s, 31);
      unsigned here = __ballot_sync(~0u, target < before) & todo;
      todo &= ~here;
      while (here) {
        const int i = __ffs(here) - 1;
        here &= here - 1;
        const u64 t = __shfl_sync(~0u, target, i);
        const unsigned passed = __ballot_sync(~0u, s > t);
        if (lane == __ffs(passed) - 1) {
          u64 run = s - sum;
          bool done = false;
#pragma unroll
          for (int e = 0; e < C::kN; ++e) {
            run += v[e];
            if (!done && run > t) {
              then(col + e, v[e], i);
              done = true;
            }
          }
        }
      }
    }
  };
  auto before_warp = [&](u64* z) {
    static_assert(kMaxCluster * kWarps == 64, "two totals a lane");
    const int me = rank * kWarps + warp, all = nb * kWarps;
    const u64 a = lane < all ? sh.tot[lane] : 0, b = 32 + lane < all ? sh.tot[32 + lane] : 0;
    *z = warp_reduce(a + b, Add());
    return warp_reduce((lane < me ? a : 0) + (32 + lane < me ? b : 0), Add());
  };
  // Edge of the shortest prefix, among the columns up to `in`, whose sum of value(x) reaches
  // target, where the scores whose key is above `khi` sum to `above` and it ends among those from
  // `klo` to there (0 if it does not): the range of keys in 256 parts, then the part where it
  // ends, until that is one score; then the column among those that hold it.
  auto reach = [&](u64 in, u64 target, u64 above, uint32_t klo, uint32_t khi, auto&& value) -> u64 {
    u64* hist = sh.wts;
    for (bool one = false; !one;) {
      const uint32_t span = khi - klo;
      const int shift = span < 256 ? 0 : 24 - __clz(span);
      one = shift == 0;
      cluster.sync();
      hist[tid] = 0;
      __syncthreads();
      const float low = keys::order_value(klo), high = keys::order_value(khi);
      uint32_t at = 0;  // equal parts in a row are added up before they go to the histogram
      u64 sum = 0;
      each([&](float y, int col) {
        if (!(y >= low) || !(y <= high)) return;
        const uint32_t k = sort_key(y);
        if (k < klo || k > khi || element(k, col) < in) return;
        const uint32_t bin = (k - klo) >> shift;
        if (bin != at && sum) {
          atomicAdd(&hist[at], sum);
          sum = 0;
        }
        at = bin;
        sum += value(y);
      });
      if (sum) atomicAdd(&hist[at], sum);
      cluster.sync();
      u64 bin = 0, all;
      for (int b = 0; b < nb; ++b) bin += cluster.map_shared_rank(hist, b)[255 - tid];
      const u64 before = above + block_scan(bin, sh.red, &all);
      if (above >= target || above + all < target) return 0;
      if (before < target && before + bin >= target) {
        sh.pick = 255 - tid;
        sh.above = before;
      }
      __syncthreads();
      klo += sh.pick << shift;
      const uint32_t rest = (1u << shift) - 1;
      khi = khi - klo > rest ? klo + rest : khi;
      above = sh.above;
    }
    const u64 v = value(keys::order_value(klo));
    const u64 ties = (target - above + v - 1) / v;
    auto tie = [&](float y, int col) {
      const uint32_t k = sort_key(y);
      return u64{k == klo && element(k, col) >= in};
    };
    u64 own_ties = 0, all;
    each([&](float y, int col) { own_ties += tie(y, col); });
    share_totals(own_ties);
    const u64 before = before_warp(&all);
    if (ties - 1 >= before && ties - 1 < before + sh.tot[rank * kWarps + warp])
      walk(before, ties - 1, 1, tie, [&](int col, u64, int) {
        for (int b = 0; b < nb; ++b) cluster.map_shared_rank(&sh, b)->found = col;
      });
    cluster.sync();
    return element(klo, static_cast<uint32_t>(sh.found));
  };

  constexpr float kLowest = -3.402823466e38f;
  const uint32_t lowest_key = sort_key(kLowest);
  const u64 everything = element(1, ~0u);  // every column that is not masked
  u64 edge = everything;
  if (o.k > 0) {
    u64 n = 0;
    each([&](float y, int) { n += y > -INFINITY; });
    n = cluster_sum(n);
    if (static_cast<u64>(o.k) < n)
      edge = reach(edge, static_cast<u64>(o.k), 0, sort_key(bound), best,
                   [](float) { return u64{1}; });
  }
  bool summed = false;  // tot holds the kept weights
  if (o.tp < 1.f) {
    const bool limited = edge != everything;
    const u64 in = edge;
    // Bins of (m - x) / T. The edge's weight is at least (1 - p) / cols of the largest, so they
    // reach that far and no further: 100 to 200 a unit. A bin sums weights relative to its upper
    // end, in 1 / unit, from a second-order series: good to half a unit and 1e-6. The unit is a
    // whole number, so that the rounded parts of a block's columns stay below 2^32 together.
    const float reach_units = logf(static_cast<float>(cols) / (1.f - fmaxf(o.tp, 0.f))) + 0.1f;
    const float bins_per_unit = kBins / reach_units;
    const float per_unit = bins_per_unit / t;
    const bool binned = !w.top_inf && per_unit > 0.f && per_unit < INFINITY;
    const float unit =
        floorf(fminf(65536.f, 4294966016.f / (static_cast<float>(block_chunks) * C::kN)));
    unsigned* hist = reinterpret_cast<unsigned*>(sh.wts);
    float* hist_total = reinterpret_cast<float*>(sh.pre);
    for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
    __syncthreads();
    const float bins_f = binned ? static_cast<float>(kBins) : 0.f;
    const float unit_per_bin = 1.f / bins_per_unit;
    float low = kLowest, high = kLowest;
    u64 z = 0;
    // unit * exp(-g * unit_per_bin) to the second order
    const float slope = -unit * unit_per_bin, bend = 0.5f * unit * unit_per_bin * unit_per_bin;
    auto weigh = [&](float y, bool in) {
      const u64 own = w.plain(y);
      // the nearest bin below, and how far into it, without a conversion
      const float v = (m - y) * per_unit, vb = __fadd_rz(v, 8388608.f);
      const float g = v - (vb - 8388608.f);
      const float q = fmaf(g, fmaf(g, bend, slope), unit + 8388608.f);
      z += in && y >= w.cut ? own : 0;
      if (v < bins_f && in)
        atomicAdd(&hist[__float_as_uint(vb) & 0x7fffffu], __float_as_uint(q) - 0x4b000000u);
    };
    if (w.top_inf)
      each([&](float y, int col) { z += element(sort_key(y), col) >= in ? w(y) : 0; });
    else if (limited)
      each([&](float y, int col) { weigh(y, element(sort_key(y), col) >= in); });
    else
      each([&](float y, int) { weigh(y, true); });
    z = cluster_sum(z);
    const u64 target = top_p_target(o.tp, z);
    if (binned) {
      const int share = kBins / nb;
      for (int i = rank * share + tid; i < (rank + 1) * share; i += kThreads) {
        unsigned part[kMaxCluster];
#pragma unroll
        for (int b = 0; b < kMaxCluster; ++b)
          part[b] = b < nb ? cluster.map_shared_rank(hist, b)[i] : 0;
        float sum = 0.f;
#pragma unroll
        for (int b = 0; b < kMaxCluster; ++b) sum += static_cast<float>(part[b]);
        sum *= expf(-static_cast<float>(i) * unit_per_bin) / unit;
#pragma unroll
        for (int b = 0; b < kMaxCluster; ++b)
          if (b < nb) cluster.map_shared_rank(hist_total, b)[i] = sum;
      }
      if (rank == 0 && tid == 0) {
        sh.list_n = 0;
        sh.cnt = 0;
      }
      if (tid == 0) {
        sh.staged = 0;
        sh.bracket[0] = sh.bracket[1] = kBins - 1;
      }
      cluster.sync();
      // the bins where the running sum surely has not, and surely has, reached the target
      constexpr int kPer = kBins / kThreads;
      constexpr double kFix = 4294967296.0;
      u64 part = 0, all;
      for (int i = 0; i < kPer; ++i)
        part += static_cast<u64>(hist_total[tid * kPer + i] * kFix);
      u64 run = block_scan(part, sh.red, &all);
      const double scale = exp2(static_cast<double>(-frac)) * kFix;
      const double goal = static_cast<double>(target) * scale;
      const double margin = (0.6 / unit + 2e-6) * static_cast<double>(z) * scale;
      for (int i = 0; i < kPer; ++i) {
        const double lo = static_cast<double>(run);
        run += static_cast<u64>(hist_total[tid * kPer + i] * kFix);
        const double hi = static_cast<double>(run);
        if (lo < goal - margin && hi >= goal - margin) sh.bracket[0] = tid * kPer + i;
        if (lo < goal + margin && hi >= goal + margin) sh.bracket[1] = tid * kPer + i;
      }
      if (tid == 0 && !(goal - margin > 0.0)) sh.bracket[0] = 0;
      __syncthreads();
      const int first = static_cast<int>(sh.bracket[0]), last = static_cast<int>(sh.bracket[1]);
      // the bracket in scores, a little wider than the bins
      const float slack = 4e-7f * (fabsf(m) + static_cast<float>(last + 1) / per_unit);
      high = m - static_cast<float>(first) / per_unit + slack;
      low = fmaxf(kLowest, m - static_cast<float>(last + 1) / per_unit - slack);
      u64 sum = 0;
      int over = 0;
      if (limited) {
        each([&](float y, int col) {
          if (!(y >= low) || element(sort_key(y), col) < in) return;
          if (y >= high) {
            sum += w(y);
            ++over;
          } else {
            stage(y, col);
          }
        });
      } else {
        sum_from(low, high, &sum, &over, stage);
      }
      hand_over();
      sum = warp_reduce(sum, Add());
      over = __reduce_add_sync(~0u, over);
      if (lane == 0) {
        zero->tot[rank * kWarps + warp] = sum;
        atomicAdd(&zero->cnt, over);
      }
      cluster.sync();
      if (rank == 0) {
        const int n = static_cast<int>(sh.list_n);
        u64 above;
        before_warp(&above);
        if (tid == 0) {
          sh.state = 0;
          sh.edge = above;  // for the way by digits
        }
        __syncthreads();
        if (n > 0 && n <= kList && above < target) {
          for (int i = tid; i < n; i += kThreads)
            sh.wts[i] = w(keys::order_value(element_key(sh.list[i])));
          __syncthreads();
          const int share = n <= 32 ? 8 : n <= 64 ? 4 : n <= 128 ? 2 : 1;
          int kept = 0;
          for (int i0 = 0; i0 < n; i0 += kThreads / share) {
            const int i = i0 + tid / share;
            const u64 e = i < n ? sh.list[i] : ~u64{0};
            u64 run = 0;
#pragma unroll 4
            for (int j = tid % share; j < n; j += share) run += sh.list[j] > e ? sh.wts[j] : 0;
            for (int s = 1; s < share; s <<= 1) run += __shfl_xor_sync(~0u, run, s);
            run += above;
            if (i >= n || tid % share || run >= target) continue;
            const u64 own = sh.wts[i];
            ++kept;
            const int g = static_cast<int>((element_col(e) + static_cast<unsigned>(head)) / C::kN);
            atomicAdd(&sh.tot[g / block_chunks * kWarps + g % block_chunks / warp_chunks], own);
            if (run + own >= target) {
              sh.edge = e;
              sh.state = o.mp_key > element_key(e) ? 1 : 2;
            }
          }
          atomicAdd(&sh.cnt, kept);
        }
        __syncthreads();
        for (int b = 1; b < nb; ++b) {
          Shared* peer = cluster.map_shared_rank(&sh, b);
          if (tid < nb * kWarps) peer->tot[tid] = sh.tot[tid];
          if (tid == 0) {
            peer->edge = sh.edge;
            peer->state = sh.state;
          }
        }
      }
      cluster.sync();
      summed = sh.state == 2;
      // more columns in the bracket than the list holds: they alone are gone through by digits
      edge = sh.state ? sh.edge
                      : reach(in, target, sh.edge, sort_key(low),
                              max(sort_key(low), sort_key(high) - 1), w);
    }
    if (!binned || !edge) edge = reach(in, target, 0, lowest_key, best, w);
  }
  if (o.mp_key > element_key(edge)) edge = element(o.mp_key, ~0u);
  auto kept_weight = [&](float y, int col) {
    return element(sort_key(y), col) >= edge ? w(y) : u64{0};
  };
  if (!summed) {
    u64 sum = 0;
    int n = 0;
    if (edge == everything) {
      each([&](float y, int) {
        sum += w(y);
        n += y > -INFINITY;
      });
    } else {
      const float last = keys::order_value(element_key(edge));
      auto take = [&](float y, int col) {
        if (y == last && static_cast<uint32_t>(col) > element_col(edge)) return;
        sum += w(y);
        ++n;
      };
      if (w.top_inf) {
        each([&](float y, int col) {
          if (y >= last) take(y, col);
        });
      } else {
        sum_from(last, keys::order_value(element_key(edge) + 1), &sum, &n, take);
      }
    }
    share_totals(sum);
    if (p.kept) {
      const u64 all = cluster_sum(static_cast<u64>(n));
      if (rank == 0 && tid == 0) p.kept[row] = static_cast<int>(all);
    }
  } else if (rank == 0 && tid == 0 && p.kept) {
    p.kept[row] = sh.cnt;
  }
  u64 z;
  const u64 before = before_warp(&z), mine = sh.tot[rank * kWarps + warp];
  for (int64_t d0 = 0; d0 < p.draws; d0 += 32) {
    const int64_t d = d0 + lane;
    const u64 target = d < p.draws ? draw_target(p.uniforms[row * p.draws + d], z) : 0;
    const unsigned todo =
        __ballot_sync(~0u, d < p.draws && target >= before && target - before < mine);
    walk(before, target, todo, kept_weight, [&](int col, u64 v, int i) {
      p.ids[row * p.draws + d0 + i] = col;
      if (p.probs)
        p.probs[row * p.draws + d0 + i] =
            static_cast<float>(static_cast<double>(v) / static_cast<double>(z));
    });
  }
}

int frac_bits(int64_t cols) {
  int log2 = 0;
  while ((int64_t{1} << log2) < cols) ++log2;
  return log2 < 12 ? 50 : 62 - log2;
}

template <class T>
cudaError_t sample(const SampleParams& p, cudaStream_t stream) {
  constexpr int kN = Chunk<T>::kN;
  constexpr size_t kFixed = (sizeof(Shared) + 15) / 16 * 16;
  const int64_t chunks = (p.cols + 2 * kN - 2) / kN;  // whatever the row's alignment
  // A batch of two rows an SM or more that may have top-k rows goes one block a row, which reads a
  // top-k row in one pass (512 rows of 100,003 fp16, top-50: 28 us against 85 by clusters of 8;
  // rows under top-p alone, which it reads again from L2, take 312 against 302, and a top-k above
  // kDirectK takes four times as long as by clusters: 1000 rows of 100,000 fp32, top-1000, 3.9 ms).
  // Otherwise a row gets a cluster: up to three blocks an SM over all rows, of 512 chunks or more
  // (16 rows of 32,000 bf16, top-p: 25 us by 8 blocks, 41 by 2), and beyond that as few as keep a
  // block's part at 2048 chunks (400 such rows: 140 us by 8 blocks, 97 by 4, 92 by 2, 117 by 1).
  const bool one_pass = p.top_k && p.rows >= 296;
  int nb = 1;
  while (nb < kMaxCluster && !one_pass && chunks / nb > 512 &&
         (p.rows * nb * 2 <= 444 || chunks / nb > 2048))
    nb *= 2;
  const int block_chunks = static_cast<int>((chunks + nb - 1) / nb);
  const int most = static_cast<int>(((one_pass ? kOneBlock : 227 * 1024) - kFixed) / 16);
  const int resident = block_chunks < most ? block_chunks : most;
  const bool many = one_pass || p.rows * nb > 592;
  auto kernel = many ? sample_kernel<T, 4> : sample_kernel<T, 3>;
  static std::atomic<uint64_t> done[2];
  const cudaError_t e = allow_smem(kernel, 227 * 1024, done[many]);
  if (e != cudaSuccess) return e;
  const LaunchShape shape{static_cast<unsigned>(p.rows * nb), kThreads,
                          kFixed + static_cast<size_t>(resident) * 16, static_cast<unsigned>(nb)};
  return launch(kernel, shape, stream, p, frac_bits(p.cols), block_chunks, resident);
}

}  // namespace

cudaError_t launch_sample_rows(const SampleParams& p, int type, cudaStream_t stream) {
  if (type == kScoreF32) return sample<float>(p, stream);
  if (type == kScoreF16) return sample<__half>(p, stream);
  return sample<__nv_bfloat16>(p, stream);
}

}  // namespace prim
}  // namespace ovvs
