// Drawing from rows of scores (see rows.cuh).
//
// Row x, temperature T, m = max x: weights w_j = exp((x_j - m) / T). Top-k, top-p and min-p each
// keep a prefix of the row in top-k order (larger first, equal ones by lower column), so what is
// kept is the shortest of the three and one (key, ties kept at that key) pair describes it. The
// draw for a uniform u is the first column whose running sum of kept weights, in column order,
// is above u times their total.
//
// Where a running sum crosses u * total, or p * total, must not hang on rounding or on the order
// of an addition: neighbouring sums differ by one weight out of up to 2^31. So a weight is a
// 64-bit integer, w_j * 2^frac rounded once, and every sum is an exact integer sum whatever its
// order. frac = min(50, 62 - ceil(log2 cols)) leaves no sum above 2^63; weights below 2^-frac of
// the row's largest (2^-45 at 131,072 columns) count as zero.
#include "rows.cuh"

#include "keys.cuh"
#include "score_load.cuh"

namespace ovvs {
namespace prim {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 256;

// Top-k order as an integer: larger is earlier; 0 marks a masked score.
__device__ __forceinline__ uint32_t sort_key(float v) {
  return v > -INFINITY ? keys::order_bits(v) : 0u;
}

struct Row {
  double m, rate;  // max; log2(e) / T
  int frac;
};

__device__ __forceinline__ uint64_t weight(const Row& r, uint32_t key) {
  const double x = keys::order_value(key);
  const double d = x == r.m ? 0.0 : x - r.m;
  const double a = d * r.rate;
  if (!(a > -64.0)) return 0;
  return static_cast<uint64_t>(__double2ll_rn(exp2(a + r.frac)));
}

template <class V, class Op>
__device__ V block_reduce(V v, Op op, V* buf) {
  for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(~0u, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  v = buf[0];
  for (int w = 1; w < kWarps; ++w) v = op(v, buf[w]);
  return v;
}

// A prefix of the row in top-k order: every score above `key`, and the first `ties` columns
// whose score is at it.
struct Edge {
  uint32_t key;
  int64_t ties;
};

template <class T>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleParams p, int frac) {
  __shared__ uint64_t red[kWarps];
  __shared__ uint64_t hist[kBins];
  __shared__ uint64_t warp_sum[kWarps];
  __shared__ uint64_t pick_sum;
  __shared__ uint32_t pick_bin;
  __shared__ int64_t found;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t cols = p.cols;
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  auto key_at = [&](int64_t j) { return sort_key(score_f32(x[j])); };
  auto add = [](uint64_t a, uint64_t b) { return a + b; };
  auto larger = [](uint64_t a, uint64_t b) { return a > b ? a : b; };

  uint64_t best = 0, n = 0;
  for (int64_t j = tid; j < cols; j += kThreads) {
    const uint32_t k = key_at(j);
    if (!k) continue;
    ++n;
    best = larger(best, (static_cast<uint64_t>(k) << 32) | static_cast<uint32_t>(~j));
  }
  best = block_reduce(best, larger, red);
  n = block_reduce(n, add, red);
  const float t = p.temperature ? p.temperature[row] : 1.f;
  if (n == 0 || !(t > 0.f)) {  // nothing to draw from, or the first in top-k order
    for (int64_t d = tid; d < p.draws; d += kThreads) {
      p.ids[row * p.draws + d] = n ? static_cast<int64_t>(~static_cast<uint32_t>(best)) : -1;
      if (p.probs) p.probs[row * p.draws + d] = n ? 1.f : 0.f;
    }
    if (tid == 0 && p.kept) p.kept[row] = n ? 1 : 0;
    return;
  }
  Row r;
  r.m = keys::order_value(static_cast<uint32_t>(best >> 32));
  r.rate = 1.4426950408889634074 / static_cast<double>(t);
  r.frac = frac;

  // The last element of the shortest prefix of `in` whose sum of value(key) reaches `target`:
  // one 8-bit digit of the key at a time, from the top.
  auto reach = [&](Edge in, uint64_t target, auto value) {
    uint64_t above = 0;
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int b = tid; b < kBins; b += kThreads) hist[b] = 0;
      __syncthreads();
      const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8);
      for (int64_t j = tid; j < cols; j += kThreads) {
        const uint32_t k = key_at(j);
        if (k > in.key && (k & mask) == prefix)
          atomicAdd(reinterpret_cast<unsigned long long*>(&hist[(k >> shift) & 255]), value(k));
      }
      if (tid == 0 && in.ties && (in.key & mask) == prefix)
        atomicAdd(reinterpret_cast<unsigned long long*>(&hist[(in.key >> shift) & 255]),
                  value(in.key) * in.ties);
      __syncthreads();
      if (tid == 0) {
        uint64_t sum = above;
        int b = kBins - 1;
        while (b > 0 && sum + hist[b] < target) sum += hist[b--];
        pick_bin = b;
        pick_sum = sum;
      }
      __syncthreads();
      prefix |= pick_bin << shift;
      above = pick_sum;
    }
    const uint64_t v = value(prefix);
    return Edge{prefix, static_cast<int64_t>((target - above + v - 1) / v)};
  };
  auto tie_count = [&](uint32_t key) {
    uint64_t c = 0;
    for (int64_t j = tid; j < cols; j += kThreads) c += key_at(j) == key;
    return static_cast<int64_t>(block_reduce(c, add, red));
  };

  Edge e{0, 0};
  const int k = p.top_k ? p.top_k[row] : 0;
  if (k > 0 && static_cast<uint64_t>(k) < n)
    e = reach(e, static_cast<uint64_t>(k), [](uint32_t) { return uint64_t{1}; });
  const float tp = p.top_p ? p.top_p[row] : 1.f;
  if (tp < 1.f) {
    uint64_t z = 0;
    for (int64_t j = tid; j < cols; j += kThreads) {
      const uint32_t kk = key_at(j);
      if (kk > e.key) z += weight(r, kk);
    }
    z = block_reduce(z, add, red);
    if (e.ties) z += weight(r, e.key) * e.ties;
    const double want = ceil(static_cast<double>(fmaxf(tp, 0.f)) * static_cast<double>(z));
    const uint64_t target = want < 1.0 ? 1 : static_cast<uint64_t>(want);
    e = reach(e, target < z ? target : z, [&](uint32_t kk) { return weight(r, kk); });
  }
  const float mp = p.min_p ? p.min_p[row] : 0.f;
  if (mp > 0.f) {
    const double edge = r.m + static_cast<double>(t) * log(fmin(static_cast<double>(mp), 1.0));
    const uint32_t ke = sort_key(__double2float_ru(edge));
    if (ke > e.key) e = Edge{ke, INT64_MAX};
  }
  uint64_t above = 0;
  for (int64_t j = tid; j < cols; j += kThreads) above += key_at(j) > e.key;
  above = block_reduce(above, add, red);
  const int64_t have = e.key ? tie_count(e.key) : 0;
  if (e.ties > have) e.ties = have;
  if (tid == 0 && p.kept) p.kept[row] = static_cast<int>(above + e.ties);

  // The column where the running sum of value(column, key) passes `target`: each warp sums a
  // contiguous range, the owner of the target walks its range again.
  const int64_t span = (cols + kThreads - 1) / kThreads * 32;
  const int64_t j0 = warp * span, j1 = j0 + span < cols ? j0 + span : cols;
  auto warp_totals = [&](auto value) {
    uint64_t s = 0;
    for (int64_t j = j0 + lane; j < j1; j += 32) s += value(j, key_at(j));
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    __syncthreads();
    if (lane == 0) warp_sum[warp] = s;
    __syncthreads();
  };
  auto walk = [&](uint64_t before, uint64_t target, auto value, auto then) {
    for (int64_t j = j0; j < j1; j += 32) {
      const uint64_t own = j + lane < j1 ? value(j + lane, key_at(j + lane)) : 0;
      uint64_t s = own;
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(~0u, s, o);
        if (lane >= o) s += y;
      }
      const unsigned hit = __ballot_sync(~0u, before + s > target);
      if (hit) {
        if (lane == __ffs(hit) - 1) then(j + lane, own);
        return;
      }
      before += __shfl_sync(~0u, s, 31);
    }
  };
  int64_t last_tie = cols;  // columns of the ties that are kept end here
  if (e.ties < have) {
    auto is_tie = [&](int64_t, uint32_t kk) { return uint64_t{kk == e.key}; };
    if (e.ties > 0) {
      warp_totals(is_tie);
      uint64_t before = 0;
      for (int w = 0; w < warp; ++w) before += warp_sum[w];
      const uint64_t target = static_cast<uint64_t>(e.ties) - 1;
      if (target >= before && target < before + warp_sum[warp])
        walk(before, target, is_tie, [&](int64_t j, uint64_t) { found = j; });
      __syncthreads();
      last_tie = found;
    } else {
      last_tie = -1;
    }
  }
  auto kept_weight = [&](int64_t j, uint32_t kk) {
    return kk > e.key || (kk && kk == e.key && j <= last_tie) ? weight(r, kk) : uint64_t{0};
  };
  warp_totals(kept_weight);
  uint64_t z = 0, before = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) before = z;
    z += warp_sum[w];
  }
  for (int64_t d = 0; d < p.draws; ++d) {
    float u = p.uniforms[row * p.draws + d];
    u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;
    const uint64_t target = static_cast<uint64_t>(static_cast<double>(u) * static_cast<double>(z));
    if (target < before || target >= before + warp_sum[warp]) continue;
    walk(before, target, kept_weight, [&](int64_t j, uint64_t own) {
      p.ids[row * p.draws + d] = j;
      if (p.probs)
        p.probs[row * p.draws + d] =
            static_cast<float>(static_cast<double>(own) / static_cast<double>(z));
    });
  }
}

int frac_bits(int64_t cols) {
  int log2 = 0;
  while ((int64_t{1} << log2) < cols) ++log2;
  return log2 < 12 ? 50 : 62 - log2;
}

}  // namespace

cudaError_t launch_sample_rows(const SampleParams& p, int type, cudaStream_t stream) {
  const unsigned grid = static_cast<unsigned>(p.rows);
  const int frac = frac_bits(p.cols);
  if (type == kScoreF32)
    sample_kernel<float><<<grid, kThreads, 0, stream>>>(p, frac);
  else if (type == kScoreF16)
    sample_kernel<__half><<<grid, kThreads, 0, stream>>>(p, frac);
  else
    sample_kernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(p, frac);
  return cudaGetLastError();
}

}  // namespace prim
}  // namespace ovvs
