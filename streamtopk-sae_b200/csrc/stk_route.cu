// Router of a routed SAE (stk_route_forward / stk_route_backward): top-k of a
// row of expert scores, the chosen experts' weights, and the gradient.
//
//   s      = softmax(l) or 1 / (1 + exp(-l))
//   choice = l without a bias (both scores rise with l), s + bias with one
//   groups rank by the sum of their two best choices (s without a bias)
//   w_j    = scale * s_j, or scale * s_j / sum of the chosen s
//
// A row is held by 1 to 32 neighbouring lanes with V (8, or 16 and 32)
// neighbouring experts each, so that a warp works on several rows at once
// where there are few experts.  A logit of -inf or NaN is no candidate.
//
// The chosen set must not depend on rounding, yet 64-bit exponentials of every
// score would cost several times the row's memory traffic.  So the choice is
// made on fp32 scores together with a bound of their error: where two choices
// that decide something (the order of the picks, the k-th against the rest,
// the last kept group against the rest) are nearer than the bound, and are not
// equal by construction (same logit, same bias), the whole warp decides the
// row again in 64 bits.
#include <cfloat>
#include <cmath>
#include <cstdio>

#include "../../include/stk_b200.h"
#include "stk_host.h"
#include "stk_vec.cuh"

namespace stk {
namespace {

constexpr int kWarps = 8;
constexpr int kWarpPicks = 256;  // picks of a warp's rows: 32 / lanes rows of at most min(32, 8 lanes) each
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxExperts = 1024;
constexpr int kMaxPicks = 32;
constexpr unsigned kFull = 0xffffffffu;
constexpr float kSumMin = 1e-20f;  // least sum that sigmoid weights are divided by

struct RouteArgs {
  const void* logits;
  const float* bias;
  const uint8_t* mask;
  float* weights;
  int32_t* experts;
  int32_t* counts;
  const float* gw;
  void* grad;
  int64_t N, ld;
  int E, k, softmax, groups, per, top_groups, renorm;
  float scale;
};

// Order-preserving key of a float that is not NaN; larger floats, larger keys,
// the two zeros alike.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key ^ (((uint32_t)~((int32_t)key >> 31)) | 0x80000000u));
}
constexpr uint32_t kNone = 0x007fffffu;  // key of -inf: no candidate at or below it

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
// exp(x - top) of a softmax whose largest logit is `top`: 1 at the top itself
// (infinite ones too), 0 where the logit is -inf.
__device__ __forceinline__ float exp_below(float x, float top) {
  return x == top ? (x == -INFINITY ? 0.f : 1.f) : (x == -INFINITY ? 0.f : expf(x - top));
}
__device__ __forceinline__ float sigmoid(float x) {
  const float t = expf(-fabsf(x));
  return x >= 0.f ? 1.f / (1.f + t) : t / (1.f + t);
}

// 1 / (1 + 2^(-x log2 e)) by the approximate exponential (two units in the last
// place and the rounding of the exponent) and reciprocal (one unit).
__device__ __forceinline__ float approx_sigmoid(float x) {
  float t, q;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(x * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(1.f + t));
  return q;
}

template <typename T>
__device__ __forceinline__ float logit_at(const T* row, int e) {
  const float x = as_f32(row[e]);
  return x == x ? x : -INFINITY;
}

// The warp's best (value, lowest index) of a 64-bit candidate per lane, by its
// order-preserving bits: the upper halves, the lower ones of those, the indices.
__device__ __forceinline__ void best_of(double v, int e, double* bv, int* be) {
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);  // (the two zeros alike)
  const uint64_t key = b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
  const uint32_t hi = (uint32_t)(key >> 32), mh = __reduce_max_sync(kFull, hi);
  const uint32_t lo = hi == mh ? (uint32_t)key : 0u, ml = __reduce_max_sync(kFull, lo);
  *be = (int)__reduce_min_sync(kFull, hi == mh && lo == ml ? (uint32_t)e : 0x7fffffffu);
  const uint64_t m = (uint64_t)mh << 32 | ml;
  *bv = __longlong_as_double((long long)(m ^ ((uint64_t)(~((int64_t)m >> 63)) | 0x8000000000000000ull)));
}

// Decides a row in 64 bits: lane j < k returns pick j (-1: none left).  `sm`:
// E doubles of this warp.
template <typename T>
__device__ __noinline__ int decide_exactly(const T* row, const RouteArgs& a, double* sm, int lane) {
  double top = -INFINITY, sum = 0.0;
  if (a.softmax) {
    for (int e = lane; e < a.E; e += 32) top = fmax(top, (double)logit_at(row, e));
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmax(top, __shfl_xor_sync(kFull, top, o));
#pragma unroll 4
    for (int e = lane; e < a.E; e += 32) {
      const double x = (double)logit_at(row, e);
      sum += x == -INFINITY ? 0.0 : x == top ? 1.0 : exp(x - top);
    }
    sum = warp_sum(sum);
  }
  __syncwarp();
#pragma unroll 4
  for (int e = lane; e < a.E; e += 32) {  // (four at once: each exponential is a long chain)
    const double x = (double)logit_at(row, e);
    const double q = exp(a.softmax ? x - top : -x);
    double s = a.softmax ? (x == top ? 1.0 : q) / sum : 1.0 / (1.0 + q);
    if (a.bias != nullptr) s += (double)a.bias[e];
    sm[e] = x > -INFINITY && s > -INFINITY ? s : -INFINITY;  // a bias of -inf or NaN: no candidate
  }
  __syncwarp();
  uint32_t kept = kFull;
  if (a.groups > 1) {
    double b1 = -INFINITY, b2 = -INFINITY;
    if (lane < a.groups)
#pragma unroll 4
      for (int i = 0; i < a.per; ++i) {
        const double c = sm[lane * a.per + (i + lane) % a.per];  // (each lane from another bank on)
        b2 = fmax(b2, fmin(b1, c));
        b1 = fmax(b1, c);
      }
    double total = b1 == -INFINITY ? -INFINITY : (b2 == -INFINITY ? b1 : b1 + b2);
    kept = 0;
    for (int t = 0; t < a.top_groups; ++t) {
      double bv;
      int bg;
      best_of(total, lane, &bv, &bg);
      if (bv == -INFINITY) break;
      kept |= 1u << bg;
      if (lane == bg) total = -INFINITY;
    }
    if (a.bias == nullptr) {  // within the groups the logits themselves decide
      __syncwarp();
      for (int e = lane; e < a.E; e += 32) sm[e] = (double)logit_at(row, e);
    }
    __syncwarp();
    for (int e = lane; e < a.E; e += 32)
      if (!((kept >> (e / a.per)) & 1u)) sm[e] = -INFINITY;
    __syncwarp();
  }
  int pick = -1;
  for (int j = 0; j < a.k; ++j) {
    double v = -INFINITY;
    int e = 0x7fffffff;
#pragma unroll 4
    for (int i = lane; i < a.E; i += 32)
      if (sm[i] > v) {
        v = sm[i];
        e = i;
      }
    double bv;
    int be;
    best_of(v, e, &bv, &be);
    if (bv == -INFINITY) break;
    if (lane == j) pick = be;
    if (lane == (be & 31)) sm[be] = -INFINITY;
    __syncwarp();
  }
  return pick;
}

// Sums and maxima over the LANES neighbouring lanes that hold a row.
template <int LANES>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
template <int LANES>
__device__ __forceinline__ float row_max(float v) {
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
template <int LANES>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  if constexpr (LANES == 32) {
    return __reduce_max_sync(kFull, v);
  } else {
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) v = max(v, __shfl_xor_sync(kFull, v, o));
    return v;
  }
}
template <int LANES>
__device__ __forceinline__ int row_min(int v) {
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) v = min(v, __shfl_xor_sync(kFull, v, o));
  return v;
}

// The exponentials of a row's softmax, and their sum.
template <int V, int LANES>
__device__ __forceinline__ float row_exp(const float (&x)[V], float top, float (&e)[V]) {
  float sum = 0.f;
  if (fabsf(top) < INFINITY) {
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = expf(x[i] - top);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = exp_below(x[i], top);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) sum += e[i];
  return row_sum<LANES>(sum);
}

// V neighbouring logits from e0 on; -inf past the row's end and for NaN.
template <typename T, int V>
__device__ __forceinline__ void load_logits(const T* row, int e0, int E, bool vec, float (&x)[V]) {
  if (vec && e0 + V <= E) {
#pragma unroll
    for (int i = 0; i < V; i += 8) {
      float w[8];
      load8(row + e0 + i, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i + j] = w[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = e0 + i < E ? as_f32(row[e0 + i]) : -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = fmaxf(x[i], -INFINITY);  // a NaN is the one operand that fmaxf passes over
}

// Sorts pairs of a small array into descending order.
__device__ __forceinline__ void order(uint32_t& a, uint32_t& b) {
  const uint32_t hi = max(a, b), lo = min(a, b);
  a = hi;
  b = lo;
}
// x[0 .. N) bitonic, or anything for N <= 2: descending afterwards.
template <int N>
__device__ __forceinline__ void bitonic_down(uint32_t* x) {
#pragma unroll
  for (int s = N / 2; s; s >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((i & s) == 0) order(x[i], x[i + s]);
}
template <int N>
__device__ __forceinline__ void sort_down(uint32_t* x) {
  if constexpr (N > 1) {
    sort_down<N / 2>(x);
    sort_down<N / 2>(x + N / 2);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) order(x[i], x[N - 1 - i]);
    bitonic_down<N / 2>(x);
    bitonic_down<N / 2>(x + N / 2);
  }
}

// The K largest of a row's keys, in descending order, in every lane of the row:
// each lane's own first, then merged over 1, 2, 4, ... lanes (of two descending
// lists the K largest are the larger of a[i] and b[K - 1 - i], a bitonic list).
// For four of 64 in eight lanes 68 comparisons and 12 shuffles, against 160 for
// four rounds that find and remove a maximum.
template <int K, int LANES>
__device__ __forceinline__ void top_of_row(uint32_t (&key)[8], uint32_t (&best)[K]) {
  if constexpr (K == 8) {
    sort_down<8>(key);
#pragma unroll
    for (int i = 0; i < K; ++i) best[i] = key[i];
  } else {
    sort_down<4>(key);
    sort_down<4>(key + 4);
#pragma unroll
    for (int i = 0; i < K; ++i) best[i] = max(key[i], key[7 - i]);
    bitonic_down<4>(best);
  }
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) {
    uint32_t other[K];
#pragma unroll
    for (int i = 0; i < K; ++i) other[i] = __shfl_xor_sync(kFull, best[i], o);
#pragma unroll
    for (int i = 0; i < K; ++i) best[i] = max(best[i], other[K - 1 - i]);
    bitonic_down<K>(best);
  }
}

// Which of a row's groups are kept, as bits, from its choices c; `unsure` is
// set where fp32 leaves that open.  Where a group is 1, 2, 4, ... whole lanes
// its two best come from the registers (256 experts in 8 groups: 40
// instructions); else from shared memory, a lane per group.
template <int V, int LANES>
__device__ __forceinline__ uint32_t keep_groups(const RouteArgs& a, const float (&c)[V], float* flat, int gl, int sub,
                                                float eps, bool* unsure) {
  constexpr int GT = LANES <= 4 ? 8 : 32 / LANES;  // groups of a lane: at most 8 lanes or 32 over all lanes
  constexpr uint32_t rows = LANES == 32 ? kFull : (1u << (LANES & 31)) - 1u;
  // Of two totals of two choices: each score's error four times, and the roundings of four sums with the bias and of
  // the totals, of the largest choice (a total may be far smaller than its two terms).
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) most = fmaxf(most, c[i] > -INFINITY ? fabsf(c[i]) : 0.f);
  const float margin = 4.f * eps + 0x1p-20f * row_max<LANES>(most);
  uint32_t kept = 0;
  float last = INFINITY;
  const int span = a.per / V;
  if (a.per % V == 0 && (span & (span - 1)) == 0) {
    float b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      b2 = fmaxf(b2, fminf(b1, c[i]));
      b1 = fmaxf(b1, c[i]);
    }
    for (int o = 1; o < span; o <<= 1) {
      const float o1 = __shfl_xor_sync(kFull, b1, o), o2 = __shfl_xor_sync(kFull, b2, o);
      b2 = fmaxf(fmaxf(b2, o2), fminf(b1, o1));
      b1 = fmaxf(b1, o1);
    }
    const float total = b2 == -INFINITY ? b1 : b1 + b2;
    const int g = gl / span;  // lanes past the last group hold nothing but -inf
    uint32_t key = total > -INFINITY ? key_of(total) : 0u;
    for (int t = 0; t < a.top_groups; ++t) {
      const uint32_t m = row_max<LANES>(key);
      const uint32_t who = (__ballot_sync(kFull, key == m) >> (sub * LANES)) & rows;
      if (m == 0u) continue;
      const int best = (__ffs(who) - 1) / span;
      kept |= 1u << best;
      last = value_of(m);
      if (g == best) key = 0u;
    }
    *unsure |= key != 0u && total > last - margin;
    return kept;
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (gl * V + i < a.E) flat[gl * V + i] = c[i];
  __syncwarp();
  float total[GT];
  uint32_t key[GT];
#pragma unroll
  for (int t = 0; t < GT; ++t) {
    const int g = gl + LANES * t;
    float b1 = -INFINITY, b2 = -INFINITY;
    if (g < a.groups)
      for (int i = 0; i < a.per; ++i) {
        const float v = flat[g * a.per + i];
        b2 = fmaxf(b2, fminf(b1, v));
        b1 = fmaxf(b1, v);
      }
    total[t] = b2 == -INFINITY ? b1 : b1 + b2;
    key[t] = total[t] > -INFINITY ? key_of(total[t]) : 0u;
  }
  for (int n = 0; n < a.top_groups; ++n) {
    uint32_t best = 0u;
    int at = 0;
#pragma unroll
    for (int t = 0; t < GT; ++t)
      if (key[t] > best) {
        best = key[t];
        at = gl + LANES * t;
      }
    const uint32_t m = row_max<LANES>(best);
    const int g = row_min<LANES>(best == m ? at : kMaxExperts);
    if (m == 0u) continue;
    kept |= 1u << g;
    last = value_of(m);
#pragma unroll
    for (int t = 0; t < GT; ++t)
      if (g == gl + LANES * t) key[t] = 0u;
  }
#pragma unroll
  for (int t = 0; t < GT; ++t)
    *unsure |= key[t] != 0u && total[t] > last - margin;
  return kept;
}

// K: 4 or 8 where the picks come from top_of_row (16-bit logits without a bias, 2 <= k <= K), else 0.
template <typename T, int V, int LANES, bool COMPLEX, int K>
__global__ void __launch_bounds__(kThreads, COMPLEX ? (V == 8 ? 3 : 2) : 5) route_kernel(const __grid_constant__ RouteArgs a, bool vec) {
  constexpr int R = 32 / LANES;
  constexpr uint32_t rows = LANES == 32 ? kFull : (1u << (LANES & 31)) - 1u;
  constexpr bool PACKED = sizeof(T) == 2 && !COMPLEX;
  extern __shared__ double smem[];
  __shared__ int hist[kMaxExperts];
  __shared__ int s_pick[kWarps][kWarpPicks];
  __shared__ float s_logit[kWarps][kWarpPicks];
  __shared__ float s_choice[COMPLEX ? kWarps : 1][COMPLEX ? kWarpPicks : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gl = lane % LANES, sub = lane / LANES;
  const int e0 = gl * V, k = a.k;
  // COMPLEX: E doubles, or R rows of E floats, a warp
  double* const wide = reinterpret_cast<double*>(reinterpret_cast<float*>(smem) + (size_t)warp * a.E * (R > 2 ? R : 2));
  float* const flat = reinterpret_cast<float*>(wide) + sub * a.E;
  int* const pick = s_pick[warp] + sub * k;
  float* const plogit = s_logit[warp] + sub * k;
  if (a.counts != nullptr) {
    for (int e = threadIdx.x; e < a.E; e += kThreads) hist[e] = 0;
    __syncthreads();
  }
  const int group0 = e0 / a.per, left0 = a.per - e0 % a.per;  // the first expert's group, and what is left of it
  float b[COMPLEX ? V : 1];  // the biases of this lane's experts
  if constexpr (COMPLEX) {
#pragma unroll
    for (int i = 0; i < V; ++i) b[i] = a.bias != nullptr && e0 + i < a.E ? a.bias[e0 + i] : 0.f;
  }
  for (int64_t r0 = ((int64_t)blockIdx.x * kWarps + warp) * R; r0 < a.N; r0 += (int64_t)gridDim.x * kWarps * R) {
    const int64_t r = r0 + sub;
    const bool inside = r < a.N;
    float x[V];
    uint32_t key[V];
    if (inside && (a.mask == nullptr || a.mask[r])) {
      load_logits<T, V>(static_cast<const T*>(a.logits) + r * a.ld, e0, a.E, vec, x);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = -INFINITY;
    }
    float top = -INFINITY, sum = 1.f, c[V];
    if (a.softmax && (COMPLEX || !a.renorm)) {
#pragma unroll
      for (int i = 0; i < V; ++i) top = fmaxf(top, x[i]);
      top = row_max<LANES>(top);
      sum = row_exp<V, LANES>(x, top, c);
    }
    bool unsure = false;
    // Error of an fp32 score, u = 2^-24.  Sigmoid: the exponential t of -x is within (4 + 2.1 |x|) u of itself (its
    // own two units in the last place, and the exponent's rounding), which moves 1 / (1 + t) by t / (1 + t)^2 <= 1/4 of
    // that and, as that falls with |x|, by 2 u at most; the sum and the reciprocal add 4 u.  Softmax, of the largest score: an exponential within
    // (4 + |x - top|) u, weighted by itself below 11 u in the sum, V + 5 additions, the division and the product.
    // A key that holds its place in the lane (log2 V bits) is up to 2 V u of its choice below it.
    float eps = 0.f;
    if constexpr (COMPLEX) {
      const float inv = 1.f / sum;
      eps = a.softmax ? (24 + V) * 0x1p-24f * inv : 0x1p-21f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        c[i] = a.softmax ? c[i] * inv : approx_sigmoid(x[i]);
        c[i] = x[i] > -INFINITY ? fmaxf(c[i] + b[i], -INFINITY) : -INFINITY;
        key[i] = a.bias != nullptr ? (key_of(c[i]) & ~(V - 1u)) | (uint32_t)(V - 1 - i) : key_of(x[i]);
      }
      if (a.groups > 1) {
        const uint32_t kept = keep_groups<V, LANES>(a, c, flat, gl, sub, eps, &unsure);
        int g = group0, left = left0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (e0 + i >= a.E || !((kept >> g) & 1u)) key[i] = 0u;
          if (--left == 0) {
            ++g;
            left = a.per;
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        key[i] = key_of(x[i]);
        // 16-bit logits leave 13 bits of their fp32 form free: with the index in ten of them no two keys are equal
        if (PACKED) key[i] = (key[i] & ~1023u) | (uint32_t)(1023 - e0 - i);
      }
    }
    if constexpr (K > 0) {
      static_assert(PACKED && V == 8, "keys with their index, eight a lane");
      uint32_t best[K];
      top_of_row<K, LANES>(key, best);
      for (int j = gl; j < k; j += LANES) {
        uint32_t m = best[0];
#pragma unroll
        for (int i = 1; i < K; ++i) m = i == j ? best[i] : m;
        pick[j] = m > kNone ? 1023 - (int)(m & 1023u) : -1;
        plogit[j] = m > kNone ? value_of((m & 0x80000000u) ? m & ~1023u : m | 1023u) : -INFINITY;
      }
    }
#pragma unroll 1
    for (int j = 0; j < (K > 0 ? 0 : k); ++j) {
      uint32_t best = key[0];
#pragma unroll
      for (int i = 1; i < V; ++i) best = max(best, key[i]);
      const bool placed = COMPLEX && a.bias != nullptr;  // keys with their place in the lane: compared without it
      const uint32_t mine_key = placed ? best | (V - 1u) : best, m = row_max<LANES>(mine_key);
      if constexpr (PACKED) {
        if (gl == 0) {
          pick[j] = m > kNone ? 1023 - (int)(m & 1023u) : -1;
          plogit[j] = m > kNone ? value_of((m & 0x80000000u) ? m & ~1023u : m | 1023u) : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) key[i] = key[i] == m ? 0u : key[i];
      } else {
        // of equals the lowest lane, and in it the first: lanes and places are in the experts' order
        const uint32_t who = (__ballot_sync(kFull, mine_key == m) >> (sub * LANES)) & rows;
        const bool mine = gl == __ffs(who) - 1;
        int at = 0;
        if (placed) {  // no two keys of a lane are equal
          at = V - 1 - (int)(best & (V - 1u));
          const uint32_t gone = mine ? best : 0u;
#pragma unroll
          for (int i = 0; i < V; ++i) key[i] = key[i] == gone ? 0u : key[i];
        } else {
#pragma unroll
          for (int i = V - 1; i > 0; --i) at = key[i] == m ? i : at;
          at = key[0] == m ? 0 : at;
          const int gone = mine ? at : -1;
#pragma unroll
          for (int i = 0; i < V; ++i) key[i] = i == gone ? 0u : key[i];
        }
        if (mine) {
          pick[j] = m > kNone ? e0 + at : -1;
          if constexpr (COMPLEX) s_choice[warp][sub * k + j] = m > kNone ? value_of(m) : -INFINITY;
          else plogit[j] = m > kNone ? value_of(m) : -INFINITY;
        }
      }
    }
    if constexpr (COMPLEX) {
      __syncwarp();
      for (int j = gl; j < k; j += LANES)
        plogit[j] = pick[j] >= 0 ? logit_at(static_cast<const T*>(a.logits) + r * a.ld, pick[j]) : -INFINITY;
    }
    __syncwarp();
    if constexpr (COMPLEX) {
      if (a.bias != nullptr) {
        // the sum with the bias, and the key's low log2 V bits: both sides of a comparison have them all set, so that
        // each is at most 2 V u above its choice and never below it
        constexpr float near = (2 * V + 4) * 0x1p-24f;
        const float* const choice = s_choice[warp] + sub * k;
        for (int j = gl; j + 1 < k; j += LANES)
          if (pick[j + 1] >= 0 && choice[j] - choice[j + 1] <= 2.f * eps + near * fabsf(choice[j]))
            unsure |= plogit[j] != plogit[j + 1] || a.bias[pick[j]] != a.bias[pick[j + 1]];
        if (pick[k - 1] >= 0) {  // the last pick against those left
          const float c = choice[k - 1], l = plogit[k - 1], pb = a.bias[pick[k - 1]];
          const uint32_t low = key_of(c - (2.f * eps + near * fabsf(c)));
#pragma unroll
          for (int i = 0; i < V; ++i)
            if ((key[i] | (V - 1u)) >= low && key[i] > kNone) unsure |= x[i] != l || b[i] != pb;
        }
      }
      uint32_t open = __ballot_sync(kFull, unsure);
      while (open != 0u) {
        const int s = (__ffs(open) - 1) / LANES;
        open &= ~(rows << (s * LANES));
        const T* const row = static_cast<const T*>(a.logits) + (r0 + s) * a.ld;
        const int e = decide_exactly(row, a, wide, lane);
        if (lane < k) {
          s_pick[warp][s * k + lane] = e;
          s_logit[warp][s * k + lane] = e >= 0 ? logit_at(row, e) : -INFINITY;
        }
        __syncwarp();
      }
    }
    // Weights: lane gl of a row's lanes has picks gl, gl + LANES, ...
    float m = -INFINITY, S = 0.f;
    if (a.renorm) {
      if (a.softmax) {
        for (int j = gl; j < k; j += LANES) m = fmaxf(m, plogit[j]);
        m = row_max<LANES>(m);
      }
      for (int j = gl; j < k; j += LANES)
        S += a.softmax ? exp_below(plogit[j], m) : (pick[j] >= 0 ? sigmoid(plogit[j]) : 0.f);
      S = row_sum<LANES>(S);
      if (!a.softmax) S = fmaxf(S, kSumMin);
    } else if (a.softmax) {
      m = top;
      S = sum;
    } else {
      S = 1.f;
    }
    for (int j = gl; j < k && inside; j += LANES) {
      const int e = pick[j];
      float w = 0.f;
      if (e >= 0) {
        w = a.scale * ((a.softmax ? exp_below(plogit[j], m) : sigmoid(plogit[j])) / S);
        if (a.counts != nullptr) atomicAdd(&hist[e], 1);
      }
      a.weights[r * k + j] = w;
      a.experts[r * k + j] = e;
    }
    __syncwarp();
  }
  if (a.counts != nullptr) {
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += kThreads) {
      if (gridDim.x == 1) a.counts[e] = hist[e];           // (not zeroed beforehand then)
      else if (hist[e]) atomicAdd(&a.counts[e], hist[e]);  // integers: any order gives the same sum
    }
  }
}

// Gradient of the weights with respect to the logits.  With g = scale * dL/dw:
//   softmax, divided by the chosen:  p_j sum_i (g_j - g_i) p_i        (chosen j; others 0)
//   softmax:                         chosen j: s_j (sum_i (g_j - g_i) s_i + g_j (1 - sum of the chosen s))
//                                    others e: -s_e sum_i g_i s_i
//   sigmoid:                         h_j s_j (1 - s_j), h = g, or (sum_i (g_j - g_i) s_i) / S^2 with S = sum of s
// The differences g_j - g_i and the sum over the others keep what would cancel
// in g_j - sum g s for a nearly certain choice.
// FEW (k <= LANES): lane j of a row's lanes has choice j in registers; else the
// choices go through shared memory.
template <typename T, int V, int LANES, bool FEW>
__global__ void __launch_bounds__(kThreads) route_grad_kernel(const __grid_constant__ RouteArgs a, bool vec, bool vec_out) {
  constexpr int R = 32 / LANES;
  constexpr int W = FEW ? 1 : kWarps, P = FEW ? 1 : kWarpPicks;
  __shared__ int s_pick[W][P];
  __shared__ float s_score[W][P], s_g[W][P], s_val[W][P];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gl = lane % LANES, sub = lane / LANES;
  const int e0 = gl * V, k = a.k;
  int* const pick = s_pick[FEW ? 0 : warp] + (FEW ? 0 : sub * k);
  float* const score = s_score[FEW ? 0 : warp] + (FEW ? 0 : sub * k);
  float* const gr = s_g[FEW ? 0 : warp] + (FEW ? 0 : sub * k);
  float* const val = s_val[FEW ? 0 : warp] + (FEW ? 0 : sub * k);
  for (int64_t r0 = ((int64_t)blockIdx.x * kWarps + warp) * R; r0 < a.N; r0 += (int64_t)gridDim.x * kWarps * R) {
    const int64_t r = r0 + sub;
    const bool inside = r < a.N;
    const T* const row = static_cast<const T*>(a.logits) + (inside ? r : 0) * a.ld;
    const bool dense = a.softmax && !a.renorm;  // every logit has a gradient
    float x[V], inv = 0.f, rest = 0.f, dot = 0.f;
    uint32_t chosen = 0;
    int mine = -1;       // FEW: this lane's choice and its gradient
    float mine_v = 0.f;
    if constexpr (FEW) {
      if (inside && gl < k) mine = a.experts[r * k + gl];
      if ((unsigned)mine >= (unsigned)a.E) mine = -1;
      float g = mine >= 0 ? a.scale * a.gw[r * k + gl] : 0.f;
      const float l = mine >= 0 ? logit_at(row, mine) : -INFINITY;
      if (!(l > -INFINITY)) {
        mine = -1;
        g = 0.f;
      }
      float s, S = 0.f;
      if (dense) {
        // rows without a choice: x stays 0, so that nothing is written but 0
        const int live = row_min<LANES>(mine >= 0 ? 0 : 1);
        if (live == 0) {
          load_logits<T, V>(row, e0, a.E, vec, x);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) x[i] = -INFINITY;
        }
        float m = x[0];
#pragma unroll
        for (int i = 1; i < V; ++i) m = fmaxf(m, x[i]);
        m = row_max<LANES>(m);
        for (int j = 0; j < k; ++j) {
          const unsigned at = (unsigned)(__shfl_sync(kFull, mine, j, LANES) - e0);
          if (at < (unsigned)V) chosen |= 1u << at;
        }
        const float all = row_exp<V, LANES>(x, m, x);
#pragma unroll
        for (int i = 0; i < V; ++i) rest += (chosen >> i) & 1u ? 0.f : x[i];
        inv = 1.f / fmaxf(all, FLT_MIN);
        rest = row_sum<LANES>(rest) * inv;
        s = mine >= 0 ? exp_below(l, m) * inv : 0.f;
      } else if (a.softmax) {
        const float m = row_max<LANES>(l);  // (by every lane, whether it has a choice or not)
        s = mine >= 0 ? exp_below(l, m) : 0.f;
        s *= 1.f / fmaxf(row_sum<LANES>(s), FLT_MIN);
      } else {
        s = mine >= 0 ? sigmoid(l) : 0.f;
        S = row_sum<LANES>(s);
      }
      for (int i = 0; i < k; ++i) {
        const float gi = __shfl_sync(kFull, g, i, LANES), si = __shfl_sync(kFull, s, i, LANES);
        mine_v += (g - gi) * si;
        dot += gi * si;
      }
      if (a.softmax) {
        mine_v = s * (mine_v + g * rest);
      } else {
        const float t = expf(-fabsf(l)), slope = t / ((1.f + t) * (1.f + t));
        mine_v = (a.renorm ? (S >= kSumMin ? mine_v / S / S : g / kSumMin) : g) * slope;
      }
    } else {
      // The chosen ones' logits (kept in `val` for the moment) and gradients.
      int any = 0;
      float m = -INFINITY;
      for (int j = gl; j < k; j += LANES) {
        int e = inside ? a.experts[r * k + j] : -1;
        if ((unsigned)e >= (unsigned)a.E) e = -1;
        const float l = e >= 0 ? logit_at(row, e) : -INFINITY;
        if (!(l > -INFINITY)) e = -1;
        pick[j] = e;
        val[j] = l;
        gr[j] = e >= 0 ? a.scale * a.gw[r * k + j] : 0.f;
        m = fmaxf(m, l);
        any |= e >= 0;
      }
      __syncwarp();
      if (dense) {
        // rows without a choice: x stays 0, so that nothing is written but 0
        const int live = row_min<LANES>(-any);
        if (live != 0) {
          load_logits<T, V>(row, e0, a.E, vec, x);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) x[i] = -INFINITY;
        }
        m = -INFINITY;
#pragma unroll
        for (int i = 0; i < V; ++i) m = fmaxf(m, x[i]);
        m = row_max<LANES>(m);
        for (int j = 0; j < k; ++j) {
          const unsigned at = (unsigned)(pick[j] - e0);
          if (at < (unsigned)V) chosen |= 1u << at;
        }
        const float all = row_exp<V, LANES>(x, m, x);
#pragma unroll
        for (int i = 0; i < V; ++i) rest += (chosen >> i) & 1u ? 0.f : x[i];
        inv = 1.f / fmaxf(all, FLT_MIN);
        rest = row_sum<LANES>(rest) * inv;
      } else if (a.softmax) {
        m = row_max<LANES>(m);
      }
      float S = 0.f;
      for (int j = gl; j < k; j += LANES) {
        const float s = pick[j] < 0 ? 0.f : (a.softmax ? exp_below(val[j], m) : sigmoid(val[j]));
        score[j] = s;
        S += s;
      }
      const float norm = a.softmax ? (dense ? inv : 1.f / fmaxf(row_sum<LANES>(S), FLT_MIN)) : 1.f;
      if (!a.softmax) S = row_sum<LANES>(S);
      __syncwarp();
      for (int j = 0; j < k; ++j) dot += gr[j] * (score[j] * norm);
      for (int j = gl; j < k; j += LANES) {
        const float g = gr[j], s = score[j] * norm;
        float v = 0.f;
        for (int i = 0; i < k; ++i) v += (g - gr[i]) * (score[i] * norm);
        if (a.softmax) {
          v = s * (v + g * rest);
        } else {
          const float t = expf(-fabsf(val[j])), slope = t / ((1.f + t) * (1.f + t));
          v = (a.renorm ? (S >= kSumMin ? v / S / S : g / kSumMin) : g) * slope;
        }
        val[j] = pick[j] >= 0 ? v : 0.f;
      }
      __syncwarp();
    }
    // The row without its choices, then those over it.
    T* const out = static_cast<T*>(a.grad) + (inside ? r : 0) * a.E;
    if (inside) {
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = dense ? -(x[i] * inv) * dot : 0.f;
      if (vec_out && e0 + V <= a.E) {
#pragma unroll
        for (int i = 0; i < V; i += 8) {
          float w[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) w[j] = x[i + j];
          store8(out + e0 + i, w);
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (e0 + i < a.E) out[e0 + i] = from_f32<T>(x[i]);
      }
    }
    __syncwarp();  // orders the lanes' stores to one row
    if constexpr (FEW) {
      if (mine >= 0) out[mine] = from_f32<T>(mine_v);
    } else {
      for (int j = gl; j < k; j += LANES)
        if (pick[j] >= 0) out[pick[j]] = from_f32<T>(val[j]);
    }
    __syncwarp();
  }
}

template <typename T, int V, int LANES>
cudaError_t launch_v(const RouteArgs& a, bool grad, int sms, cudaStream_t s) {
  constexpr int R = 32 / LANES;
  const int64_t want = (a.N + kWarps * R - 1) / (kWarps * R), most = (int64_t)sms * (grad ? 4 : a.bias != nullptr || a.groups > 1 ? (V == 8 ? 3 : 2) : 5);
  const unsigned grid = (unsigned)(want < most ? want : most);
  if (!grad && a.counts != nullptr && grid > 1) {  // one CTA writes its counts, more add theirs
    const cudaError_t e = cudaMemsetAsync(a.counts, 0, sizeof(int32_t) * (size_t)a.E, s);
    if (e != cudaSuccess) return e;
  }
  const bool vec = vec_aligned<T>(a.logits) && a.ld % 8 == 0;
  if (grad) {
    const bool vec_out = vec_aligned<T>(a.grad) && a.E % 8 == 0;
    if (a.k <= LANES) route_grad_kernel<T, V, LANES, true><<<grid, kThreads, 0, s>>>(a, vec, vec_out);
    else route_grad_kernel<T, V, LANES, false><<<grid, kThreads, 0, s>>>(a, vec, vec_out);
  } else if (a.bias != nullptr || a.groups > 1) {
    const size_t bytes = sizeof(float) * kWarps * a.E * (R > 2 ? R : 2);
    // The limit is the kernel's, and host threads may launch it with other numbers of experts at the same time: it is
    // always set to what the most experts take, never to less than another thread is about to launch with.
    constexpr int most_bytes = sizeof(float) * kWarps * V * LANES * (R > 2 ? R : 2);
    if constexpr (most_bytes > 16 * 1024) {
      const cudaError_t e = cudaFuncSetAttribute(route_kernel<T, V, LANES, true, 0>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, most_bytes);
      if (e != cudaSuccess) return e;
    }
    route_kernel<T, V, LANES, true, 0><<<grid, kThreads, bytes, s>>>(a, vec);
  } else if constexpr (sizeof(T) == 2 && V == 8) {
    if (a.k > 1 && a.k <= 4) route_kernel<T, V, LANES, false, 4><<<grid, kThreads, 0, s>>>(a, vec);
    else if (a.k > 1 && a.k <= 8) route_kernel<T, V, LANES, false, 8><<<grid, kThreads, 0, s>>>(a, vec);
    else route_kernel<T, V, LANES, false, 0><<<grid, kThreads, 0, s>>>(a, vec);
  } else {
    route_kernel<T, V, LANES, false, 0><<<grid, kThreads, 0, s>>>(a, vec);
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_t(const RouteArgs& a, bool grad, int sms, cudaStream_t s) {
  // With a bias or groups a row's fixed work (each pick, the checks, the weights) is shared by twice the rows where a
  // lane holds 16 experts.  Kernel times with 8 and with 16 a lane, in microseconds:
  //   64 experts, top 4, bias       512 rows 4.9, 5.6  4096 8.3, 8.9    8192 9.2, 9.2    20000 12.5, 10.7  65536 27, 25
  //   128 experts, top 8, bias      512 rows 5.6, 6.6  4096 10.7, 10.6  8192 14.5, 12.3  20000 23.7, 20.8  65536 59, 51
  //   256 in 8 groups, top 8, bias  512 rows 6.1, 7.9  4096 20.6, 19.6  8192 26.5, 27.0  20000 48.2, 44.2  65536 137, 127
  // They are even between 4096 and 8192 rows.  With groups that are not whole lanes of 16 eight are faster (65536 x 64 in
  // groups of 8: 39 against 45 us).
  const int per = a.groups > 1 ? a.per : 16;
  if (!grad && (a.bias != nullptr || a.groups > 1) && a.E > 32 && a.E <= 256 && a.N >= 4096 && per % 16 == 0) {
    if (a.E <= 64) return launch_v<T, 16, 4>(a, grad, sms, s);
    if (a.E <= 128) return launch_v<T, 16, 8>(a, grad, sms, s);
    return launch_v<T, 16, 16>(a, grad, sms, s);
  }
  if (a.E <= 8) return launch_v<T, 8, 1>(a, grad, sms, s);
  if (a.E <= 16) return launch_v<T, 8, 2>(a, grad, sms, s);
  if (a.E <= 32) return launch_v<T, 8, 4>(a, grad, sms, s);
  if (a.E <= 64) return launch_v<T, 8, 8>(a, grad, sms, s);
  if (a.E <= 128) return launch_v<T, 8, 16>(a, grad, sms, s);
  if (a.E <= 256) return launch_v<T, 8, 32>(a, grad, sms, s);
  if (a.E <= 512) return launch_v<T, 16, 32>(a, grad, sms, s);
  return launch_v<T, 32, 32>(a, grad, sms, s);
}

int run(const RouteArgs& a, int dtype, bool grad, cudaStream_t s) {
  int sms = 0;
  if (const int rc = host_device_sms(&sms)) return rc;
  const cudaError_t e = dtype == STK_F32   ? launch_t<float>(a, grad, sms, s)
                        : dtype == STK_F16 ? launch_t<__half>(a, grad, sms, s)
                                           : launch_t<__nv_bfloat16>(a, grad, sms, s);
  return e == cudaSuccess ? STK_OK : host_cuda_fail(e, grad ? "route_grad_kernel launch" : "route_kernel launch");
}

// What forward and backward both refuse.
int check(const char* who, int dtype, int64_t ld, int64_t N, int64_t E, int64_t k, int score, double scale) {
  static thread_local char msg[128];
  const char* bad = nullptr;
  if (dtype != STK_F32 && dtype != STK_F16 && dtype != STK_BF16) bad = "logits must be fp32, fp16, or bf16";
  else if (score != STK_SCORE_SOFTMAX && score != STK_SCORE_SIGMOID) bad = "unknown score";
  else if (N < 0 || E < 1 || E > kMaxExperts) bad = "need N >= 0 and 1 <= E <= 1024";
  else if (k < 1 || k > kMaxPicks || k > E) bad = "need 1 <= k <= min(32, E)";
  else if (ld < E) bad = "row stride below E";
  else if (!std::isfinite(scale)) bad = "scale must be finite";
  if (!bad) return STK_OK;
  snprintf(msg, sizeof msg, "%s: %s", who, bad);
  return host_fail(STK_EINVAL, msg);
}

}  // namespace
}  // namespace stk

extern "C" int stk_route_forward(const void* logits, int dtype, int64_t ld, const float* bias, const uint8_t* row_mask,
                                 float* weights, int32_t* experts, int32_t* counts, int64_t N, int64_t E, int64_t k,
                                 int score, int64_t n_groups, int64_t topk_groups, int renormalize, double scale,
                                 void* stream) {
  STK_ENTRY_BEGIN
  using namespace stk;
  if (const int rc = check("stk_route_forward", dtype, ld, N, E, k, score, scale)) return rc;
  if (n_groups < 1 || n_groups > 32 || E % n_groups || topk_groups < 1 || topk_groups > n_groups)
    return host_fail(STK_EINVAL, "stk_route_forward: need 1 <= topk_groups <= n_groups <= 32 and E a multiple of n_groups");
  if (k > topk_groups * (E / n_groups))
    return host_fail(STK_EINVAL, "stk_route_forward: k exceeds the experts of topk_groups groups");
  if (N > 0 && (!logits || !weights || !experts)) return host_fail(STK_EINVAL, "stk_route_forward: null pointer");
  if (!aligned_to(logits, dtype == STK_F32 ? 4 : 2) || !aligned_to(bias, 4) || !aligned_to(weights, 4) ||
      !aligned_to(experts, 4) || !aligned_to(counts, 4))
    return host_fail(STK_EINVAL, "stk_route_forward: pointer not aligned to its element");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (N == 0) {
    const cudaError_t e = counts != nullptr ? cudaMemsetAsync(counts, 0, sizeof(int32_t) * (size_t)E, s) : cudaSuccess;
    return e == cudaSuccess ? STK_OK : host_cuda_fail(e, "cudaMemsetAsync");
  }
  RouteArgs a = {};
  a.logits = logits;
  a.bias = bias;
  a.mask = row_mask;
  a.weights = weights;
  a.experts = experts;
  a.counts = counts;
  a.N = N;
  a.ld = ld;
  a.E = (int)E;
  a.k = (int)k;
  a.softmax = score == STK_SCORE_SOFTMAX;
  a.groups = topk_groups < n_groups ? (int)n_groups : 1;  // all groups kept: no group is left out
  a.per = (int)(E / n_groups);
  a.top_groups = (int)topk_groups;
  a.renorm = renormalize != 0;
  a.scale = (float)scale;
  return run(a, dtype, false, s);
  STK_ENTRY_END
}

extern "C" int stk_route_backward(const float* grad_weights, const void* logits, int dtype, int64_t ld,
                                  const int32_t* experts, void* grad_logits, int64_t N, int64_t E, int64_t k, int score,
                                  int renormalize, double scale, void* stream) {
  STK_ENTRY_BEGIN
  using namespace stk;
  if (const int rc = check("stk_route_backward", dtype, ld, N, E, k, score, scale)) return rc;
  if (N == 0) return STK_OK;
  if (!grad_weights || !logits || !experts || !grad_logits)
    return host_fail(STK_EINVAL, "stk_route_backward: null pointer");
  const size_t es = dtype == STK_F32 ? 4 : 2;
  if (!aligned_to(logits, es) || !aligned_to(grad_logits, es) || !aligned_to(grad_weights, 4) || !aligned_to(experts, 4))
    return host_fail(STK_EINVAL, "stk_route_backward: pointer not aligned to its element");
  RouteArgs a = {};
  a.logits = logits;
  a.gw = grad_weights;
  a.experts = const_cast<int32_t*>(experts);
  a.grad = grad_logits;
  a.N = N;
  a.ld = ld;
  a.E = (int)E;
  a.k = (int)k;
  a.softmax = score == STK_SCORE_SOFTMAX;
  a.renorm = renormalize != 0;
  a.scale = (float)scale;
  return run(a, dtype, true, static_cast<cudaStream_t>(stream));
  STK_ENTRY_END
}
