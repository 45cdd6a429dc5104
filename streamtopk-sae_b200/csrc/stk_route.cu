// Router of a routed SAE (stk_route_forward / stk_route_backward): top-k of a
// row of expert scores, the chosen experts' weights, and the gradient.
//
//   s      = softmax(l) or 1 / (1 + exp(-l))
//   choice = l without a bias (both scores rise with l), s + bias with one
//   groups rank by the sum of their two best choices (s without a bias)
//   w_j    = scale * s_j, or scale * s_j / sum of the chosen s
//
// One warp per row; lane l holds the logits l, l + 32, ...  A logit of -inf or
// NaN is no candidate.
//
// The chosen set must not depend on rounding, yet 64-bit exponentials of every
// score would cost several times the row's memory traffic.  So the choice is
// made on fp32 scores together with a bound of their error: where two choices
// that decide something (the order of the picks, the k-th against the rest,
// the last kept group against the rest) are nearer than the bound, and are not
// equal by construction (same logit, same bias), the row is decided again in
// 64 bits.  With random scores that is about one row in a thousand.
#include <cfloat>
#include <cmath>
#include <cstdio>

#include "../../include/stk_b200.h"
#include "stk_host.h"
#include "stk_vec.cuh"

namespace stk {
namespace {

constexpr int kWarps = 4;
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
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
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

template <typename T>
__device__ __forceinline__ float logit_at(const T* row, int e) {
  const float x = as_f32(row[e]);
  return x == x ? x : -INFINITY;
}

// The warp's best (value, lowest index) of a 64-bit candidate per lane.
__device__ __forceinline__ void best_of(double v, int e, double* bv, int* be) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const double ov = __shfl_xor_sync(kFull, v, o);
    const int oe = __shfl_xor_sync(kFull, e, o);
    if (ov > v || (ov == v && oe < e)) {
      v = ov;
      e = oe;
    }
  }
  *bv = v;
  *be = e;
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
    for (int e = lane; e < a.E; e += 32) {
      const double x = (double)logit_at(row, e);
      if (x > -INFINITY) sum += x == top ? 1.0 : exp(x - top);
    }
    sum = warp_sum(sum);
  }
  __syncwarp();
  for (int e = lane; e < a.E; e += 32) {
    const double x = (double)logit_at(row, e);
    double s = -INFINITY;
    if (x > -INFINITY) {
      s = a.softmax ? (x == top ? 1.0 : exp(x - top)) / sum : 1.0 / (1.0 + exp(-x));
      if (a.bias != nullptr) s += (double)a.bias[e];
      if (!(s > -INFINITY)) s = -INFINITY;  // a bias of -inf or NaN
    }
    sm[e] = s;
  }
  __syncwarp();
  uint32_t kept = kFull;
  if (a.groups > 1) {
    double b1 = -INFINITY, b2 = -INFINITY;
    if (lane < a.groups)
      for (int i = 0; i < a.per; ++i) {
        const double c = sm[lane * a.per + i];
        if (c > b1) {
          b2 = b1;
          b1 = c;
        } else if (c > b2) {
          b2 = c;
        }
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

template <typename T, int V, bool COMPLEX>
__global__ void __launch_bounds__(kThreads) route_kernel(const __grid_constant__ RouteArgs a) {
  extern __shared__ double smem[];
  __shared__ int hist[kMaxExperts];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double* const wide = smem + (size_t)warp * a.E;   // COMPLEX: E doubles a warp, first used as E floats
  float* const flat = reinterpret_cast<float*>(wide);
  if (a.counts != nullptr)
    for (int e = threadIdx.x; e < a.E; e += kThreads) hist[e] = 0;
  __syncthreads();
  for (int64_t r = (int64_t)blockIdx.x * kWarps + warp; r < a.N; r += (int64_t)gridDim.x * kWarps) {
    float w = 0.f;
    int pick = -1;
    if (a.mask == nullptr || a.mask[r]) {
      const T* const row = static_cast<const T*>(a.logits) + r * a.ld;
      float x[V];
      uint32_t key[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int e = lane + 32 * i;
        x[i] = e < a.E ? logit_at(row, e) : -INFINITY;
        key[i] = x[i] > -INFINITY ? key_of(x[i]) : 0u;
      }
      float top = -INFINITY, sum = 1.f;
      if (a.softmax && (COMPLEX || !a.renorm)) {
#pragma unroll
        for (int i = 0; i < V; ++i) top = fmaxf(top, x[i]);
        top = warp_max(top);
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) sum += exp_below(x[i], top);
        sum = warp_sum(sum);
      }
      bool unsure = false;
      float eps = 0.f;
      if constexpr (COMPLEX) {
        // fp32 error of a score: the exponential, a sum of E terms and a division, within 2^-18 of the largest score
        eps = 0x1p-18f * (a.softmax ? 1.f / sum : 1.f);
        float c[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int e = lane + 32 * i;
          c[i] = a.softmax ? exp_below(x[i], top) / sum : sigmoid(x[i]);
          if (a.bias != nullptr && e < a.E) c[i] += a.bias[e];
          if (key[i] == 0u || !(c[i] > -INFINITY)) {
            c[i] = -INFINITY;
            key[i] = 0u;
          } else if (a.bias != nullptr) {
            key[i] = key_of(c[i]);
          }
        }
        if (a.groups > 1) {
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (lane + 32 * i < a.E) flat[lane + 32 * i] = c[i];
          __syncwarp();
          float b1 = -INFINITY, b2 = -INFINITY;
          int e1 = -1, e2 = -1;
          if (lane < a.groups)
            for (int i = 0; i < a.per; ++i) {
              const float v = flat[lane * a.per + i];
              if (v > b1) {
                b2 = b1;
                e2 = e1;
                b1 = v;
                e1 = lane * a.per + i;
              } else if (v > b2) {
                b2 = v;
                e2 = lane * a.per + i;
              }
            }
          __syncwarp();
          const float total = e1 < 0 ? -INFINITY : (e2 < 0 ? b1 : b1 + b2);
          const float l1 = e1 < 0 ? 0.f : logit_at(row, e1), l2 = e2 < 0 ? -INFINITY : logit_at(row, e2);
          const float c1 = a.bias != nullptr && e1 >= 0 ? a.bias[e1] : 0.f,
                      c2 = a.bias != nullptr && e2 >= 0 ? a.bias[e2] : 0.f;
          uint32_t gkey = e1 < 0 ? 0u : key_of(total), kept = 0;
          int last = -1;
          for (int t = 0; t < a.top_groups; ++t) {
            const uint32_t m = __reduce_max_sync(kFull, gkey);
            if (m == 0u) break;
            last = __ffs(__ballot_sync(kFull, gkey == m)) - 1;
            kept |= 1u << last;
            if (lane == last) gkey = 0u;
          }
          if (last >= 0) {
            const float lt = __shfl_sync(kFull, total, last);
            // (every lane takes part in every shuffle: none behind a && that a lane may skip)
            const float k1 = __shfl_sync(kFull, l1, last), k2 = __shfl_sync(kFull, l2, last);
            const float d1 = __shfl_sync(kFull, c1, last), d2 = __shfl_sync(kFull, c2, last);
            const bool same = l1 == k1 && l2 == k2 && c1 == d1 && c2 == d2;
            // totals of two scores: twice the error each, and again for the difference
            unsure = gkey != 0u && !same && total > lt - (4.f * eps + 0x1p-20f * fabsf(lt));
          }
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const int e = lane + 32 * i;
            if (e < a.E && !((kept >> (e / a.per)) & 1u)) key[i] = 0u;
          }
        }
      }
      float picked = -INFINITY;  // lane j: the j-th choice
#pragma unroll 1
      for (int j = 0; j < a.k; ++j) {
        uint32_t best = 0u;
        int at = 0;
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (key[i] > best) {
            best = key[i];
            at = i;
          }
        const uint32_t m = __reduce_max_sync(kFull, best);
        if (m == 0u) break;
        const uint32_t e = __reduce_min_sync(kFull, best == m ? (uint32_t)(lane + 32 * at) : 0xffffffffu);
        if ((e & 31u) == (uint32_t)lane) {
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (i == (int)(e >> 5)) key[i] = 0u;
        }
        if (lane == j) {
          pick = (int)e;
          picked = __uint_as_float((m & 0x80000000u) ? m ^ 0x80000000u : ~m);
        }
      }
      float l = pick >= 0 ? logit_at(row, pick) : -INFINITY;
      if constexpr (COMPLEX) {
        if (a.bias != nullptr) {
          const float b = pick >= 0 ? a.bias[pick] : 0.f;
          const float nl = __shfl_down_sync(kFull, l, 1), nb = __shfl_down_sync(kFull, b, 1),
                      np = __shfl_down_sync(kFull, picked, 1);
          const int ne = __shfl_down_sync(kFull, pick, 1);
          const float near = 2.f * eps + 0x1p-21f * fabsf(picked);
          if (lane + 1 < a.k && ne >= 0) unsure |= picked - np <= near && !(nl == l && nb == b);
          // the k-th pick against those left
          const float kl = __shfl_sync(kFull, l, a.k - 1), kb = __shfl_sync(kFull, b, a.k - 1),
                      kp = __shfl_sync(kFull, picked, a.k - 1);
          if (kp > -INFINITY) {
            const uint32_t floor_key = key_of(kp - (2.f * eps + 0x1p-21f * fabsf(kp)));
#pragma unroll
            for (int i = 0; i < V; ++i)
              if (key[i] >= floor_key) unsure |= !(x[i] == kl && a.bias[lane + 32 * i] == kb);
          }
        }
        if (__any_sync(kFull, unsure)) {
          pick = decide_exactly(row, a, wide, lane);
          l = pick >= 0 ? logit_at(row, pick) : -INFINITY;
        }
      }
      if (a.softmax) {
        if (a.renorm) {
          const float m = warp_max(l);
          const float e = exp_below(l, m);
          w = a.scale * (e / warp_sum(e));
        } else {
          w = a.scale * (exp_below(l, top) / sum);
        }
      } else {
        w = pick >= 0 ? sigmoid(l) : 0.f;
        if (a.renorm) w /= fmaxf(warp_sum(w), kSumMin);
        w *= a.scale;
      }
      if (pick < 0) w = 0.f;
    }
    if (lane < a.k) {
      a.weights[r * a.k + lane] = w;
      a.experts[r * a.k + lane] = pick;
      if (a.counts != nullptr && pick >= 0) atomicAdd(&hist[pick], 1);
    }
    __syncwarp();
  }
  if (a.counts != nullptr) {
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += kThreads)
      if (hist[e]) atomicAdd(&a.counts[e], hist[e]);  // integers: any order gives the same sum
  }
}

// Gradient of the weights with respect to the logits.  With g = scale * dL/dw:
//   softmax, divided by the chosen:  p_j sum_i (g_j - g_i) p_i        (chosen j; others 0)
//   softmax:                         chosen j: s_j (sum_i (g_j - g_i) s_i + g_j (1 - sum of the chosen s))
//                                    others e: -s_e sum_i g_i s_i
//   sigmoid:                         h_j s_j (1 - s_j), h = g, or (sum_i (g_j - g_i) s_i) / S^2 with S = sum of s
// The differences g_j - g_i and the sum over the others keep what would cancel
// in g_j - sum g s for a nearly certain choice.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) route_grad_kernel(const __grid_constant__ RouteArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t r = (int64_t)blockIdx.x * kWarps + warp; r < a.N; r += (int64_t)gridDim.x * kWarps) {
    const T* const row = static_cast<const T*>(a.logits) + r * a.ld;
    T* const out = static_cast<T*>(a.grad) + r * a.E;
    int pick = lane < a.k ? a.experts[r * a.k + lane] : -1;
    if ((unsigned)pick >= (unsigned)a.E) pick = -1;
    const bool live = __any_sync(kFull, pick >= 0);
    const float l = pick >= 0 ? logit_at(row, pick) : -INFINITY;
    if (!(l > -INFINITY)) pick = -1;
    const float g = pick >= 0 ? a.scale * a.gw[r * a.k + lane] : 0.f;
    float x[V], top = -INFINITY, s = 0.f, inv = 1.f, rest = 0.f, val = 0.f, dot = 0.f;
    const bool dense = a.softmax && !a.renorm && live;
    if (dense) {
      float all = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        x[i] = lane + 32 * i < a.E ? logit_at(row, lane + 32 * i) : -INFINITY;
        top = fmaxf(top, x[i]);
      }
      top = warp_max(top);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        x[i] = exp_below(x[i], top);
        bool chosen = false;
        for (int j = 0; j < a.k; ++j) chosen |= __shfl_sync(kFull, pick, j) == lane + 32 * i;
        all += x[i];
        rest += chosen ? 0.f : x[i];
      }
      inv = 1.f / warp_sum(all);
      rest = warp_sum(rest) * inv;
      s = exp_below(l, top) * inv;
    } else if (a.softmax) {
      const float m = warp_max(pick >= 0 ? l : -INFINITY);
      s = pick >= 0 ? exp_below(l, m) : 0.f;
      s /= fmaxf(warp_sum(s), FLT_MIN);
    } else {
      s = pick >= 0 ? sigmoid(l) : 0.f;
    }
    for (int i = 0; i < a.k; ++i) {
      const float gi = __shfl_sync(kFull, g, i), si = __shfl_sync(kFull, s, i);
      val += (g - gi) * si;
      dot += gi * si;
    }
    if (a.softmax) {
      val = s * (val + g * rest);
    } else {
      const float t = expf(-fabsf(l)), slope = t / ((1.f + t) * (1.f + t));
      if (a.renorm) {
        const float S = warp_sum(s);
        val = S >= kSumMin ? val / S / S : g / kSumMin;
      } else {
        val = g;
      }
      val *= slope;
    }
    if (pick < 0) val = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = lane + 32 * i;
      float o = 0.f;
      bool chosen = false;
      for (int j = 0; j < a.k; ++j) {
        const bool here = __shfl_sync(kFull, pick, j) == e;
        const float v = __shfl_sync(kFull, val, j);
        chosen |= here;
        o += here ? v : 0.f;
      }
      if (dense && !chosen) o = -(x[i] * inv) * dot;
      if (e < a.E) out[e] = from_f32<T>(o);
    }
  }
}

template <typename T, int V>
cudaError_t launch_v(const RouteArgs& a, bool grad, int sms, cudaStream_t s) {
  const int64_t want = (a.N + kWarps - 1) / kWarps, most = (int64_t)sms * 12;
  const unsigned grid = (unsigned)(want < most ? want : most);
  if (grad)
    route_grad_kernel<T, V><<<grid, kThreads, 0, s>>>(a);
  else if (a.bias != nullptr || a.groups > 1)
    route_kernel<T, V, true><<<grid, kThreads, sizeof(double) * kWarps * a.E, s>>>(a);
  else
    route_kernel<T, V, false><<<grid, kThreads, 0, s>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_t(const RouteArgs& a, bool grad, int sms, cudaStream_t s) {
  if (a.E <= 32) return launch_v<T, 1>(a, grad, sms, s);
  if (a.E <= 64) return launch_v<T, 2>(a, grad, sms, s);
  if (a.E <= 128) return launch_v<T, 4>(a, grad, sms, s);
  if (a.E <= 256) return launch_v<T, 8>(a, grad, sms, s);
  if (a.E <= 512) return launch_v<T, 16>(a, grad, sms, s);
  return launch_v<T, 32>(a, grad, sms, s);
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
  if (counts != nullptr) {
    const cudaError_t e = cudaMemsetAsync(counts, 0, sizeof(int32_t) * (size_t)E, s);
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaMemsetAsync");
  }
  if (N == 0) return STK_OK;
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
