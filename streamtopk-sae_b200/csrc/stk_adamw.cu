// One AdamW step over many tensors (stk_adamw_step).
//
//   m' = b1 m + (1 - b1) g          v' = b2 v + (1 - b2) g^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// Each element's work is a dozen fp32 operations on up to 28 bytes, so the
// step is bound by memory: everything is read once and written once, and all
// tensors go in one launch (tables of kTensors tensors travel as kernel
// parameters, so a captured launch needs no table in memory).
//
// 8-bit states: m and sqrt(v) as E4M3 codes with one fp32 scale per 256
// elements (scale = largest finite magnitude / 448).  The square root halves
// v's range in octaves, which E4M3's 17 octaves then hold.  A warp owns a
// block of 256 elements, so the block's largest magnitude is one warp
// reduction and the state is requantized in the same pass.  sqrt(v) > 0 is
// never stored as 0: m / sqrt(v) could not be bounded in the next step.
//
// Every fp32 operation on the states is rounded by itself (the _rn intrinsics
// keep the compiler from contracting them), so that a state's code depends on
// the formula alone, not on how the kernel was compiled.  The division of the
// update is a product with an approximate reciprocal (one unit in the last
// place each): it reaches the parameter alone, scaled by lr.
#include <cuda_fp8.h>

#include <cmath>

#include "../../include/stk_b200.h"
#include "stk_host.h"
#include "stk_vec.cuh"

namespace stk {
namespace {

constexpr int kTensors = 48;        // per launch: the table stays below the 4 KB of kernel parameters
constexpr int kThreads = 256;
constexpr int kBlock = 256;         // elements per scale, and per warp
constexpr int kChunk = 8 * kBlock;  // elements per CTA: a block per warp
constexpr float kTiny = 0x1p-100f;  // a block below this is stored as zeros
constexpr float kE4M3Min = 0x1p-9f;

struct Table {
  stk_adamw_tensor t[kTensors];
  int first[kTensors + 1];  // first chunk of each tensor
  int count;
};

struct Hyper {
  double lr, beta1, beta2, weight_decay;
  float b1, omb1, b2, omb2, eps;
  float decay, step_size, rbc2;  // of the host's lr and step; recomputed where the device holds either
  const float* lr_dev;
  const int64_t* step_dev;
  const float* grad_scale;
  int64_t step;
  int copy_dtype;  // -1: no copies
};

struct Scalars {
  float decay, step_size, rbc2, gscale;
};

__host__ __device__ inline void derive(double lr, double wd, double b1, double b2, double t, float* decay,
                                       float* step_size, float* rbc2) {
  *decay = (float)(1.0 - lr * wd);
  *step_size = (float)(lr / (1.0 - pow(b1, t)));
  *rbc2 = (float)(1.0 / sqrt(1.0 - pow(b2, t)));
}

__device__ __forceinline__ float approx_rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// (Step by step over the eight elements: one loop over all of it took 702 instead
// of 675 us for 65536 x 2048 with 8-bit states, launches that follow an idle GPU;
// one after the other for seconds they take 745 us, 0.90 of a copy's bandwidth.)
__device__ __forceinline__ void update(const float (&g)[8], float (&p)[8], float (&m)[8], float (&v)[8], float (&root)[8],
                                       const Hyper& h, const Scalars& s) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = __fmul_rn(g[j], s.gscale);
    m[j] = __fadd_rn(__fmul_rn(m[j], h.b1), __fmul_rn(x, h.omb1));
    v[j] = __fadd_rn(__fmul_rn(v[j], h.b2), __fmul_rn(__fmul_rn(x, x), h.omb2));
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) root[j] = __fsqrt_rn(v[j]);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    // (A denominator is 0, or at least the smaller of eps >= 2^-126 and the least root, 2^-75; it is below 2^126, as the
    // root is at most 2^64, rbc2 below 2^27 and eps at most 2^125: neither it nor its reciprocal is flushed.)
    const float size = __fmul_rn(m[j], approx_rcp(__fadd_rn(__fmul_rn(root[j], s.rbc2), h.eps)));
    p[j] = __fsub_rn(__fmul_rn(p[j], s.decay), __fmul_rn(size, s.step_size));
  }
}

// Largest finite magnitude of a warp's 8 x 32 values.  That an infinity or a
// NaN is among them is rare: they are left out in a second look (fmaxf passes
// over a NaN by itself).
__device__ __forceinline__ float block_top(const float (&x)[8]) {
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[j]));
  uint32_t t = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
  if (t >= 0x7f800000u) {
    top = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[j]) < INFINITY ? fabsf(x[j]) : 0.f);
    t = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
  }
  return __uint_as_float(t);
}

// Scale and multiplier of a block whose largest finite magnitude is `top`.
__device__ __forceinline__ void block_scale(float t, float* scale, float* mul) {
  const bool some = t >= kTiny;
  *scale = some ? __fdiv_rn(t, 448.f) : 1.f;
  *mul = some ? __fdiv_rn(448.f, t) : 0.f;
}

// x * 0 is 0 for finite x and NaN otherwise: infinities and NaN get the NaN code.
__device__ __forceinline__ float code_value(float x, float mul) { return __fmaf_rn(x, 0.f, __fmul_rn(x, mul)); }
// The same of a root, which is positive or 0: what is positive is not stored as
// 0.  (A positive root is at least 2^-75, so its block's `mul` is not 0.)
__device__ __forceinline__ float root_value(float x, float mul) {
  const float q = __fmul_rn(x, mul);
  return __fmaf_rn(x, 0.f, x > 0.f ? fmaxf(q, kE4M3Min) : q);
}

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float2 from_e4m3x2(uint32_t u) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)u, __NV_E4M3);
  return __half22float2(__half2(h));
}

__device__ __forceinline__ void store_copy(void* copy, int dtype, int64_t i, float v) {
  if (dtype == STK_BF16) static_cast<__nv_bfloat16*>(copy)[i] = __float2bfloat16_rn(v);
  if (dtype == STK_F16) static_cast<__half*>(copy)[i] = __float2half_rn(v);
  if (dtype == STK_F32) static_cast<float*>(copy)[i] = v;
}
__device__ __forceinline__ void store_copy8(void* copy, int dtype, int64_t i, const float (&v)[8]) {
  if (dtype == STK_BF16) store8(static_cast<__nv_bfloat16*>(copy) + i, v);
  if (dtype == STK_F16) store8(static_cast<__half*>(copy) + i, v);
  if (dtype == STK_F32) store8(static_cast<float*>(copy) + i, v);
}

// 256 elements from `base`, all in range and aligned to eight: lane l has the
// eight from base + 8 l on.
template <typename P, typename G, bool EIGHT>
__device__ __forceinline__ void whole_block(const stk_adamw_tensor& t, int64_t base, int lane, const Hyper& h,
                                            const Scalars& s) {
  const int64_t i = base + lane * 8;
  P* const pp = static_cast<P*>(t.param) + i;
  float p[8], g[8], m[8], v[8], root[8];
  load8(pp, p);
  load8(static_cast<const G*>(t.grad) + i, g);
  if constexpr (EIGHT) {
    uint8_t* const mp = static_cast<uint8_t*>(t.exp_avg) + i;
    uint8_t* const vp = static_cast<uint8_t*>(t.exp_avg_sq) + i;
    const uint2 mq = *reinterpret_cast<const uint2*>(mp), vq = *reinterpret_cast<const uint2*>(vp);
    const float ms = t.exp_avg_scale[base / kBlock], vs = t.exp_avg_sq_scale[base / kBlock];
    const uint32_t mw[2] = {mq.x, mq.y}, vw[2] = {vq.x, vq.y};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 a = from_e4m3x2((mw[j >> 1] >> (16 * (j & 1))) & 0xffffu);
      const float2 r = from_e4m3x2((vw[j >> 1] >> (16 * (j & 1))) & 0xffffu);
      m[2 * j] = __fmul_rn(a.x, ms);
      m[2 * j + 1] = __fmul_rn(a.y, ms);
      const float r0 = __fmul_rn(r.x, vs), r1 = __fmul_rn(r.y, vs);
      v[2 * j] = __fmul_rn(r0, r0);
      v[2 * j + 1] = __fmul_rn(r1, r1);
    }
    update(g, p, m, v, root, h, s);
    float mscale, mmul, vscale, vmul;
    block_scale(block_top(m), &mscale, &mmul);
    block_scale(block_top(root), &vscale, &vmul);
    uint32_t mo[2] = {0, 0}, vo[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      mo[j >> 1] |= e4m3x2(code_value(m[2 * j], mmul), code_value(m[2 * j + 1], mmul)) << (16 * (j & 1));
      vo[j >> 1] |= e4m3x2(root_value(root[2 * j], vmul), root_value(root[2 * j + 1], vmul)) << (16 * (j & 1));
    }
    *reinterpret_cast<uint2*>(mp) = make_uint2(mo[0], mo[1]);
    *reinterpret_cast<uint2*>(vp) = make_uint2(vo[0], vo[1]);
    if (lane == 0) {
      t.exp_avg_scale[base / kBlock] = mscale;
      t.exp_avg_sq_scale[base / kBlock] = vscale;
    }
  } else {
    float* const mp = static_cast<float*>(t.exp_avg) + i;
    float* const vp = static_cast<float*>(t.exp_avg_sq) + i;
    load8(mp, m);
    load8(vp, v);
    update(g, p, m, v, root, h, s);
    store8(mp, m);
    store8(vp, v);
  }
  store8(pp, p);
  if (h.copy_dtype >= 0) store_copy8(t.copy, h.copy_dtype, i, p);
}

// The same for a block that ends early or whose tensors are not aligned so: lane l has elements base + l + 32 j, one access each.
template <typename P, typename G, bool EIGHT>
__device__ __forceinline__ void ragged_block(const stk_adamw_tensor& t, int64_t base, int lane, const Hyper& h,
                                             const Scalars& s) {
  P* const pp = static_cast<P*>(t.param) + base + lane;
  const G* const gp = static_cast<const G*>(t.grad) + base + lane;
  const int n = (int)(t.n - base < kBlock ? t.n - base : kBlock) - lane;
  float p[8], g[8], m[8], v[8], root[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {  // all loads before the first store
    p[j] = g[j] = 0.f;
    if (32 * j < n) {
      p[j] = as_f32(pp[32 * j]);
      g[j] = as_f32(gp[32 * j]);
    }
  }
  if constexpr (EIGHT) {
    uint8_t* const mp = static_cast<uint8_t*>(t.exp_avg) + base + lane;
    uint8_t* const vp = static_cast<uint8_t*>(t.exp_avg_sq) + base + lane;
    uint32_t mq[8], vq[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      mq[j] = 32 * j < n ? mp[32 * j] : 0u;
      vq[j] = 32 * j < n ? vp[32 * j] : 0u;
    }
    const float ms = t.exp_avg_scale[base / kBlock], vs = t.exp_avg_sq_scale[base / kBlock];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m[j] = __fmul_rn(from_e4m3x2(mq[j]).x, ms);
      const float r = __fmul_rn(from_e4m3x2(vq[j]).x, vs);
      v[j] = __fmul_rn(r, r);
    }
    update(g, p, m, v, root, h, s);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (32 * j >= n) m[j] = root[j] = 0.f;  // past the end (a scale may be NaN)
    float mscale, mmul, vscale, vmul;
    block_scale(block_top(m), &mscale, &mmul);
    block_scale(block_top(root), &vscale, &vmul);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (32 * j < n) {
        mp[32 * j] = (uint8_t)e4m3x2(code_value(m[j], mmul), 0.f);
        vp[32 * j] = (uint8_t)e4m3x2(root_value(root[j], vmul), 0.f);
      }
    if (lane == 0) {
      t.exp_avg_scale[base / kBlock] = mscale;
      t.exp_avg_sq_scale[base / kBlock] = vscale;
    }
  } else {
    float* const mp = static_cast<float*>(t.exp_avg) + base + lane;
    float* const vp = static_cast<float*>(t.exp_avg_sq) + base + lane;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m[j] = 32 * j < n ? mp[32 * j] : 0.f;
      v[j] = 32 * j < n ? vp[32 * j] : 0.f;
    }
    update(g, p, m, v, root, h, s);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (32 * j < n) {
        mp[32 * j] = m[j];
        vp[32 * j] = v[j];
      }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (32 * j < n) {
      pp[32 * j] = from_f32<P>(p[j]);
      if (h.copy_dtype >= 0) store_copy(t.copy, h.copy_dtype, base + lane + 32 * j, p[j]);
    }
}

// One CTA per 2048 elements and no loop: against CTAs that stay and walk over
// 8192 at a time, the same accesses run at 6.8 instead of 4.7 TB/s (the memory
// alone, 8-bit states).
template <typename P, typename G, bool EIGHT>
__global__ void __launch_bounds__(kThreads, 5) adamw_kernel(const __grid_constant__ Table tab,
                                                            const __grid_constant__ Hyper h) {
  Scalars s = {h.decay, h.step_size, h.rbc2, 1.f};
  if (h.grad_scale != nullptr) s.gscale = *h.grad_scale;
  // (By one thread of each CTA, before its loads: 65536 x 2048 with 8-bit states and no copies takes 612 to 632 us with
  // the host's values and 829 to 861 with the device's, with 32-bit states 1024 to 1078 and 1145 to 1160.)
  if (h.lr_dev != nullptr || h.step_dev != nullptr) {
    __shared__ Scalars sh;
    if (threadIdx.x == 0)
      derive(h.lr_dev != nullptr ? (double)*h.lr_dev : h.lr, h.weight_decay, h.beta1, h.beta2,
             h.step_dev != nullptr ? (double)*h.step_dev : (double)h.step, &sh.decay, &sh.step_size, &sh.rbc2);
    __syncthreads();
    s.decay = sh.decay, s.step_size = sh.step_size, s.rbc2 = sh.rbc2;
  }
  const int lane = threadIdx.x & 31, c = blockIdx.x;
  int lo = 0, hi = tab.count - 1;  // the last tensor whose first chunk is <= c
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.first[mid] <= c) lo = mid;
    else hi = mid - 1;
  }
  const stk_adamw_tensor& t = tab.t[lo];
  const int64_t base = (int64_t)(c - tab.first[lo]) * kChunk + (threadIdx.x >> 5) * kBlock;
  if (base >= t.n) return;
  const bool aligned = vec_aligned<P>(t.param) && vec_aligned<G>(t.grad) && vec_aligned<float>(t.copy) &&
                       (EIGHT ? vec_aligned<uint8_t>(t.exp_avg) && vec_aligned<uint8_t>(t.exp_avg_sq)
                              : vec_aligned<float>(t.exp_avg) && vec_aligned<float>(t.exp_avg_sq));
  if (aligned && base + kBlock <= t.n)
    whole_block<P, G, EIGHT>(t, base, lane, h, s);
  else
    ragged_block<P, G, EIGHT>(t, base, lane, h, s);
}

template <typename P, typename G>
cudaError_t launch(const Table& tab, const Hyper& h, int bits, cudaStream_t stream) {
  const int grid = tab.first[tab.count];
  if (bits == 8)
    adamw_kernel<P, G, true><<<grid, kThreads, 0, stream>>>(tab, h);
  else
    adamw_kernel<P, G, false><<<grid, kThreads, 0, stream>>>(tab, h);
  return cudaGetLastError();
}

template <typename P>
cudaError_t launch_grad(const Table& tab, const Hyper& h, int gdtype, int bits, cudaStream_t stream) {
  if (gdtype == STK_F32) return launch<P, float>(tab, h, bits, stream);
  if (gdtype == STK_F16) return launch<P, __half>(tab, h, bits, stream);
  return launch<P, __nv_bfloat16>(tab, h, bits, stream);
}

bool float_dtype(int t) { return t == STK_F32 || t == STK_F16 || t == STK_BF16; }
size_t size_of(int t) { return t == STK_F32 ? 4 : 2; }

}  // namespace
}  // namespace stk

extern "C" int stk_adamw_step(const stk_adamw_tensor* tensors, int64_t count, int param_dtype, int grad_dtype,
                              int copy_dtype, int state_bits, const stk_adamw_args* args, void* stream) {
  STK_ENTRY_BEGIN
  using namespace stk;
  if (!float_dtype(param_dtype) || !float_dtype(grad_dtype) || (copy_dtype >= 0 && !float_dtype(copy_dtype)))
    return host_fail(STK_EINVAL, "stk_adamw_step: params, grads and copies must be fp32, fp16 or bf16");
  if (state_bits != 8 && state_bits != 32) return host_fail(STK_EINVAL, "stk_adamw_step: state_bits must be 8 or 32");
  if (count < 0 || !args || (count > 0 && !tensors))
    return host_fail(STK_EINVAL, "stk_adamw_step: need args and `count` tensors");
  // Negated comparisons, so that a NaN is refused too.
  if (!(args->beta1 >= 0 && args->beta1 < 1) || !(args->beta2 >= 0 && args->beta2 < 1))
    return host_fail(STK_EINVAL, "stk_adamw_step: betas must be in [0, 1)");
  if (!(args->eps >= 0 && args->eps <= 0x1p125) || (args->eps > 0 && args->eps < 0x1p-126))
    return host_fail(STK_EINVAL, "stk_adamw_step: eps must be 0 or from 2^-126 to 2^125");
  if (!args->lr_dev && !(args->lr >= 0)) return host_fail(STK_EINVAL, "stk_adamw_step: lr must be >= 0");
  if (!(args->weight_decay >= 0)) return host_fail(STK_EINVAL, "stk_adamw_step: weight_decay must be >= 0");
  if (!args->step_dev && args->step < 1) return host_fail(STK_EINVAL, "stk_adamw_step: step must be >= 1");
  const size_t state_size = state_bits == 8 ? 1 : 4;
  for (int64_t i = 0; i < count; ++i) {
    const stk_adamw_tensor& t = tensors[i];
    if (t.n < 0 || t.n > ((int64_t)1 << 41)) return host_fail(STK_EINVAL, "stk_adamw_step: tensor size out of range");
    if (t.n == 0) continue;
    if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq || (copy_dtype >= 0 && !t.copy) ||
        (state_bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale)))
      return host_fail(STK_EINVAL, "stk_adamw_step: null tensor pointer");
    if (!aligned_to(t.param, size_of(param_dtype)) || !aligned_to(t.grad, size_of(grad_dtype)) ||
        !aligned_to(t.exp_avg, state_size) || !aligned_to(t.exp_avg_sq, state_size) ||
        (copy_dtype >= 0 && !aligned_to(t.copy, size_of(copy_dtype))) ||
        (state_bits == 8 && (!aligned_to(t.exp_avg_scale, 4) || !aligned_to(t.exp_avg_sq_scale, 4))))
      return host_fail(STK_EINVAL, "stk_adamw_step: pointer not aligned to its element");
  }
  Hyper h = {};
  h.lr = args->lr;
  h.beta1 = args->beta1;
  h.beta2 = args->beta2;
  h.weight_decay = args->weight_decay;
  h.b1 = (float)args->beta1;
  h.omb1 = (float)(1.0 - args->beta1);
  h.b2 = (float)args->beta2;
  h.omb2 = (float)(1.0 - args->beta2);
  h.eps = (float)args->eps;
  h.lr_dev = args->lr_dev;
  h.step_dev = args->step_dev;
  h.grad_scale = args->grad_scale;
  h.step = args->step;
  h.copy_dtype = copy_dtype;
  if (!h.lr_dev && !h.step_dev)
    derive(h.lr, h.weight_decay, h.beta1, h.beta2, (double)h.step, &h.decay, &h.step_size, &h.rbc2);
  Table tab;
  tab.count = 0;
  int64_t chunks = 0;
  for (int64_t i = 0; i <= count; ++i) {
    const int64_t nc = i < count ? (tensors[i].n + kChunk - 1) / kChunk : 0;
    if (tab.count > 0 && (i == count || tab.count == kTensors || chunks + nc > 0x7fffffff)) {
      tab.first[tab.count] = (int)chunks;
      const cudaStream_t s = static_cast<cudaStream_t>(stream);
      const cudaError_t e = param_dtype == STK_F32   ? launch_grad<float>(tab, h, grad_dtype, state_bits, s)
                            : param_dtype == STK_F16 ? launch_grad<__half>(tab, h, grad_dtype, state_bits, s)
                                                     : launch_grad<__nv_bfloat16>(tab, h, grad_dtype, state_bits, s);
      if (e != cudaSuccess) return host_cuda_fail(e, "adamw_kernel launch");
      tab.count = 0;
      chunks = 0;
    }
    if (i == count || nc == 0) continue;
    tab.t[tab.count] = tensors[i];
    if (copy_dtype < 0) tab.t[tab.count].copy = nullptr;
    tab.first[tab.count++] = (int)chunks;
    chunks += nc;
  }
  return STK_OK;
  STK_ENTRY_END
}
