// Eight consecutive elements of fp32 / fp16 / bf16 as fp32 registers: one
// 16-byte access for the 16-bit types, two for fp32.  Aligned to eight elements:
// vec_aligned.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <cstring>

namespace stk {

// Two fp32 values in one 64-bit register, for the packed operations (each half
// rounded as the scalar operation rounds it).
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 halves(uint64_t p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

template <typename T>
__host__ __device__ __forceinline__ bool vec_aligned(const void* p) {
  return (reinterpret_cast<uintptr_t>(p) & (8 * sizeof(T) - 1)) == 0;
}

template <typename T>
__device__ __forceinline__ float as_f32(T v);
template <>
__device__ __forceinline__ float as_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float as_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float as_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& u, float (&w)[8]);
template <>
__device__ __forceinline__ void unpack8<__nv_bfloat16>(const uint4& u, float (&w)[8]) {
  const uint32_t q[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[2 * i] = __uint_as_float(q[i] << 16);
    w[2 * i + 1] = __uint_as_float(q[i] & 0xffff0000u);
  }
}
template <>
__device__ __forceinline__ void unpack8<__half>(const uint4& u, float (&w)[8]) {
  const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    w[2 * i] = f.x;
    w[2 * i + 1] = f.y;
  }
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&w)[8]) {
  unpack8<T>(*reinterpret_cast<const uint4*>(p), w);
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&w)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], c = reinterpret_cast<const float4*>(p)[1];
  w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
  w[4] = c.x; w[5] = c.y; w[6] = c.z; w[7] = c.w;
}

// The same for memory that no thread writes during the kernel (non-coherent
// loads, which the compiler may move across stores), fp32 in one access of 32
// bytes: two of 16 each touch every sector that the warp reads, which doubles
// the L1's work where rows are gathered from the L2 (the SAE gradient's kernel:
// 434 to 403 us).  Stores are of 16 bytes: an attempt with 32 wrote only some of
// the values in one place, and its cause was not found.
template <typename T>
__device__ __forceinline__ void ldg8(const T* p, float (&w)[8]) {
  unpack8<T>(__ldg(reinterpret_cast<const uint4*>(p)), w);
}
template <>
__device__ __forceinline__ void ldg8<float>(const float* p, float (&w)[8]) {
  asm("ld.global.nc.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=f"(w[0]), "=f"(w[1]), "=f"(w[2]), "=f"(w[3]), "=f"(w[4]), "=f"(w[5]), "=f"(w[6]), "=f"(w[7])
      : "l"(p));
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&w)[8]) {
  T h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = from_f32<T>(w[i]);
  uint4 u;
  memcpy(&u, h, 16);
  *reinterpret_cast<uint4*>(p) = u;
}
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&w)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(w[0], w[1], w[2], w[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(w[4], w[5], w[6], w[7]);
}

// Streams, read or written once: marked to leave the caches first.
template <typename T>
__device__ __forceinline__ void ldcs8(const T* p, float (&w)[8]) {
  unpack8<T>(__ldcs(reinterpret_cast<const uint4*>(p)), w);
}
template <>
__device__ __forceinline__ void ldcs8<float>(const float* p, float (&w)[8]) {
  const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), c = __ldcs(reinterpret_cast<const float4*>(p) + 1);
  w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
  w[4] = c.x; w[5] = c.y; w[6] = c.z; w[7] = c.w;
}
template <typename T>
__device__ __forceinline__ void stcs8(T* p, const float (&w)[8]) {
  T h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = from_f32<T>(w[i]);
  uint4 u;
  memcpy(&u, h, 16);
  __stcs(reinterpret_cast<uint4*>(p), u);
}
template <>
__device__ __forceinline__ void stcs8<float>(float* p, const float (&w)[8]) {
  __stcs(reinterpret_cast<float4*>(p), make_float4(w[0], w[1], w[2], w[3]));
  __stcs(reinterpret_cast<float4*>(p) + 1, make_float4(w[4], w[5], w[6], w[7]));
}

}  // namespace stk
