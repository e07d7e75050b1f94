// Element access of the elementwise and row kernels: eight consecutive elements
// of a bf16, fp16 or fp32 tensor as fp32 registers, with 16-byte accesses, and
// warp reductions.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace es {

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// Raw 16-byte words of eight elements: one for 16-bit types, two for fp32.
template <typename T>
struct Raw8 {
  uint4 w[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}

// Read once: keep it out of L1.
template <typename T>
__device__ __forceinline__ Raw8<T> load8_stream(const T* p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.w[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  return r;
}

template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float (&f)[8]) {
  const T* e = reinterpret_cast<const T*>(r.w);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = to_float<T>(e[i]);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  Raw8<T> r;
  T* e = reinterpret_cast<T*>(r.w);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = from_float<T>(f[i]);
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = r.w[i];
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

}  // namespace es
