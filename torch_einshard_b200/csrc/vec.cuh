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

// To be read again by this SM or another: kept in L2, out of L1.
template <typename T>
__device__ __forceinline__ Raw8<T> load8_l2(const T* p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.w[i] = __ldcg(reinterpret_cast<const uint4*>(p) + i);
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

// Two elements of a 16-bit type from one word, and back.
template <typename T>
__device__ __forceinline__ float2 word_to_floats(uint32_t w);
template <>
__device__ __forceinline__ float2 word_to_floats<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 word_to_floats<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t floats_to_word(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t floats_to_word<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t floats_to_word<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) {
    const uint32_t w[4] = {r.w[i].x, r.w[i].y, r.w[i].z, r.w[i].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (sizeof(T) == 4) {
        f[4 * i + k] = __uint_as_float(w[k]);
      } else {
        const float2 v = word_to_floats<T>(w[k]);
        f[2 * k] = v.x;
        f[2 * k + 1] = v.y;
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (sizeof(T) == 4)
        w[k] = __float_as_uint(f[4 * i + k]);
      else
        w[k] = floats_to_word<T>(f[2 * k], f[2 * k + 1]);
    }
    r.w[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = r.w[i];
}

// ------------------------------------------------------------------ packed fp32 pairs
// Two fp32 operations an instruction (sm_100's f32x2 forms).  A pair is kept as
// one 64-bit value, so that it stays in one aligned pair of registers.

using Pair = unsigned long long;

__device__ __forceinline__ Pair pair(float lo, float hi) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(lo), "f"(hi));
  return p;
}
__device__ __forceinline__ Pair pair(float v) { return pair(v, v); }
__device__ __forceinline__ float2 both(Pair p) {
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ float lo_of(Pair p) { return both(p).x; }
__device__ __forceinline__ float hi_of(Pair p) { return both(p).y; }

__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Eight elements as four pairs.
template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, Pair* f) {
  float v[8];
  unpack8(r, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = pair(v[2 * i], v[2 * i + 1]);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const Pair* f) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 e = both(f[i]);
    v[2 * i] = e.x;
    v[2 * i + 1] = e.y;
  }
  store8(p, v);
}

// ------------------------------------------------------------------ asynchronous copies

// 16 bytes to shared memory, past the registers; only the first `bytes` are read, the rest is zero.
__device__ __forceinline__ void copy16_async(void* shared, const void* global, int bytes = 16) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(shared))),
               "l"(global), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

}  // namespace es
