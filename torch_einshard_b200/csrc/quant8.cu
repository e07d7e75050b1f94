// Activations kept for backward in 8 bits.
//
// A row is cut into blocks of 32 channels that share a power of two:
//   e = floor(log2 amax) - 6, one more if rint(amax 2^-e) would be 128;  q = rint(x 2^-e) in -127 .. 127
//   x^ = q 2^e, at most half a step 2^(e-1) from x
// Products with a power of two are exact, so every machine rounds the same way
// and a stored code never depends on how a division rounds.  The exponent is
// kept as e + 127 in a byte (the smallest e is -126; smaller steps would be
// subnormal).  A block that holds an infinity or a NaN gets exponent byte 255
// and reads back as NaN: a diverged activation stays visible in the gradients.
//
// silu(x) = x s, silu'(x) = s (1 + x (1 - s)), s = 1 / (1 + e^-x); the
// pre-activation kept here serves both the gradient of the activation and the
// activation's value in the next product's weight gradient.
//
// All kernels are bound by memory: 3 + 1/32 bytes a 16-bit element to write the
// codes, the same to read them back.  Eight elements a thread (one 16-byte
// access of a 16-bit type), four lanes a block, so the block's maximum is two
// shuffles; rows whose start is not 16-byte aligned take one element a lane,
// one block a warp.
#include "quant8.h"

#include "gemm.h"
#include "quant8.cuh"

namespace es {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;

template <typename T>
struct Limit;
template <>
struct Limit<float> {
  static constexpr float value = 3.402823466e38f;
};
template <>
struct Limit<__nv_bfloat16> {
  static constexpr float value = 3.389531389e38f;
};
template <>
struct Limit<__half> {
  static constexpr float value = 65504.0f;
};

// A code's value; next to the type's largest value it may round past it: clamped, still within half a step.
template <typename T>
__device__ __forceinline__ float value_of(float code, float scale) {
  const float v = code * scale;
  return v > Limit<T>::value ? Limit<T>::value : (v < -Limit<T>::value ? -Limit<T>::value : v);  // NaN stays
}

// Two values through kMode.
template <typename T, int kMode>
__device__ __forceinline__ void restored2(float& x1, float& x2, float g1, float g2) {
  if (kMode == kRestoreValue) return;
  float s1, s2;
  if constexpr (sizeof(T) == 4) {
    s1 = 1.0f / (1.0f + expf(-x1));
    s2 = 1.0f / (1.0f + expf(-x2));
  } else {
    sigmoid_pair(x1, x2, s1, s2);
  }
  if (kMode == kRestoreSilu) {
    x1 *= s1;
    x2 *= s2;
  } else {
    x1 = g1 * silu_slope(x1, s1);
    x2 = g2 * silu_slope(x2, s2);
  }
}

template <typename T, int kMode>
__device__ __forceinline__ float decoded(float code, float scale) {
  return kMode == kRestoreValue ? value_of<T>(code, scale) : value_of<float>(code, scale);  // pre-activations: 32 bits
}

// Work of a warp in the vector kernels: kUnroll groups of 32 chunks of eight
// elements.  kFlat (d a multiple of 32): chunks run through the whole tensor;
// otherwise a row is padded to whole blocks and a warp stays inside one row.
struct Place {
  long long elem;   // first element of this lane's chunk, or -1
  long long block;  // its block
};

template <bool kFlat>
struct Walk {
  long long units;  // warp units
  long long per_row, d, nb, total;
  __device__ __forceinline__ Walk(long long rows, long long d_) : d(d_) {
    nb = (d + kQuantBlock - 1) / kQuantBlock;
    total = rows * nb * 4;
    per_row = (nb * 4 + 32 * kUnroll - 1) / (32 * kUnroll);
    units = kFlat ? (total + 32 * kUnroll - 1) / (32 * kUnroll) : rows * per_row;
  }
  __device__ __forceinline__ Place at(long long unit, int u, int lane) const {
    if (kFlat) {
      const long long c = (unit * kUnroll + u) * 32 + lane;
      return {c < total ? c * 8 : -1, c >> 2};
    }
    const long long row = unit / per_row;
    const long long c = ((unit - row * per_row) * kUnroll + u) * 32 + lane;
    return {c * 8 < d ? row * d + c * 8 : -1, c < nb * 4 ? row * nb + (c >> 2) : -1};
  }
};

template <typename T, typename OutT, bool kSilu, bool kFlat>
__global__ void __launch_bounds__(kThreads) quant8_kernel(const T* __restrict__ x, OutT* __restrict__ out,
                                                          int8_t* __restrict__ codes, uint8_t* __restrict__ exps,
                                                          long long rows, long long d) {
  const int lane = threadIdx.x & 31;
  const long long warp = (static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const long long warps = (static_cast<long long>(gridDim.x) * kThreads) >> 5;
  const Walk<kFlat> walk(rows, d);
  for (long long unit = warp; unit < walk.units; unit += warps) {
    Raw8<T> raw[kUnroll];
    Place pl[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      pl[u] = walk.at(unit, u, lane);
      if (pl[u].elem >= 0) raw[u] = load8_stream(x + pl[u].elem);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float f[8];
      uint32_t m = 0;
      if (pl[u].elem >= 0) {
        unpack8(raw[u], f);
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
      }
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
      if (pl[u].elem < 0) continue;
      const Step8 s = step8_of(m);
      *reinterpret_cast<uint2*>(codes + pl[u].elem) =
          make_uint2(codes8_of(f[0], f[1], f[2], f[3], s), codes8_of(f[4], f[5], f[6], f[7], s));
      if ((lane & 3) == 0) exps[pl[u].block] = static_cast<uint8_t>(s.byte);
      if (kSilu) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) restored2<OutT, kRestoreSilu>(f[i], f[i + 1], 0.0f, 0.0f);
        store8(out + pl[u].elem, f);
      }
    }
  }
}

// Any width and alignment: one block a warp, one element a lane.
template <typename T, typename OutT, bool kSilu>
__global__ void __launch_bounds__(kThreads) quant8_any_kernel(const T* __restrict__ x, OutT* __restrict__ out,
                                                              int8_t* __restrict__ codes,
                                                              uint8_t* __restrict__ exps, long long rows,
                                                              long long d) {
  const int lane = threadIdx.x & 31;
  const long long warp = (static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const long long warps = (static_cast<long long>(gridDim.x) * kThreads) >> 5;
  const long long nb = (d + kQuantBlock - 1) / kQuantBlock;
  const long long per_row = (nb + kUnroll - 1) / kUnroll;
  for (long long unit = warp; unit < rows * per_row; unit += warps) {
    const long long row = unit / per_row;
    const long long b0 = (unit - row * per_row) * kUnroll;
    float f[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const long long c = (b0 + u) * kQuantBlock + lane;
      f[u] = c < d ? to_float<T>(x[row * d + c]) : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(f[u]) & 0x7fffffffu);
      const long long c = (b0 + u) * kQuantBlock + lane;
      if (b0 + u >= nb) break;  // uniform
      const Step8 s = step8_of(m);
      if (c < d) {
        codes[row * d + c] = static_cast<int8_t>(codes8_of(f[u], 0.0f, 0.0f, 0.0f, s));
        if (kSilu) {
          float none = 0.0f;
          restored2<OutT, kRestoreSilu>(f[u], none, 0.0f, 0.0f);
          out[row * d + c] = from_float<OutT>(f[u]);
        }
      }
      if (lane == 0) exps[row * nb + b0 + u] = static_cast<uint8_t>(s.byte);
    }
  }
}

template <typename T, int kMode, bool kFlat>
__global__ void __launch_bounds__(kThreads) restore8_kernel(const int8_t* __restrict__ codes,
                                                            const uint8_t* __restrict__ exps,
                                                            const T* __restrict__ grad, T* __restrict__ out,
                                                            long long rows, long long d) {
  const int lane = threadIdx.x & 31;
  const long long warp = (static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const long long warps = (static_cast<long long>(gridDim.x) * kThreads) >> 5;
  const Walk<kFlat> walk(rows, d);
  for (long long unit = warp; unit < walk.units; unit += warps) {
    uint2 q[kUnroll];
    float scale[kUnroll];
    Raw8<T> g[kUnroll];
    Place pl[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      pl[u] = walk.at(unit, u, lane);
      if (pl[u].elem < 0) continue;
      q[u] = __ldcs(reinterpret_cast<const uint2*>(codes + pl[u].elem));
      scale[u] = scale8_of(exps[pl[u].block]);
      if (kMode == kRestoreSiluGrad) g[u] = load8_stream(grad + pl[u].elem);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (pl[u].elem < 0) continue;
      float f[8], gf[8];
      if (kMode == kRestoreSiluGrad) unpack8(g[u], gf);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (kMode != kRestoreSiluGrad) gf[i] = 0.0f;
        f[i] = decoded<T, kMode>(code8_at(i < 4 ? q[u].x : q[u].y, i & 3), scale[u]);
      }
#pragma unroll
      for (int i = 0; i < 8; i += 2) restored2<T, kMode>(f[i], f[i + 1], gf[i], gf[i + 1]);
      store8(out + pl[u].elem, f);
    }
  }
}

template <typename T, int kMode>
__global__ void __launch_bounds__(kThreads) restore8_any_kernel(const int8_t* __restrict__ codes,
                                                                const uint8_t* __restrict__ exps,
                                                                const T* __restrict__ grad, T* __restrict__ out,
                                                                long long rows, long long d) {
  const int lane = threadIdx.x & 31;
  const long long warp = (static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const long long warps = (static_cast<long long>(gridDim.x) * kThreads) >> 5;
  const long long nb = (d + kQuantBlock - 1) / kQuantBlock;
  const long long per_row = (nb + kUnroll - 1) / kUnroll;
  for (long long unit = warp; unit < rows * per_row; unit += warps) {
    const long long row = unit / per_row;
    const long long b0 = (unit - row * per_row) * kUnroll;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const long long c = (b0 + u) * kQuantBlock + lane;
      if (c >= d) break;
      const float scale = scale8_of(exps[row * nb + b0 + u]);
      const float g = kMode == kRestoreSiluGrad ? to_float<T>(grad[row * d + c]) : 0.0f;
      float x = decoded<T, kMode>(static_cast<float>(codes[row * d + c]), scale), none = 0.0f;
      restored2<T, kMode>(x, none, g, 0.0f);
      out[row * d + c] = from_float<T>(x);
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Enough warps for every unit, at most eight blocks of 256 threads an SM.
int grid_for(long long units, int sms) {
  const long long want = (units + kThreads / 32 - 1) / (kThreads / 32);
  const long long cap = static_cast<long long>(sms) * 8;
  return static_cast<int>(want < 1 ? 1 : (want > cap ? cap : want));
}

long long vector_units(long long rows, long long d) {
  const long long nb = (d + kQuantBlock - 1) / kQuantBlock;
  if (d % kQuantBlock == 0) return (rows * nb * 4 + 32 * kUnroll - 1) / (32 * kUnroll);
  return rows * ((nb * 4 + 32 * kUnroll - 1) / (32 * kUnroll));
}

long long any_units(long long rows, long long d) {
  const long long nb = (d + kQuantBlock - 1) / kQuantBlock;
  return rows * ((nb + kUnroll - 1) / kUnroll);
}

template <typename T, typename OutT, bool kSilu>
int launch_quant(const T* x, OutT* out, int8_t* codes, uint8_t* exps, long long rows, long long d, int sms,
                 cudaStream_t stream) {
  if (rows <= 0 || d <= 0) return 0;
  const bool vec = d % 8 == 0 && aligned16(x) && aligned16(codes) && (!kSilu || aligned16(out));
  if (!vec)
    quant8_any_kernel<T, OutT, kSilu>
        <<<grid_for(any_units(rows, d), sms), kThreads, 0, stream>>>(x, out, codes, exps, rows, d);
  else if (d % kQuantBlock == 0)
    quant8_kernel<T, OutT, kSilu, true>
        <<<grid_for(vector_units(rows, d), sms), kThreads, 0, stream>>>(x, out, codes, exps, rows, d);
  else
    quant8_kernel<T, OutT, kSilu, false>
        <<<grid_for(vector_units(rows, d), sms), kThreads, 0, stream>>>(x, out, codes, exps, rows, d);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int kMode>
int launch_restore(const int8_t* codes, const uint8_t* exps, const T* grad, T* out, long long rows, long long d,
                   int sms, cudaStream_t stream) {
  if (rows <= 0 || d <= 0) return 0;
  const bool vec =
      d % 8 == 0 && aligned16(out) && aligned16(codes) && (kMode != kRestoreSiluGrad || aligned16(grad));
  if (!vec)
    restore8_any_kernel<T, kMode>
        <<<grid_for(any_units(rows, d), sms), kThreads, 0, stream>>>(codes, exps, grad, out, rows, d);
  else if (d % kQuantBlock == 0)
    restore8_kernel<T, kMode, true>
        <<<grid_for(vector_units(rows, d), sms), kThreads, 0, stream>>>(codes, exps, grad, out, rows, d);
  else
    restore8_kernel<T, kMode, false>
        <<<grid_for(vector_units(rows, d), sms), kThreads, 0, stream>>>(codes, exps, grad, out, rows, d);
  return static_cast<int>(cudaGetLastError());
}

template <typename T>
int restore_mode(const int8_t* codes, const uint8_t* exps, const void* grad, void* out, int mode, long long rows,
                 long long d, int sms, cudaStream_t stream) {
  const T* g = static_cast<const T*>(grad);
  T* o = static_cast<T*>(out);
  switch (mode) {
    case kRestoreValue:
      return launch_restore<T, kRestoreValue>(codes, exps, g, o, rows, d, sms, stream);
    case kRestoreSilu:
      return launch_restore<T, kRestoreSilu>(codes, exps, g, o, rows, d, sms, stream);
    case kRestoreSiluGrad:
      return launch_restore<T, kRestoreSiluGrad>(codes, exps, g, o, rows, d, sms, stream);
    default:
      return static_cast<int>(cudaErrorInvalidValue);
  }
}

}  // namespace

int quant8(const void* x, int dtype, int8_t* codes, uint8_t* exps, long long rows, long long d, int sms,
           cudaStream_t stream) {
  switch (dtype) {
    case kDtypeBF16:
      return launch_quant<__nv_bfloat16, __nv_bfloat16, false>(static_cast<const __nv_bfloat16*>(x), nullptr, codes,
                                                               exps, rows, d, sms, stream);
    case kDtypeF16:
      return launch_quant<__half, __half, false>(static_cast<const __half*>(x), nullptr, codes, exps, rows, d, sms,
                                                 stream);
    case kDtypeF32:
      return launch_quant<float, float, false>(static_cast<const float*>(x), nullptr, codes, exps, rows, d, sms,
                                               stream);
    default:
      return static_cast<int>(cudaErrorInvalidValue);
  }
}

int quant8_silu(const float* h, void* out, int out_dtype, int8_t* codes, uint8_t* exps, long long rows, long long d,
                int sms, cudaStream_t stream) {
  switch (out_dtype) {
    case kDtypeBF16:
      return launch_quant<float, __nv_bfloat16, true>(h, static_cast<__nv_bfloat16*>(out), codes, exps, rows, d, sms,
                                                      stream);
    case kDtypeF16:
      return launch_quant<float, __half, true>(h, static_cast<__half*>(out), codes, exps, rows, d, sms, stream);
    case kDtypeF32:
      return launch_quant<float, float, true>(h, static_cast<float*>(out), codes, exps, rows, d, sms, stream);
    default:
      return static_cast<int>(cudaErrorInvalidValue);
  }
}

int restore8(const int8_t* codes, const uint8_t* exps, const void* grad, void* out, int dtype, int mode,
             long long rows, long long d, int sms, cudaStream_t stream) {
  switch (dtype) {
    case kDtypeBF16:
      return restore_mode<__nv_bfloat16>(codes, exps, grad, out, mode, rows, d, sms, stream);
    case kDtypeF16:
      return restore_mode<__half>(codes, exps, grad, out, mode, rows, d, sms, stream);
    case kDtypeF32:
      return restore_mode<float>(codes, exps, grad, out, mode, rows, d, sms, stream);
    default:
      return static_cast<int>(cudaErrorInvalidValue);
  }
}

}  // namespace es
