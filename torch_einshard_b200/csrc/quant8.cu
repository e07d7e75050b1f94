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
// shuffles.  Rows of any other width take aligned words through all rows;
// tensors whose own start is not aligned, and rows under eight elements, take
// one element a lane, one block a warp.
#include "quant8.h"

#include "gemm.h"
#include "quant8.cuh"

namespace es {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;
constexpr int kAnyUnroll = 16;

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
  return max_nan(min_nan(code * scale, Limit<T>::value), -Limit<T>::value);  // NaN stays
}

// Two values through kMode.
template <typename T, int kMode>
__device__ __forceinline__ void restored2(float& x1, float& x2, float g1, float g2) {
  if (kMode == kRestoreValue) return;
  if constexpr (sizeof(T) == 4) {
    const float s1 = 1.0f / (1.0f + expf(-x1)), s2 = 1.0f / (1.0f + expf(-x2));  // 1 from x = 17 on
    x1 = kMode == kRestoreSilu ? x1 * s1 : g1 * (s1 * fmaf(x1, 1.0f - s1, 1.0f));
    x2 = kMode == kRestoreSilu ? x2 * s2 : g2 * (s2 * fmaf(x2, 1.0f - s2, 1.0f));
  } else {
    float s1, s2, e1, e2;
    sigmoid_pair(x1, x2, s1, s2, e1, e2);
    x1 = kMode == kRestoreSilu ? x1 * s1 : g1 * silu_slope(x1, s1, e1);
    x2 = kMode == kRestoreSilu ? x2 * s2 : g2 * silu_slope(x2, s2, e2);
  }
}

template <typename T, int kMode>
__device__ __forceinline__ float decoded(float code, float scale) {
  return kMode == kRestoreValue ? value_of<T>(code, scale) : value_of<float>(code, scale);  // pre-activations: 32 bits
}

// Two values of different blocks, or not from codes: they share a reciprocal, and a NaN must not reach the other one.
template <typename T, int kMode>
__device__ __forceinline__ void restored_apart(float& x1, float& x2, float g1, float g2) {
  if (kMode == kRestoreValue) return;
  const bool bad1 = x1 != x1, bad2 = x2 != x2;
  if (bad1) x1 = 0.0f;
  if (bad2) x2 = 0.0f;
  restored2<T, kMode>(x1, x2, g1, g2);
  if (bad1) x1 = __uint_as_float(0x7fc00000u);
  if (bad2) x2 = __uint_as_float(0x7fc00000u);
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
        if (s.byte != kQuantNan) {
#pragma unroll
          for (int i = 0; i < 8; i += 2) restored2<OutT, kRestoreSilu>(f[i], f[i + 1], 0.0f, 0.0f);
        } else {  // the values themselves: a NaN is one value's
#pragma unroll
          for (int i = 0; i < 8; i += 2) restored_apart<OutT, kRestoreSilu>(f[i], f[i + 1], 0.0f, 0.0f);
        }
        store8(out + pl[u].elem, f);
      }
    }
  }
}

// Any width and alignment: one block a warp, one element a lane; a warp has
// kAnyUnroll blocks of a row in flight (64 bytes each of a 16-bit type).
template <typename T, typename OutT, bool kSilu>
__global__ void __launch_bounds__(kThreads) quant8_any_kernel(const T* __restrict__ x, OutT* __restrict__ out,
                                                              int8_t* __restrict__ codes,
                                                              uint8_t* __restrict__ exps, long long rows,
                                                              long long d) {
  const int lane = threadIdx.x & 31;
  const long long warp = (static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const long long warps = (static_cast<long long>(gridDim.x) * kThreads) >> 5;
  const long long nb = (d + kQuantBlock - 1) / kQuantBlock;
  const long long per_row = (nb + kAnyUnroll - 1) / kAnyUnroll;
  for (long long unit = warp; unit < rows * per_row; unit += warps) {
    const long long row = unit / per_row;
    const long long b0 = (unit - row * per_row) * kAnyUnroll;
    const long long c0 = b0 * kQuantBlock + lane;
    const int left = static_cast<int>(d - c0 < kAnyUnroll * kQuantBlock ? d - c0 : kAnyUnroll * kQuantBlock);
    const T* src = x + row * d + c0;
    float f[kAnyUnroll];
#pragma unroll
    for (int u = 0; u < kAnyUnroll; ++u) f[u] = u * kQuantBlock < left ? to_float<T>(src[u * kQuantBlock]) : 0.0f;
    int byte = 0;  // lane u: the exponent of block u
    int8_t* dst = codes + row * d + c0;
    OutT* act = kSilu ? out + row * d + c0 : nullptr;
#pragma unroll
    for (int u = 0; u < kAnyUnroll; ++u) {
      const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(f[u]) & 0x7fffffffu);
      const Step8 s = step8_of(m);
      if (lane == u) byte = s.byte;
      if (u * kQuantBlock < left) {
        dst[u * kQuantBlock] = static_cast<int8_t>(codes8_of(f[u], 0.0f, 0.0f, 0.0f, s));
        if (kSilu) {
          float none = 0.0f;
          restored2<OutT, kRestoreSilu>(f[u], none, 0.0f, 0.0f);
          act[u * kQuantBlock] = from_float<OutT>(f[u]);
        }
      }
    }
    if (lane < kAnyUnroll && b0 + lane < nb) exps[row * nb + b0 + lane] = static_cast<uint8_t>(byte);
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
  const long long per_row = (nb + kAnyUnroll - 1) / kAnyUnroll;
  for (long long unit = warp; unit < rows * per_row; unit += warps) {
    const long long row = unit / per_row;
    const long long b0 = (unit - row * per_row) * kAnyUnroll;
    const long long c0 = b0 * kQuantBlock + lane;
    const int left = static_cast<int>(d - c0 < kAnyUnroll * kQuantBlock ? d - c0 : kAnyUnroll * kQuantBlock);
    const long long at = row * d + c0;
    const int byte = lane < kAnyUnroll && b0 + lane < nb ? exps[row * nb + b0 + lane] : 127;
    int8_t q[kAnyUnroll];
    float g[kAnyUnroll];
#pragma unroll
    for (int u = 0; u < kAnyUnroll; ++u) {
      q[u] = u * kQuantBlock < left ? codes[at + u * kQuantBlock] : 0;
      g[u] = kMode == kRestoreSiluGrad && u * kQuantBlock < left ? to_float<T>(grad[at + u * kQuantBlock]) : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < kAnyUnroll; u += 2) {
      float x1 = decoded<T, kMode>(static_cast<float>(q[u]), scale8_of(__shfl_sync(0xffffffffu, byte, u)));
      float x2 = decoded<T, kMode>(static_cast<float>(q[u + 1]), scale8_of(__shfl_sync(0xffffffffu, byte, u + 1)));
      restored_apart<T, kMode>(x1, x2, g[u], g[u + 1]);
      if (u * kQuantBlock < left) out[at + u * kQuantBlock] = from_float<T>(x1);
      if ((u + 1) * kQuantBlock < left) out[at + (u + 1) * kQuantBlock] = from_float<T>(x2);
    }
  }
}

// ------------------------------------------------------------------ rows that start anywhere
//
// Where d is no multiple of eight, aligned words of eight elements run through
// the tensor regardless of its rows.  Format blocks are numbered through all
// rows, so a word (d >= 8) holds the end of one block, perhaps the start of the
// next, and behind a row's short last block one more: spans [0, p1), [p1, p2)
// and [p2, 8).  Quantising, the maxima of a tile's blocks are formed in shared
// memory (integer maxima: any order gives the same), and a tile reads 32
// elements more on both sides, for the blocks that it shares with its
// neighbours.  Against one element a lane (the kernels above), fp16: 24004 rows of
// 8191 quantised in 208 us instead of 314, restored in 152 instead of 207;
// 3000000 rows of 65 in 259 and 172 us instead of 1925 and 1427.  Aligned rows
// of 8192 take 101 and 109: the difference is instructions (78 % of the issue
// slots in the first form).  A step formed once a block in shared memory and
// 16-bit maxima of two elements at once took 267 us to 224, the third span's
// maximum only where there is one, to 208.

constexpr int kTile = kThreads * 8 * kUnroll;
constexpr int kTileStep = kTile - 2 * kQuantBlock;
constexpr int kTileBlocks = kTile / 8 + 3;

struct Spans {
  int block;   // counted from the tile's first
  int p1, p2;  // at least 1; 8 and more: behind the word
};

// A place in the tensor, and its column and block.
struct TileAt {
  long long elem, block;
  uint32_t col;
  __device__ __forceinline__ TileAt(long long e, uint32_t d, uint32_t nb) : elem(e) {
    const long long row = e < (1ll << 32) ? static_cast<uint32_t>(e) / d : e / d;
    col = static_cast<uint32_t>(e - row * d);
    block = row * nb + col / kQuantBlock;
  }
  __device__ __forceinline__ Spans at(int off, uint32_t d, uint32_t nb) const {
    uint32_t c = col + off, row = 0;
    if (c >= d) {
      row = c / d;
      c -= row * d;
    }
    const uint32_t left = d - c, p1 = min(kQuantBlock - c % kQuantBlock, left);
    const uint32_t p2 = p1 + min(static_cast<uint32_t>(kQuantBlock), left == p1 ? d : left - p1);
    return {static_cast<int>(row * nb + c / kQuantBlock - col / kQuantBlock), static_cast<int>(p1),
            static_cast<int>(p2)};
  }
};

// Eight elements' own values out of those of three spans.
__device__ __forceinline__ void spread(const float (&v)[3], const Spans& s, float* each) {
#pragma unroll
  for (int i = 0; i < 8; ++i) each[i] = i < s.p1 ? v[0] : v[1];
  if (s.p2 < 8) {
#pragma unroll
    for (int i = 2; i < 8; ++i) each[i] = i < s.p2 ? each[i] : v[2];
  }
}

// Bits [0, width) of a word; the width may lie outside 0 .. 32.
__device__ __forceinline__ uint32_t low_bits(int width) {
  uint32_t r;
  asm("bmsk.clamp.b32 %0, 0, %1;" : "=r"(r) : "r"(max(width, 0)));
  return r;
}

// The largest |x| of each span, as fp32 bits; 16-bit types as whole numbers, two a word, before they are widened.
template <typename T>
__device__ __forceinline__ void span_maxima(const Raw8<T>& raw, const Spans& s, uint32_t (&m)[3]) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t w[4] = {raw.w[0].x, raw.w[0].y, raw.w[0].z, raw.w[0].w};
    uint32_t top[3] = {0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a = w[i] & 0x7fff7fffu, below = low_bits(16 * (s.p1 - 2 * i));
      top[0] = __vmaxs2(top[0], a & below);
      top[1] = __vmaxs2(top[1], a & ~below);
    }
    if (s.p2 < 8) {  // a short block's end
      top[1] = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = w[i] & 0x7fff7fffu;
        const uint32_t below1 = low_bits(16 * (s.p1 - 2 * i)), below2 = low_bits(16 * (s.p2 - 2 * i));
        top[1] = __vmaxs2(top[1], a & below2 & ~below1);
        top[2] = __vmaxs2(top[2], a & ~below2);
      }
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const float2 f = word_to_floats<T>(max(top[k] & 0xffffu, top[k] >> 16));
      m[k] = __float_as_uint(f.x);
    }
  } else {
    float f[8];
    unpack8(raw, f);
    m[0] = m[1] = m[2] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t a = __float_as_uint(f[i]) & 0x7fffffffu;
      m[0] = max(m[0], i < s.p1 ? a : 0);
      if (i > 0) m[1] = max(m[1], i >= s.p1 && i < s.p2 ? a : 0);
      if (i > 1) m[2] = max(m[2], i >= s.p2 ? a : 0);
    }
  }
}

template <typename T, typename OutT, bool kSilu>
__global__ void __launch_bounds__(kThreads) quant8_spans_kernel(const T* __restrict__ x, OutT* __restrict__ out,
                                                                int8_t* __restrict__ codes,
                                                                uint8_t* __restrict__ exps, long long total,
                                                                uint32_t d) {
  __shared__ uint32_t amax[kTileBlocks];
  __shared__ float inv[kTileBlocks];
  const uint32_t nb = (d + kQuantBlock - 1) / kQuantBlock;
  for (int i = threadIdx.x; i < kTileBlocks; i += kThreads) amax[i] = 0;
  __syncthreads();
  for (long long emit = static_cast<long long>(blockIdx.x) * kTileStep; emit < total;
       emit += static_cast<long long>(gridDim.x) * kTileStep) {
    const long long end = emit + kTileStep < total ? emit + kTileStep : total;
    const TileAt tile(emit > 0 ? emit - kQuantBlock : 0, d, nb);
    Raw8<T> raw[kUnroll];
    Spans sp[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const long long e = tile.elem + (u * kThreads + threadIdx.x) * 8;
      if (e + 8 <= total) {
        raw[u] = load8_stream(x + e);
      } else {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) raw[u].w[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (e + i < total) reinterpret_cast<T*>(raw[u].w)[i] = x[e + i];
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int off = (u * kThreads + threadIdx.x) * 8;
      sp[u] = tile.at(off, d, nb);
      uint32_t m[3];
      span_maxima(raw[u], sp[u], m);
      if (tile.elem + off >= total) continue;
      atomicMax(amax + sp[u].block, m[0]);
      if (sp[u].p1 < 8) atomicMax(amax + sp[u].block + 1, m[1]);
      if (sp[u].p2 < 8) atomicMax(amax + sp[u].block + 2, m[2]);
    }
    // Blocks that reach into [emit, end) are complete; one that two tiles share gets the same byte from both.
    const int first = tile.at(static_cast<int>(emit - tile.elem), d, nb).block;
    const int last = tile.at(static_cast<int>(end - 1 - tile.elem), d, nb).block;
    __syncthreads();
    for (int i = first + threadIdx.x; i <= last; i += kThreads) {
      const Step8 s = step8_of(amax[i]);
      inv[i] = s.inv;
      exps[tile.block + i] = static_cast<uint8_t>(s.byte);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kTileBlocks; i += kThreads) amax[i] = 0;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const long long e = tile.elem + (u * kThreads + threadIdx.x) * 8;
      if (e < emit || e >= end) continue;
      const float* at = inv + sp[u].block;
      const float of3[3] = {at[0], at[1], at[2]};
      float f[8], by[8];
      spread(of3, sp[u], by);
      unpack8(raw[u], f);
      uint32_t q[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = code8_of(f[i], by[i]);
      if (kSilu) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) restored_apart<OutT, kRestoreSilu>(f[i], f[i + 1], 0.0f, 0.0f);
      }
      if (total - e >= 8) {
        *reinterpret_cast<uint2*>(codes + e) =
            make_uint2(bytes_of(q[0], q[1], q[2], q[3]), bytes_of(q[4], q[5], q[6], q[7]));
        if (kSilu) store8(out + e, f);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (e + i >= total) continue;
          codes[e + i] = static_cast<int8_t>(q[i]);
          if (kSilu) out[e + i] = from_float<OutT>(f[i]);
        }
      }
    }
    __syncthreads();  // the maxima are cleared, the steps read
  }
}

template <typename T, int kMode>
__global__ void __launch_bounds__(kThreads) restore8_spans_kernel(const int8_t* __restrict__ codes,
                                                                  const uint8_t* __restrict__ exps,
                                                                  const T* __restrict__ grad, T* __restrict__ out,
                                                                  long long total, uint32_t d) {
  const uint32_t nb = (d + kQuantBlock - 1) / kQuantBlock;
  for (long long first = static_cast<long long>(blockIdx.x) * kTile; first < total;
       first += static_cast<long long>(gridDim.x) * kTile) {
    const TileAt tile(first, d, nb);
    uint2 q[kUnroll];
    Raw8<T> g[kUnroll];
    Spans sp[kUnroll];
    int byte[kUnroll][3];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int off = (u * kThreads + threadIdx.x) * 8;
      const long long e = first + off;
      if (e >= total) continue;
      const int n = total - e < 8 ? static_cast<int>(total - e) : 8;
      if (n == 8) {
        q[u] = __ldcs(reinterpret_cast<const uint2*>(codes + e));
        if (kMode == kRestoreSiluGrad) g[u] = load8_stream(grad + e);
      } else {
        q[u] = make_uint2(0, 0);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (i >= n) continue;
          (i < 4 ? q[u].x : q[u].y) |= static_cast<uint32_t>(static_cast<uint8_t>(codes[e + i])) << (8 * (i & 3));
          if (kMode == kRestoreSiluGrad) reinterpret_cast<T*>(g[u].w)[i] = grad[e + i];
        }
      }
      sp[u] = tile.at(off, d, nb);
      const uint8_t* from = exps + tile.block + sp[u].block;
      byte[u][0] = from[0];
      byte[u][1] = sp[u].p1 < n ? from[1] : 127;
      byte[u][2] = sp[u].p2 < n ? from[2] : 127;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const long long e = first + (u * kThreads + threadIdx.x) * 8;
      if (e >= total) continue;
      const float scale[3] = {scale8_of(byte[u][0]), scale8_of(byte[u][1]), scale8_of(byte[u][2])};
      float f[8], gf[8], by[8];
      spread(scale, sp[u], by);
      if (kMode == kRestoreSiluGrad) unpack8(g[u], gf);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (kMode != kRestoreSiluGrad) gf[i] = 0.0f;
        f[i] = decoded<T, kMode>(code8_at(i < 4 ? q[u].x : q[u].y, i & 3), by[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; i += 2) restored_apart<T, kMode>(f[i], f[i + 1], gf[i], gf[i + 1]);
      if (total - e >= 8) {
        store8(out + e, f);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (e + i < total) out[e + i] = from_float<T>(f[i]);
      }
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
  return rows * ((nb + kAnyUnroll - 1) / kAnyUnroll);
}

// Aligned words through all rows: see above.
bool spans_fit(long long d) { return d >= 8 && d < (1ll << 31); }

int tile_grid(long long total, int tile, int sms) {
  const long long want = (total + tile - 1) / tile, cap = static_cast<long long>(sms) * 8;
  return static_cast<int>(want < cap ? want : cap);
}

template <typename T, typename OutT, bool kSilu>
int launch_quant(const T* x, OutT* out, int8_t* codes, uint8_t* exps, long long rows, long long d, int sms,
                 cudaStream_t stream) {
  if (rows <= 0 || d <= 0) return 0;
  const bool aligned = aligned16(x) && aligned16(codes) && (!kSilu || aligned16(out));
  const long long total = rows * d;
  if (aligned && d % 8 != 0 && spans_fit(d))
    quant8_spans_kernel<T, OutT, kSilu><<<tile_grid(total, kTileStep, sms), kThreads, 0, stream>>>(
        x, out, codes, exps, total, static_cast<uint32_t>(d));
  else if (!aligned || d % 8 != 0)
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
  const bool aligned = aligned16(out) && aligned16(codes) && (kMode != kRestoreSiluGrad || aligned16(grad));
  const long long total = rows * d;
  if (aligned && d % 8 != 0 && spans_fit(d))
    restore8_spans_kernel<T, kMode><<<tile_grid(total, kTile, sms), kThreads, 0, stream>>>(
        codes, exps, grad, out, total, static_cast<uint32_t>(d));
  else if (!aligned || d % 8 != 0)
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
