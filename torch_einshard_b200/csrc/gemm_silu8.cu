// GEMMs around a SiLU whose pre-activation h is kept in 8 bits (quant8.h):
//
//   forward   a = silu(x w), codes and exponents of h = x w from the 32-bit accumulator
//   backward  dh = (dy w2^T) silu'(h^) and a^ = silu(h^), the operand of the weight gradient dw2 = a^^T dy
//
// Both are epilogues of the 256 x 256 pair kernel (gemm_tc2.cuh), whose two
// accumulators and eight epilogue warps let them run under the next tile's MMAs.
// A thread reads 32 consecutive columns of its row from TMEM, which is one block
// of the format: the maximum, exponent and codes of a block never leave the
// thread, and each of its stores is a whole 32-byte sector.
//
// Without them h crosses memory as fp32 (4 bytes out, 4 back) before it is
// quantised, and dy w2^T, dh and a^ take 2 + 2 + 1 bytes more than the two results
// and the codes.  Measured (the plain pair kernel / with the epilogue / plain wide
// kernel and elementwise passes): 32768 x 2048 x 8192 forward 0.83 / 1.05 / 1.50 ms,
// backward 0.85 / 1.18 / 1.40 ms; 2048 x 2048 x 2048 21 / 24 / 34 and 21 / 28 / 36 us;
// 128 x 1024 x 2560 15 / 17 / 25 and 15 / 20 / 22 us, so every shape that fits takes
// them.  Boxes through shared memory and TMA stores instead of the threads' own
// stores: 4 % faster at the largest of these, 10 % slower at the others.  At the
// largest the card is at its power limit, where the epilogue's arithmetic (an
// exponential and half a reciprocal a column) costs clock, not issue slots.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <string.h>

#include "gemm.h"
#include "gemm_tc.cuh"
#include "gemm_tc2.cuh"
#include "quant8.cuh"
#include "tma_desc.h"

namespace es {
namespace {

constexpr int kCols = 4 * kBN / kLongEpiWarps;  // columns of a warp's part of a tile

// 32 bytes in one access (sm_100's 256-bit forms): a whole sector a thread, so
// that rows need no transposition through shared memory.
__device__ __forceinline__ void store32(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

__device__ __forceinline__ void load32(uint32_t* w, const void* p) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p));
}

// What both epilogues know of the 8-bit tensor and the 16-bit ones: rows of N
// columns, `pitch` (a multiple of 16) apart, and of `blocks` exponents.  The
// columns between N and the pitch are written (a sector at a time), not used.
struct Codes {
  int8_t* codes;
  uint8_t* exps;
  int blocks, pitch;
};

template <typename T>
struct Silu8Epilogue {
  T* out;  // [batch M, pitch]
  Codes kept;

  __device__ __forceinline__ void setup(int*, const GemmShape&) {}
  __device__ __forceinline__ void finish(const GemmShape&, volatile int*) {}

  __device__ __forceinline__ bool tile(const EpiTile& et, const GemmShape& s, volatile int*) {
    const int row = et.c.m0 + et.row;
    const long long at = static_cast<long long>(et.c.b) * s.M + row;
#pragma unroll 1
    for (int sub = 0; sub < kCols / 32; ++sub) {
      const int col = et.c.n0 + sub * 32;
      if (col >= s.N) break;  // uniform across the warp
      uint32_t r[32];
      __syncwarp();  // the load is the whole warp's
      tmem_ld32(et.tmem + sub * 32, r);
      tmem_ld_wait();
      if (row >= s.M) continue;
      // columns behind N are zero (the loads fill them so): they leave a short block's maximum alone
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) m = max(m, r[i] & 0x7fffffffu);
      const Step8 step = step8_of(m);
      uint32_t q[8], w[16];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        q[i] = codes8_of(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1]), __uint_as_float(r[4 * i + 2]),
                         __uint_as_float(r[4 * i + 3]), step);
      if (step.byte != kQuantNan) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float x1 = __uint_as_float(r[2 * i]), x2 = __uint_as_float(r[2 * i + 1]), s1, s2;
          sigmoid_pair(x1, x2, s1, s2);
          w[i] = floats_to_word<T>(x1 * s1, x2 * s2);
        }
      } else {  // a NaN column leaves the one beside it alone
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float x1 = __uint_as_float(r[2 * i]), x2 = __uint_as_float(r[2 * i + 1]), s1, s2;
          sigmoid_apart(x1, x2, s1, s2);
          w[i] = floats_to_word<T>(x1 * s1, x2 * s2);
        }
      }
      int8_t* code_row = kept.codes + at * kept.pitch + col;
      T* out_row = out + at * kept.pitch + col;
      kept.exps[at * kept.blocks + col / 32] = static_cast<uint8_t>(step.byte);
      store32(out_row, w);
      if (col + 32 <= kept.pitch) {
        store32(out_row + 16, w + 8);
        if ((reinterpret_cast<uintptr_t>(code_row) & 31) == 0) {
          store32(code_row, q);
        } else {
          reinterpret_cast<uint4*>(code_row)[0] = make_uint4(q[0], q[1], q[2], q[3]);
          reinterpret_cast<uint4*>(code_row)[1] = make_uint4(q[4], q[5], q[6], q[7]);
        }
      } else {
        reinterpret_cast<uint4*>(code_row)[0] = make_uint4(q[0], q[1], q[2], q[3]);
      }
    }
    return true;
  }
};

template <typename T>
struct Silu8GradEpilogue {
  T* out;  // [batch M, pitch]
  T* act;
  Codes kept;

  __device__ __forceinline__ void setup(int*, const GemmShape&) {}
  __device__ __forceinline__ void finish(const GemmShape&, volatile int*) {}

  __device__ __forceinline__ bool tile(const EpiTile& et, const GemmShape& s, volatile int*) {
    const int row = et.c.m0 + et.row;
    const long long at = static_cast<long long>(et.c.b) * s.M + row;
    // the row's codes and exponents of this tile: all loads in flight at once
    uint32_t code[kCols / 4];
    uint8_t byte[kCols / 32];
#pragma unroll
    for (int j = 0; j < kCols / 32; ++j) {
      const int col = et.c.n0 + 32 * j;
      const int8_t* p = kept.codes + at * kept.pitch + col;
#pragma unroll
      for (int i = 0; i < 8; ++i) code[8 * j + i] = 0;
      byte[j] = 127;
      if (row >= s.M || col >= s.N) continue;
      byte[j] = kept.exps[at * kept.blocks + col / 32];
      if (col + 32 <= kept.pitch && (reinterpret_cast<uintptr_t>(p) & 31) == 0) {
        load32(&code[8 * j], p);
      } else {
        const uint4 lo = reinterpret_cast<const uint4*>(p)[0];
        code[8 * j] = lo.x, code[8 * j + 1] = lo.y, code[8 * j + 2] = lo.z, code[8 * j + 3] = lo.w;
        if (col + 32 <= kept.pitch) {
          const uint4 hi = reinterpret_cast<const uint4*>(p)[1];
          code[8 * j + 4] = hi.x, code[8 * j + 5] = hi.y, code[8 * j + 6] = hi.z, code[8 * j + 7] = hi.w;
        }
      }
    }
#pragma unroll
    for (int sub = 0; sub < kCols / 32; ++sub) {
      const int col = et.c.n0 + sub * 32;
      if (col >= s.N) break;  // uniform across the warp
      uint32_t r[32];
      __syncwarp();  // the load is the whole warp's
      tmem_ld32(et.tmem + sub * 32, r);
      tmem_ld_wait();
      if (row >= s.M) continue;
      const float scale = finite_scale8_of(byte[sub]);
      uint32_t dh[16], aw[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t w = code[8 * sub + i / 2];
        float x1 = code8_at(w, (2 * i) & 3) * scale, x2 = code8_at(w, (2 * i + 1) & 3) * scale, s1, s2, e1, e2;
        sigmoid_pair(x1, x2, s1, s2, e1, e2);
        aw[i] = floats_to_word<T>(x1 * s1, x2 * s2);
        dh[i] = floats_to_word<T>(__uint_as_float(r[2 * i]) * silu_slope(x1, s1, e1),
                                  __uint_as_float(r[2 * i + 1]) * silu_slope(x2, s2, e2));
      }
      T* out_row = out + at * kept.pitch + col;
      T* act_row = act + at * kept.pitch + col;
      store32(out_row, dh);
      store32(act_row, aw);
      if (col + 32 <= kept.pitch) {
        store32(out_row + 16, dh + 8);
        store32(act_row + 16, aw + 8);
      }
    }
    return true;
  }
};

template <class Epi>
int launch_long(const GemmArgs& g, const Epi& epi, cudaStream_t stream) {
  CUtensorMap ma, mb;
  make_operand_maps(g, &ma, &mb, true);
  const GemmShape s = make_shape_pair(g);
  auto kernel = gemm_tc2_long_kernel<Epi>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem2LongBytes);
  if (e != cudaSuccess) return static_cast<int>(e);
  const int pairs = s.num_m * s.num_n * s.batch;
  int clusters = g.num_sms / 2;
  if (pairs < clusters) clusters = pairs;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * clusters);
  cfg.blockDim = dim3(kLongThreads);
  cfg.dynamicSmemBytes = kSmem2LongBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, ma, mb, s, epi));
}

bool aligned32(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31) == 0; }

// Whether the pair kernel takes the product: dense outputs whose rows are whole 32-byte sectors of 16-bit values.
bool fits(const GemmArgs& g, const int8_t* codes) {
  return check_gemm_args(g) == nullptr && g.ldc >= g.N && g.ldc % 16 == 0 && g.ldc < (1ll << 31) &&
         g.out_dtype == g.dtype && (g.batch == 1 || g.c_batch_stride == g.M * g.ldc) && aligned32(g.C) &&
         (reinterpret_cast<uintptr_t>(codes) & 15) == 0;
}

Codes codes_of(const GemmArgs& g, const int8_t* codes, const uint8_t* exps) {
  return {const_cast<int8_t*>(codes), const_cast<uint8_t*>(exps), (g.N + kQuantBlock - 1) / kQuantBlock,
          static_cast<int>(g.ldc)};
}

template <typename T>
int launch_silu8(const GemmArgs& g, int8_t* codes, uint8_t* exps, cudaStream_t stream) {
  const Silu8Epilogue<T> epi{static_cast<T*>(g.C), codes_of(g, codes, exps)};
  return launch_long(g, epi, stream);
}

template <typename T>
int launch_silu8_grad(const GemmArgs& g, const int8_t* codes, const uint8_t* exps, void* act, cudaStream_t stream) {
  const Silu8GradEpilogue<T> epi{static_cast<T*>(g.C), static_cast<T*>(act), codes_of(g, codes, exps)};
  return launch_long(g, epi, stream);
}

}  // namespace

int gemm_launch_silu8(const GemmArgs& g, int8_t* codes, uint8_t* exps, cudaStream_t stream) {
  if (!fits(g, codes)) return static_cast<int>(cudaErrorInvalidValue);
  return g.dtype == kDtypeBF16 ? launch_silu8<__nv_bfloat16>(g, codes, exps, stream)
                               : launch_silu8<__half>(g, codes, exps, stream);
}

int gemm_launch_silu8_grad(const GemmArgs& g, const int8_t* codes, const uint8_t* exps, void* act,
                           cudaStream_t stream) {
  if (!fits(g, codes) || !aligned32(act)) return static_cast<int>(cudaErrorInvalidValue);
  return g.dtype == kDtypeBF16 ? launch_silu8_grad<__nv_bfloat16>(g, codes, exps, act, stream)
                               : launch_silu8_grad<__half>(g, codes, exps, act, stream);
}

}  // namespace es
