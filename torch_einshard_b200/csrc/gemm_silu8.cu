// GEMMs around a SiLU whose pre-activation h is kept in 8 bits (quant8.h):
//
//   forward   a = silu(x w), codes and exponents of h = x w from the 32-bit accumulator
//   backward  dh = (dy w2^T) silu'(h^) and a^ = silu(h^), the operand of the weight gradient dw2 = a^^T dy
//
// Both are epilogues of the 256 x 256 pair kernel (gemm_tc2.cuh), whose two
// accumulators let them run under the next tile's MMAs.  A thread reads 32
// consecutive columns of its row from TMEM, which is one block of the format: the
// maximum, exponent and codes of a block never leave the thread.  Outputs go
// through the warps' staging buffers as TMA boxes (16-bit values 32 x 64, codes
// 32 x 128).
//
// Without them h crosses memory as fp32 (4 bytes out, 4 back) before it is
// quantised, and dy w2^T, dh and a^ take 2 + 2 + 1 bytes more than the two results
// and the codes.  The SiLU's exponential and reciprocal, 1.5 a pair of results and
// column, are the epilogue's longest part (128 x 256 columns a CTA at 16 a clock:
// 3100 clocks), under the 16700 that the MMAs of a K = 2048 tile take.
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

// One box of this warp, 32 rows of 128 bytes as eight 16-byte words each, written
// row `lane` of the staging buffer in the 128-byte swizzle.
__device__ __forceinline__ void stage_words(uint8_t* stage, int lane, int chunk, uint4 v) {
  reinterpret_cast<uint4*>(stage)[lane * 8 + (chunk ^ (lane & 7))] = v;
}

__device__ __forceinline__ void send_box(const CUtensorMap* map, const uint8_t* stage, int col, int row, int batch,
                                         int lane) {
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    tma_store_3d(map, stage, col, row, batch);
    bulk_commit_group();
  }
}

// Every box of this warp has left its staging buffer.
__device__ __forceinline__ void stages_free(int lane) {
  if (lane == 0) bulk_wait_group_read<0>();
  __syncwarp();
}

template <typename T>
struct Silu8Epilogue {
  uint8_t* exps;
  int blocks;  // exponents of a row

  __device__ __forceinline__ void setup(int*, const GemmShape&) {}
  __device__ __forceinline__ void finish(const GemmShape&, volatile int*) {}

  // Codes of a block (the thread's 32 columns) into the code box, its exponent byte; r becomes the block's silu.
  __device__ __forceinline__ int block(uint32_t (&r)[32], uint8_t* code_stage, int lane, int chunk) const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) m = max(m, r[i] & 0x7fffffffu);
    const Step8 s = step8_of(m);
    uint32_t q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      q[i] = codes8_of(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1]), __uint_as_float(r[4 * i + 2]),
                       __uint_as_float(r[4 * i + 3]), s);
    stage_words(code_stage, lane, chunk, make_uint4(q[0], q[1], q[2], q[3]));
    stage_words(code_stage, lane, chunk + 1, make_uint4(q[4], q[5], q[6], q[7]));
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      float x1 = __uint_as_float(r[i]), x2 = __uint_as_float(r[i + 1]), s1, s2;
      sigmoid_pair(x1, x2, s1, s2);
      r[i] = __float_as_uint(x1 * s1);
      r[i + 1] = __float_as_uint(x2 * s2);
    }
    return s.byte;
  }

  __device__ __forceinline__ bool tile(const EpiTile& et, const GemmShape& s, volatile int*) {
    const int row0 = et.c.m0 + et.q * 32;
    const int row = row0 + et.lane;
    uint8_t* code_stage = et.stage + 4 * kStage2Out;
    uint8_t* exp_row = exps + (static_cast<long long>(et.c.b) * s.M + row) * blocks;
#pragma unroll 1
    for (int sub = 0; sub < kBN / 64; ++sub) {
      const int col0 = et.c.n0 + sub * 64;
      if (col0 >= s.N) break;  // uniform across the warp
      uint32_t r0[32], r1[32];
      tmem_ld32(et.tmem + sub * 64, r0);
      tmem_ld32(et.tmem + sub * 64 + 32, r1);
      tmem_ld_wait();
      stages_free(et.lane);
      // columns behind N are zero (the loads fill them so): they leave a short block's maximum alone
      const int chunk = (sub & 1) * 4;
      const int b0 = block(r0, code_stage, et.lane, chunk);
      const int b1 = block(r1, code_stage, et.lane, chunk + 2);
      if (row < s.M) {
        exp_row[col0 / 32] = static_cast<uint8_t>(b0);
        if (col0 + 32 < s.N) exp_row[col0 / 32 + 1] = static_cast<uint8_t>(b1);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t* v = j < 4 ? &r0[8 * j] : &r1[8 * (j - 4)];
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          w[k] = floats_to_word<T>(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1]));
        stage_words(et.stage, et.lane, j, make_uint4(w[0], w[1], w[2], w[3]));
      }
      send_box(et.tmc, et.stage, col0, row0, et.c.b, et.lane);
      // two sub-tiles make a box of 128 codes a row; the last one of a row may be half filled, and what lies behind
      // the row's end is not stored
      if ((sub & 1) || col0 + 64 >= s.N) send_box(et.tmw, code_stage, col0 & ~127, row0, et.c.b, et.lane);
    }
    return true;
  }
};

template <typename T>
struct Silu8GradEpilogue {
  const int8_t* codes;
  const uint8_t* exps;
  int blocks;

  __device__ __forceinline__ void setup(int*, const GemmShape&) {}
  __device__ __forceinline__ void finish(const GemmShape&, volatile int*) {}

  // 16 columns: dh (from the accumulator) and a^ as words of two.
  __device__ __forceinline__ void columns(const uint32_t* acc, const uint4& c, float scale, uint32_t (&dh)[8],
                                          uint32_t (&act)[8]) const {
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float x1 = code8_at(w[i / 2], (2 * i) & 3) * scale, x2 = code8_at(w[i / 2], (2 * i + 1) & 3) * scale, s1, s2;
      sigmoid_pair(x1, x2, s1, s2);
      act[i] = floats_to_word<T>(x1 * s1, x2 * s2);
      dh[i] = floats_to_word<T>(__uint_as_float(acc[2 * i]) * silu_slope(x1, s1),
                                __uint_as_float(acc[2 * i + 1]) * silu_slope(x2, s2));
    }
  }

  __device__ __forceinline__ bool tile(const EpiTile& et, const GemmShape& s, volatile int*) {
    const int row0 = et.c.m0 + et.q * 32;
    const int row = row0 + et.lane;
    const long long at = static_cast<long long>(et.c.b) * s.M + row;
    uint8_t* act_stage = et.stage + 4 * kStage2Out;
    // the row's codes and exponents of this tile: all loads in flight at once
    uint4 code[kBN / 16];
    uint8_t byte[kBN / 32];
#pragma unroll
    for (int j = 0; j < kBN / 16; ++j) {
      code[j] = make_uint4(0, 0, 0, 0);
      if (row < s.M && et.c.n0 + 16 * j < s.N)
        code[j] = __ldcs(reinterpret_cast<const uint4*>(codes + at * s.N + et.c.n0 + 16 * j));
    }
#pragma unroll
    for (int j = 0; j < kBN / 32; ++j) {
      byte[j] = 127;
      if (row < s.M && et.c.n0 + 32 * j < s.N) byte[j] = exps[at * blocks + et.c.n0 / 32 + j];
    }
#pragma unroll
    for (int sub = 0; sub < kBN / 64; ++sub) {
      const int col0 = et.c.n0 + sub * 64;
      if (col0 >= s.N) break;  // uniform across the warp
      uint32_t r0[32], r1[32];
      tmem_ld32(et.tmem + sub * 64, r0);
      tmem_ld32(et.tmem + sub * 64 + 32, r1);
      tmem_ld_wait();
      stages_free(et.lane);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t dh[8], act[8];
        columns(q < 2 ? &r0[16 * q] : &r1[16 * (q - 2)], code[sub * 4 + q], scale8_of(byte[sub * 2 + q / 2]), dh, act);
        stage_words(et.stage, et.lane, 2 * q, make_uint4(dh[0], dh[1], dh[2], dh[3]));
        stage_words(et.stage, et.lane, 2 * q + 1, make_uint4(dh[4], dh[5], dh[6], dh[7]));
        stage_words(act_stage, et.lane, 2 * q, make_uint4(act[0], act[1], act[2], act[3]));
        stage_words(act_stage, et.lane, 2 * q + 1, make_uint4(act[4], act[5], act[6], act[7]));
      }
      send_box(et.tmc, et.stage, col0, row0, et.c.b, et.lane);
      send_box(et.tmw, act_stage, col0, row0, et.c.b, et.lane);
    }
    return true;
  }
};

template <class Epi>
int launch_dual(const GemmArgs& g, const CUtensorMap& mc, const CUtensorMap& md, const Epi& epi, cudaStream_t stream) {
  CUtensorMap ma, mb;
  make_operand_maps(g, &ma, &mb, true);
  const GemmShape s = make_shape_pair(g);
  auto kernel = gemm_tc2_dual_kernel<Epi>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem2DualBytes);
  if (e != cudaSuccess) return static_cast<int>(e);
  const int pairs = s.num_m * s.num_n * s.batch;
  int clusters = g.num_sms / 2;
  if (pairs < clusters) clusters = pairs;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * clusters);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem2DualBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, ma, mb, mc, md, s, epi));
}

// Whether the pair kernel takes the product: at least a half wave of pair tiles (below, the elementwise passes cost
// less than idle SMs), and rows of codes that TMA can address.
bool fits(const GemmArgs& g) {
  const long long pairs =
      static_cast<long long>((g.M + 2 * kBM - 1) / (2 * kBM)) * ((g.N + kBN - 1) / kBN) * g.batch;
  return check_gemm_args(g) == nullptr && g.N % 16 == 0 && g.out_dtype == g.dtype && 4 * pairs >= g.num_sms &&
         g.M >= kBM && g.N >= kBN;
}

template <typename T>
int launch_silu8(const GemmArgs& g, int8_t* codes, uint8_t* exps, cudaStream_t stream) {
  CUtensorMap mc;
  if (!make_output_map(g, false, &mc)) return static_cast<int>(cudaErrorNotSupported);
  const uint64_t dims[3] = {static_cast<uint64_t>(g.N), static_cast<uint64_t>(g.M), static_cast<uint64_t>(g.batch)};
  const uint64_t strides[2] = {static_cast<uint64_t>(g.N), static_cast<uint64_t>(g.N) * g.M};
  const uint32_t box[3] = {128, 32, 1};
  const CUtensorMap md = make_tmap_nd(codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, dims, strides, box);
  const Silu8Epilogue<T> epi{exps, (g.N + kQuantBlock - 1) / kQuantBlock};
  return launch_dual(g, mc, md, epi, stream);
}

template <typename T>
int launch_silu8_grad(const GemmArgs& g, const int8_t* codes, const uint8_t* exps, void* act, cudaStream_t stream) {
  GemmArgs ga = g;
  ga.C = act;
  CUtensorMap mc, md;
  if (!make_output_map(g, false, &mc) || !make_output_map(ga, false, &md))
    return static_cast<int>(cudaErrorNotSupported);
  const Silu8GradEpilogue<T> epi{codes, exps, (g.N + kQuantBlock - 1) / kQuantBlock};
  return launch_dual(g, mc, md, epi, stream);
}

}  // namespace

int gemm_launch_silu8(const GemmArgs& g, int8_t* codes, uint8_t* exps, cudaStream_t stream) {
  if (!fits(g) || (reinterpret_cast<uintptr_t>(codes) & 15) != 0) return static_cast<int>(cudaErrorNotSupported);
  return g.dtype == kDtypeBF16 ? launch_silu8<__nv_bfloat16>(g, codes, exps, stream)
                               : launch_silu8<__half>(g, codes, exps, stream);
}

int gemm_launch_silu8_grad(const GemmArgs& g, const int8_t* codes, const uint8_t* exps, void* act,
                           cudaStream_t stream) {
  if (!fits(g) || (reinterpret_cast<uintptr_t>(codes) & 15) != 0) return static_cast<int>(cudaErrorNotSupported);
  return g.dtype == kDtypeBF16 ? launch_silu8_grad<__nv_bfloat16>(g, codes, exps, act, stream)
                               : launch_silu8_grad<__half>(g, codes, exps, act, stream);
}

}  // namespace es
