// Norms before and after a block, fused with its gate and the scaled residual
// stream (norm.cu).  dtype codes as in gemm.h.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace es {

// Column vectors: of the streams' type or fp32; null where absent.
struct NormParam {
  const void* p = nullptr;
  int f32 = 0;
};

struct NormArgs {
  int dtype = 0;
  long long rows = 0, d = 0;
  const void* x = nullptr;  // [rows, d], row pitch ldx
  const void* y = nullptr;  // [rows, d], row pitch ldy; null: n = norm(x) alone
  long long ldx = 0, ldy = 0;
  NormParam w, b, pw, pb, gate;
  // the gate's row for a stream row r: (r / gate_inner) % gate_count
  long long gate_inner = 1, gate_count = 1;
  int post = 0;    // norm y first
  int center = 1;  // 1: layer norm, 0: rms norm
  float scale = 1.0f, eps = 1e-5f;
  int sms = 148;
};

struct NormForward {
  void* h = nullptr;      // [rows, d]; null without y
  void* n = nullptr;      // [rows, d]
  float* stats = nullptr; // [rows][4]: mean and 1/deviation of y, of h; null: not kept
};

// Partial column sums: `units` slices of rows.  Grouped gate (one gate row for
// gate_inner consecutive rows): units are slices of single groups.
struct NormPlan {
  int full = 0;             // bias sums as well
  int grouped = 0;          // sums of D yh and D instead of their products with the gate
  long long groups = 1, slices = 1, len = 0;
  __host__ __device__ long long units() const { return groups * slices; }
  __host__ __device__ int sums() const { return full ? 4 : 2; }
  // floats from one row of sums to the next
  __host__ __device__ static long long pitch(long long d) { return (d + 7) / 8 * 8; }
};

struct NormBackward {
  const void* dh = nullptr;  // [rows, d] or null (zero)
  const void* dn = nullptr;
  const float* stats = nullptr;
  void* dx = nullptr;        // null: not wanted
  void* dy = nullptr;
  void* dgate_rows = nullptr;  // [rows, d] products of a gate that is not grouped; null: not wanted
  int dgate_f32 = 0;
  float* ws = nullptr;       // [units][sums][pitch(d)], null when no column sum is wanted
  float* coef = nullptr;     // [rows][4], for widths that take several passes (not norm_in_registers)
};

struct NormSums {
  void* dw = nullptr;  // outputs in the parameters' types; null: not wanted
  void* db = nullptr;
  void* dpw = nullptr;
  void* dpb = nullptr;
  void* dgate = nullptr;  // [groups, d] of a grouped gate
};

bool norm_in_registers(const NormArgs& a);  // one pass over a row; otherwise several
NormPlan norm_plan(const NormArgs& a);
int norm_forward(const NormArgs& a, const NormForward& f, cudaStream_t stream);
// Returns the launches in *launches.
int norm_backward(const NormArgs& a, const NormPlan& plan, const NormBackward& b, const NormSums& s,
                  cudaStream_t stream, int* launches);

}  // namespace es
