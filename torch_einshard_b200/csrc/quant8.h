// Activations kept for backward in 8 bits (quant8.cu).  dtype codes as in gemm.h.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace es {

constexpr int kQuantBlock = 32;  // channels that share one exponent
constexpr int kQuantNan = 255;   // exponent byte of a block that held an infinity or a NaN

// codes[rows][d], exps[rows][ceil(d / 32)] of x[rows][d] (contiguous).
int quant8(const void* x, int dtype, int8_t* codes, uint8_t* exps, long long rows, long long d, int sms,
           cudaStream_t stream);
// The same of an fp32 pre-activation h, and out = silu(h) in out_dtype.
int quant8_silu(const float* h, void* out, int out_dtype, int8_t* codes, uint8_t* exps, long long rows, long long d,
                int sms, cudaStream_t stream);

enum Restore8Mode : int {
  kRestoreValue = 0,     // out = x^
  kRestoreSilu = 1,      // out = silu(x^)
  kRestoreSiluGrad = 2,  // out = grad * silu'(x^)
};
// x^ = codes 2^exps, through `mode`, in dtype; grad[rows][d] is read by kRestoreSiluGrad alone.
int restore8(const int8_t* codes, const uint8_t* exps, const void* grad, void* out, int dtype, int mode,
             long long rows, long long d, int sms, cudaStream_t stream);

}  // namespace es
