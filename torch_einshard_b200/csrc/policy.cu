// Clipped policy loss with a KL term, from logits.
//
//   lp = z_a / T - log sum_j e^(z_j / T)      r = e^(lp - old)
//   loss_t = -min(r A, clip(r, 1 - lo, 1 + hi) A) + beta (e^(ref - lp) - (ref - lp) - 1)
//   c_t = dloss_t / dlp = -(r A where r A <= clip(r) A) + beta (1 - e^(ref - lp))
//   dz_j = g w_t c_t / T (1[j = a] - e^(z_j / T - lse))
//
// with weights w from the reduction: 1 / tokens, 1 / (sequences x the
// sequence's tokens) or 1.  A masked token has no loss and a gradient of zeros,
// whatever its logits, id and other inputs hold: its row is not read.
//
// Forward, a block reads a token's row once with a running maximum m and sum s
// of 2^((z - m) log2(e) / T) a thread; z - m is formed before the scaling, so
// rows of the type's lowest value or of very large logits keep their
// differences.  Bound by the read: 2 bytes a 16-bit logit, against 16
// exponentials a clock and SM.  Backward reads the row again and writes the
// gradient (a row whose c is 0, masked or clipped, is written without being read).
// Rows need no alignment: up to seven logits at either end are taken one by one.
#include "policy.h"

#include "gemm.h"
#include "vec.cuh"

namespace es {
namespace {

constexpr int kThreads = 512;
constexpr int kUnroll = 4;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Running maximum and sum of 2^((z - m) c).
struct Running {
  float m, s;
  __device__ __forceinline__ static float base(float m) { return m == -INFINITY ? 0.0f : m; }
  __device__ __forceinline__ void raise(float top, float c) {
    if (top > m) {
      s *= exp2_fast((m - base(top)) * c);  // m = -inf: s is 0 and stays it
      m = top;
    }
  }
  __device__ __forceinline__ void add(float z, float c) {
    raise(z, c);
    s += exp2_fast((z - base(m)) * c);
  }
  __device__ __forceinline__ void merge(float m2, float s2, float c) {
    const float top = fmaxf(m, m2);
    const float b = base(top);
    s = s * exp2_fast((m - b) * c) + s2 * exp2_fast((m2 - b) * c);
    m = top;
  }
};

// Elements before the first 16-byte boundary of a row.
template <typename T>
__device__ __forceinline__ int head_of(const T* row, long long n) {
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const int head = off == 0 ? 0 : static_cast<int>(16 / sizeof(T)) - off;
  return head < n ? head : static_cast<int>(n);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) policy_rows_kernel(const PolicyArgs a, const PolicyState o) {
  __shared__ float2 red[kThreads / 32];
  const float c = a.inv_temp * kLog2e;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (long long t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    if (a.mask != nullptr && !a.mask[t]) {  // uniform
      if (threadIdx.x == 0) {
        o.logp[t] = 0.0f;
        o.terms[t] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        o.norm[t] = make_float2(0.0f, 0.0f);
      }
      continue;
    }
    const T* row = static_cast<const T*>(a.logits) + t * a.ld;
    const int head = head_of(row, a.vocab);
    const T* body = row + head;
    const long long chunks = (a.vocab - head) / 8;
    Running r{-INFINITY, 0.0f};
    for (long long i = threadIdx.x; i < chunks; i += kThreads * kUnroll) {
      Raw8<T> raw[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (i + u * kThreads < chunks) raw[u] = load8_stream(body + (i + u * kThreads) * 8);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (i + u * kThreads >= chunks) break;
        float z[8];
        unpack8(raw[u], z);
        float top = z[0];
#pragma unroll
        for (int k = 1; k < 8; ++k) top = fmaxf(top, z[k]);
        r.raise(top, c);
        const float b = Running::base(r.m);
#pragma unroll
        for (int k = 0; k < 8; ++k) r.s += exp2_fast((z[k] - b) * c);
      }
    }
    // the ends of the row
    const int tail = static_cast<int>(a.vocab - head - chunks * 8);
    if (static_cast<int>(threadIdx.x) < head) r.add(to_float<T>(row[threadIdx.x]), c);
    if (static_cast<int>(threadIdx.x) < tail) r.add(to_float<T>(body[chunks * 8 + threadIdx.x]), c);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
      r.merge(__shfl_xor_sync(0xffffffffu, r.m, off), __shfl_xor_sync(0xffffffffu, r.s, off), c);
    __syncthreads();  // the previous token's words are read
    if (lane == 0) red[warp] = make_float2(r.m, r.s);
    __syncthreads();
    if (warp == 0) {
      const float2 v = lane < kThreads / 32 ? red[lane] : make_float2(-INFINITY, 0.0f);
      r.m = v.x;
      r.s = v.y;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1)
        r.merge(__shfl_xor_sync(0xffffffffu, r.m, off), __shfl_xor_sync(0xffffffffu, r.s, off), c);
      if (lane == 0) {
        const int64_t id = a.ids[t];
        // an id outside the vocabulary makes the loss NaN
        const float z = id >= 0 && id < a.vocab ? to_float<T>(row[id]) : __uint_as_float(0x7fc00000u);
        const float lp = (z - r.m) * a.inv_temp - logf(r.s);
        const float adv = a.adv[a.adv_per_sequence ? t / a.length : t];
        const float ratio = a.old != nullptr ? expf(lp - a.old[t]) : expf(lp - lp);
        const float kept = fminf(fmaxf(ratio, 1.0f - a.lo), 1.0f + a.hi);
        const float s1 = ratio * adv, s2 = kept * adv;
        const bool clipped = s1 > s2;
        float loss = 0.0f, slope = 0.0f, kl = 0.0f;
        if (adv != 0.0f) {
          loss = clipped ? -s2 : -s1;
          slope = clipped ? 0.0f : -s1;
        }
        if (a.ref != nullptr) {
          const float away = a.ref[t] - lp;
          const float rise = expm1f(away);
          kl = rise - away;
          loss += a.kl * kl;
          slope -= a.kl * rise;
        }
        o.logp[t] = lp;
        o.terms[t] = make_float4(loss, kl, clipped ? 1.0f : 0.0f, slope);
        o.norm[t] = make_float2(r.m, log2f(r.s));
      }
    }
  }
}

// Sums of a sequence's terms: block a sequence.
__global__ void __launch_bounds__(256) policy_sequence_kernel(const PolicyArgs a, const PolicyState o) {
  __shared__ float4 red[8];
  const long long q = blockIdx.x;
  float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (long long i = threadIdx.x; i < a.length; i += 256) {
    const long long t = q * a.length + i;
    if (a.mask != nullptr && !a.mask[t]) continue;
    const float4 v = o.terms[t];
    s.x += v.x, s.y += v.y, s.z += v.z, s.w += 1.0f;
  }
  s = make_float4(warp_sum(s.x), warp_sum(s.y), warp_sum(s.z), warp_sum(s.w));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) s.x += red[i].x, s.y += red[i].y, s.z += red[i].z, s.w += red[i].w;
    o.sums[q] = s;
  }
}

// The reduction over sequences and the weights of their tokens: one block.
__global__ void __launch_bounds__(256) policy_reduce_kernel(const PolicyArgs a, const PolicyState o) {
  __shared__ float4 red[8];
  __shared__ float total;
  const long long sequences = a.tokens / a.length;
  const bool each = a.reduction == kReduceSequence;
  float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (long long q = threadIdx.x; q < sequences; q += 256) {
    const float4 v = o.sums[q];
    if (v.w == 0.0f) continue;
    const float f = each ? 1.0f / v.w : 1.0f;
    s.x += v.x * f, s.y += v.y * f, s.z += v.z * f, s.w += each ? 1.0f : v.w;
  }
  s = make_float4(warp_sum(s.x), warp_sum(s.y), warp_sum(s.z), warp_sum(s.w));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) s.x += red[i].x, s.y += red[i].y, s.z += red[i].z, s.w += red[i].w;
    const float f = a.reduction == kReduceSum ? 1.0f : 1.0f / fmaxf(s.w, 1.0f);
    *o.loss = a.weight * s.x * f;
    *o.kl = s.y * f;
    *o.clipped = s.z * f;
    total = a.weight * f;
  }
  __syncthreads();
  for (long long q = threadIdx.x; q < sequences; q += 256)
    o.weight[q] = each ? total / fmaxf(o.sums[q].w, 1.0f) : total;
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    policy_backward_kernel(const PolicyArgs a, const PolicyState o, const float* grad, T* __restrict__ dlogits) {
  const float c = a.inv_temp * kLog2e;
  const float g = *grad;
  for (long long t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    const T* row = static_cast<const T*>(a.logits) + t * a.ld;
    T* out = dlogits + t * a.vocab;
    const bool live = a.mask == nullptr || a.mask[t];
    const float slope = live ? o.terms[t].w : 0.0f;
    const float k = slope == 0.0f ? 0.0f : g * o.weight[t / a.length] * slope * a.inv_temp;
    const bool zero = k == 0.0f;  // NaN is not zero
    const float2 norm = o.norm[t];
    const long long id = zero ? -1 : a.ids[t];
    const int head = head_of(out, a.vocab);
    const bool vec = !zero && ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    const long long chunks = (a.vocab - head) / 8;
    auto one = [&](long long j) {
      float v = 0.0f;
      if (!zero) {
        const float p = exp2_fast((to_float<T>(row[j]) - norm.x) * c - norm.y);
        v = k * ((j == id ? 1.0f : 0.0f) - p);
      }
      out[j] = from_float<T>(v);
    };
    if (zero) {
      const float nil[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
      for (long long i = threadIdx.x; i < chunks; i += kThreads) store8(out + head + i * 8, nil);
    } else if (vec) {
      for (long long i = threadIdx.x; i < chunks; i += kThreads * kUnroll) {
        Raw8<T> raw[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (i + u * kThreads < chunks) raw[u] = load8_stream(row + head + (i + u * kThreads) * 8);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          if (i + u * kThreads >= chunks) break;
          const long long j0 = head + (i + u * kThreads) * 8;
          float z[8];
          unpack8(raw[u], z);
#pragma unroll
          for (int e = 0; e < 8; ++e) z[e] = -k * exp2_fast((z[e] - norm.x) * c - norm.y);
          if (id >= j0 && id < j0 + 8) {
            const int at = static_cast<int>(id - j0);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (e == at) z[e] += k;
          }
          store8(out + j0, z);
        }
      }
    } else {
      for (long long j = head + threadIdx.x; j < head + chunks * 8; j += kThreads) one(j);
    }
    const int tail = static_cast<int>(a.vocab - head - chunks * 8);
    if (static_cast<int>(threadIdx.x) < head) one(threadIdx.x);
    if (static_cast<int>(threadIdx.x) < tail) one(head + chunks * 8 + threadIdx.x);
  }
}

int grid_for(const PolicyArgs& a) {
  const long long cap = a.sms * (2048ll / kThreads);
  return static_cast<int>(a.tokens < cap ? a.tokens : cap);
}

template <typename T>
int forward_type(const PolicyArgs& a, const PolicyState& s, cudaStream_t stream, int* launches) {
  policy_rows_kernel<T><<<grid_for(a), kThreads, 0, stream>>>(a, s);
  policy_sequence_kernel<<<static_cast<unsigned>(a.tokens / a.length), 256, 0, stream>>>(a, s);
  policy_reduce_kernel<<<1, 256, 0, stream>>>(a, s);
  *launches = 3;
  return static_cast<int>(cudaGetLastError());
}

template <typename T>
int backward_type(const PolicyArgs& a, const PolicyState& s, const float* grad, void* dlogits, cudaStream_t stream) {
  policy_backward_kernel<T><<<grid_for(a), kThreads, 0, stream>>>(a, s, grad, static_cast<T*>(dlogits));
  return static_cast<int>(cudaGetLastError());
}

}  // namespace

int policy_forward(const PolicyArgs& a, const PolicyState& s, cudaStream_t stream, int* launches) {
  *launches = 0;
  if (a.tokens <= 0) return 0;
  if (a.vocab <= 0 || a.length <= 0 || a.tokens % a.length != 0) return static_cast<int>(cudaErrorInvalidValue);
  switch (a.dtype) {
    case kDtypeBF16:
      return forward_type<__nv_bfloat16>(a, s, stream, launches);
    case kDtypeF16:
      return forward_type<__half>(a, s, stream, launches);
    case kDtypeF32:
      return forward_type<float>(a, s, stream, launches);
    default:
      return static_cast<int>(cudaErrorInvalidValue);
  }
}

int policy_backward(const PolicyArgs& a, const PolicyState& s, const float* grad, void* dlogits,
                    cudaStream_t stream) {
  if (a.tokens <= 0) return 0;
  switch (a.dtype) {
    case kDtypeBF16:
      return backward_type<__nv_bfloat16>(a, s, grad, dlogits, stream);
    case kDtypeF16:
      return backward_type<__half>(a, s, grad, dlogits, stream);
    case kDtypeF32:
      return backward_type<float>(a, s, grad, dlogits, stream);
    default:
      return static_cast<int>(cudaErrorInvalidValue);
  }
}

}  // namespace es
