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
// A block reads a token's row with a running maximum and a sum of powers of two
// a thread.  The weights depend on the mask alone, so a training step's forward pass goes on to
// write the row's gradient for g = 1 while the row is still in L2: memory moves
// 2 + 2 bytes a 16-bit logit instead of the 2 + 2 + 2 of separate passes.  The
// backward pass then only looks at g; where it is not 1 it forms the gradient
// again from the logits, in 32 bits, so that nothing is rounded twice and a small
// fp16 gradient is scaled before it could vanish.  What a row's gradient was formed
// for is kept beside it (`factors`), so that running the backward pass again, as
// the replay of a captured graph does, gives the gradient for the g of that run.
// A row whose c is 0 (clipped) is written without a second read.
//
// Bounds: memory, then the exponentials (one a logit and pass, 16 a clock and SM)
// and the instructions around them.  bf16 with gradient, 58 % of the tokens kept:
// 12288 rows of 128257 take 0.92 ms, 8192 rows of 32000 150 us, 5.4 and 5.5 TB/s of
// what has to move (84 % of a copy's rate; part of the second reads misses L2); fp32
// without, 4084 rows of 50257: 74 us, a copy's rate.  Pairs of fp32 operations up to
// the exponentials, where the scale
// takes two FMAs, saved 7 % (behind them their results would have to be moved
// into pairs).  Rows need no alignment: up to seven logits at either end are taken
// one by one.
#include "policy.h"

#include "gemm.h"
#include "vec.cuh"

#include <type_traits>

namespace es {
namespace {

constexpr int kUnroll = 4;
constexpr int kRun = 128;  // tokens whose terms a block adds
constexpr double kLog2e = 1.4426950408889634;
constexpr float kLn2 = 0.6931471805599453f;

// log2(e) / T, and what its first 24 bits leave: rounded towards zero, so that an infinite logit gives the same
// infinity with both.
__device__ __forceinline__ float scale_of(const PolicyArgs& a) { return __double2float_rz(a.inv_temp * kLog2e); }
__device__ __forceinline__ float scale_rest_of(const PolicyArgs& a, float c) {
  return fmaxf(static_cast<float>(a.inv_temp * kLog2e - c), 1e-30f);
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Sums are relative to 2^q, q the whole number above m c (c = log2(e) / T): a larger maximum scales them by an exact
// power of two, and z c - q takes one FMA.  Where m c is so large that its rounding would show (rows of mask values),
// q is infinite and sums are relative to 2^(m c), of differences that are formed before they are scaled.
constexpr float kLarge = 4194304.0f;

__device__ __forceinline__ float base_of(float m, float c) {
  const float p = m * c;
  return fabsf(p) < kLarge ? ceilf(p) : INFINITY;
}

// A logit's power.  The rest of the scale is one FMA more: without it a log-probability is off by up to 6e-8 of how
// far the logit lies from the row's mean, with one sign for all tokens.
__device__ __forceinline__ float power_of(float z, float q, float c, float rest) {
  return exp2_fast(fmaf(z, rest, fmaf(z, c, -q)));
}

// The factor that takes a sum from (m, q) to a larger maximum's (m2, q2).
__device__ __forceinline__ float rebased(float m, float q, float m2, float q2, float c, float rest) {
  if (m == -INFINITY) return 0.0f;  // nothing summed yet but zeros
  if (q != INFINITY && q2 != INFINITY)
    return __int_as_float(static_cast<int>(fmaxf(q - q2, -127.0f) + 127.0f) << 23);
  if (q == INFINITY && q2 == INFINITY) return exp2_fast((m - m2) * c);
  return exp2_fast(q == INFINITY ? fmaf(m, rest, fmaf(m, c, -q2)) : fmaf(-m2, rest, fmaf(-m2, c, q)));
}

// Largest logit and sum of powers.
struct Running {
  float m, s;
  // Joined over the warp: the maximum as an integer of the same order (a NaN ends up in s), one scaling, the sum.
  __device__ __forceinline__ void over_warp(float c, float rest) {
    const int bits = __float_as_int(m);
    const int top = __reduce_max_sync(0xffffffffu, bits ^ ((bits >> 31) & 0x7fffffff));
    const float largest = __int_as_float(top ^ ((top >> 31) & 0x7fffffff));
    s = warp_sum(s * rebased(m, base_of(m, c), largest, base_of(largest, c), c, rest));
    m = largest;
  }
};

// The same over a thread's chunks.
struct ChunkSum {
  float m = -INFINITY, q = 0.0f, s = 0.0f;
  __device__ __forceinline__ void raise(float top, float c, float rest) {
    if (top > m) {
      const float next = base_of(top, c);
      s *= rebased(m, q, top, next, c, rest);
      m = top;
      q = next;
    }
  }
  __device__ __forceinline__ void add(float z, float c, float rest) {
    raise(z, c, rest);
    s += q == INFINITY ? exp2_fast((z - m) * c) : power_of(z, q, c, rest);
  }
};

// Elements before the first 16-byte boundary of a row.
template <typename T>
__device__ __forceinline__ int head_of(const T* row, int n) {
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const int head = off == 0 ? 0 : static_cast<int>(16 / sizeof(T)) - off;
  return head < n ? head : n;
}

// Eight columns from j0 of a token's gradient k (1[j = id] - p_j), with p_j from the row's maximum and sum.
struct GradientRow {
  float k, c, off, factor, m;
  int id;
  bool large;
  __device__ __forceinline__ GradientRow(float k_, Running row, int id_, float c_, float rest)
      : k(k_), c(c_), m(row.m), id(id_) {
    const float q = base_of(row.m, c);
    large = q == INFINITY;
    off = -q;
    factor = -k / row.s * (large ? 1.0f : exp2_fast(m * rest));  // the scale's rest: at the largest logit for all
  }
  __device__ __forceinline__ float minus_p(float z) const {
    return factor * exp2_fast(large ? (z - m) * c : fmaf(z, c, off));
  }
  // (scalar arithmetic: the exponentials' results would have to be moved into pairs)
  template <typename T>
  __device__ __forceinline__ void put(T* out, int j0, const Raw8<T>& raw) const {
    float z[8];
    unpack8(raw, z);
    if (large) {  // uniform
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = minus_p(z[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = factor * exp2_fast(fmaf(z[e], c, off));
    }
    const uint32_t at = static_cast<uint32_t>(id - j0);
    if (at < 8u) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e == static_cast<int>(at)) z[e] += k;
    }
    store8(out, z);
  }
  __device__ __forceinline__ float one(float z, int j) const { return minus_p(z) + (j == id ? k : 0.0f); }
};

// A token's gradient row; zeros for k = 0 without reading the logits.
template <typename T>
__device__ __forceinline__ void gradient_row(const T* row, T* out, int vocab, float k, Running sum, int id, float c,
                                             float rest) {
  const bool zero = k == 0.0f;  // NaN is not zero
  const int head = head_of(out, vocab);
  const bool vec = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  const int chunks = (vocab - head) / 8, threads = static_cast<int>(blockDim.x), tid = static_cast<int>(threadIdx.x);
  const GradientRow g(k, sum, id, c, rest);
  auto one = [&](int j) { out[j] = from_float<T>(zero ? 0.0f : g.one(to_float<T>(row[j]), j)); };
  if (zero) {
    const Pair nil[4] = {0ull, 0ull, 0ull, 0ull};
    for (int i = tid; i < chunks; i += threads) store8(out + head + i * 8, nil);
  } else if (vec) {
    const int stride = threads * 8;
    int i = tid, j = head + tid * 8;
    const T* p = row + j;
    T* q = out + j;
    for (; i + (kUnroll - 1) * threads < chunks; i += kUnroll * threads) {
      Raw8<T> raw[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) raw[u] = load8_stream(p + u * stride);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) g.put(q + u * stride, j + u * stride, raw[u]);
      p += kUnroll * stride, q += kUnroll * stride, j += kUnroll * stride;
    }
    for (; i < chunks; i += threads, p += stride, q += stride, j += stride) g.put(q, j, load8_stream(p));
  } else {
    for (int j = head + tid; j < head + chunks * 8; j += threads) one(j);
  }
  const int tail = vocab - head - chunks * 8;
  if (tid < head) one(tid);
  if (tid < tail) one(head + chunks * 8 + tid);
}

// The largest of eight elements.
template <typename T>
__device__ __forceinline__ float largest_of(const Raw8<T>& r) {
  if constexpr (sizeof(T) == 4) {
    float f[8];
    unpack8(r, f);
    return fmaxf(fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])), fmaxf(fmaxf(f[4], f[5]), fmaxf(f[6], f[7])));
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T2* e = reinterpret_cast<const T2*>(r.w);
    const T2 m = __hmax2(__hmax2(e[0], e[1]), __hmax2(e[2], e[3]));
    const float2 f = word_to_floats<T>(*reinterpret_cast<const uint32_t*>(&m));
    return fmaxf(f.x, f.y);
  }
}

// An id as a column, or -1.
__device__ __forceinline__ int in_vocabulary(int64_t id, long long vocab) {
  return id >= 0 && id < vocab ? static_cast<int>(id) : -1;
}

// A token's sequence.
__device__ __forceinline__ long long sequence_of(const PolicyArgs& a, long long t) {
  if (a.tokens < (1ll << 31)) return static_cast<uint32_t>(t) / static_cast<uint32_t>(a.length);
  return t / a.length;
}

// A token's share in the reduction.
__device__ __forceinline__ float share_of(const PolicyArgs& a, const PolicyState& o, long long t) {
  if (a.reduction == kReduceSum) return 1.0f;
  if (a.mask == nullptr) return 1.0f / static_cast<float>(a.tokens);  // both means: sequences of one length
  return o.share[a.reduction == kReduceSequence ? sequence_of(a, t) : 0];
}

// A token's other inputs, on their way to the first thread while the row is read.
struct Inputs {
  float z, adv, old, ref, share;
};

template <bool kGrad, typename T>
__device__ __forceinline__ Inputs inputs_of(const PolicyArgs& a, const PolicyState& o, const T* row, long long t, int id) {
  Inputs in{__uint_as_float(0x7fc00000u), 0.0f, 0.0f, 0.0f, 0.0f};
  if (threadIdx.x == 0 && id >= 0) in.z = to_float<T>(row[id]);  // an id outside the vocabulary makes the loss NaN
  if (kGrad && threadIdx.x == 0) {
    in.share = share_of(a, o, t);
    in.adv = a.adv[a.adv_per_sequence ? sequence_of(a, t) : t];
    if (a.old != nullptr) in.old = a.old[t];
    if (a.ref != nullptr) in.ref = a.ref[t];
  }
  return in;
}

// The derivative of the token's loss by its log-probability (without weights).
__device__ __forceinline__ float slope_of(const PolicyArgs& a, const Inputs& in, const Running& r, float c, float rest) {
  const float q = base_of(r.m, c);
  const float d = q == INFINITY ? (in.z - r.m) * c : fmaf(in.z, rest, fmaf(in.z, c, -q));
  const float lp = d * kLn2 - logf(r.s);
  const float ratio = expf(lp - (a.old != nullptr ? in.old : lp));
  const float kept = fminf(fmaxf(ratio, static_cast<float>(a.least)), static_cast<float>(a.most));
  const float s1 = ratio * in.adv;
  float slope = (in.adv == 0.0f && lp == lp) || s1 > kept * in.adv ? 0.0f : -s1;  // a NaN stays
  if (a.ref != nullptr) slope -= a.kl * expm1f(in.ref - lp);
  return slope;
}

__device__ __forceinline__ float coefficient(const PolicyArgs& a, float share, float slope) {
  return slope == 0.0f ? 0.0f : a.weight * share * slope * static_cast<float>(a.inv_temp);
}

// What a token leaves behind for a row's blocks: shared words.
struct RowWords {
  float2 red[32];
  Running sum;
  float k;
};

// The block's maxima and sums joined and stored with the logit; with kGrad the slope, too, and the row's sum and the
// gradient's coefficient go to w (behind a barrier of the caller's).
template <bool kGrad>
__device__ __forceinline__ void finish_token(const PolicyArgs& a, const PolicyState& o, RowWords& w, Running r, float c,
                                             float rest, const Inputs& in, long long t) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  r.over_warp(c, rest);
  __syncthreads();  // the previous token's words are read
  if (lane == 0) w.red[warp] = make_float2(r.m, r.s);
  __syncthreads();
  if (warp != 0) return;
  const float2 v = lane < static_cast<int>(blockDim.x >> 5) ? w.red[lane] : make_float2(-INFINITY, 0.0f);
  r.m = v.x;
  r.s = v.y;
  r.over_warp(c, rest);
  if (lane != 0) return;
  const float slope = kGrad ? slope_of(a, in, r, c, rest) : 0.0f;
  o.terms[t] = make_float4(in.z, r.m, r.s, slope);
  if (!kGrad) return;
  o.factors[t] = 1.0f;
  w.sum = r;
  w.k = coefficient(a, in.share, slope);
}

// Exponentials of kCount chunks of eight under one maximum.
template <typename T, int kCount>
__device__ __forceinline__ void add_chunks(ChunkSum& r, const Raw8<T> (&raw)[kCount], float c, float rest) {
  float largest = largest_of(raw[0]);
#pragma unroll
  for (int u = 1; u < kCount; ++u) largest = fmaxf(largest, largest_of(raw[u]));
  r.raise(largest, c, rest);
  float s[2] = {0.0f, 0.0f};
  if (r.q != INFINITY) {
#pragma unroll
    for (int u = 0; u < kCount; ++u) {
      Pair z[4];
      unpack8(raw[u], z);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 y = both(fma2(z[k], pair(rest), fma2(z[k], pair(c), pair(-r.q))));
        s[0] += exp2_fast(y.x);
        s[1] += exp2_fast(y.y);
      }
    }
  } else {
#pragma unroll
    for (int u = 0; u < kCount; ++u) {
      float z[8];
      unpack8(raw[u], z);
#pragma unroll
      for (int k = 0; k < 8; ++k) s[k & 1] += exp2_fast((z[k] - r.m) * c);
    }
  }
  r.s += s[0] + s[1];
}

// Any alignment.  kGrad: the gradient as well, for an upstream gradient of 1, from a second read of the row.
template <typename T, bool kGrad>
__global__ void __maxnreg__(kGrad && sizeof(T) == 2 ? 40 : 64)
    policy_rows_kernel(const PolicyArgs a, const PolicyState o, const long long run) {
  __shared__ RowWords w;
  const float c = scale_of(a), rest = scale_rest_of(a, c);
  const int threads = static_cast<int>(blockDim.x), tid = static_cast<int>(threadIdx.x);
  const int vocab = static_cast<int>(a.vocab);
  if (blockIdx.x == 0 && tid == 0) *o.done = 0u;  // for the kernel behind this one
  const long long last = min(a.tokens, (blockIdx.x + 1) * run);
  for (long long t = blockIdx.x * run; t < last; ++t) {
    const T* row = static_cast<const T*>(a.logits) + t * a.ld;
    T* out = kGrad ? static_cast<T*>(o.dlogits) + t * a.vocab : nullptr;
    if (a.mask != nullptr && !a.mask[t]) {  // uniform
      if (kGrad) {
        if (tid == 0) {
          o.terms[t] = make_float4(0.0f, 0.0f, 1.0f, 0.0f);
          o.factors[t] = 1.0f;
        }
        gradient_row(row, out, vocab, 0.0f, {0.0f, 1.0f}, -1, c, rest);
      }
      continue;
    }
    const int id = in_vocabulary(a.ids[t], a.vocab);
    const Inputs in = inputs_of<kGrad>(a, o, row, t, id);
    const int head = head_of(row, vocab);
    const T* body = row + head;
    const int chunks = (vocab - head) / 8;
    ChunkSum sum;
    auto load = [&](const T* p) { return kGrad ? load8_l2(p) : load8_stream(p); };
    const int stride = threads * 8;
    const T* p = body + tid * 8;
    int i = tid;
    for (; i + (kUnroll - 1) * threads < chunks; i += kUnroll * threads, p += kUnroll * stride) {
      Raw8<T> raw[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) raw[u] = load(p + u * stride);
      add_chunks(sum, raw, c, rest);
    }
    for (; i < chunks; i += threads, p += stride) {
      const Raw8<T> raw[1] = {load(p)};
      add_chunks(sum, raw, c, rest);
    }
    // the ends of the row
    const int tail = vocab - head - chunks * 8;
    if (tid < head) sum.add(to_float<T>(row[tid]), c, rest);
    if (tid < tail) sum.add(to_float<T>(body[chunks * 8 + tid]), c, rest);
    finish_token<kGrad>(a, o, w, {sum.m, sum.s}, c, rest, in, t);
    if (kGrad) {
      __syncthreads();
      gradient_row(row, out, vocab, w.k, w.sum, id, c, rest);
    }
  }
}

// Shares of a masked batch's tokens, one a sequence ("sequence") or one for all
// ("mean"): one block counts the mask.  Counts are whole numbers, so their order
// does not matter.
__global__ void __launch_bounds__(1024) policy_shares_kernel(const PolicyArgs a, const PolicyState o) {
  __shared__ int red[32];
  __shared__ int counts[1024];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long sequences = a.tokens / a.length;
  const bool each = a.reduction == kReduceSequence;
  int mine = 0;  // counted tokens, or sequences that have any
  if (!each || sequences <= 1024) {
    counts[threadIdx.x] = 0;
    __syncthreads();
    for (long long base = warp * 32ll; base < a.tokens; base += 1024 * 4) {
      bool on[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const long long t = base + u * 1024 + lane;
        on[u] = t < a.tokens && a.mask[t];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const long long t0 = base + u * 1024;
        if (!each) {
          mine += on[u] ? 1 : 0;
        } else if (t0 < a.tokens) {
          const uint32_t votes = __ballot_sync(0xffffffffu, on[u]);
          const int q = static_cast<int>(sequence_of(a, t0)), left = static_cast<int>(min((q + 1) * a.length - t0, 32ll));
          if (left == 32) {
            if (lane == 0) atomicAdd(&counts[q], __popc(votes));
          } else if (on[u]) {
            atomicAdd(&counts[static_cast<int>(sequence_of(a, t0 + lane))], 1);
          }
        }
      }
    }
    __syncthreads();
    if (each && static_cast<int>(threadIdx.x) < sequences) {
      const int n = counts[threadIdx.x];
      mine = n > 0 ? 1 : 0;
      o.share[threadIdx.x] = 1.0f / static_cast<float>(n > 0 ? n : 1);
    }
  } else {
    for (long long q = warp; q < sequences; q += 32) {
      int n = 0;
      for (long long i = lane; i < a.length; i += 32) n += a.mask[q * a.length + i] ? 1 : 0;
      n = __reduce_add_sync(0xffffffffu, n);
      if (lane == 0) {
        mine += n > 0 ? 1 : 0;
        o.share[q] = 1.0f / static_cast<float>(n > 0 ? n : 1);
      }
    }
  }
  mine = __reduce_add_sync(0xffffffffu, mine);
  if (lane == 0) red[warp] = mine;
  __syncthreads();
  const int total = __reduce_add_sync(0xffffffffu, red[lane]);
  const float share = 1.0f / static_cast<float>(total > 0 ? total : 1);
  if (!each) {
    if (threadIdx.x == 0) o.share[0] = share;
  } else {
    for (long long q = threadIdx.x; q < sequences; q += 1024) o.share[q] *= share;
  }
}

// Sum over a block, in its first thread.
__device__ __forceinline__ PolicySums block_total(PolicySums s, PolicySums* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  s = {warp_sum(s.loss), warp_sum(s.kl), warp_sum(s.clipped)};
  if (lane == 0) red[warp] = s;
  __syncthreads();
  s = lane < static_cast<int>(blockDim.x >> 5) ? red[lane] : PolicySums{0.0, 0.0, 0.0};
  return {warp_sum(s.loss), warp_sum(s.kl), warp_sum(s.clipped)};
}

__device__ __forceinline__ void store_total(const PolicyArgs& a, const PolicyState& o, const PolicySums& s) {
  *o.loss = static_cast<float>(a.weight * s.loss);
  *o.kl = static_cast<float>(s.kl);
  *o.clipped = static_cast<float>(s.clipped);
}

// A token's terms from what its row left, in 64 bits: terms of both signs cancel in the loss, and what 32 bits lose
// in a log-probability has one sign for all tokens (over 12288 tokens a sum was off by 3e-5, and is by 3e-6 like this).
// kExpLow is what the row's exponentials are too small by on the average, measured over whole powers of two: a row
// that one logit dominates has that logit's own error instead (a token that is certain reads up to 6e-8 below 0).  The
// row kernel's slope is formed in 32 bits without it: within 2^-20 or so of a clip border the loss and the clipped
// share may take one side and the gradient the other.
__device__ __forceinline__ PolicySums terms_of(const PolicyArgs& a, const PolicyState& o, long long t, double* logp) {
  constexpr double kExpLow = 5.05e-8;
  const float4 row = o.terms[t];  // logit, largest logit, sum
  const float c = scale_of(a);
  const float q = base_of(row.y, c);
  const double z = row.x, d = q == INFINITY ? z - row.y : z - q / (a.inv_temp * kLog2e);
  double lp = d * a.inv_temp - log(static_cast<double>(row.z)) - kExpLow;
  if (lp > 0.0) lp = 0.0;  // a token that is certain
  const double ratio = a.old != nullptr ? exp(lp - a.old[t]) : (lp == lp ? 1.0 : lp);
  const double adv = a.adv[a.adv_per_sequence ? sequence_of(a, t) : t];
  const double s1 = ratio * adv, s2 = fmin(fmax(ratio, a.least), a.most) * adv;
  PolicySums r{0.0, 0.0, s1 > s2 ? 1.0 : 0.0};
  if (adv != 0.0 || lp != lp) r.loss = s1 > s2 ? -s2 : -s1;  // a NaN stays
  if (a.ref != nullptr) {
    const double away = a.ref[t] - lp;
    r.kl = expm1(away) - away;
    r.loss += a.kl * r.kl;
  }
  *logp = lp;
  return r;
}

// Loss, KL and clipped share: a token a thread, every block kRun of them; the block that is done last adds the
// blocks' sums in their order.
__global__ void __launch_bounds__(kRun) policy_sum_kernel(const PolicyArgs a, const PolicyState o) {
  __shared__ PolicySums red[32];
  __shared__ bool last;
  PolicySums s{0.0, 0.0, 0.0};
  const long long t = static_cast<long long>(blockIdx.x) * kRun + threadIdx.x;
  if (t < a.tokens) {
    double lp = 0.0;
    if (a.mask == nullptr || a.mask[t]) {
      s = terms_of(a, o, t, &lp);
      const double share = share_of(a, o, t);
      s = {share * s.loss, share * s.kl, share * s.clipped};
    }
    o.logp[t] = static_cast<float>(lp);
  }
  s = block_total(s, red);
  if (gridDim.x == 1) {
    if (threadIdx.x == 0) store_total(a, o, s);
    return;
  }
  if (threadIdx.x == 0) {
    o.sums[blockIdx.x] = s;
    __threadfence();
    last = atomicAdd(o.done, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  s = {0.0, 0.0, 0.0};
  for (unsigned i = threadIdx.x; i < gridDim.x; i += kRun) {
    const double* v = &o.sums[i].loss;
    s.loss += __ldcg(v), s.kl += __ldcg(v + 1), s.clipped += __ldcg(v + 2);
  }
  s = block_total(s, red);
  if (threadIdx.x == 0) store_total(a, o, s);
}

template <typename T>
__global__ void __launch_bounds__(1024)
    policy_backward_kernel(const PolicyArgs a, const PolicyState o, const float* grad) {
  const float c = scale_of(a), rest = scale_rest_of(a, c);
  const float g = *grad;
  if (o.factors != nullptr) {
    // rows of this block whose gradient is not for g (a NaN is for nothing)
    int stale = 0;
    for (long long t = blockIdx.x + static_cast<long long>(threadIdx.x) * gridDim.x; t < a.tokens;
         t += static_cast<long long>(blockDim.x) * gridDim.x)
      stale |= o.factors[t] == g ? 0 : 1;
    if (!__syncthreads_or(stale)) return;
  }
  for (long long t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    if (o.factors != nullptr && o.factors[t] == g) continue;  // uniform
    const T* row = static_cast<const T*>(a.logits) + t * a.ld;
    const bool live = a.mask == nullptr || a.mask[t];
    const float4 term = o.terms[t];
    const float slope = live ? term.w : 0.0f;
    const float k = slope == 0.0f ? 0.0f : g * coefficient(a, share_of(a, o, t), slope);
    gradient_row(row, static_cast<T*>(o.dlogits) + t * a.vocab, static_cast<int>(a.vocab), k, {term.y, term.z},
                 k == 0.0f ? -1 : in_vocabulary(a.ids[t], a.vocab), c, rest);
    if (o.factors != nullptr) {
      __syncthreads();  // every thread has read the factor
      if (threadIdx.x == 0) o.factors[t] = g;
    }
  }
}

// Threads of a row's block: about sixteen chunks each.  Without gradient many
// small blocks are best (1024 bf16 rows of 32000: 15.5 us with 128 threads, 16.9 with 256, 18.5 with
// 512).  With it a block waits between its two passes, and rows
// between their reads have to fit in L2 (126 MB): 1500 threads an SM (40
// registers each) with one or two rows of a large vocabulary.  bf16, 128 / 256 / 512 / 768 / 1024 threads: 8192
// rows of 32000 175 / 152 / 161 / 193 / 241 us, 6144 of 100000 427 / 408 / 374 /
// 348 / 410, 6144 of 128257 484 / 464 / 433 / 402 / 445; fp32, 6144 of 64001 558 /
// 543 / 522 / 622 / 590.  Few rows take larger blocks, until the SMs are full (33 rows of
// 32000: 8.8 us with 256, 6.5 with 1024).
int threads_for(const PolicyArgs& a, bool grad) {
  const int most = grad ? 512 : 128;
  int threads = 64;
  while (threads < most && threads * 128ll < a.vocab) threads *= 2;
  if (grad && a.dtype != kDtypeF32 && threads * 128ll < a.vocab) threads = 768;
  while (threads <= 512 && threads * 8ll < a.vocab && 2 * threads * a.tokens <= a.sms * 1536ll) threads *= 2;
  return threads;
}

template <typename T>
int forward_type(const PolicyArgs& a, const PolicyState& s, cudaStream_t stream, int* launches) {
  const bool grad = s.dlogits != nullptr;
  *launches = 2;
  if (a.mask != nullptr && a.reduction != kReduceSum) {
    policy_shares_kernel<<<1, 1024, 0, stream>>>(a, s);
    ++*launches;
  }
  const int threads = threads_for(a, grad);
  const long long resident = a.sms * (1536ll / threads);
  const long long run = a.tokens / (resident * 16) < 1 ? 1 : a.tokens / (resident * 16);
  const unsigned grid = static_cast<unsigned>((a.tokens + run - 1) / run);
  if (grad)
    policy_rows_kernel<T, true><<<grid, threads, 0, stream>>>(a, s, run);
  else
    policy_rows_kernel<T, false><<<grid, threads, 0, stream>>>(a, s, run);
  policy_sum_kernel<<<static_cast<unsigned>(policy_sum_blocks(a.tokens)), kRun, 0, stream>>>(a, s);
  return static_cast<int>(cudaGetLastError());
}

template <typename T>
int backward_type(const PolicyArgs& a, const PolicyState& s, const float* grad, cudaStream_t stream) {
  const int threads = threads_for(a, true);
  const long long cap = a.sms * (1024ll / threads);
  policy_backward_kernel<T><<<static_cast<unsigned>(a.tokens < cap ? a.tokens : cap), threads, 0, stream>>>(a, s, grad);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace

long long policy_sum_blocks(long long tokens) { return (tokens + kRun - 1) / kRun; }

int policy_forward(const PolicyArgs& a, const PolicyState& s, cudaStream_t stream, int* launches) {
  *launches = 0;
  if (a.tokens <= 0) return 0;
  if (a.vocab <= 0 || a.vocab > 0x7fffff00ll || a.length <= 0 || a.tokens % a.length != 0) return static_cast<int>(cudaErrorInvalidValue);
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

int policy_backward(const PolicyArgs& a, const PolicyState& s, const float* grad, cudaStream_t stream) {
  if (a.tokens <= 0) return 0;
  switch (a.dtype) {
    case kDtypeBF16:
      return backward_type<__nv_bfloat16>(a, s, grad, stream);
    case kDtypeF16:
      return backward_type<__half>(a, s, grad, stream);
    case kDtypeF32:
      return backward_type<float>(a, s, grad, stream);
    default:
      return static_cast<int>(cudaErrorInvalidValue);
  }
}

}  // namespace es
