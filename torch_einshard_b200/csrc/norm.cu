// Norms before and after a block, with its gate and the scaled residual stream:
//
//   yh = (y - m_y) r_y      p = yh pw + pb      (post; otherwise p = y)
//   h  = scale x + gate p
//   hh = (h - m_h) r_h      n = hh w + b        (rms: the means m are 0)
//
// and its gradients, with gn = dn w and E the mean over a row:
//
//   D  = dh + r_h (gn - E[gn] - hh E[gn hh])     (rms: without E[gn])
//   dx = scale D     dgate = D p      t = gate pw
//   dy = r_y (t D - E[t D] - yh E[t D yh])
//   dw = sum dn hh   db = sum dn      dpw = sum gate D yh   dpb = sum gate D
//
// D is linear in the two means, so E[t D] and E[t D yh] come from sums that do
// not wait for them: with A = t (dh + r_h gn), B = t r_h, C = t r_h hh,
//   E[t D ..] = E[A ..] - E[gn] E[B ..] - E[gn hh] E[C ..]
// and a row takes ONE reduction of eight sums (three for rms) instead of two
// dependent ones.  h is formed again from x and y in 32 bits, never read back
// rounded.
//
// The kernels are bound by memory (8 bytes a 16-bit element forward, 12
// backward).  A block of d / 8 threads holds a row in registers, eight elements
// a thread; the column sums of the parameters' gradients stay in registers
// (in shared memory above 4096 columns, where registers run out) over the
// block's rows, go to a workspace once a block, and a second kernel adds them
// in a fixed order.  A gate that is constant over the block's rows leaves its
// own sum and dpw's: S1 = sum D yh gives dgate = pw S1 + pb S0 and gate S1.
//
// Rows wider than 8192 take several passes over the row through the caches.
#include "norm.h"

#include "gemm.h"
#include "vec.cuh"

namespace es {
namespace {

constexpr int kE = 8;             // elements of a row a thread holds
constexpr long long kMaxD = 8192; // 1024 threads
constexpr long long kRegSums = 4096;
constexpr long long kMinGroup = 16;
constexpr int kWideThreads = 512; // block of the several-pass kernels

// ------------------------------------------------------------------ element access

// The thread's eight elements of a row: consecutive with kVec, else strided by the block.
template <bool kVec>
__device__ __forceinline__ long long column(int i) {
  return kVec ? static_cast<long long>(threadIdx.x) * kE + i : static_cast<long long>(i) * blockDim.x + threadIdx.x;
}

template <typename T, bool kVec>
struct Elems {
  Raw8<T> raw;
  T e[kVec ? 1 : kE];
  __device__ __forceinline__ void load(const T* row, long long d) {
    if (kVec) {
      if (column<true>(0) < d) raw = load8_stream(row + column<true>(0));
    } else {
#pragma unroll
      for (int i = 0; i < kE; ++i)
        if (column<false>(i) < d) e[kVec ? 0 : i] = row[column<false>(i)];
    }
  }
  __device__ __forceinline__ void get(float (&f)[kE], long long d) const {
    if (kVec) {
      if (column<true>(0) < d) {
        unpack8(raw, f);
        return;
      }
#pragma unroll
      for (int i = 0; i < kE; ++i) f[i] = 0.0f;
    } else {
#pragma unroll
      for (int i = 0; i < kE; ++i) f[i] = column<false>(i) < d ? to_float<T>(e[kVec ? 0 : i]) : 0.0f;
    }
  }
};

template <typename T, bool kVec>
__device__ __forceinline__ void put(T* row, const float (&f)[kE], long long d) {
  if (kVec) {
    if (column<true>(0) < d) store8(row + column<true>(0), f);
  } else {
#pragma unroll
    for (int i = 0; i < kE; ++i)
      if (column<false>(i) < d) row[column<false>(i)] = from_float<T>(f[i]);
  }
}

// A column vector's elements in fp32 (`other` where it is absent).
template <typename T, bool kVec>
__device__ __forceinline__ void param(const NormParam& q, long long offset, float other, float (&f)[kE], long long d) {
  if (q.p == nullptr) {
#pragma unroll
    for (int i = 0; i < kE; ++i) f[i] = other;
    return;
  }
  if (kVec) {
    const long long c = column<true>(0);
    if (c >= d) {
#pragma unroll
      for (int i = 0; i < kE; ++i) f[i] = 0.0f;
    } else if (q.f32) {
      unpack8(load8(static_cast<const float*>(q.p) + offset + c), f);
    } else {
      unpack8(load8(static_cast<const T*>(q.p) + offset + c), f);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kE; ++i) {
      const long long c = column<false>(i);
      f[i] = c >= d ? 0.0f
                    : (q.f32 ? static_cast<const float*>(q.p)[offset + c]
                             : to_float<T>(static_cast<const T*>(q.p)[offset + c]));
    }
  }
}

template <typename T>
__device__ __forceinline__ float param1(const NormParam& q, long long i, float other) {
  if (q.p == nullptr) return other;
  return q.f32 ? static_cast<const float*>(q.p)[i] : to_float<T>(static_cast<const T*>(q.p)[i]);
}

__device__ __forceinline__ long long gate_row(const NormArgs& a, long long row) {
  return a.gate.p == nullptr ? 0 : (row / a.gate_inner) % a.gate_count;
}

// ------------------------------------------------------------------ block reductions

// Sum over the block, in every thread.  `red` holds two sets of 32 words used in
// turn: one barrier a reduction is enough.
struct Reducer {
  float* red;
  int turn = 0;
  __device__ __forceinline__ float sum(float v) {
    v = warp_sum(v);
    const int warps = blockDim.x >> 5;
    if (warps == 1) return v;
    float* set = red + (turn & 1) * 32;
    ++turn;
    if ((threadIdx.x & 31) == 0) set[threadIdx.x >> 5] = v;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    return warp_sum(lane < warps ? set[lane] : 0.0f);
  }
};

// kN sums at once (kN a power of two up to 8): a warp halves the number of
// values a lane carries with every exchange, so eight sums take nine shuffles.
template <int kN>
__device__ __forceinline__ float warp_sums(float (&v)[kN]) {
  const int lane = threadIdx.x & 31;
  int off = 16;
#pragma unroll
  for (int n = kN; n > 1; n >>= 1, off >>= 1) {
    const bool up = (lane & off) != 0;
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const float give = up ? v[i] : v[i + n / 2];
      const float keep = up ? v[i + n / 2] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, off);
    }
  }
  float r = v[0];
  for (; off > 0; off >>= 1) r += __shfl_xor_sync(0xffffffffu, r, off);
  return r;  // lane l holds the sum whose index is its top log2(kN) bits
}

// The kN sums of the block in every thread; red: 2 x 32 x kN words, in turn.
template <int kN>
__device__ __forceinline__ void block_sums(float (&v)[kN], float* red, int& turn) {
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  constexpr int kSpan = 32 / kN;  // lanes that hold one sum
  const float mine = warp_sums<kN>(v);
  if (warps == 1) {
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = __shfl_sync(0xffffffffu, mine, i * kSpan);
    return;
  }
  float* set = red + (turn & 1) * 32 * kN;
  ++turn;
  if (lane % kSpan == 0) set[(threadIdx.x >> 5) * kN + lane / kSpan] = mine;
  __syncthreads();
  // warp w's sum i at set[w kN + i]: every lane adds one index over some warps, then exchanges
  const int i = lane % kN;
  float s = 0.0f;
  for (int w = lane / kN; w < warps; w += kSpan) s += set[w * kN + i];
#pragma unroll
  for (int off = kN; off < 32; off <<= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
#pragma unroll
  for (int k = 0; k < kN; ++k) v[k] = __shfl_sync(0xffffffffu, s, k);
}

// ------------------------------------------------------------------ forward

template <typename T, bool kVec, bool kPost>
__global__ void __launch_bounds__(1024) norm_forward_kernel(const NormArgs a, const NormForward o) {
  __shared__ float red[64];
  Reducer r{red};
  const float inv_d = 1.0f / static_cast<float>(a.d);
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    Elems<T, kVec> ex, ey;
    ex.load(static_cast<const T*>(a.x) + row * a.ldx, a.d);
    if (a.y != nullptr) ey.load(static_cast<const T*>(a.y) + row * a.ldy, a.d);
    float h[kE], q[kE];
    ex.get(h, a.d);
    float my = 0.0f, ry = 1.0f;
    if (a.y != nullptr) {
      float p[kE];
      ey.get(p, a.d);
      if (kPost) {
        if (a.center) {
          float s = 0.0f;
#pragma unroll
          for (int i = 0; i < kE; ++i) s += p[i];
          my = r.sum(s) * inv_d;
        }
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kE; ++i) {
          p[i] = column<kVec>(i) < a.d ? p[i] - my : 0.0f;
          s += p[i] * p[i];
        }
        ry = 1.0f / sqrtf(r.sum(s) * inv_d + a.eps);
        param<T, kVec>(a.pw, 0, 1.0f, q, a.d);
#pragma unroll
        for (int i = 0; i < kE; ++i) p[i] = p[i] * ry * q[i];
        if (a.pb.p != nullptr) {
          param<T, kVec>(a.pb, 0, 0.0f, q, a.d);
#pragma unroll
          for (int i = 0; i < kE; ++i) p[i] += q[i];
        }
      }
      if (a.gate.p != nullptr) {
        param<T, kVec>(a.gate, gate_row(a, row) * a.d, 1.0f, q, a.d);
#pragma unroll
        for (int i = 0; i < kE; ++i) p[i] *= q[i];
      }
#pragma unroll
      for (int i = 0; i < kE; ++i) h[i] = a.scale * h[i] + p[i];
      put<T, kVec>(static_cast<T*>(o.h) + row * a.d, h, a.d);
    }
    float mh = 0.0f;
    if (a.center) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < kE; ++i) s += column<kVec>(i) < a.d ? h[i] : 0.0f;
      mh = r.sum(s) * inv_d;
    }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kE; ++i) {
      h[i] = column<kVec>(i) < a.d ? h[i] - mh : 0.0f;
      s += h[i] * h[i];
    }
    const float rh = 1.0f / sqrtf(r.sum(s) * inv_d + a.eps);
    param<T, kVec>(a.w, 0, 1.0f, q, a.d);
#pragma unroll
    for (int i = 0; i < kE; ++i) h[i] = h[i] * rh * q[i];
    if (a.b.p != nullptr) {
      param<T, kVec>(a.b, 0, 0.0f, q, a.d);
#pragma unroll
      for (int i = 0; i < kE; ++i) h[i] += q[i];
    }
    put<T, kVec>(static_cast<T*>(o.n) + row * a.d, h, a.d);
    if (o.stats != nullptr && threadIdx.x == 0)
      reinterpret_cast<float4*>(o.stats)[row] = make_float4(my, ry, mh, rh);
  }
}

// Row of any width: several passes through the caches.
template <typename T>
__global__ void __launch_bounds__(kWideThreads) norm_forward_wide_kernel(const NormArgs a, const NormForward o) {
  __shared__ float red[64];
  Reducer r{red};
  const float inv_d = 1.0f / static_cast<float>(a.d);
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* y = a.y == nullptr ? nullptr : static_cast<const T*>(a.y) + row * a.ldy;
    const long long g0 = gate_row(a, row) * a.d;
    float my = 0.0f, ry = 1.0f, mh = 0.0f, s = 0.0f;
    if (a.post) {
      if (a.center) {
        for (long long c = threadIdx.x; c < a.d; c += blockDim.x) s += to_float<T>(y[c]);
        my = r.sum(s) * inv_d;
      }
      s = 0.0f;
      for (long long c = threadIdx.x; c < a.d; c += blockDim.x) {
        const float v = to_float<T>(y[c]) - my;
        s += v * v;
      }
      ry = 1.0f / sqrtf(r.sum(s) * inv_d + a.eps);
    }
    auto stream = [&](long long c) {
      float h = to_float<T>(x[c]);
      if (y == nullptr) return h;
      float p = to_float<T>(y[c]);
      if (a.post) p = (p - my) * ry * param1<T>(a.pw, c, 1.0f) + param1<T>(a.pb, c, 0.0f);
      return a.scale * h + param1<T>(a.gate, g0 + c, 1.0f) * p;
    };
    if (a.center) {
      s = 0.0f;
      for (long long c = threadIdx.x; c < a.d; c += blockDim.x) s += stream(c);
      mh = r.sum(s) * inv_d;
    }
    s = 0.0f;
    for (long long c = threadIdx.x; c < a.d; c += blockDim.x) {
      const float v = stream(c) - mh;
      s += v * v;
    }
    const float rh = 1.0f / sqrtf(r.sum(s) * inv_d + a.eps);
    for (long long c = threadIdx.x; c < a.d; c += blockDim.x) {
      const float h = stream(c);
      if (y != nullptr) static_cast<T*>(o.h)[row * a.d + c] = from_float<T>(h);
      static_cast<T*>(o.n)[row * a.d + c] =
          from_float<T>((h - mh) * rh * param1<T>(a.w, c, 1.0f) + param1<T>(a.b, c, 0.0f));
    }
    if (o.stats != nullptr && threadIdx.x == 0)
      reinterpret_cast<float4*>(o.stats)[row] = make_float4(my, ry, mh, rh);
  }
}

// ------------------------------------------------------------------ backward

// Rows of a unit.
__device__ __forceinline__ void unit_rows(const NormArgs& a, const NormPlan& p, long long unit, long long* first,
                                          long long* last) {
  const long long group = unit / p.slices, slice = unit - group * p.slices;
  const long long per = a.rows / p.groups;
  *first = group * per + slice * p.len;
  *last = slice * p.len + p.len < per ? *first + p.len : (group + 1) * per;
}

// Column sums of a thread: kFull 0: S1 (of D yh), W1 (of dn hh); 1: S0, W0 as well.
// In registers, or in shared memory [sum][column].
template <int kSums, bool kShared>
struct Sums {
  float acc[kShared ? 1 : kSums][kE];
  float* mem;
  long long d;
  __device__ __forceinline__ void init(float* shared, long long d_) {
    mem = shared;
    d = d_;
    if (kShared) {
      for (long long i = threadIdx.x; i < kSums * d; i += blockDim.x) mem[i] = 0.0f;
      __syncthreads();
    } else {
#pragma unroll
      for (int k = 0; k < kSums; ++k)
#pragma unroll
        for (int i = 0; i < kE; ++i) acc[kShared ? 0 : k][i] = 0.0f;
    }
  }
  template <bool kVec>
  __device__ __forceinline__ void add(int k, const float (&v)[kE]) {
    if (!kShared) {
#pragma unroll
      for (int i = 0; i < kE; ++i) acc[kShared ? 0 : k][i] += v[i];
    } else if (kVec) {
      const long long c = column<true>(0);
      if (c < d) {
        float4* m = reinterpret_cast<float4*>(mem + k * d + c);
        float4 u = m[0], w = m[1];
        u.x += v[0], u.y += v[1], u.z += v[2], u.w += v[3];
        w.x += v[4], w.y += v[5], w.z += v[6], w.w += v[7];
        m[0] = u;
        m[1] = w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kE; ++i)
        if (column<false>(i) < d) mem[k * d + column<false>(i)] += v[i];
    }
  }
  template <bool kVec>
  __device__ __forceinline__ void flush(float* ws) {
#pragma unroll
    for (int k = 0; k < kSums; ++k) {
      if (kShared) {
#pragma unroll
        for (int i = 0; i < kE; ++i)
          if (column<kVec>(i) < d) ws[k * d + column<kVec>(i)] = mem[k * d + column<kVec>(i)];
      } else {
        put<float, kVec>(ws + k * d, acc[kShared ? 0 : k], d);
      }
    }
  }
};

template <typename T, bool kVec, bool kPost, bool kFull, bool kShared>
__global__ void __launch_bounds__(kShared ? 1024 : kRegSums / kE)
    norm_backward_kernel(const NormArgs a, const NormPlan plan, const NormBackward o) {
  extern __shared__ float shared[];
  constexpr int kN = kFull ? 8 : 4;
  constexpr int kSums = kFull ? 4 : 2;
  float* red = shared;  // 2 x 32 x kN
  Sums<kSums, kShared> sums;
  sums.init(shared + 64 * kN, a.d);
  const bool want = o.ws != nullptr;
  int turn = 0;
  const float inv_d = 1.0f / static_cast<float>(a.d);
  long long first, last;
  unit_rows(a, plan, blockIdx.x, &first, &last);
  for (long long row = first; row < last; ++row) {
    Elems<T, kVec> ex, ey, eh, en;
    ex.load(static_cast<const T*>(a.x) + row * a.ldx, a.d);
    if (a.y != nullptr) ey.load(static_cast<const T*>(a.y) + row * a.ldy, a.d);
    if (o.dh != nullptr) eh.load(static_cast<const T*>(o.dh) + row * a.d, a.d);
    if (o.dn != nullptr) en.load(static_cast<const T*>(o.dn) + row * a.d, a.d);
    const float4 st = reinterpret_cast<const float4*>(o.stats)[row];
    float x[kE], yh[kE], g[kE], t[kE], u[kE], q[kE];
    ex.get(x, a.d);
#pragma unroll
    for (int i = 0; i < kE; ++i) yh[i] = 0.0f;
    param<T, kVec>(a.gate, gate_row(a, row) * a.d, 1.0f, g, a.d);
    // x becomes hh; t = gate pw
#pragma unroll
    for (int i = 0; i < kE; ++i) t[i] = g[i];
    if (a.y != nullptr) {
      ey.get(yh, a.d);
      float p[kE];
      if (kPost) {
        param<T, kVec>(a.pw, 0, 1.0f, q, a.d);
#pragma unroll
        for (int i = 0; i < kE; ++i) {
          yh[i] = column<kVec>(i) < a.d ? (yh[i] - st.x) * st.y : 0.0f;
          t[i] *= q[i];
          p[i] = yh[i] * q[i];
        }
        if (kFull && a.pb.p != nullptr) {
          param<T, kVec>(a.pb, 0, 0.0f, q, a.d);
#pragma unroll
          for (int i = 0; i < kE; ++i) p[i] += q[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < kE; ++i) p[i] = yh[i];
      }
#pragma unroll
      for (int i = 0; i < kE; ++i) x[i] = a.scale * x[i] + g[i] * p[i];
    }
#pragma unroll
    for (int i = 0; i < kE; ++i) x[i] = column<kVec>(i) < a.d ? (x[i] - st.z) * st.w : 0.0f;
    // u = dh + r_h gn; q = gn
    if (o.dn != nullptr) {
      float dn[kE];
      en.get(dn, a.d);
      param<T, kVec>(a.w, 0, 1.0f, q, a.d);
      if (want) {
        if (kFull) sums.template add<kVec>(3, dn);
#pragma unroll
        for (int i = 0; i < kE; ++i) u[i] = dn[i] * x[i];
        sums.template add<kVec>(1, u);
      }
#pragma unroll
      for (int i = 0; i < kE; ++i) q[i] *= dn[i];
    } else {
#pragma unroll
      for (int i = 0; i < kE; ++i) q[i] = 0.0f;
    }
    if (o.dh != nullptr) {
      eh.get(u, a.d);
    } else {
#pragma unroll
      for (int i = 0; i < kE; ++i) u[i] = 0.0f;
    }
    float v[kN];
#pragma unroll
    for (int k = 0; k < kN; ++k) v[k] = 0.0f;
#pragma unroll
    for (int i = 0; i < kE; ++i) {
      u[i] += st.w * q[i];
      v[0] += q[i] * x[i];
      if (kPost) {
        const float A = t[i] * u[i], B = t[i] * st.w;
        v[1] += A * yh[i];
        v[2] += B * x[i] * yh[i];
        if constexpr (kFull) {
          v[4] += A;
          v[5] += B;
          v[6] += B * x[i];
          v[7] += B * yh[i];
        }
      }
      if constexpr (kFull) v[3] += q[i];
    }
    block_sums<kN>(v, red, turn);
    const float m2 = v[0] * inv_d;
    const float m1 = kFull && a.center ? v[3] * inv_d : 0.0f;
    // u becomes D
#pragma unroll
    for (int i = 0; i < kE; ++i) u[i] = column<kVec>(i) < a.d ? u[i] - st.w * (m1 + m2 * x[i]) : 0.0f;
    if (o.dx != nullptr) {
#pragma unroll
      for (int i = 0; i < kE; ++i) q[i] = a.scale * u[i];
      put<T, kVec>(static_cast<T*>(o.dx) + row * a.d, q, a.d);
    }
    if (a.y == nullptr) continue;
    if (want) {
      if (plan.grouped) {
        if (kFull) sums.template add<kVec>(2, u);
#pragma unroll
        for (int i = 0; i < kE; ++i) q[i] = u[i] * yh[i];
        sums.template add<kVec>(0, q);
      } else {
#pragma unroll
        for (int i = 0; i < kE; ++i) q[i] = u[i] * g[i];
        if (kFull) sums.template add<kVec>(2, q);
#pragma unroll
        for (int i = 0; i < kE; ++i) q[i] *= yh[i];
        sums.template add<kVec>(0, q);
      }
    }
    if (o.dgate_rows != nullptr) {
      // D p, with p formed again
#pragma unroll
      for (int i = 0; i < kE; ++i) q[i] = yh[i];
      if (kPost) {
        float pw[kE];
        param<T, kVec>(a.pw, 0, 1.0f, pw, a.d);
#pragma unroll
        for (int i = 0; i < kE; ++i) q[i] *= pw[i];
        if (kFull && a.pb.p != nullptr) {
          param<T, kVec>(a.pb, 0, 0.0f, pw, a.d);
#pragma unroll
          for (int i = 0; i < kE; ++i) q[i] += pw[i];
        }
      }
#pragma unroll
      for (int i = 0; i < kE; ++i) q[i] *= u[i];
      if (o.dgate_f32)
        put<float, kVec>(static_cast<float*>(o.dgate_rows) + row * a.d, q, a.d);
      else
        put<T, kVec>(static_cast<T*>(o.dgate_rows) + row * a.d, q, a.d);
    }
    if (o.dy != nullptr) {
      if (kPost) {
        float e2 = (v[1] - m2 * v[2]) * inv_d, e1 = 0.0f;
        if constexpr (kFull) {
          if (a.center) {
            e2 -= m1 * v[7] * inv_d;
            e1 = (v[4] - m1 * v[5] - m2 * v[6]) * inv_d;
          }
        }
#pragma unroll
        for (int i = 0; i < kE; ++i) q[i] = st.y * (t[i] * u[i] - e1 - yh[i] * e2);
      } else {
#pragma unroll
        for (int i = 0; i < kE; ++i) q[i] = g[i] * u[i];
      }
      put<T, kVec>(static_cast<T*>(o.dy) + row * a.d, q, a.d);
    }
  }
  if (want) sums.template flush<kVec>(o.ws + blockIdx.x * static_cast<long long>(kSums) * a.d);
}

// Terms of one element, for the several-pass kernels.
template <typename T>
struct Terms {
  float yh, g, t, p, hh, gn, dn, dh;
  __device__ __forceinline__ Terms(const NormArgs& a, const NormBackward& o, long long row, long long c,
                                   const float4& st, long long g0) {
    const float x = to_float<T>(static_cast<const T*>(a.x)[row * a.ldx + c]);
    yh = a.y == nullptr ? 0.0f : to_float<T>(static_cast<const T*>(a.y)[row * a.ldy + c]);
    g = t = param1<T>(a.gate, g0 + c, 1.0f);
    p = yh;
    if (a.post) {
      const float pw = param1<T>(a.pw, c, 1.0f);
      yh = (yh - st.x) * st.y;
      t *= pw;
      p = yh * pw + param1<T>(a.pb, c, 0.0f);
    }
    hh = ((a.y == nullptr ? x : a.scale * x + g * p) - st.z) * st.w;
    dn = o.dn == nullptr ? 0.0f : to_float<T>(static_cast<const T*>(o.dn)[row * a.d + c]);
    dh = o.dh == nullptr ? 0.0f : to_float<T>(static_cast<const T*>(o.dh)[row * a.d + c]);
    gn = dn * param1<T>(a.w, c, 1.0f);
  }
};

template <typename T>
__global__ void __launch_bounds__(kWideThreads)
    norm_backward_wide_kernel(const NormArgs a, const NormBackward o) {
  __shared__ float red[64];
  Reducer r{red};
  const float inv_d = 1.0f / static_cast<float>(a.d);
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float4 st = reinterpret_cast<const float4*>(o.stats)[row];
    const long long g0 = gate_row(a, row) * a.d;
    float s1 = 0.0f, s2 = 0.0f;
    for (long long c = threadIdx.x; c < a.d; c += blockDim.x) {
      const Terms<T> e(a, o, row, c, st, g0);
      s1 += e.gn;
      s2 += e.gn * e.hh;
    }
    const float c2 = r.sum(s2) * inv_d * st.w;
    const float c1 = a.center ? r.sum(s1) * inv_d * st.w : 0.0f;
    float e1 = 0.0f, e2 = 0.0f;
    if (a.post) {
      s1 = s2 = 0.0f;
      for (long long c = threadIdx.x; c < a.d; c += blockDim.x) {
        const Terms<T> e(a, o, row, c, st, g0);
        const float tD = e.t * (e.dh + st.w * e.gn - c1 - c2 * e.hh);
        s1 += tD;
        s2 += tD * e.yh;
      }
      e2 = r.sum(s2) * inv_d;
      e1 = a.center ? r.sum(s1) * inv_d : 0.0f;
    }
    if (threadIdx.x == 0) reinterpret_cast<float4*>(o.coef)[row] = make_float4(c1, c2, e1, e2);
    for (long long c = threadIdx.x; c < a.d; c += blockDim.x) {
      const Terms<T> e(a, o, row, c, st, g0);
      const float D = e.dh + st.w * e.gn - c1 - c2 * e.hh;
      if (o.dx != nullptr) static_cast<T*>(o.dx)[row * a.d + c] = from_float<T>(a.scale * D);
      if (a.y == nullptr) continue;
      if (o.dy != nullptr)
        static_cast<T*>(o.dy)[row * a.d + c] =
            from_float<T>(a.post ? st.y * (e.t * D - e1 - e.yh * e2) : e.g * D);
      if (o.dgate_rows != nullptr) {
        if (o.dgate_f32)
          static_cast<float*>(o.dgate_rows)[row * a.d + c] = D * e.p;
        else
          static_cast<T*>(o.dgate_rows)[row * a.d + c] = from_float<T>(D * e.p);
      }
    }
  }
}

// Column sums of one unit for 256 columns: block (column tile, unit), a thread a column.
template <typename T>
__global__ void __launch_bounds__(256)
    norm_columns_kernel(const NormArgs a, const NormPlan plan, const NormBackward o) {
  const long long c = blockIdx.x * 256ll + threadIdx.x;
  if (c >= a.d) return;
  long long first, last;
  for (long long unit = blockIdx.y; unit < plan.units(); unit += gridDim.y) {
    unit_rows(a, plan, unit, &first, &last);
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (long long row = first; row < last; ++row) {
      const float4 st = reinterpret_cast<const float4*>(o.stats)[row];
      const float4 cf = reinterpret_cast<const float4*>(o.coef)[row];
      const Terms<T> e(a, o, row, c, st, gate_row(a, row) * a.d);
      const float D = (e.dh + st.w * e.gn - cf.x - cf.y * e.hh) * (plan.grouped ? 1.0f : e.g);
      s[0] += D * e.yh;
      s[1] += e.dn * e.hh;
      s[2] += D;
      s[3] += e.dn;
    }
    for (int k = 0; k < plan.sums(); ++k) o.ws[(unit * plan.sums() + k) * a.d + c] = s[k];
  }
}

// The units' sums to gradients: block (tile of 32 columns, y): y = 0 the
// parameters, y = 1 + group the gate's row.  32 threads walk the columns, 32 the
// units; fixed order.
__device__ __forceinline__ void put1(void* p, int f32, int dtype, long long i, float v) {
  if (f32)
    static_cast<float*>(p)[i] = v;
  else if (dtype == kDtypeBF16)
    static_cast<__nv_bfloat16*>(p)[i] = from_float<__nv_bfloat16>(v);
  else if (dtype == kDtypeF16)
    static_cast<__half*>(p)[i] = from_float<__half>(v);
  else
    static_cast<float*>(p)[i] = v;
}

template <typename T>
__global__ void __launch_bounds__(1024)
    norm_finish_kernel(const NormArgs a, const NormPlan plan, const float* ws, const NormSums o) {
  __shared__ float part[4][32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const long long c = blockIdx.x * 32ll + lane;
  const int n = plan.sums();
  for (long long job = blockIdx.y; job <= (o.dgate != nullptr ? plan.groups : 0); job += gridDim.y) {
    const long long first = job == 0 ? 0 : (job - 1) * plan.slices;
    const long long last = job == 0 ? plan.units() : job * plan.slices;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (c < a.d) {
      for (long long unit = first + w; unit < last; unit += 32) {
        const float* u = ws + unit * n * a.d + c;
        const float g = job == 0 && plan.grouped ? param1<T>(a.gate, unit / plan.slices * a.d + c, 1.0f) : 1.0f;
        s[0] += g * u[0];
        s[1] += u[a.d];
        if (n == 4) {
          s[2] += g * u[2 * a.d];
          s[3] += u[3 * a.d];
        }
      }
    }
    __syncthreads();  // the previous job's sums are read
#pragma unroll
    for (int k = 0; k < 4; ++k) part[k][w][lane] = s[k];
    __syncthreads();
    if (w < 4) {
      float v = 0.0f;
#pragma unroll 8
      for (int i = 0; i < 32; ++i) v += part[w][i][lane];
      part[w][0][lane] = v;  // read and written by this warp alone
    }
    __syncthreads();
    if (w == 0 && c < a.d) {
      const float s1 = part[0][0][lane], w1 = part[1][0][lane], s0 = part[2][0][lane], w0 = part[3][0][lane];
      if (job == 0) {
        if (o.dw != nullptr) put1(o.dw, a.w.f32, a.dtype, c, w1);
        if (o.db != nullptr) put1(o.db, a.b.f32, a.dtype, c, w0);
        if (o.dpw != nullptr) put1(o.dpw, a.pw.f32, a.dtype, c, s1);
        if (o.dpb != nullptr) put1(o.dpb, a.pb.f32, a.dtype, c, s0);
      } else {
        const float v = a.post ? param1<T>(a.pw, c, 1.0f) * s1 + (n == 4 ? param1<T>(a.pb, c, 0.0f) * s0 : 0.0f) : s1;
        put1(o.dgate, a.gate.f32, a.dtype, (job - 1) * a.d + c, v);
      }
    }
  }
}

// ------------------------------------------------------------------ launches

int threads_for(long long d) { return static_cast<int>(((d + kE - 1) / kE + 31) / 32 * 32); }

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

bool vector_rows(const NormArgs& a) {
  const int per = a.dtype == kDtypeF32 ? 4 : 8;
  return a.d % 8 == 0 && a.ldx % per == 0 && a.ldy % per == 0 && aligned(a.x) && aligned(a.y) && aligned(a.w.p) &&
         aligned(a.b.p) && aligned(a.pw.p) && aligned(a.pb.p) && aligned(a.gate.p);
}

int sum_bytes(const NormArgs& a, const NormPlan& plan) {
  return a.d > kRegSums ? static_cast<int>(plan.sums() * a.d * sizeof(float)) : 0;
}

template <typename T, bool kVec, bool kPost>
int forward_rows(const NormArgs& a, const NormForward& f, cudaStream_t stream) {
  const int threads = threads_for(a.d);
  // enough blocks to fill the SMs' 2048 threads (at most 32 blocks an SM), rows in turn
  const long long per_sm = 2048 / threads < 32 ? 2048 / threads : 32;
  const long long cap = a.sms * per_sm;
  const int grid = static_cast<int>(a.rows < cap ? a.rows : cap);
  norm_forward_kernel<T, kVec, kPost><<<grid, threads, 0, stream>>>(a, f);
  return static_cast<int>(cudaGetLastError());
}

template <typename T>
int forward_type(const NormArgs& a, const NormForward& f, cudaStream_t stream) {
  if (!norm_in_registers(a)) {
    const long long cap = a.sms * 4ll;
    norm_forward_wide_kernel<T><<<static_cast<int>(a.rows < cap ? a.rows : cap), kWideThreads, 0, stream>>>(a, f);
    return static_cast<int>(cudaGetLastError());
  }
  const bool vec = vector_rows(a) && aligned(f.h) && aligned(f.n);
  if (vec) return a.post ? forward_rows<T, true, true>(a, f, stream) : forward_rows<T, true, false>(a, f, stream);
  return a.post ? forward_rows<T, false, true>(a, f, stream) : forward_rows<T, false, false>(a, f, stream);
}

template <typename T, bool kVec, bool kPost, bool kFull, bool kShared>
int backward_rows(const NormArgs& a, const NormPlan& plan, const NormBackward& b, cudaStream_t stream) {
  auto kernel = norm_backward_kernel<T, kVec, kPost, kFull, kShared>;
  const int bytes = 64 * (kFull ? 8 : 4) * static_cast<int>(sizeof(float)) + (kShared ? sum_bytes(a, plan) : 0);
  if (bytes > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  kernel<<<static_cast<unsigned>(plan.units()), threads_for(a.d), bytes, stream>>>(a, plan, b);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, bool kVec, bool kPost>
int backward_sums(const NormArgs& a, const NormPlan& plan, const NormBackward& b, cudaStream_t stream) {
  if (a.d > kRegSums)
    return plan.full ? backward_rows<T, kVec, kPost, true, true>(a, plan, b, stream)
                     : backward_rows<T, kVec, kPost, false, true>(a, plan, b, stream);
  return plan.full ? backward_rows<T, kVec, kPost, true, false>(a, plan, b, stream)
                   : backward_rows<T, kVec, kPost, false, false>(a, plan, b, stream);
}

template <typename T>
int backward_type(const NormArgs& a, const NormPlan& plan, const NormBackward& b, const NormSums& s,
                  cudaStream_t stream, int* launches) {
  *launches = 1;
  int rc;
  if (norm_in_registers(a)) {
    const bool vec = vector_rows(a) && aligned(b.dh) && aligned(b.dn) && aligned(b.dx) && aligned(b.dy) &&
                     aligned(b.dgate_rows) && aligned(b.ws);
    if (vec)
      rc = a.post ? backward_sums<T, true, true>(a, plan, b, stream) : backward_sums<T, true, false>(a, plan, b, stream);
    else
      rc = a.post ? backward_sums<T, false, true>(a, plan, b, stream)
                  : backward_sums<T, false, false>(a, plan, b, stream);
  } else {
    const long long cap = a.sms * 4ll;
    norm_backward_wide_kernel<T><<<static_cast<int>(a.rows < cap ? a.rows : cap), kWideThreads, 0, stream>>>(a, b);
    rc = static_cast<int>(cudaGetLastError());
    if (rc == 0 && b.ws != nullptr) {
      const dim3 grid(static_cast<unsigned>((a.d + 255) / 256),
                      static_cast<unsigned>(plan.units() < 65535 ? plan.units() : 65535));
      norm_columns_kernel<T><<<grid, 256, 0, stream>>>(a, plan, b);
      rc = static_cast<int>(cudaGetLastError());
      ++*launches;
    }
  }
  if (rc != 0 || b.ws == nullptr) return rc;
  const long long jobs = 1 + (s.dgate != nullptr ? plan.groups : 0);
  const dim3 grid(static_cast<unsigned>((a.d + 31) / 32), static_cast<unsigned>(jobs < 65535 ? jobs : 65535));
  norm_finish_kernel<T><<<grid, 1024, 0, stream>>>(a, plan, b.ws, s);
  ++*launches;
  return static_cast<int>(cudaGetLastError());
}

}  // namespace

bool norm_in_registers(const NormArgs& a) { return a.d <= kMaxD; }

NormPlan norm_plan(const NormArgs& a) {
  NormPlan p;
  p.full = a.center || a.b.p != nullptr || a.pb.p != nullptr;
  // a gate of one row, or of a row for every gate_inner consecutive ones (a unit's sums are as long as 2 to 4
  // rows in fp32: shorter groups are left to a sum over the rows' products)
  p.grouped = a.gate.p != nullptr && a.gate_inner * a.gate_count == a.rows && a.gate_inner >= kMinGroup;
  p.groups = p.grouped ? a.gate_count : 1;
  const long long per = a.rows / p.groups;
  // resident blocks: about 96 registers a thread, or the shared sums' bytes
  const int threads = a.d <= kMaxD ? threads_for(a.d) : kWideThreads;
  long long per_sm = 65536 / (96ll * threads);
  if (a.d > kRegSums) per_sm = 1;
  if (per_sm > 16) per_sm = 16;
  long long slices = a.sms * per_sm / p.groups;
  if (slices > per) slices = per;
  if (slices < 1) slices = 1;
  p.len = (per + slices - 1) / slices;
  p.slices = (per + p.len - 1) / p.len;
  return p;
}

int norm_forward(const NormArgs& a, const NormForward& f, cudaStream_t stream) {
  if (a.rows <= 0 || a.d <= 0) return 0;
  switch (a.dtype) {
    case kDtypeBF16:
      return forward_type<__nv_bfloat16>(a, f, stream);
    case kDtypeF16:
      return forward_type<__half>(a, f, stream);
    case kDtypeF32:
      return forward_type<float>(a, f, stream);
    default:
      return static_cast<int>(cudaErrorInvalidValue);
  }
}

int norm_backward(const NormArgs& a, const NormPlan& plan, const NormBackward& b, const NormSums& s,
                  cudaStream_t stream, int* launches) {
  *launches = 0;
  if (a.rows <= 0 || a.d <= 0) return 0;
  switch (a.dtype) {
    case kDtypeBF16:
      return backward_type<__nv_bfloat16>(a, plan, b, s, stream, launches);
    case kDtypeF16:
      return backward_type<__half>(a, plan, b, s, stream, launches);
    case kDtypeF32:
      return backward_type<float>(a, plan, b, s, stream, launches);
    default:
      return static_cast<int>(cudaErrorInvalidValue);
  }
}

}  // namespace es
