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
// Memory is the bound (8 bytes a 16-bit element forward, 12 backward), and a
// row's fixed work (reductions, addresses) comes next: a thread holds 16
// elements, arithmetic is in fp32 pairs, and rows come through shared memory by
// asynchronous copies, up to three ahead of the one at work.  The column sums of
// the parameters' gradients stay in registers (in shared memory above 4096
// columns a block) over a block's rows, go to a workspace once a block, and a
// second kernel adds them in a fixed order.  A gate that is constant over the
// block's rows leaves its own sum and dpw's: S1 = sum D yh gives
// dgate = pw S1 + pb S0 and gate S1.  Rows too wide for a block are shared by a
// cluster, still wider ones take several passes through the caches.
//
// Measured, forward / backward with the finishing pass: 8192 rows of 2048 bf16
// (layer, both norms, a gate a channel) 31 / 67 us, 4.4 and 3.0 TB/s of what has to
// move; 16387 rows of 8192 (rms, a gate a sequence) 232 / 320 us, 4.6 and 5.0 TB/s;
// 5331 rows of 1001 fp32, not aligned (layer, a gate a token) 31 / 55 us.  A
// division a row to find its gate's row cost 8 % of the second.  What is
// left is the time between a row's last load and its reductions' results: with 16
// elements a thread an SM has one to four rows at work.
#include "norm.h"

#include "gemm.h"
#include "ptx.cuh"
#include "vec.cuh"

#include <type_traits>

namespace es {
namespace {

// A thread holds 2 kP columns of a row, as kP pairs.
constexpr int kThreads = 512;       // most threads a block has
constexpr int kRowPairs = 8;
constexpr int kNarrow = kThreads * kRowPairs;  // columns of a block whose threads hold half as many
constexpr int kMaxCluster = 8;
constexpr int kWideThreads = 512;   // block of the several-pass kernels
constexpr long long kMinGroup = 16;
constexpr int kMaxStages = 4;       // rows in flight

// How a block reads a row: every thread runs of eight columns (kExact), the last threads fewer (kVec), or
// strided columns of a row without alignment (kAny).
enum Access : int { kAny = 0, kVec = 1, kExact = 2 };

// ------------------------------------------------------------------ element access

// The block's part of a row: columns [c0, c0 + n); a row's blocks take `per` each, the last ones what is left.
struct Span {
  int d, per, c0, n;
  __device__ __forceinline__ int columns_of(int rank) const {
    const int left = d - rank * per;
    return left < per ? (left > 0 ? left : 0) : per;
  }
};

__host__ __device__ __forceinline__ int columns_per_block(long long d, int blocks) {
  return static_cast<int>(((d + blocks - 1) / blocks + 7) / 8 * 8);
}

__device__ __forceinline__ Span span_of(const NormArgs& a, int rank, int blocks) {
  Span s;
  s.d = static_cast<int>(a.d);
  s.per = columns_per_block(a.d, blocks);
  s.c0 = rank * s.per;
  s.n = s.columns_of(rank);
  return s;
}

// First column of the thread's run r of eight (kVec, kExact).
__device__ __forceinline__ int run_of(int r) {
  return (r * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * 8;
}

// Column of the thread's element i.
template <int kA>
__device__ __forceinline__ int column(int i) {
  return kA != kAny ? run_of(i / 8) + i % 8 : i * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x);
}

template <int kA>
__device__ __forceinline__ bool has(int i, const Span& s) {
  return kA == kExact || (kA == kVec ? run_of(i / 8) : column<kAny>(i)) < s.n;
}

// Pair i of a thread's values where its columns exist, else zero.
template <int kA>
__device__ __forceinline__ Pair only(Pair v, int i, const Span& s) {
  if (kA == kExact) return v;
  if (kA == kVec) return has<kVec>(2 * i, s) ? v : 0ull;
  const float2 f = both(v);
  return pair(has<kAny>(2 * i, s) ? f.x : 0.0f, has<kAny>(2 * i + 1, s) ? f.y : 0.0f);
}

// A stream's rows on their way through shared memory.  With runs of eight a
// thread copies its own 16 (32) bytes to its own place and needs no barrier to
// read them.  Otherwise the block copies the aligned 16-byte words that cover its
// columns, and a barrier comes before the read; nothing behind the row's end is read.
template <typename T, int kA, int kP>
struct Stream {
  static constexpr int kW = static_cast<int>(sizeof(T) / 2);  // 16-byte words of a run
  static constexpr int kRuns = kP / 4;
  const T* base;
  long long ld;
  uint4* slots;  // [stages][words]
  int words;
  __device__ __forceinline__ static int words_of(int n) {
    return kA != kAny ? static_cast<int>(blockDim.x) * kRuns * kW
                      : (n * static_cast<int>(sizeof(T)) + 15) / 16 + 1;
  }
  __device__ __forceinline__ void fetch(long long row, int stage, const Span& s) const {
    const T* src = base + row * ld + s.c0;
    uint4* dst = slots + stage * words;
    if (kA != kAny) {
#pragma unroll
      for (int r = 0; r < kRuns; ++r) {
        if (!has<kA>(8 * r, s)) continue;
#pragma unroll
        for (int i = 0; i < kW; ++i)
          copy16_async(dst + (r * kW + i) * blockDim.x + threadIdx.x,
                       reinterpret_cast<const uint4*>(src + run_of(r)) + i);
      }
    } else {
      const uintptr_t first = reinterpret_cast<uintptr_t>(src) & ~static_cast<uintptr_t>(15);
      const uintptr_t end = reinterpret_cast<uintptr_t>(src + s.n);
      for (uintptr_t p = first + 16 * threadIdx.x; p < end; p += 16 * blockDim.x) {
        const int bytes = end - p < 16 ? static_cast<int>(end - p) : 16;
        copy16_async(dst + (p - first) / 16, reinterpret_cast<const void*>(p), bytes);
      }
    }
  }
  __device__ __forceinline__ void read(long long row, int stage, const Span& s, Pair (&f)[kP]) const {
    const uint4* src = slots + stage * words;
    if (kA != kAny) {
#pragma unroll
      for (int r = 0; r < kRuns; ++r) {
        Raw8<T> raw;
#pragma unroll
        for (int i = 0; i < kW; ++i) raw.w[i] = src[(r * kW + i) * blockDim.x + threadIdx.x];
        unpack8(raw, f + 4 * r);
      }
    } else {
      const int off = static_cast<int>((reinterpret_cast<uintptr_t>(base + row * ld + s.c0) & 15) / sizeof(T));
      const T* e = reinterpret_cast<const T*>(src) + off;
#pragma unroll
      for (int i = 0; i < kP; ++i)
        f[i] = pair(has<kAny>(2 * i, s) ? to_float<T>(e[column<kAny>(2 * i)]) : 0.0f,
                    has<kAny>(2 * i + 1, s) ? to_float<T>(e[column<kAny>(2 * i + 1)]) : 0.0f);
    }
  }
};

template <typename T, int kA, int kP>
__device__ __forceinline__ void put(T* row, const Pair (&f)[kP], const Span& s) {
  T* out = row + s.c0;
  if (kA != kAny) {
#pragma unroll
    for (int r = 0; r < kP / 4; ++r)
      if (has<kA>(8 * r, s)) store8(out + run_of(r), f + 4 * r);
  } else {
#pragma unroll
    for (int i = 0; i < kP; ++i) {
      if (has<kAny>(2 * i, s)) out[column<kAny>(2 * i)] = from_float<T>(lo_of(f[i]));
      if (has<kAny>(2 * i + 1, s)) out[column<kAny>(2 * i + 1)] = from_float<T>(hi_of(f[i]));
    }
  }
}

template <int kP>
__device__ __forceinline__ void fill(Pair (&f)[kP], float v) {
#pragma unroll
  for (int i = 0; i < kP; ++i) f[i] = pair(v);
}

template <typename T>
__device__ __forceinline__ float param1(const NormParam& q, long long i, float other) {
  if (q.p == nullptr) return other;
  return q.f32 ? static_cast<const float*>(q.p)[i] : to_float<T>(static_cast<const T*>(q.p)[i]);
}

// A column vector's elements in fp32, `other` where there is none; zero in columns that the row does not have (sums
// over a row take a vector's elements as they are).
template <typename T, int kA, int kP>
__device__ __forceinline__ void param(const NormParam& q, long long offset, float other, Pair (&f)[kP],
                                      const Span& s) {
  if (q.p == nullptr) {
    const Pair v = pair(other);
#pragma unroll
    for (int i = 0; i < kP; ++i) f[i] = only<kA>(v, i, s);
  } else if (kA != kAny) {
#pragma unroll
    for (int r = 0; r < kP / 4; ++r) {
      const long long c = offset + s.c0 + run_of(r);
      if (!has<kA>(8 * r, s)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[4 * r + i] = 0ull;
      } else if (q.f32) {
        unpack8(load8(static_cast<const float*>(q.p) + c), f + 4 * r);
      } else {
        unpack8(load8(static_cast<const T*>(q.p) + c), f + 4 * r);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kP; ++i) {
      float v[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = column<kAny>(2 * i + h);
        v[h] = k < s.n ? param1<T>(q, offset + s.c0 + k, other) : 0.0f;
      }
      f[i] = pair(v[0], v[1]);
    }
  }
}

// f times a column vector, where there is one.
template <typename T, int kA, int kP>
__device__ __forceinline__ void times(const NormParam& q, long long offset, Pair (&f)[kP], const Span& s) {
  if (q.p == nullptr) return;
  Pair v[kP];
  param<T, kA>(q, offset, 1.0f, v, s);
#pragma unroll
  for (int i = 0; i < kP; ++i) f[i] = mul2(f[i], v[i]);
}

// All copies but those of the rows behind the next one have landed.
__device__ __forceinline__ void wait_row(int stages) {
  if (stages >= 4)
    copy_wait<2>();
  else if (stages == 3)
    copy_wait<1>();
  else
    copy_wait<0>();
}

// A row's row of the gate, and the first row behind it that may have another: found by division once a run of rows.
struct GateRow {
  long long at, end;
};

__device__ __forceinline__ GateRow gate_of(const NormArgs& a, long long row) {
  if (a.gate_count == 1) return {0, a.rows};
  if (a.gate_count == a.rows) return {row, row + 1};
  if (a.rows < (1ll << 31)) {
    const uint32_t q = static_cast<uint32_t>(row) / static_cast<uint32_t>(a.gate_inner);
    return {q % static_cast<uint32_t>(a.gate_count), (q + 1ll) * a.gate_inner};
  }
  const long long q = row / a.gate_inner;
  return {q % a.gate_count, (q + 1) * a.gate_inner};
}

// ------------------------------------------------------------------ reductions over a row

// Sum over the block, in every thread, for the several-pass kernels.  `red` holds
// two sets of 32 words used in turn: one barrier a reduction is enough.
struct Reducer {
  float* red;
  int turn = 0;
  __device__ __forceinline__ float sum(float v) {
    v = warp_sum(v);
    const int warps = blockDim.x >> 5;
    float* set = red + (turn & 1) * 32;
    ++turn;
    if ((threadIdx.x & 31) == 0) set[threadIdx.x >> 5] = v;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    return warp_sum(lane < warps ? set[lane] : 0.0f);
  }
};

// Words of the warps of a row's blocks: a warp's words are stored in every block
// of the cluster, one barrier later every thread adds them all in the same
// order.  Two sets in turn: a block writes a set again only behind the next
// barrier, which every reader of it has passed.
constexpr int kMaxWarps = kThreads / 32;

template <int kWords>
struct Exchange {
  float* mem;  // [2][kMaxCluster x kMaxWarps][kWords], at the same place in every block
  int rank, blocks, warps, turn = 0;
  static constexpr int kSet = kMaxCluster * kMaxWarps * kWords;
  // lane l of a warp stores word l of its kWords
  __device__ __forceinline__ const float* share(float word, int lane) {
    float* set = mem + (turn & 1) * kSet;
    ++turn;
    float* at = set + (rank * warps + static_cast<int>(threadIdx.x >> 5)) * kWords + lane;
    if (blocks == 1) {
      if (lane < kWords) *at = word;
      __syncthreads();
    } else {
      if (lane < kWords)
        for (int b = 0; b < blocks; ++b) st_cluster_f32(map_to_cta(at, b), word);
      cluster_sync();
    }
    return set;
  }
};

__host__ __device__ constexpr int exchange_bytes(int words) { return 2 * kMaxCluster * kMaxWarps * words * 4; }

// Mean and sum of squared differences from it (center), or 0 and the sum of
// squares, over a row: the warp's own mean and differences first, then the warps' are
// joined, M2 = sum M2_w + n_w (m_w - m)^2; no difference of large sums is taken.
template <int kA, int kP>
__device__ __forceinline__ void row_stats(const Pair (&v)[kP], const Span& s, const NormArgs& a, float inv_d,
                                          Exchange<2>& ex, float* mean, float* m2) {
  const int lane = threadIdx.x & 31;
  // columns of warp w of block b: counted over the runs or strided passes
  auto count = [&](int b, int w) {
    if (kA == kExact) return 64 * kP;
    const int all = s.columns_of(b);
    int n = 0;
    constexpr int kPasses = kA == kVec ? kP / 4 : 2 * kP, kStep = kA == kVec ? 8 : 1;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int left = all - (i * static_cast<int>(blockDim.x) + w * 32) * kStep;
      n += left < 0 ? 0 : (left < 32 * kStep ? left : 32 * kStep);
    }
    return n;
  };
  Pair t = 0ull;
  float mw = 0.0f;
  if (a.center) {
#pragma unroll
    for (int i = 0; i < kP; ++i) t = add2(t, v[i]);
    const int n = count(ex.rank, threadIdx.x >> 5);
    mw = warp_sum(lo_of(t) + hi_of(t)) *
         (kA == kExact ? 1.0f / (64 * kP) : __fdividef(1.0f, static_cast<float>(n > 0 ? n : 1)));
    t = 0ull;
  }
  const Pair off = pair(-mw);
#pragma unroll
  for (int i = 0; i < kP; ++i) {
    const Pair e = only<kA>(add2(v[i], off), i, s);
    t = fma2(e, e, t);
  }
  const float sq = warp_sum(lo_of(t) + hi_of(t));
  const int entries = ex.warps * ex.blocks;
  if (entries == 1) {
    *mean = mw;
    *m2 = sq;
    return;
  }
  const float2* set = reinterpret_cast<const float2*>(ex.share(lane == 0 ? mw : sq, lane));
  float m = 0.0f, q = 0.0f;
  if (entries <= 4) {
    // few words, of one block: every thread adds them all
    float2 w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = e < entries ? set[e] : make_float2(0.0f, 0.0f);
      q += w[e].y;
    }
    if (a.center) {
      float n[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        n[e] = e < entries ? static_cast<float>(count(0, e)) : 0.0f;
        m += w[e].x * n[e];
      }
      m *= inv_d;
#pragma unroll
      for (int e = 0; e < 4; ++e) q += (w[e].x - m) * (w[e].x - m) * n[e];
    }
  } else if (!a.center) {
    for (int e = lane; e < entries; e += 32) q += set[e].y;
    q = warp_sum(q);
  } else {
    auto of = [&](int e) { return ex.blocks == 1 ? count(0, e) : count(e / ex.warps, e % ex.warps); };
    for (int e = lane; e < entries; e += 32) m += set[e].x * of(e);
    m = warp_sum(m) * inv_d;
    for (int e = lane; e < entries; e += 32) {
      const float2 w = set[e];
      q += w.y + (w.x - m) * (w.x - m) * of(e);
    }
    q = warp_sum(q);
  }
  *mean = m;
  *m2 = q;
}

// kN sums at once (kN 4 or 8): a warp halves the number of values a lane carries
// with every exchange, so eight sums take nine shuffles instead of forty.
template <int kN>
__device__ __forceinline__ void row_sums(float (&v)[kN], Exchange<kN>& ex) {
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
  float mine = v[0];
#pragma unroll
  for (int o = 16 / kN; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  // lane l holds the sum whose number is its top log2(kN) bits: bring sum k to lane k
  mine = __shfl_sync(0xffffffffu, mine, (lane % kN) * (32 / kN));
  const int entries = ex.warps * ex.blocks;
  if (entries > 1) {
    const float* set = ex.share(mine, lane);
    float s = 0.0f;
    for (int e = lane / kN; e < entries; e += 32 / kN) s += set[e * kN + lane % kN];
#pragma unroll
    for (int o = kN; o < 32; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    mine = s;
  }
#pragma unroll
  for (int k = 0; k < kN; ++k) v[k] = __shfl_sync(0xffffffffu, mine, k);
}

// ------------------------------------------------------------------ forward

// Dynamic shared memory: exchange words, then the streams' slots.
template <typename T, int kA, bool kPost>
__global__ void __launch_bounds__(kThreads)
    norm_forward_kernel(const NormArgs a, const NormForward o, const int blocks, const int stages) {
  extern __shared__ __align__(16) unsigned char shared[];
  constexpr int kP = kRowPairs;
  using Rows = Stream<T, kA, kP>;
  const int rank = blocks == 1 ? 0 : static_cast<int>(cluster_ctarank());
  const Span s = span_of(a, rank, blocks);
  Exchange<2> ex{reinterpret_cast<float*>(shared), rank, blocks, static_cast<int>(blockDim.x >> 5)};
  const int words = Rows::words_of(s.columns_of(0));
  uint4* slots = reinterpret_cast<uint4*>(shared + exchange_bytes(2));
  const Rows sx{static_cast<const T*>(a.x), a.ldx, slots, words};
  const Rows sy{static_cast<const T*>(a.y), a.ldy, slots + stages * words, words};
  const float inv_d = 1.0f / static_cast<float>(a.d);
  const long long first = blockIdx.x / blocks, step = gridDim.x / blocks;
  const int ahead = stages - 1;
  auto fetch = [&](long long row, int stage) {
    if (row < a.rows) {
      sx.fetch(row, stage, s);
      if (a.y != nullptr) sy.fetch(row, stage, s);
    }
    copy_commit();
  };
  for (int k = 0; k < ahead; ++k) fetch(first + k * step, k);
  // column vectors in registers: t = gate pw, u = gate pb (t = gate without post), formed anew where the gate's
  // row changes
  Pair t[kP], u[kP], w[kP], b[kP];
  param<T, kA>(a.w, 0, 1.0f, w, s);
  param<T, kA>(a.b, 0, 0.0f, b, s);
  long long gate_until = a.y != nullptr ? 0 : a.rows;
  if (blocks > 1) cluster_sync();  // every block runs before one writes another's words
  int stage = 0;
  for (long long row = first; row < a.rows; row += step) {
    if (row >= gate_until) {
      const GateRow g = gate_of(a, row);
      gate_until = g.end;
      param<T, kA>(a.gate, g.at * a.d, 1.0f, t, s);
      if (kPost) {
        param<T, kA>(a.pb, 0, 0.0f, u, s);
#pragma unroll
        for (int i = 0; i < kP; ++i) u[i] = mul2(u[i], t[i]);
        times<T, kA>(a.pw, 0, t, s);
      }
    }
    wait_row(stages);
    if (kA == kAny) __syncthreads();
    Pair h[kP], p[kP];
    sx.read(row, stage, s, h);
    float my = 0.0f, ry = 1.0f, m2;
    if (a.y != nullptr) sy.read(row, stage, s, p);
    // the slot read a row ago; with kAny every thread has read it before the barrier above
    fetch(row + ahead * step, stage == 0 ? ahead : stage - 1);
    if (a.y != nullptr) {
      const Pair scale = pair(a.scale);
      if (kPost) {
#pragma unroll
        for (int i = 0; i < kP; ++i) p[i] = only<kA>(p[i], i, s);
        row_stats<kA>(p, s, a, inv_d, ex, &my, &m2);
        ry = rsqrtf(m2 * inv_d + a.eps);
        const Pair off = pair(-my), unit = pair(ry);
#pragma unroll
        for (int i = 0; i < kP; ++i)
          h[i] = fma2(scale, h[i], fma2(mul2(add2(p[i], off), unit), t[i], u[i]));
      } else {
#pragma unroll
        for (int i = 0; i < kP; ++i) h[i] = fma2(scale, h[i], mul2(p[i], t[i]));
      }
      put<T, kA>(static_cast<T*>(o.h) + row * a.d, h, s);
    }
#pragma unroll
    for (int i = 0; i < kP; ++i) h[i] = only<kA>(h[i], i, s);
    float mh;
    row_stats<kA>(h, s, a, inv_d, ex, &mh, &m2);
    const float rh = rsqrtf(m2 * inv_d + a.eps);
    const Pair off = pair(-mh), unit = pair(rh);
#pragma unroll
    for (int i = 0; i < kP; ++i) h[i] = fma2(mul2(add2(h[i], off), unit), w[i], b[i]);
    put<T, kA>(static_cast<T*>(o.n) + row * a.d, h, s);
    if (o.stats != nullptr && threadIdx.x == 0 && rank == 0)
      reinterpret_cast<float4*>(o.stats)[row] = make_float4(my, ry, mh, rh);
    stage = stage == ahead ? 0 : stage + 1;
  }
  copy_wait<0>();
  if (blocks > 1) cluster_sync();  // no block leaves while another may still write its words
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
    const long long g0 = gate_of(a, row).at * a.d;
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

// A thread's column sums in registers, or in shared memory [sum][two pairs][thread].
template <int kSums, int kP, bool kShared>
struct Sums {
  Pair acc[kShared ? 1 : kSums][kP];
  ulonglong2* mem;
  __device__ __forceinline__ ulonglong2* at(int k, int q) const {
    return mem + (k * (kP / 2) + q) * blockDim.x + threadIdx.x;
  }
  __device__ __forceinline__ void init(void* shared) {
    mem = static_cast<ulonglong2*>(shared);
#pragma unroll
    for (int k = 0; k < kSums; ++k) {
      if (kShared) {
#pragma unroll
        for (int q = 0; q < kP / 2; ++q) *at(k, q) = make_ulonglong2(0ull, 0ull);
      } else {
#pragma unroll
        for (int i = 0; i < kP; ++i) acc[kShared ? 0 : k][i] = 0ull;
      }
    }
  }
  // sum k += v w
  __device__ __forceinline__ void add(int k, const Pair (&v)[kP], const Pair (&w)[kP]) {
    if (kShared) {
#pragma unroll
      for (int q = 0; q < kP / 2; ++q) {
        const ulonglong2 m = *at(k, q);
        *at(k, q) = make_ulonglong2(fma2(v[2 * q], w[2 * q], m.x), fma2(v[2 * q + 1], w[2 * q + 1], m.y));
      }
    } else {
#pragma unroll
      for (int i = 0; i < kP; ++i) acc[kShared ? 0 : k][i] = fma2(v[i], w[i], acc[kShared ? 0 : k][i]);
    }
  }
  __device__ __forceinline__ void add(int k, const Pair (&v)[kP]) {
    if (kShared) {
#pragma unroll
      for (int q = 0; q < kP / 2; ++q) {
        const ulonglong2 m = *at(k, q);
        *at(k, q) = make_ulonglong2(add2(v[2 * q], m.x), add2(v[2 * q + 1], m.y));
      }
    } else {
#pragma unroll
      for (int i = 0; i < kP; ++i) acc[kShared ? 0 : k][i] = add2(v[i], acc[kShared ? 0 : k][i]);
    }
  }
  template <int kA>
  __device__ __forceinline__ void flush(float* ws, long long pitch, const Span& s) const {
#pragma unroll
    for (int k = 0; k < kSums; ++k) {
      Pair v[kP];
#pragma unroll
      for (int q = 0; q < kP / 2; ++q) {
        if (kShared) {
          const ulonglong2 m = *at(k, q);
          v[2 * q] = m.x;
          v[2 * q + 1] = m.y;
        } else {
          v[2 * q] = acc[kShared ? 0 : k][2 * q];
          v[2 * q + 1] = acc[kShared ? 0 : k][2 * q + 1];
        }
      }
      put<float, kA>(ws + k * pitch, v, s);
    }
  }
};

// Sums: 0 S1 (of D yh, or of gate D yh), 1 W1 (dn hh); kFull: 2 S0, 3 W0 as well.
// kWide: twice the columns a thread.  Its four sums do not fit the registers, and in shared memory they leave no
// room for the column vectors, which then come from the caches row by row.
template <typename T, int kA, bool kPost, bool kFull, bool kWide>
__global__ void __launch_bounds__(kThreads)
    norm_backward_kernel(const NormArgs a, const NormPlan plan, const NormBackward o, const int blocks,
                         const int stages) {
  extern __shared__ __align__(16) unsigned char shared[];
  constexpr int kN = kFull ? 8 : 4;
  constexpr int kSums = kFull ? 4 : 2;
  constexpr int kP = kWide ? kRowPairs : kRowPairs / 2;
  constexpr bool kShared = kWide && kFull;
  using Rows = Stream<T, kA, kP>;
  const int rank = blocks == 1 ? 0 : static_cast<int>(cluster_ctarank());
  const Span s = span_of(a, rank, blocks);
  Exchange<kN> ex{reinterpret_cast<float*>(shared), rank, blocks, static_cast<int>(blockDim.x >> 5)};
  Sums<kSums, kP, kShared> sums;
  sums.init(shared + exchange_bytes(kN));
  const int words = Rows::words_of(s.columns_of(0));
  uint4* slots = reinterpret_cast<uint4*>(shared + exchange_bytes(kN)) + (kShared ? kSums * (kP / 2) * blockDim.x : 0);
  const Rows sx{static_cast<const T*>(a.x), a.ldx, slots, words};
  const Rows sy{static_cast<const T*>(a.y), a.ldy, slots + stages * words, words};
  const Rows sh{static_cast<const T*>(o.dh), a.d, slots + 2 * stages * words, words};
  const Rows sn{static_cast<const T*>(o.dn), a.d, slots + 3 * stages * words, words};
  const float inv_d = 1.0f / static_cast<float>(a.d);
  const long long unit = blockIdx.x / blocks;
  long long first, last;
  unit_rows(a, plan, unit, &first, &last);
  auto fetch = [&](long long row, int stage) {
    if (row < last) {
      sx.fetch(row, stage, s);
      if (a.y != nullptr) sy.fetch(row, stage, s);
      if (o.dh != nullptr) sh.fetch(row, stage, s);
      if (o.dn != nullptr) sn.fetch(row, stage, s);
    }
    copy_commit();
  };
  // with one stage the next row goes to the slot just read
  const int ahead = stages > 1 ? stages - 1 : 1;
  for (int k = 0; k < ahead; ++k) fetch(first + k, k);
  const Pair scale = pair(a.scale);
  // column vectors in shared memory, a thread's own: w, t = gate pw (gate without post) and gate pb, these two
  // formed anew where the gate's row changes
  constexpr int kVectors = kFull ? 3 : 2;
  ulonglong2* vectors = reinterpret_cast<ulonglong2*>(slots + 4 * stages * words);
  auto keep = [&](int k, const Pair (&f)[kP]) {
#pragma unroll
    for (int q = 0; q < kP / 2; ++q)
      vectors[(k * (kP / 2) + q) * blockDim.x + threadIdx.x] = make_ulonglong2(f[2 * q], f[2 * q + 1]);
  };
  long long g0 = 0;  // the gate's row
  auto kept = [&](int k, Pair (&f)[kP]) {
    if constexpr (kShared) {
      param<T, kA>(k == 0 ? a.w : a.gate, k == 0 ? 0 : g0, 1.0f, f, s);
      if (k == 1 && kPost) times<T, kA>(a.pw, 0, f, s);
      if (k == 2) times<T, kA>(a.pb, 0, f, s);
    } else {
#pragma unroll
      for (int q = 0; q < kP / 2; ++q) {
        const ulonglong2 v = vectors[(k * (kP / 2) + q) * blockDim.x + threadIdx.x];
        f[2 * q] = v.x;
        f[2 * q + 1] = v.y;
      }
    }
  };
  if (!kShared) {
    Pair f[kP];
    param<T, kA>(a.w, 0, 1.0f, f, s);
    keep(0, f);
  }
  const bool each = a.y != nullptr && a.gate_count == a.rows;
  long long gate_until = a.y != nullptr ? 0 : a.rows;
  if (blocks > 1) cluster_sync();  // every block runs before one writes another's words
  int stage = 0;
  float4 next_st = first < last ? reinterpret_cast<const float4*>(o.stats)[first] : make_float4(0.0f, 1.0f, 0.0f, 1.0f);
  for (long long row = first; row < last; ++row) {
    const float4 st = next_st;
    if (row + 1 < last) next_st = reinterpret_cast<const float4*>(o.stats)[row + 1];
    const bool turn = each || row >= gate_until;  // another row of the gate
    if (each) {
      g0 = row * a.d;
    } else if (turn) {
      const GateRow g = gate_of(a, row);
      gate_until = g.end;
      g0 = g.at * a.d;
    }
    Pair hh[kP], yh[kP], t[kP], u[kP];
    if (!kShared && turn) {
      param<T, kA>(a.gate, g0, 1.0f, t, s);
      if (kPost) {
        if constexpr (kFull) {
          param<T, kA>(a.pb, 0, 0.0f, u, s);
#pragma unroll
          for (int i = 0; i < kP; ++i) u[i] = mul2(u[i], t[i]);
          keep(2, u);
        }
        times<T, kA>(a.pw, 0, t, s);
      }
      keep(1, t);
    }
    wait_row(stages);
    if (kA == kAny) __syncthreads();
    Pair v[kN];
#pragma unroll
    for (int k = 0; k < kN; ++k) v[k] = 0ull;
    sx.read(row, stage, s, hh);
    if (a.y != nullptr) {
      kept(1, t);
      sy.read(row, stage, s, yh);
      if (kPost && kFull && a.pb.p != nullptr) {
        kept(kVectors - 1, u);
#pragma unroll
        for (int i = 0; i < kP; ++i) hh[i] = fma2(hh[i], scale, u[i]);
      } else {
#pragma unroll
        for (int i = 0; i < kP; ++i) hh[i] = mul2(hh[i], scale);
      }
      if (kPost) {
        const Pair off = pair(-st.x), unit_y = pair(st.y);
#pragma unroll
        for (int i = 0; i < kP; ++i) yh[i] = only<kA>(mul2(add2(yh[i], off), unit_y), i, s);
      }
#pragma unroll
      for (int i = 0; i < kP; ++i) hh[i] = fma2(t[i], yh[i], hh[i]);
    } else {
      fill(yh, 0.0f);
    }
    const Pair rh = pair(st.w);
    {
      const Pair off = pair(-st.z);
#pragma unroll
      for (int i = 0; i < kP; ++i) hh[i] = only<kA>(mul2(add2(hh[i], off), rh), i, s);
    }
    if (o.dh != nullptr) {
      sh.read(row, stage, s, u);
#pragma unroll
      for (int i = 0; i < kP; ++i) u[i] = only<kA>(u[i], i, s);
    } else {
      fill(u, 0.0f);
    }
    if (o.dn != nullptr) {
      Pair dn[kP];
      sn.read(row, stage, s, dn);
#pragma unroll
      for (int i = 0; i < kP; ++i) dn[i] = only<kA>(dn[i], i, s);
      sums.add(1, dn, hh);
      if constexpr (kFull) sums.add(3, dn);
      kept(0, t);
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        dn[i] = mul2(dn[i], t[i]);
        u[i] = fma2(rh, dn[i], u[i]);  // dh + r_h gn
        v[0] = fma2(dn[i], hh[i], v[0]);
        if constexpr (kFull) v[3] = add2(v[3], dn[i]);
      }
    }
    if (kA == kAny && stages == 1) __syncthreads();  // every thread has read the slot
    // the slot read a row ago (a barrier lies between, or it is the thread's own); one stage: this row's, read above
    fetch(row + ahead, stages == 1 ? 0 : (stage == 0 ? ahead : stage - 1));
    if (a.y != nullptr) kept(1, t);
    if (kPost) {
      // B and C without their factor r_h
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        const Pair A = mul2(t[i], u[i]), C = mul2(t[i], hh[i]);
        v[1] = fma2(A, yh[i], v[1]);
        v[2] = fma2(C, yh[i], v[2]);
        if constexpr (kFull) {
          v[4] = add2(v[4], A);
          v[5] = add2(v[5], t[i]);
          v[6] = add2(v[6], C);
          v[7] = fma2(t[i], yh[i], v[7]);
        }
      }
    }
    float e[kN];
#pragma unroll
    for (int k = 0; k < kN; ++k) e[k] = lo_of(v[k]) + hi_of(v[k]);
    row_sums<kN>(e, ex);
#pragma unroll
    for (int k = 0; k < kN; ++k) e[k] *= inv_d;
    const float m2 = e[0];
    float m1 = 0.0f;
    if constexpr (kFull) m1 = a.center ? e[3] : 0.0f;
    // u becomes D
    {
      const Pair c1 = pair(-st.w * m1), c2 = pair(-st.w * m2);
#pragma unroll
      for (int i = 0; i < kP; ++i) u[i] = only<kA>(fma2(c2, hh[i], add2(u[i], c1)), i, s);
    }
    if (o.dx != nullptr) {
#pragma unroll
      for (int i = 0; i < kP; ++i) hh[i] = mul2(scale, u[i]);
      put<T, kA>(static_cast<T*>(o.dx) + row * a.d, hh, s);
    }
    if (a.y != nullptr) {
      if (plan.grouped || a.gate.p == nullptr) {
        sums.add(0, u, yh);
        if constexpr (kFull) sums.add(2, u);
      } else if (kPost) {
        Pair gd[kP];
#pragma unroll
        for (int i = 0; i < kP; ++i) gd[i] = u[i];
        times<T, kA>(a.gate, g0, gd, s);
        sums.add(0, gd, yh);
        if constexpr (kFull) sums.add(2, gd);
      }
      if (o.dgate_rows != nullptr) {
#pragma unroll
        for (int i = 0; i < kP; ++i) hh[i] = yh[i];
        if (kPost) {
          times<T, kA>(a.pw, 0, hh, s);
          if (kFull && a.pb.p != nullptr) {
            Pair c[kP];
            param<T, kA>(a.pb, 0, 0.0f, c, s);
#pragma unroll
            for (int i = 0; i < kP; ++i) hh[i] = add2(hh[i], c[i]);
          }
        }
#pragma unroll
        for (int i = 0; i < kP; ++i) hh[i] = mul2(hh[i], u[i]);
        if (o.dgate_f32)
          put<float, kA>(static_cast<float*>(o.dgate_rows) + row * a.d, hh, s);
        else
          put<T, kA>(static_cast<T*>(o.dgate_rows) + row * a.d, hh, s);
      }
      if (o.dy != nullptr) {
#pragma unroll
        for (int i = 0; i < kP; ++i) u[i] = mul2(t[i], u[i]);
        if (kPost) {
          float e2 = e[1] - st.w * m2 * e[2], e1 = 0.0f;
          if constexpr (kFull) {
            if (a.center) {
              e2 -= st.w * m1 * e[7];
              e1 = e[4] - st.w * (m1 * e[5] + m2 * e[6]);
            }
          }
          const Pair c1 = pair(-e1), c2 = pair(-e2), unit_y = pair(st.y);
#pragma unroll
          for (int i = 0; i < kP; ++i) u[i] = mul2(unit_y, fma2(c2, yh[i], add2(u[i], c1)));
        }
        put<T, kA>(static_cast<T*>(o.dy) + row * a.d, u, s);
      }
    }
    if (stages > 1) stage = stage == ahead ? 0 : stage + 1;
  }
  if (o.ws != nullptr) sums.template flush<kA>(o.ws + unit * kSums * plan.pitch(a.d), plan.pitch(a.d), s);
  copy_wait<0>();
  if (blocks > 1) cluster_sync();  // no block leaves while another may still write its words
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
    const long long g0 = gate_of(a, row).at * a.d;
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
      const Terms<T> e(a, o, row, c, st, gate_of(a, row).at * a.d);
      const float D = (e.dh + st.w * e.gn - cf.x - cf.y * e.hh) * (plan.grouped ? 1.0f : e.g);
      s[0] += D * e.yh;
      s[1] += e.dn * e.hh;
      s[2] += D;
      s[3] += e.dn;
    }
    for (int k = 0; k < plan.sums(); ++k) o.ws[(unit * plan.sums() + k) * plan.pitch(a.d) + c] = s[k];
  }
}

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

// The units' sums to gradients: block (tile of 4 kQuads columns, job).  Job 0: the
// parameters, and the gate's row where it has one; then a job a gate row.  kQuads
// threads walk the columns four at a time, the others the units; the order is
// fixed.  Tiles of 32 columns where there are two for every SM, else of 8 (a
// sector): 592 units of 2048 columns 11.9 us with tiles of 16 and 6.9 with 8; 148
// units in seven gate rows of 8192 columns 44 us with 8, 20 with 16 and 11.4 with 32.
constexpr int kFinishThreads = 256;

template <typename T, int kQuads>
__global__ void __launch_bounds__(kFinishThreads)
    norm_finish_kernel(const NormArgs a, const NormPlan plan, const float* __restrict__ ws, const NormSums o) {
  constexpr int kTile = 4 * kQuads;
  __shared__ float part[4][kFinishThreads / 32][kTile];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int quad = lane % kQuads;  // columns 4 quad .. 4 quad + 3 of the tile
  const int walker = w * (32 / kQuads) + lane / kQuads;
  const long long c4 = static_cast<long long>(blockIdx.x) * kTile + quad * 4;
  const long long c = static_cast<long long>(blockIdx.x) * kTile + threadIdx.x % kTile;
  const int n = plan.sums();
  const long long pitch = plan.pitch(a.d);
  const long long jobs = o.dgate != nullptr && plan.groups > 1 ? 1 + plan.groups : 1;
  for (long long job = blockIdx.y; job < jobs; job += gridDim.y) {
    const long long first = job == 0 ? 0 : (job - 1) * plan.slices;
    const long long last = job == 0 ? plan.units() : job * plan.slices;
    const bool weigh = job == 0 && plan.grouped && plan.groups > 1;  // with the gate of the unit's group
    float s[4][4] = {};
#pragma unroll 4
    for (long long unit = first + walker; unit < last; unit += kFinishThreads / kQuads) {
      float g[4] = {1.0f, 1.0f, 1.0f, 1.0f};
      if (weigh)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c4 + j < a.d) g[j] = param1<T>(a.gate, static_cast<uint32_t>(unit) / static_cast<uint32_t>(plan.slices) * a.d + c4 + j, 1.0f);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (k >= n) break;
        if (c4 >= pitch) break;
        const float4 f = *reinterpret_cast<const float4*>(ws + (unit * n + k) * pitch + c4);
        const float v[4] = {f.x, f.y, f.z, f.w};  // columns behind d hold nothing and go nowhere
        const bool gated = k == 0 || k == 2;
#pragma unroll
        for (int j = 0; j < 4; ++j) s[k][j] += gated ? g[j] * v[j] : v[j];
      }
    }
    __syncthreads();  // the previous job's sums are read
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float v = s[k][j];
#pragma unroll
        for (int o = kQuads; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane < kQuads) part[k][w][quad * 4 + j] = v;
      }
    __syncthreads();
    if (threadIdx.x < kTile && c < a.d) {
      float e[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        e[k] = 0.0f;
#pragma unroll
        for (int i = 0; i < kFinishThreads / 32; ++i) e[k] += part[k][i][threadIdx.x];
      }
      const float s1 = e[0], w1 = e[1], s0 = e[2], w0 = e[3];
      if (job == 0) {
        // one group: the sums of D become those of gate D here
        const float g = plan.grouped && plan.groups == 1 ? param1<T>(a.gate, c, 1.0f) : 1.0f;
        if (o.dw != nullptr) put1(o.dw, a.w.f32, a.dtype, c, w1);
        if (o.db != nullptr) put1(o.db, a.b.f32, a.dtype, c, w0);
        if (o.dpw != nullptr) put1(o.dpw, a.pw.f32, a.dtype, c, g * s1);
        if (o.dpb != nullptr) put1(o.dpb, a.pb.f32, a.dtype, c, g * s0);
      }
      if (o.dgate != nullptr && (job > 0 || plan.groups == 1)) {
        const float v = a.post ? param1<T>(a.pw, c, 1.0f) * s1 + (n == 4 ? param1<T>(a.pb, c, 0.0f) * s0 : 0.0f) : s1;
        put1(o.dgate, a.gate.f32, a.dtype, (job > 0 ? job - 1 : 0) * a.d + c, v);
      }
    }
  }
}

// ------------------------------------------------------------------ launches

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

bool vector_rows(const NormArgs& a) {
  const int per = a.dtype == kDtypeF32 ? 4 : 8;
  return a.d % 8 == 0 && a.ldx % per == 0 && a.ldy % per == 0 && aligned(a.x) && aligned(a.y) && aligned(a.w.p) &&
         aligned(a.b.p) && aligned(a.pw.p) && aligned(a.pb.p) && aligned(a.gate.p);
}

// Columns a block holds: 512 threads' of a 16-bit type, half of them of fp32, whose rows take twice the shared
// memory.
long long block_columns(const NormArgs& a) { return a.dtype == kDtypeF32 ? kNarrow : 2 * kRowPairs * kThreads; }

// Blocks that share a row: one, or a cluster.
int blocks_for(const NormArgs& a) { return static_cast<int>((a.d + block_columns(a) - 1) / block_columns(a)); }

int threads_for(const NormArgs& a, int pairs) {
  const int columns = columns_per_block(a.d, blocks_for(a));
  return ((columns + 2 * pairs - 1) / (2 * pairs) + 31) / 32 * 32;
}

// Backward: 512 threads of four pairs, or of eight.
bool wide_rows(const NormArgs& a) { return columns_per_block(a.d, blocks_for(a)) > kNarrow; }
int backward_pairs(const NormArgs& a) { return wide_rows(a) ? kRowPairs : kRowPairs / 2; }

Access access_of(const NormArgs& a, int pairs, bool others_aligned) {
  if (!vector_rows(a) || !others_aligned) return kAny;
  return a.d == 2ll * pairs * threads_for(a, pairs) * blocks_for(a) ? kExact : kVec;
}

// Bytes of a row's slots in `streams` streams.
int slot_bytes(const NormArgs& a, int pairs, bool vec, int streams) {
  const int size = a.dtype == kDtypeF32 ? 4 : 2;
  const long long per = columns_per_block(a.d, blocks_for(a));
  const long long n = per < a.d ? per : a.d;
  const long long words = vec ? static_cast<long long>(threads_for(a, pairs)) * (pairs / 4) * (size / 2) : (n * size + 15) / 16 + 1;
  return static_cast<int>(streams * words * 16);
}

constexpr int kSharedBytes = 227 * 1024;

// What the row kernels launch with.
struct Launch {
  int threads;
  int fixed;      // bytes of the exchange words and shared sums
  int vectors = 0;  // bytes of the column vectors behind the slots
  int stages;
  int bytes;
  long long resident;  // blocks an SM holds, about
};

Launch backward_launch(const NormArgs& a, const NormPlan& plan, bool vec) {
  Launch l;
  const bool shared = wide_rows(a) && plan.full;
  const int pairs = backward_pairs(a);
  const int threads = l.threads = threads_for(a, pairs);
  l.fixed = exchange_bytes(plan.full ? 8 : 4) + (shared ? plan.sums() * pairs * 8 * threads : 0);
  l.vectors = shared ? 0 : (plan.full ? 3 : 2) * pairs * 8 * threads;
  const int slot = slot_bytes(a, pairs, vec, 4);
  const long long regs = plan.full || wide_rows(a) ? 128 : 112;
  l.resident = 65536 / (regs * threads);
  if (l.resident > 12) l.resident = 12;
  if (l.resident < 1) l.resident = 1;
  // as many rows in flight as an SM's shared memory allows its resident blocks, two at least where one block can
  for (;; --l.resident) {
    l.stages = static_cast<int>((kSharedBytes / l.resident - 1024 - l.fixed - l.vectors) / slot);
    if (l.stages >= 2 || l.resident == 1) break;
  }
  if (l.stages > kMaxStages) l.stages = kMaxStages;
  l.bytes = l.fixed + l.vectors + l.stages * slot;
  return l;
}

Launch forward_launch(const NormArgs& a, bool vec) {
  Launch l;
  l.fixed = exchange_bytes(2);
  const int slot = slot_bytes(a, kRowPairs, vec, 2);
  const int threads = l.threads = threads_for(a, kRowPairs);
  l.resident = 65536 / (128ll * threads);
  if (l.resident < 1) l.resident = 1;
  for (;; --l.resident) {
    l.stages = static_cast<int>((kSharedBytes / l.resident - 1024 - l.fixed) / slot);
    if (l.stages >= 3 || l.resident == 1) break;
  }
  if (l.stages > kMaxStages) l.stages = kMaxStages;
  l.bytes = l.fixed + l.stages * slot;
  return l;
}

template <class Kernel, class... Args>
int launch_rows(Kernel kernel, long long units, const NormArgs& a, const Launch& l, cudaStream_t stream,
                unsigned long long* prepared, Args... args) {
  // the kernel's shared memory limit, once a device (`prepared`: a bit each)
  int dev = 0;
  cudaGetDevice(&dev);
  if (!(*prepared >> dev & 1ull)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedBytes);
    if (e != cudaSuccess) return static_cast<int>(e);
    *prepared |= 1ull << dev;
  }
  const int blocks = blocks_for(a);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(units * blocks));
  cfg.blockDim = dim3(static_cast<unsigned>(l.threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(l.bytes);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(blocks);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = blocks > 1 ? 1 : 0;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, a, args..., blocks, l.stages));
}

template <typename T, int kA, bool kPost>
int forward_rows(const NormArgs& a, const NormForward& f, cudaStream_t stream) {
  const Launch l = forward_launch(a, kA != kAny);
  const long long cap = a.sms * l.resident / blocks_for(a);
  static unsigned long long prepared = 0;
  return launch_rows(norm_forward_kernel<T, kA, kPost>, a.rows < cap ? a.rows : cap, a, l, stream, &prepared, f);
}

template <typename T>
int forward_type(const NormArgs& a, const NormForward& f, cudaStream_t stream) {
  if (!norm_in_registers(a)) {
    const long long cap = a.sms * 4ll;
    norm_forward_wide_kernel<T><<<static_cast<int>(a.rows < cap ? a.rows : cap), kWideThreads, 0, stream>>>(a, f);
    return static_cast<int>(cudaGetLastError());
  }
  switch (access_of(a, kRowPairs, aligned(f.h) && aligned(f.n))) {
    case kExact:
      return a.post ? forward_rows<T, kExact, true>(a, f, stream) : forward_rows<T, kExact, false>(a, f, stream);
    case kVec:
      return a.post ? forward_rows<T, kVec, true>(a, f, stream) : forward_rows<T, kVec, false>(a, f, stream);
    default:
      return a.post ? forward_rows<T, kAny, true>(a, f, stream) : forward_rows<T, kAny, false>(a, f, stream);
  }
}

template <typename T, int kA, bool kPost, bool kFull, bool kWide>
int backward_rows(const NormArgs& a, const NormPlan& plan, const NormBackward& b, cudaStream_t stream) {
  const Launch l = backward_launch(a, plan, kA != kAny);
  static unsigned long long prepared = 0;
  return launch_rows(norm_backward_kernel<T, kA, kPost, kFull, kWide>, plan.units(), a, l, stream, &prepared, plan, b);
}

template <typename T, int kA, bool kPost>
int backward_sums(const NormArgs& a, const NormPlan& plan, const NormBackward& b, cudaStream_t stream) {
  if (wide_rows(a))
    return plan.full ? backward_rows<T, kA, kPost, true, true>(a, plan, b, stream)
                     : backward_rows<T, kA, kPost, false, true>(a, plan, b, stream);
  return plan.full ? backward_rows<T, kA, kPost, true, false>(a, plan, b, stream)
                   : backward_rows<T, kA, kPost, false, false>(a, plan, b, stream);
}

template <typename T>
int backward_type(const NormArgs& a, const NormPlan& plan, const NormBackward& b, const NormSums& s,
                  cudaStream_t stream, int* launches) {
  *launches = 1;
  int rc;
  if (norm_in_registers(a)) {
    switch (access_of(a, backward_pairs(a), aligned(b.dh) && aligned(b.dn) && aligned(b.dx) && aligned(b.dy) &&
                             aligned(b.dgate_rows) && aligned(b.ws))) {
      case kExact:
        rc = a.post ? backward_sums<T, kExact, true>(a, plan, b, stream)
                    : backward_sums<T, kExact, false>(a, plan, b, stream);
        break;
      case kVec:
        rc = a.post ? backward_sums<T, kVec, true>(a, plan, b, stream) : backward_sums<T, kVec, false>(a, plan, b, stream);
        break;
      default:
        rc = a.post ? backward_sums<T, kAny, true>(a, plan, b, stream) : backward_sums<T, kAny, false>(a, plan, b, stream);
    }
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
  const long long jobs = s.dgate != nullptr && plan.groups > 1 ? 1 + plan.groups : 1;
  const auto finish = [&](auto quads) {
    constexpr int kQuads = decltype(quads)::value, kTile = 4 * kQuads;
    const dim3 grid(static_cast<unsigned>((a.d + kTile - 1) / kTile), static_cast<unsigned>(jobs < 65535 ? jobs : 65535));
    norm_finish_kernel<T, kQuads><<<grid, kFinishThreads, 0, stream>>>(a, plan, b.ws, s);
  };
  if ((a.d + 31) / 32 * jobs >= 2 * a.sms)
    finish(std::integral_constant<int, 8>());
  else
    finish(std::integral_constant<int, 2>());
  ++*launches;
  return static_cast<int>(cudaGetLastError());
}

}  // namespace

bool norm_in_registers(const NormArgs& a) { return a.d <= block_columns(a) * kMaxCluster; }

NormPlan norm_plan(const NormArgs& a) {
  NormPlan p;
  p.full = a.center || a.b.p != nullptr || a.pb.p != nullptr;
  // a gate of one row, or of a row for every gate_inner consecutive ones (a unit's sums are as long as 2 to 4
  // rows in fp32: shorter groups are left to a sum over the rows' products)
  p.grouped = a.gate.p != nullptr && a.gate_inner * a.gate_count == a.rows && a.gate_inner >= kMinGroup;
  p.groups = p.grouped ? a.gate_count : 1;
  const long long per = a.rows / p.groups;
  // a unit a resident block (or cluster)
  long long all = a.sms * 4ll;
  if (norm_in_registers(a)) all = a.sms * backward_launch(a, p, vector_rows(a)).resident / blocks_for(a);
  long long slices = all / p.groups;
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
