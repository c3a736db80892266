// Log probabilities of given tokens, entropies and the likeliest tokens of rows of logits, and their gradient.
//
// With m = max x, S = sum e^(x - m): log p_j = x_j - m - log S, and the entropy is log S + sum (m - x) e^(x - m) / S, a sum of terms that are not
// negative, so nothing cancels where a distribution is narrow.  The sums are taken in one pass with a running maximum: y = log2(e) x - R in one
// rounding, S = sum 2^y, E = sum y 2^y, and a larger R moves them by S' = f S, E' = f (E + d S), d = R - R', f = 2^d.  R is log2(e) times the maximum,
// rounded, and a warp's: it moves about five times a row, where one of each lane's own would move in most turns of a warp.  Its rounding, which would
// be 2^-24 of the largest logit in log S, is taken out at the end: log2(e) m - R is known to its last bit.
//
// The bytes of the logits bound both directions (an exponential takes 72 % of the special-function rate at that speed, the arithmetic 45 % of issue).
// The k likeliest tokens cost next to nothing in the pass: each thread keeps the maximum of what it saw.  The k-th largest of the maxima of 64 groups of
// threads is a bound that k logits reach, so only the pieces of threads whose maximum reaches it are looked at again (about k of 256, unless
// logits are equal).
//
// Compiled without fast math: the logarithms at a row's end are the exact ones, the exponentials of its elements the hardware's.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <math_constants.h>

#include "f32x2.cuh"
#include "host.cuh"

namespace {
namespace cg = cooperative_groups;
typedef __nv_bfloat16 bf16;
typedef unsigned long long u64;
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kUnroll = 4;                // 16-byte loads of a thread in flight
constexpr int kTopMax = 32;               // tokens that the selection gives
constexpr int kBuffer = 1024;             // candidates for them
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLow = -1e30f;            // logits below it count as this in the pass: 2^-inf times -inf is no number

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The same with results below 2^-126 kept: a gradient is a probability times numbers that may be large
__device__ __forceinline__ float ex2_small(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float lower(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float upper(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ float value(const bf16* p, long i) { return __bfloat162float(p[i]); }
__device__ __forceinline__ float value(const float* p, long i) { return p[i]; }
__device__ __forceinline__ void store(bf16* p, long i, float x) { p[i] = __float2bfloat16(x); }
__device__ __forceinline__ void store(float* p, long i, float x) { p[i] = x; }

// 16 bytes of a row
template <class T>
struct Vec;
template <>
struct Vec<bf16> {
  static constexpr int kN = 8;
  uint4 w;
  __device__ __forceinline__ float top() const {
    const uint32_t m = max2_nan(max2_nan(w.x, w.y), max2_nan(w.z, w.w));
    return max_nan(lower(m), upper(m));
  }
  __device__ __forceinline__ void floats(float2 (&x)[4]) const {       // none below kLow
    const uint32_t v[4] = {w.x, w.y, w.z, w.w}, low = 0xf149f149u;     // bf16 of -1e30
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t c = max2_nan(v[i], low);
      x[i] = make_float2(lower(c), upper(c));
    }
  }
};
template <>
struct Vec<float> {
  static constexpr int kN = 4;
  float4 w;
  __device__ __forceinline__ float top() const { return max_nan(max_nan(w.x, w.y), max_nan(w.z, w.w)); }
  __device__ __forceinline__ void floats(float2 (&x)[2]) const {
    x[0] = make_float2(max_nan(w.x, kLow), max_nan(w.y, kLow));
    x[1] = make_float2(max_nan(w.z, kLow), max_nan(w.w, kLow));
  }
};
template <class T>
__device__ __forceinline__ Vec<T> load(const T* p) {                   // 16-byte aligned
  Vec<T> v;
  *reinterpret_cast<uint4*>(&v.w) = __ldcs(reinterpret_cast<const uint4*>(p));
  return v;
}

// Order of the likeliest tokens as whole numbers: larger logits first, NaN before all, -0 as 0, then the lower index
__device__ __forceinline__ unsigned ordered(float x) {
  const int bits = x != x ? 0x7fffffff : __float_as_int(x + 0.f);
  return bits >= 0 ? static_cast<unsigned>(bits) | 0x80000000u : ~static_cast<unsigned>(bits);
}
__device__ __forceinline__ u64 rank_of(float x, int i) { return static_cast<u64>(ordered(x)) << 32 | (0xffffffffu - static_cast<unsigned>(i)); }
__device__ __forceinline__ int index_of(u64 r) { return static_cast<int>(0xffffffffu - static_cast<unsigned>(r)); }

// Sums over some logits, of which m is the largest; none yet (or none above kLow) where m is kLow
struct Sums {
  float m, R, S, E;
  __device__ __forceinline__ void move(float to, float to_R) {         // to >= m
    if (m > kLow) {
      const float d = R - to_R, f = ex2(d);
      E = f * fmaf(d, S, E);
      S *= f;
    }
    m = to;
    R = to_R;
  }
  __device__ __forceinline__ void add(Sums o) {
    if (!(o.m > kLow)) return;
    if (o.m > m) move(o.m, o.R); else o.move(m, R);
    S += o.S;
    E += o.E;
  }
};

// A CTA's part of a row: columns lo .. hi, as 16-byte pieces, the first and last of which may reach beyond it.  Piece j is thread j % kThreads'.
template <class T>
struct Part {
  static constexpr int kN = Vec<T>::kN;
  const T* x;           // column 0
  int lo, hi, base;     // the first piece begins at column base <= lo, which is 16-byte aligned
  int pieces;
  __device__ __forceinline__ Part(const T* row, int l, int h) : x(row), lo(l), hi(h) {
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(row + lo) % 16 / sizeof(T));
    base = lo - off;
    pieces = hi > lo ? (hi - base + kN - 1) / kN : 0;
  }
  __device__ __forceinline__ bool whole(int j) const { return (j > 0 || base == lo) && base + (j + 1) * kN <= hi; }
  __device__ __forceinline__ float at(int c) const { return c >= lo && c < hi ? value(x, c) : -CUDART_INF_F; }
};

struct Smem {
  Sums sums[kWarps], all;
  float top[kThreads];
  unsigned group[64], kth;                 // maxima of neighbouring threads; the bound, as `ordered`
  int count, reach, above;
  short list[kThreads];                    // threads whose pieces are looked at again
  u64 buffer[kBuffer];
  u64 best[kTopMax];
  u64 red[kWarps];
};

__device__ __forceinline__ void warp_reduce(Sums& s) {                 // lanes share m
  for (int o = 16; o; o >>= 1) {
    s.S += __shfl_xor_sync(0xffffffffu, s.S, o);
    s.E += __shfl_xor_sync(0xffffffffu, s.E, o);
  }
}

// The sums of a part and the thread's own maximum
template <class T>
__device__ __forceinline__ Sums pass(const Part<T>& p, float& top) {
  constexpr int kN = Vec<T>::kN;
  Sums s{kLow, 0.f, 0.f, 0.f};
  top = -CUDART_INF_F;
  float2 S2 = make_float2(0.f, 0.f), E2 = make_float2(0.f, 0.f);
  auto flush = [&]() {
    s.S += S2.x + S2.y;
    s.E += E2.x + E2.y;
    S2 = E2 = make_float2(0.f, 0.f);
  };
  auto raise = [&](float m) {                                          // of the warp, where a lane's logits exceed it
    if (__any_sync(0xffffffffu, m > s.m)) {
      flush();
      for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      s.move(m, m * kLog2e);
    }
  };
  auto add = [&](const float2 (&x)[kN / 2]) {
    if (s.m == kLow) return;                                           // the same in all lanes
    const float2 a = make_float2(kLog2e, kLog2e), c = make_float2(-s.R, -s.R);
#pragma unroll
    for (int i = 0; i < kN / 2; ++i) {
      const float2 y = fma2(x[i], a, c), e = make_float2(ex2(y.x), ex2(y.y));
      S2 = add2(S2, e);
      E2 = fma2(y, e, E2);
    }
  };
  const T* first = p.x + p.base;
  const int turns = (p.pieces + kThreads - 1) / kThreads;
  int j = threadIdx.x, done = 0;
  // pieces 1 .. pieces - 2 are whole; a turn of kUnroll that all lie there is loaded at once
  for (; done < turns;) {
    const bool all = done > 0 && (done + kUnroll) * kThreads < p.pieces;
    if (all) {
      Vec<T> v[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) v[u] = load(first + static_cast<long>(j + u * kThreads) * kN);
      float m = v[0].top();
#pragma unroll
      for (int u = 1; u < kUnroll; ++u) m = max_nan(m, v[u].top());
      top = max_nan(top, m);
      raise(m);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        float2 x[kN / 2];
        v[u].floats(x);
        add(x);
      }
      j += kUnroll * kThreads;
      done += kUnroll;
    } else {
      float2 x[kN / 2];
      float m = -CUDART_INF_F;
      if (j < p.pieces && p.whole(j)) {
        const Vec<T> v = load(first + static_cast<long>(j) * kN);
        m = v.top();
        v.floats(x);
      } else {
#pragma unroll
        for (int i = 0; i < kN / 2; ++i) {
          const int c = p.base + j * kN + 2 * i;
          const float a = j < p.pieces ? p.at(c) : -CUDART_INF_F, b = j < p.pieces ? p.at(c + 1) : -CUDART_INF_F;
          m = max_nan(m, max_nan(a, b));
          x[i] = make_float2(max_nan(a, kLow), max_nan(b, kLow));
        }
      }
      top = max_nan(top, m);
      raise(m);
      add(x);
      j += kThreads;
      done += 1;
    }
  }
  flush();
  warp_reduce(s);
  if (__any_sync(0xffffffffu, top != top)) s = Sums{fmaxf(s.m, 0.f), s.m > 0.f ? s.R : 0.f, CUDART_NAN_F, CUDART_NAN_F};     // also where no other number was seen
  return s;
}

// The part's k first in rank order, in sm.best (0 behind them).  top: the maximum of the thread's pieces.
template <class T>
__device__ void select(Smem& sm, const Part<T>& p, float top, int k) {
  constexpr int kN = Vec<T>::kN;
  const int t = threadIdx.x, lane = t & 31, have = min(k, p.hi - p.lo);
  const unsigned mine = ordered(top);
  unsigned group = mine;
#pragma unroll
  for (int o = 1; o < kThreads / 64; o *= 2) group = max(group, __shfl_xor_sync(0xffffffffu, group, o));
  if (t % (kThreads / 64) == 0) sm.group[t / (kThreads / 64)] = group;
  if (t == 0) sm.count = sm.reach = sm.above = 0;
  if (t < kTopMax) sm.best[t] = 0;
  __syncthreads();
  if (t < 64) {
    const unsigned g = sm.group[t];
    int before = 0;
#pragma unroll 16
    for (int i = 0; i < 64; ++i) before += sm.group[i] > g || (sm.group[i] == g && i < t);
    if (before == have - 1) sm.kth = g;
  }
  __syncthreads();
  // Logits that reach the bound.  Where many threads' do, logits are equal: then only those above it, and the first of the equal ones in order.
  const unsigned kth = sm.kth;
  if (mine >= kth) atomicAdd(&sm.reach, 1);
  __syncthreads();
  const bool ties = sm.reach > 3 * kTopMax;
  const unsigned bound = ties ? kth : kth - 1;                         // candidates are larger than this (no logit's order is 0)
  if (mine > bound) sm.list[atomicAdd(&sm.above, 1)] = static_cast<short>(t);
  __syncthreads();
  const int turns = (p.pieces + kThreads - 1) / kThreads, again = sm.above * turns;
  for (int i = t; i < again; i += kThreads) {
    const int j = sm.list[i / turns] + i % turns * kThreads;
    if (j >= p.pieces) continue;
    for (int c = 0; c < kN; ++c) {
      const int col = p.base + j * kN + c;
      if (col < p.lo || col >= p.hi) continue;
      const float x = value(p.x, col);
      if (ordered(x) > bound) {
        const int at = atomicAdd(&sm.count, 1);
        if (at < kBuffer) sm.buffer[at] = rank_of(x, col);
      }
    }
  }
  __syncthreads();
  int count = sm.count;
  if (count <= kBuffer) {
    if (ties && count < have) {
      const int missing = have - count;
      int found = 0;
      for (int c0 = p.lo; c0 < p.hi && found < missing; c0 += kThreads) {
        const bool is = c0 + t < p.hi && ordered(value(p.x, c0 + t)) == kth;
        const unsigned mask = __ballot_sync(0xffffffffu, is);
        if (lane == 0) sm.red[t >> 5] = __popc(mask);
        __syncthreads();
        int before = found;
        for (int w = 0; w < kWarps; ++w) {
          if (w < (t >> 5)) before += static_cast<int>(sm.red[w]);
          found += static_cast<int>(sm.red[w]);
        }
        const int at = before + __popc(mask & ((1u << lane) - 1));
        if (is && at < missing) sm.buffer[count + at] = rank_of(value(p.x, c0 + t), c0 + t);
        __syncthreads();
      }
      count += min(found, missing);
    }
    for (int i = t; i < count; i += kThreads) {
      const u64 r = sm.buffer[i];
      int before = 0;
      for (int o = 0; o < count; ++o) before += sm.buffer[o] > r;
      if (before < have) sm.best[before] = r;
    }
    __syncthreads();
    return;
  }
  // more candidates than are kept (the largest logits all in one thread's pieces): one after another
  u64 last = ~0ull;
  for (int n = 0; n < have; ++n) {
    u64 r = 0;
    for (int c = p.lo + t; c < p.hi; c += kThreads) {
      const u64 a = rank_of(value(p.x, c), c);
      if (a < last && a > r) r = a;
    }
    for (int o = 16; o; o >>= 1) {
      const u64 a = __shfl_xor_sync(0xffffffffu, r, o);
      r = a > r ? a : r;
    }
    __syncthreads();
    if (lane == 0) sm.red[t >> 5] = r;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) r = sm.red[w] > r ? sm.red[w] : r;
    last = r;
    if (t == 0) sm.best[n] = r;
  }
  __syncthreads();
}

// One row per cluster, its columns in even parts.
template <class T>
__global__ void __launch_bounds__(kThreads, 4) logprobs_fwd_kernel(const T* __restrict__ logits, long ld, const long long* __restrict__ tokens,
                                                                   float* __restrict__ logprob, float* __restrict__ entropy, float2* __restrict__ stats,
                                                                   float* __restrict__ top_out, long long* __restrict__ index, int V, int k,
                                                                   long long ignore, int parts, KernelStatus* status) {
  __shared__ Smem sm;
  const int t = threadIdx.x, part = blockIdx.x % parts;
  const long row = blockIdx.x / parts;
  const T* x = logits + row * ld;
  const int each = (V + parts - 1) / parts;
  const Part<T> p(x, min(part * each, V), min((part + 1) * each, V));
  float top;
  const Sums s = pass(p, top);
  if ((t & 31) == 0) sm.sums[t >> 5] = s;
  if (k > 0) select(sm, p, top, k);
  __syncthreads();
  if (t == 0) {
    Sums a = sm.sums[0];
    for (int w = 1; w < kWarps; ++w) a.add(sm.sums[w]);
    sm.all = a;
  }
  if (parts > 1) {
    cg::this_cluster().sync();
  } else {
    __syncthreads();
  }
  if (part == 0) {
    Sums a = sm.all;
    for (int c = 1; c < parts; ++c) a.add(*cg::this_cluster().map_shared_rank(&sm.all, c));
    // near kLow the pass has not told logits apart
    float m = a.m, logS = logf(a.S) - fmaf(m, kLog2e, -a.R) * kLn2, H = logf(a.S);
    bool empty = false;
    if (m <= 0.1f * kLow) {
      m = -CUDART_INF_F;
      for (int c = t; c < V; c += kThreads) m = max_nan(m, value(x, c));
      sm.top[t] = m;
      __syncthreads();
      for (int i = 0; i < kThreads; ++i) m = max_nan(m, sm.top[i]);
      empty = m == -CUDART_INF_F;
      float S = 0.f, E = 0.f;
      for (int c = t; c < V && !empty; c += kThreads) {
        const float y = (value(x, c) - m) * kLog2e, e = ex2(y);
        S += e;
        E += e > 0.f ? y * e : e;
      }
      Sums b{0.f, 0.f, S, E};
      warp_reduce(b);
      __syncthreads();
      if ((t & 31) == 0) sm.sums[t >> 5] = b;
      __syncthreads();
      b = Sums{0.f, 0.f, 0.f, 0.f};
      for (int w = 0; w < kWarps; ++w) {
        b.S += sm.sums[w].S;
        b.E += sm.sums[w].E;
      }
      a = b;
      H = logS = empty ? 0.f : logf(a.S);
    }
    H = empty ? 0.f : H - a.E * kLn2 / a.S;
    if (t == 0) {
      const long long tok = tokens[row];
      NSA_CHECK_INDEX(tok == ignore || (tok >= 0 && tok < V), status, tok);
      logprob[row] = tok == ignore || tok < 0 || tok >= V ? 0.f : empty ? m : value(x, tok) - m - logS;
      entropy[row] = H;
      stats[row] = make_float2(m, logS);                               // apart: their sum would round a probability by |m| 2^-24
    }
    // each part's best are in order: a candidate's place is the number of larger ones
    const int n = parts * k;
    for (int i = t; i < n; i += kThreads) sm.buffer[i] = *cg::this_cluster().map_shared_rank(&sm.best[i % k], i / k);
    __syncthreads();
    for (int i = t; i < n; i += kThreads) {
      const u64 r = sm.buffer[i];
      if (r == 0) continue;
      int before = 0;
      for (int o = 0; o < n; ++o) before += sm.buffer[o] > r;
      if (before < k) {
        const int c = index_of(r);
        index[row * k + before] = c;
        top_out[row * k + before] = empty ? m : value(x, c) - m - logS;
      }
    }
  }
  if (parts > 1) cg::this_cluster().sync();                            // the others' memory is read until here
}

// dx_j = -p_j (G + g_H (log p_j + H)), G the sum of the row's other gradients; theirs are added at their tokens.  One CTA per kBwdPieces pieces of a row.
constexpr int kBwdTurns = 4, kBwdPieces = kThreads * kBwdTurns;
template <class T>
__global__ void __launch_bounds__(kThreads) logprobs_bwd_kernel(const T* __restrict__ logits, long ld, const long long* __restrict__ tokens,
                                                                const float2* __restrict__ stats, const float* __restrict__ entropy,
                                                                const long long* __restrict__ index, const float* __restrict__ dlogprob,
                                                                const float* __restrict__ dentropy, const float* __restrict__ dtop,
                                                                T* __restrict__ dx_all, int V, int k, long long ignore, int chunks) {
  constexpr int kN = Vec<T>::kN;
  const int t = threadIdx.x;
  const long row = blockIdx.x / chunks;
  const int chunk = static_cast<int>(blockIdx.x - row * chunks);
  const T* x = logits + row * ld;
  T* dx = dx_all + row * V;
  const float m = stats[row].x, logS = stats[row].y, H = entropy[row], gH = dentropy ? dentropy[row] : 0.f;
  const long long tok = tokens[row];
  const bool counts = !(tok == ignore || tok < 0 || tok >= V), empty = m == -CUDART_INF_F;
  const float g = counts && dlogprob ? dlogprob[row] : 0.f;
  float G = g;
  if (dtop)
    for (int j = 0; j < k; ++j) G += dtop[row * k + j];
  // log2 p = a x + c is taken as (x - m) log2(e) - log2 S: the difference is exact enough where x is large
  const float log2S = logS * kLog2e, c1 = -fmaf(gH, H, G), c2 = -gH * kLn2;
  auto grad = [&](float v) {
    const float y = max_nan(fmaf(v - m, kLog2e, -log2S), -1000.f);
    return ex2_small(y) * fmaf(c2, y, c1);
  };
  // pieces where dx is 16-byte aligned; x is as well, or its elements are loaded one by one
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(dx) % 16 / sizeof(T)), pieces = (V + off + kN - 1) / kN;
  const bool same = (reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) % 16 == 0;
  const int j0 = chunk * kBwdPieces;
  Vec<T> v[kBwdTurns];
  bool whole[kBwdTurns];
#pragma unroll
  for (int u = 0; u < kBwdTurns; ++u) {
    const int j = j0 + u * kThreads + t, c = j * kN - off;
    whole[u] = same && c >= 0 && c + kN <= V;
    if (whole[u]) v[u] = load(x + c);
  }
#pragma unroll
  for (int u = 0; u < kBwdTurns; ++u) {
    const int j = j0 + u * kThreads + t, c = j * kN - off;
    if (j >= pieces) break;
    if (whole[u]) {
      const T* in = reinterpret_cast<const T*>(&v[u].w);
      Vec<T> out;
      T* o = reinterpret_cast<T*>(&out.w);
#pragma unroll
      for (int i = 0; i < kN; ++i) store(o, i, empty ? 0.f : grad(value(in, i)));
      __stcs(reinterpret_cast<uint4*>(dx + c), *reinterpret_cast<const uint4*>(&out.w));
    } else {
      for (int i = 0; i < kN; ++i)
        if (c + i >= 0 && c + i < V) store(dx, c + i, empty ? 0.f : grad(value(x, c + i)));
    }
  }
  if (empty || (!counts && !dtop)) return;
  __syncthreads();
  // the chosen token (t = k) and the likeliest ones, each column once
  const int n = dtop ? k : 0;
  for (int i = t; i <= n; i += kThreads) {
    if (i == n && !counts) continue;
    const long long c = i == n ? tok : index[row * k + i];
    const long piece = (c + off) / kN;
    if (piece < j0 || piece >= j0 + kBwdPieces) continue;
    float d = counts && c == tok ? g : 0.f;
    bool seen = false;
    for (int o = 0; o < n; ++o)
      if (index[row * k + o] == c) {
        d += dtop[row * k + o];
        seen |= o < i;
      }
    if (!seen) store(dx, c, grad(value(x, c)) + d);
  }
}

template <class T>
cudaError_t forward(const void* logits, long ld, const long long* tokens, float* logprob, float* entropy, float* stats, float* top, long long* index,
                    long rows, int V, int k, long long ignore, cudaStream_t st) {
  // CTAs of a row: with fewer rows than SMs up to 8, of 4096 columns at least
  const int sms = nsa::sm_count();
  int parts = 1;
  while (parts < 8 && rows * parts * 2 <= 2l * sms && V / (2 * parts) >= 4096) parts *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = static_cast<unsigned>(rows * parts);
  cfg.blockDim = kThreads;
  cfg.stream = st;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = parts;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cfg.attrs = &cluster;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, logprobs_fwd_kernel<T>, static_cast<const T*>(logits), ld, tokens, logprob, entropy, reinterpret_cast<float2*>(stats), top,
                            index, V, k, ignore, parts, nsa::status_ptr());
}
}  // namespace

extern "C" int nsa_logprobs_fwd(const void* logits, long ld, int fp32, const long long* tokens, float* logprob, float* entropy, float* stats, float* top,
                                long long* index, long rows, int V, int k, long long ignore, cudaStream_t st) {
  if (rows <= 0) return 0;
  if (V <= 0 || V > 0x7fff0000 || k < 0 || k > V || k > kTopMax || rows > 0x7fffffff) return nsa::fail(NSA_ERR_SHAPE, "logprobs: unsupported shape");
  const cudaError_t e = fp32 ? forward<float>(logits, ld, tokens, logprob, entropy, stats, top, index, rows, V, k, ignore, st)
                             : forward<bf16>(logits, ld, tokens, logprob, entropy, stats, top, index, rows, V, k, ignore, st);
  if (e != cudaSuccess) return nsa::fail_cuda(e, "nsa_logprobs_fwd launch");
  nsa::count_launch();
  return 0;
}

extern "C" int nsa_logprobs_bwd(const void* logits, long ld, int fp32, const long long* tokens, const float* stats, const float* entropy,
                                const long long* index, const float* dlogprob, const float* dentropy, const float* dtop, void* dx, long rows, int V,
                                int k, long long ignore, cudaStream_t st) {
  if (rows <= 0) return 0;
  if (V <= 0 || V > 0x7fff0000 || k < 0 || k > V) return nsa::fail(NSA_ERR_SHAPE, "logprobs: unsupported shape");
  const int n = fp32 ? 4 : 8, chunks = ((V + 2 * n - 1) / n + kBwdPieces - 1) / kBwdPieces;
  if (rows * chunks > 0x7fffffff) return nsa::fail(NSA_ERR_SHAPE, "logprobs: unsupported shape");
  const unsigned grid = static_cast<unsigned>(rows * chunks);
  if (fp32)
    logprobs_bwd_kernel<<<grid, kThreads, 0, st>>>(static_cast<const float*>(logits), ld, tokens, reinterpret_cast<const float2*>(stats), entropy, index,
                                                   dlogprob, dentropy, dtop, static_cast<float*>(dx), V, k, ignore, chunks);
  else
    logprobs_bwd_kernel<<<grid, kThreads, 0, st>>>(static_cast<const bf16*>(logits), ld, tokens, reinterpret_cast<const float2*>(stats), entropy, index,
                                                   dlogprob, dentropy, dtop, static_cast<bf16*>(dx), V, k, ignore, chunks);
  nsa::count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : nsa::fail_cuda(e, "nsa_logprobs_bwd launch");
}
