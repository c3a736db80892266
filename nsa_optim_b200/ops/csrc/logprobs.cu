// Log probabilities of given tokens, entropies and the likeliest tokens of rows of logits, and their gradient.
//
// With m = max x, S = sum e^(x - m): log p_j = x_j - m - log S, and the entropy is log S + sum (m - x) e^(x - m) / S, a sum of terms that are not
// negative, so nothing cancels where a distribution is narrow.  The sums are taken in one pass with a running maximum: y = log2(e) x - R in one
// rounding, S = sum 2^y, E = sum y 2^y, and a larger R moves them by S' = f S, E' = f (E + d S), d = R - R', f = 2^d.  R is log2(e) times the maximum,
// rounded, and a warp's: it moves about five times a row, where one of each lane's own would move in most turns of a warp.  Its rounding, which would
// be 2^-24 of the largest logit in log S, is taken out at the end: log2(e) m - R is known to its last bit.
//
// The bytes of the logits bound both directions (an exponential takes 72 % of the special-function rate at that speed, the arithmetic 45 % of issue).
// The k likeliest tokens cost next to nothing in the pass: each thread keeps the largest logit of what it saw, the four pieces it was in, and the largest
// of the other pieces.  The k-th largest of the maxima of 64 pairs of threads is a bound that k logits reach, so only the four pieces of threads whose
// maximum reaches it are read again (few more than k of 128 threads), and all pieces of a thread where a second four do.  A warp of its own does that,
// and the row's end, while the others are in the next row.  What it waits for counts: behind 24 MB of copies a load takes 4 us, so that it reads what it
// needs at once (when it read whole threads' pieces in turns, 4096 x 151936 logits with k = 8 took 413 us, with k = 1 230).  What it executes counts as well:
// where each CTA has one row, nothing hides its end, and its instructions come from memory the first time (8 in about 50 cycles of a lone warp); where
// it has many, they share the issue slots.  So loops stay loops, maxima are ranked by counting, and a single token's bound is one maximum.
//
// Measured, kernels alone: 4096 x 151936 bf16, k = 8: 232 us, 5.4 TB/s (backward 371 us, 6.7 TB/s, some of it from L2); 8192 x 32000, k = 1: 114 to 116 us, 4.5 TB/s; 511 x 50257
// fp32, k = 5: 26 to 28 us;
// 64 x 151936, k = 20: 19 us, of which 5.5 to 7 until the last logit has been seen, 4.5 for the candidates, 2 for the slowest CTA of a cluster, 2 for places.
//
// Compiled without fast math: the logarithms at a row's end are the exact ones, the exponentials of its elements the hardware's.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <math_constants.h>

#include <atomic>

#include "f32x2.cuh"
#include "host.cuh"
#include "tc5.cuh"

namespace {
namespace cg = cooperative_groups;
typedef __nv_bfloat16 bf16;
typedef unsigned long long u64;
constexpr int kThreads = 128, kWarps = kThreads / 32;        // of the pass over the logits; a warp more for the copies, one for the rows' ends
constexpr int kCtas = 5;                  // per SM
constexpr int kUnroll = 4, kHalves = 2;   // 16-byte pieces of a thread at a time; of a chunk
constexpr int kChunk = kThreads * kUnroll * kHalves, kStages = 2;      // pieces that a bulk copy brings (16 KB); chunks on their way or in use
// 4096 x 151936, k = 8, forward and backward (an older one) 669 us, 8192 x 32000, k = 1 126 and 511 x 50257 27 when these were tried instead: four CTAs of three stages
// 740 and 170; five of four stages of half a chunk 689, 124 and 29; six of three such stages 684, 121 and 31; halves in a loop 677, 122 and 29.
constexpr int kTopMax = 32;               // tokens that the selection gives
constexpr int kBuffer = 480;              // candidates for them
constexpr int kParts = 8;                 // CTAs of a cluster
constexpr int kWidest = 32767 * kThreads * kUnroll * 4;      // columns: halves of chunks are counted in 16 bits
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Logits below -kFar count as it in the pass, and rows whose maximum is above kFar or within a factor of ten of -kFar are looked at again at their end: R's rounding
// is 4 at most then, so that S, which has 2 to the power of it, is a number.  (With -1e30 for it, stretches of masks of -1e10 and the like made rows NaN.)
constexpr float kFar = 0x1p26f, kLow = -kFar;

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
  static __device__ __forceinline__ float top(const Vec (&v)[kUnroll]) {
    uint4 m = v[0].w;
#pragma unroll
    for (int u = 1; u < kUnroll; ++u) m = make_uint4(max2_nan(m.x, v[u].w.x), max2_nan(m.y, v[u].w.y), max2_nan(m.z, v[u].w.z), max2_nan(m.w, v[u].w.w));
    return Vec{m}.top();
  }
  __device__ __forceinline__ float top() const {
    const uint32_t m = max2_nan(max2_nan(w.x, w.y), max2_nan(w.z, w.w));
    return max_nan(lower(m), upper(m));
  }
  __device__ __forceinline__ void exact(float2 (&x)[4]) const {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = make_float2(lower(v[i]), upper(v[i]));
  }
  static __device__ __forceinline__ uint32_t two(float2 x) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x.x, x.y);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&x)[4]) { return make_uint4(two(x[0]), two(x[1]), two(x[2]), two(x[3])); }
  __device__ __forceinline__ void clear() { w = make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
  __device__ __forceinline__ void floats(float2 (&x)[4]) const {       // none below kLow
    const uint32_t v[4] = {w.x, w.y, w.z, w.w}, low = 0xcc80cc80u;     // bf16 of kLow
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
  static __device__ __forceinline__ float top(const Vec (&v)[kUnroll]) {
    float m = v[0].top();
#pragma unroll
    for (int u = 1; u < kUnroll; ++u) m = max_nan(m, v[u].top());
    return m;
  }
  __device__ __forceinline__ float top() const { return max_nan(max_nan(w.x, w.y), max_nan(w.z, w.w)); }
  __device__ __forceinline__ void exact(float2 (&x)[2]) const {
    x[0] = make_float2(w.x, w.y);
    x[1] = make_float2(w.z, w.w);
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&x)[2]) {
    return make_uint4(__float_as_uint(x[0].x), __float_as_uint(x[0].y), __float_as_uint(x[1].x), __float_as_uint(x[1].y));
  }
  __device__ __forceinline__ void clear() { w = make_float4(-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F); }
  __device__ __forceinline__ void floats(float2 (&x)[2]) const {
    x[0] = make_float2(max_nan(w.x, kLow), max_nan(w.y, kLow));
    x[1] = make_float2(max_nan(w.z, kLow), max_nan(w.w, kLow));
  }
};
template <class T>
__device__ __forceinline__ Vec<T> load(const T* p) {                   // 16-byte aligned
  Vec<T> v;
  *reinterpret_cast<uint4*>(&v.w) = __ldg(reinterpret_cast<const uint4*>(p));
  return v;
}

// Order of the likeliest tokens as whole numbers: larger logits first, NaN before all, -0 as 0, then the lower index
__device__ __forceinline__ unsigned ordered(float x) {
  const int bits = x != x ? 0x7fffffff : __float_as_int(x + 0.f);
  return bits >= 0 ? static_cast<unsigned>(bits) | 0x80000000u : ~static_cast<unsigned>(bits);
}
__device__ __forceinline__ u64 rank_of(float x, int i) { return static_cast<u64>(ordered(x)) << 32 | (0xffffffffu - static_cast<unsigned>(i)); }
__device__ __forceinline__ float number_of(unsigned o) { return __uint_as_float(o >> 31 ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ float logit_of(u64 r) { return number_of(static_cast<unsigned>(r >> 32)); }
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

// A CTA's part of a row: columns lo .. hi, as 16-byte pieces, the first and last of which may reach beyond it.  Of the whole ones, w0 .. w1, piece w0 + j is
// thread j % kThreads'; a first one that is not whole is thread 0's, a last one thread 32's.
template <class T>
struct Part {
  static constexpr int kN = Vec<T>::kN;
  const T* x;           // column 0
  int lo, hi, base;     // the first piece begins at column base <= lo, which is 16-byte aligned
  int pieces, w0, w1;
  __device__ __forceinline__ Part(const T* row, int l, int h) : x(row), lo(l), hi(h) {
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(row + lo) % 16 / sizeof(T));
    base = lo - off;
    pieces = hi > lo ? (hi - base + kN - 1) / kN : 0;
    w0 = off > 0 && pieces > 0 ? 1 : 0;
    w1 = max((hi - base) / kN, w0);
  }
  __device__ __forceinline__ int chunks() const { return (w1 - w0 + kChunk - 1) / kChunk; }
  __device__ __forceinline__ const T* chunk(int c) const { return x + base + static_cast<long>(w0 + c * kChunk) * kN; }
  __device__ __forceinline__ int chunk_pieces(int c) const { return min(kChunk, w1 - w0 - c * kChunk); }
  // The piece of a thread that is not whole, -1: none
  __device__ __forceinline__ int odd_piece(int t) const { return t == 0 && w0 == 1 ? 0 : t == 32 && w1 < pieces ? w1 : -1; }
  __device__ __forceinline__ float at(int c) const { return c >= lo && c < hi ? value(x, c) : -CUDART_INF_F; }
};

struct Smem {
  // what the pass leaves for a row's end, of two rows in turn
  Sums sums[2][kWarps];
  alignas(16) unsigned top[2][kThreads];   // maxima of threads, as `ordered`
  alignas(16) unsigned other[2][kThreads]; // of the pieces that do not lie with it
  alignas(8) short where[2][kThreads];     // the chunk half that it lies in; -1: a piece that is not whole
  uint64_t ready[2], taken[2];
  // what the cluster's CTAs leave here
  Sums all[kParts];
  u64 lists[kParts][kTopMax];
  // of the warp of the rows' ends
  alignas(16) uint2 pairs[32];
  short list[kThreads], rest[kThreads];    // threads of which four pieces, or all, are looked at again
  u64 buffer[kBuffer];
  uint4 piece[4][33];                      // of lanes, where their hits are read by number
  u64 best[kTopMax];
  uint64_t full[kStages], empty[kStages];
  int abort_flag;
};

__device__ __forceinline__ void warp_reduce(Sums& s) {                 // lanes share m
  for (int o = 16; o; o >>= 1) {
    s.S += __shfl_xor_sync(0xffffffffu, s.S, o);
    s.E += __shfl_xor_sync(0xffffffffu, s.E, o);
  }
}

// Of n lanes that lie together, n a power of two: in all of them
__device__ __forceinline__ Sums join(Sums s, int n) {
#pragma unroll 1
  for (int o = n >> 1; o; o >>= 1)
    s.add(Sums{__shfl_xor_sync(0xffffffffu, s.m, o), __shfl_xor_sync(0xffffffffu, s.R, o), __shfl_xor_sync(0xffffffffu, s.S, o),
               __shfl_xor_sync(0xffffffffu, s.E, o)});
  return s;
}

// The sums of a part and the thread's own maximum.  get: chunks that the CTA has read
template <class T>
__device__ __forceinline__ Sums pass(const Part<T>& p, Smem& sm, const uint4* ring, uint32_t& get, bool& ok, float& top, float& other, int& where,
                                     KernelStatus* status) {
  constexpr int kN = Vec<T>::kN;
  Sums s{kLow, 0.f, 0.f, 0.f};
  top = other = -CUDART_INF_F;
  where = -1;
  float2 S2 = make_float2(0.f, 0.f), E2 = make_float2(0.f, 0.f);
  auto flush = [&]() {
    s.S += S2.x + S2.y;
    s.E += E2.x + E2.y;
    S2 = E2 = make_float2(0.f, 0.f);
  };
  auto raise = [&](float m, int at) {                                  // of the warp, where a lane's logits exceed it
    const bool larger = top == top && !(m <= top);                     // NaN before all
    other = larger ? top : max_nan(other, m);
    where = larger ? at : where;
    top = larger ? m : top;
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
  const int chunks = p.chunks();
#pragma unroll 1
  for (int c = 0; c < chunks; ++c, ++get) {
    const int st = get % kStages, n = p.chunk_pieces(c) - static_cast<int>(threadIdx.x);
    ok = ok && tc5::mbar_wait_warp(&sm.full[st], get / kStages & 1, &sm.abort_flag, status, STATUS_TIMEOUT_SMEM_FULL);
    const uint4* at = ring + st * kChunk + threadIdx.x;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      Vec<T> v[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) *reinterpret_cast<uint4*>(&v[u].w) = at[(h * kUnroll + u) * kThreads];
      if (h == kHalves - 1) tc5::arrive_warp(&sm.empty[st]);
      if ((h + 1) * kUnroll * kThreads > n) {                          // what is behind the last piece is not this part's
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if ((h * kUnroll + u) * kThreads >= n) v[u].clear();
      }
      raise(Vec<T>::top(v), c * kHalves + h);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        float2 x[kN / 2];
        v[u].floats(x);
        add(x);
      }
    }
  }
  // the first and the last piece, where they are not whole
  if (threadIdx.x < 64 && (p.w0 == 1 || p.w1 < p.pieces)) {
    float2 x[kN / 2];
    float m = -CUDART_INF_F;
    const int j = p.odd_piece(threadIdx.x);
#pragma unroll
    for (int i = 0; i < kN / 2; ++i) {
      const int c = p.base + j * kN + 2 * i;
      const float a = j < 0 ? -CUDART_INF_F : p.at(c), b = j < 0 ? -CUDART_INF_F : p.at(c + 1);
      m = max_nan(m, max_nan(a, b));
      x[i] = make_float2(max_nan(a, kLow), max_nan(b, kLow));
    }
    raise(m, -1);
    add(x);
  }
  flush();
  warp_reduce(s);
  if (__any_sync(0xffffffffu, top != top)) s = Sums{fmaxf(s.m, 0.f), s.m > 0.f ? s.R : 0.f, CUDART_NAN_F, CUDART_NAN_F};     // also where no other number was seen
  return s;
}

// The part's k first in rank order, in sm.best (0 behind them), by one warp.  top: the threads' maxima.
template <class T>
__device__ __noinline__ void select(Smem& sm, const Part<T>& p, int b, int k) {
  constexpr int kN = Vec<T>::kN, kEach = kThreads / 32;
  constexpr unsigned kAll = 0xffffffffu;
  static_assert(kEach == 4, "four maxima a lane");
  const int lane = threadIdx.x & 31, have = min(k, p.hi - p.lo);
  const uint4 four = *reinterpret_cast<const uint4*>(sm.top[b] + lane * 4), others = *reinterpret_cast<const uint4*>(sm.other[b] + lane * 4);
  const unsigned mine[kEach] = {four.x, four.y, four.z, four.w}, second[kEach] = {others.x, others.y, others.z, others.w};
  // the have-th largest of the pairs: the smallest of those with fewer than so many larger ones
  const unsigned g0 = max(four.x, four.y), g1 = max(four.z, four.w);
  unsigned kth;
  if (have == 1) {
    kth = __reduce_max_sync(kAll, max(g0, g1));
  } else {
    int before0 = 0, before1 = 0;
    sm.pairs[lane] = make_uint2(g0, g1);
    __syncwarp();
#pragma unroll 4
    for (int i = 0; i < 16; ++i) {
      const uint4 o = reinterpret_cast<const uint4*>(sm.pairs)[i];
      before0 += (o.x > g0) + (o.y > g0) + (o.z > g0) + (o.w > g0);
      before1 += (o.x > g1) + (o.y > g1) + (o.z > g1) + (o.w > g1);
    }
    kth = __reduce_min_sync(kAll, min(before0 < have ? g0 : kAll, before1 < have ? g1 : kAll));
  }
  int reach = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) reach += __popc(__ballot_sync(kAll, mine[i] >= kth));
  // Logits that reach the bound.  Where far more threads' do than are asked for, logits are equal: then only those above it, and the first of the
  // equal ones in order.
  const bool ties = reach > 2 * have + 16;
  const unsigned bound = ties ? kth : kth - 1;                         // candidates are larger than this
  // the same as a test of numbers, !(x <= under): NaN is larger than any (bound < NaN's order: no number lies between infinity's and it), zeros are equal
  const bool none = bound == 0xffffffffu;
  const float under = bound >= 0xff800000u ? CUDART_INF_F : bound == 0x7fffffffu ? -1.401298e-45f : number_of(bound);
  int n = 0, n_rest = 0, count = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const bool all = second[i] > bound, is = mine[i] > bound && !all;
    const unsigned mask = __ballot_sync(kAll, is), mask_all = __ballot_sync(kAll, all), below = (1u << lane) - 1;
    if (is) sm.list[n + __popc(mask & below)] = static_cast<short>(lane * 4 + i);
    if (all) sm.rest[n_rest + __popc(mask_all & below)] = static_cast<short>(lane * 4 + i);
    n += __popc(mask);
    n_rest += __popc(mask_all);
  }
  sm.best[lane] = 0;
  __syncwarp();
  auto candidate = [&](bool is, float x, int col) {                    // of all lanes at once
    is = is && col >= p.lo && col < p.hi;
    const unsigned mask = __ballot_sync(kAll, is);
    const int at = count + __popc(mask & ((1u << lane) - 1));
    if (is && at < kBuffer) sm.buffer[at] = rank_of(x, col);
    count += __popc(mask);
  };
  // A lane takes four pieces of a thread at a time: those of its largest logit, or four after four of all
  const int turns = (p.w1 - p.w0 + kThreads - 1) / kThreads, fours = (turns + kUnroll - 1) / kUnroll, items = n + n_rest * fours;
#pragma unroll 1
  for (int e = lane; e - lane < items; e += 32) {
    int who = -1, four = 0;
    if (e < n) {
      who = sm.list[e];
      four = sm.where[b][who];
    } else if (e < items) {
      who = sm.rest[(e - n) / fours];
      four = (e - n) % fours;
    }
    const int j0 = p.w0 + who + four * (kUnroll * kThreads), there = who < 0 || four < 0 ? 0 : min((p.w1 - j0 + kThreads - 1) / kThreads, kUnroll);
    __syncwarp();
    {
      Vec<T> v[kUnroll];
#pragma unroll
      for (int i = 0; i < kUnroll; ++i)
        if (i < there) v[i] = load(p.x + p.base + (j0 + i * kThreads) * kN);
#pragma unroll
      for (int i = 0; i < kUnroll; ++i)
        if (i < there) sm.piece[i][lane] = *reinterpret_cast<const uint4*>(&v[i].w);
    }
    __syncwarp();
    unsigned hits = 0;
#pragma unroll 1
    for (int i = 0; i < there; ++i) {
      Vec<T> v;
      float2 x[kN / 2];
      *reinterpret_cast<uint4*>(&v.w) = sm.piece[i][lane];
      v.exact(x);
      unsigned some = 0;
#pragma unroll
      for (int c = 0; c < kN / 2; ++c) {
        if (!(x[c].x <= under)) some |= 1u << (2 * c);
        if (!(x[c].y <= under)) some |= 2u << (2 * c);
      }
      hits |= some << (i * kN);
    }
    if (none) hits = 0;
#pragma unroll 1
    while (__any_sync(kAll, hits)) {                                   // one of each lane's
      const int at = hits ? __ffs(hits) - 1 : 0;
      candidate(hits != 0, value(reinterpret_cast<const T*>(&sm.piece[at / kN][lane]), at % kN), p.base + (j0 + at / kN * kThreads) * kN + at % kN);
      hits &= hits - 1;
    }
  }
  if (p.w0 == 1 || p.w1 < p.pieces) {                                  // pieces that are not whole: a column per lane
    const int j = p.odd_piece(lane < kN ? 0 : 32), col = p.base + j * kN + lane % kN;
    const float x = j >= 0 && lane < 2 * kN ? p.at(col) : -CUDART_INF_F;
    candidate(j >= 0 && lane < 2 * kN && ordered(x) > bound, x, col);
  }
  if (count <= kBuffer - kTopMax) {
    if (ties)
      for (int c0 = p.lo; c0 < p.hi && count < have; c0 += 32) {
        const float x = p.at(c0 + lane);
        candidate(ordered(x) == kth, x, c0 + lane);
      }
    __syncwarp();
#pragma unroll 1
    for (int i = lane; i < count; i += 32) {
      const u64 r = sm.buffer[i];
      int before = 0;
#pragma unroll 8
      for (int o = 0; o < count; ++o) before += sm.buffer[o] > r;
      if (before < have) sm.best[before] = r;
    }
    __syncwarp();
    return;
  }
  // more candidates than are kept (the largest logits all in few threads' pieces): one after another
  u64 last = ~0ull;
  for (int m = 0; m < have; ++m) {
    u64 r = 0;
    for (int c = p.lo + lane; c < p.hi; c += 32) {
      const u64 a = rank_of(value(p.x, c), c);
      if (a < last && a > r) r = a;
    }
    for (int o = 16; o; o >>= 1) {
      const u64 a = __shfl_xor_sync(kAll, r, o);
      r = a > r ? a : r;
    }
    last = r;
    if (lane == 0) sm.best[m] = r;
  }
  __syncwarp();
}

// A row's end, by one warp of each CTA: a are the row's sums, lists its parts' best in order.  Each CTA places its own, the first one writes the rest.
template <class T>
__device__ __noinline__ void finish(const u64* lists, Sums a, const T* x, long row, long long tok, float chosen, float* logprob, float* entropy, float2* stats, float* top_out,
                                    long long* index, int V, int k, long long ignore, int part, int parts, KernelStatus* status) {
  const int lane = threadIdx.x & 31;
  float m = a.m, logS = logf(a.S) - fmaf(m, kLog2e, -a.R) * kLn2, H = logf(a.S);
  bool empty = false;
  if (m <= 0.1f * kLow || m > kFar) {                                  // the pass has not told logits apart, or its sums are none
    m = -CUDART_INF_F;
    for (int c = lane; c < V; c += 32) m = max_nan(m, value(x, c));
    for (int o = 16; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    empty = m == -CUDART_INF_F;
    Sums b{0.f, 0.f, 0.f, 0.f};
    for (int c = lane; c < V && !empty; c += 32) {
      const float y = (value(x, c) - m) * kLog2e, e = ex2(y);
      b.S += e;
      b.E += e > 0.f ? y * e : e;
    }
    warp_reduce(b);
    a = b;
    H = logS = empty ? 0.f : logf(a.S);
  }
  H = empty ? 0.f : H - a.E * kLn2 / a.S;
  if (lane == 0 && part == 0) {
    NSA_CHECK_INDEX(tok == ignore || (tok >= 0 && tok < V), status, tok);
    logprob[row] = tok == ignore || tok < 0 || tok >= V ? 0.f : empty ? m : chosen - m - logS;
    entropy[row] = H;
    stats[row] = make_float2(m, logS);                                 // apart: their sum would round a probability by |m| 2^-24
  }
  if (k == 0) return;
  // a token's place is the number of larger ones in all lists: 32 ranks each, that of no token is 0
  const u64 mine = lists[part * kTopMax + lane];
  int place = lane;
  if (parts > 1) {
    int n[kParts] = {};
#pragma unroll 1
    for (int step = kTopMax / 2; step; step >>= 1)
#pragma unroll
      for (int c = 0; c < kParts; ++c)
        if (c < parts) n[c] += lists[c * kTopMax + n[c] + step - 1] > mine ? step : 0;
    place = 0;
#pragma unroll
    for (int c = 0; c < kParts; ++c)
      if (c < parts) place += n[c] + (lists[c * kTopMax + n[c]] > mine);
  }
  if (mine != 0 && place < k) {
    index[row * k + place] = index_of(mine);
    top_out[row * k + place] = empty ? m : logit_of(mine) - m - logS;
  }
  __syncwarp();
}

// Of all threads of a cluster's CTAs: what came before their arrival is seen behind the wait, and an arrival follows the wait for the one before it
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// A CTA takes a row at a time; or a cluster its only one, each CTA an even part of the columns.
template <class T>
__global__ void __launch_bounds__(kThreads + 64, kCtas) logprobs_fwd_kernel(const T* __restrict__ logits, long ld, const long long* __restrict__ tokens,
                                                                            float* __restrict__ logprob, float* __restrict__ entropy,
                                                                            float2* __restrict__ stats, float* __restrict__ top_out,
                                                                            long long* __restrict__ index, long rows, int V, int k, long long ignore,
                                                                            int parts, KernelStatus* status) {
  extern __shared__ __align__(128) uint4 ring[];
  __shared__ Smem sm;
  const int t = threadIdx.x, lane = t & 31, warp = tc5::warp_index(), part = blockIdx.x % parts;
  const long first = blockIdx.x / parts, step = gridDim.x / parts;
  const int each = (V + parts - 1) / parts, lo = min(part * each, V), hi = min((part + 1) * each, V);
  if (t == 0) {
    sm.abort_flag = 0;
    for (int i = 0; i < kStages; ++i) {
      tc5::mbar_init(&sm.full[i], 1);
      tc5::mbar_init(&sm.empty[i], kWarps);
    }
    for (int i = 0; i < 2; ++i) {
      tc5::mbar_init(&sm.ready[i], kWarps);
      tc5::mbar_init(&sm.taken[i], 1);
    }
    tc5::fence_barrier_init();
  }
  __syncthreads();
  if (parts > 1) cluster_arrive();                                     // the CTA runs: its memory may be written
  bool ok = true;
  uint32_t n = 0;                                                      // rows that this CTA has had
  if (warp < kWarps) {
    uint32_t get = 0;
#pragma unroll 1
    for (long row = first; row < rows; row += step, ++n) {
      const Part<T> p(logits + row * ld, lo, hi);
      float top, other;
      int where;
      const Sums s = pass(p, sm, ring, get, ok, top, other, where, status);
      const int b = n & 1;
      if (n >= 2) ok = ok && tc5::mbar_wait_warp(&sm.taken[b], (n / 2 - 1) & 1, &sm.abort_flag, status, STATUS_TIMEOUT_SMEM_EMPTY);
      sm.top[b][t] = ordered(top);
      sm.other[b][t] = ordered(other);
      sm.where[b][t] = static_cast<short>(where);
      if (lane == 0) sm.sums[b][warp] = s;
      tc5::arrive_warp(&sm.ready[b]);
    }
    if (parts > 1) {
      cluster_wait();
      cluster_arrive();
    }
  } else if (warp == kWarps) {                                         // the copies
    uint32_t put = 0;
#pragma unroll 1
    for (long row = first; row < rows; row += step) {
      if (lane == 0) {
        const Part<T> p(logits + row * ld, lo, hi);
        const int chunks = p.chunks();
        for (int c = 0; c < chunks && ok; ++c, ++put) {
          const int st = put % kStages, bytes = p.chunk_pieces(c) * 16;
          if (put >= kStages) ok = tc5::mbar_wait(&sm.empty[st], (put / kStages - 1) & 1, &sm.abort_flag, status, STATUS_TIMEOUT_SMEM_EMPTY);
          if (!ok) break;
          tc5::mbar_expect_tx(&sm.full[st], bytes);
          asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(tc5::smem_u32(ring + st * kChunk)),
                       "l"(p.chunk(c)), "r"(bytes), "r"(tc5::smem_u32(&sm.full[st]))
                       : "memory");
        }
      }
      __syncwarp();
    }
    if (parts > 1) {
      cluster_wait();
      cluster_arrive();
    }
    if (lane == 0 && sm.abort_flag)
      for (int i = 0; i < kStages; ++i) tc5::mbar_drain(&sm.full[i]);
  } else {                                                             // the rows' ends
    // the given token of the row after the next and its logit of the next one are on their way meanwhile
    auto token = [&](long row) { return row < rows ? tokens[row] : -1ll; };
    auto logit = [&](long row, long long tok) { return tok >= 0 && tok < V ? value(logits + row * ld, tok) : 0.f; };
    long long tok = token(first), tok1 = token(first + step);
    float chosen = logit(first, tok);
#pragma unroll 1
    for (long row = first; row < rows; row += step, ++n) {
      const T* x = logits + row * ld;
      const int b = n & 1;
      const long long tok2 = token(row + 2 * step);
      const float chosen1 = logit(row + step, tok1);
      // most of the time there is nothing to do: polling would take the others' issue slots
      for (int i = 0; i < 20000 && !__all_sync(0xffffffffu, tc5::mbar_try_wait(&sm.ready[b], n / 2 & 1)); ++i) __nanosleep(100);
      ok = ok && tc5::mbar_wait_warp(&sm.ready[b], n / 2 & 1, &sm.abort_flag, status, STATUS_TIMEOUT_SMEM_FULL);
      Sums a{kLow, 0.f, 0.f, 0.f};
      if (ok) {
        a = join(sm.sums[b][lane % kWarps], kWarps);
        if (k > 0) select(sm, Part<T>(x, lo, hi), b, k);
      }
      if (parts > 1) {
        cluster_wait();
        if (ok) {
          if (lane < parts) *cg::this_cluster().map_shared_rank(&sm.all[part], lane) = a;
          if (k > 0)
#pragma unroll 1
            for (int c = 0; c < parts; ++c) *cg::this_cluster().map_shared_rank(&sm.lists[part][lane], c) = sm.best[lane];
        }
        cluster_arrive();
        cluster_wait();
        a = join(sm.all[lane & (parts - 1)], parts);                // a power of two
      }
      if (ok && (k > 0 || part == 0))
        finish(parts > 1 ? sm.lists[0] : sm.best, a, x, row, tok, chosen, logprob, entropy, stats, top_out, index, V, k, ignore, part, parts, status);
      tc5::arrive_warp(&sm.taken[b]);
      tok = tok1;
      tok1 = tok2;
      chosen = chosen1;
    }
  }
}

// dx_j = -p_j (G + g_H (log p_j + H)), G the sum of the row's other gradients; theirs are added at their tokens.  One CTA per kBwdPieces pieces of a row.
// Bytes bound it, and how they are asked for: 4096 x 151936 bf16, forward and backward in turn on the same memory, with 8 loads of each of 128 threads 606 us, 8 of 96, 160, 192 and 256
// 608, 610, 632 and 652, 4 of 256 667, 7 and 9 of 128 622, 16 of 64 772; loads that leave the caches first 618, stores that do not 617; rows from the
// first on, not from the last, which the forward pass has left in L2, 608.
constexpr int kBwdThreads = 128, kBwdTurns = 8, kBwdPieces = kBwdThreads * kBwdTurns;
template <class T>
__global__ void __launch_bounds__(kBwdThreads) logprobs_bwd_kernel(const T* __restrict__ logits, long ld, const long long* __restrict__ tokens,
                                                                const float2* __restrict__ stats, const float* __restrict__ entropy,
                                                                const long long* __restrict__ index, const float* __restrict__ dlogprob,
                                                                const float* __restrict__ dentropy, const float* __restrict__ dtop,
                                                                T* __restrict__ dx_all, int V, int k, long long ignore, int chunks) {
  constexpr int kN = Vec<T>::kN;
  const int t = threadIdx.x;
  const long row = (gridDim.x - 1 - blockIdx.x) / chunks;
  const int chunk = static_cast<int>(gridDim.x - 1 - blockIdx.x - row * chunks);
  const T* x = logits + row * ld;
  T* dx = dx_all + row * V;
  // pieces where dx is 16-byte aligned; x is as well, or its elements are loaded one by one
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(dx) % 16 / sizeof(T)), pieces = (V + off + kN - 1) / kN;
  const bool same = (reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) % 16 == 0;
  const int j0 = chunk * kBwdPieces;
  Vec<T> v[kBwdTurns];
  bool whole[kBwdTurns];
#pragma unroll
  for (int u = 0; u < kBwdTurns; ++u) {
    const int j = j0 + u * kBwdThreads + t, c = j * kN - off;
    whole[u] = same && c >= 0 && c + kN <= V;
    if (whole[u]) v[u] = load(x + c);
  }
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
#pragma unroll
  for (int u = 0; u < kBwdTurns; ++u) {
    const int j = j0 + u * kBwdThreads + t, c = j * kN - off;
    if (j >= pieces) break;
    if (whole[u]) {
      float2 a[kN / 2];
      v[u].exact(a);
#pragma unroll
      for (int i = 0; i < kN / 2; ++i) a[i] = empty ? make_float2(0.f, 0.f) : make_float2(grad(a[i].x), grad(a[i].y));
      __stcs(reinterpret_cast<uint4*>(dx + c), Vec<T>::pack(a));
    } else {
      for (int i = 0; i < kN; ++i)
        if (c + i >= 0 && c + i < V) store(dx, c + i, empty ? 0.f : grad(value(x, c + i)));
    }
  }
  if (empty || (!counts && !dtop)) return;
  __syncthreads();
  // the chosen token (t = k) and the likeliest ones, each column once
  const int n = dtop ? k : 0;
  for (int i = t; i <= n; i += kBwdThreads) {
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
  // CTAs of a row: up to 8 where the GPU holds them all at once, of 4096 columns at least: a cluster's start and end cost about 1.5 us, a CTA reads 9000 columns
  // a us.  Rows of 8192 columns are faster whole, rows of 32000 in more parts; one row, k = 1, in parts of 4096 / 8192 / 16384 columns at least / whole: 8192
  // columns 8.0 / 6.7 / 6.6 / 6.7 us, 16384 8.6 / 8.3 / 7.7 / 7.9, 32000 8.7 / 9.3 / 9.9 / 9.9, 50257 9.9 / 10.6 / 11.9 / 13.0, 151936 10.7 / 10.7 / 10.7 / 22.7; 64 rows, k = 20:
  // 8192 10.3 / 8.4 / 8.7 / 8.4, 32000 11.7 / 11.9 / 13.2 / 13.8, 151936 18.2 / 18.5 / 18.3 / 34.7
  const int sms = nsa::sm_count();
  int parts = 1;
  while (parts < kParts && rows * parts * 2 <= static_cast<long>(kCtas) * sms && V / (2 * parts) >= 4096) parts *= 2;
  cudaLaunchConfig_t cfg{};
  const long most = static_cast<long>(kCtas) * sms / parts;
  cfg.gridDim = static_cast<unsigned>((rows < most ? rows : most) * parts);
  cfg.dynamicSmemBytes = kStages * kChunk * 16;
  cfg.blockDim = kThreads + 64;
  cfg.stream = st;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = parts;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cfg.attrs = &cluster;
  cfg.numAttrs = 1;
  static std::atomic<unsigned long long> ready{0};                     // devices on which the kernel may have this much shared memory
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev > 63 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    const cudaError_t e = cudaFuncSetAttribute(logprobs_fwd_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kStages * kChunk * 16);
    if (e != cudaSuccess) return e;
    if (dev <= 63) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  return cudaLaunchKernelEx(&cfg, logprobs_fwd_kernel<T>, static_cast<const T*>(logits), ld, tokens, logprob, entropy, reinterpret_cast<float2*>(stats), top,
                            index, rows, V, k, ignore, parts, nsa::status_ptr());
}
}  // namespace

extern "C" int nsa_logprobs_fwd(const void* logits, long ld, int fp32, const long long* tokens, float* logprob, float* entropy, float* stats, float* top,
                                long long* index, long rows, int V, int k, long long ignore, cudaStream_t st) {
  if (rows <= 0) return 0;
  if (V <= 0 || V > kWidest || k < 0 || k > V || k > kTopMax || rows > 0x7fffffff) return nsa::fail(NSA_ERR_SHAPE, "logprobs: unsupported shape");
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
    logprobs_bwd_kernel<<<grid, kBwdThreads, 0, st>>>(static_cast<const float*>(logits), ld, tokens, reinterpret_cast<const float2*>(stats), entropy, index,
                                                   dlogprob, dentropy, dtop, static_cast<float*>(dx), V, k, ignore, chunks);
  else
    logprobs_bwd_kernel<<<grid, kBwdThreads, 0, st>>>(static_cast<const bf16*>(logits), ld, tokens, reinterpret_cast<const float2*>(stats), entropy, index,
                                                   dlogprob, dentropy, dtop, static_cast<bf16*>(dx), V, k, ignore, chunks);
  nsa::count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : nsa::fail_cuda(e, "nsa_logprobs_bwd launch");
}
