// Attention of a step's queries over the paged 8-bit key / value cache.
//
// o = sum_j 2^(x_j - M) v_j / sum_j 2^(x_j - M), x_j = log2(e) scale q k_j, in one pass with a running M.  Rows are (query token, head of the KV head's
// group) pairs, 16 to a warp's matrix product (m16n8k16 on f16), so a group shares what it reads.  With few rows the bytes of the codes bound it;
// every other choice serves that:
//  * Work is counted in units of 64 keys, over all requests, KV heads and row tiles, and dealt out evenly to workers, a warp each: ragged requests cost
//    no more than even ones.  A worker's range may end inside a request; such parts meet in shared memory at the CTA's end, and across CTAs in
//    cache_attn_join_kernel.
//  * Each worker has its own ring of key and value tiles that asynchronous copies fill two tiles ahead: 130 KB in flight per SM, no registers, and no
//    synchronisation between workers.
//  * The cache's orders are those of the product's operands.  Of a unit, lane 4c+r of a warp scores token 2j + c%2 of sub-block c/2 in tile j and holds
//    the probabilities of sub-block r's tokens 2j, 2j+1, so its value operand is 16 neighbouring bytes.
//  * A code u becomes an f16 operand by a byte permutation alone: the bits 0x00uu are the (subnormal) number 2^-24 u.  The offset of 128 comes out
//    of sums: 128 sum(q) of a row's scores, and 128 sum(p) of its outputs, which one more product per step leaves in the accumulators' format and
//    which is taken off every fourth unit, before it outgrows them.  (With a subtraction per pair of codes, 256 of 1170 instructions a unit, drafts for
//    32 contexts of up to 12000 tokens took 268 us, then 240.)
//  * Codes and their products are exact, and so is a query row scaled by a power of two to 2^13 .. 2^14 (bf16's 8 bits; what is 2^-28 of the row's
//    largest value rounds).  Probabilities are rounded to 11 bits, relative to the row's largest product of probability and value scale: the value
//    scale's exponent is added to x, and taken out again of the sum.  Of products below 2^-29 of the largest fewer bits are kept, none below 2^-40.  Sums
//    are fp32.  Scores may be of any size up to 2^119.
//
// Measured, with the join: 8 contexts of 65 K tokens, 32 heads of 128 on 2: 55 us, 4.7 TB/s of codes; one token of each of 64 requests with 1 to 8192 tokens,
// the same heads: 40 us, 3.4 TB/s, since a worker has 7 units, of which the first and the last few leave the memory idle (workers end between 24 and 32
// us), and the join follows; eight drafted tokens of each of 32 requests with up to 12000 tokens, 32 heads on 8: 125 us, two tiles of 16 rows, 4600
// cycles a unit of a worker (2700 for scores, 1800 for values), bounded by the latency of its products and exponentials: two workers per scheduler issue 44 % of the time.
// Prompts are right but slow, since every tile of 16 rows passes over the keys, and since work is dealt out by all of a request's units, of which a tile's rows see the
// first ones only: a fresh prompt of 512 tokens, 32 heads of 128 on 2, 40 us, of 2048 315 us, of 8192 4.5 ms, 54 to 122 TFLOP/s (the forward over whole texts takes 14, 47 and
// 484 us); 2048 tokens behind 6000 in each of 4 requests 4.5 ms, 211 TFLOP/s.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include <atomic>

#include "cache.cuh"
#include "f32x2.cuh"
#include "host.cuh"
#include "tc5.cuh"

namespace {
typedef __nv_bfloat16 bf16;
constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kMaxRequests = 768;                        // of one launch: their prefix sums are in shared memory

struct AttnParams {
  const bf16* q;
  long ldq;
  CachePages c;
  CacheStep s;
  bf16* o;
  float* head;          // (CTA, worker, rows, D): parts of requests that end inside a worker's range and began before it
  float* part;          // (CTA, 2, rows, D): parts of requests that go beyond a CTA: one that began before it, one that goes on behind it
  float2* part_ml;      // (CTA, 2, rows)
  struct Join* join;    // (CTA)
  int Hq, G, window;
  int ends;             // 1: the first request of the call is among these, 2: the last one
  unsigned long long per_g;   // ceil(2^32 / G): row / G of rows below 2^32 / G is a multiplication
  float scale;          // times log2(e)
  KernelStatus* status;
};

// The item that begins in a CTA and ends in another, if there is one
struct alignas(16) Join {
  int any, h, row0, n, q0, pad;
  long long end, each;  // the unit at which it ends, units of a worker
};

template <int D>
struct Shape {
  static constexpr int kSub = 16 * D, kPitch = kSub + 32;              // a sub-block of 16 tokens; the pitch spreads four of them over the banks
  static constexpr int kSlot = 4 * kPitch;                             // a unit's keys or values
  static constexpr int kSlots = 3 * (128 / D);                         // of a worker
  static constexpr int kRing = kSlots * kSlot;
  static_assert(kRing >= 16 * D * 4, "a worker's sums go where its ring was");
};

__device__ __forceinline__ int token_of(const AttnParams& p, int row) { return static_cast<int>(static_cast<unsigned>(row) * p.per_g >> 32); }

// What a worker has left in memory at the end
struct Left {
  int head, tail;       // whether there is a part that began before the range and ended in it; whether the last part is open at either end
  int began, open;      // of the last part: began before the range; goes on behind it
  int head_item[3], tail_item[3];                                      // request, KV head, first row
  long long tail_end;   // the unit at which the last part's item ends
  int some;             // the range is not empty
};

struct Request {
  int n, q0;            // queries, the first one's row in q
  int past, cap;        // tokens before them, keys that the table can hold
  // 64-key units that any of them sees
  __device__ __forceinline__ int unit0(int window) const { return window > 0 ? max(past - window + 1, 0) >> 6 : 0; }
  __device__ __forceinline__ int units(int window) const { return n > 0 ? max(((cap + 63) >> 6) - unit0(window), 1) : 0; }
};

template <int D, int R>
struct Smem {
  using S = Shape<D>;
  alignas(128) uint8_t ring[kWarps][S::kRing];
  float2 scale[kWarps][S::kSlots][4];
  uint64_t full[kWarps][S::kSlots];
  float2 ml[kWarps][2][R];
  Left left[kWarps];
  long long before[kMaxRequests + 1];                                  // units of the requests before b
  Request request[kMaxRequests];
  long long warps[kWarps];
  int abort_flag;
};

// ------------------------------------------------------------------------------------- work
__device__ __forceinline__ Request request_of(const AttnParams& p, int b) {
  Request r;
  const int lo = p.s.query_start[b], hi = p.s.query_start[b + 1], len = p.s.lengths[b];
  r.q0 = min(max(lo, 0), p.s.N);
  r.n = max(min(hi, p.s.N) - r.q0, 0);
  r.past = len - (hi - lo);
  r.cap = static_cast<int>(min(static_cast<long long>(max(len, 0)), static_cast<long long>(p.s.W) << p.c.shift));
  return r;
}

// A worker's share of one item (request, KV head, row tile): units lo .. hi of those that a row of the tile sees
struct Piece {
  int b, h, row0, n, q0, past, cap;
  int lo, hi;
  bool began, open;     // the item has units before, behind
  long long item_end;
};

template <int ROWS>
struct Cursor {
  long long at, end;    // the range that is left
  int b, h, tile, first;                                               // the item in which it begins, and its unit
  Piece p;

  __device__ __forceinline__ void init(const AttnParams& a, const long long* before, const Request* request, long long from, long long to) {
    at = from;
    end = to;
    int lo = 0, hi = a.s.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before[mid] <= at) lo = mid; else hi = mid;
    }
    b = lo;
    h = tile = first = 0;
    if (at < end) {
      const int units = request[b].units(a.window), tiles = (request[b].n * a.G + ROWS - 1) / ROWS;
      unsigned long long rel = at - before[b], item;
      if (rel >> 32) {
        item = rel / units;
        h = static_cast<int>(item / tiles);
      } else {
        item = static_cast<unsigned>(rel) / static_cast<unsigned>(units);
        h = static_cast<int>(static_cast<unsigned>(item) / static_cast<unsigned>(tiles));
      }
      tile = static_cast<int>(item - static_cast<unsigned long long>(h) * tiles);
      first = static_cast<int>(rel - item * units);
    }
  }

  // The next piece of the range; false at its end
  __device__ __forceinline__ bool next_piece(const AttnParams& a, const long long* before, const Request* request) {
    if (at >= end) return false;
    const Request r = request[b];
    const int units = r.units(a.window), tiles = (r.n * a.G + ROWS - 1) / ROWS, rest = units - first;
    const int count = static_cast<int>(min(static_cast<long long>(rest), end - at));
    p.b = b;
    p.h = h;
    p.row0 = tile * ROWS;
    p.n = r.n;
    p.q0 = r.q0;
    p.past = r.past;
    p.cap = r.cap;
    p.began = first > 0;
    p.open = count < rest;
    p.item_end = at + rest;
    // units that some row of the tile sees
    const int t0 = token_of(a, p.row0), t1 = min(token_of(a, p.row0 + ROWS - 1), r.n - 1), unit0 = r.unit0(a.window);
    const int from = a.window > 0 ? max(r.past + t0 - a.window + 1, 0) >> 6 : 0;
    const int to = min(r.past + t1 >= 0 ? ((r.past + t1) >> 6) + 1 : 0, (r.cap + 63) >> 6);
    p.lo = max(unit0 + first, from);
    p.hi = min(unit0 + first + count, to);
    at += count;
    first += count;
    if (count == rest) {
      first = 0;
      if (++tile == tiles) {
        tile = 0;
        if (++h == a.c.H) {
          h = 0;
          ++b;
          while (at < end && before[b + 1] <= at) ++b;
        }
      }
    }
    return true;
  }
};

// ------------------------------------------------------------------------------------- arithmetic
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Four codes as f16 numbers, 2^-24 of their values
__device__ __forceinline__ void decode(uint32_t w, uint32_t& b0, uint32_t& b1) {
  b0 = __byte_perm(w, 0u, 0x4140);
  b1 = __byte_perm(w, 0u, 0x4342);
}
constexpr uint32_t kMinus128 = 0x80808080u;              // two of -128 in that form
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void load4(uint32_t (&w)[4], const uint8_t* p) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  w[0] = v.x;
  w[1] = v.y;
  w[2] = v.z;
  w[3] = v.w;
}
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 1);
  return x + __shfl_xor_sync(0xffffffffu, x, 2);
}
// Exponent of a power of two (NaN for NaN)
__device__ __forceinline__ float log2_of_scale(float s) {
  const int e = static_cast<int>(__float_as_uint(s) >> 23) - 127;
  return e > 60 ? CUDART_NAN_F : static_cast<float>(e);
}

// Queries of one row, columns 16 r .. 16 r + 15 of each 64 for lane r of a quad.  Asked for first, taken up when the copies are under way: behind them
// they would wait for 30 MB (7000 cycles).
template <int D>
struct Query {
  uint4 v[D / 64][2];
  __device__ __forceinline__ void ask(const AttnParams& p, const Piece& it, int row) {
    const int t = token_of(p, row);
    const bf16* src = p.q + static_cast<long>(it.q0 + t) * p.ldq + static_cast<long>(it.h * p.G + row - t * p.G) * D + (threadIdx.x & 3) * 16;
#pragma unroll
    for (int h = 0; h < D / 64; ++h)
#pragma unroll
      for (int k = 0; k < 2; ++k) v[h][k] = t < it.n ? *reinterpret_cast<const uint4*>(src + h * 64 + k * 8) : make_uint4(0, 0, 0, 0);
  }
  // As f16 numbers, scaled; factor takes a product with code numbers to 2^-24 x / key scale, off is what the codes' offset adds to such a product
  __device__ __forceinline__ void take(float softmax_scale, uint32_t (&q)[D / 16][2], float& factor, float& off) const {
    unsigned top = 0;
#pragma unroll
    for (int h = 0; h < D / 64; ++h)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t w[4] = {v[h][k].x, v[h][k].y, v[h][k].z, v[h][k].w};
#pragma unroll
        for (int y = 0; y < 4; ++y) top = max(top, max(w[y] & 0x7fffu, (w[y] >> 16) & 0x7fffu));
      }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = static_cast<int>(top >> 7);                          // the largest magnitude is 2^(e - 127) at least
    const int up = min(140 - e, 126);
    const float f = softmax_scale < 0.f ? -__int_as_float((up + 127) << 23) : __int_as_float((up + 127) << 23);
    factor = e == 255 ? CUDART_NAN_F : __int_as_float((127 - up) << 23) * fabsf(softmax_scale);
    float sum = 0.f;
#pragma unroll
    for (int h = 0; h < D / 64; ++h)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t w[4] = {v[h][k].x, v[h][k].y, v[h][k].z, v[h][k].w};
#pragma unroll
        for (int y = 0; y < 4; ++y) {                                  // columns 16 r + 8 k + 2 y, + 1 of this half
          const float a = __int_as_float(w[y] << 16) * f, b = __int_as_float(w[y] & 0xffff0000u) * f;
          sum += a + b;
          q[h * 4 + k * 2 + (y >> 1)][y & 1] = pack_half(a, b);
        }
      }
    off = quad_sum(sum) * 0x1p-17f;
  }
};

// Scores s of two rows and some keys of a lane become probabilities.  get(row, n) is the reference to its n-th score, key(n) that one's token in the
// lane's sub-block, N of them; reduce() the maximum over the lanes that share the rows, rescale(f) multiplies their outputs.
// Where x or c is so large that m, b and x may round apart by a part of 1, scores are taken relative to the lane's largest first, so that no x is above 0; what
// fp32 then loses, it loses of scores that are as far apart.
constexpr float kFar = 0x1p19f;
// The largest probability is held as 2^15, near the end of f16's range: others have 11 bits down to 2^-29 of it.  Outputs and sums share the factor.
constexpr float kUp = 15.f;
struct Running {
  float factor[2], off[2];   // of the lane's two rows
  int pos[2];                // their positions; -1: no row
  float m[2], l[2];
};
template <int N, class Get, class Key, class Reduce, class Rescale>
__device__ __forceinline__ void references(Running& w, Get get, Key key, Reduce reduce, Rescale rescale, float2 scale, bool masked, int key0, int window,
                                           float (&a)[2], float (&b)[2], float& out) {
  const bool there = scale.x != 0.f;                                   // else a sub-block without a page
  const float ev = there ? log2_of_scale(scale.y) : 0.f, sk = there ? scale.x * 0x1p24f : 0.f;
  float c[2], top[2], ref[2];                                          // x = a s + c, a > 0
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    a[i] = w.factor[i] * sk;
    a[i] = a[i] == 0.f ? 0x1p-126f : a[i];
    c[i] = fmaf(-w.off[i], a[i], ev);
    top[i] = -CUDART_INF_F;
  }
  if (masked) {                                                        // some key of the unit is not seen by some row: such scores become -inf
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int to = there ? w.pos[i] - key0 : -1, from = window > 0 ? w.pos[i] - window - key0 : -1;      // from < key <= to
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (key(n) > to || key(n) <= from) get(i, n) = -CUDART_INF_F;
      if (to < 0 || from >= 15 || from >= to) {                        // a row that sees nothing of a page does not see that its scale is NaN
        a[i] = 1.f;
        c[i] = 0.f;
      }
    }
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    top[0] = fmaxf(top[0], get(0, n));
    top[1] = fmaxf(top[1], get(1, n));
  }
  float m[2];
  bool moved = false, far = false;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    m[i] = fmaxf(w.m[i], reduce(fmaf(top[i], a[i], c[i])));
    moved |= m[i] != w.m[i];
    ref[i] = m[i] == -CUDART_INF_F ? 0.f : m[i];
    far |= fmaxf(fabsf(ref[i]), fabsf(c[i])) > kFar;
    b[i] = c[i] - ref[i] + kUp;
  }
  if (__any_sync(0xffffffffu, moved || far)) {
    const float2 f = make_float2(ex2(w.m[0] - ref[0]), ex2(w.m[1] - ref[1]));
    w.m[0] = m[0];
    w.m[1] = m[1];
    w.l[0] *= f.x;
    w.l[1] *= f.y;
    rescale(f);
    if (far) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (top[i] == -CUDART_INF_F) continue;
        b[i] = fmaf(top[i], a[i], c[i]) - ref[i] + kUp;
#pragma unroll
        for (int n = 0; n < N; ++n) get(i, n) -= top[i];
      }
    }
  }
  out = ex2(-ev);
}
__device__ __forceinline__ void add_sum(float& l, float t, float out) { l += t == 0.f ? 0.f : t * out; }

// A warp's rows: queries as f16 operands, running maximum and sum, outputs.  The outputs have 128 times the sum of probabilities still in them, whose
// negative is off_o.
template <int D, int R>
struct Rows;

// 16 rows: scores S = Q K^T, lane 4c + r has rows c and c + 8, keys of sub-block r; outputs P V, the same rows, columns 8 d + 2 r, + 1
template <int D>
struct Rows<D, 16> : Running {
  using S = Shape<D>;
  Query<D> raw[2];
  uint32_t q[D / 16][4], pr[8][2];
  float o[D / 8][4], off_o[4];
  static __device__ __forceinline__ int sub_block() { return threadIdx.x & 3; }          // of a lane's keys
  static __device__ __forceinline__ int row(int i) { return (threadIdx.x & 31) / 4 + 8 * i; }

  __device__ __forceinline__ void clear() {
    m[0] = m[1] = -CUDART_INF_F;
    l[0] = l[1] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    off_o[0] = off_o[1] = off_o[2] = off_o[3] = 0.f;
  }
  __device__ __forceinline__ void settle() {             // takes the offset out of the outputs
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      float2* x = reinterpret_cast<float2*>(o[i]);
      x[0] = add2(x[0], make_float2(off_o[0], off_o[1]));
      x[1] = add2(x[1], make_float2(off_o[2], off_o[3]));
    }
    off_o[0] = off_o[1] = off_o[2] = off_o[3] = 0.f;
  }
  __device__ __forceinline__ void ask(const AttnParams& p, const Piece& it, int row0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) raw[i].ask(p, it, row0 + row(i));
  }
  __device__ __forceinline__ void take(float softmax_scale) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t half[D / 16][2];
      raw[i].take(softmax_scale, half, factor[i], off[i]);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        q[k][i] = half[k][0];
        q[k][i + 2] = half[k][1];
      }
    }
  }
  __device__ __forceinline__ void keys(const uint8_t* tile, float2 scale, bool masked, int key0, int window) {
    const int lane = threadIdx.x & 31, c = lane >> 2, r = lane & 3;
    const uint8_t* base = tile + (c >> 1) * S::kPitch + (c & 1) * 64 + r * 16;
    float s[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
    for (int g = 0; g < 8; g += 4)                                     // four tiles at a time: their products do not wait for one another
#pragma unroll
      for (int h = 0; h < D / 64; ++h) {
        uint32_t words[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) load4(words[j], base + ((g + j) * (D / 64) + h) * 128);
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t b0, b1;
            decode(words[j][y], b0, b1);
            mma(s[g + j], q[h * 4 + y], b0, b1);
          }
      }
    float a[2], b[2], out;
    references<16>(
        *this, [&](int i, int n) -> float& { return s[n >> 1][2 * i + (n & 1)]; }, [](int n) { return n; }, [](float x) { return quad_max(x); },
        [&](float2 f) {
#pragma unroll
          for (int i = 0; i < 4; ++i) off_o[i] *= i < 2 ? f.x : f.y;
#pragma unroll
          for (int d = 0; d < D / 8; ++d) {
            float2* x = reinterpret_cast<float2*>(o[d]);
            x[0] = mul2(x[0], make_float2(f.x, f.x));
            x[1] = mul2(x[1], make_float2(f.y, f.y));
          }
        },
        scale, masked, key0, window, a, b, out);
    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 x = fma2(make_float2(s[j][2 * i], s[j][2 * i + 1]), make_float2(a[i], a[i]), make_float2(b[i], b[i]));
        const float2 e = make_float2(ex2(x.x), ex2(x.y));
        sum[i] = add2(sum[i], e);
        pr[j][i] = pack_half(e.x, e.y);
      }
#pragma unroll
    for (int i = 0; i < 2; ++i) add_sum(l[i], sum[i].x + sum[i].y, out);
  }
  __device__ __forceinline__ void values(const uint8_t* tile) {
    const int lane = threadIdx.x & 31;
    const uint8_t* base = tile + (lane & 3) * S::kPitch + (lane >> 2) * 16;
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const uint32_t a[4] = {pr[2 * y][0], pr[2 * y][1], pr[2 * y + 1][0], pr[2 * y + 1][1]};
      mma(off_o, a, kMinus128, kMinus128);
    }
#pragma unroll
    for (int g = 0; g < D / 8; g += 4) {
      uint32_t words[4][4];
#pragma unroll
      for (int d = 0; d < 4; ++d) load4(words[d], base + (g + d) * 128);
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const uint32_t a[4] = {pr[2 * y][0], pr[2 * y][1], pr[2 * y + 1][0], pr[2 * y + 1][1]};
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          uint32_t b0, b1;
          decode(words[d][y], b0, b1);
          mma(o[g + d], a, b0, b1);
        }
      }
    }
  }
  __device__ __forceinline__ void sums() {
    settle();
    l[0] = quad_sum(l[0]);
    l[1] = quad_sum(l[1]);
  }
  __device__ __forceinline__ bool writes_sums() const { return (threadIdx.x & 3) == 0; }
  // Row i's outputs times f: as bf16, and as they are
  __device__ __forceinline__ void store(bf16* out, int i, float f) const {
#pragma unroll
    for (int d = 0; d < D / 8; ++d)
      *reinterpret_cast<__nv_bfloat162*>(out + d * 8 + (threadIdx.x & 3) * 2) = __floats2bfloat162_rn(o[d][2 * i] * f, o[d][2 * i + 1] * f);
  }
  __device__ __forceinline__ void store(float* out, int i) const {
#pragma unroll
    for (int d = 0; d < D / 8; ++d) *reinterpret_cast<float2*>(out + d * 8 + (threadIdx.x & 3) * 2) = make_float2(o[d][2 * i], o[d][2 * i + 1]);
  }
};

// 8 rows: scores transposed, S^T = K Q^T, lane 4c + r has rows 2r and 2r + 1, keys of sub-block c / 2; outputs O^T = V^T P^T, the same rows, columns
// 16 d + c, + 8.  Half the products and exponentials for the same codes; the probabilities change lanes once (movmatrix).
template <int D>
struct Rows<D, 8> : Running {
  using S = Shape<D>;
  Query<D> raw;
  uint32_t q[D / 16][2], pr[4][2];
  float o[D / 16][4], off_o[4];
  static __device__ __forceinline__ int sub_block() { return (threadIdx.x & 31) >> 3; }
  static __device__ __forceinline__ int row(int i) { return (threadIdx.x & 3) * 2 + i; }

  __device__ __forceinline__ void clear() {
    m[0] = m[1] = -CUDART_INF_F;
    l[0] = l[1] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    off_o[0] = off_o[1] = off_o[2] = off_o[3] = 0.f;
  }
  __device__ __forceinline__ void settle() {
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      float2* x = reinterpret_cast<float2*>(o[i]);
      x[0] = add2(x[0], make_float2(off_o[0], off_o[1]));
      x[1] = add2(x[1], make_float2(off_o[2], off_o[3]));
    }
    off_o[0] = off_o[1] = off_o[2] = off_o[3] = 0.f;
  }
  __device__ __forceinline__ void ask(const AttnParams& p, const Piece& it, int row0) { raw.ask(p, it, row0 + (threadIdx.x & 31) / 4); }
  __device__ __forceinline__ void take(float softmax_scale) {
    float f, c;
    raw.take(softmax_scale, q, f, c);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      factor[i] = __shfl_sync(0xffffffffu, f, row(i) * 4);
      off[i] = __shfl_sync(0xffffffffu, c, row(i) * 4);
    }
  }
  static __device__ __forceinline__ float over_keys(float x, bool sum) {
#pragma unroll
    for (int d = 4; d < 32; d *= 2) {
      const float y = __shfl_xor_sync(0xffffffffu, x, d);
      x = sum ? x + y : fmaxf(x, y);
    }
    return x;
  }
  __device__ __forceinline__ void keys(const uint8_t* tile, float2 scale, bool masked, int key0, int window) {
    const int lane = threadIdx.x & 31, c = lane >> 2, r = lane & 3;
    const uint8_t* base = tile + (c >> 1) * S::kPitch + (c & 1) * 64 + r * 16;
    float s[4][4];
#pragma unroll
    for (int y = 0; y < 4; ++y) s[y][0] = s[y][1] = s[y][2] = s[y][3] = 0.f;
#pragma unroll
    for (int h = 0; h < D / 64; ++h) {
      uint32_t words[8][4];
#pragma unroll
      for (int j = 0; j < 8; ++j) load4(words[j], base + (j * (D / 64) + h) * 128);
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          uint32_t a[4];
          decode(words[2 * y][k], a[0], a[2]);
          decode(words[2 * y + 1][k], a[1], a[3]);
          mma(s[y], a, q[h * 4 + k][0], q[h * 4 + k][1]);
        }
    }
    float a[2], b[2], out;
    // score n of row i: token 2n + c % 2
    references<8>(
        *this, [&](int i, int n) -> float& { return s[n >> 1][2 * (n & 1) + i]; }, [&](int n) { return 2 * n + (c & 1); },
        [](float x) { return over_keys(x, false); },
        [&](float2 f) {
          float2* t = reinterpret_cast<float2*>(off_o);
          t[0] = mul2(t[0], f);
          t[1] = mul2(t[1], f);
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            float2* x = reinterpret_cast<float2*>(o[d]);
            x[0] = mul2(x[0], f);
            x[1] = mul2(x[1], f);
          }
        },
        scale, masked, key0, window, a, b, out);
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int y = 0; y < 4; ++y)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float2 x = fma2(make_float2(s[y][2 * t], s[y][2 * t + 1]), make_float2(a[0], a[1]), make_float2(b[0], b[1]));
        const float2 e = make_float2(ex2(x.x), ex2(x.y));
        sum = add2(sum, e);
        asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(pr[y][t]) : "r"(pack_half(e.x, e.y)));
      }
    add_sum(l[0], sum.x, out);
    add_sum(l[1], sum.y, out);
  }
  __device__ __forceinline__ void values(const uint8_t* tile) {
    const int lane = threadIdx.x & 31;
    const uint8_t* base = tile + (lane & 3) * S::kPitch + (lane >> 2) * 16;
    const uint32_t minus[4] = {kMinus128, kMinus128, kMinus128, kMinus128};
#pragma unroll
    for (int y = 0; y < 4; ++y) mma(off_o, minus, pr[y][0], pr[y][1]);
#pragma unroll
    for (int g = 0; g < D / 16; g += 4) {
      uint32_t words[8][4];
#pragma unroll
      for (int d = 0; d < 8; ++d) load4(words[d], base + (2 * g + d) * 128);
#pragma unroll
      for (int y = 0; y < 4; ++y)
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          uint32_t a[4];
          decode(words[2 * d][y], a[0], a[2]);
          decode(words[2 * d + 1][y], a[1], a[3]);
          mma(o[g + d], a, pr[y][0], pr[y][1]);
        }
    }
  }
  __device__ __forceinline__ void sums() {
    settle();
    l[0] = over_keys(l[0], true);
    l[1] = over_keys(l[1], true);
  }
  __device__ __forceinline__ bool writes_sums() const { return (threadIdx.x & 31) < 4; }
  __device__ __forceinline__ void store(bf16* out, int i, float f) const {
#pragma unroll
    for (int d = 0; d < D / 8; ++d) out[d * 8 + (threadIdx.x & 31) / 4] = __float2bfloat16(o[d / 2][i + 2 * (d & 1)] * f);
  }
  __device__ __forceinline__ void store(float* out, int i) const {
#pragma unroll
    for (int d = 0; d < D / 8; ++d) out[d * 8 + (threadIdx.x & 31) / 4] = o[d / 2][i + 2 * (d & 1)];
  }
};

// Where row r of an item goes; nullptr: there is no such row
__device__ __forceinline__ bf16* row_of(const AttnParams& p, int n, int q0, int h, int row, int D) {
  const int t = token_of(p, row);
  return t < n ? p.o + (static_cast<long>(q0 + t) * p.Hq + h * p.G + row - t * p.G) * D : nullptr;
}
// What takes sums of probabilities and code numbers to the output
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 0x1p24f / l; }

template <int D, int R>
__global__ void __launch_bounds__(kThreads, 1) cache_attn_kernel(const __grid_constant__ AttnParams p) {
  using S = Shape<D>;
  extern __shared__ __align__(128) uint8_t raw_smem[];
  Smem<D, R>& sm = *reinterpret_cast<Smem<D, R>*>(raw_smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tc5::warp_index(), B = p.s.B;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- the units of all requests
  if (tid == 0) sm.abort_flag = 0;
  for (int i = tid; i < kWarps * S::kSlots; i += kThreads) tc5::mbar_init(&sm.full[0][0] + i, 32);
  tc5::fence_barrier_init();
  asm volatile("griddepcontrol.wait;" ::: "memory");                   // until here the kernel may run beside the one before it
  long long total = 0;
  for (int base = 0; base < B; base += kThreads) {
    const int b = base + tid;
    long long x = 0;
    if (b < B) {
      const Request r = request_of(p, b);
      sm.request[b] = r;
      x = static_cast<long long>(r.units(p.window)) * p.c.H * ((r.n * p.G + R - 1) / R);
    }
    const long long mine = x;
    for (int d = 1; d < 32; d <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    if (lane == 31) sm.warps[warp] = x;
    __syncthreads();
    long long below = total;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) below += sm.warps[w];
      total += sm.warps[w];
    }
    if (b < B) sm.before[b] = below + x - mine;
    __syncthreads();
  }
  if (tid == 0) sm.before[B] = total;
  __syncthreads();

  // ---- this worker's range
  const long long workers = static_cast<long long>(gridDim.x) * kWarps, each = max((total + workers - 1) / workers, 1ll);
  const long long begin = min((static_cast<long long>(blockIdx.x) * kWarps + warp) * each, total);
  Cursor<R> use, get;
  use.init(p, sm.before, sm.request, begin, min(begin + each, total));
  get = use;

  // ---- the producer's side: tile t of the range is the keys (even) or values (odd) of its unit t / 2
  uint8_t* ring = sm.ring[warp];
  int get_unit = 0, get_stop = 0;                                      // of the piece that `get` is in
  struct Where {
    int page, blk, head;
    bool have;
  };
  Where now{-1, 0, 0, false}, next = now, after = now;
  // Looks up the pages of the unit two ahead: one sub-block per lane, four of them
  auto look = [&]() {
    now = next;
    next = after;
    after.have = false;
    while (get_unit >= get_stop) {
      if (!get.next_piece(p, sm.before, sm.request)) return;
      get_unit = get.p.lo;
      get_stop = get.p.hi;
    }
    after.have = true;
    after.blk = get_unit * 4 + (lane & 3);
    after.head = get.p.h;
    // (no test of the entry here: that would wait for it)
    after.page = after.blk * 16 < get.p.cap ? p.s.table[static_cast<long>(get.p.b) * p.s.W + (after.blk >> (p.c.shift - 4))] : -1;
    ++get_unit;
  };
  int put = 0;                                                         // the slot of the next tile
  bool values = false;
  auto issue = [&]() {                                         // the next tile, if there is one
    if (!values) look();
    if (!now.have) return;
    const int slot = put;
    if (++put == S::kSlots) put = 0;
    // 16 bytes at a time by all lanes: a 2 KB bulk copy per sub-block took its lane 110 cycles, 520 a tile, in the way of the products
    const bool there = now.page >= 0 && now.page < p.c.pages;
    const long ph = static_cast<long>(there ? now.page : 0) * p.c.H + now.head;
    const uint8_t* mine = (values ? p.c.v : p.c.k) + ((ph << (p.c.shift - 4)) + (now.blk & ((1 << (p.c.shift - 4)) - 1))) * S::kSub;
    const unsigned mask = __ballot_sync(0xffffffffu, there);
    const uint32_t dst = tc5::smem_u32(ring + slot * S::kSlot) + lane * 16;
#pragma unroll
    for (int sub = 0; sub < 4; ++sub) {
      const uint8_t* src = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), sub)) + lane * 16;
      if (mask >> sub & 1)
#pragma unroll
        for (int k = 0; k < S::kSub / 512; ++k)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + sub * S::kPitch + k * 512), "l"(src + k * 512) : "memory");
    }
    if (!values && lane < 4)                                           // zeros where there is no page
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(tc5::smem_u32(&sm.scale[warp][slot][lane])), "l"(p.c.scale + ph * 2),
                   "r"(there ? 8 : 0)
                   : "memory");
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(tc5::smem_u32(&sm.full[warp][slot])) : "memory");
    values = !values;
  };
  bool ok = true;

  // ---- the consumer's side
  Rows<D, R> w;
  int slot = 0;                                                        // of the next tile, and how often the ring has gone round
  uint32_t round = 0;
  Left left{};
  left.some = use.at < use.end;
  Piece it{};
  bool held = false;                                                   // whether there is a piece whose sums are in w
  int u2 = 0, u2_end = 0, p0 = -1, p1 = -1, ahead = S::kSlots + 1;
  bool full = false, start = true, fresh = false;
  // One copy of the code at each place: 99 KB of instructions, with two, cost 10000 cycles a call in first fetches.  A turn issues a tile and takes one
  // up; keys and values of a unit take turns.  The first turn asks for queries, the next only issue (two of them only look up pages), so that a
  // tile is issued when the one that was in its place has been taken up.
#pragma unroll 1
  for (;;) {
    if (!start) {
      issue();
      if (ahead > 0) {
        --ahead;
        continue;
      }
    }
    while (u2 >= u2_end) {
      const long long piece_end = use.at;
      const bool more = use.next_piece(p, sm.before, sm.request);
      if (more) w.ask(p, use.p, use.p.row0);                           // arrives while the sums before are stored
      if (held) {
        w.sums();
        if (!it.began && !it.open) {                                   // the whole item: its rows are done
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            bf16* out = row_of(p, it.n, it.q0, it.h, it.row0 + w.row(i), D);
            if (out) w.store(out, i, inverse(w.l[i]));
          }
        } else {
          const bool is_head = it.began && !it.open && piece_end < use.end;                // more pieces follow
          float* dst = is_head ? p.head + (static_cast<long>(blockIdx.x) * kWarps + warp) * R * D : reinterpret_cast<float*>(ring);
          int* item = is_head ? left.head_item : left.tail_item;
          item[0] = it.b;
          item[1] = it.h;
          item[2] = it.row0;
          if (is_head) {
            left.head = 1;
          } else {                                                     // (the sums go where the ring was)
            left.tail = 1;
            left.began = it.began;
            left.open = it.open;
            left.tail_end = it.item_end;
            __syncwarp();
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (w.writes_sums()) sm.ml[warp][is_head ? 0 : 1][w.row(i)] = make_float2(w.m[i], w.l[i]);
            w.store(dst + w.row(i) * D, i);
          }
        }
      }
      held = more;
      if (!more) break;
      it = use.p;
      fresh = true;
      w.clear();
      // positions of the lane's two rows, and of the first and last one
      const int rows = it.n * p.G;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = token_of(p, it.row0 + w.row(i));
        w.pos[i] = at < it.n ? it.past + at : -1;
      }
      p0 = it.past + token_of(p, it.row0);
      p1 = it.past + token_of(p, min(it.row0 + R, rows) - 1);
      full = it.row0 + R <= rows;
      u2 = 2 * it.lo;
      u2_end = 2 * it.hi;
    }
    if (start) {
      start = false;
      continue;
    }
    ok = ok && held && tc5::mbar_wait_warp(&sm.full[warp][slot], round & 1, &sm.abort_flag, p.status, STATUS_TIMEOUT_SMEM_FULL);
    if (!ok) break;
    if (fresh) {
      w.take(p.scale);
      fresh = false;
    }
    const int key0 = (u2 >> 1) * 64;
    if (key0 <= p1 && (p.window == 0 || key0 + 63 > p0 - p.window)) {
      if (u2 & 1) {
        w.values(ring + slot * S::kSlot);
        if ((u2 & 7) == 7) w.settle();
      } else {
        const float2 scale = sm.scale[warp][slot][w.sub_block()];
        const bool whole = full && key0 + 63 <= p0 && (p.window == 0 || key0 > p1 - p.window);
        w.keys(ring + slot * S::kSlot, scale, !whole || __any_sync(0xffffffffu, scale.x == 0.f), key0 + 16 * w.sub_block(), p.window);
      }
    }
    __syncwarp();
    if (++slot == S::kSlots) {
      slot = 0;
      ++round;
    }
    ++u2;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (lane == 0) sm.left[warp] = left;
  __syncthreads();
  if (sm.abort_flag) {
    if (tid == 0) p.join[blockIdx.x].any = 0;
    return;
  }

  // ---- parts of one item in several workers meet; those of an item that goes beyond the CTA are left for the join
  const Left mine = sm.left[lane < kWarps ? lane : 0];
  const bool is = lane < kWarps;
  const unsigned some = __ballot_sync(0xffffffffu, is && mine.some), heads = __ballot_sync(0xffffffffu, is && mine.head);
  const unsigned tails = __ballot_sync(0xffffffffu, is && mine.tail), began = __ballot_sync(0xffffffffu, is && mine.tail && mine.began);
  const unsigned opens = __ballot_sync(0xffffffffu, is && mine.tail && mine.open);
  // Chains of contributions to one item: lane g looks at the one that worker g's last part begins (it begins its item, or is the first worker's), lane
  // kGroups at the first worker's head.
  int g1 = is ? lane : 0;
  bool open = is && (opens >> lane & 1);
  const bool chain = is ? (tails >> lane & 1) && (lane == 0 || !(began >> lane & 1)) : lane == kWarps && (heads & 1);
  unsigned from = is ? 0u : 1u;                                        // workers whose contribution is a head
  while (open && g1 + 1 < kWarps && (some >> (g1 + 1) & 1)) {
    ++g1;
    from |= heads & (1u << g1);
    open = !(heads >> g1 & 1) && (opens >> g1 & 1);
  }
  const bool before = !is || (began >> lane & 1), goes_on = chain && !before && open;
  if (warp == 0) {
    if (goes_on) {
      const Request rq = sm.request[mine.tail_item[0]];
      p.join[blockIdx.x] = Join{1, mine.tail_item[1], mine.tail_item[2], rq.n, rq.q0, 0, mine.tail_end, each};
    }
    if (!__any_sync(0xffffffffu, goes_on) && lane == 0) p.join[blockIdx.x].any = 0;
  }
  // A warp takes a row of a chain at a time, a lane D / 32 columns of it, all contributions at once.  Only the last of a chain, which closes it, may be a
  // head.
  constexpr int kCols = D / 32;
  for (unsigned chains = __ballot_sync(0xffffffffu, chain); chains; chains &= chains - 1) {
    const int which = __ffs(chains) - 1, first = which < kWarps ? which : 0, last = __shfl_sync(0xffffffffu, g1, which);
    const bool closed = __shfl_sync(0xffffffffu, static_cast<int>(from != 0), which);              // by a head
    const bool began_before = __shfl_sync(0xffffffffu, static_cast<int>(before), which), ends = !__shfl_sync(0xffffffffu, static_cast<int>(open), which);
    const int* item = which < kWarps ? sm.left[first].tail_item : sm.left[first].head_item;
    const Request rq = sm.request[item[0]];
    const int stop = last + !closed;                                   // tails: first .. stop - 1
    const float* head = p.head + (static_cast<long>(blockIdx.x) * kWarps + last) * R * D;
    const long part = (static_cast<long>(blockIdx.x) * 2 + (began_before ? 0 : 1)) * R;
#pragma unroll 2
    for (int row = warp; row < R; row += kWarps) {
      float2 x[kWarps + 1][kCols / 2], ml[kWarps + 1];
      const int at = row * D + lane * 2;
      ml[kWarps] = closed ? sm.ml[last][0][row] : make_float2(-CUDART_INF_F, 0.f);
#pragma unroll
      for (int c = 0; c < kCols / 2; ++c)
        x[kWarps][c] = closed ? *reinterpret_cast<const float2*>(head + at + c * 64) : make_float2(0.f, 0.f);
#pragma unroll
      for (int g = 0; g < kWarps; ++g) {
        const bool in = g >= first && g < stop;
        ml[g] = in ? sm.ml[g][1][row] : make_float2(-CUDART_INF_F, 0.f);
#pragma unroll
        for (int c = 0; c < kCols / 2; ++c)
          x[g][c] = in ? *reinterpret_cast<const float2*>(sm.ring[g] + (at + c * 64) * 4) : make_float2(0.f, 0.f);
      }
      float m = -CUDART_INF_F, l = 0.f;
#pragma unroll
      for (int g = 0; g <= kWarps; ++g) m = fmaxf(m, ml[g].x);
      const float ref = m == -CUDART_INF_F ? 0.f : m;
      float2 o[kCols / 2] = {};
#pragma unroll
      for (int g = 0; g <= kWarps; ++g) {
        const float f = ex2(ml[g].x - ref);
        l = fmaf(ml[g].y, f, l);
#pragma unroll
        for (int c = 0; c < kCols / 2; ++c) o[c] = fma2(x[g][c], make_float2(f, f), o[c]);
      }
      if (!began_before && ends) {
        bf16* out = row_of(p, rq.n, rq.q0, item[1], item[2] + row, D);
        const float n = inverse(l);
        if (out)
#pragma unroll
          for (int c = 0; c < kCols / 2; ++c) *reinterpret_cast<__nv_bfloat162*>(out + lane * 2 + c * 64) = __floats2bfloat162_rn(o[c].x * n, o[c].y * n);
      } else {
#pragma unroll
        for (int c = 0; c < kCols / 2; ++c) *reinterpret_cast<float2*>(p.part + part * D + at + c * 64) = o[c];
        if (lane == 0) p.part_ml[part + row] = make_float2(m, l);
      }
    }
  }
}

// Parts of items that several CTAs worked on: CTA (c, part) takes some rows of the item that begins in CTA c of the kernel before.  Rows of no request, before
// the first one's and behind the last one's, are in no item: all CTAs together set them to zero.
constexpr int kJoinParts = 4;
__device__ __forceinline__ void clear_rows(const AttnParams& p, long from, long to, long width) {      // width: 16-byte pieces of a row
  uint4* out = reinterpret_cast<uint4*>(p.o);
  const long step = static_cast<long>(gridDim.x) * kJoinParts * 128;
  for (long i = from * width + (static_cast<long>(blockIdx.x) * kJoinParts + blockIdx.y) * 128 + threadIdx.x; i < to * width; i += step)
    out[i] = make_uint4(0, 0, 0, 0);
}
template <int D, int R>
__global__ void __launch_bounds__(128) cache_attn_join_kernel(const __grid_constant__ AttnParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = blockIdx.x;
  const Join j = p.join[c];
  const int first = p.ends & 1 ? p.s.query_start[0] : 0, behind = p.ends & 2 ? p.s.query_start[p.s.B] : p.s.N;
  clear_rows(p, 0, min(first, p.s.N), static_cast<long>(p.Hq) * D / 8);
  clear_rows(p, max(behind, 0), p.s.N, static_cast<long>(p.Hq) * D / 8);
  if (!j.any) return;
  const int last = static_cast<int>((j.end - 1) / j.each / kWarps);
  for (int e = blockIdx.y * 128 + threadIdx.x; e < R * (D / 4); e += kJoinParts * 128) {
    const int row = e / (D / 4), d = (e % (D / 4)) * 4;
    bf16* out = row_of(p, j.n, j.q0, j.h, j.row0 + row, D);
    if (!out) continue;
    float m = -CUDART_INF_F, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int g0 = c; g0 <= last; g0 += 8) {                            // CTA c's second part, the first parts of those behind it, eight at once
      float2 ml[8];
      float4 x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int g = min(g0 + i, last);
        const long slot = (static_cast<long>(g) * 2 + (g == c)) * R + row;
        ml[i] = p.part_ml[slot];
        x[i] = *reinterpret_cast<const float4*>(p.part + slot * D + d);
        if (g0 + i > last) ml[i] = make_float2(-CUDART_INF_F, 0.f);
      }
      float mn = m;
#pragma unroll
      for (int i = 0; i < 8; ++i) mn = fmaxf(mn, ml[i].x);
      const float ref = mn == -CUDART_INF_F ? 0.f : mn, keep = ex2(m - ref);
      m = mn;
      l *= keep;
      o = make_float4(o.x * keep, o.y * keep, o.z * keep, o.w * keep);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float f = ex2(ml[i].x - ref);
        if (g0 + i > last) continue;
        l = fmaf(ml[i].y, f, l);
        o.x = fmaf(x[i].x, f, o.x);
        o.y = fmaf(x[i].y, f, o.y);
        o.z = fmaf(x[i].z, f, o.z);
        o.w = fmaf(x[i].w, f, o.w);
      }
    }
    const float f = inverse(l);
    __nv_bfloat162 y[2] = {__floats2bfloat162_rn(o.x * f, o.y * f), __floats2bfloat162_rn(o.z * f, o.w * f)};
    *reinterpret_cast<uint2*>(out + d) = *reinterpret_cast<uint2*>(y);
  }
}

template <int D, int R>
cudaError_t run(const AttnParams& p, int grid, cudaStream_t st) {
  constexpr int bytes = sizeof(Smem<D, R>);
  static_assert(bytes <= 232448, "shared memory of one CTA");
  int dev = 0;
  cudaGetDevice(&dev);
  static std::atomic<unsigned long long> ready{0};                     // devices on which the kernel may have this much shared memory
  cudaError_t e = cudaSuccess;
  if (dev > 63 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    e = cudaFuncSetAttribute(cache_attn_kernel<D, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    // the same division of shared memory for the join: an SM changes it only when it is empty
    if (e == cudaSuccess) e = cudaFuncSetAttribute(cache_attn_join_kernel<D, R>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return e;
    if (dev <= 63) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = kThreads;
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, cache_attn_kernel<D, R>, p);
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3(grid, kJoinParts);
  cfg.blockDim = 128;
  cfg.dynamicSmemBytes = 0;
  e = cudaLaunchKernelEx(&cfg, cache_attn_join_kernel<D, R>, p);
  nsa::count_launch(2);
  return e;
}

// Rows of a tile: 8 where a request's queries of one KV head are that many at most (16 heads of 128 on 2, 16 contexts of 16000 tokens: 22.2 us, with 16 28.0), else
// 16.  More rows are more tiles, each with its own pass over the keys, which L2 holds for the next one: two, four or eight warps with a tile each on the
// same copies were slower (32 rows 125 -> 170 us, 64 rows 42 -> 69, 128 rows 130 -> 202), since they wait for one another.
int tile_rows(long rows) { return rows <= 8 ? 8 : 16; }
}  // namespace

// Floats of scratch that nsa_cache_attention needs
extern "C" long nsa_cache_attention_scratch(int Hq, int H, int D, int max_new) {
  const long grid = nsa::sm_count(), rows = tile_rows(static_cast<long>(H > 0 ? Hq / H : 1) * max_new);
  return grid * kWarps * rows * D + grid * 2 * rows * (D + 2) + grid * static_cast<long>(sizeof(Join) / 4);
}

extern "C" int nsa_cache_attention(const void* q, long ldq, const void* kc, const void* vc, const float* scale, const int* table, const int* query_start,
                                   const int* lengths, void* o, float* scratch, int B, int W, int N, int pages, int Hq, int H, int D, int page_size,
                                   int window, float softmax_scale, int max_new, cudaStream_t st) {
  if (N == 0) return 0;
  if (B <= 0 || N < 0 || H <= 0 || Hq % H || (D != 64 && D != 128) || max_new < 1) return nsa::fail(NSA_ERR_SHAPE, "cache_attention: unsupported shape");
  AttnParams p{};
  p.q = static_cast<const bf16*>(q);
  p.ldq = ldq;
  p.c = CachePages{static_cast<uint8_t*>(const_cast<void*>(kc)), static_cast<uint8_t*>(const_cast<void*>(vc)), const_cast<float*>(scale), pages, H, D,
                   __builtin_ctz(page_size)};
  p.o = static_cast<bf16*>(o);
  p.Hq = Hq;
  p.G = Hq / H;
  p.per_g = ((1ull << 32) + p.G - 1) / p.G;
  p.window = window;
  p.scale = softmax_scale * 1.4426950408889634f;
  p.status = nsa::status_ptr();
  const int grid = nsa::sm_count(), rows = tile_rows(static_cast<long>(p.G) * max_new);
  p.part = scratch;
  p.part_ml = reinterpret_cast<float2*>(p.part + static_cast<long>(grid) * 2 * rows * D);
  p.join = reinterpret_cast<Join*>(p.part_ml + static_cast<long>(grid) * 2 * rows);
  p.head = reinterpret_cast<float*>(p.join + grid);
  cudaError_t e = cudaSuccess;
  for (int b = 0; b < B && e == cudaSuccess; b += kMaxRequests) {      // a launch for each 768 requests, on the same scratch
    p.s = CacheStep{table + static_cast<long>(b) * W, query_start + b, lengths + b, B - b < kMaxRequests ? B - b : kMaxRequests, W, N};
    p.ends = (b == 0 ? 1 : 0) | (b + kMaxRequests >= B ? 2 : 0);
    if (D == 128)
      e = rows == 8 ? run<128, 8>(p, grid, st) : run<128, 16>(p, grid, st);
    else
      e = rows == 8 ? run<64, 8>(p, grid, st) : run<64, 16>(p, grid, st);
  }
  return e == cudaSuccess ? 0 : nsa::fail_cuda(e, "nsa_cache_attention launch");
}
