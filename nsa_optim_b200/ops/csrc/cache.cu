// The paged 8-bit key / value cache: pages and slots of a step, appending, reading back.
#include <cuda_bf16.h>

#include <type_traits>

#include "cache.cuh"
#include "host.cuh"
#include "packed.cuh"
#include "rope.cuh"

namespace {
typedef __nv_bfloat16 bf16;

// ------------------------------------------------------------------------------------- pages and slots of a step
// A few thousand numbers at most: what counts is the chain of dependent loads (lengths and counts together, then a page number) and barriers, so each
// CTA scans all requests by itself and no CTA waits for another.  64 requests of one token 3.3 us, 512 requests with 65 K tokens 4.8 us.
constexpr int kPlanThreads = 1024;

// Exclusive prefix of a value per thread over the CTA, and the total
template <class T>
__device__ __forceinline__ T scan(T mine, T& total, T* warps) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, n = blockDim.x >> 5;
  T x = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const T u = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += u;
  }
  if (lane == 31) warps[w] = x;
  __syncthreads();
  T y = lane < n ? warps[lane] : 0;                                    // each warp scans the warps' sums
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const T u = __shfl_up_sync(0xffffffffu, y, d);
    if (lane >= d) y += u;
  }
  total = __shfl_sync(0xffffffffu, y, 31);
  const T before = __shfl_sync(0xffffffffu, y, w ? w - 1 : 0);
  return x - mine + (w ? before : 0);
}

__device__ __forceinline__ int pages_for(long long tokens, int shift) { return static_cast<int>((tokens + (1 << shift) - 1) >> shift); }

// Every CTA scans all requests (first token, first new page and length of each in shared memory) and writes its share of the table's new entries and of
// the slots.
__global__ void __launch_bounds__(kPlanThreads) cache_plan_kernel(const int* __restrict__ lengths, const int* __restrict__ add, int* __restrict__ table,
                                                                  const int* __restrict__ free_pages, const int* __restrict__ free_count, int F,
                                                                  int* __restrict__ query_start, int* __restrict__ total,
                                                                  long long* __restrict__ slots, long long* __restrict__ positions,
                                                                  int* __restrict__ free_left, int* __restrict__ shortfall, int B, int W, int N,
                                                                  int shift) {
  extern __shared__ int plan_smem[];
  __shared__ long long warps[3][32];
  int *start = plan_smem, *first = start + B + 1, *length = first + B + 1;
  const int t = threadIdx.x, threads = blockDim.x, have = *free_count;
  long long tokens = 0, pages = 0, wanted = 0;
  for (int base = 0; base < B; base += threads) {
    const int b = base + t, len = b < B ? max(lengths[b], 0) : 0;
    const long long mine = b < B ? max(add[b], 0) : 0;
    long long all, all_take, all_lack;
    const long long from = tokens + scan(mine, all, warps[0]);
    const long long lo = min(from, static_cast<long long>(N)), hi = min(from + mine, static_cast<long long>(N));
    const int held = pages_for(len, shift), need = pages_for(len + (hi - lo), shift);
    const long long take = min(need, W) - min(held, W), lack = need - held;
    const long long before = pages + scan(take, all_take, warps[1]);
    scan(lack, all_lack, warps[2]);
    if (b < B) {
      start[b] = static_cast<int>(lo);
      first[b] = static_cast<int>(before);
      length[b] = len;
      if (blockIdx.x == 0) {
        query_start[b] = static_cast<int>(lo);
        total[b] = static_cast<int>(len + (hi - lo));
      }
    }
    tokens += all;
    pages += all_take;
    wanted += all_lack;
    if (base + threads < B) __syncthreads();                           // the sums have been read
  }
  const int count = min(max(have, 0), F);
  if (t == 0) {
    start[B] = static_cast<int>(min(tokens, static_cast<long long>(N)));
    first[B] = static_cast<int>(pages);
    if (blockIdx.x == 0) {
      const int got = static_cast<int>(min(pages, static_cast<long long>(count)));
      query_start[B] = start[B];
      *free_left = count - got;
      *shortfall = static_cast<int>(wanted - got);
    }
  }
  __syncthreads();
  // new entries: entry `order` belongs to the last request whose first one is not behind it
  auto find = [&](const int* from, long long what) {
    int lo = 0, hi = B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (from[mid] <= what) lo = mid; else hi = mid;
    }
    return lo;
  };
  const int step = gridDim.x * threads, me = blockIdx.x * threads + t;
  for (long long order = me; order < pages; order += step) {
    const int b = find(first, order);
    table[static_cast<long>(b) * W + pages_for(length[b], shift) + (order - first[b])] = order < count ? free_pages[count - 1 - order] : -1;
  }
  for (long long i = me; i < N; i += step) {
    long long slot = -1, pos = 0;
    if (i < start[B]) {
      const int b = find(start, i), len = length[b], held = pages_for(len, shift);
      pos = len + (i - start[b]);
      const long long j = pos >> shift;
      int page = -1;
      if (j < W) {
        const long long order = first[b] + (j - held);
        page = j < held ? table[static_cast<long>(b) * W + j] : order < count ? free_pages[count - 1 - order] : -1;
      }
      if (page >= 0) slot = (static_cast<long long>(page) << shift) + (pos & ((1 << shift) - 1));
    }
    slots[i] = slot;
    positions[i] = pos;
  }
}

// One CTA: the pages of finished requests go on the stack in the order of requests and pages.
__global__ void __launch_bounds__(kPlanThreads) cache_release_kernel(const uint8_t* __restrict__ finished, const int* __restrict__ lengths,
                                                                     int* __restrict__ table, int* __restrict__ free_pages,
                                                                     const int* __restrict__ free_count, int F, int* __restrict__ total,
                                                                     int* __restrict__ free_left, int B, int W, int shift) {
  __shared__ int have[kPlanThreads];
  __shared__ long long warps[32];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  long long at = min(max(*free_count, 0), F);
  for (int base = 0; base < B; base += kPlanThreads) {
    const int end = min(B - base, kPlanThreads);
    for (int i = warp; i < end; i += kPlanThreads / 32) {
      const int b = base + i;
      int n = 0;
      if (finished[b]) {
        const int held = min(pages_for(max(lengths[b], 0), shift), W);
        for (int j = lane; j < (held + 31) / 32 * 32; j += 32)
          n += __popc(__ballot_sync(0xffffffffu, j < held && table[static_cast<long>(b) * W + j] >= 0));
      }
      if (lane == 0) have[i] = n;
    }
    __syncthreads();
    long long all;
    const long long before = scan(static_cast<long long>(t < end ? have[t] : 0), all, warps);
    if (t < end) have[t] = static_cast<int>(before);
    __syncthreads();
    for (int i = warp; i < end; i += kPlanThreads / 32) {
      const int b = base + i;
      if (finished[b]) {
        const int held = min(pages_for(max(lengths[b], 0), shift), W);
        long long place = at + have[i];
        for (int j = lane; j < (W + 31) / 32 * 32; j += 32) {
          const int page = j < W ? table[static_cast<long>(b) * W + j] : -1;
          const bool give = j < held && page >= 0;
          const unsigned mask = __ballot_sync(0xffffffffu, give);
          const long long p = place + __popc(mask & ((1u << lane) - 1));
          if (give && p < F) free_pages[p] = page;
          if (j < W) table[static_cast<long>(b) * W + j] = -1;
          place += __popc(mask);
        }
      }
      if (lane == 0) total[b] = finished[b] ? 0 : lengths[b];
    }
    at += all;
    __syncthreads();
  }
  if (t == 0) *free_left = static_cast<int>(min(at, static_cast<long long>(F)));
}

// ------------------------------------------------------------------------------------- appending
// The exponent e of the smallest power of two of which no value up to amax needs more than 127 (bits of amax: 127 * 2^e has the mantissa
// 1.984375, 0x7e0000 in fp32), -60 at least; kNoStep where amax is not finite or needs more than 2^60.
constexpr int kMinExp = -60, kMaxExp = 60, kNoStep = 1 << 20;
__device__ __forceinline__ int step_exponent(unsigned amax_bits) {
  const int x = static_cast<int>(amax_bits >> 23) - 127;           // amax = 1.m * 2^x; 127 * 2^e = 1.984375 * 2^(e+6)
  const int e = (amax_bits & 0x7fffffu) <= 0x7e0000u ? x - 6 : x - 5;
  return amax_bits >= 0x7f800000u || e > kMaxExp ? kNoStep : max(e, kMinExp);
}
__device__ __forceinline__ float power2(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ int exponent_of(float scale) {
  const int e = static_cast<int>(__float_as_uint(scale) >> 23) - 127;
  return e > kMaxExp ? kNoStep : max(e, kMinExp);
}
// 128 + x * step, rounded to the nearest whole number (half to even), in the low byte: 1.5 * 2^23 leaves no bits behind the point
__device__ __forceinline__ uint32_t code_of(float x, float step) { return __float_as_uint(fmaf(x, step, 12583040.f)); }
__device__ __forceinline__ uint32_t bytes4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
__device__ __forceinline__ float low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// Codes of one byte each on the grid that is `ratio` times coarser
__device__ __forceinline__ uint32_t coarser(uint32_t w, float ratio) {
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = code_of(static_cast<float>(w >> (8 * i) & 0xff) - 128.f, ratio);
  return bytes4(c[0], c[1], c[2], c[3]);
}

// Quotient of numbers that are the same for all threads or nearly so: most often there is nothing to divide, or a power of two to divide by
__device__ __forceinline__ int over(int y, int n) { return n == 1 ? y : (n & (n - 1)) == 0 ? y >> (31 - __clz(n)) : y / n; }

// One CTA per window of packed tokens, head and side.  The tokens of a request that lie in one page are a group, handled by the CTA in whose window the
// first of them lies: their largest magnitude gives the page's scale, codes that are there are rounded again where it grows, then the new ones are
// stored.  A warp takes 16 tokens of 32 * C columns at a time, a lane C columns of them, so that it reads whole rows of 64 or 128 columns, its 16 tokens are
// 16 bytes of each column of the values, and what it holds in registers between the maximum and the codes is read once (one such block; pages of
// 256 tokens with more than 128 columns read the rest again).  The request, its length and the total come from one load each, side by side, and the page
// number beside the tokens: what is left in a row is that, the tokens, a barrier and the codes.  34.7 K tokens of 8 heads of 128 columns: 50 us, 4.4 TB/s
// of what it moves (142 MB read, 75 written), half of the issue slots (820 instructions for a warp's 64 codes a lane).  64 registers: twice as many warps as
// 128 would allow are worth the 20 words that do not fit (with reading back, when that took 89, 48 101, 56 91.5, 80 92.2, 128 96.3).
template <int C>
struct Block {                             // 16 tokens, C columns of a lane
  uint32_t w[16][C / 2];
};
// Tokens from .. to of t0 .. t0 + 15; FULL: all of them.  src: token t0's row, which may lie outside.
template <int C, bool FULL>
__device__ __forceinline__ void load_block(Block<C>& x, const bf16* src, long ld, int t0, int from, int to) {
#pragma unroll
  for (int t = 0; t < 16; ++t) {
    const bool in = FULL || (t0 + t >= from && t0 + t < to);
    if (C == 4) {
      const uint2 v = in ? __ldcs(reinterpret_cast<const uint2*>(src + t * ld)) : make_uint2(0, 0);
      x.w[t][0] = v.x;
      x.w[t][C / 2 - 1] = v.y;
    } else {
      x.w[t][0] = in ? __ldcs(reinterpret_cast<const uint32_t*>(src + t * ld)) : 0u;
    }
  }
}
// Rotary positions on the way in: tables of cosines and sines (L, R/2), fp32
enum { kAsIs, kHalves, kPairs };
struct Turning {
  const float *cs, *sn;
  int L, R;
};
// Columns d .. d + C - 1 of a token at position pos, turned and rounded as the kernel of rope.cu does it.  A warp has whole rows of 32 C columns, R at most,
// so a column's other half is in another lane.
template <int C, int MODE>
__device__ __forceinline__ void turn_columns(uint32_t (&w)[C / 2], const Turning& z, long pos, int d) {
  const bool in = pos >= 0 && pos < z.L, mine = d < z.R;
  const int half = z.R / 2, lane = threadIdx.x & 31;
  float x[C];
#pragma unroll
  for (int c = 0; c < C / 2; ++c) x[2 * c] = low(w[c]), x[2 * c + 1] = high(w[c]);
  if constexpr (MODE == kPairs) {
    float cc[C / 2], ss[C / 2];
    const long at = pos * half + d / 2;
#pragma unroll
    for (int c = 0; c < C / 2; ++c) {
      cc[c] = mine ? (in ? __ldg(z.cs + at + c) : rope::nan()) : 1.f;
      ss[c] = mine ? (in ? __ldg(z.sn + at + c) : rope::nan()) : 0.f;
    }
    if (!mine) return;
#pragma unroll
    for (int c = 0; c < C / 2; ++c) {
      rope::turn(x[2 * c], x[2 * c + 1], cc[c], ss[c]);
      w[c] = rope::pack(x[2 * c], x[2 * c + 1]);
    }
  } else {
    const bool second = d >= half;
    const int from = mine ? (second ? lane - half / C : lane + half / C) : lane;
    const long at = pos * half + (second ? d - half : d);
    float o[C], cc[C], ss[C];
    if constexpr (C == 4) {
      const float4 nan = make_float4(rope::nan(), rope::nan(), rope::nan(), rope::nan());
      const float4 a = mine && in ? __ldg(reinterpret_cast<const float4*>(z.cs + at)) : nan, b = mine && in ? __ldg(reinterpret_cast<const float4*>(z.sn + at)) : nan;
      cc[0] = a.x, cc[1] = a.y, cc[C - 2] = a.z, cc[C - 1] = a.w;
      ss[0] = b.x, ss[1] = b.y, ss[C - 2] = b.z, ss[C - 1] = b.w;
    } else {
      const float2 nan = make_float2(rope::nan(), rope::nan());
      const float2 a = mine && in ? __ldg(reinterpret_cast<const float2*>(z.cs + at)) : nan, b = mine && in ? __ldg(reinterpret_cast<const float2*>(z.sn + at)) : nan;
      cc[0] = a.x, cc[1] = a.y;
      ss[0] = b.x, ss[1] = b.y;
    }
#pragma unroll
    for (int c = 0; c < C / 2; ++c) {
      const uint32_t v = __shfl_sync(0xffffffffu, w[c], from);
      o[2 * c] = low(v), o[2 * c + 1] = high(v);
    }
    if (!mine) return;
    const float2 sign = second ? make_float2(1.f, 1.f) : make_float2(-1.f, -1.f);      // the half's own side of the turn: the same roundings
#pragma unroll
    for (int c = 0; c < C; c += 2) {
      const float2 y = fma2(make_float2(x[c], x[c + 1]), make_float2(cc[c], cc[c + 1]),
                            mul2(make_float2(o[c], o[c + 1]), mul2(make_float2(ss[c], ss[c + 1]), sign)));
      x[c] = y.x, x[c + 1] = y.y;
    }
#pragma unroll
    for (int c = 0; c < C / 2; ++c) w[c] = rope::pack(x[2 * c], x[2 * c + 1]);
  }
}
// The tokens from .. to of a block in columns d ..; its token t is at position base + t0 + t.
template <int C, int MODE>
__device__ __forceinline__ void turn_block(Block<C>& x, const Turning& z, long base, int d, int t0, int from, int to) {
#pragma unroll 4
  for (int t = 0; t < 16; ++t)
    if (t0 + t >= from && t0 + t < to) turn_columns<C, MODE>(x.w[t], z, base + t0 + t, d);
}
// Queries of a window of tokens, heads h0 .. h1.  The tokens' positions are looked up first; then a thread has 2 V columns of a head at a time, two pieces of
// V (their halves, or neighbours), and two heads or tokens in flight.
constexpr int kMostWindow = 256;
template <int MODE, int V>
__device__ __forceinline__ void turn_queries(const bf16* __restrict__ q, long ldq, bf16* __restrict__ y, const Turning& z, const CacheStep& s, int Hq, int h0,
                                             int h1, int D, int i0, int i1) {
  __shared__ int at[kMostWindow];                                      // a token's row of the tables; -1: outside of them; -2: of no request
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, half = z.R / 2;
  if (i0 + warp < i1) {
    Request r = request_at(s.query_start, s.lengths, s.B, i0 + warp);
    for (int i = i0 + warp; i < i1; i += warps) {
      if (i >= r.next) r = request_at(s.query_start, s.lengths, s.B, i);
      const long pos = static_cast<long>(r.length) - r.next + i;
      if (lane == 0) at[i - i0] = i < r.first || i >= r.next ? -2 : pos >= 0 && pos < z.L ? static_cast<int>(pos) : -1;
    }
  }
  __syncthreads();
  const int units = D / (2 * V), heads = h1 - h0, n = (i1 - i0) * heads * units;
  using Piece = typename std::conditional<V == 8, uint4, uint2>::type;
#pragma unroll 2
  for (int k = threadIdx.x; k < n; k += blockDim.x) {
    const int rest = over(k, units), u = k - rest * units, tok = over(rest, heads), h = h0 + rest - tok * heads, pos = at[tok];
    const bool turned = u * 2 * V < z.R;
    const int da = turned && MODE == kHalves ? u * V : u * 2 * V, db = turned && MODE == kHalves ? da + half : da + V;
    const bf16* src = q + static_cast<long>(i0 + tok) * ldq + h * D;
    bf16* dst = y + (static_cast<long>(i0 + tok) * Hq + h) * D;
    union {
      Piece p[2];
      uint32_t w[V];
    } x;
    x.p[0] = __ldcs(reinterpret_cast<const Piece*>(src + da));
    x.p[1] = __ldcs(reinterpret_cast<const Piece*>(src + db));
    if (turned) {
      float v[2 * V], c[V], d[V];
#pragma unroll
      for (int e = 0; e < V; ++e) v[2 * e] = low(x.w[e]), v[2 * e + 1] = high(x.w[e]);
#pragma unroll
      for (int e = 0; e < V; e += 4) {
        const float4 nan = make_float4(rope::nan(), rope::nan(), rope::nan(), rope::nan());
        const float4 a = pos >= 0 ? __ldg(reinterpret_cast<const float4*>(z.cs + static_cast<long>(pos) * half + u * V + e)) : nan;
        const float4 b = pos >= 0 ? __ldg(reinterpret_cast<const float4*>(z.sn + static_cast<long>(pos) * half + u * V + e)) : nan;
        c[e] = a.x, c[e + 1] = a.y, c[e + 2] = a.z, c[e + 3] = a.w;
        d[e] = b.x, d[e + 1] = b.y, d[e + 2] = b.z, d[e + 3] = b.w;
      }
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        constexpr int A = MODE == kHalves ? 1 : 2, B = MODE == kHalves ? V : 1;        // between pairs, and between the two columns of one
        float2 a = make_float2(v[A * e], v[A * e + A]), b = make_float2(v[A * e + B], v[A * e + A + B]);
        rope::turn(a, b, make_float2(c[e], c[e + 1]), make_float2(d[e], d[e + 1]));
        v[A * e] = a.x, v[A * e + A] = a.y, v[A * e + B] = b.x, v[A * e + A + B] = b.y;
      }
#pragma unroll
      for (int e = 0; e < V; ++e) x.w[e] = rope::pack(v[2 * e], v[2 * e + 1]);
    }
    if (pos == -2)
#pragma unroll
      for (int e = 0; e < V; ++e) x.w[e] = 0;
    __stcs(reinterpret_cast<Piece*>(dst + da), x.p[0]);
    __stcs(reinterpret_cast<Piece*>(dst + db), x.p[1]);
  }
}

template <int C>
__device__ __forceinline__ unsigned amax_of(const Block<C>& x) {
  unsigned m = 0;                          // magnitudes as bits, two 16-bit numbers at a time: NaN above infinity above all numbers
#pragma unroll
  for (int t = 0; t < 16; ++t)
#pragma unroll
    for (int c = 0; c < C / 2; ++c) m = __vmaxu2(m, x.w[t][c] & 0x7fff7fffu);
  return max(m << 16, m & 0xffff0000u);
}
// Codes of a block whose 16 tokens are all new
template <int C>
__device__ __forceinline__ void store_full(uint8_t* codes, const Block<C>& x, bool values, int D, int d, int t0, float inv) {
  if (values) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      uint32_t w[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t n[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t v = x.w[4 * q + i][c / 2];
          n[i] = code_of(c & 1 ? high(v) : low(v), inv);
        }
        w[q] = bytes4(n[0], n[1], n[2], n[3]);
      }
      *reinterpret_cast<uint4*>(codes + value_at(t0, d + c, D)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  } else {
    uint8_t* at = codes + key_at(t0, d, D);
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      const uint32_t a = code_of(low(x.w[t][0]), inv), b = code_of(high(x.w[t][0]), inv);
      uint8_t* to = at + (t >> 1) * 2 * D + (t & 1) * 64;
      if (C == 4) *reinterpret_cast<uint32_t*>(to) = bytes4(a, b, code_of(low(x.w[t][C / 2 - 1]), inv), code_of(high(x.w[t][C / 2 - 1]), inv));
      else *reinterpret_cast<uint16_t*>(to) = static_cast<uint16_t>(__byte_perm(a, b, 0x0040));
    }
  }
}
// Codes of a block, and of what is in its place: tokens before `from` are rounded to a grid coarser by `ratio` (1: left), from .. to are new.
template <int C>
__device__ __forceinline__ void store_keys(uint8_t* codes, const Block<C>& x, int D, int d, int t0, int from, int to, float ratio, float inv, bool bad) {
#pragma unroll
  for (int t = 0; t < 16; ++t) {
    const int tok = t0 + t;
    uint8_t* at = codes + key_at(tok, d, D);
    uint32_t w = 0x80808080u;
    if (tok >= from && tok < to) {
      if (!bad) {
        const uint32_t a = code_of(low(x.w[t][0]), inv), b = code_of(high(x.w[t][0]), inv);
        w = bytes4(a, b, C == 4 ? code_of(low(x.w[t][C / 2 - 1]), inv) : 0, C == 4 ? code_of(high(x.w[t][C / 2 - 1]), inv) : 0);
      }
    } else if (tok < from && ratio != 1.f) {
      w = coarser(C == 4 ? *reinterpret_cast<const uint32_t*>(at) : *reinterpret_cast<const uint16_t*>(at), ratio);
    } else {
      continue;
    }
    if (C == 4) *reinterpret_cast<uint32_t*>(at) = w;
    else *reinterpret_cast<uint16_t*>(at) = static_cast<uint16_t>(w);
  }
}
template <int C>
__device__ __forceinline__ void store_values(uint8_t* codes, const Block<C>& x, int D, int d, int t0, int from, int to, float ratio, float inv, bool bad) {
#pragma unroll
  for (int c = 0; c < C; ++c) {
    uint4* at = reinterpret_cast<uint4*>(codes + value_at(t0, d + c, D));
    uint32_t w[4] = {0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u};
    if (t0 < from || t0 + 16 > to) {                                   // some of the 16 are others
      const uint4 v = *at;
      w[0] = v.x;
      w[1] = v.y;
      w[2] = v.z;
      w[3] = v.w;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t n[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t v = x.w[4 * q + i][c / 2];
        n[i] = bad ? 128u : code_of(c & 1 ? high(v) : low(v), inv);
      }
      const uint32_t fresh = bytes4(n[0], n[1], n[2], n[3]), old = ratio != 1.f ? coarser(w[q], ratio) : w[q];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tok = t0 + 4 * q + i;
        const uint32_t byte = 0xffu << (8 * i);
        w[q] = tok >= to ? w[q] : (w[q] & ~byte) | ((tok >= from ? fresh : old) & byte);
      }
    }
    *at = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// MODE other than kAsIs: keys are turned on the way, and the CTAs behind those of a window's keys and values turn its queries, kQueryHeads heads each: the
// ones wait for their groups, the others for memory.  (A block's 16 tokens are turned in a loop that indexes them, so that blocks lie in local memory, the values' too:
// 64 bytes of C = 2 and 128 of C = 4 beside spills.)  31.7 K tokens of 32 query and 8 cache heads of 128 (714 MB) 155 us, 4.6 TB/s; with all windows of keys
// and values first 167; with 2 / 8 / 16 heads of queries 163 / 160 / 182, with one or three of them in flight 155 and 157 and four 165, in 56 or 80 registers 165 and
// 182.
constexpr int kQueryHeads = 4;
struct Queries {
  const bf16* q;
  long ld;
  bf16* y;
  int H;
};
template <int C, int MODE>
__device__ __forceinline__ void append_window(const bf16* __restrict__ k, const bf16* __restrict__ v, long ldk, long ldv, const CachePages& c, const CacheStep& s,
                                              int at, int window, const Turning& turning, int h, bool values) {
  __shared__ unsigned red[16];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, warps = blockDim.x >> 5, D = c.D, P = 1 << c.shift;
  const bf16* x = (values ? v : k) + h * D;
  const long ld = values ? ldv : ldk;
  const int slabs = D / (32 * C), all = s.query_start[s.B];
  int i = at * window;
  Request r = request_at(s.query_start, s.lengths, s.B, i);
  const int total = min(all, s.N), end = min(i + window, total);
  while (i < end) {
    if (i >= r.next) r = request_at(s.query_start, s.lengths, s.B, i);
    if (i < r.first) {                                                 // of no request: the first one begins behind it
      i = r.first;
      continue;
    }
    const long pos = static_cast<long>(r.length) - r.next + i;
    const int off = static_cast<int>(pos & (P - 1)), m = max(min(min(r.next, total) - i, P - off), 1);
    if (off != 0 && i != r.first) {                                    // of a group that began in another window
      i += m;
      continue;
    }
    const int page = page_of(s, c, r.b, pos);                          // on its way beside the tokens
    // blocks of the group: 16 tokens each from off / 16 on, by columns
    const int g0 = off >> 4, blocks = (((off + m - 1) >> 4) - g0 + 1) * slabs;
    const bf16* src = x + static_cast<long>(i) * ld;
    Block<C> held;
    unsigned top = 0;
    auto full = [&](int t0) { return t0 >= off && t0 + 16 <= off + m; };
    auto get = [&](int y) {
      const int yt = over(y, slabs), t0 = (g0 + yt) * 16;
      const bf16* row = src + (t0 - off) * ld + (y - yt * slabs) * 32 * C + lane * C;
      if (full(t0)) load_block<C, true>(held, row, ld, t0, off, off + m);
      else load_block<C, false>(held, row, ld, t0, off, off + m);
      if (MODE != kAsIs && !values) turn_block<C, MODE>(held, turning, pos - off, (y - yt * slabs) * 32 * C + lane * C, t0, off, off + m);
    };
    for (int y = warp + warps; y < blocks; y += warps) {
      get(y);
      top = max(top, amax_of(held));
    }
    if (warp < blocks) {
      get(warp);
      top = max(top, amax_of(held));
    }
    const long ph = static_cast<long>(max(page, 0)) * c.H + h;
    const float before = c.scale[ph * 2 + values];
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) red[warp] = top;
    __syncthreads();
    for (int w = 0; w < warps; ++w) top = max(top, red[w]);
    i += m;
    __syncthreads();                                                   // the maxima have been read; and the scale
    if (page < 0) continue;
    int e = step_exponent(top), old = e;
    if (off) {
      old = exponent_of(before);
      e = max(e, old);
    }
    const bool bad = e == kNoStep;
    const float inv = bad ? 0.f : power2(-e), ratio = bad ? 1.f : power2(max(old - e, -126));
    uint8_t* codes = (values ? c.v : c.k) + ph * P * D;
    for (int y = warp; y < blocks; y += warps) {
      if (y != warp) get(y);
      const int yt = over(y, slabs), d = (y - yt * slabs) * 32 * C + lane * C, t0 = (g0 + yt) * 16;
      if (full(t0) && !bad) store_full(codes, held, values, D, d, t0, inv);
      else if (values) store_values(codes, held, D, d, t0, off, off + m, ratio, inv, bad);
      else store_keys(codes, held, D, d, t0, off, off + m, ratio, inv, bad);
    }
    if (ratio != 1.f)                                                  // all codes before the group's blocks: bytes, whatever their order
      for (int y = t * 16; y < g0 * 16 * D; y += blockDim.x * 16) {
        uint4* at = reinterpret_cast<uint4*>(codes + y);
        const uint4 w = *at;
        *at = make_uint4(coarser(w.x, ratio), coarser(w.y, ratio), coarser(w.z, ratio), coarser(w.w, ratio));
      }
    if (t == 0) c.scale[ph * 2 + values] = bad ? __int_as_float(0x7fc00000) : power2(e);
  }
}
template <int C>
__global__ void __maxnreg__(64) cache_append_kernel(const bf16* __restrict__ k, const bf16* __restrict__ v, long ldk, long ldv, CachePages c, CacheStep s,
                                                    int window) {
  append_window<C, kAsIs>(k, v, ldk, ldv, c, s, blockIdx.x, window, Turning{}, blockIdx.y, blockIdx.z);
}
template <int C, int MODE>
__global__ void __maxnreg__(64) cache_append_rope_kernel(const bf16* __restrict__ k, const bf16* __restrict__ v, long ldk, long ldv, CachePages c, CacheStep s,
                                                         int window, int jobs, Queries q, Turning turning) {
  const int at = blockIdx.x / jobs, job = blockIdx.x - at * jobs;
  if (job >= 2 * c.H) {
    const int h0 = (job - 2 * c.H) * kQueryHeads, i0 = at * window;
    const int h1 = min(h0 + kQueryHeads, q.H), i1 = min(i0 + window, s.N);
    if (turning.R % 16 == 0) turn_queries<MODE, 8>(q.q, q.ld, q.y, turning, s, q.H, h0, h1, c.D, i0, i1);
    else turn_queries<MODE, 4>(q.q, q.ld, q.y, turning, s, q.H, h0, h1, c.D, i0, i1);
    return;
  }
  append_window<C, MODE>(k, v, ldk, ldv, c, s, at, window, turning, job < c.H ? job : job - c.H, job >= c.H);
}

// One CTA per page, head and side: bf16 values (n, P, H, D).  Keys 8 codes of a token at a time, four such loads before the first store; values 16 tokens of
// C columns, so that a warp's stores are whole rows.  Bytes bound it: the same 34.7 K tokens (52 MB of the codes from memory, the rest from L2, 144 MB written)
// 37 us, 39 in one CTA for both sides with keys by 16 and codes converted as whole numbers.  Its results leave the caches first: appending and reading back
// 89.5 -> 82.2 us.
__device__ __forceinline__ float number_of(uint32_t w, int i, float s) {   // (code i of a word - 128) s, s a power of two: 2^23 + u by its bits
  return fmaf(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + i)), s, -8388736.f * s);
}
__device__ __forceinline__ uint32_t two_of(float a, float b) {
  const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <int C>
__global__ void __launch_bounds__(128) cache_values_kernel(CachePages c, const int* __restrict__ ids, bf16* __restrict__ k, bf16* __restrict__ v) {
  const int h = blockIdx.y, P = 1 << c.shift, D = c.D, page = ids[blockIdx.x], t = threadIdx.x, lane = t & 31;
  const bool there = page >= 0 && page < c.pages;
  const long ph = static_cast<long>(there ? page : 0) * c.H + h, row = static_cast<long>(c.H) * D, out = static_cast<long>(blockIdx.x) * P * row + h * D;
  const float s = there ? c.scale[ph * 2 + blockIdx.z] : 0.f;
  if (blockIdx.z == 0) {
    const uint8_t* codes = c.k + ph * P * D;
    for (int y0 = t * 8; y0 < P * D; y0 += 4 * 128 * 8) {
      uint2 w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int y = y0 + j * 128 * 8;
        w[j] = there && y < P * D ? __ldg(reinterpret_cast<const uint2*>(codes + y)) : make_uint2(0x80808080u, 0x80808080u);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int y = y0 + j * 128 * 8, two = over(y, 2 * D), token = two * 2 + (y >> 6 & 1), d = (y - two * 2 * D >> 7) * 64 + (y & 63);
        if (y >= P * D) break;
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t u = i < 2 ? w[j].x : w[j].y;
          o[i] = two_of(number_of(u, 2 * (i & 1), s), number_of(u, 2 * (i & 1) + 1, s));
        }
        __stcs(reinterpret_cast<uint4*>(k + out + token * row + d), make_uint4(o[0], o[1], o[2], o[3]));
      }
    }
    return;
  }
  const uint8_t* codes = c.v + ph * P * D;
  const int slabs = D / (32 * C);
  for (int y = t >> 5; y < P / 16 * slabs; y += 4) {
    const int yt = over(y, slabs), t0 = yt * 16, d = (y - yt * slabs) * 32 * C + lane * C;
    uint32_t w[C][4];
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const uint4 u = there ? __ldg(reinterpret_cast<const uint4*>(codes + value_at(t0, d + i, D))) : make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
      w[i][0] = u.x;
      w[i][1] = u.y;
      w[i][2] = u.z;
      w[i][3] = u.w;
    }
#pragma unroll
    for (int tok = 0; tok < 16; ++tok) {
      bf16* to = v + out + (t0 + tok) * row + d;
      const uint32_t a = two_of(number_of(w[0][tok >> 2], tok & 3, s), number_of(w[1][tok >> 2], tok & 3, s));
      if (C == 4) __stcs(reinterpret_cast<uint2*>(to), make_uint2(a, two_of(number_of(w[C - 2][tok >> 2], tok & 3, s), number_of(w[C - 1][tok >> 2], tok & 3, s))));
      else *reinterpret_cast<uint32_t*>(to) = a;
    }
  }
}
}  // namespace

extern "C" int nsa_cache_plan(const int* lengths, const int* add, int* table, const int* free_pages, const int* free_count, int F, int* query_start,
                              int* total, long long* slots, long long* positions, int* free_left, int* shortfall, int B, int W, int N,
                              int page_size, cudaStream_t st) {
  if (B <= 0 || W <= 0 || N < 0 || F < 0) return nsa::fail(NSA_ERR_SHAPE, "cache_plan: empty problem");
  if (B > nsa_cache_plan_limit()) return nsa::fail(NSA_ERR_LIMIT, "cache_plan: more requests than shared memory holds");
  const int bytes = 3 * (B + 1) * 4;
  if (bytes > 40000) {
    const cudaError_t e = cudaFuncSetAttribute(cache_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200000);
    if (e != cudaSuccess) return nsa::fail_cuda(e, "nsa_cache_plan");
  }
  // as many threads as requests, up to 1024: fewer scan in turns, more wait for one another.  One token each, with 128 / 512 / 1024 threads: 64 requests 3.3 / 3.5 /
  // 4.1 us, 256 4.5 / 3.8 / 4.4, 512 6.6 / 4.1 / 4.7, 4096 34.7 / 12.9 / 11.1 (65536 tokens of 64 requests, which write more than they scan: 5.8 / 4.4 / 5.5)
  const int threads = B <= 128 ? 128 : B <= 512 ? 512 : kPlanThreads;
  const int want = (N + threads - 1) / threads, most = nsa::sm_count();
  const int grid = want < 1 ? 1 : want < most ? want : most;
  cache_plan_kernel<<<grid, threads, bytes, st>>>(lengths, add, table, free_pages, free_count, F, query_start, total, slots, positions, free_left,
                                                       shortfall, B, W, N, __builtin_ctz(page_size));
  nsa::count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : nsa::fail_cuda(e, "nsa_cache_plan launch");
}
extern "C" int nsa_cache_plan_limit(void) { return 16384; }

extern "C" int nsa_cache_release(const void* finished, const int* lengths, int* table, int* free_pages, const int* free_count, int F, int* total,
                                 int* free_left, int B, int W, int page_size, cudaStream_t st) {
  if (B <= 0 || W <= 0 || F < 0) return nsa::fail(NSA_ERR_SHAPE, "cache_release: empty problem");
  cache_release_kernel<<<1, kPlanThreads, 0, st>>>(static_cast<const uint8_t*>(finished), lengths, table, free_pages, free_count, F, total, free_left, B,
                                                   W, __builtin_ctz(page_size));
  nsa::count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : nsa::fail_cuda(e, "nsa_cache_release launch");
}

static void append_shape(int N, int B, int D, int page_size, int& window, int& warps) {
  // Up to 2048 tokens: one a CTA, which passes over all but a group's first; else a page's worth, since for long groups those CTAs cost more than they do, while
  // a window of single tokens takes them one after another.  Pages of 64, 8 heads of 128, a token / a page's worth a CTA: 64 requests of one token 7.5 / 263 us, 512
  // 18.6 / 289, 2048 62.8 / 351, 64 requests of 8 13.6 / 35; 4 of 512 23.3 / 9.4, 4 of 1024 40 / 10.5, 8 of 4096 277 / 41.  More than 2048 single tokens are on the
  // wrong side of it (4096 122 / 360).  Warps for the 16-token blocks of a page; one where a group can have only one (512 requests 18.6
  // us, with as many as the page has blocks 34)
  window = N <= 2048 ? 1 : page_size;
  const int blocks = page_size / 16 * (D / (D % 128 ? 64 : 128));
  warps = window == 1 && N <= B ? 1 : blocks < 16 ? blocks : 16;
}
extern "C" int nsa_cache_append(const void* k, const void* v, long ldk, long ldv, void* kc, void* vc, float* scale, const int* table,
                                const int* query_start, const int* lengths, int B, int W, int N, int pages, int H, int D, int page_size,
                                cudaStream_t st) {
  if (N == 0) return 0;
  if (B <= 0 || H <= 0 || H > 65535 || D % 64 || N < 0) return nsa::fail(NSA_ERR_SHAPE, "cache_append: unsupported shape");
  const CachePages c{static_cast<uint8_t*>(kc), static_cast<uint8_t*>(vc), scale, pages, H, D, __builtin_ctz(page_size)};
  const CacheStep s{table, query_start, lengths, B, W, N};
  int window, warps;
  append_shape(N, B, D, page_size, window, warps);
  const int C = D % 128 ? 2 : 4;
  const dim3 grid((N + window - 1) / window, H, 2);
  if (C == 4)
    cache_append_kernel<4><<<grid, 32 * warps, 0, st>>>(static_cast<const bf16*>(k), static_cast<const bf16*>(v), ldk, ldv, c, s, window);
  else
    cache_append_kernel<2><<<grid, 32 * warps, 0, st>>>(static_cast<const bf16*>(k), static_cast<const bf16*>(v), ldk, ldv, c, s, window);
  nsa::count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : nsa::fail_cuda(e, "nsa_cache_append launch");
}

// cos, sin (L, R/2) fp32, R a multiple of 8 up to 128 columns (64 where D is no multiple of 128); q (N, Hq, D) of pitch ldq, yq dense
extern "C" int nsa_cache_append_rope(const void* q, long ldq, void* yq, int Hq, const void* k, const void* v, long ldk, long ldv, void* kc, void* vc,
                                     float* scale, const float* cos_t, const float* sin_t, int L, int R, int paired, const int* table, const int* query_start,
                                     const int* lengths, int B, int W, int N, int pages, int H, int D, int page_size, cudaStream_t st) {
  if (N == 0) return 0;
  if (B <= 0 || H <= 0 || Hq <= 0 || H > 16384 || Hq > 65536 || D % 64 || N < 0) return nsa::fail(NSA_ERR_SHAPE, "cache_append_rope: unsupported shape");
  if (R <= 0 || R % 8 || R > D || R > (D % 128 ? 64 : 128)) return nsa::fail(NSA_ERR_SHAPE, "cache_append_rope: columns to be turned");
  const CachePages c{static_cast<uint8_t*>(kc), static_cast<uint8_t*>(vc), scale, pages, H, D, __builtin_ctz(page_size)};
  const CacheStep s{table, query_start, lengths, B, W, N};
  int window, warps;
  append_shape(N, B, D, page_size, window, warps);
  const int jobs = 2 * H + (Hq + kQueryHeads - 1) / kQueryHeads;
  const long grid = static_cast<long>((N + window - 1) / window) * jobs;
  if (grid > 0x7fffffffl) return nsa::fail(NSA_ERR_SHAPE, "cache_append_rope: too many tokens and heads");
  const Queries qs{static_cast<const bf16*>(q), ldq, static_cast<bf16*>(yq), Hq};
  auto* kernel = D % 128 ? (paired ? cache_append_rope_kernel<2, kPairs> : cache_append_rope_kernel<2, kHalves>)
                         : (paired ? cache_append_rope_kernel<4, kPairs> : cache_append_rope_kernel<4, kHalves>);
  kernel<<<static_cast<unsigned>(grid), 32 * warps, 0, st>>>(static_cast<const bf16*>(k), static_cast<const bf16*>(v), ldk, ldv, c, s, window, jobs, qs, Turning{cos_t, sin_t, L, R});
  nsa::count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : nsa::fail_cuda(e, "nsa_cache_append_rope launch");
}

extern "C" int nsa_cache_values(const void* kc, const void* vc, const float* scale, const int* ids, void* k, void* v, int n, int pages, int H, int D,
                                int page_size, cudaStream_t st) {
  if (n == 0) return 0;
  if (H <= 0 || H > 65535 || D % 64 || n < 0) return nsa::fail(NSA_ERR_SHAPE, "cache_values: unsupported shape");
  const CachePages c{static_cast<uint8_t*>(const_cast<void*>(kc)), static_cast<uint8_t*>(const_cast<void*>(vc)), const_cast<float*>(scale), pages, H, D,
                     __builtin_ctz(page_size)};
  if (D % 128)
    cache_values_kernel<2><<<dim3(n, H, 2), 128, 0, st>>>(c, ids, static_cast<bf16*>(k), static_cast<bf16*>(v));
  else
    cache_values_kernel<4><<<dim3(n, H, 2), 128, 0, st>>>(c, ids, static_cast<bf16*>(k), static_cast<bf16*>(v));
  nsa::count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : nsa::fail_cuda(e, "nsa_cache_values launch");
}
