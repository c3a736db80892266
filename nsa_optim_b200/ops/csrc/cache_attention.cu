// Attention of a step's queries over the paged 8-bit key / value cache.
//
// o = sum_j 2^(x_j - M) v_j / sum_j 2^(x_j - M), x_j = log2(e) scale q k_j, in one pass with a running M.  Rows are (query token, head of the KV head's
// group) pairs, 16 to a warp's matrix product (m16n8k16 on f16), so a group shares what it reads.  With few rows the bytes of the codes bound it;
// every other choice serves that:
//  * Work is counted in units of 64 keys, over all requests, KV heads and row tiles, and dealt out evenly to workers (a warp with 16 rows, more
//    warps on the same keys where a request has more rows): ragged requests cost no more than even ones.  A worker's range may end inside a request;
//    such parts meet in shared memory at the CTA's end, and across CTAs in cache_attn_join_kernel.
//  * Each worker has its own ring of key and value tiles that bulk copies fill two tiles ahead: 130 KB in flight per SM, no registers, and no
//    synchronisation between workers.
//  * The cache's orders are those of the product's operands.  Of a unit, lane 4c+r of a warp scores token 2j + c%2 of sub-block c/2 in tile j and holds
//    the probabilities of sub-block r's tokens 2j, 2j+1, so its value operand is 16 neighbouring bytes; a code becomes f16 by a byte permutation and one subtraction.
//  * f16 holds a code exactly, and a query row scaled by a power of two to 2^13 .. 2^14 (bf16's 8 bits; what is 2^-28 of the row's largest
//    value rounds).  Probabilities are rounded to 11 bits, relative to the row's largest product of probability and value scale: the value scale's
//    exponent is added to x, and taken out again of the sum.  Sums are fp32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "cache.cuh"
#include "host.cuh"
#include "tc5.cuh"

namespace {
typedef __nv_bfloat16 bf16;
constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kMaxRequests = 1024;                       // of one launch: their prefix sums are in shared memory

struct AttnParams {
  const bf16* q;
  long ldq;
  CachePages c;
  CacheStep s;
  bf16* o;
  float* head;          // (CTA, worker, rows, D): parts of requests that end inside a worker's range and began before it
  float* part;          // (CTA, 2, rows, D): parts of requests that go beyond a CTA: one that began before it, one that goes on behind it
  float2* part_ml;      // (CTA, 2, rows)
  int4* join;           // (CTA): request, KV head and first row that begin in the CTA and end in CTA .w; .w = 0: none
  int Hq, G, window;
  float scale;          // times log2(e)
  KernelStatus* status;
};

template <int D, int MT>
struct Shape {
  static constexpr int kRows = 16 * MT, kGroups = kWarps / MT;         // rows and workers of a CTA
  static constexpr int kSub = 16 * D, kPitch = kSub + 32;              // a sub-block of 16 tokens; the pitch spreads four of them over the banks
  static constexpr int kSlot = 4 * kPitch;                             // a unit's keys or values
  static constexpr int kSlots = 24 * (128 / D) / kGroups;              // of a worker
  static constexpr int kRing = kSlots * kSlot;
  static_assert(kRing >= kRows * D * 4, "a worker's sums go where its ring was");
};

// What a worker has left in memory at the end
struct Left {
  int head, tail;       // whether there is a part that began before the range and ended in it; whether the last part is open at either end
  int began, open;      // of the last part: began before the range; goes on behind it
  int head_item[3], tail_item[3];                                      // request, KV head, first row
  int tail_last;        // the CTA in which the last part's item ends
  int some;             // the range is not empty
};

template <int D, int MT>
struct Smem {
  using S = Shape<D, MT>;
  alignas(128) uint8_t ring[S::kGroups][S::kRing];
  float2 scale[S::kGroups][S::kSlots][4];
  uint64_t full[S::kGroups][S::kSlots], empty[S::kGroups][S::kSlots];
  float2 ml[S::kGroups][2][S::kRows];
  Left left[S::kGroups];
  long long before[kMaxRequests + 1];                                  // units of the requests before b
  long long warps[kWarps];
  int abort_flag;
};

// ------------------------------------------------------------------------------------- work
struct Request {
  int n, q0;            // queries, the first one's row in q
  int past, cap;        // tokens before them, keys that the table can hold
  int unit0, units;     // 64-key units that any of them sees
};
__device__ __forceinline__ Request request_of(const AttnParams& p, int b) {
  Request r;
  const int lo = p.s.query_start[b], hi = p.s.query_start[b + 1], len = p.s.lengths[b];
  r.q0 = min(max(lo, 0), p.s.N);
  r.n = max(min(hi, p.s.N) - r.q0, 0);
  r.past = len - (hi - lo);
  r.cap = static_cast<int>(min(static_cast<long long>(max(len, 0)), static_cast<long long>(p.s.W) << p.c.shift));
  r.unit0 = p.window > 0 ? max(r.past - p.window + 1, 0) >> 6 : 0;
  r.units = r.n > 0 ? max(((r.cap + 63) >> 6) - r.unit0, 1) : 0;
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
  long long at, end;
  int b;
  Piece p;

  // The next piece of the range; false at its end
  __device__ __forceinline__ bool next_piece(const AttnParams& a, const long long* before) {
    if (at >= end) return false;
    while (before[b + 1] <= at) ++b;
    const Request r = request_of(a, b);
    const int tiles = (r.n * a.G + ROWS - 1) / ROWS;
    const long long rel = at - before[b], item = rel / r.units;
    const int h = static_cast<int>(item / tiles), tile = static_cast<int>(item - static_cast<long long>(h) * tiles);
    const int first = static_cast<int>(rel - item * r.units);
    const long long item_at = before[b] + item * r.units, stop = min(item_at + r.units, end);
    p.b = b;
    p.h = h;
    p.row0 = tile * ROWS;
    p.n = r.n;
    p.q0 = r.q0;
    p.past = r.past;
    p.cap = r.cap;
    p.began = first > 0;
    p.open = stop < item_at + r.units;
    p.item_end = item_at + r.units;
    // units that some row of the tile sees
    const int t0 = p.row0 / a.G, t1 = min((p.row0 + ROWS - 1) / a.G, r.n - 1);
    const int from = a.window > 0 ? max(r.past + t0 - a.window + 1, 0) >> 6 : 0;
    const int to = min(r.past + t1 >= 0 ? ((r.past + t1) >> 6) + 1 : 0, (r.cap + 63) >> 6);
    p.lo = max(r.unit0 + first, from);
    p.hi = min(r.unit0 + static_cast<int>(stop - item_at), to);
    at = stop;
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
// Four codes as f16 numbers: 0x6400 + u is 1024 + u, less 1152
__device__ __forceinline__ void decode(uint32_t w, uint32_t& b0, uint32_t& b1) {
  const uint32_t lo = __byte_perm(w, 0x64646464u, 0x4140), hi = __byte_perm(w, 0x64646464u, 0x4342), off = 0x64806480u;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(b0) : "r"(lo), "r"(off));
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(b1) : "r"(hi), "r"(off));
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 1);
  return x + __shfl_xor_sync(0xffffffffu, x, 2);
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
               "r"(tc5::smem_u32(bar))
               : "memory");
}
// Exponent of a power of two (NaN for NaN)
__device__ __forceinline__ float log2_of_scale(float s) {
  const int e = static_cast<int>(__float_as_uint(s) >> 23) - 127;
  return e > 60 ? CUDART_NAN_F : static_cast<float>(e);
}

// A warp's 16 rows: queries as f16 operands, running maximum, sum, output
template <int D>
struct Rows {
  uint32_t q[D / 16][4];
  float factor[2];      // of lane rows r and r + 8: takes a product of f16 queries and codes to x / key scale
  int pos[2];           // their positions; -1: no row
  float m[2], l[2];
  float o[D / 8][4];

  __device__ __forceinline__ void clear() {
    m[0] = m[1] = -CUDART_INF_F;
    l[0] = l[1] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  }

  // Row r of the item is query token r / G, head r % G of the group
  __device__ __forceinline__ void load(const AttnParams& p, const Piece& it, int row0) {
    const int lane = threadIdx.x & 31, r = lane & 3;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = row0 + (lane >> 2) + 8 * i, t = row / p.G;
      const bool there = t < it.n;
      pos[i] = there ? it.past + t : -1;
      uint4 raw[D / 64][2];
      unsigned top = 0;
      const bf16* src = p.q + static_cast<long>(it.q0 + t) * p.ldq + static_cast<long>(it.h * p.G + row - t * p.G) * D + r * 16;
#pragma unroll
      for (int h = 0; h < D / 64; ++h)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          raw[h][k] = there ? *reinterpret_cast<const uint4*>(src + h * 64 + k * 8) : make_uint4(0, 0, 0, 0);
          const uint32_t w[4] = {raw[h][k].x, raw[h][k].y, raw[h][k].z, raw[h][k].w};
#pragma unroll
          for (int y = 0; y < 4; ++y) top = max(top, max(w[y] & 0x7fffu, (w[y] >> 16) & 0x7fffu));
        }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = static_cast<int>(top >> 7);                        // the largest magnitude is 2^(e - 127) at least
      const int up = min(140 - e, 126);
      const float f = __int_as_float((up + 127) << 23);
      factor[i] = e == 255 ? CUDART_NAN_F : __int_as_float((127 - up) << 23) * p.scale;
#pragma unroll
      for (int h = 0; h < D / 64; ++h)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t w[4] = {raw[h][k].x, raw[h][k].y, raw[h][k].z, raw[h][k].w};
#pragma unroll
          for (int y = 0; y < 4; ++y) {                                // columns 16 r + 8 k + 2 y, + 1 of this half
            const uint32_t v = pack_half(__int_as_float(w[y] << 16) * f, __int_as_float(w[y] & 0xffff0000u) * f);
            q[h * 4 + k * 2 + (y >> 1)][i + 2 * (y & 1)] = v;
          }
        }
    }
  }
};

// Scores of one unit (codes' products): s[j] are tile j's
template <int D, class S>
__device__ __forceinline__ void scores(const Rows<D>& w, const uint8_t* keys, float (&s)[8][4]) {
  const int lane = threadIdx.x & 31, c = lane >> 2, r = lane & 3;
  const uint8_t* base = keys + (c >> 1) * S::kPitch + (c & 1) * 64 + r * 16;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
    for (int h = 0; h < D / 64; ++h) {
      const uint4 k = *reinterpret_cast<const uint4*>(base + (j * (D / 64) + h) * 128);
      const uint32_t words[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        uint32_t b0, b1;
        decode(words[y], b0, b1);
        mma(s[j], w.q[h * 4 + y], b0, b1);
      }
    }
  }
}

// Scores to probabilities, in f16 pairs, with the running maximum and sum.  MASKED: some key of the unit is not seen by some row.
template <int D, bool MASKED>
__device__ __forceinline__ void softmax(Rows<D>& w, float (&s)[8][4], uint32_t (&pr)[8][2], float2 scale, int key0, int window) {
  const bool there = scale.x >= 0.f || scale.x != scale.x;             // a sub-block without a page has -1
  const float ev = there ? log2_of_scale(scale.y) : 0.f;
  const float a[2] = {there ? w.factor[0] * scale.x : 0.f, there ? w.factor[1] * scale.x : 0.f};
  float top[2] = {-CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x = fmaf(s[j][i], a[i >> 1], ev);
      if (MASKED) {
        const int key = key0 + 2 * j + (i & 1), pos = w.pos[i >> 1];
        if (!there || key > pos || (window > 0 && key <= pos - window)) x = -CUDART_INF_F;
      }
      s[j][i] = x;
      top[i >> 1] = fmaxf(top[i >> 1], x);
    }
  float ref[2];
  bool moved = false;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float m = fmaxf(w.m[i], quad_max(top[i]));
    moved |= m != w.m[i];
    ref[i] = m == -CUDART_INF_F ? 0.f : m;
    top[i] = m;
  }
  if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float f = ex2(w.m[i] - ref[i]);
      w.m[i] = top[i];
      w.l[i] *= f;
#pragma unroll
      for (int d = 0; d < D / 8; ++d) {
        w.o[d][2 * i] *= f;
        w.o[d][2 * i + 1] *= f;
      }
    }
  }
  float sum[2] = {0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[j][i] = ex2(s[j][i] - ref[i >> 1]);
      sum[i >> 1] += s[j][i];
    }
    pr[j][0] = pack_half(s[j][0], s[j][1]);
    pr[j][1] = pack_half(s[j][2], s[j][3]);
  }
  const float out = ex2(-ev);                                          // NaN in a page of which a row sees nothing
  w.l[0] += sum[0] == 0.f ? 0.f : sum[0] * out;
  w.l[1] += sum[1] == 0.f ? 0.f : sum[1] * out;
}

template <int D, class S>
__device__ __forceinline__ void accumulate(Rows<D>& w, const uint8_t* values, const uint32_t (&pr)[8][2]) {
  const int lane = threadIdx.x & 31;
  const uint8_t* base = values + (lane & 3) * S::kPitch + (lane >> 2) * 16;
#pragma unroll
  for (int d = 0; d < D / 8; ++d) {
    const uint4 v = *reinterpret_cast<const uint4*>(base + d * 128);
    const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      uint32_t b0, b1;
      decode(words[y], b0, b1);
      const uint32_t a[4] = {pr[2 * y][0], pr[2 * y][1], pr[2 * y + 1][0], pr[2 * y + 1][1]};
      mma(w.o[d], a, b0, b1);
    }
  }
}

// Where row r of an item goes; nullptr: there is no such row
__device__ __forceinline__ bf16* row_of(const AttnParams& p, int n, int q0, int h, int row, int D) {
  const int t = row / p.G;
  return t < n ? p.o + (static_cast<long>(q0 + t) * p.Hq + h * p.G + row - t * p.G) * D : nullptr;
}
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }

template <int D, int MT>
__global__ void __launch_bounds__(kThreads, 1) cache_attn_kernel(const __grid_constant__ AttnParams p) {
  using S = Shape<D, MT>;
  extern __shared__ __align__(128) uint8_t raw_smem[];
  Smem<D, MT>& sm = *reinterpret_cast<Smem<D, MT>*>(raw_smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tc5::warp_index(), grp = warp / MT, mt = warp % MT, B = p.s.B;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- the units of all requests
  if (tid == 0) sm.abort_flag = 0;
  for (int i = tid; i < S::kGroups * S::kSlots; i += kThreads) {
    tc5::mbar_init(&sm.full[0][0] + i, 5);
    tc5::mbar_init(&sm.empty[0][0] + i, MT);
  }
  tc5::fence_barrier_init();
  long long total = 0;
  for (int base = 0; base < B; base += kThreads) {
    const int b = base + tid;
    long long x = 0;
    if (b < B) {
      const Request r = request_of(p, b);
      x = static_cast<long long>(r.units) * p.c.H * ((r.n * p.G + S::kRows - 1) / S::kRows);
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
  const long long workers = static_cast<long long>(gridDim.x) * S::kGroups, each = max((total + workers - 1) / workers, 1ll);
  Cursor<S::kRows> use, get;
  use.at = min((static_cast<long long>(blockIdx.x) * S::kGroups + grp) * each, total);
  use.end = min(use.at + each, total);
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sm.before[mid] <= use.at) lo = mid; else hi = mid;
  }
  use.b = lo;
  get = use;

  // ---- the producer's side: tile t of the range is the keys (even) or values (odd) of its unit t / 2
  uint8_t* ring = sm.ring[grp];
  int get_unit = 0, get_stop = 0;                                      // of the piece that `get` is in
  int page = -1, page_next = -1, blk = 0, blk_next = 0, head = 0, head_next = 0;
  bool have = false, have_next = false;
  // Looks up the pages of the unit after the next: one sub-block per lane, four of them
  auto look = [&]() {
    page = page_next;
    blk = blk_next;
    head = head_next;
    have = have_next;
    have_next = false;
    while (get_unit >= get_stop) {
      if (!get.next_piece(p, sm.before)) return;
      get_unit = get.p.lo;
      get_stop = get.p.hi;
    }
    have_next = true;
    blk_next = get_unit * 4 + (lane & 3);
    head_next = get.p.h;
    page_next = blk_next * 16 < get.p.cap ? page_of(p.s, p.c, get.p.b, static_cast<long>(blk_next) * 16) : -1;
    ++get_unit;
  };
  uint32_t issued = 0;
  auto issue = [&](bool& ok) {                                         // the next tile, if there is one
    const bool values = issued & 1;
    if (!values) look();
    if (!have) return;
    const uint32_t slot = issued % S::kSlots, round = issued / S::kSlots;
    if (MT > 1 && round > 0)
      ok = ok && tc5::mbar_wait_warp(&sm.empty[grp][slot], (round - 1) & 1, &sm.abort_flag, p.status, STATUS_TIMEOUT_SMEM_EMPTY);
    if (!ok) return;
    ++issued;
    uint64_t* bar = &sm.full[grp][slot];
    const bool there = page >= 0;
    const unsigned mask = __ballot_sync(0xffffffffu, there) & 0xf;
    const long ph = static_cast<long>(there ? page : 0) * p.c.H + head;
    if (lane < 4) {
      if (there) {
        const long off = ((ph << (p.c.shift - 4)) + (blk & ((1 << (p.c.shift - 4)) - 1))) * S::kSub;
        bulk_load(tc5::smem_u32(ring + slot * S::kSlot + lane * S::kPitch), (values ? p.c.v : p.c.k) + off, S::kSub, bar);
      }
      if (!values && there) {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(tc5::smem_u32(&sm.scale[grp][slot][lane])), "l"(p.c.scale + ph * 2) : "memory");
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(tc5::smem_u32(bar)) : "memory");
      } else {
        if (!values) sm.scale[grp][slot][lane] = make_float2(-1.f, 1.f);
        tc5::mbar_arrive(bar);
      }
      if (lane == 0) tc5::mbar_expect_tx(bar, __popc(mask) * S::kSub);
    }
  };
  bool ok = true;
  if (mt == 0) {
    look();                                                            // the first unit's pages are the "next" ones now
    for (int i = 0; i < S::kSlots; ++i) issue(ok);
  }

  // ---- the consumer's side
  Rows<D> w;
  uint32_t tile = 0;
  Left left{};
  left.some = use.at < use.end;
  float* ring_f = reinterpret_cast<float*>(ring);
  while (ok && use.next_piece(p, sm.before)) {
    const Piece& it = use.p;
    const int row0 = it.row0 + mt * 16;
    w.load(p, it, row0);
    w.clear();
    // positions of the warp's first and last row
    const int rows = it.n * p.G, p0 = row0 < rows ? it.past + row0 / p.G : -1, p1 = row0 < rows ? it.past + min(row0 + 15, rows - 1) / p.G : -1;
    for (int u = it.lo; u < it.hi && ok; ++u) {
      const int key0 = u * 64;
      const bool seen = key0 <= p1 && (p.window == 0 || key0 + 63 > p0 - p.window);
      uint32_t slot = tile % S::kSlots;
      ok = tc5::mbar_wait_warp(&sm.full[grp][slot], (tile / S::kSlots) & 1, &sm.abort_flag, p.status, STATUS_TIMEOUT_SMEM_FULL);
      if (!ok) break;
      uint32_t pr[8][2];
      if (seen) {
        const float2 scale = sm.scale[grp][slot][lane & 3];
        float s[8][4];
        scores<D, S>(w, ring + slot * S::kSlot, s);
        const bool whole = key0 + 63 <= p0 && (p.window == 0 || key0 > p1 - p.window) && row0 + 15 < rows;
        if (whole && !__any_sync(0xffffffffu, scale.x == -1.f))
          softmax<D, false>(w, s, pr, scale, 0, 0);
        else
          softmax<D, true>(w, s, pr, scale, key0 + 16 * (lane & 3), p.window);
      }
      __syncwarp();
      if (MT > 1 && lane == 0) tc5::mbar_arrive(&sm.empty[grp][slot]);
      ++tile;
      if (mt == 0) issue(ok);
      slot = tile % S::kSlots;
      ok = ok && tc5::mbar_wait_warp(&sm.full[grp][slot], (tile / S::kSlots) & 1, &sm.abort_flag, p.status, STATUS_TIMEOUT_SMEM_FULL);
      if (!ok) break;
      if (seen) accumulate<D, S>(w, ring + slot * S::kSlot, pr);
      __syncwarp();
      if (MT > 1 && lane == 0) tc5::mbar_arrive(&sm.empty[grp][slot]);
      ++tile;
      if (mt == 0) issue(ok);
    }
    if (!ok) break;
    w.l[0] = quad_sum(w.l[0]);
    w.l[1] = quad_sum(w.l[1]);
    const int r = lane >> 2, col = (lane & 3) * 2;
    if (!it.began && !it.open) {                                       // the whole item: its rows are done
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        bf16* out = row_of(p, it.n, it.q0, it.h, row0 + r + 8 * i, D);
        if (out) {
          const float f = inverse(w.l[i]);
#pragma unroll
          for (int d = 0; d < D / 8; ++d)
            *reinterpret_cast<__nv_bfloat162*>(out + d * 8 + col) = __floats2bfloat162_rn(w.o[d][2 * i] * f, w.o[d][2 * i + 1] * f);
        }
      }
    } else {
      const bool is_head = it.began && !it.open && use.at < use.end;   // more pieces follow
      float* dst = is_head ? p.head + (static_cast<long>(blockIdx.x) * S::kGroups + grp) * S::kRows * D : ring_f;
      int* item = is_head ? left.head_item : left.tail_item;
      item[0] = it.b;
      item[1] = it.h;
      item[2] = it.row0;
      if (is_head) {
        left.head = 1;
      } else {
        left.tail = 1;
        left.began = it.began;
        left.open = it.open;
        left.tail_last = static_cast<int>(((it.item_end - 1) / each) / S::kGroups);
        // the sums go where the ring is: every warp of the worker has let go of its last tiles
        if (MT > 1)
          for (uint32_t t = tile > S::kSlots ? tile - S::kSlots : 0; t < tile; ++t)
            ok = ok && tc5::mbar_wait_warp(&sm.empty[grp][t % S::kSlots], (t / S::kSlots) & 1, &sm.abort_flag, p.status, STATUS_TIMEOUT_SMEM_EMPTY);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = mt * 16 + r + 8 * i;
        if ((lane & 3) == 0) sm.ml[grp][is_head ? 0 : 1][row] = make_float2(w.m[i], w.l[i]);
#pragma unroll
        for (int d = 0; d < D / 8; ++d)
          *reinterpret_cast<float2*>(dst + row * D + d * 8 + col) = make_float2(w.o[d][2 * i], w.o[d][2 * i + 1]);
      }
    }
  }
  if (!ok && mt == 0)
    for (int i = 0; i < S::kSlots; ++i) tc5::mbar_drain(&sm.full[grp][i]);
  if (mt == 0 && lane == 0) sm.left[grp] = left;
  __syncthreads();
  if (sm.abort_flag) {
    if (tid == 0) p.join[blockIdx.x] = make_int4(0, 0, 0, 0);
    return;
  }

  // ---- parts of one item in several workers meet; those of an item that goes beyond the CTA are left for the join
  int4 join = make_int4(0, 0, 0, 0);
  for (int g0 = 0; g0 < S::kGroups; ++g0)
    for (int side = 0; side < 2; ++side) {                             // a chain begins with the first worker's head, or with a last part
      const Left& a = sm.left[g0];
      const bool begins = side == 0 ? g0 == 0 && a.head : a.tail && (g0 == 0 || !a.began);
      if (!begins) continue;
      const int* item = side == 0 ? a.head_item : a.tail_item;
      const bool began = side == 0 || a.began;
      int g1 = g0;
      bool open = side == 1 && a.open;
      unsigned heads = side == 0 ? 1u << g0 : 0u;                      // which workers' contributions are heads
      while (open && g1 + 1 < S::kGroups && sm.left[g1 + 1].some) {
        const Left& c = sm.left[++g1];
        if (c.head) heads |= 1u << g1;
        open = !c.head && c.open;
      }
      const Request rq = request_of(p, item[0]);
      const bool done = !began && !open;
      for (int e = tid; e < S::kRows * (D / 4); e += kThreads) {
        const int row = e / (D / 4), d = (e % (D / 4)) * 4;
        float m = -CUDART_INF_F;
        for (int g = g0; g <= g1; ++g) m = fmaxf(m, sm.ml[g][heads >> g & 1 ? 0 : 1][row].x);
        const float ref = m == -CUDART_INF_F ? 0.f : m;
        float l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int g = g0; g <= g1; ++g) {
          const bool is_head = heads >> g & 1;
          const float2 ml = sm.ml[g][is_head ? 0 : 1][row];
          const float* src = is_head ? p.head + (static_cast<long>(blockIdx.x) * S::kGroups + g) * S::kRows * D : reinterpret_cast<float*>(sm.ring[g]);
          const float4 x = *reinterpret_cast<const float4*>(src + row * D + d);
          const float f = ex2(ml.x - ref);
          l = fmaf(ml.y, f, l);
          o.x = fmaf(x.x, f, o.x);
          o.y = fmaf(x.y, f, o.y);
          o.z = fmaf(x.z, f, o.z);
          o.w = fmaf(x.w, f, o.w);
        }
        if (done) {
          bf16* out = row_of(p, rq.n, rq.q0, item[1], item[2] + row, D);
          if (out) {
            const float f = inverse(l);
            __nv_bfloat162 y[2] = {__floats2bfloat162_rn(o.x * f, o.y * f), __floats2bfloat162_rn(o.z * f, o.w * f)};
            *reinterpret_cast<uint2*>(out + d) = *reinterpret_cast<uint2*>(y);
          }
        } else {
          const long slot = static_cast<long>(blockIdx.x) * 2 + (began ? 0 : 1);
          *reinterpret_cast<float4*>(p.part + (slot * S::kRows + row) * D + d) = o;
          if (d == 0) p.part_ml[slot * S::kRows + row] = make_float2(m, l);
        }
      }
      if (!began && open) join = make_int4(item[0], item[1], item[2], sm.left[g0].tail_last);
    }
  if (tid == 0) p.join[blockIdx.x] = join;
}

// Parts of items that several CTAs worked on: CTA (c, part) takes some rows of the item that begins in CTA c of the kernel before.
constexpr int kJoinParts = 4;
template <int D, int MT>
__global__ void __launch_bounds__(128) cache_attn_join_kernel(const __grid_constant__ AttnParams p) {
  constexpr int kRows = 16 * MT;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = blockIdx.x;
  const int4 j = p.join[c];
  if (j.w <= c) return;
  const Request rq = request_of(p, j.x);
  for (int e = blockIdx.y * 128 + threadIdx.x; e < kRows * (D / 4); e += kJoinParts * 128) {
    const int row = e / (D / 4), d = (e % (D / 4)) * 4;
    bf16* out = row_of(p, rq.n, rq.q0, j.y, j.z + row, D);
    if (!out) continue;
    float m = -CUDART_INF_F, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int g = c; g <= j.w; ++g) {
      const long slot = static_cast<long>(g) * 2 + (g == c);
      const float2 ml = p.part_ml[slot * kRows + row];
      const float4 x = *reinterpret_cast<const float4*>(p.part + (slot * kRows + row) * D + d);
      const float mn = fmaxf(m, ml.x), ref = mn == -CUDART_INF_F ? 0.f : mn, f = ex2(m - ref), h = ex2(ml.x - ref);
      m = mn;
      l = l * f + ml.y * h;
      o.x = o.x * f + x.x * h;
      o.y = o.y * f + x.y * h;
      o.z = o.z * f + x.z * h;
      o.w = o.w * f + x.w * h;
    }
    const float f = inverse(l);
    __nv_bfloat162 y[2] = {__floats2bfloat162_rn(o.x * f, o.y * f), __floats2bfloat162_rn(o.z * f, o.w * f)};
    *reinterpret_cast<uint2*>(out + d) = *reinterpret_cast<uint2*>(y);
  }
}

template <int D, int MT>
cudaError_t run(const AttnParams& p, int grid, cudaStream_t st) {
  constexpr int bytes = sizeof(Smem<D, MT>);
  static_assert(bytes <= 232448, "shared memory of one CTA");
  cudaError_t e = cudaFuncSetAttribute(cache_attn_kernel<D, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return e;
  cache_attn_kernel<D, MT><<<grid, kThreads, bytes, st>>>(p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid, kJoinParts);
  cfg.blockDim = 128;
  cfg.stream = st;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, cache_attn_join_kernel<D, MT>, p);
  nsa::count_launch(2);
  return e;
}

// Warps on the same keys: rows of a request over 16, up to 8
int row_tiles(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : rows <= 64 ? 4 : 8; }
}  // namespace

// Floats of scratch that nsa_cache_attention needs
extern "C" long nsa_cache_attention_scratch(int Hq, int H, int D, int max_new) {
  const long G = H > 0 ? Hq / H : 1, mt = row_tiles(static_cast<int>(G * max_new < 1024 ? G * max_new : 1024)), grid = nsa::sm_count(), rows = 16 * mt;
  return grid * (kWarps / mt) * rows * D + grid * 2 * rows * (D + 2) + grid * 4;
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
  p.window = window;
  p.scale = softmax_scale * 1.4426950408889634f;
  p.status = nsa::status_ptr();
  const long most = static_cast<long>(p.G) * max_new;
  const int mt = row_tiles(static_cast<int>(most < 1024 ? most : 1024)), grid = nsa::sm_count(), rows = 16 * mt;
  p.part = scratch;
  p.part_ml = reinterpret_cast<float2*>(p.part + static_cast<long>(grid) * 2 * rows * D);
  p.join = reinterpret_cast<int4*>(p.part_ml + static_cast<long>(grid) * 2 * rows);
  p.head = reinterpret_cast<float*>(p.join + grid);
  cudaError_t e = cudaSuccess;
  for (int b = 0; b < B && e == cudaSuccess; b += kMaxRequests) {      // a launch for each 1024 requests, on the same scratch
    p.s = CacheStep{table + static_cast<long>(b) * W, query_start + b, lengths + b, B - b < kMaxRequests ? B - b : kMaxRequests, W, N};
    if (D == 128)
      e = mt == 1 ? run<128, 1>(p, grid, st) : mt == 2 ? run<128, 2>(p, grid, st) : mt == 4 ? run<128, 4>(p, grid, st) : run<128, 8>(p, grid, st);
    else
      e = mt == 1 ? run<64, 1>(p, grid, st) : mt == 2 ? run<64, 2>(p, grid, st) : mt == 4 ? run<64, 4>(p, grid, st) : run<64, 8>(p, grid, st);
  }
  return e == cudaSuccess ? 0 : nsa::fail_cuda(e, "nsa_cache_attention launch");
}
