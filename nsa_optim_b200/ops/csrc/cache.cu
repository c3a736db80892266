// The paged 8-bit key / value cache: pages and slots of a step, appending, reading back.
#include <cuda_bf16.h>

#include "cache.cuh"
#include "host.cuh"

namespace {
typedef __nv_bfloat16 bf16;

// ------------------------------------------------------------------------------------- pages and slots of a step
constexpr int kPlanThreads = 1024;

// Exclusive prefix of two values per thread over the CTA, and their totals
__device__ __forceinline__ void scan2(long long& a, long long& b, long long& ta, long long& tb, long long (*warps)[2]) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  long long x = a, y = b;
  for (int d = 1; d < 32; d <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, x, d), v = __shfl_up_sync(0xffffffffu, y, d);
    if (lane >= d) { x += u; y += v; }
  }
  if (lane == 31) { warps[w][0] = x; warps[w][1] = y; }
  __syncthreads();
  long long bx = 0, by = 0;
  ta = tb = 0;
  for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) {
    if (i < w) { bx += warps[i][0]; by += warps[i][1]; }
    ta += warps[i][0];
    tb += warps[i][1];
  }
  __syncthreads();
  a = bx + x - a;
  b = by + y - b;
}

__device__ __forceinline__ int pages_for(long long tokens, int shift) { return static_cast<int>((tokens + (1 << shift) - 1) >> shift); }

// Every CTA scans all requests (start[b], and first[b]: new pages of the requests before b, both in shared memory) and writes its share of the
// table's new entries and of the slots.
__global__ void __launch_bounds__(kPlanThreads) cache_plan_kernel(const int* __restrict__ lengths, const int* __restrict__ add, int* __restrict__ table,
                                                                  const int* __restrict__ free_pages, const int* __restrict__ free_count, int F,
                                                                  int* __restrict__ query_start, int* __restrict__ total,
                                                                  long long* __restrict__ slots, long long* __restrict__ positions,
                                                                  int* __restrict__ free_left, int* __restrict__ shortfall, int B, int W, int N,
                                                                  int shift) {
  extern __shared__ int plan_smem[];
  __shared__ long long warps[kPlanThreads / 32][2];
  int *start = plan_smem, *first = plan_smem + B + 1;
  const int t = threadIdx.x, count = min(max(*free_count, 0), F);
  long long tokens = 0, pages = 0, wanted = 0;
  for (int base = 0; base < B; base += kPlanThreads) {
    const int b = base + t;
    const int len = b < B ? max(lengths[b], 0) : 0;
    long long n = b < B ? max(add[b], 0) : 0, zero = 0, all, none;
    const long long mine = n;
    scan2(n, zero, all, none, warps);
    const long long lo = min(tokens + n, static_cast<long long>(N)), hi = min(tokens + n + mine, static_cast<long long>(N));
    const int held = pages_for(len, shift), need = pages_for(len + (hi - lo), shift);
    long long take = min(need, W) - min(held, W), lack = need - held, all_take, all_lack;
    scan2(take, lack, all_take, all_lack, warps);
    if (b < B) {
      start[b] = static_cast<int>(lo);
      first[b] = static_cast<int>(pages + take);
      if (blockIdx.x == 0) {
        query_start[b] = static_cast<int>(lo);
        total[b] = static_cast<int>(len + (hi - lo));
      }
    }
    tokens += all;
    pages += all_take;
    wanted += all_lack;
  }
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
  const int lane = t & 31, warp = blockIdx.x * (kPlanThreads / 32) + (t >> 5), warps_all = gridDim.x * (kPlanThreads / 32);
  for (int b = warp; b < B; b += warps_all) {
    const int held = pages_for(max(lengths[b], 0), shift), n = first[b + 1] - first[b];
    for (int j = lane; j < n; j += 32) {
      const int order = first[b] + j;
      table[static_cast<long>(b) * W + held + j] = order < count ? free_pages[count - 1 - order] : -1;
    }
  }
  for (long i = static_cast<long>(blockIdx.x) * kPlanThreads + t; i < N; i += static_cast<long>(gridDim.x) * kPlanThreads) {
    long long slot = -1, pos = 0;
    if (i < start[B]) {
      int lo = 0, hi = B;                       // the last request that begins at i or before and is not empty
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= i) lo = mid; else hi = mid;
      }
      const int len = max(lengths[lo], 0), held = pages_for(len, shift);
      pos = len + (i - start[lo]);
      const long long j = pos >> shift;
      int page = -1;
      if (j < W) {
        const long long order = first[lo] + (j - held);
        page = j < held ? table[static_cast<long>(lo) * W + j] : order < count ? free_pages[count - 1 - order] : -1;
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
  __shared__ long long warps[kPlanThreads / 32][2];
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
    long long mine = t < end ? have[t] : 0, zero = 0, all, none;
    scan2(mine, zero, all, none, warps);
    if (t < end) have[t] = static_cast<int>(mine);
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
__device__ __forceinline__ uint8_t code_of(float x, float inv) { return static_cast<uint8_t>(static_cast<int>(rintf(x * inv)) + 128); }

constexpr int kAppendThreads = 128;

// One CTA per window of packed tokens and head.  The tokens of a request that lie in one page are a group, handled by the CTA
// in whose window the first of them lies: their largest magnitudes give the page's scales, codes that are there are rounded again where
// a scale grows, then the new ones are stored.
__global__ void __launch_bounds__(kAppendThreads) cache_append_kernel(const bf16* __restrict__ k, const bf16* __restrict__ v, long ldk, long ldv, CachePages c,
                                                                      CacheStep s, int window) {
  __shared__ unsigned red[kAppendThreads / 32][2];
  const int h = blockIdx.y, t = threadIdx.x, D = c.D, P = 1 << c.shift;
  const int total = min(s.query_start[s.B], s.N);
  int i = blockIdx.x * window;
  const int end = min(i + window, total);
  while (i < end) {
    int lo = 0, hi = s.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s.query_start[mid] <= i) lo = mid; else hi = mid;
    }
    const int first = s.query_start[lo], last = min(s.query_start[lo + 1], total);
    const long pos = static_cast<long>(s.lengths[lo]) - s.query_start[lo + 1] + i;
    const int off = static_cast<int>(pos & (P - 1));
    const int m = max(min(last - i, P - off), 1);
    const int page = page_of(s, c, lo, pos);
    if ((off != 0 && i != first) || page < 0) {
      i += m;
      continue;
    }
    unsigned ak = 0, av = 0;                     // magnitudes as bits: NaN above infinity above all numbers
    for (int x = t; x < m * D; x += kAppendThreads) {
      const long r = i + x / D;
      const int d = x % D;
      ak = max(ak, __float_as_uint(__bfloat162float(k[r * ldk + h * D + d])) & 0x7fffffffu);
      av = max(av, __float_as_uint(__bfloat162float(v[r * ldv + h * D + d])) & 0x7fffffffu);
    }
    for (int o = 16; o; o >>= 1) {
      ak = max(ak, __shfl_xor_sync(0xffffffffu, ak, o));
      av = max(av, __shfl_xor_sync(0xffffffffu, av, o));
    }
    if ((t & 31) == 0) { red[t >> 5][0] = ak; red[t >> 5][1] = av; }
    __syncthreads();
    for (int w = 0; w < kAppendThreads / 32; ++w) { ak = max(ak, red[w][0]); av = max(av, red[w][1]); }
    const long ph = static_cast<long>(page) * c.H + h;
    int e[2] = {step_exponent(ak), step_exponent(av)}, old[2] = {e[0], e[1]};
    if (off)
      for (int x = 0; x < 2; ++x) {
        old[x] = exponent_of(c.scale[ph * 2 + x]);
        e[x] = max(e[x], old[x]);
      }
    __syncthreads();                             // the scales have been read
    uint8_t *kc = c.k + ph * P * D, *vc = c.v + ph * P * D;
    for (int x = 0; x < 2; ++x) {
      uint8_t* codes = x ? vc : kc;
      if (e[x] != old[x] && e[x] != kNoStep) {
        const float ratio = power2(max(old[x] - e[x], -126));
        for (int y = t; y < off * D; y += kAppendThreads) {
          const int at = x ? value_at(y / D, y % D, D) : key_at(y / D, y % D, D);
          codes[at] = code_of(static_cast<float>(codes[at]) - 128.f, ratio);
        }
      }
      const float inv = e[x] == kNoStep ? 0.f : power2(-e[x]);
      for (int y = t; y < m * D; y += kAppendThreads) {
        const long r = i + y / D;
        const int d = y % D, tok = off + y / D;
        const float f = __bfloat162float(x ? v[r * ldv + h * D + d] : k[r * ldk + h * D + d]);
        codes[x ? value_at(tok, d, D) : key_at(tok, d, D)] = e[x] == kNoStep ? 128 : code_of(f, inv);
      }
    }
    if (t < 2) c.scale[ph * 2 + t] = e[t] == kNoStep ? __int_as_float(0x7fc00000) : power2(e[t]);
    i += m;
  }
}

// One CTA per page and head: bf16 values (n, P, H, D) of both sides.
__global__ void __launch_bounds__(128) cache_values_kernel(CachePages c, const int* __restrict__ ids, bf16* __restrict__ k, bf16* __restrict__ v) {
  const int h = blockIdx.y, P = 1 << c.shift, D = c.D, page = ids[blockIdx.x];
  const bool there = page >= 0 && page < c.pages;
  const long ph = static_cast<long>(there ? page : 0) * c.H + h;
  const float sk = c.scale[ph * 2], sv = c.scale[ph * 2 + 1];
  for (int x = threadIdx.x; x < P * D; x += 128) {
    const int tok = x / D, d = x % D;
    const long at = ((static_cast<long>(blockIdx.x) * P + tok) * c.H + h) * D + d;
    k[at] = __float2bfloat16(there ? (c.k[ph * P * D + key_at(tok, d, D)] - 128.f) * sk : 0.f);
    v[at] = __float2bfloat16(there ? (c.v[ph * P * D + value_at(tok, d, D)] - 128.f) * sv : 0.f);
  }
}
}  // namespace

extern "C" int nsa_cache_plan(const int* lengths, const int* add, int* table, const int* free_pages, const int* free_count, int F, int* query_start,
                              int* total, long long* slots, long long* positions, int* free_left, int* shortfall, int B, int W, int N,
                              int page_size, cudaStream_t st) {
  if (B <= 0 || W <= 0 || N < 0 || F < 0) return nsa::fail(NSA_ERR_SHAPE, "cache_plan: empty problem");
  if (B > nsa_cache_plan_limit()) return nsa::fail(NSA_ERR_LIMIT, "cache_plan: more requests than shared memory holds");
  const int bytes = 2 * (B + 1) * 4;
  if (bytes > 40000) {
    const cudaError_t e = cudaFuncSetAttribute(cache_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200000);
    if (e != cudaSuccess) return nsa::fail_cuda(e, "nsa_cache_plan");
  }
  const int want = (N + 4 * kPlanThreads - 1) / (4 * kPlanThreads), most = nsa::sm_count();
  const int grid = want < 1 ? 1 : want < most ? want : most;
  cache_plan_kernel<<<grid, kPlanThreads, bytes, st>>>(lengths, add, table, free_pages, free_count, F, query_start, total, slots, positions, free_left,
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

extern "C" int nsa_cache_append(const void* k, const void* v, long ldk, long ldv, void* kc, void* vc, float* scale, const int* table,
                                const int* query_start, const int* lengths, int B, int W, int N, int pages, int H, int D, int page_size,
                                cudaStream_t st) {
  if (N == 0) return 0;
  if (B <= 0 || H <= 0 || H > 65535 || D % 64 || N < 0) return nsa::fail(NSA_ERR_SHAPE, "cache_append: unsupported shape");
  const CachePages c{static_cast<uint8_t*>(kc), static_cast<uint8_t*>(vc), scale, pages, H, D, __builtin_ctz(page_size)};
  const CacheStep s{table, query_start, lengths, B, W, N};
  const int window = N <= 2048 ? 1 : page_size;
  cache_append_kernel<<<dim3((N + window - 1) / window, H), kAppendThreads, 0, st>>>(static_cast<const bf16*>(k), static_cast<const bf16*>(v), ldk, ldv, c, s,
                                                                                     window);
  nsa::count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : nsa::fail_cuda(e, "nsa_cache_append launch");
}

extern "C" int nsa_cache_values(const void* kc, const void* vc, const float* scale, const int* ids, void* k, void* v, int n, int pages, int H, int D,
                                int page_size, cudaStream_t st) {
  if (n == 0) return 0;
  if (H <= 0 || H > 65535 || D % 64 || n < 0) return nsa::fail(NSA_ERR_SHAPE, "cache_values: unsupported shape");
  const CachePages c{static_cast<uint8_t*>(const_cast<void*>(kc)), static_cast<uint8_t*>(const_cast<void*>(vc)), const_cast<float*>(scale), pages, H, D,
                     __builtin_ctz(page_size)};
  cache_values_kernel<<<dim3(n, H), 128, 0, st>>>(c, ids, static_cast<bf16*>(k), static_cast<bf16*>(v));
  nsa::count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : nsa::fail_cuda(e, "nsa_cache_values launch");
}
