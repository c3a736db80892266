// Attention of a step's queries over the paged 8-bit key / value cache.
#include <cuda_bf16.h>
#include <math_constants.h>

#include "cache.cuh"
#include "host.cuh"

namespace {
typedef __nv_bfloat16 bf16;
constexpr int kWarps = 4;

// One CTA per query token and head.  A warp takes 32 keys at a time: a lane scores one key, then owns D / 32 columns of the output; the four
// warps' sums meet in shared memory.
template <int D>
__global__ void __launch_bounds__(32 * kWarps) cache_attn_kernel(const bf16* __restrict__ q, long ldq, CachePages c, CacheStep s, bf16* __restrict__ o,
                                                                 int Hq, int window, float scale_log2) {
  constexpr int kCols = D / 32;
  __shared__ float qs[D], os[kWarps][D], ms[kWarps], ls[kWarps];
  const int n = blockIdx.x, hq = blockIdx.y, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int b = 0, hi = s.B;
  while (hi - b > 1) {
    const int mid = (b + hi) >> 1;
    if (s.query_start[mid] <= n) b = mid; else hi = mid;
  }
  const bool inside = n < s.query_start[s.B] && n >= s.query_start[b];
  const long pos = inside ? static_cast<long>(s.lengths[b]) - s.query_start[b + 1] + n : -1;
  for (int d = threadIdx.x; d < D; d += 32 * kWarps) qs[d] = __bfloat162float(q[n * ldq + static_cast<long>(hq) * D + d]);
  __syncthreads();
  const int P = 1 << c.shift, h = hq / (Hq / c.H);
  float m = -CUDART_INF_F, l = 0.f, acc[kCols] = {};
  const long from = window > 0 && pos >= window ? pos - window + 1 : 0;
  for (long base = from / 32 * 32 + 32 * w; base <= pos; base += 32 * kWarps) {
    const long at = base + lane;
    const int page = at <= pos && at >= from ? page_of(s, c, b, at) : -1;
    float x = -CUDART_INF_F;
    if (page >= 0) {
      const long ph = static_cast<long>(page) * c.H + h;
      float dot = 0.f;
      for (int d = 0; d < D; ++d) dot += qs[d] * (c.k[ph * P * D + key_at(static_cast<int>(at & (P - 1)), d, D)] - 128.f);
      x = dot * c.scale[ph * 2] * scale_log2;
    }
    float top = x;
    bool nan = x != x;
    for (int i = 16; i; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
    nan = __any_sync(0xffffffffu, nan);
    const float mn = nan ? CUDART_NAN_F : fmaxf(m, top);
    if (mn == -CUDART_INF_F) continue;
    const float keep = m == -CUDART_INF_F ? 0.f : exp2f(m - mn), p = page >= 0 ? exp2f(x - mn) : 0.f;
    float sum = p;
    for (int i = 16; i; i >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
    l = l * keep + sum;
    m = mn;
    for (int i = 0; i < kCols; ++i) acc[i] *= keep;
    for (int j = 0; j < 32; ++j) {
      const float pj = __shfl_sync(0xffffffffu, p, j);
      const int page_j = __shfl_sync(0xffffffffu, page, j);
      if (page_j < 0) continue;
      const long ph = static_cast<long>(page_j) * c.H + h;
      const float f = pj * c.scale[ph * 2 + 1];
      for (int i = 0; i < kCols; ++i)
        acc[i] += f * (c.v[ph * P * D + value_at(static_cast<int>((base + j) & (P - 1)), lane * kCols + i, D)] - 128.f);
    }
  }
  for (int i = 0; i < kCols; ++i) os[w][lane * kCols + i] = acc[i];
  if (lane == 0) { ms[w] = m; ls[w] = l; }
  __syncthreads();
  float mm = -CUDART_INF_F, ll = 0.f;
  bool nan = false;
  for (int i = 0; i < kWarps; ++i) { mm = fmaxf(mm, ms[i]); nan |= ms[i] != ms[i]; }
  float f[kWarps];
  for (int i = 0; i < kWarps; ++i) {
    f[i] = nan ? CUDART_NAN_F : ms[i] == -CUDART_INF_F ? 0.f : exp2f(ms[i] - mm);
    ll += ls[i] * f[i];
  }
  for (int d = threadIdx.x; d < D; d += 32 * kWarps) {
    float r = 0.f;
    for (int i = 0; i < kWarps; ++i) r += os[i][d] * f[i];
    o[(static_cast<long>(n) * Hq + hq) * D + d] = __float2bfloat16(ll == 0.f ? 0.f : r / ll);
  }
}
}  // namespace

extern "C" int nsa_cache_attention(const void* q, long ldq, const void* kc, const void* vc, const float* scale, const int* table, const int* query_start,
                                   const int* lengths, void* o, int B, int W, int N, int pages, int Hq, int H, int D, int page_size, int window,
                                   float softmax_scale, int max_new, cudaStream_t st) {
  if (N == 0) return 0;
  if (B <= 0 || N < 0 || H <= 0 || Hq % H || Hq > 65535 || (D != 64 && D != 128) || max_new < 1)
    return nsa::fail(NSA_ERR_SHAPE, "cache_attention: unsupported shape");
  const CachePages c{static_cast<uint8_t*>(const_cast<void*>(kc)), static_cast<uint8_t*>(const_cast<void*>(vc)), const_cast<float*>(scale), pages, H, D,
                     __builtin_ctz(page_size)};
  const CacheStep s{table, query_start, lengths, B, W, N};
  auto* kernel = D == 128 ? cache_attn_kernel<128> : cache_attn_kernel<64>;
  kernel<<<dim3(N, Hq), 32 * kWarps, 0, st>>>(static_cast<const bf16*>(q), ldq, c, s, static_cast<bf16*>(o), Hq, window,
                                              softmax_scale * 1.4426950408889634f);
  nsa::count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : nsa::fail_cuda(e, "nsa_cache_attention launch");
}
