// Log probabilities of given tokens, entropies and the likeliest tokens of rows of logits, and their gradient.
//
// With m = max x, S = sum e^(x - m): log p_j = x_j - m - log S, and the entropy is log S + sum (m - x) e^(x - m) / S, a sum of terms that are not
// negative, so nothing cancels where a distribution is narrow.  Compiled without fast math: the logarithms at a row's end are the exact ones,
// the exponentials of its elements the hardware's.
#include <cuda_bf16.h>
#include <math_constants.h>

#include "host.cuh"

namespace {
typedef __nv_bfloat16 bf16;
constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

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
__device__ __forceinline__ float value(const bf16* p, long i) { return __bfloat162float(p[i]); }
__device__ __forceinline__ float value(const float* p, long i) { return p[i]; }
__device__ __forceinline__ void store(bf16* p, long i, float x) { p[i] = __float2bfloat16(x); }
__device__ __forceinline__ void store(float* p, long i, float x) { p[i] = x; }

// Order of the likeliest tokens as whole numbers: larger logits first, NaN before all, -0 as 0, then the lower index
__device__ __forceinline__ unsigned long long rank_of(float x, int i) {
  const int bits = x != x ? 0x7fffffff : __float_as_int(x + 0.f);
  const unsigned ordered = bits >= 0 ? static_cast<unsigned>(bits) | 0x80000000u : ~static_cast<unsigned>(bits);
  return static_cast<unsigned long long>(ordered) << 32 | (0xffffffffu - static_cast<unsigned>(i));
}

template <class F>
__device__ __forceinline__ float block_reduce(float x, F op, float* red) {
  for (int o = 16; o; o >>= 1) x = op(x, __shfl_xor_sync(0xffffffffu, x, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
  __syncthreads();
  x = red[0];
  for (int i = 1; i < kThreads / 32; ++i) x = op(x, red[i]);
  return x;
}

// One CTA per row; the k best by k passes.
template <class T>
__global__ void __launch_bounds__(kThreads) logprobs_fwd_kernel(const T* __restrict__ logits, long ld, const long long* __restrict__ tokens,
                                                                float* __restrict__ logprob, float* __restrict__ entropy, float2* __restrict__ stats,
                                                                float* __restrict__ top, long long* __restrict__ index, int V, int k,
                                                                long long ignore, KernelStatus* status) {
  __shared__ float red[kThreads / 32];
  __shared__ unsigned long long best[kThreads / 32];
  const long row = blockIdx.x;
  const T* x = logits + row * ld;
  auto larger = [](float a, float b) { return a != a || a > b ? a : b; };        // NaN stays
  auto plus = [](float a, float b) { return a + b; };
  float m = -CUDART_INF_F;
  for (int i = threadIdx.x; i < V; i += kThreads) m = larger(m, value(x, i));
  m = block_reduce(m, larger, red);
  const bool empty = m == -CUDART_INF_F;
  float S = 0.f, E = 0.f;
  for (int i = threadIdx.x; i < V; i += kThreads) {
    const float d = value(x, i) - m, e = empty ? 0.f : ex2(d * kLog2e);
    S += e;
    E += e > 0.f ? -d * e : e;                   // a NaN stays one
  }
  S = block_reduce(S, plus, red);
  E = block_reduce(E, plus, red);
  if (threadIdx.x == 0) {
    const long long t = tokens[row];
    NSA_CHECK_INDEX(t == ignore || (t >= 0 && t < V), status, t);
    logprob[row] = t == ignore || t < 0 || t >= V ? 0.f : empty ? m : value(x, t) - m - logf(S);
    entropy[row] = empty ? 0.f : logf(S) + E / S;
    stats[row] = make_float2(m, empty ? 0.f : logf(S));      // apart: their sum would round a probability by |m| 2^-24
  }
  unsigned long long last = ~0ull;
  for (int j = 0; j < k; ++j) {
    unsigned long long r = 0;
    for (int i = threadIdx.x; i < V; i += kThreads) {
      const unsigned long long a = rank_of(value(x, i), i);
      if (a < last && a > r) r = a;
    }
    for (int o = 16; o; o >>= 1) {
      const unsigned long long a = __shfl_xor_sync(0xffffffffu, r, o);
      r = a > r ? a : r;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) best[threadIdx.x >> 5] = r;
    __syncthreads();
    for (int i = 0; i < kThreads / 32; ++i) r = best[i] > r ? best[i] : r;
    last = r;
    if (threadIdx.x == 0) {
      const int i = static_cast<int>(0xffffffffu - static_cast<unsigned>(r));
      index[row * k + j] = i;
      top[row * k + j] = empty ? m : value(x, i) - m - logf(S);
    }
  }
}

// dx_j = -p_j (G + g_H (log p_j + H)), G the sum of the row's other gradients; theirs are added at their tokens.
template <class T>
__global__ void __launch_bounds__(kThreads) logprobs_bwd_kernel(const T* __restrict__ logits, long ld, const long long* __restrict__ tokens,
                                                                const float2* __restrict__ stats, const float* __restrict__ entropy,
                                                                const long long* __restrict__ index, const float* __restrict__ dlogprob,
                                                                const float* __restrict__ dentropy, const float* __restrict__ dtop,
                                                                T* __restrict__ dx, int V, int k, long long ignore) {
  const long row = blockIdx.x;
  const T* x = logits + row * ld;
  const float m = stats[row].x, logS = stats[row].y, H = entropy[row], gH = dentropy ? dentropy[row] : 0.f;
  const long long t = tokens[row];
  const bool counts = !(t == ignore || t < 0 || t >= V), empty = m == -CUDART_INF_F;
  const float g = counts && dlogprob ? dlogprob[row] : 0.f;
  float G = g;
  for (int j = 0; j < k; ++j) G += dtop ? dtop[row * k + j] : 0.f;
  for (int i = threadIdx.x; i < V; i += kThreads) {
    const float lp = value(x, i) - m - logS, p = ex2_small(lp * kLog2e);
    float d = p > 0.f || p != p ? -p * (G + gH * (lp + H)) : 0.f;
    if (counts && i == t) d += g;
    if (dtop)
      for (int j = 0; j < k; ++j)
        if (index[row * k + j] == i) d += dtop[row * k + j];
    store(dx, row * V + i, empty ? 0.f : d);
  }
}
}  // namespace

extern "C" int nsa_logprobs_fwd(const void* logits, long ld, int fp32, const long long* tokens, float* logprob, float* entropy, float* stats, float* top,
                                long long* index, long rows, int V, int k, long long ignore, cudaStream_t st) {
  if (rows <= 0) return 0;
  if (V <= 0 || k < 0 || k > V || rows > 0x7fffffff) return nsa::fail(NSA_ERR_SHAPE, "logprobs: unsupported shape");
  KernelStatus* status = nsa::status_ptr();
  const unsigned grid = static_cast<unsigned>(rows);
  if (fp32)
    logprobs_fwd_kernel<<<grid, kThreads, 0, st>>>(static_cast<const float*>(logits), ld, tokens, logprob, entropy, reinterpret_cast<float2*>(stats), top, index, V, k, ignore, status);
  else
    logprobs_fwd_kernel<<<grid, kThreads, 0, st>>>(static_cast<const bf16*>(logits), ld, tokens, logprob, entropy, reinterpret_cast<float2*>(stats), top, index, V, k, ignore, status);
  nsa::count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : nsa::fail_cuda(e, "nsa_logprobs_fwd launch");
}

extern "C" int nsa_logprobs_bwd(const void* logits, long ld, int fp32, const long long* tokens, const float* stats, const float* entropy,
                                const long long* index, const float* dlogprob, const float* dentropy, const float* dtop, void* dx, long rows, int V,
                                int k, long long ignore, cudaStream_t st) {
  if (rows <= 0) return 0;
  if (V <= 0 || k < 0 || k > V || rows > 0x7fffffff) return nsa::fail(NSA_ERR_SHAPE, "logprobs: unsupported shape");
  const unsigned grid = static_cast<unsigned>(rows);
  if (fp32)
    logprobs_bwd_kernel<<<grid, kThreads, 0, st>>>(static_cast<const float*>(logits), ld, tokens, reinterpret_cast<const float2*>(stats), entropy, index, dlogprob, dentropy, dtop,
                                                   static_cast<float*>(dx), V, k, ignore);
  else
    logprobs_bwd_kernel<<<grid, kThreads, 0, st>>>(static_cast<const bf16*>(logits), ld, tokens, reinterpret_cast<const float2*>(stats), entropy, index, dlogprob, dentropy, dtop,
                                                   static_cast<bf16*>(dx), V, k, ignore);
  nsa::count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : nsa::fail_cuda(e, "nsa_logprobs_bwd launch");
}
