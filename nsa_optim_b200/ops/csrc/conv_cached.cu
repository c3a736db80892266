// The short causal convolution of packed tokens that continue their requests (see ops/states.py):
//     y_t = act(bias + sum_j w_j u_{t - W + 1 + j}),
// u the request's inputs, of which the last W - 1 before the step are in its row of the state.
#include <cuda_bf16.h>

#include "f32x2.cuh"
#include "host.cuh"
#include "packed.cuh"

namespace {
typedef __nv_bfloat16 bf16;
constexpr int kThreads = 128;

// V channels of a row as they are in memory
template <int V>
struct Row {
  uint32_t w[(V + 1) / 2];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (auto& x : w) x = 0;
  }
  __device__ __forceinline__ void load(const bf16* p) {
    if constexpr (V == 4) {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      w[0] = u.x, w[1] = u.y;
    } else {
      w[0] = *reinterpret_cast<const unsigned short*>(p);
    }
  }
  __device__ __forceinline__ void store(bf16* p) const {
    if constexpr (V == 4) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<unsigned short*>(p) = static_cast<unsigned short>(w[0]);
  }
  __device__ __forceinline__ float at(int i) const { return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16); }
};
// The same as numbers, two at a time
template <int V>
struct Numbers {
  float2 v[(V + 1) / 2];
  __device__ __forceinline__ void operator=(const Row<V>& r) {
#pragma unroll
    for (int i = 0; i < (V + 1) / 2; ++i) v[i] = make_float2(r.at(2 * i), V > 1 ? r.at(2 * i + 1) : 0.f);
  }
};
__device__ __forceinline__ uint32_t two(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// z / (1 + exp(-z)) of two numbers
__device__ __forceinline__ float2 silu2(float2 z) {
  const float2 x = mul2(z, make_float2(-1.4426950408889634f, -1.4426950408889634f));
  const float2 d = add2(make_float2(1.f, 1.f), make_float2(exp2f(x.x), exp2f(x.y)));
  return make_float2(__fdividef(z.x, d.x), __fdividef(z.y, d.y));
}

// A thread has V channels of a window of tokens.  The window in which a request begins has its first W - 1 tokens too, wherever it ends: they alone need the
// old state, and the same thread then writes the new one, so nobody reads a row that another has changed.  The next eight rows are in flight while these are
// worked on.  Bound by memory and what hides it: 14.4 K tokens of 4352 channels (268 MB) 50 us, 5.4 TB/s; 60 with an address worked out for every row, 61 with
// four rows ahead, 57 with twelve.
template <int W, int V, bool act>
__global__ void __launch_bounds__(kThreads) conv_cached_kernel(const bf16* __restrict__ x, long ldx, const bf16* __restrict__ weight,
                                                               const bf16* __restrict__ bias, bf16* __restrict__ state, bf16* __restrict__ y,
                                                               const int* __restrict__ query_start, const int* __restrict__ lengths, int B, int N, int C,
                                                               int window) {
  constexpr int K = W - 1, AHEAD = 8, PAIRS = (V + 1) / 2;
  const int c = (blockIdx.y * kThreads + threadIdx.x) * V, i0 = blockIdx.x * window, i1 = min(i0 + window, N);
  const bool mine = c < C;
  Request r = request_at(query_start, lengths, B, i0);
  float2 w[W][PAIRS], b[PAIRS];
  if (mine) {
    Row<V> taps[W], own;                                               // V * W numbers side by side: a channel's taps are neighbours
    own.zero();
    if (bias) own.load(bias + c);
#pragma unroll
    for (int j = 0; j < W; ++j) taps[j].load(weight + static_cast<long>(c) * W + j * V);
    auto tap = [&](int v, int j) { return v < V ? taps[(v * W + j) / V].at((v * W + j) % V) : 0.f; };
#pragma unroll
    for (int v = 0; v < PAIRS; ++v) {
      b[v] = make_float2(own.at(2 * v), V > 1 ? own.at(2 * v + 1) : 0.f);
#pragma unroll
      for (int j = 0; j < W; ++j) w[j][v] = make_float2(tap(2 * v, j), tap(2 * v + 1, j));
    }
  }
  int i = i0;
  while (i < i1) {
    if (i >= r.next) r = request_at(query_start, lengths, B, i);
    if (i < r.first || i >= r.next) {                                  // of no request
      Row<V> none;
      none.zero();
      if (mine) none.store(y + static_cast<long>(i) * C + c);
      ++i;
      continue;
    }
    const int t = i - max(r.first, 0), last = min(r.next, N);
    if (i == i0 && t > 0 && t < K) {                                   // of the window before
      i = min(max(r.first, 0) + K, last);
      continue;
    }
    const int end = t == 0 ? min(last, max(i1, i + K)) : min(last, i1);
    if (mine) {
      Row<V> h[K];                                                     // the inputs before, the oldest first
      const bf16* at = x + static_cast<long>(i) * ldx + c;
      if (t > 0) {
#pragma unroll
        for (int j = 0; j < K; ++j) {
          if (t >= K - j) h[j].load(at - (K - j) * ldx);
          else h[j].zero();                                            // requests that overlap, which no step has: nothing in front of x is read
        }
      } else {
        const bool fresh = r.length <= r.next - r.first;
        bf16* own = state + static_cast<long>(r.b) * K * C + c;
        const int m = last - i;                                        // new tokens
#pragma unroll
        for (int j = 0; j < K; ++j) {
          if (fresh) h[j].zero();
          else h[j].load(own + j * C);
        }
#pragma unroll
        for (int j = 0; j < K; ++j) {
          Row<V> s;
          if (m - K + j >= 0) {
            s.load(at + static_cast<long>(m - K + j) * ldx);
          } else {
            s = h[K - 1];
#pragma unroll
            for (int e = 0; e < K; ++e)
              if (e == m + j) s = h[e];
          }
          s.store(own + j * C);
        }
      }
      bf16* to = y + static_cast<long>(i) * C + c;
      Numbers<V> u[W];                                                 // the last W inputs
#pragma unroll
      for (int j = 0; j < K; ++j) u[j + 1] = h[j];
      Row<V> next[AHEAD];
      auto fetch = [&](int k) {
        if (k + AHEAD <= end) {
#pragma unroll
          for (int e = 0; e < AHEAD; ++e) next[e].load(at + e * ldx);
        } else {
#pragma unroll
          for (int e = 0; e < AHEAD; ++e)
            if (k + e < end) next[e].load(at + e * ldx);
        }
        at += AHEAD * ldx;
      };
      auto finish = [&](const Row<V>& row) {
#pragma unroll
        for (int j = 0; j < K; ++j) u[j] = u[j + 1];
        u[K] = row;
        Row<V> out;
#pragma unroll
        for (int v = 0; v < PAIRS; ++v) {
          float2 z = b[v];
#pragma unroll
          for (int j = 0; j < W; ++j) z = fma2(w[j][v], u[j].v[v], z);
          if (act) z = silu2(z);
          out.w[v] = two(z.x, z.y);
        }
        out.store(to);
        to += C;
      };
      fetch(i);
      for (int k = i; k < end; k += AHEAD) {
        Row<V> g[AHEAD];
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) g[e] = next[e];
        fetch(k + AHEAD);
        if (k + AHEAD <= end) {
#pragma unroll
          for (int e = 0; e < AHEAD; ++e) finish(g[e]);
        } else {
#pragma unroll
          for (int e = 0; e < AHEAD; ++e) {
            if (k + e >= end) break;
            finish(g[e]);
          }
        }
      }
    }
    i = end;
  }
}

template <int V, bool act>
auto* kernel_of(int W) { return W == 4 ? conv_cached_kernel<4, V, act> : W == 3 ? conv_cached_kernel<3, V, act> : conv_cached_kernel<2, V, act>; }
}  // namespace

// x (N, C) of pitch ldx, weight (C, W) and bias (C; or null) bf16 dense, state (B, W - 1, C), y (N, C) dense.
extern "C" int nsa_conv1d_cached(const void* x, long ldx, const void* weight, const void* bias, void* state, void* y, const int* query_start,
                                 const int* lengths, int B, int N, int C, int W, int act, cudaStream_t st) {
  if (N == 0) return 0;
  if (B <= 0 || N < 0 || C <= 0 || W < 2 || W > 4) return nsa::fail(NSA_ERR_SHAPE, "conv1d_cached: 2 to 4 taps, and requests and channels, are needed");
  const uintptr_t places = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(state) | reinterpret_cast<uintptr_t>(y) |
                           reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(bias);
  const bool wide = C % 4 == 0 && ldx % 4 == 0 && places % 8 == 0;       // whole 8-byte pieces
  const int columns = (C + kThreads * (wide ? 4 : 1) - 1) / (kThreads * (wide ? 4 : 1));
  if (columns > 65535) return nsa::fail(NSA_ERR_SHAPE, "conv1d_cached: too many channels");
  // Longer windows read fewer rows twice and weights seldomer, as long as two CTAs for each SM are left: 256 / 1024 / 4096 tokens of 4352 channels 3.8 / 5.7 / 15.8 us; with
  // eight left 7.4 / 9.2 / 16.8, with one 3.6 / 5.8 / 15.9
  int window = 1;
  while (window < 64 && static_cast<long>((N + 2 * window - 1) / (2 * window)) * columns >= 2l * nsa::sm_count()) window *= 2;
  auto* kernel = wide ? (act ? kernel_of<4, true>(W) : kernel_of<4, false>(W)) : act ? kernel_of<1, true>(W) : kernel_of<1, false>(W);
  kernel<<<dim3((N + window - 1) / window, columns), kThreads, 0, st>>>(static_cast<const bf16*>(x), ldx, static_cast<const bf16*>(weight),
                                                                       static_cast<const bf16*>(bias), static_cast<bf16*>(state), static_cast<bf16*>(y),
                                                                       query_start, lengths, B, N, C, window);
  nsa::count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : nsa::fail_cuda(e, "nsa_conv1d_cached launch");
}
