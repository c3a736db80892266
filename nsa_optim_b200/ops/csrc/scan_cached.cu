// The selective scan of packed tokens that continue their requests (see ops/states.py), for each head
//     d = softplus(dt + bias),   h <- exp(-exp(A_log) d) h + d x B^T   (P x S),   y = h C + D x.
// Compiled without fast math: decays are powers of numbers next to one.
#include <cuda_bf16.h>

#include "host.cuh"
#include "ssd.cuh"

namespace {

struct Scan {
  const bf16 *x, *dt, *Bm, *Cm;
  long ldx, ldt, ldb, ldc;                 // pitches of tokens; a token's heads, and its groups, are dense
  const void *A_log, *bias, *D;            // D may be null
  int A_fp32, bias_fp32, D_fp32;
  float* state;                            // (B, H, P, S)
  bf16* y;                                 // (N, H, P)
  const int *query_start, *lengths;
  int B, N, H, P, G;
};

__device__ __forceinline__ float param(const void* p, int i, int fp32) {
  return fp32 ? static_cast<const float*>(p)[i] : __bfloat162float(static_cast<const bf16*>(p)[i]);
}
__device__ __forceinline__ float softplus(float x) { return x > 20.f ? x : log1pf(expf(x)); }

// n consecutive bf16 numbers as they are in memory, n * 2 bytes aligned, and a pair of them as numbers
template <int n>
struct Raw {
  uint32_t w[(n + 1) / 2];
  __device__ __forceinline__ void load(const bf16* p) {
    if constexpr (n == 8) {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    } else if constexpr (n == 4) {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      w[0] = u.x, w[1] = u.y;
    } else if constexpr (n == 2) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      w[0] = *reinterpret_cast<const unsigned short*>(p);
    }
  }
  __device__ __forceinline__ float at(int i) const { return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16); }
  __device__ __forceinline__ float2 two(int i) const { return make_float2(at(2 * i), at(2 * i + 1)); }
};

// Sums of R numbers over LANES neighbouring lanes, R <= LANES: in each step a lane gives half of its numbers away, so that lane l of the group ends with
// number l / (LANES / R)
template <int R, int LANES>
__device__ __forceinline__ float sums(const float (&v)[R]) {
  const int lane = threadIdx.x & 31;
  if constexpr (R == 1) {
    float s = v[0];
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
  } else {
    float half[R / 2];
    const bool up = lane & (LANES / 2);
#pragma unroll
    for (int i = 0; i < R / 2; ++i) half[i] = (up ? v[i + R / 2] : v[i]) + __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + R / 2], LANES / 2);
    return sums<R / 2, LANES / 2>(half);
  }
}

// Token by token, the state in registers: a CTA has up to 64 rows (32 of 256 states) of one head's state of one request, a lane R rows of four or eight
// states, two at a time.  One token: the state passes through memory once, which is what bounds it (64 requests x 64 heads, 269 MB: 41 us, 6.5 TB/s; 48 with a
// state an instruction and 80 registers).  Several: instructions, of which a token's step size and decay, the same for all lanes, are worked out once, 64
// tokens at a time (48 requests of up to 8 tokens, 206 MB: 56 us, 82 with the step size in every lane).
template <int S>
struct Tile {
  static constexpr int LANES = S >= 128 ? 32 : S / 4, COLS = S / LANES, R = S == 256 ? 4 : S / 16, ROWS = 8 * R * (32 / LANES);
};
// What is left to the products: requests of more than `longest` new tokens, the ones with the most first (up to kRanked of them), and their chunks of 128
// tokens.  As whole numbers: how many requests, how many chunks; of each request itself and its first chunk; of each chunk its first token and how many.
// Behind them a record of numbers for each chunk and head (chunk_numbers), and the states in front of each chunk and head in bf16.
constexpr int kRanked = 1024, kChunk = 128;
struct Plan {
  int* at;                                 // null: there is none
  int room, chunks;                        // places for requests and for chunks
  __host__ __device__ long words() const { return (2 + 2l * room + 2l * chunks + 31) / 32 * 32; }
  __host__ __device__ float* records() const { return reinterpret_cast<float*>(at + words()); }
  __device__ int2* requests() const { return reinterpret_cast<int2*>(at + 2); }
  __device__ int2* table() const { return reinterpret_cast<int2*>(at + 2) + room; }
};
__device__ __forceinline__ int new_tokens(const Scan& a, int b) { return min(a.query_start[b + 1], a.N) - max(a.query_start[b], 0); }
// Exclusive prefix over the CTA's 256 threads, and the total
__device__ __forceinline__ int prefix256(int mine, int& total, int* warps) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int x = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += u;
  }
  __syncthreads();
  if (lane == 31) warps[w] = x;
  __syncthreads();
  int before = 0;
  total = 0;
  for (int i = 0; i < 8; ++i) {
    if (i < w) before += warps[i];
    total += warps[i];
  }
  return before + x - mine;
}
__device__ __forceinline__ void find_prompts(const Scan& a, int longest, const Plan& plan) {
  __shared__ int2 requests[kRanked];
  __shared__ int sizes[kRanked], warps[8];
  const int t = threadIdx.x, lane = t & 31;
  int found = 0, chunks = 0, total;
  for (int base = 0; base < a.B; base += 256) {                        // chunks are counted in the order of the requests
    const int b = base + t, n = b < a.B ? new_tokens(a, b) : 0;
    const int at = found + prefix256(n > longest, total, warps);
    found += total;
    const bool ours = n > longest && at < plan.room;                   // all of them, where requests do not overlap
    const int chunk = chunks + prefix256(ours ? (n + kChunk - 1) / kChunk : 0, total, warps);
    chunks += total;
    if (ours) {
      const int2 r = make_int2(b, min(chunk, plan.chunks));
      if (at < kRanked) requests[at] = r, sizes[at] = n;
      plan.requests()[at] = r;
    }
  }
  found = min(found, plan.room);
  if (t == 0) plan.at[0] = found, plan.at[1] = min(chunks, plan.chunks);
  __syncthreads();
  if (found <= kRanked)
    for (int i = t; i < found; i += 256) {
      int rank = 0;
      for (int j = 0; j < found; ++j) rank += sizes[j] > sizes[i] || (sizes[j] == sizes[i] && j < i);
      plan.requests()[rank] = requests[i];
    }
  __syncthreads();
  for (int i = t >> 5; i < found; i += 8) {
    const int2 r = plan.requests()[i];
    const int n = new_tokens(a, r.x), lo = max(a.query_start[r.x], 0);
    for (int k = lane; k * kChunk < n && r.y + k < plan.chunks; k += 32) plan.table()[r.y + k] = make_int2(lo + k * kChunk, min(n - k * kChunk, kChunk));
  }
}
// The same for one chunk, by a warp: its first token and how many, none where there are fewer chunks
__device__ __forceinline__ int2 chunk_at(const Scan& a, int longest, int c) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int base = 0; base < a.B; base += 32) {
    const int b = base + lane, n = b < a.B ? new_tokens(a, b) : 0, mine = n > longest ? (n + kChunk - 1) / kChunk : 0;
    int end = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, end, d);
      if (lane >= d) end += u;
    }
    const unsigned behind = __ballot_sync(0xffffffffu, before + end > c);
    if (behind) {
      const int at = __ffs(behind) - 1, k = c - before - __shfl_sync(0xffffffffu, end - mine, at);
      return make_int2(max(a.query_start[base + at], 0) + k * kChunk, min(__shfl_sync(0xffffffffu, n, at) - k * kChunk, kChunk));
    }
    before += __shfl_sync(0xffffffffu, end, 31);
  }
  return make_int2(0, 0);
}

__device__ __forceinline__ float ex2(float x) {                        // two steps of fp32 off at most
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Numbers of a chunk and head, by a warp, four neighbouring tokens a lane: what both kernels need of the step sizes is worked out once.  (With these sums in a
// warp of the kernels themselves its 600 instructions took longer than everything beside them: 3000 cycles a chunk in both.)  It does not wait for the plan.
// The sums of a chunk's logarithms are kept in two fp32 numbers each, formed in 64 bits: rows need differences of them, of which long steps in front would take the
// bits (in one number a token's own weight, its step size, was off by 0.5 % at steps of 60 and decays of 16).  Decays of less than 2^-kMostDecay are that: all that
// they multiply, a weight of 2^128 at most, is zero in fp32 either way, and the sums stay finite for any step size.
constexpr float kMostDecay = 512.f;
constexpr int kCum = 0, kLess = L, kCumLow = 2 * L, kLessLow = 3 * L, kCols = 4 * L, kRowFloats = 4 * L + 192, kWeight = kRowFloats, kDecay = kWeight + L,
              kRecord = kDecay + 4;
__device__ __forceinline__ float rest_of(double x) {                   // what the number rounded to fp32 leaves
  const float high = static_cast<float>(x);
  return isfinite(high) ? static_cast<float>(x - high) : 0.f;
}
__device__ __forceinline__ void chunk_numbers(const Scan& a, const Plan& plan, int longest, int c, int h) {
  const int lane = threadIdx.x & 31, blk = lane >> 3;
  const float rate = -expf(param(a.A_log, h, a.A_fp32)) * LOG2E, bias = param(a.bias, h, a.bias_fp32);
  const int2 chunk = chunk_at(a, longest, c);
  if (chunk.y > 0) {
    float raw[4], d[4], v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      raw[i] = 4 * lane + i < chunk.y ? __bfloat162float(a.dt[static_cast<long>(chunk.x + 4 * lane + i) * a.ldt + h]) : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {                      // 0 behind the request's last token
      d[i] = 4 * lane + i < chunk.y ? softplus(raw[i] + bias) : 0.f;
      v[i] = d[i] * rate;
      if (v[i] < -kMostDecay) v[i] = -kMostDecay;      // NaN stays
    }
    // inclusive sums from the chunk's start, exclusive ones from its end, in units of log 2
    double up[4] = {v[0], static_cast<double>(v[0]) + v[1], 0., 0.};
    up[2] = up[1] + v[2], up[3] = up[2] + v[3];
    float down[4] = {v[3] + v[2] + v[1], v[3] + v[2], v[3], 0.f};
    double run = up[3];
    float back = down[0] + v[0];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double x = __shfl_up_sync(0xffffffffu, run, o);
      const float y = __shfl_down_sync(0xffffffffu, back, o);
      if (lane >= o) run += x;
      if (lane + o < 32) back += y;
    }
    double before = __shfl_up_sync(0xffffffffu, run, 1);
    float behind = __shfl_down_sync(0xffffffffu, back, 1);
    if (lane == 0) before = 0.;
    if (lane == 31) behind = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) up[i] += before, down[i] += behind;
    float* to = plan.records() + (static_cast<long>(c) * a.H + h) * kRecord;
    auto keep = [&](int high, int low, const double (&x)[4]) {
      *reinterpret_cast<float4*>(to + high + 4 * lane) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4*>(to + low + 4 * lane) = make_float4(rest_of(x[0]), rest_of(x[1]), rest_of(x[2]), rest_of(x[3]));
    };
    keep(kCum, kCumLow, up);
    keep(kLess, kLessLow, {up[0] - log2f(d[0]), up[1] - log2f(d[1]), up[2] - log2f(d[2]), up[3] - log2f(d[3])});
    // Pairs of rows in different blocks of 32 need no exponential of their own: with m the sum at the end of an earlier block, exp(c_i - c_j) = exp(c_i - m)
    // exp(m - c_j), and both exponents are <= 0: the factors of columns j for row block p + 1, j < 32 (p + 1), at 16 p (p + 1) + j
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      const double mid = __shfl_sync(0xffffffffu, up[3], 8 * p + 7);
      auto factor = [&](int i) { return ex2(fminf(static_cast<float>(mid - up[i]), 0.f)) * d[i]; };
      if (blk <= p) *reinterpret_cast<float4*>(to + kCols + 16 * p * (p + 1) + 4 * lane) = make_float4(factor(0), factor(1), factor(2), factor(3));
    }
    *reinterpret_cast<float4*>(to + kWeight + 4 * lane) =
        make_float4(d[0] * exp2f(down[0]), d[1] * exp2f(down[1]), d[2] * exp2f(down[2]), d[3] * exp2f(down[3]));
    if (lane == 0) to[kDecay] = exp2f(back);
  }
}
// plan: where what is left to the products is written down, by one more CTA, and its chunks' numbers, by eight heads of a chunk a CTA
constexpr int kAtOnce = 64;
template <int S>
__global__ void __launch_bounds__(256, S == 256 ? 2 : 4) scan_tokens_kernel(const Scan a, int parts, int longest, const Plan plan) {
  if constexpr (S == NS) {
    const int more = static_cast<int>(blockIdx.x) - a.B * a.H * parts, blocks = (a.H + 7) / 8;
    if (more == 0) {
      find_prompts(a, longest, plan);
      return;
    }
    if (more > 0) {
      const int c = (more - 1) / blocks, h = (more - 1 - c * blocks) * 8 + (threadIdx.x >> 5);
      if (h < a.H) chunk_numbers(a, plan, longest, c, h);
      return;
    }
  }
  constexpr int LANES = Tile<S>::LANES, COLS = Tile<S>::COLS, R = Tile<S>::R, ROWS = Tile<S>::ROWS;
  __shared__ float2 sized[kAtOnce];                                    // step size and decay of each token
  const int part = blockIdx.x % parts, hb = blockIdx.x / parts, h = hb % a.H, b = hb / a.H, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = a.query_start[b], next = a.query_start[b + 1], lo = max(first, 0), hi = min(next, a.N);
  if (b == 0 || b == a.B - 1) {                                        // rows of no request
    const int before = b == 0 ? min(max(first, 0), a.N) : 0, behind = b == a.B - 1 ? max(hi, 0) : a.N, rows = min(ROWS, a.P - part * ROWS);
    for (long i = threadIdx.x; i < static_cast<long>(before + a.N - behind) * rows; i += 256) {
      const long k = i / rows, n = k < before ? k : behind + k - before;
      a.y[(n * a.H + h) * a.P + part * ROWS + i - k * rows] = __float2bfloat16(0.f);
    }
  }
  if (hi <= lo || hi - lo > longest) return;
  const int row = part * ROWS + (warp * (32 / LANES) + lane / LANES) * R, col = lane % LANES * COLS, g = h / (a.H / a.G);
  const bool mine = row < a.P;                                         // P is a multiple of 8, R divides 8
  float* own_state = a.state + ((static_cast<long>(b) * a.H + h) * a.P + row) * S + col;
  float2 st[R][COLS / 2];
  const bool fresh = a.lengths[b] <= next - first;
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int c = 0; c < COLS; c += 4) {
      const float4 u = mine && !fresh ? *reinterpret_cast<const float4*>(own_state + r * S + c) : make_float4(0.f, 0.f, 0.f, 0.f);
      st[r][c / 2] = make_float2(u.x, u.y), st[r][c / 2 + 1] = make_float2(u.z, u.w);
    }
  const float D = a.D ? param(a.D, h, a.D_fp32) : 0.f;
  const int sub = lane % LANES / (LANES / R);                          // the row whose sum the lane gets
  const bf16 *px = a.x + static_cast<long>(lo) * a.ldx + h * a.P + (mine ? row : 0);
  const bf16 *pb = a.Bm + static_cast<long>(lo) * a.ldb + g * S + col, *pc = a.Cm + static_cast<long>(lo) * a.ldc + g * S + col;
  bf16* py = a.y + (static_cast<long>(lo) * a.H + h) * a.P + row + sub;
  Raw<R> x;
  Raw<COLS> Bv, Cv;
  float skip;
  auto fetch = [&](int k) {
    x.load(px + k * a.ldx);
    Bv.load(pb + k * a.ldb);
    Cv.load(pc + k * a.ldc);
    skip = __bfloat162float(px[k * a.ldx + sub]);
  };
  fetch(0);
  for (int k0 = 0; k0 < hi - lo; k0 += kAtOnce) {
    const int m = min(hi - lo - k0, kAtOnce);
    if (k0) __syncthreads();
    if (threadIdx.x < m) {
      const float d = softplus(__bfloat162float(a.dt[(lo + k0 + static_cast<long>(threadIdx.x)) * a.ldt + h]) + param(a.bias, h, a.bias_fp32));
      sized[threadIdx.x] = make_float2(d, expf(d * -expf(param(a.A_log, h, a.A_fp32))));
    }
    __syncthreads();
    for (int j = 0; j < m; ++j) {
      const int k = k0 + j;
      const float2 size = sized[j], decay = make_float2(size.y, size.y);
      float2 Bk[COLS / 2], Ck[COLS / 2], xd[R], part[R];
#pragma unroll
      for (int c = 0; c < COLS / 2; ++c) Bk[c] = Bv.two(c), Ck[c] = Cv.two(c);
#pragma unroll
      for (int r = 0; r < R; ++r) xd[r].x = xd[r].y = size.x * x.at(r), part[r] = make_float2(0.f, 0.f);
      const float own = D * skip;
      if (k + 1 < hi - lo) fetch(k + 1);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < COLS / 2; ++c) {
          st[r][c] = fma2(decay, st[r][c], mul2(xd[r], Bk[c]));
          part[r] = fma2(st[r][c], Ck[c], part[r]);
        }
      float sum[R];
#pragma unroll
      for (int r = 0; r < R; ++r) sum[r] = part[r].x + part[r].y;
      const float out = sums<R, LANES>(sum) + own;
      if (mine && lane % (LANES / R) == 0) py[static_cast<long>(k) * a.H * a.P] = __float2bfloat16(out);
    }
  }
  if (mine) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int c = 0; c < COLS; c += 4)
        *reinterpret_cast<float4*>(own_state + r * S + c) = make_float4(st[r][c / 2].x, st[r][c / 2].y, st[r][c / 2 + 1].x, st[r][c / 2 + 1].y);
  }
}

// ------------------------------------------------------------------------------------- prompts
// 128 tokens at a time on the tensor cores, for S = 128 states and P = 64 columns.  With c the inclusive sums of d A over a chunk and H the state before it:
//     H <- exp(c_last) H + sum_j B_j (exp(c_last - c_j) d_j x_j)^T                                              (scan_states_kernel)
//     y_i = sum_{j <= i} (C_i . B_j) exp(c_i - c_j) d_j x_j + exp(c_i) C_i H + D x_i                            (scan_rows_kernel)
// The first kernel walks the chunks of a request's head with the state in registers, from the request's own state and back to it, and leaves the state in
// front of each chunk in bf16; the second has all chunks at once.  Operands of the rows' products are bf16 (scores and states are rounded to it), as where
// the scan trains: a rounding of 2^-8 in each term of a row, as in the row itself, that a hint of 16 new tokens at most avoids.  The state itself is fp32 and is handed on, so nothing is lost there: scaled x goes into its product as three bf16 numbers that add up
// to it exactly.  Its weights come from sums that run back from the chunk's end: differences c_last - c_j would lose the last tokens' bits where c is large.

// `bytes` consecutive bytes to shared memory; addresses and size are multiples of 16
__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(tc5::smem_u32(smem_dst)), "l"(src), "r"(bytes), "r"(tc5::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ uint32_t raw_param(const void* p, int i, int fp32) {          // of either type, to be made a number when it is there
  return fp32 ? static_cast<const uint32_t*>(p)[i] : static_cast<const unsigned short*>(p)[i];
}
__device__ __forceinline__ float param_of(uint32_t raw, int fp32) { return __uint_as_float(fp32 ? raw : raw << 16); }

// The chunks that a CTA walks one after another: items are (request, head, part of its columns), heads fastest, dealt out in turns of alternating direction
struct Walk {
  const Scan& a;
  const Plan& plan;
  int parts, round, total, h, part, group, b, lo, n, nc, k, chunk;
  bool fresh;
  __device__ Walk(const Scan& a_, const Plan& plan_, int parts_) : a(a_), plan(plan_), parts(parts_), round(0), total(plan_.at[0] * a_.H * parts_) { load(); }
  __device__ void load() {
    const int G = gridDim.x, c = blockIdx.x, at = round * G + (round & 1 ? G - 1 - c : c);
    k = nc = 0;
    if (at >= total) return;
    const int each = a.H * parts;
    h = at % each / parts;
    part = at % parts;
    group = h / (a.H / a.G) * NS;            // first column of its B and C
    const int2 r = plan.requests()[at / each];
    b = r.x;
    chunk = r.y;
    const int first = a.query_start[b], next = a.query_start[b + 1];
    lo = max(first, 0);
    n = min(next, a.N) - lo;
    nc = min((n + L - 1) / L, plan.chunks - chunk);
    fresh = a.lengths[b] <= next - first;
  }
  __device__ bool more() const { return k < nc; }
  __device__ void next() {
    if (++k == nc) {
      ++round;
      load();
    }
  }
  __device__ int t0() const { return lo + k * L; }
  __device__ int valid() const { return min(n - k * L, L); }
  __device__ bool last() const { return k + 1 == nc; }
};

// COLS: columns of the head that a CTA has, all 64 or half of them.  Of 24 warps eight for every 32 columns keep the state and the others scale x: eight all
// chunks or, in two groups, every other one.  Four more issue products, load and store.  Bound by shared memory: a chunk's 64 columns move 230 KB through it
// (B and x in, x read and its parts written, both operands of the product, the states out), 1800 of the 2100 cycles that it takes; 32 columns 145 KB, 1150 of
// 1300, in which the warps that keep the state and the one that issues products are busy too.  13.0 K tokens of 64 heads in 8 requests 65 us; one of 16 K 90 us
// in halves, 130 with one group that scales and two stages of B.
constexpr int kGroup = 8, kStatesWarps = 3 * kGroup + 4;
template <int COLS>
struct StatesSmem {
  static constexpr int kStagesB = COLS == 64 ? 2 : 3;                  // a load of B takes as long as two products
  static constexpr int kXBytes = L * COLS * 2, kXsBytes = 3 * COLS / 64 * BOXB + (COLS == 64 ? 0 : BOXB), kHBytes = NS * COLS * 2;
  static constexpr int kB = 0, kX = kB + kStagesB * 2 * BOXB, kXs = kX + 2 * kXBytes, kH = kXs + 2 * kXsBytes, kW = kH + 2 * kHBytes, kBars = kW + 2 * L * 4,
                       kBytes = kBars + 22 * 8;
};
static_assert(StatesSmem<64>::kBytes <= 232448 && StatesSmem<32>::kBytes <= 232448, "shared memory of a CTA");
template <int COLS>
__global__ void __launch_bounds__(32 * kStatesWarps, 1)
scan_states_kernel(const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_h, const Scan a,
                   const Plan plan, KernelStatus* status) {
  extern __shared__ __align__(1024) uint8_t smem[];                    // the tiles leave no room to align by hand
  if (tc5::smem_u32(smem) & 1023u) {                                   // the swizzle needs it; never seen otherwise
    if (threadIdx.x == 0) status_report(status, STATUS_BAD_ARGUMENT, blockIdx.x, static_cast<int>(tc5::smem_u32(smem)));
    return;
  }
  typedef StatesSmem<COLS> M;
  constexpr int kKeep = kGroup * COLS / 32, kGroups = 3 - COLS / 32;     // warps of the state; groups that scale
  float* weights = reinterpret_cast<float*>(smem + M::kW);             // of the tokens of even and odd chunks
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + M::kBars);       // two of each, for even and odd chunks
  uint64_t *full_x = bars, *xs_ready = bars + 2, *x_read = bars + 4, *done = bars + 6, *read = bars + 8, *written = bars + 10, *left = bars + 12;
  uint64_t *full_b = bars + 14, *empty_b = bars + 17;                  // of each stage of B
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 20);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = tc5::warp_index(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < 2; ++i) {
      for (uint64_t* bar : {full_x, done, left}) tc5::mbar_init(bar + i, 1);
      for (uint64_t* bar : {xs_ready, x_read}) tc5::mbar_init(bar + i, kGroup);
      for (uint64_t* bar : {read, written}) tc5::mbar_init(bar + i, kKeep);
    }
    for (int i = 0; i < M::kStagesB; ++i) { tc5::mbar_init(full_b + i, 1); tc5::mbar_init(empty_b + i, 1); }
    tc5::fence_barrier_init();
  }
  if (warp == 24) { tc5::tmem_alloc(tmem_slot, 512); tc5::tmem_relinquish(); }
  tc5::fence_before_sync();
  __syncthreads();
  tc5::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  // chunk q's phase of a pair's barrier, and of the one of its stage of B
  auto wait = [&](uint64_t* pair, int q, int code) { return tc5::mbar_wait_warp(pair + (q & 1), (q >> 1) & 1, abort_flag, status, code); };
  auto wait_b = [&](uint64_t* bar, int q, int code) { return tc5::mbar_wait_warp(bar + q % M::kStagesB, q / M::kStagesB & 1, abort_flag, status, code); };
  auto swizzled = [](int row) { return COLS == 64 ? row & 7 : row >> 1 & 3; };         // of rows of 128 and of 64 bytes
  Walk w(a, plan, PD / COLS);
  if (warp < kGroups * kGroup) {                       // x, row r, half of the columns
    constexpr int PIECES = COLS / 2 / 8;               // of 16 bytes
    const int r = threadIdx.x & 127, half = (warp >> 2) & 1;
    for (int q = 0; w.more(); ++q, w.next()) {
      const int group = q & 1;
      if (kGroups == 2 && group != warp >> 3) continue;
      uint8_t *sX = smem + M::kX + group * M::kXBytes + r * COLS * 2, *sB = smem + M::kB + (q % M::kStagesB * 2 + half) * BOXB + r * 128;
      uint8_t* sXs = smem + M::kXs + group * M::kXsBytes + r * 128;
      const int valid = w.valid();
      if (!wait(full_x, q, STATUS_TIMEOUT_SMEM_FULL)) break;
      const float ws = weights[group * L + r];
      uint4 xr[PIECES];
#pragma unroll
      for (int j = 0; j < PIECES; ++j) xr[j] = *reinterpret_cast<const uint4*>(sX + ((half * PIECES + j) ^ swizzled(r)) * 16);
      // Without the fence the arrival, and the copy that waits for it, may overtake loads that are still on their way: wrong pieces of x in one chunk of a hundred
      tc5::fence_proxy_async();
      tc5::arrive_warp(x_read + group);
      if (q > 1 && !wait(done, q - 2, STATUS_TIMEOUT_TMEM_FULL)) break;
      if (valid < L) {                                 // rows of other requests, whatever they hold, are no part of the sums
        // Behind the product before the last: until then the place of B may still wait for an earlier chunk's, and the phase before it would look like this one
        if (!wait_b(full_b, q, STATUS_TIMEOUT_SMEM_FULL)) break;
        if (r >= valid) {
#pragma unroll
          for (int j = 0; j < PIECES; ++j) xr[j] = make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int j = 0; j < 8; ++j) *reinterpret_cast<uint4*>(sB + (j << 4)) = make_uint4(0, 0, 0, 0);
        }
      }
      const float2 w2 = make_float2(ws, ws), minus = make_float2(-1.f, -1.f);
      // in three parts that add up to it, each with the upper eight of the bits that are left, side by side in tiles of 64 columns
#pragma unroll
      for (int j = 0; j < PIECES; ++j) {
        const uint32_t word[4] = {xr[j].x, xr[j].y, xr[j].z, xr[j].w};
        uint32_t part[3][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float2 v = mul2(unpack2(word[i]), w2);
#pragma unroll
          for (int m = 0; m < 3; ++m) {
            const uint32_t a0 = __float_as_uint(v.x), a1 = __float_as_uint(v.y);
            part[m][i] = __byte_perm(a0, a1, 0x7632);
            if (m < 2) v = fma2(make_float2(__uint_as_float(a0 & 0xffff0000u), __uint_as_float(a1 & 0xffff0000u)), minus, v);
          }
        }
#pragma unroll
        for (int m = 0; m < 3; ++m)
          *reinterpret_cast<uint4*>(sXs + m * COLS / 64 * BOXB + (((m * COLS % 64 / 8 + half * PIECES + j) ^ (r & 7)) << 4)) =
              make_uint4(part[m][0], part[m][1], part[m][2], part[m][3]);
      }
      tc5::fence_proxy_async();
      tc5::arrive_warp(xs_ready + group);
    }
  } else if (warp < 3 * kGroup) {                      // the state: row n, sixteen columns
    constexpr int MINE = 16, PIECES = MINE / 8;
    const int n = threadIdx.x & 127, part = (warp >> 2) & (COLS / 16 - 1);
    const uint32_t acc = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + part * MINE;
    float2 st[MINE / 2];
    const float* decay = nullptr;                      // of the next chunk, fetched one ahead: a number that is not there yet holds everything up
    float g_next = 0.f;
    for (int q = 0; w.more(); ++q, w.next()) {
      float* own = a.state + ((static_cast<long>(w.b) * a.H + w.h) * PD + w.part * COLS + part * MINE) * NS + n;
      if (w.k == 0) {
        decay = plan.records() + (static_cast<long>(w.chunk) * a.H + w.h) * kRecord + kDecay;
        g_next = __ldg(decay);
#pragma unroll
        for (int j = 0; j < MINE / 2; ++j) st[j] = w.fresh ? make_float2(0.f, 0.f) : make_float2(own[2 * j * NS], own[(2 * j + 1) * NS]);
      }
      const float g = g_next;
      decay += a.H * kRecord;
      if (!w.last()) g_next = __ldg(decay);
      uint32_t pk[MINE / 2];
#pragma unroll
      for (int j = 0; j < MINE / 2; ++j) pk[j] = tc5::pack_bf16(st[j].x, st[j].y);
      if (q > 1 && !wait(left, q - 2, STATUS_TIMEOUT_SMEM_EMPTY)) break;
      uint8_t* row = smem + M::kH + (q & 1) * M::kHBytes + n * COLS * 2;
#pragma unroll
      for (int j = 0; j < PIECES; ++j) {
        *reinterpret_cast<uint4*>(row + ((part * PIECES + j) ^ swizzled(n)) * 16) = make_uint4(pk[4 * j], pk[4 * j + 1], pk[4 * j + 2], pk[4 * j + 3]);
      }
      tc5::fence_proxy_async();
      tc5::arrive_warp(written + (q & 1));
      if (!wait(done, q, STATUS_TIMEOUT_TMEM_FULL)) break;
      tc5::fence_after_sync();
      const float2 g2 = make_float2(g, g);
#pragma unroll
      for (int j = 0; j < MINE / 2; ++j) st[j] = mul2(g2, st[j]);
      uint32_t v[2][MINE];                             // the smallest parts first
      tc5::tmem_ld_x16(acc + (q & 1) * 192 + 2 * COLS, v[0]);
      tc5::tmem_ld_x16(acc + (q & 1) * 192 + COLS, v[1]);
      tc5::tmem_ld_wait();
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int j = 0; j < MINE / 2; ++j) st[j] = add2(st[j], make_float2(__uint_as_float(v[m][2 * j]), __uint_as_float(v[m][2 * j + 1])));
      tc5::tmem_ld_x16(acc + (q & 1) * 192, v[0]);
      tc5::tmem_ld_wait();
      tc5::fence_before_sync();
      tc5::arrive_warp(read + (q & 1));
#pragma unroll
      for (int j = 0; j < MINE / 2; ++j) st[j] = add2(st[j], make_float2(__uint_as_float(v[0][2 * j]), __uint_as_float(v[0][2 * j + 1])));
      if (w.last()) {
#pragma unroll
        for (int j = 0; j < MINE / 2; ++j) own[2 * j * NS] = st[j].x, own[(2 * j + 1) * NS] = st[j].y;
      }
    }
  } else if (warp == 24) {                             // products
    constexpr uint32_t idesc = tc5::make_idesc_bf16(128, 3 * COLS, 1, 1);                // the three parts side by side: B is read once for them
    const bool lead = tc5::elect_one();                // converged warp, elected lane issues
    for (int q = 0; w.more(); ++q, w.next()) {
      const int s = q & 1;
      const uint64_t bt = tc5::desc_mnmajor(tc5::smem_u32(smem + M::kB + q % M::kStagesB * 2 * BOXB), BOXB);
      const uint64_t xs = tc5::desc_mnmajor(tc5::smem_u32(smem + M::kXs + s * M::kXsBytes), BOXB);
      if (!wait_b(full_b, q, STATUS_TIMEOUT_SMEM_FULL) || !wait(xs_ready, q, STATUS_TIMEOUT_SMEM_FULL) ||
          (q > 1 && !wait(read, q - 2, STATUS_TIMEOUT_TMEM_EMPTY)))
        break;
      tc5::fence_after_sync();
      if (lead) {
#pragma unroll
        for (int kk = 0; kk < L / 16; ++kk)
          tc5::mma_ss(tmem + s * 192, bt + static_cast<uint64_t>((kk * 2048) >> 4), xs + static_cast<uint64_t>((kk * 2048) >> 4), idesc, kk > 0 ? 1u : 0u);
        tc5::mma_commit(done + s);
        tc5::mma_commit(empty_b + q % M::kStagesB);
      }
      __syncwarp();
    }
  } else if (warp == 25) {                             // loads of x and its weights
    const bool lead = tc5::elect_one();
    bool ok = true;
    const float* from = nullptr;
    for (int q = 0; w.more(); ++q, w.next()) {
      const int s = q & 1;
      from = w.k ? from + a.H * kRecord : plan.records() + (static_cast<long>(w.chunk) * a.H + w.h) * kRecord + kWeight;
      if (q > 1 && !(ok = wait(x_read, q - 2, STATUS_TIMEOUT_SMEM_EMPTY))) break;
      if (lead) {
        tc5::mbar_expect_tx(full_x + s, M::kXBytes + L * 4);
        tc5::tma_load_2d(smem + M::kX + s * M::kXBytes, &tm_x, full_x + s, w.h * PD + w.part * COLS, w.t0());
        bulk_load(weights + s * L, from, L * 4, full_x + s);
      }
      __syncwarp();
    }
    if (!ok && lead)                                   // loads may still be in flight
      for (int i = 0; i < 2; ++i) tc5::mbar_drain(full_x + i);
    __syncwarp();
  } else if (warp == 26) {                             // loads of B, and everything into L2 a few chunks ahead
    const bool lead = tc5::elect_one();
    Walk ahead = w;
    auto prefetch = [&] {
      if (!ahead.more()) return;
      if (lead) {
        tc5::tma_prefetch_2d(&tm_x, ahead.h * PD + ahead.part * COLS, ahead.t0());
        tc5::tma_prefetch_2d(&tm_b, ahead.group, ahead.t0());
        tc5::tma_prefetch_2d(&tm_b, ahead.group + 64, ahead.t0());
      }
      ahead.next();
    };
    for (int i = 0; i < 4; ++i) prefetch();
    bool ok = true;
    for (int q = 0; w.more(); ++q, w.next()) {
      const int s = q % M::kStagesB;
      if (q >= M::kStagesB && !(ok = wait_b(empty_b, q - M::kStagesB, STATUS_TIMEOUT_SMEM_EMPTY))) break;
      if (lead) {
        tc5::mbar_expect_tx(full_b + s, 2 * BOXB);
        tc5::tma_load_2d(smem + M::kB + 2 * s * BOXB, &tm_b, full_b + s, w.group, w.t0());
        tc5::tma_load_2d(smem + M::kB + (2 * s + 1) * BOXB, &tm_b, full_b + s, w.group + 64, w.t0());
      }
      __syncwarp();
      prefetch();
    }
    if (!ok && lead)
      for (int i = 0; i < M::kStagesB; ++i) tc5::mbar_drain(full_b + i);
    __syncwarp();
  } else {                                             // states to memory
    for (int q = 0; w.more(); ++q, w.next()) {
      if (!wait(written, q, STATUS_TIMEOUT_SMEM_FULL)) break;
      if (lane == 0) {
        tc5::tma_store_2d(&tm_h, smem + M::kH + (q & 1) * M::kHBytes, w.part * COLS, ((w.chunk + w.k) * a.H + w.h) * NS);
        tc5::tma_store_commit();
        tc5::tma_store_wait_read<1>();                 // the one before has left its buffer
      }
      if (q > 0) tc5::arrive_warp(left + ((q - 1) & 1));
      __syncwarp();
    }
    if (lane == 0) tc5::tma_store_wait_read<0>();
    __syncwarp();
  }
  tc5::fence_before_sync();
  __syncthreads();
  if (warp == 24) { tc5::fence_after_sync(); tc5::tmem_dealloc(tmem, 512); }
}

// Items (chunk, head), heads fastest, in equal runs: what the heads of a group share (B, C and the scores C B^T) is loaded and computed once per run of
// one chunk and group ("segment"), and the next items' tiles are in flight meanwhile.
struct Items {
  const int2* table;
  int n, h, c, H, in_group, shared, last;  // items of the run; head and chunk of the current one; heads that share B and C, and which of them
  int2 now, then;                          // first token and number of tokens of its chunk and of the next
  __device__ Items(const Plan& plan, int H_, int G) : table(plan.table()), H(H_), shared(H_ / G), last(plan.at[1] - 1) {
    const int total = plan.at[1] * H, quota = (total + gridDim.x - 1) / gridDim.x, first = blockIdx.x * quota;
    n = max(min(quota, total - first), 0);
    h = first % H;
    c = first / H;
    in_group = h % shared;
    if (n > 0) now = table[c], then = table[min(c + 1, last)];
  }
  __device__ void next() {
    if (++in_group == shared) in_group = 0;
    if (++h < H) return;
    h = 0;
    ++c;
    now = then;
    then = table[min(c + 1, last)];
  }
  __device__ bool opens(int k) const { return k == 0 || in_group == 0; }     // first item of a segment
};

// Warps of block q of 32 rows, the ones whose index is q modulo four (a warp reaches no other rows of tensor memory): q of them compute the weights of 32
// columns each in front of the block, two those of the block itself, of even and odd items (their exponentials take twice as long), and two finish the
// block's rows.  Two of the warps that are left issue products, and load and store.  C B^T stays in registers for all heads of a segment, the weights go to
// tensor memory as the A operand, y leaves from the place of x.  Bound by memory and the handoffs of an item: one request of 16 K tokens and 64 heads
// (411 MB) 73 us, 5.6 TB/s, 13.0 K in 8 (331 MB) 62; before the sums had two numbers each 71 and 61, then with warps that weigh an item and then finish the one before 88 and 76, with three
// stages of x and H together 80, with a last chunk's rows stored one by one 75 for the eight.
constexpr int kRowsWarps = 28, kWeigh = 14, kFinish = 8, kIssue = 16, kCopy = 20;
constexpr int kStages = 4, kStagesH = 3;               // of x and the sums, which stay until an item's rows are finished; of H, which its first product reads
struct RowsSmem {
  static constexpr int kC = 0, kB = kC + 4 * BOXB, kX = kB + 2 * BOXB, kH = kX + kStages * BOXB, kSums = kH + kStagesH * BOXB,
                       kBars = kSums + kStages * kRowFloats * 4, kBytes = kBars + 24 * 8;
};
static_assert(kStages == kStagesH + 1 && RowsSmem::kBytes <= 232448, "shared memory of a CTA");
__global__ void __launch_bounds__(32 * kRowsWarps, 1)
scan_rows_kernel(const __grid_constant__ CUtensorMap tm_c, const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ CUtensorMap tm_x,
                 const __grid_constant__ CUtensorMap tm_h, const __grid_constant__ CUtensorMap tm_y, const __grid_constant__ CUtensorMap tm_y8,
                 const Scan a, const Plan plan, KernelStatus* status) {
  extern __shared__ __align__(1024) uint8_t smem[];
  if (tc5::smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) status_report(status, STATUS_BAD_ARGUMENT, blockIdx.x, static_cast<int>(tc5::smem_u32(smem)));
    return;
  }
  typedef RowsSmem M;
  uint8_t *sC = smem + M::kC, *sB = smem + M::kB, *sX = smem + M::kX, *sH = smem + M::kH;    // C of even and odd segments, B; x [128 t][64]; H [128 n][64]
  float* sums = reinterpret_cast<float*>(smem + M::kSums);             // of each stage: sums, the same less the step's size, factors of columns
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + M::kBars);
  uint64_t *full = bars, *left = bars + kStages, *full_h = left + kStages, *left_h = full_h + kStagesH, *cb = left_h + kStagesH, *ms = cb + 2, *sread = cb + 3;
  uint64_t *ready = cb + 4, *done = cb + 6;                            // even and odd items
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(cb + 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = tc5::warp_index(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < kStages; ++i) { tc5::mbar_init(full + i, 1); tc5::mbar_init(left + i, kFinish); }
    for (int i = 0; i < kStagesH; ++i) { tc5::mbar_init(full_h + i, 1); tc5::mbar_init(left_h + i, 1); }
    tc5::mbar_init(ms, 1);
    tc5::mbar_init(sread, kWeigh);
    for (int i = 0; i < 2; ++i) {
      tc5::mbar_init(cb + i, 1);
      tc5::mbar_init(ready + i, kWeigh - 4);
      tc5::mbar_init(done + i, 1);
    }
    tc5::fence_barrier_init();
  }
  if (warp == kIssue) { tc5::tmem_alloc(tmem_slot, 512); tc5::tmem_relinquish(); }
  tc5::fence_before_sync();
  __syncthreads();
  tc5::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  constexpr uint32_t cS = 0, cP = 128, cYi = 256, cYo = 384;           // the last three: 64 columns for even and odd items each
  auto wait = [&](uint64_t* bar, int phase, int code) { return tc5::mbar_wait_warp(bar, phase & 1, abort_flag, status, code); };
  Items cur(plan, a.H, a.G);
  const int n = cur.n;
  const int quad = warp & 3, place = warp >> 2, r = quad * 32 + lane;                  // block of rows, place among its warps, row
  if (place < quad + 2) {
    const bool before = place < quad;                  // columns in front of the block
    const int grp = min(place, quad), own = place - quad;                              // column block; own: even or odd items
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    float s[32];                                       // C_i . B_j of the segment: row i = r, columns j = 32 grp ..
    int seg = 0;
    for (int k = 0; k < n; ++k, cur.next()) {
      const int buf = k & 1;
      if (cur.opens(k)) {
        if (!wait(ms, seg, STATUS_TIMEOUT_TMEM_FULL)) break;
        tc5::fence_after_sync();
        tld32(lanes + cS + grp * 32, s);
        tc5::fence_before_sync();
        tc5::arrive_warp(sread);
        ++seg;
      }
      if (!before && buf != own) continue;
      if (!wait(full + k % kStages, k / kStages, STATUS_TIMEOUT_SMEM_FULL)) break;
      const float *cum = sums + k % kStages * kRowFloats + kCum, *low = cum + kCumLow - kCum, *colf = cum + kCols - kCum;
      const float ci = cum[r], ci_low = low[r];
      uint32_t pk[16];
      if (before) {                                    // every column is before every row
        const float rowf = ex2(fminf((ci - cum[32 * quad - 1]) + (ci_low - low[32 * quad - 1]), 0.f));
        const float2 r2 = make_float2(rowf, rowf);
        const float* f = colf + 16 * quad * (quad - 1) + grp * 32;
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 v = *reinterpret_cast<const float4*>(f + j);
          const float2 x = mul2(make_float2(s[j], s[j + 1]), mul2(r2, make_float2(v.x, v.y)));
          const float2 y = mul2(make_float2(s[j + 2], s[j + 3]), mul2(r2, make_float2(v.z, v.w)));
          pk[j / 2] = tc5::pack_bf16(x.x, x.y);
          pk[j / 2 + 1] = tc5::pack_bf16(y.x, y.y);
        }
      } else {
        const float2 c2 = make_float2(ci, ci), low2 = make_float2(ci_low, ci_low), minus = make_float2(-1.f, -1.f);
        const float *less = cum + kLess - kCum + grp * 32, *less_low = cum + kLessLow - kCum + grp * 32;
#pragma unroll
        for (int j = 0; j < 32; j += 2) {              // exponents are <= 0 but for the step size where they count
          const float2 x = add2(fma2(*reinterpret_cast<const float2*>(less + j), minus, c2), fma2(*reinterpret_cast<const float2*>(less_low + j), minus, low2));
          const float2 v = mul2(make_float2(s[j], s[j + 1]), make_float2(ex2(x.x), ex2(x.y)));
          pk[j / 2] = tc5::pack_bf16(j <= lane ? v.x : 0.f, j + 1 <= lane ? v.y : 0.f);
        }
        if (cur.now.y < L) {                           // rows of x of other requests, whatever they hold, are no part of the sums
          if (r >= cur.now.y) {
            uint4* row = reinterpret_cast<uint4*>(sX + k % kStages * BOXB + r * 128);
#pragma unroll
            for (int j = 0; j < 8; ++j) row[j ^ (r & 7)] = make_uint4(0, 0, 0, 0);         // neighbouring rows in different banks
          }
          tc5::fence_proxy_async();
        }
        if (k < 2) {                                   // columns behind the block, once: nobody writes there
          const uint32_t none[16] = {};
          for (int j = quad + 1; j < 4; ++j) tc5::tmem_st_x16(lanes + cP + buf * 64 + j * 16, none);
        }
      }
      if (k > 1 && !wait(done + buf, (k - 2) >> 1, STATUS_TIMEOUT_TMEM_FULL)) break;      // these columns' products
      tc5::fence_after_sync();
      tc5::tmem_st_x16(lanes + cP + buf * 64 + grp * 16, pk);
      tc5::tmem_st_wait();
      tc5::fence_before_sync();
      tc5::arrive_warp(ready + buf);
    }
  } else if (place < quad + 4) {                       // rows, whose products ran while the next item's weights were computed
    constexpr int MINE = PD * 4 / kFinish;             // columns
    const int part = place - quad - 2;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16) + part * MINE;
    for (int k = 0; k < n; ++k, cur.next()) {
      const int buf = k & 1, valid = cur.now.y;
      const uint32_t D = a.D ? raw_param(a.D, cur.h, a.D_fp32) : 0u;
      if (!wait(full + k % kStages, k / kStages, STATUS_TIMEOUT_SMEM_FULL)) break;
      const float e = ex2(sums[k % kStages * kRowFloats + kCum + r]);
      if (!wait(done + buf, k >> 1, STATUS_TIMEOUT_TMEM_FULL)) break;
      tc5::fence_after_sync();
      uint8_t* base = sX + k % kStages * BOXB + r * 128;                                   // the thread's own pieces of x, which the products have read
      const float skip = param_of(D, a.D_fp32);
      const float2 e2 = make_float2(e, e), D2 = make_float2(skip, skip);
#pragma unroll
      for (int c = 0; c < MINE; c += 16) {
        uint32_t yo[16], yi[16], xr[8], o[8];
        tc5::tmem_ld_x16(lanes + cYo + buf * 64 + c, yo);
        tc5::tmem_ld_x16(lanes + cYi + buf * 64 + c, yi);
        uint8_t* piece[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          piece[j] = base + ((((part * MINE + c) / 8 + j) ^ (r & 7)) << 4);
          const uint4 u = *reinterpret_cast<const uint4*>(piece[j]);
          xr[4 * j] = u.x, xr[4 * j + 1] = u.y, xr[4 * j + 2] = u.z, xr[4 * j + 3] = u.w;
        }
        tc5::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 in = make_float2(__uint_as_float(yi[2 * i]), __uint_as_float(yi[2 * i + 1]));
          const float2 y = fma2(D2, unpack2(xr[i]), fma2(e2, in, make_float2(__uint_as_float(yo[2 * i]), __uint_as_float(yo[2 * i + 1]))));
          o[i] = tc5::pack_bf16(y.x, y.y);
        }
        if (r < (valid & ~7)) {
#pragma unroll
          for (int j = 0; j < 2; ++j) *reinterpret_cast<uint4*>(piece[j]) = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
        } else if (r < valid) {                        // less than eight; those behind the request are another's
          uint4* to = reinterpret_cast<uint4*>(a.y + (static_cast<long>(cur.now.x + r) * a.H + cur.h) * PD + part * MINE + c);
          to[0] = make_uint4(o[0], o[1], o[2], o[3]);
          to[1] = make_uint4(o[4], o[5], o[6], o[7]);
        }
      }
      tc5::fence_proxy_async();
      tc5::fence_before_sync();
      tc5::arrive_warp(left + k % kStages);
    }
  } else if (warp == kIssue) {                         // products
    constexpr uint32_t id_s = tc5::make_idesc_bf16(128, 128, 0, 0), id_y = tc5::make_idesc_bf16(128, PD, 0, 1);
    const bool lead = tc5::elect_one();                // converged warp, elected lane issues
    uint64_t cc = 0;
    int seg = 0;
    for (int k = 0; k < n; ++k, cur.next()) {
      const int buf = k & 1;
      if (cur.opens(k)) {
        if (k > 0 && !wait(sread, seg - 1, STATUS_TIMEOUT_TMEM_EMPTY)) break;
        if (!wait(cb + (seg & 1), seg >> 1, STATUS_TIMEOUT_SMEM_FULL)) break;
        tc5::fence_after_sync();
        cc = tc5::desc_kmajor(tc5::smem_u32(sC + (seg & 1) * 2 * BOXB));
        const uint64_t bb = tc5::desc_kmajor(tc5::smem_u32(sB));
        if (lead) {
#pragma unroll
          for (int kk = 0; kk < NS / 16; ++kk) {
            const uint64_t off = static_cast<uint64_t>(((kk >> 2) * BOXB + (kk & 3) * 32) >> 4);
            tc5::mma_ss(tmem + cS, cc + off, bb + off, id_s, kk > 0 ? 1u : 0u);
          }
          tc5::mma_commit(ms);
        }
        __syncwarp();
        ++seg;
      }
      if (k > 1 && !wait(left + (k - 2) % kStages, (k - 2) / kStages, STATUS_TIMEOUT_TMEM_EMPTY)) break;      // its columns are free
      if (!wait(full_h + k % kStagesH, k / kStagesH, STATUS_TIMEOUT_SMEM_FULL)) break;
      tc5::fence_after_sync();
      const uint64_t xx = tc5::desc_mnmajor(tc5::smem_u32(sX + k % kStages * BOXB), BOXB);
      const uint64_t hh = tc5::desc_mnmajor(tc5::smem_u32(sH + k % kStagesH * BOXB), BOXB);
      if (lead) {
#pragma unroll
        for (int kk = 0; kk < NS / 16; ++kk)
          tc5::mma_ss(tmem + cYi + buf * 64, cc + static_cast<uint64_t>(((kk >> 2) * BOXB + (kk & 3) * 32) >> 4),
                      hh + static_cast<uint64_t>((kk * 2048) >> 4), id_y, kk > 0 ? 1u : 0u);
        tc5::mma_commit(left_h + k % kStagesH);
      }
      __syncwarp();
      if (!wait(full + k % kStages, k / kStages, STATUS_TIMEOUT_SMEM_FULL) || !wait(ready + buf, k >> 1, STATUS_TIMEOUT_TMEM_EMPTY)) break;
      tc5::fence_after_sync();
      if (lead) {
#pragma unroll
        for (int kk = 0; kk < L / 16; ++kk)
          tc5::mma_ts(tmem + cYo + buf * 64, tmem + cP + buf * 64 + kk * 8, xx + static_cast<uint64_t>((kk * 2048) >> 4), id_y, kk > 0 ? 1u : 0u);
        tc5::mma_commit(done + buf);
      }
      __syncwarp();
    }
  } else if (warp == kCopy) {                          // loads and stores
    const bool lead = tc5::elect_one();
    Items ahead = cur, behind = cur;                   // the next item to be loaded, the next to be stored
    auto load = [&](int k) {                           // x and sums of item k, which is `ahead`
      const int at = k % kStages;
      tc5::mbar_expect_tx(full + at, BOXB + kRowFloats * 4);
      bulk_load(sums + at * kRowFloats, plan.records() + (static_cast<long>(ahead.c) * a.H + ahead.h) * kRecord, kRowFloats * 4, full + at);
      tc5::tma_load_2d(sX + at * BOXB, &tm_x, full + at, ahead.h * PD, ahead.now.x);
    };
    auto load_h = [&](int k) {
      const int at = k % kStagesH;
      tc5::mbar_expect_tx(full_h + at, BOXB);
      tc5::tma_load_2d(sH + at * BOXB, &tm_h, full_h + at, 0, (ahead.c * a.H + ahead.h) * NS);
    };
    auto store = [&](int k) {                          // item k, which is `behind`: a whole chunk, or eight rows a lane
      const uint8_t* from = sX + k % kStages * BOXB;
      if (behind.now.y == L) {
        if (lead) tc5::tma_store_2d(&tm_y, from, behind.h * PD, behind.now.x);
      } else if (8 * lane + 8 <= behind.now.y) {
        tc5::tma_store_2d(&tm_y8, from + lane * 1024, behind.h * PD, behind.now.x + 8 * lane);
      }
      tc5::tma_store_commit();
    };
    auto load_cb = [&](int seg, int t0, int group) {   // C and B of a segment
      tc5::mbar_expect_tx(cb + (seg & 1), 4 * BOXB);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        tc5::tma_load_2d(sC + ((seg & 1) * 2 + i) * BOXB, &tm_c, cb + (seg & 1), group * NS + i * 64, t0);
        tc5::tma_load_2d(sB + i * BOXB, &tm_b, cb + (seg & 1), group * NS + i * 64, t0);
      }
    };
    bool ok = true, more = false;
    int seg = 0, next_t0 = 0, next_group = 0;          // segments opened; what the next one is of, whose loads start an item after the last one opened
    if (n > 0 && lead) load_cb(0, cur.now.x, cur.h / cur.shared);
    __syncwarp();
    for (int k = 0; k < n; ++k, cur.next()) {
      if (more) {                                      // over the B that the scores were made of, and the C of the segment before, whose rows have left
        if (!(ok = wait(ms, seg - 1, STATUS_TIMEOUT_TMEM_FULL))) break;
        if (lead) load_cb(seg, next_t0, next_group);
        more = false;
        __syncwarp();
      }
      if (cur.opens(k)) {
        const int on = cur.shared - cur.in_group;
        const bool same = cur.h + on < cur.H;
        more = k + on < n;
        next_t0 = same ? cur.now.x : cur.then.x;
        next_group = same ? cur.h / cur.shared + 1 : 0;
        ++seg;
      }
      if (k == 0)
        for (int i = 0; i < kStagesH && i < n; ++i, ahead.next())
          if (lead) load(i), load_h(i);
      const bool next = k + kStagesH < n;
      if (!(ok = wait(left_h + k % kStagesH, k / kStagesH, STATUS_TIMEOUT_SMEM_EMPTY))) break;
      if (lead && next) load_h(k + kStagesH);
      if (k > 0) {
        if (!(ok = wait(left + (k - 1) % kStages, (k - 1) / kStages, STATUS_TIMEOUT_TMEM_EMPTY))) break;
        store(k - 1);
        behind.next();
      }
      if (next) {                                      // over the stage of item k - 1
        tc5::tma_store_wait_read<0>();
        __syncwarp();
        if (lead) load(k + kStagesH);
      }
      ahead.next();
      __syncwarp();
    }
    if (n > 0) {
      if (ok && wait(left + (n - 1) % kStages, (n - 1) / kStages, STATUS_TIMEOUT_TMEM_EMPTY)) {
        store(n - 1);
      } else if (lead) {                               // loads may still be in flight
        for (int i = 0; i < kStages; ++i) tc5::mbar_drain(full + i);
        for (int i = 0; i < kStagesH; ++i) tc5::mbar_drain(full_h + i);
        for (int i = 0; i < 2; ++i) tc5::mbar_drain(cb + i);
      }
    }
    tc5::tma_store_wait_read<0>();
    __syncwarp();
  }
  tc5::fence_before_sync();
  __syncthreads();
  if (warp == kIssue) { tc5::fence_after_sync(); tc5::tmem_dealloc(tmem, 512); }
}

template <int S>
int tokens(const Scan& a, int longest, const Plan& plan, cudaStream_t st) {
  const int parts = (a.P + Tile<S>::ROWS - 1) / Tile<S>::ROWS;
  const long blocks = static_cast<long>(a.B) * a.H * parts + (plan.at ? 1 + static_cast<long>(plan.chunks) * ((a.H + 7) / 8) : 0);
  if (blocks > 0x7fffffffl) return nsa::fail(NSA_ERR_SHAPE, "ssd_scan_cached: too many requests and heads");
  scan_tokens_kernel<S><<<static_cast<unsigned>(blocks), 256, 0, st>>>(a, parts, longest, plan);
  nsa::count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : nsa::fail_cuda(e, "nsa_ssd_scan_cached launch");
}

// Requests of more new tokens than this go through the products, which read and write the states in front of chunks too but take 128 tokens about as fast as
// one.  It is where both are alike for many requests, whose steps take longest; one request of 17 to 28 tokens loses up to 7 us by it, 8 of 17 to 23 up to 15.
// 64 heads, requests of 8 / 16 / 24 / 32 / 64 tokens, token by token: one request 7.6 / 11.7 / 15.8 / 20.0 / 36.4 us, 8 requests 14.8 / 24.9 / 34.9 / 44.9 /
// 86.7, 64 requests 98 / 161 / 226 / 290 / 547; by the products 19 / 19 / 18 / 18 / 17, 41 / 38 / 35 / 34 / 32 and 161 / 156 / 155 / 152 / 144.
constexpr int kLongest = 16;

Plan plan_of(int B, int N, int P, int S, int max_new) {
  const int room = N / (kLongest + 1) < B ? N / (kLongest + 1) : B;
  return S == NS && P == PD && max_new > kLongest ? Plan{nullptr, room, N / kChunk + room} : Plan{};
}

template <int COLS>
int launch_states(const CUtensorMap& tb, const Scan& a, const Plan& plan, void* states, cudaStream_t st) {
  CUtensorMap th, tx;
  const uint64_t dims[2] = {PD, static_cast<uint64_t>(plan.chunks) * a.H * NS}, strides[1] = {PD * 2};
  const uint64_t dims_x[2] = {static_cast<uint64_t>(a.H) * PD, static_cast<uint64_t>(a.N)}, strides_x[1] = {static_cast<uint64_t>(a.ldx) * 2};
  const uint32_t box[2] = {COLS, NS}, box_x[2] = {COLS, L};
  if (const int rc = nsa::make_tmap_bf16(&th, states, 2, dims, strides, box, COLS * 2)) return rc;
  if (const int rc = nsa::make_tmap_bf16(&tx, a.x, 2, dims_x, strides_x, box_x, COLS * 2)) return rc;
  const cudaError_t e = cudaFuncSetAttribute(scan_states_kernel<COLS>, cudaFuncAttributeMaxDynamicSharedMemorySize, StatesSmem<COLS>::kBytes);
  if (e != cudaSuccess) return nsa::fail_cuda(e, "ssd_scan_cached: shared memory attribute");
  const long sms = nsa::sm_count(), walks = static_cast<long>(plan.room) * a.H * (PD / COLS);
  scan_states_kernel<COLS><<<static_cast<unsigned>(walks < sms ? walks : sms), 32 * kStatesWarps, StatesSmem<COLS>::kBytes, st>>>(tb, tx, th, a, plan, nsa::status_ptr());
  return 0;
}

int prompts(const Scan& a, const Plan& plan, int max_new, cudaStream_t st) {
  void* states = plan.records() + static_cast<long>(plan.chunks) * a.H * kRecord;
  CUtensorMap tc, tb, tx, ty, ty8, th;
  int rc;
  const uint64_t cols = static_cast<uint64_t>(a.H) * PD;
  if ((rc = nsa::make_tmap_2d_bf16(&tc, a.Cm, static_cast<uint64_t>(a.G) * NS, a.N, a.ldc, 64, L))) return rc;
  if ((rc = nsa::make_tmap_2d_bf16(&tb, a.Bm, static_cast<uint64_t>(a.G) * NS, a.N, a.ldb, 64, L))) return rc;
  if ((rc = nsa::make_tmap_2d_bf16(&tx, a.x, cols, a.N, a.ldx, 64, L))) return rc;
  if ((rc = nsa::make_tmap_2d_bf16(&ty, a.y, cols, a.N, cols, 64, L))) return rc;
  if ((rc = nsa::make_tmap_2d_bf16(&ty8, a.y, cols, a.N, cols, 64, 8))) return rc;
  if ((rc = nsa::make_tmap_2d_bf16(&th, states, PD, static_cast<uint64_t>(plan.chunks) * a.H * NS, PD, 64, NS))) return rc;
  const cudaError_t attr = cudaFuncSetAttribute(scan_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RowsSmem::kBytes);
  if (attr != cudaSuccess) return nsa::fail_cuda(attr, "ssd_scan_cached: shared memory attribute");
  const long sms = nsa::sm_count(), items = static_cast<long>(plan.chunks) * a.H;
  // Half of a head's columns a CTA as long as the heads of the fewest requests that there can be leave SMs for it: the whole call with halves / all 64, 16 K
  // tokens of 64 heads 175 / 212 us, three times 8 K of 24 heads 101 / 120; above, two times 8 K of 64 heads 177 / 154, 8 K of 128 heads 176 / 154
  const long least = (a.N + max_new - 1) / max_new;
  rc = 2 * least * a.H <= sms ? launch_states<32>(tb, a, plan, states, st) : launch_states<64>(tb, a, plan, states, st);
  if (rc) return rc;
  scan_rows_kernel<<<static_cast<unsigned>(items < sms ? items : sms), 32 * kRowsWarps, RowsSmem::kBytes, st>>>(tc, tb, tx, th, ty, ty8, a, plan, nsa::status_ptr());
  nsa::count_launch(2);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : nsa::fail_cuda(e, "nsa_ssd_scan_cached launch");
}
}  // namespace

// Scratch of a call in bytes, 0: none
extern "C" long nsa_ssd_scan_cached_scratch(int B, int N, int H, int P, int S, int max_new) {
  const Plan plan = plan_of(B, N, P, S, max_new);
  return plan.room ? plan.words() * 4 + static_cast<long>(plan.chunks) * H * (kRecord * 4 + NS * PD * 2) : 0;
}

// x (N, H, P), dt (N, H), Bm and Cm (N, G, S) bf16 with the given pitches of tokens, 16-byte aligned rows in all but dt; A_log, bias, D (H; D or null) bf16 or
// fp32; state (B, H, P, S) fp32; y (N, H, P) dense; scratch: nsa_ssd_scan_cached_scratch(...) bytes at a 128-byte place, or null where it is 0.
extern "C" int nsa_ssd_scan_cached(const void* x, long ldx, const void* dt, long ldt, const void* Bm, long ldb, const void* Cm, long ldc, const void* A_log,
                                   int A_fp32, const void* bias, int bias_fp32, const void* D, int D_fp32, float* state, void* y, const int* query_start,
                                   const int* lengths, void* scratch, int B, int N, int H, int P, int G, int S, int max_new, cudaStream_t st) {
  if (N == 0) return 0;
  if (B <= 0 || N < 0 || H <= 0 || P <= 0 || G <= 0 || H % G || P % 8) return nsa::fail(NSA_ERR_SHAPE, "ssd_scan_cached: unsupported shape");
  if ((ldx | ldb | ldc) & 7) return nsa::fail(NSA_ERR_ALIGNMENT, "ssd_scan_cached: token pitches must be multiples of 8 elements");
  const Scan a{static_cast<const bf16*>(x), static_cast<const bf16*>(dt), static_cast<const bf16*>(Bm), static_cast<const bf16*>(Cm), ldx, ldt, ldb, ldc,
               A_log, bias, D, A_fp32, bias_fp32, D_fp32, state, static_cast<bf16*>(y), query_start, lengths, B, N, H, P, G};
  Plan plan = plan_of(B, N, P, S, max_new);
  const bool both = plan.room > 0;
  if (both && (scratch == nullptr || reinterpret_cast<uintptr_t>(scratch) % 128)) return nsa::fail(NSA_ERR_ALIGNMENT, "ssd_scan_cached: scratch is missing or unaligned");
  if (both && static_cast<long>(plan.chunks) * H > 0x7fffffffl / NS) return nsa::fail(NSA_ERR_SHAPE, "ssd_scan_cached: too many chunks and heads");
  if (both) plan.at = static_cast<int*>(scratch);
  const int longest = both ? kLongest : N;
  int rc = NSA_ERR_SHAPE;
  switch (S) {
    case 16: rc = tokens<16>(a, longest, plan, st); break;
    case 32: rc = tokens<32>(a, longest, plan, st); break;
    case 64: rc = tokens<64>(a, longest, plan, st); break;
    case 128: rc = tokens<128>(a, longest, plan, st); break;
    case 256: rc = tokens<256>(a, longest, plan, st); break;
    default: return nsa::fail(NSA_ERR_SHAPE, "ssd_scan_cached: 16, 32, 64, 128 or 256 states");
  }
  return rc || !both ? rc : prompts(a, plan, max_new, st);
}
