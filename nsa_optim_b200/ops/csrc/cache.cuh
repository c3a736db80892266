// The paged 8-bit key / value cache as its kernels see it (the layout is described in ops/cache.py): a page-head holds P tokens of one KV head,
// P * D bytes of keys and as many of values; codes are offset by 128, scales are powers of two, one for keys and one for values.
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

struct CachePages {
  uint8_t* k;       // (pages, H, P/2, D/64, 2, 64)
  uint8_t* v;       // (pages, H, P/16, D, 16)
  float* scale;     // (pages, H, 2)
  int pages, H, D, shift;   // P = 1 << shift
};

struct CacheStep {
  const int* table;         // (B, W)
  const int* query_start;   // (B + 1)
  const int* lengths;       // (B)
  int B, W, N;
};

#ifdef __CUDACC__
// Byte of token t, column d in a page-head's keys and in its values
__device__ __forceinline__ int key_at(int t, int d, int D) { return (t >> 1) * 2 * D + (d >> 6) * 128 + (t & 1) * 64 + (d & 63); }
__device__ __forceinline__ int value_at(int t, int d, int D) { return (t >> 4) * 16 * D + d * 16 + (t & 15); }

// Page that holds a position of request b, -1 where there is none
__device__ __forceinline__ int page_of(const CacheStep& s, const CachePages& c, int b, long pos) {
  const long j = pos >> c.shift;
  if (pos < 0 || j >= s.W) return -1;
  const int page = s.table[static_cast<long>(b) * s.W + j];
  return page < c.pages ? page : -1;
}
#endif
