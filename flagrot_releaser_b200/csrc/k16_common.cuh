// Shared device helpers of the 16-bit paged key-value cache (libflagrot_kv16.so): the pool's addressing, 16-bit element
// traits and the visibility rule of the attention kernels.
//
// Pool [num_pages, Hkv, 2, page, D]: the rows of one (page, kv head) are contiguous, keys first.  A row of D elements is
// 128 or 256 bytes, so every row is a whole number of 128-byte lines.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#ifndef FR_DEVI
#define FR_DEVI __device__ __forceinline__
#endif

namespace k16 {

// what every kernel that reads pages through a block table needs to know about the cache
struct Cache {
  const uint16_t* pool;
  long long num_pages;
  const int* bt;
  long long bt_stride;
  int bt_width;
  const int* seq_lens;
  int Hkv, page_sh;                 // page = 1 << page_sh
  FR_DEVI int page() const { return 1 << page_sh; }
  FR_DEVI int len(int b) const { return min(max(seq_lens[b], 0), bt_width << page_sh); }
  // pool page of position j of row b, or -1
  FR_DEVI int page_of(int b, int j) const {
    const int pg = bt[b * bt_stride + (j >> page_sh)];
    return pg >= 0 && pg < num_pages ? pg : -1;
  }
};

// first element of row `off` of (page pg, head h, kv 0 key | 1 value)
FR_DEVI long long row_at(long long pg, int Hkv, int h, int kv, int page_sh, int off, int D) {
  return ((((pg * Hkv + h) * 2 + kv) << page_sh) + off) * D;
}

// visible keys of a query at position pos (pos + 1 keys up to itself): [0, s1) and [lo, pos + 1)
struct Span {
  int s1, lo;
  FR_DEVI Span(int pos, int window, int sinks) {
    lo = window > 0 ? max(pos + 1 - window, 0) : 0;
    s1 = min(sinks, lo);
  }
};

template <int DT> struct Elem;      // 0 bf16, 1 fp16
template <> struct Elem<0> {
  FR_DEVI static float2 f2(uint32_t w) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w)); }
  FR_DEVI static uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&r);
  }
};
template <> struct Elem<1> {
  FR_DEVI static float2 f2(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
  FR_DEVI static uint32_t pack(float lo, float hi) {
    const __half2 r = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&r);
  }
};

FR_DEVI float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace k16
