// Eviction from the 16-bit cache: per (row, kv head) the tokens with the largest accumulated attention weight stay.
#include "k16_kernels.h"

namespace k16 {
namespace {

constexpr int NT = 256;

// order-preserving key of a weight: a > b as floats iff key(a) > key(b); -0 equals +0, NaN is below everything
FR_DEVI uint32_t key_of(float w) {
  if (isnan(w)) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);        // -0 + 0 = +0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
FR_DEVI int block_sum(int v, int* red) {
  for (int x = 16; x; x >>= 1) v += __shfl_xor_sync(~0u, v, x);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  int s = 0;
  for (int i = 0; i < NT / 32; ++i) s += red[i];
  return s;
}

// CTA per (row, kv head): the threshold key by 32 rounds of bisection on its bits, the kept positions by a scan over
// the row in order, then the rows in order (in place a step's reads end before its writes begin; a kept row only moves down).
__global__ void __launch_bounds__(NT) k_evict(EvictArgs a) {
  __shared__ int red[NT / 32], s_base, s_ties;
  const int b = blockIdx.x / a.c.Hkv, h = blockIdx.x % a.c.Hkv, tid = threadIdx.x;
  const int len = min(a.c.len(b), a.w_len), m = min(len, a.budget);
  const float* w = a.weights + b * a.w_bs + h * a.w_hs;
  int* kept = a.kept + (static_cast<long long>(b) * a.c.Hkv + h) * a.budget;
  float* nw = a.new_weights + (static_cast<long long>(b) * a.c.Hkv + h) * a.nw_len;
  if (h == 0 && tid == 0) a.new_lens[b] = m;
  if (len <= a.budget) {
    for (int i = tid; i < len; i += NT) kept[i] = i, nw[i] = w[i];
  } else {
    const int lo = a.sinks, hi = len - a.recent, want = a.budget - a.sinks - a.recent;
    uint32_t T = 0;                                     // the want-th largest key
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t c = T | (1u << bit);
      int n = 0;
      for (int i = lo + tid; i < hi; i += NT) n += key_of(w[i]) >= c;
      if (block_sum(n, red) >= want && want > 0) T = c;
    }
    int n = 0;
    for (int i = lo + tid; i < hi; i += NT) n += key_of(w[i]) > T;
    const int above = block_sum(n, red);
    if (tid == 0) s_base = 0, s_ties = want - above;    // ties still to take, lowest position first
    __syncthreads();
    for (int i0 = 0; i0 < len; i0 += NT) {
      const int i = i0 + tid;
      const bool forced = i < len && (i < lo || i >= hi);
      const uint32_t k = i < len ? key_of(w[i]) : 0u;
      const bool tie = i < len && !forced && want > 0 && k == T;
      bool take = forced || (i < len && !forced && want > 0 && k > T);
      // exclusive scans over the CTA: ties first, then what is taken
      __shared__ int wt[NT / 32], wk[NT / 32];
      const unsigned mt = __ballot_sync(~0u, tie), below = (1u << (tid & 31)) - 1;
      if ((tid & 31) == 0) wt[tid >> 5] = __popc(mt);
      __syncthreads();
      int tb = __popc(mt & below), tt = 0;
      for (int x = 0; x < NT / 32; ++x) tt += wt[x], tb += x < (tid >> 5) ? wt[x] : 0;
      take = take || (tie && tb < s_ties);
      const unsigned mk = __ballot_sync(~0u, take);
      if ((tid & 31) == 0) wk[tid >> 5] = __popc(mk);
      __syncthreads();
      int kb = __popc(mk & below), kt = 0;
      for (int x = 0; x < NT / 32; ++x) kt += wk[x], kb += x < (tid >> 5) ? wk[x] : 0;
      if (take) kept[s_base + kb] = i, nw[s_base + kb] = w[i];
      __syncthreads();
      if (tid == 0) s_base += kt, s_ties -= min(s_ties, tt);
      __syncthreads();
    }
  }
  for (int i = m + tid; i < a.budget; i += NT) kept[i] = -1;
  for (int i = m + tid; i < a.nw_len; i += NT) nw[i] = 0.f;
  if (len <= a.budget && !a.dst_bt) return;
  __threadfence_block();
  __syncthreads();
  // rows: 16-byte pieces, NT at a time; a step covers whole tokens (D / 4 pieces: key row, then value row)
  const int ppt = a.D >> 2, tps = NT / ppt;
  for (int r0 = 0; r0 < m; r0 += tps) {
    const int r = r0 + tid / ppt, piece = tid % ppt, kv = piece >= ppt / 2, e = (piece - kv * (ppt / 2)) * 8;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (r < m) {
      const int src = kept[r], pg = a.c.page_of(b, src);
      if (pg >= 0) x = *reinterpret_cast<const uint4*>(a.c.pool + row_at(pg, a.c.Hkv, h, kv, a.c.page_sh, src & (a.c.page() - 1), a.D) + e);
    }
    __syncthreads();
    if (r < m) {
      const int pg = a.dst_bt ? a.dst_bt[b * a.dst_stride + (r >> a.c.page_sh)] : a.c.page_of(b, r);
      if (pg >= 0 && pg < a.dst_pages)
        *reinterpret_cast<uint4*>(a.dst + row_at(pg, a.c.Hkv, h, kv, a.c.page_sh, r & (a.c.page() - 1), a.D) + e) = x;
    }
    __syncthreads();
  }
}

}  // namespace

cudaError_t evict(const EvictArgs& a, cudaStream_t st) {
  k_evict<<<a.B * a.c.Hkv, NT, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace k16
