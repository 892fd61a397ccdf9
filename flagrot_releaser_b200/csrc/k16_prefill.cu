// Attention of many new tokens over the 16-bit cache: causal, with an optional sliding window and sink tokens.
#include "k16_kernels.h"

namespace k16 {
namespace {

// One warp per (token, q head); a lane holds D / 32 dims; running maximum and sum.
template <int DT, int D>
__global__ void __launch_bounds__(128) k_prefill(PrefillArgs a) {
  constexpr int N = D / 64;
  const int Hq = a.c.Hkv * a.G, lane = threadIdx.x & 31;
  const long long item = blockIdx.x * 4ll + (threadIdx.x >> 5);
  const int t = static_cast<int>(item / Hq), hq = static_cast<int>(item % Hq), h = hq / a.G;
  if (t >= a.T) return;
  // the sequence of token t: the last row that begins at or before it
  int b0 = 0, b1 = a.B;              // cu_q[b0] <= t < cu_q[b1] when t belongs to any
  while (b1 - b0 > 1) {
    const int mid = (b0 + b1) >> 1;
    if (a.cu_q[mid] <= t) b0 = mid; else b1 = mid;
  }
  const int beg = a.cu_q[b0], end = a.cu_q[b0 + 1];
  if (t < beg || t >= end) return;
  const int len = a.c.len(b0), pos = len - end + t;
  const Span sp(pos, a.window, a.sinks);
  const uint32_t* qr = reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(a.q) + t * a.q_ts + hq * D) + lane * N;
  float2 q[N], o[N];
  for (int i = 0; i < N; ++i) {
    q[i] = Elem<DT>::f2(qr[i]);
    o[i] = make_float2(0.f, 0.f);
  }
  float m = -INFINITY, l = 0.f;
  const int nvis = pos < 0 ? 0 : sp.s1 + pos + 1 - sp.lo;
  for (int i = 0; i < nvis; ++i) {
    const int j = i < sp.s1 ? i : i - sp.s1 + sp.lo;
    const int pg = a.c.page_of(b0, j), off = j & (a.c.page() - 1);
    const uint32_t* kr = reinterpret_cast<const uint32_t*>(a.c.pool + row_at(pg, a.c.Hkv, h, 0, a.c.page_sh, off, D)) + lane * N;
    const uint32_t* vr = reinterpret_cast<const uint32_t*>(a.c.pool + row_at(pg, a.c.Hkv, h, 1, a.c.page_sh, off, D)) + lane * N;
    float s = 0.f;
    for (int e = 0; e < N; ++e) {
      const float2 k = pg >= 0 ? Elem<DT>::f2(kr[e]) : make_float2(0.f, 0.f);
      s = fmaf(q[e].x, k.x, fmaf(q[e].y, k.y, s));
    }
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(~0u, s, x);
    s *= a.qscale;
    const float mn = fmaxf(m, s), c = ex2(m - mn), p = ex2(s - mn);
    m = mn;
    l = fmaf(l, c, p);
    for (int e = 0; e < N; ++e) {
      const float2 v = pg >= 0 ? Elem<DT>::f2(vr[e]) : make_float2(0.f, 0.f);
      o[e].x = fmaf(p, v.x, o[e].x * c);
      o[e].y = fmaf(p, v.y, o[e].y * c);
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  uint32_t* out = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + t * a.o_ts + hq * D) + lane * N;
  for (int e = 0; e < N; ++e) out[e] = Elem<DT>::pack(o[e].x * inv, o[e].y * inv);
}

}  // namespace

long long prefill_ws_bytes(int, int, int, int, long long) { return 0; }
long long prefill_tickets(int, int, int, long long) { return 0; }

cudaError_t prefill(int dtype, const PrefillArgs& a, cudaStream_t st) {
  const long long n = static_cast<long long>(a.T) * a.c.Hkv * a.G;
  const unsigned grid = static_cast<unsigned>((n + 3) / 4);
  if (dtype == 0) {
    if (a.D == 128) k_prefill<0, 128><<<grid, 128, 0, st>>>(a);
    else k_prefill<0, 64><<<grid, 128, 0, st>>>(a);
  } else {
    if (a.D == 128) k_prefill<1, 128><<<grid, 128, 0, st>>>(a);
    else k_prefill<1, 64><<<grid, 128, 0, st>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace k16
