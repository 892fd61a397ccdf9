// Decode attention over the 16-bit cache: one new token per row.
#include "k16_kernels.h"

namespace k16 {
namespace {

// One CTA of four warps per (row, q head): warp w takes visible keys w, w + 4, ...; a lane holds D / 32 dims.  Running maximum
// and sum per warp, joined through shared memory.
template <int DT, int D>
__global__ void __launch_bounds__(128) k_decode(AttnArgs a, float* scores, float* lse) {
  constexpr int N = D / 64;          // 32-bit words (pairs of dims) per lane
  const int Hq = a.c.Hkv * a.G, b = blockIdx.x / Hq, hq = blockIdx.x % Hq, h = hq / a.G;
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int len = a.c.len(b);
  const Span sp(len - 1, a.window, a.sinks);
  const uint32_t* qr = reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(a.q) + b * a.q_bs + hq * D) + lane * N;
  float2 q[N], o[N];
  for (int i = 0; i < N; ++i) {
    q[i] = Elem<DT>::f2(qr[i]);
    o[i] = make_float2(0.f, 0.f);
  }
  const long long max_len = static_cast<long long>(a.c.bt_width) << a.c.page_sh;
  float m = -INFINITY, l = 0.f;
  const int nvis = sp.s1 + len - sp.lo;
  for (int i = w; i < nvis; i += 4) {
    const int j = i < sp.s1 ? i : i - sp.s1 + sp.lo;
    const int pg = a.c.page_of(b, j), off = j & (a.c.page() - 1);
    float s = 0.f;
    const uint32_t* kr = reinterpret_cast<const uint32_t*>(a.c.pool + row_at(pg, a.c.Hkv, h, 0, a.c.page_sh, off, D)) + lane * N;
    const uint32_t* vr = reinterpret_cast<const uint32_t*>(a.c.pool + row_at(pg, a.c.Hkv, h, 1, a.c.page_sh, off, D)) + lane * N;
    for (int e = 0; e < N; ++e) {
      const float2 k = pg >= 0 ? Elem<DT>::f2(kr[e]) : make_float2(0.f, 0.f);
      s = fmaf(q[e].x, k.x, fmaf(q[e].y, k.y, s));
    }
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(~0u, s, x);
    s *= a.qscale;
    if (scores && lane == 0) scores[(static_cast<long long>(b) * Hq + hq) * max_len + j] = s;
    const float mn = fmaxf(m, s), c = ex2(m - mn), p = ex2(s - mn);
    m = mn;
    l = fmaf(l, c, p);
    for (int e = 0; e < N; ++e) {
      const float2 v = pg >= 0 ? Elem<DT>::f2(vr[e]) : make_float2(0.f, 0.f);
      o[e].x = fmaf(p, v.x, o[e].x * c);
      o[e].y = fmaf(p, v.y, o[e].y * c);
    }
  }
  __shared__ float sm[4], sl[4], so[4][D];
  if (lane == 0) sm[w] = m, sl[w] = l;
  for (int e = 0; e < N; ++e) so[w][(lane * N + e) * 2] = o[e].x, so[w][(lane * N + e) * 2 + 1] = o[e].y;
  __syncthreads();
  const float M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float f[4], L = 0.f;
  for (int i = 0; i < 4; ++i) {
    f[i] = sl[i] > 0.f ? ex2(sm[i] - M) : 0.f;
    L += sl[i] * f[i];
  }
  const float inv = L > 0.f ? 1.f / L : 0.f;
  if (threadIdx.x < D / 2) {
    const int d = 2 * threadIdx.x;
    float x = 0.f, y = 0.f;
    for (int i = 0; i < 4; ++i) x = fmaf(f[i], so[i][d], x), y = fmaf(f[i], so[i][d + 1], y);
    reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + b * a.o_bs + hq * D)[threadIdx.x] = Elem<DT>::pack(x * inv, y * inv);
  }
  if (lse && threadIdx.x == 0) lse[b * Hq + hq] = M + log2f(L);
}

// weights[b, h, j] += sum over the head group of 2^(score - lse)
__global__ void __launch_bounds__(256) k_weights(AttnArgs a, const float* scores, const float* lse) {
  const int b = blockIdx.y / a.c.Hkv, h = blockIdx.y % a.c.Hkv, Hq = a.c.Hkv * a.G;
  const int len = a.c.len(b), j = blockIdx.x * 256 + threadIdx.x;
  const Span sp(len - 1, a.window, a.sinks);
  if (j >= len || (j >= sp.s1 && j < sp.lo)) return;
  const long long max_len = static_cast<long long>(a.c.bt_width) << a.c.page_sh;
  float w = 0.f;
  for (int g = 0; g < a.G; ++g) {
    const long long r = static_cast<long long>(b) * Hq + h * a.G + g;
    w += ex2(scores[r * max_len + j] - lse[r]);
  }
  a.weights[b * a.w_bs + h * a.w_hs + j] += w;
}

}  // namespace

long long attn_ws_bytes(int rows, int Hkv, int G, int D, long long max_len, int weights) {
  return 256 + (weights ? static_cast<long long>(rows) * Hkv * G * (max_len + 1) * 4 : 0);
}

cudaError_t attn(int dtype, const AttnArgs& a, cudaStream_t st) {
  const long long R = static_cast<long long>(a.B) * a.c.Hkv * a.G;
  float* lse = a.weights ? reinterpret_cast<float*>(a.ws) : nullptr;
  float* scores = a.weights ? lse + R : nullptr;
  const unsigned grid = static_cast<unsigned>(R);
  if (dtype == 0) {
    if (a.D == 128) k_decode<0, 128><<<grid, 128, 0, st>>>(a, scores, lse);
    else k_decode<0, 64><<<grid, 128, 0, st>>>(a, scores, lse);
  } else {
    if (a.D == 128) k_decode<1, 128><<<grid, 128, 0, st>>>(a, scores, lse);
    else k_decode<1, 64><<<grid, 128, 0, st>>>(a, scores, lse);
  }
  if (a.weights && a.c.bt_width > 0) {
    const unsigned nb = static_cast<unsigned>((((static_cast<long long>(a.c.bt_width) << a.c.page_sh)) + 255) / 256);
    k_weights<<<dim3(nb, a.B * a.c.Hkv), 256, 0, st>>>(a, scores, lse);
  }
  return cudaGetLastError();
}

}  // namespace k16
