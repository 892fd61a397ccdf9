// Row writer of the 16-bit cache: a copy of 16-byte pieces from the projection's output to the pages.  HBM bound (every byte is
// read once and written once: 65536 rows of 8 heads x 128 dims in 83 us, 0.99 of the measured copy rate); a decode step's few
// rows are bound by the launch (64 rows: 1.5 us on the device).
#include "k16_kernels.h"
#include "k16_launch.cuh"

namespace k16 {
namespace {

// A CTA copies PER * CT consecutive pieces (piece = token, row, 16 bytes of it), PER of them in flight per thread.
constexpr int CT = 256;
template <int PER>
__global__ void __launch_bounds__(CT) k_write(const uint16_t* kv, long long kv_ts, long long kv_hs,
                                              const long long* slots, int T, int Hkv, int D, int page_sh, long long nslots,
                                              uint16_t* pool) {
  const int psh = D == 128 ? 4 : 3, ppt = 2 * Hkv << psh;      // pieces per row (log2), per token
  const long long first = static_cast<long long>(blockIdx.x) * (PER * CT);
  const int tok0 = static_cast<int>(first / ppt);
  const unsigned rem = static_cast<unsigned>(first - static_cast<long long>(tok0) * ppt) + threadIdx.x;
  uint4 x[PER];
  uint16_t* to[PER];
  let_next_start();
  after_previous();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const unsigned p = rem + i * CT, dt = p / ppt, r = p - dt * ppt;
    const int t = tok0 + static_cast<int>(dt), row = static_cast<int>(r >> psh), piece = static_cast<int>(r & ((1 << psh) - 1));
    to[i] = nullptr;
    if (t >= T) continue;
    const long long s = slots[t];
    if (s < 0 || s >= nslots) continue;
    const int h = row < Hkv ? row : row - Hkv;
    to[i] = pool + row_at(s >> page_sh, Hkv, h, row >= Hkv, page_sh, static_cast<int>(s & ((1 << page_sh) - 1)), D) + piece * 8;
    x[i] = __ldcs(reinterpret_cast<const uint4*>(kv + t * kv_ts + row * kv_hs + piece * 8));
  }
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (to[i]) *reinterpret_cast<uint4*>(to[i]) = x[i];
}

}  // namespace

cudaError_t write_rows(const uint16_t* kv, long long kv_ts, long long kv_hs, const long long* slots, int T, int Hkv, int D,
                       int page_sh, long long num_pages, uint16_t* pool, cudaStream_t st) {
  const long long n = static_cast<long long>(T) * 2 * Hkv * (D >> 3), nslots = num_pages << page_sh;
  const int per = n > 148ll * 8 * 4 * CT ? 4 : 1;   // more than four pieces for every thread the SMs hold: four in flight
                                                      // (65536 rows: 83 us, 111 one by one; 64 rows: the same)
  return launch(per == 4 ? k_write<4> : k_write<1>, static_cast<unsigned>((n + per * CT - 1) / (per * CT)), CT, 0, 0, st, kv, kv_ts, kv_hs,
                slots, T, Hkv, D, page_sh, nslots, pool);
}

}  // namespace k16
