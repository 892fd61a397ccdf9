// Row writer of the 16-bit cache: a copy of 16-byte pieces from the projection's output to the pages.
#include "k16_kernels.h"

namespace k16 {
namespace {

// One thread per 16-byte piece.
__global__ void k_write(const uint16_t* __restrict__ kv, long long kv_ts, long long kv_hs, const long long* __restrict__ slots, int T,
                        int Hkv, int D, int page_sh, long long nslots, uint16_t* __restrict__ pool) {
  const int ppr = D >> 3, ppt = 2 * Hkv * ppr;          // pieces per row, per token
  const long long i = blockIdx.x * 256ll + threadIdx.x;
  const long long t = i / ppt;
  if (t >= T) return;
  const int r = static_cast<int>(i - t * ppt), row = r / ppr, piece = r - row * ppr;
  const long long s = slots[t];
  if (s < 0 || s >= nslots) return;
  const int h = row < Hkv ? row : row - Hkv;
  const uint4 x = *reinterpret_cast<const uint4*>(kv + t * kv_ts + row * kv_hs + piece * 8);
  *reinterpret_cast<uint4*>(pool + row_at(s >> page_sh, Hkv, h, row >= Hkv, page_sh, static_cast<int>(s & ((1 << page_sh) - 1)), D) +
                            piece * 8) = x;
}

}  // namespace

cudaError_t write_rows(const uint16_t* kv, long long kv_ts, long long kv_hs, const long long* slots, int T, int Hkv, int D,
                       int page_sh, long long num_pages, uint16_t* pool, cudaStream_t st) {
  const long long n = static_cast<long long>(T) * 2 * Hkv * (D >> 3);
  k_write<<<static_cast<unsigned>((n + 255) / 256), 256, 0, st>>>(kv, kv_ts, kv_hs, slots, T, Hkv, D, page_sh, num_pages << page_sh,
                                                                  pool);
  return cudaGetLastError();
}

}  // namespace k16
