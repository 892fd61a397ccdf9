// Decode attention over the 16-bit cache: one new token per row, keys and values streamed from the pages once.
//
//   s_j = qscale q . k_j,   p_j = 2^(s_j - ref),   o = sum_j p_j v_j / sum_j p_j
//
// HBM bound: a (key, kv head) costs 4 D bytes and 4 D G flops, so the kernel is a stream through shared memory with the
// products on mma.sync (m16n8k16): the contraction has at most 8 to 32 query rows, a small share of what the tensor pipe
// does in the time the bytes take, and its operands come straight out of the swizzled tiles with ldmatrix.
//
// Work: the visible keys of a (row, kv head, group of up to 32 q heads) are a segment of 32-key blocks; the segments of all
// rows, each rounded up to four blocks, form one list which is cut into equal contiguous ranges, one per CTA.  So uneven
// lengths need no host plan (the lengths may change under a captured graph), one long row fills the card, and many short
// rows are not split.  A range's pieces of segments are joined through the workspace by the last CTA to arrive (in the order
// of the pieces: the result does not depend on which one that is).
//
// CTA: four consumer warps and a producer warp that fills a ring of 16 KB stages (one block: 32 keys and their values) with
// two tensor copies each; two CTAs per SM, so that a CTA's start and joins are covered by the other's stream.  A block goes to
// NT warps, one per tile of TR q heads: one tile of 8 for G up to 8, up to 16 two of 8 (D 128) or one of 16 (D 64), two of 16
// above.  A weight meets the values as p = hi + lo, both of the cache's type, with an error of 2^-17 instead of 2^-9: in a tile
// of 8 the other 8 rows of the second MMA carry lo, at no extra cost; in a tile of 16 lo is a product of its own.  Per head that
// is a quarter fewer MMAs and half the reads of shared memory: G 32 (64 rows of 4096 tokens, 4 kv heads, D 128) 122 us, with
// four tiles of 8 157; D 64 43 and 53.  G 16 as one tile of 16: D 128 191 us where two of 8 take 177, for then all four stages are being worked on;
// D 64, with eight stages, 109 and 112.
//
// Measured (bf16, D 128, G 4, page 16, of the measured copy rate of 6.55 TB/s): 64 rows of up to 4096 tokens 153 us = 0.95; one
// row of 131072 94 us = 0.87; 32 rows x 1028 visible of 16384 29 us = 0.72; one row of 77 tokens 5 us on the device.  What is
// left: 4 to 6 us from the launch to a CTA's first block, 2 us for a join's fence and ticket, and the CTAs' uneven ends.
#include "k16_kernels.h"
#include "k16_launch.cuh"
#include "k16_tma.cuh"

namespace k16 {
namespace {

constexpr int NW = 4, THREADS = 32 * (NW + 1);
constexpr int BLK = 32;                  // keys per block
constexpr int MAX_CTAS = 2 * 148;        // partial slots of the workspace: two per CTA
constexpr int MAX_GT = 32;               // q heads per segment
constexpr float LAZY = 8.f;              // the softmax reference moves when a score exceeds it by more than this (log2)
// the reference before the first score: finite, so that a weight against it is 0 and not NaN where every score is -inf
constexpr float NO_REF = -3.402823466e38f;

__device__ int g_status;

// a workspace slot: sums [GT][D], then (reference, denominator) [GT]; a multiple of 16 bytes
__host__ __device__ __forceinline__ long long slot_floats(int GT, int D) { return (static_cast<long long>(GT) * (D + 2) + 3) & ~3ll; }

template <int D, int TR> struct Smem {   // TR: q heads of a tile
  // a multiple of NW: a stage always goes to the same warps, whose waits on its barrier then follow its phases one by one
  // (copies of different stages may land in any order, and a parity wait cannot tell a phase from the one two before)
  static constexpr int STAGES = D == 128 ? 4 : 8;
  static constexpr int STAGE = BLK * D * 4;                    // keys, values
  static constexpr int MERGE = STAGES * STAGE;                 // float [NW][TR][D]
  static constexpr int ML = MERGE + NW * TR * D * 4;           // float2 [NW][TR]
  static constexpr int BAR = ML + NW * TR * 8;                 // full[STAGES], empty[STAGES]
  static constexpr int RED = BAR + 2 * STAGES * 8;             // long long [NW + 1]; int [2 (NW + 1)]; abort flag; last-arriver flag
  static constexpr int TOTAL = RED + 96 + 1024;                // slack: the ring starts on a 1024-byte boundary
};

// a row's visible keys as blocks: [0, nsb) cover the sinks, the others start at block wb
struct Row {
  int len, s1, lo, nsb, wb, nblk, nv;    // nv: its room in the list
  FR_DEVI void set(int len_, int window, int sinks, int pad) {
    len = len_;
    const Span sp(len - 1, window, sinks);
    s1 = sp.s1;
    lo = sp.lo;
    wb = lo / BLK;
    nsb = min((s1 + BLK - 1) / BLK, wb);
    nblk = len > 0 ? nsb + (len + BLK - 1) / BLK - wb : 0;
    nv = nblk > 0 ? max((nblk + 3) & ~3, pad) : 0;
  }
  FR_DEVI int block(int k) const { return k < nsb ? k : wb + k - nsb; }
  FR_DEVI bool visible(int j) const { return j < len && (j < s1 || j >= lo); }
  FR_DEVI bool any(int j0, int j1) const { return j0 < s1 || max(j0, lo) < min(j1, len); }
  FR_DEVI bool whole(int blk) const { return (blk + 1) * BLK <= len && (blk * BLK >= lo || (blk + 1) * BLK <= s1); }
};

// the pieces of a CTA's range, in order; every warp walks them for itself
struct Walk {
  const AttnArgs& a;
  int Hv, pad, b;
  long long f, fend, row0, quota;
  Row r;
  int seg, k0, k1;                       // piece: blocks [k0, k1) of segment seg (kv head, head group) of row b
  long long f0;                          // where the segment begins
  FR_DEVI Walk(const AttnArgs& a_, int Hv_, int pad_, long long quota_, long long begin, long long total)
      : a(a_), Hv(Hv_), pad(pad_), quota(quota_) {
    f = begin;
    fend = min(begin + quota, total);
    row0 = 0;
    b = 0;
    if (f >= fend) return;
    const int lane = threadIdx.x & 31;
    for (int r0 = 0;; r0 += 32) {        // the row that holds f: 32 rows at a time
      long long n = 0;
      if (r0 + lane < a.B) {
        Row x;
        x.set(a.c.len(r0 + lane), a.window, a.sinks, pad);
        n = static_cast<long long>(x.nv) * Hv;
      }
      long long s = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long y = __shfl_up_sync(~0u, s, d);
        if (lane >= d) s += y;
      }
      const unsigned hit = __ballot_sync(~0u, row0 + s > f);
      if (hit) {
        const int w = __ffs(hit) - 1;
        b = r0 + w;
        row0 += __shfl_sync(~0u, s - n, w);
        break;
      }
      row0 += __shfl_sync(~0u, s, 31);
    }
    r.set(a.c.len(b), a.window, a.sinks, pad);
  }
  FR_DEVI bool next() {
    while (f < fend) {
      while (f - row0 >= static_cast<long long>(r.nv) * Hv) {
        row0 += static_cast<long long>(r.nv) * Hv;
        r.set(a.c.len(++b), a.window, a.sinks, pad);
      }
      const long long off = f - row0;
      seg = static_cast<int>(off / r.nv);
      k0 = static_cast<int>(off - static_cast<long long>(seg) * r.nv);
      f0 = f - k0;
      const int n = static_cast<int>(min(static_cast<long long>(r.nv - k0), fend - f));
      f += n;
      k1 = min(k0 + n, r.nblk);
      if (k1 > k0) return true;
    }
    return false;
  }
  FR_DEVI int first_cta() const { return static_cast<int>(f0 / quota); }
  FR_DEVI int last_cta() const { return static_cast<int>((f0 + r.nblk - 1) / quota); }
};

FR_DEVI void ldsm4(uint32_t a, uint32_t (&v)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a) : "memory");
}
FR_DEVI void ldsm4t(uint32_t a, uint32_t (&v)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a) : "memory");
}
template <int DT> FR_DEVI void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (DT == 0)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
FR_DEVI void bar_consumers() { asm volatile("bar.sync 1, %0;\n" ::"n"(32 * NW) : "memory"); }

// a bounded wait of a whole warp; one that runs out records its line, after which every wait of the CTA returns at once
FR_DEVI void wait_at(uint32_t bar, uint32_t parity, volatile uint32_t* abort, int line) {
  if (!*abort && !tc5::mbar_wait_abortable(bar, parity, abort)) atomicCAS(&g_status, 0, line);
  __syncwarp();
}
#define k16_wait(bar, parity, abort) wait_at(bar, parity, abort, __LINE__)

// a row whose scores are all -inf has no weights: zeros, and nothing added to its sums
FR_DEVI float inverse(float sum) { return sum == 0.f ? 0.f : 1.f / sum; }
template <int DT> FR_DEVI float log_sum(float ref, float sum) { return sum == 0.f ? INFINITY : ref + log2f(sum) - (DT == 1 ? 6.f : 0.f); }

// The pieces of CTAs c0 .. c1 of the segment that begins at f0, in order: four dims of a head per thread, eight pieces in flight;
// few heads: the threads also share the pieces, and their sums meet in shared memory (scr).
template <int DT, int D>
FR_DEVI void join(const AttnArgs& a, const float* part, long long quota, long long f0, int c0, int c1, int heads, int GT, float* scr,
                  uint16_t* out, float* lse) {
  constexpr int NTH = 32 * NW, IN = 8;
  const int cols = heads * (D / 4), tid = threadIdx.x, sets = max(NTH / cols, 1), stride = sets > 1 ? cols * sets : NTH;
  const auto finish = [&](int col, float M, float L, float4 v) {
    const float inv = inverse(L);
    uint2 r;
    r.x = Elem<DT>::pack(v.x * inv, v.y * inv);
    r.y = Elem<DT>::pack(v.z * inv, v.w * inv);
    *reinterpret_cast<uint2*>(out + 4 * col) = r;              // (col = head * D / 4 + dims)
    if (lse && col % (D / 4) == 0) lse[col / (D / 4)] = log_sum<DT>(M, L);
  };
  for (int i = tid; i < (sets > 1 ? stride : cols); i += stride) {
    const int col = i % cols, set = i / cols, hh = col / (D / 4), d = 4 * (col - hh * (D / 4));
    float M = -INFINITY, L = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = c0 + set; c <= c1; c += IN * sets) {
      float2 e[IN];
      float4 y[IN];
#pragma unroll
      for (int k = 0; k < IN; ++k) {
        const int cc = c + k * sets;
        const float* p = part + (static_cast<long long>(cc) * 2 + (cc == c0 && f0 != c0 * quota ? 1 : 0)) * slot_floats(GT, D);
        e[k] = cc <= c1 ? __ldcg(reinterpret_cast<const float2*>(p + GT * D + 2 * hh)) : make_float2(-INFINITY, 0.f);
        y[k] = cc <= c1 ? __ldcg(reinterpret_cast<const float4*>(p + hh * D + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float nm = M;
#pragma unroll
      for (int k = 0; k < IN; ++k) nm = fmaxf(nm, e[k].x);
      const float f = ex2(M - nm);
      M = nm;
      L *= f;
      v = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
#pragma unroll
      for (int k = 0; k < IN; ++k) {
        const float x = ex2(e[k].x - nm);
        L = fmaf(x, e[k].y, L);
        v.x = fmaf(x, y[k].x, v.x);
        v.y = fmaf(x, y[k].y, v.y);
        v.z = fmaf(x, y[k].z, v.z);
        v.w = fmaf(x, y[k].w, v.w);
      }
    }
    if (sets == 1) {
      finish(col, M, L, v);
    } else {
      *reinterpret_cast<float4*>(scr + 4 * i) = v;
      *reinterpret_cast<float2*>(scr + 4 * NTH + 2 * i) = make_float2(M, L);
    }
  }
  if (sets == 1) return;                                       // (all threads)
  bar_consumers();
  if (tid < cols) {
    float M = -INFINITY, L = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    const int n = min(sets, c1 - c0 + 1);                      // the others had no piece
    for (int s = 0; s < n; ++s) M = fmaxf(M, scr[4 * NTH + 2 * (s * cols + tid)]);
    for (int s = 0; s < n; ++s) {
      const float2 e = *reinterpret_cast<const float2*>(scr + 4 * NTH + 2 * (s * cols + tid));
      const float4 y = *reinterpret_cast<const float4*>(scr + 4 * (s * cols + tid));
      const float x = ex2(e.x - M);
      L = fmaf(x, e.y, L);
      v.x = fmaf(x, y.x, v.x);
      v.y = fmaf(x, y.y, v.y);
      v.z = fmaf(x, y.z, v.z);
      v.w = fmaf(x, y.w, v.w);
    }
    finish(tid, M, L, v);
  }
}

template <int DT, int D, int TR, int NT>
__global__ void __launch_bounds__(THREADS, 2) k_decode(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap map, int nhg,
                                                       float* part, float* lse, float* scores, long long score_ld) {
  using S = Smem<D, TR>;
  constexpr int STAGES = S::STAGES, KS = D / 16, ND = D / 8;                       // k steps of q . k, dim tiles of p . v
  constexpr int R = TR / 8;                                    // q heads of a thread: rows g and g + 8 of the tile
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = static_cast<uint32_t>(__cvta_generic_to_shared(smem_raw));
  const uint32_t sm = (raw + 1023) & ~1023u;
  unsigned char* base = smem_raw + (sm - raw);
  const uint32_t full = sm + S::BAR, empty = full + 8 * STAGES;
  long long* red = reinterpret_cast<long long*>(base + S::RED);
  int* redm = reinterpret_cast<int*>(base + S::RED + 40);
  volatile uint32_t* abort = reinterpret_cast<volatile uint32_t*>(base + S::RED + 80);
  volatile uint32_t* flag = abort + 1;
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int Hv = a.c.Hkv * nhg, Hq = a.c.Hkv * a.G;
  const int GT = min(a.G, MAX_GT);                             // q heads of a workspace slot

  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      tc5::mbar_init(full + 8 * i, 1);
      tc5::mbar_init(empty + 8 * i, NT);
    }
    tc5::mbar_init_fence();
    *abort = 0;
    tma_prefetch_map(&map);
  }
  let_next_start();
  after_previous();
  // the list's length; rows that see nothing are written as zeros here
  long long total = 0;
  int most = 0, rows = 0;                                      // the longest segment; rows that see something
  for (int b = tid; b < a.B; b += THREADS) {
    Row r;
    r.set(a.c.len(b), a.window, a.sinks, 0);
    total += r.nv;
    most = max(most, r.nv);
    rows += r.nv > 0;
  }
  total = (static_cast<long long>(__reduce_add_sync(~0u, static_cast<unsigned>(total >> 20))) << 20) +
          __reduce_add_sync(~0u, static_cast<unsigned>(total & 0xFFFFF));
  most = __reduce_max_sync(~0u, most);
  rows = __reduce_add_sync(~0u, rows);
  if (lane == 0) red[w] = total, redm[2 * w] = most, redm[2 * w + 1] = rows;
  for (int b = blockIdx.x; b < a.B; b += gridDim.x)
    if (a.c.len(b) == 0)
      for (int i = tid; i < Hq * D / 2; i += THREADS)
        reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + b * a.o_bs)[i] = 0;
  __syncthreads();
  total = rows = 0;
#pragma unroll
  for (int i = 0; i <= NW; ++i) total += red[i], most = max(most, redm[2 * i]), rows += redm[2 * i + 1];
  total *= Hv;
  long long quota = max(((total + gridDim.x - 1) / gridDim.x + 3) & ~3ll, 4ll);
  int pad = 0;
  // No more segments than CTAs and none much longer than a range: a whole segment each, and nothing to join (32 rows x 8 heads
  // x 1028 visible keys: 34.4 -> 29.4 us; where it does not hold the ranges stay equal).
  if (static_cast<long long>(rows) * Hv <= gridDim.x && 4 * most <= 5 * quota) {
    pad = most;
    quota = max(most, 4);
    total = static_cast<long long>(rows) * Hv * most;
  }
  Walk wk(a, Hv, pad, quota, static_cast<long long>(blockIdx.x) * quota, total);

  // where a block's 16-key half, dim half and values are in a stage: pages of 16 tokens come as [dim half][16 keys | 16 values]
  // per page, larger ones as [dim half][32 keys] and the same of values
  const bool p16 = a.c.page_sh == 4;
  const uint32_t a16 = p16 ? BLK * D * 2 : 2048u, ahalf = 4096u, av = p16 ? 2048u : BLK * D * 2;

  if (w == NW) {                                               // ------------------------------------------- producer
    const int rows_all = static_cast<int>((a.c.num_pages * a.c.Hkv * 2) << a.c.page_sh);
    int n = 0;                                                 // blocks issued
    while (wk.next()) {
      const int h = wk.seg / nhg;
      const int* bt = a.c.bt + wk.b * a.c.bt_stride;
      for (int kb = wk.k0; kb < wk.k1; kb += 32) {
        // lane i: the pool rows of block kb + i
        int y0 = rows_all, y1 = rows_all;
        bool v0 = false, v1 = false;
        if (kb + lane < wk.k1) {
          const int blk = wk.r.block(kb + lane), j = blk * BLK;
          if (p16) {
            const int p = 2 * blk;
            v0 = wk.r.any(j, j + 16);                          // a page without a visible key is not fetched
            v1 = wk.r.any(j + 16, j + 32);
            if (v0) {
              const int pg = bt[p];
              if (pg >= 0 && pg < a.c.num_pages) y0 = (pg * a.c.Hkv + h) * 32;
            }
            if (v1) {
              const int pg = bt[p + 1];
              if (pg >= 0 && pg < a.c.num_pages) y1 = (pg * a.c.Hkv + h) * 32;
            }
          } else {
            v0 = v1 = true;
            const int pg = bt[j >> a.c.page_sh];
            if (pg >= 0 && pg < a.c.num_pages) {
              y0 = (((pg * a.c.Hkv + h) * 2) << a.c.page_sh) + (j & (a.c.page() - 1));
              y1 = y0 + a.c.page();
            }
          }
        }
        const int cnt = min(32, wk.k1 - kb);
        for (int i = 0; i < cnt; ++i, ++n) {
          const int st = n % STAGES;
          const int r0 = __shfl_sync(~0u, y0, i), r1 = __shfl_sync(~0u, y1, i);
          const int n0 = __shfl_sync(~0u, static_cast<int>(v0), i), n1 = __shfl_sync(~0u, static_cast<int>(v1), i);
          if (n >= STAGES) k16_wait(empty + 8 * st, (n / STAGES - 1) & 1, abort);
          if (lane == 0 && !*abort) {
            const uint32_t dst = sm + st * S::STAGE;
            tc5::mbar_expect(full + 8 * st, (n0 + n1) * (BLK * D * 2));
            if (n0) tma3(dst, &map, 0, r0, 0, full + 8 * st);
            if (n1) tma3(dst + BLK * D * 2, &map, 0, r1, 0, full + 8 * st);
          }
          __syncwarp();
        }
      }
    }
    if (*abort && lane == 0)                                   // copies in flight end before the CTA does
      for (int i = max(0, n - STAGES); i < n; ++i) tc5::mbar_wait(full + 8 * (i % STAGES), (i / STAGES) & 1);
    return;
  }

  // -------------------------------------------------------------------------------------------------------- consumers
  constexpr int GROUPS = NW / NT;                              // blocks worked on at once
  const int tile = w / GROUPS, grp = w % GROUPS;
  const int g = lane >> 2, t = lane & 3, l8 = lane & 7, lm = lane >> 3;
  const uint32_t kx = l8 * 128 + ((lm ^ l8) << 4);             // K: matrix lm = 16-byte piece, row l8 = key
  const uint32_t vx = ((lm & 1) * 8 + l8) * 128 + (((lm >> 1) ^ l8) << 4);   // V: matrix = (dim piece, key half)
  float* mo = reinterpret_cast<float*>(base + S::MERGE);
  float2* ml = reinterpret_cast<float2*>(base + S::ML);
  int n = 0;                                                   // blocks before this piece
  while (wk.next()) {
    const int h = wk.seg / nhg, hg = wk.seg - h * nhg;
    const int heads = min(a.G - hg * MAX_GT, MAX_GT);          // q heads of the segment
    const int hq0 = h * a.G + hg * MAX_GT;
    const int hv = heads - tile * TR;                          // ... and of this warp's tile (may be <= 0)
    uint32_t q[KS][2 * R];
    // scores of row g (R = 2, and of row g + 8, which need not be one of the segment's)
    float* const srow = scores && g < hv ? scores + (static_cast<long long>(wk.b) * Hq + hq0 + tile * TR + g) * score_ld + 2 * t : nullptr;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool mine = g + 8 * r < hv;
      const int hq = hq0 + tile * TR + g + 8 * r;
      const uint32_t* qr = reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(a.q) + wk.b * a.q_bs + hq * D);
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        q[i][r] = mine ? qr[i * 8 + t] : 0u;
        q[i][R + r] = mine ? qr[i * 8 + 4 + t] : 0u;
      }
    }
    float o[ND][4], ref[R], l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) ref[r] = NO_REF, l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < ND; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    const int cnt = wk.k1 - wk.k0;
    for (int i = ((grp - n) % GROUPS + GROUPS) % GROUPS; i < cnt; i += GROUPS) {
      const int st = (n + i) % STAGES;
      const int blk = wk.r.block(wk.k0 + i);
      const uint32_t kt = sm + st * S::STAGE, vt = kt + av;
      k16_wait(full + 8 * st, ((n + i) / STAGES) & 1, abort);
      float s[4][4];
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) {
        s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {                     // 32 dims: pieces 4 c .. 4 c + 3
          uint32_t kf[4];
          ldsm4(kt + (nt >> 1) * a16 + (c >> 1) * ahalf + (nt & 1) * 1024 + (kx ^ ((c & 1) << 6)), kf);
          if constexpr (R == 1) {
            mma<DT>(s[nt], q[2 * c][0], 0u, q[2 * c][1], 0u, kf[0], kf[1]);
            mma<DT>(s[nt], q[2 * c + 1][0], 0u, q[2 * c + 1][1], 0u, kf[2], kf[3]);
          } else {
            mma<DT>(s[nt], q[2 * c][0], q[2 * c][1], q[2 * c][2], q[2 * c][3], kf[0], kf[1]);
            mma<DT>(s[nt], q[2 * c + 1][0], q[2 * c + 1][1], q[2 * c + 1][2], q[2 * c + 1][3], kf[2], kf[3]);
          }
        }
      }
      const bool whole = wk.r.whole(blk);
      uint32_t vm[4] = {~0u, ~0u, ~0u, ~0u};                   // values of hidden keys are zeroed: 0 * NaN is NaN
      float mx[R];
#pragma unroll
      for (int r = 0; r < R; ++r) mx[r] = -INFINITY;
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          s[nt][2 * r] *= a.qscale;
          s[nt][2 * r + 1] *= a.qscale;
          if (srow && (r == 0 || g + 8 < hv))
            *reinterpret_cast<float2*>(srow + r * 8 * score_ld + blk * BLK + nt * 8) = make_float2(s[nt][2 * r], s[nt][2 * r + 1]);
        }
        if (!whole) {
          const int j = blk * BLK + nt * 8 + 2 * t;
          const bool a0 = wk.r.visible(j), a1 = wk.r.visible(j + 1);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            if (!a0) s[nt][2 * r] = -INFINITY;
            if (!a1) s[nt][2 * r + 1] = -INFINITY;
          }
          vm[nt] = (a0 ? 0xFFFFu : 0u) | (a1 ? 0xFFFF0000u : 0u);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) mx[r] = fmaxf(mx[r], fmaxf(s[nt][2 * r], s[nt][2 * r + 1]));
      }
      bool moves = false;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(~0u, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(~0u, mx[r], 2));
        moves |= mx[r] > ref[r] + LAZY;
      }
      if (__any_sync(~0u, moves)) {                            // (the first block: ref = NO_REF)
        float f[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float nr = fmaxf(mx[r], ref[r]);
          f[r] = ex2(ref[r] - nr);
          ref[r] = nr;
          l[r] *= f[r];
        }
#pragma unroll
        for (int x = 0; x < ND; ++x) o[x][0] *= f[0], o[x][1] *= f[0], o[x][2] *= f[R - 1], o[x][3] *= f[R - 1];
      }
      // fp16 weights are carried times 2^6: below 2^-24 its steps are absolute
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        uint32_t hi[2][R], lo[2][R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float off = DT == 1 ? 6.f - ref[r] : -ref[r];
#pragma unroll
          for (int n2 = 0; n2 < 2; ++n2) {
            const float p0 = ex2(s[2 * ks + n2][2 * r] + off), p1 = ex2(s[2 * ks + n2][2 * r + 1] + off);
            l[r] += p0 + p1;
            hi[n2][r] = Elem<DT>::pack(p0, p1);
            const float2 e = Elem<DT>::f2(hi[n2][r]);
            lo[n2][r] = Elem<DT>::pack(p0 - e.x, p1 - e.y);
          }
        }
#pragma unroll
        for (int c = 0; c < ND; c += 2) {                      // 16 dims: pieces c, c + 1
          uint32_t vf[4];
          ldsm4t(vt + ks * a16 + (c >> 3) * ahalf + (vx ^ ((c & 7) << 4)), vf);
          if (!whole) vf[0] &= vm[2 * ks], vf[1] &= vm[2 * ks + 1], vf[2] &= vm[2 * ks], vf[3] &= vm[2 * ks + 1];
          if constexpr (R == 1) {
            mma<DT>(o[c], hi[0][0], lo[0][0], hi[1][0], lo[1][0], vf[0], vf[1]);
            mma<DT>(o[c + 1], hi[0][0], lo[0][0], hi[1][0], lo[1][0], vf[2], vf[3]);
          } else {
            mma<DT>(o[c], hi[0][0], hi[0][1], hi[1][0], hi[1][1], vf[0], vf[1]);
            mma<DT>(o[c + 1], hi[0][0], hi[0][1], hi[1][0], hi[1][1], vf[2], vf[3]);
            mma<DT>(o[c], lo[0][0], lo[0][1], lo[1][0], lo[1][1], vf[0], vf[1]);
            mma<DT>(o[c + 1], lo[0][0], lo[0][1], lo[1][0], lo[1][1], vf[2], vf[3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) tc5::mbar_arrive(empty + 8 * st);
    }
    n += cnt;
    // ---- join the warps of a tile, then the CTAs of a segment
#pragma unroll
    for (int r = 0; r < R; ++r) {
      l[r] += __shfl_xor_sync(~0u, l[r], 1);
      l[r] += __shfl_xor_sync(~0u, l[r], 2);
      if (t == 0) ml[w * TR + 8 * r + g] = make_float2(ref[r], l[r]);
      float* mw = mo + (w * TR + 8 * r + g) * D + 2 * t;
      if (g + 8 * r < hv)
#pragma unroll
        for (int x = 0; x < ND; ++x)
          *reinterpret_cast<float2*>(mw + x * 8) = R == 1 ? make_float2(o[x][0] + o[x][2], o[x][1] + o[x][3]) : make_float2(o[x][2 * r], o[x][2 * r + 1]);
    }
    bar_consumers();
    const int c0 = wk.first_cta(), c1 = wk.last_cta();
    float* slot = part + (static_cast<long long>(blockIdx.x) * 2 + (wk.f0 + wk.k0 == blockIdx.x * quota ? 0 : 1)) * slot_floats(GT, D);
    for (int i = tid; i < heads * (D / 2); i += 32 * NW) {
      const int hh = i / (D / 2), d = 2 * (i - hh * (D / 2)), w0 = hh / TR * GROUPS;
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int x = 0; x < GROUPS; ++x) M = fmaxf(M, ml[(w0 + x) * TR + hh % TR].x);
      float2 v = make_float2(0.f, 0.f);
#pragma unroll
      for (int x = 0; x < GROUPS; ++x) {
        const float2 e = ml[(w0 + x) * TR + hh % TR];
        if (e.y == 0.f) continue;                              // this warp had no block of the piece
        const float f = ex2(e.x - M);
        const float2 y = *reinterpret_cast<const float2*>(mo + ((w0 + x) * TR + hh % TR) * D + d);
        L = fmaf(f, e.y, L);
        v.x = fmaf(f, y.x, v.x);
        v.y = fmaf(f, y.y, v.y);
      }
      if (c0 == c1) {
        const float inv = inverse(L);
        reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + wk.b * a.o_bs + (hq0 + hh) * D)[d >> 1] = Elem<DT>::pack(v.x * inv, v.y * inv);
        if (lse && d == 0) lse[static_cast<long long>(wk.b) * Hq + hq0 + hh] = log_sum<DT>(M, L);
      } else {
        *reinterpret_cast<float2*>(slot + hh * D + d) = v;
        if (d == 0) *reinterpret_cast<float2*>(slot + GT * D + 2 * hh) = make_float2(M, L);
      }
    }
    if (c0 != c1) {
      __threadfence();
      bar_consumers();
      const long long sg = static_cast<long long>(wk.b) * Hv + wk.seg;
      if (tid == 0) {
        const int old = atomicAdd(a.tickets + sg, 1);
        *flag = old == c1 - c0;
        if (old == c1 - c0) a.tickets[sg] = 0;
        __threadfence();
      }
      bar_consumers();
      if (*flag) join<DT, D>(a, part, quota, wk.f0, c0, c1, heads, GT, mo, static_cast<uint16_t*>(a.out) + wk.b * a.o_bs + hq0 * D,
                             lse ? lse + static_cast<long long>(wk.b) * Hq + hq0 : nullptr);
    }
    bar_consumers();                                           // the merge area and the flag are free again
  }
}

// weights[b, h, j] += sum over the head group of 2^(score - lse): four keys per thread; VEC: the weights' rows are 16-byte
// aligned (32 x 8192: 160.6 us for the call, 161.9 without).
template <bool VEC> __global__ void __launch_bounds__(256) k_weights(AttnArgs a, const float* scores, long long score_ld, const float* lse, int chunks) {
  const int bh = blockIdx.x / chunks, b = bh / a.c.Hkv, h = bh - b * a.c.Hkv, Hq = a.c.Hkv * a.G;
  let_next_start();
  after_previous();
  const int len = a.c.len(b), j = (blockIdx.x - bh * chunks) * 1024 + 4 * threadIdx.x;
  const Span sp(len - 1, a.window, a.sinks);
  if (j >= len || (j >= sp.s1 && j + 4 <= sp.lo)) return;
  float* w = a.weights + b * a.w_bs + h * a.w_hs + j;
  const bool all = j + 4 <= len && (j >= sp.lo || j + 4 <= sp.s1);
  float4 old;
  if (VEC && all) old = *reinterpret_cast<const float4*>(w);
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  const long long r0 = static_cast<long long>(b) * Hq + h * a.G;
#pragma unroll 4
  for (int g = 0; g < a.G; ++g) {
    const float4 s = __ldcs(reinterpret_cast<const float4*>(scores + (r0 + g) * score_ld + j));
    const float m = lse[r0 + g];
    x.x += ex2(s.x - m);
    x.y += ex2(s.y - m);
    x.z += ex2(s.z - m);
    x.w += ex2(s.w - m);
  }
  if (VEC && all) {
    *reinterpret_cast<float4*>(w) = make_float4(old.x + x.x, old.y + x.y, old.z + x.z, old.w + x.w);
  } else {
    const float y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (j + e < len && (j + e < sp.s1 || j + e >= sp.lo)) w[e] += y[e];
  }
}

long long up(long long n, long long m) { return (n + m - 1) / m * m; }

template <int DT, int D, int TR, int NT>
cudaError_t launch_d(const AttnArgs& a, const CUtensorMap& map, int dev, int grid, int nhg, float* part, float* lse, float* scores, long long ld,
                   cudaStream_t st) {
  const auto k = k_decode<DT, D, TR, NT>;
  static std::atomic<bool> done[MAX_DEVICES];
  if (cudaError_t e = allow_smem(k, Smem<D, TR>::TOTAL, dev, done)) return e;
  return launch(k, grid, THREADS, Smem<D, TR>::TOTAL, 0, st, a, map, nhg, part, lse, scores, ld);
}
template <int DT, int D>
cudaError_t launch_nt(const AttnArgs& a, const CUtensorMap& map, int dev, int grid, int nhg, float* part, float* lse, float* scores, long long ld,
                      cudaStream_t st) {
  if (a.G <= 8) return launch_d<DT, D, 8, 1>(a, map, dev, grid, nhg, part, lse, scores, ld, st);
  if (a.G <= 16) return launch_d<DT, D, D == 64 ? 16 : 8, D == 64 ? 1 : 2>(a, map, dev, grid, nhg, part, lse, scores, ld, st);
  return launch_d<DT, D, 16, 2>(a, map, dev, grid, nhg, part, lse, scores, ld, st);
}

}  // namespace

// partials of two pieces per CTA | lse [rows, Hq] | scores [rows, Hq, max_len rounded up to blocks]
static long long part_bytes(int G, int D) { return up(2ll * MAX_CTAS * slot_floats(G < MAX_GT ? G : MAX_GT, D) * 4, 256); }
long long attn_ws_bytes(int rows, int Hkv, int G, int D, long long max_len, int weights) {
  const long long r = static_cast<long long>(rows) * Hkv * G;
  return part_bytes(G, D) + (weights ? up(r * 4, 256) + r * up(max_len, BLK) * 4 : 0);
}

int decode_status() {
  int v = -1;
  return cudaMemcpyFromSymbol(&v, g_status, sizeof(v)) == cudaSuccess ? v : -1;
}

cudaError_t attn(int dtype, const AttnArgs& a, cudaStream_t st) {
  int dev = 0, sms = 0;
  cudaError_t e = device_sms(dev, sms);
  if (e != cudaSuccess) return e;
  CUtensorMap map;
  e = pool_map(&map, dtype, a.c.pool, (a.c.num_pages * a.c.Hkv * 2) << a.c.page_sh, a.D, 32);
  if (e != cudaSuccess) return e;
  const long long R = static_cast<long long>(a.B) * a.c.Hkv * a.G, width = static_cast<long long>(a.c.bt_width) << a.c.page_sh;
  const long long ld = up(width, BLK);
  float* part = reinterpret_cast<float*>(a.ws);
  float* lse = a.weights ? reinterpret_cast<float*>(a.ws + part_bytes(a.G, a.D)) : nullptr;
  float* scores = a.weights ? lse + up(R * 4, 256) / 4 : nullptr;
  const int nhg = (a.G + MAX_GT - 1) / MAX_GT, grid = 2 * sms < MAX_CTAS ? 2 * sms : MAX_CTAS;
  if (dtype == 0)
    e = a.D == 128 ? launch_nt<0, 128>(a, map, dev, grid, nhg, part, lse, scores, ld, st) : launch_nt<0, 64>(a, map, dev, grid, nhg, part, lse, scores, ld, st);
  else
    e = a.D == 128 ? launch_nt<1, 128>(a, map, dev, grid, nhg, part, lse, scores, ld, st) : launch_nt<1, 64>(a, map, dev, grid, nhg, part, lse, scores, ld, st);
  if (e != cudaSuccess || !a.weights || width == 0) return e;
  const long long chunks = (width + 1023) / 1024;
  if (chunks * a.B * a.c.Hkv > 0x7FFFFFFFll) return cudaErrorInvalidValue;
  const bool vec = (reinterpret_cast<uintptr_t>(a.weights) & 15) == 0 && a.w_bs % 4 == 0 && a.w_hs % 4 == 0;
  return launch(vec ? k_weights<true> : k_weights<false>, static_cast<unsigned>(chunks * a.B * a.c.Hkv), 256, 0, 0, st, a,
                static_cast<const float*>(scores), ld, static_cast<const float*>(lse), static_cast<int>(chunks));
}

}  // namespace k16
