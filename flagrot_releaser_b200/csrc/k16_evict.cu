// Eviction from the 16-bit cache: per (row, kv head) the tokens with the largest accumulated attention weight stay, in order.
//
// HBM bound: 8 D bytes move per kept (token, kv head) (key and value row, read and written), 4 bytes are read per weight.
// Two launches:
//   k_select  a cluster of 1 to 8 CTAs per (row, kv head), the weights' order-preserving keys in registers: the threshold by a
//             radix search (four digits of 8 bits; the CTAs' histograms are added through distributed shared memory), then the
//             kept positions and their weights are written in order;
//   k_copy    (other pages) a CTA per 64 kept tokens, or
//   k_move    (in place) a cluster per (row, kv head) that moves the rows down step by step: a kept token only moves to a lower
//             position, so a step's writes hit no row that a later step reads, and one cluster barrier per step is enough.
//
// Measured (D 128): 32 rows of up to 4096 tokens x 8 heads to 2048: 99 us, of which the copy 82 (the measured copy rate); one row of
// 60000 x 8 heads to 7500: 28.5 us, of which the copy 10 and the selection 14: eight clusters of eight CTAs that meet five times
// (1.9 us a digit, half of it the barrier and the others' histograms).  With the keys in shared memory instead of registers the
// selection took 19 us.  In place: 117 and 48 us (a step's reads and the writes of the step before it overlap, the next one's
// do not).
#include <cooperative_groups.h>

#include "k16_kernels.h"
#include "k16_launch.cuh"

namespace cg = cooperative_groups;

namespace k16 {
namespace {

constexpr int NT = 512, NWARP = NT / 32;
constexpr int DIGIT = 8, BINS = 1 << DIGIT, PASSES = 32 / DIGIT;
constexpr int MAX_KEYS = 32 * NT;                     // keys of a CTA that registers hold

// order-preserving key of a weight: a > b as floats iff key(a) > key(b); -0 equals +0, NaN is below everything
FR_DEVI uint32_t key_of(float w) {
  if (isnan(w)) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);        // -0 + 0 = +0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
FR_DEVI float weight_of(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k); }   // (0: a NaN)
// one more in a counter of shared memory, under a predicate (a branch around each: the first two passes a fifth longer)
FR_DEVI void count_if(uint32_t on, uint32_t counter) {
  asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %0, 0;\n @p red.shared.add.u32 [%1], 1;\n}\n" ::"r"(on), "r"(counter) : "memory");
}
// the n lowest of 32 bits
FR_DEVI uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; }

// A warp's positions are consecutive; lane l has every 32nd of them from the l-th on, KPT keys in registers.  ONCE: that is all
// of them, read once; else (more than MAX_KEYS to a CTA) every pass reads them again, KPT at a time.
// CL: the cluster has more than one CTA.
template <int KPT, bool ONCE, bool CL> __global__ void __launch_bounds__(NT, KPT <= 16 ? 2 : 1) k_select(EvictArgs a, int C) {
  static_assert(ONCE || KPT == 32, "a mask of 32 positions to a lane");
  __shared__ alignas(16) int hist[PASSES][BINS];
  __shared__ alignas(16) int total[BINS];             // the cluster's histogram of a pass
  __shared__ int s_sure[NWARP], s_ties[NWARP];
  __shared__ int s_count[2];                          // this CTA's sure tokens and ties, read by the cluster
  cg::cluster_group cl = cg::this_cluster();
  const auto sync = [&]() {
    if (CL) cl.sync();
    else __syncthreads();
  };
  const int g = blockIdx.x / C, rank = blockIdx.x - g * C, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int b = g / a.c.Hkv, h = g - b * a.c.Hkv;
  for (int i = tid; i < PASSES * BINS; i += NT) (&hist[0][0])[i] = 0;
  let_next_start();
  after_previous();
  const int len = min(a.c.len(b), a.w_len), m = min(len, a.budget);
  const float* w = a.weights + b * a.w_bs + h * a.w_hs;
  int* kept = a.kept + static_cast<long long>(g) * a.budget;
  float* nw = a.new_weights + static_cast<long long>(g) * a.nw_len;
  const int seg = (len + C - 1) / C, s0 = min(rank * seg, len), s1 = min(s0 + seg, len);
  const int wseg = ((seg + NWARP - 1) / NWARP + 31) & ~31, i0 = min(s0 + wid * wseg, s1), i1 = min(i0 + wseg, s1);
  uint32_t k[KPT];
  const auto load = [&](int i) {                      // the keys of positions i + 32 e + lane, all loads in flight
    float x[KPT];
#pragma unroll
    for (int e = 0; e < KPT; ++e) x[e] = i + 32 * e + lane < i1 ? w[i + 32 * e + lane] : 0.f;
#pragma unroll
    for (int e = 0; e < KPT; ++e) k[e] = key_of(x[e]);
  };
  if (ONCE && len > a.budget) load(i0);
  if (h == 0 && rank == 0 && tid == 0) a.new_lens[b] = m;
  for (int i = m + rank * NT + tid; i < a.budget; i += C * NT) kept[i] = -1;
  for (int i = m + rank * NT + tid; i < a.nw_len; i += C * NT) nw[i] = 0.f;
  if (len <= a.budget) {                              // (the whole cluster)
    for (int i = rank * NT + tid; i < len; i += C * NT) kept[i] = i, nw[i] = w[i];
    return;
  }
  const int lo = a.sinks, hi = len - a.recent, want = a.budget - a.sinks - a.recent;   // [lo, hi) is chosen from
  // bit e: position i + 32 e + lane is among those before n
  const auto before = [&](int i, int n) { return low_bits((n - i - lane + 31) >> 5); };
  const auto chosen_from = [&](int i) { return want > 0 ? before(i, min(hi, i1)) & ~before(i, lo) : 0u; };
  uint32_t T = 0;                                     // the want-th largest key
  int left = want;                                    // ... of whose ties this many are taken
  __syncthreads();
  if (want > 0) {
#pragma unroll 1
    for (int p = 0; p < PASSES; ++p) {
      const int sh = 32 - DIGIT * (p + 1);
      const uint32_t h0 = static_cast<uint32_t>(__cvta_generic_to_shared(&hist[p][0]));
      for (int i = i0; i < i1; i += 32 * KPT) {
        if (!ONCE) load(i);
        const uint32_t cand = chosen_from(i), top = p == 0 ? 0u : ~0u << (sh + DIGIT);
#pragma unroll
        for (int e = 0; e < KPT; ++e) {
          if (i + 32 * e >= i1) break;
          count_if(((k[e] ^ T) & top) == 0 ? cand & (1u << e) : 0u, h0 + 4 * ((k[e] >> sh) & (BINS - 1)));
        }
      }
      sync();
      const int* cnt = hist[p];
      if (CL) {                                       // every CTA of a cluster adds all histograms up for itself
        if (tid < BINS) {
          int x[8], n = 0;
#pragma unroll
          for (int r = 0; r < 8; ++r) x[r] = r < C ? cl.map_shared_rank(&hist[p][0], r)[tid] : 0;
#pragma unroll
          for (int r = 0; r < 8; ++r) n += x[r];
          total[tid] = n;
        }
        __syncthreads();
        cnt = total;
      }
      // counts from the top bin down, eight bins a lane, every warp for itself: the one bin in which the count reaches `left`
      const int4* c4 = reinterpret_cast<const int4*>(cnt + BINS - 8 * (lane + 1));
      const int4 x = c4[0], y = c4[1];
      const int c8[8] = {y.w, y.z, y.y, y.x, x.w, x.z, x.y, x.x};
      int n = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) n += c8[e];
      int cum = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(~0u, cum, d);
        if (lane >= d) cum += v;
      }
      const int src = __ffs(__ballot_sync(~0u, cum >= left)) - 1;
      int digit = BINS - 1 - 8 * lane, rest = left - (cum - n);
#pragma unroll
      for (int e = 0; e < 7; ++e) {
        const bool on = digit == BINS - 1 - 8 * lane - e && rest > c8[e];
        rest -= on ? c8[e] : 0;
        digit -= on ? 1 : 0;
      }
      T |= static_cast<uint32_t>(__shfl_sync(~0u, digit, src)) << sh;
      left = __shfl_sync(~0u, rest, src);
    }
  }
  // sure tokens (forced, or above T) and ties are counted, then written in order, 32 at a time
  uint32_t msure = 0, mtie = 0;                       // bit e: position i + 32 e + lane is one
  const auto mark = [&](int i) {
    const uint32_t cand = chosen_from(i);
    msure = before(i, i1) & (~before(i, hi) | before(i, lo));
    mtie = 0;
#pragma unroll
    for (int e = 0; e < KPT; ++e) {
      msure |= k[e] > T ? cand & (1u << e) : 0u;
      mtie |= k[e] == T ? cand & (1u << e) : 0u;
    }
  };
  int sure = 0, ties = 0;
  for (int i = i0; i < i1; i += 32 * KPT) {
    if (!ONCE) load(i);
    mark(i);
    sure += __popc(msure);
    ties += __popc(mtie);
  }
  sure = __reduce_add_sync(~0u, sure);
  ties = __reduce_add_sync(~0u, ties);
  if (lane == 0) s_sure[wid] = sure, s_ties[wid] = ties;
  __syncthreads();
  int pos = 0, tie0 = 0;                              // this CTA's before this warp
  sure = ties = 0;
#pragma unroll
  for (int i = 0; i < NWARP; ++i) {
    if (i == wid) pos = sure, tie0 = ties;
    sure += s_sure[i];
    ties += s_ties[i];
  }
  int cta_tie = 0, cta_pos = 0;                       // ties and kept tokens before this CTA
  if (CL) {
    if (tid == 0) s_count[0] = sure, s_count[1] = ties;
    cl.sync();
    int x[8], t[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int* c = cl.map_shared_rank(&s_count[0], r < rank ? r : rank);
      x[r] = r < rank ? c[0] : 0;
      t[r] = r < rank ? c[1] : 0;
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      cta_pos += x[r] + min(max(left - cta_tie, 0), t[r]);
      cta_tie += t[r];
    }
    cl.barrier_arrive();                              // the last look at the others' memory
  }
  int tie_at = cta_tie + tie0;
  pos += cta_pos + min(tie_at, left) - min(cta_tie, left);
  const unsigned below = (1u << lane) - 1;
  for (int i = i0; i < i1; i += 32 * KPT) {
    if (!ONCE) load(i), mark(i);
    if (__any_sync(~0u, mtie != 0)) {                 // of the ties the first left - tie_at are taken
#pragma unroll 1
      for (int e = 0; e < KPT; ++e) {
        const unsigned mt = __ballot_sync(~0u, mtie >> e & 1);
        if ((mtie >> e & 1) && tie_at + __popc(mt & below) < left) msure |= 1u << e;
        tie_at += __popc(mt);
      }
    }
#pragma unroll
    for (int e = 0; e < KPT; ++e) {
      if (i + 32 * e >= i1) break;
      const unsigned mk = __ballot_sync(~0u, msure >> e & 1);
      const int at = pos + __popc(mk & below);
      if ((msure >> e & 1) && at < m) {               // (at < m: unless another stream changes the weights meanwhile)
        kept[at] = i + 32 * e + lane;
        nw[at] = weight_of(k[e]);
      }
      pos += __popc(mk);
    }
  }
  if (CL) cl.barrier_wait();                          // the others have read this CTA's counts
}

// Rows to other pages: a CTA copies TOK kept tokens, 16-byte pieces, eight of each thread's in flight.
constexpr int CT = 256, TOK = 64;
template <int D> __global__ void __launch_bounds__(CT) k_copy(EvictArgs a, int chunks) {
  constexpr int PPR = D / 8, PPT = 2 * PPR;           // pieces per row, per token (key row, then value row)
  __shared__ long long src[TOK], dst[TOK];            // element offsets of the key rows, or -1 | -2
  const int g = blockIdx.x / chunks, b = g / a.c.Hkv, h = g - b * a.c.Hkv, r0 = (blockIdx.x - g * chunks) * TOK;
  after_previous();
  const int m = a.new_lens[b];
  if (r0 >= m) return;
  const int n = min(TOK, m - r0);
  if (threadIdx.x < TOK) {
    const int r = r0 + threadIdx.x, t = threadIdx.x;
    long long s = -1, d = -1;
    if (t < n) {
      const int j = a.kept[static_cast<long long>(g) * a.budget + r], ps = a.c.page_of(b, j);
      const int pd = a.dst_bt[b * a.dst_stride + (r >> a.c.page_sh)];
      if (ps >= 0) s = row_at(ps, a.c.Hkv, h, 0, a.c.page_sh, j & (a.c.page() - 1), D);
      if (pd >= 0 && pd < a.dst_pages) d = row_at(pd, a.c.Hkv, h, 0, a.c.page_sh, r & (a.c.page() - 1), D);
    }
    src[t] = s;
    dst[t] = d;
  }
  __syncthreads();
  const long long v = static_cast<long long>(D) << a.c.page_sh;   // from a key row to its value row
  constexpr int IT = TOK * PPT / CT;
  uint4 x[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int p = i * CT + threadIdx.x, t = p / PPT, e = p % PPT;
    x[i] = make_uint4(0, 0, 0, 0);
    if (src[t] >= 0) x[i] = __ldcs(reinterpret_cast<const uint4*>(a.c.pool + src[t] + (e / PPR) * v + (e % PPR) * 8));
  }
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int p = i * CT + threadIdx.x, t = p / PPT, e = p % PPT;
    if (dst[t] >= 0) *reinterpret_cast<uint4*>(a.dst + dst[t] + (e / PPR) * v + (e % PPR) * 8) = x[i];
  }
}

// In place: step s moves the kept tokens [s C R, (s + 1) C R).  A step's sources are read into registers before the barrier
// behind which it writes, while the step before it writes: those writes end below every position that is being read.  The
// positions and pages of a step are looked up two steps ahead (they are two dependent loads from L2).
constexpr int MT = 256;
template <int D, bool CL> __global__ void __launch_bounds__(MT, 2) k_move(EvictArgs a, int C) {
  constexpr int PPR = D / 8, PPT = 2 * PPR, IT = 8, R = IT * MT / PPT;   // tokens per CTA and step
  static_assert(R <= MT, "a thread per token");
  __shared__ long long src[3][R], dst[3][R];          // element offsets of the key rows; src -1: reads as zeros; dst -1: stays
  cg::cluster_group cl = cg::this_cluster();
  const auto sync = [&]() {
    if (CL) cl.sync();
    else __syncthreads();
  };
  const int g = blockIdx.x / C, rank = blockIdx.x - g * C, b = g / a.c.Hkv, h = g - b * a.c.Hkv, tid = threadIdx.x;
  after_previous();
  const int len = min(a.c.len(b), a.w_len), m = a.new_lens[b];
  if (len <= a.budget) return;                        // (the whole cluster)
  const int* kept = a.kept + static_cast<long long>(g) * a.budget;
  uint16_t* pool = a.dst;
  const int steps = (m + C * R - 1) / (C * R);
  const auto row = [&](int j) -> long long {
    const int pg = a.c.page_of(b, j);
    return pg < 0 ? -1 : row_at(pg, a.c.Hkv, h, 0, a.c.page_sh, j & (a.c.page() - 1), D);
  };
  const auto look = [&](int s, long long& from, long long& to) {   // thread t < R: token t of step s
    const int r = (s * C + rank) * R + tid;
    from = to = -1;
    if (tid < R && r < m) {
      const int j = kept[r];
      if (j != r) from = row(j), to = row(r);
    }
  };
  const long long v = static_cast<long long>(D) << a.c.page_sh;
  const int e = tid % PPT, t0 = tid / PPT;
  const long long eo = (e / PPR) * v + (e % PPR) * 8;
  const auto read = [&](int s, uint4 (&y)[IT]) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const long long o = src[s % 3][i * (MT / PPT) + t0];
      y[i] = make_uint4(0, 0, 0, 0);
      if (o >= 0) y[i] = __ldcg(reinterpret_cast<const uint4*>(pool + o + eo));
    }
  };
  for (int s = 0; s < 2; ++s) {
    long long from, to;
    look(s, from, to);
    if (tid < R) src[s][tid] = from, dst[s][tid] = to;
  }
  __syncthreads();
  uint4 x[IT];
  read(0, x);
  for (int s = 0; s < steps; ++s) {
    long long from, to;
    look(s + 2, from, to);
    sync();                                           // every source of this step is in registers
    uint4 y[IT];
    read(s + 1, y);
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const long long o = dst[s % 3][i * (MT / PPT) + t0];
      if (o >= 0) __stcg(reinterpret_cast<uint4*>(pool + o + eo), x[i]);
    }
    if (tid < R) src[(s + 2) % 3][tid] = from, dst[(s + 2) % 3][tid] = to;
#pragma unroll
    for (int i = 0; i < IT; ++i) x[i] = y[i];
  }
}

// CTAs per (row, kv head): as many as the SMs hold at once, of at least 2048 positions each, and enough to hold the weights in
// registers.  32 x 4096 x 8 heads: 99 us with one CTA, 114 with two, 186 with eight; 16 x 16000 x 8: 41 with one, 42 with two, 52 with
// four; 4 x 30000 x 8: 27 with two, 21 with four, 23 with eight; 1 x 60000 x 8: 35 with four, 28.5 with eight.
// (20 x 32769 x 4, one position more than two CTAs' registers hold: 55 with four, 73 with two that read the weights in every pass.)
int cluster_of(long long groups, long long positions) {
  int c = 1;
  while (c < 8 && ((groups * c * 2 <= 148 && positions / c > 2048) || (positions + c - 1) / c > MAX_KEYS)) c *= 2;
  return c;
}

}  // namespace

cudaError_t evict(const EvictArgs& a, cudaStream_t st) {
  const long long groups = static_cast<long long>(a.B) * a.c.Hkv;
  const long long width = static_cast<long long>(a.c.bt_width) << a.c.page_sh;
  const long long most = width < a.w_len ? width : a.w_len;
  const int c = cluster_of(groups, most);
  const long long seg = (most + c - 1) / c;
  // as many registers as the longest row's keys take: two CTAs to an SM up to 8192 keys
  const auto k = seg > MAX_KEYS      ? k_select<32, false, true>    // (the largest cluster)
                 : seg > MAX_KEYS / 2 ? (c > 1 ? k_select<32, true, true> : k_select<32, true, false>)
                 : seg > MAX_KEYS / 4 ? (c > 1 ? k_select<16, true, true> : k_select<16, true, false>)
                                      : (c > 1 ? k_select<8, true, true> : k_select<8, true, false>);
  const cudaError_t e = launch(k, static_cast<unsigned>(groups * c), NT, 0, c, st, a, c);
  if (e != cudaSuccess) return e;
  if (!a.dst_bt) {
    // a CTA per (row, kv head) where they fill the SMs, else a cluster (256 of them: 117 us with one CTA, 125 with two, 136 with
    // eight; 8 of them: 206, 134 and 48 us)
    int cm = 1;
    while (cm < 8 && groups * cm < 148 && a.budget / cm > 256) cm *= 2;
    const auto k = a.D == 128 ? (cm > 1 ? k_move<128, true> : k_move<128, false>) : (cm > 1 ? k_move<64, true> : k_move<64, false>);
    return launch(k, static_cast<unsigned>(groups * cm), MT, 0, cm, st, a, cm);
  }
  const long long longest = width < a.budget ? width : a.budget, chunks = (longest + TOK - 1) / TOK;
  if (chunks == 0) return cudaSuccess;
  if (chunks * groups > 0x7FFFFFFFll) return cudaErrorInvalidValue;
  return a.D == 128 ? launch(k_copy<128>, static_cast<unsigned>(groups * chunks), CT, 0, 0, st, a, static_cast<int>(chunks))
                    : launch(k_copy<64>, static_cast<unsigned>(groups * chunks), CT, 0, 0, st, a, static_cast<int>(chunks));
}

}  // namespace k16
