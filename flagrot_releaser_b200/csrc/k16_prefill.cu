// Attention of many new tokens over the 16-bit cache: causal, with an optional sliding window and sink tokens, on the
// 5th-generation tensor cores.
//
//   S = Q K^T,   p = 2^(qscale S - ref),   O += P V,   out = O / sum p          (running reference and sum per row)
//
// Tensor bound: 4 D flops per (q head, query, visible key).  A work item is a pair of 128-row query tiles of one (sequence,
// kv head): rows are tokens times the G q heads of the group, so all heads of a group share every key and value tile that is
// fetched.  S (128 keys at a time), P and O of both tiles live in tensor memory (512 columns: S0 S1 O0 O1, P over its own S).
//
// CTA (one per SM, persistent): warps 0-3 and 4-7 are the softmax of tile 0 and 1 (a thread per row), warp 8 issues the
// MMAs, warp 9 takes work items and issues the tensor copies (Q once per item, K and V tiles of 128 keys through one ring).
// The tensor pipe alternates  P0 V(j-1), Q0 K(j), P1 V(j-1), Q1 K(j):  while one tile's softmax runs, the other's products do.
// The softmax reference is lazy: it moves when a row's maximum has grown by more than 2^8, and only then is O rescaled.
//
// V is taken as it lies (keys by dims): the second product's B operand is MN-major, K = keys.
// P is rounded to the cache's type (2^-9 relative in bf16, 2^-12 in fp16: one rounding, like the output's own); the row sums,
// S and O are 32-bit.
#include "k16_kernels.h"
#include "k16_tma.cuh"

namespace k16 {
namespace {

constexpr int BN = 128;                  // keys per block
constexpr int THREADS = 384;            // three warpgroups: two of softmax, one of MMA, copies and two idle warps
constexpr int W_MMA = 8, W_TMA = 9;
constexpr int REGS_SOFT = 216, REGS_REST = 72;   // 256 x 216 + 128 x 72 = 384 x 168, what the launch has
constexpr int MAX_HEADS = 128;           // q heads per item
constexpr float LAZY = 8.f;
constexpr int MAX_SPLIT = 32;            // pieces of a pair's key blocks
constexpr int SLOTS = 2 * 148;           // workspace slots: pieces of split pairs
constexpr int SPLIT_COST = 4;            // what a piece costs besides its blocks, in blocks

__device__ int g_status;

struct Item {
  int b, h, hq0, heads;                  // sequence, kv head, first q head and their number
  int tok0, tok1;                        // tokens of the pair
  int pos0;                              // position of tok0
  int len;
  int nsb, wb;                           // key blocks: the first nsb hold the sinks, the others start at block wb
  int k0, k1;                            // ... of which this item takes [k0, k1)
  int ns, part, slot, stride;            // pieces of the pair, this one's number and workspace slot, slots between pieces
  FR_DEVI int block(int k) const { return k < nsb ? k : wb + k - nsb; }
};
// the tokens of one tile, as positions [pa, pb]
struct Tile {
  int pa, pb, last, window, sinks;       // last: index of the last block that the tile needs (-1: none)
  FR_DEVI Tile(const Item& it, int i, int tpt, int window_, int sinks_) : last(-1), window(window_), sinks(sinks_) {
    pa = it.pos0 + i * tpt;
    pb = min(it.pos0 + it.tok1 - it.tok0, pa + tpt) - 1;
    if (pb >= max(pa, 0))
      for (int k = it.k1 - 1; k >= it.k0 && last < 0; --k)
        if (needs(it.block(k) * BN)) last = k;
    if (last < 0) pb = -1;                                     // nothing in this item's blocks
  }
  FR_DEVI bool needs(int kb) const { return kb <= pb && (window <= 0 || kb + BN > pa - window + 1 || kb < sinks); }
  FR_DEVI bool whole(int kb) const { return kb + BN - 1 <= pa && (window <= 0 || kb > pb - window || kb + BN <= sinks); }
};

template <int D> struct Smem {
  static constexpr int QT = 128 * D * 2;                       // one query tile
  static constexpr int STAGE = BN * D * 2;                     // one K or V tile
  static constexpr int STAGES = D == 128 ? 5 : 10;
  static constexpr int RING = 2 * QT;
  static constexpr int BAR = RING + STAGES * STAGE;            // full[STAGES] empty[STAGES] qfull qempty sfull[2] pfull[2] ofull[2]
  static constexpr int NBAR = 2 * STAGES + 2 + 6 + 4;          // ... items: full[2], empty[2]
  static constexpr int ITEMS = BAR + NBAR * 8;                 // Item[2]
  static constexpr int MISC = ITEMS + 2 * 64;                  // tensor-memory base, abort flag
  static constexpr int TOTAL = MISC + 16 + 1024;
};
static_assert(sizeof(Item) <= 64, "item slot");
static_assert(Smem<128>::TOTAL <= 232448, "shared memory");

FR_DEVI bool wait_at(uint32_t bar, uint32_t parity, volatile uint32_t* abort, int line) {
  bool ok = true;
  if (!tc5::mbar_try(bar, parity)) {
    ok = !*abort && tc5::mbar_wait_abortable(bar, parity, abort);
    if (!ok) atomicCAS(&g_status, 0, line);
  }
  return __all_sync(~0u, ok);
}
#define k16_wait(bar, parity) wait_at(bar, parity, abort, __LINE__)

// MN-major operand in 128-byte swizzle: lbo = bytes between 64-element chunks along N, sbo = bytes between groups of 8 keys
FR_DEVI uint64_t desc_mn(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return tc5::DESC_VERSION | tc5::DESC_SW128 | (static_cast<uint64_t>(sbo >> 4) << 32) | (static_cast<uint64_t>(lbo >> 4) << 16) |
         ((saddr & 0x3FFFFu) >> 4);
}
constexpr uint32_t B_MN_MAJOR = 1u << 16;                      // instruction descriptor: B is MN-major

// two floats in one register pair; each half is rounded like the scalar operation
FR_DEVI uint64_t pk(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
FR_DEVI float2 un(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
FR_DEVI uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
FR_DEVI uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
FR_DEVI float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// the n lowest of 32 bits
FR_DEVI uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; }

FR_DEVI float4 f4(const uint32_t* v) {
  return make_float4(__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2]), __uint_as_float(v[3]));
}
template <int DT> FR_DEVI void put8(uint16_t* out, float4 x, float4 y, float inv, bool any) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (any) {
    v.x = Elem<DT>::pack(x.x * inv, x.y * inv);
    v.y = Elem<DT>::pack(x.z * inv, x.w * inv);
    v.z = Elem<DT>::pack(y.x * inv, y.y * inv);
    v.w = Elem<DT>::pack(y.z * inv, y.w * inv);
  }
  *reinterpret_cast<uint4*>(out) = v;
}
FR_DEVI void tile_sync(int i) {                                // the softmax warps of a tile
  if (i == 0) asm volatile("bar.sync 1, 128;\n" ::: "memory");
  else asm volatile("bar.sync 2, 128;\n" ::: "memory");
}

template <int DT, int D>
__global__ void __launch_bounds__(THREADS, 1) k_prefill(const __grid_constant__ PrefillArgs a, const __grid_constant__ CUtensorMap qmap,
                                                        const __grid_constant__ CUtensorMap kvmap, int hb, int nhg, int box_rows) {
  using S = Smem<D>;
  constexpr int STAGES = S::STAGES, HALVES = D / 64;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = static_cast<uint32_t>(__cvta_generic_to_shared(smem_raw));
  const uint32_t sm = (raw + 1023) & ~1023u;
  unsigned char* base = smem_raw + (sm - raw);
  const uint32_t full = sm + S::BAR, empty = full + 8 * STAGES, qfull = empty + 8 * STAGES, qempty = qfull + 8, sfull = qempty + 8,
                 pfull = sfull + 16, ofull = pfull + 16, ifull = ofull + 16, iempty = ifull + 16;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(base + S::MISC);
  volatile uint32_t* abort = tmem_slot + 1;
  volatile uint32_t* flag = tmem_slot + 2;                     // [2]: this CTA joins the pieces of the tile
  Item* items = reinterpret_cast<Item*>(base + S::ITEMS);
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      tc5::mbar_init(full + 8 * i, 1);
      tc5::mbar_init(empty + 8 * i, 1);
    }
    tc5::mbar_init(qfull, 1);
    tc5::mbar_init(qempty, 1);
    for (int i = 0; i < 2; ++i) {
      tc5::mbar_init(sfull + 8 * i, 1);
      tc5::mbar_init(pfull + 8 * i, 4);
      tc5::mbar_init(ofull + 8 * i, 1);
      tc5::mbar_init(ifull + 8 * i, 1);
      tc5::mbar_init(iempty + 8 * i, 9);
    }
    tc5::mbar_init_fence();
    *abort = 0;
    tma_prefetch_map(&qmap);
    tma_prefetch_map(&kvmap);
  }
  if (w == W_MMA) {
    tc5::tmem_alloc(sm + S::MISC, 512);
    tc5::tmem_relinquish();
  }
  tc5::fence_before_sync();
  __syncthreads();
  tc5::fence_after_sync();
  const uint32_t tm = *tmem_slot;
  const uint32_t tS = tm, tO = tm + 256;                       // columns: S0 128 | S1 128 | O0 128 | O1 128
  const int tpt = 128 / hb;                                    // tokens per tile; row = token * hb + head

  if (w >= 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(REGS_REST));
  if (w > W_TMA) {
    // (idle)
  } else if (w == W_TMA) {                                            // ----------------------------------- items and tensor copies
    const int Hv = a.c.Hkv * nhg;
    const int rows_all = static_cast<int>((a.c.num_pages * a.c.Hkv * 2) << a.c.page_sh);
    const int nbox = BN / box_rows, box_sh = __ffs(box_rows) - 1;
    int n = 0, qc = 0;                                         // ring tiles and query pairs issued
    // blocks of the pair at tok0 of a sequence with tokens up to end
    const auto blocks = [&](int tok0, int end, int len, int& wb, int& nsb) {
      const int pos0 = len - end + tok0, p1 = pos0 + min(2 * tpt, end - tok0) - 1;
      const Span sp(max(pos0, 0), a.window, a.sinks);
      wb = sp.lo / BN;
      nsb = min((min(a.sinks, sp.lo) + BN - 1) / BN, wb);
      return p1 >= 0 ? nsb + p1 / BN - wb + 1 : 0;
    };
    // blocks of the longest pair of a sequence: without a window the last pair's; with one the largest count that any pair
    // can have (its keys span at most window + 2 tpt - 1 positions, which touch one block more than they fill)
    const auto most_blocks = [&](int beg, int end, int len, int np) {
      int wb, nsb;
      const int last = blocks(beg + (np - 1) * 2 * tpt, end, len, wb, nsb);
      return a.window <= 0 ? last : nsb + min((max(len, 1) - 1) / BN + 1, (min(a.window, 1 << 30) + 2 * tpt - 2) / BN + 2);
    };
    // few pairs: their key blocks are cut into pieces of `chunk` so that the grid is full, by the number of pieces that
    // costs the least of max(one piece, waves of pieces); each piece of a pair has a workspace slot
    int chunk = 1 << 30;
    {
      long long pairs = 0;
      int most = 0;
      float all = 0.f;
      for (int b = lane; b < a.B; b += 32) {
        const int beg = min(max(a.cu_q[b], 0), a.T), end = min(max(a.cu_q[b + 1], beg), a.T), len = a.c.len(b);
        if (end == beg) continue;
        const int np = (end - beg + 2 * tpt - 1) / (2 * tpt);
        int x, y;
        pairs += static_cast<long long>(np) * Hv;
        most = max(most, most_blocks(beg, end, len, np));
        all += 0.5f * (blocks(beg, end, len, x, y) + blocks(beg + (np - 1) * 2 * tpt, end, len, x, y)) * np * Hv;
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) {
        pairs += __shfl_xor_sync(~0u, pairs, d);
        most = max(most, __shfl_xor_sync(~0u, most, d));
        all += __shfl_xor_sync(~0u, all, d);
      }
      if (pairs > 0 && 2 * pairs <= SLOTS && most > 1) {
        const int sp = lane + 1, c = (most + sp - 1) / sp;     // lane i: i + 1 pieces
        const float avg = all / static_cast<float>(pairs), per = ceilf(avg / c);
        float cost = fmaxf(static_cast<float>(c + (sp > 1 ? SPLIT_COST : 0)),
                           ceilf(pairs * per / gridDim.x) * (avg / fmaxf(per, 1.f) + (sp > 1 ? SPLIT_COST : 0)));
        if (pairs * ((most + c - 1) / c) > SLOTS) cost = INFINITY;
        float best = cost;
#pragma unroll
        for (int d = 16; d; d >>= 1) best = fminf(best, __shfl_xor_sync(~0u, best, d));
        const int at = __ffs(__ballot_sync(~0u, cost == best)) - 1;
        if (at > 0) chunk = __shfl_sync(~0u, c, at);
      }
    }
    // 32 sequences at a time: lane i has sequence r0 + i, its tokens, its items (pairs x pieces of the longest pair x heads)
    // and the items up to and with it
    int r0 = -32, beg = 0, end = 0, pieces = 1;
    long long mine = 0, upto = 0, row0 = 0, group = 0;         // row0: items before the 32
    long long idx = blockIdx.x;
    for (int ic = 0;; ++ic, idx += gridDim.x) {
      Item it;
      it.b = -1;
      while (r0 < a.B && idx >= row0 + group) {                // (indices only grow)
        row0 += group;
        r0 += 32;
        const int b = r0 + lane;
        beg = end = 0;
        if (b < a.B) {
          beg = min(max(a.cu_q[b], 0), a.T);
          end = min(max(a.cu_q[b + 1], beg), a.T);
        }
        const int np = (end - beg + 2 * tpt - 1) / (2 * tpt);
        pieces = 1;
        if (chunk < 1 << 30 && np > 0) {
          pieces = max((most_blocks(beg, end, a.c.len(b), np) + chunk - 1) / chunk, 1);
        }
        mine = static_cast<long long>(np) * pieces * Hv;
        upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const long long y = __shfl_up_sync(~0u, upto, d);
          if (lane >= d) upto += y;
        }
        group = __shfl_sync(~0u, upto, 31);
      }
      if (r0 < a.B) {                                          // a head's pairs side by side, the longest first
        const int src = __ffs(__ballot_sync(~0u, row0 + upto > idx)) - 1, b = r0 + src;
        const int off = static_cast<int>(idx - row0 - __shfl_sync(~0u, upto - mine, src));
        const int sbeg = __shfl_sync(~0u, beg, src), send = __shfl_sync(~0u, end, src), np = __shfl_sync(~0u, pieces, src);
        const int npairs = (send - sbeg + 2 * tpt - 1) / (2 * tpt);
        const int hv = off / (npairs * np), rem = off - hv * npairs * np, part = rem / npairs, pr = npairs - 1 - (rem - part * npairs);
        it.b = b;
        it.h = hv / nhg;
        const int hg = hv - it.h * nhg;
        it.hq0 = it.h * a.G + hg * hb;
        it.heads = min(a.G - hg * hb, hb);
        it.tok0 = sbeg + pr * 2 * tpt;
        it.tok1 = min(it.tok0 + 2 * tpt, send);
        it.len = a.c.len(b);
        it.pos0 = it.len - send + it.tok0;
        const int nblk = blocks(it.tok0, send, it.len, it.wb, it.nsb);
        it.k0 = part > 0 ? part * chunk : 0;
        it.k1 = min(it.k0 + min(chunk, nblk), nblk);
        it.ns = np > 1 ? max((nblk + chunk - 1) / chunk, 1) : 1;
        it.part = part;
        it.slot = static_cast<int>(idx);
        it.stride = npairs;
        if (part > 0 && it.k0 >= nblk) {                       // a shorter pair than the sequence's longest
          --ic;
          continue;
        }
      }
      const int sl = ic & 1;
      if (ic >= 2 && !k16_wait(iempty + 8 * sl, (ic / 2 - 1) & 1)) break;
      if (lane == 0) {
        items[sl] = it;
        tc5::mbar_arrive(ifull + 8 * sl);
      }
      __syncwarp();
      if (it.b < 0) break;
      if (it.k0 == it.k1) continue;
      // queries: [D half][token][head] = rows of 128 bytes; what lies outside q arrives as zeros
      if (qc > 0 && !k16_wait(qempty, (qc - 1) & 1)) break;
      if (lane == 0) {
        tc5::mbar_expect(qfull, 2 * HALVES * tpt * hb * 128);
        for (int i = 0; i < 2; ++i)
          for (int x = 0; x < HALVES; ++x)
            tma4(sm + i * S::QT + x * 128 * 128, &qmap, 0, it.hq0, it.tok0 + i * tpt, x, qfull);
      }
      ++qc;
      const int* bt = a.c.bt + it.b * a.c.bt_stride;
      bool ok = true;
      for (int k = it.k0; k < it.k1 && ok; ++k) {
        const int j = it.block(k) * BN + lane * box_rows;      // lane i < nbox: box i of the block
        int y = rows_all;
        if (lane < nbox && j < it.len) {
          const int pg = bt[j >> a.c.page_sh];
          if (pg >= 0 && pg < a.c.num_pages)
            y = ((pg * a.c.Hkv + it.h) * 2 << a.c.page_sh) + (j & (a.c.page() - 1));
        }
        for (int kv = 0; kv < 2; ++kv, ++n) {
          const int st = n % STAGES;
          if (n >= STAGES && !k16_wait(empty + 8 * st, (n / STAGES - 1) & 1)) {
            ok = false;
            break;
          }
          if (lane == 0) tc5::mbar_expect(full + 8 * st, S::STAGE);
          __syncwarp();
          if (lane < nbox) {
            const uint32_t dst = sm + S::RING + st * S::STAGE + (lane << (box_sh + 7));
            const int yy = y == rows_all ? y : y + (kv << a.c.page_sh);
            for (int x = 0; x < HALVES; ++x) tma3(dst + x * BN * 128, &kvmap, 0, yy, x, full + 8 * st);
          }
          __syncwarp();
        }
      }
      if (!ok) break;
    }
    // the CTA ends after its copies and its commits on the ring have arrived (bounded, also when a wait has run out)
    for (int i = max(0, n - STAGES); i < n && lane == 0; ++i) {
      if (!*abort && tc5::mbar_wait(empty + 8 * (i % STAGES), (i / STAGES) & 1)) continue;
      tc5::mbar_wait(full + 8 * (i % STAGES), (i / STAGES) & 1);
    }
    if (*abort && lane == 0 && qc) tc5::mbar_wait(qfull, (qc - 1) & 1);
  } else if (w == W_MMA) {                                     // ------------------------------------------------------ MMAs
    constexpr uint32_t ID_QK = tc5::idesc(1, DT == 0 ? 1 : 0, DT == 0 ? 1 : 0, 128, BN);
    constexpr uint32_t ID_PV = tc5::idesc(1, DT == 0 ? 1 : 0, DT == 0 ? 1 : 0, 128, D) | B_MN_MAJOR;
    int n = 0, qc = 0, pc[2] = {0, 0};                         // ring tiles, query pairs, P tiles consumed
    bool run = true;
    for (int ic = 0; run; ++ic) {
      const int sl = ic & 1;
      if (!k16_wait(ifull + 8 * sl, (ic / 2) & 1)) break;
      const Item it = items[sl];
      __syncwarp();
      if (lane == 0) tc5::mbar_arrive(iempty + 8 * sl);
      if (it.b < 0) break;
      if (it.k0 == it.k1) continue;
      const Tile t0(it, 0, tpt, a.window, a.sinks), t1(it, 1, tpt, a.window, a.sinks);
      if (!k16_wait(qfull, qc & 1)) break;
      ++qc;
      tc5::fence_after_sync();
      bool started[2] = {false, false};
      for (int k = it.k0; k <= it.k1 && run; ++k) {
        const int nv = n + 2 * (k - it.k0) - 1, nk = nv + 1;          // ring tiles of V(k - 1) and K(k)
        const uint32_t sv = sm + S::RING + (nv % STAGES) * S::STAGE, sk = sm + S::RING + (nk % STAGES) * S::STAGE;
        const int kbv = k > it.k0 ? it.block(k - 1) * BN : 0, kbk = k < it.k1 ? it.block(k) * BN : 0;
        if (k > it.k0) {
          if (!(run = k16_wait(full + 8 * (nv % STAGES), (nv / STAGES) & 1))) break;
          if (kbv + BN > it.len) {                             // values behind the sequence: 0 * NaN would be NaN
            for (int i = (it.len - kbv) * 8 + lane; i < BN * 8; i += 32)
#pragma unroll
              for (int x = 0; x < HALVES; ++x)
                asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};\n" ::"r"(sv + x * BN * 128 + i * 16), "r"(0) : "memory");
            tc5::fence_async_smem();
            __syncwarp();
          }
        }
        bool have_k = false;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const Tile& t = i ? t1 : t0;
          if (k > it.k0 && t.needs(kbv)) {
            if (!(run = k16_wait(pfull + 8 * i, pc[i] & 1))) break;
            ++pc[i];
            tc5::fence_after_sync();
            if (tc5::elect_one()) {
#pragma unroll
              for (int s = 0; s < BN / 16; ++s)
                tc5::mma_f16_ts(tO + i * 128, tS + i * 128 + s * 8, desc_mn(sv + s * 2048, BN * 128, 1024), ID_PV, started[i] || s > 0);
              if (k - 1 == t.last) tc5::mma_commit(ofull + 8 * i);
            }
            __syncwarp();
            started[i] = true;
          }
          if (k < it.k1 && !have_k) {
            if (!(run = k16_wait(full + 8 * (nk % STAGES), (nk / STAGES) & 1))) break;
            have_k = true;
            tc5::fence_after_sync();
          }
          if (k < it.k1 && t.needs(kbk)) {
            if (tc5::elect_one()) {
#pragma unroll
              for (int s = 0; s < D / 16; ++s)
                tc5::mma_f16_ss(tS + i * 128, tc5::desc_sw128(sm + i * S::QT + (s >> 2) * 128 * 128 + (s & 3) * 32, 1024),
                                tc5::desc_sw128(sk + (s >> 2) * BN * 128 + (s & 3) * 32, 1024), ID_QK, s > 0);
              tc5::mma_commit(sfull + 8 * i);
            }
            __syncwarp();
          }
        }
        if (!run) break;
        if (tc5::elect_one()) {
          if (k > it.k0) tc5::mma_commit(empty + 8 * (nv % STAGES));
          if (k < it.k1) tc5::mma_commit(empty + 8 * (nk % STAGES));
          if (k == it.k1 - 1) tc5::mma_commit(qempty);
        }
        __syncwarp();
      }
      n += 2 * (it.k1 - it.k0);
    }
  } else {                                                     // --------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(REGS_SOFT));
    const int i = w >> 2, r = tid & 127, tok = r / hb, head = r - tok * hb;
    const uint32_t lanes = static_cast<uint32_t>(w & 3) << 21;  // tensor-memory lanes of this warp
    const uint32_t ts = tS + i * 128 + lanes, to = tO + i * 128 + lanes;
    const bool neg = a.qscale < 0.f;                           // the maximum is taken of |qscale| (+-S)
    const float qs = fmaxf(fabsf(a.qscale), 1e-37f);           // a scale of 0: all scores alike, and -inf * qs stays -inf
    constexpr float BIAS = DT == 1 ? 6.f : 0.f;                // fp16 weights are carried times 2^6: their steps below 2^-14 are absolute
    int sc = 0, oc = 0;                                        // S and O tiles consumed
    bool run = true;
    for (int ic = 0; run; ++ic) {
      const int sl = ic & 1;
      if (!k16_wait(ifull + 8 * sl, (ic / 2) & 1)) break;
      const Item it = items[sl];
      __syncwarp();
      if (lane == 0) tc5::mbar_arrive(iempty + 8 * sl);
      if (it.b < 0) break;
      const Tile t(it, i, tpt, a.window, a.sinks);
      const int mytok = it.tok0 + i * tpt + tok;
      const bool live = tok < tpt && head < it.heads && mytok < it.tok1;
      const int pos = live ? it.pos0 + i * tpt + tok : -1;
      float ref = -INFINITY, l = 0.f;
      for (int k = it.k0; k < it.k1; ++k) {
        const int kb = it.block(k) * BN;
        if (!t.needs(kb)) continue;
        if (!(run = k16_wait(sfull + 8 * i, sc & 1))) break;
        ++sc;
        tc5::fence_after_sync();
        uint32_t v[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tc5::tmem_ld32(ts + 32 * c, v[c]);
        tc5::tmem_ld_wait();
        if (neg)
#pragma unroll
          for (int c = 0; c < 128; ++c) v[c >> 5][c & 31] ^= 0x80000000u;
        if (!t.whole(kb)) {
          const int hi = pos + 1 - kb, lo = a.window > 0 ? pos - a.window + 1 - kb : 0, sk = a.sinks - kb;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t see = low_bits(hi - 32 * c) & (~low_bits(lo - 32 * c) | low_bits(sk - 32 * c));
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(see & (1u << e))) v[c][e] = 0xFF800000u;
          }
        }
        float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          m0 = max3(m0, __uint_as_float(v[0][c]), __uint_as_float(v[0][c + 1]));
          m1 = max3(m1, __uint_as_float(v[1][c]), __uint_as_float(v[1][c + 1]));
          m2 = max3(m2, __uint_as_float(v[2][c]), __uint_as_float(v[2][c + 1]));
          m3 = max3(m3, __uint_as_float(v[3][c]), __uint_as_float(v[3][c + 1]));
        }
        const float m = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)) * qs;
        if (__any_sync(~0u, m > ref + LAZY)) {
          const float nr = fmaxf(m, ref), f = ref == -INFINITY ? 0.f : ex2(ref - nr);
          // S(k) is complete, so every product into O before it is; the next one waits for this P
          if (__any_sync(~0u, l > 0.f)) {
            l *= f;
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tc5::tmem_ld32(to + 32 * c, o);
              tc5::tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tc5::tmem_st32(to + 32 * c, o);
            }
          }
          ref = nr;
        }
        const float off = (ref == -INFINITY ? 0.f : -ref) + BIAS;
        const uint64_t q2 = pk(qs, qs), off2 = pk(off, off);
        uint64_t sum = 0, sum1 = 0;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t p[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const int x = 64 * c + 2 * e;
            const float2 y = un(fma2(pk(__uint_as_float(v[x >> 5][x & 31]), __uint_as_float(v[x >> 5][(x & 31) + 1])), q2, off2));
            const float p0 = ex2(y.x), p1 = ex2(y.y);
            if (e & 1) sum1 = add2(sum1, pk(p0, p1));
            else sum = add2(sum, pk(p0, p1));
            p[e] = Elem<DT>::pack(p0, p1);
          }
          tc5::tmem_st32(ts + 32 * c, p);
        }
        const float2 l2 = un(add2(sum, sum1));
        l += l2.x + l2.y;
        tc5::tmem_st_wait();
        tc5::fence_before_sync();
        __syncwarp();
        if (lane == 0) tc5::mbar_arrive(pfull + 8 * i);
      }
      if (!run) break;
      const bool any = t.last >= 0;
      if (any) {
        if (!(run = k16_wait(ofull + 8 * i, oc & 1))) break;
        ++oc;
        tc5::fence_after_sync();
      }
      uint16_t* out = static_cast<uint16_t*>(a.out) + mytok * a.o_ts + (it.hq0 + head) * D;
      if (it.ns == 1) {
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;   // a row that sees nothing gives zeros; NaN stays NaN
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          if (any) {
            tc5::tmem_ld32(to + 32 * c, o);
            tc5::tmem_ld_wait();
          }
          if (live) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) put8<DT>(out + 32 * c + e, f4(o + e), f4(o + e + 4), inv, any && inv != 0.f);
          }
          __syncwarp();
        }
      } else {
        // this piece's sums to its slot, [dims / 4][row] x 16 bytes; the last piece of the tile to arrive joins them in order
        const int rr = i * (D / 4) * 128 + r;
        float4* po = reinterpret_cast<float4*>(a.ws) + static_cast<long long>(it.slot) * (2 * (D / 4) * 128) + rr;
        float2* pl = reinterpret_cast<float2*>(a.ws + static_cast<long long>(SLOTS) * (2 * D * 128 * 4));
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          if (any) {
            uint32_t o[32];
            tc5::tmem_ld32(to + 32 * c, o);
            tc5::tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 8; ++e) __stcg(po + (c * 8 + e) * 128, f4(o + 4 * e));
          }
        }
        __stcg(pl + static_cast<long long>(it.slot) * 256 + i * 128 + r, make_float2(ref, l));
        __threadfence();
        tile_sync(i);
        const int slot0 = it.slot - it.part * it.stride;
        if (r == 0) {
          int* tk = a.tickets + 2 * slot0 + i;
          const int old = atomicAdd(tk, 1);
          if (old == it.ns - 1) *tk = 0;
          flag[i] = old == it.ns - 1;
          __threadfence();
        }
        tile_sync(i);
        if (flag[i]) {
          const float2* ml = pl + static_cast<long long>(slot0) * 256 + i * 128 + r;
          const float4* pq = reinterpret_cast<const float4*>(a.ws) + static_cast<long long>(slot0) * (2 * (D / 4) * 128) + rr;
          float M = -INFINITY, L = 0.f;
          for (int s = 0; s < it.ns; ++s) M = fmaxf(M, __ldcg(ml + static_cast<long long>(s * it.stride) * 256).x);
          for (int s = 0; s < it.ns; ++s) {
            const float2 e = __ldcg(ml + static_cast<long long>(s * it.stride) * 256);
            if (e.y != 0.f) L = fmaf(ex2(e.x - M), e.y, L);    // (0: the piece has no key that this row sees)
          }
          const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
#pragma unroll 1
          for (int c = 0; c < D / 4; c += 8) {
            float4 acc[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int s = 0; s < it.ns; ++s) {
              const float2 e2 = __ldcg(ml + static_cast<long long>(s * it.stride) * 256);
              if (e2.y == 0.f) continue;
              const float f = ex2(e2.x - M);
              const float4* q = pq + static_cast<long long>(s * it.stride) * (2 * (D / 4) * 128) + c * 128;
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float4 x = __ldcg(q + e * 128);
                acc[e].x = fmaf(f, x.x, acc[e].x);
                acc[e].y = fmaf(f, x.y, acc[e].y);
                acc[e].z = fmaf(f, x.z, acc[e].z);
                acc[e].w = fmaf(f, x.w, acc[e].w);
              }
            }
            if (live)
#pragma unroll
              for (int e = 0; e < 8; e += 2) put8<DT>(out + 4 * (c + e), acc[e], acc[e + 1], inv, inv != 0.f);
          }
          __syncwarp();
        }
        tile_sync(i);                                          // (the flag is free again)
      }
      tc5::fence_before_sync();
    }
  }
  tc5::fence_before_sync();
  __syncthreads();
  if (w == W_MMA) {
    tc5::fence_after_sync();
    tc5::tmem_dealloc(tm, 512);
  }
}

template <int DT, int D>
cudaError_t launch(const PrefillArgs& a, const CUtensorMap& qm, const CUtensorMap& kv, int hb, int nhg, int box, int grid, cudaStream_t st) {
  const auto k = k_prefill<DT, D>;
  if (cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D>::TOTAL)) return e;
  k<<<grid, THREADS, Smem<D>::TOTAL, st>>>(a, qm, kv, hb, nhg, box);
  return cudaGetLastError();
}

}  // namespace

static void groups(int G, int& nhg, int& hb, int& tpt) {       // q heads per item, tokens per tile
  nhg = (G + MAX_HEADS - 1) / MAX_HEADS;
  hb = (G + nhg - 1) / nhg;
  tpt = 128 / hb;
}
// pairs at most: every sequence may end inside one
static long long max_pairs(int rows, int Hkv, int G, long long new_tokens) {
  int nhg, hb, tpt;
  groups(G, nhg, hb, tpt);
  return (new_tokens / (2 * tpt) + rows) * Hkv * nhg;
}
// sums and (reference, denominator) of every slot; a pair is split into MAX_SPLIT pieces at most
long long prefill_ws_bytes(int, int, int, int D, long long) { return static_cast<long long>(SLOTS) * 256 * (D * 4 + 8); }
long long prefill_tickets(int, int, int, long long) { return 2 * SLOTS; }

int prefill_status() {
  int v = -1;
  return cudaMemcpyFromSymbol(&v, g_status, sizeof(v)) == cudaSuccess ? v : -1;
}

cudaError_t prefill(int dtype, const PrefillArgs& a, cudaStream_t st) {
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return e;
  int nhg, hb, tpt;
  groups(a.G, nhg, hb, tpt);
  const int Hq = a.c.Hkv * a.G;
  const int box = 1 << a.c.page_sh;                            // page <= 128 = BN rows
  CUtensorMap qm, kv;
  e = encode4(&qm, dtype, a.q, Hq, a.D * 2ull, a.T, a.T > 1 ? a.q_ts * 2ull : Hq * a.D * 2ull, a.D / 64, 128, hb, tpt);
  if (e == cudaSuccess)
    e = encode3(&kv, dtype, a.c.pool, static_cast<uint64_t>((a.c.num_pages * a.c.Hkv * 2) << a.c.page_sh), a.D * 2ull, a.D / 64, 128, box, 1);
  if (e != cudaSuccess) return e;
  const long long items = max_pairs(a.B, a.c.Hkv, a.G, a.T) * MAX_SPLIT;
  const int grid = static_cast<int>(items < sms ? items : sms);
  if (dtype == 0)
    return a.D == 128 ? launch<0, 128>(a, qm, kv, hb, nhg, box, grid, st) : launch<0, 64>(a, qm, kv, hb, nhg, box, grid, st);
  return a.D == 128 ? launch<1, 128>(a, qm, kv, hb, nhg, box, grid, st) : launch<1, 64>(a, qm, kv, hb, nhg, box, grid, st);
}

}  // namespace k16
