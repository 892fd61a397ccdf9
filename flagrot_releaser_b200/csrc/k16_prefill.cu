// Attention of many new tokens over the 16-bit cache: causal, with an optional sliding window and sink tokens, on the
// 5th-generation tensor cores.
//
//   S = Q K^T,   p = 2^(qscale S - ref),   O += P V,   out = O / sum p          (running reference and sum per row)
//
// Tensor bound: 4 D flops per (q head, query, visible key).  A work item is a pair of 128-row query tiles of one (sequence,
// kv head): rows are tokens times the G q heads of the group, so all heads of a group share every key and value tile that is
// fetched.  S, P and O of both tiles live in tensor memory (512 columns: S0 S1 O0 O1; P over its own S).
//
// CTA (one per SM, persistent): warps 0-3 and 4-7 are the softmax of tile 0 and 1 (a thread per row), warps 8 and 9 issue
// the MMAs of tile 0 and 1, warp 10 takes work items and issues the tensor copies (Q once per item, K and V tiles of 128
// keys through one ring).  S and P go in halves of 64 keys: a half's scores are computed while the other half's weights
// are, and a half that no query of the tile sees is left out.  The softmax reference is lazy: it moves when a row's
// maximum has grown by more than 2^8, and only then is O rescaled.
// Full waves of pairs run whole; the pairs of the last, partly filled wave are cut along their keys and joined where that is
// shorter (4 x 512 over 32768: 1083 us with, 1182 without; prompts through a window, whose pairs have 10 blocks: 395 with, 394
// without).
//
// V is taken as it lies (keys by dims): the second product's B operand is MN-major, K = keys.
// P is rounded to the cache's type (2^-9 relative in bf16, 2^-12 in fp16: one rounding, like the output's own, which makes
// the output's rms error up to sqrt 2 of its own rounding's: 0.0022 of the output's rms in bf16 where its own rounding is
// 0.0017); the row sums, S and O are 32-bit.
//
// Measured (bf16, D 128, G 4, page 16): 4 x 512 new tokens over 32768: 1.08 to 1.12 ms = 0.99 to 1.02 PFLOP/s under the power cap,
// where the same pipeline without its softmax runs at 1.30 and cuBLAS at 1.40; prompts of 5544 to 7033 tokens through a window of
// 1024: 0.39 to 0.41 ms = 0.72 to 0.75 PFLOP/s of visible pairs (1216 keys are computed for 1028 visible ones; zeroing the values
// that no query of a pair sees is 0.5 to 1 % of it, and nothing measurable of the other).  A step of 128 keys takes about
// 3900 cycles, 2500 of them tensor (the N = 64 products of the halves cost 48 cycles instead of 32); the rest is latency of
// the one softmax warp per tile and scheduler.  Measured and not kept: a polynomial 2^x for part of the weights (the MUFU is
// half idle), two threads per row (104 registers a thread: spills), whole 128-key S tiles (the same time, windows 8 % slower),
// turns between the tiles' exponentials (the same), output by warps of its own (2 % and 8 % slower), one loop over the halves that
// a tile needs, with the half chosen at run time (3 % slower).
#include "k16_kernels.h"
#include "k16_launch.cuh"
#include "k16_tma.cuh"

namespace k16 {
namespace {

constexpr int BN = 128;                  // keys per block, fetched together
constexpr int HN = 64;                   // keys per half block, the unit of S, P and the softmax
constexpr int THREADS = 384;            // three warpgroups: two of softmax, one of MMA (a warp per tile), copies and an idle warp
constexpr int W_MMA = 8, W_TMA = 10;
constexpr int REGS_SOFT = 216, REGS_REST = 72;   // 256 x 216 + 128 x 72 = 384 x 168, what the launch has
constexpr int MAX_HEADS = 128;           // q heads per item
constexpr float LAZY = 8.f;
constexpr int MAX_SPLIT = 32;            // pieces of a pair's key blocks
constexpr int SLOTS = 4 * 148;           // workspace slots at most: pieces of split pairs
constexpr int SPLIT_COST = 8;            // what a piece costs besides its blocks, in blocks: its start, its sums' way through the workspace

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
  // the pair's queries see nothing of [sinks, unseen)
  FR_DEVI int unseen(int window, int sinks) const { return Span(max(pos0, 0), window, sinks).lo; }
};
// the tokens of one tile, as positions [pa, pb]
struct Tile {
  int pa, pb, last, window, sinks;       // last: the last half block that the tile needs (2 k + half; -1: none)
  FR_DEVI Tile(const Item& it, int i, int tpt, int window_, int sinks_) : last(-1), window(window_), sinks(sinks_) {
    pa = it.pos0 + i * tpt;
    pb = min(it.pos0 + it.tok1 - it.tok0, pa + tpt) - 1;
    if (pb >= max(pa, 0))
      for (int k = 2 * it.k1 - 1; k >= 2 * it.k0 && last < 0; --k)
        if (needs(it.block(k >> 1) * BN + (k & 1) * HN)) last = k;
    if (last < 0) pb = -1;                                     // nothing in this item's blocks
  }
  // whether a query of the tile sees any of the HN keys from kh on, and whether all of them see them all
  FR_DEVI bool needs(int kh) const { return kh <= pb && (window <= 0 || kh + HN > pa - window + 1 || kh < sinks); }
  FR_DEVI bool whole(int kh) const { return kh + HN - 1 <= pa && (window <= 0 || kh > pb - window || kh + HN <= sinks); }
};

template <int D> struct Smem {
  static constexpr int QT = 128 * D * 2;                       // one query tile
  static constexpr int STAGE = BN * D * 2;                     // one K or V tile
  static constexpr int STAGES = D == 128 ? 5 : 10;
  static constexpr int RING = 2 * QT;
  static constexpr int BAR = RING + STAGES * STAGE;            // full[STAGES] empty[STAGES] qfull qempty sfull[2][2] pfull[2][2] ofull[2]
  static constexpr int NBAR = 2 * STAGES + 2 + 10 + 4 + 2 + 2;          // ... items: full[2], empty[2]; tile sync[2], pvdone[2]
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

// Operand descriptors in 128-byte swizzle as two words, of which only the low one (the address) changes: K-major with 1024
// bytes between groups of 8 rows; MN-major (V) with BN * 128 bytes between 64-dim chunks and 1024 between groups of 8 keys.
constexpr uint32_t DESC_HI = static_cast<uint32_t>((tc5::DESC_VERSION | tc5::DESC_SW128) >> 32) | (1024 >> 4);
constexpr uint32_t DESC_LO_K = 1u << 16, DESC_LO_MN = static_cast<uint32_t>(BN * 128 >> 4) << 16;
FR_DEVI uint32_t desc_lo(uint32_t saddr, uint32_t bits) { return bits | ((saddr & 0x3FFFFu) >> 4); }
FR_DEVI void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 x, y;\n setp.ne.b32 p, %4, 0;\n mov.b64 x, {%1, %5};\n mov.b64 y, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(id), "r"(accumulate), "n"(DESC_HI)
      : "memory");
}
FR_DEVI void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 y;\n setp.ne.b32 p, %4, 0;\n mov.b64 y, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(id), "r"(accumulate), "n"(DESC_HI)
      : "memory");
}
constexpr uint32_t A_NEGATE = 1u << 13, B_MN_MAJOR = 1u << 16;  // bits of the instruction descriptor

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
// the registers of an earlier tmem_ld32 hold their values from here on
FR_DEVI void ld_wait(uint32_t (&v)[32]) {
#define K16_RW4(o) "+r"(v[o]), "+r"(v[o + 1]), "+r"(v[o + 2]), "+r"(v[o + 3])
  asm volatile("tcgen05.wait::ld.sync.aligned;\n"
               : K16_RW4(0), K16_RW4(4), K16_RW4(8), K16_RW4(12), K16_RW4(16), K16_RW4(20), K16_RW4(24), K16_RW4(28)::"memory");
#undef K16_RW4
}
// scores of hidden keys -> -inf
FR_DEVI void hide(uint32_t (&v)[32], uint32_t see) {
#pragma unroll
  for (int e = 0; e < 32; ++e)
    if (!(see & (1u << e))) v[e] = 0xFF800000u;
}
// the n lowest of 32 bits
FR_DEVI uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; }

FR_DEVI float4 f4(const uint32_t* v) {
  return make_float4(__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2]), __uint_as_float(v[3]));
}
// 16 dims of an output row times inv (zeros when !any); wide: rows are 32-byte aligned, a whole sector per store (prompts through
// a window: 395 us with, 413 without; 4 x 512 over 32768, whose output is small: 1083 with, 1062 without)
template <int DT> FR_DEVI void put16(uint16_t* out, float4 x, float4 y, float4 z, float4 t, float inv, bool any, bool wide) {
  uint32_t v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (any) {
    v[0] = Elem<DT>::pack(x.x * inv, x.y * inv);
    v[1] = Elem<DT>::pack(x.z * inv, x.w * inv);
    v[2] = Elem<DT>::pack(y.x * inv, y.y * inv);
    v[3] = Elem<DT>::pack(y.z * inv, y.w * inv);
    v[4] = Elem<DT>::pack(z.x * inv, z.y * inv);
    v[5] = Elem<DT>::pack(z.z * inv, z.w * inv);
    v[6] = Elem<DT>::pack(t.x * inv, t.y * inv);
    v[7] = Elem<DT>::pack(t.z * inv, t.w * inv);
  }
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"l"(out), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
                 "r"(v[6]), "r"(v[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(out)[0] = make_uint4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<uint4*>(out)[1] = make_uint4(v[4], v[5], v[6], v[7]);
  }
}

template <int DT, int D>
__global__ void __launch_bounds__(THREADS, 1) k_prefill(const __grid_constant__ PrefillArgs a, const __grid_constant__ CUtensorMap qmap,
                                                        const __grid_constant__ CUtensorMap kvmap, int hb, int nhg, int box_rows,
                                                        int slots) {
  using S = Smem<D>;
  constexpr int STAGES = S::STAGES, HALVES = D / 64;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = static_cast<uint32_t>(__cvta_generic_to_shared(smem_raw));
  const uint32_t sm = (raw + 1023) & ~1023u;
  unsigned char* base = smem_raw + (sm - raw);
  const uint32_t full = sm + S::BAR, empty = full + 8 * STAGES, qfull = empty + 8 * STAGES, qempty = qfull + 8, sfull = qempty + 8,
                 pfull = sfull + 32, ofull = pfull + 32, ifull = ofull + 16, iempty = ifull + 16, tsync = iempty + 16, pvdone = tsync + 16;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(base + S::MISC);
  volatile uint32_t* abort = tmem_slot + 1;
  volatile uint32_t* flag = tmem_slot + 2;                     // [2]: this CTA joins the pieces of the tile
  Item* items = reinterpret_cast<Item*>(base + S::ITEMS);
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      tc5::mbar_init(full + 8 * i, 1);
      tc5::mbar_init(empty + 8 * i, 2);
    }
    tc5::mbar_init(qfull, 1);
    tc5::mbar_init(qempty, 2);
    for (int i = 0; i < 2; ++i) {
      tc5::mbar_init(sfull + 16 * i, 1);
      tc5::mbar_init(sfull + 16 * i + 8, 1);
      tc5::mbar_init(pvdone + 8 * i, 1);
      tc5::mbar_init(pfull + 16 * i, 4);
      tc5::mbar_init(pfull + 16 * i + 8, 4);
      tc5::mbar_init(ofull + 8 * i, 1);
      tc5::mbar_init(ifull + 8 * i, 1);
      tc5::mbar_init(tsync + 8 * i, 4);
      tc5::mbar_init(iempty + 8 * i, 10);
    }
    tc5::mbar_init_fence();
    *abort = 0;
    tma_prefetch_map(&qmap);
    tma_prefetch_map(&kvmap);
  }
  let_next_start();
  after_previous();
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
    // The list: all pairs; those of the last, partly filled wave are cut into `split` pieces by their key blocks (the number
    // that costs least: waves of pieces times a piece), each with a workspace slot, so that the whole grid ends together.
    long long pairs = 0;
    float all = 0.f;
    for (int b = lane; b < a.B; b += 32) {
      const int beg = min(max(a.cu_q[b], 0), a.T), end = min(max(a.cu_q[b + 1], beg), a.T), len = a.c.len(b);
      if (end == beg) continue;
      const int np = (end - beg + 2 * tpt - 1) / (2 * tpt);
      int x, y;
      pairs += static_cast<long long>(np) * Hv;
      all += 0.5f * (blocks(beg, end, len, x, y) + blocks(beg + (np - 1) * 2 * tpt, end, len, x, y)) * np * Hv;
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      pairs += __shfl_xor_sync(~0u, pairs, d);
      all += __shfl_xor_sync(~0u, all, d);
    }
    const int rest = static_cast<int>(pairs % gridDim.x);
    const long long whole = pairs - rest;
    int split = 1;
    if (rest > 0) {
      const int sp = lane + 1;                                 // lane i: i + 1 pieces
      const float avg = all / static_cast<float>(pairs), n = ceilf(fminf(avg, static_cast<float>(sp)));
      float cost = ceilf(rest * n / gridDim.x) * (avg / n + (sp > 1 ? SPLIT_COST : 0));
      if (rest * sp > slots || avg < 1.f) cost = sp == 1 ? 1e30f : INFINITY;
      float best = cost;
#pragma unroll
      for (int d = 16; d; d >>= 1) best = fminf(best, __shfl_xor_sync(~0u, best, d));
      split = __ffs(__ballot_sync(~0u, cost == best));
    }
    const long long units = whole + static_cast<long long>(rest) * split;
    // 32 sequences at a time: lane i has sequence r0 + i, its tokens, its pairs (times heads) and the pairs up to and with it
    int r0 = -32, beg = 0, end = 0;
    long long mine = 0, upto = 0, row0 = 0, group = 0;         // row0: pairs before the 32
    long long unit = blockIdx.x, before = -1;
    for (int ic = 0;; ++ic, unit += gridDim.x) {
      Item it;
      it.b = -1;
      const int extra = static_cast<int>(max(unit - whole, 0ll));
      const int part = rest > 0 ? extra / rest : 0;
      const long long idx = unit < whole ? unit : unit < units ? whole + extra - part * rest : pairs;
      if (idx < before) {                                      // the next pieces of the last pairs: from the front again
        r0 = -32;
        row0 = group = 0;
      }
      before = idx;
      while (r0 < a.B && idx >= row0 + group) {                // (indices only grow)
        row0 += group;
        r0 += 32;
        const int b = r0 + lane;
        beg = end = 0;
        if (b < a.B) {
          beg = min(max(a.cu_q[b], 0), a.T);
          end = min(max(a.cu_q[b + 1], beg), a.T);
        }
        mine = static_cast<long long>((end - beg + 2 * tpt - 1) / (2 * tpt)) * Hv;
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
        const int sbeg = __shfl_sync(~0u, beg, src), send = __shfl_sync(~0u, end, src);
        const int npairs = (send - sbeg + 2 * tpt - 1) / (2 * tpt);
        const int hv = off / npairs, pr = npairs - 1 - (off - hv * npairs);
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
        const int sp = unit < whole ? 1 : max(min(split, nblk), 1), chunk = (nblk + sp - 1) / sp;
        it.k0 = min(part * chunk, nblk);
        it.k1 = min(it.k0 + chunk, nblk);
        it.ns = nblk > 0 ? (nblk + chunk - 1) / chunk : 1;
        it.part = part;
        it.slot = extra;
        it.stride = rest;
        if (part > 0 && it.k0 >= nblk) {                       // a pair of fewer blocks than pieces
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
  } else if (w == W_MMA || w == W_MMA + 1) {                   // ------------------------------------- MMAs, a warp per tile
    // the softmax takes |qscale|: a negative scale negates the A operand
    const uint32_t ID_QK = tc5::idesc(1, DT == 0 ? 1 : 0, DT == 0 ? 1 : 0, 128, HN) | (a.qscale < 0.f ? A_NEGATE : 0u);
    constexpr uint32_t ID_PV = tc5::idesc(1, DT == 0 ? 1 : 0, DT == 0 ? 1 : 0, 128, D) | B_MN_MAJOR;
    const int i = w - W_MMA;
    const uint32_t tSi = tS + i * 128, tOi = tO + i * 128, qlo = desc_lo(sm + i * S::QT, DESC_LO_K), pf = pfull + 16 * i;
    int qc = 0, pc0 = 0, pc1 = 0;                              // query pairs and P halves consumed
    int st = 0, ph = 0;                                        // the ring's next tile: K(k0), V(k0), K(k0 + 1), ... of every item
    bool run = true;
    for (int ic = 0; run; ++ic) {
      const int sl = ic & 1;
      if (!k16_wait(ifull + 8 * sl, (ic / 2) & 1)) break;
      const Item it = items[sl];
      __syncwarp();
      if (lane == 0) tc5::mbar_arrive(iempty + 8 * sl);
      if (it.b < 0) break;
      if (it.k0 == it.k1) continue;
      const Tile t(it, i, tpt, a.window, a.sinks);
      if (!k16_wait(qfull, qc & 1)) break;
      ++qc;
      tc5::fence_after_sync();
      const int unseen = it.unseen(a.window, a.sinks);
      bool dirty = false;                                      // block k - 1 holds values that no query of the pair sees
      int was = 0;                                             // bit c: the tile needs half c of V(k - 1)
      uint32_t begun = 0;                                      // its O has begun
      int kbv = 0;                                             // first key of block k - 1
      for (int k = it.k0; k <= it.k1; ++k) {
        const int kb = k < it.k1 ? it.block(k) * BN : 0;
        const int now = k < it.k1 ? (t.needs(kb) ? 1 : 0) | (t.needs(kb + HN) ? 2 : 0) : 0;
        // Every tile of the ring is waited for, needed or not: the parity of a later phase would not tell.
        const uint32_t sv = sm + S::RING + st * S::STAGE, vlo = desc_lo(sv, DESC_LO_MN), vbar = empty + 8 * st;
        if (k > it.k0) {
          if (!(run = k16_wait(full + 8 * st, ph))) break;
          if (++st == STAGES) st = 0, ph ^= 1;
          // Values that no query of the pair sees become zeros, whatever the cache holds there: 0 * NaN would be NaN.  (Both
          // tiles' warps write them: the same zeros, each before its own product.)
          if (dirty) {
            int j0 = min(max(a.sinks - kbv, 0), BN), j1 = min(unseen - kbv, BN);   // behind the window, then behind the sequence
#pragma unroll 1
            for (int part = 0; part < 2; ++part) {
#pragma unroll 1
              for (int j = j0 * 8 + lane; j < j1 * 8; j += 32)
#pragma unroll
                for (int x = 0; x < HALVES; ++x)
                  asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};\n" ::"r"(sv + x * BN * 128 + j * 16), "r"(0) : "memory");
              j0 = min(it.len - kbv, BN);
              j1 = BN;
            }
            tc5::fence_async_smem();
            __syncwarp();
          }
        }
        const uint32_t klo = desc_lo(sm + S::RING + st * S::STAGE, DESC_LO_K), kbar = empty + 8 * st;
        if (k < it.k1) {
          if (!(run = k16_wait(full + 8 * st, ph))) break;
          if (++st == STAGES) st = 0, ph ^= 1;
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if ((was >> c & 1) && !(run = k16_wait(pf + 8 * c, (c ? pc1 : pc0) & 1))) break;
          tc5::fence_after_sync();
          if (tc5::elect_one()) {
            if (was >> c & 1) {
#pragma unroll
              for (int s = 0; s < HN / 16; ++s)
                mma_ts(tOi, tSi + HN * c + s * 8, vlo + (4 * c + s) * (2048 >> 4), ID_PV, s > 0 ? 1u : begun);
              tc5::mma_commit(pvdone + 8 * i);
              if (2 * (k - 1) + c == t.last) tc5::mma_commit(ofull + 8 * i);
            }
            if (now >> c & 1) {
#pragma unroll
              for (int s = 0; s < D / 16; ++s)
                mma_ss(tSi + HN * c, qlo + (((s >> 2) * 128 * 128 + (s & 3) * 32) >> 4),
                       klo + (((s >> 2) * BN * 128 + c * HN * 128 + (s & 3) * 32) >> 4), ID_QK, s > 0);
              tc5::mma_commit(sfull + 16 * i + 8 * c);
            }
            if (c == 1) {                                      // (a commit without products before it arrives at once)
              if (k > it.k0) tc5::mma_commit(vbar);
              if (k < it.k1) tc5::mma_commit(kbar);
              if (k == it.k1 - 1) tc5::mma_commit(qempty);     // after this tile's last product with Q, whichever it was
            }
          }
          __syncwarp();
          if (was >> c & 1) begun = 1, c ? ++pc1 : ++pc0;
        }
        if (!run) break;
        was = now, kbv = kb;
        dirty = now && (kb + BN > it.len || kb < unseen);
      }
    }
  } else {                                                     // --------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(REGS_SOFT));
    const int i = w >> 2, r = tid & 127, tok = r / hb, head = r - tok * hb;
    const uint32_t lanes = static_cast<uint32_t>(w & 3) << 21;  // tensor-memory lanes of this warp
    const uint32_t ts = tS + i * 128 + lanes, to = tO + i * 128 + lanes;
    const float qs = fmaxf(fabsf(a.qscale), 1e-37f);           // a scale of 0: all scores alike, and -inf * qs stays -inf
    constexpr float BIAS = DT == 1 ? 6.f : 0.f;                // fp16 weights are carried times 2^6: their steps below 2^-14 are absolute
    const bool wide = ((reinterpret_cast<uintptr_t>(a.out) | static_cast<uintptr_t>(2 * a.o_ts)) & 31) == 0;
    int syncs = 0;
    const auto tile_sync = [&]() {                             // the softmax warps of a tile (bounded, unlike a named barrier)
      __syncwarp();
      if (lane == 0) tc5::mbar_arrive(tsync + 8 * i);
      return k16_wait(tsync + 8 * i, syncs++ & 1);
    };
    int sc[2] = {0, 0}, oc = 0;                                // S halves and O tiles consumed
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
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int kh = kb + HN * c;
          if (!t.needs(kh)) continue;
          const bool whole = t.whole(kh);
          if (!(run = k16_wait(sfull + 16 * i + 8 * c, sc[c] & 1))) break;
          ++sc[c];
          tc5::fence_after_sync();
          uint32_t v[2][32];
          tc5::tmem_ld32(ts + HN * c, v[0]);
          tc5::tmem_ld32(ts + HN * c + 32, v[1]);
          ld_wait(v[0]);
          ld_wait(v[1]);
          if (__builtin_expect(!whole, 0)) {
            const int hi = pos + 1 - kh, lo = a.window > 0 ? pos - a.window + 1 - kh : 0, sk = a.sinks - kh;
#pragma unroll
            for (int d = 0; d < 2; ++d) hide(v[d], low_bits(hi - 32 * d) & (~low_bits(lo - 32 * d) | low_bits(sk - 32 * d)));
          }
          float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            m0 = max3(m0, __uint_as_float(v[0][e]), __uint_as_float(v[0][e + 1]));
            m1 = max3(m1, __uint_as_float(v[0][e + 2]), __uint_as_float(v[0][e + 3]));
            m2 = max3(m2, __uint_as_float(v[1][e]), __uint_as_float(v[1][e + 1]));
            m3 = max3(m3, __uint_as_float(v[1][e + 2]), __uint_as_float(v[1][e + 3]));
          }
          const float m = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)) * qs;
          if (__builtin_expect(__any_sync(~0u, m > ref + LAZY), 0)) {
            const float nr = fmaxf(m, ref), f = ref == -INFINITY ? 0.f : ex2(ref - nr);
            const bool some = l > 0.f;                         // (a row that has seen a key has a sum of about 1 at least)
            l *= f;
            ref = nr;
            if (__any_sync(~0u, some)) {                       // O holds the products of every earlier half; the next ones wait for this P
              if (!(run = k16_wait(pvdone + 8 * i, (sc[0] + sc[1]) & 1))) break;
              tc5::fence_after_sync();
#pragma unroll 1
              for (int d = 0; d < D / 32; ++d) {
                uint32_t o[32];
                tc5::tmem_ld32(to + 32 * d, o);
                tc5::tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tc5::tmem_st32(to + 32 * d, o);
              }
            }
          }
          const float off = (ref == -INFINITY ? 0.f : -ref) + BIAS;
          const uint64_t q2 = pk(qs, qs), off2 = pk(off, off);
          uint64_t sum[4] = {0, 0, 0, 0};
          uint32_t p[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float2 y = un(fma2(pk(__uint_as_float(v[e >> 4][2 * (e & 15)]), __uint_as_float(v[e >> 4][2 * (e & 15) + 1])), q2, off2));
            const float p0 = ex2(y.x), p1 = ex2(y.y);
            sum[e & 3] = add2(sum[e & 3], pk(p0, p1));
            p[e] = Elem<DT>::pack(p0, p1);
          }
          tc5::tmem_st32(ts + HN * c, p);                      // over scores that have been read
          const float2 l2 = un(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])));
          l += l2.x + l2.y;
          tc5::tmem_st_wait();
          tc5::fence_before_sync();
          __syncwarp();
          if (lane == 0) tc5::mbar_arrive(pfull + 16 * i + 8 * c);
        }
        if (!run) break;
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
            for (int e = 0; e < 32; e += 16)
              put16<DT>(out + 32 * c + e, f4(o + e), f4(o + e + 4), f4(o + e + 8), f4(o + e + 12), inv, any && inv != 0.f, wide);
          }
          __syncwarp();
        }
      } else {
        // this piece's sums to its slot, [dims / 4][row] x 16 bytes; the last piece of the tile to arrive joins them in order
        const int rr = i * (D / 4) * 128 + r;
        float4* po = reinterpret_cast<float4*>(a.ws) + static_cast<long long>(it.slot) * (2 * (D / 4) * 128) + rr;
        float2* pl = reinterpret_cast<float2*>(a.ws + static_cast<long long>(slots) * (2 * D * 128 * 4));
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
        if (!(run = tile_sync())) break;
        const int slot0 = it.slot - it.part * it.stride;
        if (r == 0) {
          int* tk = a.tickets + 2 * slot0 + i;
          const int old = atomicAdd(tk, 1);
          if (old == it.ns - 1) *tk = 0;
          flag[i] = old == it.ns - 1;
          __threadfence();
        }
        if (!(run = tile_sync())) break;
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
          for (int c = 0; c < D / 4; c += 4) {                 // 16 dims of four pieces in flight
            float4 acc[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int s = 0; s < it.ns; s += 4) {
              float4 x[4][4];
              float f[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const bool in = s + q < it.ns;
                const float2 e2 = in ? __ldcg(ml + static_cast<long long>((s + q) * it.stride) * 256) : make_float2(0.f, 0.f);
                const bool use = in && e2.y != 0.f;            // (0: the piece has no key that this row sees)
                f[q] = use ? ex2(e2.x - M) : 0.f;
                const float4* src = pq + static_cast<long long>((s + q) * it.stride) * (2 * (D / 4) * 128) + c * 128;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[q][e] = use ? __ldcg(src + e * 128) : make_float4(0.f, 0.f, 0.f, 0.f);
              }
#pragma unroll
              for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  acc[e].x = fmaf(f[q], x[q][e].x, acc[e].x);
                  acc[e].y = fmaf(f[q], x[q][e].y, acc[e].y);
                  acc[e].z = fmaf(f[q], x[q][e].z, acc[e].z);
                  acc[e].w = fmaf(f[q], x[q][e].w, acc[e].w);
                }
            }
            if (live) put16<DT>(out + 4 * c, acc[0], acc[1], acc[2], acc[3], inv, inv != 0.f, wide);
          }
          __syncwarp();
        }
        if (!(run = tile_sync())) break;                       // (the flag is free again)
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
cudaError_t launch_p(const PrefillArgs& a, const CUtensorMap& qm, const CUtensorMap& kv, int hb, int nhg, int box, int slots, int dev, int grid, cudaStream_t st) {
  const auto k = k_prefill<DT, D>;
  static std::atomic<bool> done[MAX_DEVICES];
  if (cudaError_t e = allow_smem(k, Smem<D>::TOTAL, dev, done)) return e;
  return launch(k, grid, THREADS, Smem<D>::TOTAL, 0, st, a, qm, kv, hb, nhg, box, slots);
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
static int max_slots(int rows, int Hkv, int G, long long new_tokens) {
  const long long n = max_pairs(rows, Hkv, G, new_tokens) * MAX_SPLIT;
  return static_cast<int>(n < SLOTS ? n : SLOTS);
}
// sums, then (reference, denominator), of every slot
long long prefill_ws_bytes(int rows, int Hkv, int G, int D, long long new_tokens) {
  return static_cast<long long>(max_slots(rows, Hkv, G, new_tokens)) * 256 * (D * 4 + 8);
}
long long prefill_tickets(int rows, int Hkv, int G, long long new_tokens) { return 2 * max_slots(rows, Hkv, G, new_tokens); }

int prefill_status() {
  int v = -1;
  return cudaMemcpyFromSymbol(&v, g_status, sizeof(v)) == cudaSuccess ? v : -1;
}

cudaError_t prefill(int dtype, const PrefillArgs& a, cudaStream_t st) {
  int dev = 0, sms = 0;
  cudaError_t e = device_sms(dev, sms);
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
  const int grid = static_cast<int>(items < sms ? items : sms), slots = max_slots(a.B, a.c.Hkv, a.G, a.T);
  if (dtype == 0)
    return a.D == 128 ? launch_p<0, 128>(a, qm, kv, hb, nhg, box, slots, dev, grid, st) : launch_p<0, 64>(a, qm, kv, hb, nhg, box, slots, dev, grid, st);
  return a.D == 128 ? launch_p<1, 128>(a, qm, kv, hb, nhg, box, slots, dev, grid, st) : launch_p<1, 64>(a, qm, kv, hb, nhg, box, slots, dev, grid, st);
}

}  // namespace k16
