// C ABI of libflagrot_kv16.so: argument checks and dispatch (contract in include/flagrot_kv16.h).
#include "../../include/flagrot_kv16.h"

#include <climits>

#include "k16_kernels.h"

using namespace k16;

namespace {
thread_local char g_err[256];

int fail(cudaError_t e) {
  if (e == cudaSuccess) return 0;
  const char* s = cudaGetErrorString(e);
  int i = 0;
  for (; s[i] && i < 255; ++i) g_err[i] = s[i];
  g_err[i] = 0;
  cudaGetLastError();
  return -1;
}
bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
int page_shift(int page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : page == 128 ? 7 : -1; }
// a cache the kernels can index: pool rows below 2^31 (tensor-map coordinates), positions below 2^30
int check_cache(const void* pool, long long num_pages, const int* bt, long long bt_stride, int bt_width, const int* lens, int B,
                int Hkv, int D, int page) {
  if ((D != 64 && D != 128) || page_shift(page) < 0) return -2;
  if (B < 0 || Hkv < 1 || Hkv > 4096 || num_pages < 1 || bt_width < 0 || bt_stride < 0) return -3;
  if (static_cast<long long>(bt_width) * page > (1 << 30)) return -3;
  if (num_pages > (static_cast<long long>(INT_MAX) / 2) / (static_cast<long long>(Hkv) * page)) return -3;
  if (B > 0 && (!pool || !al16(pool) || !lens || (bt_width > 0 && !bt))) return -3;
  return 0;
}
// whether the n 4-byte entries at x share any with `rows` rows of `width` such entries, `stride` entries apart, at p
bool meets(const void* x, long long n, const void* p, long long rows, long long stride, long long width) {
  const long long a = static_cast<long long>(reinterpret_cast<uintptr_t>(x)) - static_cast<long long>(reinterpret_cast<uintptr_t>(p));
  if (!p || n <= 0 || rows <= 0 || width <= 0) return false;
  if (stride <= width) {                                 // no gaps: one row
    width += (rows - 1) * stride;
    rows = 1;
    stride = width;
  }
  const long long k = a < 4 * width ? 0 : (a - 4 * width) / (4 * stride) + 1;   // the first row that ends behind a
  return k < rows && 4 * k * stride < a + 4 * n;
}
Cache make_cache(const void* pool, long long num_pages, const int* bt, long long bt_stride, int bt_width, const int* lens, int Hkv,
                 int page) {
  Cache c;
  c.pool = static_cast<const uint16_t*>(pool);
  c.num_pages = num_pages;
  c.bt = bt;
  c.bt_stride = bt_stride;
  c.bt_width = bt_width;
  c.seq_lens = lens;
  c.Hkv = Hkv;
  c.page_sh = page_shift(page);
  return c;
}
}  // namespace

extern "C" {

int k16_abi_version(void) { return 1; }
const char* k16_last_error(void) { return g_err; }
int k16_device_status(void) {
  if (fail(cudaDeviceSynchronize())) return -1;   // the copies below do not wait for non-blocking streams
  const int d = decode_status();
  return d ? d : prefill_status();
}
int k16_chunk_bytes(int page, int D) { return 4 * page * D; }

int k16_write(const void* kv, long long kv_ts, long long kv_hs, const long long* slots, int T, int Hkv, int D, int page,
              long long num_pages, void* pool, void* stream) {
  if ((D != 64 && D != 128) || page_shift(page) < 0) return -2;
  if (T < 0 || Hkv < 1 || Hkv > 4096 || num_pages < 1) return -3;
  if (num_pages > (static_cast<long long>(INT_MAX) / 2) / (static_cast<long long>(Hkv) * page)) return -3;
  if (T == 0) return 0;
  if (!kv || !slots || !pool || !al16(kv) || !al16(pool) || kv_ts % 8 || kv_hs % 8) return -3;
  return fail(write_rows(static_cast<const uint16_t*>(kv), kv_ts, kv_hs, slots, T, Hkv, D, page_shift(page), num_pages,
                         static_cast<uint16_t*>(pool), static_cast<cudaStream_t>(stream)));
}

long long k16_ws_bytes(int rows, int Hkv, int G, int D, long long max_len, int weights, long long new_tokens) {
  if (rows < 0 || Hkv < 1 || G < 1 || G > 4096 || (D != 64 && D != 128) || max_len < 0 || new_tokens < 0) return -3;
  const long long a = attn_ws_bytes(rows, Hkv, G, D, max_len, weights);
  const long long p = new_tokens > 0 ? prefill_ws_bytes(rows, Hkv, G, D, new_tokens) : 0;
  return a > p ? a : p;
}
long long k16_ws_tickets(int rows, int Hkv, int G, long long new_tokens) {
  if (rows < 0 || Hkv < 1 || G < 1 || G > 4096 || new_tokens < 0) return -3;
  const long long a = static_cast<long long>(rows) * Hkv * G;
  const long long p = new_tokens > 0 ? prefill_tickets(rows, Hkv, G, new_tokens) : 0;
  return a > p ? a : p;
}

int k16_attn(int dtype, const void* q, long long q_bs, const void* pool, long long num_pages, const int* block_table,
             long long bt_stride, int bt_width, const int* seq_lens, int B, int Hkv, int G, int D, int page, float qscale,
             int window, int sinks, float* weights, long long w_bs, long long w_hs, int* tickets, long long n_tickets, void* ws,
             long long ws_bytes, void* out, long long o_bs, void* stream) {
  if (dtype != 0 && dtype != 1) return -2;
  if (int rc = check_cache(pool, num_pages, block_table, bt_stride, bt_width, seq_lens, B, Hkv, D, page)) return rc;
  if (G < 1 || G > 4096 || sinks < 0 || static_cast<long long>(B) * Hkv * G > (1 << 28)) return -3;
  if (B == 0) return 0;
  if (!q || !out || !al16(q) || !al16(out) || q_bs % 8 || o_bs % 8) return -3;
  // rows that are written must not be one another's
  if (B > 1 && o_bs < static_cast<long long>(Hkv) * G * D) return -3;
  if (weights && (w_bs < 0 || w_hs < 0 || (B > 1 && w_bs == 0) || (Hkv > 1 && w_hs == 0))) return -3;
  if (!tickets || !ws || !al16(ws) || n_tickets < k16_ws_tickets(B, Hkv, G, 0) ||
      ws_bytes < attn_ws_bytes(B, Hkv, G, D, static_cast<long long>(bt_width) * page, weights != nullptr))
    return -4;
  AttnArgs a;
  a.c = make_cache(pool, num_pages, block_table, bt_stride, bt_width, seq_lens, Hkv, page);
  a.q = q;
  a.q_bs = q_bs;
  a.B = B;
  a.G = G;
  a.D = D;
  a.qscale = qscale;
  a.window = window < (1 << 30) ? window : 1 << 30;    // positions are below 2^30
  a.sinks = sinks < (1 << 30) ? sinks : 1 << 30;
  a.weights = weights;
  a.w_bs = w_bs;
  a.w_hs = w_hs;
  a.tickets = tickets;
  a.ws = static_cast<unsigned char*>(ws);
  a.out = out;
  a.o_bs = o_bs;
  return fail(attn(dtype, a, static_cast<cudaStream_t>(stream)));
}

int k16_prefill(int dtype, const void* q, long long q_ts, int T, const int* cu_q, const void* pool, long long num_pages,
                const int* block_table, long long bt_stride, int bt_width, const int* seq_lens, int B, int Hkv, int G, int D,
                int page, float qscale, int window, int sinks, int* tickets, long long n_tickets, void* ws, long long ws_bytes,
                void* out, long long o_ts, void* stream) {
  if (dtype != 0 && dtype != 1) return -2;
  if (int rc = check_cache(pool, num_pages, block_table, bt_stride, bt_width, seq_lens, B, Hkv, D, page)) return rc;
  if (G < 1 || G > 4096 || sinks < 0 || T < 0 || static_cast<long long>(T) * Hkv * G > INT_MAX / 2) return -3;
  if (B == 0 || T == 0) return 0;
  if (!q || !out || !cu_q || !al16(q) || !al16(out) || q_ts % 8 || o_ts % 8) return -3;
  if (T > 1 && (q_ts < 1 || o_ts < static_cast<long long>(Hkv) * G * D)) return -3;
  if (!tickets || !ws || !al16(ws) || n_tickets < prefill_tickets(B, Hkv, G, T) || ws_bytes < prefill_ws_bytes(B, Hkv, G, D, T))
    return -4;
  PrefillArgs a;
  a.c = make_cache(pool, num_pages, block_table, bt_stride, bt_width, seq_lens, Hkv, page);
  a.q = q;
  a.q_ts = q_ts;
  a.T = T;
  a.cu_q = cu_q;
  a.B = B;
  a.G = G;
  a.D = D;
  a.qscale = qscale;
  a.window = window < (1 << 30) ? window : 1 << 30;    // positions are below 2^30
  a.sinks = sinks < (1 << 30) ? sinks : 1 << 30;
  a.tickets = tickets;
  a.ws = static_cast<unsigned char*>(ws);
  a.out = out;
  a.o_ts = o_ts;
  return fail(prefill(dtype, a, static_cast<cudaStream_t>(stream)));
}

int k16_evict(const void* pool, long long num_pages, const int* block_table, long long bt_stride, int bt_width,
              const int* seq_lens, int B, int Hkv, int D, int page, const float* weights, long long w_bs, long long w_hs,
              int w_len, int budget, int sinks, int recent, int* kept, int* new_lens, float* new_weights, int nw_len,
              void* dst_pool, long long dst_pages, const int* dst_table, long long dst_stride, int dst_width, void* stream) {
  if (int rc = check_cache(pool, num_pages, block_table, bt_stride, bt_width, seq_lens, B, Hkv, D, page)) return rc;
  if (budget < 1 || budget > (1 << 30) || sinks < 0 || recent < 0 || static_cast<long long>(sinks) + recent > budget) return -3;
  if (w_len < 0 || w_bs < 0 || w_hs < 0 || nw_len < budget || static_cast<long long>(B) * Hkv > 65535 * 16ll) return -3;
  if (B == 0) return 0;
  if ((w_len > 0 && !weights) || !kept || !new_lens || !new_weights) return -3;
  EvictArgs a;
  a.dst = static_cast<uint16_t*>(dst_pool);
  a.dst_pages = dst_pages;
  a.dst_bt = dst_table;
  a.dst_stride = dst_stride;
  if (dst_table) {
    if (!dst_pool || !al16(dst_pool) || dst_pages < 1 || dst_stride < 0 || dst_width < 0) return -3;
    if (static_cast<long long>(dst_width) * page < budget || (B > 1 && dst_stride < dst_width)) return -3;
    if (dst_pages > (static_cast<long long>(INT_MAX) / 2) / (static_cast<long long>(Hkv) * page)) return -3;
  } else {
    if (B > 1 && bt_stride < bt_width) return -3;        // rows that share their table would move each other's tokens
    a.dst = static_cast<uint16_t*>(const_cast<void*>(pool));
    a.dst_pages = num_pages;
  }
  // Some CTAs write results while others still read the inputs (a row's heads and a cluster's CTAs run apart).
  const long long groups = static_cast<long long>(B) * Hkv, w_span = w_len > 0 ? (B - 1) * w_bs + (Hkv - 1) * w_hs + w_len : 0;
  const void* result[3] = {kept, new_lens, new_weights};
  const long long count[3] = {groups * budget, B, groups * nw_len};
  for (int i = 0, j = 1; i < 3; ++i, j = (j + 1) % 3)
    if (meets(result[i], count[i], seq_lens, 1, B, B) || meets(result[i], count[i], weights, 1, w_span, w_span) ||
        meets(result[i], count[i], block_table, B, bt_stride, bt_width) ||
        meets(result[i], count[i], dst_table, B, dst_stride, dst_width) || meets(result[i], count[i], result[j], 1, count[j], count[j]))
      return -3;
  a.c = make_cache(pool, num_pages, block_table, bt_stride, bt_width, seq_lens, Hkv, page);
  a.B = B;
  a.D = D;
  a.weights = weights;
  a.w_bs = w_bs;
  a.w_hs = w_hs;
  a.w_len = w_len;
  a.budget = budget;
  a.sinks = sinks;
  a.recent = recent;
  a.kept = kept;
  a.new_lens = new_lens;
  a.new_weights = new_weights;
  a.nw_len = nw_len;
  return fail(evict(a, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
