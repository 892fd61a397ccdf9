/* C ABI of libflagrot_kv16.so for NVIDIA B200 (sm_100a), ABI version 1: the 16-bit paged key-value cache.
 *
 * The cache of layers that are not quantised (sliding-window layers, first / last layers, the uncompressed arm a quantised
 * format is compared with), beside the quantised pages of the other libraries.  No counterpart in the reference's C ABI.
 *
 * Pool: [num_pages, Hkv, 2, page, D] elements of one 16-bit type, contiguous, 16-byte aligned: per (page, kv head) the keys
 * of `page` tokens, then their values.  dtype 0 bf16, 1 fp16; D 64 | 128; page 16 | 32 | 64 | 128; any GQA group G.
 * Block tables int32 [B, bt_width] (row stride bt_stride elements, 0: every row reads row 0); an entry outside
 * [0, num_pages) reads as a page of zeros.  seq_lens int32 [B], taken as min(max(len, 0), bt_width * page).
 * What lies in a page behind a sequence's length is never used, whatever it holds (NaN included).
 *
 * Every entry takes raw DEVICE pointers, element strides and the caller's cudaStream_t (as void*); launches are
 * asynchronous, allocate nothing and may be captured in CUDA graphs (after a first call on the device outside a capture, which
 * loads the kernels).  The stream must belong to the current device.
 * Return: 0 ok, -1 launch error (text in k16_last_error), -2 unsupported dtype / head dim / page, -3 bad argument (null or
 * misaligned pointer, negative or too large size), -4 workspace too small.  Nothing is launched when the code is not 0. */
#ifndef FLAGROT_KV16_H
#define FLAGROT_KV16_H
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

int k16_abi_version(void);
const char* k16_last_error(void);
/* 0, or the source line of a bounded device-side wait that gave up (sticky); -1 when the device cannot be asked.  Waits for
 * everything launched on the current device, on every stream: not during a capture. */
int k16_device_status(void);
/* bytes per (page, kv head): 4 * page * D */
int k16_chunk_bytes(int page, int D);

/* Appends rows: kv [T, 2*Hkv, D] (K rows of all heads, then V rows; token stride kv_ts, row stride kv_hs elements, both
 * multiples of 8, 16-byte aligned) -> pool at slots int64 [T] (slot = page_id * page + offset; outside [0, num_pages * page)
 * skipped).  The slots that are written must be distinct. */
int k16_write(const void* kv, long long kv_ts, long long kv_hs, const long long* slots, int T, int Hkv, int D, int page,
              long long num_pages, void* pool, void* stream);

/* Workspace of k16_attn / k16_prefill (-3: bad argument): bytes for up to `rows` sequences of up to max_len cached tokens; weights != 0 when
 * k16_attn is called with weights; new_tokens: the largest T of k16_prefill (0: k16_attn only).  tickets: int32, zero before
 * the first call, left zero by every call (a workspace whose call's wait gave up is void).  Calls that may overlap on the device
 * need workspaces of their own. */
long long k16_ws_bytes(int rows, int Hkv, int G, int D, long long max_len, int weights, long long new_tokens);
long long k16_ws_tickets(int rows, int Hkv, int G, long long new_tokens);

/* Attention of one new token per row.  q [B, G*Hkv, D] (row stride q_bs elements), key j of row b is visible when j < len
 * and (window <= 0 or j >= len - window or j < sinks); qscale = softmax scale * log2(e); out [B, G*Hkv*D] (row stride
 * o_bs); q and out rows 16-byte aligned.  A row that sees no key, or only keys whose score is -inf, is written as zeros (and adds
 * nothing to weights); beside others a key whose score is -inf has weight 0.  The same in k16_prefill.
 * weights fp32 (or null): weights[b * w_bs + h * w_hs + j] += the softmax weights of visible key j summed over the G heads of
 * kv head h; other entries are left as they are.  Each row needs at least bt_width * page entries, rows of its own. */
int k16_attn(int dtype, const void* q, long long q_bs, const void* pool, long long num_pages, const int* block_table,
             long long bt_stride, int bt_width, const int* seq_lens, int B, int Hkv, int G, int D, int page, float qscale,
             int window, int sinks, float* weights, long long w_bs, long long w_hs, int* tickets, long long n_tickets, void* ws,
             long long ws_bytes, void* out, long long o_bs, void* stream);

/* Attention of many new tokens per row, which are the last ones of their sequences and whose rows are in the pages already.
 * q [T, G*Hkv, D] (row stride q_ts), row b's tokens at [cu_q[b], cu_q[b + 1]) (int32 [B + 1], ascending, taken within
 * [0, T]); token i of n is at position p = len - n + i and sees key j <= p when (window <= 0 or j > p - window or j < sinks);
 * out [T, G*Hkv*D] (row stride o_ts).  A token that sees no key (p < 0) is written as zeros; rows of out that belong to no
 * sequence are left as they are.  The softmax weights meet the values in the pool's type (a rounding each, beside the output's
 * own; sums are 32-bit), where k16_attn keeps them to 2^-17.  Rows that none of the sequence's new tokens sees (behind the window of the first of them and
 * not sinks) may hold anything, and their pages may belong to others by now; the values of rows that some of them see must be
 * finite (a weight of 0 times infinity is NaN: the sums run over whole blocks). */
int k16_prefill(int dtype, const void* q, long long q_ts, int T, const int* cu_q, const void* pool, long long num_pages,
                const int* block_table, long long bt_stride, int bt_width, const int* seq_lens, int B, int Hkv, int G, int D,
                int page, float qscale, int window, int sinks, int* tickets, long long n_tickets, void* ws, long long ws_bytes,
                void* out, long long o_ts, void* stream);

/* Evicts: of every (row, kv head) with more than `budget` cached tokens keeps the first `sinks`, the last `recent` and, of
 * the others, the budget - sinks - recent with the largest weights (ties: the lower position; NaN counts as the smallest),
 * in their order.  weights fp32 as in k16_attn, of w_len entries per row; len is taken within w_len (the newest tokens of a row
 * that is longer are dropped).
 * kept int32 [B, Hkv, budget]: the kept positions, then -1; new_lens int32 [B] = min(len, w_len, budget); new_weights fp32
 * [B, Hkv, nw_len] (contiguous, nw_len >= budget): the kept tokens' weights, then zeros.  The three results overlap neither one
 * another nor seq_lens, weights (from their first entry to their last) and the tables: -3 otherwise.
 * dst_table null: the kept rows move to the front of the row's own pages (no page may belong to two rows).  Else they are
 * copied to the pages of dst_table [B, dst_width] in dst_pool (distinct pages, dst_width * page >= budget; entries outside
 * [0, dst_pages) are not written), which share no page with the ones that are read; slots behind the kept rows are left as
 * they are. */
int k16_evict(const void* pool, long long num_pages, const int* block_table, long long bt_stride, int bt_width,
              const int* seq_lens, int B, int Hkv, int D, int page, const float* weights, long long w_bs, long long w_hs,
              int w_len, int budget, int sinks, int recent, int* kept, int* new_lens, float* new_weights, int nw_len,
              void* dst_pool, long long dst_pages, const int* dst_table, long long dst_stride, int dst_width, void* stream);

#ifdef __cplusplus
}
#endif
#endif
