// host-side launchers of the 16-bit cache kernels, called by k16_capi.cu after it has checked the arguments
#pragma once
#include <cuda_runtime.h>

#include "k16_common.cuh"

namespace k16 {

struct AttnArgs {
  Cache c;
  const void* q;
  long long q_bs;
  int B, G, D;
  float qscale;
  int window, sinks;
  float* weights;                   // may be null
  long long w_bs, w_hs;
  int* tickets;
  unsigned char* ws;
  void* out;
  long long o_bs;
};
struct PrefillArgs {
  Cache c;
  const void* q;
  long long q_ts;
  int T;
  const int* cu_q;
  int B, G, D;
  float qscale;
  int window, sinks;
  int* tickets;
  unsigned char* ws;
  void* out;
  long long o_ts;
};
struct EvictArgs {
  Cache c;
  int B, D;
  const float* weights;
  long long w_bs, w_hs;
  int w_len, budget, sinks, recent;
  int* kept;
  int* new_lens;
  float* new_weights;
  int nw_len;
  uint16_t* dst;                    // == c.pool when in place
  long long dst_pages;
  const int* dst_bt;                // null: in place
  long long dst_stride;
};

cudaError_t write_rows(const uint16_t* kv, long long kv_ts, long long kv_hs, const long long* slots, int T, int Hkv, int D,
                       int page_sh, long long num_pages, uint16_t* pool, cudaStream_t st);
long long attn_ws_bytes(int rows, int Hkv, int G, int D, long long max_len, int weights);
cudaError_t attn(int dtype, const AttnArgs& a, cudaStream_t st);
int decode_status();
long long prefill_ws_bytes(int rows, int Hkv, int G, int D, long long new_tokens);
long long prefill_tickets(int rows, int Hkv, int G, long long new_tokens);
cudaError_t prefill(int dtype, const PrefillArgs& a, cudaStream_t st);
int prefill_status();
cudaError_t evict(const EvictArgs& a, cudaStream_t st);

}  // namespace k16
