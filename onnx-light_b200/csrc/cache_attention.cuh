// Shared by the kernels of b2_cache_attention: attention over a paged 8-bit KV cache.
#pragma once
#include "quant8.cuh"

namespace b2 {

struct CaArgs {
  const void *q;
  void *y;
  int64_t q_b, q_h, q_s; // strides (elements) of Q and Y over batch, head, position
  const uint8_t *k, *v;  // [pages, Hkv, T, D] codes
  const float *ks, *vs;  // [pages, Hkv]
  const int32_t *table, *lengths, *counts;
  int64_t pages;
  int B, Hq, Hkv, group, S, T, D, max_pages;
  int causal, window, sinks; // window -1: unbounded
  float scale;               // of Q.K
  float softcap;             // <= 0: none
};

constexpr float kLog2E = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Tokens before the call and new ones of sequence b, brought into the table's range; *bad tells
// that they were not (the kernels record it for b2_kernel_status).
struct CaSpan {
  int past, count, total; // total = past + count: keys the sequence has
};
__device__ __forceinline__ CaSpan ca_span(const CaArgs &a, int b, bool *bad) {
  const int64_t room = (int64_t)a.max_pages * a.T;
  int64_t p = a.lengths[b], n = a.counts ? a.counts[b] : a.S;
  *bad = p < 0 || n < 0 || n > a.S || p + n > room;
  p = min(max(p, (int64_t)0), room);
  n = min(min(max(n, (int64_t)0), (int64_t)a.S), room - p);
  return CaSpan{(int)p, (int)n, (int)(p + n)};
}

// Whether the query at position p sees key j (j < total is checked by the caller).
__device__ __forceinline__ bool ca_sees(const CaArgs &a, int p, int j) {
  if (!a.causal) return true;
  return j <= p && (a.window < 0 || p - j <= a.window || j < a.sinks);
}

// Few query rows, keys split over the GPU (cache_attention_split.cu).
bool cache_attn_split_eligible(const CaArgs &a);
size_t cache_attn_split_workspace(const CaArgs &a);
int cache_attn_split_launch(const CaArgs &a, bool f16, bool f8, void *ws, cudaStream_t st);

// Prompts on tcgen05 (cache_attention_prefill.cu).
bool cache_attn_prefill_eligible(const CaArgs &a);
size_t cache_attn_prefill_workspace(const CaArgs &a);
int cache_attn_prefill_launch(const CaArgs &a, bool f16, bool f8, void *ws, cudaStream_t st);

} // namespace b2
