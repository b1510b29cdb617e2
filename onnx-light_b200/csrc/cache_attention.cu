// Attention over a paged 8-bit KV cache (b2_cache_attention): checks, the choice of the kernel,
// and the kernel for every shape the others do not take.
//
//   y_i = sum_j softmax_j(scale q_i . k_j) v_j,  k_j = code * k_scale[page, head], same for v,
//   over the keys j the query at position p = length + i sees: j <= p and, with a window,
//   p - j <= window or j < sink_tokens.  A query that sees no key, or i >= new_length, gives 0.
//
// cache_attn_any: one warp owns one (sequence, query head, query).  32 keys at a time each lane
// scores one key (fp32), the warp keeps a running maximum and sum, and the lanes then own the head's
// columns for P.V.  It reads a key's codes byte by byte and shares nothing between the heads of a
// group: right for any head size, page size and alignment, bound by its own loads (32 sequences of up to
// 8192 tokens, 32 / 8 heads of 128, pages of 12: 15.7 ms).
#include "cache_attention.cuh"

namespace b2 {

int check_quantized_cache(const char *op, const b2_quantized_cache *c, const b2_tensor *counts);

// 1: a length, a count or a page number was out of range.
__device__ int g_cache_attention_status;

namespace {

using namespace q8;

constexpr int CAA_WARPS = 4;
constexpr int CAA_DMAX = 512;
constexpr float CAA_DOWN = 0x1p-24f; // of what is summed: the sum of large values passes FLOAT's range before their mean

template <typename T, typename Q>
__global__ void __launch_bounds__(CAA_WARPS * 32) cache_attn_any(const CaArgs a) {
  __shared__ float qs[CAA_WARPS][CAA_DMAX];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t u = (int64_t)blockIdx.x * CAA_WARPS + warp;
  if (u >= (int64_t)a.B * a.Hq * a.S) return;
  const int i = (int)(u % a.S), hq = (int)(u / a.S % a.Hq), b = (int)(u / ((int64_t)a.S * a.Hq));
  const int kvh = hq / a.group;
  bool bad;
  const CaSpan sp = ca_span(a, b, &bad);
  const T *qp = static_cast<const T *>(a.q) + b * a.q_b + hq * a.q_h + i * a.q_s;
  T *yp = static_cast<T *>(a.y) + b * a.q_b + hq * a.q_h + i * a.q_s;
  for (int d = lane; d < a.D; d += 32) qs[warp][d] = ld1<T>(qp, d);
  __syncwarp();
  float o[CAA_DMAX / 32];
#pragma unroll
  for (int c = 0; c < CAA_DMAX / 32; ++c) o[c] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  const int p = sp.past + i;
  const int end = i < sp.count ? (a.causal ? min(sp.total, p + 1) : sp.total) : 0;
  const int edge = a.causal && a.window >= 0 ? max(0, p - a.window) : 0; // first key of the window
  for (int j0 = 0; j0 < end; j0 += 32) {
    if (j0 >= a.sinks && j0 + 32 <= edge) { // nothing until the window
      j0 = edge / 32 * 32 - 32;
      continue;
    }
    const int j = j0 + lane;
    bool seen = j < end && ca_sees(a, p, j);
    int64_t row = 0; // of the key, in rows of D codes
    float s = -INFINITY, vs = 0.0f;
    if (seen) {
      const int64_t id = a.table[(int64_t)b * a.max_pages + j / a.T];
      if (id < 0 || id >= a.pages) {
        seen = false;
        bad = true;
      } else {
        row = (id * a.Hkv + kvh) * a.T + j % a.T;
        const uint8_t *kp = a.k + row * a.D;
        float acc = 0.0f;
        for (int d = 0; d < a.D; ++d) acc = fmaf(qs[warp][d], Code<Q>::dec(kp[d]), acc);
        s = acc * a.ks[id * a.Hkv + kvh] * a.scale;
        if (a.softcap > 0.0f) s = a.softcap * tanhf(s / a.softcap);
        s *= kLog2E;
        vs = a.vs[id * a.Hkv + kvh];
      }
    }
    float mx = seen ? s : -INFINITY;
#pragma unroll
    for (int w = 16; w; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
    const float mn = fmaxf(m, mx);
    const float base = mn == -INFINITY ? 0.0f : mn;
    const float pj = seen ? exp2f(s - base) : 0.0f;
    const float corr = exp2f(m - base);
    m = mn;
    float ls = pj;
#pragma unroll
    for (int w = 16; w; w >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, w);
    l = l * corr + ls;
#pragma unroll
    for (int c = 0; c < CAA_DMAX / 32; ++c) o[c] *= corr;
    const float pv = seen ? pj * (vs * CAA_DOWN) : 0.0f;
    const unsigned any = __ballot_sync(0xffffffffu, seen);
    for (unsigned rest = any; rest; rest &= rest - 1) {
      const int src = __ffs(rest) - 1;
      const float w = __shfl_sync(0xffffffffu, pv, src);
      const uint8_t *vp = a.v + __shfl_sync(0xffffffffu, row, src) * a.D;
#pragma unroll
      for (int c = 0; c < CAA_DMAX / 32; ++c)
        if (c * 32 + lane < a.D) o[c] = fmaf(w, Code<Q>::dec(vp[c * 32 + lane]), o[c]);
    }
  }
  if (bad) atomicExch(&g_cache_attention_status, 1);
  const float inv = l == 0.0f ? 0.0f : 1.0f / CAA_DOWN / l; // a NaN in l stays
#pragma unroll
  for (int c = 0; c < CAA_DMAX / 32; ++c)
    if (c * 32 + lane < a.D) st1<T>(yp, c * 32 + lane, o[c] * inv);
}

} // namespace

int status_read_cache_attention(int reset) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_cache_attention_status, sizeof(int)) != cudaSuccess) return -1;
  if (reset && v) {
    const int z = 0;
    if (cudaMemcpyToSymbol(g_cache_attention_status, &z, sizeof(int)) != cudaSuccess) return -1;
  }
  return v;
}

} // namespace b2

using namespace b2;

extern "C" int b2_cache_attention(const b2_tensor *q, const b2_quantized_cache *cache,
                                  const b2_tensor *new_lengths,
                                  const b2_cache_attention_attrs *attrs, b2_tensor *y,
                                  void *workspace, size_t *workspace_bytes, void *stream) {
  const char *op = "b200::QuantizedCacheAttention";
  if (!q || !y || !attrs) B2_FAIL(B2_ERR_INVALID_ARGUMENT, "%s: null tensor", op);
  if (int rc = check_quantized_cache(op, cache, new_lengths)) return rc;
  B2_ENFORCE(q->dtype == kFloat16 || q->dtype == kBfloat16, "%s: Q must be FLOAT16 or BFLOAT16.", op);
  B2_ENFORCE(q->ndim == 3 || q->ndim == 4,
             "%s: Q must be [batch, heads, new, head_size] or [batch, new, heads * head_size].", op);
  B2_ENFORCE(y->dtype == q->dtype && shape_of(y) == shape_of(q), "%s: Y must have Q's dtype and shape.", op);
  const int64_t B = cache->lengths->shape[0], Hkv = cache->k->shape[1], T = cache->k->shape[2],
                D = cache->k->shape[3];
  B2_ENFORCE(q->shape[0] == B, "%s: Q does not fit the cache's batch.", op);
  CaArgs a{};
  int64_t S, Hq;
  if (q->ndim == 4) {
    Hq = q->shape[1];
    S = q->shape[2];
    B2_ENFORCE(q->shape[3] == D, "%s: Q does not fit the cache's head_size.", op);
    a.q_s = D;
    a.q_h = S * D;
    a.q_b = Hq * S * D;
  } else {
    S = q->shape[1];
    B2_ENFORCE(q->shape[2] % D == 0, "%s: Q does not fit the cache's head_size.", op);
    Hq = q->shape[2] / D;
    a.q_h = D;
    a.q_s = Hq * D;
    a.q_b = S * Hq * D;
  }
  B2_ENFORCE(Hq >= 1 && Hq % Hkv == 0, "%s: the query heads must be a multiple of the cache's kv_heads.", op);
  B2_ENFORCE(attrs->left_window_size >= -1, "%s: left_window_size must be -1 (unbounded) or more.", op);
  B2_ENFORCE(attrs->sink_tokens >= 0, "%s: sink_tokens must not be negative.", op);
  B2_ENFORCE(attrs->is_causal || attrs->left_window_size < 0,
             "%s: left_window_size needs is_causal.", op);
  if (D > CAA_DMAX) B2_FAIL(B2_ERR_UNSUPPORTED, "%s: head sizes above %d are not handled", op, CAA_DMAX);
  const int64_t lim = (int64_t)1 << 30;
  if (B >= lim || S >= lim || Hq >= lim || B * Hq * S >= lim * 2)
    B2_FAIL(B2_ERR_UNSUPPORTED, "%s: too many queries", op);
  a.q = q->data;
  a.y = y->data;
  a.k = static_cast<const uint8_t *>(cache->k->data);
  a.v = static_cast<const uint8_t *>(cache->v->data);
  a.ks = static_cast<const float *>(cache->k_scale->data);
  a.vs = static_cast<const float *>(cache->v_scale->data);
  a.table = static_cast<const int32_t *>(cache->block_table->data);
  a.lengths = static_cast<const int32_t *>(cache->lengths->data);
  a.counts = new_lengths ? static_cast<const int32_t *>(new_lengths->data) : nullptr;
  a.pages = cache->k->shape[0];
  a.B = (int)B;
  a.Hq = (int)Hq;
  a.Hkv = (int)Hkv;
  a.group = (int)(Hq / Hkv);
  a.S = (int)S;
  a.T = (int)T;
  a.D = (int)D;
  a.max_pages = (int)cache->block_table->shape[1];
  a.causal = attrs->is_causal != 0;
  // positions stay below 2^30, so a wider window or more sinks change nothing
  a.window = (int)std::min<int64_t>(attrs->left_window_size, lim);
  a.sinks = (int)std::min<int64_t>(attrs->sink_tokens, lim);
  a.scale = attrs->has_scale ? attrs->scale : 1.0f / sqrtf((float)D);
  a.softcap = attrs->softcap;
  const bool empty = B == 0 || S == 0;
  // Up to 16 query rows per KV head the split kernel is the faster one, past that the tensor-core kernel
  // (8 heads, group 4, 6144 keys, us split / prefill: 1 x 4 positions 21 / 25, 1 x 5 33 / 25, 32 x 4
  // 93 / 134, 32 x 8 217 / 134).
  const bool prefill = !empty && (int64_t)a.S * a.group > 16 && cache_attn_prefill_eligible(a);
  const bool split = !empty && !prefill && cache_attn_split_eligible(a);
  const int wr = workspace_check(workspace, workspace_bytes,
                                 split ? cache_attn_split_workspace(a) : prefill ? cache_attn_prefill_workspace(a) : 0);
  if (wr != 0) return wr > 0 ? B2_OK : wr;
  if (empty) return B2_OK;
  B2_ENFORCE(q->data && y->data, "%s: a tensor has no data.", op);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool f8 = cache->k->dtype == kF8E4M3FN;
  B2_ENFORCE(q8::aligned(workspace, 16), "%s: the workspace must be 16-byte aligned.", op);
  if (prefill) return cache_attn_prefill_launch(a, q->dtype == kFloat16, f8, workspace, st);
  if (split) return cache_attn_split_launch(a, q->dtype == kFloat16, f8, workspace, st);
  const unsigned grid = (unsigned)((B * Hq * S + CAA_WARPS - 1) / CAA_WARPS);
  if (q->dtype == kFloat16) {
    if (f8) cache_attn_any<__half, Fp8><<<grid, CAA_WARPS * 32, 0, st>>>(a);
    else cache_attn_any<__half, Int8><<<grid, CAA_WARPS * 32, 0, st>>>(a);
  } else {
    if (f8) cache_attn_any<__nv_bfloat16, Fp8><<<grid, CAA_WARPS * 32, 0, st>>>(a);
    else cache_attn_any<__nv_bfloat16, Int8><<<grid, CAA_WARPS * 32, 0, st>>>(a);
  }
  B2_LAUNCH_CHECK();
  return B2_OK;
}
