// Append of new keys and values to a paged 8-bit KV cache (b2_kv_cache_append).
//
// Position p of sequence b lies in row p % T of page block_table[b][p / T]; a page holds T tokens
// of every KV head, [Hkv, T, D] codes, with one scale per head.  For each page that gets new
// tokens, with a = max |new value| / 127 or 448 and s the scale of the older tokens in the page
// (0 when it has none):
//   s' = max(s, a); new codes round(x / s'); where s' > s the older codes become
//   round(code * (s / s')), so one scale serves the page and grows only when it has to.
//
// Bound: HBM for prompts (2 or 4 bytes read and 1 written per value), latency for single tokens.
// One CTA owns one (sequence, page, head, K or V), so no two CTAs write the same page rows or
// scale; a page's values stay in registers between the maximum and the codes when there are at
// most 8192 of them (64 tokens of 128), and are read again (from cache) past that.
// Measured (8 heads of 128, pages of 64, FLOAT8): prompts of 4 ragged sequences of up to 2048 BFLOAT16
// tokens 12.5 us, 3.1 TB/s; one token for each of 32 sequences 3.7 us in a graph.
#include "quant8.cuh"

namespace b2 {

// 1: a page number, a length or a count of new tokens was out of range.
__device__ int g_cache_append_status;

namespace {

using namespace q8;

// Threads x vectors of 8 values that a thread keeps in registers.  128 x 8, 256 x 4 and 64 x 16 take the
// prompts above 8.8, 10.7 and 11.4 us in a graph, pages of 16 tokens 21, 28 and 19, of 256 tokens 15, 13 and 23.
constexpr int KA_THREADS = 128;
constexpr int KA_HELD = 8;

struct KaArgs {
  const void *src[2];
  uint8_t *pool[2];
  float *scale[2];
  const int32_t *table, *lengths, *counts;
  int64_t s_b, s_h, s_s; // strides (elements) of the new tokens over batch, head, position
  int64_t pages;
  int B, H, S, T, D, max_pages, slots;
  FastDiv div_t, div_h, div_slots, div_row; // by T, H, slots, vectors (or values) in a row
};

// Four codes times the ratio of the old scale to the new one.
template <typename Q> __device__ __forceinline__ uint32_t rescale4(uint32_t c, float ratio) {
  uint32_t r = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    r |= Code<Q>::enc(__fmul_rn(Code<Q>::dec((c >> (8 * e)) & 0xffu), ratio)) << (8 * e);
  return r;
}

template <typename T, typename Q, bool VEC>
__global__ void __launch_bounds__(KA_THREADS) kv_cache_append_kernel(const KaArgs a) {
  __shared__ uint32_t red[32];
  const int side = (int)(blockIdx.x & 1);
  const uint32_t u = blockIdx.x >> 1, uh = a.div_h.div(u), ub = a.div_slots.div(uh);
  const int h = (int)(u - uh * a.H), slot = (int)(uh - ub * a.slots), b = (int)ub;
  int64_t past = a.lengths[b];
  int64_t n = a.counts ? a.counts[b] : a.S;
  const int64_t room = (int64_t)a.max_pages * a.T;
  bool bad = past < 0 || n < 0 || n > a.S || past + n > room;
  past = max(past, (int64_t)0);
  n = min(min(max(n, (int64_t)0), (int64_t)a.S), room - past);
  const int64_t page = (int64_t)a.div_t.div((uint32_t)past) + slot; // place in the table
  const int64_t lo = max(past, page * a.T), hi = min(past + n, (page + 1) * a.T);
  if (lo >= hi) {
    if (bad && threadIdx.x == 0) atomicExch(&g_cache_append_status, 1);
    return;
  }
  // The page number and the new values are read together: neither needs the other.
  const int64_t id = a.table[(int64_t)b * a.max_pages + page];
  const int older = (int)(lo - page * a.T), rows = (int)(hi - lo);
  const T *src = static_cast<const T *>(a.src[side]) + (int64_t)b * a.s_b + (int64_t)h * a.s_h +
                 (lo - past) * a.s_s;
  const int dv = VEC ? a.D >> 3 : a.D, nv = rows * dv;
  auto at = [&](int v) { // element offset of vector (or value) v of the new rows
    const int r = (int)a.div_row.div((uint32_t)v);
    return (int64_t)r * a.s_s + (int64_t)(v - r * dv) * (VEC ? 8 : 1);
  };
  Raw8<T> held[KA_HELD];
  if constexpr (VEC) {
#pragma unroll
    for (int k = 0; k < KA_HELD; ++k) {
      const int v = threadIdx.x + k * KA_THREADS;
      if (v < nv) held[k].load(src + at(v));
      else held[k].zero();
    }
  }
  if (id < 0 || id >= a.pages) bad = true;
  if (bad && threadIdx.x == 0) atomicExch(&g_cache_append_status, 1);
  if (id < 0 || id >= a.pages) return;
  float *sp = a.scale[side] + id * a.H + h;
  uint8_t *dst = a.pool[side] + (id * a.H + h) * (int64_t)a.T * a.D;
  const float before = older ? *sp : 0.0f;
  // ---- the largest magnitude of the new values ----
  uint32_t m = 0u;
  if constexpr (VEC) {
#pragma unroll
    for (int k = 0; k < KA_HELD; ++k) m = max(m, mag8(held[k]));
    for (int v = threadIdx.x + KA_HELD * KA_THREADS; v < nv; v += KA_THREADS) {
      Raw8<T> x;
      x.load(src + at(v));
      m = max(m, mag8(x));
    }
  } else {
    for (int v = threadIdx.x; v < nv; v += KA_THREADS) m = max(m, mag(ld1<T>(src, at(v))));
  }
  m = block_max(m, red); // every thread has read *sp before this barrier
  const float amax = __fdiv_rn(__uint_as_float(m), Code<Q>::kMax);
  // the larger of the two; a NaN on either side stays
  const float s = before != before || amax != amax ? __uint_as_float(0x7fc00000u)
                                                   : fmaxf(before, amax);
  if (threadIdx.x == 0) *sp = s;
  // ---- the older tokens of a page whose scale grew ----
  if (s > before && older) {
    const float ratio = __fdiv_rn(before, s);
    if constexpr (VEC) { // four vectors in flight a thread: one by one each waits for the last's store
      const int no = older * dv;
      for (int i = threadIdx.x; i < no; i += 4 * KA_THREADS) {
        uint2 c[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (i + k * KA_THREADS < no) c[k] = reinterpret_cast<const uint2 *>(dst)[i + k * KA_THREADS];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (i + k * KA_THREADS < no) {
            c[k].x = rescale4<Q>(c[k].x, ratio);
            c[k].y = rescale4<Q>(c[k].y, ratio);
            reinterpret_cast<uint2 *>(dst)[i + k * KA_THREADS] = c[k];
          }
      }
    } else {
      for (int i = threadIdx.x; i < older * a.D; i += KA_THREADS)
        dst[i] = (uint8_t)Code<Q>::enc(__fmul_rn(Code<Q>::dec(dst[i]), ratio));
    }
  }
  // ---- the new codes ----
  dst += (int64_t)older * a.D;
  const Divisor<Q> by(s);
  if constexpr (VEC) {
    auto put = [&](int v, const Raw8<T> &x) {
      float f[8];
      x.get(f);
      by.divide(f);
      *reinterpret_cast<uint2 *>(dst + (int64_t)v * 8) = enc8<Q>(f);
    };
#pragma unroll
    for (int k = 0; k < KA_HELD; ++k) {
      const int v = threadIdx.x + k * KA_THREADS;
      if (v < nv) put(v, held[k]);
    }
    for (int v = threadIdx.x + KA_HELD * KA_THREADS; v < nv; v += KA_THREADS) {
      Raw8<T> x;
      x.load(src + at(v));
      put(v, x);
    }
  } else {
    for (int v = threadIdx.x; v < nv; v += KA_THREADS)
      dst[v] = (uint8_t)Code<Q>::enc(by.one(ld1<T>(src, at(v))));
  }
}

template <typename T> int launch(const KaArgs &a, bool f8, bool vec, unsigned grid, cudaStream_t st) {
  if (vec) {
    if (f8) kv_cache_append_kernel<T, Fp8, true><<<grid, KA_THREADS, 0, st>>>(a);
    else kv_cache_append_kernel<T, Int8, true><<<grid, KA_THREADS, 0, st>>>(a);
  } else {
    if (f8) kv_cache_append_kernel<T, Fp8, false><<<grid, KA_THREADS, 0, st>>>(a);
    else kv_cache_append_kernel<T, Int8, false><<<grid, KA_THREADS, 0, st>>>(a);
  }
  B2_LAUNCH_CHECK();
  return B2_OK;
}

} // namespace

// Checks shared by the operators on a quantized cache; `op` prefixes the messages.
int check_quantized_cache(const char *op, const b2_quantized_cache *c, const b2_tensor *counts) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || !c->block_table || !c->lengths)
    B2_FAIL(B2_ERR_INVALID_ARGUMENT, "%s: null cache tensor", op);
  B2_ENFORCE(q8::is_q8(c->k->dtype) && c->v->dtype == c->k->dtype,
             "%s: the cache must be INT8 or FLOAT8E4M3FN.", op);
  B2_ENFORCE(c->k->ndim == 4 && shape_of(c->v) == shape_of(c->k),
             "%s: cache keys and values must be [pages, kv_heads, page_size, head_size] of one shape.", op);
  const int64_t *s = c->k->shape;
  B2_ENFORCE(s[1] >= 1 && s[2] >= 1 && s[3] >= 1, "%s: the cache has an empty dimension.", op);
  for (const b2_tensor *t : {c->k_scale, c->v_scale})
    B2_ENFORCE(t->dtype == kFloat && t->ndim == 2 && t->shape[0] == s[0] && t->shape[1] == s[1],
               "%s: cache scales must be FLOAT [pages, kv_heads].", op);
  B2_ENFORCE(c->block_table->dtype == kInt32 && c->block_table->ndim == 2,
             "%s: block_table must be INT32 [batch, max_pages].", op);
  B2_ENFORCE(c->lengths->dtype == kInt32 && c->lengths->ndim == 1 &&
                 c->lengths->shape[0] == c->block_table->shape[0],
             "%s: lengths must be INT32 [batch].", op);
  if (counts)
    B2_ENFORCE(counts->dtype == kInt32 && shape_of(counts) == shape_of(c->lengths),
               "%s: new_lengths must be INT32 [batch].", op);
  for (const b2_tensor *t : {c->k, c->v, c->k_scale, c->v_scale, c->block_table, c->lengths, counts})
    B2_ENFORCE(!t || q8::has_data(t), "%s: a cache tensor has no data.", op);
  const int64_t lim = (int64_t)1 << 30;
  if (s[0] * s[1] >= lim || s[2] >= lim || s[2] * s[3] >= lim ||
      c->block_table->shape[1] * s[2] >= lim)
    B2_FAIL(B2_ERR_UNSUPPORTED, "%s: cache too large", op);
  return B2_OK;
}

int status_read_cache_append(int reset) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_cache_append_status, sizeof(int)) != cudaSuccess) return -1;
  if (reset && v) {
    const int z = 0;
    if (cudaMemcpyToSymbol(g_cache_append_status, &z, sizeof(int)) != cudaSuccess) return -1;
  }
  return v;
}

} // namespace b2

using namespace b2;

extern "C" int b2_kv_cache_append(const b2_tensor *k, const b2_tensor *v,
                                  const b2_quantized_cache *cache, const b2_tensor *new_lengths,
                                  void *stream) {
  const char *op = "b200::KVCacheAppend";
  if (!k || !v) B2_FAIL(B2_ERR_INVALID_ARGUMENT, "%s: null tensor", op);
  if (int rc = check_quantized_cache(op, cache, new_lengths)) return rc;
  B2_ENFORCE(q8::is_float_type(k->dtype) && v->dtype == k->dtype,
             "%s: K and V must be FLOAT, FLOAT16 or BFLOAT16 of one dtype.", op);
  B2_ENFORCE((k->ndim == 3 || k->ndim == 4) && shape_of(v) == shape_of(k),
             "%s: K and V must be [batch, kv_heads, new, head_size] or [batch, new, kv_heads * head_size].", op);
  const int64_t B = cache->lengths->shape[0], H = cache->k->shape[1], T = cache->k->shape[2],
                D = cache->k->shape[3];
  KaArgs a{};
  int64_t S;
  if (k->ndim == 4) {
    S = k->shape[2];
    B2_ENFORCE(k->shape[0] == B && k->shape[1] == H && k->shape[3] == D,
               "%s: K and V do not fit the cache's batch, kv_heads or head_size.", op);
    a.s_s = D;
    a.s_h = S * D;
    a.s_b = H * S * D;
  } else {
    S = k->shape[1];
    B2_ENFORCE(k->shape[0] == B && k->shape[2] == H * D,
               "%s: K and V do not fit the cache's batch, kv_heads or head_size.", op);
    a.s_h = D;
    a.s_s = H * D;
    a.s_b = S * H * D;
  }
  if (B == 0 || S == 0) return B2_OK;
  B2_ENFORCE(k->data && v->data, "%s: a tensor has no data.", op);
  if (S >= (int64_t)1 << 30 || B >= (int64_t)1 << 30) B2_FAIL(B2_ERR_UNSUPPORTED, "%s: too many tokens", op);
  a.src[0] = k->data;
  a.src[1] = v->data;
  a.pool[0] = static_cast<uint8_t *>(cache->k->data);
  a.pool[1] = static_cast<uint8_t *>(cache->v->data);
  a.scale[0] = static_cast<float *>(cache->k_scale->data);
  a.scale[1] = static_cast<float *>(cache->v_scale->data);
  a.table = static_cast<const int32_t *>(cache->block_table->data);
  a.lengths = static_cast<const int32_t *>(cache->lengths->data);
  a.counts = new_lengths ? static_cast<const int32_t *>(new_lengths->data) : nullptr;
  a.pages = cache->k->shape[0];
  a.B = (int)B;
  a.H = (int)H;
  a.S = (int)S;
  a.T = (int)T;
  a.D = (int)D;
  a.max_pages = (int)cache->block_table->shape[1];
  a.slots = (int)((S + T - 2) / T + 1); // pages that S consecutive positions can touch
  const int64_t grid = 2 * B * H * a.slots;
  if (grid >= (int64_t)1 << 31) B2_FAIL(B2_ERR_UNSUPPORTED, "%s: too many pages", op);
  const bool vec = D % 8 == 0 && q8::aligned(k->data, 16) && q8::aligned(v->data, 16) &&
                   q8::aligned(cache->k->data, 8) && q8::aligned(cache->v->data, 8);
  const bool f8 = cache->k->dtype == kF8E4M3FN;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  a.div_t = FastDiv((uint32_t)a.T);
  a.div_h = FastDiv((uint32_t)a.H);
  a.div_slots = FastDiv((uint32_t)a.slots);
  a.div_row = FastDiv((uint32_t)(vec ? D / 8 : D));
  if (k->dtype == kFloat16) return launch<__half>(a, f8, vec, (unsigned)grid, st);
  if (k->dtype == kBfloat16) return launch<__nv_bfloat16>(a, f8, vec, (unsigned)grid, st);
  return launch<float>(a, f8, vec, (unsigned)grid, st);
}
