// RMS normalization with the residual's addition and an 8-bit output with scales
// (b2_rms_normalization_quantize), the operator before a projection of 8-bit activations:
//   h = x + residual            (fp32; written to `sum` rounded to x's type)
//   n = h / sqrt(mean(h^2) + epsilon) * weight
//   s = max |n| over the row or over each group of columns, divided by 127 or 448
//   code = round(n / s)
//
// Bound: HBM, (1 + residual + sum) elements and 1 code per element.  One CTA owns one row and holds
// it in registers between the three steps (statistic, largest magnitude, codes), so x and the
// residual are read once and nothing is read back.  The norm is taken of the unrounded sum.  All
// sums are fp32 in a fixed order; the maxima are integer maxima of magnitudes, which keep a NaN.
// n itself is never formed: 1 / sqrt(...) is split into a power of two, which scales h exactly, and a
// rest in [1, 2) that only the scale takes, so a code is h w over the largest h w and carries the
// rounding of h w and of the quotient alone.
// Measured: 8192 x 4096 BFLOAT16 with residual and FLOAT8 codes 44 us, 5.3 TB/s (in a graph 40, and 32
// without residual, where the issue slots bind); one such row 2.5 us in a graph.
#include "attn_math.cuh"
#include "quant8.cuh"

namespace b2 {
namespace {

using namespace q8;

struct RnqArgs {
  const void *x, *res, *w;
  void *sum;
  uint8_t *y;
  float *y_scale;
  int width, group, groups;
  float eps;
};

// Sum over the block, the same value in every thread; `red` has 32 words.
__device__ __forceinline__ float block_sum(float v, float *red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int n = blockDim.x >> 5;
  v = (int)(threadIdx.x & 31) < n ? red[threadIdx.x & 31] : 0.0f;
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ void unpack2(uint64_t v, float &x, float &y) {
  const float2 f = f2unpack(v);
  x = f.x;
  y = f.y;
}

// 1 / sqrt(mean + epsilon) as p2 * rest: p2 a power of two, 1 <= rest < 2 (0, infinity and NaN are p2).
struct Rms {
  float p2, rest;
  __device__ __forceinline__ Rms(float ss, int width, float eps) {
    const float r = 1.0f / sqrtf(ss / (float)width + eps);
    const uint32_t u = __float_as_uint(r);
    const bool split = r > 0.0f && r < INFINITY; // never subnormal: a root is at most 2^64
    p2 = split ? __uint_as_float(u & 0x7f800000u) : r;
    rest = split ? __uint_as_float((u & 0x007fffffu) | 0x3f800000u) : 1.0f;
  }
};
template <typename Q> __device__ __forceinline__ float scale_of(uint32_t top, float rest) {
  return __fdiv_rn(__uint_as_float(top) * rest, Code<Q>::kMax);
}

// Quotients by top / 127 or 448, kept as the sum of two floats: q = v inv is within some ulps,
// v - q (hi + lo) comes from two FMAs, and q + that * inv is the quotient rounded once, but for a
// second-order term.  A ratio next to a tie between two codes so mostly falls on the side where the
// inputs put it: of 10^8 FLOAT8 codes 204 are a neighbour of the exact one (311 by the rounded scale's
// chain), of INT8 codes 33 (40).  Zeros where the group's scale is 0, infinite or not a number.
template <typename Q> struct ByTop {
  float hi, lo, inv;
  int kind; // 0 zeros, 1 products, 2 divisions
  __device__ __forceinline__ ByTop(uint32_t top, float rest) {
    const float t = __uint_as_float(top), s = scale_of<Q>(top, rest);
    hi = __fdiv_rn(t, Code<Q>::kMax);
    kind = !(s > 0.0f && s < INFINITY) ? 0 : hi > 1e-25f && hi < 1e30f ? 1 : 2;
    lo = fmaf(-hi, Code<Q>::kMax, t) * (1.0f / Code<Q>::kMax);
    if (kind == 2) { // a quotient of v lo and hi; top / 127 may be subnormal, then by the stored scale itself
      lo = hi < 1e-36f ? rest : 1.0f;
      hi = hi < 1e-36f ? s : hi;
    }
    inv = kind == 1 ? __frcp_rn(hi) : 0.0f;
  }
  __device__ __forceinline__ float one(float v) const {
    if (kind != 1) return kind == 0 ? 0.0f : quotient_by_rounded<Q>(v * lo, hi);
    const float q = v * inv;
    return fmaf(fmaf(-q, lo, fmaf(-q, hi, v)), inv, q);
  }
  __device__ __forceinline__ void divide(float (&v)[8]) const {
    if (kind == 1) {
      const uint64_t i2 = f2pack(inv, inv), h2 = f2pack(-hi, -hi), l2 = f2pack(-lo, -lo);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const uint64_t x = f2pack(v[e], v[e + 1]), q = fmul2(x, i2);
        unpack2(ffma2(ffma2(q, l2, ffma2(q, h2, x)), i2, q), v[e], v[e + 1]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = one(v[e]);
    }
  }
};

// Groups of columns: kRow one group per row; kLanes a group is 8 * seg columns with seg a power
// of two up to 32, so it lies in seg neighbouring lanes of one warp; kShared any other multiple
// of 8, by integer maxima in shared memory.
enum Mode { kRow, kLanes, kShared };

// width a multiple of 8, 16-byte aligned rows: thread t holds the 8-column vectors t + k blockDim.
template <typename T, typename Q, int KV, int MODE>
__global__ void __launch_bounds__(1024) rms_norm_q_vec(const RnqArgs a) {
  extern __shared__ uint32_t gmax[]; // kShared: [groups]
  __shared__ float red_f[32];
  __shared__ uint32_t red_u[32];
  const int64_t row = blockIdx.x, base = row * a.width;
  const int nv = a.width >> 3, tid = threadIdx.x, nt = blockDim.x;
  // Wide FLOAT rows load residual and weights where they are used: ahead of the statistic they do not
  // fit a thread's 64 registers (1024 x 32768 with residual: 156 us spilling, 91 like this; 4.8 TB/s).
  constexpr bool kAhead = KV < 4 || sizeof(T) == 2;
  Raw8<T> xr[KV], rr[KV], wr[KV];
#pragma unroll
  for (int k = 0; k < KV; ++k) {
    const int v = tid + k * nt;
    if (v < nv) {
      xr[k].load(static_cast<const T *>(a.x) + base + 8 * v);
      if (kAhead && a.res) rr[k].load(static_cast<const T *>(a.res) + base + 8 * v);
    }
  }
#pragma unroll
  for (int k = 0; k < KV; ++k)
    if (kAhead && tid + k * nt < nv) wr[k].load(static_cast<const T *>(a.w) + 8 * (tid + k * nt));
  if (MODE == kShared)
    for (int g = tid; g < a.groups; g += nt) gmax[g] = 0u;
  float h[KV][8];
  uint64_t ss2 = 0; // sums of the even and of the odd columns
#pragma unroll
  for (int k = 0; k < KV; ++k) {
    const int v = tid + k * nt;
    if (v < nv) {
      xr[k].get(h[k]);
      if (a.res) {
        float r[8];
        if (!kAhead) rr[k].load(static_cast<const T *>(a.res) + base + 8 * v);
        rr[k].get(r);
#pragma unroll
        for (int e = 0; e < 8; e += 2)
          unpack2(fadd2(f2pack(h[k][e], h[k][e + 1]), f2pack(r[e], r[e + 1])), h[k][e], h[k][e + 1]);
      }
      if (a.sum) Raw8<T>::store(static_cast<T *>(a.sum) + base + 8 * v, h[k]);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const uint64_t x = f2pack(h[k][e], h[k][e + 1]);
        ss2 = ffma2(x, x, ss2);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) h[k][e] = 0.0f;
    }
  }
  float ss, odd;
  unpack2(ss2, ss, odd);
  ss = block_sum(ss + odd, red_f);
  const Rms r(ss, a.width, a.eps);
  const uint64_t p2 = f2pack(r.p2, r.p2);
  uint32_t m[KV];
#pragma unroll
  for (int k = 0; k < KV; ++k) {
    m[k] = 0u;
    if (tid + k * nt < nv) {
      float w[8];
      if (!kAhead) wr[k].load(static_cast<const T *>(a.w) + 8 * (tid + k * nt));
      wr[k].get(w);
#pragma unroll
      for (int e = 0; e < 8; e += 2)
        unpack2(fmul2(fmul2(f2pack(h[k][e], h[k][e + 1]), p2), f2pack(w[e], w[e + 1])), h[k][e], h[k][e + 1]);
#pragma unroll
      for (int e = 0; e < 8; ++e) m[k] = max(m[k], mag(h[k][e]));
    }
  }
  // m: the largest magnitude of the group that vector k lies in
  if (MODE == kRow) {
    uint32_t mm = 0u;
#pragma unroll
    for (int k = 0; k < KV; ++k) mm = max(mm, m[k]);
    mm = block_max(mm, red_u);
    if (tid == 0) a.y_scale[row] = scale_of<Q>(mm, r.rest);
    const ByTop<Q> by(mm, r.rest);
#pragma unroll
    for (int k = 0; k < KV; ++k) {
      const int v = tid + k * nt;
      if (v < nv) {
        by.divide(h[k]);
        *reinterpret_cast<uint2 *>(a.y + base + 8 * v) = enc8<Q>(h[k]);
      }
    }
    return;
  }
  if (MODE == kLanes) {
    const int seg = a.group >> 3;
#pragma unroll
    for (int k = 0; k < KV; ++k) {
      for (int o = seg >> 1; o; o >>= 1) m[k] = max(m[k], __shfl_xor_sync(0xffffffffu, m[k], o));
      const int v = tid + k * nt;
      if (v < nv && v % seg == 0) a.y_scale[row * a.groups + v / seg] = scale_of<Q>(m[k], r.rest);
    }
  } else {
    // gmax was cleared before block_sum's barrier
#pragma unroll
    for (int k = 0; k < KV; ++k)
      if (tid + k * nt < nv) atomicMax(&gmax[(8 * (tid + k * nt)) / a.group], m[k]);
    __syncthreads();
    for (int g = tid; g < a.groups; g += nt)
      a.y_scale[row * a.groups + g] = scale_of<Q>(gmax[g], r.rest);
#pragma unroll
    for (int k = 0; k < KV; ++k)
      if (tid + k * nt < nv) m[k] = gmax[(8 * (tid + k * nt)) / a.group];
  }
#pragma unroll
  for (int k = 0; k < KV; ++k) {
    const int v = tid + k * nt;
    if (v < nv) {
      ByTop<Q>(m[k], r.rest).divide(h[k]);
      *reinterpret_cast<uint2 *>(a.y + base + 8 * v) = enc8<Q>(h[k]);
    }
  }
}

// Any width, group and alignment: the row's fp32 values stay in shared memory.  8192 x 4097 BFLOAT16 with
// residual and FLOAT8 codes 227 us, 1.0 TB/s, bound by its one-value loads and maxima in shared memory.
template <typename T, typename Q>
__global__ void __launch_bounds__(256) rms_norm_q_any(const RnqArgs a) {
  extern __shared__ uint32_t gmax[]; // [groups], then the row [width]
  float *hs = reinterpret_cast<float *>(gmax + a.groups);
  __shared__ float red_f[32];
  const int64_t row = blockIdx.x, base = row * a.width;
  for (int g = threadIdx.x; g < a.groups; g += 256) gmax[g] = 0u;
  float ss = 0.0f;
  for (int c = threadIdx.x; c < a.width; c += 256) {
    float v = ld1<T>(a.x, base + c);
    if (a.res) v += ld1<T>(a.res, base + c);
    if (a.sum) st1<T>(a.sum, base + c, v);
    hs[c] = v;
    ss = fmaf(v, v, ss);
  }
  ss = block_sum(ss, red_f);
  const Rms r(ss, a.width, a.eps);
  for (int c = threadIdx.x; c < a.width; c += 256) {
    const float v = hs[c] * r.p2 * ld1<T>(a.w, c);
    hs[c] = v;
    atomicMax(&gmax[c / a.group], mag(v));
  }
  __syncthreads();
  for (int g = threadIdx.x; g < a.groups; g += 256)
    a.y_scale[row * a.groups + g] = scale_of<Q>(gmax[g], r.rest);
  for (int c = threadIdx.x; c < a.width; c += 256)
    a.y[base + c] = (uint8_t)Code<Q>::enc(ByTop<Q>(gmax[c / a.group], r.rest).one(hs[c]));
}

constexpr int kMaxShared = 220 * 1024;

template <typename T, typename Q, int KV>
int launch_vec(const RnqArgs &a, int64_t rows, int threads, cudaStream_t st) {
  const int seg = a.group >> 3;
  if (a.groups == 1) rms_norm_q_vec<T, Q, KV, kRow><<<(unsigned)rows, threads, 0, st>>>(a);
  else if (seg <= 32 && (seg & (seg - 1)) == 0)
    rms_norm_q_vec<T, Q, KV, kLanes><<<(unsigned)rows, threads, 0, st>>>(a);
  else // at most 4096 groups of 8 columns: 16 KB
    rms_norm_q_vec<T, Q, KV, kShared><<<(unsigned)rows, threads, (size_t)a.groups * 4, st>>>(a);
  B2_LAUNCH_CHECK();
  return B2_OK;
}

template <typename T, typename Q> int launch(const RnqArgs &a, int64_t rows, cudaStream_t st) {
  const bool vec = a.width % 8 == 0 && a.group % 8 == 0 && a.width <= 32768 && aligned(a.x, 16) &&
                   (!a.res || aligned(a.res, 16)) && (!a.sum || aligned(a.sum, 16)) &&
                   aligned(a.w, 16) && aligned(a.y, 8);
  if (vec) {
    // Vectors per thread: 2 up to a width of 16384, then 4.  One up to a width of 8192 is slower where rows
    // count (8192 x 4096 in a graph 49 us against 42) and 0.1 us faster for a single row.
    const int nv = a.width / 8, kv = nv <= 32 ? 1 : nv <= 2048 ? 2 : 4;
    const int threads = ((nv + kv - 1) / kv + 31) / 32 * 32;
    if (kv == 1) return launch_vec<T, Q, 1>(a, rows, threads, st);
    if (kv == 2) return launch_vec<T, Q, 2>(a, rows, threads, st);
    return launch_vec<T, Q, 4>(a, rows, threads, st);
  }
  const size_t smem = ((size_t)a.width + a.groups) * 4;
  if (smem > kMaxShared)
    B2_FAIL(B2_ERR_UNSUPPORTED, "b200::RMSNormalizationQuantize: rows of %d columns are too wide",
            a.width);
  auto kern = rms_norm_q_any<T, Q>;
  B2_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxShared));
  kern<<<(unsigned)rows, 256, smem, st>>>(a);
  B2_LAUNCH_CHECK();
  return B2_OK;
}

} // namespace
} // namespace b2

using namespace b2;

extern "C" int b2_rms_normalization_quantize(const b2_tensor *x, const b2_tensor *residual,
                                             const b2_tensor *scale, float epsilon,
                                             int64_t group_size, b2_tensor *y, b2_tensor *y_scale,
                                             b2_tensor *sum, void *stream) {
#define RNQ "b200::RMSNormalizationQuantize: "
  if (!x || !scale || !y || !y_scale) B2_FAIL(B2_ERR_INVALID_ARGUMENT, RNQ "null tensor");
  B2_ENFORCE(q8::is_float_type(x->dtype), RNQ "X must be FLOAT, FLOAT16 or BFLOAT16.");
  B2_ENFORCE(x->ndim >= 1, RNQ "X must have rank >= 1.");
  const int64_t width = x->shape[x->ndim - 1];
  B2_ENFORCE(scale->dtype == x->dtype && scale->ndim == 1 && scale->shape[0] == width,
             RNQ "scale must have X's dtype and one value per column of X.");
  if (residual)
    B2_ENFORCE(residual->dtype == x->dtype && shape_of(residual) == shape_of(x),
               RNQ "residual must have X's dtype and shape.");
  if (sum)
    B2_ENFORCE(sum->dtype == x->dtype && shape_of(sum) == shape_of(x),
               RNQ "sum must have X's dtype and shape.");
  B2_ENFORCE(q8::is_q8(y->dtype) && shape_of(y) == shape_of(x),
             RNQ "Y must be INT8 or FLOAT8E4M3FN of X's shape.");
  const int64_t rows = width > 0 ? numel(x) / width : 0;
  const int64_t group = group_size == 0 ? width : group_size;
  B2_ENFORCE(group_size >= 0 && (width == 0 || width % group == 0),
             RNQ "group_size must divide the number of columns (0: one group per row).");
  const int64_t groups = width > 0 ? width / group : 1;
  std::vector<int64_t> want = shape_of(x);
  want.back() = groups;
  B2_ENFORCE(y_scale->dtype == kFloat && shape_of(y_scale) == want,
             RNQ "Y_scale must be FLOAT with one value per group of columns.");
  if (rows == 0) return B2_OK;
  B2_ENFORCE(x->data && scale->data && y->data && y_scale->data && (!residual || residual->data) &&
                 (!sum || sum->data),
             RNQ "a tensor has no data.");
  if (rows >= (int64_t)1 << 31) B2_FAIL(B2_ERR_UNSUPPORTED, RNQ "too many rows");
  if (width >= (int64_t)1 << 30) B2_FAIL(B2_ERR_UNSUPPORTED, RNQ "rows too wide");
  RnqArgs a{};
  a.x = x->data;
  a.res = residual ? residual->data : nullptr;
  a.w = scale->data;
  a.sum = sum ? sum->data : nullptr;
  a.y = static_cast<uint8_t *>(y->data);
  a.y_scale = static_cast<float *>(y_scale->data);
  a.width = (int)width;
  a.group = (int)group;
  a.groups = (int)groups;
  a.eps = epsilon;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool f8 = y->dtype == kF8E4M3FN;
  if (x->dtype == kFloat16)
    return f8 ? launch<__half, q8::Fp8>(a, rows, st) : launch<__half, q8::Int8>(a, rows, st);
  if (x->dtype == kBfloat16)
    return f8 ? launch<__nv_bfloat16, q8::Fp8>(a, rows, st)
              : launch<__nv_bfloat16, q8::Int8>(a, rows, st);
  return f8 ? launch<float, q8::Fp8>(a, rows, st) : launch<float, q8::Int8>(a, rows, st);
#undef RNQ
}
