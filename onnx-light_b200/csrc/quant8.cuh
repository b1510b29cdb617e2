// 8-bit codes with a scale: INT8 (|code| <= 127) and FLOAT8E4M3FN (|code| <= 448).
// A code stands for code * scale.  The scale of a group of values is their largest magnitude
// divided by 127 or 448, the code the value divided by that scale, rounded to nearest even.  A
// scale of 0 (the values are 0, or so small that it rounds to 0), an infinite one and a NaN (a value is
// not a number) give zero codes, so no NaN code is ever written; the scale carries it.
#pragma once
#include <cuda_fp8.h>

#include <type_traits>

#include "b2_common.cuh"

namespace b2 {
namespace q8 {

struct Int8 {};
struct Fp8 {};

template <typename Q> struct Code;
template <> struct Code<Int8> {
  static constexpr float kMax = 127.0f;
  static __device__ __forceinline__ uint32_t enc(float v) { // NaN -> 0
    return (uint32_t)max(-127, min(127, __float2int_rn(v))) & 0xffu;
  }
  static __device__ __forceinline__ float dec(uint32_t c) { return (float)(int8_t)c; }
};
template <> struct Code<Fp8> {
  static constexpr float kMax = 448.0f;
  static __device__ __forceinline__ uint32_t enc(float v) {
    return (uint32_t)__nv_cvt_float_to_fp8(v == v ? v : 0.0f, __NV_SATFINITE, __NV_E4M3);
  }
  static __device__ __forceinline__ float dec(uint32_t c) { return dec_f8e4m3fn(c); }
};

// Eight finite values of at most kMax (and a rounding) -> eight code bytes, the first value in the
// lowest byte.
template <typename Q> __device__ __forceinline__ uint2 enc8(const float (&v)[8]) {
  uint2 r;
  if constexpr (std::is_same<Q, Fp8>::value) {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      h[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i], v[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    r.x = h[0] | (h[1] << 16);
    r.y = h[2] | (h[3] << 16);
  } else {
    // adding 1.5 * 2^23 rounds to nearest even and leaves the integer in the low bits
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = __float_as_uint(v[i] + 12582912.0f);
    r.x = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    r.y = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
  }
  return r;
}

// Division by one scale.  A scale of a few units of 2^-149 is rounded so coarsely that quotients by it
// pass 127 or 448 by up to a half; they are held to the largest code.
template <typename Q> __device__ __forceinline__ float quotient_by_rounded(float v, float s) {
  return fminf(fmaxf(__fdiv_rn(v, s), -Code<Q>::kMax), Code<Q>::kMax);
}

// Division of many values by one scale, correctly rounded: with inv the correctly rounded 1 / s,
// q = x inv is within an ulp or two, x - q s is exact in one FMA, and q + (x - q s) inv rounds to the
// nearest quotient (P. Markstein, "Computation of elementary functions on the IBM RISC System/6000
// processor", 1990, theorem on division by a correctly rounded reciprocal).  That needs s and inv
// well inside the normal range; other scales take the division itself, and a scale that is 0, infinite
// or not a number gives zeros, the code of such a group.
template <typename Q> struct Divisor {
  float s, inv;
  int kind; // 0 zeros, 1 products, 2 divisions
  __device__ __forceinline__ explicit Divisor(float scale) : s(scale) {
    kind = !(scale > 0.0f && scale < INFINITY) ? 0 : scale > 1e-30f && scale < 1e30f ? 1 : 2;
    inv = kind == 1 ? __frcp_rn(scale) : 0.0f;
  }
  __device__ __forceinline__ float one(float v) const {
    if (kind != 1) return kind == 0 ? 0.0f : quotient_by_rounded<Q>(v, s);
    const float q = v * inv;
    return fmaf(fmaf(-q, s, v), inv, q);
  }
  __device__ __forceinline__ void divide(float (&v)[8]) const {
    if (kind == 1) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float q = v[e] * inv;
        v[e] = fmaf(fmaf(-q, s, v[e]), inv, q);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = one(v[e]);
    }
  }
};

// Eight consecutive FLOAT16 / BFLOAT16 / FLOAT values as loaded (16-byte aligned).
template <typename T> struct Raw8 {
  uint4 a;
  __device__ __forceinline__ void load(const void *p) { a = *static_cast<const uint4 *>(p); }
  __device__ __forceinline__ void zero() { a = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        const float2 t = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        f[2 * i] = t.x;
        f[2 * i + 1] = t.y;
      } else {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
  static __device__ __forceinline__ void store(void *p, const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&h);
      }
    }
    *static_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const void *p) {
    a = static_cast<const float4 *>(p)[0];
    b = static_cast<const float4 *>(p)[1];
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
  static __device__ __forceinline__ void store(void *p, const float (&f)[8]) {
    static_cast<float4 *>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    static_cast<float4 *>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
};

template <typename T> __device__ __forceinline__ float ld1(const void *p, int64_t i) {
  if constexpr (std::is_same<T, float>::value) return static_cast<const float *>(p)[i];
  else if constexpr (std::is_same<T, __half>::value) return __half2float(static_cast<const __half *>(p)[i]);
  else return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
template <typename T> __device__ __forceinline__ void st1(void *p, int64_t i, float v) {
  if constexpr (std::is_same<T, float>::value) static_cast<float *>(p)[i] = v;
  else if constexpr (std::is_same<T, __half>::value) static_cast<__half *>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

// |v| as an unsigned integer: orders like the magnitude, with every NaN above infinity, so an
// integer maximum over a group keeps a NaN.
__device__ __forceinline__ uint32_t mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Largest magnitude over a block whose threads all call it (blockDim.x a multiple of 32, at most
// 1024); `red` has 32 words.  The maximum does not depend on the order.
__device__ __forceinline__ uint32_t block_max(uint32_t m, uint32_t *red) {
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  const uint32_t n = blockDim.x >> 5;
  m = __reduce_max_sync(0xffffffffu, (threadIdx.x & 31) < n ? red[threadIdx.x & 31] : 0u);
  return m;
}

// The largest magnitude of eight values as loaded, as mag() gives it.
template <typename T> __device__ __forceinline__ uint32_t mag8(const Raw8<T> &x) {
  if constexpr (std::is_same<T, float>::value) {
    float f[8];
    x.get(f);
    uint32_t m = 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, mag(f[e]));
    return m;
  } else {
    // 16-bit magnitudes order like unsigned integers, every NaN above infinity
    const uint32_t m = __vmaxu2(__vmaxu2(x.a.x & 0x7fff7fffu, x.a.y & 0x7fff7fffu),
                                __vmaxu2(x.a.z & 0x7fff7fffu, x.a.w & 0x7fff7fffu));
    const uint32_t h = max(m & 0xffffu, m >> 16);
    if constexpr (std::is_same<T, __half>::value) return __float_as_uint(__half2float(__ushort_as_half((unsigned short)h)));
    else return h << 16;
  }
}

inline bool is_q8(int dt) { return dt == kInt8 || dt == kF8E4M3FN; }
inline bool is_float_type(int dt) { return dt == kFloat || dt == kFloat16 || dt == kBfloat16; }
inline bool has_data(const b2_tensor *t) { return t->data != nullptr || numel(t) == 0; }
inline bool aligned(const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

} // namespace q8
} // namespace b2
