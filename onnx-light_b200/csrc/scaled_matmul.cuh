// Shared by the kernels of b2_scaled_matmul: the product of two 8-bit operands with scales.
#pragma once
#include "quant8.cuh"

namespace b2 {

struct SmArgs {
  const uint8_t *a, *w;  // [M, K], [N, K]
  const float *as, *ws;
  void *y;               // [M, N]
  int64_t M, N, K;
  int a_per_row, w_per_col; // scales per row / column (else one for all)
};

// Few rows (scaled_matmul_skinny.cu).
bool scaled_skinny_eligible(const SmArgs &g, bool f8);
int scaled_skinny_launch(const SmArgs &g, int y_dtype, bool f8, cudaStream_t st);

// Pairs of SMs (scaled_matmul_pair.cu).
bool scaled_pair_eligible(const SmArgs &g);
int scaled_pair_launch(const SmArgs &g, int y_dtype, bool f8, cudaStream_t st);

// Tensor-core tiles (scaled_matmul_tc.cu).
bool scaled_tc_eligible(const SmArgs &g);
int scaled_tc_launch(const SmArgs &g, int y_dtype, bool f8, cudaStream_t st);

// 32 columns of one row: the sums times the row's scale and the columns' (in shared memory).
template <typename T, typename Q>
__device__ __forceinline__ void store_scaled32(T *y, int left, float as, const float *ws, const uint32_t (&r)[32], bool vec) {
  float v[32];
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    const float4 w = *reinterpret_cast<const float4 *>(ws + j);
    const float f[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      v[j + e] = (std::is_same<Q, q8::Int8>::value ? (float)(int)r[j + e] : __uint_as_float(r[j + e])) * (as * f[e]);
  }
  if (vec && left >= 32) {
#pragma unroll
    for (int j = 0; j < 32; j += 8) {
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = v[j + e];
      q8::Raw8<T>::store(y + j, f);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < left) q8::st1<T>(y, j, v[j]);
  }
}

} // namespace b2
