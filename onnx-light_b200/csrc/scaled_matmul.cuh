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

// Tensor-core tiles (scaled_matmul_tc.cu).
bool scaled_tc_eligible(const SmArgs &g);
int scaled_tc_launch(const SmArgs &g, int y_dtype, bool f8, cudaStream_t st);

} // namespace b2
