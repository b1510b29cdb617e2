// Product of two 8-bit operands with scales (b2_scaled_matmul):
//   y[m, n] = a_scale[m] * w_scale[n] * sum_k a[m, k] w[n, k]
// INT8 x INT8 summed exactly in int32, FLOAT8E4M3FN x FLOAT8E4M3FN in fp32; the scales multiply the
// sum in fp32 and the result is rounded once.
//
// This file: checks, the choice of the kernel, and scaled_mm_any, the CUDA-core kernel for shapes the
// others do not take (64 x 64 tiles, 32 columns of K staged in shared memory, 4 x 4 sums a thread), bound by
// its shared-memory reads: 1024 x 4097 x 4096 FLOAT8 1.83 ms, 19 TFLOP/s.
#include "scaled_matmul.cuh"

namespace b2 {
namespace {

using namespace q8;

constexpr int SA_TILE = 64, SA_K = 32;

template <typename T, typename Q>
__global__ void __launch_bounds__(256) scaled_mm_any(const SmArgs g) {
  using Acc = typename std::conditional<std::is_same<Q, Int8>::value, int, float>::type;
  __shared__ Acc sa[SA_K][SA_TILE + 1], sw[SA_K][SA_TILE + 1];
  const int64_t tiles = (g.N + SA_TILE - 1) / SA_TILE;
  const int64_t m0 = blockIdx.x / tiles * SA_TILE, n0 = blockIdx.x % tiles * SA_TILE;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  Acc acc[4][4] = {};
  for (int64_t k0 = 0; k0 < g.K; k0 += SA_K) {
    for (int e = threadIdx.x; e < SA_TILE * SA_K; e += 256) {
      const int r = e / SA_K, c = e % SA_K;
      const bool in = k0 + c < g.K;
      sa[c][r] = in && m0 + r < g.M ? (Acc)Code<Q>::dec(g.a[(m0 + r) * g.K + k0 + c]) : (Acc)0;
      sw[c][r] = in && n0 + r < g.N ? (Acc)Code<Q>::dec(g.w[(n0 + r) * g.K + k0 + c]) : (Acc)0;
    }
    __syncthreads();
#pragma unroll 8
    for (int c = 0; c < SA_K; ++c) {
      Acc av[4], wv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        av[i] = sa[c][ty + 16 * i];
        wv[i] = sw[c][tx + 16 * i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += av[i] * wv[j];
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty + 16 * i;
    if (m >= g.M) continue;
    const float as = g.as[g.a_per_row ? m : 0];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tx + 16 * j;
      if (n < g.N) st1<T>(g.y, m * g.N + n, (float)acc[i][j] * (as * g.ws[g.w_per_col ? n : 0]));
    }
  }
}

template <typename T> int launch_any(const SmArgs &g, bool f8, cudaStream_t st) {
  const int64_t grid = (g.M + SA_TILE - 1) / SA_TILE * ((g.N + SA_TILE - 1) / SA_TILE);
  if (grid >= (int64_t)1 << 31) B2_FAIL(B2_ERR_UNSUPPORTED, "b200::ScaledMatMul: output too large");
  if (f8) scaled_mm_any<T, Fp8><<<(unsigned)grid, 256, 0, st>>>(g);
  else scaled_mm_any<T, Int8><<<(unsigned)grid, 256, 0, st>>>(g);
  B2_LAUNCH_CHECK();
  return B2_OK;
}

} // namespace
} // namespace b2

using namespace b2;

extern "C" int b2_scaled_matmul(const b2_tensor *a, const b2_tensor *a_scale, const b2_tensor *w,
                                const b2_tensor *w_scale, b2_tensor *y, void *workspace,
                                size_t *workspace_bytes, void *stream) {
#define SMM "b200::ScaledMatMul: "
  if (!a || !a_scale || !w || !w_scale || !y) B2_FAIL(B2_ERR_INVALID_ARGUMENT, SMM "null tensor");
  B2_ENFORCE(q8::is_q8(a->dtype) && w->dtype == a->dtype,
             SMM "A and W must be INT8 or FLOAT8E4M3FN of one dtype.");
  B2_ENFORCE(a->ndim >= 1 && w->ndim == 2 && w->shape[1] == a->shape[a->ndim - 1],
             SMM "W must be [N, K] with K the last dimension of A.");
  const int64_t K = w->shape[1], N = w->shape[0];
  int64_t M = 1;
  for (int i = 0; i + 1 < a->ndim; ++i) M *= a->shape[i];
  B2_ENFORCE(a_scale->dtype == kFloat && w_scale->dtype == kFloat, SMM "scales must be FLOAT.");
  const int64_t na = numel(a_scale), nw = numel(w_scale);
  B2_ENFORCE(na == M || na == 1, SMM "A_scale must have one value, or one per row of A.");
  B2_ENFORCE(nw == N || nw == 1, SMM "W_scale must have one value, or one per row of W.");
  std::vector<int64_t> want = shape_of(a);
  want.back() = N;
  B2_ENFORCE(q8::is_float_type(y->dtype) && shape_of(y) == want,
             SMM "Y must be FLOAT, FLOAT16 or BFLOAT16 of A's shape with N columns.");
  // |sum| <= 128 * 128 * K stays in int32
  if (a->dtype == kInt8 && K > 131071) B2_FAIL(B2_ERR_UNSUPPORTED, SMM "K above 131071 with INT8");
  const int wr = workspace_check(workspace, workspace_bytes, 0);
  if (wr != 0) return wr > 0 ? B2_OK : wr;
  if (M == 0 || N == 0) return B2_OK;
  B2_ENFORCE(q8::has_data(a) && q8::has_data(w) && a_scale->data && w_scale->data && y->data,
             SMM "a tensor has no data.");
  SmArgs g{};
  g.a = static_cast<const uint8_t *>(a->data);
  g.w = static_cast<const uint8_t *>(w->data);
  g.as = static_cast<const float *>(a_scale->data);
  g.ws = static_cast<const float *>(w_scale->data);
  g.y = y->data;
  g.M = M;
  g.N = N;
  g.K = K;
  g.a_per_row = na == M && M > 1;
  g.w_per_col = nw == N && N > 1;
  const bool f8 = a->dtype == kF8E4M3FN;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (scaled_skinny_eligible(g, f8)) return scaled_skinny_launch(g, y->dtype, f8, st);
  if (scaled_pair_eligible(g)) return scaled_pair_launch(g, y->dtype, f8, st);
  if (scaled_tc_eligible(g)) return scaled_tc_launch(g, y->dtype, f8, st);
  if (y->dtype == kFloat16) return launch_any<__half>(g, f8, st);
  if (y->dtype == kBfloat16) return launch_any<__nv_bfloat16>(g, f8, st);
  return launch_any<float>(g, f8, st);
#undef SMM
}
