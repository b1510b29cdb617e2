// The scaled 8-bit product (b2_scaled_matmul) for few rows of A: decode steps.
//
// Bound: HBM, the weight's N x K bytes read once.  A CTA owns 16 RT rows of W (output columns) over
// the whole K, so nothing is merged between CTAs; its eight warps take the 128-byte segments of K in
// turn and stream them straight into registers, UNROLL segments ahead.  The weights are the 16-row M
// side of mma.sync m16n8k32 and the rows of A its 8-wide N side.  A dot product does not care in
// which order it takes k, so a lane's 32 consecutive bytes of a row serve as the k indices of four
// MMA steps, for both operands alike: every load is a full 16 bytes and no byte moves between lanes.
// Measured: one row, 4096 x 4096 FLOAT8, 5.1 us in a graph, 3.3 TB/s (launch and first loads 2 of it).
#include "scaled_matmul.cuh"

namespace b2 {
namespace {

using namespace q8;

constexpr int SK_WARPS = 8;

template <typename Q, typename Acc>
__device__ __forceinline__ void mma_k32(Acc (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<Q, Int8>::value)
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
                 "{%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
                 "{%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 ldg_stream(const uint8_t *p) { // read once
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

template <typename T, typename Q, int NT, int RT, int UNROLL>
__global__ void __launch_bounds__(SK_WARPS * 32) scaled_mm_skinny(const SmArgs g) {
  using Acc = typename std::conditional<std::is_same<Q, Int8>::value, int, float>::type;
  __shared__ Acc red[SK_WARPS][16 * RT][8 * NT + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, t = lane & 3;
  const int64_t n0 = (int64_t)blockIdx.x * (16 * RT);
  Acc acc[RT][NT][4] = {};
  const uint8_t *wp[RT][2];
  bool wv[RT][2];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t n = n0 + r * 16 + h * 8 + gq;
      wv[r][h] = n < g.N;
      wp[r][h] = g.w + (wv[r][h] ? n : 0) * g.K + 32 * t;
    }
  const uint8_t *ap[NT];
  bool av[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int m = j * 8 + gq;
    av[j] = m < g.M;
    ap[j] = g.a + (int64_t)(av[j] ? m : 0) * g.K + 32 * t;
  }
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  for (int64_t k0 = (int64_t)warp * 128; k0 < g.K; k0 += SK_WARPS * 128 * UNROLL) {
    uint4 w[UNROLL][RT][2][2];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int64_t k = k0 + (int64_t)u * SK_WARPS * 128;
      const bool in0 = k + 32 * t < g.K, in1 = k + 32 * t + 16 < g.K; // K is a multiple of 16
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          w[u][r][h][0] = wv[r][h] && in0 ? ldg_stream(wp[r][h] + k) : zero;
          w[u][r][h][1] = wv[r][h] && in1 ? ldg_stream(wp[r][h] + k + 16) : zero;
        }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int64_t k = k0 + (int64_t)u * SK_WARPS * 128;
      if (k >= g.K) break;
      const bool in0 = k + 32 * t < g.K, in1 = k + 32 * t + 16 < g.K;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const uint4 x0 = av[j] && in0 ? __ldg(reinterpret_cast<const uint4 *>(ap[j] + k)) : zero;
        const uint4 x1 = av[j] && in1 ? __ldg(reinterpret_cast<const uint4 *>(ap[j] + k + 16)) : zero;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const uint4 *lo = w[u][r][0], *hi = w[u][r][1];
          mma_k32<Q>(acc[r][j], lo[0].x, hi[0].x, lo[0].y, hi[0].y, x0.x, x0.y);
          mma_k32<Q>(acc[r][j], lo[0].z, hi[0].z, lo[0].w, hi[0].w, x0.z, x0.w);
          mma_k32<Q>(acc[r][j], lo[1].x, hi[1].x, lo[1].y, hi[1].y, x1.x, x1.y);
          mma_k32<Q>(acc[r][j], lo[1].z, hi[1].z, lo[1].w, hi[1].w, x1.z, x1.w);
        }
      }
    }
  }
  // sum over the warps in order
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[warp][r * 16 + (e >> 1) * 8 + gq][j * 8 + 2 * t + (e & 1)] = acc[r][j][e];
  __syncthreads();
  for (int e = threadIdx.x; e < 16 * RT * 8 * NT; e += SK_WARPS * 32) {
    const int nn = e % (16 * RT), m = e / (16 * RT);
    const int64_t n = n0 + nn;
    if (m >= g.M || n >= g.N) continue;
    Acc s = 0;
#pragma unroll
    for (int w = 0; w < SK_WARPS; ++w) s += red[w][nn][m];
    st1<T>(g.y, (int64_t)m * g.N + n, (float)s * (g.as[g.a_per_row ? m : 0] * g.ws[g.w_per_col ? n : 0]));
  }
}

template <typename T, typename Q> int pick(const SmArgs &g, cudaStream_t st) {
  const int64_t tiles = (g.N + 15) / 16;
  if (g.M <= 8) scaled_mm_skinny<T, Q, 1, 1, 4><<<(unsigned)tiles, SK_WARPS * 32, 0, st>>>(g);
  else if (g.M <= 16) scaled_mm_skinny<T, Q, 2, 1, 4><<<(unsigned)tiles, SK_WARPS * 32, 0, st>>>(g);
  else scaled_mm_skinny<T, Q, 4, 1, 2><<<(unsigned)tiles, SK_WARPS * 32, 0, st>>>(g);
  B2_LAUNCH_CHECK();
  return B2_OK;
}

} // namespace

// Against the tcgen05 kernel (us in a graph with weights from HBM, K x N, here / there).  Up to two
// million codes, where a launch counts: 32 rows 1024 x 1024 3.1 / 4.1, 4096 x 512 4.9 / 7.2.  4096 x 4096:
// INT8 1 row 5.4 / 9.4, 16 rows 6.2 / 8.4, 32 rows 8.0 / 8.3; FLOAT8, whose mma.sync is slower, 8 rows
// 6.1 / 8.8, 16 rows 8.6 / 8.6, 32 rows 11.8 / 8.5.  4096 x 11008: INT8 1 row 11.9 / 12.2, 16 rows
// 15.0 / 12.1; FLOAT8 1 row 13.0 / 12.4, 8 rows 14.5 / 12.4.  So the limits of 16 and 8 rows hold for
// weights of some ten million codes and are up to 3 us late for the largest.
bool scaled_skinny_eligible(const SmArgs &g, bool f8) {
  const int64_t rows = g.N * g.K <= (1 << 21) ? 32 : f8 ? 8 : 16;
  return g.M <= rows && g.K > 0 && g.K % 16 == 0 && aligned(g.a, 16) && aligned(g.w, 16) &&
         g.N < ((int64_t)1 << 34);
}

int scaled_skinny_launch(const SmArgs &g, int y_dtype, bool f8, cudaStream_t st) {
  if (y_dtype == kFloat16) return f8 ? pick<__half, Fp8>(g, st) : pick<__half, Int8>(g, st);
  if (y_dtype == kBfloat16) return f8 ? pick<__nv_bfloat16, Fp8>(g, st) : pick<__nv_bfloat16, Int8>(g, st);
  return f8 ? pick<float, Fp8>(g, st) : pick<float, Int8>(g, st);
}

} // namespace b2
