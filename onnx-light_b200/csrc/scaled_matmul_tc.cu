// The scaled 8-bit product (b2_scaled_matmul) on tcgen05 tensor cores: prompts and batches.
//
// Bound: tensor pipe for prompts.  A tile is 128 rows of A by BN rows of W; both are K-major, so one
// 128-byte-wide TMA box each (128-byte swizzle) feeds kind::i8 or kind::f8f6f4 with K = 32 a step.
// Persistent CTAs, one per SM, 192 threads:
//   warp 0     TMA producer: a ring of [128 + BN] x 128-byte stages that runs on across tiles;
//   warp 1     MMA issuer: BN columns of TMEM per tile, two buffers, so the next tile's sums start
//              while the last tile's are read;
//   warps 2-5  read TMEM, multiply by the two scales in fp32, round once and store.
// Tiles are numbered in bands of 8 tile rows, column by column, so that a wave of CTAs shares its
// rows of A and W in L2.  Every wait is bounded; after a time-out the CTA records a code, lets
// its own copies and MMAs in flight finish, frees its TMEM and returns.
#include <algorithm>

#include "scaled_matmul.cuh"
#include "tc_common.cuh"

namespace b2 {

__device__ int g_scaled_tc_status;

namespace {

using namespace q8;

constexpr int ST_BM = 128, ST_BK = 128, ST_THREADS = 192, ST_BAND = 8;
constexpr uint32_t ST_A = ST_BM * ST_BK;

template <int BN> struct StLayout {
  static constexpr uint32_t STAGE = ST_A + BN * ST_BK;
  static constexpr int STAGES = BN == 256 ? 4 : BN == 128 ? 6 : 8;
  static constexpr size_t SMEM = (size_t)STAGES * STAGE + 1024 + 512;
};

struct StArgs {
  SmArgs p;
  int mt, nt; // tiles
};

__device__ __forceinline__ void mma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\t"
               "setp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
               "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
               : "memory");
}

// Tile t of the numbering: bands of ST_BAND tile rows, column by column inside a band.
__device__ __forceinline__ void tile_of(const StArgs &g, int t, int *m, int *n) {
  const int band = t / (ST_BAND * g.nt), first = band * ST_BAND, height = min(ST_BAND, g.mt - first);
  const int r = t - band * ST_BAND * g.nt;
  *n = r / height;
  *m = first + r - *n * height;
}

template <typename T, typename Q>
__device__ __forceinline__ void store32(const SmArgs &p, int64_t m, int64_t n0, float as,
                                        const uint32_t (&r)[32], bool vec) {
  float v[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const float s = std::is_same<Q, Int8>::value ? (float)(int)r[j] : __uint_as_float(r[j]);
    const int64_t n = n0 + j;
    v[j] = s * (as * (p.w_per_col ? (n < p.N ? __ldg(p.ws + n) : 0.0f) : __ldg(p.ws)));
  }
  T *y = static_cast<T *>(p.y) + m * p.N + n0;
  if (vec && n0 + 32 <= p.N) {
#pragma unroll
    for (int j = 0; j < 32; j += 8) {
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = v[j + e];
      Raw8<T>::store(y + j, f);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (n0 + j < p.N) st1<T>(y, j, v[j]);
  }
}

template <typename T, typename Q, int BN>
__global__ void __launch_bounds__(ST_THREADS, 1)
    scaled_mm_tc(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                 const StArgs g) {
  using L = StLayout<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *full = reinterpret_cast<uint64_t *>(sm + L::STAGES * L::STAGE);
  uint64_t *empty = full + L::STAGES;
  uint64_t *acc_full = empty + L::STAGES; // 2
  uint64_t *acc_empty = acc_full + 2;     // 2
  uint64_t *all_done = acc_empty + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(all_done + 1);
  __shared__ volatile int abort_flag;
  const SmArgs &p = g.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = g.mt * g.nt, kt_count = (int)((p.K + ST_BK - 1) / ST_BK);
  constexpr uint32_t COLS = 2 * BN < 32 ? 32 : 2 * BN;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < L::STAGES; ++s) {
      tc::mbar_init(&full[s], 1);
      tc::mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(&acc_full[b], 1);
      tc::mbar_init(&acc_empty[b], 4);
    }
    tc::mbar_init(all_done, 1);
    tc::fence_barrier_init();
  }
  if (warp == 1) {
    tc::tmem_alloc(tmem_slot, COLS);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (tc::elect_one()) {
      tc::prefetch_tensormap(&map_a);
      tc::prefetch_tensormap(&map_w);
      int i = 0; // stages filled so far
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
        int mt, nt;
        tile_of(g, tile, &mt, &nt);
        for (int kt = 0; kt < kt_count; ++kt, ++i) {
          const int s = i % L::STAGES;
          if (abort_flag || (i >= L::STAGES && !tc::mbar_wait(&empty[s], ((i / L::STAGES) - 1) & 1))) {
            if (!abort_flag) atomicExch(&g_scaled_tc_status, tc::kTimeoutEmpty);
            abort_flag = 1;
            ok = false;
            break;
          }
          uint8_t *st = sm + s * L::STAGE;
          tc::mbar_expect_tx(&full[s], L::STAGE);
          tc::tma_load_2d(st, &map_a, &full[s], kt * ST_BK, mt * ST_BM);
          tc::tma_load_2d(st + ST_A, &map_w, &full[s], kt * ST_BK, nt * BN);
        }
      }
      // no copy may land after the CTA has left: wait (bounded) for each stage's last fill
      for (int j = max(0, i - L::STAGES); j < i; ++j) tc::mbar_wait(&full[j % L::STAGES], (j / L::STAGES) & 1);
    }
  } else if (warp == 1) {
    if (tc::elect_one()) {
      const uint32_t id = std::is_same<Q, Int8>::value ? tc::idesc(2, 1, 1, 0, 0, ST_BM, BN)
                                                       : tc::idesc(1, 0, 0, 0, 0, ST_BM, BN);
      int i = 0, c = 0; // stages, tiles consumed
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x, ++c) {
        const int b = c & 1;
        if (c >= 2 && !tc::mbar_wait(&acc_empty[b], ((c >> 1) - 1) & 1)) {
          ok = false;
          break;
        }
        tc::tc_fence_after();
        for (int kt = 0; kt < kt_count; ++kt, ++i) {
          const int s = i % L::STAGES;
          if (abort_flag || !tc::mbar_wait(&full[s], (i / L::STAGES) & 1)) {
            ok = false;
            break;
          }
          tc::tc_fence_after();
          const uint32_t ab = tc::smem_u32(sm + s * L::STAGE), wb = ab + ST_A;
#pragma unroll
          for (int kk = 0; kk < ST_BK / 32; ++kk) {
            const uint64_t ad = tc::sdesc_sw128(ab + kk * 32, 16, 1024);
            const uint64_t wd = tc::sdesc_sw128(wb + kk * 32, 16, 1024);
            const uint32_t more = (kt > 0 || kk > 0) ? 1u : 0u;
            if constexpr (std::is_same<Q, Int8>::value) tc::mma_i8(tmem + b * BN, ad, wd, id, more);
            else mma_f8(tmem + b * BN, ad, wd, id, more);
          }
          tc::tc_commit(&empty[s]);
        }
        if (ok) tc::tc_commit(&acc_full[b]);
      }
      if (!ok) {
        atomicExch(&g_scaled_tc_status, tc::kTimeoutFull);
        abort_flag = 1;
      }
      // TMEM is freed below: wait (bounded) until every issued MMA is done
      tc::tc_commit(all_done);
      tc::mbar_wait(all_done, 0);
    }
  } else {
    const int q = warp & 3; // TMEM lanes 32 q ..
    const bool vec = p.N % 8 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
    int c = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++c) {
      const int b = c & 1;
      const bool ok = !abort_flag && tc::mbar_wait(&acc_full[b], (c >> 1) & 1, 2 * kWaitNs);
      if (!__all_sync(0xffffffffu, ok)) {
        if (lane == 0 && !abort_flag) {
          atomicExch(&g_scaled_tc_status, tc::kTimeoutMma);
          abort_flag = 1;
        }
        break;
      }
      tc::tc_fence_after();
      int mt, nt;
      tile_of(g, tile, &mt, &nt);
      const int64_t m = (int64_t)mt * ST_BM + q * 32 + lane;
      const float as = m < p.M ? __ldg(p.as + (p.a_per_row ? m : 0)) : 0.0f;
#pragma unroll 1
      for (int ch = 0; ch < BN / 32; ++ch) {
        uint32_t r[32];
        tc::tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(b * BN + ch * 32), r);
        tc::tmem_ld_wait();
        const int64_t n0 = (int64_t)nt * BN + ch * 32;
        if (m < p.M && n0 < p.N) store32<T, Q>(p, m, n0, as, r, vec);
      }
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&acc_empty[b]);
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) tc::tmem_dealloc(tmem, COLS);
}

template <typename T, typename Q, int BN>
int launch(const CUtensorMap &ma, const CUtensorMap &mw, const StArgs &g, cudaStream_t st) {
  auto kern = scaled_mm_tc<T, Q, BN>;
  B2_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)StLayout<BN>::SMEM));
  const int grid = std::min(g.mt * g.nt, sm_count());
  kern<<<grid, ST_THREADS, StLayout<BN>::SMEM, st>>>(ma, mw, g);
  B2_LAUNCH_CHECK();
  return B2_OK;
}

template <typename T, typename Q>
int pick(int bn, const CUtensorMap &ma, const CUtensorMap &mw, const StArgs &g, cudaStream_t st) {
  if (bn == 256) return launch<T, Q, 256>(ma, mw, g, st);
  if (bn == 128) return launch<T, Q, 128>(ma, mw, g, st);
  return launch<T, Q, 64>(ma, mw, g, st);
}

} // namespace

bool scaled_tc_eligible(const SmArgs &g) {
  const int64_t tiles = (g.M + ST_BM - 1) / ST_BM * ((g.N + 63) / 64);
  return g.K > 0 && g.K % 16 == 0 && aligned(g.a, 16) && aligned(g.w, 16) && tiles < ((int64_t)1 << 30) &&
         g.K < ((int64_t)1 << 30);
}

int scaled_tc_launch(const SmArgs &p, int y_dtype, bool f8, cudaStream_t st) {
  StArgs g{};
  g.p = p;
  g.mt = (int)((p.M + ST_BM - 1) / ST_BM);
  // the widest tile that still gives every SM one
  int bn = 256;
  while (bn > 64 && (int64_t)g.mt * ((p.N + bn - 1) / bn) < sm_count()) bn /= 2;
  g.nt = (int)((p.N + bn - 1) / bn);
  CUtensorMap ma, mw;
  const uint64_t strides[1] = {(uint64_t)p.K};
  const uint64_t da[2] = {(uint64_t)p.K, (uint64_t)p.M}, dw[2] = {(uint64_t)p.K, (uint64_t)p.N};
  const uint32_t ba[2] = {ST_BK, ST_BM}, bw[2] = {ST_BK, (uint32_t)bn};
  if (int rc = make_tensor_map(&ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, p.a, da, strides, ba, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  if (int rc = make_tensor_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, p.w, dw, strides, bw, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  if (y_dtype == kFloat16) return f8 ? pick<__half, Fp8>(bn, ma, mw, g, st) : pick<__half, Int8>(bn, ma, mw, g, st);
  if (y_dtype == kBfloat16)
    return f8 ? pick<__nv_bfloat16, Fp8>(bn, ma, mw, g, st) : pick<__nv_bfloat16, Int8>(bn, ma, mw, g, st);
  return f8 ? pick<float, Fp8>(bn, ma, mw, g, st) : pick<float, Int8>(bn, ma, mw, g, st);
}

int status_read_scaled_tc(int reset) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_scaled_tc_status, sizeof(int)) != cudaSuccess) return -1;
  if (reset && v) {
    const int z = 0;
    if (cudaMemcpyToSymbol(g_scaled_tc_status, &z, sizeof(int)) != cudaSuccess) return -1;
  }
  return v;
}

} // namespace b2
