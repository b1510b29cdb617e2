// The scaled 8-bit product (b2_scaled_matmul) on tcgen05 tensor cores: prompts and batches.
//
// Bound: tensor pipe for prompts, the ring's loads for few rows.  K = 4096, FLOAT8, in a graph: 32 x 11008
// outputs 10.7 us, 4.2 TB/s; 512 x 9472 18.7 us, 2130 TFLOP/s.
// A tile is 128 rows of A by BN rows of W; both are K-major, so one 128-byte-wide TMA box each (128-byte swizzle) feeds kind::i8 or kind::f8f6f4 with K = 32 a step.
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

// AR rows of A are loaded: with fewer rows than a tile's 128 the MMA reads past them whatever
// shared memory holds, which reaches no row that is stored.
template <int BN, int AR> struct StLayout {
  // 128-byte-wide blocks of K per stage: narrow tiles take two, so a stage's fixed cost in the
  // issuing threads (about 0.2 us) moves more bytes
  static constexpr int KB = BN <= 64 ? 2 : 1;
  static constexpr uint32_t A = AR * ST_BK, W = BN * ST_BK; // one block of each operand
  static constexpr uint32_t STAGE = KB * (A + W);           // A blocks, W blocks
  static constexpr uint32_t PAD = (ST_BM - AR) * ST_BK; // what the last stage's A is read past
  static constexpr int FIT = (int)((232448 - 4096 - PAD) / STAGE);
  static constexpr int STAGES = FIT < 16 ? FIT : 16;
  static constexpr size_t SMEM = (size_t)STAGES * STAGE + PAD + 1024 + 512 + 2 * 4 * BN; // and W's scales, twice
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

template <typename T, typename Q, int BN, int AR>
__global__ void __launch_bounds__(ST_THREADS, 1)
    scaled_mm_tc(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                 const StArgs g) {
  using L = StLayout<BN, AR>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *full = reinterpret_cast<uint64_t *>(sm + L::STAGES * L::STAGE + L::PAD);
  uint64_t *empty = full + L::STAGES;
  uint64_t *acc_full = empty + L::STAGES; // 2
  uint64_t *acc_empty = acc_full + 2;     // 2
  uint64_t *all_done = acc_empty + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(all_done + 1);
  float *scales = reinterpret_cast<float *>(sm + L::STAGES * L::STAGE + L::PAD + 512); // [2][BN]
  __shared__ volatile int abort_flag;
  const SmArgs &p = g.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = g.mt * g.nt, kt_count = (int)((p.K + L::KB * ST_BK - 1) / (L::KB * ST_BK));
  constexpr uint32_t BUF = BN <= 32 ? 32 : BN <= 64 ? 64 : BN <= 128 ? 128 : 256; // columns per buffer of sums
  constexpr uint32_t COLS = 2 * BUF;

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
      int i = 0, s = 0; // stages filled so far; the next one
      uint32_t phase = 1; // parity of its last release
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
        int mt, nt;
        tile_of(g, tile, &mt, &nt);
        for (int kt = 0; kt < kt_count; ++kt, ++i) {
          if (abort_flag || (i >= L::STAGES && !tc::mbar_wait(&empty[s], phase))) {
            if (!abort_flag) atomicExch(&g_scaled_tc_status, tc::kTimeoutEmpty);
            abort_flag = 1;
            ok = false;
            break;
          }
          uint8_t *st = sm + s * L::STAGE;
          tc::mbar_expect_tx(&full[s], L::STAGE);
#pragma unroll
          for (int b = 0; b < L::KB; ++b) { // blocks past K read as zeros
            tc::tma_load_2d(st + b * L::A, &map_a, &full[s], (kt * L::KB + b) * ST_BK, mt * ST_BM);
            tc::tma_load_2d(st + L::KB * L::A + b * L::W, &map_w, &full[s], (kt * L::KB + b) * ST_BK, nt * BN);
          }
          if (++s == L::STAGES) {
            s = 0;
            phase ^= 1;
          }
        }
      }
      // no copy may land after the CTA has left: wait (bounded) for each stage's last fill
      for (int j = max(0, i - L::STAGES); j < i; ++j) tc::mbar_wait(&full[j % L::STAGES], (j / L::STAGES) & 1);
    }
  } else if (warp == 1) {
    if (tc::elect_one()) {
      const uint32_t id = std::is_same<Q, Int8>::value ? tc::idesc(2, 1, 1, 0, 0, ST_BM, BN)
                                                       : tc::idesc(1, 0, 0, 0, 0, ST_BM, BN);
      // descriptors of stage 0's operands; a stage or 32 bytes of K further is an addition
      const uint64_t a0 = tc::sdesc_sw128(tc::smem_u32(sm), 16, 1024);
      const uint64_t w0 = tc::sdesc_sw128(tc::smem_u32(sm) + L::KB * L::A, 16, 1024);
      int s = 0, c = 0; // next stage; tiles consumed
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x, ++c) {
        const int b = c & 1;
        if (c >= 2 && !tc::mbar_wait(&acc_empty[b], ((c >> 1) - 1) & 1)) {
          ok = false;
          break;
        }
        tc::tc_fence_after();
        for (int kt = 0; kt < kt_count; ++kt) {
          if (abort_flag || !tc::mbar_wait(&full[s], phase)) {
            ok = false;
            break;
          }
          tc::tc_fence_after();
          const uint64_t at = (uint64_t)(s * (L::STAGE >> 4));
#pragma unroll
          for (int kb = 0; kb < L::KB; ++kb)
#pragma unroll
            for (int kk = 0; kk < ST_BK / 32; ++kk) {
              const uint64_t ad = a0 + at + kb * (L::A >> 4) + kk * 2, wd = w0 + at + kb * (L::W >> 4) + kk * 2;
              const uint32_t more = (kt > 0 || kb > 0 || kk > 0) ? 1u : 0u;
              if constexpr (std::is_same<Q, Int8>::value) tc::mma_i8(tmem + b * BUF, ad, wd, id, more);
              else mma_f8(tmem + b * BUF, ad, wd, id, more);
            }
          tc::tc_commit(&empty[s]);
          if (++s == L::STAGES) {
            s = 0;
            phase ^= 1;
          }
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
    bool failed = false;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++c) {
      const int b = c & 1;
      int mt, nt;
      tile_of(g, tile, &mt, &nt);
      // the tile's scales, while its sums are still under way; two buffers, so one barrier a tile
      // keeps a slow warp's from being overwritten
      const int64_t m = (int64_t)mt * ST_BM + q * 32 + lane, n0 = (int64_t)nt * BN;
      const float as = m < p.M ? __ldg(p.as + (p.a_per_row ? m : 0)) : 0.0f;
      float *ws = scales + b * BN;
      for (int e = threadIdx.x - 64; e < BN; e += 128)
        ws[e] = n0 + e < p.N ? __ldg(p.ws + (p.w_per_col ? n0 + e : 0)) : 0.0f;
      asm volatile("bar.sync 1, 128;" ::: "memory");
      const bool ok = !abort_flag && tc::mbar_wait(&acc_full[b], (c >> 1) & 1, 2 * kWaitNs);
      if (!__all_sync(0xffffffffu, ok)) {
        if (lane == 0 && !abort_flag) atomicExch(&g_scaled_tc_status, tc::kTimeoutMma);
        abort_flag = 1;
        failed = true;
      }
      if (failed) continue; // the other warps still count on the barrier
      tc::tc_fence_after();
      const int left = (int)min(p.N - n0, (int64_t)BN);
      T *y = static_cast<T *>(p.y) + m * p.N + n0;
#pragma unroll 1
      for (int ch = 0; ch < BN / 32; ++ch) {
        if (ch * 32 >= left) break;
        uint32_t r[32];
        tc::tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(b * BUF + ch * 32), r);
        tc::tmem_ld_wait();
        if (m < p.M) store_scaled32<T, Q>(y + ch * 32, left - ch * 32, as, ws + ch * 32, r, vec);
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

template <typename T, typename Q, int BN, int AR>
int launch(const CUtensorMap &ma, const CUtensorMap &mw, const StArgs &g, cudaStream_t st) {
  using L = StLayout<BN, AR>;
  auto kern = scaled_mm_tc<T, Q, BN, AR>;
  B2_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::SMEM));
  const int grid = std::min(g.mt * g.nt, sm_count());
  kern<<<grid, ST_THREADS, L::SMEM, st>>>(ma, mw, g);
  B2_LAUNCH_CHECK();
  return B2_OK;
}

template <typename T, typename Q>
int pick(int bn, int ar, const CUtensorMap &ma, const CUtensorMap &mw, const StArgs &g, cudaStream_t st) {
  switch (bn) {
#define B2_WIDTH(BN)                                                                                                    \
  case BN:                                                                                                             \
    return ar == 32 ? launch<T, Q, BN, 32>(ma, mw, g, st) : launch<T, Q, BN, 128>(ma, mw, g, st)
    B2_WIDTH(256);
    B2_WIDTH(192);
    B2_WIDTH(160);
    B2_WIDTH(128);
    B2_WIDTH(96);
    B2_WIDTH(64);
#undef B2_WIDTH
  }
  return ar == 32 ? launch<T, Q, 32, 32>(ma, mw, g, st) : launch<T, Q, 32, 128>(ma, mw, g, st);
}

} // namespace

bool scaled_tc_eligible(const SmArgs &g) {
  const int64_t tiles = (g.M + ST_BM - 1) / ST_BM * ((g.N + 31) / 32);
  return g.K > 0 && g.K % 16 == 0 && aligned(g.a, 16) && aligned(g.w, 16) && tiles < ((int64_t)1 << 30) &&
         g.K < ((int64_t)1 << 30);
}

int scaled_tc_launch(const SmArgs &p, int y_dtype, bool f8, cudaStream_t st) {
  StArgs g{};
  g.p = p;
  g.mt = (int)((p.M + ST_BM - 1) / ST_BM);
  // Tile width: a tile's time grows like its width plus a fixed part (K = 4096, one tile per SM: 4.4,
  // 5.0, 8 and 11 us past the launch for 32, 64, 128 and 256 columns), and the busiest SM sets the
  // call's.  32 x 11008 outputs: 16.6, 14.6, 12.3 and 16.6 us with 3, 2, 1 and 1 tiles on it.  The widths
  // between the powers of two fill a last round: 200 x 11008 16.7 -> 13.0 us (192 columns), 600 x 4096
  // 15.8 -> 12.4 (160), 512 x 11008 29.1 -> 22.3 (160), 128 x 11008 11.9 -> 11.4 (96).
  int bn = 256;
  int64_t best = INT64_MAX;
  for (const int w : {256, 192, 160, 128, 96, 64, 32}) {
    const int64_t tiles = g.mt * ((p.N + w - 1) / w), cost = (tiles + sm_count() - 1) / sm_count() * (w + 96);
    if (cost < best) {
      best = cost;
      bn = w;
    }
  }
  // (128-row boxes over fewer than 32 rows are slow: 17 rows 17.9 us, with 32-row boxes 11.6)
  const int ar = p.M <= 32 ? 32 : ST_BM;
  g.nt = (int)((p.N + bn - 1) / bn);
  CUtensorMap ma, mw;
  const uint64_t strides[1] = {(uint64_t)p.K};
  const uint64_t da[2] = {(uint64_t)p.K, (uint64_t)p.M}, dw[2] = {(uint64_t)p.K, (uint64_t)p.N};
  const uint32_t ba[2] = {ST_BK, (uint32_t)ar}, bw[2] = {ST_BK, (uint32_t)bn};
  if (int rc = make_tensor_map(&ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, p.a, da, strides, ba, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  if (int rc = make_tensor_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, p.w, dw, strides, bw, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  if (y_dtype == kFloat16) return f8 ? pick<__half, Fp8>(bn, ar, ma, mw, g, st) : pick<__half, Int8>(bn, ar, ma, mw, g, st);
  if (y_dtype == kBfloat16)
    return f8 ? pick<__nv_bfloat16, Fp8>(bn, ar, ma, mw, g, st) : pick<__nv_bfloat16, Int8>(bn, ar, ma, mw, g, st);
  return f8 ? pick<float, Fp8>(bn, ar, ma, mw, g, st) : pick<float, Int8>(bn, ar, ma, mw, g, st);
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
