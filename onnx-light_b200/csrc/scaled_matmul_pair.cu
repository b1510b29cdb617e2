// The scaled 8-bit product (b2_scaled_matmul) on pairs of SMs: large products.
//
// Bound: tensor pipe.  One SM alone is held back by its shared memory: a 128 x 256 tile writes 48 KB and
// reads 48 KB per 128 columns of K, 190 bytes a cycle at the full MMA rate of which an SM moves 128.
// Here two CTAs of a cluster share a 256 x 256 tile (tcgen05 cta_group::2): each loads its 128 rows
// of A and its half of W (32 KB per 128 columns), and every MMA, issued by the first CTA, multiplies
// both halves of A by both halves of W.  Each CTA's TMEM holds the sums of its own 128 rows, two
// buffers, so the epilogue of a tile runs under the next one's sums.
//   warp 0     TMA producer of the CTA's own operands; both CTAs' copies count on the first CTA's barrier
//   warp 1     of the first CTA: MMA issuer; its commits release the stage and hand over the sums in
//              both CTAs
//   warps 2-5  the CTA's epilogue, as in the one-CTA kernel
// Measured: 8192 x 4096 x 11008 FLOAT8 264 us for a launch alone (2795 TFLOP/s, tensor pipe 84 % active),
// 323 to 346 us back to back, where the power limit lowers the clock.
// Tile numbering, scales and rounding are the one-CTA kernel's.  Every wait is bounded; the CTAs of a
// pair leave together, after each has seen its own copies consumed (or given up waiting).
#include <algorithm>

#include "scaled_matmul.cuh"
#include "tc_common.cuh"

namespace b2 {

__device__ int g_scaled_pair_status;

namespace {

using namespace q8;

constexpr int SP_BM = 128, SP_BN = 256, SP_BK = 128, SP_THREADS = 192, SP_STAGES = 6, SP_BAND = 8;
constexpr uint32_t SP_A = SP_BM * SP_BK, SP_STAGE = 2 * SP_A; // A rows, half of W's rows
constexpr size_t SP_SMEM = (size_t)SP_STAGES * SP_STAGE + 1024 + 512 + 2 * 4 * SP_BN;

struct SpArgs {
  SmArgs p;
  int mt, nt; // tiles of 256 x 256
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Address of this CTA's shared-memory object in the cluster's CTA `rank`.
__device__ __forceinline__ uint32_t map_rank(const void *p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(tc::smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A tile into this CTA's shared memory, its bytes counted on a barrier of either CTA of the pair.
__device__ __forceinline__ void pair_load(void *dst, const CUtensorMap *map, uint32_t bar, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
               " [%0], [%1, {%3, %4}], [%2];" ::"r"(tc::smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
               : "memory");
}
template <typename Q>
__device__ __forceinline__ void pair_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t more) {
  if constexpr (std::is_same<Q, Int8>::value)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(more)
                 : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(more)
                 : "memory");
}
// Arrives on both CTAs' barrier once every MMA issued so far is done.
__device__ __forceinline__ void pair_commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                   tc::smem_u32(bar)),
               "h"((uint16_t)3)
               : "memory");
}

__device__ __forceinline__ void pair_tile(const SpArgs &g, int t, int *m, int *n) {
  const int band = t / (SP_BAND * g.nt), first = band * SP_BAND, height = min(SP_BAND, g.mt - first);
  const int r = t - band * SP_BAND * g.nt;
  *n = r / height;
  *m = first + r - *n * height;
}

template <typename T, typename Q>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(SP_THREADS, 1)
    scaled_mm_pair(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                   const SpArgs g) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *full = reinterpret_cast<uint64_t *>(sm + SP_STAGES * SP_STAGE); // counted in the first CTA
  uint64_t *empty = full + SP_STAGES;     // in both
  uint64_t *acc_full = empty + SP_STAGES; // 2, in both
  uint64_t *acc_empty = acc_full + 2;     // 2, counted in the first CTA
  uint64_t *all_done = acc_empty + 2;     // in both
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(all_done + 1);
  float *scales = reinterpret_cast<float *>(sm + SP_STAGES * SP_STAGE + 512); // [2][SP_BN]
  __shared__ volatile int abort_flag;
  const SmArgs &p = g.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int tiles = g.mt * g.nt, kt_count = (int)((p.K + SP_BK - 1) / SP_BK);
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < SP_STAGES; ++s) {
      tc::mbar_init(&full[s], 1);
      tc::mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(&acc_full[b], 1);
      tc::mbar_init(&acc_empty[b], 8); // four epilogue warps of each CTA
    }
    tc::mbar_init(all_done, 1);
    tc::fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(tmem_slot)), "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc::tc_fence_before();
  __syncthreads();
  cluster_sync(); // both CTAs' barriers are ready
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (tc::elect_one()) {
      tc::prefetch_tensormap(&map_a);
      tc::prefetch_tensormap(&map_w);
      int i = 0, s = 0;
      uint32_t phase = 1; // parity of the next stage's last release
      bool ok = true;
      for (int tile = pair; ok && tile < tiles; tile += pairs) {
        int mt, nt;
        pair_tile(g, tile, &mt, &nt);
        const int row_a = (2 * mt + (int)rank) * SP_BM, row_w = nt * SP_BN + (int)rank * (SP_BN / 2);
        for (int kt = 0; kt < kt_count; ++kt, ++i) {
          if (abort_flag || (i >= SP_STAGES && !tc::mbar_wait(&empty[s], phase))) {
            if (!abort_flag) atomicExch(&g_scaled_pair_status, tc::kTimeoutEmpty);
            abort_flag = 1;
            ok = false;
            break;
          }
          // the first CTA expects both CTAs' bytes (the other's may land first: the phase stays open)
          if (rank == 0) tc::mbar_expect_tx(&full[s], 2 * SP_STAGE);
          const uint32_t bar = map_rank(&full[s], 0);
          uint8_t *st = sm + s * SP_STAGE;
          pair_load(st, &map_a, bar, kt * SP_BK, row_a);
          pair_load(st + SP_A, &map_w, bar, kt * SP_BK, row_w);
          if (++s == SP_STAGES) {
            s = 0;
            phase ^= 1;
          }
        }
      }
      // No copy may land after the CTA has left: each stage's last fill is consumed before its release
      // (bounded; after a give-up the copies have long landed when the wait runs out).
      for (int j = max(0, i - SP_STAGES); j < i; ++j) tc::mbar_wait(&empty[j % SP_STAGES], (j / SP_STAGES) & 1);
    }
  } else if (warp == 1) {
    if (rank == 0 && tc::elect_one()) {
      const uint32_t id = std::is_same<Q, Int8>::value ? tc::idesc(2, 1, 1, 0, 0, 2 * SP_BM, SP_BN)
                                                       : tc::idesc(1, 0, 0, 0, 0, 2 * SP_BM, SP_BN);
      const uint64_t a0 = tc::sdesc_sw128(tc::smem_u32(sm), 16, 1024);
      const uint64_t w0 = tc::sdesc_sw128(tc::smem_u32(sm) + SP_A, 16, 1024);
      int s = 0, c = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < tiles; tile += pairs, ++c) {
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
          const uint64_t at = (uint64_t)(s * (SP_STAGE >> 4));
#pragma unroll
          for (int kk = 0; kk < SP_BK / 32; ++kk)
            pair_mma<Q>(tmem + b * SP_BN, a0 + at + kk * 2, w0 + at + kk * 2, id, (kt > 0 || kk > 0) ? 1u : 0u);
          pair_commit(&empty[s]);
          if (++s == SP_STAGES) {
            s = 0;
            phase ^= 1;
          }
        }
        if (ok) pair_commit(&acc_full[b]);
      }
      if (!ok) {
        atomicExch(&g_scaled_pair_status, tc::kTimeoutFull);
        abort_flag = 1;
      }
      // TMEM is freed below: wait (bounded) until every issued MMA is done
      pair_commit(all_done);
      tc::mbar_wait(all_done, 0);
    }
  } else {
    const int q = warp & 3; // TMEM lanes 32 q ..
    const bool vec = p.N % 8 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
    int c = 0;
    bool failed = false;
    for (int tile = pair; tile < tiles; tile += pairs, ++c) {
      const int b = c & 1;
      int mt, nt;
      pair_tile(g, tile, &mt, &nt);
      const int64_t m = (int64_t)(2 * mt + rank) * SP_BM + q * 32 + lane, n0 = (int64_t)nt * SP_BN;
      const float as = m < p.M ? __ldg(p.as + (p.a_per_row ? m : 0)) : 0.0f;
      float *ws = scales + b * SP_BN;
      for (int e = threadIdx.x - 64; e < SP_BN; e += 128)
        ws[e] = n0 + e < p.N ? __ldg(p.ws + (p.w_per_col ? n0 + e : 0)) : 0.0f;
      asm volatile("bar.sync 1, 128;" ::: "memory");
      const bool ok = !abort_flag && !failed && tc::mbar_wait(&acc_full[b], (c >> 1) & 1, 2 * kWaitNs);
      if (!__all_sync(0xffffffffu, ok)) {
        if (lane == 0 && !abort_flag) atomicExch(&g_scaled_pair_status, tc::kTimeoutMma);
        abort_flag = 1;
        failed = true;
        continue; // the other warps still count on the barrier
      }
      tc::tc_fence_after();
      const int left = (int)min(p.N - n0, (int64_t)SP_BN);
      T *y = static_cast<T *>(p.y) + m * p.N + n0;
#pragma unroll 1
      for (int ch = 0; ch < SP_BN / 32; ++ch) {
        if (ch * 32 >= left) break;
        uint32_t r[32];
        tc::tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(b * SP_BN + ch * 32), r);
        tc::tmem_ld_wait();
        if (m < p.M) store_scaled32<T, Q>(y + ch * 32, left - ch * 32, as, ws + ch * 32, r, vec);
      }
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0)
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(map_rank(&acc_empty[b], 0)) : "memory");
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  cluster_sync(); // the other CTA's copies, MMAs and arrivals are done with this one
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

template <typename T, typename Q>
int launch(const CUtensorMap &ma, const CUtensorMap &mw, const SpArgs &g, cudaStream_t st) {
  auto kern = scaled_mm_pair<T, Q>;
  B2_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SP_SMEM));
  const int grid = 2 * std::min(g.mt * g.nt, sm_count() / 2);
  kern<<<grid, SP_THREADS, SP_SMEM, st>>>(ma, mw, g);
  B2_LAUNCH_CHECK();
  return B2_OK;
}

} // namespace

// From two rounds of tiles on every pair of SMs: 8192 x 4096 x 11008 takes the one-CTA kernel 355 us and
// this one 346 on the same box.  With fewer tiles neither is ahead (K = 4096, FLOAT8, one CTA against
// pairs, us: 512 x 9472 22.5 / 24.6, 2048 x 4096 32.8 / 32.8), and the one-CTA kernel has narrower tiles to
// fill a round with (512 x 11008 23.2 / 34.8, 1536 x 4096 24.1 / 32.8).
bool scaled_pair_eligible(const SmArgs &g) {
  const int64_t tiles = (g.M + 2 * SP_BM - 1) / (2 * SP_BM) * ((g.N + SP_BN - 1) / SP_BN);
  return g.K > 0 && g.K % 16 == 0 && aligned(g.a, 16) && aligned(g.w, 16) && g.K < ((int64_t)1 << 30) &&
         tiles >= sm_count() && tiles < ((int64_t)1 << 30);
}

int scaled_pair_launch(const SmArgs &p, int y_dtype, bool f8, cudaStream_t st) {
  SpArgs g{};
  g.p = p;
  g.mt = (int)((p.M + 2 * SP_BM - 1) / (2 * SP_BM));
  g.nt = (int)((p.N + SP_BN - 1) / SP_BN);
  CUtensorMap ma, mw;
  const uint64_t strides[1] = {(uint64_t)p.K};
  const uint64_t da[2] = {(uint64_t)p.K, (uint64_t)p.M}, dw[2] = {(uint64_t)p.K, (uint64_t)p.N};
  const uint32_t box[2] = {SP_BK, SP_BM};
  if (int rc = make_tensor_map(&ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, p.a, da, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  if (int rc = make_tensor_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, p.w, dw, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  if (y_dtype == kFloat16) return f8 ? launch<__half, Fp8>(ma, mw, g, st) : launch<__half, Int8>(ma, mw, g, st);
  if (y_dtype == kBfloat16) return f8 ? launch<__nv_bfloat16, Fp8>(ma, mw, g, st) : launch<__nv_bfloat16, Int8>(ma, mw, g, st);
  return f8 ? launch<float, Fp8>(ma, mw, g, st) : launch<float, Int8>(ma, mw, g, st);
}

int status_read_scaled_pair(int reset) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_scaled_pair_status, sizeof(int)) != cudaSuccess) return -1;
  if (reset && v) {
    const int z = 0;
    if (cudaMemcpyToSymbol(g_scaled_pair_status, &z, sizeof(int)) != cudaSuccess) return -1;
  }
  return v;
}

} // namespace b2
