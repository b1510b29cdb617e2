// Attention of prompts over a paged 8-bit KV cache (b2_cache_attention) on tcgen05 tensor cores:
// FLOAT16 / BFLOAT16 queries, head sizes that are multiples of 16 up to 128, pages of whole 16s.
//
// Bound: the softmax warps (exponentials, conversions), then the tensor pipe.  2048 positions after 6144,
// 32 / 8 heads of 128: 343 us, 702 TFLOP/s, tensor pipe 37 % active.
//
// One CTA owns 128 query rows -- pk heads of one GQA group (a power of two that divides it, up to 8 or
// as few positions leave room for) x 128 / pk positions -- and walks the 128-key tiles that any of them sees (the
// sinks' tiles, then the window's up to the diagonal):
//   warp 9     (pages) looks up the tiles' pages and scales ahead of use and brings the codes by TMA,
//              one box per run of a page's tokens, K and V through two buffers each;
//   warps 10-15 (converters) widen the codes to FLOAT16 (exact for both code types) and write the
//              128-byte-swizzled K and V operands, two buffers each; rows without a token become zeros;
//   warp 8     (MMA) issues S = Q K^T into one of two TMEM buffers and O += P V with P read from TMEM;
//   warps 0-7  (softmax) two threads per query row, one per half of the columns.
// Scales never touch an element: within 16 keys of one page the key scale is part of the exponent's
// factor and log2 of the value scale part of its offset, p' = 2^(s k_scale + log2 v_scale - m), so O
// sums p' code and the denominator sums p' / v_scale, one multiplication per 16 keys.  m follows
// the row's largest exponent lazily: it is moved only when p' would pass 2^15, then to 2^7, and O
// and l are rescaled; p' in FLOAT16 keeps 11 bits down to 2^-21 of the row's largest and more.  In fp32
// p' ends at 2^-126, so a page whose value scale is 2^-110 of another's leaves keys of less than about
// 2^-23 of the row's largest weight out of the denominator.
// BFLOAT16 queries become FLOAT16 after a power of two per row (8 significant bits fit in 11; columns
// 2^-14 below the row's largest lose low bits).
//
// Every mbarrier is waited phase by phase by the threads that depend on it, and no barrier can run
// two phases ahead of a waiter.  All waits are bounded; after a time-out the CTA records a code,
// waits for its MMAs in flight, frees its TMEM and returns.
#include <algorithm>
#include <type_traits>

#include "attn_math.cuh"
#include "cache_attention.cuh"
#include "tc_common.cuh"

namespace b2 {

__device__ int g_cache_attn_prefill_status; // time-out code
__device__ int g_cache_attn_prefill_range;  // 1: a length, count or page number was out of range

namespace {

using namespace q8;

constexpr int CP_M = 128, CP_N = 128;             // query rows, keys per tile
constexpr int CP_SOFT = 8, CP_MMA = 8, CP_PAGES = 9, CP_CONV = 10, CP_NCONV = 6;
// Registers: 16 warps start with 128 each; the two softmax warpgroups take 160, the other two keep
// 96 (2 x 160 + 2 x 96 = 4 x 128).
constexpr int CP_REG_SOFT = 160, CP_REG_REST = 96;
constexpr int CP_THREADS = (CP_CONV + CP_NCONV) * 32;
constexpr uint32_t CP_HALF = 128 * 128;           // [128 rows][64 FLOAT16]: 16 KB
constexpr uint32_t CP_RAW = 128 * 128;            // a tile's codes, 128 bytes a key
constexpr uint32_t CP_TMEM_COLS = 512, CP_COL_O = 256;
constexpr float CP_TOP = 15.0f, CP_BASE = 7.0f;   // log2 of the largest p', and after a move of m
constexpr float CP_LV_MIN = -60.0f;

template <int DP> struct CpLayout {
  static constexpr int NH = DP / 64;              // 64-column halves
  static constexpr uint32_t TILE = NH * CP_HALF;  // a K or V operand
  static constexpr uint32_t OFF_Q = 0;
  static constexpr uint32_t OFF_K = TILE, OFF_V = 3 * TILE; // two buffers each
  static constexpr uint32_t OFF_RAW = 5 * TILE;             // codes [128][128 B]: K, K, V, V
  static constexpr uint32_t OFF_RED = OFF_RAW + 4 * CP_RAW;  // float [2][2][128]
  static constexpr uint32_t OFF_SC = OFF_RED + 2 * 2 * CP_M * 4; // float4 [4 tiles][8 runs of 16 keys]
  static constexpr uint32_t OFF_FAC = OFF_SC + 4 * 8 * 16;       // float [4][8], then int [4]
  static constexpr uint32_t OFF_BAR = OFF_FAC + 4 * 8 * 4 + 16;
  static constexpr int NBAR = 24;
  static constexpr size_t SMEM = OFF_BAR + NBAR * 8 + 16;
};

struct CpArgs {
  CaArgs c;
  int qtiles, pk, np, hpacks;
  int splits;         // CTAs that share a query tile's keys, at most
  float *partials;    // [query tile][splits][128][DP + 4]: O, m, l
  float scale_log2;
  FastDiv div_t; // by the page size
  int chunk;     // keys per TMA box: a power of two, 16 to 128, that divides the page
};

// Four codes -> two FLOAT16 pairs, exactly.
template <typename Q> __device__ __forceinline__ void widen4(uint32_t w, uint32_t &lo, uint32_t &hi) {
  if constexpr (std::is_same<Q, Fp8>::value) {
    asm("{\n\t.reg .b16 a, b;\n\t"
        "mov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    const uint32_t u = w ^ 0x80808080u; // 1024 + (code + 128), minus 1152
    const __half2 k = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&a), k);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2 *>(&b), k);
    lo = *reinterpret_cast<const uint32_t *>(&x);
    hi = *reinterpret_cast<const uint32_t *>(&y);
  }
}

__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// What a query tile's CTAs have to do.
struct CpTile {
  int b, h0, q0;                 // sequence, first query head, first query
  CaSpan sp;
  int first, sink_tiles, tiles;  // key tiles: the window's first, the sinks' before it, all
  int parts;                     // CTAs that share them
};
__device__ __forceinline__ CpTile cp_tile(const CpArgs &g, int qtile, bool *bad) {
  const CaArgs &a = g.c;
  CpTile t{};
  const int bhp = qtile / g.qtiles;
  t.b = bhp / g.hpacks;
  t.h0 = (bhp % g.hpacks) * g.pk;
  t.q0 = (g.qtiles - 1 - qtile % g.qtiles) * g.np; // long rows first
  t.sp = ca_span(a, t.b, bad);
  if (t.q0 >= t.sp.count) return t; // no query of this tile counts
  const int p_first = t.sp.past + t.q0, p_last = t.sp.past + min(t.q0 + g.np, t.sp.count) - 1;
  const int kend = a.causal ? min(t.sp.total, p_last + 1) : t.sp.total;
  const bool win = a.causal && a.window >= 0;
  t.first = win ? max(0, p_first - a.window) / CP_N : 0;
  t.sink_tiles = win ? min((min(a.sinks, kend) + CP_N - 1) / CP_N, t.first) : 0;
  t.tiles = t.sink_tiles + (kend + CP_N - 1) / CP_N - t.first;
  t.parts = min(g.splits, t.tiles);
  return t;
}

template <typename T, typename Q, int DP>
__global__ void __launch_bounds__(CP_THREADS, 1)
    cache_attn_prefill(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                       const CpArgs g) {
  using L = CpLayout<DP>;
  extern __shared__ __align__(1024) uint8_t sm[];
  if (tc::smem_u32(sm) & 1023u) { // the operands need a 1024-byte aligned base
    if (threadIdx.x == 0) atomicExch(&g_cache_attn_prefill_status, tc::kTimeoutFull);
    return;
  }
  const CaArgs &a = g.c;
  uint64_t *bars = reinterpret_cast<uint64_t *>(sm + L::OFF_BAR);
  float *red = reinterpret_cast<float *>(sm + L::OFF_RED);
  float4 *sc = reinterpret_cast<float4 *>(sm + L::OFF_SC);
  float *fac = reinterpret_cast<float *>(sm + L::OFF_FAC);           // of value scales below 2^-60
  volatile int *look = reinterpret_cast<volatile int *>(sm + L::OFF_FAC + 4 * 8 * 4); // [4] per tile: what converters check
  uint64_t *q_full = bars;       // 1
  uint64_t *k_full = bars + 1;   // 2
  uint64_t *k_empty = bars + 3;  // 2: S of the buffer's tile done
  uint64_t *v_full = bars + 5;   // 2
  uint64_t *v_empty = bars + 7;  // 2: P.V of the buffer's tile done
  uint64_t *s_full = bars + 9;   // 2
  uint64_t *p_full = bars + 11;  // 2
  uint64_t *o_done = bars + 13;  // 2
  uint64_t *mma_done = bars + 15;
  uint64_t *raw_full = bars + 16;  // 4: the codes of K (0, 1) and V (2, 3) landed
  uint64_t *raw_empty = bars + 20; // 4: converted
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + L::NBAR);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = (int)(blockIdx.x % g.splits), qtile = (int)(blockIdx.x / g.splits);
  bool bad;
  const CpTile tile = cp_tile(g, qtile, &bad);
  const int b = tile.b, h0 = tile.h0, kvh = h0 / a.group, q0 = tile.q0;
  const CaSpan sp = tile.sp;
  if (bad && threadIdx.x == 0) atomicExch(&g_cache_attn_prefill_range, 1);
  T *yb = static_cast<T *>(a.y) + (int64_t)b * a.q_b;
  if (q0 >= sp.count) { // no query of this tile counts
    if (part) return;
    const int cols = a.D / 8;
    for (int e = threadIdx.x; e < CP_M * cols; e += CP_THREADS) {
      const int row = e / cols, i = q0 + row % g.np;
      if (i < a.S)
        *reinterpret_cast<uint4 *>(yb + (int64_t)(h0 + row / g.np) * a.q_h + (int64_t)i * a.q_s + e % cols * 8) =
            make_uint4(0u, 0u, 0u, 0u);
    }
    return;
  }
  // positions of the first and last query that counts; this CTA's share of the key tiles
  const int p_first = sp.past + q0, p_last = sp.past + min(q0 + g.np, sp.count) - 1;
  const bool win = a.causal && a.window >= 0;
  const int first = tile.first, sink_tiles = tile.sink_tiles, parts = tile.parts;
  if (part >= parts) return;
  const int t0 = (int)((int64_t)part * tile.tiles / parts);
  const int ntiles = (int)((int64_t)(part + 1) * tile.tiles / parts) - t0;
  auto key0_of = [&](int j) { return (t0 + j < sink_tiles ? t0 + j : first + t0 + j - sink_tiles) * CP_N; };

  if (threadIdx.x == 0) {
    tc::mbar_init(q_full, CP_SOFT);
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&k_full[i], CP_NCONV);
      tc::mbar_init(&k_empty[i], 1);
      tc::mbar_init(&v_full[i], CP_NCONV);
      tc::mbar_init(&v_empty[i], 1);
      tc::mbar_init(&s_full[i], 1);
      tc::mbar_init(&p_full[i], CP_SOFT);
      tc::mbar_init(&o_done[i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      tc::mbar_init(&raw_full[i], 1);
      tc::mbar_init(&raw_empty[i], CP_NCONV);
    }
    tc::mbar_init(mma_done, 1);
    *abort_flag = 0;
    tc::fence_barrier_init();
  }
  if (warp == CP_MMA) {
    tc::tmem_alloc(tmem_slot, CP_TMEM_COLS);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= CP_SOFT) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(CP_REG_REST));
    if (warp >= CP_CONV) {
      // ------------------------------ converters --------------------------------
      // 16-code units: lanes cover DP / 16 units of 512 / DP keys; a warp takes every sixth group.
      // Eight neighbouring lanes have four units of two rows, so no bank is hit twice.
      const int cw = warp - CP_CONV;
      constexpr int UPR = DP / 16, KPW = 32 / UPR, GROUPS = CP_N / KPW, MINE = (GROUPS + CP_NCONV - 1) / CP_NCONV;
      const int u = DP == 64 ? lane & 3 : (lane & 3) | (lane >> 1 & 4);
      const int sub = DP == 64 ? lane >> 2 : (lane >> 2 & 1) | (lane >> 4) * 2;
      auto widen = [&](uint32_t raw, uint32_t base, int j, bool values) {
        const int check = look[j & 3];
        uint4 r[MINE];
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
          const int row = (cw + i * CP_NCONV) * KPW + sub;
          if (row < CP_N) r[i] = *reinterpret_cast<const uint4 *>(sm + raw + row * 128 + ((u ^ (row & 7)) << 4));
        }
        if (check) { // zero codes widen to zeros
#pragma unroll
          for (int i = 0; i < MINE; ++i) {
            const int row = (cw + i * CP_NCONV) * KPW + sub;
            if (row < CP_N && (key0_of(j) + row >= sp.total || sc[(j & 3) * 8 + row / 16].w == 0.0f))
              r[i] = make_uint4(0u, 0u, 0u, 0u);
          }
        }
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
          const int row = (cw + i * CP_NCONV) * KPW + sub;
          if (row < CP_N) {
            const uint32_t w[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
            uint32_t h[8];
#pragma unroll
            for (int q = 0; q < 4; ++q) widen4<Q>(w[q], h[2 * q], h[2 * q + 1]);
            if (values && (check & 2)) {
              // value scales below 2^-60: what 2^-60 does not hold goes into the codes
              const float f = fac[(j & 3) * 8 + row / 16];
#pragma unroll
              for (int q = 0; q < 8; ++q) {
                const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&h[q]));
                h[q] = half2_of(v.x * f, v.y * f);
              }
            }
            uint8_t *p = sm + base + (u >> 2) * CP_HALF + row * 128;
            const int c = (u & 3) * 2;
            *reinterpret_cast<uint4 *>(p + ((c ^ (row & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
            *reinterpret_cast<uint4 *>(p + (((c + 1) ^ (row & 7)) << 4)) = make_uint4(h[4], h[5], h[6], h[7]);
          }
        }
        tc::fence_proxy_async();
        __syncwarp();
      };
      bool ok = true;
      for (int j = 0; ok && j < ntiles; ++j) {
        const int s = j & 1;
        const uint32_t ph = (j >> 1) & 1;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          uint64_t *empty = v ? v_empty : k_empty;
          ok = ok && !*abort_flag && tc::mbar_wait(&raw_full[2 * v + s], ph) &&
               (j < 2 || tc::mbar_wait(&empty[s], ph ^ 1));
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          widen(L::OFF_RAW + (2 * v + s) * CP_RAW, (v ? L::OFF_V : L::OFF_K) + s * L::TILE, j, v == 1);
          if (lane == 0) {
            tc::mbar_arrive(&raw_empty[2 * v + s]);
            tc::mbar_arrive(v ? &v_full[s] : &k_full[s]);
          }
        }
      }
      if (!ok && lane == 0) {
        atomicExch(&g_cache_attn_prefill_status, tc::kTimeoutEmpty);
        *abort_flag = 1;
      }
    } else if (warp == CP_PAGES) {
      // ------------------------------ pages --------------------------------------
      // Lane (my, ch) has box ch of tile my of each batch of `per` tiles; page numbers are read two
      // batches ahead and scales one.  A tile's scales go to sc, four tiles deep: both buffers of tile
      // j - 2 are converted before tile j is written, so P.V of tile j - 4 is done, and its softmax.
      const int nch = CP_N / g.chunk, per = 32 / nch, my = lane / nch, ch = lane % nch;
      const uint32_t box_bytes = (uint32_t)g.chunk * 128;
      if (lane == 0) {
        tc::prefetch_tensormap(&map_k);
        tc::prefetch_tensormap(&map_v);
      }
      struct Box {
        int id, row; // page as the table has it, first row in it
        bool live;   // the sequence has tokens there
      };
      auto find = [&](int j) {
        Box x{0, 0, false};
        if (j < ntiles) {
          const int key = key0_of(j) + ch * g.chunk;
          if (key < sp.total) {
            const int page = (int)g.div_t.div(key);
            x.id = a.table[(int64_t)b * a.max_pages + page];
            x.row = key - page * a.T;
            x.live = true;
          }
        }
        return x;
      };
      // the page's place among pages and heads, -1 when there is none; reports pages out of range
      auto place = [&](const Box &x) {
        if (!x.live) return -1;
        if (x.id >= 0 && x.id < a.pages) return x.id * a.Hkv + kvh;
        atomicExch(&g_cache_attn_prefill_range, 1);
        return -1;
      };
      auto scales = [&](int z) { return z >= 0 ? make_float2(a.ks[z], a.vs[z]) : make_float2(0.0f, 0.0f); };
      bool ok = true;
      int issued = 0;
      Box x0 = find(my), x1 = find(per + my);
      int z0 = place(x0);
      float2 s0 = scales(z0);
      for (int j0 = 0; ok && j0 < ntiles; j0 += per) {
        const int z1 = place(x1);
        const float2 s1 = scales(z1);
        const Box x2 = find(j0 + 2 * per + my);
        float4 f = make_float4(0.0f, CP_LV_MIN, 0.0f, 0.0f);
        if (z0 >= 0) {
          f.x = s0.x * g.scale_log2;
          f.y = fmaxf(log2f(s0.y), CP_LV_MIN); // a NaN gives the bound
          f.z = exp2f(-f.y);
          // 1: scales of ordinary values; 2: the softmax looks at each score
          f.w = f.x > 0.0f && f.x < INFINITY && fabsf(s0.y) < INFINITY ? 1.0f : 2.0f;
          if (!(fabsf(s0.y) < INFINITY)) f.z = __uint_as_float(0x7fc00000u);
        }
        const bool tiny = z0 >= 0 && f.y <= CP_LV_MIN;
        const bool holes = z0 < 0 || key0_of(min(j0 + my, ntiles - 1)) + (ch + 1) * g.chunk > sp.total;
        const uint32_t tinies = __ballot_sync(0xffffffffu, tiny), holed = __ballot_sync(0xffffffffu, holes);
        const uint32_t have = __ballot_sync(0xffffffffu, z0 >= 0);
        for (int k = 0; ok && k < per && j0 + k < ntiles; ++k) {
          const int j = j0 + k, s = j & 1;
          if (j >= 2) {
            ok = tc::mbar_wait(&raw_empty[s], ((j >> 1) - 1) & 1) && tc::mbar_wait(&raw_empty[2 + s], ((j >> 1) - 1) & 1);
          }
          ok = __all_sync(0xffffffffu, ok && !*abort_flag);
          if (!ok) break;
          const uint32_t bits = (nch == 32 ? 0xffffffffu : (1u << nch) - 1u) << (k * nch);
          const uint32_t bytes = (uint32_t)__popc(have & bits) * box_bytes;
          if (my == k) {
            for (int e = 0; e < g.chunk / 16; ++e) {
              sc[(j & 3) * 8 + ch * (g.chunk / 16) + e] = f;
              fac[(j & 3) * 8 + ch * (g.chunk / 16) + e] = tiny && fabsf(s0.y) < INFINITY ? s0.y * exp2f(-CP_LV_MIN) : tiny ? 0.0f : 1.0f;
            }
          }
          if (lane == 0) look[j & 3] = ((holed & bits) ? 1 : 0) | ((tinies & bits) ? 2 : 0);
          __syncwarp();
          if (lane == 0) {
            tc::mbar_expect_tx(&raw_full[s], bytes);
            tc::mbar_expect_tx(&raw_full[2 + s], bytes);
          }
          __syncwarp();
          if (my == k && z0 >= 0) {
            tc::tma_load_3d(sm + L::OFF_RAW + s * CP_RAW + ch * box_bytes, &map_k, &raw_full[s], 0, x0.row, z0);
            tc::tma_load_3d(sm + L::OFF_RAW + (2 + s) * CP_RAW + ch * box_bytes, &map_v, &raw_full[2 + s], 0, x0.row, z0);
          }
          issued = j + 1;
        }
        x0 = x1;
        z0 = z1;
        x1 = x2;
        s0 = s1;
      }
      if (!ok && lane == 0) {
        atomicExch(&g_cache_attn_prefill_status, tc::kTimeoutEmpty);
        *abort_flag = 1;
      }
      // no copy may land once the CTA has left: wait (bounded) for the last fills of both buffers
      for (int j = max(0, issued - 2); j < issued; ++j) {
        tc::mbar_wait(&raw_full[j & 1], (j >> 1) & 1);
        tc::mbar_wait(&raw_full[2 + (j & 1)], (j >> 1) & 1);
      }
    } else {
      // ------------------------------ MMA issuer --------------------------------
      if (tc::elect_one()) {
        const uint32_t id_s = tc::idesc(1, 0, 0, 0, 0, CP_M, CP_N);
        const uint32_t id_o = tc::idesc(1, 0, 0, 0, 1, CP_M, DP);
        const uint32_t q_base = tc::smem_u32(sm + L::OFF_Q);
        bool ok = tc::mbar_wait(q_full, 0);
        auto issue_pv = [&](int j) { // O (+)= P_j V_j, V read MN-major over the head's columns
          if (!tc::mbar_wait(&p_full[j & 1], (j >> 1) & 1)) return false;
          if (!tc::mbar_wait(&v_full[j & 1], (j >> 1) & 1)) return false;
          tc::tc_fence_after();
          const uint32_t p_col = tmem + (uint32_t)(j & 1) * CP_N;
          const uint32_t v_base = tc::smem_u32(sm + L::OFF_V + (j & 1) * L::TILE);
  #pragma unroll
          for (int kk = 0; kk < CP_N / 16; ++kk) {
            const uint64_t bd = tc::sdesc_sw128(v_base + kk * 16 * 128, CP_HALF, 1024);
            tc::mma_f16_ts(tmem + CP_COL_O, p_col + kk * 8, bd, id_o, (j > 0 || kk > 0) ? 1u : 0u);
          }
          tc::tc_commit(&o_done[j & 1]);
          tc::tc_commit(&v_empty[j & 1]);
          return true;
        };
        for (int j = 0; ok && j < ntiles; ++j) {
          if (*abort_flag || !tc::mbar_wait(&k_full[j & 1], (j >> 1) & 1)) {
            ok = false;
            break;
          }
          // S buffer j & 1 holds P_{j-2} until P.V of tile j - 2 is done
          if (j >= 2 && !tc::mbar_wait(&o_done[j & 1], ((j - 2) >> 1) & 1)) {
            ok = false;
            break;
          }
          tc::tc_fence_after();
          const uint32_t k_base = tc::smem_u32(sm + L::OFF_K + (j & 1) * L::TILE);
  #pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk) {
            const uint64_t ad = tc::sdesc_sw128(q_base + (kk >> 2) * CP_HALF + (kk & 3) * 32, 16, 1024);
            const uint64_t bd = tc::sdesc_sw128(k_base + (kk >> 2) * CP_HALF + (kk & 3) * 32, 16, 1024);
            tc::mma_f16(tmem + (j & 1) * CP_N, ad, bd, id_s, kk > 0 ? 1u : 0u);
          }
          tc::tc_commit(&s_full[j & 1]);
          tc::tc_commit(&k_empty[j & 1]);
          if (j >= 1 && !issue_pv(j - 1)) ok = false;
        }
        if (ok && !issue_pv(ntiles - 1)) ok = false;
        if (!ok) {
          atomicExch(&g_cache_attn_prefill_status, tc::kTimeoutFull);
          *abort_flag = 1;
        }
        // TMEM is freed below: wait (bounded) until every issued MMA is done
        tc::tc_commit(mma_done);
        tc::mbar_wait(mma_done, 0);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(CP_REG_SOFT));
    // ------------------------------ softmax warps -----------------------------
    // Warps w and w + 4 share TMEM lanes 32 (w % 4) .. + 31; each thread has one half of its row's
    // columns.  Control flow stays warp-uniform around the TMEM accesses, and every softmax warp
    // takes every named barrier even after a time-out, so none can hang.
    const int quarter = warp & 3, half = warp >> 2;
    const int row = quarter * 32 + lane;           // query row = TMEM lane
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const int qi = q0 + row % g.np, pos = sp.past + qi; // position of the row's query
    const bool counts = qi < sp.count;
    // keys the row sees: first_key .. last_key, and the sinks
    const int last_key = a.causal ? min(pos, sp.total - 1) : sp.total - 1;
    const int first_key = win ? pos - a.window : 0;
    auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }; // bits < n
    auto softmax_sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(CP_SOFT * 32) : "memory"); };
    float qf = 1.0f; // power of two taken out of the row's queries
    {
      // this thread's 64 columns of Q -> FLOAT16 in the swizzled operand
      uint32_t w[32];
      const T *qp = static_cast<const T *>(a.q) + (int64_t)b * a.q_b + (int64_t)(h0 + row / g.np) * a.q_h +
                    (int64_t)qi * a.q_s;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const int d = half * 64 + c * 8;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (counts && d < a.D) v = __ldg(reinterpret_cast<const uint4 *>(qp + d));
        w[4 * c] = v.x;
        w[4 * c + 1] = v.y;
        w[4 * c + 2] = v.z;
        w[4 * c + 3] = v.w;
      }
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        uint32_t e = 0u;
#pragma unroll
        for (int c = 0; c < 32; ++c) e = max(e, max(w[c] & 0x7f80u, (w[c] >> 16) & 0x7f80u));
        uint32_t *re = reinterpret_cast<uint32_t *>(red);
        re[half * CP_M + row] = e;
        softmax_sync();
        e = max(e, re[(half ^ 1) * CP_M + row]);
        softmax_sync(); // red is free again
        const int ex = min(max((int)(e >> 7) - 127, -126), 126);
        const float down = __uint_as_float((uint32_t)(127 - ex) << 23);
        qf = __uint_as_float((uint32_t)(127 + ex) << 23);
#pragma unroll
        for (int c = 0; c < 32; ++c)
          w[c] = half2_of(__uint_as_float(w[c] << 16) * down, __uint_as_float(w[c] & 0xffff0000u) * down);
      }
      if (half < L::NH) {
        uint8_t *p = sm + L::OFF_Q + half * CP_HALF + row * 128;
#pragma unroll
        for (int c = 0; c < 8; ++c)
          *reinterpret_cast<uint4 *>(p + ((c ^ (row & 7)) << 4)) = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
      }
      tc::fence_proxy_async();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(q_full);
    }
    float m_ref = -INFINITY, l_part = 0.0f;
    bool ok = true;
    auto uniform_wait = [&](uint64_t *bar, uint32_t parity) {
      const bool w = ok && !*abort_flag && tc::mbar_wait(bar, parity);
      return __all_sync(0xffffffffu, w);
    };
    constexpr int OC = DP / 2; // O columns per thread
    for (int j = 0; j < ntiles; ++j) {
      if (!uniform_wait(&s_full[j & 1], (j >> 1) & 1)) ok = false;
      tc::tc_fence_after();
      const int key0 = key0_of(j) + half * 64;
      const uint32_t s_col = tmem + lane_off + (j & 1) * CP_N + half * 64;
      // the scores of this half row stay in registers; vk, lv: factor and offset of each 16 keys' exponents
      float v[64], vk[4], lv[4], inv[4];
      float mx = -INFINITY;
      bool poison = false;
      if (ok) {
        bool plain = g.scale_log2 > 0.0f && a.softcap <= 0.0f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float4 f = sc[(j & 3) * 8 + half * 4 + c];
          vk[c] = f.x * qf;
          lv[c] = f.y;
          inv[c] = f.z;
          plain = plain && f.w == 1.0f;
        }
        const bool need_mask = key0 + 64 > sp.total || (a.causal && key0 + 63 > p_first) ||
                               (win && key0 < p_last - a.window && key0 + 64 > a.sinks);
        uint32_t r0[32], r1[32];
        tc::tmem_ld32(s_col, r0);
        tc::tmem_ld32(s_col + 32, r1);
        tc::tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          v[e] = __uint_as_float(r0[e]);
          v[32 + e] = __uint_as_float(r1[e]);
        }
        if (!__all_sync(0xffffffffu, plain && !need_mask)) {
          // every score in base-2 units, -inf where the row does not see the key: one bit per key;
          // pages out of range (flag 0) hold no keys
          uint32_t bits[2];
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const int base = key0 + w * 32;
            bits[w] = below(last_key + 1 - base) & (~below(first_key - base) | below(a.sinks - base));
          }
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 16; ++e) v[c * 16 + e] *= vk[c];
          if (a.softcap > 0.0f) { // on its own: its code would be fetched past by every masked tile
#pragma unroll
            for (int e = 0; e < 64; ++e) v[e] = a.softcap * tanhf(v[e] * kLn2 / a.softcap) * kLog2E;
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t flag = __float_as_uint(sc[(j & 3) * 8 + half * 4 + c].w);
            const uint32_t seen = flag ? (bits[c >> 1] >> ((c & 1) * 16)) & 0xffffu : 0u;
#pragma unroll
            for (int e = 0; e < 16; ++e) v[c * 16 + e] = seen >> e & 1u ? v[c * 16 + e] : -INFINITY;
            poison = poison || (seen != 0u && inv[c] != inv[c]); // it sees values that are not finite
            // its infinite offset must not meet the -inf of the rows that do not see them
            if (inv[c] != inv[c]) inv[c] = lv[c] = 0.0f;
            vk[c] = 1.0f;
          }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float m = -INFINITY;
#pragma unroll
          for (int e = 0; e < 16; e += 2) m = max3f(m, v[c * 16 + e], v[c * 16 + e + 1]);
          mx = fmaxf(mx, fmaf(m, vk[c], lv[c])); // vk > 0
        }
      }
      float *rm = red + (j & 1) * 2 * CP_M;
      rm[half * CP_M + row] = mx;
      softmax_sync();
      mx = fmaxf(mx, rm[(half ^ 1) * CP_M + row]);
      if (!ok) continue;
      const bool reb = mx > m_ref + CP_TOP;
      float corr = 1.0f;
      if (reb) {
        const float to = mx - CP_BASE;
        corr = exp2f(m_ref - to);
        l_part *= corr;
        m_ref = to;
      }
      if (j >= 1 && __any_sync(0xffffffffu, reb)) {
        if (!uniform_wait(&o_done[(j - 1) & 1], ((j - 1) >> 1) & 1)) {
          ok = false;
          continue;
        }
        tc::tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < OC / 32; ++c) {
          const uint32_t o_col = tmem + lane_off + CP_COL_O + half * OC + c * 32;
          uint32_t r[32];
          tc::tmem_ld32(o_col, r);
          tc::tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * corr);
          tc::tmem_st32(o_col, r);
        }
        tc::tmem_st_wait();
      }
      // P over the S buffer the scores came from (every thread of the row has read its S half
      // before the barrier above)
      const float ref = m_ref == -INFINITY ? 0.0f : m_ref;
      const uint32_t p_col = tmem + lane_off + (j & 1) * CP_N + half * 32;
#pragma unroll
      for (int c2 = 0; c2 < 2; ++c2) {
        uint32_t ph[16];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int c = c2 * 2 + h;
          const uint64_t k2 = f2pack(vk[c], vk[c]), o2 = f2pack(lv[c] - ref, lv[c] - ref);
          uint64_t ls = f2pack(0.0f, 0.0f);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 x = f2unpack(ffma2(f2pack(v[c * 16 + 2 * e], v[c * 16 + 2 * e + 1]), k2, o2));
            const float p0 = ex2(x.x), p1 = ex2(x.y);
            ls = fadd2(ls, f2pack(p0, p1));
            ph[h * 8 + e] = half2_of(p0, p1);
          }
          const float2 l2 = f2unpack(ls);
          l_part = fmaf(l2.x + l2.y, inv[c], l_part);
        }
        tc::tmem_st16(p_col + c2 * 16, ph);
      }
      if (poison) l_part = __uint_as_float(0x7fc00000u);
      tc::tmem_st_wait();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&p_full[j & 1]);
    }
    const int last = ntiles - 1;
    const bool fin = uniform_wait(&o_done[last & 1], (last >> 1) & 1);
    softmax_sync();
    red[half * CP_M + row] = l_part;
    softmax_sync();
    const float l_sum = l_part + red[(half ^ 1) * CP_M + row];
    if (fin) {
      tc::tc_fence_after();
      const float scale = l_sum == 0.0f ? 0.0f : 1.0f / l_sum; // a NaN stays
      T *yr = yb + (int64_t)(h0 + row / g.np) * a.q_h + (int64_t)qi * a.q_s;
      float *mine = g.partials + (((size_t)qtile * g.splits + part) * CP_M + row) * (DP + 4);
      if (parts > 1 && half == 0) *reinterpret_cast<float2 *>(mine + DP) = make_float2(m_ref, l_sum);
#pragma unroll 1
      for (int c = 0; c < OC / 32; ++c) {
        uint32_t r[32];
        tc::tmem_ld32(tmem + lane_off + CP_COL_O + half * OC + c * 32, r);
        tc::tmem_ld_wait();
        const int d0 = half * OC + c * 32;
        if (parts > 1) { // several CTAs share the tile: cache_attn_prefill_join adds their O, m, l
          if (counts) {
#pragma unroll
            for (int q = 0; q < 8; ++q)
              *reinterpret_cast<float4 *>(mine + d0 + q * 4) =
                  make_float4(__uint_as_float(r[q * 4]), __uint_as_float(r[q * 4 + 1]), __uint_as_float(r[q * 4 + 2]),
                              __uint_as_float(r[q * 4 + 3]));
          }
        } else if (qi < a.S) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = counts ? __uint_as_float(r[q * 8 + e]) * scale : 0.0f;
            if (d0 + q * 8 < a.D) Raw8<T>::store(yr + d0 + q * 8, f);
          }
        }
      }
    }
    if (!fin) {
      atomicExch(&g_cache_attn_prefill_status, tc::kTimeoutFull);
      *abort_flag = 1;
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == CP_MMA) tc::tmem_dealloc(tmem, CP_TMEM_COLS);
}

// Adds the parts of query tiles whose keys several CTAs shared, in order: one warp per query row, a
// lane for four columns at a time.  Bound by latency: 4 us and 0.02 per part.
template <typename T, int DP> __global__ void __launch_bounds__(256) cache_attn_prefill_join(const CpArgs g) {
  const int row = (int)(blockIdx.x % (CP_M / 8)) * 8 + (threadIdx.x >> 5), qtile = (int)(blockIdx.x / (CP_M / 8));
  const int d = (threadIdx.x & 31) * 4;
  bool bad;
  const CpTile t = cp_tile(g, qtile, &bad);
  const int qi = t.q0 + row % g.np;
  if (t.parts <= 1 || qi >= g.c.S || d >= g.c.D) return;
  T *y = static_cast<T *>(g.c.y) + (int64_t)t.b * g.c.q_b + (int64_t)(t.h0 + row / g.np) * g.c.q_h +
         (int64_t)qi * g.c.q_s + d;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (qi < t.sp.count) {
    constexpr int W = DP + 4;
    const float *p = g.partials + ((size_t)qtile * g.splits * CP_M + row) * W;
    float M = -INFINITY, l = 0.0f;
    for (int c = 0; c < t.parts; c += 8) {
      float2 ml[8];
      float4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        ml[k] = make_float2(-INFINITY, 0.0f);
        v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (c + k < t.parts) {
          const float *src = p + (size_t)(c + k) * CP_M * W;
          ml[k] = __ldcg(reinterpret_cast<const float2 *>(src + DP));
          v[k] = __ldcg(reinterpret_cast<const float4 *>(src + d));
        }
      }
      float mn = M;
#pragma unroll
      for (int k = 0; k < 8; ++k) mn = fmaxf(mn, ml[k].x);
      const float base = mn == -INFINITY ? 0.0f : mn, keep = exp2f(M - base);
      l *= keep;
      acc = make_float4(acc.x * keep, acc.y * keep, acc.z * keep, acc.w * keep);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float w = exp2f(ml[k].x - base);
        l = fmaf(ml[k].y, w, l);
        acc.x = fmaf(v[k].x, w, acc.x);
        acc.y = fmaf(v[k].y, w, acc.y);
        acc.z = fmaf(v[k].z, w, acc.z);
        acc.w = fmaf(v[k].w, w, acc.w);
      }
      M = mn;
    }
    const float scale = l == 0.0f ? 0.0f : 1.0f / l;
    acc = make_float4(acc.x * scale, acc.y * scale, acc.z * scale, acc.w * scale);
  }
  st1<T>(y, 0, acc.x);
  st1<T>(y, 1, acc.y);
  st1<T>(y, 2, acc.z);
  st1<T>(y, 3, acc.w);
}

// Heads per CTA: a power of two that divides the group, up to 8, and more where few positions would
// leave rows empty.
int cp_pk(const CaArgs &a) {
  int most = 8, pk = 1;
  while (most < CP_M && (int64_t)a.S * 2 * most <= CP_M) most *= 2;
  while (pk < most && a.group % (2 * pk) == 0) pk *= 2;
  return pk;
}

template <typename T, typename Q, int DP>
int cp_launch_dp(const CUtensorMap &mk, const CUtensorMap &mv, const CpArgs &g, int64_t tiles, cudaStream_t st) {
  auto kern = cache_attn_prefill<T, Q, DP>;
  B2_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)CpLayout<DP>::SMEM));
  kern<<<(unsigned)(tiles * g.splits), CP_THREADS, CpLayout<DP>::SMEM, st>>>(mk, mv, g);
  B2_LAUNCH_CHECK();
  if (g.splits > 1) {
    cache_attn_prefill_join<T, DP><<<(unsigned)(tiles * (CP_M / 8)), 256, 0, st>>>(g);
    B2_LAUNCH_CHECK();
  }
  return B2_OK;
}
template <typename T, typename Q>
int cp_launch(const CUtensorMap &mk, const CUtensorMap &mv, const CpArgs &g, int64_t tiles, cudaStream_t st) {
  return g.c.D <= 64 ? cp_launch_dp<T, Q, 64>(mk, mv, g, tiles, st) : cp_launch_dp<T, Q, 128>(mk, mv, g, tiles, st);
}

int cp_read(int reset, const int &symbol) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, symbol, sizeof(int)) != cudaSuccess) return -1;
  if (reset && v) {
    const int z = 0;
    if (cudaMemcpyToSymbol(symbol, &z, sizeof(int)) != cudaSuccess) return -1;
  }
  return v;
}

} // namespace

// Query tiles of a call.
static int64_t cp_tiles(const CaArgs &a) {
  const int pk = cp_pk(a), np = CP_M / pk;
  return (int64_t)((a.S + np - 1) / np) * a.B * (a.Hq / pk);
}

// CTAs that share a query tile's keys, from the longest the table (and the window) can hold: a key
// tile takes about 1.3 us, a CTA's start and end 6, the joining kernel 4 and 0.02 per part, and the
// busiest SM sets the time.  64 queries over 6208 keys (16 query tiles): 84 us with one, 31 with 9.
static int cp_splits(const CaArgs &a) {
  const int64_t tiles = cp_tiles(a), sms = sm_count();
  int64_t keys = (int64_t)a.max_pages * a.T;
  if (a.causal && a.window >= 0) keys = std::min<int64_t>(keys, (int64_t)a.window + a.sinks + 3 * CP_N);
  const double per = 1.3 * (double)((keys + CP_N - 1) / CP_N);
  int best = 1;
  double least = 0.0;
  for (int s = 1; s <= 32 && tiles * (s - 1) < 4 * sms; ++s) {
    const double cost = (double)((tiles * s + sms - 1) / sms) * (per / s + 6.0) + (s > 1 ? 4.0 + 0.02 * (double)(tiles * s) : 0.0);
    if (s == 1 || cost < least) {
      least = cost;
      best = s;
    }
  }
  return best;
}

bool cache_attn_prefill_eligible(const CaArgs &a) {
  return a.D % 16 == 0 && a.D <= 128 && a.T % 16 == 0 && aligned(a.q, 16) && aligned(a.y, 16) && aligned(a.k, 16) &&
         aligned(a.v, 16) && a.pages > 0 && a.q_h % 8 == 0 && a.q_s % 8 == 0 && cp_tiles(a) < ((int64_t)1 << 31);
}

size_t cache_attn_prefill_workspace(const CaArgs &a) {
  const int splits = cp_splits(a);
  return splits > 1 ? kCounterBytes + (size_t)cp_tiles(a) * splits * CP_M * ((a.D <= 64 ? 64 : 128) + 4) * 4 : 0;
}

int cache_attn_prefill_launch(const CaArgs &a, bool f16, bool f8, void *ws, cudaStream_t st) {
  CpArgs g{};
  g.c = a;
  g.pk = cp_pk(a);
  g.np = CP_M / g.pk;
  g.qtiles = (a.S + g.np - 1) / g.np;
  g.hpacks = a.Hq / g.pk;
  g.scale_log2 = a.scale * kLog2E;
  g.div_t = FastDiv((uint32_t)a.T);
  g.chunk = a.T % 128 == 0 ? 128 : a.T % 64 == 0 ? 64 : a.T % 32 == 0 ? 32 : 16;
  g.splits = cp_splits(a);
  g.partials = ws ? reinterpret_cast<float *>(static_cast<uint8_t *>(ws) + kCounterBytes) : nullptr;
  const int64_t tiles = cp_tiles(a);
  // [pages * Hkv][T][D] codes; columns past D read as zeros
  CUtensorMap mk, mv;
  const uint64_t dims[3] = {(uint64_t)a.D, (uint64_t)a.T, (uint64_t)a.pages * a.Hkv};
  const uint64_t strides[2] = {(uint64_t)a.D, (uint64_t)a.T * a.D};
  const uint32_t box[3] = {128, (uint32_t)g.chunk, 1};
  if (int rc = make_tensor_map(&mk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, a.k, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  if (int rc = make_tensor_map(&mv, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, a.v, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  if (f16) return f8 ? cp_launch<__half, Fp8>(mk, mv, g, tiles, st) : cp_launch<__half, Int8>(mk, mv, g, tiles, st);
  return f8 ? cp_launch<__nv_bfloat16, Fp8>(mk, mv, g, tiles, st) : cp_launch<__nv_bfloat16, Int8>(mk, mv, g, tiles, st);
}

int status_read_cache_attn_prefill(int reset) { return cp_read(reset, g_cache_attn_prefill_status); }
int range_read_cache_attn_prefill(int reset) { return cp_read(reset, g_cache_attn_prefill_range); }

} // namespace b2
