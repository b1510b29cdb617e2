// Attention over a paged 8-bit KV cache for few query rows: single tokens and short runs of them
// (b2_cache_attention), with the keys split over the whole GPU.
//
// Bound: HBM, the visible codes of K and V once; for one short sequence, latency.
//
// A KV head's queries -- the heads of its group times the new positions, a pack of 8 NT rows -- are
// the 8-wide N side of mma.sync m16n8k16 and the tokens (Q.K) or head columns (P.V) its 16-row M side,
// so a code read from HBM serves all of them and the padding is at most 7 columns of N (half of them for
// one position of a group of 4 heads):
//   S^T[16 tokens x 8 rows] += K[16 x 16 columns] Q^T     O^T[16 columns x 8 rows] += V^T[16 x 16 tokens] P^T
// Codes become FLOAT16 in registers, exactly (INT8 and FLOAT8E4M3FN values both fit), and the page
// scales multiply in fp32: the key scale the score, the value scale the probability.  Sums and the
// softmax state are fp32.  Three roundings to FLOAT16 remain: BFLOAT16 queries, after a power of two
// per row brings them to [-2, 2) (8 significant bits fit in 11; columns 2^-14 below the row's largest
// lose low bits); and p * v_scale, relative to the largest such product of the row, so 2^-11 of
// what it contributes.  The denominator sums the unrounded p.
//
// The running reference of a row is m ~ max_j (s_j + log2 v_scale_j): with p_j = 2^(s_j - m + 19) in
// fp32, p_j times 2^-12 v_scale_j is at most 2^15 for every token, however far the pages' scales lie
// apart, and keeps its 11 bits down to 2^-21 of the largest and below (FLOAT16's normal range ends at
// 2^-14).  log2 v_scale is held to [-60, 122]: below, p would overflow (a smaller scale only makes its
// products smaller); no scale of finite values is above 2^128 / 127.  The 2^12 keeps p, which the
// denominator sums, normal down to 2^-23 of the largest even there.
//
// Data path: tiles of 32 tokens (K and V, 128 bytes a token, 128-byte swizzle) through a TMA ring
// filled by two producer warps, one for the keys and scales and one for the values.  Page numbers and
// scales are fetched for the next 8 to 32 tiles at once, one page chunk a lane; the first tiles' copies start before their scales arrive.  Each
// tile is one consumer warp's: the swizzle makes the fragment reads (16 bytes a lane) free of
// bank conflicts, for K along a token's columns and for V across four tokens.
//
// Split: (sequence, KV head, pack, tile) units are numbered in order and the CTAs (one per SM) take
// equal ranges, worked out on the device from the lengths, so ragged batches balance and the host
// never waits.  A CTA merges its warps' (m, l, O) per pair; a pair that spans CTAs is merged
// by its last arriver in CTA order, so results do not depend on timing.
//
// Measured (32 / 8 heads of 128): 32 sequences of up to 8192 tokens (344 MB of codes)
// 75.7 us, 4.5 TB/s; 8 sequences with a window of 4096 28.7 us, 2.3 TB/s; one sequence of 4097 tokens
// 13.3 us.  The consumer warps' dependent chain per tile (widen, MMA, exponentials) bounds the first two,
// the walk's fixed start and merge the last.
#include <algorithm>

#include "attn_math.cuh"
#include "cache_attention.cuh"
#include "tc_common.cuh"

namespace b2 {

__device__ int g_cache_attn_split_status; // time-out code of a bounded wait
__device__ int g_cache_attn_split_range;  // 1: a length, count or page number was out of range

namespace {

using namespace q8;

constexpr int KEYS = 32; // tokens per tile
constexpr float CS_TOP = 15.0f, CS_BASE = 7.0f; // log2 of the largest product of p, and after a move of m
constexpr float CS_UP = 12.0f, CS_UP_F = 4096.0f; // power of two that p carries and its product does not
constexpr float CS_LV_MIN = -60.0f, CS_LV_MAX = 122.0f; // of log2 v_scale
constexpr size_t CS_SMEM_MAX = 232448;
constexpr int CS_CTAS = 160; // at most, one per SM

template <int DP, int NT> struct CsLayout {
  static constexpr uint32_t BOX = KEYS * 128;             // a 128-byte-wide tile of codes
  static constexpr int NB = DP == 256 ? 2 : 1;            // 128-byte boxes per row
  // Consumer warps: 10 and the two producers share the register file at 168 each, 6 at 255.
  static constexpr int WARPS = NT == 1 && DP <= 128 ? 10 : DP <= 128 || NT == 1 ? 6 : 4;
  static constexpr int THREADS = (WARPS + 2) * 32;
  static constexpr uint32_t STAGE = 2 * NB * BOX;      // K boxes, V boxes
  static constexpr int W = DP + 4;                        // a row's O, m, l (16-byte rows)
  static constexpr uint32_t MERGE = WARPS * 8 * NT * W * 4;
  static constexpr uint32_t FIXED = 1024 + MERGE + 4096;  // alignment, merge, barriers, scales
  // Each stage belongs to one consumer warp (see the parity note in the kernel).
  static constexpr int STAGES = (int)((CS_SMEM_MAX - FIXED) / STAGE) / WARPS * WARPS < 24
                                    ? (int)((CS_SMEM_MAX - FIXED) / STAGE) / WARPS * WARPS
                                    : 24;
  static constexpr uint32_t OFF_MERGE = STAGES * STAGE;
  static constexpr uint32_t OFF_BAR = OFF_MERGE + MERGE;  // full, empty
  static constexpr uint32_t OFF_SC = OFF_BAR + 24 * 16;   // float4 [STAGES][KEYS / 8]
  static constexpr uint32_t OFF_MISC = OFF_SC + STAGES * KEYS * 2;
  static constexpr size_t SMEM = OFF_MISC + 256 + 1024;
  static_assert(STAGES >= WARPS && STAGES >= 4 && SMEM <= CS_SMEM_MAX, "shared memory");
};

struct CsArgs {
  CaArgs c;
  int packs, rows;  // packs of 8 NT rows of a KV head's `rows` = S * group
  int chunk, shift; // tokens per TMA box: a power of two (2^shift), 8 to KEYS, that divides the page
  int align_pairs;  // CTA ranges start at pair boundaries (more pairs than counters)
  float *partials;  // [grid][2][8 NT][DP + 4]: O, m, l
  uint32_t *counters;
};

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, "
               "{%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transposes an 8 x 8 matrix of 16-bit elements held one row of pairs a lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// Codes in a word -> exact FLOAT16 pairs: bytes 0 and 1 to lo, 2 and 3 to hi.
template <typename Q> __device__ __forceinline__ void to_half(uint32_t w, uint32_t &lo, uint32_t &hi) {
  if constexpr (std::is_same<Q, Fp8>::value) {
    asm("{\n\t.reg .b16 a, b;\n\t"
        "mov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    // code + 128 as the low byte of 1024 + (code + 128), an exact FLOAT16, minus 1152
    const uint32_t u = w ^ 0x80808080u;
    const __half2 k = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&a), k);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2 *>(&b), k);
    lo = *reinterpret_cast<const uint32_t *>(&x);
    hi = *reinterpret_cast<const uint32_t *>(&y);
  }
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
// The tiles of sequence b: the window's (from the first query's) and the sinks' before it.
struct CsSeq {
  CaSpan sp;
  int first, sink_tiles, tiles; // first window tile; tiles before it; all tiles (at least 1)
};
__device__ __forceinline__ CsSeq cs_seq(const CaArgs &a, int b, bool *bad) {
  CsSeq s;
  s.sp = ca_span(a, b, bad);
  const bool win = a.causal && a.window >= 0;
  s.first = win ? max(0, s.sp.past - a.window) / KEYS : 0;
  s.sink_tiles = win ? min((min(a.sinks, s.sp.total) + KEYS - 1) / KEYS, s.first) : 0;
  s.tiles = s.sp.count > 0 ? s.sink_tiles + (s.sp.total + KEYS - 1) / KEYS - s.first : 0;
  s.tiles = max(s.tiles, 1); // a sequence without new tokens still gets its zeros written
  return s;
}
__device__ __forceinline__ int cs_key0(const CsSeq &s, int tile) {
  return (tile < s.sink_tiles ? tile : s.first + tile - s.sink_tiles) * KEYS;
}

// A walk over the units in order.
struct CsWalk {
  int b, before; // sequence, tiles (per pair) of the sequences before it
  CsSeq s;
  int pair, tile; // of the unit: KV head * packs + pack, tile
};
__device__ __forceinline__ void cs_seek(const CsArgs &g, CsWalk &w, int u) {
  const int hp = g.c.Hkv * g.packs;
  bool bad;
  while (u >= (w.before + w.s.tiles) * hp) { // all units together stay below 2^30
    w.before += w.s.tiles;
    w.s = cs_seq(g.c, ++w.b, &bad);
  }
  const int r = u - w.before * hp;
  w.pair = r / w.s.tiles;
  w.tile = r - w.pair * w.s.tiles;
}
// Positions of the pack's first and last query (last < first: none counts).
__device__ __forceinline__ void cs_pack(const CsArgs &g, const CsSeq &s, int pack, int rows_per_pack,
                                        int *first, int *last) {
  const int r0 = pack * rows_per_pack, r1 = min(g.rows, r0 + rows_per_pack) - 1;
  *first = s.sp.past + r0 / g.c.group;
  *last = s.sp.past + min(r1 / g.c.group, s.sp.count - 1);
}
// Whether any query of the pack may see a key of the tile.
__device__ __forceinline__ bool cs_live(const CsArgs &g, const CsSeq &s, int first, int last, int key0) {
  if (last < first || key0 >= s.sp.total) return false;
  if (!g.c.causal) return true;
  if (key0 > last) return false;
  return g.c.window < 0 || key0 + KEYS > first - g.c.window || key0 < g.c.sinks;
}

// Sum of v over the lanes before this one, and over the warp.
__device__ __forceinline__ int warp_scan(int v, int *total) {
  const int lane = threadIdx.x & 31;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += t;
  }
  *total = __shfl_sync(0xffffffffu, inc, 31);
  return inc - v;
}
// Sum of v over the block and the sum over the threads before this one; every thread calls it.
template <int THREADS> __device__ __forceinline__ int block_scan(int v, int *total, int *red) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += t;
  }
  __syncthreads(); // red is free
  if (lane == 31) red[warp] = inc;
  __syncthreads();
  int base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    const int t = red[w];
    if (w < warp) base += t;
    all += t;
  }
  *total = all;
  return base + inc - v;
}

__device__ __forceinline__ uint32_t arrive_acq_rel(uint32_t *p, uint32_t v) {
  uint32_t old;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], %2;" : "=r"(old) : "l"(p), "r"(v) : "memory");
  return old;
}

template <typename T, typename Q, int DP, int NT>
__global__ void __launch_bounds__(CsLayout<DP, NT>::THREADS, 1)
    cache_attn_split(const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v, const CsArgs g) {
  using L = CsLayout<DP, NT>;
  constexpr uint32_t BOX = L::BOX;
  constexpr int CHUNKS = KEYS / 8; // at most, per tile
  constexpr int MT = KEYS / 16;    // 16-token tiles
  constexpr int STAGES = L::STAGES, WARPS = L::WARPS, NB = L::NB, RP = 8 * NT;
  constexpr int KS = DP / 16;                 // k16 steps of Q.K; M tiles of P.V
  extern __shared__ uint8_t dsm[];
  uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(dsm) + 1023) & ~uintptr_t(1023));
  uint64_t *full = reinterpret_cast<uint64_t *>(sm + L::OFF_BAR);
  uint64_t *empty = full + STAGES;
  float4 *sc = reinterpret_cast<float4 *>(sm + L::OFF_SC);
  float *mrg = reinterpret_cast<float *>(sm + L::OFF_MERGE);
  int *misc = reinterpret_cast<int *>(sm + L::OFF_MISC); // [0..15] scan, [16] b, [17] before
  volatile int *flags = misc + 24;                       // [0] abort [1] last
  const CaArgs &a = g.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hp = a.Hkv * g.packs; // pairs per sequence

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      tc::mbar_init(&full[i], 2);  // both producers
      tc::mbar_init(&empty[i], 1); // one consumer warp per stage
    }
    flags[0] = 0;
    flags[1] = 0;
    tc::fence_barrier_init();
  }
  // ---- this CTA's range of units ----
  // Up to 32 sequences every warp works it out for itself, a lane for a sequence; up to a block's
  // threads the block does, a thread for a sequence; past that it takes them in runs.
  const bool by_warp = a.B <= 32, at_once = a.B <= L::THREADS;
  const int me = by_warp ? lane : threadIdx.x;
  auto scan = [&](int v, int *total) { // sum of v before this sequence, and over all
    return by_warp ? warp_scan(v, total) : block_scan<L::THREADS>(v, total, misc);
  };
  bool bad = false;
  int tiles_all = 0, before = 0; // all sequences' tiles (per pair); those before sequence `me`
  CsSeq mine{};                  // sequence `me`, when all are looked at at once
  for (int b0 = 0; b0 < a.B; b0 += L::THREADS) {
    const int b = b0 + me;
    bool bb = false;
    mine = b < a.B ? cs_seq(a, b, &bb) : CsSeq{};
    bad |= bb;
    int t;
    before = scan(mine.tiles, &t);
    tiles_all += t;
  }
  if (bad) atomicExch(&g_cache_attn_split_range, 1);
  // No more CTAs than units take part, so each of them has one and every contributor arrives.
  const int U = tiles_all * hp, G = min((int)gridDim.x, U), cta = blockIdx.x;
  if (cta >= G) return;
  const int share = U / G, extra = U - share * G; // the first `extra` CTAs take one more
  int u0 = cta * share + min(cta, extra), u1 = u0 + share + (cta < extra);
  // With few pairs, CTAs of one pair each where that costs at most a quarter more units per CTA: a CTA
  // on a boundary would do two pairs' work and merges one after the other (for 8 pairs of 129 tiles
  // it finished at 21 us, the others at 8).  The fewest units per CTA that will do, by bisection.
  bool own_pair = false;
  int parts = 0, at = 0;            // CTAs per pair of sequence `me`, its first CTA
  int own_first = 0, own_count = 0; // the CTAs of this CTA's pair
  if (at_once && a.B * hp <= G && !g.align_pairs) {
    int lo = (U + G - 1) / G, hi = lo + max(1, lo / 4);
    auto fits = [&](int q) {
      parts = (mine.tiles + q - 1) / q;
      int all;
      at = scan(parts, &all) * hp;
      own_count = all * hp;
      return own_count <= G;
    };
    own_pair = fits(lo);
    if (!own_pair && fits(hi)) {
      own_pair = true;
      ++lo;
      bool last = true; // whether parts and at are those of hi
      while (lo < hi) {
        const int q = (lo + hi) / 2;
        last = fits(q);
        if (last) hi = q;
        else lo = q + 1;
      }
      if (!last) fits(hi);
    }
    if (own_pair && cta >= own_count) return;
  }
  CsWalk walk;
  if (at_once) {
    const bool here = mine.tiles && (own_pair ? cta >= at && cta < at + parts * hp
                                              : u0 >= before * hp && u0 < (before + mine.tiles) * hp);
    if (by_warp) {
      const int src = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
      walk.b = src;
      walk.before = __shfl_sync(0xffffffffu, before, src);
      at = __shfl_sync(0xffffffffu, at, src);
      parts = __shfl_sync(0xffffffffu, parts, src);
      walk.s.sp.past = __shfl_sync(0xffffffffu, mine.sp.past, src);
      walk.s.sp.count = __shfl_sync(0xffffffffu, mine.sp.count, src);
      walk.s.sp.total = __shfl_sync(0xffffffffu, mine.sp.total, src);
      walk.s.first = __shfl_sync(0xffffffffu, mine.first, src);
      walk.s.sink_tiles = __shfl_sync(0xffffffffu, mine.sink_tiles, src);
      walk.s.tiles = __shfl_sync(0xffffffffu, mine.tiles, src);
    } else if (here) {
      misc[16] = threadIdx.x;
      misc[17] = before;
      misc[18] = at;
      misc[19] = parts;
    }
  } else {
    int run = 0;
    for (int b0 = 0; b0 < a.B; b0 += L::THREADS) {
      const int b = b0 + threadIdx.x;
      bool bb;
      const int n = b < a.B ? cs_seq(a, b, &bb).tiles : 0;
      int t;
      const int first = run + block_scan<L::THREADS>(n, &t, misc);
      run += t;
      if (n && u0 >= first * hp && u0 < (first + n) * hp) {
        misc[16] = b;
        misc[17] = first;
      }
    }
  }
  __syncthreads(); // the barriers, and what another thread found
  if (!by_warp) {
    walk.b = misc[16];
    walk.before = misc[17];
    walk.s = cs_seq(a, walk.b, &bad);
    if (own_pair) {
      at = misc[18];
      parts = misc[19];
    }
  }
  if (own_pair) {
    const int pair = (cta - at) / parts, part = cta - at - pair * parts;
    own_first = cta - part;
    own_count = parts;
    const int n = walk.s.tiles, first = walk.before * hp + pair * n, q = n / parts, x = n - q * parts;
    u0 = first + part * q + min(part, x);
    u1 = u0 + q + (part < x);
  } else if (g.align_pairs) {
    // whole pairs only: a range starts and ends at the next pair's first unit
    CsWalk w = walk;
    cs_seek(g, w, u0);
    if (w.tile) u0 += w.s.tiles - w.tile;
    if (u1 < U) {
      cs_seek(g, w, u1);
      if (w.tile) u1 += w.s.tiles - w.tile;
    }
    if (u0 >= u1) return;
    cs_seek(g, walk, u0);
  }
  const int nun = u1 - u0;

  if (warp >= WARPS) {
    // ------------------------------ producers ------------------------------
    // One warp brings the keys and the scales, the other the values (a lane's copies are issued one
    // after the other, at about 170 cycles each: with one warp for both they set the pace).
    // Lane (my, ch) brings chunk ch of tile my of each batch of `per` tiles.  Page numbers are
    // read two batches ahead and scales one, so no batch waits for them; within a batch, groups of
    // up to 8 tiles go through the ring's protocol together, one tile a lane
    // (at most half the ring, so that a group's stages are distinct and the others stay in flight).
    const int nch = KEYS >> g.shift, per = 32 / nch, grp = min(per, min(8, STAGES / 2));
    const int my = lane / nch, ch = lane % nch;
    const bool values = warp > WARPS;
    const uint32_t chunk_bytes = (uint32_t)(g.chunk * 128 * NB);
    const CUtensorMap *map = values ? &map_v : &map_k;
    if (lane == 0) tc::prefetch_tensormap(map);
    struct Chunk {
      int id, row, kvh; // page, row in the page
      bool live;        // a key of it may be seen
    };
    // the page of this lane's chunk of tile i (of this CTA's)
    auto find = [&](int i) {
      Chunk c{0, 0, 0, false};
      if (i < nun) {
        cs_seek(g, walk, u0 + i);
        const int pack = walk.pair % g.packs, key0 = cs_key0(walk.s, walk.tile), j = key0 + ch * g.chunk;
        int pf, pl;
        cs_pack(g, walk.s, pack, RP, &pf, &pl);
        if (cs_live(g, walk.s, pf, pl, key0) && j < walk.s.sp.total) {
          const int page = j / a.T;
          c.id = a.table[(int64_t)walk.b * a.max_pages + page];
          c.row = j - page * a.T;
          c.kvh = walk.pair / g.packs;
          c.live = true;
        }
      }
      return c;
    };
    // its row of the pool in pages and heads, -1 when there is none; reports pages out of range
    auto place = [&](const Chunk &c) {
      if (!c.live) return -1;
      if (c.id >= 0 && c.id < a.pages) return c.id * a.Hkv + c.kvh;
      atomicExch(&g_cache_attn_split_range, 1);
      return -1;
    };
    bool stop = false;
    int issued = 0;
    Chunk c0 = find(my), c1 = find(per + my);
    int z0 = place(c0);
    float ks = !values && z0 >= 0 ? a.ks[z0] : 0.0f, vs = !values && z0 >= 0 ? a.vs[z0] : 0.0f;
    for (int i0 = 0; i0 < nun && !stop; i0 += per) {
      const int i = i0 + my, s = i % STAGES;
      const uint32_t have = __ballot_sync(0xffffffffu, z0 >= 0);
      auto copy = [&] { // this lane's boxes
        uint8_t *st = sm + s * L::STAGE + (values ? NB * BOX : 0) + ch * g.chunk * 128;
#pragma unroll
        for (int x = 0; x < NB; ++x) tc::tma_load_3d(st + x * BOX, map, &full[s], x * 128, c0.row, z0);
      };
      // The first fill of the ring: every copy starts before its scales are waited for (a copy may
      // land before its bytes are expected; the phase stays open until the arrival below).
      const bool early = i < STAGES;
      if (early && z0 >= 0) copy();
      // the next batch's scales, and the pages of the one after
      const int z1 = place(c1);
      const float ks1 = !values && z1 >= 0 ? a.ks[z1] : 0.0f, vs1 = !values && z1 >= 0 ? a.vs[z1] : 0.0f;
      const Chunk c2 = find(i + 2 * per);
      for (int k = 0; k < per && i0 + k < nun; k += grp) {
        const bool act = my >= k && my < k + grp && i < nun;
        bool ok = true;
        if (act && i >= STAGES) ok = tc::mbar_wait(&empty[s], ((i / STAGES) - 1) & 1);
        ok = ok && !flags[0]; // consumers that gave up free stages without reading them
        if (!__all_sync(0xffffffffu, ok)) {
          if (lane == 0) {
            atomicExch(&g_cache_attn_split_status, tc::kTimeoutEmpty);
            flags[0] = 1;
          }
          // early copies that are not expected yet: the wait below has to see them land
          if (early && i >= issued && i < nun && ch == 0)
            tc::mbar_expect_tx(&full[s], (uint32_t)__popc(have >> lane & ((1u << nch) - 1u)) * chunk_bytes);
          issued = max(issued, min(min(nun, STAGES), i0 + per));
          __syncwarp();
          stop = true;
          break;
        }
        if (act && !values) // key scale in score units; value scale times 2^-12; its logarithm; validity
          sc[s * CHUNKS + ch] = make_float4(ks * a.scale * kLog2E, vs * (1.0f / CS_UP_F),
                                            fminf(fmaxf(log2f(vs), CS_LV_MIN), CS_LV_MAX), z0 >= 0 ? 1.0f : 0.0f);
        __syncwarp();
        if (act && ch == 0)
          tc::mbar_expect_tx(&full[s], (uint32_t)__popc(have >> lane & ((1u << nch) - 1u)) * chunk_bytes);
        __syncwarp();
        if (act && !early && z0 >= 0) copy();
        issued = min(nun, i0 + k + grp);
      }
      c0 = c1;
      c1 = c2;
      z0 = z1;
      ks = ks1;
      vs = vs1;
    }
    // No copy may land once the CTA has left: wait (bounded) for each stage's last fill.  They
    // are done already unless a wait gave up.
    for (int i = max(0, issued - STAGES); i < issued; ++i) tc::mbar_wait(&full[i % STAGES], (i / STAGES) & 1);
    return;
  }

  // ------------------------------ consumers -------------------------------
  const int gq = lane >> 2, t = lane & 3;
  bool ok = true;
  int first_pair = -1; // number of the range's first pair
  const uint32_t smem0 = tc::smem_u32(sm);
  const uint32_t k_at = gq * 128 + (((DP == 64 ? t : 2 * t) ^ gq) << 4);
  const uint32_t v_at = 2 * t * 128 + ((DP == 64 ? (gq >> 1) ^ (2 * t) : gq ^ (2 * t)) << 4) + (DP == 64 ? (gq & 1) * 8 : 0);
  int seg0 = 0;
  while (seg0 < nun) {
    cs_seek(g, walk, u0 + seg0);
    const CsSeq seq = walk.s;
    const int seg1 = min(nun, seg0 + seq.tiles - walk.tile);
    const int kvh = walk.pair / g.packs, pack = walk.pair % g.packs;
    const int pair = walk.b * hp + walk.pair;
    if (first_pair < 0) first_pair = pair;
    const int rows = min(RP, g.rows - pack * RP);
    int pos_first, pos_last;
    cs_pack(g, seq, pack, RP, &pos_first, &pos_last);

    // ---- queries: B fragments, lane (gq, t) holds row gq of each 8-row tile ----
    // k step s of box x covers columns 128 x + 32 t + 4 s .. + 3 of lane t (16 t + 4 s when DP is 64).
    uint32_t qb[NT][KS][2];
    float qf[NT][2]; // power of two of the columns' rows 2t, 2t + 1
    int hi[NT][2], lo[NT][2]; // last key seen, first key of the window
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = pack * RP + nt * 8 + gq;
      const bool in = r < g.rows;
      const T *qp = static_cast<const T *>(a.q) + (int64_t)walk.b * a.q_b +
                    (in ? (int64_t)(kvh * a.group + r % a.group) * a.q_h + (int64_t)(r / a.group) * a.q_s : 0);
      constexpr int COLS = DP == 64 ? 16 : 32;
      float f = 1.0f;
#pragma unroll
      for (int x = 0; x < NB; ++x)
#pragma unroll
        for (int c = 0; c < COLS / 8; ++c) {
          const int d = x * 128 + COLS * t + 8 * c;
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (in && d < a.D) v = *reinterpret_cast<const uint4 *>(qp + d); // D is a multiple of 16
          const int k = x * 8 + 2 * c;
          qb[nt][k][0] = v.x;
          qb[nt][k][1] = v.y;
          qb[nt][k + 1][0] = v.z;
          qb[nt][k + 1][1] = v.w;
        }
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        // the row's largest exponent, over the four lanes of the row
        uint32_t e = 0u;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i) e = max(e, max(qb[nt][k][i] & 0x7f80u, (qb[nt][k][i] >> 16) & 0x7f80u));
        e = max(e, __shfl_xor_sync(0xffffffffu, e, 1));
        e = max(e, __shfl_xor_sync(0xffffffffu, e, 2));
        const int ex = min(max((int)(e >> 7) - 127, -126), 126);
        const float down = __uint_as_float((uint32_t)(127 - ex) << 23);
        f = __uint_as_float((uint32_t)(127 + ex) << 23);
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            qb[nt][k][i] = half2_of(__uint_as_float(qb[nt][k][i] << 16) * down,
                                    __uint_as_float(qb[nt][k][i] & 0xffff0000u) * down);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        qf[nt][e] = __shfl_sync(0xffffffffu, f, (2 * t + e) * 4);
        const int rc = pack * RP + nt * 8 + 2 * t + e, i = rc / a.group, p = seq.sp.past + i;
        const bool counts = rc < g.rows && i < seq.sp.count;
        hi[nt][e] = !counts ? -1 : a.causal ? min(p, seq.sp.total - 1) : seq.sp.total - 1;
        lo[nt][e] = a.causal && a.window >= 0 ? p - a.window : 0;
      }
    }
    float o[NT][KS][4]; // [columns 16 gq + 2 i (+1)][rows 2t, 2t + 1]; 8 gq + 2 i when DP is 64
    float m_run[NT][2], l_run[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][k][e] = 0.0f;
      m_run[nt][0] = m_run[nt][1] = -INFINITY;
      l_run[nt][0] = l_run[nt][1] = 0.0f;
    }

    // A stage is always the same warp's, which frees its last fill before it waits for the next, so
    // a parity wait cannot be satisfied by the fill before last.
    for (int i = seg0 + ((warp - seg0 % WARPS + WARPS) % WARPS); i < seg1; i += WARPS) {
      const int s = i % STAGES;
      if (ok && !tc::mbar_wait(&full[s], (i / STAGES) & 1)) {
        atomicExch(&g_cache_attn_split_status, tc::kTimeoutFull);
        flags[0] = 1;
        ok = false;
      }
      ok = __all_sync(0xffffffffu, ok);
      const int key0 = cs_key0(seq, walk.tile + (i - seg0));
      if (ok && cs_live(g, seq, pos_first, pos_last, key0)) {
        // The 16-byte unit u of row r of a box lies at r * 128 + ((u ^ (r & 7)) << 4).  A lane's K rows
        // are gq (mod 8), its V rows 2t and 2t + 1, so the exclusive or leaves two places for each.
        const uint32_t kb = smem0 + s * L::STAGE, vb = kb + NB * BOX;
        const uint32_t ka = kb + k_at, va[2] = {vb + v_at, vb + (v_at ^ 16) + 128};
        // scales of the tokens of this lane's S rows (gq and gq + 8 of each 16)
        auto scales = [&](int mt, int h) { return sc[s * CHUNKS + ((mt * 16 + h * 8 + gq) >> g.shift)]; };
        const bool all = __all_sync(0xffffffffu, lane >= KEYS >> g.shift || sc[s * CHUNKS + lane].w != 0.0f);
        const bool whole = all && key0 + KEYS <= seq.sp.total;
        if (!whole) {
          // rows that hold no token of this sequence: their V codes must not reach the MMA
#pragma unroll 1
          for (int r = lane >> 3; r < KEYS; r += 4) {
            if (key0 + r >= seq.sp.total || sc[s * CHUNKS + (r >> g.shift)].w == 0.0f)
#pragma unroll
              for (int x = 0; x < NB; ++x)
                *reinterpret_cast<uint4 *>(sm + s * L::STAGE + (NB + x) * BOX + r * 128 + (lane & 7) * 16) =
                    make_uint4(0u, 0u, 0u, 0u);
          }
          tc::fence_proxy_async(); // before the stage's next TMA fill
          __syncwarp();
        }
        const bool need_mask =
            !whole || (a.causal && (key0 + KEYS - 1 > pos_first ||
                                    (a.window >= 0 && key0 < pos_last - a.window && key0 + KEYS > a.sinks))) ||
            pos_last - seq.sp.past != (pack * RP + rows - 1) / a.group; // rows that do not count
        // ---- S^T = K . Q^T ----
        // With one tile of rows, even and odd steps have sums of their own: four short chains of MMAs.
        constexpr int CH = NT == 1 ? 2 : 1;
        float sv[MT][NT][4];
#pragma unroll
        for (int m2 = 0; m2 < MT; m2 += 2) {
          float sx[CH][2][NT][4];
#pragma unroll
          for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) sx[c][mt][nt][e] = 0.0f;
#pragma unroll
          for (int x = 0; x < NB; ++x)
#pragma unroll
            for (int h = 0; h < (DP == 64 ? 1 : 2); ++h) {
              uint32_t w[2][2][4];
#pragma unroll
              for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                  const uint4 v = lds128((h ? ka ^ 16 : ka) + x * BOX + (m2 + mt) * 2048 + r * 1024);
                  w[mt][r][0] = v.x;
                  w[mt][r][1] = v.y;
                  w[mt][r][2] = v.z;
                  w[mt][r][3] = v.w;
                }
#pragma unroll
              for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
                  uint32_t a0, a1, a2, a3;
                  to_half<Q>(w[mt][0][q], a0, a2);
                  to_half<Q>(w[mt][1][q], a1, a3);
                  const int k = x * 8 + h * 4 + q;
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt)
                    mma16816(sx[q % CH][mt][nt], a0, a1, a2, a3, qb[nt][k][0], qb[nt][k][1]);
                }
            }
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                sv[m2 + mt][nt][e] = CH == 2 ? sx[0][mt][nt][e] + sx[CH - 1][mt][nt][e] : sx[0][mt][nt][e];
        }
        // ---- scores in base 2, masks, the running reference ----
        float mx[NT][2], lz[MT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mx[nt][0] = mx[nt][1] = -INFINITY;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float4 c = scales(mt, h);
            lz[mt][h] = c.z;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                sv[mt][nt][2 * h + e] *= std::is_same<T, __half>::value ? c.x : c.x * qf[nt][e];
          }
        if (a.softcap > 0.0f) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                sv[mt][nt][e] = a.softcap * tanhf(sv[mt][nt][e] * kLn2 / a.softcap) * kLog2E;
        }
        if (need_mask) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int j = key0 + mt * 16 + h * 8 + gq;
              const bool has = scales(mt, h).w != 0.0f;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  if (!(has && j <= hi[nt][e] && (j >= lo[nt][e] || j < a.sinks))) sv[mt][nt][2 * h + e] = -INFINITY;
            }
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[nt][e & 1] = fmaxf(mx[nt][e & 1], sv[mt][nt][e] + lz[mt][e >> 1]);
        // m moves only when a product would pass 2^15 (then to 2^7), so most tiles cost one vote instead
        // of a maximum over the lanes and a pass over the sums
        bool over = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) over = over || mx[nt][e] > m_run[nt][e] + (CS_TOP - CS_BASE);
        if (__any_sync(0xffffffffu, over)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
              for (int w = 4; w < 32; w <<= 1) mx[nt][e] = fmaxf(mx[nt][e], __shfl_xor_sync(0xffffffffu, mx[nt][e], w));
              const float mn = fmaxf(m_run[nt][e], mx[nt][e]);
              const float corr = ex2(m_run[nt][e] - (mn == -INFINITY ? 0.0f : mn));
              m_run[nt][e] = mn;
              l_run[nt][e] *= corr;
#pragma unroll
              for (int k = 0; k < KS; ++k) {
                o[nt][k][e] *= corr;
                o[nt][k][2 + e] *= corr;
              }
            }
        }
        float ref[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) ref[nt][e] = (m_run[nt][e] == -INFINITY ? 0.0f : m_run[nt][e]) - (CS_BASE + CS_UP);
        // ---- P^T fragments ----
        uint32_t pb[MT][NT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float vs = scales(mt, h).y;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float p[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float v = sv[mt][nt][2 * h + e];
                p[e] = ex2(v - ref[nt][e]);
                l_run[nt][e] += p[e];
                p[e] *= vs;
                // a key that is not seen has p = 0 whatever its page's scale is
                if (need_mask && v == -INFINITY) p[e] = 0.0f;
              }
              pb[mt][nt][h] = transpose8(half2_of(p[0], p[1]));
            }
          }
        // ---- O^T += V^T . P^T ----
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int x = 0; x < NB; ++x) {
            uint32_t w[4][4]; // [token 2t, 2t + 1, 2t + 8, 2t + 9][4 columns each]
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint32_t at = va[q & 1] + mt * 2048 + (q >> 1) * 1024;
              if constexpr (DP == 64) {
                const uint2 v = lds64(at);
                w[q][0] = v.x;
                w[q][1] = v.y;
              } else {
                const uint4 v = lds128(at + x * BOX);
                w[q][0] = v.x;
                w[q][1] = v.y;
                w[q][2] = v.z;
                w[q][3] = v.w;
              }
            }
#pragma unroll
            for (int c = 0; c < (DP == 64 ? 2 : 4); ++c) {
#pragma unroll
              for (int h = 0; h < 2; ++h) { // columns 4c + 2h, 4c + 2h + 1
                const uint32_t sel = h ? 0x7362u : 0x5140u;
                uint32_t a0, a1, a2, a3;
                to_half<Q>(__byte_perm(w[0][c], w[1][c], sel), a0, a1);
                to_half<Q>(__byte_perm(w[2][c], w[3][c], sel), a2, a3);
                const int k = x * 8 + 2 * c + h;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][k], a0, a1, a2, a3, pb[mt][nt][0], pb[mt][nt][1]);
              }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&empty[s]);
    }

    // ---------------- end of a pair's segment: merge the warps ----------------
    auto consumers_sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory"); };
    consumers_sync(); // the merge buffer is free
    constexpr int W = L::W;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l_run[nt][e] += __shfl_xor_sync(0xffffffffu, l_run[nt][e], 4);
        l_run[nt][e] += __shfl_xor_sync(0xffffffffu, l_run[nt][e], 8);
        l_run[nt][e] += __shfl_xor_sync(0xffffffffu, l_run[nt][e], 16);
        float *mw = mrg + (size_t)(warp * RP + nt * 8 + 2 * t + e) * W;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const int d = DP == 64 ? 8 * gq + 2 * k : (k >> 3) * 128 + 16 * gq + 2 * (k & 7);
          *reinterpret_cast<float2 *>(mw + d) = make_float2(o[nt][k][e], o[nt][k][2 + e]);
        }
        if (gq == 0) {
          mw[DP] = m_run[nt][e];
          mw[DP + 1] = l_run[nt][e];
        }
      }
    consumers_sync();
    // the pair's units, and the CTAs cf .. cl that hold some of them
    const int pu = walk.before * hp + walk.pair * seq.tiles;
    auto cta_of = [&](int u) {
      const int thr = extra * (share + 1);
      return u < thr ? u / (share + 1) : extra + (u - thr) / share;
    };
    const int cf = own_pair ? own_first : cta_of(pu);
    const int cl = own_pair ? own_first + own_count - 1 : cta_of(pu + seq.tiles - 1);
    const bool one = g.align_pairs || cf == cl;
    // Only cf can hold the pair in its second slot: every later CTA's range starts inside it.
    const int cf_slot = !own_pair && cf * share + min(cf, extra) < pu ? 1 : 0;
    float *part = g.partials + ((size_t)cta * 2 + (pair == first_pair ? 0 : 1)) * RP * W;
    auto put = [&](int r, int d, float4 v, float l) { // four columns of row r
      const int rr = pack * RP + r;
      T *y = static_cast<T *>(a.y) + (int64_t)walk.b * a.q_b + (int64_t)(kvh * a.group + rr % a.group) * a.q_h +
             (int64_t)(rr / a.group) * a.q_s + d;
      const float inv = l == 0.0f ? 0.0f : CS_UP_F / l;
      uint2 w;
      if constexpr (std::is_same<T, __half>::value) {
        w.x = half2_of(v.x * inv, v.y * inv);
        w.y = half2_of(v.z * inv, v.w * inv);
      } else {
        const __nv_bfloat162 b0 = __floats2bfloat162_rn(v.x * inv, v.y * inv);
        const __nv_bfloat162 b1 = __floats2bfloat162_rn(v.z * inv, v.w * inv);
        w.x = *reinterpret_cast<const uint32_t *>(&b0);
        w.y = *reinterpret_cast<const uint32_t *>(&b1);
      }
      *reinterpret_cast<uint2 *>(y) = w;
    };
    auto add = [](float4 &acc, const float4 &v, float w) {
      acc.x = fmaf(v.x, w, acc.x);
      acc.y = fmaf(v.y, w, acc.y);
      acc.z = fmaf(v.z, w, acc.z);
      acc.w = fmaf(v.w, w, acc.w);
    };
    const int nw = min(WARPS, seg1 - seg0), w0 = seg0 % WARPS, n4 = rows * (DP / 4);
    for (int e = threadIdx.x; e < n4; e += WARPS * 32) {
      const int r = e / (DP / 4), d = e % (DP / 4) * 4;
      if (d >= a.D) continue;
      float M = -INFINITY;
      for (int k = 0; k < nw; ++k) {
        const int w = w0 + k < WARPS ? w0 + k : w0 + k - WARPS;
        M = fmaxf(M, mrg[(w * RP + r) * W + DP]);
      }
      const float base = M == -INFINITY ? 0.0f : M;
      float l = 0.0f;
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int k = 0; k < nw; ++k) {
        const int w = w0 + k < WARPS ? w0 + k : w0 + k - WARPS;
        const float *row = mrg + (w * RP + r) * W;
        const float2 ml = *reinterpret_cast<const float2 *>(row + DP);
        const float c = exp2f(ml.x - base);
        l = fmaf(ml.y, c, l);
        add(acc, *reinterpret_cast<const float4 *>(row + d), c);
      }
      if (one) {
        if (ok) put(r, d, acc, l);
      } else {
        *reinterpret_cast<float4 *>(part + r * W + d) = acc;
        if (d == 0) *reinterpret_cast<float2 *>(part + r * W + DP) = make_float2(M, l);
      }
    }
    if (!one) {
      consumers_sync();
      if (threadIdx.x == 0) {
        const uint32_t inc = flags[0] ? kAbortMark + 1u : 1u;
        const uint32_t now = arrive_acq_rel(g.counters + pair, inc) + inc;
        const bool last = (now & (kAbortMark - 1u)) == (uint32_t)(cl - cf + 1);
        if (last) g.counters[pair] = 0u;
        flags[1] = last && (now >> 16) == 0u ? 1 : 0;
      }
      consumers_sync();
      if (flags[1] && ok) {
        // The last CTA of this pair: the partials in CTA order.  With threads to spare, `teams` of
        // them share the CTAs (every teams-th each) and are joined in order through the merge
        // buffer; a thread has up to eight partials in flight.
        const int nc = cl - cf + 1, teams = max(1, WARPS * 32 / n4);
        for (int x = threadIdx.x; x < (teams > 1 ? n4 * teams : n4); x += WARPS * 32) {
          const int team = teams > 1 ? x / n4 : 0, e = x - team * n4;
          const int r = e / (DP / 4), d = e % (DP / 4) * 4;
          float M = -INFINITY, l = 0.0f;
          float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          for (int c = team; c < nc; c += 8 * teams) {
            float2 ml[8];
            float4 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int cc = c + k * teams;
              ml[k] = make_float2(-INFINITY, 0.0f);
              v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              if (cc < nc) {
                const float *row = g.partials + ((size_t)(cf + cc) * 2 + (cc ? 0 : cf_slot)) * RP * W + r * W;
                ml[k] = __ldcg(reinterpret_cast<const float2 *>(row + DP));
                if (d < a.D) v[k] = __ldcg(reinterpret_cast<const float4 *>(row + d));
              }
            }
            float mn = M;
#pragma unroll
            for (int k = 0; k < 8; ++k) mn = fmaxf(mn, ml[k].x);
            const float base = mn == -INFINITY ? 0.0f : mn, keep = exp2f(M - base);
            l *= keep;
            acc.x *= keep;
            acc.y *= keep;
            acc.z *= keep;
            acc.w *= keep;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float w = exp2f(ml[k].x - base);
              l = fmaf(ml[k].y, w, l);
              add(acc, v[k], w);
            }
            M = mn;
          }
          if (teams > 1) {
            *reinterpret_cast<float4 *>(mrg + 8 * x) = acc;
            *reinterpret_cast<float2 *>(mrg + 8 * x + 4) = make_float2(M, l);
          } else if (d < a.D) {
            put(r, d, acc, l);
          }
        }
        if (teams > 1) {
          consumers_sync();
          for (int e = threadIdx.x; e < n4; e += WARPS * 32) {
            const int r = e / (DP / 4), d = e % (DP / 4) * 4;
            float M = -INFINITY, l = 0.0f;
            for (int team = 0; team < teams; ++team) M = fmaxf(M, mrg[8 * (team * n4 + e) + 4]);
            const float base = M == -INFINITY ? 0.0f : M;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int team = 0; team < teams; ++team) {
              const float *p = mrg + 8 * (team * n4 + e);
              const float w = exp2f(p[4] - base);
              l = fmaf(p[5], w, l);
              add(acc, *reinterpret_cast<const float4 *>(p), w);
            }
            if (d < a.D) put(r, d, acc, l);
          }
        }
      }
    }
    seg0 = seg1;
  }
}

// Rows of a pack in eights: as few as hold all rows, up to 32 (16 for heads above 128, whose
// accumulators fill the registers).
int cs_nt(int64_t rows, int dp) { return rows <= 8 ? 1 : rows <= 16 || dp == 256 ? 2 : 4; }

template <typename T, typename Q, int DP, int NT>
int cs_launch(const CUtensorMap &mk, const CUtensorMap &mv, const CsArgs &g, unsigned grid, cudaStream_t st) {
  using L = CsLayout<DP, NT>;
  auto kern = cache_attn_split<T, Q, DP, NT>;
  B2_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::SMEM));
  kern<<<grid, L::THREADS, L::SMEM, st>>>(mk, mv, g);
  B2_LAUNCH_CHECK();
  return B2_OK;
}

template <typename T, typename Q>
int cs_pick(int dp, int nt, const CUtensorMap &mk, const CUtensorMap &mv, const CsArgs &g, unsigned grid,
            cudaStream_t st) {
  if (dp == 64) {
    if (nt == 1) return cs_launch<T, Q, 64, 1>(mk, mv, g, grid, st);
    if (nt == 2) return cs_launch<T, Q, 64, 2>(mk, mv, g, grid, st);
    return cs_launch<T, Q, 64, 4>(mk, mv, g, grid, st);
  }
  if (dp == 128) {
    if (nt == 1) return cs_launch<T, Q, 128, 1>(mk, mv, g, grid, st);
    if (nt == 2) return cs_launch<T, Q, 128, 2>(mk, mv, g, grid, st);
    return cs_launch<T, Q, 128, 4>(mk, mv, g, grid, st);
  }
  if (nt == 1) return cs_launch<T, Q, 256, 1>(mk, mv, g, grid, st);
  return cs_launch<T, Q, 256, 2>(mk, mv, g, grid, st);
}

int cs_grid() { return std::min(sm_count(), CS_CTAS); }
int dp_of(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

} // namespace

// Head sizes that are multiples of 16 up to 256, pages that are multiples of 8 tokens, 16-byte
// aligned Q and cache (TMA), and counts that fit 32 bits.
bool cache_attn_split_eligible(const CaArgs &a) {
  const int64_t rows = (int64_t)a.S * a.group, nt = cs_nt(rows, dp_of(a.D));
  const int64_t packs = (rows + 8 * nt - 1) / (8 * nt);
  const int64_t tiles = (int64_t)a.max_pages * a.T / KEYS + 2;
  return a.D % 16 == 0 && a.D <= 256 && a.T % 8 == 0 && aligned(a.q, 16) && aligned(a.k, 16) &&
         aligned(a.v, 16) && aligned(a.y, 8) && a.pages > 0 && rows < ((int64_t)1 << 30) &&
         (double)a.B * a.Hkv * packs * tiles < 1e9;
}

size_t cache_attn_split_workspace(const CaArgs &a) {
  const int dp = dp_of(a.D), nt = cs_nt((int64_t)a.S * a.group, dp);
  return kCounterBytes + (size_t)cs_grid() * 2 * 8 * nt * (dp + 4) * 4;
}

int cache_attn_split_launch(const CaArgs &a, bool f16, bool f8, void *ws, cudaStream_t st) {
  const int dp = dp_of(a.D), nt = cs_nt((int64_t)a.S * a.group, dp);
  CsArgs g{};
  g.c = a;
  g.rows = a.S * a.group;
  g.packs = (g.rows + 8 * nt - 1) / (8 * nt);
  g.shift = 3;
  while ((1 << g.shift) < KEYS && a.T % (2 << g.shift) == 0) ++g.shift;
  g.chunk = 1 << g.shift;
  g.align_pairs = (int64_t)a.B * a.Hkv * g.packs > (int64_t)kMaxCounters;
  g.counters = static_cast<uint32_t *>(ws);
  g.partials = reinterpret_cast<float *>(static_cast<uint8_t *>(ws) + kCounterBytes);
  // [pages * Hkv][T][D] codes; columns past D read as zeros
  CUtensorMap mk, mv;
  const uint64_t dims[3] = {(uint64_t)a.D, (uint64_t)a.T, (uint64_t)a.pages * a.Hkv};
  const uint64_t strides[2] = {(uint64_t)a.D, (uint64_t)a.T * a.D};
  const uint32_t box[3] = {128, (uint32_t)g.chunk, 1};
  if (int rc = make_tensor_map(&mk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, a.k, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  if (int rc = make_tensor_map(&mv, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, a.v, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  const unsigned grid = (unsigned)cs_grid();
  if (f16) return f8 ? cs_pick<__half, Fp8>(dp, nt, mk, mv, g, grid, st) : cs_pick<__half, Int8>(dp, nt, mk, mv, g, grid, st);
  return f8 ? cs_pick<__nv_bfloat16, Fp8>(dp, nt, mk, mv, g, grid, st)
            : cs_pick<__nv_bfloat16, Int8>(dp, nt, mk, mv, g, grid, st);
}

namespace {
int read_word(int reset, const int &symbol) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, symbol, sizeof(int)) != cudaSuccess) return -1;
  if (reset && v) {
    const int z = 0;
    if (cudaMemcpyToSymbol(symbol, &z, sizeof(int)) != cudaSuccess) return -1;
  }
  return v;
}
} // namespace
int status_read_cache_attn_split(int reset) { return read_word(reset, g_cache_attn_split_status); }
int range_read_cache_attn_split(int reset) { return read_word(reset, g_cache_attn_split_range); }

} // namespace b2
