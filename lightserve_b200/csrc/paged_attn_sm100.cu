// Paged attention for many rows per sequence (chunked prefill) on the
// 5th-generation tensor cores.
//
// One CTA: two query tiles of up to 128 pairs (row, head of the group) of one
// (sequence, cache head), and one chunk of the keys they see, in tiles of 128.
// The inner loop is the one of the contiguous forward kernel: S_t = Q_t K^T
// (tcgen05 SS, fp32 in TMEM), softmax with one thread per row (TMEM lane) and a
// conditional rescale, P packed to 16 bits over S in two halves, O_t += P_t V
// (TS), the two query tiles' MMA batches and softmaxes alternating. What
// differs is where K and V come from and which keys count:
//  * 16-bit cache: one TMA box per page and head (the cache is a tensor of
//    8-row groups, so the box's atoms land as the MMA's descriptors want them; a
//    box per 64-column half took 13% longer over pages of 16). Pages that do not
//    exist, or that no row sees, are fetched past the end: zeros.
//  * e4m3 cache: TMA stages the raw tile, and a converter warpgroup multiplies
//    each row by its power of two, rounds to q's type (exact in bf16, and in fp16
//    for a cache written from fp16 rows; values below 2^-21 of one written from a
//    wider type lose bits) and writes the swizzled tiles. (Two converter warpgroups
//    took the registers of the softmax and were 12% slower; loading the raw
//    rows into registers instead of staging them, 25%.)
//  * V rows that no row of the item sees (past the context, between sinks and
//    window) are zeroed in shared memory, so that what such cells hold never
//    meets a weight of 0; the tiles that need it are the ends of a span.
//  * A pair's heads of one group share the K/V tiles: row r of a tile is
//    token r / G, head r % G.
//
// What bounds it, per step of 128 keys at D = 128: the softmax's exponentials
// (2 x 128 x 128 at 16 a clock, 2048 clocks) and the MMAs (2100 clocks at the
// dense rate), overlapped but for the chain S -> P -> PV -> next S: about 3000
// clocks, 65% of the tensor pipe and 65% of the exponential unit busy. At D = 64
// the MMAs halve and the step stays. An e4m3 step is 17% longer: the converters
// share shared memory and issue slots with the rest. Measured, 16 heads, one chunk
// of 8192 tokens: D 128 bf16 222 us (1240 TFLOP/s), over e4m3 259; D 64 209 and 232.
// (Tried: a share of the exponentials on the FMA pipe, D 128 +2% at an eighth to
// +16% at a half, D 64 -2% to +22%; an MMA warp per
// query tile, +25%, the tiles fall into step; three S buffers at D = 64, +8%;
// six converter warps, +3 to +11%.)
//
// Warps: 0 loads (Q; K, V of a 16-bit cache, raw tiles of an e4m3 one), 1 issues
// MMAs and owns TMEM, 4-7 and 8-11 softmax of query tile 0 and 1, 12-15 convert (e4m3 only).
// TMEM: S0 [0,128), S1 [128,256), O0 [256,384), O1 [384,512) columns. Every
// mbarrier wait is bounded; on a timeout the error word is set, the role ends,
// TMEM is freed and the CTA exits.
#include "paged_attn.cuh"
#include "sm100.cuh"
#include "tma_host.cuh"

#include <algorithm>
#include <type_traits>

namespace lsb {
namespace pa {
namespace tc {

using namespace sm100;

constexpr int BM = 128;
constexpr int BN = TC_TK;
constexpr int TILES = 2;
constexpr int NS = 2;  // K/V ring stages
constexpr int CHUNK_BYTES = 128 * 128;  // Q: [128 rows][64 columns] of 16 bits
// K and V tiles are rows of 128-byte-swizzled atoms (8 keys x 64 columns, 1024
// bytes): [key / 8][column / 64][8 keys][64 columns], the order in which one
// TMA box over [cache rows / 8, D / 64, 8, 64] delivers a whole page.
constexpr int ATOM = 1024;
constexpr float RESCALE_THRESHOLD = 8.0f;

template <int D, bool FP8>
struct Smem {
  static constexpr int KC = D / 64;
  static constexpr int TILE = KC * CHUNK_BYTES;  // bytes of a K or V tile
  static constexpr int RAW = BN * D;             // bytes of an e4m3 tile
  static constexpr int Q_OFF = 0;
  static constexpr int K_OFF = Q_OFF + TILES * KC * CHUNK_BYTES;
  static constexpr int V_OFF = K_OFF + NS * KC * CHUNK_BYTES;
  static constexpr int RAW_OFF = V_OFF + NS * KC * CHUNK_BYTES;  // e4m3 K, V, then their scales
  static constexpr int SCALE_OFF = RAW_OFF + (FP8 ? 2 * RAW : 0);
  static constexpr int BAR_OFF = SCALE_OFF + (FP8 ? 2 * BN : 0);
  // q_full[2], k_full[NS], v_full[NS], k_empty[NS], v_empty[NS], s_full[2], p_full[2][2],
  // pv_done[2], edge, raw_full[2], raw_empty[2]
  static constexpr int NBAR = TILES + 4 * NS + 4 * TILES + 1 + 4;
  static constexpr int TMEM_SLOT_OFF = BAR_OFF + NBAR * 8;
  static constexpr int BYTES = TMEM_SLOT_OFF + 16;
  static constexpr int ALLOC = BYTES + 1024;  // slack for 1024-byte alignment
};

__device__ __forceinline__ float max3f(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

__device__ __forceinline__ void st_global_v8(void* dst, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "r"(w[0]), "r"(w[1]),
               "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// The n lowest bits set (none for n <= 0, all for n >= 32).
__device__ __forceinline__ uint32_t low_bits(int n) {
  return n >= 32 ? 0xffffffffu : (1u << max(n, 0)) - 1u;
}

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0,
                                            int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1)
      : "memory");
}

// A 128-byte-swizzle descriptor by its words (smem_desc_sw128's layout): byte
// offsets / 16 are added to the low one, which holds the address and the leading
// offset. Building each descriptor from its address took 2% of the loop.
__device__ __forceinline__ uint64_t desc(uint32_t lo, uint32_t hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
  return d;
}
__device__ __forceinline__ uint32_t desc_lo(const void* p, int lbo) {
  return (smem_u32(p) >> 4) | (uint32_t)(lbo >> 4) << 16;
}
constexpr uint32_t desc_hi(int sbo) { return (uint32_t)(sbo >> 4) | 1u << 14 | 2u << 29; }

// Two fp16 values times an fp16 factor, in fp32 (exact), without widening them
// first (bf16 over e4m3, one chunk of 8192 tokens, D 128: 281 us against 272).
__device__ __forceinline__ float2 mul_widen(uint32_t z, uint16_t f) {
  float2 y;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
      "fma.rn.f32.f16 %0, l, %3, %4;\n\tfma.rn.f32.f16 %1, h, %3, %4;\n\t}"
      : "=f"(y.x), "=f"(y.y)
      : "r"(z), "h"(f), "f"(-0.f));
  return y;
}

template <int N>
__device__ __forceinline__ float row_max(const uint32_t (&sr)[N][32]) {
  float mx8[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) mx8[u] = -INFINITY;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int cc = 0; cc < 32; cc += 2)
      mx8[(cc >> 1) & 7] = max3f(mx8[(cc >> 1) & 7], __uint_as_float(sr[i][cc]),
                                 __uint_as_float(sr[i][cc + 1]));
  return fmaxf(max3f(mx8[0], mx8[1], mx8[2]),
               max3f(max3f(mx8[3], mx8[4], mx8[5]), mx8[6], mx8[7]));
}

// Everything a role needs to know about the CTA's work; each thread derives
// it from the lengths in device memory.
struct Item {
  Seq q;
  int hk, pairs, R;         // R: pairs per query tile
  int c0;                   // the item's first query tile
  int pos_lo, pos_hi;       // positions of its rows
  KeySpan span;
  int v0, nkv, nkv_t[TILES];  // first span tile, tiles visited by the item and by each query tile
  int chunk, chunks;
};

// False: this CTA has nothing to do.
__device__ __forceinline__ bool make_item(const Params& p, Item& w) {
  w.q = load_seq(p, blockIdx.z);
  w.hk = blockIdx.x / p.P;
  w.chunk = blockIdx.x % p.P;
  w.R = BM / p.G * p.G;
  w.pairs = w.q.n * p.G;
  w.c0 = (gridDim.y - 1 - blockIdx.y) * TILES;  // later rows see more keys: they start first
  if (w.c0 * w.R >= w.pairs) return false;
  tile_positions(p, w.q, w.c0 / TILES, TILES * w.R, w.pos_lo, w.pos_hi);
  w.span = KeySpan(p, w.q, w.pos_lo, w.pos_hi, BN);
  const int tiles = w.span.count(), per = p.chunk / BN;
  w.chunks = chunks_of(p, tiles, BN);
  if (w.chunk >= w.chunks) return false;
  w.v0 = w.chunk * per;
  const int v1 = w.chunk + 1 == w.chunks ? tiles : min(tiles, w.v0 + per);
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    int lo, hi, n = 0;
    if ((w.c0 + t) * w.R < w.pairs) {
      // Span tiles whose first key the tile's last row reaches, a prefix.
      tile_positions(p, w.q, w.c0 + t, w.R, lo, hi);
      const int last = min(hi, w.q.ctx - 1);
      const int reach = last < 0 ? 0 : last / BN + 1;  // key tiles from 0 on
      n = min(w.span.s_tiles, reach) + max(0, min(w.span.hi, reach) - w.span.lo);
    }
    w.nkv_t[t] = max(0, min(n, v1) - w.v0);
  }
  w.nkv = max(w.nkv_t[0], w.nkv_t[1]);
  return true;
}

template <int D, int FMT, bool FP8>
__global__ void __launch_bounds__(FP8 ? 512 : 384, 1)
paged_chunk_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                   const __grid_constant__ CUtensorMap tv, const Params p, const int box_log2) {
  using L = Smem<D, FP8>;
  using T = typename std::conditional<FMT == 1, __nv_bfloat16, __half>::type;
  constexpr int KC = L::KC;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
  uint64_t* q_full = bars;                // [TILES]
  uint64_t* k_full = q_full + TILES;      // [NS]
  uint64_t* v_full = k_full + NS;         // [NS]
  // K is free after its QK, V a step later after its PV: the next K's load or
  // conversion has a whole step to hide behind.
  uint64_t* k_empty = v_full + NS;        // [NS]
  uint64_t* v_empty = k_empty + NS;       // [NS]
  uint64_t* s_full = v_empty + NS;        // [TILES]
  uint64_t* p_full = s_full + TILES;      // [TILES][2]
  uint64_t* pv_done = p_full + 2 * TILES; // [TILES]
  uint64_t* edge = pv_done + TILES;       // V boxes of a tile that is zeroed in places
  uint64_t* raw_full = edge + 1;          // [K, V]: the e4m3 tile is in shared memory
  uint64_t* raw_empty = raw_full + 2;     // [K, V]: its converters have read it
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::TMEM_SLOT_OFF);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    prefetch_tmap(&tq);
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
  }
  allow_dependents();
  wait_prerequisites();
  Item w;
  if (!make_item(p, w)) return;  // the whole CTA alike

  if (threadIdx.x == 0) {
    for (int t = 0; t < TILES; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[2 * t], BM);
      mbar_init(&p_full[2 * t + 1], BM);
      mbar_init(&pv_done[t], 1);
    }
    for (int s = 0; s < NS; ++s) {
      mbar_init(&k_full[s], FP8 ? 4 : 1);
      mbar_init(&v_full[s], FP8 ? 4 : 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    mbar_init(edge, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], 4);
    }
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  uint8_t* sQ = smem + L::Q_OFF;
  uint8_t* sK = smem + L::K_OFF;
  uint8_t* sV = smem + L::V_OFF;
  const int32_t* bt = p.block_tables + (int64_t)blockIdx.z * p.max_blocks;
  // First key of the item's j-th tile.
  auto key0_of = [&](int j) { return w.span.tile(w.v0 + j) * BN; };
  // Whether some key of [a, a + n) is seen by a row of the item.
  auto any_seen = [&](int a, int n) {
    return a <= w.pos_hi && a < w.q.ctx &&
           (p.window == 0 || w.pos_lo - (a + n - 1) < p.window || a < p.sinks);
  };
  auto all_seen_by_some = [&](int a, int n) {  // no key of [a, a + n) is unseen by every row
    const int b = a + n - 1;
    return b <= w.pos_hi && b < w.q.ctx && (p.window == 0 || w.pos_lo - a < p.window || b < p.sinks);
  };

  // Page ids of the item's j-th tile, lane b < 16 holding that of keys
  // [8 b, 8 b + 8); -1: no such page. Fetched a tile ahead of their use.
  auto fetch_ids = [&](int j) -> int {
    if (lane >= BN / 8 || j >= w.nkv) return -1;
    const int key = key0_of(j) + 8 * lane;
    if (key >= w.q.ctx) return -1;
    const int id = bt[key >> p.bs_log2];
    return id >= 0 && id < p.num_blocks ? id : -1;
  };

  // Register split, 384 threads x 168 at launch: 128 x 56 + 256 x 224 = 64,512
  // (with 200 the softmax spilled: one chunk of 8192 tokens, D 128, 229 us against
  // 222). e4m3: 512 x 128 at launch: 128 x (48 + 80) + 256 x 192 = 65,536.
  if (warp == 0) {
    // ------------------------------------------------------------- loads --
    reg_dealloc<FP8 ? 48 : 56>();
    if (lane == 0) {
      const int tokens = w.R / p.G;
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        if (w.nkv_t[t] == 0) continue;
        mbar_arrive_expect_tx(&q_full[t], KC * w.R * 128);
        for (int kc = 0; kc < KC; ++kc)
          tma_load_4d(sQ + (t * KC + kc) * CHUNK_BYTES, &tq, &q_full[t], kc * 64, 0, w.hk,
                      w.q.row0 + (w.c0 + t) * tokens);
      }
    }
    if constexpr (!FP8) {
      const int box = 1 << box_log2;          // rows per TMA box: a page, 128 of a larger one
      const int per_tile = BN >> box_log2;    // boxes per tile (at most 16): one lane each
      int edges = 0;
      int ids = fetch_ids(0);
      for (int j = 0; j < w.nkv; ++j) {
        const int s = j % NS;
        const int next = fetch_ids(j + 1);
        const int key0 = key0_of(j), key = key0 + lane * box, row = key & ((1 << p.bs_log2) - 1);
        int id = __shfl_sync(0xffffffffu, ids, (lane * box >> 3) & 15);
        if (lane < per_tile && !any_seen(key, box)) id = -1;
        // Eight-row groups of the cache; one past its end reads as zeros.
        const int at = id >= 0 ? (int)((((int64_t)id * p.Hkv + w.hk) << (p.bs_log2 - 3)) + (row >> 3))
                               : (int)(((int64_t)p.num_blocks * p.Hkv) << (p.bs_log2 - 3));
        const bool clean = all_seen_by_some(key0, BN);
        if (j >= NS && !mbar_wait_warp(&k_empty[s], ((j / NS) - 1) & 1, 0x501)) break;
        if (lane == 0) mbar_arrive_expect_tx(&k_full[s], L::TILE);
        __syncwarp();
        if (lane < per_tile)
          tma_load_4d(sK + s * L::TILE + lane * box * (KC * 128), &tk, &k_full[s], 0, 0, 0, at);
        if (j >= NS && !mbar_wait_warp(&v_empty[s], ((j / NS) - 1) & 1, 0x503)) break;
        if (lane == 0) mbar_arrive_expect_tx(clean ? &v_full[s] : edge, L::TILE);
        __syncwarp();
        if (lane < per_tile)
          tma_load_4d(sV + s * L::TILE + lane * box * (KC * 128), &tv, clean ? &v_full[s] : edge, 0, 0,
                      0, at);
        if (!clean) {
          if (!mbar_wait_warp(edge, edges & 1, 0x502)) break;
          ++edges;
          for (int r = lane; r < BN; r += 32)
            if (!seen_by_any(p, w.pos_lo, w.pos_hi, w.q.ctx, key0 + r))
              for (int kc = 0; kc < KC; ++kc)
                for (int c = 0; c < 8; ++c)
                  *reinterpret_cast<uint4*>(sV + s * L::TILE + ((r >> 3) * KC + kc) * ATOM + (r & 7) * 128 +
                                            c * 16) = make_uint4(0u, 0u, 0u, 0u);
          fence_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_full[s]);
        }
        ids = next;
      }
    } else {
      const int box = 1 << box_log2, per_tile = BN >> box_log2;
      // Scales of 8 keys a lane (0-15 of K, 16-31 of V), a tile ahead; their page
      // ids two.
      auto fetch_scales = [&](int j, int ids) -> uint2 {
        const int id = __shfl_sync(0xffffffffu, ids, lane & 15);
        if (id < 0) return make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
        const int key = key0_of(j) + 8 * (lane & 15);
        const int64_t cell = (((int64_t)id * p.Hkv + w.hk) << p.bs_log2) + (key & ((1 << p.bs_log2) - 1));
        return __ldg(reinterpret_cast<const uint2*>((lane < 16 ? p.k_scale : p.v_scale) + cell));
      };
      int ids = fetch_ids(0), ids1 = fetch_ids(1);
      uint2 sc = fetch_scales(0, ids);
      for (int j = 0; j < w.nkv; ++j) {
        const int ids2 = fetch_ids(j + 2);
        const uint2 sc1 = fetch_scales(j + 1, ids1);
        const int key = key0_of(j) + lane * box;
        int id = __shfl_sync(0xffffffffu, ids, (lane * box >> 3) & 15);
        if (lane < per_tile && !any_seen(key, box)) id = -1;
        // Rows of the cache; one past its end reads as zeros.
        const int at = (int)((((int64_t)(id >= 0 ? id : p.num_blocks) * p.Hkv + (id >= 0 ? w.hk : 0))
                              << p.bs_log2) + (id >= 0 ? key & ((1 << p.bs_log2) - 1) : 0));
        bool ok = true;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          if (j > 0 && !mbar_wait_warp(&raw_empty[kv], (j - 1) & 1, 0x504)) { ok = false; break; }
          if (lane >> 4 == kv) *reinterpret_cast<uint2*>(smem + L::SCALE_OFF + lane * 8) = sc;
          __syncwarp();
          if (lane == 0) mbar_arrive_expect_tx(&raw_full[kv], L::RAW);
          __syncwarp();
          if (lane < per_tile)
            tma_load_2d(smem + L::RAW_OFF + kv * L::RAW + lane * box * D, kv == 0 ? &tk : &tv,
                        &raw_full[kv], 0, at);
        }
        if (!ok) break;
        ids = ids1;
        ids1 = ids2;
        sc = sc1;
      }
    }
  } else if (warp == 1) {
    // --------------------------------------------------------- MMA issue --
    // The whole warp walks this path and its elected lane issues. A lane alone on
    // it computed every descriptor outside the uniform registers, which paced the
    // loop: one chunk of 8192 tokens, 16 heads of 128, took 240 us against 229
    // (e4m3 325 against 281).
    reg_dealloc<FP8 ? 48 : 56>();
    constexpr uint32_t IDESC_QK = idesc_f16(BM, BN, FMT, 0, 0);
    constexpr uint32_t IDESC_PV = idesc_f16(BM, D, FMT, 0, 1);
    const uint32_t q_lo = desc_lo(sQ, 16), k_lo = desc_lo(sK, 16), v_lo = desc_lo(sV, ATOM);
    auto issue_qk = [&](int t, int j) {
      const int s = j % NS;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t qo = (t * KC + kk / 4) * CHUNK_BYTES + (kk % 4) * 32;
        const uint32_t ko = (kk / 4) * ATOM + (kk % 4) * 32;
        mma_ss_warp(tmem + t * 128, desc(q_lo + (qo >> 4), desc_hi(ATOM)),
                    desc(k_lo + s * (L::TILE >> 4) + (ko >> 4), desc_hi(KC * ATOM)), IDESC_QK, kk > 0);
      }
      mma_commit_warp(&s_full[t]);
    };
    // PV over keys [64 h, 64 h + 64) of the tile; the second half commits pv_done.
    auto issue_pv_half = [&](int t, int j, int h) {
      const int s = j % NS;
#pragma unroll
      for (int k4 = 0; k4 < BN / 32; ++k4) {
        const int kk = h * (BN / 32) + k4;
        mma_ts_warp(tmem + 256 + t * 128, tmem + t * 128 + kk * 8,
                    desc(v_lo + s * (L::TILE >> 4) + kk * (2 * KC * ATOM >> 4), desc_hi(KC * ATOM)),
                    IDESC_PV, (j > 0 || kk > 0) ? 1u : 0u);
      }
      if (h == 1) mma_commit_warp(&pv_done[t]);
    };
    bool ok = true;
    for (int t = 0; t < TILES && ok; ++t)
      if (w.nkv_t[t] > 0 && !mbar_wait_warp(&q_full[t], 0, 0x511)) ok = false;
    if (ok && w.nkv > 0 && !mbar_wait_warp(&k_full[0], 0, 0x512)) ok = false;
    tc_fence_after();
    for (int t = 0; ok && t < TILES; ++t)
      if (w.nkv_t[t] > 0) issue_qk(t, 0);
    if (ok && w.nkv > 0) mma_commit_warp(&k_empty[0]);
    for (int j = 0; ok && j < w.nkv; ++j) {
      const int s = j % NS;
      if (!mbar_wait_warp(&v_full[s], (j / NS) & 1, 0x513)) { ok = false; break; }
      for (int t = 0; t < TILES; ++t) {
        if (j >= w.nkv_t[t]) continue;
        if (!mbar_wait_warp(&p_full[2 * t], j & 1, 0x514)) { ok = false; break; }
        tc_fence_after();
        issue_pv_half(t, j, 0);
        if (!mbar_wait_warp(&p_full[2 * t + 1], j & 1, 0x515)) { ok = false; break; }
        tc_fence_after();
        issue_pv_half(t, j, 1);
        if (j + 1 < w.nkv_t[t]) {
          // (Waited for once: by tile 0 where it visits these keys.)
          if ((t == 0 || j + 1 >= w.nkv_t[0]) &&
              !mbar_wait_warp(&k_full[(j + 1) % NS], ((j + 1) / NS) & 1, 0x516)) {
            ok = false;
            break;
          }
          tc_fence_after();
          issue_qk(t, j + 1);
        }
      }
      if (!ok) break;
      mma_commit_warp(&v_empty[s]);
      if (j + 1 < w.nkv) mma_commit_warp(&k_empty[(j + 1) % NS]);
    }
  } else if (warp < 4) {
    reg_dealloc<FP8 ? 48 : 56>();  // idle members of the first warpgroup
  } else if (warp < 12) {
    // ----------------------------------------------------------- softmax --
    reg_alloc<FP8 ? 192 : 224>();
    const int t = (warp >> 2) - 1;
    const int row = threadIdx.x - 128 * (t + 1);  // TMEM lane
    const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const float sl2 = p.scale_log2;
    const int nkv_t = t == 0 ? w.nkv_t[0] : w.nkv_t[1];
    const int pr = (w.c0 + t) * w.R + row;
    const bool mine = row < w.R && pr < w.pairs;
    const int pos = w.q.pos0 + pr / p.G;
    int tile_lo = 0, tile_hi = 0;
    if ((w.c0 + t) * w.R < w.pairs) tile_positions(p, w.q, w.c0 + t, w.R, tile_lo, tile_hi);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    int ids = fetch_ids(0);
    for (int j = 0; j < nkv_t; ++j) {
      const uint32_t have = __ballot_sync(0xffffffffu, ids >= 0);  // bit per 8 keys: page there
      ids = fetch_ids(j + 1);
      if (!mbar_wait_warp(&s_full[t], j & 1, 0x521)) { ok = false; break; }
      tc_fence_after();
      const int kv0 = key0_of(j), last = kv0 + BN - 1;
      const bool whole = last <= tile_lo && last < w.q.ctx && have == 0xffffu &&
                         (p.window == 0 || tile_hi - kv0 < p.window || last < p.sinks);
      // Visible columns as bits, 32 columns a word: below hi, from lo on (or a
      // sink, below sk), and in a page that is there.
      uint32_t bits[4];
      if (!whole) {
        const int hi = min(w.q.ctx, pos + 1) - kv0;
        const int lo = p.window > 0 ? pos - p.window + 1 - kv0 : 0;
        const int sk = p.window > 0 ? p.sinks - kv0 : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t pg = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b) pg |= (0u - ((have >> (4 * i + b)) & 1u)) & (0xffu << (8 * b));
          bits[i] = low_bits(hi - 32 * i) & (~low_bits(lo - 32 * i) | low_bits(sk - 32 * i)) & pg;
        }
      }
      // Scores of columns [32 i, 32 i + 32), hidden ones at -inf (after the wait).
      auto fetch = [&](int i, uint32_t (&x)[32]) { tmem_ld32(lane_addr + t * 128 + 32 * i, x); };
      auto hide = [&](int i, uint32_t (&x)[32]) {
#pragma unroll
        for (int cc = 0; cc < 32; ++cc)
          if (!((bits[i] >> cc) & 1)) x[cc] = __float_as_uint(-INFINITY);
      };
      uint32_t sr[4][32];
#pragma unroll
      for (int i = 0; i < 4; ++i) fetch(i, sr[i]);
      tmem_ld_wait();
      if (!whole) {
#pragma unroll
        for (int i = 0; i < 4; ++i) hide(i, sr[i]);
      }
      const float mx = row_max(sr);
      const float m_new = fmaxf(m, mx * sl2);
      float alpha = 1.f;
      const bool rescale = m_new > m + RESCALE_THRESHOLD;
      if (rescale) {
        alpha = ex2(m - m_new);
        m = m_new;
        l *= alpha;
      }
      const float m_use = (m == -INFINITY) ? 0.f : m;
      const float neg_m = FMT == 0 ? F16_LIFT - m_use : -m_use;
      float2 l2[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f),
                      make_float2(0.f, 0.f)};
      const float2 sl2_2 = make_float2(sl2, sl2), negm2 = make_float2(neg_m, neg_m);
      auto weigh = [&](const uint32_t (&x)[32], uint32_t* pk) {  // 32 scores to 16 packed pairs
#pragma unroll
        for (int cc = 0; cc < 16; ++cc) {
          const float2 y = __ffma2_rn(
              make_float2(__uint_as_float(x[2 * cc]), __uint_as_float(x[2 * cc + 1])), sl2_2, negm2);
          const float2 pp = make_float2(ex2(y.x), ex2(y.y));
          l2[cc & 3] = __fadd2_rn(l2[cc & 3], pp);
          pk[cc] = FMT == 1 ? pack_bf16(pp.x, pp.y) : pack_f16(pp.x, pp.y);
        }
      };
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t pk[32];
        weigh(sr[2 * h], pk);
        weigh(sr[2 * h + 1], pk + 16);
        tmem_st32(lane_addr + t * 128 + 32 * h, pk);
        // O is rescaled before the first half's PV accumulates into it; PV_t(j-1)
        // has completed: s_full(j) follows it in issue order.
        if (h == 0 && __any_sync(0xffffffffu, rescale && j > 0)) {
          const float a = (rescale && j > 0) ? alpha : 1.f;
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            uint32_t ov[32];
            tmem_ld32(lane_addr + 256 + t * 128 + 32 * i, ov);
            tmem_ld_wait();
#pragma unroll
            for (int cc = 0; cc < 32; ++cc) ov[cc] = __float_as_uint(__uint_as_float(ov[cc]) * a);
            tmem_st32(lane_addr + 256 + t * 128 + 32 * i, ov);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_full[2 * t + h]);
      }
      const float2 a2 = __fadd2_rn(__fadd2_rn(l2[0], l2[1]), __fadd2_rn(l2[2], l2[3]));
      l += a2.x + a2.y;
    }
    if (ok && nkv_t > 0) {
      if (!mbar_wait_warp(&pv_done[t], (nkv_t - 1) & 1, 0x523)) ok = false;
      tc_fence_after();
    }
    if (ok) {
      const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;  // NaN sums give NaN
      const bool none = l == 0.f;  // a row without keys: 0, whatever V holds
      const int tok = w.q.row0 + pr / p.G, h = w.hk * p.G + pr % p.G;
      const int64_t at = ((int64_t)tok * p.Hq + h) * p.P + w.chunk;
      uint8_t* orow = static_cast<uint8_t*>(p.o) +
                      2 * ((int64_t)tok * p.so_t + (int64_t)h * p.so_h);
      const bool st32 = (reinterpret_cast<uintptr_t>(orow) & 31) == 0;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        uint32_t ov[32];
        if (nkv_t > 0) {
          tmem_ld32(lane_addr + 256 + t * 128 + 32 * i, ov);
          tmem_ld_wait();
        }
#pragma unroll
        for (int cc = 0; cc < 32; ++cc)
          ov[cc] = none ? 0u : __float_as_uint(__uint_as_float(ov[cc]) * inv);
        if (mine && w.chunks > 1) {
#pragma unroll
          for (int v8 = 0; v8 < 4; ++v8) st_global_v8(p.part_o + at * D + 32 * i + 8 * v8, &ov[8 * v8]);
        } else if (mine) {
          uint32_t pk[16];
#pragma unroll
          for (int cc = 0; cc < 16; ++cc) {
            float a0 = __uint_as_float(ov[2 * cc]), a1 = __uint_as_float(ov[2 * cc + 1]);
            if constexpr (FP8 && FMT == 0) {  // P's rounding can lift O past fp16's largest value
              a0 = clamp_finite<T>(a0);
              a1 = clamp_finite<T>(a1);
            }
            pk[cc] = FMT == 1 ? pack_bf16(a0, a1) : pack_f16(a0, a1);
          }
          if (st32) {
#pragma unroll
            for (int v8 = 0; v8 < 2; ++v8) st_global_v8(orow + 64 * i + 32 * v8, &pk[8 * v8]);
          } else {
            uint4* dst = reinterpret_cast<uint4*>(orow + 64 * i);
#pragma unroll
            for (int v4 = 0; v4 < 4; ++v4)
              dst[v4] = make_uint4(pk[4 * v4], pk[4 * v4 + 1], pk[4 * v4 + 2], pk[4 * v4 + 3]);
          }
        }
        __syncwarp();
      }
      if (mine) {
        const float lse2 = none ? -INFINITY : m + log2f(l) - (FMT == 0 ? F16_LIFT : 0.f);
        if (w.chunks > 1)
          p.part_lse[at] = lse2;
        else if (p.lse != nullptr)
          p.lse[(int64_t)h * p.T + tok] = lse2 * 0.69314718055994531f;
      }
      tc_fence_before();
    }
  } else {
    // ----------------------------------------------------------- convert --
    reg_dealloc<80>();
    if constexpr (FP8) {
      constexpr int CPR = D / 16;           // 16-byte pieces of a cached row
      constexpr int RPP = 128 / CPR;        // rows per pass of the 128 threads
      constexpr int PASSES = BN / RPP;
      const int tid = threadIdx.x & 127, c = tid % CPR, r0 = tid / CPR;
      auto store = [&](int i, const uint4& raw16, int scale, auto plain, uint8_t* tile) {
        const int kc = c / 4, row = r0 + i * RPP;
        const uint32_t words[4] = {raw16.x, raw16.y, raw16.z, raw16.w};
        uint32_t o[8];
        // plain: the scale is an fp16, and no product leaves fp16's range (nor is its
        // byte one of e8m0's special ones).
        if constexpr (FMT == 0 && decltype(plain)::value) {
          const __half2 f = __half2half2(__float2half_rn(__uint_as_float((uint32_t)scale << 23)));
#pragma unroll
          for (int i2 = 0; i2 < 8; ++i2) {
            const uint32_t z = cvt_e4m3x2_f16x2((uint16_t)(words[i2 / 2] >> (16 * (i2 & 1))));
            const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&z), f);
            o[i2] = *reinterpret_cast<const uint32_t*>(&y);
          }
        } else if constexpr (decltype(plain)::value) {
          const uint16_t f = __half_as_ushort(__float2half_rn(__uint_as_float((uint32_t)scale << 23)));
#pragma unroll
          for (int i2 = 0; i2 < 8; ++i2) {
            const float2 y = mul_widen(cvt_e4m3x2_f16x2((uint16_t)(words[i2 / 2] >> (16 * (i2 & 1)))), f);
            o[i2] = pack_bf16(y.x, y.y);
          }
        } else {
          const float f = e8m0_to_float(scale);
#pragma unroll
          for (int i2 = 0; i2 < 8; ++i2) {
            const float2 y = __fmul2_rn(
                f16x2_to_float2(cvt_e4m3x2_f16x2((uint16_t)(words[i2 / 2] >> (16 * (i2 & 1))))),
                make_float2(f, f));
            if constexpr (FMT == 1) {
              o[i2] = pack_bf16(y.x, y.y);
            } else {  // a value lifted past fp16's range stays at its largest
              const __half2 top = __float2half2_rn(65504.f);
              const uint32_t z = pack_f16(y.x, y.y);
              const __half2 c2 =
                  __hmax2_nan(__hmin2_nan(*reinterpret_cast<const __half2*>(&z), top), __hneg2(top));
              o[i2] = *reinterpret_cast<const uint32_t*>(&c2);
            }
          }
        }
        uint8_t* base = tile + ((row >> 3) * KC + kc) * ATOM + (row & 7) * 128;
        // Halves in alternating order, so that 8 lanes of a row touch every bank once.
        const int first = (c >> 2) & 1, piece = (c & 3) * 2;
        const uint4 lo = make_uint4(o[0], o[1], o[2], o[3]), hi = make_uint4(o[4], o[5], o[6], o[7]);
        *reinterpret_cast<uint4*>(base + (((piece + first) ^ (row & 7)) << 4)) = first ? hi : lo;
        *reinterpret_cast<uint4*>(base + (((piece + 1 - first) ^ (row & 7)) << 4)) = first ? lo : hi;
      };
      bool ok = true;
      for (int j = 0; ok && j < w.nkv; ++j) {
        const int s = j % NS, key0 = key0_of(j);
        const bool clean = all_seen_by_some(key0, BN);
#pragma unroll 1
        for (int kv = 0; kv < 2; ++kv) {
          const uint8_t* raw = smem + L::RAW_OFF + kv * L::RAW;
          const uint8_t* scales = smem + L::SCALE_OFF + kv * BN;
          uint8_t* tile = smem + (kv ? L::V_OFF : L::K_OFF) + s * L::TILE;
          if (!mbar_wait_warp(&raw_full[kv], j & 1, 0x531)) { ok = false; break; }
          uint4 x[PASSES];
          int e[PASSES];
#pragma unroll
          for (int i = 0; i < PASSES; ++i) {
            x[i] = *reinterpret_cast<const uint4*>(raw + (r0 + i * RPP) * D + c * 16);
            e[i] = scales[r0 + i * RPP];
          }
          if (!clean) {
#pragma unroll
            for (int i = 0; i < PASSES; ++i)
              if (!seen_by_any(p, w.pos_lo, w.pos_hi, w.q.ctx, key0 + r0 + i * RPP)) {
                x[i] = make_uint4(0u, 0u, 0u, 0u);
                e[i] = 127;
              }
          }
          if (j >= NS && !mbar_wait_warp(kv ? &v_empty[s] : &k_empty[s], ((j / NS) - 1) & 1, 0x532)) {
            ok = false;
            break;
          }
          // Every scale between 2^-24 and 2^7 (448 2^7 is below 65504).
          bool plain = true;
#pragma unroll
          for (int i = 0; i < PASSES; ++i) plain = plain && e[i] >= 103 && e[i] <= 134;
          plain = __all_sync(0xffffffffu, plain);
          // One branch for the tile: a branch per pass kept the passes apart (fp16 over
          // e4m3, one chunk of 8192 tokens, D 128: 288 us against 252).
          if (plain) {
#pragma unroll
            for (int i = 0; i < PASSES; ++i) store(i, x[i], e[i], std::true_type{}, tile);
          } else {
#pragma unroll
            for (int i = 0; i < PASSES; ++i) store(i, x[i], e[i], std::false_type{}, tile);
          }
          fence_async_shared();
          __syncwarp();
          // The raw tile is released once its values have been used: an arrival does
          // not wait for shared-memory loads still under way, and the next tile's
          // copy could overtake them.
          if (lane == 0) {
            mbar_arrive(kv ? &v_full[s] : &k_full[s]);
            mbar_arrive(&raw_empty[kv]);
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// q as [T, Hkv, G, D]: boxes of 64 columns, G heads, the tokens of one tile.
static int make_q_map(CUtensorMap* map, const Params& p, int dtype) {
  EncodeTiledFn enc = get_encode_tiled();
  if (!enc) {
    set_error("cuTensorMapEncodeTiled unavailable (no CUDA driver?)");
    return LSB_ERR_CUDA;
  }
  cuuint64_t dims[4] = {(cuuint64_t)p.D, (cuuint64_t)p.G, (cuuint64_t)p.Hkv, (cuuint64_t)p.T};
  // A dim of one has no stride of its own: any multiple of 16 bytes will do.
  const int64_t sg = p.Hq > 1 ? p.sq_h : p.D, st = p.T > 1 ? p.sq_t : p.D;
  cuuint64_t strides[3] = {(cuuint64_t)(sg * 2), (cuuint64_t)(sg * p.G * 2), (cuuint64_t)(st * 2)};
  cuuint32_t box[4] = {64, (cuuint32_t)p.G, 1, (cuuint32_t)(BM / p.G)};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = enc(map, dtype == LSB_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                   4, const_cast<void*>(p.q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed (%d)", (int)r);
    return LSB_ERR_CUDA;
  }
  return LSB_OK;
}

// The cache as [rows / 8, D / 64, 8, 64]: a box is `groups` row groups of one page.
static int make_cache_map(CUtensorMap* map, const void* base, const Params& p, int dtype, int groups) {
  EncodeTiledFn enc = get_encode_tiled();
  if (!enc) {
    set_error("cuTensorMapEncodeTiled unavailable (no CUDA driver?)");
    return LSB_ERR_CUDA;
  }
  const int64_t rows8 = ((int64_t)p.num_blocks * p.Hkv) << (p.bs_log2 - 3);
  cuuint64_t dims[4] = {64, 8, (cuuint64_t)(p.D / 64), (cuuint64_t)rows8};
  cuuint64_t strides[3] = {(cuuint64_t)p.D * 2, 128, (cuuint64_t)p.D * 16};
  cuuint32_t box[4] = {64, 8, (cuuint32_t)(p.D / 64), (cuuint32_t)groups};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = enc(map, dtype == LSB_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                   4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed (%d)", (int)r);
    return LSB_ERR_CUDA;
  }
  return LSB_OK;
}

// An e4m3 cache as [rows, D] bytes: a box is the rows of a page.
static int make_raw_map(CUtensorMap* map, const void* base, const Params& p, int rows_per_box) {
  EncodeTiledFn enc = get_encode_tiled();
  if (!enc) {
    set_error("cuTensorMapEncodeTiled unavailable (no CUDA driver?)");
    return LSB_ERR_CUDA;
  }
  cuuint64_t dims[2] = {(cuuint64_t)p.D, (cuuint64_t)(((int64_t)p.num_blocks * p.Hkv) << p.bs_log2)};
  cuuint64_t strides[1] = {(cuuint64_t)p.D};
  cuuint32_t box[2] = {(cuuint32_t)p.D, (cuuint32_t)rows_per_box};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed (%d)", (int)r);
    return LSB_ERR_CUDA;
  }
  return LSB_OK;
}

template <int D, int FMT, bool FP8>
static int launch(const Params& p, int dtype, cudaStream_t st) {
  CUtensorMap mq, mk, mv;
  int rc = make_q_map(&mq, p, dtype);
  const int box_log2 = std::min(p.bs_log2, 7);
  if (!FP8) {
    if (!rc) rc = make_cache_map(&mk, p.k_cache, p, dtype, 1 << (box_log2 - 3));
    if (!rc) rc = make_cache_map(&mv, p.v_cache, p, dtype, 1 << (box_log2 - 3));
  } else {
    if (!rc) rc = make_raw_map(&mk, p.k_cache, p, 1 << box_log2);
    if (!rc) rc = make_raw_map(&mv, p.v_cache, p, 1 << box_log2);
  }
  if (rc) return rc;
  auto kern = paged_chunk_kernel<D, FMT, FP8>;
  static SmemLimit limit;
  if (int rc_ = limit.ensure(kern, Smem<D, FP8>::ALLOC, "paged_attn smem attribute")) return rc_;
  const int64_t R = (int64_t)(BM / p.G * p.G) * TILES;
  const dim3 grid((unsigned)(p.Hkv * p.P), (unsigned)(((int64_t)p.max_q * p.G + R - 1) / R), (unsigned)p.S);
  LSB_CUDA_OK(launch_kernel(kern, grid, dim3(FP8 ? 512 : 384), Smem<D, FP8>::ALLOC, st, mq, mk, mv, p, box_log2),
              "paged_attn");
  return LSB_OK;
}

}  // namespace tc

bool tc_eligible(const Params& p, int dtype, bool kv_fp8) {
  if (dtype != LSB_DTYPE_BF16 && dtype != LSB_DTYPE_F16) return false;
  if ((p.D != 64 && p.D != 128) || p.bs_log2 < 3 || p.G > tc::BM) return false;
  if (!(p.scale_log2 > 0.f)) return false;  // the running maximum is taken before the scale
  // TMA: 16-byte aligned bases and strides; rows of o are written 16 bytes at a time.
  if (!aligned16(p.q) || p.sq_t % 8 != 0 || p.sq_h % 8 != 0 || p.sq_t < 0 || p.sq_h < 0) return false;
  if (!aligned16(p.o) || p.so_t % 8 != 0 || p.so_h % 8 != 0) return false;
  if (!aligned16(p.k_cache) || !aligned16(p.v_cache)) return false;
  if (p.T > 1 && p.sq_t == 0) return false;
  if (p.Hq > 1 && p.sq_h == 0) return false;
  // The cache's 8-row groups (e4m3: rows) are a 32-bit TMA coordinate; scales are
  // read 8 keys at a time.
  if ((((int64_t)p.num_blocks * p.Hkv) << (kv_fp8 ? p.bs_log2 : p.bs_log2 - 3)) > 0x7fffffff) return false;
  if (kv_fp8 && ((reinterpret_cast<uintptr_t>(p.k_scale) | reinterpret_cast<uintptr_t>(p.v_scale)) & 7))
    return false;
  const int64_t R = (int64_t)(tc::BM / p.G * p.G) * tc::TILES;
  return ((int64_t)p.max_q * p.G + R - 1) / R <= 65535 && (int64_t)p.Hkv * p.P <= 0x7fffffff;
}

int launch_tc(const Params& p, int dtype, bool kv_fp8, cudaStream_t st) {
  const bool bf = dtype == LSB_DTYPE_BF16;
  if (p.D == 128) {
    if (kv_fp8) return bf ? tc::launch<128, 1, true>(p, dtype, st) : tc::launch<128, 0, true>(p, dtype, st);
    return bf ? tc::launch<128, 1, false>(p, dtype, st) : tc::launch<128, 0, false>(p, dtype, st);
  }
  if (kv_fp8) return bf ? tc::launch<64, 1, true>(p, dtype, st) : tc::launch<64, 0, true>(p, dtype, st);
  return bf ? tc::launch<64, 1, false>(p, dtype, st) : tc::launch<64, 0, false>(p, dtype, st);
}

}  // namespace pa

int paged_attn_tc_device_error(bool reset) { return sm100::tu_device_error(reset); }

}  // namespace lsb
