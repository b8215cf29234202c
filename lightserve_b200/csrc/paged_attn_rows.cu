// Paged attention for a few rows per sequence (decode, drafted tokens): the
// cache is read once at HBM speed, the arithmetic rides along on mma.sync.
//
// One CTA: a query tile of 8 NH pairs (row, head of the group) of one
// (sequence, cache head) and one chunk of its keys; its 4 warps take groups of
// 16 keys (e4m3: 32) in turn and merge at the end. Bound by HBM for a 16-bit
// cache; over e4m3 by latency (65% of the DRAM rate, 43% of the issue slots, 12
// warps an SM at 151 registers): half the bytes a key, the same number of MMAs,
// 16 m16n8k16 per 16 keys and 8 pairs. The warp-level MMA is the right size
// here: tcgen05's 128-row tiles would hold one row of use per key read.
// Measured: 64 sequences, 16 heads of 128, 512-4096 keys, e4m3 114 us (5.2 TB/s);
// 4096 keys each, 16-bit, 312 us (6.9 TB/s with what L2 keeps), e4m3 196 (5.5).
//
// Both products keep the cache on the MMA's 16-row side and the pairs on its
// 8-column side, so a single query head wastes 7 of 8 columns and nothing else:
//  * S^T = K Q^T (16 keys x pairs): lane (g, t) = (lane / 4, lane % 4) reads
//    16-byte runs of the rows of keys g and 8 + g at dims (4 i + t) EK. A
//    contraction's index order is free as long as both operands agree on it, so
//    the runs' 4-element pieces serve as its slots of consecutive k steps as they
//    are; Q is laid out by the same rule, once.
//  * O^T += V^T P^T (dims x pairs): P^T's fragment is S^T's, each 8 x 8 quarter
//    transposed in registers (movmatrix). Lane (g, t) reads V of keys 2t, 2t + 1,
//    8 + 2t and 9 + 2t at dims (8 i + g) EV and interleaves key pairs with byte
//    permutes; its dims are rows g and 8 + g of the m-tiles in turn.
//
// Each warp streams its groups through a ring of its own in shared memory, a TMA
// box per page, tensor and group issued by one lane (copying 16 bytes a lane
// with cp.async took a third of all instructions). The boxes' swizzle and the
// order in which a group's keys are the MMA's rows (sigma) make both kinds of
// read touch every bank once.
//
// e4m3 cache: bytes convert to fp16 in one instruction per pair (exactly; the
// MMAs run in fp16), unscaled. K's power-of-two scale multiplies the score. V's
// is added to the score as an exponent: w_j = 2^(x_j + e_j - m'), with a running
// maximum m' of x + e of its own, so weights stay near 1 whatever the scales,
// beside p_j = 2^(x_j - m) for the denominator. A bf16 q is scaled by a power
// of two per row into fp16's range (exact down to 2^-28 of the row's largest
// value; below that the error is under 2^-39 of it).
//
// The running maximum is raised only when a score exceeds it by 2^8 (a vote
// per group instead of shuffles and a rescale). Weights of an fp16 P carry 2^7
// (paged_attn.cuh): rounding P to 16 bits is off by half a step of the operand
// type relative to each weight, as in the framework's other tensor-core attention
// kernels (the plain decode kernel, on the CUDA cores, keeps P in fp32).
#include "paged_attn.cuh"
#include "sm100.cuh"
#include "tma_host.cuh"

#include <type_traits>

namespace lsb {
namespace pa {

namespace rows {

constexpr int WARPS = 4;
constexpr float RAISE = 8.f;   // log2: how far a score may exceed the reference maximum

// (volatile: a group's MMAs, and with them the uses of its loads, stay ahead of
// the next group's wait and copies.)
template <bool F16>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The transpose of an 8 x 8 tile of 16-bit values held two to a lane.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// N words from shared memory (8 or 16 bytes).
template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const void* p) {
  static_assert(N == 2 || N == 4, "8 or 16 bytes");
  if constexpr (N == 4) {
    const uint4 x = *static_cast<const uint4*>(p);
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
  } else {
    const uint2 x = *static_cast<const uint2*>(p);
    w[0] = x.x; w[1] = x.y;
  }
}

// Key of a half group that is the MMA's row r, such that the rows read by eight
// consecutive lanes have swizzle patterns that do not collide.
__device__ __forceinline__ int sigma(int r) { return r ^ ((r & 1) << 2); }

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(sm100::smem_u32(bar)), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1,
                                            int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(sm100::smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

template <bool FP8, int D>
struct Shape {
  static constexpr int EB = FP8 ? 1 : 2;           // bytes per cached element
  static constexpr int TK = rows_tk(FP8);          // keys per group
  static constexpr int NU = TK / 16;               // MMA row blocks of a group
  static constexpr int GR = TK / 8;                // runs of 8 keys, each within a page
  static constexpr int EK = 16 / EB;               // K elements per lane and load
  static constexpr int NK = D / (4 * EK);          // K loads per key and lane
  static constexpr int EV = FP8 ? D / 8 : 8;       // V elements per lane and load
  static constexpr int NV = D / (8 * EV);          // V loads per key and lane
  static constexpr int WV = EV * EB / 4;           // words per V load
  static constexpr int STEPS = D / 16;             // k steps of S^T
  static constexpr int MT = D / 16;                // m-tiles of O^T
  static constexpr int CPR = D * EB / 16;          // 16-byte pieces of a row: 4, 8 or 16
  static constexpr int TILE = TK * CPR * 16;       // bytes of a group's K (and V)
  static constexpr int STAGE = 2 * TILE;
  // Groups in flight per warp and CTAs per SM (registers): 96 to 196 KB of ring
  // an SM. e4m3, D 64, one block of pairs: 5 CTAs 78 us, 3 CTAs 86 (64 sequences,
  // 16 heads, 512-4096 keys).
  static constexpr int STAGES = FP8 ? 2 : (D == 64 ? 4 : 3);
  static constexpr int ctas(int nh) {
    return FP8 ? (D == 64 ? (nh == 1 ? 5 : 3) : (nh == 3 ? 2 : 3)) : (D == 64 ? 3 : 2);
  }
  // Byte offset of 16-byte piece c of key k's row in its tile, as the boxes of
  // up to 16 rows and their swizzle leave it (256-byte rows come in two halves
  // of 128).
  static __device__ __forceinline__ int at(int k, int c) {
    if constexpr (CPR == 4) return k * 64 + ((c ^ ((k >> 1) & 3)) << 4);
    return (k >> 4) * (CPR * 256) + (c >> 3) * 2048 + (k & 15) * 128 + (((c & 7) ^ (k & 7)) << 4);
  }
};

// Dynamic shared memory of a CTA: the rings, which the merge reuses.
template <bool FP8, int D, int NH>
constexpr int smem_bytes() {
  const int ring = WARPS * Shape<FP8, D>::STAGES * Shape<FP8, D>::STAGE;
  const int merge = WARPS * 8 * NH * (D + 4 + 3) * 4;
  return (ring > merge ? ring : merge) + 1024;  // slack for 1024-byte alignment
}

template <typename T, bool FP8, int D, int NH, bool ONE>
__global__ void __launch_bounds__(WARPS * 32, (Shape<FP8, D>::ctas(NH)))
paged_rows_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                  const Params p) {
  if (threadIdx.x == 0) {
    sm100::prefetch_tmap(&tk);
    sm100::prefetch_tmap(&tv);
  }
  allow_dependents();
  wait_prerequisites();
  using S = Shape<FP8, D>;
  constexpr bool F16 = FP8 || std::is_same<T, __half>::value;  // MMA operand type
  constexpr float LIFT = F16 ? F16_LIFT : 0.f;                 // log2: factor on every weight
  // NE: of a lane's pairs 8 h + 2 t and + 1, those that can be in use (ONE: the
  // call has one pair per cache head, plain decode).
  constexpr int R = 8 * NH, TK = S::TK, NU = S::NU, NE = ONE ? 1 : 2;
  static_assert(!ONE || NH == 1, "one pair fits one block");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (sm100::smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ uint64_t bars[WARPS][S::STAGES];  // a group's boxes have arrived

  const int chunk = blockIdx.x % p.P, hk = blockIdx.x / p.P, tile = blockIdx.y, s = blockIdx.z;
  const Seq q = load_seq(p, s);
  const int pairs = q.n * p.G;
  if (tile * R >= pairs) return;
  int pos_lo, pos_hi;
  tile_positions(p, q, tile, R, pos_lo, pos_hi);
  const KeySpan span(p, q, pos_lo, pos_hi, TK);
  const int tiles = span.count(), per = p.chunk / TK;
  const int chunks = chunks_of(p, tiles, TK);
  if (chunk >= chunks) return;
  const int v0 = chunk * per, v1 = chunk + 1 == chunks ? tiles : min(tiles, v0 + per);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int32_t* bt = p.block_tables + (int64_t)s * p.max_blocks;
  const int bs = 1 << p.bs_log2;

  // ------------------------------------------------------------- loads ----
  // Page ids of the next BATCH of this warp's groups from v on, one run of 8 keys
  // per lane; -1: no such page.
  constexpr int BATCH = 32 / S::GR;
  auto fetch_ids = [&](int v) -> int {
    const int vv = v + lane / S::GR * WARPS;
    if (vv >= v1) return -1;
    const int tok = span.tile(vv) * TK + 8 * (lane % S::GR);
    if (tok >= q.ctx) return -1;
    const int id = bt[tok >> p.bs_log2];
    return id >= 0 && id < p.num_blocks ? id : -1;
  };
  uint8_t* ring = smem + warp * (S::STAGES * S::STAGE);
  uint64_t* full = bars[warp];
  if (lane == 0) {
    for (int i = 0; i < S::STAGES; ++i) sm100::mbar_init(&full[i], 1);
    sm100::fence_barrier_init();
  }
  __syncwarp();
  // Whether every pair sees all TK keys at tok0 (pages apart).
  auto all_seen = [&](int tok0) -> bool {
    const int last = tok0 + TK - 1;
    return last <= pos_lo && last < q.ctx &&
           (p.window == 0 || pos_hi - tok0 < p.window || last < p.sinks);
  };
  // Copies the group at keys [tok0, tok0 + TK) into a stage; `id` holds, in lanes
  // base, base + 1, ..., the page of each run of 8 keys. A lane per box; rows past
  // the cache arrive as zeros: missing pages.
  const int box = min(16, bs);  // rows of a box
  const int none = (int)(((int64_t)p.num_blocks * p.Hkv) << p.bs_log2);
  auto copy_group = [&](int stage, int tok0, int id, int base) {
    uint64_t* bar = &full[stage];
    const int r = lane * box;  // this lane's first row
    const int mine_id = __shfl_sync(0xffffffffu, id, base + (r >> 3) % S::GR);
    if (lane == 0) sm100::mbar_arrive_expect_tx(bar, S::STAGE);
    __syncwarp();
    if (r >= TK) return;
    const uint32_t dst = sm100::smem_u32(ring + stage * S::STAGE) +
                         (S::CPR == 16 ? (r >> 4) * 4096 + (r & 15) * 128 : r * (S::CPR * 16));
    const int row =
        mine_id >= 0 ? (int)(((int64_t)mine_id * p.Hkv + hk) << p.bs_log2) + ((tok0 + r) & (bs - 1)) : none;
    if constexpr (S::CPR == 16) {  // both halves of 16 rows, or each half of 8
      for (int z = 0; z < (box == 16 ? 1 : 2); ++z) {
        tma_load_3d(dst + z * 2048, &tk, bar, 0, row, z);
        tma_load_3d(dst + z * 2048 + S::TILE, &tv, bar, 0, row, z);
      }
    } else {
      tma_load_2d(dst, &tk, bar, 0, row);
      tma_load_2d(dst + S::TILE, &tv, bar, 0, row);
    }
  };
  // e4m3: this lane's scale bytes of the group, of K (low) and V, key lane;
  // 127 (a scale of 1) where there is no page.
  auto fetch_scales = [&](int tok0, int id, int base) -> int {
    const int my = __shfl_sync(0xffffffffu, id, base + (lane >> 3) % S::GR);
    if (my < 0) return 127 | 127 << 8;
    const int64_t cell = (((int64_t)my * p.Hkv + hk) << p.bs_log2) + ((tok0 + lane) & (bs - 1));
    return p.k_scale[cell] | p.v_scale[cell] << 8;
  };

  // Group n of this warp is v0 + warp + n WARPS and sits in stage n % STAGES.
  constexpr int AHEAD = S::STAGES - 1;
  const int first = v0 + warp;
  const int mine = v1 > first ? (v1 - first + WARPS - 1) / WARPS : 0;
  int near = fetch_ids(first), far = fetch_ids(first + BATCH * WARPS);
  int scale_of[AHEAD + 1];  // scale bytes of the groups in flight
  auto copy_next = [&](int n) -> uint32_t {  // called for n = 0, 1, 2, ... in turn
    if (n > 0 && n % BATCH == 0) {
      near = far;
      far = fetch_ids(first + (n + BATCH) * WARPS);
    }
    const int base = n % BATCH * S::GR;
    if (n < mine) {
      const int tok0 = span.tile(first + n * WARPS) * TK;
      copy_group(n % S::STAGES, tok0, near, base);
      if constexpr (FP8) scale_of[AHEAD] = fetch_scales(tok0, near, base);
    }
    return __ballot_sync(0xffffffffu, near >= 0) >> base & ((1u << S::GR) - 1u);
  };
  // Which runs of 8 keys have a page, GR bits per group in flight.
  uint32_t there = 0;
#pragma unroll
  for (int n = 0; n < AHEAD; ++n) {
    there |= copy_next(n) << (S::GR * n);
    if constexpr (FP8) scale_of[n] = scale_of[AHEAD];
  }

  // ---------------------------------------------------------------- Q ----
  // B fragments: pair 8 h + g of the tile, its 4-element piece per k step.
  uint32_t qb[NH][S::STEPS][2];
  // Of pairs 8 h + 2 t and 8 h + 2 t + 1, whose scores this lane holds: the
  // score's factor (scale log2(e), and the row's power of two) and position.
  float fac[NH][NE];
  int pos[NH][NE];
#pragma unroll
  for (int h = 0; h < NH; ++h) {
    const int pr = tile * R + h * 8 + g;
    const bool in = pr < pairs;
    const T* row = static_cast<const T*>(p.q) + (int64_t)(q.row0 + (in ? pr / p.G : 0)) * p.sq_t +
                   (int64_t)(hk * p.G + (in ? pr % p.G : 0)) * p.sq_h;
    uint2 raw[S::STEPS];
#pragma unroll
    for (int st = 0; st < S::STEPS; ++st) {
      const int i = st / (S::EK / 4), w = st % (S::EK / 4);
      raw[st] = in ? *reinterpret_cast<const uint2*>(row + (4 * i + t) * S::EK + 4 * w)
                   : make_uint2(0u, 0u);
    }
    float f = p.scale_log2;
    if constexpr (FP8 && std::is_same<T, __nv_bfloat16>::value) {
      float amax = 0.f;
#pragma unroll
      for (int st = 0; st < S::STEPS; ++st) {
        const T* x = reinterpret_cast<const T*>(&raw[st]);
#pragma unroll
        for (int e = 0; e < 4; ++e) amax = fmaxf(amax, finite_abs(to_f(x[e])));
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // The row's largest value goes to [2^14, 2^15); x is its biased exponent,
      // held where 2^(x - 141) and its inverse are normal.
      const int x = min(max((int)(__float_as_uint(amax) >> 23), 16), 254);
      const float down = __uint_as_float((uint32_t)(268 - x) << 23);  // 2^(141 - x)
      f *= __uint_as_float((uint32_t)(x - 14) << 23);                 // 2^(x - 141)
#pragma unroll
      for (int st = 0; st < S::STEPS; ++st) {
        const T* y = reinterpret_cast<const T*>(&raw[st]);
        qb[h][st][0] = sm100::pack_f16(to_f(y[0]) * down, to_f(y[1]) * down);
        qb[h][st][1] = sm100::pack_f16(to_f(y[2]) * down, to_f(y[3]) * down);
      }
    } else {
#pragma unroll
      for (int st = 0; st < S::STEPS; ++st) {
        qb[h][st][0] = raw[st].x;
        qb[h][st][1] = raw[st].y;
      }
    }
#pragma unroll
    for (int e = 0; e < NE; ++e) {  // lane 4 (2 t + e) holds pair 8 h + 2 t + e
      fac[h][e] = __shfl_sync(0xffffffffu, f, 4 * (2 * t + e));
      const int pe = tile * R + h * 8 + 2 * t + e;
      pos[h][e] = pe < pairs ? q.pos0 + pe / p.G : -1;  // position -1 sees nothing
    }
  }

  // ----------------------------------------------------------- compute ----
  // Running maxima m (of scores) and mw (of scores + V exponents), held as the
  // thresholds that raise them; sums and outputs are relative to them.
  float m[NH][NE], mw[NH][NE], l[NH][NE], acc[NH][S::MT][4];
#pragma unroll
  for (int h = 0; h < NH; ++h) {
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      m[h][e] = mw[h][e] = -INFINITY;
      l[h][e] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < S::MT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[h][j][e] = 0.f;
  }

  // S^T of the group: sc[h][u][2 n + e] = key 16 u + 8 n + sigma(g), pair
  // 8 h + 2 t + e.
  auto scores = [&](const uint8_t* kt, float (&sc)[NH][NU][4]) {
    float odd[NH][NU][4];  // odd k steps: half as long a chain of MMAs
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[h][u][e] = odd[h][u][e] = 0.f;
#pragma unroll
    for (int i = 0; i < S::NK; ++i) {
      uint32_t k[NU][2][4];
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int n = 0; n < 2; ++n) load_words(k[u][n], kt + S::at(16 * u + 8 * n + sigma(g), 4 * i + t));
#pragma unroll
      for (int w = 0; w < S::EK / 4; ++w) {
        const int st = i * (S::EK / 4) + w;
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          uint32_t a[4];  // keys g, 8 + g; then their second halves of the step
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            if constexpr (FP8) {
              a[n] = cvt_e4m3x2_f16x2((uint16_t)(k[u][n][w] & 0xffff));
              a[2 + n] = cvt_e4m3x2_f16x2((uint16_t)(k[u][n][w] >> 16));
            } else {
              a[n] = k[u][n][2 * w];
              a[2 + n] = k[u][n][2 * w + 1];
            }
          }
#pragma unroll
          for (int h = 0; h < NH; ++h)
            mma16816<F16>(st % 2 == 0 ? sc[h][u] : odd[h][u], a[0], a[1], a[2], a[3], qb[h][st][0],
                          qb[h][st][1]);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[h][u][e] += odd[h][u][e];
  };

  // Weights of the group's keys as B fragments of O^T: pb[h][u][n] = pair 8 h + g,
  // rows 16 u + 8 n + 2 t and + 1. Scores go to log2 units, to -inf for keys that
  // a row does not see.
  auto weights = [&](int scale, float (&sc)[NH][NU][4], int tok0, uint32_t pages,
                     uint32_t (&pb)[NH][NU][2]) {
    float ev[NU][2];
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        float f = 1.f, bad = 0.f;
        ev[u][n] = 0.f;
        if constexpr (FP8) {
          const int b = __shfl_sync(0xffffffffu, scale, 16 * u + 8 * n + sigma(g));
          f = __uint_as_float((uint32_t)(b & 0xff) << 23);  // 255, e8m0's NaN, gives infinity here
          bad = f - f;                                      // and NaN here
          ev[u][n] = (b >> 8) == 255 ? __int_as_float(0x7fc00000)
                                     : __uint_as_float(0x4b000000u | (b >> 8)) - (8388608.f + 127.f);
        }
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
          for (int e = 0; e < NE; ++e)
            sc[h][u][2 * n + e] = FP8 ? fmaf(sc[h][u][2 * n + e] * fac[h][e], f, bad)
                                      : sc[h][u][2 * n + e] * fac[h][e];
      }
    if (pages != (1u << S::GR) - 1u || !all_seen(tok0)) {
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int j = tok0 + 16 * u + 8 * n + sigma(g);
          const bool page = (pages >> (2 * u + n)) & 1;
#pragma unroll
          for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int e = 0; e < NE; ++e)
              if (!page || !sees(p, pos[h][e], q.ctx, j)) sc[h][u][2 * n + e] = -INFINITY;
          if (!page || !seen_by_any(p, pos_lo, pos_hi, q.ctx, j)) ev[u][n] = 0.f;
        }
    }
    bool raise = false;
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < NE; ++e) {
            raise |= sc[h][u][2 * n + e] > m[h][e] + RAISE;
            if constexpr (FP8) raise |= sc[h][u][2 * n + e] + ev[u][n] > mw[h][e] + RAISE;
          }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          float a = m[h][e], b = mw[h][e];
#pragma unroll
          for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              a = fmaxf(a, sc[h][u][2 * n + e]);
              if constexpr (FP8) b = fmaxf(b, sc[h][u][2 * n + e] + ev[u][n]);
            }
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
            if constexpr (FP8) b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, o));
          }
          if constexpr (!FP8) b = a;
          const float ra = exp2f(m[h][e] - (a == -INFINITY ? 0.f : a));
          const float rb = exp2f(mw[h][e] - (b == -INFINITY ? 0.f : b));
          m[h][e] = a;
          mw[h][e] = b;
          l[h][e] *= ra;
#pragma unroll
          for (int j = 0; j < S::MT; ++j) {
            acc[h][j][e] *= rb;
            acc[h][j][2 + e] *= rb;
          }
        }
    }
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      float mm[NE], mmw[NE];
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        mm[e] = m[h][e] == -INFINITY ? 0.f : m[h][e] - LIFT;
        mmw[e] = mw[h][e] == -INFINITY ? 0.f : mw[h][e] - LIFT;
      }
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float x0 = sc[h][u][2 * n], x1 = sc[h][u][2 * n + 1];
          const float p0 = sm100::ex2(x0 - mm[0]), p1 = ONE ? 0.f : sm100::ex2(x1 - mm[NE - 1]);
          l[h][0] += p0;
          if constexpr (!ONE) l[h][NE - 1] += p1;
          uint32_t w;
          if constexpr (FP8)
            w = sm100::pack_f16(sm100::ex2(x0 + (ev[u][n] - mmw[0])),
                                ONE ? 0.f : sm100::ex2(x1 + (ev[u][n] - mmw[NE - 1])));
          else
            w = F16 ? sm100::pack_f16(p0, p1) : sm100::pack_bf16(p0, p1);
          pb[h][u][n] = transpose8x8(w);
        }
    }
  };

  auto weigh_v = [&](const uint8_t* vt, const uint32_t (&pb)[NH][NU][2]) {
#pragma unroll
    for (int ui = 0; ui < NU * S::NV; ++ui) {
      const int u = ui / S::NV, i = ui % S::NV;
      uint32_t vw[4][S::WV];  // the keys of rows 2t, 2t + 1, 8 + 2t, 9 + 2t
      const int byte = (8 * i + g) * (S::EV * S::EB);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        load_words(vw[e], vt + S::at(16 * u + (e >> 1) * 8 + sigma(2 * t + (e & 1)), byte / 16) + byte % 16);
      // m-tile j's rows g and 8 + g are dims 2 j' and 2 j' + 1 of the lane's run.
#pragma unroll
      for (int w = 0; w < S::WV; ++w) {
        const uint32_t a = vw[0][w], b = vw[1][w], c = vw[2][w], d = vw[3][w];
        if constexpr (FP8) {
          const int j = (i * S::EV + 4 * w) / 2;
          const uint32_t lo0 = __byte_perm(a, b, 0x5140), lo1 = __byte_perm(c, d, 0x5140);
          const uint32_t hi0 = __byte_perm(a, b, 0x7362), hi1 = __byte_perm(c, d, 0x7362);
          const uint32_t l0 = cvt_e4m3x2_f16x2((uint16_t)(lo0 & 0xffff));
          const uint32_t l1 = cvt_e4m3x2_f16x2((uint16_t)(lo0 >> 16));
          const uint32_t l2 = cvt_e4m3x2_f16x2((uint16_t)(lo1 & 0xffff));
          const uint32_t l3 = cvt_e4m3x2_f16x2((uint16_t)(lo1 >> 16));
          const uint32_t h0 = cvt_e4m3x2_f16x2((uint16_t)(hi0 & 0xffff));
          const uint32_t h1 = cvt_e4m3x2_f16x2((uint16_t)(hi0 >> 16));
          const uint32_t h2 = cvt_e4m3x2_f16x2((uint16_t)(hi1 & 0xffff));
          const uint32_t h3 = cvt_e4m3x2_f16x2((uint16_t)(hi1 >> 16));
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            mma16816<F16>(acc[h][j], l0, l1, l2, l3, pb[h][u][0], pb[h][u][1]);
            mma16816<F16>(acc[h][j + 1], h0, h1, h2, h3, pb[h][u][0], pb[h][u][1]);
          }
        } else {
          const int j = (i * S::EV + 2 * w) / 2;
          const uint32_t x0 = __byte_perm(a, b, 0x5410), x1 = __byte_perm(a, b, 0x7632);
          const uint32_t x2 = __byte_perm(c, d, 0x5410), x3 = __byte_perm(c, d, 0x7632);
#pragma unroll
          for (int h = 0; h < NH; ++h)
            mma16816<F16>(acc[h][j], x0, x1, x2, x3, pb[h][u][0], pb[h][u][1]);
        }
      }
    }
  };

  for (int n = 0; n < mine; ++n) {
    const int tok0 = span.tile(first + n * WARPS) * TK;
    if (!sm100::mbar_wait_warp(&full[n % S::STAGES], (n / S::STAGES) & 1, 0x601)) {
      // The error word is set; no copy may be in flight when the rings are reused.
      for (int i = n; i < min(mine, n + AHEAD); ++i)
        sm100::mbar_wait_warp(&full[i % S::STAGES], (i / S::STAGES) & 1, 0x601);
      break;
    }
    // The next boxes go where group n - 1 was, by another proxy than the one
    // that read (and, at a span's ends, zeroed) it. The reads are plain loads, for
    // which a vote does not wait: each lane's fence orders them before the boxes,
    // which the warp issues behind a __syncwarp. (No cost measured.)
    sm100::fence_async_shared();
    there |= copy_next(n + AHEAD) << (S::GR * AHEAD);
    uint8_t* st = ring + (n % S::STAGES) * S::STAGE;
    if (!all_seen(tok0)) {
      // V rows that no row of the tile sees: what such cells hold must not meet
      // a weight of 0.
      const int k = lane % TK;
      if (!seen_by_any(p, pos_lo, pos_hi, q.ctx, tok0 + k))
        for (int c = lane / TK; c < S::CPR; c += 32 / TK)
          *reinterpret_cast<uint4*>(st + S::TILE + S::at(k, c)) = make_uint4(0u, 0u, 0u, 0u);
      __syncwarp();
    }
    float sc[NH][NU][4];
    scores(st, sc);
    uint32_t pb[NH][NU][2];
    weights(FP8 ? scale_of[0] : 0, sc, tok0, there & ((1u << S::GR) - 1u), pb);
    weigh_v(st + S::TILE, pb);
    there >>= S::GR;
    if constexpr (FP8) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) scale_of[i] = scale_of[i + 1];
    }
  }
  __syncthreads();  // the merge reuses the rings

  // ------------------------------------------------------------- merge ----
  float(*sm_acc)[R][D + 4] = reinterpret_cast<float(*)[R][D + 4]>(smem);
  float(*sm_m)[R] = reinterpret_cast<float(*)[R]>(smem + sizeof(float) * WARPS * R * (D + 4));
  float(*sm_l)[R] = sm_m + WARPS;
  float(*sm_w)[R] = sm_l + WARPS;
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int e = 0; e < NE; ++e) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[h][e] += __shfl_xor_sync(0xffffffffu, l[h][e], o);
      const int r = h * 8 + 2 * t + e;
      if (tile * R + r < pairs) {
        if (g == 0) {
          sm_m[warp][r] = m[h][e];
          sm_l[warp][r] = l[h][e];
          sm_w[warp][r] = mw[h][e];
        }
#pragma unroll
        for (int i = 0; i < S::NV; ++i)
#pragma unroll
          for (int d = 0; d < S::EV; d += 2)
            *reinterpret_cast<float2*>(&sm_acc[warp][r][(8 * i + g) * S::EV + d]) =
                make_float2(acc[h][(i * S::EV + d) / 2][e], acc[h][(i * S::EV + d) / 2][2 + e]);
      }
    }
  __syncthreads();
  const int here = min(R, pairs - tile * R);
  for (int r = warp; r < here; r += WARPS) {
    float M = -INFINITY, MW = -INFINITY, L = 0.f, wt[WARPS];
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      M = fmaxf(M, sm_m[w][r]);
      MW = fmaxf(MW, sm_w[w][r]);
    }
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      L += sm_m[w][r] == -INFINITY ? sm_l[w][r] : exp2f(sm_m[w][r] - M) * sm_l[w][r];
      wt[w] = sm_w[w][r] == -INFINITY ? 1.f : exp2f(sm_w[w][r] - MW);
    }
    // 2^(MW - M): V's scale, back on the result (1 for a 16-bit cache).
    const float back = FP8 && MW != -INFINITY ? exp2f(MW - M) : 1.f;
    const float inv = L > 0.f || L != L ? back / L : 0.f;  // NaN sums give NaN
    const int pr = tile * R + r;
    const int row = q.row0 + pr / p.G, h = hk * p.G + pr % p.G;
    const float lse2 = L == 0.f ? -INFINITY : M + log2f(L) - LIFT;
    const int64_t at = ((int64_t)row * p.Hq + h) * p.P + chunk;
    T* dst = static_cast<T*>(p.o) + (int64_t)row * p.so_t + (int64_t)h * p.so_h;
    for (int d = lane; d < D; d += 32) {
      float a = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) a = fmaf(wt[w], sm_acc[w][r][d], a);
      a *= inv;
      if (chunks == 1)
        dst[d] = from_f<T>(FP8 ? clamp_finite<T>(a) : a);
      else
        p.part_o[at * D + d] = a;
    }
    if (lane == 0) {
      if (chunks > 1)
        p.part_lse[at] = lse2;
      else if (p.lse != nullptr)
        p.lse[(int64_t)h * p.T + row] = lse2 * 0.69314718055994531f;
    }
  }
}

// The cache as rows: 64- or 128-byte rows, or the two 128-byte halves of
// 256-byte ones; a box is the rows of a group that one page holds.
template <bool FP8, int D>
static int make_map(CUtensorMap* map, const void* base, const Params& p, bool bf16) {
  EncodeTiledFn enc = get_encode_tiled();
  if (!enc) {
    set_error("cuTensorMapEncodeTiled unavailable (no CUDA driver?)");
    return LSB_ERR_CUDA;
  }
  using S = Shape<FP8, D>;
  const int inner = FP8 ? D : 64, rank = S::CPR == 16 ? 3 : 2;
  cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)(((int64_t)p.num_blocks * p.Hkv) << p.bs_log2), 2};
  cuuint64_t strides[2] = {(cuuint64_t)(D * S::EB), 128};
  // (pages of 8: a box per half row, whose 16-row halves two boxes share)
  cuuint32_t box[3] = {(cuuint32_t)inner, (cuuint32_t)(p.bs_log2 >= 4 ? 16 : 8), p.bs_log2 >= 4 ? 2u : 1u};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUtensorMapDataType type = FP8    ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                          : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUresult r = enc(map, type, rank, const_cast<void*>(base), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE,
                   S::CPR == 4 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed (%d)", (int)r);
    return LSB_ERR_CUDA;
  }
  return LSB_OK;
}

template <typename T, bool FP8, int D, int NH, bool ONE>
static int launch_tile(const Params& p, cudaStream_t st) {
  constexpr int smem = smem_bytes<FP8, D, NH>();
  constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
  CUtensorMap mk, mv;
  if (int rc = make_map<FP8, D>(&mk, p.k_cache, p, BF)) return rc;
  if (int rc = make_map<FP8, D>(&mv, p.v_cache, p, BF)) return rc;
  auto kern = paged_rows_kernel<T, FP8, D, NH, ONE>;
  static SmemLimit limit;
  if (int rc = limit.ensure(kern, smem, "paged_attn smem attribute")) return rc;
  const int64_t pairs = (int64_t)p.max_q * p.G;
  const dim3 grid((unsigned)(p.Hkv * p.P), (unsigned)((pairs + 8 * NH - 1) / (8 * NH)), (unsigned)p.S);
  LSB_CUDA_OK(launch_kernel(kern, grid, dim3(WARPS * 32), smem, st, mk, mv, p), "paged_attn");
  return LSB_OK;
}

template <typename T, bool FP8, int D>
static int launch(const Params& p, cudaStream_t st) {
  const int64_t pairs = (int64_t)p.max_q * p.G;
  if (pairs == 1) return launch_tile<T, FP8, D, 1, true>(p, st);
  switch (rows_tile(pairs)) {
    case 8: return launch_tile<T, FP8, D, 1, false>(p, st);
    case 16: return launch_tile<T, FP8, D, 2, false>(p, st);
    default: return launch_tile<T, FP8, D, 3, false>(p, st);
  }
}

}  // namespace rows

bool rows_eligible(const Params& p, int dtype) {
  if (dtype != LSB_DTYPE_BF16 && dtype != LSB_DTYPE_F16) return false;
  if ((p.D != 64 && p.D != 128) || p.bs_log2 < 3) return false;
  // q rows are read in 8-byte pieces; the cache's rows are a 32-bit TMA
  // coordinate, its base 16-byte aligned.
  auto at = [](const void* x, uintptr_t a) { return (reinterpret_cast<uintptr_t>(x) & (a - 1)) == 0; };
  if (!at(p.q, 8) || p.sq_t % 4 != 0 || p.sq_h % 4 != 0) return false;
  if (!at(p.k_cache, 16) || !at(p.v_cache, 16)) return false;
  if ((((int64_t)p.num_blocks * p.Hkv) << p.bs_log2) > 0x7fffffff) return false;
  return (int64_t)p.max_q * p.G / 8 < 65535 && (int64_t)p.Hkv * p.P <= 0x7fffffff;
}

int launch_rows(const Params& p, int dtype, bool kv_fp8, cudaStream_t st) {
  const bool bf = dtype == LSB_DTYPE_BF16;
  if (p.D == 128) {
    if (kv_fp8) return bf ? rows::launch<__nv_bfloat16, true, 128>(p, st) : rows::launch<__half, true, 128>(p, st);
    return bf ? rows::launch<__nv_bfloat16, false, 128>(p, st) : rows::launch<__half, false, 128>(p, st);
  }
  if (kv_fp8) return bf ? rows::launch<__nv_bfloat16, true, 64>(p, st) : rows::launch<__half, true, 64>(p, st);
  return bf ? rows::launch<__nv_bfloat16, false, 64>(p, st) : rows::launch<__half, false, 64>(p, st);
}

}  // namespace pa

int paged_attn_rows_device_error(bool reset) { return sm100::tu_device_error(reset); }

}  // namespace lsb
