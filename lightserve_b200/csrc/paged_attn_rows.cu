// Paged attention for a few rows per sequence (decode, drafted tokens): the
// cache is read once at HBM speed, the arithmetic rides along on mma.sync.
//
// One CTA: a query tile of 8 NH pairs (row, head of the group) of one
// (sequence, cache head) and one chunk of its keys; its 4 warps take groups of
// 16 keys in turn and merge at the end. Bound by HBM and, for e4m3, close to it
// by instruction issue: per 16 keys a warp moves 4 KiB (D = 128) and issues 16
// m16n8k16 MMAs per 8 pairs. The warp-level MMA is the right size here:
// tcgen05's 128-row tiles would hold one row of use per key read.
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
// Each warp streams its groups through a ring of its own in shared memory
// (cp.async, 16 bytes a lane: STAGES groups in flight cost no registers and no
// barrier beyond the warp's). Rows are stored with their 16-byte pieces permuted
// (Shape::at) so that both kinds of read touch every bank once.
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
// per group instead of shuffles and a rescale). Weights carry a factor 2^7, so
// an fp16 weight keeps its precision down to 2^-21 of the maximum and vanishes
// below 2^-32: rounding P to 16 bits is off by half a step of the operand type
// relative to each weight, as in the framework's other attention kernels.
#include "paged_attn.cuh"
#include "sm100.cuh"

#include <type_traits>

namespace lsb {
namespace pa {

namespace rows {

constexpr int TK = ROWS_TK;  // keys per group
constexpr int WARPS = 4;
constexpr float RAISE = 8.f;   // log2: how far a score may exceed the reference maximum
constexpr float LIFT = 7.f;    // log2: factor on every weight

template <bool F16>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm(
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

// 16 bytes (8: scales) from global to shared memory, zeros when !there.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(src)), "r"(there ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy8(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(src)), "r"(there ? 8 : 0)
               : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <bool FP8, int D>
struct Shape {
  static constexpr int EB = FP8 ? 1 : 2;           // bytes per cached element
  static constexpr int EK = 16 / EB;               // K elements per lane and load
  static constexpr int NK = D / (4 * EK);          // K loads per key and lane
  static constexpr int EV = FP8 ? D / 8 : 8;       // V elements per lane and load
  static constexpr int NV = D / (8 * EV);          // V loads per key and lane
  static constexpr int WV = EV * EB / 4;           // words per V load
  static constexpr int STEPS = D / 16;             // k steps of S^T
  static constexpr int MT = D / 16;                // m-tiles of O^T
  static constexpr int CPR = D * EB / 16;          // 16-byte pieces of a row: 4, 8 or 16
  static constexpr int HALF = 8 * CPR;             // pieces of 8 keys
  static constexpr int TILE = TK * CPR * 16;       // bytes of a group's K (and V)
  // A stage: K, V, and for e4m3 the scales (16 of K, 16 of V).
  static constexpr int STAGE = 2 * TILE + (FP8 ? 32 : 0);
  // Groups in flight per warp, sized so that an SM holds about 190 KB of ring.
  static constexpr int STAGES = FP8 ? 4 : (D == 64 ? 4 : 3);
  static constexpr int ctas(int nh) {
    return FP8 ? (D == 64 ? 6 - nh : (nh == 3 ? 2 : 3)) : (D == 64 ? 3 : 2);
  }
  // Byte offset of piece c of key k's row in its tile.
  static __device__ __forceinline__ int at(int k, int c) {
    if constexpr (CPR == 4) {  // two rows to a 128-byte line
      const int line = k >> 1;
      return (line * 8 + ((((k & 1) << 2) | c) ^ ((line & 3) << 1))) * 16;
    } else {
      return (k * CPR + (c ^ ((((k >> 1) & 3) << 1) ^ ((k & 1) << 2)))) * 16;
    }
  }
};

// Dynamic shared memory of a CTA: the rings, which the merge reuses.
template <bool FP8, int D, int NH>
constexpr int smem_bytes() {
  const int ring = WARPS * Shape<FP8, D>::STAGES * Shape<FP8, D>::STAGE;
  const int merge = WARPS * 8 * NH * (D + 4 + 3) * 4;
  return ring > merge ? ring : merge;
}

template <typename T, bool FP8, int D, int NH>
__global__ void __launch_bounds__(WARPS * 32, (Shape<FP8, D>::ctas(NH)))
paged_rows_kernel(const Params p) {
  allow_dependents();
  wait_prerequisites();
  using S = Shape<FP8, D>;
  constexpr bool F16 = FP8 || std::is_same<T, __half>::value;  // MMA operand type
  constexpr int R = 8 * NH;
  extern __shared__ __align__(16) uint8_t smem[];

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
  // Page ids of 16 of this warp's groups from v on, one half group per lane;
  // -1: no such page.
  auto fetch_ids = [&](int v) -> int {
    const int vv = v + (lane >> 1) * WARPS;
    if (vv >= v1) return -1;
    const int tok = span.tile(vv) * TK + 8 * (lane & 1);
    if (tok >= q.ctx) return -1;
    const int id = bt[tok >> p.bs_log2];
    return id >= 0 && id < p.num_blocks ? id : -1;
  };
  const uint8_t* kc = static_cast<const uint8_t*>(p.k_cache) + lane * 16;
  const uint8_t* vc = static_cast<const uint8_t*>(p.v_cache) + lane * 16;
  uint8_t* ring = smem + warp * (S::STAGES * S::STAGE);
  // Whether every pair sees all 16 keys at tok0 (pages apart).
  auto all_seen = [&](int tok0) -> bool {
    const int last = tok0 + TK - 1;
    return last <= pos_lo && last < q.ctx &&
           (p.window == 0 || pos_hi - tok0 < p.window || last < p.sinks);
  };
  // Copies the group at keys [tok0, tok0 + 16) into a stage. Missing pages and
  // V rows that no row of the tile sees arrive as zeros, so what such cells
  // hold never meets a weight of 0.
  auto copy_group = [&](int stage, int tok0, int id0, int id1) {
    const uint32_t dst = sm100::smem_u32(ring + stage * S::STAGE);
    const bool clean = id0 >= 0 && id1 >= 0 && all_seen(tok0);
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int id = hf == 0 ? id0 : id1;
      const int64_t cell =
          ((int64_t)max(id, 0) * p.Hkv + hk) * bs + ((tok0 + 8 * hf) & (bs - 1));
      const uint8_t* ks = kc + cell * (D * S::EB);
      const uint8_t* vs = vc + cell * (D * S::EB);
#pragma unroll
      for (int i = 0; i < S::HALF / 32; ++i) {
        const int piece = i * 32 + lane, k = hf * 8 + piece / S::CPR;
        const uint32_t to = dst + S::at(k, piece % S::CPR);
        bool kt = true, vt = true;
        if (!clean) {
          kt = id >= 0;
          vt = kt && seen_by_any(p, pos_lo, pos_hi, q.ctx, tok0 + k);
        }
        copy16(to, ks + i * 512, kt);
        copy16(to + S::TILE, vs + i * 512, vt);
      }
      if constexpr (FP8) {
        if (lane < 2)
          copy8(dst + 2 * S::TILE + lane * 16 + hf * 8, (lane == 0 ? p.k_scale : p.v_scale) + cell,
                id >= 0);
      }
    }
  };

  // Group n of this warp is v0 + warp + n WARPS and sits in stage n % STAGES.
  constexpr int AHEAD = S::STAGES - 1;
  const int first = v0 + warp;
  const int mine = v1 > first ? (v1 - first + WARPS - 1) / WARPS : 0;
  int near = fetch_ids(first), far = fetch_ids(first + 16 * WARPS);
  auto copy_next = [&](int n) -> uint32_t {  // called for n = 0, 1, 2, ... in turn
    if (n > 0 && n % 16 == 0) {
      near = far;
      far = fetch_ids(first + (n + 16) * WARPS);
    }
    const int a = __shfl_sync(0xffffffffu, near, 2 * (n % 16));
    const int b = __shfl_sync(0xffffffffu, near, 2 * (n % 16) + 1);
    if (n < mine) copy_group(n % S::STAGES, span.tile(first + n * WARPS) * TK, a, b);
    copies_commit();  // a group of copies per n, empty past the end
    return (a >= 0 ? 1u : 0u) | (b >= 0 ? 2u : 0u);
  };
  uint32_t there = 0;  // two bits per group in flight: which halves have a page
#pragma unroll
  for (int n = 0; n < AHEAD; ++n) there |= copy_next(n) << (2 * n);

  // ---------------------------------------------------------------- Q ----
  // B fragments: pair 8 h + g of the tile, its 4-element piece per k step.
  uint32_t qb[NH][S::STEPS][2];
  // Of pairs 8 h + 2 t and 8 h + 2 t + 1, whose scores this lane holds: the
  // score's factor (scale log2(e), and the row's power of two) and position.
  float fac[NH][2];
  int pos[NH][2];
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
    for (int e = 0; e < 2; ++e) {  // lane 4 (2 t + e) holds pair 8 h + 2 t + e
      fac[h][e] = __shfl_sync(0xffffffffu, f, 4 * (2 * t + e));
      const int pe = tile * R + h * 8 + 2 * t + e;
      pos[h][e] = pe < pairs ? q.pos0 + pe / p.G : -1;  // position -1 sees nothing
    }
  }

  // ----------------------------------------------------------- compute ----
  // Running maxima m (of scores) and mw (of scores + V exponents), held as the
  // thresholds that raise them; sums and outputs are relative to them.
  float m[NH][2], mw[NH][2], l[NH][2], acc[NH][S::MT][4];
#pragma unroll
  for (int h = 0; h < NH; ++h) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      m[h][e] = mw[h][e] = -INFINITY;
      l[h][e] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < S::MT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[h][j][e] = 0.f;
  }

  // S^T of the group: sc[h][2 n + e] = key 8 n + g, pair 8 h + 2 t + e.
  auto scores = [&](const uint8_t* kt, float (&sc)[NH][4]) {
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[h][e] = 0.f;
#pragma unroll
    for (int i = 0; i < S::NK; ++i) {
      uint32_t k[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n) load_words(k[n], kt + S::at(8 * n + g, 4 * i + t));
#pragma unroll
      for (int w = 0; w < S::EK / 4; ++w) {
        const int st = i * (S::EK / 4) + w;
        uint32_t a[4];  // keys g, 8 + g; then their second halves of the step
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          if constexpr (FP8) {
            a[n] = cvt_e4m3x2_f16x2((uint16_t)(k[n][w] & 0xffff));
            a[2 + n] = cvt_e4m3x2_f16x2((uint16_t)(k[n][w] >> 16));
          } else {
            a[n] = k[n][2 * w];
            a[2 + n] = k[n][2 * w + 1];
          }
        }
#pragma unroll
        for (int h = 0; h < NH; ++h)
          mma16816<F16>(sc[h], a[0], a[1], a[2], a[3], qb[h][st][0], qb[h][st][1]);
      }
    }
  };

  // Weights of the group's keys as B fragments of O^T: pb[h][n] = pair 8 h + g,
  // keys 8 n + 2 t, 8 n + 2 t + 1. Scores go to log2 units, to -inf for keys
  // that a row does not see.
  auto weights = [&](const uint8_t* scales, float (&sc)[NH][4], int tok0, uint32_t pages,
                     uint32_t (&pb)[NH][2]) {
    float ev[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      float f = 1.f, bad = 0.f;
      if constexpr (FP8) {
        const int kb = scales[8 * n + g], vb = scales[16 + 8 * n + g];
        f = __uint_as_float((uint32_t)kb << 23);  // 255, e8m0's NaN, gives infinity here
        bad = f - f;                              // and NaN here
        ev[n] = vb == 255 ? __int_as_float(0x7fc00000)
                          : __uint_as_float(0x4b000000u | vb) - (8388608.f + 127.f);
      }
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          sc[h][2 * n + e] =
              FP8 ? fmaf(sc[h][2 * n + e] * fac[h][e], f, bad) : sc[h][2 * n + e] * fac[h][e];
    }
    if (pages != 3u || !all_seen(tok0)) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int j = tok0 + 8 * n + g;
        const bool page = (pages >> n) & 1;
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (!page || !sees(p, pos[h][e], q.ctx, j)) sc[h][2 * n + e] = -INFINITY;
        if (!page || !seen_by_any(p, pos_lo, pos_hi, q.ctx, j)) ev[n] = 0.f;
      }
    }
    bool raise = false;
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          raise |= sc[h][2 * n + e] > m[h][e] + RAISE;
          if constexpr (FP8) raise |= sc[h][2 * n + e] + ev[n] > mw[h][e] + RAISE;
        }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float a = fmaxf(m[h][e], fmaxf(sc[h][e], sc[h][2 + e]));
          float b = FP8 ? fmaxf(mw[h][e], fmaxf(sc[h][e] + ev[0], sc[h][2 + e] + ev[1])) : 0.f;
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
      float mm[2], mmw[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mm[e] = m[h][e] == -INFINITY ? 0.f : m[h][e] - LIFT;
        mmw[e] = mw[h][e] == -INFINITY ? 0.f : mw[h][e] - LIFT;
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float p0 = sm100::ex2(sc[h][2 * n] - mm[0]), p1 = sm100::ex2(sc[h][2 * n + 1] - mm[1]);
        l[h][0] += p0;
        l[h][1] += p1;
        uint32_t w;
        if constexpr (FP8)
          w = sm100::pack_f16(sm100::ex2(sc[h][2 * n] + (ev[n] - mmw[0])),
                              sm100::ex2(sc[h][2 * n + 1] + (ev[n] - mmw[1])));
        else
          w = F16 ? sm100::pack_f16(p0, p1) : sm100::pack_bf16(p0, p1);
        pb[h][n] = transpose8x8(w);
      }
    }
  };

  auto weigh_v = [&](const uint8_t* vt, const uint32_t (&pb)[NH][2]) {
#pragma unroll
    for (int i = 0; i < S::NV; ++i) {
      uint32_t vw[4][S::WV];  // keys 2t, 2t + 1, 8 + 2t, 9 + 2t
      const int byte = (8 * i + g) * (S::EV * S::EB);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        load_words(vw[e], vt + S::at((e >> 1) * 8 + 2 * t + (e & 1), byte / 16) + byte % 16);
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
            mma16816<F16>(acc[h][j], l0, l1, l2, l3, pb[h][0], pb[h][1]);
            mma16816<F16>(acc[h][j + 1], h0, h1, h2, h3, pb[h][0], pb[h][1]);
          }
        } else {
          const int j = (i * S::EV + 2 * w) / 2;
          const uint32_t x0 = __byte_perm(a, b, 0x5410), x1 = __byte_perm(a, b, 0x7632);
          const uint32_t x2 = __byte_perm(c, d, 0x5410), x3 = __byte_perm(c, d, 0x7632);
#pragma unroll
          for (int h = 0; h < NH; ++h)
            mma16816<F16>(acc[h][j], x0, x1, x2, x3, pb[h][0], pb[h][1]);
        }
      }
    }
  };

  for (int n = 0; n < mine; ++n) {
    copies_wait<AHEAD - 1>();  // this lane's copies of group n are in
    __syncwarp();              // every lane's are, and group n - 1 has been read by all
    there |= copy_next(n + AHEAD) << (2 * AHEAD);
    const uint8_t* st = ring + (n % S::STAGES) * S::STAGE;
    float sc[NH][4];
    scores(st, sc);
    uint32_t pb[NH][2];
    weights(st + 2 * S::TILE, sc, span.tile(first + n * WARPS) * TK, there & 3u, pb);
    weigh_v(st + S::TILE, pb);
    there >>= 2;
  }
  copies_wait<0>();
  __syncthreads();  // the merge reuses the rings

  // ------------------------------------------------------------- merge ----
  float(*sm_acc)[R][D + 4] = reinterpret_cast<float(*)[R][D + 4]>(smem);
  float(*sm_m)[R] = reinterpret_cast<float(*)[R]>(smem + sizeof(float) * WARPS * R * (D + 4));
  float(*sm_l)[R] = sm_m + WARPS;
  float(*sm_w)[R] = sm_l + WARPS;
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
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

template <typename T, bool FP8, int D, int NH>
static int launch_tile(const Params& p, cudaStream_t st) {
  constexpr int smem = smem_bytes<FP8, D, NH>();
  auto kern = paged_rows_kernel<T, FP8, D, NH>;
  static SmemLimit limit;
  if (int rc = limit.ensure(kern, smem, "paged_attn smem attribute")) return rc;
  const int64_t pairs = (int64_t)p.max_q * p.G;
  const dim3 grid((unsigned)(p.Hkv * p.P), (unsigned)((pairs + 8 * NH - 1) / (8 * NH)), (unsigned)p.S);
  LSB_CUDA_OK(launch_kernel(kern, grid, dim3(WARPS * 32), smem, st, p), "paged_attn");
  return LSB_OK;
}

template <typename T, bool FP8, int D>
static int launch(const Params& p, cudaStream_t st) {
  switch (rows_tile((int64_t)p.max_q * p.G)) {
    case 8: return launch_tile<T, FP8, D, 1>(p, st);
    case 16: return launch_tile<T, FP8, D, 2>(p, st);
    default: return launch_tile<T, FP8, D, 3>(p, st);
  }
}

}  // namespace rows

bool rows_eligible(const Params& p, int dtype, bool kv_fp8) {
  if (dtype != LSB_DTYPE_BF16 && dtype != LSB_DTYPE_F16) return false;
  if ((p.D != 64 && p.D != 128) || p.bs_log2 < 3) return false;
  // q rows are read in 8-byte pieces, the cache in 16-byte ones, the scales of
  // 8 keys at a time.
  auto at = [](const void* x, uintptr_t a) { return (reinterpret_cast<uintptr_t>(x) & (a - 1)) == 0; };
  if (!at(p.q, 8) || p.sq_t % 4 != 0 || p.sq_h % 4 != 0) return false;
  if (!at(p.k_cache, 16) || !at(p.v_cache, 16)) return false;
  if (kv_fp8 && (!at(p.k_scale, 8) || !at(p.v_scale, 8))) return false;
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
}  // namespace lsb
