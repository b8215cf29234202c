// Attention of new tokens over a paged KV cache: the C entry, the choice of
// kernel, the CUDA-core kernel (any type, head dim up to 256, any alignment)
// and the kernel that joins split key ranges. paged_attn.cuh has the
// definitions.
#include "paged_attn.cuh"

#include <algorithm>
#include <type_traits>

namespace lsb {
namespace pa {

// ------------------------------------------------------- CUDA-core kernel --
// One CTA: a query tile of 4 ROWS pairs of one (sequence, cache head) and one
// chunk of its keys; its 4 warps own ROWS pairs each. K and V tiles of STK = 32
// keys are staged in shared memory as fp32 (dequantised there; ROWS = 1: from
// registers that were loaded a tile ahead). Scores: lane = key, so a K row is read
// once as float4s (row stride D + 4: conflict-free) for ROWS pairs whose q values
// are broadcast reads. P V: lane = dim, each V element serving the warp's pairs.
// All arithmetic is fp32, as the fp32 model's parity with the reference needs
// (tensor-core TF32 does not reach it).
// ROWS = 1 serves up to 4 pairs (a tile of 16 took 197 us against 87 for 4
// sequences of 2000-9000 fp32 keys, 8 cache heads of 128, 4 pairs: 39% of HBM), and
// a single pair is shared by the warps (32 sequences of 512-4096 fp32 keys, 8
// heads of 128, a window of 2048: 158 us against 126, 55% of HBM). ROWS = 8 where
// half the CTAs still fill the GPU: shared-memory reads, 4 + ROWS wavefronts per
// 4 ROWS FMAs of a warp, and issue slots bound it (4 chunks of 300-700 tokens over
// 1000-4000, 8 x 2 heads of 128: 1610 us, 19 TFLOP/s, against 2010 with 4; three
// short prompts 19 against 13).
constexpr int STK = 32;
constexpr int S_WARPS = 4;
static int simt_rows(int64_t S, int64_t Hkv, int64_t pairs) {
  if (pairs <= 4) return 1;
  return pairs > 16 && S * Hkv * ((pairs + 31) / 32) >= 2 * 148 ? 8 : 4;
}

// Four elements of a cached row as they are stored, in whole words: unpacking
// them where they are loaded waited for each load in turn (64 sequences of
// 512-4096 e4m3 keys, 16 heads of 128, fp32 q: 1995 us against 586).
template <typename KV>
struct alignas(4 * sizeof(KV)) Quad {
  uint32_t w[sizeof(KV)];
};

// `left` of the elements exist.
template <typename KV>
__device__ __forceinline__ Quad<KV> load4(const KV* p, bool vec, int left) {
  if (vec) return *reinterpret_cast<const Quad<KV>*>(p);
  Quad<KV> x = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i >= left) break;
    if constexpr (sizeof(KV) == 1)
      x.w[0] |= (uint32_t)reinterpret_cast<const uint8_t*>(p)[i] << (8 * i);
    else if constexpr (sizeof(KV) == 2)
      x.w[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << (16 * (i % 2));
    else
      x.w[i] = reinterpret_cast<const uint32_t*>(p)[i];
  }
  return x;
}

template <typename KV>
__device__ __forceinline__ float4 widen(const Quad<KV>& x) {
  if constexpr (sizeof(KV) == 1) {
    float f[4];
    e4m3x4_to_float(x.w[0], f);
    return make_float4(f[0], f[1], f[2], f[3]);
  } else if constexpr (sizeof(KV) == 2) {
    KV e[4];
    memcpy(e, x.w, sizeof(e));
    return make_float4(to_f(e[0]), to_f(e[1]), to_f(e[2]), to_f(e[3]));
  } else {
    return make_float4(__uint_as_float(x.w[0]), __uint_as_float(x.w[1]), __uint_as_float(x.w[2]),
                       __uint_as_float(x.w[3]));
  }
}

// DC: 32-dim columns per lane (head dim up to 32 DC). ONE: the call has one pair per
// cache head, which the warps share: a quarter of the dims of each score, then a
// quarter of the keys of P V.
template <typename T, typename KV, int DC, int ROWS, bool ONE>
__global__ void __launch_bounds__(S_WARPS * 32)
paged_simt_kernel(const Params p, const bool vec) {
  constexpr bool FP8 = std::is_same<KV, uint8_t>::value;
  static_assert(!ONE || ROWS == 1, "one pair");
  constexpr int SR = S_WARPS * ROWS;
  // Staging: a warp's 8 keys of a tile, QL lanes per key, QPL quads per lane.
  constexpr int QL = DC == 2 ? 16 : 32, QPL = DC == 8 ? 2 : 1;
  constexpr int PASSES = STK / S_WARPS * QL / 32, N = PASSES * QPL;
  constexpr bool AHEAD = ROWS == 1 && DC <= 4;  // (elsewhere its registers cost more than it hides)
  extern __shared__ float sm[];
  const int D = p.D, Dp = (D + 3) & ~3, ldk = Dp + 4;
  float* sQ = sm;                    // [SR][Dp]
  float* sK = sQ + SR * Dp;          // [STK][ldk]
  float* sV = sK + STK * ldk;        // [STK][Dp]
  float* sP = sV + STK * Dp;         // [SR][STK]

  const int s = blockIdx.z;
  const Seq q = load_seq(p, s);
  // blockIdx.x runs over (cache head, chunk), blockIdx.y over query tiles.
  const int hk = blockIdx.x / p.P, chunk = blockIdx.x % p.P;
  const int pairs = q.n * p.G, tile = blockIdx.y;
  if (tile * SR >= pairs) return;
  int pos_lo, pos_hi;
  tile_positions(p, q, tile, SR, pos_lo, pos_hi);
  const KeySpan span(p, q, pos_lo, pos_hi, STK);
  const int per = p.chunk / STK, tiles = span.count();
  const int chunks = chunks_of(p, tiles, STK);
  if (chunk >= chunks) return;
  const int v0 = chunk * per, v1 = chunk + 1 == chunks ? tiles : min(tiles, v0 + per);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < SR * Dp; i += blockDim.x) {
    const int r = tile * SR + i / Dp, d = i % Dp;
    float x = 0.f;
    if (r < pairs && d < D)
      x = to_f(static_cast<const T*>(p.q)[(int64_t)(q.row0 + r / p.G) * p.sq_t +
                                          (int64_t)(hk * p.G + r % p.G) * p.sq_h + d]);
    sQ[i] = x;
  }
  // Pair r of this warp is pair r S_WARPS + warp of the tile.
  int pos[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int pr = ONE ? 0 : tile * SR + r * S_WARPS + warp;
    pos[r] = pr < pairs ? q.pos0 + pr / p.G : -1;  // position -1 sees nothing
  }
  const bool live = ONE || tile * SR + warp < pairs;
  float m[ROWS], l[ROWS], acc[ROWS][DC];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int c = 0; c < DC; ++c) acc[r][c] = 0.f;
  }
  const int32_t* bt = p.block_tables + (int64_t)s * p.max_blocks;
  const int bs = 1 << p.bs_log2;

  // Page of key `lane` of span tile v; -1: none, or no row of the tile sees it.
  auto fetch_id = [&](int v) -> int {
    if (v >= v1) return -1;
    const int key = span.tile(v) * STK + lane;
    if (!seen_by_any(p, pos_lo, pos_hi, q.ctx, key)) return -1;
    const int id = bt[key >> p.bs_log2];
    return id >= 0 && id < p.num_blocks ? id : -1;
  };
  auto cell_of = [&](int id, int key) {
    return (((int64_t)id * p.Hkv + hk) << p.bs_log2) + (key & (bs - 1));
  };
  // This thread's quads of a tile: n = pass QPL + u is key `row` + pass 32 / QL of
  // the tile, dims from `dim` + 128 u on.
  const int row = warp * (STK / S_WARPS) + lane / QL, dim = lane % QL * 4;
  auto load = [&](const void* cache, int key0, int id, Quad<KV> (&x)[N]) {
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
      const int j = row + pass * (32 / QL), jd = __shfl_sync(0xffffffffu, id, j);
#pragma unroll
      for (int u = 0; u < QPL; ++u) {
        const int d = dim + 128 * u;
        x[pass * QPL + u] = Quad<KV>{};
        if (jd >= 0 && d < D)
          x[pass * QPL + u] = load4(static_cast<const KV*>(cache) + cell_of(jd, key0 + j) * D + d, vec, D - d);
      }
    }
  };
  // scale: the byte of key `lane`.
  auto store = [&](float* dst, int ld, const Quad<KV> (&x)[N], int scale) {
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
      const int j = row + pass * (32 / QL);
      const float f = FP8 ? e8m0_to_float(__shfl_sync(0xffffffffu, scale, j)) : 1.f;
#pragma unroll
      for (int u = 0; u < QPL; ++u) {
        const int d = dim + 128 * u;
        float4 y = widen(x[pass * QPL + u]);
        if constexpr (FP8) y = make_float4(y.x * f, y.y * f, y.z * f, y.w * f);
        if (d < Dp) *reinterpret_cast<float4*>(dst + j * ld + d) = y;
      }
    }
  };

  Quad<KV> xk[N], xv[N];
  int id = fetch_id(v0), id1 = fetch_id(v0 + 1), scales = 127 | 127 << 8;
  auto load_tile = [&](int v, int ids) {
    const int key0 = span.tile(v) * STK;
    if constexpr (FP8) {
      scales = 127 | 127 << 8;
      if (ids >= 0) {
        const int64_t cell = cell_of(ids, key0 + lane);
        scales = p.k_scale[cell] | p.v_scale[cell] << 8;
      }
    }
    load(p.k_cache, key0, ids, xk);
    if constexpr (AHEAD) load(p.v_cache, key0, ids, xv);
  };
  if (AHEAD && v0 < v1) load_tile(v0, id);
  for (int v = v0; v < v1; ++v) {
    const int key0 = span.tile(v) * STK;
    __syncthreads();  // the previous tile (and, at first, nothing) has been read
    if constexpr (!AHEAD) load_tile(v, id);
    store(sK, ldk, xk, scales & 0xff);
    if constexpr (!AHEAD) load(p.v_cache, key0, id, xv);
    store(sV, Dp, xv, scales >> 8);
    __syncthreads();
    const bool key_ok = id >= 0;
    id = id1;
    id1 = fetch_id(v + 2);
    if (AHEAD && v + 1 < v1) load_tile(v + 1, id);
    if (!live) continue;
    float sc[ROWS] = {};
#pragma unroll 2
    for (int d = ONE ? 4 * warp : 0; d < Dp; d += ONE ? 4 * S_WARPS : 4) {
      const float4 kx = *reinterpret_cast<const float4*>(sK + lane * ldk + d);
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const float4 qx = *reinterpret_cast<const float4*>(sQ + (ONE ? 0 : r * S_WARPS + warp) * Dp + d);
        sc[r] = fmaf(qx.x, kx.x, sc[r]);
        sc[r] = fmaf(qx.y, kx.y, sc[r]);
        sc[r] = fmaf(qx.z, kx.z, sc[r]);
        sc[r] = fmaf(qx.w, kx.w, sc[r]);
      }
    }
    if constexpr (ONE) {
      sP[warp * STK + lane] = sc[0];
      __syncthreads();
      sc[0] = (sP[lane] + sP[STK + lane]) + (sP[2 * STK + lane] + sP[3 * STK + lane]);
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float x = key_ok && sees(p, pos[r], q.ctx, key0 + lane) ? sc[r] * p.scale_log2 : -INFINITY;
      // A NaN score stays visible: fmaxf drops it, but exp2f below returns it.
      const float mx = fmaxf(m[r], warp_max(x));
      const float m_use = mx == -INFINITY ? 0.f : mx;
      const float a = exp2f(m[r] - m_use);
      const float e = exp2f(x - m_use);
      m[r] = mx;
      l[r] = l[r] * a + e;  // per-lane partial sum
#pragma unroll
      for (int c = 0; c < DC; ++c) acc[r][c] *= a;
      if constexpr (ONE) {
        const float* vt = sV + warp * (STK / S_WARPS) * Dp;
#pragma unroll
        for (int j = 0; j < STK / S_WARPS; ++j) {
          const float pe = __shfl_sync(0xffffffffu, e, warp * (STK / S_WARPS) + j);
#pragma unroll
          for (int c = 0; c < DC; ++c)
            if (c * 32 + lane < Dp) acc[r][c] = fmaf(pe, vt[j * Dp + c * 32 + lane], acc[r][c]);
        }
      } else {
        sP[(warp * ROWS + r) * STK + lane] = e;
      }
    }
    if constexpr (ONE) continue;
    __syncwarp();
    for (int j = 0; j < STK; j += 4) {
      float4 pr[ROWS];
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
        pr[r] = *reinterpret_cast<const float4*>(sP + (warp * ROWS + r) * STK + j);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int c = 0; c < DC; ++c) {
          const int d = c * 32 + lane;
          const float vx = d < Dp ? sV[(j + e) * Dp + d] : 0.f;
#pragma unroll
          for (int r = 0; r < ROWS; ++r) {
            const float pe = e == 0 ? pr[r].x : e == 1 ? pr[r].y : e == 2 ? pr[r].z : pr[r].w;
            acc[r][c] = fmaf(pe, vx, acc[r][c]);
          }
        }
      }
    }
  }
  if constexpr (ONE) {  // the warps' shares of P V (every warp has the statistics)
    __syncthreads();
#pragma unroll
    for (int c = 0; c < DC; ++c) sK[warp * (DC * 32) + c * 32 + lane] = acc[0][c];
    __syncthreads();
    if (warp > 0) return;
#pragma unroll
    for (int c = 0; c < DC; ++c)
#pragma unroll
      for (int w = 1; w < S_WARPS; ++w) acc[0][c] += sK[w * (DC * 32) + c * 32 + lane];
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int pr = tile * SR + r * S_WARPS + warp;
    if (pr >= pairs) continue;
    const int row = q.row0 + pr / p.G, h = hk * p.G + pr % p.G;
    const float lsum = warp_sum(l[r]);
    const float inv = lsum > 0.f || lsum != lsum ? 1.f / lsum : 0.f;  // NaN sums give NaN
    const float lse2 = lsum == 0.f ? -INFINITY : m[r] + log2f(lsum);
    if (chunks == 1) {
      T* dst = static_cast<T*>(p.o) + (int64_t)row * p.so_t + (int64_t)h * p.so_h;
#pragma unroll
      for (int c = 0; c < DC; ++c)
        if (c * 32 + lane < D) dst[c * 32 + lane] = from_f<T>(FP8 ? clamp_finite<T>(acc[r][c] * inv) : acc[r][c] * inv);
      if (p.lse != nullptr && lane == 0) p.lse[(int64_t)h * p.T + row] = lse2 * 0.69314718055994531f;
    } else {
      const int64_t at = ((int64_t)row * p.Hq + h) * p.P + chunk;
#pragma unroll
      for (int c = 0; c < DC; ++c)
        if (c * 32 + lane < D) p.part_o[at * D + c * 32 + lane] = acc[r][c] * inv;
      if (lane == 0) p.part_lse[at] = lse2;
    }
  }
}

int launch_simt(const Params& p, int dtype, bool kv_fp8, cudaStream_t st) {
  const int Dp = (p.D + 3) & ~3, rows = simt_rows(p.S, p.Hkv, (int64_t)p.max_q * p.G);
  const int SR = S_WARPS * rows;
  const size_t smem = sizeof(float) * (SR * Dp + STK * (Dp + 4) + STK * Dp + SR * STK);
  const int64_t tiles = ((int64_t)p.max_q * p.G + SR - 1) / SR;
  LSB_CHECK_ARG(tiles <= 65535 && (int64_t)p.Hkv * p.P <= 0x7fffffff,
                "paged_attn: %lld query tiles per head exceed 65535 (CUDA-core kernel)", (long long)tiles);
  const dim3 grid((unsigned)(p.Hkv * p.P), (unsigned)tiles, (unsigned)p.S);
  auto go = [&](auto tag, auto kvtag, auto dc, auto nr, auto one) -> int {
    using T = decltype(tag);
    using KV = decltype(kvtag);
    constexpr int DC = decltype(dc)::value;
    // 4-element loads: every cache row starts on such a boundary.
    const bool vec = p.D % 4 == 0 &&
                     ((reinterpret_cast<uintptr_t>(p.k_cache) | reinterpret_cast<uintptr_t>(p.v_cache)) &
                      (4 * sizeof(KV) - 1)) == 0;
    auto kern = paged_simt_kernel<T, KV, DC, decltype(nr)::value, decltype(one)::value>;
    static SmemLimit limit;
    if (smem > 48 * 1024)
      if (int rc = limit.ensure(kern, smem, "paged_attn smem attribute")) return rc;
    kern<<<grid, S_WARPS * 32, smem, st>>>(p, vec);
    LSB_CHECK_LAUNCH("paged_attn");
    return LSB_OK;
  };
  auto by_rows = [&](auto tag, auto kvtag, auto dc) -> int {
    using std::integral_constant;
    if ((int64_t)p.max_q * p.G == 1) return go(tag, kvtag, dc, integral_constant<int, 1>{}, std::true_type{});
    if (rows == 1) return go(tag, kvtag, dc, integral_constant<int, 1>{}, std::false_type{});
    if (rows == 4) return go(tag, kvtag, dc, integral_constant<int, 4>{}, std::false_type{});
    return go(tag, kvtag, dc, integral_constant<int, 8>{}, std::false_type{});
  };
  auto by_dim = [&](auto tag, auto kvtag) -> int {
    if (p.D <= 64) return by_rows(tag, kvtag, std::integral_constant<int, 2>{});
    if (p.D <= 128) return by_rows(tag, kvtag, std::integral_constant<int, 4>{});
    return by_rows(tag, kvtag, std::integral_constant<int, 8>{});
  };
  return LSB_DISPATCH_DTYPE(dtype, T, [&] {
    if (kv_fp8) return by_dim(T{}, uint8_t{});
    return by_dim(T{}, T{});
  });
}

// ----------------------------------------------------------------- combine --
// One CTA per (row, head): the grid is (row, head) pairs of the longest
// sequence by sequences, so no row has to look its sequence up. Its 4 warps
// take the chunks in turn (4 of them in flight per warp: a few hundred chunks
// would otherwise be as many dependent trips to L2), then join.
constexpr int C_WARPS = 4;

template <typename T, int DC>
__global__ void __launch_bounds__(C_WARPS * 32)
paged_combine_kernel(const Params p, int R, int tk) {
  allow_dependents();
  wait_prerequisites();
  __shared__ float sm[C_WARPS][DC * 32];
  const Seq q = load_seq(p, blockIdx.y);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i = blockIdx.x / p.Hq, h = blockIdx.x % p.Hq;
  if (i >= q.n) return;
  int pos_lo, pos_hi;
  tile_positions(p, q, (i * p.G + h % p.G) / R, R, pos_lo, pos_hi);
  const KeySpan span(p, q, pos_lo, pos_hi, tk);
  const int chunks = chunks_of(p, span.count(), tk);
  if (chunks == 1) return;  // written directly
  const int row = q.row0 + i;
  const int64_t at = ((int64_t)row * p.Hq + h) * p.P;
  float mx = -INFINITY, bad = 0.f;
  for (int c = lane; c < chunks; c += 32) {
    const float x = p.part_lse[at + c];
    if (x != x) bad = x;
    mx = fmaxf(mx, x);
  }
  mx = warp_max(mx);
  bad = warp_sum(bad);  // NaN when a chunk's is
  const float m_use = mx == -INFINITY ? 0.f : mx;
  float sum = 0.f;
  for (int c = lane; c < chunks; c += 32) sum += exp2f(p.part_lse[at + c] - m_use);
  sum = warp_sum(sum);
  float acc[DC];
#pragma unroll
  for (int d = 0; d < DC; ++d) acc[d] = 0.f;
#pragma unroll 4
  for (int c = warp; c < chunks; c += C_WARPS) {
    const float w = exp2f(p.part_lse[at + c] - m_use);
#pragma unroll
    for (int d = 0; d < DC; ++d)
      if (d * 32 + lane < p.D) acc[d] = fmaf(w, p.part_o[(at + c) * p.D + d * 32 + lane], acc[d]);
  }
#pragma unroll
  for (int d = 0; d < DC; ++d) sm[warp][d * 32 + lane] = acc[d];
  __syncthreads();
  const float inv = (sum > 0.f ? 1.f / sum : 0.f) + bad;
  T* dst = static_cast<T*>(p.o) + (int64_t)row * p.so_t + (int64_t)h * p.so_h;
  for (int d = threadIdx.x; d < p.D; d += C_WARPS * 32) {
    float a = 0.f;
#pragma unroll
    for (int w = 0; w < C_WARPS; ++w) a += sm[w][d];
    a *= inv;
    dst[d] = from_f<T>(p.v_scale != nullptr ? clamp_finite<T>(a) : a);
  }
  if (p.lse != nullptr && threadIdx.x == 0)
    p.lse[(int64_t)h * p.T + row] =
        (sum > 0.f ? (mx + log2f(sum)) * 0.69314718055994531f : -INFINITY) + bad;
}

int launch_combine(const Params& p, int rows_per_tile, int tk, int dtype, cudaStream_t st) {
  const int64_t blocks = (int64_t)p.max_q * p.Hq;
  return LSB_DISPATCH_DTYPE(dtype, T, [&] {
    auto go = [&](auto dc) -> int {
      LSB_CUDA_OK(launch_kernel(paged_combine_kernel<T, decltype(dc)::value>,
                                dim3((unsigned)blocks, (unsigned)p.S), dim3(C_WARPS * 32), 0, st, p,
                                rows_per_tile, tk),
                  "paged_attn combine");
      return LSB_OK;
    };
    if (p.D <= 64) return go(std::integral_constant<int, 2>{});
    if (p.D <= 128) return go(std::integral_constant<int, 4>{});
    return go(std::integral_constant<int, 8>{});
  });
}

// -------------------------------------------------------------- dispatch ---
// How a call's keys are cut, from its sizes alone: with fewer query tiles
// than the GPU holds CTAs (8 on each of a B200's 148 SMs for the CUDA-core
// kernel), each tile's keys go to P CTAs of `chunk` keys.
struct Plan {
  int chunk, P;
};

static Plan plan_split(int64_t tiles, int64_t max_keys, int64_t want, int64_t min_chunk) {
  int64_t P = tiles > 0 ? std::max<int64_t>(1, want / tiles) : 1;
  int64_t chunk = (max_keys + P - 1) / P;
  chunk = std::max<int64_t>(min_chunk, (chunk + 127) / 128 * 128);
  P = std::max<int64_t>(1, (max_keys + chunk - 1) / chunk);
  return {(int)std::min<int64_t>(chunk, 1 << 30), (int)P};
}

// Keys a row tile may visit: the block table's capacity, or with a window the
// window, the tile's own rows and the sinks (each rounded up to a key tile).
static int64_t max_visible(int64_t max_q, int64_t max_keys, int64_t window, int64_t sinks) {
  if (window <= 0 || window >= max_keys || sinks >= max_keys) return max_keys;
  return std::min<int64_t>(max_keys, window + max_q + sinks + 3 * 128);
}

static Plan plan_simt(int64_t S, int64_t max_q, int64_t Hkv, int64_t G, int64_t keys) {
  const int64_t SR = S_WARPS * simt_rows(S, Hkv, max_q * G);
  return plan_split(S * Hkv * ((max_q * G + SR - 1) / SR), keys, 8 * 148, 128);
}

// Pairs up to which the few-rows kernel is taken where it serves the call: one
// of its tiles. Measured against the tcgen05 kernel, bf16, 8 cache heads of 128 and 4
// query heads each: 32 sequences of 512-4096 keys with 1-5 / 5 / 6 new tokens 82 /
// 91 / 95 us against 94 / 90 / 91, over e4m3 91 / 101 / 106 against 120; 16 heads of
// 64, 20 pairs 110 against 127; above, 32 pairs 90 against 74. One sequence would
// cross at 16 pairs (16000 keys: 17 / 23 us at 16 / 24 pairs against 20). So one
// bound for both caches and all batches gives up 1 to 4% over a 16-bit cache where
// every sequence brings 20 to 24 pairs, and 15% for one sequence, for the 11 to
// 24% that ragged batches and e4m3 gain.
constexpr int64_t ROWS_MAX_PAIRS = 24;

// The few-rows kernel's chunks: as many as give 3 CTAs per SM, of at most 1024
// keys so that ragged batches end together (and at least a 64th of the span:
// what the join reads). At 512 / 768 / 1024 / 1536 / 2048 keys: 64 sequences of
// 512-4096 e4m3 keys, 16 heads of 128, 131 / 124 / 117 / 119 / 115 us; of 4096
// keys each 218 / 202 / 196 / 193 / 196; 32 sequences of drafted tokens, 16-bit,
// 86 / 79 / 80 / 80 / 82.
static Plan plan_rows(int64_t S, int64_t max_q, int64_t Hkv, int64_t G, int64_t keys) {
  if (max_q * G > ROWS_MAX_PAIRS) return {1 << 30, 1};
  const int64_t R = rows_tile(max_q * G);
  const int64_t tiles = S * Hkv * ((max_q * G + R - 1) / R);
  const int64_t P = std::max<int64_t>(1, 3 * 148 / tiles);
  int64_t chunk = std::min<int64_t>(1024, ((keys + P - 1) / P + 127) / 128 * 128);
  chunk = std::max<int64_t>(chunk, (keys / std::max<int64_t>(64, P) + 127) / 128 * 128);
  return {(int)std::min<int64_t>(chunk, 1 << 30),
          (int)std::max<int64_t>(1, (keys + chunk - 1) / chunk)};
}

// Pairs of a CTA of the tcgen05 kernel: two query tiles.
static int64_t tc_pairs(int64_t G) { return 2 * std::max<int64_t>(1, 128 / G) * G; }

static Plan plan_tc(int64_t S, int64_t max_q, int64_t Hkv, int64_t G, int64_t keys) {
  const int64_t items = S * Hkv * ((max_q * G + tc_pairs(G) - 1) / tc_pairs(G));
  return plan_split(items, keys, 148, 512);
}

}  // namespace pa
}  // namespace lsb

extern "C" int64_t lsb_paged_attn_workspace_size(int64_t num_seqs, int64_t total_q,
                                                 int64_t max_seqlen_q, int64_t Hq, int64_t Hkv,
                                                 int64_t D, int64_t max_blocks_per_seq,
                                                 int64_t block_size, int64_t window,
                                                 int64_t num_sinks) {
  using namespace lsb::pa;
  if (num_seqs <= 0 || total_q <= 0 || max_seqlen_q <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 ||
      D <= 0 || max_blocks_per_seq <= 0 || block_size <= 0)
    return 0;
  const int64_t keys =
      max_visible(max_seqlen_q, max_blocks_per_seq * block_size, window, num_sinks);
  const int64_t G = Hq / Hkv;
  const int64_t P = std::max(plan_simt(num_seqs, max_seqlen_q, Hkv, G, keys).P,
                             std::max(plan_rows(num_seqs, max_seqlen_q, Hkv, G, keys).P,
                                      plan_tc(num_seqs, max_seqlen_q, Hkv, G, keys).P));
  if (P <= 1) return 0;
  return lsb::align256(4 * total_q * Hq * P) + 4 * total_q * Hq * P * D;
}

extern "C" int lsb_paged_attn(const void* q, const void* k_cache, const void* v_cache,
                              const void* k_scale, const void* v_scale,
                              const int32_t* block_tables, const int32_t* context_lens,
                              const int32_t* cu_seqlens_q, void* o, float* lse, int64_t num_seqs,
                              int64_t total_q, int64_t max_seqlen_q, int64_t Hq, int64_t Hkv,
                              int64_t D, int64_t max_blocks_per_seq, int64_t block_size,
                              int64_t num_blocks, int64_t sq_t, int64_t sq_h, int64_t so_t,
                              int64_t so_h, int64_t window, int64_t num_sinks, float scale,
                              int dtype, int kv_dtype, int impl, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  using namespace lsb::pa;
  LSB_CHECK_ARG(num_seqs >= 0 && total_q >= 0 && max_seqlen_q >= 0 && Hq > 0 && Hkv > 0 && D > 0 &&
                    max_blocks_per_seq > 0 && num_blocks > 0,
                "paged_attn: bad sizes num_seqs=%lld total_q=%lld max_seqlen_q=%lld Hq=%lld Hkv=%lld "
                "D=%lld max_blocks=%lld num_blocks=%lld",
                (long long)num_seqs, (long long)total_q, (long long)max_seqlen_q, (long long)Hq,
                (long long)Hkv, (long long)D, (long long)max_blocks_per_seq, (long long)num_blocks);
  LSB_CHECK_ARG(Hq % Hkv == 0, "paged_attn: %lld query heads are no multiple of the cache's %lld",
                (long long)Hq, (long long)Hkv);
  LSB_CHECK_ARG(block_size > 0 && (block_size & (block_size - 1)) == 0,
                "paged_attn: block_size %lld must be a power of two", (long long)block_size);
  const int esz = lsb::dtype_size(dtype);
  LSB_CHECK_ARG(esz > 0, "paged_attn: unsupported dtype %d", dtype);
  const bool fp8 = kv_dtype == LSB_DTYPE_E4M3;
  LSB_CHECK_ARG(fp8 || kv_dtype == dtype, "paged_attn: the cache holds q's type or e4m3, got %d", kv_dtype);
  LSB_CHECK_ARG(window >= 0 && num_sinks >= 0 && (window > 0 || num_sinks == 0),
                "paged_attn: window %lld and num_sinks %lld: neither is negative, and sinks need a window",
                (long long)window, (long long)num_sinks);
  LSB_CHECK_ARG(max_seqlen_q <= total_q, "paged_attn: max_seqlen_q %lld above total_q %lld",
                (long long)max_seqlen_q, (long long)total_q);
  LSB_CHECK_ARG(cu_seqlens_q != nullptr || total_q == num_seqs,
                "paged_attn: without cu_seqlens_q there is one row per sequence");
  if (num_seqs == 0 || total_q == 0 || max_seqlen_q == 0) return LSB_OK;
  LSB_CHECK_ARG(q && k_cache && v_cache && block_tables && context_lens && o,
                "paged_attn: null pointer");
  LSB_CHECK_ARG(!fp8 || (k_scale && v_scale), "paged_attn: an e4m3 cache needs its scales");
  constexpr int64_t kMax = 1LL << 30;
  LSB_CHECK_ARG(num_seqs <= 65535 && total_q < kMax && Hq < 65536 && num_blocks < kMax &&
                    total_q * Hq < kMax && max_blocks_per_seq < kMax && block_size < kMax &&
                    max_blocks_per_seq * block_size < kMax,
                "paged_attn: sizes too large (65535 sequences; 2^30 rows x heads, blocks, keys per "
                "sequence)");
  if (D > 256) {
    lsb::set_error("paged_attn: head dim %lld above 256", (long long)D);
    return LSB_ERR_UNSUPPORTED;
  }
  LSB_CHECK_ARG(impl == LSB_IMPL_AUTO || impl == LSB_IMPL_SIMT || impl == LSB_IMPL_ROWS ||
                    impl == LSB_IMPL_TCGEN05,
                "paged_attn: bad impl %d", impl);

  Params p = {};
  p.q = q; p.k_cache = k_cache; p.v_cache = v_cache;
  p.k_scale = static_cast<const uint8_t*>(k_scale);
  p.v_scale = static_cast<const uint8_t*>(v_scale);
  p.block_tables = block_tables; p.context_lens = context_lens; p.cu_seqlens_q = cu_seqlens_q;
  p.o = o; p.lse = lse;
  p.sq_t = sq_t; p.sq_h = sq_h; p.so_t = so_t; p.so_h = so_h;
  p.S = (int)num_seqs; p.T = (int)total_q; p.max_q = (int)max_seqlen_q;
  p.Hq = (int)Hq; p.Hkv = (int)Hkv; p.G = (int)(Hq / Hkv); p.D = (int)D;
  p.max_blocks = (int)max_blocks_per_seq; p.num_blocks = (int)num_blocks;
  while ((1LL << p.bs_log2) < block_size) ++p.bs_log2;
  // A window or sinks past every position change nothing.
  p.window = (int)std::min<int64_t>(window, kMax);
  p.sinks = (int)std::min<int64_t>(num_sinks, kMax);
  p.scale_log2 = scale * LOG2E;
  const int64_t keys = max_visible(max_seqlen_q, max_blocks_per_seq * block_size, p.window, p.sinks);
  const Plan rows_plan = plan_rows(num_seqs, max_seqlen_q, Hkv, p.G, keys);
  const Plan tc_plan = plan_tc(num_seqs, max_seqlen_q, Hkv, p.G, keys);
  p.P = std::max(rows_plan.P, tc_plan.P);  // (the grids' limits)
  const bool rows_ok = rows_eligible(p, dtype), tc_ok = tc_eligible(p, dtype, fp8);
  LSB_CHECK_ARG(impl != LSB_IMPL_ROWS || rows_ok,
                "paged_attn: the few-rows kernel needs bf16/fp16, D in {64,128}, pages of 8 keys or "
                "more, q strides that are multiples of 4 elements and 16-byte aligned caches");
  LSB_CHECK_ARG(impl != LSB_IMPL_TCGEN05 || tc_ok,
                "paged_attn: the tcgen05 kernel needs bf16/fp16, D in {64,128}, pages of 8 keys or "
                "more, a positive scale, at most 128 heads per group and 16-byte aligned tensors "
                "and strides");
  // Few rows: bandwidth decides, and the few-rows kernel reads the cache at
  // full rate. Many: the tensor cores. Tensors whose alignment rules a kernel
  // out take the other one, then the CUDA cores.
  if (impl == LSB_IMPL_AUTO) {
    const bool few = max_seqlen_q * p.G <= ROWS_MAX_PAIRS;
    impl = rows_ok && (few || !tc_ok) ? LSB_IMPL_ROWS : tc_ok ? LSB_IMPL_TCGEN05 : LSB_IMPL_SIMT;
  }
  const Plan plan = impl == LSB_IMPL_ROWS      ? rows_plan
                    : impl == LSB_IMPL_TCGEN05 ? tc_plan
                                               : plan_simt(num_seqs, max_seqlen_q, Hkv, p.G, keys);
  p.chunk = plan.chunk;
  p.P = plan.P;
  if (p.P > 1) {
    const int64_t need = lsb_paged_attn_workspace_size(num_seqs, total_q, max_seqlen_q, Hq, Hkv, D,
                                                       max_blocks_per_seq, block_size, window,
                                                       num_sinks);
    LSB_CHECK_ARG(workspace != nullptr && workspace_bytes >= need &&
                      (reinterpret_cast<uintptr_t>(workspace) & 31) == 0,
                  "paged_attn: workspace of %lld bytes (32-byte aligned) required, got %lld",
                  (long long)need, (long long)workspace_bytes);
    p.part_lse = static_cast<float*>(workspace);
    p.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                        lsb::align256(4 * total_q * Hq * p.P));
  }
  cudaStream_t st = (cudaStream_t)stream;
  if (impl == LSB_IMPL_ROWS) {
    const int rc = launch_rows(p, dtype, fp8, st);
    if (rc != LSB_OK || p.P == 1) return rc;
    return launch_combine(p, rows_tile(max_seqlen_q * p.G), rows_tk(fp8), dtype, st);
  }
  if (impl == LSB_IMPL_TCGEN05) {
    const int rc = launch_tc(p, dtype, fp8, st);
    if (rc != LSB_OK || p.P == 1) return rc;
    return launch_combine(p, (int)tc_pairs(p.G), TC_TK, dtype, st);
  }
  const int rc = launch_simt(p, dtype, fp8, st);
  if (rc != LSB_OK || p.P == 1) return rc;
  return launch_combine(p, S_WARPS * simt_rows(num_seqs, Hkv, max_seqlen_q * p.G), STK, dtype, st);
}
