// Quantised paged KV cache: writing rows, writing rows with the rotary
// embedding fused in, and reading rows back (all HBM-bound).
//
// Layout, per layer: K and V as e4m3 [num_blocks, H, block_size, D] and their
// scales as e8m0 [num_blocks, H, block_size] (fp8.cuh has the format), so the
// block tables and slots of the 16-bit cache address it unchanged.
//
// Vectorised kernels: LPR = D * sizeof(T) / 16 lanes hold one row of K, V or
// q as one 16-byte vector each, so a warp's loads are whole contiguous
// sectors; the row's maximum is a butterfly over those lanes, and a lane's 8
// (16-bit types) or 4 (fp32) bytes make the row's 32- to 256-byte run in the
// cache. The rotary partner x[i +- D/2] sits LPR / 2 lanes away and comes by
// shuffle. Any other head dim or alignment takes the warp-per-row kernels.
//
// Bound by HBM: 16384 tokens of 16 heads of 128 in bf16 written and read back, two
// launches, 63.7 us for 404 MB (6.3 TB/s, 97% of the copy rate); 12001 tokens
// rotated, written and read back 66.3 us for 400 MB (6.0 TB/s). A decode step's 64
// tokens take 3 us a launch.
#include "common.cuh"
#include "fp8.cuh"

#include <type_traits>

namespace lsb {
namespace kvq {

constexpr int THREADS = 256;

// n / d for n < 2^31 by a multiplication (round-up method: with s the smallest
// shift that has 2^s >= d and m = floor(2^32 (2^s - d) / d) + 1, n / d =
// (mulhi(n, m) + n) >> s).
struct FastDiv {
  uint32_t d, m, s;
  explicit FastDiv(uint32_t div) : d(div), s(0) {
    while ((1ull << s) < d) ++s;
    m = (uint32_t)((((1ull << s) - d) << 32) / d + 1);
  }
  __device__ __forceinline__ void split(uint32_t n, uint32_t& q, uint32_t& r) const {
    q = (__umulhi(n, m) + n) >> s;
    r = n - q * d;
  }
};

// Where one token's rows go: row `cell` of the cache seen as [blocks * H * bs]
// rows of D, or -1 for none. The divisions by the page size are shifts when
// it is a power of two (64-bit divisions were a third of the kernels' issue
// slots).
struct CellOf {
  const int64_t* slots;          // [T] block * bs + offset, or NULL
  const int64_t* positions;      // with block tables
  const int32_t* block_tables;   // [T, max_blocks]
  int64_t max_blocks;
  int64_t num_blocks;
  int bs, bs_log2;               // bs_log2 < 0: no power of two
  uint32_t H;
  CellOf(const int64_t* sl, const int64_t* pos, const int32_t* bt, int64_t mb, int64_t nb, int64_t b,
         int64_t heads)
      : slots(sl), positions(pos), block_tables(bt), max_blocks(mb), num_blocks(nb), bs((int)b),
        bs_log2(-1), H((uint32_t)heads) {
    if ((b & (b - 1)) == 0)
      for (bs_log2 = 0; (1LL << bs_log2) < b;) ++bs_log2;
  }
  __device__ __forceinline__ int64_t page(int64_t x) const { return bs_log2 >= 0 ? x >> bs_log2 : x / bs; }
  __device__ __forceinline__ int64_t operator()(int64_t t, uint32_t h) const {
    int64_t blk, at;
    if (slots != nullptr) {
      const int64_t s = slots[t];
      if (s < 0 || s >= num_blocks * bs) return -1;
      blk = page(s);
      at = s - blk * bs;
    } else {
      const int64_t pos = positions[t];
      const int64_t i = page(pos);
      if (pos < 0 || i >= max_blocks) return -1;
      blk = block_tables[t * max_blocks + i];
      if (blk < 0 || blk >= num_blocks) return -1;
      at = pos - i * bs;
    }
    return (blk * H + h) * bs + at;
  }
};

// The magnitude of a 16-byte vector's largest element as the bits of its
// type (ordered like the values; infinity and NaN on top), by packed integer
// maxima.
template <typename T>
__device__ __forceinline__ uint32_t top_bits(const Vec16<T>& x) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&x);
  uint32_t m = 0;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, w[i] & 0x7fffffffu);
    return m;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
    return max(m >> 16, m & 0xffffu);
  }
}

template <typename T> struct Bits;
template <> struct Bits<float> {
  static constexpr uint32_t inf = 0x7f800000u;
  static __device__ __forceinline__ float value(uint32_t b) { return __uint_as_float(b); }
};
template <> struct Bits<__nv_bfloat16> {
  static constexpr uint32_t inf = 0x7f80u;
  static __device__ __forceinline__ float value(uint32_t b) { return __uint_as_float(b << 16); }
};
template <> struct Bits<__half> {
  static constexpr uint32_t inf = 0x7c00u;
  static __device__ __forceinline__ float value(uint32_t b) { return __half2float(__ushort_as_half((unsigned short)b)); }
};

template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Quantises the row whose LANES lanes hold `x`, writing 8 (16-bit types) or 4
// bytes per lane and the scale byte. Every lane of the warp takes part;
// `cell` < 0: the row is not stored.
template <int LANES, typename T>
__device__ __forceinline__ void store_row(const Vec16<T>& x, int64_t cell, int lane_in_row, int D,
                                          uint8_t* __restrict__ cache, uint8_t* __restrict__ scale) {
  constexpr int VEC = 16 / sizeof(T);
  uint32_t top = top_bits(x);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  float amax = Bits<T>::value(top), f[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) f[e] = to_f(x.v[e]);
  const bool special = __any_sync(0xffffffffu, top >= Bits<T>::inf);
  if (special) {  // some row of the warp holds a NaN or an infinity
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) m = fmaxf(m, finite_abs(f[e]));
    amax = lanes_max<LANES>(m);
  }
  const int e8 = e8m0_of_amax(amax);
  const float inv = e8m0_inverse(e8);
  if (special) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = scaled_for_e4m3(f[e], inv);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; e += 2) {
      const float2 y = __fmul2_rn(make_float2(f[e], f[e + 1]), make_float2(inv, inv));
      f[e] = y.x;
      f[e + 1] = y.y;
    }
  }
  uint32_t w[VEC / 4];
#pragma unroll
  for (int i = 0; i < VEC / 4; ++i)
    w[i] = cvt_e4m3x2(f[4 * i], f[4 * i + 1]) | (cvt_e4m3x2(f[4 * i + 2], f[4 * i + 3]) << 16);
  if (cell < 0) return;
  uint8_t* row = cache + cell * D + lane_in_row * VEC;
  if constexpr (VEC == 8)
    *reinterpret_cast<uint2*>(row) = make_uint2(w[0], w[1]);
  else
    *reinterpret_cast<uint32_t*>(row) = w[0];
  if (lane_in_row == 0) scale[cell] = (uint8_t)e8;
}

// A group of lanes writes QPT heads of one token, their loads all in flight.
constexpr int QPT = 2;

template <typename T, int D>
__global__ void __launch_bounds__(THREADS)
quantize_vec_kernel(const T* __restrict__ k, const T* __restrict__ v, uint8_t* __restrict__ k_cache,
                    uint8_t* __restrict__ v_cache, uint8_t* __restrict__ k_scale,
                    uint8_t* __restrict__ v_scale, const CellOf cell_of, uint32_t units,
                    const FastDiv head_groups, int64_t sk_t, int64_t sk_h, int64_t sv_t, int64_t sv_h) {
  allow_dependents();
  wait_prerequisites();
  constexpr int VEC = 16 / sizeof(T);
  constexpr int LPR = D / VEC;
  const uint64_t g = (uint64_t)blockIdx.x * THREADS + threadIdx.x;
  const bool in = g / LPR < units;
  const int c = (int)(g % LPR);
  uint32_t t, hg;
  head_groups.split(in ? (uint32_t)(g / LPR) : units - 1, t, hg);  // lanes past the end repeat the last unit
  const uint32_t H = cell_of.H;
  Vec16<T> kx[QPT], vx[QPT];
#pragma unroll
  for (int i = 0; i < QPT; ++i) {
    const uint32_t h = min(hg * QPT + i, H - 1);
    kx[i] = ld_vec16_stream(k + t * sk_t + h * sk_h + c * VEC);
    vx[i] = ld_vec16_stream(v + t * sv_t + h * sv_h + c * VEC);
  }
  const int64_t cell = in ? cell_of(t, hg * QPT) : -1;
#pragma unroll
  for (int i = 0; i < QPT; ++i) {
    const int64_t at = cell >= 0 && hg * QPT + i < H ? cell + (int64_t)i * cell_of.bs : -1;
    store_row<LPR>(kx[i], at, c, D, k_cache, k_scale);
    store_row<LPR>(vx[i], at, c, D, v_cache, v_scale);
  }
}

// One warp per (token, head) row, any head dim and alignment.
template <typename T>
__device__ __forceinline__ void store_row_any(const T* __restrict__ x, int D, uint8_t* __restrict__ row,
                                              uint8_t* __restrict__ scale) {
  const int lane = threadIdx.x & 31;
  float amax = 0.f;
  for (int d = lane; d < D; d += 32) amax = fmaxf(amax, finite_abs(to_f(x[d])));
  const int e8 = e8m0_of_amax(warp_max(amax));
  const float inv = e8m0_inverse(e8);
  for (int d = lane; d < D; d += 32)
    row[d] = (uint8_t)cvt_e4m3x2(scaled_for_e4m3(to_f(x[d]), inv), 0.f);
  if (lane == 0) *scale = (uint8_t)e8;
}

template <typename T>
__global__ void __launch_bounds__(THREADS)
quantize_any_kernel(const T* __restrict__ k, const T* __restrict__ v, uint8_t* __restrict__ k_cache,
                    uint8_t* __restrict__ v_cache, uint8_t* __restrict__ k_scale,
                    uint8_t* __restrict__ v_scale, const CellOf cell_of, uint32_t rows, const FastDiv heads,
                    int D, int64_t sk_t, int64_t sk_h, int64_t sv_t, int64_t sv_h) {
  allow_dependents();
  wait_prerequisites();
  const uint64_t row = ((uint64_t)blockIdx.x * THREADS + threadIdx.x) >> 5;
  if (row >= rows) return;
  uint32_t t, h;
  heads.split((uint32_t)row, t, h);
  const int64_t cell = cell_of(t, h);
  if (cell < 0) return;
  store_row_any(k + t * sk_t + h * sk_h, D, k_cache + cell * D, k_scale + cell);
  store_row_any(v + t * sv_t + h * sv_h, D, v_cache + cell * D, v_scale + cell);
}

// ------------------------------------------------------------ read back ---
// Words of e4m3 times the row's scale f, in T. Only scales near the top of T's
// range can take a product past it (448 f above T's largest).
template <typename T, int W>
__device__ __forceinline__ void dequantize_vec(const uint32_t (&w)[W], float f, Vec16<T>& out) {
  const bool top = !(f * 448.f <= FiniteMax<T>::v);
#pragma unroll
  for (int i = 0; i < W; ++i) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float2 y = __fmul2_rn(f16x2_to_float2(cvt_e4m3x2_f16x2((uint16_t)(w[i] >> (16 * e)))),
                            make_float2(f, f));
      if (top) {
        y.x = clamp_finite<T>(y.x);
        y.y = clamp_finite<T>(y.y);
      }
      out.v[4 * i + 2 * e] = from_f<T>(y.x);
      out.v[4 * i + 2 * e + 1] = from_f<T>(y.y);
    }
  }
}

// A group of lanes reads HPT heads of one token: one trip for the slot, then
// all their loads at once.
constexpr int HPT = 4;

template <typename T, int D>
__global__ void __launch_bounds__(THREADS)
dequantize_vec_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache,
                      const uint8_t* __restrict__ k_scale, const uint8_t* __restrict__ v_scale,
                      const CellOf cell_of, T* __restrict__ k_out, T* __restrict__ v_out,
                      uint32_t units, const FastDiv head_groups) {
  allow_dependents();
  wait_prerequisites();
  constexpr int VEC = 16 / sizeof(T), W = VEC / 4;
  constexpr int LPR = D / VEC;
  const uint64_t g = (uint64_t)blockIdx.x * THREADS + threadIdx.x;
  if (g / LPR >= units) return;
  const int c = (int)(g % LPR);
  uint32_t t, hg;
  head_groups.split((uint32_t)(g / LPR), t, hg);
  const uint32_t h0 = hg * HPT, H = cell_of.H;
  const int64_t cell = cell_of(t, h0);
  uint32_t kw[HPT][W], vw[HPT][W];
  int ke[HPT], ve[HPT];
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    if (cell < 0 || h0 + i >= H) {
      ke[i] = ve[i] = 127;
#pragma unroll
      for (int w = 0; w < W; ++w) kw[i][w] = vw[i][w] = 0u;
      continue;
    }
    const int64_t at = cell + (int64_t)i * cell_of.bs;
    ke[i] = k_scale[at];
    ve[i] = v_scale[at];
    if constexpr (VEC == 8) {
      const uint2 a = __ldcs(reinterpret_cast<const uint2*>(k_cache + at * D + c * VEC));
      const uint2 b = __ldcs(reinterpret_cast<const uint2*>(v_cache + at * D + c * VEC));
      kw[i][0] = a.x; kw[i][1] = a.y; vw[i][0] = b.x; vw[i][1] = b.y;
    } else {
      kw[i][0] = __ldcs(reinterpret_cast<const uint32_t*>(k_cache + at * D + c * VEC));
      vw[i][0] = __ldcs(reinterpret_cast<const uint32_t*>(v_cache + at * D + c * VEC));
    }
  }
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    if (h0 + i >= H) break;
    Vec16<T> ko, vo;
    dequantize_vec(kw[i], e8m0_to_float(ke[i]), ko);
    dequantize_vec(vw[i], e8m0_to_float(ve[i]), vo);
    const int64_t o = ((int64_t)t * H + h0 + i) * D + c * VEC;
    __stcs(reinterpret_cast<uint4*>(k_out + o), *reinterpret_cast<const uint4*>(&ko));
    __stcs(reinterpret_cast<uint4*>(v_out + o), *reinterpret_cast<const uint4*>(&vo));
  }
}

template <typename T>
__global__ void __launch_bounds__(THREADS)
dequantize_any_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache,
                      const uint8_t* __restrict__ k_scale, const uint8_t* __restrict__ v_scale,
                      const CellOf cell_of, T* __restrict__ k_out, T* __restrict__ v_out,
                      uint32_t rows, const FastDiv heads, int D) {
  allow_dependents();
  wait_prerequisites();
  const uint64_t row = ((uint64_t)blockIdx.x * THREADS + threadIdx.x) >> 5;
  if (row >= rows) return;
  const int lane = threadIdx.x & 31;
  uint32_t t, h;
  heads.split((uint32_t)row, t, h);
  const int64_t cell = cell_of(t, h);
  const float ks = cell < 0 ? 0.f : e8m0_to_float(k_scale[cell]);
  const float vs = cell < 0 ? 0.f : e8m0_to_float(v_scale[cell]);
  for (int d = lane; d < D; d += 32) {
    float a = 0.f, b = 0.f;
    if (cell >= 0) {
      a = f16x2_to_float2(cvt_e4m3x2_f16x2(k_cache[cell * D + d])).x * ks;
      b = f16x2_to_float2(cvt_e4m3x2_f16x2(v_cache[cell * D + d])).x * vs;
    }
    k_out[(int64_t)row * D + d] = from_f<T>(clamp_finite<T>(a));
    v_out[(int64_t)row * D + d] = from_f<T>(clamp_finite<T>(b));
  }
}

// ------------------------------------------------- rotary + quantisation ---
// rotate_half(x) = [-x2, x1]; each product and the sum rounded to T, as the
// 16-bit cache's rotary write does, so q and the k that is quantised equal
// its q and k bit for bit.
template <typename T>
__device__ __forceinline__ T rope1(float x, float turned, float c, float s) {
  const float a = to_f(from_f<T>(__fmul_rn(x, c)));
  const float b = to_f(from_f<T>(__fmul_rn(turned, s)));
  return from_f<T>(__fadd_rn(a, b));
}

// The same for a 16-byte vector; `s` has its sign turned where the partner's is.
// Products and sums of 16-bit pairs round once, like the scalar form: an fp32
// product of two 16-bit values is exact, and their fp32 sum is too, or lies too
// far from a halfway point for its rounding to matter.
template <typename T>
__device__ __forceinline__ void rope_vec(const Vec16<T>& x, const Vec16<T>& p, const Vec16<T>& c,
                                         const Vec16<T>& s, Vec16<T>& out) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) out.v[e] = rope1<T>(x.v[e], p.v[e], c.v[e], s.v[e]);
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T2 *x2 = reinterpret_cast<const T2*>(&x), *p2 = reinterpret_cast<const T2*>(&p);
    const T2 *c2 = reinterpret_cast<const T2*>(&c), *s2 = reinterpret_cast<const T2*>(&s);
    T2* o2 = reinterpret_cast<T2*>(&out);
#pragma unroll
    for (int i = 0; i < 4; ++i) o2[i] = __hadd2_rn(__hmul2_rn(x2[i], c2[i]), __hmul2_rn(p2[i], s2[i]));
  }
}

struct RopeArgs {
  int64_t s_s, s_part, s_h;  // qkv strides
  int64_t s_pos, max_pos;    // cos / sin row stride and rows
  const int64_t* positions;
  int32_t* context_lens;     // may be NULL
};

template <typename T, int D>
__global__ void __launch_bounds__(THREADS)
rope_quantize_vec_kernel(const T* __restrict__ qkv, const T* __restrict__ cos_t,
                         const T* __restrict__ sin_t, const RopeArgs a, T* __restrict__ q_out,
                         T* __restrict__ k_out, uint8_t* __restrict__ k_cache,
                         uint8_t* __restrict__ v_cache, uint8_t* __restrict__ k_scale,
                         uint8_t* __restrict__ v_scale, const CellOf cell_of, uint32_t units,
                         const FastDiv head_groups) {
  allow_dependents();
  wait_prerequisites();
  constexpr int VEC = 16 / sizeof(T);
  constexpr int LPR = D / VEC;
  static_assert(LPR >= 2 && LPR <= 32, "a row and its rotary partner live in one warp");
  const uint64_t g = (uint64_t)blockIdx.x * THREADS + threadIdx.x;
  const bool in = g / LPR < units;
  const int c = (int)(g % LPR);
  uint32_t t, hg;
  head_groups.split(in ? (uint32_t)(g / LPR) : units - 1, t, hg);
  const uint32_t h0 = hg * QPT, H = cell_of.H;
  Vec16<T> qx[QPT], kx[QPT], vx[QPT];
#pragma unroll
  for (int i = 0; i < QPT; ++i) {
    const T* x = qkv + t * a.s_s + min(h0 + i, H - 1) * a.s_h + c * VEC;
    qx[i] = ld_vec16_stream(x);
    kx[i] = ld_vec16_stream(x + a.s_part);
    vx[i] = ld_vec16_stream(x + 2 * a.s_part);
  }
  const int64_t pos = a.positions[t];
  // A position outside the table has no angle: q (and k_out) become NaN and
  // nothing is cached.
  const bool known = pos >= 0 && pos < a.max_pos;
  const Vec16<T> cx = ld_vec16(cos_t + (known ? pos : 0) * a.s_pos + c * VEC);
  const Vec16<T> sx = ld_vec16(sin_t + (known ? pos : 0) * a.s_pos + c * VEC);
  const int64_t cell = in && known ? cell_of(t, h0) : -1;
  if (in && h0 == 0 && c == 0 && a.context_lens != nullptr)
    a.context_lens[t] = known ? (int32_t)(pos + 1) : 0;
  Vec16<T> sn;  // the first half takes -x2, the second x1
  {
    const uint32_t flip = c < LPR / 2 ? (sizeof(T) == 4 ? 0x80000000u : 0x80008000u) : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<uint32_t*>(&sn)[i] = reinterpret_cast<const uint32_t*>(&sx)[i] ^ flip;
  }
  auto turn = [&](const Vec16<T>& v, Vec16<T>& out) {
    Vec16<T> p;
    const uint32_t* src = reinterpret_cast<const uint32_t*>(&v);
    uint32_t* dst = reinterpret_cast<uint32_t*>(&p);
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i] = __shfl_xor_sync(0xffffffffu, src[i], LPR / 2);
    rope_vec(v, p, cx, sn, out);
    if (!known) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) out.v[e] = from_f<T>(__int_as_float(0x7fc00000));
    }
  };
#pragma unroll
  for (int i = 0; i < QPT; ++i) {
    const bool here = in && h0 + i < H;
    const int64_t o = ((int64_t)t * H + h0 + i) * D + c * VEC;
    const int64_t at = cell >= 0 && here ? cell + (int64_t)i * cell_of.bs : -1;
    Vec16<T> r;
    turn(qx[i], r);
    if (here) st_vec16(q_out + o, r);
    turn(kx[i], r);
    if (here && k_out != nullptr) st_vec16(k_out + o, r);
    store_row<LPR>(r, at, c, D, k_cache, k_scale);
    store_row<LPR>(vx[i], at, c, D, v_cache, v_scale);
  }
}

template <typename T>
__global__ void __launch_bounds__(THREADS)
rope_quantize_any_kernel(const T* __restrict__ qkv, const T* __restrict__ cos_t,
                         const T* __restrict__ sin_t, const RopeArgs a, T* __restrict__ q_out,
                         T* __restrict__ k_out, uint8_t* __restrict__ k_cache,
                         uint8_t* __restrict__ v_cache, uint8_t* __restrict__ k_scale,
                         uint8_t* __restrict__ v_scale, const CellOf cell_of, uint32_t rows,
                         const FastDiv heads, int D) {
  allow_dependents();
  wait_prerequisites();
  const uint64_t row = ((uint64_t)blockIdx.x * THREADS + threadIdx.x) >> 5;
  if (row >= rows) return;
  const int lane = threadIdx.x & 31, half = D / 2;
  uint32_t t, h;
  heads.split((uint32_t)row, t, h);
  const int64_t pos = a.positions[t];
  const bool known = pos >= 0 && pos < a.max_pos;
  const T* cs = cos_t + (known ? pos : 0) * a.s_pos;
  const T* sn = sin_t + (known ? pos : 0) * a.s_pos;
  const int64_t cell = known ? cell_of(t, h) : -1;
  if (h == 0 && lane == 0 && a.context_lens != nullptr)
    a.context_lens[t] = known ? (int32_t)(pos + 1) : 0;
  const T* q = qkv + t * a.s_s + h * a.s_h;
  auto turned = [&](const T* x, int d) -> T {
    if (!known) return from_f<T>(__int_as_float(0x7fc00000));
    const float p = d < half ? -to_f(x[d + half]) : to_f(x[d - half]);
    return rope1<T>(to_f(x[d]), p, to_f(cs[d]), to_f(sn[d]));
  };
  float amax = 0.f;
  for (int d = lane; d < D; d += 32) {
    q_out[(int64_t)row * D + d] = turned(q, d);
    const T kr = turned(q + a.s_part, d);
    if (k_out != nullptr) k_out[(int64_t)row * D + d] = kr;
    amax = fmaxf(amax, finite_abs(to_f(kr)));
  }
  if (cell < 0) return;
  const int e8 = e8m0_of_amax(warp_max(amax));
  const float inv = e8m0_inverse(e8);
  for (int d = lane; d < D; d += 32)  // the rotation again, instead of D registers
    k_cache[cell * D + d] =
        (uint8_t)cvt_e4m3x2(scaled_for_e4m3(to_f(turned(q + a.s_part, d)), inv), 0.f);
  if (lane == 0) k_scale[cell] = (uint8_t)e8;
  store_row_any(q + 2 * a.s_part, D, v_cache + cell * D, v_scale + cell);
}

// Blocks for `rows` rows of `lanes` lanes each; 0 when the grid cannot hold them.
static unsigned blocks_for(int64_t rows, int lanes) {
  const int64_t b = (rows * lanes + THREADS - 1) / THREADS;
  return b <= 0x7fffffff ? (unsigned)b : 0;
}

// Calls f(head dim constant) for the head dims the vectorised kernels serve.
template <typename T, class F>
static int with_dim(int64_t D, F&& f) {
  if (D == 64) return f(std::integral_constant<int, 64>{});
  if (D == 128) return f(std::integral_constant<int, 128>{});
  if constexpr (sizeof(T) == 2) {
    if (D == 256) return f(std::integral_constant<int, 256>{});
  } else {
    if (D == 32) return f(std::integral_constant<int, 32>{});
  }
  return -1;
}

static bool strides16(int esz, std::initializer_list<int64_t> s) {
  for (int64_t x : s)
    if ((x * esz) % 16 != 0) return false;
  return true;
}

static bool aligned(std::initializer_list<const void*> p, uintptr_t to) {
  for (const void* x : p)
    if ((reinterpret_cast<uintptr_t>(x) & (to - 1)) != 0) return false;
  return true;
}

static int check_sizes(const char* who, int64_t T, int64_t H, int64_t D, int64_t num_blocks,
                       int64_t block_size, int dtype) {
  LSB_CHECK_ARG(T >= 0 && H > 0 && D > 0 && num_blocks > 0 && block_size > 0,
                "%s: bad sizes T=%lld H=%lld D=%lld num_blocks=%lld block_size=%lld", who,
                (long long)T, (long long)H, (long long)D, (long long)num_blocks,
                (long long)block_size);
  LSB_CHECK_ARG(dtype_size(dtype) > 0, "%s: unsupported dtype %d", who, dtype);
  LSB_CHECK_ARG(D <= 65536 && block_size <= 0x7fffffff && num_blocks <= 0x7fffffff &&
                    H <= 0x7fffffff && T <= 0x7fffffff && T * H <= 0x7fffffff,
                "%s: sizes too large (T * H is limited to 2^31 - 1)", who);
  return LSB_OK;
}

}  // namespace kvq
}  // namespace lsb

extern "C" int lsb_kv_quantize(const void* k, const void* v, void* k_cache, void* v_cache,
                               void* k_scale, void* v_scale, const int64_t* slot_mapping, int64_t T,
                               int64_t H, int64_t D, int64_t num_blocks, int64_t block_size,
                               int64_t sk_t, int64_t sk_h, int64_t sv_t, int64_t sv_h, int dtype,
                               void* stream) {
  using namespace lsb::kvq;
  if (int rc = check_sizes("kv_quantize", T, H, D, num_blocks, block_size, dtype)) return rc;
  if (T == 0) return LSB_OK;
  LSB_CHECK_ARG(k && v && k_cache && v_cache && k_scale && v_scale && slot_mapping,
                "kv_quantize: null pointer");
  const CellOf cell_of(slot_mapping, nullptr, nullptr, 0, num_blocks, block_size, H);
  const FastDiv heads((uint32_t)H);
  const uint32_t rows = (uint32_t)(T * H);
  cudaStream_t st = (cudaStream_t)stream;
  return LSB_DISPATCH_DTYPE(dtype, Tt, [&] {
    const bool vec = aligned({k, v}, 16) && aligned({k_cache, v_cache}, 8) &&
                     strides16(sizeof(Tt), {sk_t, sk_h, sv_t, sv_h});
    const int rc = vec ? with_dim<Tt>(D, [&](auto dim) -> int {
      constexpr int DD = decltype(dim)::value;
      const uint32_t groups = (uint32_t)((H + QPT - 1) / QPT), units = (uint32_t)T * groups;
      const unsigned blocks = blocks_for(units, DD * (int)sizeof(Tt) / 16);
      LSB_CHECK_ARG(blocks > 0, "kv_quantize: too many rows");
      LSB_CUDA_OK(lsb::launch_kernel(quantize_vec_kernel<Tt, DD>, dim3(blocks), dim3(THREADS), 0, st,
                                     (const Tt*)k, (const Tt*)v, (uint8_t*)k_cache,
                                     (uint8_t*)v_cache, (uint8_t*)k_scale, (uint8_t*)v_scale,
                                     cell_of, units, FastDiv(groups), sk_t, sk_h, sv_t, sv_h),
                  "kv_quantize");
      return LSB_OK;
    }) : -1;
    if (rc >= 0) return rc;
    const unsigned blocks = blocks_for(rows, 32);
    LSB_CHECK_ARG(blocks > 0, "kv_quantize: too many rows");
    LSB_CUDA_OK(lsb::launch_kernel(quantize_any_kernel<Tt>, dim3(blocks), dim3(THREADS), 0, st,
                                   (const Tt*)k, (const Tt*)v, (uint8_t*)k_cache, (uint8_t*)v_cache,
                                   (uint8_t*)k_scale, (uint8_t*)v_scale, cell_of, rows, heads,
                                   (int)D, sk_t, sk_h, sv_t, sv_h),
                "kv_quantize");
    return LSB_OK;
  });
}

extern "C" int lsb_kv_dequantize(const void* k_cache, const void* v_cache, const void* k_scale,
                                 const void* v_scale, const int64_t* slot_mapping, void* k_out,
                                 void* v_out, int64_t T, int64_t H, int64_t D, int64_t num_blocks,
                                 int64_t block_size, int dtype, void* stream) {
  using namespace lsb::kvq;
  if (int rc = check_sizes("kv_dequantize", T, H, D, num_blocks, block_size, dtype)) return rc;
  if (T == 0) return LSB_OK;
  LSB_CHECK_ARG(k_cache && v_cache && k_scale && v_scale && slot_mapping && k_out && v_out,
                "kv_dequantize: null pointer");
  const CellOf cell_of(slot_mapping, nullptr, nullptr, 0, num_blocks, block_size, H);
  const FastDiv heads((uint32_t)H);
  const uint32_t rows = (uint32_t)(T * H);
  cudaStream_t st = (cudaStream_t)stream;
  return LSB_DISPATCH_DTYPE(dtype, Tt, [&] {
    const bool vec = aligned({k_out, v_out}, 16) && aligned({k_cache, v_cache}, 8);
    const int rc = vec ? with_dim<Tt>(D, [&](auto dim) -> int {
      constexpr int DD = decltype(dim)::value;
      const uint32_t groups = (uint32_t)((H + HPT - 1) / HPT), units = (uint32_t)T * groups;
      const unsigned blocks = blocks_for(units, DD * (int)sizeof(Tt) / 16);
      LSB_CHECK_ARG(blocks > 0, "kv_dequantize: too many rows");
      LSB_CUDA_OK(lsb::launch_kernel(dequantize_vec_kernel<Tt, DD>, dim3(blocks), dim3(THREADS), 0,
                                     st, (const uint8_t*)k_cache, (const uint8_t*)v_cache,
                                     (const uint8_t*)k_scale, (const uint8_t*)v_scale, cell_of,
                                     (Tt*)k_out, (Tt*)v_out, units, FastDiv(groups)),
                  "kv_dequantize");
      return LSB_OK;
    }) : -1;
    if (rc >= 0) return rc;
    const unsigned blocks = blocks_for(rows, 32);
    LSB_CHECK_ARG(blocks > 0, "kv_dequantize: too many rows");
    LSB_CUDA_OK(lsb::launch_kernel(dequantize_any_kernel<Tt>, dim3(blocks), dim3(THREADS), 0, st,
                                   (const uint8_t*)k_cache, (const uint8_t*)v_cache,
                                   (const uint8_t*)k_scale, (const uint8_t*)v_scale, cell_of,
                                   (Tt*)k_out, (Tt*)v_out, rows, heads, (int)D),
                "kv_dequantize");
    return LSB_OK;
  });
}

extern "C" int lsb_rope_kv_quantize(const void* qkv, int64_t s_s, int64_t s_part, int64_t s_h,
                                    const void* cos_table, const void* sin_table, int64_t s_pos,
                                    int64_t max_pos, const int64_t* positions,
                                    const int64_t* slot_mapping, const int32_t* block_tables,
                                    int64_t max_blocks_per_seq, void* q_out, void* k_out,
                                    void* k_cache, void* v_cache, void* k_scale, void* v_scale,
                                    int32_t* context_lens, int64_t T, int64_t H, int64_t D,
                                    int64_t num_blocks, int64_t block_size, int dtype,
                                    void* stream) {
  using namespace lsb::kvq;
  if (int rc = check_sizes("rope_kv_quantize", T, H, D, num_blocks, block_size, dtype)) return rc;
  LSB_CHECK_ARG(D % 2 == 0 && max_pos > 0, "rope_kv_quantize: D=%lld must be even, max_pos=%lld positive",
                (long long)D, (long long)max_pos);
  LSB_CHECK_ARG((slot_mapping == nullptr) != (block_tables == nullptr) || T == 0,
                "rope_kv_quantize: give slot_mapping or block_tables, not both");
  LSB_CHECK_ARG(block_tables == nullptr || max_blocks_per_seq > 0,
                "rope_kv_quantize: max_blocks_per_seq=%lld must be positive",
                (long long)max_blocks_per_seq);
  if (T == 0) return LSB_OK;
  LSB_CHECK_ARG(qkv && cos_table && sin_table && positions && q_out && k_cache && v_cache &&
                    k_scale && v_scale,
                "rope_kv_quantize: null pointer");
  const CellOf cell_of(slot_mapping, positions, block_tables, max_blocks_per_seq, num_blocks, block_size, H);
  const FastDiv heads((uint32_t)H);
  const RopeArgs args{s_s, s_part, s_h, s_pos, max_pos, positions, context_lens};
  const uint32_t rows = (uint32_t)(T * H);
  cudaStream_t st = (cudaStream_t)stream;
  return LSB_DISPATCH_DTYPE(dtype, Tt, [&] {
    const bool vec = aligned({qkv, cos_table, sin_table, q_out, k_out}, 16) &&
                     aligned({k_cache, v_cache}, 8) &&
                     strides16(sizeof(Tt), {s_s, s_part, s_h, s_pos});
    const int rc = vec ? with_dim<Tt>(D, [&](auto dim) -> int {
      constexpr int DD = decltype(dim)::value;
      const uint32_t groups = (uint32_t)((H + QPT - 1) / QPT), units = (uint32_t)T * groups;
      const unsigned blocks = blocks_for(units, DD * (int)sizeof(Tt) / 16);
      LSB_CHECK_ARG(blocks > 0, "rope_kv_quantize: too many rows");
      LSB_CUDA_OK(lsb::launch_kernel(rope_quantize_vec_kernel<Tt, DD>, dim3(blocks), dim3(THREADS),
                                     0, st, (const Tt*)qkv, (const Tt*)cos_table,
                                     (const Tt*)sin_table, args, (Tt*)q_out, (Tt*)k_out,
                                     (uint8_t*)k_cache, (uint8_t*)v_cache, (uint8_t*)k_scale,
                                     (uint8_t*)v_scale, cell_of, units, FastDiv(groups)),
                  "rope_kv_quantize");
      return LSB_OK;
    }) : -1;
    if (rc >= 0) return rc;
    const unsigned blocks = blocks_for(rows, 32);
    LSB_CHECK_ARG(blocks > 0, "rope_kv_quantize: too many rows");
    LSB_CUDA_OK(lsb::launch_kernel(rope_quantize_any_kernel<Tt>, dim3(blocks), dim3(THREADS), 0, st,
                                   (const Tt*)qkv, (const Tt*)cos_table, (const Tt*)sin_table, args,
                                   (Tt*)q_out, (Tt*)k_out, (uint8_t*)k_cache, (uint8_t*)v_cache,
                                   (uint8_t*)k_scale, (uint8_t*)v_scale, cell_of, rows, heads,
                                   (int)D),
                "rope_kv_quantize");
    return LSB_OK;
  });
}
