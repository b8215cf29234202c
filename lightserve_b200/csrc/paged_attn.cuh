// Attention of new tokens over a paged KV cache: what its kernels share.
//
// Sequence s has context_lens[s] cached tokens, the last n_s of which are the
// call's new tokens (rows [cu_seqlens_q[s], cu_seqlens_q[s + 1]) of q; one row
// per sequence when cu_seqlens_q is NULL). Row i stands at position
// p = context_lens[s] - n_s + i and sees key j when
//     j <= p,  j < context_lens[s],  page of j inside the cache,
//     and, with a window w > 0, p - j < w or j < num_sinks.
// O = softmax(scale Q K^T) V over the keys it sees, 0 when it sees none.
//
// The keys of a sequence are walked in tiles of TK keys. With a window, the
// tiles that no row of a query tile can see are not visited: the visited
// ones are the tiles of [0, num_sinks) followed by the tiles from the
// window's first key on (KeySpan). A span is cut into chunks of
// `chunk` keys, one per CTA along the grid, when there are few rows: each
// chunk then leaves its normalised output and log2-sum-exp in the workspace
// and paged_combine_kernel joins them. A span of one chunk is written
// directly.
#pragma once

#include <stdint.h>

#include "common.cuh"
#include "fp8.cuh"

namespace lsb {
namespace pa {

constexpr float LOG2E = 1.4426950408889634f;

// The tensor-core kernels' running maximum may lag a score by 2^8 (it is raised,
// and the outputs rescaled, only beyond that). An fp16 P also carries 2^7 on every
// weight: 2^15 at most, and full precision down to 2^-21 of the running maximum
// instead of 2^-14, nothing below 2^-32 instead of 2^-25 (a key that takes
// nearly all the weight beside tens of thousands of small ones: they are still
// summed). bf16 has fp32's range and carries nothing, so a sum passes fp32's
// only where values times keys pass 2^120.
constexpr float F16_LIFT = 7.f;

struct Params {
  const void* q;
  const void* k_cache;
  const void* v_cache;
  const uint8_t* k_scale;       // e4m3 cache: e8m0 scales; else NULL
  const uint8_t* v_scale;
  const int32_t* block_tables;  // [S, max_blocks]
  const int32_t* context_lens;  // [S]
  const int32_t* cu_seqlens_q;  // [S + 1] or NULL
  void* o;
  float* lse;                   // [Hq, T] or NULL
  float* part_lse;              // [T, Hq, P] log2-sum-exp of each chunk
  float* part_o;                // [T, Hq, P, D] normalised
  int64_t sq_t, sq_h, so_t, so_h;
  int S, T, max_q, Hq, Hkv, G, D;
  int max_blocks, num_blocks, bs_log2;
  int window, sinks;            // window 0: none
  int chunk, P;                 // keys per chunk, chunks per row at most
  float scale_log2;
};

// Rows and keys of sequence s, read from device memory and clamped to the
// tensors, so malformed lengths cannot reach outside them.
struct Seq {
  int row0;   // first row in q
  int n;      // rows computed (at most max_q)
  int pos0;   // position of row 0 (negative: more rows than cached tokens)
  int ctx;    // keys addressable through the block table
};

__device__ __forceinline__ Seq load_seq(const Params& p, int s) {
  Seq r;
  int n_all = 1;
  if (p.cu_seqlens_q != nullptr) {
    r.row0 = min(max(p.cu_seqlens_q[s], 0), p.T);
    n_all = min(max(p.cu_seqlens_q[s + 1], r.row0), p.T) - r.row0;
  } else {
    r.row0 = s;
  }
  r.n = min(n_all, p.max_q);
  const int len = max(p.context_lens[s], 0);
  r.pos0 = len - n_all;
  r.ctx = min(len, p.max_blocks << p.bs_log2);
  return r;
}

// The key tiles (of tk keys) that the rows at positions [pos_lo, pos_hi] see:
// s_tiles tiles from key 0 on, then the tiles [lo, hi).
struct KeySpan {
  int s_tiles, lo, hi;
  KeySpan() = default;
  __device__ __forceinline__ KeySpan(const Params& p, const Seq& q, int pos_lo, int pos_hi, int tk) {
    const int end = max(min(q.ctx, pos_hi + 1), 0);  // keys from here on are seen by none
    hi = (end + tk - 1) / tk;
    lo = 0;
    s_tiles = 0;
    if (p.window > 0) {
      lo = min(max(pos_lo - p.window + 1, 0) / tk, hi);
      s_tiles = min((min(p.sinks, end) + tk - 1) / tk, lo);
    }
  }
  __device__ __forceinline__ int count() const { return s_tiles + hi - lo; }
  __device__ __forceinline__ int tile(int v) const { return v < s_tiles ? v : v - s_tiles + lo; }
};

__device__ __forceinline__ bool sees(const Params& p, int pos, int ctx, int j) {
  return j <= pos && j < ctx && (p.window == 0 || pos - j < p.window || j < p.sinks);
}

// Whether a row between positions pos_lo and pos_hi sees key j. Kernels zero the
// staged V of a key that none of a tile's rows sees, so that what such a cell
// holds (nothing yet, another sequence's values, NaN) never meets a weight of 0.
__device__ __forceinline__ bool seen_by_any(const Params& p, int pos_lo, int pos_hi, int ctx, int j) {
  return j <= pos_hi && j < ctx && (p.window == 0 || pos_lo - j < p.window || j < p.sinks);
}

// Chunks that a span of `tiles` tiles of tk keys is cut into (at least one).
__device__ __forceinline__ int chunks_of(const Params& p, int tiles, int tk) {
  const int per = p.chunk / tk;
  return min(max((tiles + per - 1) / per, 1), p.P);
}

// Query tile `tile` of a (sequence, cache head): the (row, head of the group)
// pairs r in [tile R, tile R + R), pair r being row r / G and head r % G of
// the group, so the group's heads share the K/V tiles. Its rows' positions.
__device__ __forceinline__ void tile_positions(const Params& p, const Seq& q, int tile, int R,
                                               int& lo, int& hi) {
  lo = q.pos0 + tile * R / p.G;
  hi = q.pos0 + min((tile * R + R - 1) / p.G, q.n - 1);
}

// Joins the chunks of one (row, head): o = sum_c w_c o_c / sum_c w_c with
// w_c = 2^(lse_c - max lse). The grid covers every row and head; a row whose
// span was one chunk was written directly and is skipped, as are rows that
// belong to no sequence (left as they were). rows_per_tile: the (row, query
// head of the group) pairs of a query tile in the kernel that wrote the
// chunks, which fixes the spans; tk: its key tile.
int launch_combine(const Params& p, int rows_per_tile, int tk, int dtype, cudaStream_t st);

// Each kernel's launcher. `kv_fp8`: the cache holds e4m3.
int launch_simt(const Params& p, int dtype, bool kv_fp8, cudaStream_t st);

// paged_attn_rows.cu's key group, and the pairs of its query tile: 8, 16 or 24,
// the fewest that hold a sequence's (more pairs take several tiles, each of
// which reads the cache again).
constexpr int rows_tk(bool kv_fp8) { return kv_fp8 ? 32 : 16; }
inline int rows_tile(int64_t pairs) { return pairs <= 8 ? 8 : pairs <= 16 ? 16 : 24; }
constexpr int TC_TK = 128;  // paged_attn_sm100.cu's key tile; a query tile holds (128 / G) G pairs
bool tc_eligible(const Params& p, int dtype, bool kv_fp8);
int launch_tc(const Params& p, int dtype, bool kv_fp8, cudaStream_t st);
bool rows_eligible(const Params& p, int dtype);
int launch_rows(const Params& p, int dtype, bool kv_fp8, cudaStream_t st);

}  // namespace pa
}  // namespace lsb
