// Shared by the kernels of the chunk attention (attn_chunk.cu, attn_chunk_tile.cu): parameters, the visible range of a
// query token, the scores' cap and bias.
#pragma once

#include "common.cuh"
#include "devfn.cuh"

namespace lsvd {

constexpr float kChunkLog2e = 1.4426950408889634f;
constexpr int kStreamRows = 8;      // query rows of a block of the stream form
constexpr int kStreamMost = 2 * kStreamRows;      // of a request of the stream form: one or two blocks
constexpr int kChunkTileRows = 256;  // and of the tile form
constexpr int kFoldKeys = 8192;      // keys that an accumulator in tensor memory sums before it is folded into the workspace

// Weights are 2^(x - R + kWeightShift) with R, the row's reference, the largest x + exponent of |V scale| among the keys that the row
// SEES when R was last moved (x: score in units of log2).  R moves when that has grown by more than kLazy, so |weight * scale| stays
// below 2^15, fits fp16, and keeps its bits down to 2^-31 of the largest.  Keys that a row does not see have no part in it, nor has
// a large scale whose weight is nothing.  R and the weights' sum go through splits and joins like a maximum and its sum.
constexpr float kWeightShift = 6.f;
constexpr float kLazy = 8.f;
constexpr int kLeastExponent = -24;      // of a finite fp16 scale; also for zero, infinity and NaN

struct ChunkHead {
  int32_t k_col, v_col;      // byte offsets of the head inside a K / V cache row
  int16_t nk, nv;            // 16-entry pieces of K and V
};

struct ChunkParams {
  const __half* q;
  int64_t q_stride_t, q_stride_h;
  const int8_t* cache_k;
  const int8_t* cache_v;
  const __half* scale_k;
  const __half* scale_v;
  int64_t cache_k_row_stride, cache_v_row_stride, scale_k_row_stride, scale_v_row_stride;
  const __half* up_k;
  const __half* up_v;
  int64_t up_k_row_stride, up_v_row_stride;
  const int32_t* req_to_token;
  int64_t req_to_token_stride;
  const int32_t* b_req_idx;
  const int32_t* b_seq_len;
  const int32_t* b_start_loc;
  __half* out;
  int64_t out_stride_t, out_stride_h;
  __half* out_latent;
  int64_t out_latent_stride_t;
  // partial results, for the merge: reference (log2 domain) and sum of weights [split][row][head], unnormalised sums
  // [split][row][sum r_v]; a row is request * stream_stride + i in the stream form, the token's row in the tile form
  float2* stream_ml;
  float* stream_o;
  float2* tile_ml;
  float* tile_o;
  int32_t* status_word;
  const float* alibi_slopes;
  const int32_t* b_prefix_len;
  const int32_t* key_begin;
  const int32_t* mem_index;
  float score_scale;         // sm_scale
  float softcap;             // 0: none
  float cap_u, cap_log2e;    // 2 / softcap, softcap * log2(e)
  int32_t batch, num_heads, head_dim, max_len, num_tokens, max_new, num_slots, r2t_rows;
  int32_t causal, window, head_major, sum_rv;
  int32_t q_vec, up_k_vec;   // rows of q / up_k can be read in 8-byte pieces
  int32_t up_v_vec, out_vec2, out_lat_vec16;     // rows of up_v in 8-byte, of out in 4-byte, of out_latent in 16-byte pieces
  // split s takes the keys [s * split_len, (s + 1) * split_len)
  int32_t stream_splits, stream_split_len, stream_stride;
  int32_t tile_splits, tile_split_len;
  int32_t stream_partials;   // the stream form leaves its results to the merge (the tile form: when it is split)
  // (a block of the tile form with more than kFoldKeys keys also folds its sums into its rows of tile_o as it goes, and keeps the
  // reference that they are relative to in tile_ml)
  int32_t tile_min;          // the tile form takes requests of more rows than this
  ChunkHead head[LSVD_MAX_HEADS];
};

cudaError_t launch_chunk_tile(const ChunkParams& p, int tiles, cudaStream_t st);

#ifdef __CUDACC__
// A request, checked: its first row, its new tokens (0: skip it), its length and its row of the slot table.
struct ChunkRequest {
  int start, n, len, req;
};

// `report`: one thread per request says what was wrong.  A request whose rows do not lie in the step's, or that has more of them than
// the bound, is skipped: rows are its LAST tokens, so a part of them would stand at other positions.
__device__ __forceinline__ ChunkRequest chunk_request(const ChunkParams& p, int b, bool report) {
  ChunkRequest r;
  const int start = p.b_start_loc[b], end = p.b_start_loc[b + 1];
  const bool fits = start >= 0 && end >= start && end <= p.num_tokens;
  r.start = fits ? start : 0;
  r.n = fits ? end - start : 0;
  r.len = p.b_seq_len[b];
  r.req = p.b_req_idx[b];
  bool bad = !fits || r.len > p.max_len || r.n > p.max_new;
  if (r.len > p.max_len) r.len = p.max_len;
  if (r.n > p.max_new) r.n = 0;
  if (r.len < 0) r.len = 0;
  if (r.len < r.n) {                 // fewer tokens than rows: no row has a position (they see nothing)
    bad = true;
    r.len = 0;
  }
  if (static_cast<uint32_t>(r.req) >= static_cast<uint32_t>(p.r2t_rows)) {
    bad = true;
    r.req = 0;
    r.len = 0;
  }
  if (bad && report) report_status(p.status_word, LSVD_ERR_BOUNDS);
  return r;
}

struct KeyRange {
  int lo, hi;      // keys lo <= t < hi are seen; lo >= hi: none
};

// Causal, sliding-window, prefix and document masks all leave a query token one run of keys.
__device__ __forceinline__ KeyRange visible_keys(const ChunkParams& p, const ChunkRequest& r, int prefix, int i) {
  const int pos = r.len - r.n + i;
  KeyRange k;
  k.lo = 0;
  k.hi = r.len;
  if (p.causal) k.hi = min(r.len, max(pos + 1, prefix));
  if (p.window > 0) {
    k.lo = max(0, static_cast<int>(max(static_cast<int64_t>(pos) + 1 - p.window, static_cast<int64_t>(0))));
    if (!p.causal) k.hi = static_cast<int>(min(static_cast<int64_t>(r.len), static_cast<int64_t>(pos) + p.window));
  }
  if (p.key_begin != nullptr) k.lo = max(k.lo, p.key_begin[r.start + i]);
  if (p.mem_index != nullptr && p.mem_index[r.start + i] < 0) k.hi = 0;      // a token that was refused is not in the cache
  if (k.hi <= k.lo) k.lo = k.hi = 0;
  return k;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// cap * tanh(x / cap) in units of log2, of v = x * log2(e), by u = 2 v / cap (so e^(2 x / cap) = 2^u).  For |x / cap| below a quarter the
// series of tanh(y) / y up to y^6 (what follows is below 2^-21 of it): v stands as a factor, so a cap far above the scores leaves
// them as they are.  Above it 1 - 2 / (1 + 2^u), whose rounding, 2^-22 of the cap, is below 2^-19 of such a score.
// (The hardware's tanh is off by 2^-11 of the cap, half a unit of a score at a cap of 1000, 2 % of a weight at 50.)
constexpr float kCapSeries = 0.5f * kChunkLog2e;      // u at x / cap = 1/4
__device__ __forceinline__ float2 capped_series(float2 v, float2 u) {
  auto both = [](float c) { return make_float2(c, c); };
  const float2 s = mul2(u, u);
  return mul2(v, fma2(fma2(fma2(s, both(-9.35214345e-5f), both(1.92362582e-3f)), s, both(-4.00377512e-2f)), s, both(1.f)));
}
__device__ __forceinline__ float2 capped_log2(float2 v, float2 u, float cap_log2e) {
  const float2 y = capped_series(v, u);
  return make_float2(fabsf(u.x) < kCapSeries ? y.x : fmaf(__fdividef(-2.f, 1.f + ex2(u.x)), cap_log2e, cap_log2e),
                     fabsf(u.y) < kCapSeries ? y.y : fmaf(__fdividef(-2.f, 1.f + ex2(u.y)), cap_log2e, cap_log2e));
}

// Exponent e with 2^e <= x < 2^(e+1) for a positive normal x (0 for what is not positive and finite).
__device__ __forceinline__ int exponent_of(float x) {
  return (x > 0.f && x < INFINITY) ? static_cast<int>((__float_as_uint(x) >> 23) & 255u) - 127 : 0;
}
__device__ __forceinline__ float scale_exponent(float x) {
  const int e = static_cast<int>((__float_as_uint(x) >> 23) & 255u);
  return static_cast<float>(e > 0 && e < 255 ? e - 127 : kLeastExponent);
}
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float(static_cast<uint32_t>(min(max(e, -126), 127) + 127) << 23); }

// Four int8 codes (already xored with 0x80808080, i.e. code + 128) as two fp16 pairs: 0x6400 | u is 1024 + u, exactly.
__device__ __forceinline__ void codes_to_half(uint32_t u, uint32_t& lo, uint32_t& hi) {
  const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
  const __half2 off = __floats2half2_rn(-1152.f, -1152.f);
  const __half2 x = __hadd2(*reinterpret_cast<const __half2*>(&a), off), y = __hadd2(*reinterpret_cast<const __half2*>(&b), off);
  lo = *reinterpret_cast<const uint32_t*>(&x);
  hi = *reinterpret_cast<const uint32_t*>(&y);
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Two values as fp16 and what that leaves of them, as fp16 too.  (An infinity or a NaN leaves nothing.)
__device__ __forceinline__ void pack_half2_rest(float a, float b, uint32_t& most, uint32_t& rest) {
  most = pack_half2(a, b);
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&most));
  const float x = a - h.x, y = b - h.y;
  rest = pack_half2(fabsf(x) < INFINITY ? x : 0.f, fabsf(y) < INFINITY ? y : 0.f);
}

// Four consecutive halves, zero beyond `n` of them.
__device__ __forceinline__ uint2 load_halves4(const __half* src, int n, bool vec) {
  uint2 v = make_uint2(0u, 0u);
  if (n >= 4 && vec) return __ldg(reinterpret_cast<const uint2*>(src));
  uint32_t h[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < n) h[e] = __half_as_ushort(src[e]);
  v.x = h[0] | (h[1] << 16);
  v.y = h[2] | (h[3] << 16);
  return v;
}

__device__ __forceinline__ void store_halves8(__half* dst, uint4 v, bool vec) {
  if (vec) {
    *reinterpret_cast<uint4*>(dst) = v;
    return;
  }
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 8; ++e) dst[e] = __ushort_as_half(static_cast<unsigned short>(w[e >> 1] >> (16 * (e & 1))));
}

template <int kN>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kN) : "memory"); }
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// 16 bytes global -> shared, or 16 zero bytes (nothing is read).
__device__ __forceinline__ void copy16_or_zero(void* dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(real ? 16 : 0) : "memory");
}

// Where codes lie in shared memory (32 keys a group).  Column c = 2 t + e of the 8-key score tile j = 2 m + jj stands for key
// 16 m + 8 jj + t + 4 e, so that lane (g, t)'s weights are those of keys t, t + 4, t + 8, t + 12 of a 16-key step and its V
// operand comes from rows four apart.  K rows are stored in column order (lane (g, t) reads row 8 j + g), V rows in key order.
// The 16-byte pieces of rows of 64 and 128 bytes are swizzled so that the rows read together lie in different banks.
__device__ __forceinline__ int k_row_of(int key) { return (key & ~7) | ((key & 3) << 1) | ((key >> 2) & 1); }
__device__ __forceinline__ int k_piece_at(int row, int piece, int nk) { return nk == 8 ? piece ^ ((row & 1) << 2) : piece; }
__device__ __forceinline__ int v_piece_at(int key, int piece, int nv) {
  return nv == 8 ? piece ^ ((key & 3) << 1) : (nv == 4 ? piece ^ (key & 2) : piece);
}
#endif

}  // namespace lsvd
