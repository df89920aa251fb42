// Attention of new tokens over the paged int8 latent cache ("absorb" form): entry points, the stream form, the merge.
//
// The query is folded into the per-head K up-factor once per row (q~ = B_k q), so that a score is a dot product of r_k int8
// latents with q~, and the values stay in the latent space until the end:
//   x_t = sm_scale scale_k[t] (z_k[t] . q~) [capped, biased],  o_lat = sum_t softmax(x)_t scale_v[t] z_v[t],  o = B_v^T o_lat.
//
// Stream form (8 query rows of a request share one pass over its cache): a block owns (request, head, the rows,
// split of the keys); each of its four warps walks its own 32-key tiles.  The rows arrive by 16-byte asynchronous copies in
// a ring of shared memory per warp (gathered slot by slot: any page table, both cache layouts); codes become fp16 exactly
// (|code| <= 128) and meet q~ and the weights on the tensor cores (mma m16n8k16, fp32 accumulators).  With few rows the bytes
// of the cache would bound it, r_k + r_v + 4 bytes per key and head; what does is the instruction stream of a tile (widening,
// two products of 16-row fragments that few rows fill, softmax) at twelve warps an SM.  Measured: 16 single tokens over 4096 keys, 32
// heads, mean ranks 64 + 64: 200 us (268 MB, 1.3 TB/s); five tokens of eight requests over 4091 keys 136 us.  Before the value loop
// was rolled for the instruction cache (215 -> 201 us for the single tokens), sixteen rows a block, with the lower half of the
// fragments for rows 9 to 16, took them 230 us against 215.
//
// Roundings.  q~ enters the products as two fp16 numbers, what fp16 keeps of it and the rest, relative to its row's largest entry (a
// power of two taken out, so no entry overflows and small ones keep their bits down to 2^-23 of the largest).  The weights
// p * scale_v enter as two fp16 numbers as well, relative to the largest one that the row sees (attn_chunk.cuh); the stream form
// carries the second ones in the half of the fragment that its few rows leave free, the tile form in a product of their own.
// References, sums and accumulators are fp32.  Scales are applied in fp32 to scores and weights, never to the codes: a masked key's
// scale, were it huge, infinite or NaN, touches nothing.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstring>

#include "attn_chunk.cuh"
#include "devfn.cuh"

namespace lsvd {

constexpr int kChunkWarps = 4;
constexpr int kChunkThreads = kChunkWarps * 32;
constexpr int kRingBytes = 16 * 1024;         // per warp: 2 to 8 stages of 32 keys x (r_k + r_v) bytes
constexpr int kMaxStages = 8;

// Absorbed query row `row` [128] fp32: four rows in the last 2 KB of every warp's ring, which no copy reaches before the
// first tile is consumed (stages 0 .. n - 2 are requested ahead of that; the last stage, or what lies behind it, is free).
__device__ __forceinline__ float* absorbed_row(uint8_t* ring_mem, int row) {
  return reinterpret_cast<float*>(ring_mem + ((row >> 2) + 1) * kRingBytes - 2048 + (row & 3) * 512);
}

struct __align__(16) ChunkShared {
  float sk[kChunkWarps][32], sv[kChunkWarps][32];             // scales of the tile in hand
  float se[kChunkWarps][32];                                  // exponents of the V scales
  int32_t slot[kChunkWarps][kMaxStages][32];                  // slot of every key in the ring, -1: none
  float m[kChunkWarps][kStreamRows], l[kChunkWarps][kStreamRows];
  int32_t lo[kStreamRows], hi[kStreamRows];
};

// q~ of up to 8 rows into shared memory, by all warps of the block: warp w takes the 8-rank tiles w, w + 4, ...
// (mma lane (g, t): row g, rows 8 .. 15 zero, k = halves 4t .. 4t + 3 of a 16-wide step, ranks 8 j + g).
__device__ __forceinline__ void absorb_rows(const ChunkParams& p, const ChunkHead& H, int h, const ChunkRequest& r, int row0, int rows,
                                            uint8_t* ring_mem) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const __half* qa = p.q + static_cast<int64_t>(r.start + row0 + min(g, rows - 1)) * p.q_stride_t + h * p.q_stride_h;
  const int tiles = H.nk * 2;
  for (int j = warp; j < tiles; j += kChunkWarps) {
    const __half* up = p.up_k + static_cast<int64_t>(H.k_col + j * 8 + g) * p.up_k_row_stride;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int d0 = 0; d0 < p.head_dim; d0 += 64) {
      uint2 a0[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = d0 + 16 * i + 4 * t;
        a0[i] = load_halves4(qa + d, p.head_dim - d, p.q_vec);
        b[i] = load_halves4(up + d, p.head_dim - d, p.up_k_vec);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) mma_f16_16x8x16(acc, a0[i].x, 0u, a0[i].y, 0u, b[i].x, b[i].y);
    }
    *reinterpret_cast<float2*>(absorbed_row(ring_mem, g) + j * 8 + 2 * t) = make_float2(acc[0], acc[1]);
  }
}

// grid: (heads, requests' first rows and, where some request may have more than 8, their second ones, splits)
template <bool kCap, bool kBias>
__global__ void __launch_bounds__(kChunkThreads, 3) chunk_stream_kernel(const __grid_constant__ ChunkParams p) {
  extern __shared__ __align__(16) uint8_t ring_mem[];
  __shared__ ChunkShared s;
  grid_dependency_release();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
  const int h = blockIdx.x, split = blockIdx.z;
  const int row0 = static_cast<int>(blockIdx.y) >= p.batch ? kStreamRows : 0, b = blockIdx.y - (row0 > 0 ? p.batch : 0);
  const ChunkRequest r = chunk_request(p, b, h == 0 && split == 0 && row0 == 0 && threadIdx.x == 0);
  if (r.n <= row0 || r.n > kStreamMost) return;      // none, or the tile form's
  const int rows = min(r.n - row0, kStreamRows);
  const ChunkHead H = p.head[h];
  const int rk = H.nk * 16, rv = H.nv * 16;

  // the rows' visible keys, and the block's: from the smallest lo to the largest hi, cut to the split
  if (threadIdx.x < kStreamRows) {
    KeyRange k;
    k.lo = k.hi = 0;
    if (static_cast<int>(threadIdx.x) < rows)
      k = visible_keys(p, r, p.b_prefix_len != nullptr ? p.b_prefix_len[b] : 0, row0 + threadIdx.x);
    s.lo[threadIdx.x] = k.lo;
    s.hi[threadIdx.x] = k.hi;
  }
  __syncthreads();
  int kbeg = 0x7fffffff, kend = 0, inner_lo = 0, inner_hi = 0x7fffffff;    // inner: keys that every live row sees
  for (int i = 0; i < rows; ++i) {
    if (s.hi[i] > s.lo[i]) kbeg = min(kbeg, s.lo[i]);
    kend = max(kend, s.hi[i]);
    inner_lo = max(inner_lo, s.lo[i]);
    inner_hi = min(inner_hi, s.hi[i]);
  }
  kbeg = max(kbeg & ~31, split * p.stream_split_len);
  if (p.stream_splits > 1) kend = static_cast<int>(min(static_cast<int64_t>(kend), (static_cast<int64_t>(split) + 1) * p.stream_split_len));
  const int ntiles = kend > kbeg ? (kend - kbeg + 31) / 32 : 0;

  if (ntiles == 0 && p.stream_partials) {      // the merge reads no sums where the weights' sum is zero
    if (static_cast<int>(threadIdx.x) < rows)
      p.stream_ml[(static_cast<int64_t>(split) * p.batch * p.stream_stride + b * p.stream_stride + row0 + threadIdx.x) * p.num_heads + h] =
          make_float2(-INFINITY, 0.f);
    return;
  }

  const int32_t* r2t = p.req_to_token + static_cast<int64_t>(r.req) * p.req_to_token_stride;
  const int8_t* kbase = p.cache_k + (p.head_major ? static_cast<int64_t>(H.k_col) * p.num_slots : H.k_col);
  const int8_t* vbase = p.cache_v + (p.head_major ? static_cast<int64_t>(H.v_col) * p.num_slots : H.v_col);
  const uint32_t kstride = static_cast<uint32_t>(p.head_major ? rk : p.cache_k_row_stride);      // (the host has checked the strides)
  const uint32_t vstride = static_cast<uint32_t>(p.head_major ? rv : p.cache_v_row_stride);
  const __half* ksc = p.scale_k + (p.head_major ? static_cast<int64_t>(h) * p.num_slots : h);
  const __half* vsc = p.scale_v + (p.head_major ? static_cast<int64_t>(h) * p.num_slots : h);
  const int64_t kss = p.head_major ? 1 : p.scale_k_row_stride, vss = p.head_major ? 1 : p.scale_v_row_stride;

  const int stage_bytes = 32 * (rk + rv);
  const int stages = stage_bytes * 8 <= kRingBytes ? 8 : (stage_bytes * 4 <= kRingBytes ? 4 : 2);
  uint8_t* ring = ring_mem + warp * kRingBytes;
  const int mine = ntiles > warp ? (ntiles - warp + kChunkWarps - 1) / kChunkWarps : 0;

  // slot of this lane's key in tile `i` of the warp (-1: behind the end, unmapped or out of range)
  auto fetch_slot = [&](int i) {
    int slot = -1;
    const int key = kbeg + (warp + i * kChunkWarps) * 32 + lane;
    if (i < mine && key < kend) slot = r2t[key];
    return slot;
  };
  const uint32_t inv_k = 65536u / H.nk + 1, inv_v = 65536u / H.nv + 1;     // x / n = x * inv >> 16 for x < 256, n <= 8
  auto request = [&](int i, int slot) {
    if (slot >= p.num_slots) {
      report_status(p.status_word, LSVD_ERR_BOUNDS);
      slot = -1;
    }
    const int st = i & (stages - 1);
    s.slot[warp][st][lane] = slot;
    uint8_t* kd = ring + st * stage_bytes;
    uint8_t* vd = kd + 32 * rk;
    for (int x = lane; x < 32 * H.nk; x += 32) {
      const int tok = (x * inv_k) >> 16, piece = x - tok * H.nk;
      const int sl = __shfl_sync(0xffffffffu, slot, tok);
      const int row = k_row_of(tok);
      copy16_or_zero(kd + row * rk + k_piece_at(row, piece, H.nk) * 16, kbase + static_cast<uint64_t>(static_cast<uint32_t>(max(sl, 0))) * kstride + piece * 16, sl >= 0);
    }
    for (int x = lane; x < 32 * H.nv; x += 32) {
      const int tok = (x * inv_v) >> 16, piece = x - tok * H.nv;
      const int sl = __shfl_sync(0xffffffffu, slot, tok);
      copy16_or_zero(vd + tok * rv + v_piece_at(tok, piece, H.nv) * 16, vbase + static_cast<uint64_t>(static_cast<uint32_t>(max(sl, 0))) * vstride + piece * 16, sl >= 0);
    }
  };
  // (kept as loaded until the tile is in hand: a conversion here would wait for the load)
  auto load_scales = [&](int i, __half& a, __half& c) {
    if (i >= mine) return;
    const int sl = max(s.slot[warp][i & (stages - 1)][lane], 0);
    a = ksc[sl * kss];
    c = vsc[sl * vss];
  };

  // the first stages are on their way while the query rows are absorbed
  int slot_next = fetch_slot(0);
  for (int i = 0; i < stages - 1; ++i) {
    const int slot = slot_next;
    slot_next = fetch_slot(i + 1);
    if (i < mine) request(i, slot);
    copy_commit();
  }
  __half sk_next = __ushort_as_half(0), sv_next = sk_next;
  load_scales(0, sk_next, sv_next);

  absorb_rows(p, H, h, r, row0, rows, ring_mem);
  __syncthreads();
  const float* qt = absorbed_row(ring_mem, g);
  // q~ as fp16 A fragments: step (mb, i) of a 64-rank block holds ranks 64 mb + 16 t + 4 i .. + 3 of lane (g, t).  Row g is what
  // fp16 keeps of q~, row g + 8 of the fragment the rest, so that the products see 22 bits of it at no further cost.
  uint32_t qa[2][4][4];
  float f;                            // score scale of the row, with the power of two that was taken out
  {
    float big = 0.f;
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int rank = 64 * mb + 16 * t4 + 4 * i;
        if (rank < rk) {
          const float4 x = *reinterpret_cast<const float4*>(qt + rank);
          big = fmaxf(big, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
        }
      }
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
    const int ex = exponent_of(big) - 8;                                 // entries end up below 2^9
    const float by = pow2i(-ex);
    f = p.score_scale * pow2i(ex);
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int rank = 64 * mb + 16 * t4 + 4 * i;
        qa[mb][i][0] = qa[mb][i][1] = qa[mb][i][2] = qa[mb][i][3] = 0u;
        if (rank < rk) {
          const float4 x = *reinterpret_cast<const float4*>(qt + rank);
          pack_half2_rest(x.x * by, x.y * by, qa[mb][i][0], qa[mb][i][1]);
          pack_half2_rest(x.z * by, x.w * by, qa[mb][i][2], qa[mb][i][3]);
        }
      }
  }
  __syncthreads();                    // the rings' last stages may be written from here on
  f *= kChunkLog2e;
  const int lo = s.lo[g], hi = s.hi[g], pos = r.len - r.n + row0 + g;
  const float slope = kBias ? p.alibi_slopes[h] * kChunkLog2e : 0.f;

  float R = -INFINITY, l = 0.f;       // reference and sum of the weights
  float o[2][8][4];
#pragma unroll
  for (int vb = 0; vb < 2; ++vb)
#pragma unroll
    for (int j = 0; j < 8; ++j) o[vb][j][0] = o[vb][j][1] = o[vb][j][2] = o[vb][j][3] = 0.f;

  for (int i = 0; i < mine; ++i) {
    {
      const int slot = slot_next;
      slot_next = fetch_slot(i + stages);
      __syncwarp();                   // every lane is done with the stage that is refilled now
      if (i + stages - 1 < mine) request(i + stages - 1, slot);
      copy_commit();
    }
    const int st = i & (stages - 1);
    const int my_slot = s.slot[warp][st][lane];
    const float sk = my_slot >= 0 ? __half2float(sk_next) : 0.f, sv = my_slot >= 0 ? __half2float(sv_next) : 0.f;
    const uint32_t valid = __ballot_sync(0xffffffffu, my_slot >= 0);
    load_scales(i + 1, sk_next, sv_next);
    const float se = scale_exponent(sv);
    const float e_top = static_cast<float>(__reduce_max_sync(0xffffffffu, static_cast<int>(se)));      // of all keys, seen or not
    s.sk[warp][lane] = sk;
    s.sv[warp][lane] = sv;
    s.se[warp][lane] = se;
    if (stages == 8) copy_wait<7>();
    else if (stages == 4) copy_wait<3>();
    else copy_wait<1>();
    __syncwarp();
    const uint8_t* kd = ring + st * stage_bytes;
    const uint8_t* vd = kd + 32 * rk;

    // scores of 32 keys in four 8-key tiles; column c = 2 t' + e of tile j = 2 m + jj is key 16 m + 8 jj + t' + 4 e
    float x[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j][0] = x[j][1] = x[j][2] = x[j][3] = 0.f;
#pragma unroll
      for (int mb = 0; mb < 2; ++mb) {
        if (mb * 4 < H.nk) {
          uint4 w = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
          if (mb * 4 + t4 < H.nk) {
            w = *reinterpret_cast<const uint4*>(kd + (8 * j + g) * rk + k_piece_at(8 * j + g, mb * 4 + t4, H.nk) * 16);
            w.x ^= 0x80808080u; w.y ^= 0x80808080u; w.z ^= 0x80808080u; w.w ^= 0x80808080u;
          }
          uint32_t b0, b1;
          codes_to_half(w.x, b0, b1);
          mma_f16_16x8x16(x[j], qa[mb][0][0], qa[mb][0][1], qa[mb][0][2], qa[mb][0][3], b0, b1);
          codes_to_half(w.y, b0, b1);
          mma_f16_16x8x16(x[j], qa[mb][1][0], qa[mb][1][1], qa[mb][1][2], qa[mb][1][3], b0, b1);
          codes_to_half(w.z, b0, b1);
          mma_f16_16x8x16(x[j], qa[mb][2][0], qa[mb][2][1], qa[mb][2][2], qa[mb][2][3], b0, b1);
          codes_to_half(w.w, b0, b1);
          mma_f16_16x8x16(x[j], qa[mb][3][0], qa[mb][3][1], qa[mb][3][2], qa[mb][3][3], b0, b1);
        }
      }
    }
    const int key0 = kbeg + (warp + i * kChunkWarps) * 32;
    const bool masked = key0 < inner_lo || key0 + 32 > inner_hi || valid != 0xffffffffu;
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (kCap) {
        const float2 v = mul2(make_float2(x[j][0] + x[j][2], x[j][1] + x[j][3]),
                              make_float2(s.sk[warp][8 * j + t4] * f, s.sk[warp][8 * j + t4 + 4] * f));
        const float2 y = capped_log2(v, mul2(v, make_float2(p.cap_u, p.cap_u)), p.cap_log2e);
        x[j][0] = y.x;
        x[j][1] = y.y;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int k = 8 * j + t4 + 4 * e;
        const float c = s.sk[warp][k];
        float v = kCap ? x[j][e] : (x[j][e] + x[j][2 + e]) * (c * f);
        if (kBias) v -= slope * fabsf(static_cast<float>(pos - key0 - k));
        if (masked && (!((valid >> k) & 1u) || key0 + k < lo || key0 + k >= hi)) v = -INFINITY;
        x[j][e] = v;
        top = fmaxf(top, v);
      }
    }
    // top + e_top bounds what the row sees here: only where that is past the reference is the row's own value looked for
    if (__any_sync(0xffffffffu, R == -INFINITY ? top > -INFINITY : top + e_top > R + kLazy)) {
      float need = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) need = fmaxf(need, x[j][e] + s.se[warp][8 * j + t4 + 4 * e]);
      need = fmaxf(need, __shfl_xor_sync(0xffffffffu, need, 1));
      need = fmaxf(need, __shfl_xor_sync(0xffffffffu, need, 2));
      const bool first = R == -INFINITY;
      const bool grown = first ? need > -INFINITY : need > R + kLazy;
      if (__any_sync(0xffffffffu, grown && !first)) {
        const float by = grown && !first ? ex2(R - need) : 1.f;
        l *= by;
#pragma unroll
        for (int vb = 0; vb < 2; ++vb)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            o[vb][j][0] *= by;
            o[vb][j][1] *= by;
            o[vb][j][2] *= by;
            o[vb][j][3] *= by;
          }
      }
      if (grown) R = need;
    }
    const float base = R == -INFINITY ? 0.f : R - kWeightShift;
    uint32_t w[4][2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float p0 = ex2(x[j][0] - base), p1 = ex2(x[j][1] - base);
      l += p0 + p1;
      const float v0 = s.sv[warp][8 * j + t4], v1 = s.sv[warp][8 * j + t4 + 4];
      // a masked key's weight is zero whatever its scale holds; what fp16 leaves of a weight goes to row g + 8
      pack_half2_rest(p0 == 0.f ? 0.f : p0 * v0, p1 == 0.f ? 0.f : p1 * v1, w[j][0], w[j][1]);
    }
    // values: rank 64 vb + 8 g + n of lane (g, t) is column g of tile n; the keys of step m are the score columns' keys
#pragma unroll 1
    for (int m = 0; m < 2; ++m) {
#pragma unroll
      for (int vb = 0; vb < 2; ++vb) {
        if (vb * 4 < H.nv) {
          uint2 ra = make_uint2(0x80808080u, 0x80808080u), rb = ra, rc = ra, rd = ra;
          if (64 * vb + 8 * g < rv) {
            // (keys four apart share their swizzle)
            const uint8_t* at = vd + (16 * m + t4) * rv + v_piece_at(t4, 4 * vb + (g >> 1), H.nv) * 16 + 8 * (g & 1);
            ra = *reinterpret_cast<const uint2*>(at);
            rb = *reinterpret_cast<const uint2*>(at + 4 * rv);
            rc = *reinterpret_cast<const uint2*>(at + 8 * rv);
            rd = *reinterpret_cast<const uint2*>(at + 12 * rv);
            ra.x ^= 0x80808080u; ra.y ^= 0x80808080u; rb.x ^= 0x80808080u; rb.y ^= 0x80808080u;
            rc.x ^= 0x80808080u; rc.y ^= 0x80808080u; rd.x ^= 0x80808080u; rd.y ^= 0x80808080u;
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) {       // two ranks at a time: bytes 2 (q & 1), + 1 of word q >> 1
            const uint32_t sel = (q & 1) ? 0x7362u : 0x5140u;
            const uint32_t u = __byte_perm(q < 2 ? ra.x : ra.y, q < 2 ? rb.x : rb.y, sel);
            const uint32_t v = __byte_perm(q < 2 ? rc.x : rc.y, q < 2 ? rd.x : rd.y, sel);
            uint32_t b0, b1, c0, c1;
            codes_to_half(u, b0, c0);         // {key t, key t + 4} of the first rank, of the second
            codes_to_half(v, b1, c1);         // {key t + 8, key t + 12}
            mma_f16_16x8x16(o[vb][2 * q], w[0][0], w[0][1], w[1][0], w[1][1], b0, b1);
            mma_f16_16x8x16(o[vb][2 * q + 1], w[0][0], w[0][1], w[1][0], w[1][1], c0, c1);
          }
        }
      }
      w[0][0] = w[2][0];
      w[0][1] = w[2][1];
      w[1][0] = w[3][0];
      w[1][1] = w[3][1];
    }
  }
  copy_wait<0>();

  // join the four warps: common reference per row, sums in shared memory (the rings are done with)
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  if (t4 == 0) {
    s.m[warp][g] = R;
    s.l[warp][g] = l;
  }
  __syncthreads();
  float* sums = reinterpret_cast<float*>(ring_mem) + warp * (kStreamRows * LSVD_MAX_RANK);
  float top = s.m[0][g];
#pragma unroll
  for (int w = 1; w < kChunkWarps; ++w) top = fmaxf(top, s.m[w][g]);
  const float by = ex2(R - (top == -INFINITY ? 0.f : top));
#pragma unroll
  for (int vb = 0; vb < 2; ++vb)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int rank = 64 * vb + 16 * t4 + 8 * e;
      if (rank < rv) {
        float4* dst = reinterpret_cast<float4*>(sums + g * LSVD_MAX_RANK + rank);
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = (o[vb][j][e] + o[vb][j][2 + e]) * by;
        dst[0] = make_float4(y[0], y[1], y[2], y[3]);
        dst[1] = make_float4(y[4], y[5], y[6], y[7]);
      }
    }
  __syncthreads();
  const float* all = reinterpret_cast<const float*>(ring_mem);
  for (int x = threadIdx.x; x < rows * rv; x += kChunkThreads) {
    const int row = x / rv, rank = x - row * rv;
    const int token = r.start + row0 + row;
    float top = s.m[0][row], sum = 0.f, v = 0.f;
#pragma unroll
    for (int w = 1; w < kChunkWarps; ++w) top = fmaxf(top, s.m[w][row]);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < kChunkWarps; ++w) {
      sum += s.l[w][row] * ex2(s.m[w][row] - base);
      v += all[w * (kStreamRows * LSVD_MAX_RANK) + row * LSVD_MAX_RANK + rank];
    }
    if (p.stream_partials) {
      const int64_t at = (static_cast<int64_t>(split) * p.batch + b) * p.stream_stride + row0 + row;
      p.stream_o[at * p.sum_rv + H.v_col + rank] = v;
      if (rank == 0) p.stream_ml[at * p.num_heads + h] = make_float2(top, sum);
    } else {
      p.out_latent[token * p.out_latent_stride_t + H.v_col + rank] = __float2half_rn(sum == 0.f ? 0.f : v / sum);
    }
  }
}

// Joins the splits of a row and applies the V up-factor: grid (heads, tiles of 8 rows).
constexpr int kMergeRows = 8;
__global__ void __launch_bounds__(128) chunk_merge_kernel(const __grid_constant__ ChunkParams p) {
  __shared__ float lat[kMergeRows][LSVD_MAX_RANK];
  __shared__ int64_t first[kMergeRows], step[kMergeRows];      // row of the first split, rows between splits
  __shared__ int splits[kMergeRows];                            // 0: not a row for the merge; < 0: of the tile form
  grid_dependency_release();
  grid_dependency_wait();
  const int h = blockIdx.x, token0 = blockIdx.y * kMergeRows;
  const ChunkHead H = p.head[h];
  const int rv = H.nv * 16;
  if (threadIdx.x < kMergeRows) {
    const int token = token0 + threadIdx.x;
    int lo = 0, hi = p.batch - 1;               // last request whose first row is not behind the token
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (p.b_start_loc[mid] <= token) lo = mid; else hi = mid - 1;
    }
    const ChunkRequest r = chunk_request(p, lo, false);
    int n = 0;
    if (token < p.num_tokens && token >= r.start && token < r.start + r.n) {
      if (r.n > p.tile_min) {
        n = p.tile_splits > 1 ? -p.tile_splits : 0;
        first[threadIdx.x] = token;
        step[threadIdx.x] = p.num_tokens;
      } else {
        n = p.stream_partials ? p.stream_splits : 0;
        first[threadIdx.x] = static_cast<int64_t>(lo) * p.stream_stride + token - r.start;
        step[threadIdx.x] = static_cast<int64_t>(p.batch) * p.stream_stride;
      }
    }
    splits[threadIdx.x] = n;
  }
  __syncthreads();
  bool any = false;
  for (int i = 0; i < kMergeRows; ++i) any = any || splits[i] != 0;
  if (!any) return;
  for (int x = threadIdx.x; x < kMergeRows * rv; x += blockDim.x) {
    const int row = x / rv, rank = x - row * rv, token = token0 + row;
    if (splits[row] == 0) continue;
    const bool tile = splits[row] < 0;
    const int n = abs(splits[row]);
    const float2* ml = (tile ? p.tile_ml : p.stream_ml) + first[row] * p.num_heads + h;
    const float* po = (tile ? p.tile_o : p.stream_o) + first[row] * p.sum_rv + H.v_col + rank;
    float top = -INFINITY;
    for (int s = 0; s < n; ++s) top = fmaxf(top, ml[s * step[row] * p.num_heads].x);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, v = 0.f;
    for (int s = 0; s < n; ++s) {
      const float2 part = ml[s * step[row] * p.num_heads];
      if (part.y == 0.f) continue;                // nothing seen in this split
      const float c = ex2(part.x - base);
      sum += part.y * c;
      v += po[s * step[row] * p.sum_rv] * c;
    }
    v = sum == 0.f ? 0.f : v / sum;
    lat[row][rank] = v;
    if (p.out_latent != nullptr) p.out_latent[token * p.out_latent_stride_t + H.v_col + rank] = __float2half_rn(v);
  }
  if (p.out == nullptr) return;
  __syncthreads();
  for (int d = threadIdx.x; d < p.head_dim; d += blockDim.x) {
    float acc[kMergeRows];
#pragma unroll
    for (int i = 0; i < kMergeRows; ++i) acc[i] = 0.f;
    for (int rank = 0; rank < rv; ++rank) {
      const float w = __half2float(p.up_v[static_cast<int64_t>(H.v_col + rank) * p.up_v_row_stride + d]);
#pragma unroll
      for (int i = 0; i < kMergeRows; ++i) acc[i] = fmaf(w, lat[i][rank], acc[i]);
    }
#pragma unroll
    for (int i = 0; i < kMergeRows; ++i)
      if (splits[i] != 0) p.out[(token0 + i) * p.out_stride_t + h * p.out_stride_h + d] = __float2half_rn(acc[i]);
  }
}

struct ChunkPlan {
  bool stream, tile;                       // which forms are launched
  int stream_splits, stream_split_len, stream_stride;
  int tiles, tile_splits, tile_split_len, tile_min;
  bool tile_rows;                          // the tile form needs rows for partial results: it is split, or a piece is folded
};

static void chunk_split(int64_t blocks, int64_t want, int least, int unit, int max_len, int* splits, int* len) {
  const int64_t most = std::max(1, max_len / least);
  const int64_t n = std::max<int64_t>(1, std::min(most, std::min<int64_t>(want / std::max<int64_t>(1, blocks), 128)));
  const int64_t piece = std::max<int64_t>(unit, (max_len + n - 1) / n);
  *len = static_cast<int>((piece + unit - 1) / unit * unit);
  *splits = std::max(1, (max_len + *len - 1) / *len);
}

// Requests of up to 16 new tokens go to the stream form (from 9 on as two blocks, each with its own pass over the keys), longer ones
// to the tile form: eight requests over 4091 keys with 8, 9 and 16 new tokens each take 139, 226 and 230 us so, 392 from 9 on in the
// tile form.  A single request of a step that may bring more than 16 always goes to the tile form (one launch).  The keys are split
// where the rows alone are too few blocks: stream form, four rounds of the resident blocks (three per SM), pieces of 256 keys or more
// (at two, three, four, six and eight rounds: eight requests of five tokens 128, 131, 136, 151, 169 us, 16 single tokens 232, 206, 200,
// 210, 217 us); tile form, two rounds (one per SM), 512 keys or more.
static ChunkPlan chunk_plan(int batch, int num_heads, int num_tokens, int max_new, int max_len) {
  ChunkPlan c{};
  const int64_t sms = std::max(1, device_sm_count());
  const int longest = std::max(1, std::min(max_new, num_tokens));
  c.tile = longest > kStreamMost;
  c.stream = !c.tile || batch > 1;
  c.tile_min = c.stream ? kStreamMost : 0;
  c.stream_stride = std::min(kStreamMost, longest);
  chunk_split(static_cast<int64_t>(num_heads) * batch, 4 * 3 * sms, 256, 128, max_len, &c.stream_splits, &c.stream_split_len);
  const int64_t of_tokens = num_tokens / kChunkTileRows + std::min<int64_t>(batch, num_tokens / (c.tile_min + 1));
  const int64_t of_requests = static_cast<int64_t>(batch) * ((static_cast<int64_t>(longest) + kChunkTileRows - 1) / kChunkTileRows);
  c.tiles = static_cast<int>(std::max<int64_t>(1, std::min(of_tokens, of_requests)));
  chunk_split(static_cast<int64_t>(num_heads) * c.tiles, 2 * sms, 512, 64, max_len, &c.tile_splits, &c.tile_split_len);
  if (!c.stream) c.stream_splits = 0;
  if (!c.tile) c.tile_splits = 0;
  c.tile_rows = c.tile && (c.tile_splits > 1 || max_len > kFoldKeys);
  return c;
}

struct ChunkWorkspace {
  size_t stream_ml, stream_o, tile_ml, tile_o, total;
};

// The stream form always has room for partial results (its up-projection is the merge's), the tile form when it is split or its
// rows may have more keys than one accumulator sums.
static ChunkWorkspace chunk_workspace(const ChunkPlan& c, int batch, int num_heads, int sum_rv, int num_tokens) {
  auto align = [](size_t x) { return (x + 255) / 256 * 256; };
  const size_t srows = static_cast<size_t>(c.stream_splits) * batch * c.stream_stride;
  const size_t trows = c.tile_rows ? static_cast<size_t>(c.tile_splits) * num_tokens : 0;
  ChunkWorkspace w{};
  w.stream_o = align(srows * num_heads * sizeof(float2));
  w.tile_ml = w.stream_o + align(srows * sum_rv * sizeof(float));
  w.tile_o = w.tile_ml + align(trows * num_heads * sizeof(float2));
  w.total = w.tile_o + align(trows * sum_rv * sizeof(float));
  return w;
}

}  // namespace lsvd

extern "C" size_t lsvd_attn_chunk_workspace_bytes(int32_t batch, int32_t num_heads, int32_t sum_rank_v, int32_t num_tokens,
                                                  int32_t max_new_in_batch, int32_t max_len_in_batch) {
  using namespace lsvd;
  if (batch <= 0 || num_heads <= 0 || sum_rank_v <= 0 || num_tokens < 0 || max_new_in_batch < 0 || max_len_in_batch < 0) return 0;
  const ChunkWorkspace w = chunk_workspace(chunk_plan(batch, num_heads, num_tokens, max_new_in_batch, max_len_in_batch), batch, num_heads,
                                           sum_rank_v, num_tokens);
  return w.total;
}

extern "C" int lsvd_attn_chunk(const lsvd_attn_chunk_args* a, void* stream) {
  using namespace lsvd;
  if (a == nullptr) return LSVD_ERR_INVALID_ARG;
  if (a->batch <= 0 || a->num_heads <= 0 || a->num_heads > LSVD_MAX_HEADS) return LSVD_ERR_INVALID_ARG;
  if (a->head_dim <= 0 || a->head_dim > 256 || (a->head_dim % 8) != 0) return LSVD_ERR_INVALID_ARG;
  if (a->num_slots <= 0 || a->max_len_in_batch < 0 || a->num_tokens < 0 || a->max_new_in_batch < 0) return LSVD_ERR_INVALID_ARG;
  if (!a->k_off || !a->v_off || a->k_off[0] != 0 || a->v_off[0] != 0) return LSVD_ERR_INVALID_ARG;
  ChunkParams p{};
  for (int h = 0; h < a->num_heads; ++h) {
    const int rk = a->k_off[h + 1] - a->k_off[h], rv = a->v_off[h + 1] - a->v_off[h];
    if (rk <= 0 || rv <= 0 || rk > LSVD_MAX_RANK || rv > LSVD_MAX_RANK || (rk % 16) != 0 || (rv % 16) != 0) return LSVD_ERR_INVALID_ARG;
    p.head[h] = {a->k_off[h], a->v_off[h], static_cast<int16_t>(rk / 16), static_cast<int16_t>(rv / 16)};
  }
  const int sum_rk = a->k_off[a->num_heads], sum_rv = a->v_off[a->num_heads];
  if (a->num_tokens == 0) return LSVD_OK;
  if (!a->q || !a->cache_k || !a->cache_v || !a->scale_k || !a->scale_v || !a->up_k || !a->req_to_token || !a->b_req_idx ||
      !a->b_seq_len || !a->b_start_loc)
    return LSVD_ERR_INVALID_ARG;
  if ((a->out == nullptr && a->out_latent == nullptr) || (a->out != nullptr && a->up_v == nullptr)) return LSVD_ERR_INVALID_ARG;
  if (a->cache_layout != LSVD_CACHE_SLOT_MAJOR && a->cache_layout != LSVD_CACHE_HEAD_MAJOR) return LSVD_ERR_INVALID_ARG;
  if (!aligned(a->cache_k, 16) || !aligned(a->cache_v, 16)) return LSVD_ERR_INVALID_ARG;
  if (a->cache_layout == LSVD_CACHE_SLOT_MAJOR &&
      ((a->cache_k_row_stride % 16) != 0 || (a->cache_v_row_stride % 16) != 0 || a->cache_k_row_stride < sum_rk ||
       a->cache_v_row_stride < sum_rv || a->scale_k_row_stride < a->num_heads || a->scale_v_row_stride < a->num_heads))
    return LSVD_ERR_INVALID_ARG;
  if (a->cache_layout == LSVD_CACHE_SLOT_MAJOR && (a->cache_k_row_stride > 0x7fffffffLL || a->cache_v_row_stride > 0x7fffffffLL))
    return LSVD_ERR_UNSUPPORTED;
  const void* halves[] = {a->q, a->up_k, a->up_v, a->scale_k, a->scale_v, a->out, a->out_latent};
  for (const void* x : halves)
    if (!aligned(x, 2)) return LSVD_ERR_INVALID_ARG;
  const void* words[] = {a->req_to_token, a->b_req_idx, a->b_seq_len, a->b_start_loc, a->alibi_slopes, a->b_prefix_len, a->key_begin,
                         a->mem_index, a->status_word};
  for (const void* x : words)
    if (!aligned(x, 4)) return LSVD_ERR_INVALID_ARG;
  if (a->up_k_row_stride < a->head_dim || (a->out != nullptr && a->up_v_row_stride < a->head_dim)) return LSVD_ERR_INVALID_ARG;
  if (a->req_to_token_rows <= 0 || (a->req_to_token_rows > 1 && a->req_to_token_stride < a->max_len_in_batch)) return LSVD_ERR_INVALID_ARG;
  if (a->max_len_in_batch > (1 << 30)) return LSVD_ERR_UNSUPPORTED;
  if (!std::isfinite(a->softcap) || !std::isfinite(a->sm_scale) || a->softcap < 0.f || a->window < 0) return LSVD_ERR_INVALID_ARG;
  if (a->softcap > 0.f && a->softcap < 1e-6f) return LSVD_ERR_UNSUPPORTED;      // (2 / softcap times a score has to stay in range)
  const ChunkPlan c = chunk_plan(a->batch, a->num_heads, a->num_tokens, a->max_new_in_batch, a->max_len_in_batch);
  const int64_t stream_blocks = static_cast<int64_t>(a->batch) * (c.stream_stride > kStreamRows ? 2 : 1);
  if (a->batch > 65535 || stream_blocks > 65535 || c.tiles > 65535 || (a->num_tokens + kMergeRows - 1) / kMergeRows > 65535) return LSVD_ERR_UNSUPPORTED;
  const bool stream_partials = c.stream && (c.stream_splits > 1 || a->out != nullptr);
  const bool merge = stream_partials || c.tile_splits > 1;
  const ChunkWorkspace w = chunk_workspace(c, a->batch, a->num_heads, sum_rv, a->num_tokens);
  if ((merge || c.tile_rows) && (a->workspace == nullptr || a->workspace_bytes < w.total || !aligned(a->workspace, 256))) return LSVD_ERR_WORKSPACE;

  p.q = static_cast<const __half*>(a->q);
  p.q_stride_t = a->q_stride_t;
  p.q_stride_h = a->q_stride_h;
  p.cache_k = a->cache_k;
  p.cache_v = a->cache_v;
  p.scale_k = static_cast<const __half*>(a->scale_k);
  p.scale_v = static_cast<const __half*>(a->scale_v);
  p.cache_k_row_stride = a->cache_k_row_stride;
  p.cache_v_row_stride = a->cache_v_row_stride;
  p.scale_k_row_stride = a->scale_k_row_stride;
  p.scale_v_row_stride = a->scale_v_row_stride;
  p.up_k = static_cast<const __half*>(a->up_k);
  p.up_v = static_cast<const __half*>(a->up_v);
  p.up_k_row_stride = a->up_k_row_stride;
  p.up_v_row_stride = a->up_v_row_stride;
  p.req_to_token = a->req_to_token;
  p.req_to_token_stride = a->req_to_token_stride;
  p.b_req_idx = a->b_req_idx;
  p.b_seq_len = a->b_seq_len;
  p.b_start_loc = a->b_start_loc;
  p.out = static_cast<__half*>(a->out);
  p.out_stride_t = a->out_stride_t;
  p.out_stride_h = a->out_stride_h;
  p.out_latent = static_cast<__half*>(a->out_latent);
  p.out_latent_stride_t = a->out_latent_stride_t;
  p.status_word = a->status_word;
  p.alibi_slopes = a->alibi_slopes;
  p.b_prefix_len = a->b_prefix_len;
  p.key_begin = a->key_begin;
  p.mem_index = a->mem_index;
  p.score_scale = a->sm_scale > 0.f ? a->sm_scale : 1.0f / std::sqrt(static_cast<float>(a->head_dim));
  p.softcap = a->softcap;
  p.cap_u = a->softcap > 0.f ? 2.f / a->softcap : 0.f;
  p.cap_log2e = std::min(a->softcap * kChunkLog2e, FLT_MAX);
  p.batch = a->batch;
  p.num_heads = a->num_heads;
  p.head_dim = a->head_dim;
  p.max_len = a->max_len_in_batch;
  p.num_tokens = a->num_tokens;
  p.max_new = a->max_new_in_batch;
  p.num_slots = a->num_slots;
  p.r2t_rows = a->req_to_token_rows;
  p.causal = a->causal;
  p.window = a->window;
  p.head_major = a->cache_layout == LSVD_CACHE_HEAD_MAJOR ? 1 : 0;
  p.sum_rv = sum_rv;
  p.q_vec = aligned(a->q, 8) && (a->q_stride_t % 4) == 0 && (a->q_stride_h % 4) == 0;
  p.up_k_vec = aligned(a->up_k, 8) && (a->up_k_row_stride % 4) == 0;
  p.up_v_vec = aligned(a->up_v, 8) && (a->up_v_row_stride % 4) == 0;
  p.out_vec2 = aligned(a->out, 4) && (a->out_stride_t % 2) == 0 && (a->out_stride_h % 2) == 0;
  p.out_lat_vec16 = aligned(a->out_latent, 16) && (a->out_latent_stride_t % 8) == 0;
  p.stream_splits = c.stream_splits;
  p.stream_split_len = c.stream_split_len;
  p.stream_stride = c.stream_stride;
  p.tile_splits = c.tile_splits;
  p.tile_split_len = c.tile_split_len;
  p.tile_min = c.tile_min;
  p.stream_partials = stream_partials;
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  p.stream_ml = reinterpret_cast<float2*>(ws + w.stream_ml);
  p.stream_o = reinterpret_cast<float*>(ws + w.stream_o);
  p.tile_ml = reinterpret_cast<float2*>(ws + w.tile_ml);
  p.tile_o = reinterpret_cast<float*>(ws + w.tile_o);

  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (c.stream) {
    const bool cap = a->softcap > 0.f, bias = a->alibi_slopes != nullptr;
    void (*kern)(ChunkParams) = cap ? (bias ? chunk_stream_kernel<true, true> : chunk_stream_kernel<true, false>)
                                    : (bias ? chunk_stream_kernel<false, true> : chunk_stream_kernel<false, false>);
    const int smem = kChunkWarps * kRingBytes;
    LSVD_CUDA_TRY(ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem));
    LSVD_CUDA_TRY(launch_chained(kern, dim3(a->num_heads, static_cast<unsigned>(stream_blocks), c.stream_splits), dim3(kChunkThreads), smem, st, 1, true, p));
  }
  if (c.tile) LSVD_CUDA_TRY(launch_chunk_tile(p, c.tiles, st));
  if (merge)
    LSVD_CUDA_TRY(launch_chained(chunk_merge_kernel, dim3(a->num_heads, (a->num_tokens + kMergeRows - 1) / kMergeRows), dim3(128), 0, st, 1,
                                 true, p));
  return LSVD_OK;
}
