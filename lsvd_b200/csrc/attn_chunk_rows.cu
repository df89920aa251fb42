// Attention of new tokens over the paged int8 latent cache, row-tile form: 128 query rows of one request and head per block.
// (The mathematics and the stream form, for requests of few rows, are in attn_chunk.cu.)
//
// The block's warps share every 64 keys: the rows of codes arrive by 16-byte asynchronous copies in a ring of four stages, and
// each warp works on its own query rows against them, so a block reads a key once for 128 rows.  Nothing is exchanged between
// warps: a warp folds its rows into q~ = B_k q with the tensor cores, keeps q~, the running maxima, sums and outputs in
// registers, and finishes with o = B_v^T o_lat.  Two shapes of the same loop:
//   ranks up to 64    32 rows a warp (two m16 tiles), four warps: a code is widened to fp16 once for two products
//   ranks up to 128   16 rows a warp, so that q~ and o stay in registers; the block does its 128 rows in two passes
// Codes are widened in registers (two operations per pair), which costs about a third of the softmax's issue slots and
// saves the shared-memory round trip of a widened copy.
#include <algorithm>

#include "attn_chunk.cuh"
#include "devfn.cuh"

namespace lsvd {

constexpr int kRowsPerBlock = 128;
constexpr int kRowWarps = 4;
constexpr int kRowThreads = kRowWarps * 32;
constexpr int kRowKeys = 64;                  // keys of a stage
constexpr int kRowStages = 4;
constexpr int kSlotRing = 8;
constexpr int kRowSmem = kRowStages * kRowKeys * 2 * LSVD_MAX_RANK;       // 64 KB: ranks of 128 + 128
constexpr int kRowShift = 10;

struct __align__(16) RowShared {
  float sk[kRowWarps][32], sv[kRowWarps][32];     // scales of the warp's 32 keys in hand
  int32_t slot[kSlotRing][kRowKeys];              // slots of the stages' keys, -1: none
  int32_t lo[kRowsPerBlock], hi[kRowsPerBlock];
  int32_t b, tile;
};

// One pass of the block: rows row0 .. of the request, MT * 16 of them per warp; kNB 64-rank blocks of K and of V.
template <int MT, int kNB, bool kCap, bool kBias>
__device__ __forceinline__ void row_pass(const ChunkParams& p, const ChunkRequest& r, const ChunkHead& H, int h, int split, int row0,
                                         int rows, RowShared& s, uint8_t* ring) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int rk = H.nk * 16, rv = H.nv * 16;
  // visible keys of the rows, and of the pass
  __syncthreads();
  for (int i = tid; i < MT * 16 * kRowWarps; i += kRowThreads) {
    KeyRange k;
    k.lo = k.hi = 0;
    if (i < rows) k = visible_keys(p, r, p.b_prefix_len != nullptr ? p.b_prefix_len[s.b] : 0, row0 + i);
    s.lo[i] = k.lo;
    s.hi[i] = k.hi;
  }
  __syncthreads();
  int kbeg = 0x7fffffff, kend = 0;
  for (int i = lane; i < MT * 16 * kRowWarps; i += 32) {
    if (s.hi[i] > s.lo[i]) kbeg = min(kbeg, s.lo[i]);
    kend = max(kend, s.hi[i]);
  }
  kbeg = __reduce_min_sync(0xffffffffu, kbeg) & ~31;
  kend = __reduce_max_sync(0xffffffffu, kend);
  if (p.tile_splits > 1) {
    kbeg = static_cast<int>(max(static_cast<int64_t>(kbeg), static_cast<int64_t>(split) * p.tile_split_len));
    kend = static_cast<int>(min(static_cast<int64_t>(kend), (static_cast<int64_t>(split) + 1) * p.tile_split_len));
  }
  const int ntiles = kend > kbeg ? (kend - kbeg + kRowKeys - 1) / kRowKeys : 0;
  const int wrow = warp * MT * 16;              // the warp's first row in the pass
  const bool live = wrow < rows;
  // keys that any / every row of the warp sees
  int outer_lo, outer_hi, inner_lo, inner_hi;
  {
    const int i = wrow + min(lane, MT * 16 - 1);
    const bool on = i < rows;
    outer_lo = __reduce_min_sync(0xffffffffu, on && s.hi[i] > s.lo[i] ? s.lo[i] : 0x7fffffff);
    outer_hi = __reduce_max_sync(0xffffffffu, on ? s.hi[i] : 0);
    inner_lo = __reduce_max_sync(0xffffffffu, on ? s.lo[i] : 0);
    inner_hi = __reduce_min_sync(0xffffffffu, on ? s.hi[i] : 0x7fffffff);
  }

  const int32_t* r2t = p.req_to_token + static_cast<int64_t>(r.req) * p.req_to_token_stride;
  const int8_t* kbase = p.cache_k + (p.head_major ? static_cast<int64_t>(H.k_col) * p.num_slots : H.k_col);
  const int8_t* vbase = p.cache_v + (p.head_major ? static_cast<int64_t>(H.v_col) * p.num_slots : H.v_col);
  const int64_t kstride = p.head_major ? rk : p.cache_k_row_stride, vstride = p.head_major ? rv : p.cache_v_row_stride;
  const __half* ksc = p.scale_k + (p.head_major ? static_cast<int64_t>(h) * p.num_slots : h);
  const __half* vsc = p.scale_v + (p.head_major ? static_cast<int64_t>(h) * p.num_slots : h);
  const int64_t kss = p.head_major ? 1 : p.scale_k_row_stride, vss = p.head_major ? 1 : p.scale_v_row_stride;
  const int k_bytes = kRowKeys * rk, stage_bytes = kRowKeys * (rk + rv);
  const uint32_t inv_k = 65536u / H.nk + 1, inv_v = 65536u / H.nv + 1;       // x / n = x * inv >> 16 for x < 512, n <= 8

  auto fetch_slot = [&](int i) {
    int slot = -1;
    const int key = kbeg + i * kRowKeys + tid;
    if (tid < kRowKeys && i < ntiles && key < kend) slot = r2t[key];
    if (slot >= p.num_slots) {
      report_status(p.status_word, LSVD_ERR_BOUNDS);
      slot = -1;
    }
    return slot;
  };
  auto request = [&](int i) {
    const int32_t* slots = s.slot[i & (kSlotRing - 1)];
    uint8_t* kd = ring + (i & (kRowStages - 1)) * stage_bytes;
    uint8_t* vd = kd + k_bytes;
    for (int x = tid; x < kRowKeys * H.nk; x += kRowThreads) {
      const int tok = (x * inv_k) >> 16, piece = x - tok * H.nk, sl = slots[tok];
      copy16_or_zero(kd + k_row_of(tok) * rk + k_piece_at(k_row_of(tok), piece, H.nk) * 16,
                     kbase + static_cast<int64_t>(max(sl, 0)) * kstride + piece * 16, sl >= 0);
    }
    for (int x = tid; x < kRowKeys * H.nv; x += kRowThreads) {
      const int tok = (x * inv_v) >> 16, piece = x - tok * H.nv, sl = slots[tok];
      copy16_or_zero(vd + tok * rv + v_piece_at(tok, piece, H.nv) * 16, vbase + static_cast<int64_t>(max(sl, 0)) * vstride + piece * 16,
                     sl >= 0);
    }
  };
  // scales of this lane's key in 32-key group `c` of the pass (two groups a stage)
  auto load_scales = [&](int c, float& a, float& b) {
    a = b = 0.f;
    if (c >= 2 * ntiles) return;
    const int sl = s.slot[(c >> 1) & (kSlotRing - 1)][(c & 1) * 32 + lane];
    if (sl >= 0) {
      a = __half2float(ksc[sl * kss]);
      b = __half2float(vsc[sl * vss]);
    }
  };

  if (tid < kRowKeys)
    for (int i = 0; i < kRowStages; ++i) s.slot[i][tid] = fetch_slot(i);
  int slot_ahead = fetch_slot(kRowStages);
  __syncthreads();
  for (int i = 0; i < kRowStages - 1; ++i) {
    if (i < ntiles) request(i);
    copy_commit();
  }

  // q~ of the warp's rows as fp16 A fragments.  Column c = 2 t + e of the product's 8-rank tile (mb, i, half) is rank
  // 64 mb + 16 t + 4 i + 2 half + e: the accumulators of lane (g, t) are then the entries that its fragment of the score
  // product needs, whose k index runs over the ranks in the order in which the lane reads a row's codes.
  uint32_t qa[MT][kNB][4][4];
  float f[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m) f[m][0] = f[m][1] = 0.f;
  if (live && ntiles > 0) {
    const __half* qrow[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        qrow[m][e] = p.q + static_cast<int64_t>(r.start + row0 + min(wrow + 16 * m + g + 8 * e, rows - 1)) * p.q_stride_t + h * p.q_stride_h;
    float acc[MT][kNB][4][2][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int mb = 0; mb < kNB; ++mb)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[m][mb][i][e >> 2][e & 3] = 0.f;
    for (int d0 = 0; d0 < p.head_dim; d0 += 16) {
      const int d = d0 + 4 * t4;
      uint2 a[MT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < 2; ++e) a[m][e] = load_halves4(qrow[m][e] + d, p.head_dim - d, p.q_vec);
#pragma unroll
      for (int mb = 0; mb < kNB; ++mb)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int rank = 64 * mb + 16 * (g >> 1) + 4 * i + 2 * half + (g & 1);
            uint2 b = make_uint2(0u, 0u);
            if (rank < rk) b = load_halves4(p.up_k + static_cast<int64_t>(H.k_col + rank) * p.up_k_row_stride + d, p.head_dim - d, p.up_k_vec);
#pragma unroll
            for (int m = 0; m < MT; ++m) mma_f16_16x8x16(acc[m][mb][i][half], a[m][0].x, a[m][1].x, a[m][0].y, a[m][1].y, b.x, b.y);
          }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = 0.f;
#pragma unroll
        for (int mb = 0; mb < kNB; ++mb)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int half = 0; half < 2; ++half)
              top = fmaxf(top, fmaxf(fabsf(acc[m][mb][i][half][2 * e]), fabsf(acc[m][mb][i][half][2 * e + 1])));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int ex = exponent_of(top) - 8;                   // entries end up below 2^9
        const float x = pow2i(-ex);
        f[m][e] = fmaxf(p.score_scale * pow2i(ex) * (kCap ? 2.f * kChunkLog2e / p.softcap : kChunkLog2e), 1e-37f);
#pragma unroll
        for (int mb = 0; mb < kNB; ++mb)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            qa[m][mb][i][e] = pack_half2(acc[m][mb][i][0][2 * e] * x, acc[m][mb][i][0][2 * e + 1] * x);
            qa[m][mb][i][2 + e] = pack_half2(acc[m][mb][i][1][2 * e] * x, acc[m][mb][i][1][2 * e + 1] * x);
          }
      }
    }
  }

  int lo[MT][2], hi[MT][2];
  float top_m[MT][2], l[MT][2];
  float o[MT][kNB][8][4];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      lo[m][e] = s.lo[wrow + 16 * m + g + 8 * e];
      hi[m][e] = s.hi[wrow + 16 * m + g + 8 * e];
      top_m[m][e] = -INFINITY;
      l[m][e] = 0.f;
    }
#pragma unroll
    for (int vb = 0; vb < kNB; ++vb)
#pragma unroll
      for (int j = 0; j < 8; ++j) o[m][vb][j][0] = o[m][vb][j][1] = o[m][vb][j][2] = o[m][vb][j][3] = 0.f;
  }
  const int pos0 = r.len - r.n + row0 + wrow + g;
  const float cap_log2e = p.softcap * kChunkLog2e;
  const float slope = kBias ? p.alibi_slopes[h] * kChunkLog2e : 0.f;
  int E = -200;
  float sk_next, sv_next;
  load_scales(0, sk_next, sv_next);

  for (int i = 0; i < ntiles; ++i) {
    copy_wait<kRowStages - 2>();
    __syncthreads();                   // stage i has arrived for everyone, and everyone is done with stage i - 1
    if (tid < kRowKeys) s.slot[(i + kRowStages) & (kSlotRing - 1)][tid] = slot_ahead;
    slot_ahead = fetch_slot(i + kRowStages + 1);
    if (i + kRowStages - 1 < ntiles) request(i + kRowStages - 1);
    copy_commit();
    const uint8_t* stage = ring + (i & (kRowStages - 1)) * stage_bytes;
#pragma unroll 1
    for (int c = 0; c < 2; ++c) {
      const int key0 = kbeg + i * kRowKeys + c * 32;
      const float sk = sk_next, sv = sv_next;
      load_scales(2 * i + c + 1, sk_next, sv_next);
      if (!live || key0 >= outer_hi || key0 + 32 <= outer_lo) continue;       // nothing of this warp's
      const uint32_t valid = __ballot_sync(0xffffffffu, s.slot[i & (kSlotRing - 1)][c * 32 + lane] >= 0);
      const float av = fabsf(sv);
      const int ex = (av > 0.f && av < INFINITY) ? exponent_of(av) : -200;
      const int e_new = max(E, __reduce_max_sync(0xffffffffu, ex));
      __syncwarp();
      s.sk[warp][lane] = sk;
      s.sv[warp][lane] = sv * pow2i(kRowShift - e_new);
      __syncwarp();
      const uint8_t* kd = stage + c * 32 * rk;
      const uint8_t* vd = stage + k_bytes + c * 32 * rv;

      float x[MT][4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int m = 0; m < MT; ++m) x[m][j][0] = x[m][j][1] = x[m][j][2] = x[m][j][3] = 0.f;
#pragma unroll
        for (int mb = 0; mb < kNB; ++mb) {
          if (mb * 4 < H.nk) {
            uint4 w = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
            if (mb * 4 + t4 < H.nk) {
              w = *reinterpret_cast<const uint4*>(kd + (8 * j + g) * rk + k_piece_at(8 * j + g, mb * 4 + t4, H.nk) * 16);
              w.x ^= 0x80808080u; w.y ^= 0x80808080u; w.z ^= 0x80808080u; w.w ^= 0x80808080u;
            }
            uint32_t b0, b1;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              codes_to_half(q == 0 ? w.x : q == 1 ? w.y : q == 2 ? w.z : w.w, b0, b1);
#pragma unroll
              for (int m = 0; m < MT; ++m)
                mma_f16_16x8x16(x[m][j], qa[m][mb][q][0], qa[m][mb][q][1], qa[m][mb][q][2], qa[m][mb][q][3], b0, b1);
            }
          }
        }
      }
      const bool masked = key0 < inner_lo || key0 + 32 > inner_hi || valid != 0xffffffffu;
      float top[MT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m) top[m][0] = top[m][1] = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int k = 8 * j + t4 + 4 * e;
          const float ck = s.sk[warp][k];
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int row = 0; row < 2; ++row) {
              float y = x[m][j][2 * row + e] * (ck * f[m][row]);
              if (kCap) y = capped_log2(y, cap_log2e);
              if (kBias) y = fmaf(-slope, fabsf(static_cast<float>(pos0 + 16 * m + 8 * row - key0 - k)), y);
              if (masked && (!((valid >> k) & 1u) || key0 + k < lo[m][row] || key0 + k >= hi[m][row])) y = -INFINITY;
              x[m][j][2 * row + e] = y;
              top[m][row] = fmaxf(top[m][row], y);
            }
        }
      bool moved = e_new != E;
      float base[MT][2], fresh[MT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int row = 0; row < 2; ++row) {
          float v = top[m][row];
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
          fresh[m][row] = fmaxf(top_m[m][row], v);
          moved = moved || fresh[m][row] != top_m[m][row];
          base[m][row] = fresh[m][row] == -INFINITY ? 0.f : fresh[m][row];
        }
      if (__any_sync(0xffffffffu, moved)) {
        const float shift = pow2i(max(E - e_new, -126));
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const float c0 = ex2(top_m[m][0] - base[m][0]), c1 = ex2(top_m[m][1] - base[m][1]);
          l[m][0] *= c0;
          l[m][1] *= c1;
          const float2 s0 = make_float2(c0 * shift, c0 * shift), s1 = make_float2(c1 * shift, c1 * shift);
#pragma unroll
          for (int vb = 0; vb < kNB; ++vb)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float2 u = mul2(make_float2(o[m][vb][j][0], o[m][vb][j][1]), s0), v = mul2(make_float2(o[m][vb][j][2], o[m][vb][j][3]), s1);
              o[m][vb][j][0] = u.x; o[m][vb][j][1] = u.y; o[m][vb][j][2] = v.x; o[m][vb][j][3] = v.y;
            }
          top_m[m][0] = fresh[m][0];
          top_m[m][1] = fresh[m][1];
        }
        E = e_new;
      }
      uint32_t w[MT][4][2];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float v0 = s.sv[warp][8 * j + t4], v1 = s.sv[warp][8 * j + t4 + 4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int row = 0; row < 2; ++row) {
            const float p0 = ex2(x[m][j][2 * row] - base[m][row]), p1 = ex2(x[m][j][2 * row + 1] - base[m][row]);
            l[m][row] += p0 + p1;
            float w0 = p0 * v0, w1 = p1 * v1;
            if (masked) {                 // a masked key's weight is zero whatever its scale holds
              if (p0 == 0.f) w0 = 0.f;
              if (p1 == 0.f) w1 = 0.f;
            }
            w[m][j][row] = pack_half2(w0, w1);
          }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int vb = 0; vb < kNB; ++vb) {
          if (vb * 4 < H.nv) {
            uint2 ra = make_uint2(0x80808080u, 0x80808080u), rb = ra, rc = ra, rd = ra;
            if (64 * vb + 8 * g < rv) {
              // (keys four apart share their swizzle)
              const uint8_t* at = vd + (16 * half + t4) * rv + v_piece_at(t4, 4 * vb + (g >> 1), H.nv) * 16 + 8 * (g & 1);
              ra = *reinterpret_cast<const uint2*>(at);
              rb = *reinterpret_cast<const uint2*>(at + 4 * rv);
              rc = *reinterpret_cast<const uint2*>(at + 8 * rv);
              rd = *reinterpret_cast<const uint2*>(at + 12 * rv);
              ra.x ^= 0x80808080u; ra.y ^= 0x80808080u; rb.x ^= 0x80808080u; rb.y ^= 0x80808080u;
              rc.x ^= 0x80808080u; rc.y ^= 0x80808080u; rd.x ^= 0x80808080u; rd.y ^= 0x80808080u;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint32_t sel = (q & 1) ? 0x7362u : 0x5140u;
              const uint32_t u = __byte_perm(q < 2 ? ra.x : ra.y, q < 2 ? rb.x : rb.y, sel);
              const uint32_t v = __byte_perm(q < 2 ? rc.x : rc.y, q < 2 ? rd.x : rd.y, sel);
              uint32_t b0, b1, c0, c1;
              codes_to_half(u, b0, c0);
              codes_to_half(v, b1, c1);
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                mma_f16_16x8x16(o[m][vb][2 * q], w[m][2 * half][0], w[m][2 * half][1], w[m][2 * half + 1][0], w[m][2 * half + 1][1], b0, b1);
                mma_f16_16x8x16(o[m][vb][2 * q + 1], w[m][2 * half][0], w[m][2 * half][1], w[m][2 * half + 1][0], w[m][2 * half + 1][1], c0, c1);
              }
            }
          }
        }
      }
    }
  }
  copy_wait<0>();

  // ---- results: lane (g, t) holds ranks 64 vb + 16 t + n and + 8 + n (n = tile) of rows g and g + 8 -------------------------
  const float back = E > -200 ? pow2i(E - kRowShift) : 1.f;
  const bool to_up = p.out != nullptr && p.tile_splits == 1;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int row = 0; row < 2; ++row) {
      float sum = l[m][row];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      const int i = wrow + 16 * m + g + 8 * row;
      const int token = r.start + row0 + i;
      const float by = p.tile_splits > 1 ? back : (sum == 0.f ? 0.f : back / sum);
#pragma unroll
      for (int vb = 0; vb < kNB; ++vb)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          o[m][vb][j][2 * row] = by == 0.f ? 0.f : o[m][vb][j][2 * row] * by;
          o[m][vb][j][2 * row + 1] = by == 0.f ? 0.f : o[m][vb][j][2 * row + 1] * by;
        }
      if (i >= rows) continue;
      if (p.tile_splits > 1) {
        const int64_t part = static_cast<int64_t>(split) * p.num_tokens + token;
        if (t4 == 0) p.tile_ml[part * p.num_heads + h] = make_float2(top_m[m][row], sum);
        if (ntiles > 0) {
          float* dst = p.tile_o + part * p.sum_rv + H.v_col;
#pragma unroll
          for (int vb = 0; vb < kNB; ++vb)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int rank = 64 * vb + 16 * t4 + 8 * e, at = 2 * row + e;
              if (rank < rv) {
                *reinterpret_cast<float4*>(dst + rank) = make_float4(o[m][vb][0][at], o[m][vb][1][at], o[m][vb][2][at], o[m][vb][3][at]);
                *reinterpret_cast<float4*>(dst + rank + 4) = make_float4(o[m][vb][4][at], o[m][vb][5][at], o[m][vb][6][at], o[m][vb][7][at]);
              }
            }
        }
      } else if (p.out_latent != nullptr) {
        __half* dst = p.out_latent + token * p.out_latent_stride_t + H.v_col;
#pragma unroll
        for (int vb = 0; vb < kNB; ++vb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int rank = 64 * vb + 16 * t4 + 8 * e, at = 2 * row + e;
            if (rank < rv) {
              uint4 y;
              y.x = pack_half2(o[m][vb][0][at], o[m][vb][1][at]);
              y.y = pack_half2(o[m][vb][2][at], o[m][vb][3][at]);
              y.z = pack_half2(o[m][vb][4][at], o[m][vb][5][at]);
              y.w = pack_half2(o[m][vb][6][at], o[m][vb][7][at]);
              store_halves8(dst + rank, y, p.out_lat_vec16);
            }
          }
      }
    }
  if (!to_up) return;

  // ---- o = B_v^T o_lat: the head's factor [r_v x head_dim] in shared memory, o_lat (rounded to fp16, as the latent result
  // is) as A: tiles n = 2 i, 2 i + 1 give the k order 16 t + 2 i, + 8, 16 t + 2 i + 1, + 8 ----------------------------------
  __syncthreads();
  __half* up = reinterpret_cast<__half*>(ring);
  for (int x = tid; x < rv * (p.head_dim >> 2); x += kRowThreads) {
    const int rank = x / (p.head_dim >> 2), d = (x - rank * (p.head_dim >> 2)) * 4;
    *reinterpret_cast<uint2*>(up + rank * p.head_dim + d) =
        load_halves4(p.up_v + static_cast<int64_t>(H.v_col + rank) * p.up_v_row_stride + d, 4, p.up_v_vec);
  }
  __syncthreads();
  if (!live) return;
  for (int d0 = 0; d0 < p.head_dim; d0 += 8) {
    float y[MT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m) y[m][0] = y[m][1] = y[m][2] = y[m][3] = 0.f;
#pragma unroll
    for (int vb = 0; vb < kNB; ++vb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t b0 = 0u, b1 = 0u;
        const int rank = 64 * vb + 16 * t4 + 2 * i;
        if (rank < rv) {
          const uint16_t* at = reinterpret_cast<const uint16_t*>(up) + rank * p.head_dim + d0 + g;
          b0 = at[0] | (static_cast<uint32_t>(at[8 * p.head_dim]) << 16);
          b1 = at[p.head_dim] | (static_cast<uint32_t>(at[9 * p.head_dim]) << 16);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
          mma_f16_16x8x16(y[m], pack_half2(o[m][vb][2 * i][0], o[m][vb][2 * i][1]), pack_half2(o[m][vb][2 * i][2], o[m][vb][2 * i][3]),
                          pack_half2(o[m][vb][2 * i + 1][0], o[m][vb][2 * i + 1][1]),
                          pack_half2(o[m][vb][2 * i + 1][2], o[m][vb][2 * i + 1][3]), b0, b1);
      }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int row = 0; row < 2; ++row) {
        const int i = wrow + 16 * m + g + 8 * row;
        if (i >= rows) continue;
        __half* dst = p.out + static_cast<int64_t>(r.start + row0 + i) * p.out_stride_t + h * p.out_stride_h + d0 + 2 * t4;
        const uint32_t v = pack_half2(y[m][2 * row], y[m][2 * row + 1]);
        if (p.out_vec2) {
          *reinterpret_cast<uint32_t*>(dst) = v;
        } else {
          const __half2 hh = *reinterpret_cast<const __half2*>(&v);
          dst[0] = __low2half(hh);
          dst[1] = __high2half(hh);
        }
      }
  }
}

// grid: (heads, row tiles of all requests (a bound), splits of the keys)
template <bool kCap, bool kBias>
__global__ void __launch_bounds__(kRowThreads, 2) chunk_rows_kernel(const __grid_constant__ ChunkParams p) {
  extern __shared__ __align__(16) uint8_t row_ring[];
  __shared__ RowShared s;
  grid_dependency_release();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, h = blockIdx.x, split = blockIdx.z;
  // which request and row tile: the tiles of the requests that this form takes, in batch order, a request's last tile first
  // (it has the most keys to see)
  if (threadIdx.x < 32) {
    int before = 0, found_b = -1, found_t = 0;
    for (int b0 = 0; b0 < p.batch && found_b < 0; b0 += 32) {
      int tiles = 0;
      if (b0 + lane < p.batch) {
        const ChunkRequest r = chunk_request(p, b0 + lane, h == 0 && blockIdx.y == 0 && split == 0);
        if (r.n > p.tile_min) tiles = (r.n + kRowsPerBlock - 1) / kRowsPerBlock;
      }
      int inc = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      const int mine = static_cast<int>(blockIdx.y) - (before + inc - tiles);
      const uint32_t who = __ballot_sync(0xffffffffu, mine >= 0 && mine < tiles);
      if (who != 0) {
        found_b = b0 + __ffs(who) - 1;
        found_t = __shfl_sync(0xffffffffu, tiles - 1 - mine, __ffs(who) - 1);
      }
      before += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) {
      s.b = found_b;
      s.tile = found_t;
    }
  }
  __syncthreads();
  if (s.b < 0) return;
  const ChunkRequest r = chunk_request(p, s.b, false);
  const int row0 = s.tile * kRowsPerBlock, rows = min(kRowsPerBlock, r.n - row0);
  const ChunkHead H = p.head[h];
  if (H.nk <= 4 && H.nv <= 4) {
    row_pass<2, 1, kCap, kBias>(p, r, H, h, split, row0, rows, s, row_ring);
  } else {
#pragma unroll 1
    for (int half = 0; half < 2; ++half)
      if (rows > 64 * half) row_pass<1, 2, kCap, kBias>(p, r, H, h, split, row0 + 64 * half, min(64, rows - 64 * half), s, row_ring);
  }
}

cudaError_t launch_chunk_rows(const ChunkParams& p, int tiles, cudaStream_t st) {
  const bool cap = p.softcap > 0.f, bias = p.alibi_slopes != nullptr;
  void (*kern)(ChunkParams) = cap ? (bias ? chunk_rows_kernel<true, true> : chunk_rows_kernel<true, false>)
                                  : (bias ? chunk_rows_kernel<false, true> : chunk_rows_kernel<false, false>);
  const cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), kRowSmem);
  if (e != cudaSuccess) return e;
  return launch_chained(kern, dim3(p.num_heads, tiles, p.tile_splits), dim3(kRowThreads), kRowSmem, st, 1, true, p);
}

}  // namespace lsvd
