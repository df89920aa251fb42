// Attention of new tokens over the paged int8 latent cache, tile form: 256 query rows of one request and head per block, on
// tcgen05.  (The mathematics and the stream form, for requests of few rows, are in attn_chunk.cu.)
//
// The rows are two groups of 128.  Per 64 keys a block does, for each group, two products with the weights' softmax between them:
//   S[128 x 64] = q~[128 x r_k] . z_k^T     A and B from shared memory, accumulator in tensor memory (two buffers); A twice,
//                                           what fp16 keeps of q~ and the rest (22 bits in all)
//   O[128 x r_v] += P[128 x 64] . z_v       A = P, written over S in tensor memory (32 columns of what fp16 keeps of it, 32 of the
//                                           rest); B = the codes, ranks contiguous
// Thirteen warps: eight for the softmax (thread = row, no exchange between threads), four that gather the rows by slot, widen
// the int8 codes to fp16 (exact) and store them in the 128-byte-swizzled layouts that the products read, one that issues the
// products.  The codes are widened once for both groups; the score product of tile j + 2 runs while the softmax is at tile j + 1.
//
// What bounds it.  The 16384 exponentials of 64 keys take 1024 cycles of an SM (16 a cycle), the products 1024 at ranks of
// 64 + 64; a prompt of 8191 tokens takes 2.0 us more for each such step of an SM than one of 4096, some 3900 cycles.  The dependent
// chains of the softmax, two warps a scheduler, are what is left (fixed-latency waits lead the stalls, 43 % of the issue slots are
// used).  What moved it, for a prompt of 8191 tokens, 32 heads, ranks 64 + 64, each at its time:
//   * code size: the load warps' passes fully unrolled (compile-time widths) took 1.38 ms, as loops shared by K and V 0.97 ms:
//     with all roles unrolled a third of the instruction fetches missed the SM's cache;
//   * the prologue (q~ = B_k q) and the epilogue (o = B_v^T o_lat) with their factors read by every warp from global memory
//     were 65 of 250 thousand cycles of an average block; with the factors in shared memory 0.88 ms;
//   * four load warps instead of three 0.83 ms (five 0.85, seven 0.84): with three the softmax warps waited a quarter to a third of
//     a step for them;
//   * both halves of q~ in the products, and of o_lat in the up-projection, 0.90 ms; both halves of the weights 1.00 ms; references
//     over the keys that a row sees 1.01 ms; folds 1.03 ms.  With them the error against 64 bits is that of rounding the result
//     alone, before them 1.8 times that.
// Tried and slower: two threads a row with sixteen softmax warps (1.05 against 0.83 ms), the scores read twice instead of kept in
// registers between the maximum and the weights (1.08 ms).  128 rows a block (mma m16n8k16) took 2.6 ms.
//
// O is rescaled only when a row's reference moves (attn_chunk.cuh): a reference is looked for where a tile's largest score and largest
// V scale together are past it, over the keys that the row sees.  Each weight enters the product as two fp16 numbers, its
// first eleven bits and the rest: one rounding to fp16 instead, 2^-11 of every term, made the error against 64 bits 1.2 to 1.4 times that
// of rounding the exact result, the second half costs 4 to 15 % (a prompt of 8191 tokens, 32 heads, ranks 64 + 64: 897 -> 1000 us).
// o_lat meets the up-factor as two fp16 numbers, what fp16 keeps of it and the rest.
//
// The tensor cores cut off what an addition to an accumulator leaves: the error grows by about 2^-23.6 of the sum with each of the 8
// products of a tile where all terms have one sign (8192 keys 0.8e-4, half the error of the fp16 result; 66000 keys 6.6e-4), by a
// quarter of that for sums of both signs.  Every 8192 keys the softmax warps therefore add O to fp32 sums in the workspace, to nearest,
// and start it again from zero.  That costs 1 to 2 % where nothing is folded (code), and 3 to 4 % instead at 4096 keys.
#include <algorithm>

#include "attn_chunk.cuh"
#include "devfn.cuh"
#include "tc5.cuh"

namespace lsvd {

constexpr int kGroupRows = 128;                  // rows of one product: a softmax warpgroup's, thread = row
constexpr int kGroups = 2;
constexpr int kTileRows = kChunkTileRows;
static_assert(kTileRows == kGroups * kGroupRows, "two products' rows");
constexpr int kTileKeys = 64;
constexpr int kSoftmaxWarps = 4 * kGroups, kLoadWarps = 4;
constexpr int kMmaWarp = kSoftmaxWarps + kLoadWarps;
constexpr int kTileThreads = (kMmaWarp + 1) * 32;
constexpr int kLoadThreads = kLoadWarps * 32;
constexpr int kTileSmem = 208 * 1024 + 1024;     // q~ (or o_lat), widened stages, copied codes; 1024 to align
constexpr int kTileMaxStages = 4;
constexpr int kCodeStages = 4;                   // stages of codes on their way (one where four do not fit)
constexpr int kTileSlotRing = 8;
constexpr int kFoldTiles = kFoldKeys / kTileKeys;
static_assert((kFoldTiles & (kFoldTiles - 1)) == 0, "tiles between folds");
constexpr int kTileCols = 512;                   // tensor memory, 256 columns a group: S0 0..63, S1 64..127, O 128..255
constexpr int kGroupCols = 256;
constexpr int kColO = 128;

struct __align__(16) TileShared {
  float sk[kTileMaxStages][kTileKeys], sv[kTileMaxStages][kTileKeys], se[kTileMaxStages][kTileKeys];      // first: read in 16-byte pieces
  uint64_t full[kTileMaxStages], empty[kTileMaxStages];
  uint64_t s_full[kGroups][2], p_full[kGroups][2], o_done[kGroups], q_full[kGroups], last;
  uint32_t live[kTileMaxStages][2];              // keys with a slot, one bit each
  float e_top[kTileMaxStages];                   // largest of se
  int32_t slot[kTileSlotRing][kTileKeys];
  uint32_t tmem;
  volatile uint32_t abort;
  int32_t b, tile;
  int32_t kbeg, kend;
  float scale[kTileRows];                        // power of two taken out of each q~ row
};

// ---- tcgen05 kind::f16 ------------------------------------------------------------------------------------------------
// D = F32 (1 at bit 4), A = B = F16 (0), B's major-ness at bit 16 (1: N contiguous), N >> 3 at bit 17, M >> 4 at bit 24.
__device__ __forceinline__ uint32_t idesc_f16(int n, bool b_n_major) {
  return (1u << 4) | (b_n_major ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kGroupRows >> 4) << 24);
}
__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a_tmem), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// Descriptor of a tile whose rows are K indexes and whose N (or M) index is contiguous: rows of 128 bytes = 64 entries,
// 128-byte swizzle, groups of 8 rows 1024 bytes apart (stride offset), 64-entry blocks `block_bytes` apart (leading offset).
__device__ __forceinline__ uint64_t smem_desc_n_major_sw128(const void* tile, uint32_t block_bytes) {
  const uint64_t addr = smem_u32(tile);
  return ((addr & 0x3FFFFull) >> 4) | (static_cast<uint64_t>(block_bytes >> 4) << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void named_barrier(int id, int count) { asm volatile("barrier.sync %0, %1;" ::"r"(id), "r"(count) : "memory"); }
// True in one lane of the (converged) warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r)::"memory");
  return r != 0u;
}
// Four 8 x 8 tiles of halves, transposed: lane i gives the address of row i & 7 of tile i >> 3.
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], const uint8_t* row) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(row)) : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Two weights as fp16 numbers of their first eleven bits (cut off, not rounded: nothing waits for a conversion back, 2 % of a long
// prompt's time) and of what that leaves.  (An infinite or NaN weight leaves NaN, which a maximum turns into a number: the product is
// as infinite, or no number, as without the rest.)
__device__ __forceinline__ void pack_weights(float2 w, uint32_t& most, uint32_t& rest) {
  const float2 h = make_float2(__uint_as_float(__float_as_uint(w.x) & 0xffffe000u), __uint_as_float(__float_as_uint(w.y) & 0xffffe000u));
  most = pack_half2(h.x, h.y);
  const __half2 x = __hmax2(__float22half2_rn(fma2(h, make_float2(-1.f, -1.f), w)), __floats2half2_rn(-65504.f, -65504.f));
  rest = *reinterpret_cast<const uint32_t*>(&x);
}

// Wait for a phase, bounded by kMbarTimeoutNs; also gives up once another role has.  False: stop and leave.
__device__ __forceinline__ bool tile_wait(TileShared& s, uint64_t* bar, uint32_t parity, int32_t* status_word) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  for (uint32_t i = 0; i < kMbarMaxPolls; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if (s.abort) return false;
    if ((i & 63u) == 63u && global_timer_ns() - t0 > kMbarTimeoutNs) break;
  }
  s.abort = 1;
  report_status(status_word, LSVD_ERR_TIMEOUT);
  return false;
}

// What sums that were folded at a row's reference `at` count at its present one.
__device__ __forceinline__ float folded_factor(float at, float now) { return at == now ? 1.f : ex2(at - now); }

// 16-byte piece `chunk` (0..7) of row `row` in a swizzled [row][128 bytes] tile.
__device__ __forceinline__ uint32_t swizzled(int row, int chunk) { return static_cast<uint32_t>(row * 128 + ((chunk ^ (row & 7)) << 4)); }

// 16 codes -> 16 fp16 values, two 16-byte pieces of a swizzled row.
__device__ __forceinline__ void store_codes(uint8_t* tile, int row, int piece, uint4 w) {
  uint4 a, b;
  codes_to_half(w.x ^ 0x80808080u, a.x, a.y);
  codes_to_half(w.y ^ 0x80808080u, a.z, a.w);
  codes_to_half(w.z ^ 0x80808080u, b.x, b.y);
  codes_to_half(w.w ^ 0x80808080u, b.z, b.w);
  *reinterpret_cast<uint4*>(tile + swizzled(row, 2 * piece)) = a;
  *reinterpret_cast<uint4*>(tile + swizzled(row, 2 * piece + 1)) = b;
}

// q~ = B_k q of the block's rows (mma m16n8k16, like the stream form's; a warp has 32), as fp16 rows of the A operand relative to
// each row's largest entry; the powers of two go to s.scale.  The factor is first brought to `up`, 64 ranks at a time, by the
// `warps` warps that come here (read from global memory by every warp, 8 bytes a lane, the block's prologue took 34000 cycles).
// With more than 64 ranks the first block is computed again once the row's largest entry over both is known.
__device__ __forceinline__ void absorb_tile_rows(const ChunkParams& p, const ChunkHead& H, int h, const ChunkRequest& r, int row0, int rows,
                                                 int warps, TileShared& s, uint8_t* q_tile, int half_bytes, uint8_t* up) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int rk = H.nk * 16, blocks = rk > 64 ? 2 : 1;
  const int steps = (p.head_dim + 15) >> 4, stride = ((p.head_dim * 2 + 127) & ~127) + 32;      // (rows of lanes g on other banks)
  float top[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll 1
  for (int pass = 0; pass < (blocks == 2 ? 3 : 1); ++pass) {      // block 0, block 1, block 0 again
    const int rank0 = pass == 1 ? 64 : 0;
    if (pass > 0) named_barrier(2, warps * 32);
#pragma unroll 4
    for (int x = threadIdx.x; x < 64 * 4 * steps; x += warps * 32) {
      const int rank = x / (4 * steps), d = (x - rank * (4 * steps)) * 4;
      uint2 v = make_uint2(0u, 0u);
      if (rank0 + rank < rk) v = load_halves4(p.up_k + static_cast<int64_t>(H.k_col + rank0 + rank) * p.up_k_row_stride + d, p.head_dim - d, p.up_k_vec);
      *reinterpret_cast<uint2*>(up + rank * stride + d * 2) = v;
    }
    named_barrier(2, warps * 32);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int first = warp * 32 + 16 * m;
      const __half* qa = p.q + static_cast<int64_t>(r.start + row0 + min(first + g, rows - 1)) * p.q_stride_t + h * p.q_stride_h;
      const __half* qb = p.q + static_cast<int64_t>(r.start + row0 + min(first + 8 + g, rows - 1)) * p.q_stride_t + h * p.q_stride_h;
      float acc[8][4];
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll 1
      for (int s0 = 0; s0 < steps; s0 += 8) {
        uint2 a[8], b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int d = (s0 + i) * 16 + 4 * t;
          a[i] = load_halves4(qa + d, p.head_dim - d, p.q_vec);
          b[i] = load_halves4(qb + d, p.head_dim - d, p.q_vec);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (s0 + i >= steps) continue;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint2 u = *reinterpret_cast<const uint2*>(up + (8 * j + g) * stride + (s0 + i) * 32 + 8 * t);
            mma_f16_16x8x16(acc[j], a[i].x, b[i].x, a[i].y, b[i].y, u.x, u.y);
          }
        }
      }
      if (pass < 2) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int j = 0; j < 8; ++j) top[m][e] = fmaxf(top[m][e], fmaxf(fabsf(acc[j][2 * e]), fabsf(acc[j][2 * e + 1])));
          top[m][e] = fmaxf(top[m][e], __shfl_xor_sync(0xffffffffu, top[m][e], 1));
          top[m][e] = fmaxf(top[m][e], __shfl_xor_sync(0xffffffffu, top[m][e], 2));
        }
      }
      if (pass == 0 && blocks == 2) continue;
      uint8_t* block = q_tile + (rank0 >> 6) * kGroupRows * 128;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int ex = exponent_of(top[m][e]) - 8, row = first + 8 * e + g;      // entries end up below 2^9
        const float x = pow2i(-ex);
        if (t == 0) s.scale[row] = pow2i(ex);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (rank0 + 8 * j < rk) {
            uint32_t most, rest;
            pack_half2_rest(acc[j][2 * e] * x, acc[j][2 * e + 1] * x, most, rest);
            uint8_t* at = block + swizzled(row & (kGroupRows - 1), j) + 4 * t;
            *reinterpret_cast<uint32_t*>(at) = most;
            *reinterpret_cast<uint32_t*>(at + half_bytes) = rest;
          }
      }
    }
  }
}

// o = B_v^T o_lat of the block's rows: the factor [r_v x head_dim] in the stages' place, o_lat (fp16, where q~ was) as A
// (mma m16n8k16).  For the whole block, after its tensor memory is gone.
__device__ __forceinline__ void chunk_tile_up(const ChunkParams& p, const TileShared& s, uint8_t* smem) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, h = blockIdx.x;
  const ChunkHead H = p.head[h];
  const int rv = H.nv * 16, half_bytes = ((max(H.nk, H.nv) + 3) >> 2) * kGroupRows * 128, q_bytes = 2 * half_bytes;
  const ChunkRequest r = chunk_request(p, s.b, false);
  const int row0 = s.tile * kTileRows, rows = min(kTileRows, r.n - row0);
  const int stride = p.head_dim * 2 + 16, quads = p.head_dim >> 2;
  uint8_t* up = smem + kGroups * q_bytes;
#pragma unroll 4
  for (int x = tid; x < rv * quads; x += kTileThreads) {
    const int rank = x / quads, d = (x - rank * quads) * 4;
    *reinterpret_cast<uint2*>(up + rank * stride + d * 2) = load_halves4(p.up_v + static_cast<int64_t>(H.v_col + rank) * p.up_v_row_stride + d, 4, p.up_v_vec);
  }
  __syncthreads();
#pragma unroll 1
  for (int w = warp; w * 16 < rows; w += kTileThreads / 32) {
    const int ra = w * 16 + g, la = ra & (kGroupRows - 1), lb = la + 8;
    uint32_t a[2][8][4];             // o_lat as fp16 and what that leaves of it
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const uint8_t* block = smem + (w >> 3) * q_bytes + x * half_bytes + (q >> 2) * kGroupRows * 128 + 4 * t;
        const int c = 2 * (q & 3);
        a[x][q][0] = a[x][q][1] = a[x][q][2] = a[x][q][3] = 0u;
        if (q < H.nv) {
          a[x][q][0] = *reinterpret_cast<const uint32_t*>(block + swizzled(la, c));
          a[x][q][1] = *reinterpret_cast<const uint32_t*>(block + swizzled(lb, c));
          a[x][q][2] = *reinterpret_cast<const uint32_t*>(block + swizzled(la, c + 1));
          a[x][q][3] = *reinterpret_cast<const uint32_t*>(block + swizzled(lb, c + 1));
        }
      }
#pragma unroll 1
    for (int d0 = 0; d0 < p.head_dim; d0 += 16) {      // 16 columns: two products a step, their B fragments by one transposing load
      const bool both = d0 + 8 < p.head_dim;
      const uint8_t* from = up + (lane & 15) * stride + (d0 + (both ? (lane >> 4) * 8 : 0)) * 2;
      float y[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        if (q >= H.nv) continue;
        uint32_t b[4];
        ldmatrix_x4_trans(b, from + 16 * q * stride);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          mma_f16_16x8x16(y[0], a[x][q][0], a[x][q][1], a[x][q][2], a[x][q][3], b[0], b[1]);
          mma_f16_16x8x16(y[1], a[x][q][0], a[x][q][1], a[x][q][2], a[x][q][3], b[2], b[3]);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = ra + 8 * (e & 1), d = d0 + 8 * (e >> 1) + 2 * t;
        if (row >= rows || d >= p.head_dim) continue;
        __half* dst = p.out + static_cast<int64_t>(r.start + row0 + row) * p.out_stride_t + h * p.out_stride_h + d;
        const uint32_t v = pack_half2(y[e >> 1][2 * (e & 1)], y[e >> 1][2 * (e & 1) + 1]);
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
}

// grid: (heads, row tiles of all requests (a bound), splits of the keys)
template <bool kCap, bool kBias>
__global__ void __launch_bounds__(kTileThreads, 1) chunk_tile_kernel(const __grid_constant__ ChunkParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ TileShared s;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  // (the warp's number through a shuffle: the compiler then knows that the roles' branches take whole warps)
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int h = blockIdx.x, split = blockIdx.z;
  const ChunkHead H = p.head[h];
  const int rk = H.nk * 16, rv = H.nv * 16;
  const int kblocks = (H.nk + 3) >> 2, vblocks = (H.nv + 3) >> 2;            // 64-rank blocks
  const int half_bytes = max(kblocks, vblocks) * kGroupRows * 128, q_bytes = 2 * half_bytes;      // of a group: fp16, and the rest
  const int k_bytes = kblocks * kTileKeys * 128, stage_bytes = k_bytes + vblocks * kTileKeys * 128;
  const int code_bytes = kTileKeys * (rk + rv);
  // four stages of each kind up to ranks of 64 + 64, two and one at 128 + 128
  const int room = kTileSmem - 1024 - kGroups * q_bytes;
  const int stages = 4 * stage_bytes + kCodeStages * code_bytes <= room ? 4 : 2;
  const int code_stages = stages * stage_bytes + kCodeStages * code_bytes <= room ? kCodeStages : 1;
  uint8_t* stage0 = smem + kGroups * q_bytes;
  uint8_t* codes = stage0 + stages * stage_bytes;

  grid_dependency_wait();
  // which request and row tile: the tiles of the requests that this form takes, in batch order, a request's last tile first
  // (it has the most keys to see)
  if (warp == 0) {
    int before = 0, found_b = -1, found_t = 0;
    for (int b0 = 0; b0 < p.batch && found_b < 0; b0 += 32) {
      int tiles = 0;
      if (b0 + lane < p.batch) {
        const ChunkRequest r = chunk_request(p, b0 + lane, h == 0 && blockIdx.y == 0 && split == 0);
        if (r.n > p.tile_min) tiles = (r.n + kTileRows - 1) / kTileRows;
      }
      int inc = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      const int first = before + inc - tiles, mine = static_cast<int>(blockIdx.y) - first;
      const uint32_t who = __ballot_sync(0xffffffffu, mine >= 0 && mine < tiles);
      if (who != 0) {
        const int src = __ffs(who) - 1;
        found_b = b0 + src;
        found_t = __shfl_sync(0xffffffffu, tiles - 1 - mine, src);
      }
      before += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) {
      s.b = found_b;
      s.tile = found_t;
      s.kbeg = 0x7fffffff;
      s.kend = 0;
      s.abort = 0;
      for (int i = 0; i < kTileMaxStages; ++i) {
        mbar_init(&s.full[i], kLoadWarps);
        mbar_init(&s.empty[i], 1);
      }
      for (int i = 0; i < kGroups; ++i) {
        mbar_init(&s.s_full[i][0], 1);
        mbar_init(&s.s_full[i][1], 1);
        mbar_init(&s.o_done[i], 1);
      }
    }
  }
  __syncthreads();
  if (s.b < 0) return;
  const ChunkRequest r = chunk_request(p, s.b, false);
  const int row0 = s.tile * kTileRows, rows = min(kTileRows, r.n - row0);
  const int live_warps = (rows + 31) >> 5;                // softmax warps with rows, and groups with such warps
  const int groups = (rows + kGroupRows - 1) / kGroupRows;
  // the row of each softmax thread, and the block's keys
  KeyRange keys;
  keys.lo = keys.hi = 0;
  if (tid < rows) keys = visible_keys(p, r, p.b_prefix_len != nullptr ? p.b_prefix_len[s.b] : 0, row0 + tid);
  if (warp < kSoftmaxWarps) {
    const int lo = __reduce_min_sync(0xffffffffu, keys.hi > keys.lo ? keys.lo : 0x7fffffff);
    const int hi = __reduce_max_sync(0xffffffffu, keys.hi);
    if (lane == 0 && hi > 0) {
      atomicMin(&s.kbeg, lo);
      atomicMax(&s.kend, hi);
    }
  }
  if (tid == 0) {
    for (int i = 0; i < groups; ++i) {
      const int warps = min(4, live_warps - 4 * i);
      mbar_init(&s.p_full[i][0], warps);
      mbar_init(&s.p_full[i][1], warps);
      mbar_init(&s.q_full[i], warps);
    }
    mbar_init(&s.last, 1);
    fence_mbar_init();
  }
  __syncwarp();
  if (warp == kMmaWarp) tmem_alloc(&s.tmem, kTileCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Only now may the next kernel's blocks come in: one that takes tensor memory and then waits for this kernel must find
  // every block of it already served.
  grid_dependency_release();
  const uint32_t tmem = s.tmem;
  int kbeg = s.kbeg & ~(kTileKeys - 1), kend = s.kend;
  if (p.tile_splits > 1) {
    kbeg = static_cast<int>(max(static_cast<int64_t>(kbeg), static_cast<int64_t>(split) * p.tile_split_len));
    kend = static_cast<int>(min(static_cast<int64_t>(kend), (static_cast<int64_t>(split) + 1) * p.tile_split_len));
  }
  const int ntiles = kend > kbeg ? (kend - kbeg + kTileKeys - 1) / kTileKeys : 0;

  if (ntiles > 0 && warp == kMmaWarp) {
    // ================= products: the whole warp keeps step, one elected lane issues =================
    const uint32_t idesc_s = idesc_f16(kTileKeys, false), idesc_o = idesc_f16(rv, true);
    auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, tile_wait(s, bar, parity, p.status_word)); };
    // scores of tile j for both groups; a group's buffer still holds the weights of tile j - 2 until their product is done
    auto scores = [&](int j) {
      const int st = j & (stages - 1);
      if (!wait(&s.full[st], (j / stages) & 1)) return false;
#pragma unroll
      for (int grp = 0; grp < kGroups; ++grp) {
        if (grp >= groups) continue;
        if (j >= 2 && !wait(&s.o_done[grp], j & 1)) return false;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t qdesc = smem_desc_k_major_sw128(smem + grp * q_bytes), kdesc = smem_desc_k_major_sw128(stage0 + st * stage_bytes);
          // 16 ranks a step: 32 bytes of a row; a 64-rank block is a tile of its own.  First what fp16 keeps of q~, then the rest.
          for (int rest = 0; rest < 2; ++rest)
            for (int q = 0; q < H.nk; ++q)
              umma_f16_ss(tmem + grp * kGroupCols + (j & 1) * kTileKeys,
                          qdesc + (rest * (half_bytes >> 4) + (q >> 2) * (kGroupRows * 128 >> 4) + (q & 3) * 2),
                          kdesc + ((q >> 2) * (kTileKeys * 128 >> 4) + (q & 3) * 2), idesc_s, (rest | q) != 0 ? 1u : 0u);
          umma_commit(&s.s_full[grp][j & 1]);
        }
        __syncwarp();
      }
      return true;
    };
    bool go = true;
    for (int grp = 0; grp < groups; ++grp) go = go && wait(&s.q_full[grp], 0);
    go = go && scores(0);
    if (ntiles > 1) go = go && scores(1);
    for (int j = 0; go && j < ntiles; ++j) {
      const int st = j & (stages - 1);
#pragma unroll
      for (int grp = 0; grp < kGroups; ++grp) {
        if (!go || grp >= groups) continue;
        go = wait(&s.p_full[grp][j & 1], (j >> 1) & 1);
        if (!go) continue;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t vdesc = smem_desc_n_major_sw128(stage0 + st * stage_bytes + k_bytes, kTileKeys * 128);
          const uint32_t base = tmem + grp * kGroupCols;
#pragma unroll
          for (int q = 0; q < 2 * kTileKeys / 16; ++q)    // 16 keys a step: two groups of eight rows; 8 columns of P, then of its rest
            umma_f16_ts(base + kColO, base + (j & 1) * kTileKeys + 8 * q, vdesc + (q & 3) * (2048 >> 4), idesc_o, (j | q) != 0 ? 1u : 0u);
          umma_commit(&s.o_done[grp]);
          if (grp + 1 == groups) umma_commit(&s.empty[st]);
        }
        __syncwarp();
      }
      if (go && j + 2 < ntiles) go = scores(j + 2);
    }
  } else if (ntiles > 0 && warp >= kSoftmaxWarps) {
    // ================= gather and widen =================
    const int lt = tid - kSoftmaxWarps * 32, lw = warp - kSoftmaxWarps;
    const int32_t* r2t = p.req_to_token + static_cast<int64_t>(r.req) * p.req_to_token_stride;
    const int8_t* kbase = p.cache_k + (p.head_major ? static_cast<int64_t>(H.k_col) * p.num_slots : H.k_col);
    const int8_t* vbase = p.cache_v + (p.head_major ? static_cast<int64_t>(H.v_col) * p.num_slots : H.v_col);
    const uint32_t kstride = static_cast<uint32_t>(p.head_major ? rk : p.cache_k_row_stride);      // (the host has checked the strides)
    const uint32_t vstride = static_cast<uint32_t>(p.head_major ? rv : p.cache_v_row_stride);
    const __half* sc = lw == 0 ? p.scale_v + (p.head_major ? static_cast<int64_t>(h) * p.num_slots : h)
                               : p.scale_k + (p.head_major ? static_cast<int64_t>(h) * p.num_slots : h);
    const int64_t sc_stride = p.head_major ? 1 : (lw == 0 ? p.scale_v_row_stride : p.scale_k_row_stride);
    // What is loaded ahead is looked at one tile later, not where it is requested: a comparison or a conversion right behind
    // the load waits for it (1100 of 3700 cycles per tile).
    auto fetch_slot = [&](int j) {
      const int key = kbeg + j * kTileKeys + lt;
      return lt < kTileKeys && j < ntiles && key < kend ? r2t[key] : -1;
    };
    auto keep_slot = [&](int j, int slot) {
      if (slot >= p.num_slots) {
        report_status(p.status_word, LSVD_ERR_BOUNDS);
        slot = -1;
      }
      if (lt < kTileKeys) s.slot[j & (kTileSlotRing - 1)][lt] = slot;
    };
    // A thread's pieces of a tile: 16-byte piece `piece` of rows row0, row0 + step, ... (threads beyond the last whole row: none).
    // The passes are loops on purpose, and K and V share them: unrolled, the roles' code does not fit the instruction cache.
    const int k_step = kLoadThreads / H.nk, v_step = kLoadThreads / H.nv;
    const int k_row = lt / H.nk < k_step ? lt / H.nk : kTileKeys, v_row = lt / H.nv < v_step ? lt / H.nv : kTileKeys;
    const int k_piece = lt % H.nk, v_piece = lt % H.nv;
    auto request = [&](int j) {
      const int32_t* slots = s.slot[j & (kTileSlotRing - 1)];
      uint8_t* dst = codes + (j & (code_stages - 1)) * code_bytes;
#pragma unroll 1
      for (int part = 0; part < 2; ++part) {
        const int step = part ? v_step : k_step, bytes = part ? rv : rk;
        const uint32_t stride = part ? vstride : kstride;
        const int8_t* src = (part ? vbase + v_piece * 16 : kbase + k_piece * 16);
        uint8_t* to = dst + lt * 16;
#pragma unroll 1
        for (int row = part ? v_row : k_row; row < kTileKeys; row += step, to += step * bytes) {
          const int slot = slots[row];
          copy16_or_zero(to, src + static_cast<uint64_t>(static_cast<uint32_t>(max(slot, 0))) * stride, slot >= 0);
        }
        dst += kTileKeys * rk;
      }
    };
    auto widen = [&](const uint8_t* src, uint8_t* dst) {
#pragma unroll 1
      for (int part = 0; part < 2; ++part) {
        const int step = part ? v_step : k_step, piece = part ? v_piece : k_piece, bytes = part ? rv : rk;
        const uint8_t* from = src + lt * 16;
        uint8_t* tile = dst + (piece >> 2) * kTileKeys * 128;
#pragma unroll 1
        for (int row = part ? v_row : k_row; row < kTileKeys; row += step, from += step * bytes)
          store_codes(tile, row, piece & 3, *reinterpret_cast<const uint4*>(from));
        src += kTileKeys * rk;
        dst += k_bytes;
      }
    };
    __half raw0 = __ushort_as_half(0), raw1 = raw0;
    int sl0 = -1, sl1 = -1;
    auto load_scales = [&](int j) {
      if (lw > 1 || j >= ntiles) return;
      sl0 = s.slot[j & (kTileSlotRing - 1)][lane];
      sl1 = s.slot[j & (kTileSlotRing - 1)][lane + 32];
      raw0 = sc[max(sl0, 0) * sc_stride];
      raw1 = sc[max(sl1, 0) * sc_stride];
    };
    {
      int first[kCodeStages];
#pragma unroll
      for (int j = 0; j < kCodeStages; ++j) first[j] = fetch_slot(j);
#pragma unroll
      for (int j = 0; j < kCodeStages; ++j) keep_slot(j, first[j]);
    }
    int slot_ahead = fetch_slot(kCodeStages);
    named_barrier(1, kLoadThreads);
    const int deep = code_stages - 1;               // tiles requested ahead of the one in hand
    for (int j = 0; j < max(deep, 1); ++j) {
      if (j < ntiles) request(j);
      copy_commit();
    }
    load_scales(0);
    // the K up-factor is in the stages' place until every row is absorbed
    bool ok = true;
    for (int i = 0; i < groups; ++i) ok = ok && tile_wait(s, &s.q_full[i], 0, p.status_word);
    ok = __all_sync(0xffffffffu, ok);
    for (int j = 0; j < ntiles; ++j) {
      const int st = j & (stages - 1);
      if (deep > 0) {
        copy_wait<kCodeStages - 2>();
      } else {
        copy_wait<0>();
      }
      // tile j's codes are here for every load warp, and all are done with the stage of tile j - 1.  Every load warp comes
      // here, whatever its waits returned, and all stop together.
      if (named_barrier_or(1, kLoadThreads, !ok)) break;
      keep_slot(j + kCodeStages, slot_ahead);
      slot_ahead = fetch_slot(j + kCodeStages + 1);
      if (deep > 0) {
        if (j + deep < ntiles) request(j + deep);
        copy_commit();
      }
      uint8_t* kd = stage0 + st * stage_bytes;
      const uint8_t* kc = codes + (j & (code_stages - 1)) * code_bytes;
      ok = __all_sync(0xffffffffu, tile_wait(s, &s.empty[st], ((j / stages) & 1) ^ 1, p.status_word));
      if (!ok) continue;
      // the scales go first: the softmax reads them once K is there
      const float sc0 = sl0 >= 0 ? __half2float(raw0) : 0.f, sc1 = sl1 >= 0 ? __half2float(raw1) : 0.f;
      if (lw == 0) {
        const float e0 = scale_exponent(sc0), e1 = scale_exponent(sc1);
        const int e_top = __reduce_max_sync(0xffffffffu, static_cast<int>(fmaxf(e0, e1)));
        s.sv[st][lane] = sc0;
        s.sv[st][lane + 32] = sc1;
        s.se[st][lane] = e0;
        s.se[st][lane + 32] = e1;
        const uint32_t m0 = __ballot_sync(0xffffffffu, sl0 >= 0), m1 = __ballot_sync(0xffffffffu, sl1 >= 0);
        if (lane == 0) {
          s.e_top[st] = static_cast<float>(e_top);
          s.live[st][0] = m0;
          s.live[st][1] = m1;
        }
      } else if (lw == 1) {
        s.sk[st][lane] = sc0;
        s.sk[st][lane + 32] = sc1;
      }
      load_scales(j + 1);
      widen(kc, kd);
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.full[st]);
      if (deep == 0) {                 // (what a thread copies it has widened itself)
        if (j + 1 < ntiles) request(j + 1);
        copy_commit();
      }
    }
    copy_wait<0>();
  } else if (warp < live_warps) {
    // ================= softmax: thread = row =================
    const int grp = warp >> 2;
    uint8_t* q_tile = smem + grp * q_bytes;
    const uint32_t lane_addr = tmem + grp * kGroupCols + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const int token = r.start + row0 + tid;
    const int pos = r.len - r.n + row0 + tid;
    float f = 0.f, R = -INFINITY, l = 0.f;
    bool go = true;
    if (ntiles > 0) {
      absorb_tile_rows(p, H, h, r, row0, rows, live_warps, s, q_tile, half_bytes, stage0);
      __syncwarp();
      f = s.scale[tid];
      f = fmaxf(f * p.score_scale * kChunkLog2e, 1e-37f);
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.q_full[grp]);
    }
    const float slope = kBias ? p.alibi_slopes[h] * kChunkLog2e : 0.f;
    // keys that every row of the warp sees
    const int inner_lo = __reduce_max_sync(0xffffffffu, tid < rows ? keys.lo : 0);
    const int inner_hi = __reduce_min_sync(0xffffffffu, tid < rows ? keys.hi : 0x7fffffff);
    const int outer_lo = __reduce_min_sync(0xffffffffu, keys.hi > keys.lo ? keys.lo : 0x7fffffff);
    const int outer_hi = __reduce_max_sync(0xffffffffu, keys.hi);

    for (int j0 = 0; go && j0 < ntiles; j0 += kFoldTiles) {
      const int jend = min(ntiles, j0 + kFoldTiles);
      if (j0 > 0) {
        // the sums so far go to the workspace, added to nearest, and O starts again from zero
        go = __all_sync(0xffffffffu, tile_wait(s, &s.o_done[grp], (j0 - 1) & 1, p.status_word));
        if (!go) break;
        tc_fence_after();
        const int64_t part = static_cast<int64_t>(split) * p.num_tokens + token;
        const bool again = j0 > kFoldTiles && tid < rows;
        const float by = again ? folded_factor(p.tile_ml[part * p.num_heads + h].x, R) : 0.f;
        float4* sums = reinterpret_cast<float4*>(p.tile_o + part * p.sum_rv + H.v_col);
        __syncwarp();
#pragma unroll 1
        for (int col = 0; col < rv; col += 16) {
          uint32_t v[16];
          tmem_ld16(lane_addr + kColO + col, v);
          if (tid < rows) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float4 y = again ? sums[(col >> 2) + i] : make_float4(0.f, 0.f, 0.f, 0.f);
              y.x = fmaf(y.x, by, __uint_as_float(v[4 * i]));
              y.y = fmaf(y.y, by, __uint_as_float(v[4 * i + 1]));
              y.z = fmaf(y.z, by, __uint_as_float(v[4 * i + 2]));
              y.w = fmaf(y.w, by, __uint_as_float(v[4 * i + 3]));
              sums[(col >> 2) + i] = y;
            }
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = 0u;
          tmem_st16(lane_addr + kColO + col, v);
        }
        if (tid < rows) p.tile_ml[part * p.num_heads + h].x = R;
      }
      for (int j = j0; go && j < jend; ++j) {
        const int st = j & (stages - 1), k0 = kbeg + j * kTileKeys;
        const uint32_t s_addr = lane_addr + (j & 1) * kTileKeys;
        go = tile_wait(s, &s.full[st], (j / stages) & 1, p.status_word) && tile_wait(s, &s.s_full[grp][j & 1], (j >> 1) & 1, p.status_word);
        if (!__all_sync(0xffffffffu, go)) {
          go = false;
          break;
        }
        tc_fence_after();
        const bool nothing = k0 >= outer_hi || k0 + kTileKeys <= outer_lo;      // of this warp's rows
        const uint32_t live0 = s.live[st][0], live1 = s.live[st][1];
        const bool masked = k0 < inner_lo || k0 + kTileKeys > inner_hi || (live0 & live1) != 0xffffffffu;
        float2 x[kTileKeys / 2];
        float top = -INFINITY;
        if (!nothing) {
          // (half by half: the scales of the second half are not fetched before the first half's scores are in)
          const float4* sk = reinterpret_cast<const float4*>(s.sk[st]);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t raw[32];
            __syncwarp();
            tmem_ld32(s_addr + 32 * half, raw);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 c = sk[8 * half + i];
              x[16 * half + 2 * i] = mul2(make_float2(__uint_as_float(raw[4 * i]), __uint_as_float(raw[4 * i + 1])), make_float2(c.x, c.y));
              x[16 * half + 2 * i + 1] = mul2(make_float2(__uint_as_float(raw[4 * i + 2]), __uint_as_float(raw[4 * i + 3])), make_float2(c.z, c.w));
            }
          }
          if (kCap || kBias) {
            const float2 ff = make_float2(f, f);
#pragma unroll
            for (int i = 0; i < kTileKeys / 2; ++i) x[i] = mul2(x[i], ff);
          }
          if (kCap) {
            const float2 cu = make_float2(p.cap_u, p.cap_u);
            float far = 0.f;
#pragma unroll
            for (int i = 0; i < kTileKeys / 2; ++i) far = max3(far, fabsf(x[i].x), fabsf(x[i].y));
            if (__any_sync(0xffffffffu, far * p.cap_u >= kCapSeries)) {
#pragma unroll
              for (int i = 0; i < kTileKeys / 2; ++i) x[i] = capped_log2(x[i], mul2(x[i], cu), p.cap_log2e);
            } else {
#pragma unroll
              for (int i = 0; i < kTileKeys / 2; ++i) x[i] = capped_series(x[i], mul2(x[i], cu));
            }
          }
          if (kBias) {
            const float away = static_cast<float>(pos - k0);
#pragma unroll
            for (int i = 0; i < kTileKeys / 2; ++i)
              x[i] = make_float2(fmaf(-slope, fabsf(away - static_cast<float>(2 * i)), x[i].x),
                                 fmaf(-slope, fabsf(away - static_cast<float>(2 * i + 1)), x[i].y));
          }
          if (masked) {
            const int a = min(max(keys.lo - k0, 0), 64), b = min(max(keys.hi - k0, 0), 64);
#pragma unroll
            for (int w = 0; w < 2; ++w) {            // bits of the keys that the row sees, 32 at a time
              const int from = min(max(a - 32 * w, 0), 32), upto = min(max(b - 32 * w, 0), 32);
              const uint32_t mask = (w == 0 ? live0 : live1) & (upto >= 32 ? ~0u : (1u << upto) - 1u) & (from >= 32 ? 0u : ~0u << from);
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                if (!((mask >> (2 * i)) & 1u)) x[16 * w + i].x = -INFINITY;
                if (!((mask >> (2 * i + 1)) & 1u)) x[16 * w + i].y = -INFINITY;
              }
            }
          }
          float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
          for (int i = 0; i < kTileKeys / 2; i += 2) {
            t0 = max3(t0, x[i].x, x[i].y);
            t1 = max3(t1, x[i + 1].x, x[i + 1].y);
          }
          top = fmaxf(t0, t1);
          if (!kCap && !kBias) top *= f;
        }
        // top + e_top bounds what a row sees here: only where that is past a row's reference are the rows' own values looked for
        if (__any_sync(0xffffffffu, R == -INFINITY ? top > -INFINITY : top + s.e_top[st] > R + kLazy)) {
          float need = -INFINITY;
          if (!nothing) {
            const float4* se = reinterpret_cast<const float4*>(s.se[st]);
            const float2 ff = make_float2(f, f);
#pragma unroll
            for (int i = 0; i < kTileKeys / 4; ++i) {
              const float4 e = se[i];
              const float2 a = (kCap || kBias) ? add2(x[2 * i], make_float2(e.x, e.y)) : fma2(x[2 * i], ff, make_float2(e.x, e.y));
              const float2 b = (kCap || kBias) ? add2(x[2 * i + 1], make_float2(e.z, e.w)) : fma2(x[2 * i + 1], ff, make_float2(e.z, e.w));
              need = max3(need, a.x, a.y);
              need = max3(need, b.x, b.y);
            }
          }
          const bool first = R == -INFINITY;
          const bool grown = first ? need > -INFINITY : need > R + kLazy;
          if (__any_sync(0xffffffffu, grown && !first)) {        // (so j > 0)
            const float by = grown && !first ? ex2(R - need) : 1.f;
            l *= by;
            go = tile_wait(s, &s.o_done[grp], (j - 1) & 1, p.status_word);
            if (!__all_sync(0xffffffffu, go)) {
              go = false;
              break;
            }
            tc_fence_after();
            __syncwarp();
#pragma unroll 1
            for (int col = 0; col < rv; col += 16) {
              uint32_t v[16];
              tmem_ld16(lane_addr + kColO + col, v);
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * by);
              tmem_st16(lane_addr + kColO + col, v);
            }
          }
          if (grown) R = need;
        }
        __syncwarp();
        if (nothing) {
          uint32_t z[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) z[i] = 0u;
#pragma unroll
          for (int i = 0; i < kTileKeys; i += 16) tmem_st16(s_addr + i, z);
        } else {
          // exponentials in place, one after another without a pause between them, then the weights
          const float base = R == -INFINITY ? 0.f : R - kWeightShift;
          const float2 nb = make_float2(-base, -base), ff = make_float2(f, f);
          float2 sum[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[i] = make_float2(0.f, 0.f);
#pragma unroll
          for (int i = 0; i < kTileKeys / 2; ++i) {
            const float2 y = (kCap || kBias) ? add2(x[i], nb) : fma2(x[i], ff, nb);
            x[i] = make_float2(ex2(y.x), ex2(y.y));
            sum[i & 3] = add2(sum[i & 3], x[i]);
          }
          const float4* sv = reinterpret_cast<const float4*>(s.sv[st]);
#pragma unroll
          for (int part = 0; part < 4; ++part) {         // (16-column stores cost spills)
            uint32_t w[8], rest[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 p0 = x[8 * part + 2 * i], p1 = x[8 * part + 2 * i + 1];
              const float4 c = sv[4 * part + i];
              float2 w0 = mul2(p0, make_float2(c.x, c.y)), w1 = mul2(p1, make_float2(c.z, c.w));
              if (masked) {             // a masked key's weight is zero whatever its scale holds
                if (p0.x == 0.f) w0.x = 0.f;
                if (p0.y == 0.f) w0.y = 0.f;
                if (p1.x == 0.f) w1.x = 0.f;
                if (p1.y == 0.f) w1.y = 0.f;
              }
              pack_weights(w0, w[2 * i], rest[2 * i]);
              pack_weights(w1, w[2 * i + 1], rest[2 * i + 1]);
            }
            __syncwarp();
            tmem_st8(s_addr + 8 * part, w);
            tmem_st8(s_addr + kTileKeys / 2 + 8 * part, rest);
          }
          sum[0] = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
          l += sum[0].x + sum[0].y;
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        // Phases are told apart by parity alone: before the last product is let go, the one in front of it is seen to have ended.
        if (j > 0 && j + 1 == jend) go = go && tile_wait(s, &s.o_done[grp], (j - 1) & 1, p.status_word);
        go = __all_sync(0xffffffffu, go);
        if (go && lane == 0) mbar_arrive(&s.p_full[grp][j & 1]);
      }
    }

    // ---- results -------------------------------------------------------------------------------------------------------
    // (all that is known here is that the product of tile ntiles - 3 is done: a phase is waited for by its parity, one by one)
    if (go && ntiles > 0) go = tile_wait(s, &s.o_done[grp], (ntiles - 1) & 1, p.status_word);
    go = __all_sync(0xffffffffu, go);
    tc_fence_after();
    if (go) {
      const float by = p.tile_splits > 1 ? 1.f : (l == 0.f ? 0.f : 1.f / l);
      const bool to_up = p.out != nullptr && p.tile_splits == 1;
      const int64_t part = static_cast<int64_t>(split) * p.num_tokens + token;
      const bool folded = ntiles > kFoldTiles && tid < rows;
      const float by_folded = folded ? folded_factor(p.tile_ml[part * p.num_heads + h].x, R) : 0.f;
      if (p.tile_splits > 1 && tid < rows) p.tile_ml[part * p.num_heads + h] = make_float2(R, l);
#pragma unroll 1
      for (int c = 0; c < rv; c += 16) {
        uint32_t v[16];
        float y[16];
        __syncwarp();
        if (ntiles > 0) tmem_ld16(lane_addr + kColO + c, v);
        if (folded) {
          const float4* sums = reinterpret_cast<const float4*>(p.tile_o + part * p.sum_rv + H.v_col + c);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 y = sums[i];
            v[4 * i] = __float_as_uint(fmaf(y.x, by_folded, __uint_as_float(v[4 * i])));
            v[4 * i + 1] = __float_as_uint(fmaf(y.y, by_folded, __uint_as_float(v[4 * i + 1])));
            v[4 * i + 2] = __float_as_uint(fmaf(y.z, by_folded, __uint_as_float(v[4 * i + 2])));
            v[4 * i + 3] = __float_as_uint(fmaf(y.w, by_folded, __uint_as_float(v[4 * i + 3])));
          }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = (ntiles > 0 && by != 0.f) ? __uint_as_float(v[i]) * by : 0.f;
        if (p.tile_splits > 1) {
          if (tid < rows && ntiles > 0) {
            float4* dst = reinterpret_cast<float4*>(p.tile_o + part * p.sum_rv + H.v_col + c);
#pragma unroll
            for (int i = 0; i < 4; ++i) dst[i] = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
          }
          continue;
        }
        __align__(16) __half2 hh[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) hh[i] = __floats2half2_rn(y[2 * i], y[2 * i + 1]);
        const uint4 lo = *reinterpret_cast<const uint4*>(&hh[0]), hi = *reinterpret_cast<const uint4*>(&hh[4]);
        if (p.out_latent != nullptr && tid < rows) {
          __half* dst = p.out_latent + token * p.out_latent_stride_t + H.v_col + c;
          store_halves8(dst, lo, p.out_lat_vec16);
          store_halves8(dst + 8, hi, p.out_lat_vec16);
        }
        if (to_up && ntiles > 0) {
          uint8_t* block = smem + grp * q_bytes + (c >> 6) * kGroupRows * 128;
          uint32_t most[8], rest[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) pack_half2_rest(y[2 * i], y[2 * i + 1], most[i], rest[i]);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint8_t* at = block + swizzled(tid & (kGroupRows - 1), ((c & 63) >> 3) + i);
            *reinterpret_cast<uint4*>(at) = make_uint4(most[4 * i], most[4 * i + 1], most[4 * i + 2], most[4 * i + 3]);
            *reinterpret_cast<uint4*>(at + half_bytes) = make_uint4(rest[4 * i], rest[4 * i + 1], rest[4 * i + 2], rest[4 * i + 3]);
          }
        }
      }
      if (to_up && ntiles == 0 && tid < rows)
        for (int d = 0; d < p.head_dim; ++d) p.out[token * p.out_stride_t + h * p.out_stride_h + d] = __float2half_rn(0.f);
    } else {
      s.abort = 1;
    }
  }

  // Every role is through with its stages here (one that gave up has set the abort flag).  Block barriers and
  // tensor memory instructions take whole warps.
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) {
    if (s.abort) {
      // products may be in flight: an arrival behind all of them, waited for (bounded), before their memory goes
      if (elect_one()) umma_commit(&s.last);
      __syncwarp();
      mbar_wait_bounded(&s.last, 0);
      __syncwarp();
    }
    tmem_dealloc(tmem, kTileCols);
  }
  // (what follows is worked out anew: held over the loops above, it would not fit the registers)
  if (s.kend <= s.kbeg || p.out == nullptr || p.tile_splits > 1 || s.abort) return;
  chunk_tile_up(p, s, smem);
}

cudaError_t launch_chunk_tile(const ChunkParams& p, int tiles, cudaStream_t st) {
  const bool cap = p.softcap > 0.f, bias = p.alibi_slopes != nullptr;
  void (*kern)(ChunkParams) = cap ? (bias ? chunk_tile_kernel<true, true> : chunk_tile_kernel<true, false>)
                                  : (bias ? chunk_tile_kernel<false, true> : chunk_tile_kernel<false, false>);
  const cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), kTileSmem);
  if (e != cudaSuccess) return e;
  return launch_chained(kern, dim3(p.num_heads, tiles, p.tile_splits), dim3(kTileThreads), kTileSmem, st, 1, true, p);
}

}  // namespace lsvd
