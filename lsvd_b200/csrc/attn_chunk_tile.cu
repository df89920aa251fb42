// Attention of new tokens over the paged int8 latent cache, tile form: 128 query rows of one request and head per block, on
// tcgen05.  (The mathematics and the stream form, for requests of few rows, are in attn_chunk.cu.)
//
// Per 64 keys a block does two products with the weights' softmax between them:
//   S[128 x 64] = q~[128 x r_k] . z_k^T     A and B from shared memory, accumulator in tensor memory (two buffers)
//   O[128 x r_v] += P[128 x 64] . z_v       A = P, fp16, written over S in tensor memory; B = the codes, ranks contiguous
// 16384 exponentials per 128 x 128 scores take 1024 cycles of an SM (16 a cycle) while the products take 512 at ranks of
// 64 + 64: the exponentials bound it, then the issue slots of the softmax (about six per score).  So the softmax warps must never
// wait.  Eight warps: four for the softmax (thread = row, no exchange between threads), three that gather the rows by slot,
// widen the int8 codes to fp16 (exact) and store them in the 128-byte-swizzled layouts that the products read, one that issues
// the products.  The score product of tile j + 2 runs while the softmax is at tile j + 1, and two blocks share an SM (256 tensor
// memory columns and at most 113 KB of shared memory each), so that one's waits are the other's cycles.
//
// The prologue computes q~ = B_k q with the same unit; the epilogue applies the V up-factor likewise (o_lat rounded to fp16,
// as in the latent result).  O is rescaled only when a row's maximum has grown by more than 2^8 since its last
// reference, or when a larger V scale arrives: weights are held as p * scale_v * 2^(6 - E) with p < 2^8 and 2^E the power of
// two below the largest V scale seen, so fp16 neither overflows (< 2^15) nor loses bits above 2^-20 of the reference.
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
constexpr int kHalves = 2;                       // threads that share a row: each takes half of a tile's keys
constexpr int kSoftmaxWarps = 4 * kGroups * kHalves, kLoadWarps = 3;
constexpr int kMmaWarp = kSoftmaxWarps + kLoadWarps;
constexpr int kTileThreads = (kMmaWarp + 1) * 32;
constexpr int kLoadThreads = kLoadWarps * 32;
constexpr int kTileSmem = 192 * 1024 + 1024;     // q~ (or o_lat), widened stages, copied codes; 1024 to align
constexpr int kTileMaxStages = 4;
constexpr int kCodeStages = 4;                   // stages of codes on their way
constexpr int kTileSlotRing = 8;
constexpr int kTileCols = 512;                   // tensor memory, 256 columns a group: S0 0..63, S1 64..127, O 128..255
constexpr int kGroupCols = 256;
constexpr int kColO = 128;
constexpr float kLazy = 8.f;                     // growth of a row's maximum (log2) that rescales O
constexpr int kTileShift = 6;

struct __align__(16) TileShared {
  float sk[kTileMaxStages][kTileKeys], sv[kTileMaxStages][kTileKeys];      // first: read in 16-byte pieces
  uint64_t k_full[kTileMaxStages], k_empty[kTileMaxStages], v_full[kTileMaxStages], v_empty[kTileMaxStages];
  uint64_t s_full[kGroups][2], p_full[kGroups][2], o_done[kGroups], q_full[kGroups], last;
  uint32_t live[kTileMaxStages][2];              // keys with a slot, one bit each
  int32_t E[kTileMaxStages];
  int32_t slot[kTileSlotRing][kTileKeys];
  uint32_t tmem;
  volatile uint32_t abort;
  int32_t b, tile;
  int32_t kbeg, kend;
  int32_t first, rows;                           // the block's first row, and how many
  float scale[kTileRows];                        // power of two taken out of each q~ row
  int32_t lo[kTileRows], hi[kTileRows];          // keys that each row sees
  float both[kHalves][kTileRows];                // what the two threads of a row tell one another
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
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Wait for a phase, bounded by kMbarTimeoutNs; also gives up once another role has.  False: stop and leave.  The thread is
// suspended for up to a millisecond a poll: a dozen warps that poll at full speed take the load warps' issue slots.
__device__ __forceinline__ bool tile_poll(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity), "r"(1000000u) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool tile_wait(TileShared& s, uint64_t* bar, uint32_t parity, int32_t* status_word) {
  if (tile_poll(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  for (uint32_t i = 0; i < kMbarMaxPolls; ++i) {
    if (tile_poll(bar, parity)) return true;
    if (s.abort || global_timer_ns() - t0 > kMbarTimeoutNs) break;
  }
  if (!s.abort) report_status(status_word, LSVD_ERR_TIMEOUT);
  s.abort = 1;
  return false;
}

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

// A tile's rows of N 16-byte pieces: thread lt of the load warps has piece lt % N of rows lt / N, + kStep, ...  N is a
// compile-time number (1 to 8) so that every offset is: with runtime steps the load warps spent 3000 instructions a tile.
template <int N>
struct TileRows {
  static constexpr int kStep = kLoadThreads / N < kTileKeys ? kLoadThreads / N : kTileKeys;
  static constexpr int kPasses = (kTileKeys + kStep - 1) / kStep;
};
template <int N>
__device__ __forceinline__ void copy_rows(int lt, const int32_t* slots, uint8_t* dst, const int8_t* src, uint32_t stride) {
  using R = TileRows<N>;
  const int row = lt / N, piece = lt % N;
  if (row >= R::kStep) return;
#pragma unroll
  for (int i = 0; i < R::kPasses; ++i)
    if (row + i * R::kStep < kTileKeys) {
      const int slot = slots[row + i * R::kStep];
      copy16_or_zero(dst + lt * 16 + i * (R::kStep * N * 16), src + static_cast<uint64_t>(static_cast<uint32_t>(max(slot, 0))) * stride + piece * 16,
                     slot >= 0);
    }
}
template <int N>
__device__ __forceinline__ void widen_rows(int lt, const uint8_t* src, uint8_t* tile) {
  using R = TileRows<N>;
  const int row = lt / N, piece = lt % N;
  if (row >= R::kStep) return;
  tile += (piece >> 2) * kTileKeys * 128;
#pragma unroll
  for (int i0 = 0; i0 < R::kPasses; i0 += 2) {
    uint4 w[2];
#pragma unroll
    for (int i = i0; i < i0 + 2 && i < R::kPasses; ++i)
      if (row + i * R::kStep < kTileKeys) w[i - i0] = *reinterpret_cast<const uint4*>(src + lt * 16 + i * (R::kStep * N * 16));
#pragma unroll
    for (int i = i0; i < i0 + 2 && i < R::kPasses; ++i)
      if (row + i * R::kStep < kTileKeys) store_codes(tile, row + i * R::kStep, piece & 3, w[i - i0]);
  }
}
__device__ __forceinline__ void copy_rows(int n, int lt, const int32_t* slots, uint8_t* dst, const int8_t* src, uint32_t stride) {
  asm volatile("" : "+r"(lt));        // nothing of the eight forms is to be worked out ahead of the loop and kept (spills)
  switch (n) {
    case 1: return copy_rows<1>(lt, slots, dst, src, stride);
    case 2: return copy_rows<2>(lt, slots, dst, src, stride);
    case 3: return copy_rows<3>(lt, slots, dst, src, stride);
    case 4: return copy_rows<4>(lt, slots, dst, src, stride);
    case 5: return copy_rows<5>(lt, slots, dst, src, stride);
    case 6: return copy_rows<6>(lt, slots, dst, src, stride);
    case 7: return copy_rows<7>(lt, slots, dst, src, stride);
    default: return copy_rows<8>(lt, slots, dst, src, stride);
  }
}
__device__ __forceinline__ void widen_rows(int n, int lt, const uint8_t* src, uint8_t* tile) {
  asm volatile("" : "+r"(lt));
  switch (n) {
    case 1: return widen_rows<1>(lt, src, tile);
    case 2: return widen_rows<2>(lt, src, tile);
    case 3: return widen_rows<3>(lt, src, tile);
    case 4: return widen_rows<4>(lt, src, tile);
    case 5: return widen_rows<5>(lt, src, tile);
    case 6: return widen_rows<6>(lt, src, tile);
    case 7: return widen_rows<7>(lt, src, tile);
    default: return widen_rows<8>(lt, src, tile);
  }
}

// q~ = B_k q of the warp's 16 rows (mma m16n8k16, like the stream form's), as fp16 rows of the A operand relative to each
// row's largest entry; the powers of two go to s.scale.  Ranks in blocks of 64: with two blocks the first is computed again
// once the row's largest entry over both is known (its accumulators do not fit beside the second's).
__device__ __forceinline__ void absorb_tile_rows(const ChunkParams& p, const ChunkHead& H, int h, const ChunkRequest& r, int row0, int rows,
                                                 TileShared& s, uint8_t* q_tile) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int rk = H.nk * 16, first = warp * 16;      // rows of the block; q_tile is the group's
  const __half* qa = p.q + static_cast<int64_t>(r.start + row0 + min(first + g, rows - 1)) * p.q_stride_t + h * p.q_stride_h;
  const __half* qb = p.q + static_cast<int64_t>(r.start + row0 + min(first + 8 + g, rows - 1)) * p.q_stride_t + h * p.q_stride_h;
  float acc[8][4], top[2] = {0.f, 0.f};
  const int blocks = rk > 64 ? 2 : 1;
#pragma unroll 1
  for (int pass = 0; pass < (blocks == 2 ? 3 : 1); ++pass) {      // block 0, block 1, block 0 again
    const int rank0 = pass == 1 ? 64 : 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll 1
    for (int d0 = 0; d0 < p.head_dim; d0 += 16) {
      const int d = d0 + 4 * t;
      const uint2 a0 = load_halves4(qa + d, p.head_dim - d, p.q_vec), a1 = load_halves4(qb + d, p.head_dim - d, p.q_vec);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint2 b = make_uint2(0u, 0u);
        const int rank = rank0 + 8 * j + g;
        if (rank < rk) b = load_halves4(p.up_k + static_cast<int64_t>(H.k_col + rank) * p.up_k_row_stride + d, p.head_dim - d, p.up_k_vec);
        mma_f16_16x8x16(acc[j], a0.x, a1.x, a0.y, a1.y, b.x, b.y);
      }
    }
    if (pass < 2) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int j = 0; j < 8; ++j) top[e] = fmaxf(top[e], fmaxf(fabsf(acc[j][2 * e]), fabsf(acc[j][2 * e + 1])));
        top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
        top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
      }
    }
    if (pass == 0 && blocks == 2) continue;
    uint8_t* block = q_tile + (rank0 >> 6) * kGroupRows * 128;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int ex = exponent_of(top[e]) - 8, row = first + 8 * e + g;      // entries end up below 2^9
      const float x = pow2i(-ex);
      if (t == 0) s.scale[row] = pow2i(ex);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (rank0 + 8 * j < rk)
          *reinterpret_cast<uint32_t*>(block + swizzled(row & (kGroupRows - 1), j) + 4 * t) = pack_half2(acc[j][2 * e] * x, acc[j][2 * e + 1] * x);
    }
  }
}

// o = B_v^T o_lat of the block's rows: the factor [r_v x head_dim] in the stages' place, o_lat (fp16, where q~ was) as A
// (mma m16n8k16).  For the whole block, after its tensor memory is gone.
__device__ __forceinline__ void chunk_tile_up(const ChunkParams& p, const TileShared& s, uint8_t* smem) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, h = blockIdx.x;
  const ChunkHead H = p.head[h];
  const int rv = H.nv * 16, q_bytes = ((max(H.nk, H.nv) + 3) >> 2) * kGroupRows * 128;
  const ChunkRequest r = chunk_request(p, s.b, false);
  const int row0 = s.tile * kTileRows, rows = min(kTileRows, r.n - row0);
  __half* up = reinterpret_cast<__half*>(smem + kGroups * q_bytes);
  for (int x = tid; x < rv * (p.head_dim >> 2); x += kTileThreads) {
    const int rank = x / (p.head_dim >> 2), d = (x - rank * (p.head_dim >> 2)) * 4;
    *reinterpret_cast<uint2*>(up + rank * p.head_dim + d) =
        load_halves4(p.up_v + static_cast<int64_t>(H.v_col + rank) * p.up_v_row_stride + d, 4, p.up_v_vec);
  }
  __syncthreads();
  if (warp * 16 >= rows) return;
  {
    const int ra = warp * 16 + g, rb = ra + 8, la = ra & (kGroupRows - 1), lb = la + 8;
#pragma unroll 1
    for (int d0 = 0; d0 < p.head_dim; d0 += 8) {
      float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
      for (int q = 0; q < H.nv; ++q) {
        const uint8_t* block = smem + (warp >> 3) * q_bytes + (q >> 2) * kGroupRows * 128;
        const int c = 2 * (q & 3);
        const uint16_t* at = reinterpret_cast<const uint16_t*>(up) + (16 * q + 2 * t) * p.head_dim + d0 + g;
        const uint32_t b0 = at[0] | (static_cast<uint32_t>(at[p.head_dim]) << 16);
        const uint32_t b1 = at[8 * p.head_dim] | (static_cast<uint32_t>(at[9 * p.head_dim]) << 16);
        mma_f16_16x8x16(y, *reinterpret_cast<const uint32_t*>(block + swizzled(la, c) + 4 * t),
                        *reinterpret_cast<const uint32_t*>(block + swizzled(lb, c) + 4 * t),
                        *reinterpret_cast<const uint32_t*>(block + swizzled(la, c + 1) + 4 * t),
                        *reinterpret_cast<const uint32_t*>(block + swizzled(lb, c + 1) + 4 * t), b0, b1);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = e == 0 ? ra : rb;
        if (row >= rows) continue;
        __half* dst = p.out + static_cast<int64_t>(r.start + row0 + row) * p.out_stride_t + h * p.out_stride_h + d0 + 2 * t;
        const uint32_t v = pack_half2(y[2 * e], y[2 * e + 1]);
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
  const int q_bytes = max(kblocks, vblocks) * kGroupRows * 128;              // of a group
  const int k_bytes = kblocks * kTileKeys * 128, stage_bytes = k_bytes + vblocks * kTileKeys * 128;
  const int code_bytes = kTileKeys * (rk + rv);
  const int stages = kGroups * q_bytes + 4 * stage_bytes + kCodeStages * code_bytes <= kTileSmem - 1024 ? 4 : 2;
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
        mbar_init(&s.k_full[i], kLoadWarps);
        mbar_init(&s.k_empty[i], 1);
        mbar_init(&s.v_full[i], kLoadWarps);
        mbar_init(&s.v_empty[i], 1);
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
  const int groups = (rows + kGroupRows - 1) / kGroupRows;
  // The row of each softmax thread, and the block's keys.  Warp w of a group has the tensor memory lanes 32 (w % 4) .., that is
  // the group's rows of that number, and the keys of half w / 4 of a tile.
  const int grp = warp >> 3, half = (warp >> 2) & 1, row = grp * kGroupRows + (warp & 3) * 32 + lane;
  const bool live = warp < kSoftmaxWarps && row - lane < rows;
  KeyRange keys;
  keys.lo = keys.hi = 0;
  if (live && row < rows) keys = visible_keys(p, r, p.b_prefix_len != nullptr ? p.b_prefix_len[s.b] : 0, row0 + row);
  if (warp < kSoftmaxWarps) {
    if (half == 0) {
      s.lo[row] = keys.lo;
      s.hi[row] = keys.hi;
    }
    const int lo = __reduce_min_sync(0xffffffffu, keys.hi > keys.lo ? keys.lo : 0x7fffffff);
    const int hi = __reduce_max_sync(0xffffffffu, keys.hi);
    if (lane == 0 && hi > 0) {
      atomicMin(&s.kbeg, lo);
      atomicMax(&s.kend, hi);
    }
  }
  if (tid == 0) {
    s.first = r.start + row0;
    s.rows = rows;
    for (int i = 0; i < groups; ++i) {
      const int mine = min(kGroupRows, rows - i * kGroupRows);
      mbar_init(&s.p_full[i][0], kHalves * ((mine + 31) / 32));
      mbar_init(&s.p_full[i][1], kHalves * ((mine + 31) / 32));
      mbar_init(&s.q_full[i], (mine + 15) / 16);
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
      if (!wait(&s.k_full[st], (j / stages) & 1)) return false;
#pragma unroll
      for (int grp = 0; grp < kGroups; ++grp) {
        if (grp >= groups) continue;
        if (j >= 2 && !wait(&s.o_done[grp], j & 1)) return false;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t qdesc = smem_desc_k_major_sw128(smem + grp * q_bytes), kdesc = smem_desc_k_major_sw128(stage0 + st * stage_bytes);
          for (int q = 0; q < H.nk; ++q)        // 16 ranks a step: 32 bytes of a row; a 64-rank block is a tile of its own
            umma_f16_ss(tmem + grp * kGroupCols + (j & 1) * kTileKeys, qdesc + ((q >> 2) * (kGroupRows * 128 >> 4) + (q & 3) * 2),
                        kdesc + ((q >> 2) * (kTileKeys * 128 >> 4) + (q & 3) * 2), idesc_s, q > 0 ? 1u : 0u);
          umma_commit(&s.s_full[grp][j & 1]);
          if (grp + 1 == groups) umma_commit(&s.k_empty[st]);
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
      go = wait(&s.v_full[st], (j / stages) & 1);
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
          for (int q = 0; q < kTileKeys / 16; ++q)    // 16 keys a step: two groups of eight rows; 8 columns of P
            umma_f16_ts(base + kColO, base + (j & 1) * kTileKeys + 8 * q, vdesc + q * (2048 >> 4), idesc_o, (j | q) != 0 ? 1u : 0u);
          umma_commit(&s.o_done[grp]);
          if (grp + 1 == groups) umma_commit(&s.v_empty[st]);
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
    auto request = [&](int j) {
      const int32_t* slots = s.slot[j & (kTileSlotRing - 1)];
      uint8_t* kd = codes + (j & (kCodeStages - 1)) * code_bytes;
      copy_rows(H.nk, lt, slots, kd, kbase, kstride);
      copy_rows(H.nv, lt, slots, kd + kTileKeys * rk, vbase, vstride);
    };
    __half raw0 = __ushort_as_half(0), raw1 = raw0;
    int sl0 = -1, sl1 = -1, E = -200;
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
    for (int j = 0; j < kCodeStages - 1; ++j) {
      if (j < ntiles) request(j);
      copy_commit();
    }
    load_scales(0);
    bool ok = true;
    for (int j = 0; j < ntiles; ++j) {
      const int st = j & (stages - 1);
      copy_wait<kCodeStages - 2>();
      // tile j's codes are here for every load warp, and all are done with the stage of tile j - 1.  Every load warp comes
      // here, whatever its waits returned, and all stop together.
      if (named_barrier_or(1, kLoadThreads, !ok)) break;
      keep_slot(j + kCodeStages, slot_ahead);
      slot_ahead = fetch_slot(j + kCodeStages + 1);
      if (j + kCodeStages - 1 < ntiles) request(j + kCodeStages - 1);
      copy_commit();
      uint8_t* kd = stage0 + st * stage_bytes;
      const uint8_t* kc = codes + (j & (kCodeStages - 1)) * code_bytes;
      ok = tile_wait(s, &s.k_empty[st], ((j / stages) & 1) ^ 1, p.status_word);
      ok = ok && tile_wait(s, &s.v_empty[st], ((j / stages) & 1) ^ 1, p.status_word);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) continue;
      // the scales go first: the softmax reads them once K is there
      const float sc0 = sl0 >= 0 ? __half2float(raw0) : 0.f, sc1 = sl1 >= 0 ? __half2float(raw1) : 0.f;
      if (lw == 0) {
        const float a0 = fabsf(sc0), a1 = fabsf(sc1);
        int e = -200;
        if (a0 > 0.f && a0 < INFINITY) e = exponent_of(a0);
        if (a1 > 0.f && a1 < INFINITY) e = max(e, exponent_of(a1));
        E = max(E, __reduce_max_sync(0xffffffffu, e));
        const float x = pow2i(kTileShift - E);
        s.sv[st][lane] = sc0 * x;
        s.sv[st][lane + 32] = sc1 * x;
        const uint32_t m0 = __ballot_sync(0xffffffffu, sl0 >= 0), m1 = __ballot_sync(0xffffffffu, sl1 >= 0);
        if (lane == 0) {
          s.E[st] = E;
          s.live[st][0] = m0;
          s.live[st][1] = m1;
        }
      } else if (lw == 1) {
        s.sk[st][lane] = sc0;
        s.sk[st][lane + 32] = sc1;
      }
      load_scales(j + 1);
      widen_rows(H.nk, lt, kc, kd);
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.k_full[st]);
      widen_rows(H.nv, lt, kc + kTileKeys * rk, kd + k_bytes);
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.v_full[st]);
    }
    copy_wait<0>();
  } else if (warp < kSoftmaxWarps) {
    // ================= softmax: two threads a row =================
    if (ntiles > 0 && warp * 16 < rows) {
      absorb_tile_rows(p, H, h, r, row0, rows, s, smem + grp * q_bytes);
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.q_full[grp]);
    }
    const uint32_t lane_addr = tmem + grp * kGroupCols + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const int pos = kBias ? r.len - r.n + row0 + row : 0, partner = 2 + grp * 4 + (warp & 3);      // named barrier of the rows' two warps
    float f = 0.f, m = -INFINITY, l = 0.f;
    int E = -200;
    bool go = live;
    if (go && ntiles > 0) {
      go = __all_sync(0xffffffffu, tile_wait(s, &s.q_full[grp], 0, p.status_word));
      f = fmaxf(s.scale[row] * p.score_scale * (kCap ? 2.f * kChunkLog2e / p.softcap : kChunkLog2e), 1e-37f);
    }
    const float cap_log2e = p.softcap * kChunkLog2e;
    const float slope = kBias ? p.alibi_slopes[h] * kChunkLog2e : 0.f;
    // A wait that gave up: both warps of the rows learn of it at their next common barrier (or have no further one).
    for (int j = 0; live && j < ntiles; ++j) {
      const int st = j & (stages - 1), k0 = kbeg + j * kTileKeys;
      const uint32_t s_addr = lane_addr + (j & 1) * kTileKeys;
      go = go && tile_wait(s, &s.k_full[st], (j / stages) & 1, p.status_word) && tile_wait(s, &s.s_full[grp][j & 1], (j >> 1) & 1, p.status_word);
      go = __all_sync(0xffffffffu, go);
      tc_fence_after();
      const int e_new = s.E[st];
      const int lo = s.lo[row], hi = s.hi[row];
      const bool nothing = __all_sync(0xffffffffu, hi <= k0 || lo >= k0 + kTileKeys);      // (both warps of the rows find the same)
      const int kh = k0 + 32 * half;                                          // this thread's first key
      uint32_t mask = s.live[st][half];                                       // keys that the row sees
      {
        const int a = min(max(lo - kh, 0), 32), b = min(max(hi - kh, 0), 32);
        mask &= (b >= 32 ? ~0u : (1u << b) - 1u) & (a >= 32 ? 0u : ~0u << a);
      }
      const bool masked = __any_sync(0xffffffffu, mask != ~0u && row < s.rows);
      // O (this thread's columns) and the sum for a new reference (factor c) or a larger V scale; the product of tile j - 1 is
      // waited for
      auto rescale = [&](float c, int e) {
        l *= c;
        if (j == 0) return;
        go = go && tile_wait(s, &s.o_done[grp], (j - 1) & 1, p.status_word);
        go = __all_sync(0xffffffffu, go);
        if (!go) return;
        tc_fence_after();
        const float by = c * pow2i(max(E - e, -126));
        __syncwarp();
#pragma unroll 1
        for (int col = 16 * half; col < rv; col += 32) {
          uint32_t v[16];
          tmem_ld16(lane_addr + kColO + col, v);
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * by);
          tmem_st16(lane_addr + kColO + col, v);
        }
        tmem_wait_st();              // it may be read again in this tile
      };
      if (e_new != E) {
        rescale(1.f, e_new);
        E = e_new;
      }
      uint32_t w[2][8];
      float2 sum = make_float2(0.f, 0.f);
      if (nothing) {
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i >> 3][i & 7] = 0u;
      } else {
        const float4* sk = reinterpret_cast<const float4*>(s.sk[st] + 32 * half);
        const float4* sv = reinterpret_cast<const float4*>(s.sv[st] + 32 * half);
        const float away = static_cast<float>(pos - kh);
        // One pass: the weights against the row's reference so far, and how far the scores rise above it.  Where some row's rise
        // is more than 2^8 (the first tile, hardly any after it) the reference moves and the tile is worked through again.
#pragma unroll 1
        for (int pass = 0;; ++pass) {
          asm volatile("" : "+r"(mask));       // its tests are not to be kept across the passes (spills)
          const float base = m == -INFINITY ? 0.f : m;
          const float2 nb = make_float2(-base, -base), ff = make_float2(f, f);
          float t0 = -INFINITY, t1 = -INFINITY;
          sum = make_float2(0.f, 0.f);
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            uint32_t raw[16];
            __syncwarp();
            tmem_ld16(s_addr + 32 * half + 16 * part, raw);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float4 ck = sk[4 * part + i], cv = sv[4 * part + i];
              float2 y[2] = {mul2(make_float2(__uint_as_float(raw[4 * i]), __uint_as_float(raw[4 * i + 1])), make_float2(ck.x, ck.y)),
                             mul2(make_float2(__uint_as_float(raw[4 * i + 2]), __uint_as_float(raw[4 * i + 3])), make_float2(ck.z, ck.w))};
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int key = 16 * part + 4 * i + 2 * e;
                if (kCap || kBias) {
                  float u = y[e].x * f, v = y[e].y * f;
                  if (kCap) {
                    u = capped_log2(u, cap_log2e);
                    v = capped_log2(v, cap_log2e);
                  }
                  if (kBias) {
                    u = fmaf(-slope, fabsf(away - static_cast<float>(key)), u);
                    v = fmaf(-slope, fabsf(away - static_cast<float>(key + 1)), v);
                  }
                  y[e] = add2(make_float2(u, v), nb);
                } else {
                  y[e] = fma2(y[e], ff, nb);
                }
                if (masked) {
                  if (!((mask >> key) & 1u)) y[e].x = -INFINITY;
                  if (!((mask >> (key + 1)) & 1u)) y[e].y = -INFINITY;
                }
              }
              t0 = max3(t0, y[0].x, y[0].y);
              t1 = max3(t1, y[1].x, y[1].y);
              const float2 p0 = make_float2(ex2(y[0].x), ex2(y[0].y)), p1 = make_float2(ex2(y[1].x), ex2(y[1].y));
              sum = add2(sum, add2(p0, p1));
              float2 w0 = mul2(p0, make_float2(cv.x, cv.y)), w1 = mul2(p1, make_float2(cv.z, cv.w));
              if (masked) {             // a masked key's weight is zero whatever its scale holds
                if (p0.x == 0.f) w0.x = 0.f;
                if (p0.y == 0.f) w0.y = 0.f;
                if (p1.x == 0.f) w1.x = 0.f;
                if (p1.y == 0.f) w1.y = 0.f;
              }
              w[part][2 * i] = pack_half2(w0.x, w0.y);
              w[part][2 * i + 1] = pack_half2(w1.x, w1.y);
            }
          }
          float rise = fmaxf(t0, t1);
          const bool first = m == -INFINITY;
          // The barrier also lets no weight be stored over scores that the other warp has not read.
          const bool again = named_barrier_or(partner, 64, pass == 0 && (first ? rise > -INFINITY : rise > kLazy));
          if (!again) break;
          s.both[half][row] = rise;
          named_barrier(partner, 64);
          rise = fmaxf(rise, s.both[half ^ 1][row]);
          named_barrier(partner, 64);
          const bool moves = first ? rise > -INFINITY : rise > kLazy;
          // (a first reference finds O and the sum at zero: times 1 keeps a NaN of a row that has one)
          rescale(moves && !first ? ex2(-rise) : 1.f, E);
          if (moves) m = base + rise;
        }
      }
      l += sum.x + sum.y;
      __syncwarp();
      if (go) {
#pragma unroll
        for (int part = 0; part < 2; ++part) tmem_st8(s_addr + 16 * half + 8 * part, w[part]);
      }
      tmem_wait_st();
      tc_fence_before();
      // Phases are told apart by parity alone: before the last product is let go, the one in front of it is seen to have ended.
      if (j > 0 && j + 1 == ntiles) go = go && tile_wait(s, &s.o_done[grp], (j - 1) & 1, p.status_word);
      go = __all_sync(0xffffffffu, go);
      if (go && lane == 0) mbar_arrive(&s.p_full[grp][j & 1]);
    }

    // ---- results -------------------------------------------------------------------------------------------------------
    if (go && ntiles > 0) go = tile_wait(s, &s.o_done[grp], (ntiles - 1) & 1, p.status_word);
    go = __all_sync(0xffffffffu, go);
    tc_fence_after();
    if (live) {
      s.both[half][row] = l;
      named_barrier(partner, 64);
      l += s.both[half ^ 1][row];
    }
    if (go) {
      const int token = s.first + row;
      const float back = ntiles > 0 ? (E > -200 ? pow2i(E - kTileShift) : 1.f) : 0.f;
      const float by = p.tile_splits > 1 ? back : (l == 0.f ? 0.f : back / l);
      const bool to_up = p.out != nullptr && p.tile_splits == 1;
      const int64_t part = static_cast<int64_t>(split) * p.num_tokens + token;
      if (p.tile_splits > 1 && row < s.rows && half == 0) p.tile_ml[part * p.num_heads + h] = make_float2(m, l);
#pragma unroll 1
      for (int c = 16 * half; c < rv; c += 32) {
        uint32_t v[16];
        float y[16];
        __syncwarp();
        if (ntiles > 0) tmem_ld16(lane_addr + kColO + c, v);
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = (ntiles > 0 && by != 0.f) ? __uint_as_float(v[i]) * by : 0.f;
        if (p.tile_splits > 1) {
          if (row < s.rows && ntiles > 0) {
            float4* dst = reinterpret_cast<float4*>(p.tile_o + part * p.sum_rv + H.v_col + c);
#pragma unroll
            for (int i = 0; i < 4; ++i) dst[i] = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
          }
          continue;
        }
        const uint4 lo = make_uint4(pack_half2(y[0], y[1]), pack_half2(y[2], y[3]), pack_half2(y[4], y[5]), pack_half2(y[6], y[7]));
        const uint4 hi = make_uint4(pack_half2(y[8], y[9]), pack_half2(y[10], y[11]), pack_half2(y[12], y[13]), pack_half2(y[14], y[15]));
        if (p.out_latent != nullptr && row < s.rows) {
          __half* dst = p.out_latent + token * p.out_latent_stride_t + H.v_col + c;
          store_halves8(dst, lo, p.out_lat_vec16);
          store_halves8(dst + 8, hi, p.out_lat_vec16);
        }
        if (to_up && ntiles > 0) {
          uint8_t* block = smem + grp * q_bytes + (c >> 6) * kGroupRows * 128;
          const int piece = (c & 63) >> 3;
          *reinterpret_cast<uint4*>(block + swizzled(row & (kGroupRows - 1), piece)) = lo;
          *reinterpret_cast<uint4*>(block + swizzled(row & (kGroupRows - 1), piece + 1)) = hi;
        }
      }
      if (to_up && ntiles == 0 && half == 0 && row < s.rows)
        for (int d = 0; d < p.head_dim; ++d) p.out[token * p.out_stride_t + h * p.out_stride_h + d] = __float2half_rn(0.f);
    } else if (live) {
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
