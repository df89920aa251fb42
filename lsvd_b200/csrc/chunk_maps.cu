// Slots of the tokens that a step adds: pages taken from a free list, token maps, the requests' slot tables.
//
// Per batch entry b (row r, `ready` cached tokens, n new ones, pages of P slots) three exclusive sums over the batch give
// everything else: start[b] = sum n, page[b] = head + sum need with need = ceil((ready + n) / P) - ceil(ready / P), and, for
// a rebuild, the running sum of `ready`.  Token i of entry b then has position ready + i and the slot
// table[r][pos / P] * P + pos % P, where a page beyond ceil(ready / P) is free_pages[page[b] + ...].
//
// The work is 16 bytes per token (two maps, one table entry written, one page number read): less than a microsecond of
// memory traffic even for a 64 K-token step, so launches and dependent round trips are what counts.  Hence ONE launch: every
// block of a cluster computes the batch's sums for itself in shared memory (a few loads per entry), and the blocks share out
// the tokens, one thread per token with a binary search over start[].  The cluster barrier between "everyone has read the
// lengths and the free list's head" and "block 0 writes them" is what allows both to be updated in place.
#include "common.cuh"

namespace lsvd {

constexpr int kMapsThreads = 1024;
constexpr int kMapsPer = LSVD_MAX_BATCH / kMapsThreads;     // entries per thread in the batch's sums
constexpr int kMapsCluster = 8;
constexpr int kHashEmpty = -1;

// Exclusive sums over the block of kMapsPer values per thread (thread t owns entries t * kMapsPer ..); total in `total`.
__device__ __forceinline__ void block_exscan(int64_t (&v)[kMapsPer], int64_t* warp_sums, int64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t mine = 0;
#pragma unroll
  for (int i = 0; i < kMapsPer; ++i) {
    const int64_t x = v[i];
    v[i] = mine;
    mine += x;
  }
  int64_t inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    int64_t w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += up;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  total = warp_sums[31];
  const int64_t before = inc - mine + (warp > 0 ? warp_sums[warp - 1] : 0);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMapsPer; ++i) v[i] += before;
}

// Largest b with first[b] <= x, for a non-decreasing first[0 .. n) with first[0] <= x.
template <typename T>
__device__ __forceinline__ int owner_of(const T* first, int n, T x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ int pages_of(int tokens, int page) {
  return static_cast<int>((static_cast<uint32_t>(tokens) + static_cast<uint32_t>(page) - 1u) / static_cast<uint32_t>(page));
}

// Shared memory, in 4-byte words per entry: start, fresh, ready, row, new (refused: -1), the hash (2 x 2), ready sums (2).
struct MapsShared {
  int32_t* start;      // [B]      first token row
  int32_t* fresh;      // [B]      index into free_pages of the entry's first new page
  int32_t* nscan;      // [B]      sum of new pages before the entry
  int32_t* ready;      // [B]
  int32_t* row;        // [B]      -1: refused
  int32_t* count;      // [B]      new tokens that it gets
  int32_t* key;        // [hash]   request row
  int32_t* first;      // [hash]   smallest entry that adds tokens to it
  int64_t* old;        // [B]      sum of ready before the entry
  int hash_mask;
};

__global__ void __launch_bounds__(kMapsThreads) chunk_maps_kernel(const __grid_constant__ lsvd_chunk_maps_args p, int hash_size) {
  extern __shared__ __align__(16) uint8_t maps_smem[];
  __shared__ int64_t warp_sums[32];
  __shared__ int32_t taken_end;
  grid_dependency_release();
  grid_dependency_wait();
  const int B = p.batch, P = p.page_size;
  uint32_t cta, ctas;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(cta));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  MapsShared s;
  s.old = reinterpret_cast<int64_t*>(maps_smem);
  s.start = reinterpret_cast<int32_t*>(s.old + B);
  s.fresh = s.start + B;
  s.nscan = s.fresh + B;
  s.ready = s.nscan + B;
  s.row = s.ready + B;
  s.count = s.row + B;
  s.key = s.count + B;
  s.first = s.key + hash_size;
  s.hash_mask = hash_size - 1;
  const bool paged = p.free_head != nullptr;       // (a free list of no entries has no address)
  const int32_t head = paged ? *p.free_head : 0;
  const bool head_ok = head >= 0 && head <= p.num_free;
  if (threadIdx.x == 0) taken_end = head;
  for (int i = threadIdx.x; i < hash_size; i += kMapsThreads) {
    s.key[i] = kHashEmpty;
    s.first[i] = 0x7fffffff;
  }

  // lengths, and whether an entry fits the tables
  int32_t row[kMapsPer], ready[kMapsPer], add[kMapsPer];
  bool ok[kMapsPer];
  int64_t v[kMapsPer], total_new, total;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kMapsPer; ++i) {
    const int b = threadIdx.x * kMapsPer + i;
    row[i] = -1;
    ready[i] = add[i] = 0;
    ok[i] = false;
    v[i] = 0;
    if (b < B) {
      row[i] = p.b_req_idx[b];
      ready[i] = p.b_ready_cache_len[b];
      add[i] = p.b_new_len[b];
      const int64_t seq = static_cast<int64_t>(ready[i]) + add[i];
      ok[i] = row[i] >= 0 && row[i] < p.table_rows && ready[i] >= 0 && add[i] >= 0 && seq <= p.max_len &&
              seq <= static_cast<int64_t>(p.max_blocks) * P && (p.max_new_in_batch == 0 || add[i] <= p.max_new_in_batch);
      v[i] = add[i] > 0 ? add[i] : 0;
    }
  }
  block_exscan(v, warp_sums, total_new);
#pragma unroll
  for (int i = 0; i < kMapsPer; ++i) {
    const int b = threadIdx.x * kMapsPer + i;
    if (b >= B) continue;
    if (v[i] + (add[i] > 0 ? add[i] : 0) > p.num_tokens) ok[i] = false;
    s.start[b] = static_cast<int32_t>(min(v[i], static_cast<int64_t>(p.num_tokens)));
    // the first entry that adds tokens to a row keeps it: an open-addressing table of at least twice the batch
    if (ok[i] && add[i] > 0) {
      uint32_t at = (static_cast<uint32_t>(row[i]) * 2654435761u) >> 7;
      for (int probe = 0; probe < hash_size; ++probe, ++at) {
        const int32_t seen = atomicCAS(&s.key[at & s.hash_mask], kHashEmpty, row[i]);
        if (seen == kHashEmpty || seen == row[i]) {
          atomicMin(&s.first[at & s.hash_mask], b);
          break;
        }
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMapsPer; ++i) {
    const int b = threadIdx.x * kMapsPer + i;
    v[i] = 0;
    if (b >= B) continue;
    if (ok[i] && add[i] > 0) {
      uint32_t at = (static_cast<uint32_t>(row[i]) * 2654435761u) >> 7;
      while (s.key[at & s.hash_mask] != row[i]) ++at;      // it was entered above
      if (s.first[at & s.hash_mask] != b) ok[i] = false;
      if (ok[i] && paged) v[i] = pages_of(ready[i] + add[i], P) - pages_of(ready[i], P);
    } else if (ok[i] && paged && p.rebuild) {
      // its slots are rewritten from columns of the table: none of them may be one that another entry's pages go to
      uint32_t at = (static_cast<uint32_t>(row[i]) * 2654435761u) >> 7;
      while (s.key[at & s.hash_mask] != row[i] && s.key[at & s.hash_mask] != kHashEmpty) ++at;      // (half the table is empty)
      if (s.key[at & s.hash_mask] == row[i] && ready[i] > p.b_ready_cache_len[s.first[at & s.hash_mask]]) ok[i] = false;
    }
  }
  int32_t need[kMapsPer];
#pragma unroll
  for (int i = 0; i < kMapsPer; ++i) need[i] = static_cast<int32_t>(v[i]);
  block_exscan(v, warp_sums, total);
#pragma unroll
  for (int i = 0; i < kMapsPer; ++i) {
    const int b = threadIdx.x * kMapsPer + i;
    if (b >= B) continue;
    const int64_t first = head + v[i];
    if (need[i] > 0) {
      // the free pages run out: the sums only grow, so this and every later entry that needs a page is refused
      if (!head_ok || first + need[i] > p.num_free) ok[i] = false;
      else atomicMax(&taken_end, static_cast<int32_t>(first + need[i]));
    }
    if (!ok[i]) bad = true;
    s.fresh[b] = static_cast<int32_t>(min(first, static_cast<int64_t>(0x7fffffff)));
    s.nscan[b] = static_cast<int32_t>(min(v[i], static_cast<int64_t>(p.num_free)));
    s.ready[b] = ready[i];
    s.row[b] = ok[i] ? row[i] : -1;
    s.count[b] = ok[i] ? add[i] : 0;
    v[i] = 0;
  }
  if (p.rebuild) {
#pragma unroll
    for (int i = 0; i < kMapsPer; ++i) v[i] = ok[i] ? ready[i] : 0;
    block_exscan(v, warp_sums, total);
#pragma unroll
    for (int i = 0; i < kMapsPer; ++i) {
      const int b = threadIdx.x * kMapsPer + i;
      if (b < B) s.old[b] = v[i];
    }
  }
  __syncthreads();
  // every block of the cluster has read the lengths and the head: block 0 may write them
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (cta == 0) {
#pragma unroll
    for (int i = 0; i < kMapsPer; ++i) {
      const int b = threadIdx.x * kMapsPer + i;
      if (b >= B) continue;
      p.b_start_loc[b] = s.start[b];
      p.b_seq_len[b] = ok[i] ? ready[i] + add[i] : max(ready[i], 0);
    }
    if (threadIdx.x == 0) {
      p.b_start_loc[B] = static_cast<int32_t>(min(total_new, static_cast<int64_t>(p.num_tokens)));
      if (paged) *p.free_head_out = taken_end;
    }
    if (bad) report_status(p.status_word, LSVD_ERR_BOUNDS);
  }

  // Slot of position `pos` of entry b: an old page stands in the block table (only columns in front of the new pages are
  // read there, which no block writes), a new one in the free list.
  bool outside = false;
  auto page_of = [&](int b, int block, int have) {
    return block >= have ? p.free_pages[s.fresh[b] + block - have]
                         : p.block_table[static_cast<int64_t>(s.row[b]) * p.block_table_stride + block];
  };
  auto slot_of = [&](int b, int pos) {
    const int block = pos / P;
    const int have = paged ? pages_of(s.ready[b], P) : 0x7fffffff;
    const int page = page_of(b, block, have);
    if (page < 0 || (static_cast<int64_t>(page) + 1) * P > p.num_slots) {
      outside = true;
      return -1;
    }
    return page * P + (pos - block * P);
  };
  const int step = static_cast<int>(ctas) * kMapsThreads, tid = static_cast<int>(cta) * kMapsThreads + threadIdx.x;
  const int used = static_cast<int>(min(total_new, static_cast<int64_t>(p.num_tokens)));
  for (int64_t t64 = tid; t64 < p.num_tokens; t64 += step) {
    const int t = static_cast<int>(t64);
    int slot = -1, pos = 0;
    if (t < used) {
      // entries without new tokens share their start with the next one: the last of them owns the token
      const int b = owner_of(s.start, B, t), i = t - s.start[b];
      if (i < s.count[b]) {
        pos = s.ready[b] + i;
        slot = slot_of(b, pos);
        p.req_to_token[static_cast<int64_t>(s.row[b]) * p.req_to_token_stride + pos] = slot;
      }
    }
    p.mem_index[t] = slot;
    p.position_ids[t] = pos;
  }
  if (paged) {                                   // the new pages' columns of the block table
    const int pages = taken_end - head;          // (a refused entry's pages lie behind taken_end)
    for (int64_t j = tid; j < pages; j += step) {
      const int b = owner_of(s.nscan, B, static_cast<int32_t>(j));
      const int column = pages_of(s.ready[b], P) + static_cast<int>(j) - s.nscan[b];
      if (s.row[b] >= 0) p.block_table[static_cast<int64_t>(s.row[b]) * p.block_table_stride + column] = p.free_pages[head + j];
    }
  }
  if (p.rebuild) {
    for (int64_t j = tid; j < total; j += step) {
      const int b = owner_of(s.old, B, j);
      const int pos = static_cast<int>(j - s.old[b]);
      if (s.row[b] >= 0 && pos < s.ready[b])
        p.req_to_token[static_cast<int64_t>(s.row[b]) * p.req_to_token_stride + pos] = slot_of(b, pos);
    }
  }
  if (outside) report_status(p.status_word, LSVD_ERR_BOUNDS);
}

}  // namespace lsvd

extern "C" int lsvd_chunk_maps(const lsvd_chunk_maps_args* a, void* stream) {
  using namespace lsvd;
  if (a == nullptr || a->batch <= 0 || a->page_size <= 0 || a->num_tokens < 0 || a->num_slots <= 0 || a->max_new_in_batch < 0) return LSVD_ERR_INVALID_ARG;
  if (a->max_blocks <= 0 || a->table_rows <= 0 || a->max_len <= 0) return LSVD_ERR_INVALID_ARG;
  if (!a->b_req_idx || !a->b_ready_cache_len || !a->b_new_len || !a->block_table || !a->req_to_token || !a->b_start_loc ||
      !a->b_seq_len || (a->num_tokens > 0 && (!a->mem_index || !a->position_ids)))
    return LSVD_ERR_INVALID_ARG;
  if (a->free_pages != nullptr && !a->free_head) return LSVD_ERR_INVALID_ARG;
  if (a->free_head != nullptr && (!a->free_head_out || a->num_free < 0 || (a->num_free > 0 && !a->free_pages))) return LSVD_ERR_INVALID_ARG;
  if (a->table_rows > 1 && (a->block_table_stride < a->max_blocks || a->req_to_token_stride < a->max_len)) return LSVD_ERR_INVALID_ARG;
  const void* words[] = {a->b_req_idx, a->b_ready_cache_len, a->b_new_len, a->block_table, a->req_to_token, a->free_pages,
                         a->free_head, a->free_head_out, a->b_start_loc, a->b_seq_len, a->mem_index, a->position_ids};
  for (const void* w : words)
    if (!aligned(w, 4)) return LSVD_ERR_INVALID_ARG;
  if (a->batch > LSVD_MAX_BATCH) return LSVD_ERR_UNSUPPORTED;
  int hash = 64;
  while (hash < 2 * a->batch) hash *= 2;
  const size_t smem = static_cast<size_t>(a->batch) * (6 * 4 + 8) + static_cast<size_t>(hash) * 8;
  LSVD_CUDA_TRY(ensure_dynamic_smem(reinterpret_cast<const void*>(chunk_maps_kernel), static_cast<int>(smem)));
  // (one block and eight, replayed: 64 tokens 8.2 and 8.2 us, 2400 tokens 10.2 and 10.2, 98304 tokens 100 and 21)
  const int ctas = a->num_tokens > 2 * kMapsThreads || a->rebuild ? kMapsCluster : 1;
  LSVD_CUDA_TRY(launch_chained(chunk_maps_kernel, dim3(ctas), dim3(kMapsThreads), smem, static_cast<cudaStream_t>(stream), ctas, true,
                               *a, hash));
  return LSVD_OK;
}
