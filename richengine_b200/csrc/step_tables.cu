// step_tables.cu — what a step's kernels read, built on the GPU from request lengths: page-table entries from page ids,
// the lanes' store and attention parameter blocks, the slots of the step's new rows; and which lanes share how long a
// prefix, found from the tables.
//
// The host path these stand beside writes entries page by page (kv::PageStorage::writeEntries, rk_storage_write_entries)
// and uploads the parameter blocks each step. Neither kernel lets a dependent launch start early: the attention kernels
// read the parameter blocks before they wait for their predecessor.
#include "common.cuh"

namespace rk {
namespace {

constexpr uint32_t kMaxLanes = 1024;
constexpr uint32_t kTableThreads = 256;
constexpr uint32_t kGroupThreads = 256;

struct StepArgs {
  const uint32_t *page_ids, *page_offsets, *committed, *rows, *known_pages;
  rk_step_layout layout;
  rk_step_outputs out;
};

__device__ __forceinline__ uint32_t block_sum(uint32_t value, uint32_t *scratch) {
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) value += __shfl_xor_sync(0xffffffffu, value, o);
  if (lane == 0) scratch[warp] = value;
  __syncthreads();
  uint32_t total = 0;
  for (uint32_t w = 0; w < blockDim.x / 32; ++w) total += scratch[w];
  __syncthreads();
  return total;
}

// One block per lane. Entries are written as their ids are read; what waits for all of a lane's ids is the verdict on it (its
// parameter blocks, slots and the status word), which one block gives without a counter of blocks that have arrived. Bound by
// latency: where only the pages behind `known_pages` are new, one chain of dependent loads; where tables are built anew (4 bytes in,
// 8 out per page), two rounds of 4-byte loads and 8-byte stores a thread, with a division by the extent's size per id. 256
// threads: eight blocks of an SM hold the largest batch in one wave. Measured: 2.4 us for 8 lanes whose pages but one are known,
// 11 for 1 024 of 2 500 (31 MB, 2.8 TB/s).
__global__ void __launch_bounds__(kTableThreads)
step_tables_kernel(const __grid_constant__ StepArgs a) {
  __shared__ uint32_t scratch[kTableThreads / 32];
  const uint32_t l = blockIdx.x, tid = threadIdx.x, capacity = a.layout.row_capacity, page_count = a.layout.pool.page_count;
  const uint32_t begin = a.page_offsets[l], end = a.page_offsets[l + 1], committed = a.committed[l], rows = a.rows[l];
  const uint32_t known = a.known_pages ? a.known_pages[l] : 0;
  uint32_t before = 0; // rows of the lanes before this one
  for (uint32_t i = tid; i < l; i += kTableThreads) before += min(a.rows[i], capacity);
  const bool named = end >= begin && (!a.layout.id_count || end <= a.layout.id_count); // its ids lie in the array
  const uint32_t count = named ? end - begin : 0;
  const uint64_t tokens = uint64_t(committed) + rows;
  bool good = rows > 0 && rows <= capacity && named && tokens <= RK_MAX_PHYSICAL_TOKENS &&
              rk_pages_for(uint32_t(tokens)) <= min(count, a.layout.table_pages);
  const uint32_t pages = good ? rk_pages_for(uint32_t(tokens)) : 0;
  const uint32_t *ids = a.page_ids + begin;
  rk_page_entry *table = a.out.entries + uint64_t(l) * a.layout.table_pages;
  constexpr uint32_t kBatch = 8; // ids of a thread in flight
  for (uint32_t base = min(known, pages); base < pages; base += kTableThreads * kBatch) {
    uint32_t id[kBatch];
#pragma unroll
    for (uint32_t k = 0; k < kBatch; ++k) {
      const uint32_t j = base + k * kTableThreads + tid;
      id[k] = j < pages ? __ldg(ids + j) : 0;
    }
#pragma unroll
    for (uint32_t k = 0; k < kBatch; ++k) {
      const uint32_t j = base + k * kTableThreads + tid;
      if (j >= pages) break;
      if (id[k] >= page_count) { good = false; continue; }
      const uint32_t extent = id[k] / a.layout.pool.extent_pages;
      table[j] = rk_make_entry(a.layout.pool.base + extent * a.layout.pool.extent_stride, id[k] - extent * a.layout.pool.extent_pages);
    }
  }
  // the new rows' slots; a page among the known ones is looked at here too
  const uint32_t mine = min(rows, capacity);
  uint64_t slot = ~uint64_t(0);
  if (tid < mine && pages) {
    const uint32_t position = committed + tid, id = ids[position / kPageTokens];
    if (id >= page_count) good = false;
    slot = uint64_t(id) * kPageTokens + position % kPageTokens;
  }
  good = !__syncthreads_or(!good);
  before = block_sum(before, scratch);
  if (tid < mine) a.out.row_slots[before + tid] = good ? slot : ~uint64_t(0);
  if (tid == 0) {
    const uint32_t live = good ? rows : 0; // a lane without live rows is skipped by every kernel
    a.out.row_offsets[l] = before;
    if (l + 1 == a.layout.lanes) a.out.row_offsets[l + 1] = before + mine;
    a.out.chunk_params[l] = rk_chunk_params{committed, live, RK_VERIFY_CHUNK_STRIDE, count, rk_kv_layer{0, 0}};
    a.out.verify_params[l] = rk_verify_params{committed, count, rk_kv_layer{0, 0}, a.layout.split_count, a.layout.split_count, live, capacity, a.layout.score_scale};
    if (!good && rows) atomicOr(a.out.status, 1u); // rows == 0 is an idle lane
  }
}

// ---- groups of lanes that share a prefix ---------------------------------------------------------------------------
// A page is shared when two tables hold the same entry. leader(l) = the lowest lane whose first entry is lane l's;
// common(l) = leading entries equal to the leader's, among the pages that are full on both sides. Of the lanes of a
// leader, those with common >= p form a group that reads p pages once instead of n times: p is chosen to save most,
// (n - 1) * p, ties to the larger p. Two dependent launches, a chain of dependent loads each: bound by latency, 5 us for 32
// lanes over 32K tokens, 15 for 1 024.

// full pages of a lane that takes part
__device__ __forceinline__ uint32_t full_pages(rk_verify_params p) {
  p.kv.extent_pages = 1; // placement plays no part
  return rk_verify_contract_valid(&p) ? p.committed_tokens / kPageTokens : 0;
}

// One block per lane: its leader and their common pages, left in the two outputs.
__global__ void __launch_bounds__(kGroupThreads)
common_prefix_kernel(uint32_t lanes, const rk_page_entry *const *__restrict__ tables, const rk_verify_params *__restrict__ lane_params,
                     uint32_t *__restrict__ leaders, uint32_t *__restrict__ commons) {
  __shared__ uint32_t found, differ;
  const uint32_t l = blockIdx.x, tid = threadIdx.x;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); // the second kernel waits for this grid's writes
  const uint32_t full = full_pages(lane_params[l]);
  if (!full) {
    if (tid == 0) { leaders[l] = RK_NO_GROUP; commons[l] = 0; }
    return;
  }
  const rk_page_entry *table = tables[l];
  if (tid == 0) { found = l; differ = RK_NO_GROUP; }
  __syncthreads();
  const rk_page_entry first = table[0];
  constexpr uint32_t kRounds = kMaxLanes / kGroupThreads; // every lane's pointer, then every first entry, in flight at once
  const rk_page_entry *theirs_at[kRounds];
#pragma unroll
  for (uint32_t r = 0; r < kRounds; ++r) {
    const uint32_t i = tid + r * kGroupThreads;
    theirs_at[r] = i < l && full_pages(lane_params[i]) ? tables[i] : nullptr;
  }
  bool same[kRounds];
#pragma unroll
  for (uint32_t r = 0; r < kRounds; ++r) same[r] = theirs_at[r] && *theirs_at[r] == first;
#pragma unroll
  for (uint32_t r = 0; r < kRounds; ++r)
    if (same[r]) { atomicMin(&found, tid + r * kGroupThreads); break; } // this thread's lowest
  __syncthreads();
  const uint32_t leader = found;
  uint32_t common = full;
  if (leader != l) {
    const rk_page_entry *theirs = tables[leader];
    const uint32_t reach = min(full, full_pages(lane_params[leader]));
    constexpr uint32_t kBatch = 4; // entries of a thread in flight
    common = reach;
    for (uint32_t base = 0; base < reach; base += kGroupThreads * kBatch) {
      bool equal[kBatch];
#pragma unroll
      for (uint32_t k = 0; k < kBatch; ++k) {
        const uint32_t j = base + k * kGroupThreads + tid;
        equal[k] = j >= reach || table[j] == theirs[j];
      }
#pragma unroll
      for (uint32_t k = 0; k < kBatch; ++k)
        if (!equal[k]) atomicMin(&differ, base + k * kGroupThreads + tid);
      __syncthreads();
      const uint32_t at = differ;
      __syncthreads(); // everyone has read it before the next round moves it
      if (at != RK_NO_GROUP) { common = at; break; }
    }
  }
  if (tid == 0) { leaders[l] = leader; commons[l] = common; }
}

// One block: sorts (leader, common descending, lane), reads off how many lanes of a leader have at least a lane's common
// pages, picks each leader's best count and writes the groups.
__global__ void __launch_bounds__(kMaxLanes)
form_groups_kernel(uint32_t lanes, uint32_t size, uint32_t minimum_lanes, uint32_t minimum_pages, uint32_t *__restrict__ lane_groups,
                   uint32_t *__restrict__ group_pages) {
  __shared__ uint32_t keys[kMaxLanes]; // leader << 16 | 0xffff - common (common <= 8 192)
  __shared__ uint32_t starts[kMaxLanes];
  __shared__ unsigned long long best[kMaxLanes]; // saved pages << 32 | common
  const uint32_t tid = threadIdx.x;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint32_t leader = tid < lanes ? __ldcg(lane_groups + tid) : RK_NO_GROUP, common = tid < lanes ? __ldcg(group_pages + tid) : 0;
  keys[tid] = leader == RK_NO_GROUP ? 0xffffffffu : leader << 16 | (0xffffu - common);
  best[tid] = 0;
  // bitonic sort; steps between lanes of a warp need neither shared memory nor a barrier
  uint32_t held = keys[tid];
  for (uint32_t k = 2; k <= size; k <<= 1)
    for (uint32_t j = k >> 1; j > 0; j >>= 1) {
      uint32_t theirs;
      if (j >= 32) {
        __syncthreads();
        keys[tid] = held;
        __syncthreads();
        theirs = keys[tid ^ j];
      } else {
        theirs = __shfl_xor_sync(0xffffffffu, held, j);
      }
      const bool low = (tid & j) == 0, ascending = (tid & k) == 0;
      held = low == ascending ? min(held, theirs) : max(held, theirs);
    }
  __syncthreads();
  keys[tid] = held;
  __syncthreads();
  const uint32_t key = keys[tid];
  const bool live = key != 0xffffffffu;
  if (live && (tid == 0 || keys[tid - 1] >> 16 != key >> 16)) starts[key >> 16] = tid;
  __syncthreads();
  // the last of a run of equal keys knows how many lanes have at least that many common pages
  if (live && (tid + 1 == size || keys[tid + 1] != key)) {
    const uint32_t count = tid - starts[key >> 16] + 1, pages = 0xffffu - (key & 0xffffu);
    if (count >= minimum_lanes && pages >= minimum_pages)
      atomicMax(&best[key >> 16], static_cast<unsigned long long>(uint64_t(count - 1) * pages) << 32 | pages);
  }
  __syncthreads();
  if (tid < lanes) {
    const uint32_t pages = leader == RK_NO_GROUP ? 0 : uint32_t(best[leader]);
    lane_groups[tid] = pages && common >= pages ? leader : RK_NO_GROUP;
    group_pages[tid] = uint32_t(best[tid]);
  }
}

} // namespace
} // namespace rk

using namespace rk;

extern "C" {

int rk_step_tables(const rk_step_layout *layout, const uint32_t *page_ids, const uint32_t *page_offsets, const uint32_t *committed,
                   const uint32_t *rows, const uint32_t *known_pages, const rk_step_outputs *outputs, void *stream) {
  if (!layout || !layout->lanes || layout->lanes > kMaxLanes || !layout->table_pages || !layout->row_capacity ||
      layout->row_capacity > RK_TREE_NODES || !layout->split_count || layout->split_count > RK_VERIFY_MAX_SPLITS) {
    set_error("rk_step_tables: 1..1024 lanes, a row capacity of 1..16, 1..128 splits and at least one table page");
    return kInvalid;
  }
  const rk_step_pool &pool = layout->pool;
  if (!pool.base || (pool.base & RK_PAGE_INDEX_MASK) || !pool.extent_stride || (pool.extent_stride & RK_PAGE_INDEX_MASK) ||
      !pool.extent_pages || pool.extent_pages > RK_PAGE_INDEX_MASK + 1 || !pool.page_count) {
    set_error("rk_step_tables: extents are 16 KiB-aligned and hold at most 16 384 pages");
    return kInvalid;
  }
  if (!page_ids || !page_offsets || !committed || !rows || !outputs || !outputs->entries || !outputs->chunk_params || !outputs->verify_params ||
      !outputs->row_offsets || !outputs->row_slots || !outputs->status) {
    set_error("rk_step_tables: invalid arguments");
    return kInvalid;
  }
  step_tables_kernel<<<layout->lanes, kTableThreads, 0, static_cast<cudaStream_t>(stream)>>>(
      StepArgs{page_ids, page_offsets, committed, rows, known_pages, *layout, *outputs});
  return cuda_status(cudaGetLastError(), "step tables launch");
}

int rk_prefix_groups(uint32_t lanes, const rk_page_entry *const *tables, const rk_verify_params *lane_params, uint32_t minimum_lanes,
                     uint32_t minimum_pages, uint32_t *lane_groups, uint32_t *group_pages, void *stream) {
  if (!lanes || lanes > kMaxLanes || minimum_lanes < 2 || !minimum_pages) {
    set_error("rk_prefix_groups: 1..1024 lanes, groups of at least two lanes and one page");
    return kInvalid;
  }
  if (!tables || !lane_params || !lane_groups || !group_pages || lane_groups == group_pages) {
    set_error("rk_prefix_groups: invalid arguments");
    return kInvalid;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  common_prefix_kernel<<<lanes, kGroupThreads, 0, s>>>(lanes, tables, lane_params, lane_groups, group_pages);
  if (int st = cuda_status(cudaGetLastError(), "common prefix launch")) return st;
  uint32_t size = 32;
  while (size < lanes) size *= 2;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(1);
  config.blockDim = dim3(size);
  config.stream = s;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&config, form_groups_kernel, lanes, size, minimum_lanes, minimum_pages, lane_groups, group_pages),
                     "form groups launch");
}

} // extern "C"
