// shared_prefix.cu — decode attention for a batch in which groups of lanes share the first pages of their tables.
//
// With attention over a context split into a prefix and a rest, a lane's output is the merge of two partials
// {max, sum of exp, sum of exp * v}. The rest is the streaming kernel's business (decode_attention.cu, which leaves the
// shared pages out). The prefix part is the same keys and values for every lane of a group, so its query rows, 6 per lane
// and KV head, stand side by side as the M side of a tensor-core tile: pages are read once per tile, not once per lane,
// and a group of n lanes turns 6 multiply-adds per key element into 6 n.
//
// The kernel is the window kernel's pipeline (verify_attention.cu) with rows gathered from many lanes: TMA brings raw pages
// into a ring, expander warps turn them into 16-bit operand tiles, two warps issue S = Q.K^T and O += P.V with both A
// operands in tensor memory, sixteen warps run the online softmax. All 128 rows of a tile are real rows here.
#include "common.cuh"
#include "decode_partials.cuh"
#include "score_shape.cuh"
#include "window_tile.cuh"

#include <atomic>

namespace rk {
using namespace tile;
namespace {

constexpr uint32_t kMaxLanes = 1024;
constexpr uint32_t kNone = 0xffffu;
constexpr uint32_t kTileLanes = 24;   // lanes with a row in a 128-row tile: at most 23
constexpr uint32_t kLeastUnits = 4;   // 64-token groups of a split: shorter ones cost more in partials than they spread

struct PrefixArgs {
  const uint16_t *queries;
  float *partials;       // [row][256], rows as the lanes' descriptors say
  float *statistics;     // [row]{max, sum}
  uint32_t *descriptors; // [lane]{row of head 0 and split 0, splits, rows of the group, -}
  const rk_page_entry *const *tables;
  const rk_verify_params *lane_params;
  rk_kv_layer layer;
  uint64_t window_base;
  uint32_t lanes;
  uint32_t *status;
  uint32_t spin_limit;
  const uint32_t *lane_groups, *group_pages;
  ShapeArgs shape;
};

// One piece of work: a tile of a group's rows against a run of its 64-token groups, for one KV head.
struct Item {
  uint32_t head, split, splits, tile, group_rows, row_base; // row_base: row of (head 0, split 0, the group's first row)
  uint32_t page_begin, page_end;
  uint32_t group, first_member, leader;
};

// A group with work: its number, members and pages, and the lowest member's lane (whose table the tiles read).
struct GroupWork { uint16_t group, members, pages, leader; };

struct PlanShared {
  uint16_t member_of[kMaxLanes];  // a lane's group, kNone: none
  uint32_t count[kMaxLanes];      // members of a group
  uint32_t leader[kMaxLanes];     // its lowest member
  GroupWork list[kMaxLanes];      // the groups with work, by leader
  uint32_t words[kMaxLanes / 32]; // lanes as bits: leaders, then the members of the item's group
  uint32_t groups, chunk, items;  // groups with work; most 64-token groups of a split; items of the launch
  Item item;
  uint32_t tile_lanes[kTileLanes];
};

__device__ __forceinline__ bool lane_takes_part(rk_verify_params p) {
  p.kv.extent_pages = 1;
  return rk_verify_contract_valid(&p) && p.active_rows == 1 && p.row_capacity == 1;
}
__device__ __forceinline__ uint32_t tiles_of(uint32_t members) { return (members * kG + kM - 1) / kM; }
__device__ __forceinline__ uint32_t units_of(uint32_t pages) { return (pages + 1) / 2; }
// bits of the words before `word`, for a whole warp
__device__ __forceinline__ uint32_t bits_before(const uint32_t *words, uint32_t word) {
  const uint32_t lane = threadIdx.x % 32;
  return __reduce_add_sync(0xffffffffu, lane < word ? uint32_t(__popc(words[lane])) : 0u);
}

// How the launch is cut, the same in every CTA: members per group, the groups with work, and the shortest split length for
// which (KV heads x tiles x splits) of all groups still fit the grid. With more tiles than CTAs every tile is one item and
// the CTAs take them in turn.
__device__ __noinline__ void plan_launch(const PrefixArgs &args, PlanShared &sh) {
  const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32, lanes = args.lanes, words = (lanes + 31) / 32;
  constexpr uint32_t kRounds = (kMaxLanes + kThreads - 1) / kThreads; // warps take whole words: lane i of round r is tid + r * kThreads
  for (uint32_t i = tid; i < lanes; i += kThreads) { sh.count[i] = 0; sh.leader[i] = kMaxLanes; }
  __syncthreads();
  uint32_t group[kRounds], pages[kRounds]; // of this thread's lanes
#pragma unroll
  for (uint32_t r = 0; r < kRounds; ++r) {
    const uint32_t i = tid + r * kThreads;
    group[r] = kNone;
    if (i >= lanes) continue;
    const uint32_t g = args.lane_groups[i];
    const rk_verify_params p = args.lane_params[i];
    const uint32_t shared = g < lanes ? args.group_pages[g] : 0;
    if (shared && lane_takes_part(p)) {
      group[r] = g;
      pages[r] = min(shared, rk_pages_for(p.committed_tokens + 1));
      atomicAdd(&sh.count[g], 1u);
      atomicMin(&sh.leader[g], i);
    }
    sh.member_of[i] = uint16_t(group[r]);
  }
  __syncthreads();
#pragma unroll
  for (uint32_t r = 0; r < kRounds; ++r) {
    const uint32_t i = tid + r * kThreads;
    if (i / 32 >= words) continue; // the whole warp
    const uint32_t mask = __ballot_sync(0xffffffffu, group[r] != kNone && sh.leader[group[r]] == i);
    if (lane == 0) sh.words[i / 32] = mask;
  }
  __syncthreads();
#pragma unroll
  for (uint32_t r = 0; r < kRounds; ++r) {
    const uint32_t i = tid + r * kThreads;
    if (i / 32 >= words) continue;
    const uint32_t mask = sh.words[i / 32], at = bits_before(sh.words, i / 32) + __popc(mask & ((1u << lane) - 1u));
    if (mask >> lane & 1u) sh.list[at] = GroupWork{uint16_t(group[r]), uint16_t(sh.count[group[r]]), uint16_t(pages[r]), uint16_t(i)};
    if (i / 32 + 1 == words && lane == 31) sh.groups = at + (mask >> 31);
  }
  __syncthreads();
  if (warp == 0) {
    const uint32_t groups = sh.groups;
    uint32_t units = 0, tiles = 0; // of all groups, times the KV heads
    for (uint32_t i = lane; i < groups; i += 32) {
      const uint32_t t = kHeads * tiles_of(sh.list[i].members);
      tiles += t;
      units += t * units_of(sh.list[i].pages);
    }
    units = __reduce_add_sync(0xffffffffu, units);
    tiles = __reduce_add_sync(0xffffffffu, tiles);
    auto items_for = [&](uint32_t chunk) {
      uint32_t sum = 0;
      for (uint32_t i = lane; i < groups; i += 32)
        sum += kHeads * tiles_of(sh.list[i].members) * ((units_of(sh.list[i].pages) + chunk - 1) / chunk);
      return __reduce_add_sync(0xffffffffu, sum);
    };
    // items(chunk) <= units / chunk + tiles, and >= units / chunk: the shortest chunk that fits lies between these two
    uint32_t high = units_of(rk_pages_for(RK_MAX_PHYSICAL_TOKENS));
    if (tiles < gridDim.x) {
      high = max(kLeastUnits, units / (gridDim.x - tiles) + 1);
      uint32_t low = max(kLeastUnits, (units + gridDim.x - 1) / gridDim.x);
      while (low < high) {
        const uint32_t middle = (low + high) / 2;
        if (items_for(middle) <= gridDim.x) high = middle; else low = middle + 1;
      }
    }
    const uint32_t items = items_for(high);
    if (lane == 0) { sh.chunk = high; sh.items = items; }
  }
  __syncthreads();
}

// Item number `index` of the launch and the lanes of its tile.
__device__ __noinline__ void find_item(const PrefixArgs &args, PlanShared &sh, uint32_t index) {
  const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32, lanes = args.lanes;
  if (warp == 0) {
    uint32_t before = 0, rows = 0;
    for (uint32_t base = 0; base < sh.groups; base += 32) {
      const bool live = base + lane < sh.groups;
      const GroupWork work = live ? sh.list[base + lane] : GroupWork{0, 0, 0, 0};
      const uint32_t units = units_of(work.pages), splits = (units + sh.chunk - 1) / sh.chunk, tiles = tiles_of(work.members);
      const uint32_t items = kHeads * tiles * splits, group_rows = work.members * kG;
      uint32_t items_up = items, rows_up = kHeads * splits * group_rows;
#pragma unroll
      for (uint32_t o = 1; o < 32; o <<= 1) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, items_up, o), b = __shfl_up_sync(0xffffffffu, rows_up, o);
        if (lane >= o) { items_up += a; rows_up += b; }
      }
      const uint32_t found = __ballot_sync(0xffffffffu, live && index < before + items_up);
      if (found) {
        if (lane == uint32_t(__ffs(found) - 1)) {
          const uint32_t within = index - (before + items_up - items);
          Item &item = sh.item;
          item.head = within % kHeads;
          item.tile = within / kHeads % tiles;
          item.split = within / kHeads / tiles;
          item.splits = splits;
          item.group_rows = group_rows;
          item.row_base = rows + rows_up - kHeads * splits * group_rows;
          item.page_begin = 2 * (units * item.split / splits);
          item.page_end = min(uint32_t(work.pages), 2 * (units * (item.split + 1) / splits));
          item.group = work.group;
          item.leader = work.leader;
          item.first_member = item.tile * kM / kG;
        }
        break;
      }
      before += __shfl_sync(0xffffffffu, items_up, 31);
      rows += __shfl_sync(0xffffffffu, rows_up, 31);
    }
  }
  if (tid < kTileLanes) sh.tile_lanes[tid] = kMaxLanes;
  __syncthreads();
  for (uint32_t w = warp; w < (lanes + 31) / 32; w += kThreads / 32) {
    const uint32_t i = 32 * w + lane;
    const uint32_t mask = __ballot_sync(0xffffffffu, i < lanes && sh.member_of[i] == sh.item.group);
    if (lane == 0) sh.words[w] = mask;
  }
  __syncthreads();
  for (uint32_t w = warp; w < (lanes + 31) / 32; w += kThreads / 32) {
    const uint32_t rank = bits_before(sh.words, w) + __popc(sh.words[w] & ((1u << lane) - 1u));
    if ((sh.words[w] >> lane & 1u) && rank >= sh.item.first_member && rank < sh.item.first_member + kTileLanes)
      sh.tile_lanes[rank - sh.item.first_member] = 32 * w + lane;
  }
  __syncthreads();
}

template <uint32_t Format, bool kShaped>
__global__ void __launch_bounds__(kThreads, 1)
shared_prefix_kernel(const __grid_constant__ CUtensorMap head_map, PrefixArgs args) {
  using Kind = Traits<Format>;
  constexpr uint32_t kSlab = Kind::kSlab, kRawStages = Kind::kRawStages, kRawStageBytes = raw_stage_bytes<Format>();
  constexpr uint32_t kRawScaleOffset = 4 * kSlab;
  constexpr uint32_t kTileStages = Kind::kTileStages, kExpandThreads = kExpandWarps * 32 / kTileStages;
  extern __shared__ uint8_t dynamic_shared[];
  const uint32_t tiles = (smem_u32(dynamic_shared) + 1023u) & ~1023u;
  uint8_t *tile_ptr = dynamic_shared + (tiles - smem_u32(dynamic_shared));
  Control &ctl = *reinterpret_cast<Control *>(tile_ptr + tile_bytes<Format>());
  PlanShared &plan = *reinterpret_cast<PlanShared *>(&ctl + 1);
  volatile uint32_t *error = &ctl.error;
  const uint32_t k_tile = tiles, v_tile = k_tile + kTileStages * kKBytes, raw_tile = v_tile + kTileStages * kVBytes; // K stages | V stages | raw ring
  uint8_t *k_ptr = tile_ptr, *v_ptr = k_ptr + kTileStages * kKBytes;
  const uint8_t *raw_ptr = v_ptr + kTileStages * kVBytes;
  const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); // the streaming kernel takes the SMs that this one leaves

  if (tid == 0) {
    for (uint32_t r = 0; r < kRawStages; ++r) {
      barrier_init(smem_u32(&ctl.raw_full[r]), 1);
      barrier_init(smem_u32(&ctl.raw_free[r]), kExpandThreads);
    }
    for (uint32_t b = 0; b < 2; ++b) {
      barrier_init(smem_u32(&ctl.k_full[b]), kExpandThreads);
      barrier_init(smem_u32(&ctl.v_full[b]), kExpandThreads);
      barrier_init(smem_u32(&ctl.k_free[b]), 1);
      barrier_init(smem_u32(&ctl.v_free[b]), 1);
      barrier_init(smem_u32(&ctl.s_full[b]), 1);
      barrier_init(smem_u32(&ctl.p_free[b]), 1);
      barrier_init(smem_u32(&ctl.p_full[b]), kSoftmaxThreads);
    }
    for (uint32_t b = 0; b < kScaleStages; ++b) barrier_init(smem_u32(&ctl.scale_free[b]), kSoftmaxThreads);
    barrier_init(smem_u32(&ctl.drained[0]), 1);
    barrier_init(smem_u32(&ctl.drained[1]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    ctl.error = 0;
    ctl.spin_limit = args.spin_limit;
  }
  // The partition reads only the lanes' parameter blocks and groups, which no kernel that lets a dependent start early
  // writes; everything else waits for the predecessor.
  plan_launch(args, plan);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (blockIdx.x == 0)
    for (uint32_t i = tid; i < args.lanes; i += kThreads)
      if (plan.member_of[i] == kNone) reinterpret_cast<uint4 *>(args.descriptors)[i] = make_uint4(0, 0, 0, 0);
  if (blockIdx.x >= plan.items) return;
  if (warp == kTmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem_base)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = ctl.tmem_base;
  const uint32_t tmem_o = tmem + kTmemO, tmem_s = tmem + kTmemS, tmem_q = tmem + kTmemQ;
  const uint32_t data_bytes = kHeads * kSlab, scale_bytes = Kind::kScales ? kPageTokens * kHeads * 4 : 0;

  uint32_t done = 0; // 64-token groups of earlier items: every ring, stage and barrier counts on across items
  for (uint32_t index = blockIdx.x; index < plan.items; index += gridDim.x) {
    find_item(args, plan, index);
    const Item item = plan.item;
    const uint32_t page_begin = item.page_begin, page_end = item.page_end, groups = (page_end - page_begin + 1) / 2;
    const rk_page_entry *table = args.tables[item.leader];
    if (item.head == 0 && item.split == 0 && tid < kTileLanes && plan.tile_lanes[tid] < kMaxLanes) {
      const uint32_t first_row = (item.first_member + tid) * kG; // the tile that holds a lane's first row writes its descriptor
      if (first_row >= item.tile * kM && first_row < (item.tile + 1) * kM)
        reinterpret_cast<uint4 *>(args.descriptors)[plan.tile_lanes[tid]] = make_uint4(item.row_base + first_row, item.splits, item.group_rows, 0);
    }

    // ---- this thread's row, and the query tile into tensor memory (layout as in the window kernel) ----
    const uint32_t quarter = warp & 3u, part = warp >> 2, my_row = quarter * 32 + lane;
    const uint32_t fused = item.tile * kM + my_row; // row of the group
    const bool real = warp < kSoftmaxWarps && fused < item.group_rows;
    const uint32_t my_lane = real ? plan.tile_lanes[fused / kG - item.first_member] : 0;
    int exponent = 0; // a power of two keeps large queries inside fp16 (exact)
    if (warp < kSoftmaxWarps) {
      const uint16_t *query = args.queries + ((uint64_t(my_lane) * kHeads + item.head) * RK_VERIFY_CHUNK_STRIDE * kG + fused % kG) * kD;
      const uint32_t column = part * (128 / kRowThreads); // 32 columns = 64 dims of the row
      if (!Kind::kBf16) {
        float amax = 0.0f;
#pragma unroll 4
        for (uint32_t c = 0; c < 8; ++c) {
          if (!real) break;
          const uint4 raw = __ldg(reinterpret_cast<const uint4 *>(query + 2 * column + 8 * c));
          const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i)
            amax = fmaxf(amax, fmaxf(fabsf(bf16_bits_to_float(words[i] & 0xffffu)), fabsf(bf16_bits_to_float(words[i] >> 16))));
        }
        ctl.exchange[1][part][my_row] = amax;
        asm volatile("bar.sync %0, %1;" ::"r"(1u + quarter), "n"(32 * kRowThreads) : "memory");
#pragma unroll
        for (uint32_t i = 0; i < kRowThreads; ++i) amax = fmaxf(amax, ctl.exchange[1][i][my_row]);
        if (amax >= 8192.0f) exponent = ilogbf(amax) - 12;
      }
      const float down = ldexpf(1.0f, -exponent);
      float q_sum = 0.0f; // over the values the tensor core will see, for the key-offset correction
      float columns[32];
#pragma unroll
      for (uint32_t c = 0; c < 8; ++c) {
        uint4 raw = make_uint4(0, 0, 0, 0);
        if (real) raw = __ldg(reinterpret_cast<const uint4 *>(query + 2 * column + 8 * c));
        const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
        uint32_t chunk[4];
        if (Kind::kBf16) {
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) chunk[i] = words[i];
        } else {
          float d[8];
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) { d[2 * i] = bf16_bits_to_float(words[i] & 0xffffu) * down; d[2 * i + 1] = bf16_bits_to_float(words[i] >> 16) * down; }
          if (Format == RK_FORMAT_INT4) {
            chunk[0] = pack_half2(d[0], d[4]); chunk[1] = pack_half2(d[1] * 0.0625f, d[5] * 0.0625f);
            chunk[2] = pack_half2(d[2], d[6]); chunk[3] = pack_half2(d[3] * 0.0625f, d[7] * 0.0625f);
          } else {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) chunk[i] = pack_half2(d[2 * i], d[2 * i + 1]);
          }
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) {
            const __half2 h = *reinterpret_cast<const __half2 *>(&chunk[i]);
            q_sum += ((Format == RK_FORMAT_INT4 && (i & 1u)) ? 16.0f : 1.0f) * (__low2float(h) + __high2float(h));
          }
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) columns[c * 4 + i] = __uint_as_float(chunk[i]);
      }
      tmem_store32(tmem_q + ((quarter * 32u) << 16) + column, columns);
      ctl.exchange[0][part][my_row] = q_sum;
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    if (tid < kM) {
      float total = 0.0f;
#pragma unroll
      for (uint32_t i = 0; i < kRowThreads; ++i) total += ctl.exchange[0][i][tid];
      ctl.q_sums[tid] = total;
    }
    __syncthreads();

    if (warp == kTmaWarp) {
      // ---- TMA producer: lanes 0-7 issue one copy each (page, {K, V, key scales, value scales}) of the group ----
      const uint32_t local = (lane >> 2) & 1u, kind = lane & 3u;
      const bool copier = lane < 8 && (kind < 2 || Kind::kScales);
      const uint64_t extent_pages = args.layer.extent_pages;
      const uint64_t tensor_base = args.layer.offset +
                                   extent_pages * (kind == 0 ? 0ull : kind == 2 ? uint64_t(data_bytes)
                                                    : kind == 1 ? uint64_t(data_bytes) + scale_bytes : 2ull * data_bytes + scale_bytes) +
                                   item.head * (kind < 2 ? kSlab : 128u);
      const uint32_t page_stride = kind < 2 ? data_bytes : scale_bytes;
      rk_page_entry next = lane < 8 && page_begin + local < page_end ? table[page_begin + local] : 0;
      for (uint32_t g = 0; g < groups; ++g) {
        const uint32_t n = done + g, r = n % kRawStages, first = page_begin + 2 * g, group_pages = min(2u, page_end - first);
        const rk_page_entry entry = next;
        if (lane < 8 && first + 2 + local < page_end) next = table[first + 2 + local];
        if (n >= kRawStages) barrier_wait(&ctl.raw_free[r], n / kRawStages - 1, error);
        const uint32_t full = smem_u32(&ctl.raw_full[r]), stage = raw_tile + r * kRawStageBytes;
        if (lane == 0) barrier_expect(full, group_pages * (2 * kSlab + (Kind::kScales ? 256 : 0)));
        __syncwarp();
        if (copier && local < group_pages) {
          const uint64_t address = rk_entry_extent(entry) + tensor_base + uint64_t(rk_entry_index(entry)) * page_stride;
          if (kind < 2) tma_load_rows(stage + (2 * kind + local) * kSlab, &head_map, int32_t((address - args.window_base) >> 7), full);
          else bulk_load(stage + kRawScaleOffset + (2 * (kind - 2) + local) * 128, reinterpret_cast<const void *>(address), 128, full);
        }
      }
      // every copy of this item has landed before the CTA goes on or leaves (also after a failed wait)
      if (lane == 0)
        for (uint32_t g = groups > kRawStages ? groups - kRawStages : 0; g < groups; ++g) {
          const uint32_t n = done + g, bar = smem_u32(&ctl.raw_full[n % kRawStages]), parity = (n / kRawStages) & 1u;
          for (uint32_t i = 0; i < kSpinLimit && !barrier_try(bar, parity); ++i) __nanosleep(64);
        }
      __syncwarp();
    } else if (warp == kScoreWarp) {
      // ---- S = Q.K^T; the whole warp walks the loop, one elected lane issues ----
      const uint32_t idesc_qk = umma_instruction(kM, kGroupTokens, Kind::kBf16, Kind::kBf16);
      const uint64_t k_desc0 = umma_descriptor(k_tile), k_desc1 = umma_descriptor(k_tile + kKBytes);
      for (uint32_t g = 0; g < groups; ++g) {
        const uint32_t n = done + g, b = n & 1u, t = n % kTileStages;
        barrier_wait(&ctl.k_full[t], n / kTileStages, error);
        if (n >= 2) barrier_wait(&ctl.p_free[b], (n >> 1) - 1, error);
        tmem_fence_after();
        const uint64_t desc = t ? k_desc1 : k_desc0;
        const uint32_t target = tmem_s + b * 64;
        if (elect_one()) {
#pragma unroll
          for (uint32_t j = 0; j < 16; ++j)
            umma_f16_ts(target, tmem_q + 8 * j, desc + (((j >> 2) * (kGroupTokens * 128) + (j & 3u) * 32) >> 4), idesc_qk, j ? 1u : 0u);
          umma_commit(&ctl.s_full[b]);
          umma_commit(&ctl.k_free[t]);
        }
        __syncwarp();
      }
    } else if (warp == kValueWarp) {
      // ---- O += P.V ----
      const uint32_t idesc_pv = umma_instruction(kM, kD, Kind::kBf16, Kind::kBf16);
      const uint64_t v_desc0 = umma_descriptor(v_tile), v_desc1 = umma_descriptor(v_tile + kVBytes);
      for (uint32_t g = 0; g < groups; ++g) {
        const uint32_t n = done + g, b = n & 1u, t = n % kTileStages;
        barrier_wait(&ctl.v_full[t], n / kTileStages, error);
        barrier_wait(&ctl.p_full[b], n >> 1, error);
        tmem_fence_after();
        const uint64_t desc = t ? v_desc1 : v_desc0;
        const uint32_t source = tmem_s + b * 64;
        if (elect_one()) {
#pragma unroll
          for (uint32_t j = 0; j < 4; ++j) {
            umma_f16_ts(tmem_o, source + 8 * j, desc + ((j * 32) >> 4), idesc_pv, (g || j) ? 1u : 0u);
            if (Kind::kBf16) umma_f16_ts(tmem_o, source + 32 + 8 * j, desc + ((j * 32) >> 4), idesc_pv, 1u); // the low parts
          }
          umma_commit(&ctl.v_free[t]);
          umma_commit(&ctl.p_free[b]);
        }
        __syncwarp();
      }
    } else if (warp >= kSoftmaxWarps) {
      // ---- expanders: raw codes -> 16-bit operand tiles; the team of an operand stage ----
      const uint32_t index = tid - kSoftmaxThreads, team = index / kExpandThreads, e = index - team * kExpandThreads;
      for (uint32_t g = (team + kTileStages - done % kTileStages) % kTileStages; g < groups; g += kTileStages) {
        const uint32_t n = done + g, r = n % kRawStages, round = n / kTileStages, first = page_begin + 2 * g;
        const ValidBelow valid{min(2u, page_end - first) * kPageTokens};
        const uint8_t *raw = raw_ptr + r * kRawStageBytes;
        barrier_wait(&ctl.raw_full[r], n / kRawStages, error);
        if (e < kGroupTokens) {
          if (n >= kScaleStages) barrier_wait(&ctl.scale_free[n % kScaleStages], n / kScaleStages - 1, error);
          const uint32_t token = Expand<Format>::token_of(e);
          float3 triple = make_float3(0.0f, 0.0f, 0.0f);
          if (valid.holds(token)) {
            if (Kind::kScales) {
              const float ks = reinterpret_cast<const float *>(raw + kRawScaleOffset)[token];
              const float vs = fmaxf(reinterpret_cast<const float *>(raw + kRawScaleOffset)[64 + token], 9.094947e-13f); // 2^-40
              triple = make_float3(ks, log2_fast(vs), __fdividef(0.015625f, vs));
            } else {
              triple = make_float3(1.0f, 0.0f, 0.015625f);
            }
          }
          ctl.scales[n % kScaleStages].put(e, triple.x, triple.y, triple.z);
        }
        if (round) barrier_wait(&ctl.k_free[team], round - 1, error);
        Expand<Format>::template keys<kExpandThreads>(raw, k_ptr + team * kKBytes, e);
        async_proxy_fence();
        barrier_arrive(smem_u32(&ctl.k_full[team]));
        if (round) barrier_wait(&ctl.v_free[team], round - 1, error);
        Expand<Format>::template values<kExpandThreads>(raw, v_ptr + team * kVBytes, e, valid);
        async_proxy_fence();
        barrier_arrive(smem_u32(&ctl.v_full[team]));
        barrier_arrive(smem_u32(&ctl.raw_free[r]));
      }
    } else {
      // ---- softmax: kRowThreads threads per row, kRowTokens contraction positions each ----
      const rk_verify_params p = args.lane_params[my_lane];
      const float score_scale = rk_score_scale(p.score_scale, kD) * kLog2e;
      const float row_factor = ldexpf(score_scale, Kind::kKeyShift + exponent);
      const float row_offset = -Kind::kKeyOffset * ctl.q_sums[my_row] * ldexpf(score_scale, exponent);
      const uint32_t position = p.committed_tokens;
      const float slope = kShaped && args.shape.slopes ? __ldg(args.shape.slopes + item.head * kG + fused % kG) * kLog2e : 0.0f;
      const uint32_t row_window = kShaped && args.shape.window && position + 1 > args.shape.window ? position + 1 - args.shape.window : 0;
      const uint32_t lane_address = (quarter * 32u) << 16;
      constexpr uint32_t kOutColumns = kD / kRowThreads;
      constexpr bool kPermuted = Format == RK_FORMAT_INT4;
      const uint32_t part_token = kPermuted ? (kRowTokens / 8) * part : kRowTokens * part;
      float row_max = -1.0e30f, row_sum = 0.0f; // row_sum: this thread's tokens only
      for (uint32_t g = 0; g < groups; ++g) {
        const uint32_t n = done + g, b = n & 1u, first = page_begin + 2 * g, base = first * kPageTokens;
        const GroupView view{base, base + kPageTokens, first + 1 < page_end};
        const ScaleStage &stage = ctl.scales[n % kScaleStages];
        barrier_wait(&ctl.s_full[b], n >> 1, error);
        tmem_fence_after();
        float scores[kRowTokens];
        tmem_load_scores(tmem_s + b * 64 + lane_address + part * kRowTokens, scores);
        float group_max = -INFINITY;
        if (kShaped) {
          shape_scores<kRowTokens, kPermuted>(scores, stage, part * kRowTokens, row_factor, row_offset, part_token, args.shape, slope, view, position);
        } else {
          scale_scores(scores, stage, part * kRowTokens, row_factor, row_offset);
        }
        mask_scores<kRowTokens, kPermuted>(scores, part_token, view, position, row_window, kShaped ? args.shape.sinks : 0, real);
#pragma unroll
        for (uint32_t i = 0; i < kRowTokens; ++i) group_max = fmaxf(group_max, scores[i]);
        // the row's other parts; past this barrier every part holds its scores in registers, so the probabilities may
        // overwrite the first 32 columns of the buffer
        ctl.exchange[b][part][my_row] = group_max;
        tmem_fence_before();
        asm volatile("bar.sync %0, %1;" ::"r"(1u + quarter), "n"(32 * kRowThreads) : "memory");
        tmem_fence_after();
#pragma unroll
        for (uint32_t i = 0; i < kRowThreads; ++i) group_max = fmaxf(group_max, ctl.exchange[b][i][my_row]);
        // the reference exponent only moves when the maximum grew by more than 2^8: fp16 probabilities stay below 2^14
        const bool grow = group_max > row_max + 8.0f;
        float scale = 1.0f;
        if (grow) {
          scale = exp2_fast(row_max - group_max);
          row_max = group_max;
          row_sum *= scale;
        }
        const float exponent_base = row_max - 6.0f;
        weigh_scores(scores, stage, part * kRowTokens, exponent_base, row_sum); // row_sum: of 2^(score - row_max)
        uint32_t packed[kRowTokens / 2], packed_low[Kind::kBf16 ? kRowTokens / 2 : 1];
#pragma unroll
        for (uint32_t c = 0; c < kRowTokens / 2; ++c) {
          const float w[2] = {scores[2 * c], scores[2 * c + 1]};
          if (Kind::kBf16) { // a high and a low bf16 part: 16 bits of the probability
            packed[c] = pack_bfloat2(w[0], w[1]);
            packed_low[c] = pack_bfloat2(w[0] - __uint_as_float(packed[c] << 16), w[1] - __uint_as_float(packed[c] & 0xffff0000u));
          } else {
            packed[c] = pack_half2(w[0], w[1]);
          }
        }
        if (g && __any_sync(0xffffffffu, grow)) { // this part rescales its columns of O once P.V(g-1) has landed
          barrier_wait(&ctl.v_free[(n - 1) % kTileStages], (n - 1) / kTileStages, error);
          tmem_fence_after();
#pragma unroll 1
          for (uint32_t c = 0; c < kOutColumns / 32; ++c) {
            float o[32];
            tmem_load32(tmem_o + lane_address + part * kOutColumns + c * 32, o);
#pragma unroll
            for (uint32_t i = 0; i < 32; ++i) o[i] *= scale;
            tmem_store32(tmem_o + lane_address + part * kOutColumns + c * 32, o);
          }
        }
        tmem_store_packed(tmem_s + b * 64 + lane_address + part * (kRowTokens / 2), packed);
        if constexpr (Kind::kBf16) tmem_store_packed(tmem_s + b * 64 + 32 + lane_address + part * (kRowTokens / 2), packed_low);
        tmem_fence_before();
        barrier_arrive(smem_u32(&ctl.p_full[b]));
        barrier_arrive(smem_u32(&ctl.scale_free[n % kScaleStages]));
      }

      // ---- partial output: the row of O, un-normalised; statistics {reference exponent, sum} ----
      const uint32_t last = done + groups - 1;
      barrier_wait(&ctl.v_free[last % kTileStages], last / kTileStages, error);
      tmem_fence_after();
      const bool failed = *error != 0;
      const uint64_t row = item.row_base + uint64_t(item.head * item.splits + item.split) * item.group_rows + fused;
      float *out = args.partials + row * kD + part * kOutColumns;
#pragma unroll 1
      for (uint32_t c = 0; c < kOutColumns / 32; ++c) {
        float o[32];
        tmem_load32(tmem_o + lane_address + part * kOutColumns + c * 32, o);
        if (real) {
#pragma unroll
          for (uint32_t i = 0; i < 32; i += 4)
            *reinterpret_cast<float4 *>(out + c * 32 + i) = make_float4(o[i] * 0.015625f, o[i + 1] * 0.015625f, o[i + 2] * 0.015625f, o[i + 3] * 0.015625f);
        }
      }
      ctl.exchange[(last + 1) & 1u][part][my_row] = row_sum;
      asm volatile("bar.sync %0, %1;" ::"r"(1u + quarter), "n"(32 * kRowThreads) : "memory");
      if (part == 0 && real) {
        float total = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kRowThreads; ++i) total += ctl.exchange[(last + 1) & 1u][i][my_row];
        args.statistics[row * 2] = failed ? -INFINITY : row_max * kLn2;
        args.statistics[row * 2 + 1] = failed ? 0.0f : total;
      }
    }
    done += groups;
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
  }
  // Tensor memory is released once every contraction that was issued has completed, also when a wait gave up.
  if (warp == kScoreWarp || warp == kValueWarp) {
    uint64_t *drained = &ctl.drained[warp - kScoreWarp];
    if (elect_one()) umma_commit(drained);
    __syncwarp();
    for (uint32_t i = 0; i < kSpinLimit && !barrier_try(smem_u32(drained), 0); ++i) __nanosleep(64);
  }
  tmem_fence_before();
  __syncthreads();
  if (tid == 0 && ctl.error) atomicExch(args.status, 1u);
  if (warp == kTmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// ---- the merge: a lane's prefix splits, then its streaming partials, in that order ------------------------------------
// thread = (query head of the block's kRows, slot group, four consecutive dims). Slot t belongs to group t mod kGroups; a
// group folds its slots in rising order with a running maximum, statistics and rows of a batch in flight together, and
// the groups are merged in order: a fixed function of the slot counts.
template <uint32_t kGroups, uint32_t kRows>
__global__ void __launch_bounds__(64 * kGroups * kRows)
shared_merge_kernel(const float *__restrict__ partials, const float *__restrict__ statistics, const uint32_t *__restrict__ descriptors,
                    const float *__restrict__ prefix_partials, const float *__restrict__ prefix_statistics,
                    const uint4 *__restrict__ prefix_descriptors, uint16_t *__restrict__ output, float *__restrict__ output_f32,
                    const rk_verify_params *__restrict__ lane_params) {
  constexpr uint32_t kBatch = kGroups == 1 ? 8 : 4;
  __shared__ float4 sums[kRows][kGroups][kD / 4];
  __shared__ float2 stats[kRows][kGroups];
  const uint32_t head = blockIdx.y, l = blockIdx.z, tid = threadIdx.x, quad = tid & 63u, group = tid / 64 % kGroups, row = tid / (64 * kGroups);
  const uint32_t query_head = blockIdx.x * kRows + row;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory"); // the streaming kernel, which itself waited for the prefix kernel
  const uint2 descriptor = __ldcg(reinterpret_cast<const uint2 *>(descriptors + 2 * l));
  const uint4 prefix = __ldcg(prefix_descriptors + l);
  if (!lane_takes_part(lane_params[l])) return;
  const LaneSlots lane_slots(descriptor);
  const uint32_t splits = prefix.y, slots = splits + lane_slots.slots;
  float running = -INFINITY, denominator = 0.0f;
  float4 numerator = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (uint32_t t = group; t < slots; t += kGroups * kBatch) {
    float2 stat[kBatch];
    float4 part[kBatch];
#pragma unroll
    for (uint32_t k = 0; k < kBatch; ++k) { // every load of the batch is in flight before the first fold
      const uint32_t at = t + k * kGroups;
      stat[k] = make_float2(-INFINITY, 0.0f);
      part[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (at < slots) {
        const bool of_prefix = at < splits;
        const uint64_t where = of_prefix ? prefix.x + uint64_t(head * splits + at) * prefix.z + query_head
                                         : lane_slots.slot(at - splits, head) * kG + query_head;
        stat[k] = __ldcg(reinterpret_cast<const float2 *>(of_prefix ? prefix_statistics : statistics) + where);
        part[k] = __ldcg(reinterpret_cast<const float4 *>((of_prefix ? prefix_partials : partials) + where * kD) + quad);
      }
    }
#pragma unroll
    for (uint32_t k = 0; k < kBatch; ++k) {
      if (stat[k].x == -INFINITY) continue; // an empty partial (or past the last slot) weighs nothing
      if (stat[k].x > running) {
        const float scale = expf(running - stat[k].x); // 0 for the first slot
        numerator.x *= scale; numerator.y *= scale; numerator.z *= scale; numerator.w *= scale;
        denominator *= scale;
        running = stat[k].x;
      }
      const float weight = expf(stat[k].x - running);
      numerator.x += weight * part[k].x; numerator.y += weight * part[k].y;
      numerator.z += weight * part[k].z; numerator.w += weight * part[k].w;
      denominator += weight * stat[k].y;
    }
  }
  if (kGroups > 1) {
    sums[row][group][quad] = numerator;
    if (quad == 0) stats[row][group] = make_float2(running, denominator);
    __syncthreads();
    if (group) return;
    float maximum = stats[row][0].x;
#pragma unroll
    for (uint32_t g = 1; g < kGroups; ++g) maximum = fmaxf(maximum, stats[row][g].x);
    numerator = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    denominator = 0.0f;
#pragma unroll
    for (uint32_t g = 0; g < kGroups; ++g) {
      const float2 own = stats[row][g];
      const float weight = own.x == -INFINITY ? 0.0f : expf(own.x - maximum);
      const float4 other = sums[row][g][quad];
      numerator.x += weight * other.x; numerator.y += weight * other.y; numerator.z += weight * other.z; numerator.w += weight * other.w;
      denominator += weight * own.y;
    }
  }
  const float inverse = denominator > 0.0f ? 1.0f / denominator : 0.0f;
  const float4 value = make_float4(numerator.x * inverse, numerator.y * inverse, numerator.z * inverse, numerator.w * inverse);
  const uint64_t at = (uint64_t(l) * kHeads + head) * (RK_VERIFY_CHUNK_STRIDE * kG * kD) + query_head * kD + 4 * quad;
  *reinterpret_cast<uint2 *>(output + at) = make_uint2(uint32_t(float_to_bf16_bits(value.x)) | uint32_t(float_to_bf16_bits(value.y)) << 16,
                                                       uint32_t(float_to_bf16_bits(value.z)) | uint32_t(float_to_bf16_bits(value.w)) << 16);
  if (output_f32) *reinterpret_cast<float4 *>(output_f32 + at) = value;
}

template <uint32_t Format> constexpr size_t prefix_shared_bytes() { return 1024 + tile_bytes<Format>() + sizeof(Control) + sizeof(PlanShared); }
static_assert(prefix_shared_bytes<RK_FORMAT_INT4>() <= 227 * 1024 && prefix_shared_bytes<RK_FORMAT_INT8>() <= 227 * 1024 &&
              prefix_shared_bytes<RK_FORMAT_BF16>() <= 227 * 1024, "the tiles fit one SM");

template <typename Kernel, typename... Args>
int launch_dependent(Kernel kernel, dim3 grid, uint32_t threads, size_t shared_bytes, cudaStream_t stream, const char *what, Args... args) {
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = shared_bytes;
  config.stream = stream;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&config, kernel, args...), what);
}

template <uint32_t Format> int launch_prefix(const Window *w, uint32_t ctas, const PrefixArgs &args, bool shaped, cudaStream_t s) {
  constexpr size_t bytes = prefix_shared_bytes<Format>();
  const CUtensorMap &map = Format == RK_FORMAT_INT4 ? w->int4_head_map : Format == RK_FORMAT_BF16 ? w->int4_map : w->byte_head_map;
  auto launch = [&](auto kernel) -> int {
    if (int st = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)), "prefix kernel shared memory")) return st;
    return launch_dependent(kernel, dim3(ctas), kThreads, bytes, s, "prefix kernel launch", map, args);
  };
  return shaped ? launch(shared_prefix_kernel<Format, true>) : launch(shared_prefix_kernel<Format, false>);
}

} // namespace
} // namespace rk

using namespace rk;

extern "C" {

int rk_shared_plan_make(uint32_t format, uint32_t kv_heads, uint32_t query_heads, uint32_t head_dim, uint32_t lanes, uint32_t ctas,
                        rk_shared_plan *plan) {
  if (!plan) { set_error("rk_shared_plan_make: no plan"); return kInvalid; }
  if (int st = rk_decode_plan_make(format, kv_heads, query_heads, head_dim, lanes, ctas, &plan->decode)) return st;
  plan->prefix_ctas = plan->decode.ctas;
  plan->reserved = 0;
  // split launches have at most one item of 128 rows per CTA; otherwise every row has one partial
  const uint64_t rows = plan->prefix_ctas * uint64_t(kM) > lanes * uint64_t(kHeads * kG) ? plan->prefix_ctas * uint64_t(kM) : lanes * uint64_t(kHeads * kG);
  plan->prefix_partials_bytes = rows * kD * sizeof(float);
  plan->prefix_statistics_bytes = rows * 2 * sizeof(float);
  plan->prefix_descriptor_bytes = lanes * 4ull * sizeof(uint32_t);
  return kOk;
}

int rk_attention_decode_shared(const void *window, const rk_shared_plan *plan, uint32_t format, const void *queries, void *output,
                               float *output_f32, const rk_shared_buffers *buffers, const rk_page_entry *const *tables,
                               const rk_verify_params *lane_params, rk_kv_layer layer, const uint32_t *lane_groups,
                               const uint32_t *group_pages, const rk_score_shape *shape, void *stream) {
  const auto *w = static_cast<const Window *>(window);
  ShapeArgs shape_args;
  if (!w || !plan || !plan->decode.lanes || plan->decode.lanes > kMaxLanes || !plan->prefix_ctas || !queries || !output || !buffers ||
      !buffers->partials || !buffers->statistics || !buffers->descriptors || !buffers->prefix_partials || !buffers->prefix_statistics ||
      !buffers->prefix_descriptors || !tables || !lane_params || !layer.extent_pages || !lane_groups || !group_pages ||
      !rk_format_valid(format) || !shape_arguments(shape, shape_args)) {
    set_error("rk_attention_decode_shared: invalid arguments");
    return kInvalid;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uint32_t lanes = plan->decode.lanes;
  const PrefixArgs args{static_cast<const uint16_t *>(queries), buffers->prefix_partials, buffers->prefix_statistics, buffers->prefix_descriptors,
                        tables, lane_params, layer, w->base, lanes, buffers->descriptors + 2 * lanes, kSpinLimit, lane_groups, group_pages, shape_args};
  const bool shaped = shape_args.cap > 0.0f || shape_args.window || shape_args.slopes;
  int st = kOk;
  switch (format) {
  case RK_FORMAT_INT4: st = launch_prefix<RK_FORMAT_INT4>(w, plan->prefix_ctas, args, shaped, s); break;
  case RK_FORMAT_INT8: st = launch_prefix<RK_FORMAT_INT8>(w, plan->prefix_ctas, args, shaped, s); break;
  case RK_FORMAT_FP8E4M3: st = launch_prefix<RK_FORMAT_FP8E4M3>(w, plan->prefix_ctas, args, shaped, s); break;
  default: st = launch_prefix<RK_FORMAT_BF16>(w, plan->prefix_ctas, args, shaped, s); break;
  }
  if (st) return st;
  if ((st = launch_decode_suffix(format, plan->decode, s, w, queries, buffers->partials, buffers->statistics, buffers->descriptors, tables,
                                 lane_params, layer, shape_args, lane_groups, group_pages)))
    return st;
  auto merge = [&](auto kernel, uint32_t rows, uint32_t groups) {
    return launch_dependent(kernel, dim3(kG / rows, kHeads, lanes), 64 * groups * rows, 0, s, "shared merge launch", buffers->partials,
                            buffers->statistics, buffers->descriptors, buffers->prefix_partials, buffers->prefix_statistics,
                            reinterpret_cast<const uint4 *>(buffers->prefix_descriptors), static_cast<uint16_t *>(output), output_f32, lane_params);
  };
  // few lanes have many slots each: their blocks spread the slots; many lanes have few, and a block per (lane, KV head)
  if (lanes * kHeads * kG <= 148) return merge(shared_merge_kernel<16, 1>, 1, 16);
  if (lanes * kHeads * kG <= 8 * 148) return merge(shared_merge_kernel<4, 1>, 1, 4);
  return merge(shared_merge_kernel<1, 6>, 6, 1);
}

} // extern "C"
