// shared_prefix.cu — decode attention for a batch in which groups of lanes share the first pages of their tables.
//
// With attention over a context split into a prefix and a rest, a lane's output is the merge of two partials
// {max, sum of exp, sum of exp * v}. The rest is the streaming kernel's business (decode_attention.cu, which leaves the
// shared pages out). The prefix part is the same keys and values for every lane of a group, so its query rows, 6 per lane
// and KV head, stand side by side as the M side of a tensor-core tile: pages are read once per tile, not once per lane,
// and a group of n lanes turns 6 multiply-adds per key element into 6 n.
//
// The kernel is the row-tile kernel (row_tile.cuh) with rows gathered from many lanes. Measured, streaming kernel and merge
// included: int4, 256 lanes over one 32K prefix 272 us (770 TFLOP/s; 1 364 us lane by lane), 32 over 8K 52 us (61), four over
// 2K tokens of int8 25 us (20): three launches cost more than four short lanes' pages do. A tile takes the same time however many of
// its rows are real, so small groups lose at any length (32 groups of four over 8K, int4: 176 us, 148 lane by lane); session.py has
// the rule.
#include "common.cuh"
#include "decode_partials.cuh"
#include "row_tile.cuh"
#include "score_shape.cuh"

namespace rk {
using namespace tile;
namespace {

constexpr uint32_t kMaxLanes = 1024;
constexpr uint32_t kNone = 0xffffu;
constexpr uint32_t kTileLanes = 24;   // lanes with a row in a 128-row tile: at most 23
static_assert(kTileLanes == sizeof(RowItem::lanes) / sizeof(uint16_t), "an item names its tile's lanes");

struct PrefixArgs : RowTileArgs { // partials [row][256], statistics [row]{max, sum}, rows as the lanes' descriptors say
  uint32_t *descriptors; // [lane]{row of head 0 and split 0, splits, rows of the group, -}
  const rk_page_entry *const *tables;
  const rk_verify_params *lane_params;
  uint32_t lanes;
  const uint32_t *lane_groups, *group_pages;
};

// A group with work: its number, members and pages, the lowest member's lane (whose table the tiles read), and the smallest
// position of its rows, whose window begins first.
struct GroupWork {
  uint16_t group, members, pages, leader;
  uint32_t nearest;
  __device__ __forceinline__ uint32_t last_position() const { return pages * kPageTokens - 1; }
  // the pages of the prefix that some row sees
  __device__ __forceinline__ PageList list(const ShapeArgs &shape) const { return PageList::make(nearest, last_position(), 0, shape); }
};

struct PlanShared {
  uint16_t member_of[kMaxLanes];  // a lane's group, kNone: none
  union {
    struct {
      uint32_t count[kMaxLanes];  // members of a group
      uint32_t leader[kMaxLanes]; // its lowest member
      uint32_t nearest[kMaxLanes]; // its smallest position
    };
    GroupWork list[kMaxLanes];    // then: the groups with work, by leader
  };
  uint32_t words[kMaxLanes / 32]; // lanes as bits: the leaders
  uint32_t groups, chunk, item_count; // groups with work; most 64-token groups of a split; items of the launch
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
// which (KV heads x tiles x splits) of all groups still fit the grid. It goes down to one 64-token group: a longer chain of
// groups costs more than the partials that the merge reads (four lanes over 2K tokens: 25 us, and 29 with four groups at
// least). With more tiles than CTAs every tile is one item and the CTAs take them in turn.
__device__ __noinline__ void plan_launch(const PrefixArgs &args, PlanShared &sh) {
  const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32, lanes = args.lanes, words = (lanes + 31) / 32;
  constexpr uint32_t kRounds = (kMaxLanes + kRowTileThreads - 1) / kRowTileThreads; // warps take whole words: lane i of round r is tid + r * kRowTileThreads
  for (uint32_t i = tid; i < lanes; i += kRowTileThreads) { sh.count[i] = 0; sh.leader[i] = kMaxLanes; sh.nearest[i] = ~0u; }
  __syncthreads();
  uint32_t group[kRounds], pages[kRounds]; // of this thread's lanes
#pragma unroll
  for (uint32_t r = 0; r < kRounds; ++r) {
    const uint32_t i = tid + r * kRowTileThreads;
    group[r] = kNone;
    if (i / 32 >= words) continue; // the whole warp
    if (i < lanes) {
      const uint32_t g = args.lane_groups[i];
      const rk_verify_params p = args.lane_params[i];
      const uint32_t shared = g < lanes ? args.group_pages[g] : 0;
      if (shared && lane_takes_part(p)) {
        group[r] = g;
        pages[r] = min(shared, rk_pages_for(p.committed_tokens + 1));
        if (args.shape.window) atomicMin(&sh.nearest[g], p.committed_tokens);
      }
      sh.member_of[i] = uint16_t(group[r]);
    }
    // one pair of atomics per group and warp: every lane on one word would be a queue of 32
    const uint32_t peers = __match_any_sync(0xffffffffu, group[r]);
    if (group[r] != kNone && lane == uint32_t(__ffs(peers) - 1)) {
      atomicAdd(&sh.count[group[r]], uint32_t(__popc(peers)));
      atomicMin(&sh.leader[group[r]], i);
    }
  }
  __syncthreads();
  uint32_t members[kRounds], nearest[kRounds];
#pragma unroll
  for (uint32_t r = 0; r < kRounds; ++r) {
    const uint32_t i = tid + r * kRowTileThreads;
    if (i / 32 >= words) continue; // the whole warp
    members[r] = group[r] != kNone ? sh.count[group[r]] : 0;
    nearest[r] = group[r] != kNone ? sh.nearest[group[r]] : 0;
    const uint32_t mask = __ballot_sync(0xffffffffu, group[r] != kNone && sh.leader[group[r]] == i);
    if (lane == 0) sh.words[i / 32] = mask;
  }
  __syncthreads();
#pragma unroll
  for (uint32_t r = 0; r < kRounds; ++r) {
    const uint32_t i = tid + r * kRowTileThreads;
    if (i / 32 >= words) continue;
    const uint32_t mask = sh.words[i / 32], at = bits_before(sh.words, i / 32) + __popc(mask & ((1u << lane) - 1u));
    if (mask >> lane & 1u) sh.list[at] = GroupWork{uint16_t(group[r]), uint16_t(members[r]), uint16_t(pages[r]), uint16_t(i), nearest[r]};
    if (i / 32 + 1 == words && lane == 31) sh.groups = at + (mask >> 31);
  }
  __syncthreads();
  if (warp == 0) {
    const uint32_t groups = sh.groups;
    uint32_t units = 0, tiles = 0; // of all groups, times the KV heads
    for (uint32_t i = lane; i < groups; i += 32) {
      const uint32_t t = kHeads * tiles_of(sh.list[i].members);
      tiles += t;
      units += t * units_of(sh.list[i].list(args.shape).count);
    }
    units = __reduce_add_sync(0xffffffffu, units);
    tiles = __reduce_add_sync(0xffffffffu, tiles);
    auto items_for = [&](uint32_t chunk) {
      uint32_t sum = 0;
      for (uint32_t i = lane; i < groups; i += 32)
        sum += kHeads * tiles_of(sh.list[i].members) * ((units_of(sh.list[i].list(args.shape).count) + chunk - 1) / chunk);
      return __reduce_add_sync(0xffffffffu, sum);
    };
    // items(chunk) <= units / chunk + tiles, and >= units / chunk: the shortest chunk that fits lies between these two
    uint32_t high = units_of(rk_pages_for(RK_MAX_PHYSICAL_TOKENS));
    if (tiles < gridDim.x) {
      high = units / (gridDim.x - tiles) + 1;
      uint32_t low = max(1u, (units + gridDim.x - 1) / gridDim.x);
      while (low < high) {
        const uint32_t middle = (low + high) / 2;
        if (items_for(middle) <= gridDim.x) high = middle; else low = middle + 1;
      }
    }
    const uint32_t items = items_for(high);
    if (lane == 0) { sh.chunk = high; sh.item_count = items; }
  }
  __syncthreads();
}

// place = {tile, split, splits, rows of the group, row of (head 0, split 0, the group's first row), the tile's first member,
// group}.
struct PrefixPlacement : PlanShared {
  using Args = PrefixArgs;
  // The partition reads only the lanes' parameter blocks and groups, which no kernel that lets a dependent start early writes.
  __device__ void prepare(const Args &args) { plan_launch(args, *this); }
  __device__ void begin(const Args &args) {
    if (blockIdx.x == 0)
      for (uint32_t i = threadIdx.x; i < args.lanes; i += kRowTileThreads)
        if (member_of[i] == kNone) reinterpret_cast<uint4 *>(args.descriptors)[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ uint32_t items(const Args &) const { return item_count; }
  // Item number `index` of the launch and the lanes of its tile; the whole warp.
  __device__ void plan(const Args &args, uint32_t index, RowItem &item) {
    const uint32_t lane = threadIdx.x % 32, lanes = args.lanes;
    uint32_t before = 0, rows = 0;
    for (uint32_t base = 0; base < groups; base += 32) {
      const bool live = base + lane < groups;
      const GroupWork work = live ? list[base + lane] : GroupWork{0, 0, 1, 0, 0};
      const PageList pages = work.list(args.shape);
      const uint32_t units = units_of(pages.count), splits = (units + chunk - 1) / chunk, tiles = tiles_of(work.members);
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
          const uint32_t within = index - (before + items_up - items), split = within / kHeads / tiles, tile = within / kHeads % tiles;
          item.head = within % kHeads;
          item.ordinal_begin = 2 * (units * split / splits);
          item.ordinal_end = min(pages.count, 2 * (units * (split + 1) / splits));
          item.list = pages;
          item.last_position = work.last_position();
          item.table = args.tables[work.leader];
          item.place[0] = tile;
          item.place[1] = split;
          item.place[2] = splits;
          item.place[3] = group_rows;
          item.place[4] = rows + rows_up - kHeads * splits * group_rows;
          item.place[5] = tile * kM / kG;
          item.place[6] = work.group;
        }
        break;
      }
      before += __shfl_sync(0xffffffffu, items_up, 31);
      rows += __shfl_sync(0xffffffffu, rows_up, 31);
    }
    if (lane < kTileLanes) item.lanes[lane] = kMaxLanes;
    __syncwarp();
    const uint32_t group = item.place[6], first_member = item.place[5], first_row = item.place[0] * kM;
    for (uint32_t base = 0, rank = 0; base < lanes && rank < first_member + kTileLanes; base += 32) {
      const bool member = base + lane < lanes && member_of[base + lane] == group;
      const uint32_t mask = __ballot_sync(0xffffffffu, member), mine = rank + __popc(mask & ((1u << lane) - 1u));
      if (member && mine >= first_member && mine < first_member + kTileLanes) {
        item.lanes[mine - first_member] = uint16_t(base + lane);
        // the tile that holds a lane's first row writes its descriptor
        if (item.head == 0 && item.place[1] == 0 && mine * kG >= first_row && mine * kG < first_row + kM)
          reinterpret_cast<uint4 *>(args.descriptors)[base + lane] = make_uint4(item.place[4] + mine * kG, item.place[2], item.place[3], 0);
      }
      rank += __popc(mask);
    }
    __syncwarp();
  }
  __device__ RowPlace row(const Args &args, const RowItem &item, uint32_t r) const {
    RowPlace place;
    const uint32_t fused = item.place[0] * kM + r; // row of the group
    place.real = fused < item.place[3];
    const uint32_t lane = place.real ? item.lanes[fused / kG - item.place[5]] : item.lanes[0];
    const rk_verify_params p = args.lane_params[lane];
    place.head_row = fused % kG;
    place.position = place.real ? p.committed_tokens : item.last_position; // a row without a lane: what it sees is of no interest
    place.score_scale = p.score_scale;
    place.query = args.queries + ((uint64_t(lane) * kHeads + item.head) * (RK_VERIFY_CHUNK_STRIDE * kG) + place.head_row) * kD;
    place.slot = item.place[4] + uint64_t(item.head * item.place[2] + item.place[1]) * item.place[3] + fused;
    return place;
  }
  __device__ void empty(const Args &, const RowItem &, uint32_t) const {}
};

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
  constexpr uint32_t kBatch = kGroups == 4 ? 8 : 4; // slots of a thread in flight: what the registers of its block size allow
  __shared__ float4 sums[kRows][kGroups][kD / 4];
  __shared__ float2 stats[kRows][kGroups];
  const uint32_t head = blockIdx.y, l = blockIdx.z, tid = threadIdx.x, quad = tid & 63u, group = tid / 64 % kGroups, row = tid / (64 * kGroups);
  const uint32_t query_head = blockIdx.x * kRows + row;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory"); // the row tiles, whose blocks all waited for the streaming kernel
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
  // as the other merges: a row without a positive sum (nothing seen, or no number) is zeros
  const float4 value = denominator > 0.0f ? make_float4(numerator.x / denominator, numerator.y / denominator, numerator.z / denominator, numerator.w / denominator)
                                          : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  const uint64_t at = (uint64_t(l) * kHeads + head) * (RK_VERIFY_CHUNK_STRIDE * kG * kD) + query_head * kD + 4 * quad;
  *reinterpret_cast<uint2 *>(output + at) = make_uint2(uint32_t(float_to_bf16_bits(value.x)) | uint32_t(float_to_bf16_bits(value.y)) << 16,
                                                       uint32_t(float_to_bf16_bits(value.z)) | uint32_t(float_to_bf16_bits(value.w)) << 16);
  if (output_f32) *reinterpret_cast<float4 *>(output_f32 + at) = value;
}

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
  if (!aligned_to(16, queries, output_f32, buffers->partials, buffers->prefix_partials, buffers->prefix_descriptors) ||
      !aligned_to(8, output, buffers->statistics, buffers->descriptors, buffers->prefix_statistics, tables)) {
    set_error("rk_attention_decode_shared: queries, partials, fp32 rows and prefix descriptors start on 16-byte boundaries, the rest on 8-byte ones");
    return kInvalid;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uint32_t lanes = plan->decode.lanes;
  const PrefixArgs args{{static_cast<const uint16_t *>(queries), buffers->prefix_partials, buffers->prefix_statistics, layer, w->base,
                         buffers->descriptors + 2 * lanes, kSpinLimit, shape_args},
                        buffers->prefix_descriptors, tables, lane_params, lanes, lane_groups, group_pages};
  // The streaming kernel goes first: it leaves its SMs one by one, and the longer prologue of the row tiles (the plan, tensor
  // memory) runs beside its tail. Neither needs the other; the merge waits for the second, whose blocks all waited for the first.
  if (int st = launch_decode_suffix(format, plan->decode, s, w, queries, buffers->partials, buffers->statistics, buffers->descriptors, tables,
                                    lane_params, layer, shape_args, lane_groups, group_pages))
    return st;
  if (int st = launch_row_tile<PrefixPlacement>(format, w, plan->prefix_ctas, args, s)) return st;
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
