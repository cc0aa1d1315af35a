// shaped_attention.cu — verify windows and prefill tiles with a score shape (rk_score_shape) on the row-tile kernel.
//
// Scratch, slots and merges are those of the plain entries (rk_attention_verify_split_tc, rk_attention_prefill_split_tc);
// what differs is that a tile walks the list of pages that one of its rows sees and that every score passes the shape. Its
// merges count the splits that exist from the whole context, so the listed pages are dealt to that many, in whole 64-token
// groups, and a split that gets none leaves an empty partial.
//
// Measured: four lanes of 16 rows over 32K int4 tokens with a soft cap 112 us with the merge (86 with an empty shape, 83 on
// the plain window kernel, which needs no plan); 2 048 int8 rows behind 6K with a window of 4 096 and slopes 362 us, of
// which the merge is 24 (with an empty shape 484 us; the plain prefill kernel takes 564 for the same rows).
#include "row_tile.cuh"

#include <atomic>
#include <string>

namespace rk {
using namespace tile;
namespace {

// The run of a tile's page list that one split takes.
__device__ __forceinline__ bool split_list(RowItem &item, uint32_t first_position, uint32_t last_position, uint32_t splits, uint32_t split, const ShapeArgs &shape) {
  const uint32_t pages = last_position / kPageTokens + 1, per_split = rk_pages_per_split(pages, splits), written = (pages + per_split - 1) / per_split;
  item.ordinal_begin = item.ordinal_end = 0;
  if (split >= written) return false; // the merge does not look at it
  item.list = PageList::make(first_position, last_position, 0, shape);
  item.last_position = last_position;
  const uint32_t share = ((item.list.count + written - 1) / written + 1) & ~1u;
  item.ordinal_begin = min(item.list.count, split * share);
  item.ordinal_end = min(item.list.count, item.ordinal_begin + share);
  return true;
}
__device__ __forceinline__ void clear_slot(const RowTileArgs &args, uint64_t first_row, uint32_t rows, uint32_t tid) {
  for (uint32_t i = tid; i < rows * (kD / 4); i += kSoftmaxThreads) reinterpret_cast<float4 *>(args.partials)[first_row * (kD / 4) + i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (uint32_t i = tid; i < rows; i += kSoftmaxThreads) reinterpret_cast<float2 *>(args.statistics)[first_row + i] = make_float2(-INFINITY, 0.0f);
}

// A lane's window of up to 16 rows: place = {lane, capacity rows of a slot, slot, committed, active rows, score scale, empty}.
struct VerifyPlacement {
  struct Args : RowTileArgs {
    const rk_page_entry *const *tables;
    const rk_verify_params *lane_params;
    uint32_t lanes, splits, capacity;
  };
  __device__ void prepare(const Args &) { __syncthreads(); }
  __device__ void begin(const Args &) {}
  __device__ uint32_t items(const Args &args) const { return kHeads * args.splits * args.lanes; }
  __device__ void plan(const Args &args, uint32_t index, RowItem &item) {
    if (threadIdx.x % 32) return;
    const uint32_t lane_index = index / (kHeads * args.splits), split = index / kHeads % args.splits;
    item.head = index % kHeads;
    rk_verify_params p = args.lane_params[lane_index];
    p.kv = args.layer;
    item.ordinal_begin = item.ordinal_end = 0;
    item.place[6] = 0;
    if (!rk_verify_contract_valid(&p) || p.row_capacity != args.capacity || split >= p.split_count) return;
    item.table = args.tables[lane_index];
    item.place[0] = lane_index;
    item.place[2] = (lane_index * kHeads + item.head) * p.slot_splits + split;
    item.place[3] = p.committed_tokens;
    item.place[4] = p.active_rows;
    item.place[5] = __float_as_uint(p.score_scale);
    item.place[6] = split_list(item, p.committed_tokens, p.committed_tokens + p.active_rows - 1, p.split_count, split, args.shape);
  }
  __device__ RowPlace row(const Args &args, const RowItem &item, uint32_t r) const {
    RowPlace place;
    const uint32_t query_row = r / kG;
    place.real = query_row < item.place[4];
    place.head_row = r % kG;
    place.position = item.place[3] + min(query_row, item.place[4] - 1);
    place.score_scale = __uint_as_float(item.place[5]);
    place.query = args.queries + ((uint64_t(item.place[0]) * kHeads + item.head) * (RK_VERIFY_CHUNK_STRIDE * kG) + r) * kD;
    place.slot = uint64_t(item.place[2]) * (args.capacity * kG) + r;
    return place;
  }
  __device__ void empty(const Args &args, const RowItem &item, uint32_t tid) const {
    if (item.place[6]) clear_slot(args, uint64_t(item.place[2]) * (args.capacity * kG), args.capacity * kG, tid);
  }
};

// Consecutive rows of a prefill chunk. An unsplit plan packs 21 rows x 6 query heads into the tile's 128 (126); a split plan
// takes the merge's tiles of eight rows (48 of 128), whose splits follow from each tile's own context: for chunks too short to
// fill the GPU otherwise. The partials keep the merge's slots of eight rows either way. Tiles go from the last, whose context is the longest, to the first.
constexpr uint32_t kPackedRows = kM / kG;
struct PrefillPlacement {
  struct Args : RowTileArgs {
    const rk_page_entry *table;
    rk_prefill_params params;
    uint32_t rows, tiles; // rows of a tile; tiles of the chunk
  };
  __device__ void prepare(const Args &) { __syncthreads(); }
  __device__ void begin(const Args &) {}
  __device__ uint32_t items(const Args &args) const { return kHeads * args.params.split_count * args.tiles; }
  __device__ void plan(const Args &args, uint32_t index, RowItem &item) {
    if (threadIdx.x % 32) return;
    const uint32_t splits = args.params.split_count, start = (args.tiles - 1 - index / (kHeads * splits)) * args.rows;
    const uint32_t rows = min(args.rows, args.params.rows - start), split = index / kHeads % splits;
    item.head = index % kHeads;
    item.table = args.table;
    item.place[0] = start;
    item.place[1] = rows;
    item.place[2] = split;
    item.place[6] = split_list(item, args.params.committed_tokens + start, args.params.committed_tokens + start + rows - 1, splits, split, args.shape);
  }
  __device__ uint64_t slot(const Args &args, const RowItem &item, uint32_t row) const { // of the chunk's row `row`, its first query head
    const uint32_t merge_tile = row / RK_PREFILL_TILE_ROWS;
    return ((uint64_t(merge_tile) * kHeads + item.head) * args.params.split_count + item.place[2]) * (RK_PREFILL_TILE_ROWS * kG) + row % RK_PREFILL_TILE_ROWS * kG;
  }
  __device__ RowPlace row(const Args &args, const RowItem &item, uint32_t r) const {
    RowPlace place;
    const uint32_t within = r / kG, row = item.place[0] + within;
    place.real = within < item.place[1];
    place.head_row = r % kG;
    place.position = args.params.committed_tokens + item.place[0] + min(within, item.place[1] - 1);
    place.score_scale = args.params.score_scale;
    place.query = args.queries + ((uint64_t(item.head) * args.params.chunk_stride + row) * kG + place.head_row) * kD;
    place.slot = slot(args, item, row) + place.head_row;
    return place;
  }
  __device__ void empty(const Args &args, const RowItem &item, uint32_t tid) const {
    if (item.place[6]) clear_slot(args, slot(args, item, item.place[0]), RK_PREFILL_TILE_ROWS * kG, tid);
  }
};

int common_arguments(const char *what, const void *window, uint32_t format, uint32_t kv_heads, uint32_t query_heads, uint32_t head_dim,
                     const rk_score_shape *shape, ShapeArgs &shape_args) {
  if (kv_heads != kHeads || query_heads != kHeads * kG || head_dim != kD || !rk_format_valid(format)) {
    set_error((std::string(what) + ": built for 4 KV heads x 24 query heads x 256").c_str());
    return kUnsupported;
  }
  if (!window || !shape || !shape_arguments(shape, shape_args)) {
    set_error((std::string(what) + ": no window, or an invalid shape").c_str());
    return kInvalid;
  }
  return kOk;
}

} // namespace

// CTAs of a persistent launch: one per SM of the current device, no more than there are items.
int tile::persistent_ctas(uint64_t items, uint32_t &ctas) {
  static std::atomic<uint32_t> counts[64] = {}; // per device; written twice at worst, with the same value
  int device = 0;
  if (int st = cuda_status(cudaGetDevice(&device), "cudaGetDevice")) return st;
  if (device < 0 || device >= 64) { set_error("device index out of range"); return kInvalid; }
  uint32_t sms = counts[device].load(std::memory_order_relaxed);
  if (!sms) {
    int count = 0;
    if (int st = cuda_status(cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device), "SM count")) return st;
    counts[device].store(sms = uint32_t(count), std::memory_order_relaxed);
  }
  ctas = uint32_t(items < sms ? items : sms);
  return kOk;
}

} // namespace rk

using namespace rk;

static int verify_split_shaped(const char *what, const void *window, uint32_t format, uint32_t kv_heads, uint32_t query_heads,
                               uint32_t head_dim, uint32_t lanes, uint32_t row_capacity, uint32_t grid_splits, const void *queries,
                               float *partials, float *statistics, const rk_page_entry *const *tables, const rk_verify_params *lane_params,
                               rk_kv_layer layer, const rk_score_shape *shape, uint32_t *status, uint32_t most_ctas, uint32_t spin_limit,
                               uint32_t withheld_groups, void *stream) {
  ShapeArgs shape_args;
  if (int st = common_arguments(what, window, format, kv_heads, query_heads, head_dim, shape, shape_args)) return st;
  if (row_capacity != 8 && row_capacity != 16) {
    set_error((std::string(what) + ": row capacity 8 or 16; one row takes rk_attention_decode_shaped").c_str());
    return kUnsupported;
  }
  if (!lanes || lanes > 65535 || !grid_splits || grid_splits > RK_VERIFY_MAX_SPLITS || !queries || !partials || !statistics || !tables || !lane_params ||
      !layer.extent_pages || !status) {
    set_error((std::string(what) + ": invalid arguments").c_str());
    return kInvalid;
  }
  if (!aligned_to(16, queries, partials) || !aligned_to(8, statistics, tables)) {
    set_error((std::string(what) + ": queries and partials start on 16-byte boundaries, statistics and tables on 8-byte ones").c_str());
    return kInvalid;
  }
  const auto *w = static_cast<const Window *>(window);
  VerifyPlacement::Args args{{static_cast<const uint16_t *>(queries), partials, statistics, layer, w->base, status, spin_limit, shape_args,
                              withheld_groups},
                             tables, lane_params, lanes, grid_splits, row_capacity};
  uint32_t ctas = 0;
  if (int st = persistent_ctas(uint64_t(kHeads) * grid_splits * lanes, ctas)) return st;
  return launch_row_tile<VerifyPlacement>(format, w, ctas < most_ctas ? ctas : most_ctas, args, static_cast<cudaStream_t>(stream));
}

extern "C" int rk_attention_verify_split_shaped(const void *window, uint32_t format, uint32_t kv_heads, uint32_t query_heads,
                                                uint32_t head_dim, uint32_t lanes, uint32_t row_capacity, uint32_t grid_splits,
                                                const void *queries, float *partials, float *statistics,
                                                const rk_page_entry *const *tables, const rk_verify_params *lane_params,
                                                rk_kv_layer layer, const rk_score_shape *shape, uint32_t *status, void *stream) {
  return verify_split_shaped("rk_attention_verify_split_shaped", window, format, kv_heads, query_heads, head_dim, lanes, row_capacity, grid_splits,
                             queries, partials, statistics, tables, lane_params, layer, shape, status, ~0u, kSpinLimit, 0, stream);
}

// Test hook of the row-tile kernel's timeout path: the same launch on at most `ctas` CTAs with waits that give up after
// `spin_limit` polls and a TMA warp that streams nothing more from the last `withheld_groups` 64-token groups of its first item
// on. Every later wait of the CTA gives up at once, the copies under way land, tensor memory is released, `status` turns
// non-zero and the kernel returns; nothing faults and no wait is unbounded. The step's output is invalid.
extern "C" int rk_attention_shaped_probe_timeout(const void *window, uint32_t format, uint32_t kv_heads, uint32_t query_heads,
                                                 uint32_t head_dim, uint32_t lanes, uint32_t row_capacity, uint32_t grid_splits,
                                                 const void *queries, float *partials, float *statistics,
                                                 const rk_page_entry *const *tables, const rk_verify_params *lane_params,
                                                 rk_kv_layer layer, const rk_score_shape *shape, uint32_t *status, uint32_t ctas,
                                                 uint32_t spin_limit, uint32_t withheld_groups, void *stream) {
  if (!ctas || !spin_limit || spin_limit > kSpinLimit || withheld_groups > rk_pages_for(RK_MAX_PHYSICAL_TOKENS)) {
    set_error("rk_attention_shaped_probe_timeout: CTAs, spin limit or withheld groups out of range");
    return kInvalid;
  }
  return verify_split_shaped("rk_attention_shaped_probe_timeout", window, format, kv_heads, query_heads, head_dim, lanes, row_capacity, grid_splits,
                             queries, partials, statistics, tables, lane_params, layer, shape, status, ctas, spin_limit, withheld_groups, stream);
}

extern "C" int rk_attention_prefill_split_shaped(const void *window, uint32_t format, uint32_t kv_heads, uint32_t query_heads,
                                                 uint32_t head_dim, const void *queries, float *partials, float *statistics,
                                                 const rk_page_entry *table, const rk_prefill_params *params,
                                                 const rk_score_shape *shape, uint32_t *status, void *stream) {
  ShapeArgs shape_args;
  if (int st = common_arguments("rk_attention_prefill_split_shaped", window, format, kv_heads, query_heads, head_dim, shape, shape_args)) return st;
  if (!queries || !partials || !statistics || !table || !params || !status || !rk_prefill_contract_valid(params)) {
    set_error("rk_attention_prefill_split_shaped: invalid arguments");
    return kInvalid;
  }
  if (!aligned_to(16, queries, partials) || !aligned_to(8, statistics, table)) {
    set_error("rk_attention_prefill_split_shaped: queries and partials start on 16-byte boundaries, statistics and tables on 8-byte ones");
    return kInvalid;
  }
  const auto *w = static_cast<const Window *>(window);
  const uint32_t rows = params->split_count == 1 ? kPackedRows : RK_PREFILL_TILE_ROWS;
  PrefillPlacement::Args args{{static_cast<const uint16_t *>(queries), partials, statistics, params->kv, w->base, status, kSpinLimit, shape_args},
                              table, *params, rows, (params->rows + rows - 1) / rows};
  uint32_t ctas = 0;
  if (int st = persistent_ctas(uint64_t(kHeads) * params->split_count * args.tiles, ctas)) return st;
  return launch_row_tile<PrefillPlacement>(format, w, ctas, args, static_cast<cudaStream_t>(stream));
}
