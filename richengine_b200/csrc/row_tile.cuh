// row_tile.cuh — attention of up to 128 query rows against one run of pages, as a tcgen05 contraction; the kernel of the
// shaped windows and prefill tiles (shaped_attention.cu) and of shared prefixes (shared_prefix.cu), which differ in where the
// rows come from, which pages they meet and where the partials go (Placement).
//
//   S = Q.K^T (16 x M128 N64 K16)       w = 2^(shape(s) + log2 vscale - reference)        O += w.V (4 x M128 N256 K16)
//
// The pipeline is the window kernel's (verify_attention.cu). A block is persistent over items (a tile of rows, one KV head, a
// run of 64-token groups) and holds 28 warps:
//   warps 0-15        softmax: four threads per row (= lane of tensor memory), 16 scores each
//   warps 16-23       raw codes -> 16-bit operand tiles (Expand, window_tile.cuh)
//   warp 24           TMA: pages into the raw ring;  warps 25, 26: issue of the two contractions
//   warp 27           the plan: descriptions of the CTA's items, up to eight at a time
// Tensor memory (512 columns): O 256, two score buffers of 64 (a group's weights overwrite the first half of its scores; of
// bf16, a low part of each weight the second), the query tile 128.
//
// What bounds it: a 64-token group of int4 takes about 2 400 cycles, of which the matrix unit is busy 1 024 (the two
// contractions at M128), the schedulers 1 450 (61 % of all issue slots: softmax of 128 x 64 scores, expansion of 32 K codes)
// and shared memory about 2 100 (1 450 wavefronts of loads and stores, half of them scales that every row's thread reads, 128
// of the copies in, 512 of the matrix unit's operand reads). Work left out in a copy: without the softmax the 256-lane prefix
// takes 188 us instead of 222, without the expansion 205, without either 157, without the scales' reads 205: several limits
// lie close together. What a shape adds to the softmax shows in full (a cap 26 us of 85, slopes 20 % of a prefill chunk), for the rows
// that do not exist too: the softmax warps work on all 128, of which a 16-row window fills 96 and an 8-row one 48.
// Sixteen softmax warps because eight were latency bound (a group's chain of load, maximum,
// weights and store is shorter with 16 scores a thread than with 32); two teams of eight that alternate between groups, and a
// single score buffer beside two of weights, were 4-6 % slower. Rates: 770 TFLOP/s for 256 lanes of int4, 460 for a 16-row
// window with a soft cap (96 of 128 rows), 570 for a prefill chunk of int8 with slopes and a window of 4 096.
#pragma once

#include "common.cuh"
#include "score_shape.cuh"
#include "window_tile.cuh"

namespace rk::tile {

constexpr uint32_t kRowTileThreads = 28 * 32;
constexpr uint32_t kExpanderThreads = 256;
constexpr uint32_t kCopyWarp = 24, kScoresWarp = 25, kOutputsWarp = 26, kPlanWarp = 27;
constexpr uint32_t kBatchItems = 8; // planned at a time; the roles meet between batches only
// One piece of work. Placement fills it; `place` is its own.
struct RowItem {
  uint32_t head, ordinal_begin, ordinal_end; // of the page list; equal: nothing to stream
  PageList list;
  uint32_t last_position;         // of the tile's rows: what lies behind it, or before the list's window, no row sees
  uint32_t place[8];
  uint16_t lanes[24];
  const rk_page_entry *table;
};
// A softmax thread's row.
struct RowPlace {
  bool real;
  const uint16_t *query;
  uint32_t position, head_row;    // head_row: query head within the KV head's group
  float score_scale;              // as rk_score_scale takes it
  uint64_t slot;                  // row of partials and statistics
};

struct RowTileShared {
  uint64_t raw_full[kMaxRawStages], raw_free[kMaxRawStages];
  uint64_t k_full[2], k_free[2], v_full[2], v_free[2], s_full[2], p_full[2], p_free[2];
  uint64_t query_full, output_free, drained[2];
  uint32_t tmem_base;
  uint32_t error;
  uint32_t spin_limit; // directly after `error`: barrier_wait reads it through the error pointer
  float exchange[2][kRowThreads][kM]; // a row's part maxima; at an item's ends its query magnitudes and sums, its weights' sums
  ScaleStage scales[kScaleStages];
  RowItem items[kBatchItems];
};

int persistent_ctas(uint64_t items, uint32_t &ctas); // shaped_attention.cu

struct RowTileArgs {
  const uint16_t *queries;
  float *partials, *statistics;
  rk_kv_layer layer;
  uint64_t window_base;
  uint32_t *status;
  uint32_t spin_limit;
  ShapeArgs shape;
  uint32_t withheld_groups = 0; // timeout probe only: from an item's last groups on, nothing more is streamed
};

// ---- a softmax thread's scores --------------------------------------------------------------------------------------------
// Adds slope * (token - the group's first token) to the scores and returns slope * (the group's first token - position).
template <bool kPermuted>
__device__ __forceinline__ float bias_scores(float (&scores)[kRowTokens], uint32_t part_token, float slope, const GroupView &view, uint32_t position) {
  const float gap = slope * float(int32_t(view.second - view.first - kPageTokens)); // zero unless the list skips pages between the two
#pragma unroll
  for (uint32_t i = 0; i < kRowTokens; ++i) scores[i] = fmaf(slope, float(local_token<kPermuted>(i)), scores[i]);
  float origin = slope * float(int32_t(view.first + part_token - position));
  if (!kPermuted && part_token >= kPageTokens) origin += gap;
  if (kPermuted && gap != 0.0f) {
#pragma unroll
    for (uint32_t i = 0; i < kRowTokens; ++i)
      if (local_token<kPermuted>(i) >= kPageTokens) scores[i] += gap;
  }
  return origin;
}
// Accumulators of contraction positions first_position .. + 15 to scores + log2(value scale), the unseen ones -infinity.
// part_token: what those positions add to local_token<...>(i) of the first sixteen. Of a bias -slope * (position - token), the
// part that these tokens have in common (by their page, which is one page or two neighbours) is returned, to be added by the
// caller once instead of sixteen times; the rest is one multiply-add by a constant per score.
template <bool kPermuted>
__device__ __forceinline__ float shape_scores(float (&scores)[kRowTokens], const ScaleStage &stage, uint32_t first_position, uint32_t part_token,
                                             float row_factor, float row_offset, const ShapeArgs &shape, float slope, const GroupView &view,
                                             uint32_t position) {
  if (shape.cap == 0.0f && !shape.slopes) { // one branch for the launch
    scale_scores(scores, stage, first_position, row_factor, row_offset);
    return 0.0f;
  }
  if (shape.cap == 0.0f) {
    scale_scores(scores, stage, first_position, row_factor, row_offset);
    return bias_scores<kPermuted>(scores, part_token, slope, view, position);
  }
  const float2 factor = make_float2(row_factor, row_factor), offset = make_float2(row_offset, row_offset);
  float2 logs[kRowTokens / 2];
#pragma unroll
  for (uint32_t i = 0; i < kRowTokens; i += 2) {
    const float4 pair = stage.pairs[(first_position + i) >> 1];
    const float2 s = mul_pair(fma_pair(make_float2(scores[i], scores[i + 1]), factor, offset), make_float2(pair.x, pair.y));
    scores[i] = s.x;
    scores[i + 1] = s.y;
    logs[i / 2] = make_float2(pair.z, pair.w);
  }
  soft_cap(scores, shape.cap, shape.cap_inverse);
#pragma unroll
  for (uint32_t i = 0; i < kRowTokens; i += 2) {
    const float2 s = add_pair(make_float2(scores[i], scores[i + 1]), logs[i / 2]);
    scores[i] = s.x;
    scores[i + 1] = s.y;
  }
  return shape.slopes ? bias_scores<kPermuted>(scores, part_token, slope, view, position) : 0.0f;
}
template <bool kPermuted>
__device__ __forceinline__ void mask_scores(float (&scores)[kRowTokens], uint32_t part_token, uint32_t seen_first, uint32_t seen_second, float unseen) {
  const uint32_t mine = part_token < kPageTokens ? seen_first : seen_second;
#pragma unroll
  for (uint32_t i = 0; i < kRowTokens; ++i) {
    const uint32_t bits = kPermuted ? (local_token<kPermuted>(i) < kPageTokens ? seen_first : seen_second) : mine;
    if (!((bits >> ((local_token<kPermuted>(i) + part_token) & 31u)) & 1u)) scores[i] = unseen;
  }
}

// A warp's arrival on a barrier, behind whatever fence its lanes have executed: one operation on the word instead of 32.
__device__ __forceinline__ void warp_arrive(uint64_t *barrier, uint32_t lane) {
  __syncwarp();
  if (lane == 0) barrier_arrive(smem_u32(barrier));
}

// ---- the kernel -------------------------------------------------------------------------------------------------------
// Placement: a type with
//   Args                     derived from RowTileArgs
//   prepare(args)            every thread, before anything is read that the predecessor wrote; ends synchronised
//   begin(args)              every thread, after the wait for the predecessor
//   items(args)              of the launch, the same for every thread from then on
//   plan(args, index, item)  the plan warp: item number `index`
//   row(args, item, r)       row r of the tile
//   empty(args, item, tid)   each softmax thread, for an item without pages
// It lives in shared memory behind the kernel's own.
template <uint32_t Format, typename Placement>
__global__ void __launch_bounds__(kRowTileThreads, 1)
row_tile_kernel(const __grid_constant__ CUtensorMap head_map, const __grid_constant__ typename Placement::Args args) {
  using Kind = Traits<Format>;
  constexpr uint32_t kSlab = Kind::kSlab, kRawStages = Kind::kRawStages, kRawStageBytes = raw_stage_bytes<Format>();
  constexpr uint32_t kRawScaleOffset = 4 * kSlab, kTileStages = Kind::kTileStages, kExpandTeam = kExpanderThreads / kTileStages;
  constexpr bool kPermuted = Format == RK_FORMAT_INT4;
  static_assert(kRawStages % kTileStages == 0, "a raw stage belongs to one expander team: its barrier is never waited on two completions behind");
  extern __shared__ uint8_t dynamic_shared[];
  const uint32_t tiles = (smem_u32(dynamic_shared) + 1023u) & ~1023u;
  uint8_t *tile_ptr = dynamic_shared + (tiles - smem_u32(dynamic_shared));
  RowTileShared &sh = *reinterpret_cast<RowTileShared *>(tile_ptr + tile_bytes<Format>());
  Placement &placement = *reinterpret_cast<Placement *>(&sh + 1);
  volatile uint32_t *error = &sh.error;
  const uint32_t k_tile = tiles, v_tile = k_tile + kTileStages * kKBytes, raw_tile = v_tile + kTileStages * kVBytes; // K stages | V stages | raw ring
  uint8_t *k_ptr = tile_ptr, *v_ptr = k_ptr + kTileStages * kKBytes;
  const uint8_t *raw_ptr = v_ptr + kTileStages * kVBytes;
  const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); // what follows takes the SMs that this launch leaves

  if (tid == 0) {
    for (uint32_t r = 0; r < kRawStages; ++r) {
      barrier_init(smem_u32(&sh.raw_full[r]), 1);
      barrier_init(smem_u32(&sh.raw_free[r]), kExpandTeam / 32);
    }
    for (uint32_t b = 0; b < 2; ++b) {
      barrier_init(smem_u32(&sh.k_full[b]), kExpandTeam / 32);
      barrier_init(smem_u32(&sh.v_full[b]), kExpandTeam / 32);
      barrier_init(smem_u32(&sh.k_free[b]), 1);
      barrier_init(smem_u32(&sh.v_free[b]), 1);
      barrier_init(smem_u32(&sh.s_full[b]), 1);
      barrier_init(smem_u32(&sh.p_free[b]), 1);
      barrier_init(smem_u32(&sh.p_full[b]), kSoftmaxWarps);
      barrier_init(smem_u32(&sh.drained[b]), 1);
    }
    barrier_init(smem_u32(&sh.query_full), kSoftmaxWarps);
    barrier_init(smem_u32(&sh.output_free), kSoftmaxWarps);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    sh.error = 0;
    sh.spin_limit = args.spin_limit;
  }
  if (warp == kCopyWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  placement.prepare(args);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  placement.begin(args);
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = sh.tmem_base;
  const uint32_t tmem_o = tmem + kTmemO, tmem_s = tmem + kTmemS, tmem_q = tmem + kTmemQ;

  // Every role walks the same items, so that all of them make the same number of steps whatever a wait that gave up left
  // behind; `done` counts the groups of the items before, and every ring, stage and barrier counts on across items. Between
  // batches the roles meet and the plan warp fills the next ones in.
  const uint32_t items = placement.items(args), mine = blockIdx.x < items ? (items - blockIdx.x - 1) / gridDim.x + 1 : 0;
  auto plan_batch = [&](uint32_t first) {
    for (uint32_t k = first; k < min(mine, first + kBatchItems); ++k) placement.plan(args, blockIdx.x + k * gridDim.x, sh.items[k % kBatchItems]);
  };
  if (warp == kPlanWarp) plan_batch(0);
  __syncthreads();
  auto item_of = [&](uint32_t k) -> const RowItem & {
    if (k && k % kBatchItems == 0) { // every thread of the block comes by here
      __syncthreads();
      __syncthreads();
    }
    return sh.items[k % kBatchItems];
  };

  if (warp < kSoftmaxWarps) {
    // ---- softmax ----------------------------------------------------------------------------------------------------
    const uint32_t quarter = warp & 3u, part = warp >> 2;
    const uint32_t my_row = quarter * 32 + lane, lane_address = (quarter * 32u) << 16;
    auto row_barrier = [&] { asm volatile("bar.sync %0, %1;" ::"r"(1u + quarter), "n"(32 * kRowThreads) : "memory"); }; // the four warps of the quarter's rows
    uint32_t done = 0;
    for (uint32_t k = 0; k < mine; ++k) {
      const RowItem &item = item_of(k);
      const uint32_t begin = item.ordinal_begin, end = item.ordinal_end, groups = (end - begin + 1) / 2;
      if (!groups) {
        placement.empty(args, item, tid);
        continue;
      }
      const RowPlace row = placement.row(args, item, my_row);
      const PageList list = item.list;
      const float slope = args.shape.slopes ? __ldg(args.shape.slopes + item.head * kG + row.head_row) * kLog2e : 0.0f;

      // The query row into tensor memory, a quarter of its dims by each of its threads. int4: fp16, element order (0,4,1,5,2,6,3,7)
      // inside every 8 dims, dims 1,5,3,7 divided by 16; int8, fp8: fp16 in order; bf16: the bits. A power of two keeps large
      // queries inside fp16 (exact).
      const uint16_t *query = row.query + part * (kD / kRowThreads);
      uint4 words[8]; // 64 dims, read once: they become the operands in place
#pragma unroll
      for (uint32_t c = 0; c < 8; ++c) words[c] = row.real ? __ldg(reinterpret_cast<const uint4 *>(query + 8 * c)) : make_uint4(0, 0, 0, 0);
      int exponent = 0;
      if (!Kind::kBf16) {
        float amax = 0.0f;
#pragma unroll
        for (uint32_t c = 0; c < 8; ++c) {
          const uint32_t w[4] = {words[c].x, words[c].y, words[c].z, words[c].w};
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) amax = fmaxf(amax, fmaxf(fabsf(bf16_bits_to_float(w[i] & 0xffffu)), fabsf(bf16_bits_to_float(w[i] >> 16))));
        }
        sh.exchange[0][part][my_row] = amax;
        row_barrier();
#pragma unroll
        for (uint32_t i = 0; i < kRowThreads; ++i) amax = fmaxf(amax, sh.exchange[0][i][my_row]);
        if (amax >= 8192.0f) exponent = ilogbf(amax) - 12;
      }
      float q_sum = 0.0f; // over the values the tensor core will see, for the key-offset correction
      if (!Kind::kBf16) {
        const float down = ldexpf(1.0f, -exponent);
#pragma unroll
        for (uint32_t c = 0; c < 8; ++c) {
          const uint32_t w[4] = {words[c].x, words[c].y, words[c].z, words[c].w};
          float d[8];
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) { d[2 * i] = bf16_bits_to_float(w[i] & 0xffffu) * down; d[2 * i + 1] = bf16_bits_to_float(w[i] >> 16) * down; }
          if (Format == RK_FORMAT_INT4)
            words[c] = make_uint4(pack_half2(d[0], d[4]), pack_half2(d[1] * 0.0625f, d[5] * 0.0625f), pack_half2(d[2], d[6]), pack_half2(d[3] * 0.0625f, d[7] * 0.0625f));
          else
            words[c] = make_uint4(pack_half2(d[0], d[1]), pack_half2(d[2], d[3]), pack_half2(d[4], d[5]), pack_half2(d[6], d[7]));
          const uint32_t h[4] = {words[c].x, words[c].y, words[c].z, words[c].w};
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) {
            const __half2 pair = *reinterpret_cast<const __half2 *>(&h[i]);
            q_sum += ((Format == RK_FORMAT_INT4 && (i & 1u)) ? 16.0f : 1.0f) * (__low2float(pair) + __high2float(pair));
          }
        }
      }
      tmem_store32(tmem_q + lane_address + part * 32, reinterpret_cast<const float (&)[32]>(words));
      if (!Kind::kBf16) sh.exchange[1][part][my_row] = q_sum;
      tmem_fence_before();
      warp_arrive(&sh.query_full, lane);
      if (!Kind::kBf16) {
        row_barrier();
        q_sum = (sh.exchange[1][0][my_row] + sh.exchange[1][1][my_row]) + (sh.exchange[1][2][my_row] + sh.exchange[1][3][my_row]);
        row_barrier(); // the exchange is free for the groups' maxima
      }

      const float score_scale = rk_score_scale(row.score_scale, kD) * kLog2e;
      const float row_factor = ldexpf(score_scale, Kind::kKeyShift + exponent);
      const float row_offset = -Kind::kKeyOffset * q_sum * ldexpf(score_scale, exponent);
      const uint32_t position = row.position, sinks = args.shape.sinks;
      const uint32_t row_window = args.shape.window && position + 1 > args.shape.window ? position + 1 - args.shape.window : 0;
      constexpr uint32_t kOutColumns = kD / kRowThreads; // of O, this thread's to rescale and write out
      const uint32_t first_position = part * kRowTokens, part_token = kPermuted ? first_position / 8 : first_position;
      float row_max = -1.0e30f, row_sum = 0.0f;          // the sum of 2^(score - row_max) over this thread's tokens
      for (uint32_t g = 0; g < groups; ++g) {
        const uint32_t n = done + g, b = n & 1u, first = begin + 2 * g;
        const GroupView view{list.page(first) * kPageTokens, list.page(first + 1) * kPageTokens, first + 1 < end};
        const ScaleStage &stage = sh.scales[n % kScaleStages];
        barrier_wait(&sh.s_full[b], n >> 1, error);
        tmem_fence_after();
        float scores[kRowTokens];
        tmem_load_scores(tmem_s + b * 64 + lane_address + first_position, scores);
        // Most groups are seen whole by every row of a warp: nothing is tested then.
        const bool whole = __all_sync(0xffffffffu, view.whole(position, row_window));
        if (!whole && args.shape.cap != 0.0f) // the cap wants numbers, also where a row does not look
          mask_scores<kPermuted>(scores, part_token, view.seen_first(position, row_window, sinks), view.seen_second(position, row_window, sinks), 0.0f);
        const float common = shape_scores<kPermuted>(scores, stage, first_position, part_token, row_factor, row_offset, args.shape, slope, view, position);
        if (!whole)
          mask_scores<kPermuted>(scores, part_token, view.seen_first(position, row_window, sinks), view.seen_second(position, row_window, sinks), -INFINITY);
        float maximum = scores[0];
#pragma unroll
        for (uint32_t i = 1; i < kRowTokens; ++i) maximum = fmaxf(maximum, scores[i]);
        maximum += common;
        // the row's other parts; past this barrier every part holds its scores in registers, so the weights may overwrite the
        // first 32 columns of the buffer
        sh.exchange[b][part][my_row] = maximum;
        tmem_fence_before();
        row_barrier();
        tmem_fence_after();
#pragma unroll
        for (uint32_t i = 0; i < kRowThreads; ++i) maximum = fmaxf(maximum, sh.exchange[b][i][my_row]);
        // The reference only moves when the maximum grew by more than 2^8, so the 16-bit weights stay below 2^(8+6).
        const bool grow = maximum > row_max + 8.0f;
        float scale = 1.0f;
        if (grow) {
          scale = exp2_fast(row_max - maximum);
          row_max = maximum;
          row_sum *= scale;
        }
        weigh_scores(scores, stage, first_position, row_max - 6.0f - common, row_sum);
        uint32_t packed[kRowTokens / 2], packed_low[Kind::kBf16 ? kRowTokens / 2 : 1];
#pragma unroll
        for (uint32_t c = 0; c < kRowTokens / 2; ++c) {
          packed[c] = Kind::kBf16 ? pack_bfloat2(scores[2 * c], scores[2 * c + 1]) : pack_half2(scores[2 * c], scores[2 * c + 1]);
          if (Kind::kBf16) // what the high part left of each weight: 16 bits of it altogether, two contractions
            packed_low[c] = pack_bfloat2(scores[2 * c] - __uint_as_float(packed[c] << 16), scores[2 * c + 1] - __uint_as_float(packed[c] & 0xffff0000u));
        }
        if (g && __any_sync(0xffffffffu, grow)) { // this part rescales its columns of O once the contraction before has landed
          barrier_wait(&sh.p_free[(n - 1) & 1u], (n - 1) >> 1, error);
          tmem_fence_after();
#pragma unroll 1
          for (uint32_t c = 0; c < kOutColumns; c += 32) {
            float o[32];
            tmem_load32(tmem_o + lane_address + part * kOutColumns + c, o);
#pragma unroll
            for (uint32_t i = 0; i < 32; ++i) o[i] *= scale;
            tmem_store32(tmem_o + lane_address + part * kOutColumns + c, o);
          }
        }
        tmem_store_packed(tmem_s + b * 64 + lane_address + part * (kRowTokens / 2), packed);
        if constexpr (Kind::kBf16) tmem_store_packed(tmem_s + b * 64 + 32 + lane_address + part * (kRowTokens / 2), packed_low);
        tmem_fence_before();
        warp_arrive(&sh.p_full[b], lane);
      }

      // ---- partial output: the row of O, un-normalised, a quarter of its columns by each thread; {reference exponent, sum} ----
      const uint32_t last = done + groups - 1;
      row_barrier(); // every part is through with the exchange
      sh.exchange[1][part][my_row] = row_sum; // the next item writes [0] first, and [1] behind a barrier that follows the reads below
      // Every contraction into O has landed when the last group's has. (The completion before it on that barrier, two groups
      // earlier, preceded the last scores, so the parity is not mistaken.)
      barrier_wait(&sh.p_free[last & 1u], last >> 1, error);
      tmem_fence_after();
      const bool failed = *error != 0;
      // Lanes l and l ^ 1 swap halves of 32 bytes, so that each store instruction writes whole sectors: both write the even
      // lane's row, then both the odd one's.
      float *out = args.partials + row.slot * kD + part * kOutColumns;
      const bool odd = lane & 1u;
      float *other_out = reinterpret_cast<float *>(__shfl_xor_sync(0xffffffffu, reinterpret_cast<unsigned long long>(out), 1));
      const bool other_real = __shfl_xor_sync(0xffffffffu, row.real, 1);
      float *even_out = odd ? other_out + 4 : out, *odd_out = odd ? out + 4 : other_out;
      const bool even_real = odd ? other_real : row.real, odd_real = odd ? row.real : other_real;
#pragma unroll 1
      for (uint32_t c = 0; c < kOutColumns; c += 32) {
        float o[32];
        tmem_load32(tmem_o + lane_address + part * kOutColumns + c, o);
#pragma unroll
        for (uint32_t i = 0; i < 32; i += 8) {
          float theirs[4]; // the even lane gives its upper half away, the odd one its lower
#pragma unroll
          for (uint32_t e = 0; e < 4; ++e) theirs[e] = __shfl_xor_sync(0xffffffffu, odd ? o[i + e] : o[i + 4 + e], 1);
          const float4 mine = odd ? make_float4(o[i + 4], o[i + 5], o[i + 6], o[i + 7]) : make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          const float4 given = make_float4(theirs[0], theirs[1], theirs[2], theirs[3]);
          const float4 even = odd ? given : mine, other = odd ? mine : given;
          constexpr float kUnscale = 0.015625f; // 2^-6
          if (even_real) *reinterpret_cast<float4 *>(even_out + c + i) = make_float4(even.x * kUnscale, even.y * kUnscale, even.z * kUnscale, even.w * kUnscale);
          if (odd_real) *reinterpret_cast<float4 *>(odd_out + c + i) = make_float4(other.x * kUnscale, other.y * kUnscale, other.z * kUnscale, other.w * kUnscale);
        }
      }
      tmem_fence_before();
      warp_arrive(&sh.output_free, lane);
      row_barrier(); // the sums are there
      if (part == 0 && row.real) {
        args.statistics[row.slot * 2] = failed ? -INFINITY : row_max * kLn2;
        float total = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kRowThreads; ++i) total += sh.exchange[1][i][my_row];
        args.statistics[row.slot * 2 + 1] = failed ? 0.0f : total;
      }
      done += groups;
    }
  } else if (warp < kCopyWarp) {
    // ---- expanders: the team of an operand stage ----------------------------------------------------------------------
    const uint32_t index = tid - kSoftmaxThreads, team = index / kExpandTeam, e = index - team * kExpandTeam;
    uint32_t done = 0;
    for (uint32_t k = 0; k < mine; ++k) {
      const RowItem &item = item_of(k);
      const uint32_t begin = item.ordinal_begin, end = item.ordinal_end, groups = (end - begin + 1) / 2, last_position = item.last_position;
      const PageList list = item.list;
      for (uint32_t g = (team + kTileStages - done % kTileStages) % kTileStages; g < groups; g += kTileStages) {
        const uint32_t n = done + g, r = n % kRawStages, round = n / kTileStages, first = begin + 2 * g;
        // Positions whose token some row of the tile sees. The others may hold anything: their scales and, where a code may
        // decode to no number, their values become zeros.
        const GroupView view{list.page(first) * kPageTokens, list.page(first + 1) * kPageTokens, first + 1 < end};
        ValidBits valid{~uint64_t(0)};
        if (!view.whole(last_position, list.window_first))
          valid.bits = uint64_t(view.seen_first(last_position, list.window_first, args.shape.sinks)) |
                       uint64_t(view.seen_second(last_position, list.window_first, args.shape.sinks)) << 32;
        const uint8_t *raw = raw_ptr + r * kRawStageBytes;
        barrier_wait(&sh.raw_full[r], n / kRawStages, error);
        if (e < kGroupTokens) {
          // The slot's last readers, the softmax of group n - kScaleStages, are done: before this team expanded the values of
          // its last group it waited for the contraction two of its groups ago, which is that group's or a later one.
          static_assert(2 * kTileStages <= kScaleStages, "a scale slot outlives its readers");
          const uint32_t token = Expand<Format>::token_of(e);
          float key_scale = 0.0f, value_log = 0.0f, factor = 0.0f;
          if (valid.holds(token)) {
            if (Kind::kScales) {
              key_scale = reinterpret_cast<const float *>(raw + kRawScaleOffset)[token];
              const float value_scale = fmaxf(reinterpret_cast<const float *>(raw + kRawScaleOffset)[64 + token], 9.094947e-13f); // 2^-40
              value_log = log2_fast(value_scale);
              factor = __fdividef(0.015625f, value_scale);
            } else {
              key_scale = 1.0f;
              factor = 0.015625f;
            }
          }
          sh.scales[n % kScaleStages].put(e, key_scale, value_log, factor);
        }
        if (round) barrier_wait(&sh.k_free[team], round - 1, error);
        Expand<Format>::template keys<kExpandTeam>(raw, k_ptr + team * kKBytes, e);
        async_proxy_fence();
        warp_arrive(&sh.k_full[team], lane);
        if (round) barrier_wait(&sh.v_free[team], round - 1, error);
        Expand<Format>::template values<kExpandTeam>(raw, v_ptr + team * kVBytes, e, valid);
        async_proxy_fence();
        warp_arrive(&sh.v_full[team], lane);
        warp_arrive(&sh.raw_free[r], lane);
      }
      done += groups;
    }
  } else {
    if (warp == kCopyWarp) {
      // ---- TMA producer: lanes 0-7 issue one copy each (page, {K, V, key scales, value scales}) of the group -----------
      const uint32_t data_bytes = kHeads * kSlab, scale_bytes = Kind::kScales ? kPageTokens * kHeads * 4 : 0;
      const uint32_t local = (lane >> 2) & 1u, kind = lane & 3u;
      const bool copier = lane < 8 && (kind < 2 || Kind::kScales);
      const uint64_t extent_pages = args.layer.extent_pages;
      const uint64_t region_base = args.layer.offset + extent_pages * (kind == 0 ? 0ull : kind == 2 ? uint64_t(data_bytes)
                                                                        : kind == 1 ? uint64_t(data_bytes) + scale_bytes : 2ull * data_bytes + scale_bytes);
      const uint32_t page_stride = kind < 2 ? data_bytes : scale_bytes;
      // A wait that gave up (here or elsewhere) ends the streaming: a stage may then still be waiting for its last copy, and a
      // second one on the same barrier would leave its phases out of step with the wait for the copies below.
      uint32_t done = 0, issued = 0;
      bool stopped = false;
      for (uint32_t k = 0; k < mine; ++k) {
        const RowItem &item = item_of(k);
        const uint32_t begin = item.ordinal_begin, end = item.ordinal_end, groups = (end - begin + 1) / 2;
        const PageList list = item.list;
        const rk_page_entry *table = item.table;
        const uint64_t tensor_base = region_base + item.head * (kind < 2 ? kSlab : 128u);
        rk_page_entry next = lane < 8 && begin + local < end ? table[list.page(begin + local)] : 0;
        for (uint32_t g = 0; g < groups && !stopped; ++g) {
          const uint32_t n = done + g, r = n % kRawStages, first = begin + 2 * g, group_pages = min(2u, end - first);
          const rk_page_entry entry = next;
          if (lane < 8 && first + 2 + local < end) next = table[list.page(first + 2 + local)];
          if (n >= kRawStages) barrier_wait(&sh.raw_free[r], n / kRawStages - 1, error);
          stopped = __any_sync(0xffffffffu, *error != 0) || g + args.withheld_groups >= groups;
          if (stopped) break;
          issued = n + 1;
          const uint32_t full = smem_u32(&sh.raw_full[r]), stage = raw_tile + r * kRawStageBytes;
          if (lane == 0) barrier_expect(full, group_pages * (2 * kSlab + (Kind::kScales ? 256 : 0)));
          __syncwarp();
          if (copier && local < group_pages) {
            const uint64_t address = rk_entry_extent(entry) + tensor_base + uint64_t(rk_entry_index(entry)) * page_stride;
            if (kind < 2) tma_load_rows(stage + (2 * kind + local) * kSlab, &head_map, int32_t((address - args.window_base) >> 7), full);
            else bulk_load(stage + kRawScaleOffset + (2 * (kind - 2) + local) * 128, reinterpret_cast<const void *>(address), 128, full);
          }
        }
        done += groups;
      }
      // every copy this warp started has landed before the CTA may leave (also after a failed wait)
      if (lane == 0)
        for (uint32_t n = issued > kRawStages ? issued - kRawStages : 0; n < issued; ++n) {
          const uint32_t bar = smem_u32(&sh.raw_full[n % kRawStages]), parity = (n / kRawStages) & 1u;
          for (uint32_t i = 0; i < kSpinLimit && !barrier_try(bar, parity); ++i) __nanosleep(64);
        }
    } else if (warp == kScoresWarp) {
      // ---- S = Q.K^T: buffer n&1 is free once PV(n-2), which read its weights, has landed. The whole warp walks the loop
      // (uniform control flow); one elected lane issues ----
      const uint32_t idesc_qk = umma_instruction(kM, kGroupTokens, Kind::kBf16, Kind::kBf16);
      const uint64_t k_desc0 = umma_descriptor(k_tile), k_desc1 = umma_descriptor(k_tile + kKBytes);
      uint32_t done = 0, worked = 0;
      for (uint32_t k = 0; k < mine; ++k) {
        const RowItem &item = item_of(k);
        const uint32_t groups = (item.ordinal_end - item.ordinal_begin + 1) / 2;
        if (groups) barrier_wait(&sh.query_full, worked++, error);
        for (uint32_t g = 0; g < groups; ++g) {
          const uint32_t n = done + g, b = n & 1u, t = n % kTileStages;
          barrier_wait(&sh.k_full[t], n / kTileStages, error);
          if (n >= 2) barrier_wait(&sh.p_free[b], (n >> 1) - 1, error);
          tmem_fence_after();
          const uint64_t desc = t ? k_desc1 : k_desc0;
          if (elect_one()) {
#pragma unroll
            for (uint32_t j = 0; j < 16; ++j)
              umma_f16_ts(tmem_s + b * 64, tmem_q + 8 * j, desc + (((j >> 2) * (kGroupTokens * 128) + (j & 3u) * 32) >> 4), idesc_qk, j ? 1u : 0u);
            umma_commit(&sh.s_full[b]);
            umma_commit(&sh.k_free[t]);
          }
          __syncwarp();
        }
        done += groups;
      }
    } else if (warp == kOutputsWarp) {
      // ---- O += w.V: the first of an item overwrites O, once the item before has been read ----
      const uint32_t idesc_pv = umma_instruction(kM, kD, Kind::kBf16, Kind::kBf16); // both operands of one kind
      const uint64_t v_desc0 = umma_descriptor(v_tile), v_desc1 = umma_descriptor(v_tile + kVBytes);
      uint32_t done = 0, worked = 0;
      for (uint32_t k = 0; k < mine; ++k) {
        const RowItem &item = item_of(k);
        const uint32_t groups = (item.ordinal_end - item.ordinal_begin + 1) / 2;
        if (groups && worked) barrier_wait(&sh.output_free, worked - 1, error);
        worked += groups ? 1 : 0;
        for (uint32_t g = 0; g < groups; ++g) {
          const uint32_t n = done + g, b = n & 1u, t = n % kTileStages;
          barrier_wait(&sh.v_full[t], n / kTileStages, error);
          barrier_wait(&sh.p_full[b], n >> 1, error);
          tmem_fence_after();
          const uint64_t desc = t ? v_desc1 : v_desc0;
          const uint32_t source = tmem_s + b * 64;
          if (elect_one()) {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
              umma_f16_ts(tmem_o, source + 8 * j, desc + ((j * 32) >> 4), idesc_pv, (g || j) ? 1u : 0u);
              if (Kind::kBf16) umma_f16_ts(tmem_o, source + 32 + 8 * j, desc + ((j * 32) >> 4), idesc_pv, 1u); // the low parts
            }
            umma_commit(&sh.v_free[t]);
            umma_commit(&sh.p_free[b]);
          }
          __syncwarp();
        }
        done += groups;
      }
    } else {
      // ---- the plan -----------------------------------------------------------------------------------------------------
      for (uint32_t first = kBatchItems; first < mine; first += kBatchItems) {
        __syncthreads(); // the batch before is done
        plan_batch(first);
        __syncthreads();
      }
    }
    // Tensor memory is released once every contraction that was issued has completed, also when a wait gave up.
    if (warp == kScoresWarp || warp == kOutputsWarp) {
      uint64_t *drained = &sh.drained[warp - kScoresWarp];
      if (elect_one()) umma_commit(drained);
      __syncwarp();
      for (uint32_t i = 0; i < kSpinLimit && !barrier_try(smem_u32(drained), 0); ++i) __nanosleep(64);
    }
  }
  tmem_fence_before();
  __syncthreads();
  if (tid == 0 && sh.error) atomicExch(args.status, 1u);
  if (warp == kCopyWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

template <uint32_t Format, typename Placement> constexpr size_t row_tile_shared_bytes() { return 1024 + tile_bytes<Format>() + sizeof(RowTileShared) + sizeof(Placement); }

// Launches the kernel of a format on `ctas` persistent CTAs, as a programmatic dependent of what precedes it.
template <typename Placement, uint32_t Format>
int launch_row_tile_format(const CUtensorMap &map, uint32_t ctas, const typename Placement::Args &args, cudaStream_t stream) {
  constexpr size_t bytes = row_tile_shared_bytes<Format, Placement>();
  static_assert(bytes <= 227 * 1024, "the tiles fit one SM");
  auto kernel = row_tile_kernel<Format, Placement>;
  if (int st = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)), "row tile shared memory")) return st;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(ctas);
  config.blockDim = dim3(kRowTileThreads);
  config.dynamicSmemBytes = bytes;
  config.stream = stream;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&config, kernel, map, args), "row tile launch");
}
template <typename Placement>
int launch_row_tile(uint32_t format, const Window *w, uint32_t ctas, const typename Placement::Args &args, cudaStream_t stream) {
  switch (format) {
  case RK_FORMAT_INT4: return launch_row_tile_format<Placement, RK_FORMAT_INT4>(w->int4_head_map, ctas, args, stream);
  case RK_FORMAT_INT8: return launch_row_tile_format<Placement, RK_FORMAT_INT8>(w->byte_head_map, ctas, args, stream);
  case RK_FORMAT_FP8E4M3: return launch_row_tile_format<Placement, RK_FORMAT_FP8E4M3>(w->byte_head_map, ctas, args, stream);
  default: return launch_row_tile_format<Placement, RK_FORMAT_BF16>(w->int4_map, ctas, args, stream);
  }
}

} // namespace rk::tile
