// decode_partials.cuh — what a lane's partials look like behind a streaming decode kernel, and that kernel's launch for
// callers that merge the partials with others (shared_prefix.cu).
#pragma once

#include "common.cuh"
#include "score_shape.cuh"
#include "window.cuh"

namespace rk {

constexpr uint32_t kDecodeSlotsPerSegment = 3; // the page residues a CTA keeps apart
constexpr uint32_t kDecodeHeads = 4;

// A lane's descriptor {first segment, segments | last segment holds three slots << 31} -> its partial slots in order.
struct LaneSlots {
  uint32_t first, single, slots; // segments [first, first + single) hold one slot each; then up to three of segment first + single
  __device__ __forceinline__ explicit LaneSlots(uint2 descriptor) {
    const uint32_t segments = descriptor.y & 0x7fffffffu, triple = descriptor.y >> 31;
    first = descriptor.x;
    single = segments - (segments ? triple : 0u);
    slots = single + (segments - single) * kDecodeSlotsPerSegment;
  }
  __device__ __forceinline__ uint64_t slot(uint32_t t, uint32_t head) const {
    return t < single ? (uint64_t(first + t) * kDecodeHeads + head) * kDecodeSlotsPerSegment
                      : (uint64_t(first + single) * kDecodeHeads + head) * kDecodeSlotsPerSegment + (t - single);
  }
};

// The streaming kernel over what each lane has behind its group's shared pages, without the merge (decode_attention.cu).
int launch_decode_suffix(uint32_t format, const rk_decode_plan &plan, cudaStream_t stream, const Window *window, const void *queries,
                         float *partials, float *statistics, uint32_t *descriptors, const rk_page_entry *const *tables,
                         const rk_verify_params *lane_params, rk_kv_layer layer, const ShapeArgs &shape, const uint32_t *lane_groups,
                         const uint32_t *group_pages);

} // namespace rk
