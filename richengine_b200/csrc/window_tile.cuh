// window_tile.cuh — what the tcgen05 attention kernels share (verify_attention.cu and row_tile.cuh, with shaped_attention.cu and
// shared_prefix.cu on it): the roles' sizes, the stored formats as 16-bit tensor-core operands, and the mbarrier, TMA, tcgen05 and
// tensor-memory primitives.
#pragma once

#include "common.cuh"
#include "score_shape.cuh"
#include "window.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace rk::tile {

constexpr uint32_t kRowThreads = 4;                      // softmax threads per fused row (one per warp of the row's quarter)
constexpr uint32_t kSoftmaxWarps = 4 * kRowThreads;
constexpr uint32_t kRowTokens = 64 / kRowThreads;         // contraction positions of a group per softmax thread
constexpr uint32_t kExpandWarps = 8;   // kTileStages teams: team t expands the groups g = t (mod kTileStages) into operand stage t
constexpr uint32_t kSoftmaxThreads = kSoftmaxWarps * 32;
constexpr uint32_t kThreads = (kSoftmaxWarps + kExpandWarps + 3) * 32;
constexpr uint32_t kTmaWarp = kSoftmaxWarps + kExpandWarps, kScoreWarp = kTmaWarp + 1, kValueWarp = kTmaWarp + 2;
constexpr uint32_t kScaleStages = 4;
constexpr uint32_t kGroupTokens = 64;
constexpr uint32_t kM = 128, kD = 256, kG = 6, kHeads = 4;
constexpr uint32_t kSpinLimit = 1u << 20;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// shared-memory tiles (bytes); every tile starts 1024-aligned
constexpr uint32_t kKBytes = kGroupTokens * kD * 2;  // 4 column blocks of [64 rows][64 elements]
constexpr uint32_t kVBytes = kD * kGroupTokens * 2;  // 1 column block of [256 rows][64 elements]
constexpr uint32_t kMaxRawStages = 4;

// What differs between the stored formats: the size of one head's K (or V) slab of a page, whether
// scales exist, how codes become 16-bit tensor-core operands, and the depth of the raw ring that fits.
//   int4      fp16 operands; key codes as u * 2^-24 with u = code + 8 (the +8 leaves through sum(q)),
//             odd dims x16 against queries / 16, dims of every 8 in the order (0,4,1,5,2,6,3,7).
//   int8      fp16 operands; key codes as u * 2^-24 with u = code + 128; values exact (1024 + u - 1152).
//   fp8 e4m3  fp16 operands, exact (cvt); queries staged as fp16 like the reference's fp8 tile
//             (paged_attention_fp8_tile.h:34-60).
//   bf16      bf16 operands (bits as stored). Both operands of a contraction are of one kind, so the
//             probabilities are bf16 too: a high and a low part, contracted one after the other (16 bits).
template <uint32_t Format> struct Traits;
template <> struct Traits<RK_FORMAT_INT4> {
  static constexpr uint32_t kSlab = 4096, kRawStages = 4, kTileStages = 2;
  static constexpr bool kScales = true, kBf16 = false;
  static constexpr float kKeyOffset = 8.0f;
  static constexpr int kKeyShift = 24;
};
template <> struct Traits<RK_FORMAT_INT8> {
  static constexpr uint32_t kSlab = 8192, kRawStages = 2, kTileStages = 2;
  static constexpr bool kScales = true, kBf16 = false;
  static constexpr float kKeyOffset = 128.0f;
  static constexpr int kKeyShift = 24;
};
template <> struct Traits<RK_FORMAT_FP8E4M3> {
  static constexpr uint32_t kSlab = 8192, kRawStages = 2, kTileStages = 2;
  static constexpr bool kScales = true, kBf16 = false;
  static constexpr float kKeyOffset = 0.0f;
  static constexpr int kKeyShift = 0;
};
template <> struct Traits<RK_FORMAT_BF16> {
  static constexpr uint32_t kSlab = 16384, kRawStages = 2, kTileStages = 1; // the slabs are large: one operand stage, two raw stages
  static constexpr bool kScales = false, kBf16 = true;
  static constexpr float kKeyOffset = 0.0f;
  static constexpr int kKeyShift = 0;
};
// raw stage: K0 | K1 | V0 | V1 | ks0 ks1 vs0 vs1 (128 B each) | pad to 1 KiB
template <uint32_t Format> __host__ __device__ constexpr uint32_t raw_stage_bytes() { return 4 * Traits<Format>::kSlab + 1024; }
template <uint32_t Format> __host__ __device__ constexpr uint32_t tile_bytes() {
  return Traits<Format>::kTileStages * (kKBytes + kVBytes) + Traits<Format>::kRawStages * raw_stage_bytes<Format>();
}
// tensor-memory columns
constexpr uint32_t kTmemO = 0, kTmemS = 256, kTmemQ = 384; // S twice (64 columns each); P(g) overwrites the first half of S(g)

// The per-token scales of a group, laid out for a softmax thread's neighbouring positions: two tokens' {key scale pair, log2
// value scale pair} in one 16-byte word (operands of packed fp32 arithmetic), the factors of four tokens in another. Every
// thread of a row reads the same words, a wavefront each: 12 of them for 16 tokens instead of 32.
struct ScaleStage {
  float4 pairs[kGroupTokens / 2];   // {key scale, key scale, log2 value scale, log2 value scale}
  float4 factors[kGroupTokens / 4]; // 2^-6 / value scale
  __device__ __forceinline__ void put(uint32_t position, float key_scale, float value_log, float factor) {
    float *pair = reinterpret_cast<float *>(&pairs[position >> 1]) + (position & 1u);
    pair[0] = key_scale;
    pair[2] = value_log;
    reinterpret_cast<float *>(factors)[position] = factor;
  }
};

struct Control {
  uint64_t raw_full[kMaxRawStages], raw_free[kMaxRawStages];
  uint64_t k_full[2], k_free[2], v_full[2], v_free[2], s_full[2], p_full[2], p_free[2], scale_free[kScaleStages];
  uint64_t drained[2]; // one per issue warp: every contraction it issued has completed
  uint32_t tmem_base;
  uint32_t error;
  uint32_t spin_limit; // directly after `error`: barrier_wait reads it through the error pointer
  float q_sums[kM];
  float exchange[2][kRowThreads][kM]; // the part-row maxima of a group (and, at the end, the part-row sums); a warp's rows side by side
  ScaleStage scales[kScaleStages];
};

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return uint32_t(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void barrier_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool barrier_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
               : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0;
}
// Waits for completion number `count` (0-based) of a barrier. Bounded: gives up after the launch's poll limit,
// or at once when another wait of this CTA already gave up; either way `error` ends non-zero.
// `error` points at Control::error; the word after it holds the poll limit of this launch.
__device__ __forceinline__ void barrier_wait(uint64_t *barrier, uint32_t count, volatile uint32_t *error) {
  const uint32_t bar = smem_u32(barrier), parity = count & 1u;
  if (barrier_try(bar, parity)) return;
  const uint32_t limit = error[1];
  for (uint32_t i = 0; i < limit; ++i) {
    if (barrier_try(bar, parity)) return; // try_wait itself suspends the thread for a while
    if ((i & 63u) == 63u) {
      if (*error) return;
      if (i > 4096) __nanosleep(256);
    }
  }
  *error = 1;
}
__device__ __forceinline__ void tma_load_rows(uint32_t dst, const CUtensorMap *map, int32_t row, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               ::"r"(dst), "l"(map), "r"(0), "r"(row), "r"(bar) : "memory");
}
// Asks L2 for `bytes` of global memory (16-byte granular) without a destination: the later copy of the same
// bytes into shared memory then pays the L2 latency, not the HBM one.
__device__ __forceinline__ void prefetch_l2(uint64_t address, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(address), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// K-major, 128-byte swizzle shared-memory descriptor: 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t umma_descriptor(uint32_t address) {
  uint64_t desc = 0;
  desc |= uint64_t((address & 0x3FFFFu) >> 4);   // start address
  desc |= uint64_t(1) << 16;                      // leading byte offset (unused for swizzled K-major)
  desc |= uint64_t(1024 >> 4) << 32;              // stride byte offset
  desc |= uint64_t(1) << 46;                      // descriptor version (sm_100)
  desc |= uint64_t(2) << 61;                      // SWIZZLE_128B
  return desc;
}
// kind::f16 instruction descriptor: 16-bit operands (0 = fp16, 1 = bf16) -> fp32, both operands K-major.
__host__ __device__ constexpr uint32_t umma_instruction(uint32_t m, uint32_t n, uint32_t a_format = 0, uint32_t b_format = 0) {
  return (1u << 4) | (a_format << 7) | (b_format << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
// True in exactly one lane of a converged warp; unlike a test of the lane index it keeps the surrounding
// control flow warp-uniform, so descriptors and addresses stay on the uniform datapath.
__device__ __forceinline__ bool elect_one() {
  uint32_t pred;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(pred));
  return pred != 0;
}
// A operand from tensor memory: lane = row, each 32-bit column two consecutive K elements.
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n}"
               ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(0u) : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t *barrier) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(barrier)) : "memory");
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void async_proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tmem_load32(uint32_t address, float (&v)[32]) {
  uint32_t r[32];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
               "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                 "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                 "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(address));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_store32(uint32_t address, const float (&v)[32]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
               "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
               ::"r"(address), "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])),
                 "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])), "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7])),
                 "r"(__float_as_uint(v[8])), "r"(__float_as_uint(v[9])), "r"(__float_as_uint(v[10])), "r"(__float_as_uint(v[11])),
                 "r"(__float_as_uint(v[12])), "r"(__float_as_uint(v[13])), "r"(__float_as_uint(v[14])), "r"(__float_as_uint(v[15])),
                 "r"(__float_as_uint(v[16])), "r"(__float_as_uint(v[17])), "r"(__float_as_uint(v[18])), "r"(__float_as_uint(v[19])),
                 "r"(__float_as_uint(v[20])), "r"(__float_as_uint(v[21])), "r"(__float_as_uint(v[22])), "r"(__float_as_uint(v[23])),
                 "r"(__float_as_uint(v[24])), "r"(__float_as_uint(v[25])), "r"(__float_as_uint(v[26])), "r"(__float_as_uint(v[27])),
                 "r"(__float_as_uint(v[28])), "r"(__float_as_uint(v[29])), "r"(__float_as_uint(v[30])), "r"(__float_as_uint(v[31]))
               : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t address, float (&v)[16]) {
  uint32_t r[16];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(address));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_store8(uint32_t address, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"r"(address), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_load_scores(uint32_t address, float (&v)[16]) { tmem_load16(address, v); }
__device__ __forceinline__ void tmem_store_packed(uint32_t address, const uint32_t (&v)[8]) { tmem_store8(address, v); }
__device__ __forceinline__ float exp2_fast(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ float log2_fast(float x) { float r; asm("lg2.approx.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) { const __half2 h = __floats2half2_rn(lo, hi); return *reinterpret_cast<const uint32_t *>(&h); }
__device__ __forceinline__ uint32_t pack_bfloat2(float lo, float hi) { const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi); return *reinterpret_cast<const uint32_t *>(&h); }
__device__ __forceinline__ uint32_t sub_f16x2(uint32_t a, uint32_t b) { uint32_t r; asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
__device__ __forceinline__ uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) { uint32_t r; asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c)); return r; }
// (a & mask) ^ flip in one logic instruction; both constants sit in registers.
__device__ __forceinline__ uint32_t and_xor(uint32_t a, uint32_t mask, uint32_t flip) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(r) : "r"(a), "r"(mask), "r"(flip));
  return r;
}
__device__ __forceinline__ uint32_t register_constant(uint32_t value) {
  uint32_t r;
  asm volatile("mov.b32 %0, %1;" : "=r"(r) : "r"(value));
  return r;
}

// Byte offset of 16-byte chunk `chunk` (0..7) of row `row` inside one 128-byte-swizzled block.
__device__ __forceinline__ uint32_t swizzled(uint32_t row, uint32_t chunk) { return row * 128u + ((chunk ^ (row & 7u)) << 4); }

// Within a 16-byte operand chunk of 8 dims the element order is (0,4,1,5,2,6,3,7): the order in which
// an int4 word yields its nibble pairs; queries and keys use the same order, so the contraction is
// unchanged. Dims 1,5,3,7 of each 8 carry the 16x of a high nibble on the key side, 1/16 on the query.

// ---- raw codes -> 16-bit operand tiles, one team of `Team` threads (e = 0..Team-1) per 64-token group ---------
// K tile: four column blocks of [64 positions][64 dims], 128-byte rows, 128-byte swizzle. V^T tile: one block
// of [256 dims][64 positions]. `raw` = K0 | K1 | V0 | V1 slabs as TMA left them (128-byte rows, swizzled).
// `valid` = positions of the group whose tokens exist; formats whose stale bytes can decode to NaN or
// infinity (fp8, bf16) get zeros at value positions past it, so a zero probability meets a finite value.

template <uint32_t Format> struct Expand;

// Which positions of a group hold a token: the first `valid` ones, or, for a shaped launch, those of a bit mask (the
// tokens that some row of the tile sees).
struct ValidBelow {
  uint32_t valid;
  __device__ __forceinline__ bool holds(uint32_t token) const { return token < valid; }
  template <uint32_t N> __device__ __forceinline__ bool holds_all(uint32_t position) const { return position + N <= valid; }
};
struct ValidBits {
  uint64_t bits;
  __device__ __forceinline__ bool holds(uint32_t token) const { return (bits >> token) & 1u; }
  template <uint32_t N> __device__ __forceinline__ bool holds_all(uint32_t position) const {
    constexpr uint32_t kAll = (1u << N) - 1u;
    return (uint32_t(bits >> position) & kAll) == kAll;
  }
};
template <typename Valid> __device__ __forceinline__ uint32_t mask_pair(uint32_t value, uint32_t position, const Valid &valid) {
  return value & ((valid.holds(position) ? 0x0000FFFFu : 0u) | (valid.holds(position + 1) ? 0xFFFF0000u : 0u));
}

template <> struct Expand<RK_FORMAT_INT4> {
  // position 8r+j holds token 8j+r: every access of both transposes is conflict-free
  __device__ static uint32_t token_of(uint32_t position) { return 8 * (position & 7u) + (position >> 3); }
  template <uint32_t Team> __device__ static void keys(const uint8_t *raw, uint8_t *k_stage, uint32_t e) {
    const uint32_t low_mask = register_constant(0x000F000Fu), high_mask = register_constant(0x00F000F0u);
    const uint32_t key_low = register_constant(0x00080008u), key_high = register_constant(0x00800080u);
    // a thread takes a raw 16-byte chunk (32 dims of one token) = four operand chunks. The eight lanes of an
    // access phase take tokens 8k + t and chunks c0 ^ k.
#pragma unroll
    for (uint32_t i = 0; i < (512 + Team - 1) / Team; ++i) {
      const uint32_t item = e + i * Team;
      if (512 % Team && item >= 512) break;
      const uint32_t k8 = item & 7u, c = ((item >> 3) & 7u) ^ k8, t = item >> 6;
      const uint32_t token = 8 * k8 + t, position = 8 * t + k8;
      const uint4 x = *reinterpret_cast<const uint4 *>(raw + (token >> 5) * 4096 + swizzled(token & 31u, c));
      const uint32_t words[4] = {x.x, x.y, x.z, x.w};
      uint8_t *block = k_stage + (c >> 1) * (kGroupTokens * 128);
#pragma unroll
      for (uint32_t w = 0; w < 4; ++w) {
        const uint32_t y = words[w] >> 8;
        *reinterpret_cast<uint4 *>(block + swizzled(position, ((c & 1u) << 2) + w)) =
            make_uint4(and_xor(words[w], low_mask, key_low), and_xor(words[w], high_mask, key_high),
                       and_xor(y, low_mask, key_low), and_xor(y, high_mask, key_high));
      }
    }
  }
  template <uint32_t Team, typename Valid> __device__ static void values(const uint8_t *raw, uint8_t *v_stage, uint32_t e, const Valid &) {
    const uint32_t low_mask = register_constant(0x000F000Fu), high_mask = register_constant(0x00F000F0u);
    const uint32_t value_low = register_constant(0x64086408u), value_high = register_constant(0x64806480u);
    // thread = (r8, word w of 8 dims) takes tokens 8j + r8, j = 0..7, and transposes 8x8 in registers: each
    // dim gets a 16-byte run of eight tokens at contraction positions 8*r8 + j.
#pragma unroll
    for (uint32_t half = 0; half < (256 + Team - 1) / Team; ++half) {
      const uint32_t unit = e + half * Team, r8 = unit & 7u, w = unit >> 3;
      if ((256 % Team || Team > 256) && unit >= 256) break;
      uint32_t x[8];
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j)
        x[j] = *reinterpret_cast<const uint32_t *>(raw + (2 + (j >> 2)) * 4096 + swizzled(8 * (j & 3u) + r8, w >> 2) + (w & 3u) * 4);
#pragma unroll
      for (uint32_t byte = 0; byte < 4; ++byte) { // byte of each word = dims 8w+2*byte (low nibble), +1 (high nibble)
        uint32_t lo[4], hi[4];
        const uint32_t selector = byte | (byte << 4) | ((4 + byte) << 8) | ((4 + byte) << 12);
#pragma unroll
        for (uint32_t pair = 0; pair < 4; ++pair) {
          const uint32_t joined = __byte_perm(x[2 * pair], x[2 * pair + 1], selector);
          lo[pair] = sub_f16x2(and_xor(joined, low_mask, value_low), value_low);                                   // 1024+u - 1032
          hi[pair] = fma_f16x2(and_xor(joined, high_mask, value_high), 0x2C002C00u /* 1/16 */, 0xD480D480u /* -72 */); // (1024+16u)/16 - 72
        }
        const uint32_t dim = 8 * w + 2 * byte;
        *reinterpret_cast<uint4 *>(v_stage + swizzled(dim, r8)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        *reinterpret_cast<uint4 *>(v_stage + swizzled(dim + 1, r8)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      }
    }
  }
};

// One-byte codes (int8, fp8): K rows are 256 bytes = two 128-byte TMA rows; V rows (one dim) are 32 bytes, four
// dims to a TMA row. Positions are the tokens in order.
template <bool kFloat8> struct ExpandBytes {
  __device__ static uint32_t token_of(uint32_t position) { return position; }
  // four codes -> two registers of two 16-bit operands
  __device__ static void key_pairs(uint32_t word, uint32_t &first, uint32_t &second) {
    if (kFloat8) {
      asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %2;\ncvt.rn.f16x2.e4m3x2 %0, lo;\ncvt.rn.f16x2.e4m3x2 %1, hi;\n}" : "=r"(first), "=r"(second) : "r"(word));
    } else { // u = code + 128 as fp16 bits: u * 2^-24
      const uint32_t flipped = word ^ 0x80808080u;
      first = __byte_perm(flipped, 0, 0x4140);
      second = __byte_perm(flipped, 0, 0x4342);
    }
  }
  __device__ static void value_pairs(uint32_t word, uint32_t &first, uint32_t &second) {
    if (kFloat8) {
      key_pairs(word, first, second);
    } else { // 1024 + u, minus 1152: the code itself
      const uint32_t flipped = word ^ 0x80808080u;
      first = sub_f16x2(__byte_perm(flipped, 0x64646464u, 0x4140), 0x64806480u);
      second = sub_f16x2(__byte_perm(flipped, 0x64646464u, 0x4342), 0x64806480u);
    }
  }
  template <uint32_t Team> __device__ static void keys(const uint8_t *raw, uint8_t *k_stage, uint32_t e) {
    // item = (token, 16-byte chunk c of its 256-byte row): 16 dims -> two operand chunks. The eight lanes of a
    // shared-memory phase take chunks c..c+3 of token t and chunks c+4..c+7 of token t ^ 1: their raw rows differ by 2
    // and their chunk sets by bit 2 (eight distinct chunks to read), and their operand rows differ in bit 0 (eight
    // distinct chunks to write).
#pragma unroll
    for (uint32_t i = 0; i < (1024 + Team - 1) / Team; ++i) {
      const uint32_t item = e + i * Team, c = item & 15u, token = (item >> 4) ^ ((item >> 2) & 1u);
      if (1024 % Team && item >= 1024) break;
      const uint32_t row = 2 * (token & 31u) + (c >> 3);
      const uint4 x = *reinterpret_cast<const uint4 *>(raw + (token >> 5) * 8192 + swizzled(row, c & 7u));
      uint32_t out[8];
      key_pairs(x.x, out[0], out[1]); key_pairs(x.y, out[2], out[3]);
      key_pairs(x.z, out[4], out[5]); key_pairs(x.w, out[6], out[7]);
      uint8_t *block = k_stage + (c >> 2) * (kGroupTokens * 128);
      *reinterpret_cast<uint4 *>(block + swizzled(token, 2 * (c & 3u))) = make_uint4(out[0], out[1], out[2], out[3]);
      *reinterpret_cast<uint4 *>(block + swizzled(token, 2 * (c & 3u) + 1)) = make_uint4(out[4], out[5], out[6], out[7]);
    }
  }
  template <uint32_t Team, typename Valid> __device__ static void values(const uint8_t *raw, uint8_t *v_stage, uint32_t e, const Valid &valid) {
    // item = (page, dim, half h of its 32 tokens): 16 tokens -> two operand chunks of the dim's row. The eight lanes
    // of a shared-memory phase take eight consecutive dims of one half: two raw rows whose chunk sets have opposite
    // parity (eight distinct chunks to read), eight operand rows whose swizzles differ (eight distinct chunks to write).
#pragma unroll
    for (uint32_t i = 0; i < (1024 + Team - 1) / Team; ++i) {
      const uint32_t item = e + i * Team, h = (item >> 3) & 1u, dim = (item & 7u) | ((item >> 1) & 248u), page = item >> 9;
      if (1024 % Team && item >= 1024) break;
      const uint4 x = *reinterpret_cast<const uint4 *>(raw + (2 + page) * 8192 + swizzled(dim >> 2, 2 * (dim & 3u) + h));
      uint32_t out[8];
      value_pairs(x.x, out[0], out[1]); value_pairs(x.y, out[2], out[3]);
      value_pairs(x.z, out[4], out[5]); value_pairs(x.w, out[6], out[7]);
      const uint32_t position = 32 * page + 16 * h;
      if (kFloat8 && !valid.template holds_all<16>(position)) {
#pragma unroll
        for (uint32_t r = 0; r < 8; ++r) out[r] = mask_pair(out[r], position + 2 * r, valid);
      }
      *reinterpret_cast<uint4 *>(v_stage + swizzled(dim, 4 * page + 2 * h)) = make_uint4(out[0], out[1], out[2], out[3]);
      *reinterpret_cast<uint4 *>(v_stage + swizzled(dim, 4 * page + 2 * h + 1)) = make_uint4(out[4], out[5], out[6], out[7]);
    }
  }
};
template <> struct Expand<RK_FORMAT_INT8> : ExpandBytes<false> {};
template <> struct Expand<RK_FORMAT_FP8E4M3> : ExpandBytes<true> {};

// bf16: the stored bits are the operands; the expansion is a re-tiling copy. K rows are 512 bytes = four TMA
// rows (= the four column blocks); V rows (one dim) are 64 bytes, two dims to a TMA row.
template <> struct Expand<RK_FORMAT_BF16> {
  __device__ static uint32_t token_of(uint32_t position) { return position; }
  template <uint32_t Team> __device__ static void keys(const uint8_t *raw, uint8_t *k_stage, uint32_t e) {
#pragma unroll
    for (uint32_t i = 0; i < (2048 + Team - 1) / Team; ++i) {
      const uint32_t item = e + i * Team, c = item & 31u, token = item >> 5;
      if (2048 % Team && item >= 2048) break;
      const uint32_t row = 4 * (token & 31u) + (c >> 3);
      const uint4 x = *reinterpret_cast<const uint4 *>(raw + (token >> 5) * 16384 + swizzled(row, c & 7u));
      *reinterpret_cast<uint4 *>(k_stage + (c >> 3) * (kGroupTokens * 128) + swizzled(token, c & 7u)) = x;
    }
  }
  template <uint32_t Team, typename Valid> __device__ static void values(const uint8_t *raw, uint8_t *v_stage, uint32_t e, const Valid &valid) {
#pragma unroll
    for (uint32_t i = 0; i < (2048 + Team - 1) / Team; ++i) {
      // the eight lanes of a shared-memory phase take the four 16-byte pieces of dim d and of dim d ^ 5: raw rows two
      // apart with the other half of the row (eight distinct chunks to read), operand rows whose swizzles differ in
      // bit 2 (eight distinct chunks to write)
      const uint32_t item = e + i * Team, q = item & 3u, page = item >> 10;
      const uint32_t dim = ((item >> 2) & 255u) ^ (item & 4u); // odd dims trade places with the odd dim four further
      if (2048 % Team && item >= 2048) break;
      uint4 x = *reinterpret_cast<const uint4 *>(raw + (2 + page) * 16384 + swizzled(dim >> 1, 4 * (dim & 1u) + q));
      const uint32_t position = 32 * page + 8 * q;
      if (!valid.template holds_all<8>(position)) {
        x.x = mask_pair(x.x, position, valid); x.y = mask_pair(x.y, position + 2, valid);
        x.z = mask_pair(x.z, position + 4, valid); x.w = mask_pair(x.w, position + 6, valid);
      }
      *reinterpret_cast<uint4 *>(v_stage + swizzled(dim, 4 * page + q)) = x;
    }
  }
};

// ---- a softmax thread's N scores of a 64-token group ----------------------------------------------------------------
// Accumulators to scores + log2(value scale); `position` is the thread's first of the group.
template <uint32_t N>
__device__ __forceinline__ void scale_scores(float (&scores)[N], const ScaleStage &stage, uint32_t position, float row_factor, float row_offset) {
  const float2 factor = make_float2(row_factor, row_factor), offset = make_float2(row_offset, row_offset);
#pragma unroll
  for (uint32_t i = 0; i < N; i += 2) {
    const float4 pair = stage.pairs[(position + i) >> 1];
    const float2 s = fma_pair(fma_pair(make_float2(scores[i], scores[i + 1]), factor, offset), make_float2(pair.x, pair.y), make_float2(pair.z, pair.w));
    scores[i] = s.x;
    scores[i + 1] = s.y;
  }
}
// Scores to weights 2^(score - base); `sum` takes each weight times its token's factor, in order.
template <uint32_t N>
__device__ __forceinline__ void weigh_scores(float (&scores)[N], const ScaleStage &stage, uint32_t position, float base, float &sum) {
#pragma unroll
  for (uint32_t i = 0; i < N; i += 4) {
    const float4 factor = stage.factors[(position + i) >> 2];
    const float2 low = add_pair(make_float2(scores[i], scores[i + 1]), make_float2(-base, -base));
    const float2 high = add_pair(make_float2(scores[i + 2], scores[i + 3]), make_float2(-base, -base));
    scores[i] = exp2_fast(low.x); scores[i + 1] = exp2_fast(low.y); // 0 for a masked token
    scores[i + 2] = exp2_fast(high.x); scores[i + 3] = exp2_fast(high.y);
    sum = fmaf(scores[i], factor.x, sum); sum = fmaf(scores[i + 1], factor.y, sum);
    sum = fmaf(scores[i + 2], factor.z, sum); sum = fmaf(scores[i + 3], factor.w, sum);
  }
}
// Score i belongs to token part_token + local_token<...>(i) of the group: the first page's tokens below 32, the second's
// above. Which page that is, is known at compile time where the tokens are permuted and by the thread's part elsewhere.
template <bool kPermuted> __device__ __forceinline__ constexpr uint32_t local_token(uint32_t i) { return kPermuted ? 8 * (i & 7u) + (i >> 3) : i; }

// What a row (or all rows of a tile: the last one's position, the first one's window) sees of a group's two pages, which
// begin at tokens `first` and `second`.
struct GroupView {
  uint32_t first, second;
  bool both; // the group has a second page
  // every token, by their positions alone (the sinks aside)
  __device__ __forceinline__ bool whole(uint32_t position, uint32_t window_first) const {
    return both && first >= window_first && second + (kPageTokens - 1) <= position;
  }
  __device__ __forceinline__ uint32_t seen_first(uint32_t position, uint32_t window_first, uint32_t sinks) const {
    return seen_tokens(first, position, window_first, sinks);
  }
  __device__ __forceinline__ uint32_t seen_second(uint32_t position, uint32_t window_first, uint32_t sinks) const {
    return both ? seen_tokens(second, position, window_first, sinks) : 0u;
  }
};

} // namespace rk::tile
