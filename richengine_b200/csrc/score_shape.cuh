// score_shape.cuh — what a score goes through between the contraction and the softmax (rk_score_shape): a tanh cap, a
// bias that falls with the distance, a sliding window with sink tokens; and the pages that such a row reads.
//
//   x = scale * q.k            x = cap * tanh(x / cap)  (cap > 0)            x -= slope * (p - t)  (slopes given)
//   seen(p, t) = t <= p and (window == 0 or p - t < window or t < sink_tokens)
//
// The kernels hold scores in the log2 domain (x * log2 e), so the cap and the slopes come multiplied by log2 e.
#pragma once

#include "common.cuh"

namespace rk {

struct ShapeArgs {
  float cap = 0.0f;        // cap * log2 e; 0: none
  float cap_inverse = 0.0f; // 1 / (cap * log2 e)
  uint32_t window = 0;     // 0: every token up to the row's own
  uint32_t sinks = 0;      // with a window: tokens that stay visible at the start of the sequence
  const float *slopes = nullptr; // [query head], device memory; null: none
};

// Host side: the launch arguments of a shape (null: none). False when a field is out of range.
inline bool shape_arguments(const rk_score_shape *shape, ShapeArgs &out) {
  out = ShapeArgs{};
  if (!shape) return true;
  if (!(shape->softcap >= 0.0f) || shape->softcap > 1.0e30f || (shape->softcap > 0.0f && shape->softcap < 1.0e-30f)) return false;
  if (shape->softcap > 0.0f) {
    out.cap = shape->softcap * 1.4426950408889634f;
    out.cap_inverse = 1.0f / out.cap;
  }
  out.window = shape->window;
  out.sinks = shape->window ? shape->sink_tokens : 0;
  out.slopes = shape->slopes;
  return true;
}

// Two fp32 operations in one instruction, each rounded as on its own.
__device__ __forceinline__ float2 fma_pair(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\nfma.rn.f32x2 x, x, y, z;\nmov.b64 {%0, %1}, x;\n}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 mul_pair(float2 a, float2 b) {
  float2 r;
  asm("{\n.reg .b64 x, y;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmul.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 add_pair(float2 a, float2 b) {
  float2 r;
  asm("{\n.reg .b64 x, y;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nadd.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

// cap * tanh(s / cap) for N scores, tanh(u) = 1 - 2 / (e^2u + 1). The hardware's own tanh (2^-11) would move a score of 30
// by 0.015. Four scores share one reciprocal (1/a = b c d / (a b c d)): five special-function operations for four scores instead
// of eight; four lanes over 32K int4 tokens: 115 us, and 121 with a reciprocal each (86 without a cap: what the cap adds is the
// length of a group's chain, the special-function unit is a third busy). e^2u stops at 2^30, where the quotient is under half a
// step of one, so that four of them stay finite.
// Error of this form, in units of cap * 2^-23, from the sum of its roundings with q = 1 / (e^2u + 1) <= 1: the exponent's six
// (its scale and products) 2 * 0.67, ex2 (2^-22) and the sum with one 2 * (0.5 + 0.5), the reciprocal (2^-23) and four products
// 2 * 3, the last multiply-add 0.5: under 10, cap * 2^-19.7 (the worst of 80 million scores was cap * 2^-20.8 in a replay with
// exact ex2 and rcp). Caps up to 64 take it: under 2^-13 on a score, a quarter of what rounding the weights to 11 bits allows.
// Beyond, scores are small against the cap and the difference from one loses them: below |u| = 1/4 the odd series u (1 - u^2/3 +
// 2u^4/15 - 17u^6/315 + 62u^8/2835), whose next term is under 10^-8 there, takes over, and the result is good to about 10^-6 of
// itself (the four lanes: 123 us with a cap of 100, 110 with one of 50).
// A score that is no number stays one, and takes the three that share its reciprocal with it: callers pass scores of one query
// row, s[4i] .. s[4i + 3], and give tokens that the row does not see (their keys may hold anything) a finite score beforehand.
constexpr float kDirectCap = 64.0f * 1.4426950408889634f;
__device__ __forceinline__ float exp2_special(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// The smaller of two, a NaN when either is one (fminf would return the other).
__device__ __forceinline__ float minimum_or_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float reciprocal_special(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
template <uint32_t N> __device__ __forceinline__ void soft_cap(float (&s)[N], float cap, float cap_inverse) {
  static_assert(N % 4 == 0, "four scores share a reciprocal");
  const float factor = cap_inverse * 2.8853900817779268f; // e^2u = 2^(2u log2 e)
  if (cap <= kDirectCap) { // the same branch for the whole launch
    const float2 one = make_float2(1.0f, 1.0f), caps = make_float2(cap, cap), down = make_float2(-2.0f * cap, -2.0f * cap);
#pragma unroll
    for (uint32_t i = 0; i < N; i += 4) {
      float e[4];
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) e[k] = exp2_special(minimum_or_nan(s[i + k] * factor, 30.0f));
      const float2 a = add_pair(make_float2(e[0], e[1]), one), b = add_pair(make_float2(e[2], e[3]), one), ab = mul_pair(a, b);
      const float r = reciprocal_special(ab.x * ab.y);
      const float2 both = make_float2(r * ab.y, r * ab.x); // 1 / ab
      const float2 low = fma_pair(mul_pair(both, b), down, caps), high = fma_pair(mul_pair(both, a), down, caps);
      s[i] = low.x; s[i + 1] = low.y; s[i + 2] = high.x; s[i + 3] = high.y;
    }
  } else {
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
      const float u = s[i] * cap_inverse, u2 = u * u;
      float near = fmaf(u2, 0.021869489f, -0.053968254f);
      near = fmaf(u2, near, 0.13333333f);
      near = fmaf(u2, near, -0.33333333f);
      near = fmaf(u2 * s[i], near, s[i]);
      s[i] = fmaf(-2.0f * cap, reciprocal_special(exp2_special(s[i] * factor) + 1.0f), cap);
      // a select, not a branch: branches would keep both sides of every score alive (a NaN stays one)
      asm("{\n.reg .pred p;\nsetp.lt.f32 p, %2, 0f3D800000;\nselp.f32 %0, %1, %0, p;\n}" : "+f"(s[i]) : "f"(near), "f"(u2));
    }
  }
}

// The pages of tokens 0..last_position that rows at first_position and later read, as a list: page(o) for o < count. Pages before
// `skip` belong to someone else (a shared prefix); of the rest, those with a sink token and those from the first row's
// window on.
struct PageList {
  uint32_t begin, head, gap, count;  // page(o) = begin + o, + gap from o == head on
  uint32_t window_first;             // first token of the first row's window
  __device__ __forceinline__ static PageList make(uint32_t first_position, uint32_t last_position, uint32_t skip, const ShapeArgs &shape) {
    PageList list;
    const uint32_t pages = last_position / kPageTokens + 1;
    list.window_first = shape.window && first_position + 1 > shape.window ? first_position + 1 - shape.window : 0;
    list.begin = min(skip, pages);
    const uint32_t sinks_end = max(list.begin, rk_pages_for(min(shape.sinks, last_position + 1)));
    // (The first row may lie behind the last position and its window with it: then the list keeps the last page, seen by none.)
    const uint32_t window_begin = max(list.begin, min(list.window_first / kPageTokens, pages - 1));
    if (window_begin <= sinks_end) {
      list.head = list.count = pages - list.begin;
      list.gap = 0;
    } else {
      list.head = sinks_end - list.begin;
      list.gap = window_begin - sinks_end;
      list.count = list.head + pages - window_begin;
    }
    return list;
  }
  __device__ __forceinline__ uint32_t page(uint32_t o) const { return begin + o + (o >= head ? gap : 0); }
};

// Bit i: the token `base + i` of a page (32-aligned base) is seen by a row at first_position or by one up to `last_position`
// (`window_first` = first token of the first row's window).
__device__ __forceinline__ uint32_t seen_tokens(uint32_t base, uint32_t last_position, uint32_t window_first, uint32_t sinks) {
  auto below = [](uint32_t end) { return end >= 32 ? 0xffffffffu : (1u << end) - 1u; };
  const uint32_t present = last_position < base ? 0u : below(last_position - base + 1);
  const uint32_t old = window_first <= base ? 0u : below(window_first - base);
  const uint32_t sink = sinks <= base ? 0u : below(sinks - base);
  return present & (~old | sink);
}

} // namespace rk
