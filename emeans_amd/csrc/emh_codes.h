// 8-bit codes (e4m3) of a block that shares a scale: scale = largest magnitude / 448, code =
// the nearest to value / scale. Both quotients are correctly rounded, so that the codes
// follow from the values alone: a code one step off is a sixteenth of its value.
#pragma once

#include "emh_types.h"

namespace emh {

constexpr int CODE_BLOCK = EMH_CODE_BLOCK;  // columns that share a scale

// The largest magnitude counts finite values alone (an element that is not finite gets the
// NaN code and has no part in the scale).
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a < INFINITY ? a : 0.f;
}

// The code of a block's values. L lanes have it, v[count] each, and all of the wave's come here.
struct Coder {
  float scale, by;
  bool quick;  // (the wave's)
  // Infinite values apart, and scales whose quotients need the division, a scale is a product
  // and its remainder, and so is every quotient by it: correctly rounded.
  template <int L>
  __device__ __forceinline__ static Coder of(const float* v, int count) {
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < count; e++) top = fmaxf(top, fabsf(v[e]));  // (passes over NaN)
    return Coder(lanes_max<L>(top), [&]() __attribute__((always_inline)) {
      float t = 0.f;
#pragma unroll
      for (int e = 0; e < count; e++) t = fmaxf(t, finite_abs(v[e]));
      return lanes_max<L>(t);
    });
  }
  // top: the largest magnitude, infinite ones among it; finite(): without them.
  template <class F>
  __device__ __forceinline__ Coder(float top, F&& finite) {
    quick = __all((top > 1e-25f && top < 1e30f) || top == 0.f);
    if (quick) {
      constexpr float PER = 1.f / 448.f;
      const float q = top * PER;
      scale = fmaf(fmaf(-448.f, q, top), PER, q);
      const float s = top > 0.f ? scale : 1.f, r0 = __builtin_amdgcn_rcpf(s);
      by = fmaf(r0, fmaf(-s, r0, 1.f), r0);
    } else {
      scale = finite() / 448.f;
      by = 0.f;
    }
  }
  // A quotient: at most 448 (1 + 2^-23), which rounds to 448.
  __device__ __forceinline__ float quotient(float v) const {
    if (quick) {
      const float q = v * by;
      // (The remainder of a negative zero is a positive one.)
      return copysignf(fmaf(fmaf(-scale, q, v), by, q), v);
    }
    // (Without a scale the values are zeros, or below what a code can hold of them; one
    // among the last subnormal numbers may be small by half of itself.)
    const float q = scale > 0.f ? v / scale : v;
    return fabsf(q) < INFINITY ? fminf(fmaxf(q, -448.f), 448.f) : q;
  }
  __device__ __forceinline__ uint32_t four(const float* v) const {
    const uint32_t w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(quotient(v[0]), quotient(v[1]), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(quotient(v[2]), quotient(v[3]), (int)w, true);
  }
};

// The codes of N (4 or 8) columns from `col` on, the first `skip` of v other columns', to a
// row of codes (its start 16-byte aligned); zeros from the row's d columns to its next
// multiple of 16. through: eight codes pass through the caches at once (emh_types.h). Coding alone does
// that where rows of codes are whole 64 bytes (16,384 x 768 bf16 7.9 us, written back at the end 8.6;
// 30,000 x 1,000, whose 1,008 bytes straddle lines, 19.9 and 17.4); the norm by its rows' size
// (launch_rms_norm).
template <int N>
__device__ __forceinline__ void store_codes(uint8_t* row, int col, int skip, int d, const Coder& c,
                                            const float* v, bool through) {
  static_assert(N == 4 || N == 8, "codes of a vector");
  if constexpr (N == 8) {
    uint64_t w = (uint64_t)c.four(v) | (uint64_t)c.four(v + 4) << 32;
    w >>= 8 * skip;
    if (through)
      __hip_atomic_store(reinterpret_cast<uint64_t*>(row + col), w, __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
    else
      *reinterpret_cast<uint2*>(row + col) = make_uint2((uint32_t)w, (uint32_t)(w >> 32));
  } else {
    *reinterpret_cast<uint32_t*>(row + col) = c.four(v) >> (8 * skip);
  }
  if (col + N >= d)
    for (int t = col + N; t < ((d + 15) & ~15); t += 4) *reinterpret_cast<uint32_t*>(row + t) = 0u;
}

}  // namespace emh
