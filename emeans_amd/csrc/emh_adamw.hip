// The AdamW step over many tensors in one launch.
//
// Every workgroup takes one chunk of one tensor, which a table on the device
// names (made once, with the plan); the chunks of all tensors are one grid, so a
// hundred small tensors cost one launch. A lane takes four consecutive elements at
// a time, a wave 256: the elements that share the scale of their 8-bit states, whose
// largest magnitude is then one reduction over the wave's lanes.
//
// m and the root of v are what is held in 8 bits, as e4m3 codes times the block's
// scale. The root, because its codes reach 2^17 below the block's largest (v
// itself would need twice the exponents); a positive v never gets the code zero,
// which would divide m by eps alone.
//
// Bound by HBM: 28 bytes an element with f32 parameters, gradients and states,
// 16 with 8-bit states, 10 with those and 16-bit parameters and gradients.
#include "emh_learn.h"
#include "emh_types.h"

namespace emh {
namespace {

constexpr float F8_TOP = 448.0f;             // the largest code
constexpr float F8_LEAST = 1.953125e-3f;     // the least positive one, 2^-9

__device__ __forceinline__ void load4_kind(const void* p, int kind, size_t i, int left, float* v) {
  if (left >= 4) {
    if (kind == EMH_F32) {
      const Any16 a = *reinterpret_cast<const Any16*>(reinterpret_cast<const float*>(p) + i);
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = __uint_as_float(a.w[e]);
    } else {
      const Any8 a = *reinterpret_cast<const Any8*>(reinterpret_cast<const uint16_t*>(p) + i);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const uint16_t b = (uint16_t)(a.w[e >> 1] >> (16 * (e & 1)));
        v[e] = kind == EMH_F16 ? (float)__builtin_bit_cast(f16, b)
                               : __uint_as_float((uint32_t)b << 16);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = e < left ? load_kind(p, kind, i + e) : 0.f;
  }
}
__device__ __forceinline__ void store4_kind(void* p, int kind, size_t i, int left, const float* v) {
  if (left >= 4) {
    if (kind == EMH_F32) {
      Any16 a;
#pragma unroll
      for (int e = 0; e < 4; e++) a.w[e] = __float_as_uint(v[e]);
      *reinterpret_cast<Any16*>(reinterpret_cast<float*>(p) + i) = a;
    } else {
      Any8 a;
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const uint16_t lo = kind == EMH_F16 ? __builtin_bit_cast(uint16_t, (f16)v[2 * e])
                                            : __builtin_bit_cast(uint16_t, (bf16)v[2 * e]);
        const uint16_t hi = kind == EMH_F16 ? __builtin_bit_cast(uint16_t, (f16)v[2 * e + 1])
                                            : __builtin_bit_cast(uint16_t, (bf16)v[2 * e + 1]);
        a.w[e] = (uint32_t)lo | (uint32_t)hi << 16;
      }
      *reinterpret_cast<Any8*>(reinterpret_cast<uint16_t*>(p) + i) = a;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (e < left) store_kind(p, kind, i + e, v[e]);
  }
}

struct __attribute__((packed, aligned(1))) Any4 {
  uint32_t w;
};
__device__ __forceinline__ uint32_t load4_codes(const void* p, size_t i, int left) {
  const uint8_t* b = reinterpret_cast<const uint8_t*>(p) + i;
  if (left >= 4) return reinterpret_cast<const Any4*>(b)->w;
  uint32_t w = 0;
  for (int e = 0; e < 3; e++)
    if (e < left) w |= (uint32_t)b[e] << (8 * e);
  return w;
}
__device__ __forceinline__ void store4_codes(void* p, size_t i, int left, uint32_t w) {
  uint8_t* b = reinterpret_cast<uint8_t*>(p) + i;
  if (left >= 4) {
    reinterpret_cast<Any4*>(b)->w = w;
    return;
  }
  for (int e = 0; e < 3; e++)
    if (e < left) b[e] = (uint8_t)(w >> (8 * e));
}
__device__ __forceinline__ void decode4(uint32_t w, float scale, float* v) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  v[0] = lo[0] * scale, v[1] = lo[1] * scale, v[2] = hi[0] * scale, v[3] = hi[1] * scale;
}
// The codes of v in a block whose scale this finds (a wave's 256 values).
template <bool LEAST>
__device__ __forceinline__ uint32_t encode4(const float* v, float& scale) {
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const float m = fabsf(v[e]);
    top = fmaxf(top, m <= 3.4028235e38f ? m : 0.f);
  }
  scale = lanes_max<64>(top) * (1.f / F8_TOP);
  // (One reciprocal a block: a code near a tie may be its neighbour. Finite, or a
  // zero in a block of the least numbers would become a NaN.)
  const float by = fminf(__builtin_amdgcn_rcpf(scale), 3.4028235e38f);
  float q[4];
#pragma unroll
  for (int e = 0; e < 4; e++) {
    q[e] = v[e] * by;
    if (LEAST && v[e] > 0.f && q[e] < F8_LEAST) q[e] = F8_LEAST;
    // (A quotient that rounded past the top; infinities and NaN become the NaN code.)
    if (fabsf(v[e]) <= 3.4028235e38f)
      q[e] = fminf(fmaxf(q[e], -F8_TOP), F8_TOP);
    else
      q[e] = __builtin_nanf("");
  }
  uint32_t w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], (int)w, true);
}

// sqrt(v) within a unit in the last place, below the normal range too (where
// the instruction takes zero for v).
__device__ __forceinline__ float root(float v) {
  const bool small = v < 1.17549435e-38f;
  const float t = __builtin_amdgcn_sqrtf(small ? v * 18446744073709551616.f : v);  // 2^64
  return small ? t * 2.3283064365386963e-10f : t;                                  // 2^-32
}

template <int U>  // a chunk: 1024 U elements
__global__ __launch_bounds__(256) void k_adamw(const AdamTensor* __restrict__ tensors,
                                               const uint2* __restrict__ chunks,
                                               const AdamScalars s) {
  const uint2 at = chunks[blockIdx.x];
  const AdamTensor t = tensors[at.x];
  const size_t base = (size_t)at.y * (1024 * U);
  const size_t here = t.len - base;  // > 0
  const int lane4 = (int)threadIdx.x * 4;
  const bool eight = t.m_scale != nullptr;
  const float keep = (float)(1.0 - s.lr * t.weight_decay);
  float p[U][4], g[U][4], m[U][4], v[U][4];
  uint32_t mc[U], vc[U];
  float msc[U], vsc[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int o = u * 1024 + lane4;
    const int left = (int)min((size_t)(1024 * U), here) - o;
    const size_t i = base + o;
    load4_kind(t.param, t.param_kind, i, left, p[u]);
    load4_kind(t.grad, t.grad_kind, i, left, g[u]);
    if (eight) {
      mc[u] = load4_codes(t.m, i, left);
      vc[u] = load4_codes(t.v, i, left);
      msc[u] = left > 0 ? t.m_scale[i / EMH_ADAMW_BLOCK] : 0.f;
      vsc[u] = left > 0 ? t.v_scale[i / EMH_ADAMW_BLOCK] : 0.f;
    } else {
      load4_kind(t.m, EMH_F32, i, left, m[u]);
      load4_kind(t.v, EMH_F32, i, left, v[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int o = u * 1024 + lane4;
    const int left = (int)min((size_t)(1024 * U), here) - o;
    const size_t i = base + o;
    if (eight) {
      decode4(mc[u], msc[u], m[u]);
      decode4(vc[u], vsc[u], v[u]);
#pragma unroll
      for (int e = 0; e < 4; e++) v[u][e] *= v[u][e];
    }
    float r[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float ge = g[u][e] * s.gscale;
      m[u][e] = s.beta1 * m[u][e] + s.new1 * ge;
      v[u][e] = s.beta2 * v[u][e] + s.new2 * ge * ge;
      // The root and the quotient within two units of the last place (the correctly
      // rounded ones are twenty instructions each, which bounded the step: 595 us at
      // 134 million elements).
      r[e] = root(v[u][e]);
      const float by = m[u][e] * __builtin_amdgcn_rcpf(r[e] * s.root2 + s.eps);
      p[u][e] = p[u][e] * keep - s.rate * by;
    }
    store4_kind(t.param, t.param_kind, i, left, p[u]);
    if (t.copy) store4_kind(t.copy, t.copy_kind, i, left, p[u]);
    if (eight) {
      // (Elements past the tensor's end are zeros here and have no part in the scale.)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        r[e] = e < left ? r[e] : 0.f;
        m[u][e] = e < left ? m[u][e] : 0.f;
      }
      float ms, vs;
      const uint32_t a = encode4<false>(m[u], ms), b = encode4<true>(r, vs);
      store4_codes(t.m, i, left, a);
      store4_codes(t.v, i, left, b);
      if ((threadIdx.x & 63) == 0 && left > 0) {
        t.m_scale[i / EMH_ADAMW_BLOCK] = ms;
        t.v_scale[i / EMH_ADAMW_BLOCK] = vs;
      }
    } else {
      store4_kind(t.m, EMH_F32, i, left, m[u]);
      store4_kind(t.v, EMH_F32, i, left, v[u]);
    }
  }
}

}  // namespace

void launch_adamw(emh_ctx* c, const AdamTensor* tensors, const uint2* chunks, size_t nchunks,
                  size_t chunk, const AdamScalars& s) {
  if (nchunks == 0) return;
  const dim3 grid((unsigned)nchunks);
  if (chunk == ADAM_CHUNK)
    k_adamw<(int)(ADAM_CHUNK / 1024)><<<grid, 256, 0, c->stream>>>(tensors, chunks, s);
  else
    k_adamw<(int)(ADAM_CHUNK_FEW / 1024)><<<grid, 256, 0, c->stream>>>(tensors, chunks, s);
  EMH_HIP(hipGetLastError());
}

}  // namespace emh
