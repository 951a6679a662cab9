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
// which would divide m by eps alone. Rounded to the nearest code, a state follows its
// average only where a step moves it by half a code, which beta2 near 1 never does; a plan
// with a seed rounds at random (RANDOM), in the proportion that keeps the mean.
//
// Bound by HBM: 28 bytes an element with f32 parameters, gradients and states,
// 16 with 8-bit states, 10 with those and 16-bit parameters and gradients.
#include <type_traits>

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
// The codes of v in a block whose scale this finds (a wave's 256 values). The
// quotients are correctly rounded (one reciprocal a block, refined, then a product
// and its remainder): a code one step off changes a small root by up to half, and
// the parameter's step with it. A quotient is at most 448 (1 + 2^-23), which rounds to
// 448; infinities and NaN become the NaN code.
// RANDOM: the code above or below, as bits' top 20 decide.
template <bool LEAST, bool RANDOM>
__device__ __forceinline__ uint32_t encode4(const float* v, float& scale, const uint32_t* bits) {
  float top = lanes_max<64>(fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3]))));
  top = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(top)));  // (the wave's)
  if (!(top < INFINITY)) {  // without the infinite ones (the maximum passes over NaN)
    top = 0.f;
#pragma unroll
    for (int e = 0; e < 4; e++) top = fmaxf(top, fabsf(v[e]) < INFINITY ? fabsf(v[e]) : 0.f);
    top = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(lanes_max<64>(top))));
  }
  scale = top * (1.f / F8_TOP);
  float q[4];
  if (scale > 1e-30f && scale < 1e30f) {
    const float r0 = __builtin_amdgcn_rcpf(scale);
    const float by = fmaf(r0, fmaf(-scale, r0, 1.f), r0);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float q0 = v[e] * by;
      q[e] = fmaf(fmaf(-scale, q0, v[e]), by, q0);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) q[e] = scale > 0.f ? v[e] / scale : v[e];
  }
  if (LEAST) {
#pragma unroll
    for (int e = 0; e < 4; e++) q[e] = v[e] > 0.f && q[e] < F8_LEAST ? F8_LEAST : q[e];
  }
  if constexpr (RANDOM) {
    // (Bits below the code's last are added to and cut off; past 448 lies the NaN.)
#pragma unroll
    for (int e = 0; e < 4; e++)
      q[e] = fabsf(q[e]) < INFINITY ? fminf(fmaxf(q[e], -F8_TOP), F8_TOP) : q[e];
    int w = __builtin_amdgcn_cvt_sr_fp8_f32(q[0], (int)bits[0], 0, 0);
    w = __builtin_amdgcn_cvt_sr_fp8_f32(q[1], (int)bits[1], w, 1);
    w = __builtin_amdgcn_cvt_sr_fp8_f32(q[2], (int)bits[2], w, 2);
    return (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(q[3], (int)bits[3], w, 3);
  }
  const uint32_t w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], (int)w, true);
}

// Random bits for a lane's four elements of block `block` of a tensor: for m, and, the
// same backwards, for v (20 of 32 bits each count, the first twelve of them alone in one
// of the two). Multiplications by odd numbers between shifts; of lanes, elements,
// blocks, tensors and steps no two are correlated beyond chance over 2^20 samples.
__device__ __forceinline__ uint32_t mixed(uint32_t h) {
  h = (h ^ h >> 16) * 0x9E3779B1u;
  h = (h ^ h >> 14) * 0xA2F9836Bu;
  return h ^ h >> 15;
}
__device__ __forceinline__ void random4(const AdamScalars& s, uint32_t tensor, size_t block,
                                        uint32_t* m, uint32_t* v) {
  const uint32_t b = mixed(mixed(s.key0 + tensor) ^ (uint32_t)block) + s.key1 +
                     (uint32_t)(block >> 32) * 0x9E3779B1u;
  const uint32_t l = mixed(b ^ (threadIdx.x & 63));
#pragma unroll
  for (uint32_t e = 0; e < 4; e++) {
    uint32_t h = l + e * 0x9E3779B1u;
    h = (h ^ h >> 15) * 0xA2F9836Bu;
    m[e] = h ^ h >> 16;
    v[e] = __brev(m[e]);
  }
}

// One element's step; r: the root of the new v.
__device__ __forceinline__ void step1(const AdamScalars& s, float keep, float& p, float g, float& m,
                                      float& v, float& r) {
  const float ge = g * s.gscale;
  m = s.beta1 * m + s.new1 * ge;
  v = s.beta2 * v + s.new2 * ge * ge;
  r = sqrtf(v);
  // The quotient within two units of the last place (the correctly rounded one is
  // twenty instructions).
  p = p * keep - s.rate * (m * __builtin_amdgcn_rcpf(r * s.root2 + s.eps));
}

// Vectors in global memory (a pointer that comes from a table is otherwise taken to be
// of any address space) at any element's address.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32_any __attribute__((aligned(1)));
#define EMH_GLOBAL __attribute__((address_space(1)))
template <class V>
__device__ __forceinline__ V gload(const void* p, size_t byte) {
  return *(const EMH_GLOBAL V*)((const EMH_GLOBAL char*)p + byte);
}
template <class V>
__device__ __forceinline__ void gstore(void* p, size_t byte, V v) {
  *(EMH_GLOBAL V*)((EMH_GLOBAL char*)p + byte) = v;
}
__device__ __forceinline__ void unpack16(u32x2_any w, int kind, float* v) {
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const uint16_t b = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
    v[e] = kind == EMH_F16 ? (float)__builtin_bit_cast(f16, b) : __uint_as_float((uint32_t)b << 16);
  }
}
template <class T>
__device__ __forceinline__ u32x2_any pack16_of(const float* v) {
  u32x2_any w;
#pragma unroll
  for (int e = 0; e < 2; e++)
    w[e] = (uint32_t)__builtin_bit_cast(uint16_t, (T)v[2 * e]) |
           (uint32_t)__builtin_bit_cast(uint16_t, (T)v[2 * e + 1]) << 16;
  return w;
}
__device__ __forceinline__ u32x2_any pack16(const float* v, int kind) {
  return kind == EMH_F16 ? pack16_of<f16>(v) : pack16_of<bf16>(v);
}
__device__ __forceinline__ void unpack32(u32x4_any w, float* v) {
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = __uint_as_float(w[e]);
}
__device__ __forceinline__ u32x4_any pack32(const float* v) {
  u32x4_any w;
#pragma unroll
  for (int e = 0; e < 4; e++) w[e] = __float_as_uint(v[e]);
  return w;
}

// A whole chunk: every load goes out before the first is used.
template <int U, bool P16, bool G16, bool EIGHT, bool RANDOM>
__device__ __forceinline__ void whole_chunk(const AdamTensor& t, uint32_t tensor,
                                            const AdamScalars& s, size_t base) {
  const float keep = (float)(1.0 - s.lr * t.weight_decay);
  const size_t i0 = base + threadIdx.x * 4;
  u32x4_any p4[P16 ? 1 : U], g4[G16 ? 1 : U], m4[EIGHT ? 1 : U], v4[EIGHT ? 1 : U];
  u32x2_any p2[P16 ? U : 1], g2[G16 ? U : 1];
  uint32_t mc[U], vc[U];
  float msc[U], vsc[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const size_t i = i0 + u * 1024;
    if constexpr (P16)
      p2[u] = gload<u32x2_any>(t.param, i * 2);
    else
      p4[u] = gload<u32x4_any>(t.param, i * 4);
    if constexpr (G16)
      g2[u] = gload<u32x2_any>(t.grad, i * 2);
    else
      g4[u] = gload<u32x4_any>(t.grad, i * 4);
    if constexpr (EIGHT) {
      mc[u] = gload<u32_any>(t.m, i);
      vc[u] = gload<u32_any>(t.v, i);
      const size_t block = i / EMH_ADAMW_BLOCK;  // (a wave's)
      msc[u] = gload<float>(t.m_scale, block * 4);
      vsc[u] = gload<float>(t.v_scale, block * 4);
    } else {
      m4[u] = gload<u32x4_any>(t.m, i * 4);
      v4[u] = gload<u32x4_any>(t.v, i * 4);
    }
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    const size_t i = i0 + u * 1024;
    float p[4], g[4], m[4], v[4], r[4];
    if constexpr (P16)
      unpack16(p2[u], t.param_kind, p);
    else
      unpack32(p4[u], p);
    if constexpr (G16)
      unpack16(g2[u], t.grad_kind, g);
    else
      unpack32(g4[u], g);
    if constexpr (EIGHT) {
      decode4(mc[u], msc[u], m);
      decode4(vc[u], vsc[u], v);
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] *= v[e];
    } else {
      unpack32(m4[u], m);
      unpack32(v4[u], v);
    }
#pragma unroll
    for (int e = 0; e < 4; e++) step1(s, keep, p[e], g[e], m[e], v[e], r[e]);
    if constexpr (P16)
      gstore(t.param, i * 2, pack16(p, t.param_kind));
    else
      gstore(t.param, i * 4, pack32(p));
    if (t.copy) gstore(t.copy, i * 2, pack16(p, t.copy_kind));
    if constexpr (EIGHT) {
      float ms, vs;
      uint32_t rm[4], rv[4];
      if constexpr (RANDOM)
        random4(s, tensor, (base >> 8) + u * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6),
                rm, rv);
      const uint32_t a = encode4<false, RANDOM>(m, ms, rm), b = encode4<true, RANDOM>(r, vs, rv);
      gstore<u32_any>(t.m, i, a);
      gstore<u32_any>(t.v, i, b);
      if ((threadIdx.x & 63) == 0) {
        gstore(t.m_scale, i / EMH_ADAMW_BLOCK * 4, ms);
        gstore(t.v_scale, i / EMH_ADAMW_BLOCK * 4, vs);
      }
    } else {
      gstore(t.m, i * 4, pack32(m));
      gstore(t.v, i * 4, pack32(v));
    }
  }
}

// A tensor's last chunk: fours that may be cut short.
template <bool RANDOM>
__device__ __forceinline__ void last_chunk(const AdamTensor& t, uint32_t tensor,
                                           const AdamScalars& s, size_t base, int count) {
  const float keep = (float)(1.0 - s.lr * t.weight_decay);
  for (int o = (int)threadIdx.x * 4; o < ((count + 255) & ~255); o += 1024) {
    const int left = count - o;  // (whole waves come here together: a block's scale is theirs)
    const size_t i = base + o;
    float p[4], g[4], m[4], v[4], r[4];
    load4_kind(t.param, t.param_kind, i, left, p);
    load4_kind(t.grad, t.grad_kind, i, left, g);
    if (t.m_scale) {
      const size_t block = i / EMH_ADAMW_BLOCK;
      decode4(load4_codes(t.m, i, left), t.m_scale[block], m);
      decode4(load4_codes(t.v, i, left), t.v_scale[block], v);
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] *= v[e];
    } else {
      load4_kind(t.m, EMH_F32, i, left, m);
      load4_kind(t.v, EMH_F32, i, left, v);
    }
#pragma unroll
    for (int e = 0; e < 4; e++) step1(s, keep, p[e], g[e], m[e], v[e], r[e]);
    store4_kind(t.param, t.param_kind, i, left, p);
    if (t.copy) store4_kind(t.copy, t.copy_kind, i, left, p);
    if (t.m_scale) {
      // (Elements past the tensor's end are zeros here and have no part in the scale.)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        r[e] = e < left ? r[e] : 0.f;
        m[e] = e < left ? m[e] : 0.f;
      }
      float ms, vs;
      uint32_t rm[4], rv[4];
      if constexpr (RANDOM) random4(s, tensor, i / EMH_ADAMW_BLOCK, rm, rv);
      const uint32_t a = encode4<false, RANDOM>(m, ms, rm), b = encode4<true, RANDOM>(r, vs, rv);
      store4_codes(t.m, i, left, a);
      store4_codes(t.v, i, left, b);
      if ((threadIdx.x & 63) == 0) {
        t.m_scale[i / EMH_ADAMW_BLOCK] = ms;
        t.v_scale[i / EMH_ADAMW_BLOCK] = vs;
      }
    } else {
      store4_kind(t.m, EMH_F32, i, left, m);
      store4_kind(t.v, EMH_F32, i, left, v);
    }
  }
}

// A chunk: 1024 U elements. 131,071 x 1,024 and two layers in bf16 with 8-bit states,
// 10 bytes an element: 275 us, 4.9 TB/s, rounded at random 316; 256 x 384 f32 3.3 us, a launch.
// CLIP: the gradients times clip[1] too; a NaN there leaves everything as it is.
template <int U, bool RANDOM, bool CLIP>
__global__ __launch_bounds__(256) void k_adamw(const AdamTensor* __restrict__ tensors,
                                               const uint2* __restrict__ chunks,
                                               const AdamScalars given,
                                               const float* __restrict__ clip) {
  AdamScalars s = given;
  if constexpr (CLIP) {
    const float f = clip[1];
    if (!(f == f)) return;
    s.gscale *= f;
  }
  const uint2 at = chunks[blockIdx.x];
  const AdamTensor t = tensors[at.x];
  const size_t base = (size_t)at.y * (1024 * U);
  const size_t here = t.len - base;  // > 0
  if (here < (size_t)(1024 * U)) {
    last_chunk<RANDOM>(t, at.x, s, base, (int)here);
    return;
  }
  const bool p16 = t.param_kind != EMH_F32, g16 = t.grad_kind != EMH_F32;
  if (t.m_scale) {
    if (p16)
      g16 ? whole_chunk<U, true, true, true, RANDOM>(t, at.x, s, base)
          : whole_chunk<U, true, false, true, RANDOM>(t, at.x, s, base);
    else
      g16 ? whole_chunk<U, false, true, true, RANDOM>(t, at.x, s, base)
          : whole_chunk<U, false, false, true, RANDOM>(t, at.x, s, base);
  } else {
    if (p16)
      g16 ? whole_chunk<U, true, true, false, RANDOM>(t, at.x, s, base)
          : whole_chunk<U, true, false, false, RANDOM>(t, at.x, s, base);
    else
      g16 ? whole_chunk<U, false, true, false, RANDOM>(t, at.x, s, base)
          : whole_chunk<U, false, false, false, RANDOM>(t, at.x, s, base);
  }
}

}  // namespace

void launch_adamw(emh_ctx* c, const AdamTensor* tensors, const uint2* chunks, size_t nchunks,
                  size_t chunk, bool random, const AdamScalars& s, const float* clip) {
  if (nchunks == 0) return;
  const dim3 grid((unsigned)nchunks);
  auto go = [&](auto kernel) { kernel<<<grid, 256, 0, c->stream>>>(tensors, chunks, s, clip); };
  constexpr int MANY = (int)(ADAM_CHUNK / 1024), FEW = (int)(ADAM_CHUNK_FEW / 1024);
  auto with = [&](auto clipped) {
    constexpr bool CLIP = decltype(clipped)::value;
    if (chunk == ADAM_CHUNK)
      random ? go(k_adamw<MANY, true, CLIP>) : go(k_adamw<MANY, false, CLIP>);
    else
      random ? go(k_adamw<FEW, true, CLIP>) : go(k_adamw<FEW, false, CLIP>);
  };
  clip ? with(std::true_type{}) : with(std::false_type{});
  EMH_HIP(hipGetLastError());
}

}  // namespace emh
