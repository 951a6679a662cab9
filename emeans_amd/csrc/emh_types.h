// Loads and stores of the learning operators' element types, as f32 in
// registers: vectors of up to 16 bytes from any address that an element may
// have (the hardware takes unaligned global accesses).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace emh {

// Sixteen and eight bytes at an element's alignment.
struct __attribute__((packed, aligned(2))) Any16 {
  uint32_t w[4];
};
struct __attribute__((packed, aligned(2))) Any8 {
  uint32_t w[2];
};

typedef _Float16 f16;
typedef __bf16 bf16;

template <class T>
struct VecOf {
  static constexpr int N = 16 / sizeof(T);  // elements of a 16-byte vector
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(f16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(bf16 v) { return (float)v; }
template <class T>
__device__ __forceinline__ T from_f32(float v) {
  return (T)v;  // nearest, ties to even
}
// Two of a 16-bit type in one word, by one instruction.
template <class T>
__device__ __forceinline__ uint32_t pair_from_f32(float lo, float hi) {
  typedef float F2 __attribute__((ext_vector_type(2)));
  typedef T T2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((F2{lo, hi}), T2));
}

// A 16-byte vector's raw bits and its elements.
template <class T>
struct Vec {
  static constexpr int N = VecOf<T>::N;
  uint4 raw;
  __device__ __forceinline__ float get(int e) const {
    if constexpr (sizeof(T) == 4) {
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
      return __uint_as_float(w[e]);
    } else {
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
      const uint16_t b = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
      return to_f32(__builtin_bit_cast(T, b));
    }
  }
};
template <class T>
__device__ __forceinline__ Vec<T> load_vec(const T* p) {
  const Any16 a = *reinterpret_cast<const Any16*>(p);
  return Vec<T>{make_uint4(a.w[0], a.w[1], a.w[2], a.w[3])};
}
// The same of a 16-bit type where addresses may be odd multiples of two bytes, by whole
// words: lanes apart from each other are served a word at a time there otherwise.
// (What the words hold besides is not used; each holds an element of p's.)
template <class T>
__device__ __forceinline__ Vec<T> load_vec_words(const T* p) {
  static_assert(sizeof(T) == 2, "16 bits");
  const uint32_t odd = (uint32_t)(uintptr_t)p & 2;
  const T* from = reinterpret_cast<const T*>((uintptr_t)p - odd);
  struct __attribute__((packed, aligned(4))) Words {
    uint32_t w[4];
  };
  const Words a = *reinterpret_cast<const Words*>(from);
  const uint32_t last = *reinterpret_cast<const uint32_t*>(from + (odd ? 8 : 6));
  const uint32_t by = odd * 8;
  return Vec<T>{make_uint4(
      __builtin_amdgcn_alignbit(a.w[1], a.w[0], by), __builtin_amdgcn_alignbit(a.w[2], a.w[1], by),
      __builtin_amdgcn_alignbit(a.w[3], a.w[2], by), __builtin_amdgcn_alignbit(last, a.w[3], by))};
}
// The elements p[0 .. left), left < N; the others zero.
template <class T>
__device__ __forceinline__ Vec<T> load_some(const T* p, int left) {
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < VecOf<T>::N; e++) {
    if (e >= left) continue;
    if constexpr (sizeof(T) == 4)
      w[e] = __float_as_uint(p[e]);
    else
      w[e >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, p[e]) << (16 * (e & 1));
  }
  return Vec<T>{make_uint4(w[0], w[1], w[2], w[3])};
}
template <class T>
__device__ __forceinline__ void store_vec(T* p, const float* v) {
  Any16 a;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; e++) a.w[e] = __float_as_uint(v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) a.w[e] = pair_from_f32<T>(v[2 * e], v[2 * e + 1]);
  }
  *reinterpret_cast<Any16*>(p) = a;
}
template <class T>
__device__ __forceinline__ void store_vec(T* p, const Vec<T>& v) {
  *reinterpret_cast<Any16*>(p) = Any16{{v.raw.x, v.raw.y, v.raw.z, v.raw.w}};
}
template <class T>
__device__ __forceinline__ void store_some(T* p, const Vec<T>& v, int left) {
#pragma unroll
  for (int e = 0; e < VecOf<T>::N; e++)
    if (e < left) p[e] = from_f32<T>(v.get(e));
}
template <class T>
__device__ __forceinline__ void store_some(T* p, const float* v, int left) {
#pragma unroll
  for (int e = 0; e < VecOf<T>::N; e++)
    if (e < left) p[e] = from_f32<T>(v[e]);
}

// Stores that pass through the caches to memory at once: what a kernel leaves in them is written
// back at its end, when nothing else is left to do (a few us for the 32 MB that they hold). Where
// lines are stored in parts they cost more than they save. (Two idle cycles: the data's registers
// may be written next.)
template <class T>
__device__ __forceinline__ void through_vec(T* p, const Vec<T>& v) {
  typedef uint32_t any16 __attribute__((ext_vector_type(4)));
  const any16 q{v.raw.x, v.raw.y, v.raw.z, v.raw.w};
  asm volatile("global_store_dwordx4 %0, %1, off sc1\n\ts_nop 1" ::"v"(p), "v"(q) : "memory");
}
// Stores of what no cache need keep.
template <class T>
__device__ __forceinline__ void stream_vec(T* p, const Vec<T>& v) {
  typedef uint32_t any16 __attribute__((ext_vector_type(4), aligned(2)));
  __builtin_nontemporal_store(any16{v.raw.x, v.raw.y, v.raw.z, v.raw.w}, reinterpret_cast<any16*>(p));
}
template <class T>
__device__ __forceinline__ Vec<T> vec_of(const float* v) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; e++) {
    if constexpr (sizeof(T) == 4)
      w[e] = __float_as_uint(v[e]);
    else
      w[e] = pair_from_f32<T>(v[2 * e], v[2 * e + 1]);
  }
  return Vec<T>{make_uint4(w[0], w[1], w[2], w[3])};
}
template <class T>
__device__ __forceinline__ void stream_vec(T* p, const float* v) {
  stream_vec(p, vec_of<T>(v));
}
template <class T>
__device__ __forceinline__ void put_vec(bool through, T* p, const Vec<T>& v) {
  through ? through_vec(p, v) : store_vec(p, v);
}
template <class T>
__device__ __forceinline__ void put_vec(bool through, T* p, const float* v) {
  put_vec(through, p, vec_of<T>(v));
}

// Element i of a buffer whose kind is a run-time value (EMH_F32, EMH_F16,
// EMH_BF16).
__device__ __forceinline__ float load_kind(const void* p, int kind, size_t i) {
  if (kind == EMH_F32) return reinterpret_cast<const float*>(p)[i];
  if (kind == EMH_F16) return (float)reinterpret_cast<const f16*>(p)[i];
  return (float)reinterpret_cast<const bf16*>(p)[i];
}
__device__ __forceinline__ void store_kind(void* p, int kind, size_t i, float v) {
  if (kind == EMH_F32)
    reinterpret_cast<float*>(p)[i] = v;
  else if (kind == EMH_F16)
    reinterpret_cast<f16*>(p)[i] = (f16)v;
  else
    reinterpret_cast<bf16*>(p)[i] = (bf16)v;
}

// Reductions over groups of W consecutive lanes (16, 32 or 64), the result in
// every lane, without LDS: lane permutations within rows of 16 (neighbours, pairs,
// then mirrored halves and rows, whose lanes agree by then), and the swaps of rows
// and halves between two registers.
template <int CTRL>
__device__ __forceinline__ float lane_perm(float v) {
  return __int_as_float(
      __builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}
template <int W, class F>
__device__ __forceinline__ float lanes_reduce(float v, F&& f) {
  static_assert(W == 16 || W == 32 || W == 64, "group of lanes");
  v = f(v, lane_perm<0xB1>(v));   // quad_perm 1 0 3 2
  v = f(v, lane_perm<0x4E>(v));   // quad_perm 2 3 0 1
  v = f(v, lane_perm<0x141>(v));  // row_half_mirror
  v = f(v, lane_perm<0x140>(v));  // row_mirror
  if constexpr (W >= 32) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(s[0]), __uint_as_float(s[1]));
  }
  if constexpr (W == 64) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(s[0]), __uint_as_float(s[1]));
  }
  return v;
}
template <int W>
__device__ __forceinline__ float lanes_sum(float v) {
  return lanes_reduce<W>(v, [](float a, float b) { return a + b; });
}
template <int W>
__device__ __forceinline__ float lanes_max(float v) {
  return lanes_reduce<W>(v, [](float a, float b) { return fmaxf(a, b); });
}

}  // namespace emh
