// The global norm of many tensors, and their elements brought to a largest one.
//
// norm = |scale| sqrt(sum g^2) over all elements of all tensors, factor = min(1, max_norm /
// norm). Squares and sums are in f64: no f32 square overflows or vanishes there, and the sum of
// 2^27 elements is as good as its rounding to f32.
//
// Two launches. The first leaves one sum a workgroup (at most NORM_SUMS, over chunks that a
// table on the device names); in the second every workgroup adds those sums, in one order, and so
// has the norm and the factor, and scales its chunks, the last ones first: what the first launch
// read last is what the caches may still hold, if results that exceed them go past them (131 M
// bf16 elements 156 us, then 128). No atomics: results follow from the tensors alone.
//
// Bound by HBM: two reads and one write of an element (131,071 x 1,001 bf16 124 us, 6.3 TB/s of
// those three, the second read in part from the caches; 99,072 f32, two launches, 5.6 to 7.5 us; 4 M
// f32 10.1, results through the caches, without that 12.6; at odd addresses 10.9 and 12.7, and 50 M
// bf16 50.6 and 50.1).
// Where the gradients are scaled in place and the factor is 1 the second read and the write are
// left out.
#include "emh_answer.h"
#include "emh_types.h"

namespace emh {
namespace {

__device__ __forceinline__ double lanes_sum64(double v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// The workgroup's sum, in all of its threads.
__device__ __forceinline__ double group_sum(double v, double* red) {
  v = lanes_sum64(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

template <class T>
__device__ __forceinline__ double square_sum(const T* p, size_t count) {
  constexpr int N = VecOf<T>::N;
  double s[2] = {0.0, 0.0};
  const size_t whole = count / N;
#pragma unroll 4
  for (size_t i = threadIdx.x; i < whole; i += 256) {
    const Vec<T> v = load_vec(p + i * N);
#pragma unroll
    for (int e = 0; e < N; e++) {
      const double x = (double)v.get(e);
      s[e & 1] = fma(x, x, s[e & 1]);
    }
  }
  const size_t i = whole * N + threadIdx.x;
  if (i < count) {
    const double x = (double)to_f32(p[i]);
    s[0] = fma(x, x, s[0]);
  }
  return s[0] + s[1];
}

__global__ __launch_bounds__(256) void k_square_sums(const NormTensor* __restrict__ tensors,
                                                     const uint2* __restrict__ chunks,
                                                     uint32_t nchunks, uint32_t chunk,
                                                     double* sums) {
  __shared__ double red[4];
  double s = 0.0;
  for (uint32_t i = blockIdx.x; i < nchunks; i += gridDim.x) {
    const uint2 at = chunks[i];
    const NormTensor t = tensors[at.x];
    const size_t base = (size_t)at.y * chunk, count = min(t.len - base, (size_t)chunk);
    if (t.kind == EMH_F32)
      s += square_sum(reinterpret_cast<const float*>(t.grad) + base, count);
    else if (t.kind == EMH_F16)
      s += square_sum(reinterpret_cast<const f16*>(t.grad) + base, count);
    else
      s += square_sum(reinterpret_cast<const bf16*>(t.grad) + base, count);
  }
  s = group_sum(s, red);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

template <bool STREAM, class T>
__device__ __forceinline__ void scale_chunk(const T* p, T* o, size_t count, float f) {
  constexpr int N = VecOf<T>::N;
  const size_t whole = count / N;
  auto put = [&](size_t i, const Vec<T>& v) __attribute__((always_inline)) {
    float x[N];
#pragma unroll
    for (int e = 0; e < N; e++) x[e] = v.get(e) * f;
    STREAM ? stream_vec(o + i * N, x) : put_vec(true, o + i * N, x);
  };
  constexpr int AT_ONCE = 4;
  size_t at = threadIdx.x;
  for (; at + (AT_ONCE - 1) * 256 < whole; at += AT_ONCE * 256) {
    Vec<T> v[AT_ONCE];
#pragma unroll
    for (int b = 0; b < AT_ONCE; b++) v[b] = load_vec(p + (at + b * 256) * N);
#pragma unroll
    for (int b = 0; b < AT_ONCE; b++) put(at + b * 256, v[b]);
  }
  for (; at < whole; at += 256) put(at, load_vec(p + at * N));
  const size_t i = whole * N + threadIdx.x;
  if (i < count) o[i] = from_f32<T>(to_f32(p[i]) * f);
}

// What the sums give: all workgroups alike.
__device__ __forceinline__ float2 norm_of(const double* sums, uint32_t nsums, float scale,
                                          float max_norm, bool& finite) {
  __shared__ double red[4];
  double s = 0.0;
  for (uint32_t i = threadIdx.x; i < nsums; i += 256) s += sums[i];
  s = group_sum(s, red);
  const double norm = fabs((double)scale) * sqrt(s);
  finite = (float)norm < INFINITY;  // (as out holds it)
  float f = 1.f;
  if (!finite)
    f = NAN;
  else if (norm > (double)max_norm)
    f = (float)((double)max_norm / norm);
  return make_float2((float)norm, f);
}

__global__ __launch_bounds__(256) void k_norm_only(const double* sums, uint32_t nsums, float scale,
                                                   float max_norm, float* out) {
  bool finite;
  const float2 r = norm_of(sums, nsums, scale, max_norm, finite);
  if (threadIdx.x == 0) out[0] = r.x, out[1] = r.y;
}

template <bool STREAM>
__global__ __launch_bounds__(256) void k_clip(const NormTensor* __restrict__ tensors,
                                              const uint2* __restrict__ chunks, uint32_t nchunks,
                                              uint32_t chunk, const double* sums, uint32_t nsums,
                                              float scale, float max_norm, float* out) {
  bool finite;
  const float2 r = norm_of(sums, nsums, scale, max_norm, finite);
  if (blockIdx.x == 0 && threadIdx.x == 0) out[0] = r.x, out[1] = r.y;
  const float f = finite ? r.y : 1.f;  // (what is not finite stays as it is)
  for (uint32_t i = blockIdx.x; i < nchunks; i += gridDim.x) {
    const uint2 at = chunks[nchunks - 1 - i];
    const NormTensor t = tensors[at.x];
    if (f == 1.f && t.out == t.grad) continue;
    const size_t base = (size_t)at.y * chunk, count = min(t.len - base, (size_t)chunk);
    if (t.kind == EMH_F32)
      scale_chunk<STREAM>(reinterpret_cast<const float*>(t.grad) + base,
                          reinterpret_cast<float*>(t.out) + base, count, f);
    else if (t.kind == EMH_F16)
      scale_chunk<STREAM>(reinterpret_cast<const f16*>(t.grad) + base,
                          reinterpret_cast<f16*>(t.out) + base, count, f);
    else
      scale_chunk<STREAM>(reinterpret_cast<const bf16*>(t.grad) + base,
                          reinterpret_cast<bf16*>(t.out) + base, count, f);
  }
}

}  // namespace

void launch_grad_norm(emh_ctx* c, const NormTensor* tensors, const uint2* chunks, size_t nchunks,
                      size_t chunk, bool stream, double* sums, float scale, float max_norm, float* out,
                      bool clip) {
  const unsigned nsums = (unsigned)std::min(nchunks, NORM_SUMS);
  if (nsums > 0)
    k_square_sums<<<nsums, 256, 0, c->stream>>>(tensors, chunks, (uint32_t)nchunks, (uint32_t)chunk,
                                                sums);
  if (clip && nchunks > 0) {
    auto go = [&](auto kernel) {
      kernel<<<(unsigned)std::min(nchunks, (size_t)2048), 256, 0, c->stream>>>(
          tensors, chunks, (uint32_t)nchunks, (uint32_t)chunk, sums, nsums, scale, max_norm, out);
    };
    stream ? go(k_clip<true>) : go(k_clip<false>);
  } else
    k_norm_only<<<1, 256, 0, c->stream>>>(sums, nsums, scale, max_norm, out);
  EMH_HIP(hipGetLastError());
}

}  // namespace emh
