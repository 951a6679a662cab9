// Layer norm's forward and backward pass over the rows of a matrix.
//
// Forward, for a row x of d elements: mean = sum x / d, var = sum (x - mean)^2 /
// d, y = (x - mean) rstd w + b. The row stays in registers between the two sums
// and the result, so memory is read once; the second sum is over differences
// (sum x^2 - mean^2 would cancel where a row's mean exceeds its spread).
//
// Backward, with h = (x - mean) rstd and g = dy w: dx = rstd (g - mean(g) - h
// mean(g h)); dweight = sum over rows of dy h, dbias = sum of dy. A thread owns
// the same columns in every row that its workgroup takes, so both sums over the
// rows grow in its registers, in f32; a workgroup adds its groups' through LDS and leaves
// one row of sums, and a second launch adds those. No atomics: the order of
// every sum follows from the sizes.
//
// Bound by HBM: 2 (forward) and 3 (backward) elements moved per element.
#include <algorithm>
#include <type_traits>

#include "emh_learn.h"
#include "emh_types.h"

namespace emh {
namespace {

struct NormArgs {
  const void* x;
  size_t ldx;
  const void* dy;
  size_t lddy;
  size_t rows;
  int d;
  const void* w;
  const void* b;
  int wkind, bkind;
  float eps;
  void* y;  // forward: y; backward: dx
  size_t ldy;
  float* mean;
  float* rstd;
  float* part;  // backward: [block][2][d], or null
};

// Sums over the LPR lanes (threads, past a wave) that share a row, in all of
// them. red: LDS, one float for every wave, and a row of the workgroup's groups
// for each of the calls that may follow one another without a barrier.
template <int LPR, int TB>
__device__ __forceinline__ float row_sum(float v, float (*red)[TB / 64], int slot) {
  v = lanes_sum<(LPR < 64 ? LPR : 64)>(v);
  if constexpr (LPR > 64) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) red[slot][w] = v;
    __syncthreads();
    constexpr int NW = LPR / 64;
    const int w0 = w / NW * NW;
    v = 0.f;
#pragma unroll
    for (int i = 0; i < NW; i++) v += red[slot][w0 + i];
  }
  return v;
}

// A thread's vectors begin at columns `col`, d >= N. Where one would pass the row's end
// it is the row's last N columns instead (at): those before col are another thread's
// too, and count there (in); both store the same value. One load and one store a
// vector, whatever d is. (Element by element the last vector of 300 f16 took half of
// the forward pass.)
template <int N>
struct Cols {
  int at, from;  // in(e): at + e >= from
  __device__ __forceinline__ Cols(int col, int d) : at(min(col, d - N)), from(col) {}
  __device__ __forceinline__ bool in(int e) const { return at + e >= from; }
  __device__ __forceinline__ bool any() const { return at + N > from; }
};

// A vector of a norm's weight or bias (T or f32), `fill` without one.
template <class T>
__device__ __forceinline__ void load_affine(const void* p, int kind, int at, float fill, float* out) {
  constexpr int N = VecOf<T>::N;
  if (!p) {
#pragma unroll
    for (int e = 0; e < N; e++) out[e] = fill;
  } else if (kind == EMH_F32) {
#pragma unroll
    for (int q = 0; q < N; q += 4) {
      const Vec<float> v = load_vec(reinterpret_cast<const float*>(p) + at + q);
#pragma unroll
      for (int e = 0; e < 4; e++) out[q + e] = v.get(e);
    }
  } else {
    const Vec<T> v = load_vec(reinterpret_cast<const T*>(p) + at);
#pragma unroll
    for (int e = 0; e < N; e++) out[e] = v.get(e);
  }
}

// Forward: LPR threads a row, NV vectors of 16 bytes a thread. The next row is on
// its way while a row's sums are formed. 200,000 x 768 f32 228 us, 5.4 TB/s; 16,384 x
// 768 bf16 13.5 us, 3.7 TB/s; 16 x 384 2.5 us, a launch.
template <class T, int LPR, int NV>
__global__ __launch_bounds__(256) void k_norm(const NormArgs a) {
  constexpr int N = VecOf<T>::N, TB = 256, G = TB / LPR;
  __shared__ float red[4][TB / 64];
  const int l = threadIdx.x % LPR, g = threadIdx.x / LPR;
  const int d = a.d;
  auto cols = [&](int j) __attribute__((always_inline)) { return Cols<N>((l + LPR * j) * N, d); };
  Vec<T> next[NV];
  auto fetch = [&](size_t row) __attribute__((always_inline)) {
    const T* x = reinterpret_cast<const T*>(a.x) + (row < a.rows ? row : 0) * a.ldx;
#pragma unroll
    for (int j = 0; j < NV; j++) next[j] = load_vec(x + cols(j).at);
  };
  fetch((size_t)blockIdx.x * G + g);
  float w[NV * N], b[NV * N];
#pragma unroll
  for (int j = 0; j < NV; j++) {
    load_affine<T>(a.w, a.wkind, cols(j).at, 1.f, w + j * N);
    load_affine<T>(a.b, a.bkind, cols(j).at, 0.f, b + j * N);
  }
  const float inv = 1.0f / (float)d;
  int slot = 0;
  const size_t step = (size_t)gridDim.x * G;
  // (The bound is the workgroup's: all its threads meet at row_sum's barriers.)
  for (size_t r0 = (size_t)blockIdx.x * G; r0 < a.rows; r0 += step) {
    const size_t row = r0 + g;
    const bool live = row < a.rows;
    Vec<T> v[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) v[j] = next[j];
    if (r0 + step < a.rows) fetch(r0 + step + g);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
      for (int e = 0; e < N; e++) s += cols(j).in(e) ? v[j].get(e) : 0.f;
    const float mean = row_sum<LPR, TB>(s, red, slot) * inv;
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
      for (int e = 0; e < N; e++) {
        const float o = cols(j).in(e) ? v[j].get(e) - mean : 0.f;
        q = fmaf(o, o, q);
      }
    const float rstd = 1.0f / sqrtf(row_sum<LPR, TB>(q, red, slot ^ 1) * inv + a.eps);
    slot ^= 2;
    if (!live) continue;
    T* y = reinterpret_cast<T*>(a.y) + row * a.ldy;
#pragma unroll
    for (int j = 0; j < NV; j++) {
      float o[N];
#pragma unroll
      for (int e = 0; e < N; e++)
        o[e] = fmaf((v[j].get(e) - mean) * rstd, w[j * N + e], b[j * N + e]);
      if (cols(j).any()) store_vec(y + cols(j).at, o);
    }
    if (l == 0 && a.mean) a.mean[row] = mean;
    if (l == 0 && a.rstd) a.rstd[row] = rstd;
  }
}

// Backward, TB threads. The row's elements stay packed and are unpacked again for
// the result: what that takes is fewer registers, so more waves, whose rows are in
// flight together. AHEAD: the next row is on its way, too, where there are registers.
// 200,000 x 768 f32 371 us, 5.0 TB/s; 16,384 x 768 bf16 17.9 us, 4.2 TB/s.
template <class T, int LPR, int NV, int TB>
__global__ __launch_bounds__(TB, TB / 256) void k_norm_grad(const NormArgs a) {
  constexpr int N = VecOf<T>::N, G = TB / LPR;
  constexpr bool AHEAD = NV * N <= 12;
  __shared__ float red[4][TB / 64];
  __shared__ float fold[TB * NV * N];
  const int l = threadIdx.x % LPR, g = threadIdx.x / LPR;
  const int d = a.d;
  auto cols = [&](int j) __attribute__((always_inline)) { return Cols<N>((l + LPR * j) * N, d); };
  float w[NV * N], aw[NV * N], ab[NV * N];
#pragma unroll
  for (int j = 0; j < NV; j++) {
    load_affine<T>(a.w, a.wkind, cols(j).at, 1.f, w + j * N);
#pragma unroll
    for (int e = 0; e < N; e++) aw[j * N + e] = ab[j * N + e] = 0.f;
  }
  const float inv = 1.0f / (float)d;
  const size_t step = (size_t)gridDim.x * G;
  int slot = 0;
  struct Row {
    Vec<T> x[NV], dy[NV];
    float mean, rstd;
  };
  auto fetch = [&](size_t row, Row& o) __attribute__((always_inline)) {
    const size_t r = row < a.rows ? row : 0;
    const T* xp = reinterpret_cast<const T*>(a.x) + r * a.ldx;
    const T* dp = reinterpret_cast<const T*>(a.dy) + r * a.lddy;
#pragma unroll
    for (int j = 0; j < NV; j++) {
      o.x[j] = load_vec(xp + cols(j).at);
      o.dy[j] = load_vec(dp + cols(j).at);
    }
    o.mean = a.mean[r];
    o.rstd = a.rstd[r];
  };
  auto one = [&](const Row& o, size_t row) __attribute__((always_inline)) {
    const bool live = row < a.rows;
    float c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
      for (int e = 0; e < N; e++) {
        const int i = j * N + e;
        const float h = live ? (o.x[j].get(e) - o.mean) * o.rstd : 0.f;
        const float t = live ? o.dy[j].get(e) : 0.f;
        ab[i] += t;
        aw[i] = fmaf(t, h, aw[i]);
        const float u = cols(j).in(e) ? t * w[i] : 0.f;
        c1 += u;
        c2 = fmaf(u, cols(j).in(e) ? h : 0.f, c2);
      }
    c1 = row_sum<LPR, TB>(c1, red, slot) * inv;
    c2 = row_sum<LPR, TB>(c2, red, slot ^ 1) * inv;
    slot ^= 2;
    if (live && a.y) {
      T* y = reinterpret_cast<T*>(a.y) + row * a.ldy;
#pragma unroll
      for (int j = 0; j < NV; j++) {
        float t[N];
#pragma unroll
        for (int e = 0; e < N; e++)
          t[e] = o.rstd * (o.dy[j].get(e) * w[j * N + e] - c1 - (o.x[j].get(e) - o.mean) * o.rstd * c2);
        if (cols(j).any()) store_vec(y + cols(j).at, t);
      }
    }
  };
  size_t r0 = (size_t)blockIdx.x * G;
  if constexpr (AHEAD) {
    Row next;
    fetch(r0 + g, next);
    for (; r0 < a.rows; r0 += step) {
      const Row now = next;
      if (r0 + step < a.rows) fetch(r0 + step + g, next);
      one(now, r0 + g);
    }
  } else {
    for (; r0 < a.rows; r0 += step) {
      Row now;
      fetch(r0 + g, now);
      one(now, r0 + g);
    }
  }
  if (!a.part) return;
  // The groups' sums of a column added through LDS: dweight, then dbias.
  static_assert(G > 1, "groups to add");
#pragma unroll
  for (int which = 0; which < 2; which++) {
    if (which) __syncthreads();
#pragma unroll
    for (int i = 0; i < NV * N; i++) fold[i * TB + threadIdx.x] = which ? ab[i] : aw[i];
    __syncthreads();
    float* out = a.part + ((size_t)blockIdx.x * 2 + which) * d;
#pragma unroll
    for (int i0 = 0; i0 < NV * N; i0 += G) {
      const int i = i0 + g;
      if (i >= NV * N) continue;
      const Cols<N> c = cols(i / N);
      const int col = c.at + i % N;
      if (!c.in(i % N)) continue;
      float s = 0.f;
#pragma unroll 8
      for (int k = 0; k < G; k++) s += fold[i * TB + k * LPR + l];
      out[col] = s;
    }
  }
}

// Rows too long for the registers of a workgroup (or shorter than a vector): one
// workgroup a row, read again for every step (from L2, mostly). 4,096 x 20,001 f32: 301
// us forward (2.2 TB/s), 337 back and 151 for the sums over the rows.
template <class T>
__global__ __launch_bounds__(256) void k_norm_wide(const NormArgs a) {
  __shared__ float red[4][4];
  // (A row's second sum has a barrier between the reads of the first and the next row's.)
  for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.ldx;
    T* y = reinterpret_cast<T*>(a.y) + row * a.ldy;
    float s = 0.f;
    for (int i = threadIdx.x; i < a.d; i += 256) s += to_f32(x[i]);
    const float mean = row_sum<256, 256>(s, red, 0) / (float)a.d;
    float q = 0.f;
    for (int i = threadIdx.x; i < a.d; i += 256) {
      const float o = to_f32(x[i]) - mean;
      q = fmaf(o, o, q);
    }
    const float rstd = 1.0f / sqrtf(row_sum<256, 256>(q, red, 1) / (float)a.d + a.eps);
    for (int i = threadIdx.x; i < a.d; i += 256) {
      const float h = (to_f32(x[i]) - mean) * rstd;
      y[i] = from_f32<T>(fmaf(h, a.w ? load_kind(a.w, a.wkind, i) : 1.f,
                              a.b ? load_kind(a.b, a.bkind, i) : 0.f));
    }
    if (threadIdx.x == 0 && a.mean) a.mean[row] = mean;
    if (threadIdx.x == 0 && a.rstd) a.rstd[row] = rstd;
  }
}
template <class T>
__global__ __launch_bounds__(256) void k_norm_grad_wide(const NormArgs a) {
  __shared__ float red[4][4];
  for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.ldx;
    const T* dy = reinterpret_cast<const T*>(a.dy) + row * a.lddy;
    T* o = reinterpret_cast<T*>(a.y) + row * a.ldy;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float c1 = 0.f, c2 = 0.f;
    for (int i = threadIdx.x; i < a.d; i += 256) {
      const float u = to_f32(dy[i]) * (a.w ? load_kind(a.w, a.wkind, i) : 1.f);
      c1 += u;
      c2 = fmaf(u, (to_f32(x[i]) - mean) * rstd, c2);
    }
    c1 = row_sum<256, 256>(c1, red, 0) / (float)a.d;
    c2 = row_sum<256, 256>(c2, red, 1) / (float)a.d;
    for (int i = threadIdx.x; i < a.d; i += 256) {
      const float u = to_f32(dy[i]) * (a.w ? load_kind(a.w, a.wkind, i) : 1.f);
      o[i] = from_f32<T>(rstd * (u - c1 - (to_f32(x[i]) - mean) * rstd * c2));
    }
  }
}
// Their sums over rows: a thread a column, blockIdx.y a share of the rows.
template <class T>
__global__ __launch_bounds__(256) void k_norm_cols(const NormArgs a) {
  const int col = blockIdx.x * 256 + threadIdx.x;
  if (col >= a.d) return;
  const size_t per = (a.rows + gridDim.y - 1) / gridDim.y;
  const size_t lo = blockIdx.y * per, hi = min(a.rows, lo + per);
  float sw = 0.f, sb = 0.f;
#pragma unroll 4
  for (size_t r = lo; r < hi; r++) {
    const float t = to_f32(reinterpret_cast<const T*>(a.dy)[r * a.lddy + col]);
    const float h = (to_f32(reinterpret_cast<const T*>(a.x)[r * a.ldx + col]) - a.mean[r]) * a.rstd[r];
    sw = fmaf(t, h, sw);
    sb += t;
  }
  a.part[((size_t)blockIdx.y * 2) * a.d + col] = sw;
  a.part[((size_t)blockIdx.y * 2 + 1) * a.d + col] = sb;
}

// out = the nparts rows of sums added: 16 columns a workgroup, 64 shares of the
// rows in step and then one after another. Bound by latency: 256 rows of 2 x 768 3.9 us.
__global__ __launch_bounds__(1024) void k_norm_sums(const float* __restrict__ part, int nparts,
                                                    int d, void* dw, int dwkind, void* db,
                                                    int dbkind) {
  __shared__ float s[64][17];
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
  const size_t cols = (size_t)d * 2;
  for (size_t c0 = (size_t)blockIdx.x * 16; c0 < cols; c0 += (size_t)gridDim.x * 16) {
    const size_t col = c0 + c;
    float v = 0.f;
    if (col < cols) {
#pragma unroll 8
      for (int i = g; i < nparts; i += 64) v += part[(size_t)i * cols + col];
    }
    s[g][c] = v;
    __syncthreads();
    if (g == 0 && col < cols) {
      v = 0.f;
#pragma unroll
      for (int i = 0; i < 64; i++) v += s[i][c];
      if (col < (size_t)d) {
        if (dw) store_kind(dw, dwkind, col, v);
      } else if (db) {
        store_kind(db, dbkind, col - d, v);
      }
    }
    __syncthreads();  // the next columns' sums take their place
  }
}
// No rows: the sums are zero.
__global__ __launch_bounds__(256) void k_norm_zero(int d, void* dw, int dwkind, void* db,
                                                   int dbkind) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= d) return;
  if (dw) store_kind(dw, dwkind, i, 0.f);
  if (db) store_kind(db, dbkind, i, 0.f);
}

template <class F>
void by_kind(int kind, F&& f) {
  if (kind == EMH_F32)
    f(float{});
  else if (kind == EMH_F16)
    f(f16{});
  else
    f(bf16{});
}
template <int L, int V>
struct Shape {
  static constexpr int LPR = L, NV = V;
};
// The threads that share a row and the vectors each holds: the fewest vectors
// that hold the row. False: none does. (Rows of 300 f16 on 16 or 32 lanes with
// fewer idle ones took 8.7 us forward and 15.5 back; on 64, 8.0 and 12.6.)
template <class T, class F>
bool by_shape(size_t d, F&& f) {
  const size_t v = (d + VecOf<T>::N - 1) / VecOf<T>::N;
  if (d < (size_t)VecOf<T>::N)
    return false;
  else if (v <= 16)
    f(Shape<16, 1>{});
  else if (v <= 64)
    f(Shape<64, 1>{});
  else if (v <= 128)
    f(Shape<64, 2>{});
  else if (v <= 192)
    f(Shape<64, 3>{});
  else if (v <= 256)
    f(Shape<64, 4>{});
  else if (v <= 512)
    f(Shape<256, 2>{});
  else if (v <= 1024)
    f(Shape<256, 4>{});
  else
    return false;
  return true;
}

}  // namespace

void launch_layer_norm(emh_ctx* c, const MatIn& x, size_t rows, size_t d, const MatIn& weight,
                       const MatIn& bias, float eps, const MatOut& y, float* mean, float* rstd) {
  if (rows == 0) return;
  NormArgs a{};
  a.x = x.p, a.ldx = x.ld, a.rows = rows, a.d = (int)d;
  a.w = weight.p, a.wkind = weight.kind, a.b = bias.p, a.bkind = bias.kind;
  a.eps = eps, a.y = y.p, a.ldy = y.ld, a.mean = mean, a.rstd = rstd;
  by_kind(x.kind, [&](auto t) {
    using T = decltype(t);
    const bool held = by_shape<T>(d, [&](auto s) {
      using S = decltype(s);
      constexpr size_t G = 256 / S::LPR;
      const size_t blocks = std::min((rows + G - 1) / G, (size_t)c->cus * 8);
      k_norm<T, S::LPR, S::NV><<<dim3((unsigned)blocks), 256, 0, c->stream>>>(a);
    });
    if (!held)
      k_norm_wide<T><<<dim3((unsigned)std::min(rows, MAX_GROUPS)), 256, 0, c->stream>>>(a);
  });
  EMH_HIP(hipGetLastError());
}

void launch_layer_norm_grad(emh_ctx* c, const MatIn& dy, const MatIn& x, size_t rows, size_t d,
                            const MatIn& weight, const float* mean, const float* rstd,
                            const MatOut& dx, const MatOut& dweight, const MatOut& dbias) {
  NormArgs a{};
  a.x = x.p, a.ldx = x.ld, a.dy = dy.p, a.lddy = dy.ld, a.rows = rows, a.d = (int)d;
  a.w = weight.p, a.wkind = weight.kind, a.y = dx.p, a.ldy = dx.ld;
  a.mean = const_cast<float*>(mean), a.rstd = const_cast<float*>(rstd);
  const bool sums = dweight.p || dbias.p;
  if (rows == 0) {
    if (sums)
      k_norm_zero<<<grid1(d, 256), 256, 0, c->stream>>>((int)d, dweight.p, dweight.kind, dbias.p,
                                                        dbias.kind);
    EMH_HIP(hipGetLastError());
    return;
  }
  size_t parts = 0;
  by_kind(x.kind, [&](auto t) {
    using T = decltype(t);
    const bool held = by_shape<T>(d, [&](auto s) {
      using S = decltype(s);
      // A workgroup a CU, of as many waves as the registers allow: few rows of
      // sums to write and add. (Twelve elements a thread fill 1,024 threads' registers
      // and a few more: 30,000 x 641 f32 75 us a training pass, with 768 threads 67.)
      auto go = [&](auto threads) {
        constexpr int TB = decltype(threads)::value;
        constexpr size_t G = TB / S::LPR;
        parts = std::min((rows + G - 1) / G, (size_t)c->cus);
        if (sums) a.part = (float*)c->norm_part.get(parts * 2 * d * 4);
        k_norm_grad<T, S::LPR, S::NV, TB><<<dim3((unsigned)parts), TB, 0, c->stream>>>(a);
      };
      constexpr int HELD = S::NV * VecOf<T>::N;
      if constexpr (HELD > 16)
        go(std::integral_constant<int, 512>{});
      else if constexpr (HELD >= 12)
        go(std::integral_constant<int, 768>{});
      else
        go(std::integral_constant<int, 1024>{});
    });
    if (held) return;
    if (sums) {  // before dx, which may overwrite dy
      parts = std::min((rows + 15) / 16, (size_t)64);
      a.part = (float*)c->norm_part.get(parts * 2 * d * 4);
      k_norm_cols<T><<<dim3((unsigned)((d + 255) / 256), (unsigned)parts), 256, 0, c->stream>>>(a);
    }
    if (dx.p)
      k_norm_grad_wide<T><<<dim3((unsigned)std::min(rows, MAX_GROUPS)), 256, 0, c->stream>>>(a);
  });
  if (sums)
    k_norm_sums<<<dim3((unsigned)std::min((2 * d + 15) / 16, MAX_GROUPS)), 1024, 0, c->stream>>>(
        a.part, (int)parts, (int)d, dweight.p, dweight.kind, dbias.p, dbias.kind);
  EMH_HIP(hipGetLastError());
}

}  // namespace emh
