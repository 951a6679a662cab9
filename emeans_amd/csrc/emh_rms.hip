// Root-mean-square norm of rows and of what is added to them, its backward pass, and 8-bit
// codes of any rows.
//
// Forward, for a row of d columns: h = x + r, rounded to the rows' type (what is kept, and
// what the backward pass sees); rstd = 1 / sqrt(sum h^2 / d + eps), y = h rstd w; y in the rows'
// type, or as codes with a scale for every 128 columns (emh_codes.h), whose values are the
// unrounded y. The row stays in registers between the sum and the result: each element moves
// once.
//
// Backward, with u = h rstd and g = dy w: dx = dh + rstd (g - u mean(g u)), dweight = sum over
// rows of dy u. As layer norm's (emh_norm.hip): a thread owns the same columns in every row that
// its workgroup takes and sums dweight's terms in registers; the workgroups' sums are
// added by a second launch, in an order that follows from the sizes.
//
// Bound by HBM: 3 elements and a byte, or 4 elements, moved per element forward, 4 backward.
// 200,000 x 768 bf16: 236 us and 240, 5.2 TB/s; to codes 221 us, 4.9 TB/s; codes alone 89 us, 5.2
// TB/s. 16,384 x 768, which the caches hold in part: 16.3, 21.9, 17.9 and 7.9 us. One row of 1,024:
// 4.5 us, its launch. Rows that no workgroup holds (k_rms_wide and what follows it) are read by single
// elements: 4,096 x 16,384 bf16 206 us, backward 385, to codes 280.
#include "emh_answer.h"
#include "emh_codes.h"

namespace emh {
namespace {

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

// A thread's vectors begin at columns `from`, d >= N. Where one would pass the row's end it is
// the row's last N columns instead (at): those before `from` are another thread's too, and
// count there (in); both store the same value.
template <int N>
struct Cols {
  int at, from;
  __device__ __forceinline__ Cols(int col, int d) : at(min(col, d - N)), from(col) {}
  __device__ __forceinline__ bool in(int e) const { return at + e >= from; }
  __device__ __forceinline__ bool any() const { return at + N > from; }
};

// 1 / sqrt(v), to a unit of its last place: the instruction's and a Newton step.
__device__ __forceinline__ float root_of(float v) {
  const float r = __builtin_amdgcn_rsqf(v);
  const float better = fmaf(r * 0.5f, fmaf(-v * r, r, 1.f), r);
  return v > 1e-30f && v < 1e30f ? better : 1.0f / sqrtf(v);
}

template <class T>
__device__ __forceinline__ void load_weight(const RmsArgs& a, int at, float* out) {
  constexpr int N = VecOf<T>::N;
  if (!a.w) {
#pragma unroll
    for (int e = 0; e < N; e++) out[e] = 1.f;
  } else if (a.wkind == EMH_F32) {
#pragma unroll
    for (int q = 0; q < N; q += 4) {
      const Vec<float> v = load_vec(reinterpret_cast<const float*>(a.w) + at + q);
#pragma unroll
      for (int e = 0; e < 4; e++) out[q + e] = v.get(e);
    }
  } else {
    const Vec<T> v = load_vec(reinterpret_cast<const T*>(a.w) + at);
#pragma unroll
    for (int e = 0; e < N; e++) out[e] = v.get(e);
  }
}

// The sum of two vectors in their type.
template <class T>
__device__ __forceinline__ Vec<T> add_vec(const Vec<T>& x, const Vec<T>& r) {
  uint32_t w[4];
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; e++) w[e] = __float_as_uint(x.get(e) + r.get(e));
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++)
      w[e] = pair_from_f32<T>(x.get(2 * e) + r.get(2 * e), x.get(2 * e + 1) + r.get(2 * e + 1));
  }
  return Vec<T>{make_uint4(w[0], w[1], w[2], w[3])};
}

// Forward: LPR threads a row, NV vectors of 16 bytes a thread; the next row is on its way
// while this one's sum is formed. (A wave a row where four vectors a lane hold it, 4 KB: no
// barrier. 8,192 x 4,096 bf16 on four waves 41 us, 6.5 TB/s.)
template <class T, int LPR, int NV, bool CODES>
__global__ __launch_bounds__(256) void k_rms(const RmsArgs a) {
  constexpr int N = VecOf<T>::N, TB = 256, G = TB / LPR;
  __shared__ float red[2][TB / 64];
  const int l = threadIdx.x % LPR, g = threadIdx.x / LPR;
  const int d = a.d;
  auto cols = [&](int j) __attribute__((always_inline)) { return Cols<N>((l + LPR * j) * N, d); };
  Vec<T> nx[NV], nr[NV];
  auto fetch = [&](size_t row) __attribute__((always_inline)) {
    const size_t r = row < a.rows ? row : 0;
    const T* x = reinterpret_cast<const T*>(a.x) + r * a.ldx;
#pragma unroll
    for (int j = 0; j < NV; j++) nx[j] = load_vec(x + cols(j).at);
    if (a.r) {
      const T* p = reinterpret_cast<const T*>(a.r) + r * a.ldr;
#pragma unroll
      for (int j = 0; j < NV; j++) nr[j] = load_vec(p + cols(j).at);
    }
  };
  fetch((size_t)blockIdx.x * G + g);
  float w[NV * N];
#pragma unroll
  for (int j = 0; j < NV; j++) {
    load_weight<T>(a, cols(j).at, w + j * N);
    if constexpr (CODES) {  // columns that count elsewhere have no part in a block's scale
#pragma unroll
      for (int e = 0; e < N; e++) w[j * N + e] = cols(j).in(e) ? w[j * N + e] : 0.f;
    }
  }
  const float inv = 1.0f / (float)d;
  int slot = 0;
  const size_t step = (size_t)gridDim.x * G;
  // (The bound is the workgroup's: all its threads meet at row_sum's barriers.)
  for (size_t r0 = (size_t)blockIdx.x * G; r0 < a.rows; r0 += step) {
    const size_t row = r0 + g;
    const bool live = row < a.rows;
    Vec<T> h[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) h[j] = a.r ? add_vec<T>(nx[j], nr[j]) : nx[j];
    if (r0 + step < a.rows) fetch(r0 + step + g);
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
      for (int e = 0; e < N; e++) {
        const float o = cols(j).in(e) ? h[j].get(e) : 0.f;
        q = fmaf(o, o, q);
      }
    // (h may take x's or r's place: the row is loaded by all its threads here.)
    const float rstd = root_of(row_sum<LPR, TB>(q, red, slot) * inv + a.eps);
    slot ^= 1;
    if (live && a.h) {
      T* p = reinterpret_cast<T*>(a.h) + row * a.ldh;
#pragma unroll
      for (int j = 0; j < NV; j++)
        if (cols(j).any()) put_vec(a.through, p + cols(j).at, h[j]);
    }
    if (live && l == 0 && a.rstd) a.rstd[row] = rstd;
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const Cols<N> c = cols(j);
      float y[N];
#pragma unroll
      for (int e = 0; e < N; e++) y[e] = h[j].get(e) * rstd * w[j * N + e];
      if constexpr (CODES) {
        // A block's lanes (a row of 16 lanes has one block).
        constexpr int LPB = CODE_BLOCK / N < LPR ? CODE_BLOCK / N : LPR;
        const Coder code = Coder::of<LPB>(y, N);
        if (live && c.any()) {
          store_codes<N>(reinterpret_cast<uint8_t*>(a.y) + row * a.ldy, c.from, c.from - c.at, d,
                         code, y, a.through);
          if (c.from % CODE_BLOCK == 0) a.scale[row * a.lds + c.from / CODE_BLOCK] = code.scale;
        }
      } else {
        if (live && c.any()) put_vec(a.through, reinterpret_cast<T*>(a.y) + row * a.ldy + c.at, y);
      }
    }
  }
}

// Backward, TB threads. AHEAD: the next row is on its way, too, where there are registers.
template <class T, int LPR, int NV, int TB>
__global__ __launch_bounds__(TB, TB / 256) void k_rms_grad(const RmsArgs a) {
  constexpr int N = VecOf<T>::N, G = TB / LPR;
  constexpr bool AHEAD = NV * N <= 12;
  __shared__ float red[2][TB / 64];
  __shared__ float fold[TB * NV * N];
  const int l = threadIdx.x % LPR, g = threadIdx.x / LPR;
  const int d = a.d;
  auto cols = [&](int j) __attribute__((always_inline)) { return Cols<N>((l + LPR * j) * N, d); };
  float w[NV * N], aw[NV * N];
#pragma unroll
  for (int j = 0; j < NV; j++) {
    load_weight<T>(a, cols(j).at, w + j * N);
#pragma unroll
    for (int e = 0; e < N; e++) aw[j * N + e] = 0.f;
  }
  const float inv = 1.0f / (float)d;
  const size_t step = (size_t)gridDim.x * G;
  int slot = 0;
  struct Row {
    Vec<T> h[NV], dy[NV], dh[NV];
    float rstd;
  };
  auto fetch = [&](size_t row, Row& o) __attribute__((always_inline)) {
    const size_t r = row < a.rows ? row : 0;
    const T* hp = reinterpret_cast<const T*>(a.x) + r * a.ldx;
    const T* dp = reinterpret_cast<const T*>(a.dy) + r * a.lddy;
#pragma unroll
    for (int j = 0; j < NV; j++) {
      o.h[j] = load_vec(hp + cols(j).at);
      o.dy[j] = load_vec(dp + cols(j).at);
    }
    if (a.r) {
      const T* rp = reinterpret_cast<const T*>(a.r) + r * a.ldr;
#pragma unroll
      for (int j = 0; j < NV; j++) o.dh[j] = load_vec(rp + cols(j).at);
    }
    o.rstd = a.rstd[r];
  };
  auto one = [&](const Row& o, size_t row) __attribute__((always_inline)) {
    const bool live = row < a.rows;
    float c = 0.f;
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
      for (int e = 0; e < N; e++) {
        const int i = j * N + e;
        const float u = live ? o.h[j].get(e) * o.rstd : 0.f;
        const float t = live ? o.dy[j].get(e) : 0.f;
        aw[i] = fmaf(t, u, aw[i]);
        c = fmaf(cols(j).in(e) ? t * w[i] : 0.f, cols(j).in(e) ? u : 0.f, c);
      }
    c = row_sum<LPR, TB>(c, red, slot) * inv;
    slot ^= 1;
    if (live && a.y) {
      T* y = reinterpret_cast<T*>(a.y) + row * a.ldy;
#pragma unroll
      for (int j = 0; j < NV; j++) {
        float t[N];
#pragma unroll
        for (int e = 0; e < N; e++) {
          t[e] = o.rstd * (o.dy[j].get(e) * w[j * N + e] - o.h[j].get(e) * o.rstd * c);
          if (a.r) t[e] += o.dh[j].get(e);
        }
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
  if (!a.part && !a.dw) return;
  // The groups' sums of a column, added through LDS.
  static_assert(G > 1, "groups to add");
#pragma unroll
  for (int i = 0; i < NV * N; i++) fold[i * TB + threadIdx.x] = aw[i];
  __syncthreads();
  float* out = a.part + (size_t)blockIdx.x * d;
#pragma unroll
  for (int i0 = 0; i0 < NV * N; i0 += G) {
    const int i = i0 + g;
    if (i >= NV * N) continue;
    const Cols<N> c = cols(i / N);
    if (!c.in(i % N)) continue;
    float s = 0.f;
#pragma unroll 8
    for (int k = 0; k < G; k++) s += fold[i * TB + k * LPR + l];
    if (a.dw)
      store_kind(a.dw, a.dwkind, c.at + i % N, s);
    else
      out[c.at + i % N] = s;
  }
}

// Rows too long for the registers of a workgroup (or shorter than a vector): one workgroup a
// row, which it reads twice. What it writes an element's own thread has read (h may be x or r, y
// may be x). A thread's sum is f64 here, of up to 65,536 elements: in f32 equal ones' sum was
// off by 0.06 %.
template <class T, bool CODES>
__global__ __launch_bounds__(256) void k_rms_wide(const RmsArgs a) {
  __shared__ float red[2][4];
  int slot = 0;
  for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.ldx;
    const T* r = a.r ? reinterpret_cast<const T*>(a.r) + row * a.ldr : nullptr;
    T* hp = a.h ? reinterpret_cast<T*>(a.h) + row * a.ldh : nullptr;
    auto sum = [&](int i) __attribute__((always_inline)) {
      return r ? from_f32<T>(to_f32(x[i]) + to_f32(r[i])) : x[i];
    };
    double q = 0.0;
    for (int i = threadIdx.x; i < a.d; i += 256) {
      const double o = to_f32(sum(i));
      q = fma(o, o, q);
    }
    const float rstd = 1.0f / sqrtf(row_sum<256, 256>((float)q, red, slot) / (float)a.d + a.eps);
    slot ^= 1;
    if (threadIdx.x == 0 && a.rstd) a.rstd[row] = rstd;
    auto y_of = [&](int i) __attribute__((always_inline)) {
      const T h = sum(i);
      if (hp) hp[i] = h;
      return to_f32(h) * rstd * (a.w ? load_kind(a.w, a.wkind, i) : 1.f);
    };
    if constexpr (CODES) {
      // A wave a block, two columns a lane.
      uint8_t* out = reinterpret_cast<uint8_t*>(a.y) + row * a.ldy;
      const int blocks = (a.d + CODE_BLOCK - 1) / CODE_BLOCK, lane = threadIdx.x & 63;
      for (int b = threadIdx.x >> 6; b < blocks; b += 4) {
        const int i = b * CODE_BLOCK + 2 * lane;
        const float y0 = i < a.d ? y_of(i) : 0.f, y1 = i + 1 < a.d ? y_of(i + 1) : 0.f;
        const float v[4] = {y0, y1, 0.f, 0.f};
        const Coder code = Coder::of<64>(v, 2);
        if (i < ((a.d + 15) & ~15))
          *reinterpret_cast<uint16_t*>(out + i) = (uint16_t)code.four(v);
        if (lane == 0) a.scale[row * a.lds + b] = code.scale;
      }
    } else {
      T* y = reinterpret_cast<T*>(a.y) + row * a.ldy;
      for (int i = threadIdx.x; i < a.d; i += 256) {
        const float v = y_of(i);
        y[i] = from_f32<T>(v);
      }
    }
  }
}
template <class T>
__global__ __launch_bounds__(256) void k_rms_grad_wide(const RmsArgs a) {
  __shared__ float red[2][4];
  int slot = 0;
  for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* h = reinterpret_cast<const T*>(a.x) + row * a.ldx;
    const T* dy = reinterpret_cast<const T*>(a.dy) + row * a.lddy;
    const T* dh = a.r ? reinterpret_cast<const T*>(a.r) + row * a.ldr : nullptr;
    T* o = reinterpret_cast<T*>(a.y) + row * a.ldy;
    const float rstd = a.rstd[row];
    double sum = 0.0;
    for (int i = threadIdx.x; i < a.d; i += 256)
      sum = fma((double)(to_f32(dy[i]) * (a.w ? load_kind(a.w, a.wkind, i) : 1.f)),
                (double)(to_f32(h[i]) * rstd), sum);
    const float c = row_sum<256, 256>((float)sum, red, slot) / (float)a.d;
    slot ^= 1;
    for (int i = threadIdx.x; i < a.d; i += 256) {
      const float g = to_f32(dy[i]) * (a.w ? load_kind(a.w, a.wkind, i) : 1.f);
      float t = rstd * (g - to_f32(h[i]) * rstd * c);
      if (dh) t += to_f32(dh[i]);
      o[i] = from_f32<T>(t);
    }
  }
}
// Their sums over rows: a thread a column, blockIdx.y a share of the rows (f64: rows shorter than
// a vector may be many millions).
template <class T>
__global__ __launch_bounds__(256) void k_rms_cols(const RmsArgs a) {
  const int col = blockIdx.x * 256 + threadIdx.x;
  if (col >= a.d) return;
  const size_t per = (a.rows + gridDim.y - 1) / gridDim.y;
  const size_t lo = min(a.rows, blockIdx.y * per), hi = min(a.rows, lo + per);
  double s = 0.0;
#pragma unroll 4
  for (size_t r = lo; r < hi; r++)
    s = fma((double)to_f32(reinterpret_cast<const T*>(a.dy)[r * a.lddy + col]),
            (double)(to_f32(reinterpret_cast<const T*>(a.x)[r * a.ldx + col]) * a.rstd[r]), s);
  a.part[(size_t)blockIdx.y * a.d + col] = (float)s;
}

// out = the nparts rows of sums added: 16 columns a workgroup, 64 shares of the rows in step
// and then one after another. No rows: zeros.
__global__ __launch_bounds__(1024) void k_rms_sums(const float* __restrict__ part, int nparts,
                                                   int d, void* dw, int dwkind) {
  __shared__ float s[64][17];
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
  for (size_t c0 = (size_t)blockIdx.x * 16; c0 < (size_t)d; c0 += (size_t)gridDim.x * 16) {
    const size_t col = c0 + c;
    float v = 0.f;
    if (col < (size_t)d) {
#pragma unroll 8
      for (int i = g; i < nparts; i += 64) v += part[(size_t)i * d + col];
    }
    s[g][c] = v;
    __syncthreads();
    if (g == 0 && col < (size_t)d) {
      v = 0.f;
#pragma unroll
      for (int i = 0; i < 64; i++) v += s[i][c];
      store_kind(dw, dwkind, col, v);
    }
    __syncthreads();  // the next columns' sums take their place
  }
}

// Codes of rows: a lane a vector, 16 (f32: 32) lanes a block of 128 columns. HBM-bound: 200,000 x 768
// bf16 89 us, 5.2 TB/s.
template <class T>
__global__ __launch_bounds__(256) void k_codes_rows(const T* __restrict__ x, size_t ldx, size_t rows,
                                                    int d, int blocks, uint8_t* q, size_t ldq,
                                                    float* scale, size_t lds) {
  constexpr int N = VecOf<T>::N, LPB = CODE_BLOCK / N;
  const bool whole = ldq % 64 == 0 && (uintptr_t)q % 64 == 0;
  const size_t units = rows * blocks, step = (size_t)gridDim.x * (256 / LPB);
  const int l = threadIdx.x % LPB;
  // (Whole waves leave together: lanes_max and Coder take all lanes.)
  for (size_t u0 = (size_t)blockIdx.x * (256 / LPB); u0 < units; u0 += step) {
    const size_t u = u0 + threadIdx.x / LPB;
    const bool live = u < units;
    const size_t row = live ? u / blocks : 0;
    const int b = live ? (int)(u - row * blocks) : 0, col = b * CODE_BLOCK + l * N;
    const int left = live ? d - col : 0;
    const T* p = x + row * ldx + col;
    Vec<T> v{};
    if (left >= N)
      v = load_vec(p);
    else if (left > 0)
      v = load_some(p, left);
    float f[N];
#pragma unroll
    for (int e = 0; e < N; e++) f[e] = v.get(e);
    const Coder code = Coder::of<LPB>(f, N);
    if (left > 0) {
      store_codes<N>(q + row * ldq, col, 0, d, code, f, whole);
      if (l == 0) scale[row * lds + b] = code.scale;
    }
  }
}
// Codes of tiles of 128 x 128: a workgroup a tile, which its threads hold. HBM-bound: 131,071 x
// 1,024 f32 126 us, 5.3 TB/s.
template <class T>
__global__ __launch_bounds__(256) void k_codes_tiles(const T* __restrict__ x, size_t ldx,
                                                     size_t rows, int d, int blocks, size_t tiles,
                                                     uint8_t* q, size_t ldq, float* scale,
                                                     size_t lds) {
  constexpr int N = VecOf<T>::N, LPB = CODE_BLOCK / N, RPP = 256 / LPB, P = CODE_BLOCK / RPP;
  __shared__ float2 red[4];
  const bool whole = ldq % 64 == 0 && (uintptr_t)q % 64 == 0;
  const int l = threadIdx.x % LPB, r0 = threadIdx.x / LPB;
  for (size_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const size_t tr = t / blocks;
    const int b = (int)(t - tr * blocks), col = b * CODE_BLOCK + l * N, left = d - col;
    Vec<T> v[P];
    float top = 0.f, fine = 0.f;
#pragma unroll
    for (int p = 0; p < P; p++) {
      const size_t row = tr * CODE_BLOCK + p * RPP + r0;
      v[p] = Vec<T>{};
      if (row < rows && left >= N)
        v[p] = load_vec(x + row * ldx + col);
      else if (row < rows && left > 0)
        v[p] = load_some(x + row * ldx + col, left);
#pragma unroll
      for (int e = 0; e < N; e++) {
        top = fmaxf(top, fabsf(v[p].get(e)));
        fine = fmaxf(fine, finite_abs(v[p].get(e)));
      }
    }
    top = lanes_max<64>(top);
    fine = lanes_max<64>(fine);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_float2(top, fine);
    __syncthreads();
    const Coder code(fmaxf(fmaxf(red[0].x, red[1].x), fmaxf(red[2].x, red[3].x)), [&] {
      return fmaxf(fmaxf(red[0].y, red[1].y), fmaxf(red[2].y, red[3].y));
    });
    if (threadIdx.x == 0) scale[tr * lds + b] = code.scale;
#pragma unroll
    for (int p = 0; p < P; p++) {
      const size_t row = tr * CODE_BLOCK + p * RPP + r0;
      float f[N];
#pragma unroll
      for (int e = 0; e < N; e++) f[e] = v[p].get(e);
      if (row < rows && left > 0) store_codes<N>(q + row * ldq, col, 0, d, code, f, whole);
    }
    __syncthreads();  // red is the next tile's
  }
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
// The threads that share a row and the vectors each holds: the fewest vectors that hold the
// row. False: none does.
template <class T, class F>
bool by_shape(size_t d, F&& f) {
  constexpr size_t N = VecOf<T>::N;
  const size_t v = (d + N - 1) / N;
  // A row on as many lanes as one block of codes has: 100,000 x 256 bf16 to codes 30.2 us, x 128
  // f32 26.3 (on 64 lanes 36.9 and 29.1). Longer rows, two vectors on 32 lanes, take as long
  // or longer (10,007 x 300 f16 6.9, so 6.6, both with stores that were written back).
  constexpr int PAIR = N == 8 ? 16 : 32;
  if (d < N)
    return false;
  else if (v <= 16)
    f(Shape<16, 1>{});
  else if (v <= 32)
    f(Shape<PAIR, 32 / PAIR>{});
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

void launch_rms_norm(emh_ctx* c, RmsArgs a) {
  if (a.rows == 0) return;
  // Up to 16 MB of rows through the caches: 4,096 x 1,024 f32 8.2 us, written back 10.3; to codes 7.3
  // and 10.5; 25 MB take the same time either way, longer rows longer. At any address: 10,007 x 300
  // f16 to codes 5.8, with codes written back 6.3, h too 6.9; 8,000 x 999 bf16 10.0 and 12.1 (codes
  // 10.5 and 13.6); f32 4,000 x 1,001 9.7 and 9.3, the only one slower of a dozen.
  a.through = a.rows * (size_t)a.d * kind_bytes(a.kind) <= size_t(16) << 20;
  by_kind(a.kind, [&](auto t) {
    using T = decltype(t);
    const bool held = by_shape<T>((size_t)a.d, [&](auto s) {
      using S = decltype(s);
      constexpr size_t G = 256 / S::LPR;
      const dim3 grid((unsigned)std::min((a.rows + G - 1) / G, (size_t)c->cus * 8));
      if (a.scale)
        k_rms<T, S::LPR, S::NV, true><<<grid, 256, 0, c->stream>>>(a);
      else
        k_rms<T, S::LPR, S::NV, false><<<grid, 256, 0, c->stream>>>(a);
    });
    if (held) return;
    const dim3 grid((unsigned)std::min(a.rows, MAX_GROUPS));
    if (a.scale)
      k_rms_wide<T, true><<<grid, 256, 0, c->stream>>>(a);
    else
      k_rms_wide<T, false><<<grid, 256, 0, c->stream>>>(a);
  });
  EMH_HIP(hipGetLastError());
}

void launch_rms_norm_grad(emh_ctx* c, RmsArgs a, const MatOut& dweight) {
  const size_t d = (size_t)a.d;
  size_t parts = 0;
  if (a.rows > 0)
    by_kind(a.kind, [&](auto t) {
      using T = decltype(t);
      const bool held = by_shape<T>(d, [&](auto s) {
        using S = decltype(s);
        // A workgroup a CU, of as many waves as the registers allow: few rows of sums to write
        // and add.
        auto go = [&](auto threads) {
          constexpr int TB = decltype(threads)::value;
          constexpr size_t G = TB / S::LPR;
          parts = std::min((a.rows + G - 1) / G, (size_t)c->cus);
          if (parts == 1)
            a.dw = dweight.p, a.dwkind = dweight.kind;
          else if (dweight.p)
            a.part = (float*)c->rms_part.get(parts * d * 4, c->stream);
          k_rms_grad<T, S::LPR, S::NV, TB><<<dim3((unsigned)parts), TB, 0, c->stream>>>(a);
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
      if (dweight.p) {  // before dx, which may overwrite dy
        parts = std::min((a.rows + 15) / 16, (size_t)64);
        a.part = (float*)c->rms_part.get(parts * d * 4, c->stream);
        k_rms_cols<T><<<dim3((unsigned)((d + 255) / 256), (unsigned)parts), 256, 0, c->stream>>>(a);
      }
      if (a.y)
        k_rms_grad_wide<T><<<dim3((unsigned)std::min(a.rows, MAX_GROUPS)), 256, 0, c->stream>>>(a);
    });
  // (One workgroup's sums are dweight: 8 rows of 1,024 bf16 4.4 us, with a second launch 8.0.)
  if (dweight.p && !a.dw)
    k_rms_sums<<<dim3((unsigned)std::min((d + 15) / 16, MAX_GROUPS)), 1024, 0, c->stream>>>(
        a.part, (int)parts, (int)d, dweight.p, dweight.kind);
  EMH_HIP(hipGetLastError());
}

void launch_quantize(emh_ctx* c, const MatIn& x, size_t rows, size_t d, bool tall, uint8_t* q,
                     size_t ldq, float* scale, size_t lds) {
  if (rows == 0) return;
  const int blocks = (int)((d + CODE_BLOCK - 1) / CODE_BLOCK);
  by_kind(x.kind, [&](auto t) {
    using T = decltype(t);
    const T* p = (const T*)x.p;
    if (tall) {
      const size_t tiles = (rows + CODE_BLOCK - 1) / CODE_BLOCK * blocks;
      k_codes_tiles<T><<<dim3((unsigned)std::min(tiles, MAX_GROUPS)), 256, 0, c->stream>>>(
          p, x.ld, rows, (int)d, blocks, tiles, q, ldq, scale, lds);
    } else {
      constexpr size_t PER = 256 / (CODE_BLOCK / VecOf<T>::N);
      const size_t groups = (rows * blocks + PER - 1) / PER;
      k_codes_rows<T><<<dim3((unsigned)std::min(groups, MAX_GROUPS)), 256, 0, c->stream>>>(
          p, x.ld, rows, (int)d, blocks, q, ldq, scale, lds);
    }
  });
  EMH_HIP(hipGetLastError());
}

}  // namespace emh
