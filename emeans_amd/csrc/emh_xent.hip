// Softmax cross entropy of rows against a linear classifier's classes, and its
// gradients, without an n x k matrix of logits: which products run over what
// (emh_xent.h), the operands laid out for them, and the joins of their parts.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <vector>

#include "emh_xent.h"

namespace emh {
namespace {

constexpr float LN2 = 0.693147181f;

// A row's lse and loss from the maximum and sum of all its classes.
__device__ __forceinline__ void finish_row(uint32_t i, float m, float s, uint32_t lab, uint32_t k,
                                           float zlabel, float* loss, float* lse, uint32_t* small) {
  const float top = m == -INFINITY ? 0.f : m, ls = log2f(s) * LN2;
  if (lse) lse[i] = top + ls;
  loss[i] = lab < k ? (top - zlabel) + ls : 0.f;
  if (lab >= k && lab != NO_LABEL) small[SW_BAD_CLASS] = 1u;
}

// One matrix to lay out: rows to 16-byte aligned rows of dp elements, the rest zero
// (dp a multiple of SLAB); labels: rows without one become zeros.
struct PackOne {
  const void* x;
  size_t ld, n;
  const uint32_t* labels;
  char *hi, *lo;
  int* ex;
  uint32_t blocks;
  // A wave's first row, and from one to the next.
  __device__ __forceinline__ size_t first(uint32_t block) const {
    return (size_t)block * 4 + (threadIdx.x >> 6);
  }
  __device__ __forceinline__ size_t step() const { return (size_t)blocks * 4; }
};
struct PackArgs {  // both operands in one launch, the first's workgroups first
  PackOne m[2];
  uint32_t d, dp, k, first;
};

// 16-bit rows. A wave a row. Bound by HBM: 16,384 and 1,000 rows of 770 12.5 us, 4.3 TB/s.
template <class T>
__global__ __launch_bounds__(256) void k_pack16(const PackArgs a) {
  const bool second = blockIdx.x >= a.first;
  const PackOne& m = a.m[second ? 1 : 0];
  const uint32_t lane = threadIdx.x & 63;
  for (size_t i = m.first(blockIdx.x - (second ? a.first : 0)); i < m.n; i += m.step()) {
    const T* row = reinterpret_cast<const T*>(m.x) + i * m.ld;
    T* out = reinterpret_cast<T*>(m.hi) + i * a.dp;
    const bool zero = m.labels && m.labels[i] >= a.k;
    for (uint32_t c = lane * 8; c < a.dp; c += 512) {
      Vec<T> v{make_uint4(0u, 0u, 0u, 0u)};
      if (!zero && c < a.d) v = c + 8 <= a.d ? load_vec(row + c) : load_some(row + c, (int)(a.d - c));
      *reinterpret_cast<uint4*>(out + c) = v.raw;
    }
  }
}

// f32 rows to planes of f16 (emh_xent.h) and their exponents e (x = plane 2^e). A
// wave a row, which it holds where it has at most 1,024 elements, and reads twice
// beyond. Bound by HBM and, there, by a launch of few rows a wave: 11,007 rows of 300
// 8.7 us, 3.2 TB/s; 65,536 of 768 64 us, 6.3 TB/s.
__global__ __launch_bounds__(256) void k_pack32(const PackArgs a) {
  const bool second = blockIdx.x >= a.first;
  const PackOne& m = a.m[second ? 1 : 0];
  const uint32_t lane = threadIdx.x & 63, d = a.d, dp = a.dp;
  for (size_t i = m.first(blockIdx.x - (second ? a.first : 0)); i < m.n; i += m.step()) {
    const float* row = reinterpret_cast<const float*>(m.x) + i * m.ld;
    const bool zero = m.labels && m.labels[i] >= a.k;
    constexpr uint32_t HELD = 4;  // vectors of four a lane
    auto get = [&](uint32_t c) __attribute__((always_inline)) {
      Vec<float> v{make_uint4(0u, 0u, 0u, 0u)};
      if (!zero && c < d) v = c + 4 <= d ? load_vec(row + c) : load_some(row + c, (int)(d - c));
      return v;
    };
    auto largest = [](const Vec<float>& v, float top) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float t = fabsf(v.get(e));
        top = fmaxf(top, t < INFINITY ? t : 0.f);
      }
      return top;
    };
    Vec<float> held[HELD];
    float top = 0.f;
#pragma unroll
    for (uint32_t q = 0; q < HELD; q++) held[q] = get(lane * 4 + q * 256);
#pragma unroll
    for (uint32_t q = 0; q < HELD; q++) top = largest(held[q], top);
    for (uint32_t c = lane * 4 + HELD * 256; c < d; c += 256) top = largest(get(c), top);
    top = lanes_max<64>(top);
    // (A row of zeros takes the least exponent, which is no one's largest.)
    const int e0 = top > 0.f ? max(ilogbf(top) - 13, XENT_LEAST) : XENT_LEAST;
    const float by = ldexpf(1.f, -e0);
    auto put = [&](uint32_t c, const Vec<float>& v) __attribute__((always_inline)) {
      uint16_t h4[4], l4[4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float t = v.get(e) * by;
        const f16 h = (f16)t;
        h4[e] = __builtin_bit_cast(uint16_t, h);
        l4[e] = __builtin_bit_cast(uint16_t, (f16)((t - (float)h) * (1.f / LOW_UNIT)));
      }
      const size_t o = (i * dp + c) * 2;
      *reinterpret_cast<uint2*>(m.hi + o) =
          make_uint2(h4[0] | (uint32_t)h4[1] << 16, h4[2] | (uint32_t)h4[3] << 16);
      *reinterpret_cast<uint2*>(m.lo + o) =
          make_uint2(l4[0] | (uint32_t)l4[1] << 16, l4[2] | (uint32_t)l4[3] << 16);
    };
#pragma unroll
    for (uint32_t q = 0; q < HELD; q++)
      if (lane * 4 + q * 256 < dp) put(lane * 4 + q * 256, held[q]);
    for (uint32_t c = lane * 4 + HELD * 256; c < dp; c += 256) put(c, get(c));
    if (lane == 0) m.ex[i] = e0;
  }
}

// The call's state, by one workgroup: a pass over the labels and weights, and of f32
// operands over the exponents. Bound by latency: 16,384 rows 5.4 us, of f32 7.1. (A
// workgroup: joining several would take a launch more, or a fence and a ticket, which
// cost more. Calls that need only how many rows have a label do without: RowScale.)
__global__ __launch_bounds__(1024) void k_survey(uint32_t n, const uint32_t* __restrict__ labels,
                                                 uint32_t k, const float* __restrict__ gloss,
                                                 const int* __restrict__ ex,
                                                 const int* __restrict__ ew, XentState* st,
                                                 uint32_t* small) {
  const uint32_t lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  __shared__ int sh[5][16];
  constexpr int MANY = 1 << 20;
  int count = 0, uexp = 0, ewmax = 0, ulow = MANY, ewlow = MANY;
  bool bad = false;
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < n; i += 1024) {
    const uint32_t lab = labels[i];
    const bool has = lab < k;
    bad = bad || (!has && lab != NO_LABEL);
    count += has ? 1 : 0;
    const float g = gloss ? fabsf(gloss[i]) : 1.f;
    const int e = (ex ? ex[i] : 0) + XENT_BIAS + (gloss ? ilogbf(g) : 0);
    if (has && g > 0.f && g < INFINITY) {
      uexp = max(uexp, e);
      ulow = min(ulow, e);
    }
  }
  if (ew) {
#pragma unroll 8
    for (uint32_t j = threadIdx.x; j < k; j += 1024) {
      ewmax = max(ewmax, ew[j] + XENT_BIAS);
      ewlow = min(ewlow, ew[j] + XENT_BIAS);
    }
  }
  if (bad) small[SW_BAD_CLASS] = 1u;
  for (int o = 32; o > 0; o >>= 1) {
    count += __shfl_xor(count, o, 64);
    uexp = max(uexp, __shfl_xor(uexp, o, 64));
    ewmax = max(ewmax, __shfl_xor(ewmax, o, 64));
    ulow = min(ulow, __shfl_xor(ulow, o, 64));
    ewlow = min(ewlow, __shfl_xor(ewlow, o, 64));
  }
  if (lane == 0) sh[0][w] = count, sh[1][w] = uexp, sh[2][w] = ewmax, sh[3][w] = ulow, sh[4][w] = ewlow;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < 16; i++) {
    count += sh[0][i];
    uexp = max(uexp, sh[1][i]);
    ewmax = max(ewmax, sh[2][i]);
    ulow = min(ulow, sh[3][i]);
    ewlow = min(ewlow, sh[4][i]);
  }
  const int span = max(uexp - ulow, 0) + max(ewmax - ewlow, 0);
  *st = XentState{(uint32_t)count, uexp, ewmax, span <= XENT_SPAN ? 1 : 0};
}

typedef float v4f __attribute__((ext_vector_type(4)));

// One chunk of 16 classes (a) and 16 rows (b).
__device__ __forceinline__ v4f mfma_few(const Vec<float>& a, const Vec<float>& b, v4f c) {
#pragma unroll
  for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.get(e), b.get(e), c, 0, 0, 0);
  return c;
}
__device__ __forceinline__ v4f mfma_few(const Vec<f16>& a, const Vec<f16>& b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a.raw),
                                                __builtin_bit_cast(v8h, b.raw), c, 0, 0, 0);
}
__device__ __forceinline__ v4f mfma_few(const Vec<bf16>& a, const Vec<bf16>& b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a.raw),
                                                 __builtin_bit_cast(v8bf, b.raw), c, 0, 0, 0);
}

// Few rows (at most 16 R) against all classes, the operands read as they lie, once:
// a workgroup takes 16 C classes at a time, its four waves a quarter of the depth
// each (every fourth 64 bytes of a row), with 16 x 16 MFMAs, the classes as their A: a
// lane then holds four classes of one row. f32 in f32 MFMAs. The workgroup's maximum
// and sum of its classes go to part[row][workgroup].
// Bound by the classes' bytes from HBM (16 rows of 1,024 against 131,071 classes in
// bf16 48 us with the join, 5.6 TB/s), or by latency: 16 rows of 384 against 256 classes
// are 25 KB a CU and take 5.4 us, the join 3.2.
// Many waves do more than many loads of one: with eight chunks in flight, 16 rows of
// 384 against 20,000 took 15.0 us, now 10.0. C = 4 where there are classes enough for
// every CU: the rows' loads, which are as many as the classes' with C = 1, are shared
// (16 rows by 131,071: 64.8 us before, 64 rows 150, now 74; but 64 classes at a time,
// 16 by 4,096, take 9.8 us and 16 at a time 7.5).
// ODD: rows may begin at odd multiples of two bytes.
template <class T, int R, int C, bool ODD>
__global__ __launch_bounds__(256) void k_few(const T* __restrict__ x, size_t ldx, uint32_t n,
                                             uint32_t d, const T* __restrict__ w, size_t ldw,
                                             uint32_t k, const uint32_t* __restrict__ labels,
                                             float scale, float2* part, float* zlabel) {
  constexpr int N = VecOf<T>::N, DEEP = 4 * N;  // a chunk: DEEP of the depth, N a lane
  constexpr int U = C == 1 && R < 4 ? 2 : 1;    // chunks a wave has in flight
  __shared__ v4f sum[4][R][C][64];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t l = lane & 15, q = lane >> 4;
  const uint32_t groups = (k + 16 * C - 1) / (16 * C), chunks = (d + DEEP - 1) / DEEP;
  float m = -INFINITY, s = 0.f;  // of the row that this lane keeps (wave r: rows 16 r ..)
  const uint32_t mine = wave * 16 + l;
  const uint32_t lab = wave < R && mine < n ? labels[mine] : NO_LABEL;
  auto fetch = [&](const T* p, size_t ld, uint32_t row, uint32_t rows, uint32_t c) __attribute__((always_inline)) {
    const T* at = p + (size_t)min(row, rows - 1) * ld;
    const uint32_t col = c * DEEP + q * N;
    if constexpr (ODD) {
      if (col + N <= d) return load_vec_words(at + col);
    } else {
      if (col + N <= d) return load_vec(at + col);
    }
    return load_some(at + min(col, d), (int)d - (int)col);
  };
  for (uint32_t g = blockIdx.x; g < groups; g += gridDim.x) {
    v4f acc[R][C];
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
      for (int i = 0; i < C; i++) acc[r][i] = v4f{0.f, 0.f, 0.f, 0.f};
    for (uint32_t c0 = wave; c0 < chunks; c0 += 4 * U) {
      // (Past the last chunk it is read again, and not used: no load waits for a branch.)
      Vec<T> a[U][C], b[U][R];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const uint32_t c = min(c0 + 4 * u, chunks - 1);
#pragma unroll
        for (int i = 0; i < C; i++) a[u][i] = fetch(w, ldw, (g * C + i) * 16 + l, k, c);
#pragma unroll
        for (int r = 0; r < R; r++) b[u][r] = fetch(x, ldx, r * 16 + l, n, c);
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (c0 + 4 * u >= chunks) continue;
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
          for (int i = 0; i < C; i++) acc[r][i] = mfma_few(a[u][i], b[u][r], acc[r][i]);
      }
    }
    __syncthreads();  // the last group's sums have been read
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
      for (int i = 0; i < C; i++) sum[wave][r][i][lane] = acc[r][i];
    __syncthreads();
    if (wave >= R) continue;
    v4f z[C];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < C; i++) {
      z[i] = sum[0][wave][i][lane];
#pragma unroll
      for (int o = 1; o < 4; o++) z[i] += sum[o][wave][i][lane];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const uint32_t j = (g * C + i) * 16 + q * 4 + e;
        z[i][e] = j < k ? z[i][e] * scale : -INFINITY;
        if (j == lab && j < k) zlabel[mine] = z[i][e];
        top = fmaxf(top, z[i][e]);  // (passes over NaN: the sum keeps it)
      }
    }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float b = fmaxf(m, top), bb = b == -INFINITY ? 0.f : b;
    s *= exp_of(m, bb);
#pragma unroll
    for (int i = 0; i < C; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) s += exp_of(z[i][e], bb);
    m = b;
  }
  if (wave >= R) return;
  s += __shfl_xor(s, 16, 64);  // (the four lanes of a row share m)
  s += __shfl_xor(s, 32, 64);
  if (q == 0 && mine < n) part[(size_t)mine * gridDim.x + blockIdx.x] = make_float2(m, s);
}

// Its parts joined, a workgroup a row: 2.4 to 3.2 us, a launch.
__global__ __launch_bounds__(256) void k_join_few(const float2* __restrict__ part, uint32_t nparts,
                                                  const uint32_t* labels, uint32_t k,
                                                  const float* zlabel, float* loss, float* lse,
                                                  uint32_t* small) {
  __shared__ float2 sh[4];
  const uint32_t i = blockIdx.x;
  const uint32_t lab = labels[i];
  const float zl = zlabel[i];
  float m = -INFINITY, s = 0.f;
  auto join = [&](float2 p) __attribute__((always_inline)) { join_sums(m, s, p); };
#pragma unroll 4
  for (uint32_t t = threadIdx.x; t < nparts; t += 256) join(part[(size_t)i * nparts + t]);
  for (int o = 32; o > 0; o >>= 1) join(make_float2(__shfl_xor(m, o, 64), __shfl_xor(s, o, 64)));
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x != 0) return;
  m = sh[0].x, s = sh[0].y;
  for (int t = 1; t < 4; t++) join(sh[t]);
  finish_row(i, m, s, lab, k, zl, loss, lse, small);
}

// The parts' maxima and sums joined: 64 rows a workgroup, 16 shares of the parts. Bound
// by latency: 16,384 rows of 8 parts 4.8 us; 8,192 of 1,024 parts (67 MB) 16.5.
__global__ __launch_bounds__(1024) void k_join(const float2* __restrict__ part, uint32_t nparts,
                                               uint32_t n, const uint32_t* labels, uint32_t k,
                                               const float* zlabel, float* loss, float* lse,
                                               uint32_t* small) {
  __shared__ float2 sh[16][64];
  const uint32_t c = threadIdx.x & 63, g = threadIdx.x >> 6;
  const uint32_t i = blockIdx.x * 64 + c;
  float m = -INFINITY, s = 0.f;
  auto join = [&](float2 p) __attribute__((always_inline)) { join_sums(m, s, p); };
  if (i < n) {
    uint32_t t = g;
    for (; t + 48 < nparts; t += 64) {  // four loads in flight
      const float2 p0 = part[(size_t)t * n + i], p1 = part[(size_t)(t + 16) * n + i],
                   p2 = part[(size_t)(t + 32) * n + i], p3 = part[(size_t)(t + 48) * n + i];
      join(p0), join(p1), join(p2), join(p3);
    }
    for (; t < nparts; t += 16) join(part[(size_t)t * n + i]);
  }
  sh[g][c] = make_float2(m, s);
  __syncthreads();
  if (g != 0 || i >= n) return;
  m = -INFINITY, s = 0.f;
#pragma unroll
  for (int t = 0; t < 16; t++) join(sh[t][c]);
  finish_row(i, m, s, labels[i], k, zlabel[i], loss, lse, small);
}

// out = the splits' sums added, in their order. Bound by the parts' bytes, which the last
// product left in the caches: 5 of 1,024 x 768 (16 MB) 4.9 us, 2 of 8,192 x 1,024 (67
// MB) 17.5.
template <class T>
__global__ __launch_bounds__(256) void k_splits(const float* __restrict__ part, uint32_t splits,
                                                size_t rows, uint32_t cols, size_t ldp, T* out,
                                                size_t ldo) {
  const size_t per = ldp / 4;
  for (size_t t = (size_t)blockIdx.x * 256 + threadIdx.x; t < rows * per;
       t += (size_t)gridDim.x * 256) {
    const size_t i = t / per;
    const uint32_t j = (uint32_t)(t % per) * 4;
    if (j >= cols) continue;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (uint32_t s = 0; s < splits; s++) {
      const float4 p = *reinterpret_cast<const float4*>(part + (s * rows + i) * ldp + j);
      v[0] += p.x, v[1] += p.y, v[2] += p.z, v[3] += p.w;
    }
    T* o = out + i * ldo + j;
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (j + e < cols) o[e] = from_f32<T>(v[e]);
  }
}

// Scratch of one call, 256-byte aligned pieces (first sized, then taken).
struct Carve {
  char* base = nullptr;
  size_t used = 0;
  template <class T>
  T* take(size_t count) {
    const size_t at = used;
    used = (at + count * sizeof(T) + 255) & ~(size_t)255;
    return reinterpret_cast<T*>(base + at);
  }
};

uint32_t up(size_t v, size_t to) { return (uint32_t)((v + to - 1) / to * to); }

// Whether rows can be the tiles' operand where they lie: every row at a 16-byte
// address, whole 16-byte chunks (whole: whole slabs, for products along the row),
// and offsets in a tile that stay below 2^31.
bool direct(const MatIn& m, size_t d, bool whole) {
  return m.kind != EMH_F32 && (uintptr_t)m.p % 16 == 0 && m.ld % 8 == 0 &&
         m.ld < (size_t(1) << 22) && d % (whole ? SLAB : 8) == 0;
}

// An operand of the products: as it lies, or laid out in the call's scratch.
struct Laid {
  bool packed = false;
  uint32_t dp = 0;  // elements of a laid-out row
  char* p[2] = {nullptr, nullptr};
  int* ex = nullptr;
  void size(Carve& w, const MatIn& m, size_t rows, size_t d, bool need) {
    packed = need;
    dp = up(d, SLAB);
    if (!need) return;
    p[0] = w.take<char>(rows * dp * 2);
    if (m.kind == EMH_F32) {
      p[1] = w.take<char>(rows * dp * 2);
      ex = w.take<int>(rows + ALL_COLS);  // (the tiles read whole column tiles of them)
    }
  }
  Operand deep(const MatIn& m, size_t first, size_t rows) const {
    Operand o{};
    o.ld = packed ? dp * 2 : (uint32_t)(m.ld * 2);
    for (int i = 0; i < 2; i++)  // (of 16 bits there is one plane)
      o.p[i] = (packed ? p[p[1] ? i : 0] : (char*)m.p) + first * o.ld;
    o.rows = (uint32_t)rows;
    o.wide = packed ? dp : 0;
    return o;
  }
};

// Lays out the operands that need it; labels: see PackOne, for x.
void pack(emh_ctx* c, const XentIn& in, const Laid& x, const Laid& w, const uint32_t* labels) {
  PackArgs a{};
  unsigned blocks = 0;
  auto add = [&](PackOne& m, const MatIn& from, size_t rows, const Laid& to, const uint32_t* lab) {
    m = {from.p, from.ld, rows, lab, to.p[0], to.p[1], to.ex,
         (uint32_t)std::min((rows + 3) / 4, MAX_GROUPS)};
    blocks += m.blocks;
    a.dp = to.dp;
  };
  if (x.packed) add(a.m[0], in.x, in.n, x, labels);
  a.first = blocks;
  if (w.packed) add(a.m[1], in.w, in.k, w, nullptr);
  if (blocks == 0) return;
  a.d = (uint32_t)in.d, a.k = (uint32_t)in.k;
  if (in.x.kind == EMH_F32)
    k_pack32<<<dim3(blocks), 256, 0, c->stream>>>(a);
  else  // (16-bit words, whatever they stand for)
    k_pack16<f16><<<dim3(blocks), 256, 0, c->stream>>>(a);
}

// At most this many rows take the kernel that reads the classes once, as they lie. (64
// rows of 768 in bf16 by 16,384 classes 12.8 us, in tiles 14.0; by 131,071 56.7 and 53.0;
// f32, which the tiles have laid out first, by 65,536 87 and 129.)
constexpr size_t FEW_ROWS = 64;
constexpr uint32_t FEW_BLOCKS = 2048;
template <class T>
void few(emh_ctx* c, const XentIn& in, float* loss, float* lse) {
  const uint32_t n = (uint32_t)in.n, k = (uint32_t)in.k;
  // 16 of 768 in bf16 by 8,192: 9.8 us wide, 8.8 not; by 16,384: 9.7 and 11.2. One row,
  // which stays in the L1: by 16,384 10.1 and 9.1, f32 by 65,536 37.3 and 40.4.
  const bool wide = k >= (n > 4 ? 16384u : 65536u);
  const uint32_t per = wide ? 64 : 16;
  const uint32_t blocks = std::min((k + per - 1) / per, FEW_BLOCKS);
  char* ws = (char*)c->xent.get((size_t)blocks * n * sizeof(float2) + n * 4);
  float2* part = (float2*)ws;
  float* zlabel = (float*)(part + (size_t)blocks * n);
  auto run = [&](auto kernel) {
    kernel<<<dim3(blocks), 256, 0, c->stream>>>((const T*)in.x.p, in.x.ld, n, (uint32_t)in.d,
                                                (const T*)in.w.p, in.w.ld, k, in.labels,
                                                in.scale, part, zlabel);
  };
  auto shaped = [&](auto odd) {
    constexpr bool ODD = decltype(odd)::value;
    if (n <= 16)
      wide ? run(k_few<T, 1, 4, ODD>) : run(k_few<T, 1, 1, ODD>);
    else if (n <= 32)
      wide ? run(k_few<T, 2, 4, ODD>) : run(k_few<T, 2, 1, ODD>);
    else
      wide ? run(k_few<T, 4, 4, ODD>) : run(k_few<T, 4, 1, ODD>);
  };
  auto odd = [](const MatIn& m) { return m.ld % 2 != 0 || (uintptr_t)m.p % 4 != 0; };
  if constexpr (sizeof(T) == 2) {
    // (57 rows of 641 in bf16 by 59,673: 71 us without, 44 with.)
    odd(in.x) || odd(in.w) ? shaped(std::true_type{}) : shaped(std::false_type{});
  } else {
    shaped(std::false_type{});
  }
  // (A launch of its own: the fence and the ticket that let the last workgroup join
  // the parts cost 70 us with 1,024 workgroups, 6 with 16.)
  k_join_few<<<dim3(n), 256, 0, c->stream>>>(part, blocks, in.labels, k, zlabel, loss, lse, c->small);
  EMH_HIP(hipGetLastError());
}

// The shape and splits of a product of rows x cols over `slabs` (of f32's planes): the
// fewest rounds of workgroups times a workgroup's time, with the cost of
// writing and adding the splits' sums.
struct Plan {
  Tile tile = TILE_L;
  uint32_t rtiles = 1, ctiles = 1, splits = 1, passes = 1, slabs = 1;
};
Plan plan_of(size_t rows, size_t cols, size_t slabs, bool planes, int cus, bool may_split) {
  // us a slab on a full card (256 x 256: 1.18 PFLOP/s), workgroups a CU. 128 x 128 two
  // a CU for many tiles, else one with a deeper ring (10,007 x 300 by 1,000 f32: dx
  // without splits, dw in 10 instead of 30, 12 us less a training pass). Of a
  // slab of both of f32's planes (TILE_BOTH) STEP_BOTH.
  constexpr double STEP[TILES] = {1.8, 1.4, 1.2, 0.6}, STEP_BOTH = 1.2;
  constexpr int PER_CU[TILES] = {1, 1, 2, 1};
  Plan best;
  double least = 1e300;
  for (int tile = 0; tile < TILES; tile++) {
    const size_t rt = (rows + TILE_ROWS[tile] - 1) / TILE_ROWS[tile];
    const size_t ct = (cols + TILE_COLS[tile] - 1) / TILE_COLS[tile];
    const bool both = planes && TILE_BOTH[tile];
    const size_t passes = planes && !both ? 3 : 1, steps = passes * slabs;
    for (size_t s = 1; s <= (may_split ? 32 : 1); s++) {
      if (s > 1 && steps < 4 * s) break;
      if (rt * ct * s >= size_t(1) << 23) break;  // (512 threads each: a launch's limit)
      const double rounds = std::ceil((double)(rt * ct * s) / ((double)cus * PER_CU[tile]));
      double us = rounds * ((double)((steps + s - 1) / s) * (both ? STEP_BOTH : STEP[tile]) + 4.0);
      if (s > 1) us += 3.0 + 1.2e-6 * (double)s * (double)rows * (double)cols;
      if (us < least) {
        least = us;
        best = {(Tile)tile, (uint32_t)rt, (uint32_t)ct, (uint32_t)s, (uint32_t)passes,
                (uint32_t)slabs};
      }
    }
  }
  if (least == 1e300) throw Failure("cross_entropy: more tiles than a launch holds");
  return best;
}

void set_plan(TileIn& t, const Plan& p) {
  t.slabs = p.slabs, t.passes = p.passes;
  t.rtiles = p.rtiles, t.ctiles = p.ctiles, t.splits = p.splits;
}

// A gradient's classes in pieces and its rows in blocks, and the shapes and splits of the
// products of a whole block and piece. What bounds them is G's bytes, `workspace` (and a
// sixteenth more, for whole tiles of every shape; 256 x 768 of it at least). The
// pieces are all of one size (a small last one, in a few workgroups, took as
// long as 0.17 of a whole one: 8,192 rows of 1,024 against 131,071, 8.43 ms a training
// pass, now 8.29), whole rows of dw's tiles each. The rows are one block where 768 classes
// of them fit, else blocks of one size that hold up to CUT_COLS classes: deep enough
// for both products, whose sums over blocks and pieces are added in memory.
struct GradPlan {
  size_t n, d, planes, pieces, piece, blocks, block, grows, gcols;  // G: grows x gcols
  bool f32;
  int cus;
  Plan px, pw;
};
constexpr size_t CUT_COLS = 5 * ALL_COLS;
GradPlan grad_plan(size_t n, size_t d, size_t k, bool f32, int cus, size_t workspace) {
  GradPlan g{};
  g.n = n, g.d = d, g.f32 = f32, g.cus = cus;
  g.planes = f32 ? 4 : 1;
  const size_t room = workspace / (2 * g.planes);  // elements of G
  g.blocks = 1, g.block = n;
  if (up(n, ALL_ROWS) > room / ALL_COLS) {
    const size_t cols = std::min<size_t>(up(k, ALL_COLS), CUT_COLS);
    const size_t rows = std::max<size_t>(ALL_ROWS, room / cols / ALL_ROWS * ALL_ROWS);
    g.blocks = (n + rows - 1) / rows;
    if (g.blocks > 1) g.block = up((n + g.blocks - 1) / g.blocks, ALL_ROWS);
    g.blocks = (n + g.block - 1) / g.block;
  }
  g.grows = up(g.block, ALL_ROWS);
  size_t most = std::max<size_t>(ALL_COLS, room / g.grows);
  if (most < 16 * ALL_COLS) most -= most % ALL_COLS;
  g.pieces = (k + most - 1) / most;
  g.piece = g.pieces == 1 ? k : up((k + g.pieces - 1) / g.pieces, ALL_ROWS);
  g.pieces = (k + g.piece - 1) / g.piece;
  g.gcols = up(g.piece, ALL_COLS);
  // (dx's sums are those of all rows: in splits only where the rows are one block.)
  g.px = plan_of(g.block, d, (g.piece + SLAB - 1) / SLAB, f32, cus, g.blocks == 1);
  g.pw = plan_of(g.piece, d, (g.block + SLAB - 1) / SLAB, f32, cus, true);
  return g;
}
// The products of a block of nr rows and a piece of m classes. A last one may have fewer
// steps than the others have splits. (Their sums, of all splits, are there by then: it
// adds to the first of them.)
Plan logits_plan(const GradPlan& g, size_t nr, size_t m) {
  return plan_of(nr, m, up(g.d, SLAB) / SLAB, g.f32, g.cus, false);
}
Plan cut(Plan p, size_t rows, size_t depth) {
  p.rtiles = (uint32_t)((rows + TILE_ROWS[p.tile] - 1) / TILE_ROWS[p.tile]);
  p.slabs = (uint32_t)((depth + SLAB - 1) / SLAB);
  p.splits = std::min(p.splits, p.slabs * p.passes);
  return p;
}
Plan dx_plan(const GradPlan& g, size_t nr, size_t m) { return cut(g.px, nr, m); }
Plan dw_plan(const GradPlan& g, size_t nr, size_t m) { return cut(g.pw, m, nr); }
// f(first row, rows, first class, classes) for every block of every piece.
template <class F>
void by_part(const GradPlan& g, size_t k, F&& f) {
  for (size_t v0 = 0; v0 < k; v0 += g.piece)
    for (size_t r0 = 0; r0 < g.n; r0 += g.block)
      f(r0, std::min(g.block, g.n - r0), v0, std::min(g.piece, k - v0));
}

void join_splits(emh_ctx* c, const float* part, uint32_t splits, size_t rows, size_t cols, size_t ldp,
                 void* out, size_t ldo, int kind) {
  const dim3 grid((unsigned)std::min((rows * (ldp / 4) + 255) / 256, MAX_GROUPS));
  if (kind == EMH_F32)
    k_splits<float><<<grid, 256, 0, c->stream>>>(part, splits, rows, (uint32_t)cols, ldp, (float*)out, ldo);
  else if (kind == EMH_F16)
    k_splits<f16><<<grid, 256, 0, c->stream>>>(part, splits, rows, (uint32_t)cols, ldp, (f16*)out, ldo);
  else
    k_splits<bf16><<<grid, 256, 0, c->stream>>>(part, splits, rows, (uint32_t)cols, ldp, (bf16*)out, ldo);
}

}  // namespace

void launch_cross_entropy(emh_ctx* c, const XentIn& in, float* loss, float* lse) {
  const size_t n = in.n, d = in.d, k = in.k;
  const bool f32 = in.x.kind == EMH_F32;
  if (n <= FEW_ROWS) {
    if (f32)
      few<float>(c, in, loss, lse);
    else if (in.x.kind == EMH_F16)
      few<f16>(c, in, loss, lse);
    else
      few<bf16>(c, in, loss, lse);
    return;
  }
  const size_t slabs = up(d, SLAB) / SLAB;
  // Rows at a time: what bounds them is the parts' maxima and sums (512 MB, or those of
  // 256 rows: 32 bytes a class).
  const size_t all = (k + 127) / 128 * 2;
  const size_t rows = std::min(n, std::max<size_t>(256, ((size_t(64) << 20) / all) & ~(size_t)255));
  Carve w;
  Laid lx, lw;
  float2* part = nullptr;
  float* zlabel = nullptr;
  for (int pass = 0; pass < 2; pass++) {
    w.used = 0;
    lx.size(w, in.x, n, d, !direct(in.x, d, true));
    lw.size(w, in.w, k, d, !direct(in.w, d, true));
    part = w.take<float2>(all * rows);
    zlabel = w.take<float>(rows);
    if (pass == 0) w.base = (char*)c->xent.get(w.used);
  }
  pack(c, in, lx, lw, nullptr);
  for (size_t r0 = 0; r0 < n; r0 += rows) {
    const size_t m = std::min(rows, n - r0);
    const Plan p = plan_of(m, k, slabs, f32, c->cus, false);
    LogitArgs a{};
    a.t.r = lx.deep(in.x, r0, m);
    a.t.c = lw.deep(in.w, 0, k);
    set_plan(a.t, p);
    a.n = (uint32_t)m, a.m = a.k = (uint32_t)k;
    a.labels = in.labels + r0;
    a.scale = in.scale;
    a.ex = f32 ? lx.ex + r0 : nullptr;
    a.ew = lw.ex;
    a.part = part, a.zlabel = zlabel;
    launch_logits(c->stream, a, in.x.kind, p.tile, false);
    k_join<<<grid1(m, 64), 1024, 0, c->stream>>>(part, p.ctiles * PARTS, (uint32_t)m, in.labels + r0,
                                                 (uint32_t)k, zlabel, loss + r0,
                                                 lse ? lse + r0 : nullptr, c->small);
    EMH_HIP(hipGetLastError());
  }
}

void launch_cross_entropy_grad(emh_ctx* c, const XentIn& in, const float* lse, const float* gloss,
                               float loss_scale, const MatOut& dx, const MatOut& dw) {
  const size_t n = in.n, d = in.d, k = in.k;
  const bool f32 = in.x.kind == EMH_F32;
  if (n == 0) {  // no row, no gradient
    if (dw.p) join_splits(c, nullptr, 0, k, d, up(d, 4), dw.p, dw.ld, dw.kind);
    EMH_HIP(hipGetLastError());
    return;
  }
  const GradPlan gp = grad_plan(n, d, k, f32, c->cus, c->xent_workspace);
  const size_t planes = gp.planes, ldg = gp.gcols * 2, ldp = up(d, 4);
  const bool px_part = gp.px.splits > 1 || gp.pieces > 1, pw_part = gp.pw.splits > 1 || gp.blocks > 1;
  // Rows without a label: see OddRows. (Several blocks would need a flag each: their rows are
  // laid out for the call.)
  const bool x_as_is = direct(in.x, d, true) && gp.blocks == 1;
  Carve w;
  Laid lx, lw;
  XentState* st = nullptr;
  uint32_t* counts = nullptr;
  char* G[4] = {};
  float *partx = nullptr, *partw = nullptr;
  for (int pass = 0; pass < 2; pass++) {
    w.used = 0;
    st = w.take<XentState>(1);
    counts = w.take<uint32_t>(MANY_COUNTS);
    lx.size(w, in.x, n, d, true);
    lw.size(w, in.w, k, d, !direct(in.w, d, true));
    for (size_t i = 0; i < planes; i++) G[i] = w.take<char>(gp.grows * ldg);
    if (dx.p && px_part) partx = w.take<float>(gp.px.splits * n * ldp);
    if (dw.p && pw_part) partw = w.take<float>((size_t)gp.pw.splits * gp.piece * ldp);
    if (pass == 0) w.base = (char*)c->xent.get(w.used);
  }
  const uint32_t call = ++c->xent_calls;
  pack(c, in, x_as_is ? Laid{} : lx, lw, in.labels);
  const Plan first = logits_plan(gp, gp.block, gp.piece);
  const size_t waves = (size_t)first.rtiles * TILE_WAVES[first.tile];
  const bool counted = !f32 && !gloss && waves <= MANY_COUNTS && gp.blocks == 1;
  if (!counted) {
    k_survey<<<dim3(1), 1024, 0, c->stream>>>((uint32_t)n, in.labels, (uint32_t)k, gloss, lx.ex, lw.ex,
                                              st, c->small);
    EMH_HIP(hipGetLastError());
  }
  Laid as_is;
  const Laid& xl = x_as_is ? as_is : lx;
  by_part(gp, k, [&](size_t r0, size_t nr, size_t v0, size_t m) {
    const Plan pg = logits_plan(gp, nr, m), px = dx_plan(gp, nr, m), pw = dw_plan(gp, nr, m);
    if ((size_t)pg.rtiles * TILE_ROWS[pg.tile] > gp.grows ||
        (size_t)pg.ctiles * TILE_COLS[pg.tile] > gp.gcols)
      throw Failure("cross_entropy_grad: tiles beyond the piece");
    LogitArgs a{};
    a.t.r = xl.deep(in.x, r0, nr);
    a.t.c = lw.deep(in.w, v0, m);
    set_plan(a.t, pg);
    a.n = (uint32_t)nr, a.m = (uint32_t)m, a.col0 = (uint32_t)v0, a.k = (uint32_t)k;
    a.labels = in.labels + r0;
    a.scale = in.scale;
    a.ex = f32 ? lx.ex + r0 : nullptr, a.ew = f32 ? lw.ex + v0 : nullptr;
    a.lse = lse + r0, a.gloss = gloss ? gloss + r0 : nullptr, a.st = st;
    a.small = c->small;
    if (counted) a.counts = counts;
    OddRows odd{};
    if (x_as_is && dw.p && v0 == 0)
      odd = {c->small + SW_ODD_ROW, call, lx.p[0], lx.dp, (const char*)in.x.p, in.x.ld, d};
    a.odd = odd;
    for (int i = 0; i < 4; i++) a.g[i] = G[i];
    a.ldg = ldg;
    launch_logits(c->stream, a, in.x.kind, pg.tile, true);
    ProdArgs p{};
    p.labels = a.labels, p.k = (uint32_t)k;
    p.gloss = a.gloss, p.st = st, p.scale = in.scale * loss_scale;
    if (counted) p.counts = counts, p.ncounts = (uint32_t)waves;
    p.cols = (uint32_t)d, p.ldp = ldp;
    if (dx.p) {
      p.t.r = {{G[0], G[f32 ? 1 : 0]}, (uint32_t)ldg, (uint32_t)nr, 0};
      p.t.c = lw.deep(in.w, v0, m);
      p.t.c.wide = lw.packed ? lw.dp : (uint32_t)d;
      set_plan(p.t, px);
      p.rows = (uint32_t)nr, p.dw = false;
      p.ex = a.ex;
      p.out = (char*)dx.p + r0 * dx.ld * kind_bytes(dx.kind), p.ldo = dx.ld;
      p.part = px_part ? partx + r0 * ldp : nullptr;
      p.part_rows = n;
      p.add = v0 > 0;
      p.odd = odd;
      launch_prod(c->stream, p, in.x.kind, px.tile);
    } else if (odd.flag) {
      launch_copy_rows(c, odd, (uint32_t)n, in.labels, (uint32_t)k);
    }
    if (dw.p) {
      p.t.r = {{G[0], G[f32 ? 1 : 0]}, (uint32_t)ldg, up(nr, SLAB), (uint32_t)gp.gcols};
      p.gb[0] = G[2], p.gb[1] = G[3];
      p.ex = a.ew;
      p.t.c = xl.deep(in.x, r0, nr);
      p.t.c.wide = xl.packed ? xl.dp : (uint32_t)d;
      set_plan(p.t, pw);
      p.rows = (uint32_t)m, p.dw = true;
      p.out = (char*)dw.p + v0 * dw.ld * kind_bytes(dw.kind), p.ldo = dw.ld;
      p.part = pw_part ? partw : nullptr;
      p.part_rows = m;
      p.add = r0 > 0;
      if (x_as_is) {
        p.flag = c->small + SW_ODD_ROW;
        p.call = call;
        p.alt = lx.deep(in.x, 0, n);
      }
      launch_prod(c->stream, p, in.x.kind, pw.tile);
      if (pw_part && r0 + nr == n)
        join_splits(c, partw, gp.pw.splits, m, d, ldp, p.out, dw.ld, dw.kind);
    }
  });
  if (dx.p && px_part) join_splits(c, partx, gp.px.splits, n, d, ldp, dx.p, dx.ld, dx.kind);
  EMH_HIP(hipGetLastError());
}

std::vector<emh_xent_product> cross_entropy_products(size_t n, size_t d, size_t k, bool f32, int cus,
                                                     size_t workspace) {
  std::vector<emh_xent_product> out;
  if (n == 0) return out;
  const GradPlan gp = grad_plan(n, d, k, f32, cus, workspace);
  by_part(gp, k, [&](size_t r0, size_t nr, size_t v0, size_t m) {
    auto add = [&](int what, const Plan& p) {
      out.push_back({what, TILE_ROWS[p.tile], TILE_COLS[p.tile], p.rtiles, p.ctiles, p.splits,
                     p.slabs, p.passes, r0, nr, v0, m, gp.grows * gp.gcols * 2 * gp.planes});
    };
    add(EMH_XENT_LOGITS, logits_plan(gp, nr, m));
    add(EMH_XENT_DX, dx_plan(gp, nr, m));
    add(EMH_XENT_DW, dw_plan(gp, nr, m));
  });
  return out;
}

}  // namespace emh
