// Softmax cross entropy of rows against a linear classifier's classes, and its
// gradients, without an n x k matrix of logits.
//
// Every product is a tile of 64 x 64 dots, 4 x 4 a thread, over slabs of 16
// columns in LDS, in f32.
#include <algorithm>

#include "emh_learn.h"
#include "emh_types.h"

namespace emh {
namespace {

constexpr float LOG2E = 1.44269504f, LN2 = 0.693147181f;

// Element (i, k) of an operand at i si + k sk.
struct Side {
  const void* p;
  int kind;
  size_t si, sk, rows;
};
struct ProdArgs {
  Side a, b;
  size_t depth;
  int mode;  // 0 statistics, 1 gradients of logits, 2 f32 out (+=), 3 out in kind
  const uint32_t* labels;
  float s2;  // scale log2(e)
  float2* part;   // mode 0: [column tile][row]
  float* zlabel;  // ... the label's logit times log2(e)
  size_t col0;    // the first class of the piece
  const float* lse;
  const float* up;   // gloss, or one value for all rows
  int up_each;
  float scale;
  void* out;
  size_t ldo;
  int okind, add;
};

__global__ __launch_bounds__(256) void k_prod(const ProdArgs g) {
  __shared__ float A[16][68], B[16][68];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const size_t i0 = (size_t)blockIdx.y * 64, j0 = (size_t)blockIdx.x * 64;
  float acc[4][4] = {};
  for (size_t k0 = 0; k0 < g.depth; k0 += 16) {
    for (int t = threadIdx.x; t < 1024; t += 256) {
      // Neighbouring threads along the operand's contiguous direction.
      const int kk = g.a.sk == 1 ? t & 15 : t >> 6, r = g.a.sk == 1 ? t >> 4 : t & 63;
      const bool in = i0 + r < g.a.rows && k0 + kk < g.depth;
      A[kk][r] = in ? load_kind(g.a.p, g.a.kind, (i0 + r) * g.a.si + (k0 + kk) * g.a.sk) : 0.f;
      const int kb = g.b.sk == 1 ? t & 15 : t >> 6, q = g.b.sk == 1 ? t >> 4 : t & 63;
      const bool inb = j0 + q < g.b.rows && k0 + kb < g.depth;
      B[kb][q] = inb ? load_kind(g.b.p, g.b.kind, (j0 + q) * g.b.si + (k0 + kb) * g.b.sk) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; k++)
#pragma unroll
      for (int u = 0; u < 4; u++)
#pragma unroll
        for (int v = 0; v < 4; v++) acc[u][v] = fmaf(A[k][ty * 4 + u], B[k][tx * 4 + v], acc[u][v]);
    __syncthreads();
  }
#pragma unroll
  for (int u = 0; u < 4; u++) {
    const size_t i = i0 + ty * 4 + u;
    const bool row = i < g.a.rows;
    if (g.mode == 0) {
      const uint32_t lab = row ? g.labels[i] : NO_LABEL;
      float m = -INFINITY, s = 0.f;
#pragma unroll
      for (int v = 0; v < 4; v++) {
        const size_t j = j0 + tx * 4 + v;
        acc[u][v] = j < g.b.rows ? acc[u][v] * g.s2 : -INFINITY;
        m = fmaxf(m, acc[u][v]);
        if (row && j == lab) g.zlabel[i] = acc[u][v];
      }
      m = lanes_max<16>(m);
      const float mm = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int v = 0; v < 4; v++) s += exp2f(acc[u][v] - mm);
      s = lanes_sum<16>(s);
      if (row && tx == 0) g.part[blockIdx.x * g.a.rows + i] = make_float2(m, s);
      continue;
    }
    if (!row) continue;
#pragma unroll
    for (int v = 0; v < 4; v++) {
      const size_t j = j0 + tx * 4 + v;
      if (j >= g.b.rows) continue;
      float o = acc[u][v];
      if (g.mode == 1) {
        const uint32_t lab = g.labels[i];
        const float p = exp2f(o * g.s2 - g.lse[i] * LOG2E);
        o = (p - (g.col0 + j == lab ? 1.f : 0.f)) * (g.up[g.up_each ? i : 0] * g.scale);
        if (lab == NO_LABEL) o = 0.f;
      }
      if (g.mode == 3)
        store_kind(g.out, g.okind, i * g.ldo + j, o);
      else if (g.add)
        reinterpret_cast<float*>(g.out)[i * g.ldo + j] += o;
      else
        reinterpret_cast<float*>(g.out)[i * g.ldo + j] = o;
    }
  }
}

// The parts' maxima and sums joined, the rows' lse and loss. A label out of
// range is recorded and counts as none.
__global__ __launch_bounds__(256) void k_xent_join(const float2* part, size_t nparts, size_t n,
                                                   const uint32_t* labels, size_t k,
                                                   const float* zlabel, float* loss, float* lse,
                                                   uint32_t* small) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float m = -INFINITY, s = 0.f;
  for (size_t t = 0; t < nparts; t++) {
    const float2 p = part[t * n + i];
    const float b = fmaxf(m, p.x), mm = b == -INFINITY ? 0.f : b;
    s = s * exp2f(m - mm) + p.y * exp2f(p.x - mm);
    m = b;
  }
  const float l2 = (m == -INFINITY ? 0.f : m) + log2f(s);
  const uint32_t lab = labels[i];
  if (lse) lse[i] = l2 * LN2;
  loss[i] = lab < k ? (l2 - zlabel[i]) * LN2 : 0.f;
  if (lab >= k && lab != NO_LABEL) small[SW_BAD_CLASS] = 1u;
}

// 1 / (rows with a label), 0 when there is none.
__global__ __launch_bounds__(1024) void k_xent_count(const uint32_t* labels, size_t n, size_t k,
                                                     float* out) {
  __shared__ uint32_t c;
  if (threadIdx.x == 0) c = 0;
  __syncthreads();
  uint32_t mine = 0;
  for (size_t i = threadIdx.x; i < n; i += 1024) mine += labels[i] < k ? 1u : 0u;
  atomicAdd(&c, mine);
  __syncthreads();
  if (threadIdx.x == 0) *out = c ? 1.f / (float)c : 0.f;
}
// labels with those out of range as NONE; rows without one zeroed (f32 copies).
__global__ __launch_bounds__(256) void k_xent_rows(const void* x, int kind, size_t ldx, size_t n,
                                                   size_t d, const uint32_t* labels, size_t k,
                                                   uint32_t* lab, float* out, uint32_t* small) {
  const size_t i = blockIdx.x;
  const uint32_t l = labels[i];
  const bool has = l < k;
  if (threadIdx.x == 0) {
    lab[i] = has ? l : NO_LABEL;
    if (!has && l != NO_LABEL) small[SW_BAD_CLASS] = 1u;
  }
  for (size_t j = threadIdx.x; j < d; j += 256)
    out[i * d + j] = has ? load_kind(x, kind, i * ldx + j) : 0.f;
}
__global__ __launch_bounds__(256) void k_xent_out(const float* acc, size_t n, size_t d, void* out,
                                                  int kind, size_t ld) {
  const size_t t = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= n * d) return;
  store_kind(out, kind, t / d * ld + t % d, acc[t]);
}

void prod(emh_ctx* c, const ProdArgs& g) {
  k_prod<<<dim3((unsigned)((g.b.rows + 63) / 64), (unsigned)((g.a.rows + 63) / 64)), 256, 0,
           c->stream>>>(g);
}

}  // namespace

void launch_cross_entropy(emh_ctx* c, const XentIn& in, float* loss, float* lse) {
  const size_t parts = (in.k + 63) / 64;
  char* ws = (char*)c->xent.get(parts * in.n * 8 + in.n * 4);
  ProdArgs g{};
  g.a = {in.x.p, in.x.kind, in.x.ld, 1, in.n};
  g.b = {in.w.p, in.w.kind, in.w.ld, 1, in.k};
  g.depth = in.d;
  g.labels = in.labels;
  g.s2 = in.scale * LOG2E;
  g.part = (float2*)ws;
  g.zlabel = (float*)(ws + parts * in.n * 8);
  prod(c, g);
  k_xent_join<<<grid1(in.n, 256), 256, 0, c->stream>>>(g.part, parts, in.n, in.labels, in.k,
                                                       g.zlabel, loss, lse, c->small);
  EMH_HIP(hipGetLastError());
}

void launch_cross_entropy_grad(emh_ctx* c, const XentIn& in, const float* lse, const float* gloss,
                               const MatOut& dx, const MatOut& dw) {
  const size_t n = in.n, d = in.d, k = in.k;
  // Classes a piece: 256 MB of their gradients.
  const size_t piece = std::min(k, std::max<size_t>(64, (size_t(64) << 20) / std::max<size_t>(n, 1)));
  char* ws = (char*)c->xent.get((n * piece + 2 * n * d + n + 1) * 4);
  float* G = (float*)ws;
  float* xs = G + n * piece;
  float* acc = xs + n * d;
  uint32_t* lab = (uint32_t*)(acc + n * d);
  float* mean = (float*)(lab + n);
  if (n > 0) {
    k_xent_rows<<<dim3((unsigned)n), 256, 0, c->stream>>>(in.x.p, in.x.kind, in.x.ld, n, d,
                                                          in.labels, k, lab, xs, c->small);
    if (!gloss) k_xent_count<<<1, 1024, 0, c->stream>>>(in.labels, n, k, mean);
  }
  for (size_t v0 = 0; v0 < k; v0 += piece) {
    const size_t m = std::min(piece, k - v0);
    const char* wp = (const char*)in.w.p + v0 * in.w.ld * kind_bytes(in.w.kind);
    if (n > 0) {
      ProdArgs g{};
      g.a = {xs, EMH_F32, d, 1, n};
      g.b = {wp, in.w.kind, in.w.ld, 1, m};
      g.depth = d;
      g.mode = 1;
      g.labels = lab;
      g.s2 = in.scale * LOG2E;
      g.col0 = v0;
      g.lse = lse;
      g.up = gloss ? gloss : mean;
      g.up_each = gloss != nullptr;
      g.scale = in.scale;
      g.out = G;
      g.ldo = m;
      prod(c, g);
    }
    if (dx.p && n > 0) {
      ProdArgs g{};
      g.a = {G, EMH_F32, m, 1, n};
      g.b = {wp, in.w.kind, 1, in.w.ld, d};
      g.depth = m;
      g.mode = 2;
      g.out = acc;
      g.ldo = d;
      g.add = v0 > 0;
      prod(c, g);
    }
    if (dw.p) {
      ProdArgs g{};
      g.a = {G, EMH_F32, 1, m, m};
      g.b = {xs, EMH_F32, 1, d, d};
      g.depth = n;
      g.mode = 3;
      g.out = (char*)dw.p + v0 * dw.ld * kind_bytes(dw.kind);
      g.okind = dw.kind;
      g.ldo = dw.ld;
      prod(c, g);
    }
  }
  if (dx.p && n > 0)
    k_xent_out<<<grid1(n * d, 256), 256, 0, c->stream>>>(acc, n, d, dx.p, dx.kind, dx.ld);
  EMH_HIP(hipGetLastError());
}

}  // namespace emh
