// The cross entropy's logits in tiles: every row's maximum and sum over each tile's
// columns, or the gradients of a piece of the classes (emh_xent.h).
#include "emh_xent.h"

namespace emh {
namespace {

// f(c, v) in place of every v of the lane's row y, c its column less the lane's
// first, which is 4 (lane / 32).
template <class S, class F>
__device__ __forceinline__ void each(v16f (&acc)[S::WA][S::WB], int y, F&& f) {
#pragma unroll
  for (int b = 0; b < S::WA; b++)
#pragma unroll
    for (int r = 0; r < 16; r++) acc[b][y][r] = f(b * 32 + 8 * (r >> 2) + (r & 3), acc[b][y][r]);
}
// The v whose c it is (below 32 WA, a multiple of 8 and at most 3): its block first,
// half of the selections that a search of all takes.
template <class S>
__device__ __forceinline__ float at_column(const v16f (&acc)[S::WA][S::WB], int y, uint32_t c) {
  v16f v = acc[0][y];
#pragma unroll
  for (int b = 1; b < S::WA; b++) {
    const bool from = c >= (uint32_t)b * 32;
#pragma unroll
    for (int r = 0; r < 16; r++) v[r] = from ? acc[b][y][r] : v[r];
  }
  const uint32_t at = (c & 31) >> 3 << 2 | (c & 3);
  float out = v[0];
#pragma unroll
  for (int r = 1; r < 16; r++) out = at == (uint32_t)r ? v[r] : out;
  return out;
}
// Four classes' exponents (their buffer is a whole number of tiles long).
__device__ __forceinline__ int4 four_exps(const int* ew, uint32_t j) {
  return *reinterpret_cast<const int4*>(ew + j);
}

// A tile of logits, never in memory. !GRAD: its rows' maxima and sums of exponentials;
// GRAD: G instead of it. F32: operands are planes of f16 with exponents.
// Bound by the MFMAs (emh_tile.h), then by the exponentials (5 instructions an element)
// and G's bytes. In bf16: 16,384 x 768 by 1,024 28 us, and 35 with G, of which the
// loop takes 19; 8,192 x 1,024 by 131,071 1.91 ms (1.15 PFLOP/s), 2.47 with G (2.1 GB).
template <class T, class S, bool F32, bool GRAD>
__global__ __launch_bounds__(S::THREADS, 2) void k_logits(const LogitArgs a) {
  __shared__ __attribute__((aligned(1024))) char ring[S::RING];
  const TileAt at = tile_at(a.t);
  v16f acc[S::WA][S::WB];
  tile_sums<T, S, true, true, F32>(a.t, at, ring, acc);

  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, li = lane & 31, h = lane >> 5;
  const int wr = w % S::NWR, wc = w / S::NWR;
  const uint32_t i0 = at.rt * S::TR + wr * S::WB * 32 + li;
  const uint32_t j0 = at.ct * S::TC + wc * S::WA * 32;

  // The sums in their own units. The logits are these times the scale, which the
  // exponentials take in their difference (exp_of). (The paths that few calls take
  // are kept out of the others' way: a call's workgroups are few enough for the
  // instructions' first reads to count.)
  int ex[S::WB];
#pragma unroll
  for (int y = 0; y < S::WB; y++) ex[y] = F32 ? a.ex[min(i0 + y * 32, a.n - 1)] : 0;
  if constexpr (F32) {
#pragma unroll
    for (int b = 0; b < S::WA; b++)
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const int4 v = four_exps(a.ew, j0 + b * 32 + 8 * q + 4 * h);
        const int ew[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
          for (int y = 0; y < S::WB; y++)
            acc[b][y][4 * q + e] = ldexpf(acc[b][y][4 * q + e], ex[y] + ew[e]);
      }
  }
  float scale = a.scale;

  // Columns of the wave that there are; all of them but in the last tile.
  const int left = (int)min(a.m - min(a.m, j0), (uint32_t)(S::WA * 32));
  const bool full = left == S::WA * 32;
  if constexpr (!GRAD) {
    const uint32_t pi = at.ct * S::NWC + wc;
    if (__builtin_expect(!(scale > 0.f), 0)) {  // the largest sum is not the largest logit's
#pragma unroll
      for (int y = 0; y < S::WB; y++)
        each<S>(acc, y, [&](int, float v) { return v * scale; });
      scale = 1.f;
    }
    if (__builtin_expect(!full, 0)) {
      int have = left - 4 * h;
      asm volatile("" : "+v"(have));  // (the comparisons are made here, not kept)
#pragma unroll
      for (int y = 0; y < S::WB; y++)
        each<S>(acc, y, [&](int c, float v) { return c < have ? v : -INFINITY; });
    }
#pragma unroll
    for (int y = 0; y < S::WB; y++) {
      const uint32_t i = i0 + y * 32;
      const uint32_t lab = i < a.n ? a.labels[i] : NO_LABEL;
      const uint32_t own = lab - j0 - 4 * h;  // the label's column of the lane's, if it has it
      const bool mine = lab < a.k && own < S::WA * 32 && !(own & 4);
      if (__any(mine)) {
        const float z = at_column<S>(acc, y, own) * scale;
        if (mine) a.zlabel[i] = z;
      }
      float m = -INFINITY;
#pragma unroll
      for (int b = 0; b < S::WA; b++)
#pragma unroll
        for (int r = 0; r < 16; r++)
          m = fmaxf(m, acc[b][y][r]);  // (passes over NaN: the sum keeps it)
      m = fmaxf(m, __shfl_xor(m, 32, 64)) * scale;
      const float mm = m == -INFINITY ? 0.f : m;
      float s = 0.f;
#pragma unroll
      for (int b = 0; b < S::WA; b++)
#pragma unroll
        for (int r = 0; r < 16; r++) s += exp_of(acc[b][y][r], scale, mm);
      s += __shfl_xor(s, 32, 64);
      if (h == 0 && i < a.n) a.part[(size_t)pi * a.n + i] = make_float2(m, s);
    }
  } else {
    // G in place of the sums.
    uint32_t count = 0;
#pragma unroll
    for (int y = 0; y < S::WB; y++) {
      const uint32_t i = i0 + y * 32;
      const uint32_t ic = min(i, a.n - 1);
      const uint32_t lab = i < a.n ? a.labels[ic] : NO_LABEL;
      const bool has = lab < a.k;
      const float lse = a.lse[ic];
      if constexpr (!F32) {
        count += __popcll(__ballot(has && h == 0));
        if (a.counts && lab != NO_LABEL && !has) a.small[SW_BAD_CLASS] = 1u;
        if (a.odd.flag && i < a.n && !has && !(fabsf(acc[0][y][0]) < INFINITY))
          *a.odd.flag = a.odd.call;
      }
      // The label's column (another piece's: none of this one), and the columns
      // there are, none in a row without a label, from the lane's first.
      uint32_t own = lab - a.col0 - j0 - 4 * h;
      int have = (has ? left : 0) - 4 * h;
      asm volatile("" : "+v"(own), "+v"(have));
      each<S>(acc, y, [&](int, float v) { return exp_of(v, scale, lse); });
      // (Where there are many classes, few waves have a row's label.)
      if (__any(own < S::WA * 32))
        each<S>(acc, y, [&](int c, float v) { return own == (uint32_t)c ? v - 1.f : v; });
      if (__builtin_expect(a.gloss != nullptr, 0)) {
        const float u = a.gloss[ic];
        each<S>(acc, y, [&](int, float v) { return v * u; });
      }
      if (__builtin_expect(__any(!has) || !full, 0))
        each<S>(acc, y, [&](int c, float v) { return c < have ? v : 0.f; });
    }
    if constexpr (!F32) {
      if (a.counts && a.col0 == 0 && at.ct == 0 && wc == 0 && lane == 0)
        a.counts[at.rt * S::NWR + wr] = count;
    }
    // Through LDS (the ring is free once every wave is here), so that a row's
    // 2 TC bytes go to memory together: eight columns a lane are one 16-byte chunk,
    // XOR-swizzled by the row.
    const int gexp = __is_same(T, f16) ? RowScale::exponent(a.st, a.counts) : 0;
    int ewmax = 0;
    bool one = false;
    if constexpr (F32) {
      ewmax = a.st->ewmax - XENT_BIAS;
      one = a.st->one != 0;
    }
    constexpr int CH = S::TC / 8;
    const uint32_t r0 = wr * S::WB * 32 + li;
#pragma unroll
    for (int plane = 0; plane < (F32 ? 4 : 1); plane++) {
      if (plane == 2 && one) break;
      __syncthreads();
#pragma unroll
      for (int y = 0; y < S::WB; y++) {
        int ga = 0;
        if constexpr (F32)
          ga = (one ? ex[y] + gexp : row_exp(a.gloss, min(i0 + y * 32, a.n - 1))) - ewmax;
        const uint32_t row = r0 + y * 32;
#pragma unroll
        for (int b = 0; b < S::WA; b++)
#pragma unroll
          for (int p = 0; p < 2; p++) {
            float g[2][4];
#pragma unroll
            for (int f = 0; f < 2; f++) {
              int by[4] = {gexp, gexp, gexp, gexp};
              if (F32 && plane < 2) {
                const int4 v = four_exps(a.ew, j0 + b * 32 + 8 * (2 * p + f) + 4 * h);
                by[0] = v.x + ga, by[1] = v.y + ga, by[2] = v.z + ga, by[3] = v.w + ga;
              } else if (F32) {
                by[0] = by[1] = by[2] = by[3] = ex[y] + gexp;
              }
#pragma unroll
              for (int e = 0; e < 4; e++) {
                float t = acc[b][y][4 * (2 * p + f) + e];
                if constexpr (__is_same(T, f16)) t = ldexpf(t, by[e]);
                g[f][e] = F32 && (plane & 1) ? (t - (float)(f16)t) * (1.f / LOW_UNIT) : t;
              }
            }
            const uint32_t chunk = (wc * S::WA + b) * 4 + 2 * p + h;
            store_vec(reinterpret_cast<T*>(ring + row * S::TC * 2 + ((chunk ^ (row & 7)) << 4)),
                      eight_of<T>(g[0], g[1]));
          }
      }
      __syncthreads();
      char* const out = a.g[plane] + (size_t)at.rt * S::TR * a.ldg + (size_t)at.ct * S::TC * 2;
#pragma unroll 4
      for (int t = threadIdx.x; t < S::TR * CH; t += S::THREADS) {
        const uint32_t row = t / CH, chunk = t % CH;
        const uint4 v = *reinterpret_cast<const uint4*>(ring + row * S::TC * 2 +
                                                        ((chunk ^ (row & 7)) << 4));
        *reinterpret_cast<uint4*>(out + row * a.ldg + chunk * 16) = v;
      }
    }
  }
}

template <class T, bool F32, bool GRAD>
void launch(hipStream_t s, LogitArgs a, Tile tile) {
  const unsigned blocks = prepare(a.t);
  by_tile(tile, [&](auto shape) {
    using S = decltype(shape);
    k_logits<T, S, F32, GRAD><<<blocks, S::THREADS, 0, s>>>(a);
  });
}

}  // namespace

void launch_logits(hipStream_t s, const LogitArgs& a, int kind, Tile tile, bool grads) {
  if (kind == EMH_F32)
    grads ? launch<f16, true, true>(s, a, tile) : launch<f16, true, false>(s, a, tile);
  else if (kind == EMH_F16)
    grads ? launch<f16, false, true>(s, a, tile) : launch<f16, false, false>(s, a, tile);
  else
    grads ? launch<bf16, false, true>(s, a, tile) : launch<bf16, false, false>(s, a, tile);
  EMH_HIP(hipGetLastError());
}

}  // namespace emh
