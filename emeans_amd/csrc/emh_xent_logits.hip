// The cross entropy's logits in tiles: every row's maximum and sum over each tile's
// columns, or the gradients of a piece of the classes (emh_xent.h).
#include "emh_xent.h"

namespace emh {
namespace {

// x with zeros in rows without a label (OddRows): every workgroup its share.
template <class T>
__device__ __forceinline__ void copy_rows(const LogitArgs& a) {
  const OddRows& o = a.odd;
  for (uint32_t i = blockIdx.x; i < a.n; i += gridDim.x) {
    const T* row = reinterpret_cast<const T*>(o.x) + i * o.ld;
    const bool has = a.labels[i] < a.k;
    for (uint32_t c = threadIdx.x * 8; c < o.dp; c += blockDim.x * 8) {
      Vec<T> v{make_uint4(0u, 0u, 0u, 0u)};
      if (has && c < o.d)
        v = c + 8 <= o.d ? load_vec(row + c) : load_some(row + c, (int)(o.d - c));
      *reinterpret_cast<uint4*>(o.rows + ((size_t)i * o.dp + c) * 2) = v.raw;
    }
  }
}

// F32: operands are planes of f16 with exponents.
template <class T, class S, bool F32, bool GRAD>
__global__ __launch_bounds__(S::THREADS, 2) void k_logits(const LogitArgs a) {
  __shared__ __attribute__((aligned(1024))) char ring[S::RING];
  if constexpr (GRAD && !F32) {
    if (a.odd.flag && *a.odd.flag == a.odd.call) copy_rows<T>(a);
  }
  const TileAt at = tile_at(a.t);
  v16f acc[S::WA][S::WB];
  tile_sums<T, S, true, true>(a.t, at, ring, acc);

  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, li = lane & 31, h = lane >> 5;
  const int wr = w % S::NWR, wc = w / S::NWR;
  const uint32_t i0 = at.rt * S::TR + wr * S::WB * 32 + li;
  const uint32_t j0 = at.ct * S::TC + wc * S::WA * 32;

  // To logits.
  int ex[S::WB];
#pragma unroll
  for (int y = 0; y < S::WB; y++) ex[y] = F32 ? a.ex[min(i0 + y * 32, a.n - 1)] : 0;
#pragma unroll
  for (int b = 0; b < S::WA; b++)
#pragma unroll
    for (int q = 0; q < 4; q++) {
      int ew[4] = {0, 0, 0, 0};
      if constexpr (F32) {  // (the exponents' buffer is a whole number of tiles long)
        const int4 v = *reinterpret_cast<const int4*>(a.ew + j0 + b * 32 + 8 * q + 4 * h);
        ew[0] = v.x, ew[1] = v.y, ew[2] = v.z, ew[3] = v.w;
      }
#pragma unroll
      for (int e = 0; e < 4; e++)
#pragma unroll
        for (int y = 0; y < S::WB; y++) {
          const float z = acc[b][y][4 * q + e];
          acc[b][y][4 * q + e] = (F32 ? ldexpf(z, ex[y] + ew[e]) : z) * a.scale;
        }
    }

  // Columns of the wave that there are; all of them but in the last tile.
  const int left = (int)min(a.m - min(a.m, j0), (uint32_t)(S::WA * 32));
  const bool full = left == S::WA * 32;
  if constexpr (!GRAD) {
    const uint32_t pi = at.ct * S::NWC + wc;
    if (!full) {
      int have = left - 4 * h;
      asm volatile("" : "+v"(have));  // (the comparisons are made here, not kept)
#pragma unroll
      for (int b = 0; b < S::WA; b++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          const bool in = b * 32 + 8 * (r >> 2) + (r & 3) < have;
#pragma unroll
          for (int y = 0; y < S::WB; y++) acc[b][y][r] = in ? acc[b][y][r] : -INFINITY;
        }
    }
#pragma unroll
    for (int y = 0; y < S::WB; y++) {
      const uint32_t i = i0 + y * 32;
      const uint32_t lab = i < a.n ? a.labels[i] : NO_LABEL;
      uint32_t own = lab - j0 - 4 * h;  // the label's column of the lane's, if it has it
      asm volatile("" : "+v"(own));
      float m = -INFINITY, z = 0.f;
      bool mine = false;
#pragma unroll
      for (int b = 0; b < S::WA; b++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          const bool is = own == (uint32_t)(b * 32 + 8 * (r >> 2) + (r & 3));
          z = is ? acc[b][y][r] : z;
          mine = mine || is;
          m = fmaxf(m, acc[b][y][r]);  // (passes over NaN: the sum keeps it)
        }
      if (mine && lab < a.k) a.zlabel[i] = z;
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      const float mm = m == -INFINITY ? 0.f : m;
      float s = 0.f;
#pragma unroll
      for (int b = 0; b < S::WA; b++)
#pragma unroll
        for (int r = 0; r < 16; r++) s += exp_of(acc[b][y][r], mm);
      s += __shfl_xor(s, 32, 64);
      if (h == 0 && i < a.n) a.part[(size_t)pi * a.n + i] = make_float2(m, s);
    }
  } else {
    // G in place of the logits.
#pragma unroll
    for (int y = 0; y < S::WB; y++) {
      const uint32_t i = i0 + y * 32;
      const uint32_t ic = min(i, a.n - 1);
      const uint32_t lab = i < a.n ? a.labels[ic] : NO_LABEL;
      const bool has = lab < a.k;
      const float lse = a.lse[ic];
      const float u = a.gloss ? a.gloss[ic] : 1.f;
      // The label's column (another piece's: none of this one), and the columns
      // there are, none in a row without a label, from the lane's first.
      uint32_t own = lab - a.col0 - j0 - 4 * h;
      int have = (has ? left : 0) - 4 * h;
      asm volatile("" : "+v"(own), "+v"(have));
#pragma unroll
      for (int b = 0; b < S::WA; b++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          const int c = b * 32 + 8 * (r >> 2) + (r & 3);
          const float soft = exp_of(acc[b][y][r], lse);
          const float g = (soft - (own == (uint32_t)c ? 1.f : 0.f)) * u;
          acc[b][y][r] = c < have ? g : 0.f;
        }
    }
    // Through LDS (the ring is free once every wave is here), so that a row's
    // 2 TC bytes go to memory together: eight columns a lane are one 16-byte chunk,
    // XOR-swizzled by the row.
    RowScale rs;
    rs.init(a.st, a.gloss, a.scale);
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
          ga = one ? ex[y] + rs.gexp : row_exp(a.gloss, min(i0 + y * 32, a.n - 1));
        const uint32_t row = r0 + y * 32;
#pragma unroll
        for (int b = 0; b < S::WA; b++)
#pragma unroll
          for (int p = 0; p < 2; p++) {
            float lo[4], hi[4], g[8];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              lo[e] = acc[b][y][8 * p + e];
              hi[e] = acc[b][y][8 * p + 4 + e];
            }
            eight(lo, hi, g);
            if constexpr (F32) {
              int by[8];
              if (plane < 2) {
                const uint32_t j = j0 + b * 32 + 16 * p + 8 * h;
                const int4 w0 = *reinterpret_cast<const int4*>(a.ew + j);
                const int4 w1 = *reinterpret_cast<const int4*>(a.ew + j + 4);
                const int ew[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
                for (int e = 0; e < 8; e++) by[e] = ew[e] - ewmax + ga;
              } else {
#pragma unroll
                for (int e = 0; e < 8; e++) by[e] = ex[y] + rs.gexp;
              }
#pragma unroll
              for (int e = 0; e < 8; e++) {
                const float t = ldexpf(g[e], by[e]);
                g[e] = plane & 1 ? t - (float)(f16)t : t;
              }
            } else if constexpr (__is_same(T, f16)) {
#pragma unroll
              for (int e = 0; e < 8; e++) g[e] = ldexpf(g[e], rs.gexp);
            }
            const uint32_t chunk = (wc * S::WA + b) * 4 + 2 * p + h;
            store_vec(reinterpret_cast<T*>(ring + row * S::TC * 2 + ((chunk ^ (row & 7)) << 4)), g);
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
void launch(hipStream_t s, const LogitArgs& a, Tile tile) {
  by_tile(tile, [&](auto shape) {
    using S = decltype(shape);
    k_logits<T, S, F32, GRAD><<<a.t.rtiles * a.t.ctiles, S::THREADS, 0, s>>>(a);
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
