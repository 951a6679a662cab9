// The cross entropy's gradient products: dx = G w and dw = G^T x (emh_xent.h).
#include "emh_xent.h"

namespace emh {
namespace {

// x with zeros in rows without a label (OddRows): every workgroup of `blocks` its share.
template <class T>
__device__ __forceinline__ void copy_rows(const OddRows& o, uint32_t n, const uint32_t* labels,
                                          uint32_t k, uint32_t blocks) {
  for (uint32_t i = blockIdx.x; i < n; i += blocks) {
    const T* row = reinterpret_cast<const T*>(o.x) + i * o.ld;
    const bool has = labels[i] < k;
    for (uint32_t c = threadIdx.x * 8; c < o.dp; c += blockDim.x * 8) {
      Vec<T> v{make_uint4(0u, 0u, 0u, 0u)};
      if (has && c < o.d)
        v = c + 8 <= o.d ? load_vec(row + c) : load_some(row + c, (int)(o.d - c));
      *reinterpret_cast<uint4*>(o.rows + ((size_t)i * o.dp + c) * 2) = v.raw;
    }
  }
}
// Where no dx is asked for. (16-bit words, whatever they stand for.)
__global__ __launch_bounds__(256) void k_copy_rows(const OddRows o, uint32_t n,
                                                   const uint32_t* labels, uint32_t k) {
  if (*o.flag == o.call) copy_rows<f16>(o, n, labels, k, gridDim.x);
}

// A tile of dx (rows: G's, as they lie; columns: w's, across) or of dw (both across), or
// its sums over one split of the depth or one piece of the classes. Bound by the MFMAs
// (emh_tile.h). In bf16: 16,384 x 768 by 1,024 31 us (dx) and 38 (dw in 5 splits; in 16
// of 256 x 192 tiles 35, but their sums take 9 us instead of 5); 8,192 x 1,024 by
// 131,071 1.86 and 1.82 ms, 1.18 and 1.21 PFLOP/s.
template <class T, class S, bool F32, bool DW, class O>
__global__ __launch_bounds__(S::THREADS, 2) void k_grads(const ProdArgs a) {
  __shared__ __attribute__((aligned(1024))) char ring[S::RING];
  const bool alt = DW && a.flag && *a.flag == a.call;
  if constexpr (!DW && !F32) {
    if (a.odd.flag && *a.odd.flag == a.odd.call)
      copy_rows<T>(a.odd, a.rows, a.labels, a.k, a.t.blocks);
  }
  const TileAt at = tile_at(a.t);
  v16f acc[S::WA][S::WB];
  TileIn t = a.t;
  if (alt) t.c = a.alt;
  bool one = false;
  if constexpr (F32) {
    one = a.st->one != 0;
    if (DW && !one) t.r.p[0] = a.gb[0], t.r.p[1] = a.gb[1];
  }
  tile_sums<T, S, !DW, false, F32>(t, at, ring, acc);

  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, li = lane & 31, h = lane >> 5;
  const int wr = w % S::NWR, wc = w / S::NWR;
  const uint32_t i0 = at.rt * S::TR + wr * S::WB * 32 + li;
  const uint32_t j0 = at.ct * S::TC + wc * S::WA * 32;
  const int gexp = __is_same(T, f16) ? RowScale::exponent(a.st, a.counts) : 0;
  const float factor = RowScale::factor(a.st, a.counts, a.ncounts, a.gloss, a.scale);
  if constexpr (sizeof(O) == 2) {
    if (!a.part) {
      // Through LDS (the ring is free once every wave is here), so that a row's 2 TC
      // bytes go to memory together, as G's do (emh_xent_logits.hip). (Sixteen bytes a lane
      // from the registers are as fast where rows begin at 16-byte addresses; at odd ones,
      // 57 rows of 641 by 59,673 classes, a training pass takes 173 us so and 149.)
      constexpr int CH = S::TC / 8;
      __syncthreads();
#pragma unroll
      for (int y = 0; y < S::WB; y++) {
        const bool zero = !DW && a.labels[min(i0 + y * 32, a.rows - 1)] >= a.k;
        const uint32_t row = wr * S::WB * 32 + y * 32 + li;
#pragma unroll
        for (int b = 0; b < S::WA; b++)
#pragma unroll
          for (int p = 0; p < 2; p++) {
            float v[2][4];
#pragma unroll
            for (int f = 0; f < 2; f++)
#pragma unroll
              for (int e = 0; e < 4; e++) {
                const float t = acc[b][y][4 * (2 * p + f) + e];
                v[f][e] = zero ? 0.f : (__is_same(T, f16) ? ldexpf(t, -gexp) : t) * factor;
              }
            const uint32_t chunk = (wc * S::WA + b) * 4 + 2 * p + h;
            store_vec(reinterpret_cast<O*>(ring + row * S::TC * 2 + ((chunk ^ (row & 7)) << 4)),
                      eight_of<O>(v[0], v[1]));
          }
      }
      __syncthreads();
#pragma unroll 4
      for (int t = threadIdx.x; t < S::TR * CH; t += S::THREADS) {
        const uint32_t row = t / CH, chunk = t % CH;
        const uint32_t i = at.rt * S::TR + row, j = at.ct * S::TC + chunk * 8;
        if (i >= a.rows || j >= a.cols) continue;
        const Vec<O> v{*reinterpret_cast<const uint4*>(ring + row * S::TC * 2 +
                                                       ((chunk ^ (row & 7)) << 4))};
        O* const o = reinterpret_cast<O*>(a.out) + (size_t)i * a.ldo + j;
        if (j + 8 <= a.cols)
          store_vec(o, v);
        else
          store_some(o, v, (int)(a.cols - j));
      }
      return;
    }
  }
#pragma unroll
  for (int y = 0; y < S::WB; y++) {
    const uint32_t i = i0 + y * 32;
    if (i >= a.rows) continue;
    const bool zero = !DW && a.labels[i] >= a.k;
    int by = 0;
    if constexpr (F32) {
      const int ewmax = a.st->ewmax - XENT_BIAS;
      if (one)
        by = ewmax - a.ex[i] - gexp;
      else
        by = DW ? -gexp : ewmax - row_exp(a.gloss, i);
    } else if constexpr (__is_same(T, f16)) {
      by = -gexp;
    }
#pragma unroll
    for (int b = 0; b < S::WA; b++)
#pragma unroll
      for (int p = 0; p < 2; p++) {
        float v[2][4];
#pragma unroll
        for (int f = 0; f < 2; f++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float t = acc[b][y][4 * (2 * p + f) + e];
            v[f][e] = zero ? 0.f : (__is_same(T, f16) ? ldexpf(t, by) : t) * factor;
          }
        if (a.part) {
          // Whole fours: ldp is a multiple of 4.
#pragma unroll
          for (int f = 0; f < 2; f++) {
            const uint32_t j = j0 + b * 32 + 8 * (2 * p + f) + 4 * h;
            if (j >= a.cols) continue;
            float4* o = reinterpret_cast<float4*>(
                a.part + (at.split * a.part_rows + i) * a.ldp + j);
            float4 s = make_float4(v[f][0], v[f][1], v[f][2], v[f][3]);
            if (a.add) {
              const float4 had = *o;
              s = make_float4(had.x + s.x, had.y + s.y, had.z + s.z, had.w + s.w);
            }
            *o = s;
          }
          continue;
        }
        if constexpr (sizeof(O) == 4) {
          const uint32_t j = j0 + b * 32 + 16 * p + 8 * h;
          O* o = reinterpret_cast<O*>(a.out) + (size_t)i * a.ldo + j;
          float g[8];
          eight(v[0], v[1], g);
          if (j + 8 <= a.cols) {
            store_vec(o, g);
            store_vec(o + 4, g + 4);
          } else {
#pragma unroll
            for (int e = 0; e < 8; e++)
              if (j + e < a.cols) o[e] = g[e];
          }
        }
      }
  }
}

template <class T, bool F32, class O>
void launch(hipStream_t s, ProdArgs a, Tile tile) {
  const unsigned blocks = prepare(a.t);
  by_tile(tile, [&](auto shape) {
    using S = decltype(shape);
    if (a.dw)
      k_grads<T, S, F32, true, O><<<blocks, S::THREADS, 0, s>>>(a);
    else
      k_grads<T, S, F32, false, O><<<blocks, S::THREADS, 0, s>>>(a);
  });
}

}  // namespace

void launch_copy_rows(emh_ctx* c, const OddRows& o, uint32_t n, const uint32_t* labels, uint32_t k) {
  k_copy_rows<<<dim3(std::min<uint32_t>(n, (uint32_t)c->cus * 4)), 256, 0, c->stream>>>(o, n, labels, k);
  EMH_HIP(hipGetLastError());
}

void launch_prod(hipStream_t s, const ProdArgs& a, int kind, Tile tile) {
  if (kind == EMH_F32)
    launch<f16, true, float>(s, a, tile);
  else if (kind == EMH_F16)
    launch<f16, false, f16>(s, a, tile);
  else
    launch<bf16, false, bf16>(s, a, tile);
  EMH_HIP(hipGetLastError());
}

}  // namespace emh
