// Rows in 8 bits times classes in 8 bits: y(i, v) = sum over blocks b of 128 columns of
// xs(i, b) ws(v / 128, b) (sum over the block's columns of x(i, c) w(v, c)).
//
// A block's sum is one MFMA of depth 128 (products of codes are exact in f32); it is scaled and
// added in f32, one fused multiply-add an element.
#include "emh_answer.h"
#include "emh_codes.h"

namespace emh {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

// Eight codes as f16, which holds each exactly.
__device__ __forceinline__ v8h halves8(uint32_t lo, uint32_t hi) {
  const v2h a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.f, false);
  const v2h b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.f, true);
  const v2h c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.f, false);
  const v2h d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.f, true);
  return v8h{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// A lane's 32 codes of a block.
struct Halves {
  v8h v[4];
  __device__ __forceinline__ Halves() {}
  __device__ __forceinline__ Halves(uint4 a, uint4 b)
      : v{halves8(a.x, a.y), halves8(a.z, a.w), halves8(b.x, b.y), halves8(b.z, b.w)} {}
};
// 16 x 16 x 128. Lane l gives row l % 16 of a and of b and 32 of the depth's codes, the same
// ones of both; it gets column l % 16 (of b), rows 4 (l / 16) .. + 3 (of a).
__device__ __forceinline__ v4f block16(const Halves& a, const Halves& b) {
  v4f t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; i++)
    t = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v[i], b.v[i], t, 0, 0, 0);
  return t;
}

// The 16 codes of a row from column c on, zeros from column d on.
__device__ __forceinline__ uint4 codes16(const uint8_t* row, size_t c, size_t d) {
  if (c >= d) return make_uint4(0u, 0u, 0u, 0u);
  const uint4 v = *reinterpret_cast<const uint4*>(row + c);
  if (c + 16 <= d) return v;
  const int left = (int)(d - c);
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int have = left - 4 * i;
    w[i] = have >= 4 ? w[i] : have <= 0 ? 0u : w[i] & ((1u << (8 * have)) - 1u);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// Few rows: a workgroup takes 16 classes and 16 YB rows, its four waves the blocks of the depth
// by turns; operands come from memory as they lie.
template <int YB>
__global__ __launch_bounds__(256) void k_few8(const CodedIn x, size_t n, size_t d, const CodedIn w,
                                              size_t k, void* y, size_t ldy, int kind,
                                              uint32_t rgroups, size_t groups) {
  __shared__ v4f sums[4][YB][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, g = lane >> 4;
  const size_t blocks = (d + CODE_BLOCK - 1) / CODE_BLOCK;
  for (size_t u = blockIdx.x; u < groups; u += gridDim.x) {
    const size_t cg = u / rgroups, r0 = (u - cg * rgroups) * (16 * YB), v0 = cg * 16;
    const uint8_t* wp = w.q + min(v0 + li, k - 1) * w.ld;
    const uint8_t* xp[YB];
    const float* sp[YB];
#pragma unroll
    for (int b = 0; b < YB; b++) {
      const size_t row = min(r0 + b * 16 + li, n - 1);
      xp[b] = x.q + row * x.ld;
      sp[b] = x.scale + row * x.lds;
    }
    const float* ws = w.scale + v0 / CODE_BLOCK * w.lds;
    v4f acc[YB];
#pragma unroll
    for (int b = 0; b < YB; b++) acc[b] = v4f{0.f, 0.f, 0.f, 0.f};
    for (size_t s = wave; s < blocks; s += 4) {
      const size_t c = s * CODE_BLOCK + 16 * g;
      const Halves a(codes16(wp, c, d), codes16(wp, c + 64, d));
      const float by = ws[s];
#pragma unroll
      for (int b = 0; b < YB; b++) {
        const v4f t = block16(a, Halves(codes16(xp[b], c, d), codes16(xp[b], c + 64, d)));
        const float f = sp[b][s] * by;
#pragma unroll
        for (int e = 0; e < 4; e++) acc[b][e] = fmaf(t[e], f, acc[b][e]);
      }
    }
#pragma unroll
    for (int b = 0; b < YB; b++) sums[wave][b][lane] = acc[b];
    __syncthreads();
    for (int b = wave; b < YB; b += 4) {
      const size_t row = r0 + b * 16 + li;
      const v4f t = (sums[0][b][lane] + sums[1][b][lane]) + (sums[2][b][lane] + sums[3][b][lane]);
      if (row < n) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const size_t v = v0 + 4 * g + e;
          if (v < k) store_kind(y, kind, row * ldy + v, t[e]);
        }
      }
    }
    __syncthreads();  // the next group's sums take their place
  }
}

}  // namespace

void launch_product8(emh_ctx* c, const CodedIn& x, size_t n, size_t d, const CodedIn& w, size_t k,
                     const MatOut& y) {
  if (n == 0) return;
  auto few = [&](auto yb) {
    constexpr int YB = decltype(yb)::value;
    const size_t rg = (n + 16 * YB - 1) / (16 * YB), groups = (k + 15) / 16 * rg;
    k_few8<YB><<<dim3((unsigned)std::min(groups, MAX_GROUPS)), 256, 0, c->stream>>>(
        x, n, d, w, k, y.p, y.ld, y.kind, (uint32_t)rg, groups);
  };
  if (n <= 16)
    few(std::integral_constant<int, 1>{});
  else if (n <= 32)
    few(std::integral_constant<int, 2>{});
  else
    few(std::integral_constant<int, 4>{});
  EMH_HIP(hipGetLastError());
}

}  // namespace emh
