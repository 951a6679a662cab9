// The cross entropy's products and what they share (emh_xent.hip,
// emh_xent_logits.hip, emh_xent_grads.hip).
//
// z = scale x w^T, in tiles (emh_tile.h), twice: for every row's maximum and sum
// of exponentials, and for the gradients of a piece of the classes, G = gloss
// (softmax - onehot), which go to memory in 16 bits; then dx = G w and dw = G^T x,
// times scale (and, for a mean, 1 / rows) in f32. A factor that all rows share is
// left out of G: most rows' label has a G of nearly -1, which 16 bits hold
// better than any product, whose rounding would be one error for all of them.
//
// Types. 16-bit rows and classes are the MFMA's operands as they are; G is
// rounded once to their type (f16: times a power of two that brings the largest
// possible element to 2^13 .. 2^14, or the gradients of a mean over many rows would be
// subnormal). float32 operands are two planes of f16: a row times a power of two
// 2^-e that brings its largest element to 2^13 .. 2^14, h = f16(x), l = f16(2^11 (x - h)),
// which hold every element to 2^-22 of itself, or to 2^-49 of the row's largest where that is
// more (an element below 2^-27 of it); h h + 2^-11 (h l + l h) leaves out 2^-22 of a product,
// as f32's own rounding would over a few terms, and takes three MFMAs of the f16 rate
// where the f32 MFMA takes sixteen. (Without the 2^11, l ends in f16's subnormals from
// 2^-16 of the largest on: columns of 1e4 and 1e-4, which the classes make up for, left
// logits 2e-3 off, now 1.3e-6, as f32 does; of 1e5 and 1e-5 0.2, now 1e-4.)
// The exponents: z = sum 2^(ex_i + ew_v). The gradient products sum over the
// class or the row, whose exponent then has to be in G, and the other one's may be. Where
// all exponents together span little (XENT_SPAN; a row of zeros does not), one G
// serves both,
//   G' = G 2^(ew_v - ewmax + ex_i + gb), dx_i = 2^(ewmax - ex_i - gb) sum_v G' w_v,
//                                        dw_v = 2^(ewmax - ew_v - gb) sum_i G' x_i;
// otherwise there are two,
//   Ga = G 2^(ew_v - ewmax + ga_i)  for dx_i = 2^(ewmax - ga_i) sum_v Ga w_v,
//   Gb = G 2^(ex_i + gb)            for dw_v = 2^-gb sum_i Gb x_i,
// with ga_i and gb such that the largest element is below 2^14: what is lost of
// the others is 2^-50 of that (of G', 2^-50 of 2^SPAN times an element's own bound).
// 10,007 x 300 by 1,000: with two G, 82 MB, their kernel takes 44 us, with one 38.
#pragma once

#include "emh_learn.h"
#include "emh_tile.h"

namespace emh {

// exp(z - of) as the softmax takes it: the difference first, in z's own units, which is
// exact where it matters (z near of); a logit in units of log 2 would be rounded by
// a unit in its last place beforehand, a relative error of |z| 2^-24 in every term.
__device__ __forceinline__ float exp_of(float z, float of) {
  return __builtin_amdgcn_exp2f((z - of) * 1.44269504f);
}
// The same of z = sum scale, which is not rounded by itself.
__device__ __forceinline__ float exp_of(float sum, float scale, float of) {
  return __builtin_amdgcn_exp2f(fmaf(sum, scale, -of) * 1.44269504f);
}
// A row's maximum and sum of exponentials, joined with another's.
__device__ __forceinline__ void join_sums(float& m, float& s, float2 p) {
  const float b = fmaxf(m, p.x), bb = b == -INFINITY ? 0.f : b;
  s = s * exp_of(m, bb) + p.y * exp_of(p.x, bb);
  m = b;
}

// What a gradient call finds out about its rows, on the device.
struct XentState {
  uint32_t count;  // rows with a label
  int uexp;        // largest exponent of |gloss_i| 2^ex_i over them (no gloss: of 2^ex_i), + BIAS
  int ewmax;       // largest ew_v, + BIAS
  int one;         // f32: one G serves both products
};
constexpr int XENT_SPAN = 8;
// Rows without a label have zeros in G, which silence any finite value of x in dw.
// f32 rows are laid out for the call anyway, and are made zeros there. Of 16-bit rows
// that the tiles can read as they lie the kernel of the logits looks at a logit: where
// a row holds a value that is not finite, none of its logits is. Only when one without
// a label is so, which the call's number in `flag` then says, dx's kernel (or one of its
// own) makes the copy `rows` of x with zeros in their place, and dw reads that.
struct OddRows {
  uint32_t* flag;  // null: nothing to do
  uint32_t call;
  char* rows;
  uint32_t dp;           // elements of a row there
  const char* x;
  size_t ld, d;
};
constexpr int XENT_LEAST = -120;  // least exponent of a row (its power of two is finite)
constexpr int XENT_BIAS = 4096;  // (so that zero is less than any)

struct LogitArgs {
  TileIn t;
  uint32_t n, m;    // rows of the block, classes of the piece
  uint32_t col0, k; // its first class, all classes
  const uint32_t* labels;
  float scale;
  const int* ex;    // f32: exponents of the rows, and of the piece's classes
  const int* ew;
  float2* part;     // statistics: [part][row] (max, sum) of z
  float* zlabel;
  const float* lse; // gradients
  const float* gloss;
  const XentState* st;
  uint32_t* counts; // or null: [row tile][wave of it] rows with a label (RowScale)
  uint32_t* small;
  OddRows odd;      // flag and call
  char* g[4];       // G; f32: the planes of G' or Ga, and of Gb
  size_t ldg;       // bytes (rows and columns to full tiles)
};
void launch_logits(hipStream_t s, const LogitArgs& a, int kind, Tile tile, bool grads);

struct ProdArgs {
  TileIn t;
  uint32_t rows, cols;  // of the result
  bool dw;              // else dx
  const uint32_t* labels;  // dx: rows without one are zero
  uint32_t k;
  const float* gloss;
  const XentState* st;
  const uint32_t* counts;  // or null: as in LogitArgs
  uint32_t ncounts;
  OddRows odd;          // dx: the copy to make
  const int* ex;        // f32: as in LogitArgs (dx: of the rows, dw: of the classes)
  const char* gb[2];    // f32, dw: Gb's planes (t.r: those of G')
  float scale;
  void* out;            // the result in its kind, or
  size_t ldo;           // (elements)
  float* part;          // one split's sums: [split][part_rows][ldp] in f32
  size_t ldp, part_rows;
  bool add;             // into what an earlier piece or block left
  const uint32_t* flag; // dw: where it is `call`, x is read from alt
  uint32_t call;
  Operand alt;
};
void launch_prod(hipStream_t s, const ProdArgs& a, int kind, Tile tile);
void launch_copy_rows(emh_ctx* c, const OddRows& o, uint32_t n, const uint32_t* labels, uint32_t k);

// The powers of two of G (see above), and the factor left for the results, from the
// call's state. A mean over rows of 16 bits has all weights 1 in G and needs nothing of
// its rows but how many have a label: the kernel of the logits counts them on the way,
// in MANY_COUNTS words at most, which the products' workgroups add. (k_survey would be
// a launch, 5 us of 139 at 16,384 x 768 by 1,024.)
constexpr uint32_t MANY_COUNTS = 512;
struct RowScale {
  // f16: G's exponent; f32: gb.
  static __device__ __forceinline__ int exponent(const XentState* st, const uint32_t* counts) {
    if (counts) return 13;
    return st->uexp ? 14 - (st->uexp - XENT_BIAS + 1) : 0;  // |weight_i| 2^ex_i < 2^(uexp + 1)
  }
  // scale, and without gloss 1 / rows with a label. By whole waves.
  static __device__ __forceinline__ float factor(const XentState* st, const uint32_t* counts,
                                                 uint32_t ncounts, const float* gloss,
                                                 float scale) {
    if (gloss) return scale;
    uint32_t c = 0;
    if (counts) {
      const uint32_t i = (threadIdx.x & 63) * 4;  // (the buffer holds MANY_COUNTS)
      static_assert(MANY_COUNTS == 512, "two loads a lane");
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const uint4 v = *reinterpret_cast<const uint4*>(counts + h * 256 + i);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; e++) c += h * 256 + i + e < ncounts ? w[e] : 0u;
      }
      for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, 64);
    } else {
      c = st->count;
    }
    return c ? scale / (float)c : 0.f;
  }
};
// The exponent that brings a row's weight below 2^14.
__device__ __forceinline__ int row_exp(const float* gloss, uint32_t i) {
  const float f = gloss ? fabsf(gloss[i]) : 1.f;
  return f > 0.f && f < INFINITY ? 13 - ilogbf(f) : 0;
}

}  // namespace emh
