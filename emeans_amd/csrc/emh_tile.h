// Tiles of products of two 16-bit matrices in f32, the core of the cross
// entropy's four products (emh_xent.h): out(i, j) = sum over k of R(i, k) C(j, k).
//
// A workgroup owns a tile of TR rows x TC columns of the result. The depth goes by in
// slabs of 64, each operand's slab (TR or TC by 64, 128 bytes a row) moved to LDS by
// DMA into one of two stages, or of four for a small tile that has its CU to itself,
// whose slab is done in less than the memory takes to answer (0.6 us a slab with four
// stages, 0.75 with two). An operand lies in memory in one of two ways:
//   DEEP  its rows run along the depth (x and w for the logits): a slab is 128
//         bytes of each row, and a wave's operand is one 16-byte read a lane;
//   WIDE  its rows run across it (w and x for the gradients: the depth is the
//         class or the row): a slab is 64 rows of 2 T bytes, and the operand is two
//         reads that transpose 4 x 16 elements on the way (ds_read_b64_tr_b16), so
//         no operand is ever transposed in memory.
// In LDS the 16-byte chunks of a row are XOR-swizzled so that neither kind of
// read meets a bank twice: a DEEP row r's chunks by (r / 2) % 8 (two rows fill the
// 64 banks: sixteen rows' equal chunks are sixteen different ones), a WIDE row's
// by 4 (r % 4) (a transposing read takes 64 bytes of each of four rows; rows of
// 384 bytes lie half the banks apart already: by 4 (r / 2 % 2)).
//
// Bound by the MFMAs and the clock that they leave: a slab of 256 x 256 x 64 takes 1.56
// us on every CU, 1.38 PFLOP/s, from a tile's first to its last, at whatever clock; the
// same MFMAs without a load take 1.30 (1.65 PFLOP/s, all there are at 1.57 GHz; over
// whole large products they are busy 60 % of the time at 1.8 GHz). The memory answers in
// 0.7 us. Measured no faster: operands read a step further ahead, rings of five half as
// deep slabs (64-byte rows cost more than 128 KB in flight give), four waves of 128 x
// 128, two workgroups of 128 x 192 a CU, other orders of tiles, priorities for MFMAs.
// A launch of one round of workgroups also waits for a tile's ends, 7 to 9 us of first
// instructions, loads and results.
//
// The columns are the MFMA's A and the rows its B, so that a lane holds one
// row of each 32 x 32 block and four consecutive columns at a time.
#pragma once

#include <algorithm>

#include "emh_dma.h"
#include "emh_learn.h"
#include "emh_types.h"

namespace emh {
namespace {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef const v8s __attribute__((address_space(3)))* lds_v8s;
typedef v4s __attribute__((address_space(3)))* lds_v4s;

__device__ __forceinline__ v16f mfma16(f16, v8s a, v8s b, v16f c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a),
                                                __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}
__device__ __forceinline__ v16f mfma16(bf16, v8s a, v8s b, v16f c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a),
                                                 __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}

}  // namespace

constexpr int SLAB = 64;  // depth of a slab
// What plane 1 of an f32 operand counts of plane 0's unit (emh_xent.h).
constexpr float LOW_UNIT = 1.f / 2048;

// A workgroup's shape: waves of NWR x NWC, each WB x WA blocks of 32 x 32.
// STAGES slabs are in the ring.
template <int NWR_, int NWC_, int WB_, int WA_, int STAGES_>
struct TileShape {
  static constexpr int NWR = NWR_, NWC = NWC_, WB = WB_, WA = WA_;
  static constexpr int NW = NWR * NWC, THREADS = 64 * NW;
  static constexpr int TR = NWR * WB * 32, TC = NWC * WA * 32;
  static constexpr int RBYTES = TR * SLAB * 2, CBYTES = TC * SLAB * 2;
  static constexpr int STAGES = STAGES_, STAGE = RBYTES + CBYTES, RING = STAGES * STAGE;
  static constexpr int RD = RBYTES / (1024 * NW), CD = CBYTES / (1024 * NW);  // DMAs a wave
};
typedef TileShape<4, 2, 2, 4, 2> TileL;  // 256 x 256, 8 waves
typedef TileShape<4, 2, 2, 3, 2> TileM;  // 256 x 192, 8 waves
typedef TileShape<2, 2, 2, 2, 2> TileS;  // 128 x 128, 4 waves (two workgroups a CU)
typedef TileShape<4, 2, 1, 2, 4> TileD;  // 128 x 128, 8 waves, three slabs on their way
enum Tile : int { TILE_L, TILE_M, TILE_S, TILE_D, TILES };
constexpr uint32_t TILE_ROWS[TILES] = {TileL::TR, TileM::TR, TileS::TR, TileD::TR};
constexpr uint32_t TILE_COLS[TILES] = {TileL::TC, TileM::TC, TileS::TC, TileD::TC};
// Waves down the rows.
constexpr uint32_t TILE_WAVES[TILES] = {TileL::NWR, TileM::NWR, TileS::NWR, TileD::NWR};
// Rows and columns of whole tiles of any shape.
constexpr uint32_t ALL_ROWS = 256, ALL_COLS = 768;
constexpr uint32_t PARTS = 2;  // waves across a tile's columns
template <class S>
constexpr bool whole_tiles = ALL_ROWS % S::TR == 0 && ALL_COLS % S::TC == 0 && S::NWC == PARTS;
static_assert(whole_tiles<TileL> && whole_tiles<TileM> && whole_tiles<TileS> && whole_tiles<TileD>,
              "whole tiles, and parts of their rows");
// Whether f32's planes are taken together: where two stages of both are in the ring.
template <class S>
constexpr bool takes_both = S::STAGES >= 4;
constexpr bool TILE_BOTH[TILES] = {takes_both<TileL>, takes_both<TileM>, takes_both<TileS>,
                                   takes_both<TileD>};
// Runs f with the shape as a type.
template <class F>
void by_tile(Tile t, F&& f) {
  if (t == TILE_L)
    f(TileL{});
  else if (t == TILE_M)
    f(TileM{});
  else if (t == TILE_S)
    f(TileS{});
  else
    f(TileD{});
}

// One operand. f32 matrices come as two planes of fp16 (emh_xent.h).
struct Operand {
  const char* p[2];  // planes
  uint32_t ld;       // bytes of a row in memory (16-byte multiples, rows 16-byte aligned)
  uint32_t rows;     // rows there are: what lies past them (DEEP: of the tile, WIDE: of the
                     // last slab) reads the last
  uint32_t wide;     // WIDE: elements of a row that may be read (a multiple of 8)
};

struct TileIn {
  Operand r, c;
  uint32_t slabs;   // of the depth; one operand is zero past it
  uint32_t passes;  // 1, or 3: planes (0, 1), (1, 0), (0, 0) one after another
  uint32_t rtiles, ctiles, splits;  // workgroups: rtiles ctiles splits (at most slabs passes:
                                    // each has a step, whose loads go out unasked)
  // What a workgroup finds its tile by (prepare): divisions there, by whole words,
  // were 300 instructions that every workgroup of a launch met cold.
  uint32_t blocks, steps;  // all workgroups; steps of a split (the first `more`: one more)
  uint32_t more;
  uint32_t by_split, by_group, by_tail;
};
constexpr uint32_t GROUP = 8;  // row tiles taken together (tile_at)
// floor(v / by) as umulhi(v, m), which is that or one more (v below 2^31, by > 1).
inline uint32_t recip(uint32_t by) { return (uint32_t)((uint64_t(1) << 32) / by + 1); }
inline unsigned prepare(TileIn& t) {
  const uint32_t steps = t.slabs * t.passes;
  if (t.splits == 0 || t.splits > steps) throw Failure("a product's split without a step");
  t.blocks = t.rtiles * t.ctiles * t.splits;
  t.steps = steps / t.splits;
  t.more = steps % t.splits;
  t.by_split = recip(t.rtiles * t.ctiles);
  t.by_group = recip(GROUP * t.ctiles);
  t.by_tail = recip(std::max(1u, t.rtiles % GROUP));
  return t.blocks;
}

namespace {

__device__ __forceinline__ uint32_t quotient(uint32_t v, uint32_t by, uint32_t m) {
  if (by == 1) return v;
  const uint32_t q = __umulhi(v, m);
  return q * by > v ? q - 1 : q;
}

// Which tile, and which steps (pass, slab) of it, a workgroup takes.
struct TileAt {
  uint32_t rt, ct, split, s0, s1;
};
// Workgroups are dealt to the 8 XCDs in turn: every XCD takes a run of
// consecutive items, in which the tiles of GROUP row tiles and a column tile follow each
// other, so that what its 32 CUs read at a time is a few row and column
// slabs, shared in its L2.
__device__ __forceinline__ TileAt tile_at(const TileIn& t, uint32_t bid) {
  const uint32_t nb = t.blocks;
  const uint32_t xcd = bid & 7, q = bid >> 3, m = nb >> 3, rem = nb & 7;
  uint32_t wi = xcd * m + min(xcd, rem) + q;
  TileAt a;
  const uint32_t tiles = t.rtiles * t.ctiles;
  a.split = quotient(wi, tiles, t.by_split);
  wi -= a.split * tiles;
  const uint32_t per = GROUP * t.ctiles, g = quotient(wi, per, t.by_group);
  const uint32_t have = min(GROUP, t.rtiles - g * GROUP);
  wi -= g * per;
  a.ct = have == GROUP ? wi / GROUP : quotient(wi, have, t.by_tail);
  a.rt = g * GROUP + wi - a.ct * have;
  a.s0 = a.split * t.steps + min(a.split, t.more);
  a.s1 = a.s0 + t.steps + (a.split < t.more ? 1 : 0);
  return a;
}

__device__ __forceinline__ TileAt tile_at(const TileIn& t) { return tile_at(t, blockIdx.x); }

__device__ __forceinline__ uint32_t deep_swz(uint32_t row) { return (row >> 1) & 7; }

// A wave's DMAs of one operand's slab, and its reads of it.
template <bool DEEP, int T, int ND, int NW>
struct Side16 {
  static constexpr uint32_t RB = 2 * T;         // WIDE: bytes of a row in LDS
  static constexpr uint32_t LPR = RB / 16;      // ... its chunks
  static __device__ __forceinline__ uint32_t wide_swz(uint32_t krow) {
    return RB % 256 == 0 ? (krow & 3) << 2 : ((krow >> 1) & 1) << 2;
  }
  uint32_t off[ND];                             // DEEP: row and chunk; WIDE: chunk
  uint32_t krow[ND];                            // WIDE: row in the slab
  uint32_t at[DEEP ? 1 : 4];                    // LDS reads (WIDE: by block)

  // t0: the tile's first row (DEEP) or column (WIDE). w: the wave, uniform.
  __device__ __forceinline__ void init(const Operand& o, uint32_t t0, int w) {
    const uint32_t lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < ND; j++) {
      const uint32_t d = (uint32_t)(j * NW + w);
      if constexpr (DEEP) {
        const uint32_t row = d * 8 + (lane >> 3);
        const uint32_t r = min(t0 + row, o.rows - 1) - t0;
        off[j] = r * o.ld + (((lane & 7) ^ deep_swz(row)) << 4);
      } else {
        krow[j] = (d * 64 + lane) / LPR;
        const uint32_t chunk = ((d * 64 + lane) % LPR) ^ wide_swz(krow[j]);
        const uint32_t col = t0 + chunk * 8;
        off[j] = (col < o.wide ? col : 0u) * 2;
      }
    }
  }
  // The wave's blocks begin at block b0 of the operand's tile.
  __device__ __forceinline__ void init_reads(uint32_t lds, int b0) {
    const uint32_t lane = threadIdx.x & 63;
    if constexpr (DEEP) {
      const uint32_t li = lane & 31, h = lane >> 5;
      at[0] = lds + (uint32_t)b0 * 32 * 128 + li * 128 + ((h ^ deep_swz(li)) << 4);
    } else {
      const uint32_t g = lane >> 4, l = lane & 15;
#pragma unroll
      for (int a = 0; a < 4; a++) {
        const uint32_t chunk = (uint32_t)(b0 + a) * 4 + (g & 1) * 2 + ((l & 3) >> 1);
        at[a] = lds + (8 * (g >> 1) + (l >> 2)) * RB + ((chunk ^ wide_swz(l >> 2)) << 4) + (l & 1) * 8;
      }
    }
  }
  // DMA j of the slab that begins at `slab` (uniform) of the plane at p.
  __device__ __forceinline__ void dma(int j, const char* p, const Operand& o, uint32_t slab,
                                      uint32_t lds) const {
    if constexpr (DEEP) {
      dma16a(p + (size_t)slab * (SLAB * 2), off[j], lds);
    } else {
      const uint32_t last = o.rows - 1 - slab * SLAB;
      dma16a(p + (size_t)slab * SLAB * o.ld, min(krow[j], last) * o.ld + off[j], lds);
    }
  }
  // Block a's operand of MFMA step ks from the stage at `stage` (bytes).
  __device__ __forceinline__ v8s read(uint32_t stage, int ks, int a) const {
    if constexpr (DEEP) {
      return *(lds_v8s)(uintptr_t)(((at[0] + stage) ^ (uint32_t)(ks << 5)) + (uint32_t)a * 32 * 128);
    } else {
      const uint32_t p = at[a] + stage + (uint32_t)ks * 16 * RB;
      const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(uintptr_t)p);
      const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(uintptr_t)(p + 4 * RB));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

// The tile's sums into acc[column block][row block] of every wave.
//
// A step: the slab's four MFMA steps. Each column block's operand is replaced by the
// next step's as soon as its MFMAs are issued. The last MFMA step's operands
// are in registers before it begins, so its stage is free then: every wave has
// waited for its own reads and DMAs (the next slab's) and met the others at the
// barrier, and the DMAs of the slab that takes the stage next (the one after the next,
// with two) go out between its MFMAs.
//
// PLANES (f32): plane 1 counts LOW_UNIT, so the products with one are made first and
// scaled once, when the (0, 0) follow or the split ends.
// BOTH (f32's planes, where one pass over the depth can have them all in LDS): a stage
// holds both planes of both operands, and a step takes the three products from it: two
// thirds of the DMAs and of the LDS reads; the products with a plane 1 have sums of their
// own. (10,007 x 300 by 1,000: dx 37 us with three
// passes, 31 with both; dw 36 and 30.)
template <class T, class S, bool RDEEP, bool CDEEP, bool PLANES>
__device__ __forceinline__ void tile_sums(const TileIn& t, const TileAt& at, char* ring,
                                          v16f (&acc)[S::WA][S::WB]) {
  const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wr = w % S::NWR, wc = w / S::NWR;
  Side16<RDEEP, S::TR, S::RD, S::NW> R;
  Side16<CDEEP, S::TC, S::CD, S::NW> C;
  R.init(t.r, at.rt * S::TR, w);
  C.init(t.c, at.ct * S::TC, w);
  const uint32_t lds0 = lds_addr(ring);
  R.init_reads(lds0, wr * S::WB);
  C.init_reads(lds0 + S::RBYTES, wc * S::WA);
  const size_t r0 = RDEEP ? (size_t)at.rt * S::TR * t.r.ld : 0;
  const size_t c0 = CDEEP ? (size_t)at.ct * S::TC * t.c.ld : 0;
  const uint32_t ldst = lds0 + (uint32_t)w * 1024;
  constexpr bool BOTH = PLANES && takes_both<S>;
  constexpr int P = BOTH ? 2 : 1, STAGES = S::STAGES / P, STAGE = S::STAGE * P;
  static_assert(STAGES >= 2, "a stage to fill and one to read");

  // Load cursor: pass, slab and stage of the next DMAs; past the last step it
  // stays there, and what it fetches again nothing reads.
  uint32_t lpass = 0, lslab = at.s0, lleft = at.s1 - at.s0, lst = 0;
  auto after = [](uint32_t stage) __attribute__((always_inline)) {
    if constexpr (STAGES == 2) return STAGE - stage;
    return stage + STAGE == STAGES * STAGE ? 0u : stage + STAGE;
  };
  while (lslab >= t.slabs) lslab -= t.slabs, lpass++;
  auto dma = [&](int i) __attribute__((always_inline)) {
    const int q = i % (S::RD + S::CD), plane = i / (S::RD + S::CD);
    const uint32_t to = ldst + lst + (uint32_t)plane * S::STAGE;
    if (q < S::RD)
      R.dma(q, t.r.p[BOTH ? plane : PLANES && lpass == 1 ? 1 : 0] + r0, t.r, lslab,
            to + (uint32_t)q * S::NW * 1024);
    else
      C.dma(q - S::RD, t.c.p[BOTH ? plane : PLANES && lpass == 0 ? 1 : 0] + c0, t.c, lslab,
            to + S::RBYTES + (uint32_t)(q - S::RD) * S::NW * 1024);
  };
  auto advance = [&]() __attribute__((always_inline)) {
    lst = after(lst);
    if (lleft > 1) {
      lleft--;
      if (++lslab == t.slabs) {
        lslab = 0;
        lpass++;
      }
    }
  };
#pragma unroll
  for (int a = 0; a < S::WA; a++)
#pragma unroll
    for (int y = 0; y < S::WB; y++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[a][y][r] = 0.f;

  constexpr int PER = (S::RD + S::CD) * P;
#pragma unroll
  for (int s = 0; s < STAGES; s++) {
#pragma unroll
    for (int q = 0; q < PER; q++) dma(q);
    advance();
  }
  wait_vm<(STAGES - 1) * PER>();  // the first slab is in, the others in flight
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  // The next slab is in, and what this one's stage held is in registers.
  auto meet = [&]() __attribute__((always_inline)) {
    wait_vm<(STAGES - 2) * PER>();
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  uint32_t st = 0;
  if constexpr (BOTH) {
    constexpr int ROWS = 2 * S::WB, READS = ROWS + 2 * S::WA, MS = 3 * S::WA;
    v8s op[2][READS];  // [row block][plane], then [column block][plane]
    v16f low[S::WA][S::WB];
#pragma unroll
    for (int a = 0; a < S::WA; a++)
#pragma unroll
      for (int y = 0; y < S::WB; y++)
#pragma unroll
        for (int r = 0; r < 16; r++) low[a][y][r] = 0.f;
    auto read = [&](int i, uint32_t stage, int ks) __attribute__((always_inline)) {
      const uint32_t at_plane = stage + (uint32_t)(i & 1) * S::STAGE;
      return i < ROWS ? R.read(at_plane, ks, i / 2) : C.read(at_plane, ks, (i - ROWS) / 2);
    };
#pragma unroll
    for (int i = 0; i < READS; i++) op[0][i] = read(i, 0, 0);
    for (uint32_t s = at.s0; s < at.s1; s++) {
#pragma unroll
      for (int ks = 0; ks < 4; ks++) {
        if (ks == 3) meet();
        const uint32_t from = ks == 3 ? after(st) : st;
#pragma unroll
        for (int m = 0; m < MS; m++) {  // (h, h) of every block, (h, l), (l, h)
          const int a = m % S::WA, pass = m / S::WA;
#pragma unroll
          for (int y = 0; y < S::WB; y++) {
            v16f& to = pass == 0 ? acc[a][y] : low[a][y];
            to = mfma16(T{}, op[ks & 1][ROWS + 2 * a + (pass == 1)],
                        op[ks & 1][2 * y + (pass == 2)], to);
          }
          __builtin_amdgcn_sched_barrier(0);
          // The next step's operands by the middle of this one.
          constexpr int BY = (MS + 1) / 2;
          if (m < BY) {
#pragma unroll
            for (int i = m * READS / BY; i < (m + 1) * READS / BY; i++)
              op[(ks + 1) & 1][i] = read(i, from, (ks + 1) & 3);
          }
          if (ks == 3) {
#pragma unroll
            for (int q = m * PER / MS; q < (m + 1) * PER / MS; q++) dma(q);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      advance();
      st = after(st);
    }
#pragma unroll
    for (int a = 0; a < S::WA; a++)
#pragma unroll
      for (int y = 0; y < S::WB; y++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[a][y][r] = fmaf(low[a][y][r], LOW_UNIT, acc[a][y][r]);
  } else {
    v8s rb[2][S::WB], ca[S::WA];
#pragma unroll
    for (int y = 0; y < S::WB; y++) rb[0][y] = R.read(0, 0, y);
#pragma unroll
    for (int a = 0; a < S::WA; a++) ca[a] = C.read(0, 0, a);
    auto units = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int a = 0; a < S::WA; a++)
#pragma unroll
        for (int y = 0; y < S::WB; y++)
#pragma unroll
          for (int r = 0; r < 16; r++) acc[a][y][r] *= LOW_UNIT;
    };
    for (uint32_t s = at.s0; s < at.s1; s++) {
      if (PLANES && s == 2 * t.slabs) units();  // (at a split's first step the sums are zero)
#pragma unroll
      for (int ks = 0; ks < 4; ks++) {
        if (ks == 3) meet();
        const uint32_t from = ks == 3 ? after(st) : st;
#pragma unroll
        for (int a = 0; a < S::WA; a++) {
#pragma unroll
          for (int y = 0; y < S::WB; y++)
            acc[a][y] = mfma16(T{}, ca[a], rb[ks & 1][y], acc[a][y]);
          __builtin_amdgcn_sched_barrier(0);
          if (a == 0) {
#pragma unroll
            for (int y = 0; y < S::WB; y++) rb[(ks + 1) & 1][y] = R.read(from, (ks + 1) & 3, y);
          }
          ca[a] = C.read(from, (ks + 1) & 3, a);
          if (ks == 3) {
#pragma unroll
            for (int q = a * PER / S::WA; q < (a + 1) * PER / S::WA; q++) dma(q);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      advance();
      st = after(st);
    }
    if (PLANES && at.s1 <= 2 * t.slabs) units();
  }
  wait_vm<0>();  // the DMAs past the last step have landed
  asm volatile("" ::: "memory");
}

// A lane's pair of fours of a block's columns, 8 q + 4 h .. + 3 of q = 2 p and
// 2 p + 1, as eight consecutive ones: 16 p + 8 h .. + 7 (the lanes l and l + 32
// swap halves).
__device__ __forceinline__ void eight(const float* lo, const float* hi, float* out) {
#pragma unroll
  for (int e = 0; e < 4; e++) {
    // Lanes below 32 keep lo and take the partner's lo; the others keep hi and
    // take the partner's hi.
    const auto v = __builtin_amdgcn_permlane32_swap(__float_as_uint(lo[e]), __float_as_uint(hi[e]),
                                                    false, false);
    out[e] = __uint_as_float(v[0]);
    out[4 + e] = __uint_as_float(v[1]);
  }
}
// The same in a 16-bit type.
template <class T>
__device__ __forceinline__ Vec<T> eight_of(const float* lo, const float* hi) {
  uint32_t out[4];
#pragma unroll
  for (int e = 0; e < 2; e++) {
    const auto v = __builtin_amdgcn_permlane32_swap(pair_from_f32<T>(lo[2 * e], lo[2 * e + 1]),
                                                    pair_from_f32<T>(hi[2 * e], hi[2 * e + 1]),
                                                    false, false);
    out[e] = v[0];
    out[2 + e] = v[1];
  }
  return Vec<T>{make_uint4(out[0], out[1], out[2], out[3])};
}

}  // namespace
}  // namespace emh
