// Rows in 8 bits times classes in 8 bits: y(i, v) = sum over blocks b of 128 columns of
// xs(i, b) ws(v / 128, b) (sum over the block's columns of x(i, c) w(v, c)).
//
// A block's sum comes from the MFMAs and is scaled and added in f32, one fused multiply-add an
// element of the result and block.
//
// Two kinds of MFMA. The 8-bit ones (16 x 16 x 128, twice the 16-bit rate) align the products of
// eight neighbouring columns to the largest and cut 13 bits below it: a sum is off by up to 7
// 2^-13 of the largest product of each eight. 16-bit results take them, few rows' and tiles' alike:
// 1.4e-5 of results from normal data, and 1e-4 below results from positive codes of log-normal sizes (sigma
// 2), where bf16 rounds by up to 3.9e-3 and f16 by up to 4.9e-4 (worst of those codes in f16: 6.8e-4).
// f32 results take the f16 MFMA (an f16 holds every code exactly): 5e-8. For 16-bit results of few
// rows that costs 5.6 us instead of 5.1 (1 x 1,024 x 16,384), and 29.3 instead of 22.2 (131,071 classes).
//
// Bound by the matrix cores where all three sizes are large (8,192^3: 458 us, 2.4 PFLOP/s; f32 935 us,
// 1.2), by the results' bytes where the depth is short (8,192 x 1,024 x 131,072 bf16 1.14 ms, 2.1
// GB; k = 131,071, whose rows straddle lines and stay in the caches on their way, 1.61 ms), and
// by the classes' bytes and latency where rows are few (1 x 1,024 x 16,384: 5.1 us, from memory 5.8; 64
// rows: 9.3, f32 12.5).
//
// Few rows read the classes as they lie. More of them go in tiles: a workgroup owns 256 x
// 256 or 128 x 128 of the result, and a block of the depth, 128 bytes a row of both operands,
// goes by in one step, moved to LDS by DMA into one of two stages, its 16-byte chunks
// XOR-swizzled so that sixteen rows' equal chunks meet no bank twice. 256 x 256 takes 2 us a
// block of the depth and CU where 128 x 128, two a CU, take 1.3 for half as much; but fewer of
// them leave more of the last round idle: launch_product8 weighs that.
#include <cmath>

#include "emh_answer.h"
#include "emh_codes.h"
#include "emh_tile.h"

namespace emh {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef v4u __attribute__((address_space(3)))* lds_v4u;

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
  __device__ __forceinline__ Halves(v4u a, v4u b)
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

// The first `left` of 16 codes, then zeros.
__device__ __forceinline__ v4u first_codes(v4u v, int left) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int have = left - 4 * i;
    v[i] = have >= 4 ? v[i] : have <= 0 ? 0u : v[i] & ((1u << (8 * have)) - 1u);
  }
  return v;
}
// The 16 codes at p, of which `left` are the row's, the others zeros.
__device__ __forceinline__ v4u codes16(const uint8_t* p, int left) {
  if (left <= 0) return v4u{0u, 0u, 0u, 0u};
  const v4u v = *reinterpret_cast<const v4u*>(p);
  return left >= 16 ? v : first_codes(v, left);
}
// The same by one 8-bit MFMA.
__device__ __forceinline__ v8i codes_of(v4u a, v4u b) {
  return __builtin_bit_cast(v8i, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}
__device__ __forceinline__ v4f block8(v8i a, v8i b) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, v4f{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0,
                                                          0, 0);
}

// Few rows: a workgroup takes 16 classes and 16 YB rows, its four waves the blocks of the depth
// by turns; operands come from memory as they lie, AHEAD blocks of a wave's on their way at once.
// Bound by the classes' bytes: 1 x 1,024 x 16,384 5.1 us with its launch, 16.8 MB at 3.3 TB/s.
template <int YB, bool EXACT>
__global__ __launch_bounds__(256) void k_few8(const CodedIn x, size_t n, uint32_t d, const CodedIn w,
                                              size_t k, void* y, size_t ldy, int kind,
                                              uint32_t rgroups, size_t groups) {
  constexpr int AHEAD = YB == 1 ? 4 : 2;
  __shared__ v4f sums[4][YB][64];
  const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t blocks = (d + CODE_BLOCK - 1) / CODE_BLOCK, whole = d / CODE_BLOCK;
  for (size_t u = blockIdx.x; u < groups; u += gridDim.x) {
    size_t cg = u, r0 = 0;
    if (rgroups > 1) cg = u / rgroups, r0 = (u - cg * rgroups) * (16 * YB);
    const size_t v0 = cg * 16;
    const uint8_t* wp = w.q + min(v0 + li, k - 1) * w.ld + 16 * g;
    const uint8_t* xp[YB];
    const float* sp[YB];
#pragma unroll
    for (int b = 0; b < YB; b++) {
      const size_t row = min(r0 + b * 16 + li, n - 1);
      xp[b] = x.q + row * x.ld + 16 * g;
      sp[b] = x.scale + row * x.lds;
    }
    const float* ws = w.scale + v0 / CODE_BLOCK * w.lds;
    v4f acc[YB];
#pragma unroll
    for (int b = 0; b < YB; b++) acc[b] = v4f{0.f, 0.f, 0.f, 0.f};
    struct Block {
      v4u w[2], x[YB][2];
      float by, f[YB];
    };
    auto add = [&](const Block& o) __attribute__((always_inline)) {
      Halves wh;
      if constexpr (EXACT) wh = Halves(o.w[0], o.w[1]);
#pragma unroll
      for (int b = 0; b < YB; b++) {
        v4f t;
        if constexpr (EXACT)
          t = block16(wh, Halves(o.x[b][0], o.x[b][1]));
        else
          t = block8(codes_of(o.w[0], o.w[1]), codes_of(o.x[b][0], o.x[b][1]));
        const float f = o.f[b] * o.by;
#pragma unroll
        for (int e = 0; e < 4; e++) acc[b][e] = fmaf(t[e], f, acc[b][e]);
      }
    };
    for (uint32_t s0 = wave; s0 < whole; s0 += 4 * AHEAD) {
      Block o[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; i++) {
        const uint32_t s = s0 + 4 * i;
        if (s >= whole) continue;
        const size_t c = (size_t)s * CODE_BLOCK;
#pragma unroll
        for (int h = 0; h < 2; h++) o[i].w[h] = *reinterpret_cast<const v4u*>(wp + c + 64 * h);
        o[i].by = ws[s];
#pragma unroll
        for (int b = 0; b < YB; b++) {
#pragma unroll
          for (int h = 0; h < 2; h++)
            o[i].x[b][h] = *reinterpret_cast<const v4u*>(xp[b] + c + 64 * h);
          o[i].f[b] = sp[b][s];
        }
      }
#pragma unroll
      for (int i = 0; i < AHEAD; i++)
        if (s0 + 4 * i < whole) add(o[i]);
    }
    if (whole < blocks && (int)(whole & 3) == wave) {  // the short last block
      Block o;
      const size_t c = (size_t)whole * CODE_BLOCK;
      const int left = (int)(d - whole * CODE_BLOCK) - 16 * g;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        o.w[h] = codes16(wp + c + 64 * h, left - 64 * h);
#pragma unroll
        for (int b = 0; b < YB; b++) o.x[b][h] = codes16(xp[b] + c + 64 * h, left - 64 * h);
      }
      o.by = ws[whole];
#pragma unroll
      for (int b = 0; b < YB; b++) o.f[b] = sp[b][whole];
      add(o);
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
    if (gridDim.x < groups) __syncthreads();  // the next group's sums take their place
  }
}

// ------------------------------------------------------------------ tiles
// Waves of NWR x NWC, each 16 YB rows by 16 AB classes. A stage holds a block of the depth of
// both operands, the rows' scales of it (TR) and the classes' (64, by turns the tile's two).
template <int NWR_, int NWC_, int YB_, int AB_, int PER_CU_>
struct Shape8 {
  static constexpr int NWR = NWR_, NWC = NWC_, YB = YB_, AB = AB_, PER_CU = PER_CU_;
  static constexpr int NW = NWR * NWC, THREADS = 64 * NW;
  static constexpr int TR = NWR * YB * 16, TC = NWC * AB * 16;
  static constexpr int RBYTES = TR * CODE_BLOCK, CBYTES = TC * CODE_BLOCK;
  static constexpr int CODES = RBYTES + CBYTES, STAGE = CODES + TR * 4 + 256;
  static constexpr int RD = RBYTES / (1024 * NW), CD = CBYTES / (1024 * NW);  // DMAs a wave
  static constexpr int XW = TR / 64;  // waves that move the rows' scales; the next the classes'
  static_assert(NW % 2 == 0 && XW < NW && CODE_BLOCK % (AB * 16) == 0,
                "a wave's classes share a scale");
};
typedef Shape8<4, 2, 4, 8, 1> Large8;  // 256 x 256, 8 waves
typedef Shape8<2, 2, 4, 4, 2> Small8;  // 128 x 128, 4 waves, two workgroups a CU

struct Prod8Args {
  TileIn t;  // r: the rows, c: the classes; slabs: blocks of the depth
  uint32_t n, k, d;
  const float* xs;
  uint32_t ldxs;  // bytes
  const float* ws;
  size_t ldws;
  void* y;
  size_t ldy;
  bool odd;  // 16 bits: rows of y may begin at odd multiples of two bytes
};

struct Frag {  // a lane's 32 codes of a block's row
  v4u a, b;
  __device__ __forceinline__ void read(uint32_t at) {
    a = *(lds_v4u)(uintptr_t)at;
    b = *(lds_v4u)(uintptr_t)(at ^ 64u);
  }
  __device__ __forceinline__ v8i codes() const { return codes_of(a, b); }
};
typedef const float __attribute__((address_space(3)))* lds_f32;
// Between a wave's writes to LDS and other lanes' reads, which the LDS takes in order.
__device__ __forceinline__ void wave_fence8() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Sixteen bytes of a lane's results in the blocks from acc[0] on: f32 as they are; of 16 bits two
// blocks' fours swapped between lanes, so that each has eight columns of one.
template <class T, int YB>
__device__ __forceinline__ void sixteen(const v4f (*acc)[YB], int y, uint32_t* out) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; e++) out[e] = __float_as_uint(acc[0][y][e]);
  } else {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const auto v = __builtin_amdgcn_permlane16_swap(
          pair_from_f32<T>(acc[0][y][2 * h], acc[0][y][2 * h + 1]),
          pair_from_f32<T>(acc[1][y][2 * h], acc[1][y][2 * h + 1]), false, false);
      out[h] = v[0];
      out[2 + h] = v[1];
    }
  }
}
// Where results go: into the caches, through them or past them.
enum Way { CACHED, THROUGH, PAST };
// Sixteen bytes of a row to p; `left` elements from p on are the row's.
template <class T, Way WAY>
__device__ __forceinline__ void store_row(T* p, const v4u& v, uint32_t left) {
  const Vec<T> out{make_uint4(v[0], v[1], v[2], v[3])};
  constexpr uint32_t EL = 16 / sizeof(T);
  if (left >= EL)
    WAY == PAST ? stream_vec(p, out) : put_vec(WAY == THROUGH, p, out);
  else if (left > 0)
    store_some(p, out, (int)left);
}
// The same of a 16-bit row that may begin at an odd multiple of two bytes: then an element
// later, by whole words; after: the row's next word. The first element of what a wave has of the
// row, and the last of its last (last) sixteen bytes, are left to the caller.
template <class T, Way WAY>
__device__ __forceinline__ void store_odd_row(T* p, const v4u& v, uint32_t after, bool last,
                                              uint32_t left) {
  const uint32_t odd = (uint32_t)((uintptr_t)p >> 1) & 1, by = 16 * odd;
  v4u s;
#pragma unroll
  for (int e = 0; e < 4; e++)
    s[e] = __builtin_amdgcn_alignbit(e < 3 ? v[e < 3 ? e + 1 : 3] : after, v[e], by);
  // (`left > odd ? left - odd : 0` lets the compiler take left for at least `odd` elsewhere.)
  const uint32_t n = max(left, odd) - odd;
  if (last && odd && n >= 7) {  // six of them; the seventh goes with the first
    typedef uint32_t three __attribute__((ext_vector_type(3), aligned(4)));
    *reinterpret_cast<three*>(p + 1) = three{s[0], s[1], s[2]};
  } else {
    store_row<T, WAY>(p + odd, s, min(n, last ? 8 - odd : 8u));
  }
}

// EXACT: f32 results by f16 MFMAs; else T results by 8-bit ones.
//
// A workgroup takes tiles in turn, and the blocks of all its tiles are one stream: while a
// tile's last blocks are multiplied, the next one's first are on their way, and while its
// results go out of the registers, too. (A workgroup for every tile: 8,192^3 538 us, so 455;
// 16,384 x 768 x 1,024 bf16 21.6 us, so 18.5, and 16.7 with results through the caches.)
template <class T, class S, bool EXACT, Way WAY>
__global__ __launch_bounds__(S::THREADS, 2) void k_tile8(const Prod8Args a) {
  __shared__ __attribute__((aligned(1024))) char ring[2 * S::STAGE];
  __shared__ __attribute__((aligned(16))) char out[S::NW * 16 * 144];
  const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wr = w % S::NWR, wc = w / S::NWR;
  const uint32_t lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
  const uint32_t steps = a.t.slabs;
  const uint32_t lds0 = lds_addr(ring);
  // The last block may be short: chunks past the row's sixteens read the last one, and
  // what lies past d is made zeros in LDS. (A lane moves the same chunk of a row in all its DMAs:
  // a wave's rows are 8 apart times an even number.)
  const uint32_t tail = a.d - (steps - 1) * CODE_BLOCK, lastc = (tail + 15) / 16 - 1;
  const uint32_t chunk = (lane & 7) ^ (((uint32_t)w * 4 + (lane >> 4)) & 7);
  const uint32_t back = chunk > lastc ? (chunk - lastc) << 4 : 0u;

  // The next DMAs: their tile and block. Past the last tile they fetch its last block again.
  uint32_t lbid = blockIdx.x, lslab = 0, lst = lds0;
  const char *rp, *cp, *xp, *wp;
  uint32_t roff, rlast, coff, clast, soff;
  auto aim = [&]() __attribute__((always_inline)) {
    const TileAt at = tile_at(a.t, lbid);
    const uint32_t row = (uint32_t)w * 8 + (lane >> 3), ch = chunk << 4;
    rp = a.t.r.p[0] + (size_t)at.rt * S::TR * a.t.r.ld;
    cp = a.t.c.p[0] + (size_t)at.ct * S::TC * a.t.c.ld;
    const uint32_t r1 = a.t.r.rows - 1 - at.rt * S::TR, c1 = a.t.c.rows - 1 - at.ct * S::TC;
    roff = row * a.t.r.ld + ch;
    rlast = min(r1, (uint32_t)S::TR - 1) * a.t.r.ld + ch;
    coff = row * a.t.c.ld + ch;
    clast = min(c1, (uint32_t)S::TC - 1) * a.t.c.ld + ch;
    // Scales: waves below XW move the rows', the one after them the classes'.
    xp = reinterpret_cast<const char*>(a.xs) + (size_t)at.rt * S::TR * a.ldxs;
    const uint32_t v0 = at.ct * S::TC / CODE_BLOCK;
    wp = reinterpret_cast<const char*>(a.ws + v0 * a.ldws);
    soff = w < S::XW ? min((uint32_t)w * 64 + lane, r1) * a.ldxs
                     : (uint32_t)(min(v0 + (lane & 1), (a.k - 1) / CODE_BLOCK) - v0) *
                           (uint32_t)a.ldws * 4u;
  };
  constexpr int PER = S::RD + S::CD + 1;
  auto dma = [&](int q) __attribute__((always_inline)) {
    const uint32_t by = lslab + 1 == steps ? back : 0u;
    const size_t from = (size_t)lslab * CODE_BLOCK;
    if (q < S::RD) {
      const uint32_t o = min(roff + (uint32_t)q * S::NW * 8 * a.t.r.ld, rlast);
      dma16a(rp + from, o - by, lst + (uint32_t)(q * S::NW + w) * 1024);
    } else if (q < S::RD + S::CD) {
      const int j = q - S::RD;
      const uint32_t o = min(coff + (uint32_t)j * S::NW * 8 * a.t.c.ld, clast);
      dma16a(cp + from, o - by, lst + S::RBYTES + (uint32_t)(j * S::NW + w) * 1024);
    } else if (w <= S::XW) {
      dma4a((w < S::XW ? xp : wp) + (size_t)lslab * 4, soff, lst + S::CODES + (uint32_t)w * 256);
    }
  };
  auto advance = [&]() __attribute__((always_inline)) {
    lst = 2 * lds0 + S::STAGE - lst;
    if (++lslab == steps) {
      if (lbid + gridDim.x < a.t.blocks) {
        lbid += gridDim.x;
        lslab = 0;
        aim();
      } else {
        lslab = steps - 1;
      }
    }
  };
  auto barrier = [&]() __attribute__((always_inline)) {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // Zeros past d in the last block's stage, which has landed.
  auto cut = [&](uint32_t stage) __attribute__((always_inline)) {
    for (uint32_t r = threadIdx.x; r < (uint32_t)(S::TR + S::TC); r += S::THREADS) {
      const uint32_t row = stage + r * CODE_BLOCK;
      for (uint32_t c = tail / 16; c < 8; c++) {
        lds_v4u p = (lds_v4u)(uintptr_t)(row + ((c ^ deep_swz(r)) << 4));
        v4u v{0u, 0u, 0u, 0u};
        if (c * 16 < tail) v = first_codes(*p, (int)(tail - c * 16));
        *p = v;
      }
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    barrier();
  };

  aim();
#pragma unroll
  for (int s = 0; s < 2; s++) {
#pragma unroll
    for (int q = 0; q < PER; q++) dma(q);
    advance();
  }
  wait_vm<PER - 1>();  // the first block is in (a wave without a DMA of scales has PER - 1 a block)
  barrier();
  if (steps == 1 && tail < CODE_BLOCK) cut(lds0);

  const uint32_t swz = (g ^ deep_swz(li)) << 4;
  const uint32_t rat = (uint32_t)(wr * S::YB * 16 + li) * CODE_BLOCK + swz;
  const uint32_t cat = S::RBYTES + (uint32_t)(wc * S::AB * 16 + li) * CODE_BLOCK + swz;
  const uint32_t xat = S::CODES + (uint32_t)(wr * S::YB * 16 + li) * 4;
  const uint32_t wat = S::CODES + S::TR * 4 + (uint32_t)(wc * S::AB * 16 / CODE_BLOCK) * 4;
  constexpr uint32_t BLOCK16 = 16 * CODE_BLOCK;
  constexpr int ALL = S::AB * S::YB, SLOTS = 4, AHEAD = SLOTS - 1;
  static_assert(S::YB == 4 && S::AB % SLOTS == 0, "t and ca by turns");

  uint32_t st = lds0;
  Frag rb[S::YB], ca[SLOTS];
  float f[S::YB], fx[S::YB], fw;
  auto read_scales = [&](uint32_t stage) __attribute__((always_inline)) {
    fw = *(lds_f32)(uintptr_t)(stage + wat);
#pragma unroll
    for (int y = 0; y < S::YB; y++) fx[y] = *(lds_f32)(uintptr_t)(stage + xat + y * 64);
  };
  read_scales(st);
#pragma unroll
  for (int y = 0; y < S::YB; y++) rb[y].read(st + rat + y * BLOCK16);
#pragma unroll
  for (int i = 0; i < AHEAD; i++) ca[i].read(st + cat + i * BLOCK16);
#pragma unroll
  for (int y = 0; y < S::YB; y++) f[y] = fx[y] * fw;

  Halves rh[EXACT ? S::YB : 1], ch[EXACT ? 2 : 1];  // as f16: the rows', this and the next classes'
  if constexpr (EXACT) ch[0] = Halves(ca[0].a, ca[0].b);

  // Sixteen bytes of results a lane.
  constexpr int EL = 16 / sizeof(T), STRIDE = EL / 4, STORES = S::YB * S::AB / STRIDE;
  bool stored = false;  // the last tile's results went out in STORES stores of every wave
  for (uint32_t bid = blockIdx.x; bid < a.t.blocks; bid += gridDim.x) {
    v4f acc[S::AB][S::YB];
#pragma unroll
    for (int i = 0; i < S::AB; i++)
#pragma unroll
      for (int y = 0; y < S::YB; y++) acc[i][y] = v4f{0.f, 0.f, 0.f, 0.f};
    float fp[2] = {0.f, 0.f};  // the last block's scales of its last two sums
    v4f t[4];
#pragma unroll
    for (int i = 0; i < 4; i++) t[i] = v4f{0.f, 0.f, 0.f, 0.f};
    for (uint32_t s = 0; s < steps; s++) {
      if constexpr (EXACT) rh[0] = Halves(rb[0].a, rb[0].b);
      const uint32_t other = 2 * lds0 + S::STAGE - st;
#pragma unroll
      for (int i = 0; i < S::AB; i++) {
        // The class blocks are read AHEAD of their MFMAs: before these the last of the stage's
        // are in registers.
        constexpr int MEET = S::AB - AHEAD;
        if (i == MEET) {
          // The next block is in. (What a wave queues is done in order: stores of the last
          // tile's results went out after it.)
          if (s == 0 && stored)
            wait_vm<STORES>();
          else
            wait_vm<0>();
          __builtin_amdgcn_s_waitcnt(0xc07f);
          barrier();
          // (Of this tile, or of the next one, whose only block it then is.)
          if (tail < CODE_BLOCK && (s + 2 == steps || steps == 1)) cut(other);
          read_scales(other);
        }
        if (i + AHEAD < S::AB)
          ca[(i + AHEAD) % SLOTS].read(st + cat + (i + AHEAD) * BLOCK16);
        else
          ca[(i + AHEAD) % SLOTS].read(other + cat + (i + AHEAD - S::AB) * BLOCK16);
#pragma unroll
        for (int y = 0; y < S::YB; y++) {
          const int m = i * S::YB + y, o = (m + ALL - 2) % ALL;  // the MFMA, and whose sums are due
          if constexpr (EXACT) {
            t[m & 3] = block16(ch[i & 1], rh[y]);
            // Between these MFMAs: the next classes' codes as f16 and, once a block, the rows'.
            const Frag& next = ca[(i + 1) % SLOTS];
            const v4u from = y < 2 ? next.a : next.b;
            ch[(i + 1) & 1].v[y] = y & 1 ? halves8(from.z, from.w) : halves8(from.x, from.y);
            if (i == 0 && y + 1 < S::YB) rh[y + 1] = Halves(rb[y + 1].a, rb[y + 1].b);
          } else {
            t[m & 3] = block8(ca[i % SLOTS].codes(), rb[y].codes());
          }
          const float by = m < 2 ? fp[m] : f[o % S::YB];
#pragma unroll
          for (int e = 0; e < 4; e++)
            acc[o / S::YB][o % S::YB][e] = fmaf(t[o & 3][e], by, acc[o / S::YB][o % S::YB][e]);
          // (Here, not at the step's end, with all the blocks' sums kept until then.)
          asm volatile("" : "+v"(acc[o / S::YB][o % S::YB]));
          if (i == S::AB - 1) rb[y].read(other + rat + y * BLOCK16);
          if constexpr (EXACT) {
#pragma unroll
            for (int q = 0; q < 4; q++) {
              __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);  // an MFMA
              if (i == 0 && y + 1 < S::YB)
                __builtin_amdgcn_sched_group_barrier(0x2, 6, 0);  // VALU
              else
                __builtin_amdgcn_sched_group_barrier(0x2, 2, 0);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
          if (i >= MEET) {
            constexpr int LEFT = (S::AB - MEET) * S::YB;
            const int from = m - MEET * S::YB;
#pragma unroll
            for (int q = from * PER / LEFT; q < (from + 1) * PER / LEFT; q++) dma(q);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
      fp[0] = f[S::YB - 2];
      fp[1] = f[S::YB - 1];
#pragma unroll
      for (int y = 0; y < S::YB; y++) f[y] = fx[y] * fw;
      advance();
      st = other;
    }
#pragma unroll
    for (int m = 0; m < 2; m++) {
      const int o = ALL - 2 + m;
#pragma unroll
      for (int e = 0; e < 4; e++)
        acc[o / S::YB][o % S::YB][e] = fmaf(t[o & 3][e], fp[m], acc[o / S::YB][o % S::YB][e]);
    }

    // Through LDS, where a wave has room for 128 bytes of sixteen rows (and a word more): eight
    // lanes side by side store a row's 128 bytes. (What a wave reads there it wrote before.)
    const TileAt at = tile_at(a.t, bid);
    stored = (at.rt + 1) * S::TR <= a.n && (at.ct + 1) * S::TC <= a.k;
    constexpr int PIECES = S::AB / (2 * STRIDE);
    constexpr uint32_t PITCH = 144;
    char* const mine = out + w * 16 * PITCH;
    const uint32_t chunk_at = (sizeof(T) == 4 ? g : 2 * (g & 1) + (g >> 1)) * 16;
    const uint32_t place = lane & 7;
    const uint32_t col0 = at.ct * S::TC + (uint32_t)(wc * S::AB) * 16 + place * EL;
#pragma unroll
    for (int y = 0; y < S::YB; y++) {
      uint32_t q[PIECES + 1][2][4] = {}, single[2];
      bool some[2];
#pragma unroll
      for (int i = 0; i < PIECES; i++)
#pragma unroll
        for (int h = 0; h < 2; h++) sixteen<T>(&acc[(2 * i + h) * STRIDE], y, q[i][h]);
#pragma unroll
      for (int i = 0; i < PIECES; i++) {
#pragma unroll
        for (int h = 0; h < 2; h++)
          *reinterpret_cast<v4u*>(mine + li * PITCH + h * 64 + chunk_at) =
              v4u{q[i][h][0], q[i][h][1], q[i][h][2], q[i][h][3]};
        if (sizeof(T) == 2 && g == 0)
          *reinterpret_cast<uint32_t*>(mine + li * PITCH + 128) = q[i + 1][0][0];
        wave_fence8();
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const uint32_t in = (lane >> 3) + 8 * h;
          const uint32_t row = at.rt * S::TR + (uint32_t)(wr * S::YB + y) * 16 + in;
          const char* const from = mine + in * PITCH + place * 16;
          const v4u v = *reinterpret_cast<const v4u*>(from);
          const uint32_t col = col0 + i * 8 * EL;
          T* const p = reinterpret_cast<T*>(a.y) + (size_t)row * a.ldy + col;
          const uint32_t left = row < a.n && col < a.k ? a.k - col : 0u;
          if (sizeof(T) == 2 && a.odd) {
            if constexpr (sizeof(T) == 2) {
              const bool last = i + 1 == PIECES && place == 7;
              store_odd_row<T, WAY>(p, v, *reinterpret_cast<const uint32_t*>(from + 16), last,
                                       left);
              // The first element of the wave's, from its first piece, and the last.
              if (i == 0) single[h] = v[0], some[h] = left > 0;
              if (last) single[h] = v[3] >> 16, some[h] = left >= 8;
              if (i + 1 == PIECES && ((uintptr_t)p & 2) && (place == 0 || place == 7) && some[h])
                *(p + (last ? 7 : -i * 8 * (int)EL)) = __builtin_bit_cast(T, (uint16_t)single[h]);
            }
          } else {
            store_row<T, WAY>(p, v, stored ? EL : left);
          }
        }
        wave_fence8();
      }
    }
  }
  wait_vm<0>();  // the DMAs past the last step have landed
}

template <class T, class S, bool EXACT>
void launch_tiles(emh_ctx* c, const CodedIn& x, size_t n, size_t d, const CodedIn& w, size_t k,
                  const MatOut& y) {
  Prod8Args a{};
  a.k = (uint32_t)k, a.d = (uint32_t)d;
  a.odd = sizeof(T) == 2 && (y.ld % 2 != 0 || (uintptr_t)y.p % 4 != 0);
  a.ws = w.scale, a.ldws = w.lds, a.ldxs = (uint32_t)(x.lds * 4), a.ldy = y.ld;
  a.t.c = {{(const char*)w.q, nullptr}, (uint32_t)w.ld, (uint32_t)k, 0};
  a.t.slabs = (uint32_t)((d + CODE_BLOCK - 1) / CODE_BLOCK);
  a.t.passes = 1, a.t.splits = 1;
  // Rows that do not begin at whole 64 bytes: their pieces are put together in the caches. Others
  // go through them (16,384 x 768 x 1,024 bf16 17.0 us, written back at the end 18.5), and past
  // them where they are larger.
  const bool whole = y.ld * sizeof(T) % 64 == 0 && (uintptr_t)y.p % 64 == 0;
  a.t.ctiles = (uint32_t)((k + S::TC - 1) / S::TC);
  a.t.rtiles = (uint32_t)((n + S::TR - 1) / S::TR);
  EMH_ENSURE((size_t)a.t.ctiles * a.t.rtiles <= (size_t(1) << 30) / GROUP,
             "y is larger than any device's memory");
  a.n = (uint32_t)n;
  a.xs = x.scale;
  a.y = y.p;
  a.t.r = {{(const char*)x.q, nullptr}, (uint32_t)x.ld, (uint32_t)n, 0};
  const unsigned blocks = prepare(a.t);
  const unsigned grid = std::min(blocks, (unsigned)(c->cus * S::PER_CU));
  auto go = [&](auto kernel) { kernel<<<grid, S::THREADS, 0, c->stream>>>(a); };
  if (!whole)
    go(k_tile8<T, S, EXACT, CACHED>);
  else if (n * k * sizeof(T) < STREAM_FROM)
    go(k_tile8<T, S, EXACT, THROUGH>);
  else
    go(k_tile8<T, S, EXACT, PAST>);
}

}  // namespace

void launch_product8(emh_ctx* c, const CodedIn& x, size_t n, size_t d, const CodedIn& w, size_t k,
                     const MatOut& y) {
  if (n == 0) return;
  auto few = [&](auto yb) {
    constexpr int YB = decltype(yb)::value;
    const size_t rg = (n + 16 * YB - 1) / (16 * YB), groups = (k + 15) / 16 * rg;
    auto go = [&](auto exact) {
      k_few8<YB, decltype(exact)::value>
          <<<dim3((unsigned)std::min(groups, MAX_GROUPS)), 256, 0, c->stream>>>(
              x, n, (uint32_t)d, w, k, y.p, y.ld, y.kind, (uint32_t)rg, groups);
    };
    y.kind == EMH_F32 ? go(std::true_type{}) : go(std::false_type{});
  };
  // What each way takes, in us, from the times of 1 to 2,000 rows (tiles: 16,384) by 1,000 to 131,071
  // classes of 128 to 4,096: few rows read the classes again for every 64 rows and the rows for
  // every 16 classes, or take what their workgroups take; a tile's block of the depth takes a CU
  // as long as here, of small tiles less where a CU has but one.
  const double cus = c->cus, steps = (double)((d + CODE_BLOCK - 1) / CODE_BLOCK);
  const bool f32 = y.kind == EMH_F32;
  auto up = [](size_t v, size_t by) { return (double)((v + by - 1) / by); };
  auto tiles_take = [&](double tiles, double slots, double start, double step, double alone) {
    const double full = std::floor(tiles / slots), rest = tiles - full * slots;
    return start + steps * (full * step + (rest == 0 ? 0 : rest <= cus ? alone : step));
  };
  const double reads = n <= 64 ? (double)n / 16 + 1 : 5 * up(n, 64);
  const double few_take = 2.5 + std::max(reads * (double)k * (double)d / 5.8e6,
                                         up(k, 16) * up(n, 64) * 1.3e-3);
  const double small_take = std::max(
      tiles_take(up(n, 128) * up(k, 128), 2 * cus, f32 ? 4.5 : 4.2, f32 ? 2.05 : 1.3,
                 f32 ? 1.05 : 0.64),
      (double)k * (double)d / 4.2e6);
  const double large_take = f32 ? INFINITY : tiles_take(up(n, 256) * up(k, 256), cus, 4, 2, 2);
  // (A tile's offsets are 32 bits.)
  const bool far = std::max({x.ld, w.ld, x.lds * 4, w.lds * 4}) >= (size_t(1) << 23);
  if (far || few_take <= std::min(small_take, large_take)) {
    if (n <= 16)
      few(std::integral_constant<int, 1>{});
    else if (n <= 32)
      few(std::integral_constant<int, 2>{});
    else
      few(std::integral_constant<int, 4>{});
  } else if (f32) {
    launch_tiles<float, Small8, true>(c, x, n, d, w, k, y);
  } else {
    auto go = [&](auto t) {
      using T = decltype(t);
      large_take < small_take ? launch_tiles<T, Large8, false>(c, x, n, d, w, k, y)
                              : launch_tiles<T, Small8, false>(c, x, n, d, w, k, y);
    };
    y.kind == EMH_F16 ? go(f16{}) : go(bf16{});
  }
  EMH_HIP(hipGetLastError());
}

}  // namespace emh
