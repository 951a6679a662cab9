// Log probabilities of given classes, entropies and the likeliest classes from rows of
// logits, and the gradient of the logits.
//
// With z = scale logits: lse = log sum exp z_v, log p_v = z_v - lse, H = -sum p_v log p_v. One
// pass: a lane keeps the largest logit m of what it has seen (before the scale), S = sum exp(d)
// and E = sum exp(d) d with d = scale (x - m), both moved to a new largest by exp(scale (m - m'));
// lanes, waves and parts of a row are joined the same way, and lse = scale m + log S, H = log S - E
// / S, log p_t = scale (x_t - m) - log S. (The difference comes before the scale: then d of the
// largest is 0 however large it is. Off by a rounding of scale m, it was 1e31 in a row masked by
// f32's lowest value.) Exponents and E are in base 2.
//
// The likeliest classes: a wave keeps a sorted list in its lanes (lane i the i-th), the
// larger logit first, the lower class among equals: an entry is one key of 64 bits, the logit's
// own value (unscaled and unrounded) in an order of whole numbers above the class's complement.
// Of a chunk only lanes whose largest element would enter the list matter; of the top largest
// of those the least is a bound that no better element is below. What reaches it, a few more
// than top, goes to LDS beside the list, where every entry counts the ones before it: that is
// its place. (Many equal values overflow the LDS: then each lane offers its largest, and its
// next where that was taken.)
//
// Gradient: dz_v = scale (gl ([v = t] - p_v) - gh p_v (log p_v + H)), element by element, p_v =
// min(1, exp(z_v - lse)). lse and z_v are f32: all p of a row are off by a factor within exp(2^-23
// |lse|), 2e-6 for logits of 20 and 0.7 % for 60,000; where f32 holds no logarithm beside
// them p is 1 at each of the largest.
//
// A row is read in vectors at multiples of 16 bytes, whatever its address (a vector at
// either end may hold elements of no row of it: they count as -infinity); each vector holds an
// element of the row.
//
// Bound by HBM (one read; one read and one write): 4,096 x 131,071 bf16 190 us, 5.7 TB/s, with
// the 8 likeliest 215 us; the gradient 409 us, 5.3 TB/s. Next by the instructions, 11 issue slots an
// element forward, and with a list by its steps, a chain of some 400 instructions and ten visits
// to LDS a row and chunk, which short rows feel: 10,007 x 1,000 f32 8.8 us, with the 5
// likeliest 13.3. A few rows are latency: of 131,071 4.5 us, with
// the 8 likeliest 9.1.
#include <cfloat>

#include "emh_answer.h"
#include "emh_types.h"

namespace emh {
namespace {

constexpr float LOG2E = 1.44269504f, LN2 = 0.693147181f;
constexpr float FAR = -1e4f;  // below any logarithm of a positive f32
constexpr uint32_t NONE = 0xFFFFFFFFu;

template <class T>
__device__ __forceinline__ uint32_t minus_inf() {  // a word of them
  if constexpr (sizeof(T) == 4) return 0xFF800000u;
  return __is_same(T, f16) ? 0xFC00FC00u : 0xFF80FF80u;
}

// The vectors of a row that begins at p: `head` elements of the first lie before it.
template <class T>
struct Row {
  static constexpr int N = VecOf<T>::N;
  const T* base;  // a multiple of 16 bytes
  uint32_t head;
  size_t k;
  __device__ __forceinline__ Row(const void* z, size_t at, size_t k_) : k(k_) {
    const T* p = reinterpret_cast<const T*>(z) + at;
    head = (uint32_t)((uintptr_t)p & 15) / sizeof(T);
    base = p - head;
  }
  __device__ __forceinline__ size_t vectors() const { return (k + head + N - 1) / N; }
  __device__ __forceinline__ Vec<T> load(size_t v) const {
    return Vec<T>{*reinterpret_cast<const uint4*>(base + v * N)};
  }
  // The first element of vector v, as a column (of the first vector possibly below 0).
  __device__ __forceinline__ int64_t column(size_t v) const { return (int64_t)(v * N) - head; }
  // -infinity in place of what is not the row's.
  __device__ __forceinline__ void mask(Vec<T>& x, size_t v) const {
    const int64_t c = column(v);
    const int lo = c < 0 ? (int)-c : 0;
    const int64_t left = (int64_t)k - c;
    const int hi = left < N ? (left < 0 ? 0 : (int)left) : N;
    uint32_t w[4] = {x.raw.x, x.raw.y, x.raw.z, x.raw.w};
    const uint32_t none = minus_inf<T>();
    constexpr int PER = 4 / (int)sizeof(T);  // elements of a word
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (PER == 1) {
        if (i < lo || i >= hi) w[i] = none;
      } else {
        const bool a = 2 * i < lo || 2 * i >= hi, b = 2 * i + 1 < lo || 2 * i + 1 >= hi;
        w[i] = (a ? none & 0xFFFFu : w[i] & 0xFFFFu) | (b ? none & 0xFFFF0000u : w[i] & 0xFFFF0000u);
      }
    }
    x.raw = make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// exp(scale (x - m)) = 2^power(x, half_of(m), base2(scale)). (Halves: the difference of two finite
// logits does not overflow. Where the scale's product does it stays finite: 0 times it is 0.)
__device__ __forceinline__ float base2(float scale) { return fminf(scale * (2.f * LOG2E), FLT_MAX); }
__device__ __forceinline__ float half_of(float m) { return m == -INFINITY ? 0.f : 0.5f * m; }
__device__ __forceinline__ float power(float x, float half, float by) {
  return fmaf(x, 0.5f, -half) * by;
}

// What a lane, a wave or a part of a row has seen: the largest, S and E (see above).
struct Seen {
  float m = -INFINITY, s = 0.f, e = 0.f;
  __device__ __forceinline__ Seen() {}
  __device__ __forceinline__ explicit Seen(float4 v) : m(v.x), s(v.y), e(v.z) {}
  __device__ __forceinline__ float4 packed() const { return make_float4(m, s, e, 0.f); }
  // To the largest `to`, at least m.
  __device__ __forceinline__ void move(float to, float by) {
    const float d = fmaxf(power(m, half_of(to), by), FAR);  // (nothing seen: s is zero)
    const float f = __builtin_amdgcn_exp2f(d);
    e = f * fmaf(s, d, e);
    s *= f;
    m = to;
  }
  __device__ __forceinline__ void join(const Seen& o, float by) {
    Seen t = o;
    const float to = fmaxf(m, o.m);
    move(to, by);
    t.move(to, by);
    s += t.s;
    e += t.e;
  }
  __device__ __forceinline__ void join_lanes(float by) {
    move(lanes_max<64>(m), by);
    s = lanes_sum<64>(s);
    e = lanes_sum<64>(e);
  }
};

__device__ __forceinline__ float lane_value(float v, uint32_t lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), (int)lane));
}

__device__ __forceinline__ uint64_t key_of(float v, uint32_t id) {
  const uint32_t u = __float_as_uint(v + 0.f);  // (-0 is equal to 0)
  return (uint64_t)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (uint32_t)~id;
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t u = (uint32_t)(k >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}
__device__ __forceinline__ uint32_t key_class(uint64_t k) { return ~(uint32_t)k; }
__device__ __forceinline__ uint64_t lane_key(uint64_t k, uint32_t lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(k >> 32), (int)lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)k, (int)lane);
}
// What other lanes of the wave have written to LDS is there.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

constexpr uint32_t ROOM = 64;  // entries that a wave ranks at a time
constexpr uint32_t ROOM_END = 4;  // zeros after them

// The `top` best, sorted, in a wave's lanes; no entry: 0.
struct Best {
  uint64_t key = 0;
  // The least value that an entry must exceed.
  __device__ __forceinline__ float bound(uint32_t top) const {
    const uint64_t k = lane_key(key, top - 1);
    return k ? key_value(k) : -INFINITY;
  }
  // The list's entries behind `count` others in `room` (ROOM in all), and the best of all of
  // them the list. (Every lane reads every entry, two at a time: no lane waits for another's.)
  __device__ __forceinline__ void merge(uint32_t top, uint64_t* room, uint32_t count) {
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t old = (uint32_t)__popcll(__ballot(key != 0));
    if (lane < old + 4) room[count + lane] = lane < old ? key : 0;
    count += old;
    wave_fence();
    const uint64_t mine = lane < count ? room[lane] : 0;
    uint32_t place = 0;
    for (uint32_t j = 0; j < count; j += 4) {
      const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(room + j);
      const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(room + j + 2);
      place += (a.x > mine) + (a.y > mine) + (b.x > mine) + (b.y > mine);
    }
    wave_fence();
    if (lane < count && place < top) room[place] = mine;
    wave_fence();
    key = lane < (count < top ? count : top) ? room[lane] : 0;
    wave_fence();
  }
  // Every lane with `has` offers (cv, cid), cv > -infinity; the lanes whose offer was taken.
  __device__ __forceinline__ uint64_t offer(uint32_t top, float cv, uint32_t cid, bool has) {
    const uint32_t lane = threadIdx.x & 63;
    uint64_t taken = 0;
    for (;;) {
      const uint64_t mine = has ? key_of(cv, cid) : 0;
      const uint64_t last = lane_key(key, top - 1);
      uint64_t who = __ballot(mine > last);
      if (!who) return taken;
      uint32_t from = (uint32_t)__ffsll((unsigned long long)who) - 1;
      uint64_t best = lane_key(mine, from);
      for (who &= who - 1; who; who &= who - 1) {
        const uint32_t at = (uint32_t)__ffsll((unsigned long long)who) - 1;
        const uint64_t o = lane_key(mine, at);
        if (o > best) best = o, from = at;
      }
      taken |= uint64_t(1) << from;
      if (lane == from) has = false;
      const uint32_t r = (uint32_t)__popcll(__ballot(key > best));
      const uint32_t lo = __float_as_uint(lane_perm<0x138>(__uint_as_float((uint32_t)key)));
      const uint32_t hi = __float_as_uint(lane_perm<0x138>(__uint_as_float((uint32_t)(key >> 32))));
      const uint64_t below = (uint64_t)hi << 32 | lo;  // the lane below's
      key = lane == r ? best : lane > r ? below : key;
    }
  }
};

// Lanes' values v: a bound that at least `top` of them reach (-infinity where fewer than that
// are above it), found in groups: as many as the next power of two from top; the least of the
// groups' largest.
__device__ __forceinline__ uint32_t group_bits(uint32_t top) {  // log2 of the groups
  return top <= 1 ? 0u : 32u - (uint32_t)__clz((int)(top - 1));
}
__device__ __forceinline__ float group_bound(float v, uint32_t top) {
  const uint32_t p = group_bits(top);
  auto join = [&](uint32_t step, float a, float b) __attribute__((always_inline)) {
    return step + p < 6 ? fmaxf(a, b) : fminf(a, b);
  };
  v = join(0, v, lane_perm<0xB1>(v));
  v = join(1, v, lane_perm<0x4E>(v));
  v = join(2, v, lane_perm<0x141>(v));
  v = join(3, v, lane_perm<0x140>(v));
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = join(4, __uint_as_float(s[0]), __uint_as_float(s[1]));
  const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return join(5, __uint_as_float(h[0]), __uint_as_float(h[1]));
}
// The top-th largest of the lanes' values among those in `who` (more than top). room: LDS for 68.
__device__ __forceinline__ float exact_bound(float v, uint64_t who, uint32_t top, float* room) {
  const uint32_t lane = threadIdx.x & 63, count = (uint32_t)__popcll(who);
  const bool in = who >> lane & 1;
  if (in)
    room[__builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32),
                                   __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0u))] = v;
  if (lane < 4) room[count + lane] = -INFINITY;
  wave_fence();
  uint32_t above = 0;
  for (uint32_t j = 0; j < count; j += 4) {
    const float4 o = *reinterpret_cast<const float4*>(room + j);
    above += (o.x > v) + (o.y > v) + (o.z > v) + (o.w > v);
  }
  wave_fence();
  return lanes_reduce<64>(in && above < top ? v : INFINITY,
                          [](float a, float b) { return fminf(a, b); });
}
// The least f32 above v.
__device__ __forceinline__ float next_above(float v) {
  const uint32_t u = __float_as_uint(v);
  return __uint_as_float(v == 0.f ? 1u : u & 0x80000000u ? u - 1 : u + 1);
}

// A row's given class and its logit: asked for before the row's sums are made.
struct Given {
  uint32_t t = NONE;
  float z = 0.f;
  __device__ __forceinline__ Given(const LogpArgs& a, int kind, size_t row) {
    if (!a.logp) return;
    t = a.tokens[row];
    z = load_kind(a.z, kind, row * a.ldz + (t < a.k ? t : 0));
  }
};
// The outputs of a row, by one wave.
__device__ __forceinline__ void finish(const LogpArgs& a, size_t row, const Given& given,
                                       const Seen& all, const Best& best) {
  const uint32_t lane = threadIdx.x & 63;
  // top + off: the scaled largest, exactly.
  const float m = all.m == -INFINITY ? 0.f : all.m;
  const float top = m * a.scale, off = fmaf(m, a.scale, -top);
  // A NaN, an infinite logit, or one that the scale makes infinite.
  const bool odd = !(all.s < INFINITY) || top == INFINITY;
  const bool none = all.m == -INFINITY || top == -INFINITY;
  const float ls = logf(all.s);
  auto some = [&](float z) __attribute__((always_inline)) {  // it has a probability
    return !odd && !none && z * a.scale > -INFINITY;
  };
  auto logp_of = [&](float z) __attribute__((always_inline)) {
    return odd ? (float)NAN : some(z) ? fmaf(z, a.scale, -top) - off - ls : -INFINITY;
  };
  if (lane == 0) {
    a.lse[row] = odd ? NAN : none ? -INFINITY : top + (off + ls);
    if (a.entropy) a.entropy[row] = odd ? NAN : none ? 0.f : fmaf(-LN2, all.e / all.s, ls);
    if (a.logp) {
      float lp = 0.f;
      if (given.t < a.k)
        lp = logp_of(given.z);
      else if (given.t != NONE)
        a.small[SW_BAD_CLASS] = 1u;
      a.logp[row] = lp;
    }
  }
  if (lane < a.top) {
    // (Of a finite logit it may be -infinity: 6e38 below the largest.)
    const float z = best.key != 0 ? key_value(best.key) : -INFINITY;
    if (a.ids) a.ids[row * a.top + lane] = some(z) ? key_class(best.key) : NONE;
    if (a.tops) a.tops[row * a.top + lane] = logp_of(z);
  }
}

// What the parts of a row leave for each other lies in memory: written and read by single
// accesses that all of the GPU's caches let through, so that none of them is written back or
// emptied for it (64 rows of 131,071 with top 8: 17.6 us, by fences 24.5). A second launch that
// joins the parts took 8.0 us for a row of 131,071 without a list where this takes 4.6.
__device__ __forceinline__ void share(uint64_t* p, uint64_t v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t shared_value(const uint64_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Counters lie a line apart: side by side 64 rows' (1,024 parts) took 10.3 us, and so 7.4.
constexpr uint32_t DONE_STEP = 32;
struct PartOut {  // [row][part]
  uint64_t* seen;  // two: m and s, e
  uint64_t* best;  // [row][part][top]
  uint32_t* done;  // [row]: its parts that are there; zeros between calls
  __device__ __forceinline__ void put_seen(size_t u, const Seen& v) const {
    share(seen + 2 * u, (uint64_t)__float_as_uint(v.s) << 32 | __float_as_uint(v.m));
    share(seen + 2 * u + 1, __float_as_uint(v.e));
  }
  __device__ __forceinline__ Seen get_seen(size_t u) const {
    const uint64_t ms = shared_value(seen + 2 * u), e = shared_value(seen + 2 * u + 1);
    return Seen(make_float4(__uint_as_float((uint32_t)ms), __uint_as_float((uint32_t)(ms >> 32)),
                            __uint_as_float((uint32_t)e), 0.f));
  }
};
// One wave's, of a part of a row: whether it is the last one there.
__device__ __forceinline__ bool last_part(uint32_t* done, uint32_t parts) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // what the wave has shared is there
  uint32_t before = 0;
  if ((threadIdx.x & 63) == 0) {
    before = __hip_atomic_fetch_add(done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (before == parts - 1)
      __hip_atomic_store(done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  const bool last = (uint32_t)__builtin_amdgcn_readfirstlane((int)before) == parts - 1;
  asm volatile("" ::: "memory");
  return last;
}
// The parts of a row, by a wave. room: LDS for ROOM + ROOM_END.
template <bool TOP>
__device__ __forceinline__ void join_parts(const PartOut& in, size_t row, uint32_t parts,
                                           uint32_t top, float by, uint64_t* room, Seen& all,
                                           Best& best) {
  const uint32_t lane = threadIdx.x & 63;
  // (Entries come from lists of 64 - top at a time, so that these and a list of top have room.)
  const uint32_t count = parts * top, each = ROOM - top;
  const uint64_t* const list = in.best + row * count;
  auto entry = [&](uint32_t i0) __attribute__((always_inline)) {
    const uint32_t i = i0 + lane;
    return lane < each && i < count ? shared_value(list + i) : 0;
  };
  constexpr int AHEAD = 4;
  uint64_t o[AHEAD], first = 0;
  if constexpr (TOP) {
#pragma unroll
    for (int j = 0; j < AHEAD; j++) o[j] = entry(j * each);
    // Of a group's lanes (group_bound) the first have the parts' best, others what comes next:
    // each an entry of its own.
    const uint32_t groups = group_bits(top);
    const uint32_t e = (lane & ((64u >> groups) - 1)) << groups | lane >> (6 - groups);
    const uint32_t rank = e / parts, part = e - rank * parts;
    if (rank < top) first = shared_value(list + part * top + rank);
    for (uint32_t p = e + 64; p < parts; p += 64) {
      const uint64_t f = shared_value(list + p * top);
      first = f > first ? f : first;
    }
  }
  all = Seen();
  for (uint32_t p = lane; p < parts; p += 64) all.join(in.get_seen(row * parts + p), by);
  all.join_lanes(by);
  if constexpr (TOP) {
    best.key = 0;
    // (At least top entries reach it.)
    const float bound = group_bound(first ? key_value(first) : -INFINITY, top);
    uint32_t have = 0;
    for (uint32_t i0 = 0; i0 < count;) {
#pragma unroll
      for (int j = 0; j < AHEAD; j++, i0 += each) {
        const uint64_t them = __ballot(o[j] > lane_key(best.key, top - 1) && key_value(o[j]) >= bound);
        if (!them) continue;
        const uint32_t more = (uint32_t)__popcll(them);
        if (have + more > each) {
          best.merge(top, room, have);
          have = 0;
        }
        if (them >> lane & 1)
          room[__builtin_amdgcn_mbcnt_hi((uint32_t)(them >> 32),
                                         __builtin_amdgcn_mbcnt_lo((uint32_t)them, have))] = o[j];
        have += more;
      }
      if (i0 < count) {
#pragma unroll
        for (int j = 0; j < AHEAD; j++) o[j] = entry(i0 + j * each);
      }
    }
    if (have > 0) best.merge(top, room, have);
  }
}

// W waves take a part of a row, by turns in chunks of 64 NV vectors; the last of a row's parts
// joins them all, in their order, and writes the row's results. One wave: rows of one chunk.
// (least_waves: with lists of the likeliest a few registers fewer than the compiler would take,
// for a wave more on a SIMD. 16,384 rows of 2,000 bf16 with top 5: 24.5 us, without 26.3.)
template <class T>
constexpr int least_waves(int W, int NV, bool top, bool parts) {
  return !top || parts ? 1 : sizeof(T) == 4 ? 6 : W == 1 && NV == 4 ? 5 : 1;
}
template <class T, int W, int NV, bool TOP, bool PARTS>
__global__ __launch_bounds__(256, least_waves<T>(W, NV, TOP, PARTS)) void k_logp(
    const LogpArgs a, int kind, uint32_t parts, uint32_t each, PartOut out) {
  constexpr int N = VecOf<T>::N, ROWS = 4 / W;
  __shared__ float4 seen[4];
  __shared__ __attribute__((aligned(16))) uint64_t rooms[TOP ? 4 : 1][ROOM + ROOM_END];
  __shared__ uint64_t lists[TOP && W > 1 ? 4 : 1][MAX_TOP];
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t w = wave % W;
  const float by = base2(a.scale);
  const size_t units = PARTS ? a.n * parts : a.n;
  for (size_t u0 = (size_t)blockIdx.x * ROWS; u0 < units; u0 += (size_t)gridDim.x * ROWS) {
    const size_t u = u0 + wave / W;
    if (W == 1 && u >= units) return;  // (waves of their own)
    // (Rows in parts are few.)
    const size_t row = PARTS ? (uint32_t)u / parts : u;
    const uint32_t part = PARTS ? (uint32_t)(u - row * parts) : 0;
    const Row<T> r(a.z, row * a.ldz, a.k);
    const uint32_t nv = (uint32_t)r.vectors(), chunks = (nv + 64 * NV - 1) / (64 * NV);
    const uint32_t c0 = PARTS ? min(chunks, part * each) : 0;
    const uint32_t c1 = W == 1 ? 1 : PARTS ? min(chunks, c0 + each) : chunks;
    Seen all;
    Best best;
    Vec<T> next[NV];
    auto fetch = [&](uint32_t c) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < NV; j++) {
        const uint32_t v = c * (64 * NV) + j * 64 + lane;
        next[j] = r.load(v < nv ? v : nv - 1);
      }
    };
    if (c0 + w < c1) fetch(c0 + w);
    Given given(a, kind, row);
    for (uint32_t c = c0 + w; c < c1; c += W) {
      Vec<T> x[NV];
#pragma unroll
      for (int j = 0; j < NV; j++) x[j] = next[j];
      if (W > 1 && c + W < c1) fetch(c + W);
      const uint32_t v0 = c * (64 * NV) + lane;
      if (c == 0 || c == chunks - 1) {
#pragma unroll
        for (int j = 0; j < NV; j++) r.mask(x[j], v0 + j * 64);
      }
      float most = -INFINITY;
#pragma unroll
      for (int j = 0; j < NV; j++)
#pragma unroll
        for (int e = 0; e < N; e++) most = fmaxf(most, x[j].get(e));
      if constexpr (W == 1)
        all.m = most;  // (a row's only chunk: nothing to move)
      else
        all.move(fmaxf(all.m, most), by);
      const float half = half_of(all.m);
#pragma unroll
      for (int j = 0; j < NV; j++)
#pragma unroll
        for (int e = 0; e < N; e++) {
          const float d = power(x[j].get(e), half, by);
          const float p = __builtin_amdgcn_exp2f(d);
          all.s += p;
          all.e = fmaf(p, fmaxf(d, FAR), all.e);
        }
      if constexpr (TOP) {
        // The largest of the lane's that comes after (v, id) in the list's order. (From memory
        // again: registers for the few rows that come here would be every row's.)
        auto after = [&](float v, uint32_t id, float& cv, uint32_t& cid) {
          cv = -INFINITY;
          cid = NONE;
#pragma unroll 1
          for (int j = 0; j < NV; j++) {
            const uint32_t at = v0 + j * 64;
            Vec<T> y = r.load(at < nv ? at : nv - 1);
            r.mask(y, at);
            const uint32_t col = (uint32_t)r.column(at);
#pragma unroll
            for (int e = 0; e < N; e++) {
              const float q = y.get(e);
              const bool is = (q < v || (q == v && col + e > id)) && q > cv;
              cv = is ? q : cv;
              cid = is ? col + e : cid;
            }
          }
        };
        const float need = best.bound(a.top);
        uint64_t who = __ballot(most > need);
        if (who) {
          float least = -INFINITY;
          if ((uint32_t)__popcll(who) > a.top) {
            const float bound = group_bound(most, a.top);
            who &= __ballot(most >= bound);
            least = (uint32_t)__popcll(who) > a.top
                        ? exact_bound(most, who, a.top, reinterpret_cast<float*>(rooms[wave]))
                        : bound;
          }
          least = least > need ? least : next_above(need);
          // (A later chunk's equal of the list's last has a higher class.)
          uint64_t* const room = rooms[wave];
          const uint32_t old = (uint32_t)__popcll(__ballot(best.key != 0));
          uint32_t count = 0;
          // A bit for every element of the lane's, the first the highest.
          uint32_t bits = 0;
#pragma unroll
          for (int j = 0; j < NV; j++)
#pragma unroll
            for (int e = 0; e < N; e++) bits = bits + bits + (x[j].get(e) >= least ? 1u : 0u);
          const bool single = (bits & (bits - 1)) == 0;  // then it is the lane's largest
          for (uint64_t them; count <= ROOM && (them = __ballot(bits != 0));) {
            const uint32_t at = __builtin_amdgcn_mbcnt_hi(
                (uint32_t)(them >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)them, count));
            const uint32_t bit = 31u - (uint32_t)__clz((int)bits), slot = NV * N - 1 - bit;
            const uint32_t v = v0 + slot / N * 64, e = slot % N;
            if (bits != 0 && at < ROOM) {
              const float q = single ? most : to_f32(r.base[(size_t)v * N + e]);
              room[at] = key_of(q, (uint32_t)r.column(v) + e);
            }
            bits &= ~(1u << bit);
            count += (uint32_t)__popcll(them);
          }
          if (count + old <= ROOM) {
            best.merge(a.top, room, count);
          } else {
            wave_fence();
            float lv = INFINITY;
            uint32_t lid = 0;
            bool may = true;
            for (;;) {
              float cv;
              uint32_t cid;
              after(lv, lid, cv, cid);
              const uint64_t taken = best.offer(a.top, cv, cid, may && cid != NONE);
              if (!taken) break;
              may = taken >> lane & 1;
              lv = cv;
              lid = cid;
            }
          }
        }
      }
    }
    all.join_lanes(by);
    if constexpr (W > 1) {
      __syncthreads();  // (what the last unit left has been read)
      if (lane == 0) seen[wave] = all.packed();
      if (TOP && lane < a.top) lists[wave][lane] = best.key;
      __syncthreads();
      if (wave == 0) {
        for (int i = 1; i < W; i++) all.join(Seen(seen[i]), by);
        if constexpr (TOP) {
          // All lists at once where there is room (places without an entry count as least).
          const uint32_t lists_at = (ROOM - a.top) / a.top >= W - 1 ? W - 1 : 1;
          for (uint32_t i = 1; i < W; i += lists_at) {
            const uint32_t n = a.top * lists_at;
            if (lane < n) rooms[0][lane] = (&lists[i][0])[lane / a.top * MAX_TOP + lane % a.top];
            best.merge(a.top, rooms[0], n);
          }
        }
      }
    }
    if (W > 1 && wave != 0) continue;
    if constexpr (PARTS) {
      if (lane == 0) out.put_seen(u, all);
      if (TOP && lane < a.top) share(out.best + u * a.top + lane, best.key);
      if (!last_part(out.done + row * DONE_STEP, parts)) continue;
      join_parts<TOP>(out, row, parts, a.top, by, rooms[0], all, best);
    }
    finish(a, row, given, all, best);
  }
}

// A wave takes 64 NV vectors of a row of dz: stores of whole vectors of dz, whatever z's address,
// through the caches or not.
template <class T, int NV, bool THROUGH>
__global__ __launch_bounds__(256) void k_logp_grad(const LogpArgs a, uint32_t chunks,
                                                   uint32_t units) {
  constexpr int N = VecOf<T>::N;
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  for (uint32_t u = blockIdx.x * 4 + wave; u < units; u += gridDim.x * 4) {
    const uint32_t in = chunks == 1 ? u : u / chunks, c = u - in * chunks;
    const size_t row = in;
    const Row<T> o(a.dz, row * a.lddz, a.k);
    const T* z = reinterpret_cast<const T*>(a.z) + row * a.ldz;
    T* dz = const_cast<T*>(o.base) + o.head;
    const size_t nv = o.vectors(), v0 = (size_t)c * (64 * NV) + lane;
    // Vectors that are the row's whole.
    auto whole = [&](size_t v) __attribute__((always_inline)) {
      return (v > 0 || o.head == 0) && (v + 1) * N - o.head <= o.k;
    };
    Vec<T> x[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const size_t v = v0 + j * 64;
      if (v < nv && whole(v)) x[j] = load_vec(z + o.column(v));
    }
    uint32_t t = a.tokens ? a.tokens[row] : NONE;
    if (t >= a.k) {
      if (t != NONE && lane == 0) a.small[SW_BAD_CLASS] = 1u;
      t = NONE;
    }
    float lse = a.lse_in[row], gl = t != NONE && a.glogp ? a.glogp[row] * a.scale : 0.f;
    float gh = a.gentropy ? a.gentropy[row] * a.scale : 0.f;
    const float h = a.gentropy ? a.entropy_in[row] : 0.f;
    if (lse == -INFINITY) lse = gl = gh = 0.f;  // no class may be answered: zeros
    if (lse != lse) gl = NAN;                   // (the bounds of d hold no NaN)
    const float glh = fmaf(gh, h, gl);
    auto one = [&](float q, bool own) __attribute__((always_inline)) {
      // (Rounded as lse's largest was: a class alone has p = 1 at any size of logits. From FAR to 0.)
      const float d = __builtin_amdgcn_fmed3f(q * a.scale - lse, FAR, 0.f);
      const float p = __builtin_amdgcn_exp2f(d * LOG2E);
      const float g = -p * fmaf(gh, d, glh);
      return own ? g + gl : g;
    };
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const size_t v = v0 + j * 64;
      if (v >= nv) continue;
      const int64_t col = o.column(v);
      if (whole(v)) {
        float g[N];
#pragma unroll
        for (int e = 0; e < N; e++) g[e] = one(x[j].get(e), false);
        const int64_t own = (int64_t)t - col;
        if (own >= 0 && own < N && t != NONE) {
#pragma unroll
          for (int e = 0; e < N; e++) g[e] = own == e ? g[e] + gl : g[e];
        }
        put_vec(THROUGH, dz + col, g);
      } else {
        for (int e = 0; e < N; e++) {
          const int64_t i = col + e;
          if (i >= 0 && i < (int64_t)o.k) dz[i] = from_f32<T>(one(to_f32(z[i]), i == (int64_t)t));
        }
      }
    }
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

}  // namespace

void launch_log_probs(emh_ctx* c, LogpArgs a, int kind) {
  if (a.n == 0) return;
  a.small = c->small;
  by_kind(kind, [&](auto t) {
    using T = decltype(t);
    constexpr size_t N = VecOf<T>::N;
    // Of a row at any address one more than its elements fill.
    const bool whole = a.ldz % N == 0 && (uintptr_t)a.z % 16 == 0;
    const size_t vectors = (a.k + N - 1) / N + (whole ? 0 : 1);
    // A wave a row where the row is a chunk; otherwise four, and parts of a row where there are
    // few rows. Chunks of 128 vectors, not 256, where they leave no wave a second one anyway (a
    // row of 16,384 bf16 8.5 us, so 9.2; 16 of them 8.7, so 9.5; 131,071 with top 8 9.0, so 9.3).
    const bool small = vectors <= 256;
    const size_t per = vectors <= 1024 || a.n * vectors <= 512 * (size_t)c->cus ? 128 : 256;
    const size_t chunks = (vectors + per - 1) / per;
    size_t parts = 1;
    if (!small) parts = std::min((chunks + 3) / 4, std::max<size_t>(1, 4 * (size_t)c->cus / a.n));
    PartOut out{};
    if (parts > 1) {
      const size_t seen = (a.n * parts * 2 * sizeof(uint64_t) + 255) & ~size_t(255);
      char* p = (char*)c->logp_part.get(seen + a.n * parts * a.top * sizeof(uint64_t), c->stream);
      out.seen = (uint64_t*)p;
      out.best = (uint64_t*)(p + seen);
      // (Fewer rows than twice the CUs have parts.)
      const bool first = c->logp_done.bytes == 0;
      out.done = (uint32_t*)c->logp_done.get(2 * (size_t)c->cus * DONE_STEP * sizeof(uint32_t),
                                             c->stream);
      if (first) EMH_HIP(hipMemsetAsync(out.done, 0, c->logp_done.bytes, c->stream));
    }
    auto go = [&](auto waves, auto nv, auto top) {
      constexpr int W = decltype(waves)::value, NV = decltype(nv)::value;
      constexpr bool TOP = decltype(top)::value;
      const size_t groups = (a.n * parts + 4 / W - 1) / (4 / W);
      auto run = [&](auto kernel) {
        kernel<<<dim3((unsigned)std::min(groups, MAX_GROUPS)), 256, 0, c->stream>>>(
            a, kind, (uint32_t)parts, (uint32_t)((chunks + parts - 1) / parts), out);
      };
      if constexpr (W > 1) {
        if (parts > 1) return run(k_logp<T, W, NV, TOP, true>);
      }
      run(k_logp<T, W, NV, TOP, false>);
    };
    auto with_top = [&](auto top) {
      if (per == 256 && !small)
        go(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{}, top);
      else if (!small)
        go(std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{}, top);
      else if (vectors <= 64)
        go(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{}, top);
      else if (vectors <= 128)
        go(std::integral_constant<int, 1>{}, std::integral_constant<int, 2>{}, top);
      else
        go(std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{}, top);
    };
    if (a.top > 0)
      with_top(std::true_type{});
    else
      with_top(std::false_type{});
  });
  EMH_HIP(hipGetLastError());
}

void launch_log_probs_grad(emh_ctx* c, LogpArgs a, int kind) {
  if (a.n == 0) return;
  a.small = c->small;
  by_kind(kind, [&](auto t) {
    using T = decltype(t);
    constexpr size_t N = VecOf<T>::N, NV = 4;
    const bool whole = a.lddz % N == 0 && (uintptr_t)a.dz % 16 == 0;
    const size_t vectors = (a.k + N - 1) / N + (whole ? 0 : 1);
    const size_t chunks = (vectors + 64 * NV - 1) / (64 * NV);
    const size_t units = a.n * chunks;  // (2 KB of dz at least, or a row)
    EMH_ENSURE(units < (size_t(1) << 31), "z is larger than any device's memory");
    const dim3 grid((unsigned)std::min((units + 3) / 4, MAX_GROUPS));
    // Up to 128 MB through the caches: 16,384 x 1,024 bf16 13.4 us, written back 16.6, 512 x 131,071
    // 45.2 and 47.4; but 16,384 x 5,001, 164 MB, 66.7 and 62.4.
    if (a.n * a.k * sizeof(T) <= size_t(128) << 20)
      k_logp_grad<T, NV, true><<<grid, 256, 0, c->stream>>>(a, (uint32_t)chunks, (uint32_t)units);
    else
      k_logp_grad<T, NV, false><<<grid, 256, 0, c->stream>>>(a, (uint32_t)chunks, (uint32_t)units);
  });
  EMH_HIP(hipGetLastError());
}

}  // namespace emh
