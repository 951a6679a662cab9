// Log probabilities of given classes, entropies and the likeliest classes from rows of
// logits, and the gradient of the logits.
//
// With z = scale logits: lse = log sum exp z_v, log p_v = z_v - lse, H = -sum p_v log p_v. One
// pass: a lane keeps the maximum m of what it has seen, S = sum exp(z - m) and E = sum exp(z -
// m) (z - m), both moved to a new maximum by exp(m - m'); lanes, waves and parts of a row are
// joined the same way, and lse = m + log S, H = log S - E / S, log p_t = (z_t - m) - log S.
//
// The likeliest classes: a wave keeps a sorted list in its lanes (lane i the i-th), the
// larger logit first, the lower class among equals. A chunk is looked at again only where a
// lane's largest element would enter the list; each lane offers its largest, then, where that
// was taken, its next. The logits' own values are compared, unscaled and unrounded.
//
// Gradient: dz_v = scale (gl ([v = t] - p_v) - gh p_v (log p_v + H)), element by element.
//
// A row is read in vectors at multiples of 16 bytes, whatever its address (a vector at
// either end may hold elements of no row of it: they count as -infinity); each vector holds an
// element of the row.
//
// Bound by HBM (one read; one read and one write), and nearly by the instructions: 11
// issue slots an element forward.
#include "emh_answer.h"
#include "emh_types.h"

namespace emh {
namespace {

constexpr float LOG2E = 1.44269504f;
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

// What a lane, a wave or a part of a row has seen: maximum, S and E (see above).
struct Seen {
  float m = -INFINITY, s = 0.f, e = 0.f;
  __device__ __forceinline__ Seen() {}
  __device__ __forceinline__ explicit Seen(float4 v) : m(v.x), s(v.y), e(v.z) {}
  __device__ __forceinline__ float4 packed() const { return make_float4(m, s, e, 0.f); }
  // To the maximum `to`, at least m.
  __device__ __forceinline__ void move(float to) {
    const float b = to == -INFINITY ? 0.f : to;
    const float d = fmaxf(m - b, -1e30f);  // (nothing seen: s is zero)
    const float f = __builtin_amdgcn_exp2f(d * LOG2E);
    e = f * fmaf(s, d, e);
    s *= f;
    m = to;
  }
  __device__ __forceinline__ void join(const Seen& o) {
    Seen t = o;
    const float to = fmaxf(m, o.m);
    move(to);
    t.move(to);
    s += t.s;
    e += t.e;
  }
  __device__ __forceinline__ void join_lanes() {
    move(lanes_max<64>(m));
    s = lanes_sum<64>(s);
    e = lanes_sum<64>(e);
  }
};

__device__ __forceinline__ float lane_value(float v, uint32_t lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), (int)lane));
}

// The list of the `top` best, sorted, in a wave's lanes.
struct Best {
  float v = -INFINITY;
  uint32_t id = NONE;
  // Every lane with `has` offers (cv, cid), cv > -infinity; the lanes whose offer was taken.
  __device__ __forceinline__ uint64_t offer(uint32_t top, float cv, uint32_t cid, bool has) {
    const uint32_t lane = threadIdx.x & 63;
    uint64_t taken = 0;
    for (;;) {
      const float tv = lane_value(v, top - 1);
      const uint32_t tid = (uint32_t)__builtin_amdgcn_readlane((int)id, (int)top - 1);
      const bool better = has && (cv > tv || (cv == tv && cid < tid));
      if (!__any(better)) return taken;
      const float best = lanes_max<64>(better ? cv : -INFINITY);
      uint64_t who = __ballot(better && cv == best);
      uint32_t from = (uint32_t)__ffsll((unsigned long long)who) - 1;
      uint32_t bid = (uint32_t)__builtin_amdgcn_readlane((int)cid, (int)from);
      for (who &= who - 1; who; who &= who - 1) {  // the lowest class of equals
        const uint32_t at = (uint32_t)__ffsll((unsigned long long)who) - 1;
        const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)cid, (int)at);
        if (o < bid) bid = o, from = at;
      }
      taken |= uint64_t(1) << from;
      if (lane == from) has = false;
      const uint32_t r = (uint32_t)__popcll(__ballot(v > best || (v == best && id < bid)));
      const float pv = lane_perm<0x138>(v);  // the lane below's
      const uint32_t pid = __float_as_uint(lane_perm<0x138>(__uint_as_float(id)));
      v = lane == r ? best : lane > r ? pv : v;
      id = lane == r ? bid : lane > r ? pid : id;
    }
  }
};

// The outputs of a row, by one wave.
__device__ __forceinline__ void finish(const LogpArgs& a, int kind, size_t row, const Seen& all,
                                       const Best& best) {
  const uint32_t lane = threadIdx.x & 63;
  const float b = all.m == -INFINITY ? 0.f : all.m;
  const float ls = logf(all.s);
  const bool odd = !(all.s < INFINITY);  // a NaN, or an infinite logit
  if (lane == 0) {
    a.lse[row] = odd ? NAN : all.m == -INFINITY ? -INFINITY : all.m + ls;
    if (a.entropy) a.entropy[row] = odd ? NAN : all.s > 0.f ? ls - all.e / all.s : 0.f;
    if (a.logp) {
      const uint32_t t = a.tokens[row];
      float lp = 0.f;
      if (t < a.k) {
        lp = fmaf(load_kind(a.z, kind, row * a.ldz + t), a.scale, -b);
        lp = odd ? NAN : all.s > 0.f ? lp - ls : -INFINITY;
      } else if (t != NONE) {
        a.small[SW_BAD_CLASS] = 1u;
      }
      a.logp[row] = lp;
    }
  }
  if (lane < a.top) {
    const bool is = best.id != NONE && !odd;
    if (a.ids) a.ids[row * a.top + lane] = is ? best.id : NONE;
    if (a.tops)
      a.tops[row * a.top + lane] = odd ? NAN : is ? fmaf(best.v, a.scale, -b) - ls : -INFINITY;
  }
}

struct PartOut {  // [row][part]
  float4* seen;   // m, s, e
  float2* best;   // [row][part][top]: value, class
};

// W waves take a part of a row, by turns in chunks of 64 NV vectors; parts == 1: whole
// rows, whose results they write.
template <class T, int W, int NV, bool TOP>
__global__ __launch_bounds__(256) void k_logp(const LogpArgs a, int kind, uint32_t parts,
                                              PartOut out) {
  constexpr int N = VecOf<T>::N, ROWS = 4 / W;
  __shared__ float4 seen[4];
  __shared__ float2 lists[W > 1 ? 4 : 1][MAX_TOP];
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t w = wave % W;
  const size_t units = a.n * parts;
  for (size_t u0 = (size_t)blockIdx.x * ROWS; u0 < units; u0 += (size_t)gridDim.x * ROWS) {
    const size_t u = u0 + wave / W;
    if (W == 1 && u >= units) return;  // (waves of their own)
    const size_t row = u / parts;
    const uint32_t part = (uint32_t)(u - row * parts);
    const Row<T> r(a.z, row * a.ldz, a.k);
    const size_t nv = r.vectors(), chunks = (nv + 64 * NV - 1) / (64 * NV);
    const size_t c0 = chunks * part / parts, c1 = chunks * (part + 1) / parts;
    Seen all;
    Best best;
    Vec<T> next[NV];
    auto fetch = [&](size_t c) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < NV; j++) {
        const size_t v = c * (64 * NV) + j * 64 + lane;
        next[j] = r.load(v < nv ? v : nv - 1);
      }
    };
    if (c0 + w < c1) fetch(c0 + w);
    for (size_t c = c0 + w; c < c1; c += W) {
      Vec<T> x[NV];
#pragma unroll
      for (int j = 0; j < NV; j++) x[j] = next[j];
      if (c + W < c1) fetch(c + W);
      const size_t v0 = c * (64 * NV) + lane;
      if (c == 0 || c == chunks - 1) {
#pragma unroll
        for (int j = 0; j < NV; j++) r.mask(x[j], v0 + j * 64);
      }
      float most = -INFINITY;
#pragma unroll
      for (int j = 0; j < NV; j++)
#pragma unroll
        for (int e = 0; e < N; e++) most = fmaxf(most, x[j].get(e));
      const float to = fmaxf(all.m, most * a.scale);
      all.move(to);
      const float b = to == -INFINITY ? 0.f : to;
#pragma unroll
      for (int j = 0; j < NV; j++)
#pragma unroll
        for (int e = 0; e < N; e++) {
          const float d = fmaf(x[j].get(e), a.scale, -b);
          const float p = __builtin_amdgcn_exp2f(d * LOG2E);
          all.s += p;
          all.e = fmaf(p, fmaxf(d, FAR), all.e);
        }
      if constexpr (TOP) {
        // The largest of the lane's that comes after (v, id) in the list's order.
        auto after = [&](float v, uint32_t id, float& cv, uint32_t& cid) __attribute__((always_inline)) {
          cv = -INFINITY;
          cid = NONE;
#pragma unroll
          for (int j = 0; j < NV; j++) {
            const uint32_t col = (uint32_t)r.column(v0 + j * 64);
#pragma unroll
            for (int e = 0; e < N; e++) {
              const float q = x[j].get(e);
              const bool is = (q < v || (q == v && col + e > id)) && q > cv;
              cv = is ? q : cv;
              cid = is ? col + e : cid;
            }
          }
        };
        if (__any(most >= lane_value(best.v, a.top - 1) && most > -INFINITY)) {
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
    all.join_lanes();
    if constexpr (W > 1) {
      __syncthreads();  // (what the last unit left has been read)
      if (lane == 0) seen[wave] = all.packed();
      if (TOP && lane < a.top) lists[wave][lane] = make_float2(best.v, __uint_as_float(best.id));
      __syncthreads();
      if (wave == 0) {
        for (int i = 1; i < W; i++) {
          all.join(Seen(seen[i]));
          if constexpr (TOP) {
            const float2 o = lane < a.top ? lists[i][lane] : make_float2(-INFINITY, 0.f);
            (void)best.offer(a.top, o.x, __float_as_uint(o.y), o.x > -INFINITY);
          }
        }
      }
    }
    if (W > 1 && wave != 0) continue;
    if (parts == 1) {
      finish(a, kind, row, all, best);
    } else {
      if (lane == 0) out.seen[u] = all.packed();
      if (TOP && lane < a.top)
        out.best[u * a.top + lane] = make_float2(best.v, __uint_as_float(best.id));
    }
  }
}

// The parts of a row, by a wave.
template <bool TOP>
__global__ __launch_bounds__(64) void k_logp_join(const LogpArgs a, int kind, uint32_t parts,
                                                  PartOut in) {
  const uint32_t lane = threadIdx.x;
  for (size_t row = blockIdx.x; row < a.n; row += gridDim.x) {
    Seen all;
    for (uint32_t p = lane; p < parts; p += 64) all.join(Seen(in.seen[row * parts + p]));
    all.join_lanes();
    Best best;
    if constexpr (TOP) {
      const uint32_t count = parts * a.top;
      for (uint32_t i0 = 0; i0 < count; i0 += 64) {
        const uint32_t i = i0 + lane;
        const float2 o = i < count ? in.best[row * count + i] : make_float2(-INFINITY, 0.f);
        (void)best.offer(a.top, o.x, __float_as_uint(o.y), o.x > -INFINITY);
      }
    }
    finish(a, kind, row, all, best);
  }
}

// A wave takes 64 NV vectors of a row of dz.
template <class T, int NV>
__global__ __launch_bounds__(256) void k_logp_grad(const LogpArgs a, uint32_t chunks) {
  constexpr int N = VecOf<T>::N;
  const uint32_t lane = threadIdx.x & 63;
  const size_t wave = (size_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const size_t units = a.n * chunks;
  for (size_t u = (size_t)blockIdx.x * 4 + wave; u < units; u += (size_t)gridDim.x * 4) {
    const size_t row = u / chunks, c = u - row * chunks;
    const Row<T> o(a.dz, row * a.lddz, a.k);
    const T* z = reinterpret_cast<const T*>(a.z) + row * a.ldz;
    T* dz = const_cast<T*>(o.base) + o.head;
    const size_t nv = o.vectors(), v0 = c * (64 * NV) + lane;
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
    auto one = [&](float q, bool own) __attribute__((always_inline)) {
      const float d = fmaf(q, a.scale, -lse);
      const float p = __builtin_amdgcn_exp2f(d * LOG2E);
      const float g = -p * fmaf(gh, fmaxf(d, FAR) + h, gl);
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
        store_vec(dz + col, g);
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
    const size_t vectors = (a.k + N - 1) / N + 1;  // (of a row at any address)
    // A wave a row where the row is a chunk or two and the rows fill the GPU; otherwise four,
    // and parts of a row where there are few rows.
    const bool small = vectors <= 64 * 8 && a.n >= (size_t)c->cus;
    const size_t chunks = (vectors + 255) / 256;
    size_t parts = 1;
    if (!small) parts = std::min((chunks + 3) / 4, std::max<size_t>(1, 4 * (size_t)c->cus / a.n));
    PartOut out{};
    if (parts > 1) {
      const size_t seen = (a.n * parts * sizeof(float4) + 255) & ~size_t(255);
      char* p = (char*)c->logp_part.get(seen + a.n * parts * a.top * sizeof(float2), c->stream);
      out.seen = (float4*)p;
      out.best = (float2*)(p + seen);
    }
    auto go = [&](auto waves, auto nv, auto top) {
      constexpr int W = decltype(waves)::value, NV = decltype(nv)::value;
      constexpr bool TOP = decltype(top)::value;
      const size_t groups = (a.n * parts + 4 / W - 1) / (4 / W);
      k_logp<T, W, NV, TOP><<<dim3((unsigned)std::min(groups, MAX_GROUPS)), 256, 0, c->stream>>>(
          a, kind, (uint32_t)parts, out);
      if (parts > 1)
        k_logp_join<TOP><<<dim3((unsigned)std::min(a.n, MAX_GROUPS)), 64, 0, c->stream>>>(
            a, kind, (uint32_t)parts, out);
    };
    auto with_top = [&](auto top) {
      if (!small)
        go(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{}, top);
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
    const size_t vectors = (a.k + N - 1) / N + 1, chunks = (vectors + 64 * NV - 1) / (64 * NV);
    const size_t groups = (a.n * chunks + 3) / 4;
    k_logp_grad<T, NV><<<dim3((unsigned)std::min(groups, MAX_GROUPS)), 256, 0, c->stream>>>(
        a, (uint32_t)chunks);
  });
  EMH_HIP(hipGetLastError());
}

}  // namespace emh
