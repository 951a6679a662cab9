// The C ABI of the operators that a classifier answers and is tuned with
// (include/emeans_hip.h): their arguments, checked before anything is queued, and the plan of
// a gradient norm.

#include <algorithm>
#include <cmath>
#include <cstring>
#include <memory>
#include <mutex>
#include <vector>

#include "emh_answer.h"
#include "emh_check.h"

struct emh_grad_norm {
  emh_ctx* ctx = nullptr;  // null once it is destroyed
  double* sums = nullptr;  // a block on the device, with what follows
  emh::NormTensor* tensors = nullptr;
  uint2* chunks = nullptr;
  size_t nchunks = 0, chunk = 0;
  bool stream = false;
  std::vector<emh_buf*> written;
  std::vector<Range> ranges;  // of gradients and outputs
};

namespace {

// A context's list of plans: a plan may be destroyed on another thread than its context.
std::mutex g_norms_mu;

void free_tables(emh_grad_norm* p) {
  if (p->sums) (void)hipFree(p->sums);
  p->sums = nullptr;
}

constexpr size_t RMS_D = size_t(1) << 24, RMS_ROWS = size_t(1) << 31;

size_t code_blocks(size_t n) { return (n + EMH_CODE_BLOCK - 1) / EMH_CODE_BLOCK; }

// rows x d codes whose rows begin at multiples of 16 bytes, ld (0: d rounded up) too: their
// range goes to the end of the last row's sixteen.
Range check_codes(const emh_buf* b, size_t rows, size_t d, size_t& ld, const char* what) {
  EMH_ENSURE(b && b->kind == EMH_F8, "%s must be an f8 buffer", what);
  const size_t wide = (d + 15) & ~size_t(15);
  if (ld == 0) ld = wide;
  EMH_ENSURE(ld >= wide && ld % 16 == 0,
             "%s: the stride %zu of rows of %zu codes must be a multiple of 16 that holds them",
             what, ld, d);
  EMH_ENSURE((uintptr_t)b->ptr % 16 == 0, "%s must begin at a multiple of 16 bytes", what);
  return check_matrix(b, rows, wide, ld, what);
}
// Their scales, f32.
Range check_scales(const emh_buf* b, size_t rows, size_t d, size_t& ld, const char* what) {
  EMH_ENSURE(b && b->kind == EMH_F32, "%s must be an f32 buffer", what);
  return check_matrix(b, rows, code_blocks(d), ld, what);
}

struct Named {
  Range r;
  const char* name;
};
// No output meets an input or another output.
void all_apart(const std::vector<Named>& out, const std::vector<Named>& in) {
  for (size_t i = 0; i < out.size(); i++) {
    for (const Named& v : in) apart(out[i].r, v.r, out[i].name, v.name);
    for (size_t j = 0; j < i; j++) apart(out[i].r, out[j].r, out[i].name, out[j].name);
  }
}

}  // namespace

extern "C" {

int emh_rms_norm(emh_ctx* c, const emh_buf* x, size_t ldx, const emh_buf* residual, size_t ldr,
                 size_t rows, size_t d, const emh_buf* weight, float eps, emh_buf* h, size_t ldh,
                 emh_buf* y, size_t ldy, emh_buf* scales, size_t lds, emh_buf* rstd) {
  return guard([&] {
    EMH_ENSURE(c, "null context");
    EMH_ENSURE(d > 0 && d <= RMS_D, "d must be 1 to 2^24");
    EMH_ENSURE(rows < RMS_ROWS, "too many rows");
    EMH_ENSURE(x && real_kind(x->kind), "x must be an f32, f16 or bf16 buffer");
    EMH_ENSURE(!residual || residual->kind == x->kind, "residual must be of x's kind");
    EMH_ENSURE(!h || h->kind == x->kind, "h must be of x's kind");
    EMH_ENSURE(y && (y->kind == x->kind || y->kind == EMH_F8), "y must be of x's kind or f8");
    EMH_ENSURE((y->kind == EMH_F8) == (scales != nullptr),
               "an f8 y comes with scales, another with none");
    EMH_ENSURE(eps >= 0.f && std::isfinite(eps), "eps must be finite and not negative");
    const Range rx = check_matrix(x, rows, d, ldx, "x");
    Range rr, rh, rw, rs, rt;
    if (residual) rr = check_matrix(residual, rows, d, ldr, "residual");
    const emh::MatIn w = check_affine(weight, d, x->kind, "weight", rw);
    if (h) {
      rh = check_matrix(h, rows, d, ldh, "h");
      apart_or_same(rh, rx, ldh == ldx, "h", "x");
      apart_or_same(rh, rr, ldh == ldr, "h", "residual");
      apart(rh, rw, "h", "weight");
    }
    Range ry;
    if (scales) {
      ry = check_codes(y, rows, d, ldy, "y");
      rs = check_scales(scales, rows, d, lds, "scales");
      apart(ry, rx, "y", "x");
      apart(ry, rr, "y", "residual");
    } else {
      ry = check_matrix(y, rows, d, ldy, "y");
      apart_or_same(ry, rx, ldy == ldx, "y", "x");
      apart_or_same(ry, rr, ldy == ldr, "y", "residual");
    }
    apart(ry, rw, "y", "weight");
    apart(ry, rh, "y", "h");
    if (rstd) rt = check_f32(rstd, rows, "rstd");
    all_apart({{rs, "scales"}, {rt, "rstd"}},
              {{rx, "x"}, {rr, "residual"}, {rw, "weight"}, {rh, "h"}, {ry, "y"}});
    use_device(c);
    for (emh_buf* o : {h, y, scales, rstd})
      if (o) ++o->gen;
    emh::RmsArgs a{};
    a.x = x->ptr, a.ldx = ldx, a.rows = rows, a.d = (int)d, a.kind = x->kind;
    if (residual) a.r = residual->ptr, a.ldr = ldr;
    a.w = w.p, a.wkind = w.kind, a.eps = eps;
    if (h) a.h = h->ptr, a.ldh = ldh;
    a.y = y->ptr, a.ldy = ldy;
    if (scales) a.scale = (float*)scales->ptr, a.lds = lds;
    a.rstd = rstd ? (float*)rstd->ptr : nullptr;
    emh::launch_rms_norm(c, a);
  });
}

int emh_rms_norm_grad(emh_ctx* c, const emh_buf* dy, size_t lddy, const emh_buf* dh, size_t lddh,
                      const emh_buf* h, size_t ldh, size_t rows, size_t d, const emh_buf* weight,
                      const emh_buf* rstd, emh_buf* dx, size_t lddx, emh_buf* dweight) {
  return guard([&] {
    EMH_ENSURE(c, "null context");
    EMH_ENSURE(d > 0 && d <= RMS_D, "d must be 1 to 2^24");
    EMH_ENSURE(rows < RMS_ROWS, "too many rows");
    EMH_ENSURE(h && real_kind(h->kind), "h must be an f32, f16 or bf16 buffer");
    EMH_ENSURE(dy && dy->kind == h->kind, "dy must be of h's kind");
    EMH_ENSURE(!dh || dh->kind == h->kind, "dh must be of h's kind");
    EMH_ENSURE(!dx || dx->kind == h->kind, "dx must be of h's kind");
    EMH_ENSURE(!dweight || dweight->kind == h->kind || dweight->kind == EMH_F32,
               "dweight must be f32 or of h's kind");
    const Range rh = check_matrix(h, rows, d, ldh, "h"), ry = check_matrix(dy, rows, d, lddy, "dy");
    Range rd, rw, rx, rg;
    if (dh) rd = check_matrix(dh, rows, d, lddh, "dh");
    const emh::MatIn w = check_affine(weight, d, h->kind, "weight", rw);
    const Range rt = check_f32(rstd, rows, "rstd");
    if (dx) {
      rx = check_matrix(dx, rows, d, lddx, "dx");
      apart_or_same(rx, ry, lddx == lddy, "dx", "dy");
      apart_or_same(rx, rd, lddx == lddh, "dx", "dh");
      all_apart({{rx, "dx"}}, {{rh, "h"}, {rw, "weight"}, {rt, "rstd"}});
    }
    if (dweight) {
      rg = check_vector(dweight, d, "dweight");
      all_apart({{rg, "dweight"}}, {{rh, "h"}, {rw, "weight"}, {rt, "rstd"}, {ry, "dy"},
                                    {rd, "dh"}, {rx, "dx"}});
    }
    if (!dx && !dweight) return;
    use_device(c);
    for (emh_buf* o : {dx, dweight})
      if (o) ++o->gen;
    emh::RmsArgs a{};
    a.x = h->ptr, a.ldx = ldh, a.rows = rows, a.d = (int)d, a.kind = h->kind;
    if (dh) a.r = dh->ptr, a.ldr = lddh;
    a.dy = dy->ptr, a.lddy = lddy, a.w = w.p, a.wkind = w.kind;
    a.rstd = (float*)rstd->ptr;
    if (dx) a.y = dx->ptr, a.ldy = lddx;
    emh::MatOut g;
    if (dweight) g = {dweight->ptr, d, dweight->kind};
    emh::launch_rms_norm_grad(c, a, g);
  });
}

int emh_quantize(emh_ctx* c, const emh_buf* x, size_t ldx, size_t rows, size_t d, size_t tile_rows,
                 emh_buf* q, size_t ldq, emh_buf* scales, size_t lds) {
  return guard([&] {
    EMH_ENSURE(c, "null context");
    EMH_ENSURE(d > 0 && d <= RMS_D, "d must be 1 to 2^24");
    EMH_ENSURE(rows < RMS_ROWS, "too many rows");
    EMH_ENSURE(tile_rows == 1 || tile_rows == EMH_CODE_BLOCK, "a scale serves 1 or %d rows",
               EMH_CODE_BLOCK);
    EMH_ENSURE(x && real_kind(x->kind), "x must be an f32, f16 or bf16 buffer");
    const Range rx = check_matrix(x, rows, d, ldx, "x"), rq = check_codes(q, rows, d, ldq, "q");
    const Range rs =
        check_scales(scales, tile_rows == 1 ? rows : code_blocks(rows), d, lds, "scales");
    all_apart({{rq, "q"}, {rs, "scales"}}, {{rx, "x"}});
    use_device(c);
    ++q->gen;
    ++scales->gen;
    emh::launch_quantize(c, {x->ptr, ldx, x->kind}, rows, d, tile_rows != 1, (uint8_t*)q->ptr, ldq,
                         (float*)scales->ptr, lds);
  });
}

int emh_product8(emh_ctx* c, const emh_buf* x, size_t ldx, const emh_buf* xscales, size_t ldxs,
                 size_t n, size_t d, const emh_buf* w, size_t ldw, const emh_buf* wscales,
                 size_t ldws, size_t k, emh_buf* y, size_t ldy) {
  return guard([&] {
    EMH_ENSURE(c, "null context");
    EMH_ENSURE(d > 0 && d <= (size_t(1) << 21), "d must be 1 to 2^21");
    EMH_ENSURE(k > 0 && k <= (size_t(1) << 30), "k must be 1 to 2^30");
    EMH_ENSURE(n <= (size_t(1) << 30), "too many rows");
    EMH_ENSURE(y && real_kind(y->kind), "y must be an f32, f16 or bf16 buffer");
    const Range rx = check_codes(x, n, d, ldx, "x"), rw = check_codes(w, k, d, ldw, "w");
    const Range rxs = check_scales(xscales, n, d, ldxs, "xscales");
    const Range rws = check_scales(wscales, code_blocks(k), d, ldws, "wscales");
    const Range ry = check_matrix(y, n, k, ldy, "y");
    all_apart({{ry, "y"}}, {{rx, "x"}, {rw, "w"}, {rxs, "xscales"}, {rws, "wscales"}});
    use_device(c);
    ++y->gen;
    emh::launch_product8(c, {(const uint8_t*)x->ptr, ldx, (const float*)xscales->ptr, ldxs}, n, d,
                         {(const uint8_t*)w->ptr, ldw, (const float*)wscales->ptr, ldws}, k,
                         {y->ptr, ldy, y->kind});
  });
}

}  // extern "C"

namespace {
struct LogpCall {
  emh::LogpArgs a;
  Range z, tokens;
};
LogpCall check_logp(emh_ctx* c, const emh_buf* z, size_t ldz, size_t n, size_t k,
                    const emh_buf* tokens, float scale) {
  EMH_ENSURE(c, "null context");
  EMH_ENSURE(k > 0 && k <= (size_t(1) << 30), "k must be 1 to 2^30");
  EMH_ENSURE(n <= (size_t(1) << 30), "too many rows");
  EMH_ENSURE(z && real_kind(z->kind), "z must be an f32, f16 or bf16 buffer");
  EMH_ENSURE(scale > 0.f && std::isfinite(scale), "scale must be finite and positive");
  LogpCall t{};
  t.z = check_matrix(z, n, k, ldz, "z");
  if (tokens) {
    EMH_ENSURE(tokens->kind == EMH_U32, "tokens must be a u32 buffer");
    t.tokens = check_vector(tokens, n, "tokens");
    t.a.tokens = (const uint32_t*)tokens->ptr;
  }
  t.a.z = z->ptr, t.a.ldz = ldz, t.a.n = n, t.a.k = k, t.a.scale = scale;
  return t;
}
}  // namespace

extern "C" {

int emh_log_probs(emh_ctx* c, const emh_buf* z, size_t ldz, size_t n, size_t k,
                  const emh_buf* tokens, float scale, emh_buf* logp, emh_buf* lse,
                  emh_buf* entropy, size_t top, emh_buf* top_ids, emh_buf* top_logp) {
  return guard([&] {
    LogpCall t = check_logp(c, z, ldz, n, k, tokens, scale);
    EMH_ENSURE((tokens != nullptr) == (logp != nullptr), "tokens and logp come together");
    EMH_ENSURE(top <= EMH_MAX_TOP, "top must be at most %d", EMH_MAX_TOP);
    EMH_ENSURE(top > 0 ? top_ids || top_logp : !top_ids && !top_logp,
               "top and its outputs come together");
    std::vector<Named> out = {{check_f32(lse, n, "lse"), "lse"}};
    if (logp) out.push_back({check_f32(logp, n, "logp"), "logp"});
    if (entropy) out.push_back({check_f32(entropy, n, "entropy"), "entropy"});
    if (top_ids) {
      EMH_ENSURE(top_ids->kind == EMH_U32, "top_ids must be a u32 buffer");
      out.push_back({check_vector(top_ids, n * top, "top_ids"), "top_ids"});
    }
    if (top_logp) out.push_back({check_f32(top_logp, n * top, "top_logp"), "top_logp"});
    all_apart(out, {{t.z, "z"}, {t.tokens, "tokens"}});
    use_device(c);
    for (emh_buf* o : {logp, lse, entropy, top_ids, top_logp})
      if (o) ++o->gen;
    t.a.lse = (float*)lse->ptr;
    t.a.logp = logp ? (float*)logp->ptr : nullptr;
    t.a.entropy = entropy ? (float*)entropy->ptr : nullptr;
    t.a.top = (uint32_t)top;
    t.a.ids = top_ids ? (uint32_t*)top_ids->ptr : nullptr;
    t.a.tops = top_logp ? (float*)top_logp->ptr : nullptr;
    emh::launch_log_probs(c, t.a, z->kind);
  });
}

int emh_log_probs_grad(emh_ctx* c, const emh_buf* z, size_t ldz, size_t n, size_t k,
                       const emh_buf* tokens, float scale, const emh_buf* lse,
                       const emh_buf* entropy, const emh_buf* glogp, const emh_buf* gentropy,
                       emh_buf* dz, size_t lddz) {
  return guard([&] {
    LogpCall t = check_logp(c, z, ldz, n, k, tokens, scale);
    EMH_ENSURE(dz && dz->kind == z->kind, "dz must be of z's kind");
    EMH_ENSURE((tokens != nullptr) == (glogp != nullptr), "tokens and glogp come together");
    EMH_ENSURE((entropy != nullptr) == (gentropy != nullptr), "entropy and gentropy come together");
    const Range rd = check_matrix(dz, n, k, lddz, "dz");
    apart_or_same(rd, t.z, lddz == t.a.ldz, "dz", "z");
    std::vector<Named> in = {{t.tokens, "tokens"}, {check_f32(lse, n, "lse"), "lse"}};
    if (glogp) in.push_back({check_f32(glogp, n, "glogp"), "glogp"});
    if (entropy) in.push_back({check_f32(entropy, n, "entropy"), "entropy"});
    if (gentropy) in.push_back({check_f32(gentropy, n, "gentropy"), "gentropy"});
    all_apart({{rd, "dz"}}, in);
    use_device(c);
    ++dz->gen;
    t.a.lse_in = (const float*)lse->ptr;
    t.a.glogp = glogp ? (const float*)glogp->ptr : nullptr;
    t.a.entropy_in = entropy ? (const float*)entropy->ptr : nullptr;
    t.a.gentropy = gentropy ? (const float*)gentropy->ptr : nullptr;
    t.a.dz = dz->ptr, t.a.lddz = lddz;
    emh::launch_log_probs_grad(c, t.a, z->kind);
  });
}

int emh_grad_norm_create(emh_ctx* c, const emh_buf* const* grads, emh_buf* const* outs,
                         size_t count, emh_grad_norm** out) {
  return guard([&] {
    EMH_ENSURE(c && out, "null argument");
    EMH_ENSURE(count == 0 || grads, "null tensors");
    auto plan = std::make_unique<emh_grad_norm>();
    plan->ctx = c;
    struct Tensor {
      Range g, o;
      size_t i;
    };
    std::vector<Tensor> all;
    std::vector<emh::NormTensor> table;
    std::vector<uint2> chunks;
    size_t total = 0;
    size_t bytes = 0;
    for (size_t i = 0; i < count; i++) {
      total += grads[i] ? grads[i]->len : 0;
      bytes += grads[i] ? grads[i]->len * emh::kind_bytes(grads[i]->kind) : 0;
    }
    plan->stream = outs && bytes >= emh::STREAM_FROM / 2;  // (with what is read, twice that)
    plan->chunk = total <= emh::NORM_FEW ? emh::NORM_CHUNK_FEW : emh::NORM_CHUNK;
    for (size_t i = 0; i < count; i++) {
      const emh_buf* g = grads[i];
      EMH_ENSURE(g && real_kind(g->kind), "tensor %zu: grad must be f32, f16 or bf16", i);
      Tensor t{check_vector(g, g->len, "grad"), {}, i};
      t.o = t.g;
      if (outs) {
        EMH_ENSURE(outs[i] && outs[i]->kind == g->kind && outs[i]->len == g->len,
                   "tensor %zu: its output must be of grad's kind and length", i);
        t.o = check_vector(outs[i], g->len, "output");
        plan->written.push_back(outs[i]);
      } else {
        plan->written.push_back(const_cast<emh_buf*>(g));
      }
      EMH_ENSURE(g->len < (size_t(1) << 41), "tensor %zu is too long", i);
      for (size_t k = 0; k * plan->chunk < g->len; k++)
        chunks.push_back(make_uint2((unsigned)table.size(), (unsigned)k));
      table.push_back({g->ptr, (void*)t.o.lo, g->len, g->kind, 0});
      if (g->len > 0) all.push_back(t);
      plan->ranges.push_back(t.g);
      plan->ranges.push_back(t.o);
    }
    EMH_ENSURE(chunks.size() < (size_t(1) << 24), "too many tensors or elements for one plan");
    // What is written is written once, and read by no other tensor; gradients may overlap
    // only where nothing is written to them.
    std::sort(all.begin(), all.end(), [](const Tensor& a, const Tensor& b) { return a.o.lo < b.o.lo; });
    for (size_t i = 1; i < all.size(); i++)
      EMH_ENSURE(all[i - 1].o.hi <= all[i].o.lo, "tensors %zu and %zu: what is written overlaps",
                 all[i - 1].i, all[i].i);
    for (const Tensor& t : all) {
      auto it = std::lower_bound(all.begin(), all.end(), t.g.hi,
                                 [](const Tensor& a, const char* hi) { return a.o.lo < hi; });
      while (it != all.begin()) {
        --it;
        if (it->o.hi <= t.g.lo) break;
        EMH_ENSURE(it->i == t.i && t.o.same(t.g),
                   "tensor %zu: its gradient overlaps what is written for tensor %zu", t.i, it->i);
      }
    }
    use_device(c);
    plan->nchunks = chunks.size();
    // One block: the sums, then the tables (each entry's size is a multiple of 8).
    const size_t first = emh::NORM_SUMS * sizeof(double);
    const size_t named = table.size() * sizeof table[0], parts = chunks.size() * sizeof chunks[0];
    try {
      EMH_HIP(hipMalloc(&plan->sums, first + named + parts));
      char* p = (char*)plan->sums + first;
      plan->tensors = (emh::NormTensor*)p;
      plan->chunks = (uint2*)(p + named);
      if (parts > 0) {
        std::vector<char> host(named + parts);
        memcpy(host.data(), table.data(), named);
        memcpy(host.data() + named, chunks.data(), parts);
        EMH_HIP(hipMemcpyAsync(p, host.data(), host.size(), hipMemcpyHostToDevice, c->stream));
        EMH_HIP(hipStreamSynchronize(c->stream));  // the host's tables go away
      }
      std::lock_guard<std::mutex> g(g_norms_mu);
      c->norms.push_back(plan.get());
    } catch (...) {
      free_tables(plan.get());
      throw;
    }
    *out = plan.release();
  });
}

}  // extern "C"

namespace {
void measure(emh_grad_norm* plan, float scale, float max_norm, emh_buf* out, bool clip) {
  EMH_ENSURE(plan, "null argument");
  EMH_ENSURE(plan->ctx, "the plan's context is destroyed");
  EMH_ENSURE(std::isfinite(scale), "scale must be finite");
  EMH_ENSURE(max_norm >= 0.f, "max_norm must not be negative");
  const Range ro = check_f32(out, 2, "out");
  for (const Range& r : plan->ranges) apart(ro, r, "out", "a tensor");
  use_device(plan->ctx);
  ++out->gen;
  if (clip)
    for (emh_buf* b : plan->written) ++b->gen;
  emh::launch_grad_norm(plan->ctx, plan->tensors, plan->chunks, plan->nchunks, plan->chunk,
                        plan->stream, plan->sums, scale, max_norm, (float*)out->ptr, clip);
}
}  // namespace

extern "C" {

int emh_grad_norm_measure(emh_grad_norm* plan, float scale, float max_norm, emh_buf* out) {
  return guard([&] { measure(plan, scale, max_norm, out, false); });
}
int emh_grad_norm_clip(emh_grad_norm* plan, float scale, float max_norm, emh_buf* out) {
  return guard([&] { measure(plan, scale, max_norm, out, true); });
}

int emh_grad_norm_destroy(emh_grad_norm* plan) {
  return guard([&] {
    if (!plan) return;
    std::unique_ptr<emh_grad_norm> hold(plan);
    std::lock_guard<std::mutex> g(g_norms_mu);
    if (!plan->ctx) return;  // its context went first, and the tables with it
    auto& plans = plan->ctx->norms;
    plans.erase(std::remove(plans.begin(), plans.end(), plan), plans.end());
    use_device(plan->ctx);
    const hipError_t e = hipStreamSynchronize(plan->ctx->stream);  // a queued call may read the tables
    free_tables(plan);
    EMH_HIP(e);
  });
}

}  // extern "C"

namespace emh {
void drop_norms(emh_ctx* c) {
  std::lock_guard<std::mutex> g(g_norms_mu);
  for (emh_grad_norm* p : c->norms) {
    free_tables(p);
    p->ctx = nullptr;
  }
  c->norms.clear();
}
}  // namespace emh
