// The C ABI of the learning operators (include/emeans_hip.h): their arguments,
// checked before anything is queued, and the AdamW plan.

#include <algorithm>
#include <cmath>
#include <memory>
#include <mutex>
#include <vector>

#include "emh_check.h"

struct emh_adamw {
  emh_ctx* ctx = nullptr;  // null once it is destroyed
  emh::AdamTensor* tensors = nullptr;  // on the device
  uint2* chunks = nullptr;
  size_t nchunks = 0, chunk = emh::ADAM_CHUNK;
  bool random = false;  // emh_adamw_set_seed
  uint64_t seed = 0;
  std::vector<emh_buf*> written;
  std::vector<Range> ranges;  // of what a step writes
};

namespace {

// A context's list of plans: a plan may be destroyed on another thread than its context.
std::mutex g_plans_mu;

void free_tables(emh_adamw* p) {
  if (p->tensors) (void)hipFree(p->tensors);
  if (p->chunks) (void)hipFree(p->chunks);
  p->tensors = nullptr;
  p->chunks = nullptr;
}

}  // namespace

extern "C" {

int emh_layer_norm(emh_ctx* c, const emh_buf* x, size_t ldx, size_t rows, size_t d,
                   const emh_buf* weight, const emh_buf* bias, float eps, emh_buf* y, size_t ldy,
                   emh_buf* mean, emh_buf* rstd) {
  return guard([&] {
    EMH_ENSURE(c, "null context");
    EMH_ENSURE(d > 0 && d <= MAX_D, "d must be 1 to 2^30");
    EMH_ENSURE(rows < (size_t(1) << 31), "too many rows");
    EMH_ENSURE(x && real_kind(x->kind), "x must be an f32, f16 or bf16 buffer");
    EMH_ENSURE(y && y->kind == x->kind, "y must be of x's kind");
    EMH_ENSURE(eps >= 0.f && std::isfinite(eps), "eps must be finite and not negative");
    const Range rx = check_matrix(x, rows, d, ldx, "x"), ry = check_matrix(y, rows, d, ldy, "y");
    apart_or_same(ry, rx, ldx == ldy, "y", "x");
    Range rw, rb;
    const emh::MatIn w = check_affine(weight, d, x->kind, "weight", rw);
    const emh::MatIn b = check_affine(bias, d, x->kind, "bias", rb);
    apart(ry, rw, "y", "weight");
    apart(ry, rb, "y", "bias");
    Range rs[2];
    emh_buf* stat[2] = {mean, rstd};
    const char* name[2] = {"mean", "rstd"};
    for (int i = 0; i < 2; i++) {
      if (!stat[i]) continue;
      rs[i] = check_f32(stat[i], rows, name[i]);
      apart(rs[i], rx, name[i], "x");
      apart(rs[i], ry, name[i], "y");
      apart(rs[i], rw, name[i], "weight");
      apart(rs[i], rb, name[i], "bias");
    }
    apart(rs[0], rs[1], "mean", "rstd");
    use_device(c);
    for (emh_buf* o : {y, mean, rstd})
      if (o) ++o->gen;
    emh::launch_layer_norm(c, {x->ptr, ldx, x->kind}, rows, d, w, b, eps, {y->ptr, ldy, y->kind},
                           mean ? (float*)mean->ptr : nullptr, rstd ? (float*)rstd->ptr : nullptr);
  });
}

int emh_layer_norm_grad(emh_ctx* c, const emh_buf* dy, size_t lddy, const emh_buf* x, size_t ldx,
                        size_t rows, size_t d, const emh_buf* weight, const emh_buf* mean,
                        const emh_buf* rstd, emh_buf* dx, size_t lddx, emh_buf* dweight,
                        emh_buf* dbias) {
  return guard([&] {
    EMH_ENSURE(c, "null context");
    EMH_ENSURE(d > 0 && d <= MAX_D, "d must be 1 to 2^30");
    EMH_ENSURE(rows < (size_t(1) << 31), "too many rows");
    EMH_ENSURE(x && real_kind(x->kind), "x must be an f32, f16 or bf16 buffer");
    EMH_ENSURE(dy && dy->kind == x->kind, "dy must be of x's kind");
    const Range rx = check_matrix(x, rows, d, ldx, "x");
    const Range rdy = check_matrix(dy, rows, d, lddy, "dy");
    Range rw;
    const emh::MatIn w = check_affine(weight, d, x->kind, "weight", rw);
    const Range in[5] = {rx, rdy, rw, check_f32(mean, rows, "mean"), check_f32(rstd, rows, "rstd")};
    const char* in_name[5] = {"x", "dy", "weight", "mean", "rstd"};
    Range out[3];
    const char* out_name[3] = {"dx", "dweight", "dbias"};
    emh_buf* o[3] = {dx, dweight, dbias};
    for (int i = 0; i < 3; i++) {
      if (!o[i]) continue;
      EMH_ENSURE(o[i]->kind == x->kind || (i > 0 && o[i]->kind == EMH_F32), "%s must be %sof x's kind",
                 out_name[i], i > 0 ? "f32 or " : "");
      out[i] = i == 0 ? check_matrix(dx, rows, d, lddx, "dx") : check_vector(o[i], d, out_name[i]);
      for (int j = 0; j < 5; j++) {
        if (i == 0 && j == 1)
          apart_or_same(out[i], in[j], lddx == lddy, out_name[i], in_name[j]);
        else
          apart(out[i], in[j], out_name[i], in_name[j]);
      }
      for (int j = 0; j < i; j++) apart(out[i], out[j], out_name[i], out_name[j]);
    }
    if (!dx && !dweight && !dbias) return;
    use_device(c);
    for (emh_buf* b : o)
      if (b) ++b->gen;
    emh::MatOut mo[3];
    for (int i = 0; i < 3; i++)
      if (o[i]) mo[i] = {o[i]->ptr, i == 0 ? lddx : d, o[i]->kind};
    emh::launch_layer_norm_grad(c, {dy->ptr, lddy, dy->kind}, {x->ptr, ldx, x->kind}, rows, d, w,
                                (const float*)mean->ptr, (const float*)rstd->ptr, mo[0], mo[1],
                                mo[2]);
  });
}

}  // extern "C"

namespace {
constexpr size_t XENT_D = size_t(1) << 21, XENT_K = size_t(1) << 30, XENT_N = size_t(1) << 30;
struct XentCall {
  emh::XentIn in;
  Range x, w, labels;
};
XentCall check_xent(emh_ctx* c, const emh_buf* x, size_t ldx, size_t n, size_t d, const emh_buf* w,
                    size_t ldw, size_t k, const emh_buf* labels, float scale) {
  EMH_ENSURE(c, "null context");
  EMH_ENSURE(d > 0 && d <= XENT_D, "d must be 1 to 2^21");
  EMH_ENSURE(k > 0 && k <= XENT_K, "k must be 1 to 2^30");
  EMH_ENSURE(n <= XENT_N, "too many rows");
  EMH_ENSURE(x && real_kind(x->kind), "x must be an f32, f16 or bf16 buffer");
  EMH_ENSURE(w && w->kind == x->kind, "w must be of x's kind");
  EMH_ENSURE(labels && labels->kind == EMH_U32, "labels must be a u32 buffer");
  EMH_ENSURE(std::isfinite(scale), "scale must be finite");
  XentCall t{};
  t.x = check_matrix(x, n, d, ldx, "x");
  t.w = check_matrix(w, k, d, ldw, "w");
  t.labels = check_vector(labels, n, "labels");
  t.in = {{x->ptr, ldx, x->kind}, {w->ptr, ldw, w->kind}, n, d, k, (const uint32_t*)labels->ptr,
          scale};
  return t;
}
void apart_from_inputs(const Range& r, const XentCall& t, const char* what) {
  apart(r, t.x, what, "x");
  apart(r, t.w, what, "w");
  apart(r, t.labels, what, "labels");
}
}  // namespace

extern "C" {

int emh_cross_entropy(emh_ctx* c, const emh_buf* x, size_t ldx, size_t n, size_t d,
                      const emh_buf* w, size_t ldw, size_t k, const emh_buf* labels, float scale,
                      emh_buf* loss, emh_buf* lse) {
  return guard([&] {
    const XentCall t = check_xent(c, x, ldx, n, d, w, ldw, k, labels, scale);
    const Range rl = check_f32(loss, n, "loss");
    apart_from_inputs(rl, t, "loss");
    if (lse) {
      const Range rs = check_f32(lse, n, "lse");
      apart_from_inputs(rs, t, "lse");
      apart(rs, rl, "lse", "loss");
    }
    if (n == 0) return;
    use_device(c);
    ++loss->gen;
    if (lse) ++lse->gen;
    emh::launch_cross_entropy(c, t.in, (float*)loss->ptr, lse ? (float*)lse->ptr : nullptr);
  });
}

int emh_cross_entropy_grad(emh_ctx* c, const emh_buf* x, size_t ldx, size_t n, size_t d,
                           const emh_buf* w, size_t ldw, size_t k, const emh_buf* labels,
                           float scale, const emh_buf* lse, const emh_buf* gloss, emh_buf* dx,
                           size_t lddx, emh_buf* dw, size_t lddw) {
  return emh_cross_entropy_grad_scaled(c, x, ldx, n, d, w, ldw, k, labels, scale, lse, gloss, 1.f, dx,
                                       lddx, dw, lddw);
}

int emh_cross_entropy_grad_scaled(emh_ctx* c, const emh_buf* x, size_t ldx, size_t n, size_t d,
                                  const emh_buf* w, size_t ldw, size_t k, const emh_buf* labels,
                                  float scale, const emh_buf* lse, const emh_buf* gloss,
                                  float loss_scale, emh_buf* dx, size_t lddx, emh_buf* dw,
                                  size_t lddw) {
  return guard([&] {
    EMH_ENSURE(std::isfinite(loss_scale), "loss_scale must be finite");
    EMH_ENSURE(std::isfinite(scale * loss_scale), "scale times loss_scale must be finite");
    const XentCall t = check_xent(c, x, ldx, n, d, w, ldw, k, labels, scale);
    const Range rs = check_f32(lse, n, "lse");
    Range rg;
    if (gloss) rg = check_f32(gloss, n, "gloss");
    Range out[2];
    emh_buf* o[2] = {dx, dw};
    size_t* ld[2] = {&lddx, &lddw};
    const char* name[2] = {"dx", "dw"};
    for (int i = 0; i < 2; i++) {
      if (!o[i]) continue;
      EMH_ENSURE(o[i]->kind == x->kind, "%s must be of x's kind", name[i]);
      out[i] = check_matrix(o[i], i ? k : n, d, *ld[i], name[i]);
      apart_from_inputs(out[i], t, name[i]);
      apart(out[i], rs, name[i], "lse");
      apart(out[i], rg, name[i], "gloss");
    }
    apart(out[0], out[1], "dx", "dw");
    if (!dx && !dw) return;
    use_device(c);
    emh::MatOut mo[2];
    for (int i = 0; i < 2; i++) {
      if (!o[i]) continue;
      ++o[i]->gen;
      mo[i] = {o[i]->ptr, *ld[i], o[i]->kind};
    }
    emh::launch_cross_entropy_grad(c, t.in, (const float*)lse->ptr,
                                   gloss ? (const float*)gloss->ptr : nullptr, loss_scale, mo[0],
                                   mo[1]);
  });
}

int emh_set_xent_workspace(emh_ctx* c, uint64_t bytes) {
  return guard([&] {
    EMH_ENSURE(c, "null context");
    c->xent_workspace = bytes ? (size_t)bytes : emh::XENT_WORKSPACE;
  });
}

int emh_host_xent_products(uint64_t n, uint64_t d, uint64_t k, int kind, int cus, uint64_t workspace,
                           emh_xent_product* out, uint64_t cap, uint64_t* count) {
  return guard([&] {
    EMH_ENSURE(count && (out || cap == 0), "null argument");
    EMH_ENSURE(d > 0 && d <= XENT_D && k > 0 && k <= XENT_K && n <= XENT_N, "size out of range");
    EMH_ENSURE(real_kind(kind), "kind must be f32, f16 or bf16");
    EMH_ENSURE(cus > 0, "cus must be positive");
    const auto all = emh::cross_entropy_products(n, d, k, kind == EMH_F32, cus,
                                                 workspace ? (size_t)workspace : emh::XENT_WORKSPACE);
    *count = all.size();
    std::copy_n(all.begin(), std::min<size_t>(all.size(), cap), out);
  });
}

int emh_adamw_create(emh_ctx* c, const emh_adamw_tensor* tensors, size_t count, emh_adamw** out) {
  return guard([&] {
    EMH_ENSURE(c && out, "null argument");
    EMH_ENSURE(count == 0 || tensors, "null tensors");
    std::vector<emh::AdamTensor> table;
    std::vector<uint2> chunks;
    struct Written {
      Range r;
      size_t tensor;
    };
    std::vector<Written> written;
    std::vector<Written> read;
    auto plan = std::make_unique<emh_adamw>();
    plan->ctx = c;
    size_t total = 0;
    for (size_t i = 0; i < count; i++) total += tensors[i].param ? tensors[i].param->len : 0;
    if (total <= emh::ADAM_FEW) plan->chunk = emh::ADAM_CHUNK_FEW;
    for (size_t i = 0; i < count; i++) {
      const emh_adamw_tensor& t = tensors[i];
      EMH_ENSURE(t.param && real_kind(t.param->kind), "tensor %zu: param must be f32, f16 or bf16", i);
      EMH_ENSURE(t.grad && real_kind(t.grad->kind), "tensor %zu: grad must be f32, f16 or bf16", i);
      EMH_ENSURE(t.m && t.v, "tensor %zu: null state", i);
      const size_t len = t.param->len;
      const bool eight = t.m->kind == EMH_F8;
      EMH_ENSURE(t.m->kind == t.v->kind && (eight || t.m->kind == EMH_F32),
                 "tensor %zu: m and v must both be f32 or both f8", i);
      EMH_ENSURE(t.grad->len == len && t.m->len == len && t.v->len == len,
                 "tensor %zu: grad, m and v must be as long as param (%zu)", i, len);
      EMH_ENSURE(std::isfinite(t.weight_decay), "tensor %zu: weight_decay must be finite", i);
      const size_t blocks = (len + EMH_ADAMW_BLOCK - 1) / EMH_ADAMW_BLOCK;
      EMH_ENSURE(eight == (t.m_scale != nullptr) && eight == (t.v_scale != nullptr),
                 "tensor %zu: 8-bit states come with both scales, 32-bit states with none", i);
      emh::AdamTensor a{};
      auto writes = [&](emh_buf* b, size_t n, const char* what) {
        written.push_back({check_vector(b, n, what), i});
        plan->written.push_back(b);
        return b->ptr;
      };
      a.param = writes(t.param, len, "param");
      a.param_kind = t.param->kind;
      read.push_back({check_vector(t.grad, len, "grad"), i});
      a.grad = t.grad->ptr;
      a.grad_kind = t.grad->kind;
      a.m = writes(t.m, len, "m");
      a.v = writes(t.v, len, "v");
      if (eight) {
        EMH_ENSURE(t.m_scale->kind == EMH_F32 && t.v_scale->kind == EMH_F32,
                   "tensor %zu: the scales must be f32", i);
        a.m_scale = (float*)writes(t.m_scale, blocks, "m_scale");
        a.v_scale = (float*)writes(t.v_scale, blocks, "v_scale");
      }
      if (t.copy) {
        EMH_ENSURE(t.copy->kind == EMH_F16 || t.copy->kind == EMH_BF16,
                   "tensor %zu: copy must be f16 or bf16", i);
        EMH_ENSURE(t.copy->len == len, "tensor %zu: copy must be as long as param", i);
        a.copy = writes(t.copy, len, "copy");
        a.copy_kind = t.copy->kind;
      }
      a.len = len;
      a.weight_decay = t.weight_decay;
      EMH_ENSURE(len < (size_t(1) << 41), "tensor %zu is too long", i);
      for (size_t k = 0; k * plan->chunk < len; k++)
        chunks.push_back(make_uint2((unsigned)table.size(), (unsigned)k));
      table.push_back(a);
    }
    EMH_ENSURE(chunks.size() < (size_t(1) << 24), "too many tensors or elements for one plan");
    // What is written is written once.
    std::sort(written.begin(), written.end(),
              [](const Written& a, const Written& b) { return a.r.lo < b.r.lo; });
    std::vector<Written> kept;  // not empty
    for (const Written& w : written)
      if (w.r.lo < w.r.hi) kept.push_back(w);
    for (const Written& w : kept) plan->ranges.push_back(w.r);
    for (size_t i = 1; i < kept.size(); i++)
      EMH_ENSURE(kept[i - 1].r.hi <= kept[i].r.lo,
                 "tensors %zu and %zu: two of what the step writes overlap", kept[i - 1].tensor,
                 kept[i].tensor);
    for (const Written& g : read) {
      if (g.r.lo == g.r.hi) continue;
      auto it = std::lower_bound(kept.begin(), kept.end(), g.r.hi,
                                 [](const Written& a, const char* hi) { return a.r.lo < hi; });
      EMH_ENSURE(it == kept.begin() || std::prev(it)->r.hi <= g.r.lo,
                 "tensor %zu: its gradient overlaps what the step writes", g.tensor);
    }
    use_device(c);
    plan->nchunks = chunks.size();
    if (!chunks.empty()) {
      try {
        EMH_HIP(hipMalloc(&plan->tensors, table.size() * sizeof table[0]));
        EMH_HIP(hipMalloc(&plan->chunks, chunks.size() * sizeof chunks[0]));
        EMH_HIP(hipMemcpyAsync(plan->tensors, table.data(), table.size() * sizeof table[0],
                               hipMemcpyHostToDevice, c->stream));
        EMH_HIP(hipMemcpyAsync(plan->chunks, chunks.data(), chunks.size() * sizeof chunks[0],
                               hipMemcpyHostToDevice, c->stream));
        EMH_HIP(hipStreamSynchronize(c->stream));  // the host's tables go away
      } catch (...) {
        free_tables(plan.get());
        throw;
      }
    }
    std::lock_guard<std::mutex> g(g_plans_mu);
    try {
      c->plans.push_back(plan.get());
    } catch (...) {
      free_tables(plan.get());
      throw;
    }
    *out = plan.release();
  });
}

int emh_adamw_set_seed(emh_adamw* plan, uint64_t seed) {
  return guard([&] {
    EMH_ENSURE(plan, "null argument");
    plan->random = true;
    plan->seed = seed;
  });
}

static int adamw_step(emh_adamw* plan, const emh_adamw_config* cfg, const emh_buf* clip,
                      bool clipped) {
  return guard([&] {
    EMH_ENSURE(plan && cfg, "null argument");
    EMH_ENSURE(plan->ctx, "the plan's context is destroyed");
    if (clipped) {
      const Range r = check_f32(clip, 2, "clip");
      for (const Range& w : plan->ranges) apart(w, r, "what the step writes", "clip");
    }
    EMH_ENSURE(cfg->step >= 1, "step counts from 1");
    EMH_ENSURE(cfg->beta1 >= 0 && cfg->beta1 < 1 && cfg->beta2 >= 0 && cfg->beta2 < 1,
               "beta1 and beta2 must be in [0, 1)");
    EMH_ENSURE(std::isfinite(cfg->lr) && std::isfinite(cfg->grad_scale), "lr and grad_scale must be finite");
    EMH_ENSURE(cfg->eps >= 0 && std::isfinite(cfg->eps), "eps must be finite and not negative");
    emh::AdamScalars s{};
    s.beta1 = (float)cfg->beta1;
    s.beta2 = (float)cfg->beta2;
    s.new1 = (float)(1.0 - cfg->beta1);
    s.new2 = (float)(1.0 - cfg->beta2);
    s.rate = (float)(cfg->lr / (1.0 - std::pow(cfg->beta1, (double)cfg->step)));
    s.root2 = (float)(1.0 / std::sqrt(1.0 - std::pow(cfg->beta2, (double)cfg->step)));
    s.eps = (float)cfg->eps;
    s.gscale = (float)cfg->grad_scale;
    s.lr = cfg->lr;
    uint64_t key = plan->seed * 0xD1342543DE82EF95u + cfg->step * 0x9E3779B97F4A7C15u +
                   0x632BE59BD9B4E019u;
    for (int i = 0; i < 2; i++) key = (key ^ key >> 32) * 0xD6E8FEB86659FD93u;
    key ^= key >> 32;
    s.key0 = (uint32_t)key;
    s.key1 = (uint32_t)(key >> 32);
    use_device(plan->ctx);
    for (emh_buf* b : plan->written) ++b->gen;
    emh::launch_adamw(plan->ctx, plan->tensors, plan->chunks, plan->nchunks, plan->chunk,
                      plan->random, s, clipped ? (const float*)clip->ptr : nullptr);
  });
}
int emh_adamw_step(emh_adamw* plan, const emh_adamw_config* cfg) {
  return adamw_step(plan, cfg, nullptr, false);
}
int emh_adamw_step_clipped(emh_adamw* plan, const emh_adamw_config* cfg, const emh_buf* clip) {
  return adamw_step(plan, cfg, clip, true);
}

int emh_adamw_destroy(emh_adamw* plan) {
  return guard([&] {
    if (!plan) return;
    std::unique_ptr<emh_adamw> hold(plan);
    std::lock_guard<std::mutex> g(g_plans_mu);
    if (!plan->ctx) return;  // its context went first, and the tables with it
    auto& plans = plan->ctx->plans;
    plans.erase(std::remove(plans.begin(), plans.end(), plan), plans.end());
    use_device(plan->ctx);
    const hipError_t e = hipStreamSynchronize(plan->ctx->stream);  // a queued step may read the tables
    free_tables(plan);
    EMH_HIP(e);
  });
}

}  // extern "C"

namespace emh {
void drop_plans(emh_ctx* c) {
  std::lock_guard<std::mutex> g(g_plans_mu);
  for (emh_adamw* p : c->plans) {
    free_tables(p);
    p->ctx = nullptr;
  }
  c->plans.clear();
}
}  // namespace emh
