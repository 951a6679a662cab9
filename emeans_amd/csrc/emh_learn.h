// Launchers of the learning operators (layer norm, cross entropy, AdamW), and
// the arguments that their entry points (emh_learn.cpp) have checked.
#pragma once

#include <vector>

#include "emh_internal.h"

namespace emh {

// A row-major matrix or vector of a run-time kind.
struct MatIn {
  const void* p = nullptr;
  size_t ld = 0;
  int kind = EMH_F32;
};
struct MatOut {
  void* p = nullptr;
  size_t ld = 0;
  int kind = EMH_F32;
};

// A launch has fewer than 2^32 threads (more are cut off without an error): the most
// workgroups of 256 or 1,024 that a kernel whose work may exceed that is given, which
// strides over the rest.
constexpr size_t MAX_GROUPS = size_t(1) << 21;

// ---- emh_norm.hip
void launch_layer_norm(emh_ctx* c, const MatIn& x, size_t rows, size_t d, const MatIn& weight,
                       const MatIn& bias, float eps, const MatOut& y, float* mean, float* rstd);
void launch_layer_norm_grad(emh_ctx* c, const MatIn& dy, const MatIn& x, size_t rows, size_t d,
                            const MatIn& weight, const float* mean, const float* rstd,
                            const MatOut& dx, const MatOut& dweight, const MatOut& dbias);

// ---- emh_xent.hip
// Rows x (n x d) against classes w (k x d, x's kind); labels: n, NONE where a row
// has none.
struct XentIn {
  MatIn x, w;
  size_t n, d, k;
  const uint32_t* labels;
  float scale;
};
constexpr uint32_t NO_LABEL = 0xFFFFFFFFu;
void launch_cross_entropy(emh_ctx* c, const XentIn& in, float* loss, float* lse);
// gloss (n entries): the gradients of the rows' losses, or null: of their mean; all of
// loss_scale times it.
void launch_cross_entropy_grad(emh_ctx* c, const XentIn& in, const float* lse, const float* gloss,
                               float loss_scale, const MatOut& dx, const MatOut& dw);
// The tiled products that launch_cross_entropy_grad queues, in their order, for both
// gradients (host arithmetic alone).
std::vector<emh_xent_product> cross_entropy_products(size_t n, size_t d, size_t k, bool f32, int cus,
                                                     size_t workspace);

// ---- emh_adamw.hip
struct AdamTensor {  // as the kernel reads it
  void* param;
  const void* grad;
  void* m;
  void* v;
  float* m_scale;  // 8-bit states: not null
  float* v_scale;
  void* copy;
  uint64_t len;
  double weight_decay;
  int param_kind, grad_kind, copy_kind, pad;
};
struct AdamScalars {
  float beta1, beta2, new1, new2;  // new = 1 - beta
  float rate, root2, eps, gscale;  // lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t)
  double lr;
  uint32_t key0, key1;             // of a step whose 8-bit states are rounded at random
};
// Elements of a workgroup's share of one tensor: four loads of each array in
// flight a thread, or, in a plan of few elements, one, and four times the workgroups.
constexpr size_t ADAM_CHUNK = 4096, ADAM_CHUNK_FEW = 1024;
constexpr size_t ADAM_FEW = size_t(2) << 20;
// The plans made with c step no more, and what they hold on the device is freed (c's
// stream is idle).
void drop_plans(emh_ctx* c);
// chunks[i]: the tensor and the chunk in it that workgroup i takes. clip: a gradient norm's
// output, or null.
void launch_adamw(emh_ctx* c, const AdamTensor* tensors, const uint2* chunks, size_t nchunks,
                  size_t chunk, bool random, const AdamScalars& s, const float* clip);

}  // namespace emh
