// Launchers of the operators that a classifier answers and is tuned with (RMS norm,
// 8-bit codes and their product, log probabilities, gradient norm), and the arguments that
// their entry points (emh_answer.cpp) have checked.
#pragma once

#include "emh_learn.h"

namespace emh {

// Bytes of results from which they go past the caches (which hold as many).
constexpr size_t STREAM_FROM = size_t(256) << 20;

// ---- emh_rms.hip
struct RmsArgs {
  const void* x;   // forward: the rows; backward: their sums h
  size_t ldx;
  const void* r;   // forward: what is added; backward: the gradient dh; or null
  size_t ldr;
  const void* dy;  // backward
  size_t lddy;
  size_t rows;
  int d, kind;
  const void* w;   // or null: ones
  int wkind;
  float eps;
  void* h;         // forward: the sums, or null
  size_t ldh;
  void* y;         // forward: the result; backward: dx, or null
  size_t ldy;
  float* scale;    // not null: y is codes
  size_t lds;
  float* rstd;     // forward: or null
  bool through;    // forward: h and y pass through the caches
  float* part;     // backward: [workgroup][d], or null
  void* dw;        // backward: dweight, where one workgroup has all of its sums; or null
  int dwkind;
};
void launch_rms_norm(emh_ctx* c, RmsArgs a);
void launch_rms_norm_grad(emh_ctx* c, RmsArgs a, const MatOut& dweight);
// Codes of x (rows x d), a scale for every `tall` rows (1 or CODE_BLOCK) by CODE_BLOCK columns.
void launch_quantize(emh_ctx* c, const MatIn& x, size_t rows, size_t d, bool tall, uint8_t* q,
                     size_t ldq, float* scale, size_t lds);

// ---- emh_product8.hip
struct CodedIn {  // codes whose rows begin at multiples of 16 bytes, and their scales
  const uint8_t* q;
  size_t ld;
  const float* scale;
  size_t lds;
};
void launch_product8(emh_ctx* c, const CodedIn& x, size_t n, size_t d, const CodedIn& w, size_t k,
                     const MatOut& y);

// ---- emh_logp.hip
struct LogpArgs {
  const void* z;
  size_t ldz, n, k;
  const uint32_t* tokens;  // or null
  float scale;
  float* logp;             // forward; each but lse may be null
  float* lse;
  float* entropy;
  uint32_t top;
  uint32_t* ids;
  float* tops;
  const float* lse_in;     // backward
  const float* entropy_in;
  const float* glogp;      // or null: zeros
  const float* gentropy;
  void* dz;
  size_t lddz;
  uint32_t* small;
};
constexpr uint32_t MAX_TOP = EMH_MAX_TOP;
void launch_log_probs(emh_ctx* c, LogpArgs a, int kind);
void launch_log_probs_grad(emh_ctx* c, LogpArgs a, int kind);

// ---- emh_gradnorm.hip
struct NormTensor {  // as the kernels read it
  const void* grad;
  void* out;
  uint64_t len;
  int kind, pad;
};
// Elements of a workgroup's share of one tensor: in a plan of few elements (NORM_FEW), as
// little as fills the GPU.
constexpr size_t NORM_CHUNK = 16384, NORM_CHUNK_FEW = 2048, NORM_FEW = size_t(4) << 20;
constexpr size_t NORM_SUMS = 1024;
// chunks[i]: a tensor and the number of a chunk in it. stream: results past the caches. sums:
// NORM_SUMS; out: the norm and the factor.
void launch_grad_norm(emh_ctx* c, const NormTensor* tensors, const uint2* chunks, size_t nchunks,
                      size_t chunk, bool stream, double* sums, float scale, float max_norm,
                      float* out, bool clip);

// No plan made with c measures any more, and what they hold on the device is freed (c's
// stream is idle).
void drop_norms(emh_ctx* c);

}  // namespace emh
