// The operators that train a block's own weights: norm forward and backward with the weights' gradients, the gated
// feed-forward block, AdamW over many tensors.  Launchers enqueue on `stream` and return the launch's status; pointers
// are device pointers whose checks CudaBackend (block_ops.cc) has made.
#ifndef SEE_CUDA_BLOCK_OPS_H_
#define SEE_CUDA_BLOCK_OPS_H_

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "../../include/see_cuda.h"
#include "kernels.h"

namespace see::k {

// ---- norm (k_block_norm.cu) ------------------------------------------------
constexpr uint32_t kNormMaxCols = 16384;      // a row is held in the registers of one block
constexpr size_t kMostShared = 224 * 1024;   // bytes of shared memory that a block of these kernels asks for at most
constexpr uint32_t kNormPartials = 148;       // most rows of partial sums of the weights' gradients
struct NormArgs {
  const void *x = nullptr, *dy = nullptr, *addend = nullptr;
  const float *gamma = nullptr, *beta = nullptr;
  void *y = nullptr, *dx = nullptr;
  float *mean = nullptr, *rstd = nullptr;     // written by the forward pass, read by the backward pass
  float *dgamma = nullptr, *dbeta = nullptr;
  float* partials = nullptr;                  // [2][blocks][cols]
  uint64_t rows = 0, x_stride = 0, y_stride = 0;
  uint32_t cols = 0;
  int x_type = SEE_F32, y_type = SEE_F32;
  bool rms = false;
  float eps = 0.0f;
  DeviceStatus* status = nullptr;
};
inline uint64_t NormPartialRows(uint64_t rows) { return rows < kNormPartials ? rows : kNormPartials; }
cudaError_t NormForward(const NormArgs& a, uint32_t sms, cudaStream_t s);
cudaError_t NormBackward(const NormArgs& a, uint32_t sms, cudaStream_t s, int* launches);

// ---- AdamW (k_adamw.cu) ----------------------------------------------------
constexpr uint32_t kAdamBlock = SEE_ADAMW_BLOCK;
struct AdamStepScalars {
  float lr, beta1, beta2, om_beta1, om_beta2, eps, weight_decay, inv_bc1, inv_bc2, root_inv_bc2;
  uint32_t phase;   // the step's share of the rounding words
};
cudaError_t AdamWTensors(const see_adamw_tensor* tensors, uint64_t count, int state_bits, const AdamStepScalars& a,
                         const float* grad_scale, uint32_t sms, DeviceStatus* status, cudaStream_t s, int* launches);

// ---- a block's join to the residual stream (k_join.cu) -------------------------
struct JoinArgs {
  const void *x = nullptr, *block = nullptr;   // x: of the backward pass, what the forward pass made of it
  void *x_out = nullptr, *y = nullptr;
  const void *dy = nullptr, *dx_out = nullptr;
  void *dx = nullptr, *dblock = nullptr;
  see_join_weights w = {}, grads = {};
  see_join_stats stats = {};
  float* partials = nullptr;                   // [4][blocks][cols]
  uint64_t rows = 0, x_stride = 0, y_stride = 0;
  uint32_t cols = 0;
  int x_type = SEE_F32, y_type = SEE_F32;
  bool rms = false;
  float eps = 0.0f, scale = 1.0f;
  DeviceStatus* status = nullptr;
};
cudaError_t Join(const JoinArgs& a, bool backward, uint32_t sms, cudaStream_t s, int* launches);

// ---- losses over rows of logits (k_logit_loss.cu) ------------------------------
constexpr uint32_t kPolicyPartials = 592;     // most thread blocks' sums
struct LogitArgs {
  const void* logits;
  void* dlogits;                              // or null
  const int32_t* labels;
  uint64_t rows, stride;
  uint32_t classes;
  float scale, k, k_rest;                     // k: scale / ln 2; k_rest: what its rounding leaves, above 0 (of the policy loss: next to nothing)
  float k_up;                                 // the next power of two from k on
  double inv_k;
  DeviceStatus* status;
};
struct PolicyArgs {
  const float *old_logp, *ref_logp, *advantages, *weights, *loss_grad;
  float *loss, *logp;
  float clip_low, clip_high, kl_coef;
};
struct PreferenceArgs {
  const int32_t* starts;
  const float *ref_logp, *loss_grad;
  float *loss, *margins, *sequence_logp;
  double* losses;                             // [pairs]
  uint32_t pairs;
  int kind, average;
  float beta, smoothing, margin;
};
// kept [rows], and behind it, of the policy loss, [kPolicyPartials][3] doubles and 16 bytes.
cudaError_t PolicyLoss(const LogitArgs& a, int type, const PolicyArgs& p, float4* kept, uint32_t sms, cudaStream_t s, int* launches);
cudaError_t PreferenceLoss(const LogitArgs& a, int type, const PreferenceArgs& p, float4* kept, uint32_t sms, cudaStream_t s, int* launches);

// ---- all gradients' norm (k_grad_norm.cu) ------------------------------------
// clip: writes the tensors' out too.  partials [kGradPartials] (grad_table.h).
cudaError_t GradNorm(const see_grad_tensor* tensors, uint64_t count, bool clip, float max_norm, const float* grad_scale, float* norm,
                     float* factor, double* partials, uint32_t sms, cudaStream_t s, int* launches);

}  // namespace see::k

#endif  // SEE_CUDA_BLOCK_OPS_H_
