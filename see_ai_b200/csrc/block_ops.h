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

}  // namespace see::k

#endif  // SEE_CUDA_BLOCK_OPS_H_
