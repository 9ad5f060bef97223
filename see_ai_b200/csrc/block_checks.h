// Workspaces and refusals of the operators that train a block's own weights.  Host-only (C++23).
#ifndef SEE_CUDA_BLOCK_CHECKS_H_
#define SEE_CUDA_BLOCK_CHECKS_H_

#include "operand_checks.h"
#include "plan_abi.h"

namespace see {
// Bytes for any shape of these sizes, whatever its types and alignment (0: sizes outside the range).
uint64_t NormBackwardWorkspace(uint64_t rows, uint64_t cols);
uint64_t GatedBackwardWorkspace(uint64_t rows, uint64_t d_in, uint64_t d_hidden);
uint64_t JoinBackwardWorkspace(uint64_t rows, uint64_t cols);
uint64_t GradWorkspace();
uint64_t PreferenceWorkspace(uint64_t rows, uint64_t pairs);
uint64_t PolicyWorkspace(uint64_t rows);
// What a call for these gradients uses of it on a device of `sms`.
uint64_t GatedBackwardUses(uint64_t rows, uint64_t d_in, uint64_t d_hidden, bool dx, bool dw, uint32_t sms);

// What see_cuda.h says a call refuses, without a device.  The shapes' strides of 0 are filled in.
Status CheckNormForward(see_norm_shape* shape, const void* x, const float* gamma, const float* beta, const void* y, const float* mean,
                        const float* rstd);
Status CheckNormBackward(see_norm_shape* shape, const void* dy, const void* x, const float* gamma, const float* mean, const float* rstd,
                         const void* addend, const void* dx, const float* dgamma, const float* dbeta, const void* workspace,
                         uint64_t workspace_bytes);
Status CheckGatedForward(see_gated_shape* shape, const void* x, const void* w_gate, const void* w_up, const void* hidden, const void* gate,
                         const void* up);
Status CheckGatedBackward(see_gated_shape* shape, const void* dhidden, const void* x, const void* w_gate, const void* w_up,
                          const void* gate, const void* up, const void* dx, const void* dw_gate, const void* dw_up, const void* workspace,
                          uint64_t workspace_bytes);
Status CheckAdamW(const see_adamw_tensor* tensors, uint64_t count, int state_bits, const StepParams& params, const float* grad_scale);
Status CheckJoinForward(see_join_shape* shape, const void* x, const void* block, const see_join_weights* weights, const void* x_out,
                        const void* y, const see_join_stats* stats);
Status CheckJoinBackward(see_join_shape* shape, const void* dy, const void* dx_out, const void* x_out, const void* block,
                         const see_join_weights* weights, const see_join_stats* stats, const void* dx, const void* dblock,
                         const see_join_weights* gradients, const void* workspace, uint64_t workspace_bytes);
Status CheckPreference(see_preference_shape* shape, const void* logits, const int32_t* labels, const int32_t* starts, const float* ref_logp,
                       const float* loss_grad, const float* loss, const float* margins, const float* sequence_logp, const void* dlogits,
                       const void* workspace, uint64_t workspace_bytes);
Status CheckPolicy(see_policy_shape* shape, const void* logits, const int32_t* labels, const float* old_logp, const float* ref_logp,
                   const float* advantages, const float* weights, const float* loss_grad, const float* loss, const float* logp,
                   const void* dlogits, const void* workspace, uint64_t workspace_bytes);
Status CheckGrad(const see_grad_tensor* tensors, uint64_t count, bool clip, float max_norm, const float* grad_scale, const float* norm,
                 const float* factor, const void* workspace, uint64_t workspace_bytes);
}  // namespace see

#endif  // SEE_CUDA_BLOCK_CHECKS_H_
