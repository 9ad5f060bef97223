// The checks of the losses over rows of logits, and their dispatch.
#include <algorithm>
#include <cmath>
#include <limits>

#include "block_checks.h"
#include "block_ops.h"
#include "cuda_backend.h"

namespace see {
namespace {

constexpr double kLog2E = 1.4426950408889634;

template <typename Shape>
Status CheckLogits(const std::string& what, Shape* s) {
  if (!IsType(s->type)) return std::unexpected(what + ": unknown type");
  // (logit_scale / ln 2, the power of two above it and what its rounding leaves are f32's)
  if (!(s->logit_scale >= 0x1p-100f && s->logit_scale <= 0x1p100f)) return std::unexpected(what + ": logit_scale is not from 2^-100 to 2^100");
  if (s->classes == 0 || s->classes > (1u << 20)) return std::unexpected(what + ": 1 to 2^20 classes");
  if (s->rows > 0x7FFFFFFFull) return std::unexpected(what + ": more than 2^31 - 1 rows");
  if (s->stride == 0) s->stride = s->classes;
  if (s->stride < s->classes || s->stride > (1ull << 40)) return std::unexpected(what + ": the stride is smaller than a row, or over 2^40");
  return {};
}

template <typename Shape>
Operand Logits(const char* name, const Shape& s, const void* p, bool written) {
  const uint64_t size = SizeOfType(s.type);
  return {name, p, s.rows, s.classes * size, s.stride * size, size, written};
}

// whole: with what k's rounding leaves (a preference loss's).
template <typename Shape>
k::LogitArgs ArgsOf(const Shape& s, const void* logits, const int32_t* labels, void* dlogits, bool whole, k::DeviceStatus* status) {
  const double exact = kLog2E * static_cast<double>(s.logit_scale);
  float k = static_cast<float>(exact);
  if (whole && static_cast<double>(k) > exact) k = std::nextafter(k, 0.0f);
  const float rest = whole ? static_cast<float>(exact - static_cast<double>(k)) : 0.0f;
  int exponent;
  const bool power = std::frexp(k, &exponent) == 0.5f;
  const float up = std::ldexp(1.0f, power ? exponent - 1 : exponent);
  return {logits, s.rows ? dlogits : nullptr, labels, s.rows, s.stride, static_cast<uint32_t>(s.classes), s.logit_scale, k,
          std::max(rest, std::numeric_limits<float>::denorm_min()), up, 1.0 / (whole ? exact : static_cast<double>(k)), status};
}

}  // namespace

uint64_t PreferenceWorkspace(uint64_t rows, uint64_t pairs) {   // what is kept of a row, and each pair's loss
  return rows > 0x7FFFFFFFull || pairs == 0 || pairs > (1u << 24) ? 0 : rows * 16 + (pairs * 8 + 15) / 16 * 16;
}
uint64_t PolicyWorkspace(uint64_t rows) { return rows > 0x7FFFFFFFull ? 0 : rows * 16 + k::kPolicyPartials * 3 * sizeof(double) + 16; }

Status CheckPreference(see_preference_shape* shape, const void* logits, const int32_t* labels, const int32_t* starts, const float* ref_logp,
                       const float* loss_grad, const float* loss, const float* margins, const float* sequence_logp, const void* dlogits,
                       const void* workspace, uint64_t workspace_bytes) {
  const char* const what = "cuda: preference loss";
  auto refuse = [what](const char* why) { return std::unexpected(std::string(what) + ": " + why); };
  if (auto r = CheckLogits(what, shape); !r) return r;
  const see_preference_shape& s = *shape;
  if (s.kind != SEE_PREFERENCE_SIGMOID && s.kind != SEE_PREFERENCE_HINGE && s.kind != SEE_PREFERENCE_SQUARE) return refuse("unknown kind");
  if (s.pairs == 0 || s.pairs > (1u << 24)) return refuse("1 to 2^24 pairs");
  if (!(s.beta > 0.0f) || !std::isfinite(s.beta)) return refuse("beta is not a finite number above 0");
  if (!(s.smoothing >= 0.0f && s.smoothing < 0.5f)) return refuse("smoothing is from 0 on and below 1/2");
  if (s.smoothing != 0.0f && s.kind != SEE_PREFERENCE_SIGMOID) return refuse("smoothing belongs to the sigmoid");
  if (!std::isfinite(s.margin)) return refuse("margin is not finite");
  if (s.margin != 0.0f && s.kind == SEE_PREFERENCE_SQUARE) return refuse("the square has no margin");
  if (workspace_bytes < PreferenceWorkspace(s.rows, s.pairs)) return refuse("the workspace is too small");
  const bool in_place = dlogits && dlogits == logits;
  Operands ops = {Logits("logits", s, logits, in_place),
                  Vector("labels", labels, s.rows * 4, 4, false),
                  Vector("starts", starts, (2 * s.pairs + 1) * 4, 4, false),
                  Vector("loss", loss, 4, 4, true),
                  Vector("margins", margins, s.pairs * 4, 4, true),
                  Vector("sequence_logp", sequence_logp, s.pairs * 8, 4, true),
                  Vector("workspace", workspace, workspace_bytes, 16, true)};
  if (ref_logp) ops.Add(Vector("ref_logp", ref_logp, s.pairs * 8, 4, false));
  if (loss_grad) ops.Add(Vector("loss_grad", loss_grad, 4, 4, false));
  if (dlogits && !in_place) ops.Add(Logits("dlogits", s, dlogits, true));
  return ops.Check(what);
}

Status CudaBackend::PreferenceLoss(const see_preference_shape& given, const void* logits, const int32_t* labels, const int32_t* starts,
                                   const float* ref_logp, const float* loss_grad, float* loss, float* margins, float* sequence_logp,
                                   void* dlogits, void* workspace, uint64_t workspace_bytes) {
  see_preference_shape s = given;
  if (auto r = CheckPreference(&s, logits, labels, starts, ref_logp, loss_grad, loss, margins, sequence_logp, dlogits, workspace, workspace_bytes);
      !r)
    return r;
  float4* kept = static_cast<float4*>(workspace);
  const k::PreferenceArgs p = {starts, ref_logp, loss_grad, loss, margins, sequence_logp, reinterpret_cast<double*>(kept + s.rows),
                               static_cast<uint32_t>(s.pairs), s.kind, s.average, s.beta, s.smoothing, s.margin};
  OnDevice on(device_);
  if (!on.ok()) return Check(cudaGetLastError(), "preference loss: device");
  int launches = 0;
  const cudaError_t e = k::PreferenceLoss(ArgsOf(s, logits, labels, dlogits, true, d_status_), s.type, p, kept, sms_, stream_, &launches);
  counters_.kernel_launches += static_cast<uint64_t>(launches);
  return Check(e, "preference loss");
}

Status CheckPolicy(see_policy_shape* shape, const void* logits, const int32_t* labels, const float* old_logp, const float* ref_logp,
                   const float* advantages, const float* weights, const float* loss_grad, const float* loss, const float* logp,
                   const void* dlogits, const void* workspace, uint64_t workspace_bytes) {
  const char* const what = "cuda: policy loss";
  auto refuse = [what](const char* why) { return std::unexpected(std::string(what) + ": " + why); };
  if (auto r = CheckLogits(what, shape); !r) return r;
  const see_policy_shape& s = *shape;
  if (!(s.clip_low >= 0.0f && s.clip_low <= 1.0f)) return refuse("clip_low is from 0 to 1");
  if (!(s.clip_high >= 0.0f) || !std::isfinite(s.clip_high)) return refuse("clip_high is not a finite number from 0 on");
  if (!(s.kl_coef >= 0.0f) || !std::isfinite(s.kl_coef)) return refuse("kl_coef is not a finite number from 0 on");
  if (s.kl_coef != 0.0f && !ref_logp && s.rows) return refuse("a KL term needs ref_logp");
  if (workspace_bytes < PolicyWorkspace(s.rows)) return refuse("the workspace is too small");
  const bool in_place = dlogits && dlogits == logits;
  Operands ops = {Logits("logits", s, logits, in_place),
                  Vector("labels", labels, s.rows * 4, 4, false),
                  Vector("old_logp", old_logp, s.rows * 4, 4, false),
                  Vector("advantages", advantages, s.rows * 4, 4, false),
                  Vector("loss", loss, 12, 4, true),
                  Vector("logp", logp, s.rows * 4, 4, true),
                  Vector("workspace", workspace, workspace_bytes, 16, true)};
  if (ref_logp) ops.Add(Vector("ref_logp", ref_logp, s.rows * 4, 4, false));
  if (weights) ops.Add(Vector("weights", weights, s.rows * 4, 4, false));
  if (loss_grad) ops.Add(Vector("loss_grad", loss_grad, 4, 4, false));
  if (dlogits && !in_place) ops.Add(Logits("dlogits", s, dlogits, true));
  return ops.Check(what);
}

Status CudaBackend::PolicyLoss(const see_policy_shape& given, const void* logits, const int32_t* labels, const float* old_logp,
                               const float* ref_logp, const float* advantages, const float* weights, const float* loss_grad, float* loss,
                               float* logp, void* dlogits, void* workspace, uint64_t workspace_bytes) {
  see_policy_shape s = given;
  if (auto r = CheckPolicy(&s, logits, labels, old_logp, ref_logp, advantages, weights, loss_grad, loss, logp, dlogits, workspace,
                           workspace_bytes);
      !r)
    return r;
  const k::PolicyArgs p = {old_logp, ref_logp, advantages, weights, loss_grad, loss, logp, s.clip_low, s.clip_high, s.kl_coef};
  OnDevice on(device_);
  if (!on.ok()) return Check(cudaGetLastError(), "policy loss: device");
  int launches = 0;
  const cudaError_t e =
      k::PolicyLoss(ArgsOf(s, logits, labels, dlogits, false, d_status_), s.type, p, static_cast<float4*>(workspace), sms_, stream_, &launches);
  counters_.kernel_launches += static_cast<uint64_t>(launches);
  return Check(e, "policy loss");
}

}  // namespace see
