// The checks of the operators that train a block's own weights, and their dispatch: what see_cuda.h promises to refuse is
// refused here, before anything is enqueued.
#include "block_ops.h"

#include <algorithm>
#include <cmath>
#include <vector>

#include "block_checks.h"
#include "cuda_backend.h"

namespace see {
namespace {

// Shape checks common to both directions; fills the strides.
Status CheckNorm(const char* what, see_norm_shape* s) {
  if (s->kind != SEE_NORM_LAYER && s->kind != SEE_NORM_RMS) return std::unexpected(std::string(what) + ": unknown kind");
  if (!IsType(s->x_type) || !IsType(s->y_type) || (s->x_type != s->y_type && s->x_type != SEE_F32))
    return std::unexpected(std::string(what) + ": x_type and y_type are equal, or x_type is f32");
  if (!(s->eps >= 0.0f) || !std::isfinite(s->eps)) return std::unexpected(std::string(what) + ": eps is not a finite number from 0 on");
  if (s->cols == 0 || s->cols > k::kNormMaxCols) return std::unexpected(std::string(what) + ": 1 to 16384 columns");
  if (s->rows > 0x7FFFFFFFull) return std::unexpected(std::string(what) + ": more than 2^31 - 1 rows");
  if (s->x_stride == 0) s->x_stride = s->cols;
  if (s->y_stride == 0) s->y_stride = s->cols;
  if (s->x_stride < s->cols || s->y_stride < s->cols || s->x_stride > (1ull << 40) || s->y_stride > (1ull << 40))
    return std::unexpected(std::string(what) + ": a stride is smaller than a row, or over 2^40");
  return {};
}

k::NormArgs ArgsOf(const see_norm_shape& s) {
  k::NormArgs a;
  a.rows = s.rows;
  a.cols = static_cast<uint32_t>(s.cols);
  a.x_stride = s.x_stride;
  a.y_stride = s.y_stride;
  a.x_type = s.x_type;
  a.y_type = s.y_type;
  a.rms = s.kind == SEE_NORM_RMS;
  a.eps = s.eps;
  return a;
}

}  // namespace

uint64_t NormBackwardWorkspace(uint64_t rows, uint64_t cols) {
  if (cols == 0 || cols > k::kNormMaxCols) return 0;
  return std::max<uint64_t>(16, k::NormPartialRows(rows) * cols * 2 * sizeof(float));
}

Status CheckNormForward(see_norm_shape* shape, const void* x, const float* gamma, const float* beta, const void* y, const float* mean,
                        const float* rstd) {
  const char* const what = "cuda: norm forward";
  if (auto r = CheckNorm(what, shape); !r) return r;
  const see_norm_shape& s = *shape;
  const bool layer = s.kind == SEE_NORM_LAYER;
  if (!layer && (beta || mean)) return std::unexpected(std::string(what) + ": rms has neither beta nor mean");
  const uint64_t xs = SizeOfType(s.x_type), ys = SizeOfType(s.y_type);
  Operands ops = {{"x", x, s.rows, s.cols * xs, s.x_stride * xs, xs, false},
                              {"y", y, s.rows, s.cols * ys, s.y_stride * ys, ys, true},
                              Vector("gamma", gamma, s.cols * 4, 4, false),
                              Vector("rstd", rstd, s.rows * 4, 4, true)};
  if (layer) {
    ops.Add(Vector("beta", beta, s.cols * 4, 4, false));
    ops.Add(Vector("mean", mean, s.rows * 4, 4, true));
  }
  return ops.Check(what);
}

Status CudaBackend::NormForward(const see_norm_shape& given, const void* x, const float* gamma, const float* beta, void* y, float* mean,
                                float* rstd) {
  see_norm_shape s = given;
  if (auto r = CheckNormForward(&s, x, gamma, beta, y, mean, rstd); !r) return r;
  if (s.rows == 0) return {};
  k::NormArgs a = ArgsOf(s);
  a.x = x;
  a.gamma = gamma;
  a.beta = beta;
  a.y = y;
  a.mean = mean;
  a.rstd = rstd;
  a.status = d_status_;
  OnDevice on(device_);
  if (!on.ok()) return Check(cudaGetLastError(), "norm forward: device");
  if (auto r = Check(k::NormForward(a, sms_, stream_), "norm forward"); !r) return r;
  ++counters_.kernel_launches;
  return {};
}

Status CheckNormBackward(see_norm_shape* shape, const void* dy, const void* x, const float* gamma, const float* mean, const float* rstd,
                         const void* addend, const void* dx, const float* dgamma, const float* dbeta, const void* workspace,
                         uint64_t workspace_bytes) {
  const char* const what = "cuda: norm backward";
  if (auto r = CheckNorm(what, shape); !r) return r;
  const see_norm_shape& s = *shape;
  const bool layer = s.kind == SEE_NORM_LAYER;
  if (!layer && (dbeta || mean)) return std::unexpected(std::string(what) + ": rms has neither mean nor dbeta");
  if (workspace_bytes < NormBackwardWorkspace(s.rows, s.cols)) return std::unexpected(std::string(what) + ": the workspace is too small");
  const uint64_t xs = SizeOfType(s.x_type), ys = SizeOfType(s.y_type);
  Operands ops = {{"dy", dy, s.rows, s.cols * ys, s.y_stride * ys, ys, false},
                              {"x", x, s.rows, s.cols * xs, s.x_stride * xs, xs, false},
                              {"dx", dx, s.rows, s.cols * xs, s.x_stride * xs, xs, true},
                              Vector("gamma", gamma, s.cols * 4, 4, false),
                              Vector("rstd", rstd, s.rows * 4, 4, false),
                              Vector("dgamma", dgamma, s.cols * 4, 4, true),
                              Vector("workspace", workspace, workspace_bytes, 16, true)};
  if (addend) ops.Add({"addend", addend, s.rows, s.cols * xs, s.x_stride * xs, xs, false});
  if (layer) {
    ops.Add(Vector("mean", mean, s.rows * 4, 4, false));
    ops.Add(Vector("dbeta", dbeta, s.cols * 4, 4, true));
  }
  return ops.Check(what);
}

Status CudaBackend::NormBackward(const see_norm_shape& given, const void* dy, const void* x, const float* gamma, const float* mean,
                                 const float* rstd, const void* addend, void* dx, float* dgamma, float* dbeta, void* workspace,
                                 uint64_t workspace_bytes) {
  see_norm_shape s = given;
  if (auto r = CheckNormBackward(&s, dy, x, gamma, mean, rstd, addend, dx, dgamma, dbeta, workspace, workspace_bytes); !r) return r;
  const bool layer = s.kind == SEE_NORM_LAYER;
  OnDevice on(device_);
  if (!on.ok()) return Check(cudaGetLastError(), "norm backward: device");
  if (s.rows == 0) {
    if (auto r = Check(cudaMemsetAsync(dgamma, 0, s.cols * 4, stream_), "norm backward"); !r) return r;
    return layer ? Check(cudaMemsetAsync(dbeta, 0, s.cols * 4, stream_), "norm backward") : Status{};
  }
  k::NormArgs a = ArgsOf(s);
  a.x = x;
  a.dy = dy;
  a.addend = addend;
  a.gamma = gamma;
  a.mean = const_cast<float*>(mean);
  a.rstd = const_cast<float*>(rstd);
  a.dx = dx;
  a.dgamma = dgamma;
  a.dbeta = dbeta;
  a.partials = static_cast<float*>(workspace);
  a.status = d_status_;
  int launches = 0;
  const cudaError_t e = k::NormBackward(a, sms_, stream_, &launches);
  counters_.kernel_launches += static_cast<uint64_t>(launches);
  return Check(e, "norm backward");
}

Status CheckAdamW(const see_adamw_tensor* tensors, uint64_t count, int state_bits, const StepParams& params, const float* grad_scale) {
  const char* const what = "cuda: adamw";
  if (state_bits != 8 && state_bits != 32) return std::unexpected(std::string(what) + ": moments have 8 or 32 bits");
  if (params.step == 0) return std::unexpected(std::string(what) + ": steps count from 1");
  if (!(params.beta1 >= 0.0f && params.beta1 < 1.0f && params.beta2 >= 0.0f && params.beta2 < 1.0f))
    return std::unexpected(std::string(what) + ": beta1 and beta2 are from 0 on and below 1");
  if (count && !tensors) return std::unexpected(std::string(what) + ": tensors is null");
  if (reinterpret_cast<uint64_t>(grad_scale) % 4) return std::unexpected(std::string(what) + ": grad_scale is not aligned");
  // Seven operands a tensor.  Lists of tensors mostly follow the layout of a few buffers, so each operand's spans are tried in
  // the list's order first; only where they do not ascend, or two operands' ranges meet, is everything sorted.
  struct Span { uint64_t begin, end; };
  constexpr size_t kOperands = 7;
  static constexpr const char* kNames[kOperands] = {"p", "g", "m", "v", "m_scale", "v_scale", "copy"};
  const uint64_t state = static_cast<uint64_t>(state_bits) / 8;
  auto spans_of = [&](const see_adamw_tensor& t, Span (&out)[kOperands]) {
    const uint64_t scales = state == 1 ? (t.n + k::kAdamBlock - 1) / k::kAdamBlock * 4 : 0;
    const void* p[kOperands] = {t.p, t.g, t.m, t.v, t.m_scale, t.v_scale, t.copy};
    const uint64_t bytes[kOperands] = {t.n * 4, t.n * SizeOfType(t.g_type), t.n * state, t.n * state, scales, scales, t.copy ? t.n * 2 : 0};
    for (size_t o = 0; o < kOperands; ++o) out[o] = {reinterpret_cast<uint64_t>(p[o]), reinterpret_cast<uint64_t>(p[o]) + bytes[o]};
  };
  Span range[kOperands + 1];
  for (Span& r : range) r = {~0ull, 0};
  bool ascending = true;
  for (uint64_t i = 0; i < count; ++i) {
    const see_adamw_tensor& t = tensors[i];
    auto refuse = [&](const std::string& why) { return std::unexpected(std::string(what) + ": tensor " + std::to_string(i) + ": " + why); };
    if (!IsType(t.g_type) || !IsType(t.copy_type)) return refuse("unknown type");
    if (t.flags & ~static_cast<uint32_t>(SEE_ADAMW_NO_DECAY)) return refuse("unknown flag");
    if (t.n == 0) continue;   // (empty allocations have no address, the copy's neither)
    if ((t.copy_type == SEE_F32) != (t.copy == nullptr)) return refuse("a copy has 16 bits, and none is null with type f32");
    if (t.n > (1ull << 38)) return refuse("more than 2^38 elements");
    const uint64_t align[kOperands] = {4, SizeOfType(t.g_type), state, state, 4, 4, 2};
    Span spans[kOperands];
    spans_of(t, spans);
    for (size_t o = 0; o < kOperands; ++o) {
      if (spans[o].begin == spans[o].end) continue;
      if (!spans[o].begin) return refuse(std::string(kNames[o]) + " is null");
      if (spans[o].begin % align[o]) return refuse(std::string(kNames[o]) + " is not aligned");
      ascending = ascending && (range[o].end == 0 || spans[o].begin >= range[o].end);
      range[o] = {std::min(range[o].begin, spans[o].begin), std::max(range[o].end, spans[o].end)};
    }
  }
  if (grad_scale) range[kOperands] = {reinterpret_cast<uint64_t>(grad_scale), reinterpret_cast<uint64_t>(grad_scale) + 4};
  for (size_t i = 0; i <= kOperands && ascending; ++i)
    for (size_t j = i + 1; j <= kOperands; ++j)
      if (range[i].end && range[j].end && range[i].begin < range[j].end && range[j].begin < range[i].end) ascending = false;
  if (ascending) return {};
  struct Sorted { Span span; bool written; };
  std::vector<Sorted> all;
  all.reserve(count * kOperands + 1);
  for (uint64_t i = 0; i < count; ++i) {
    if (tensors[i].n == 0) continue;
    Span spans[kOperands];
    spans_of(tensors[i], spans);
    for (size_t o = 0; o < kOperands; ++o)
      if (spans[o].begin != spans[o].end) all.push_back({spans[o], o != 1});
  }
  if (grad_scale) all.push_back({range[kOperands], false});
  std::sort(all.begin(), all.end(), [](const Sorted& a, const Sorted& b) { return a.span.begin < b.span.begin; });
  uint64_t any = 0, written = 0;   // how far the spans so far reach
  for (const Sorted& s : all) {
    if (s.span.begin < written || (s.written && s.span.begin < any)) return std::unexpected(std::string(what) + ": operands overlap");
    any = std::max(any, s.span.end);
    if (s.written) written = std::max(written, s.span.end);
  }
  return {};
}

Status CudaBackend::AdamWTensors(const see_adamw_tensor* tensors, uint64_t count, int state_bits, const StepParams& params,
                                 const float* grad_scale) {
  if (auto r = CheckAdamW(tensors, count, state_bits, params, grad_scale); !r) return r;
  const k::AdamScalars sc = ScalarsOf(params);
  k::AdamStepScalars a;
  a.lr = sc.lr;
  a.beta1 = sc.beta1;
  a.beta2 = sc.beta2;
  a.om_beta1 = 1.0f - sc.beta1;
  a.om_beta2 = 1.0f - sc.beta2;
  a.eps = sc.eps;
  a.weight_decay = sc.weight_decay;
  a.inv_bc1 = sc.inv_bc1;
  a.inv_bc2 = sc.inv_bc2;
  a.root_inv_bc2 = std::sqrt(sc.inv_bc2);
  a.phase = static_cast<uint32_t>(params.step) * 0x6A09E667u;   // 2^32 (sqrt(2) - 1)
  OnDevice on(device_);
  if (!on.ok()) return Check(cudaGetLastError(), "adamw: device");
  int launches = 0;
  const cudaError_t e = k::AdamWTensors(tensors, count, state_bits, a, grad_scale, sms_, d_status_, stream_, &launches);
  counters_.kernel_launches += static_cast<uint64_t>(launches);
  return Check(e, "adamw");
}

}  // namespace see
