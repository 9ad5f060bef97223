// The checks of the norm over all gradients, and its dispatch.
#include <algorithm>
#include <vector>

#include "block_checks.h"
#include "block_ops.h"
#include "cuda_backend.h"
#include "grad_table.h"

namespace see {

uint64_t GradWorkspace() { return k::kGradPartials * sizeof(double); }

Status CheckGrad(const see_grad_tensor* tensors, uint64_t count, bool clip, float max_norm, const float* grad_scale, const float* norm,
                 const float* factor, const void* workspace, uint64_t workspace_bytes) {
  const char* const what = clip ? "cuda: grad clip" : "cuda: grad norm";
  if (!(max_norm > 0.0f)) return std::unexpected(std::string(what) + ": max_norm is not above 0");
  if (count && !tensors) return std::unexpected(std::string(what) + ": tensors is null");
  if (workspace_bytes < GradWorkspace()) return std::unexpected(std::string(what) + ": the workspace is too small");
  Operands ops = {Vector("norm", norm, 4, 4, true), Vector("factor", factor, 4, 4, true), Vector("workspace", workspace, workspace_bytes, 16, true)};
  if (grad_scale) ops.Add(Vector("grad_scale", grad_scale, 4, 4, false));
  if (auto r = ops.Check(what); !r) return r;
  // Tensors mostly ascend; only where they do not, or meet what else there is, is everything sorted.
  struct Span { uint64_t begin, end; bool written; };
  const Span small[4] = {{reinterpret_cast<uint64_t>(norm), reinterpret_cast<uint64_t>(norm) + 4, true},
                         {reinterpret_cast<uint64_t>(factor), reinterpret_cast<uint64_t>(factor) + 4, true},
                         {reinterpret_cast<uint64_t>(workspace), reinterpret_cast<uint64_t>(workspace) + workspace_bytes, true},
                         {reinterpret_cast<uint64_t>(grad_scale), reinterpret_cast<uint64_t>(grad_scale) + (grad_scale ? 4 : 0), false}};
  Span g = {~0ull, 0, false}, out = {~0ull, 0, true};
  bool plain = true;   // ascending, the ranges apart
  for (uint64_t i = 0; i < count; ++i) {
    const see_grad_tensor& t = tensors[i];
    auto refuse = [&](const char* why) { return std::unexpected(std::string(what) + ": tensor " + std::to_string(i) + ": " + why); };
    if (!IsType(t.type)) return refuse("unknown type");
    if (t.n == 0) continue;
    if (t.n > (1ull << 38)) return refuse("more than 2^38 elements");
    const uint64_t size = SizeOfType(t.type), at = reinterpret_cast<uint64_t>(t.g), to = reinterpret_cast<uint64_t>(t.out);
    if (!at) return refuse("g is null");
    if (at % size) return refuse("g is not aligned");
    if (at > (1ull << 57) || (clip && to > (1ull << 57))) return refuse("an address is too large");
    plain = plain && at >= g.end;
    g = {std::min(g.begin, at), std::max(g.end, at + t.n * size), false};
    if (!clip || !to || to == at) continue;
    if (to % size) return refuse("out is not aligned");
    plain = plain && to >= out.end;
    out = {std::min(out.begin, to), std::max(out.end, to + t.n * size), true};
  }
  auto meet = [](const Span& a, const Span& b) { return a.begin < b.end && b.begin < a.end; };
  for (const Span& s : small) plain = plain && !meet(s, g) && !meet(s, out);
  if (plain && !meet(g, out)) return {};
  std::vector<Span> all;
  all.reserve(2 * count + 4);
  for (const Span& s : small)
    if (s.end != s.begin) all.push_back(s);
  for (uint64_t i = 0; i < count; ++i) {
    const see_grad_tensor& t = tensors[i];
    if (t.n == 0) continue;
    const uint64_t bytes = t.n * SizeOfType(t.type), at = reinterpret_cast<uint64_t>(t.g), to = reinterpret_cast<uint64_t>(t.out);
    const bool in_place = clip && (!to || to == at);
    all.push_back({at, at + bytes, in_place});
    if (clip && !in_place) all.push_back({to, to + bytes, true});
  }
  std::sort(all.begin(), all.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
  uint64_t any = 0, written = 0;   // how far the spans so far reach
  for (const Span& s : all) {
    if (s.begin < written || (s.written && s.begin < any)) return std::unexpected(std::string(what) + ": operands overlap");
    any = std::max(any, s.end);
    if (s.written) written = std::max(written, s.end);
  }
  return {};
}

Status CudaBackend::GradNorm(const see_grad_tensor* tensors, uint64_t count, bool clip, float max_norm, const float* grad_scale, float* norm,
                             float* factor, void* workspace, uint64_t workspace_bytes) {
  if (auto r = CheckGrad(tensors, count, clip, max_norm, grad_scale, norm, factor, workspace, workspace_bytes); !r) return r;
  const char* const what = clip ? "grad clip" : "grad norm";
  OnDevice on(device_);
  if (!on.ok()) return Check(cudaGetLastError(), "grad norm: device");
  int launches = 0;
  const cudaError_t e = k::GradNorm(tensors, count, clip, max_norm, grad_scale, norm, factor, static_cast<double*>(workspace), sms_, stream_, &launches);
  counters_.kernel_launches += static_cast<uint64_t>(launches);
  return Check(e, what);
}

}  // namespace see
