// The checks of a block's join to the residual stream, and its dispatch.
#include <algorithm>
#include <cmath>

#include "block_checks.h"
#include "block_ops.h"
#include "cuda_backend.h"

namespace see {
namespace {

std::unexpected<std::string> Refuse(const char* what, const char* why) { return std::unexpected(std::string(what) + ": " + why); }

// What both directions share; fills the strides.
Status CheckJoin(const char* what, see_join_shape* s, const see_join_weights* w, const see_join_stats* stats) {
  if (s->kind != SEE_NORM_LAYER && s->kind != SEE_NORM_RMS) return Refuse(what, "unknown kind");
  if (!IsType(s->x_type) || !IsType(s->y_type) || (s->x_type != s->y_type && s->x_type != SEE_F32))
    return Refuse(what, "x_type and y_type are equal, or x_type is f32");
  if (!(s->eps >= 0.0f) || !std::isfinite(s->eps)) return Refuse(what, "eps is not a finite number from 0 on");
  if (!std::isfinite(s->residual_scale)) return Refuse(what, "residual_scale is not finite");
  if (s->cols == 0 || s->cols > k::kNormMaxCols) return Refuse(what, "1 to 16384 columns");
  if (s->rows > 0x7FFFFFFFull) return Refuse(what, "more than 2^31 - 1 rows");
  if (s->x_stride == 0) s->x_stride = s->cols;
  if (s->y_stride == 0) s->y_stride = s->cols;
  if (s->x_stride < s->cols || s->y_stride < s->cols || s->x_stride > (1ull << 40) || s->y_stride > (1ull << 40))
    return Refuse(what, "a stride is smaller than a row, or over 2^40");
  if (!w) return Refuse(what, "weights is null");
  if (!stats) return Refuse(what, "stats is null");
  if (s->kind == SEE_NORM_RMS && (w->post_beta || w->pre_beta || stats->post_mean || stats->pre_mean))
    return Refuse(what, "rms has neither beta nor mean");
  if (!w->post_gamma && (w->post_beta || stats->post_mean || stats->post_rstd)) return Refuse(what, "post_beta and post's stats go with post_gamma");
  return {};
}

void AddStats(Operands* ops, const see_join_shape& s, const see_join_weights& w, const see_join_stats& stats, bool written) {
  const bool layer = s.kind == SEE_NORM_LAYER;
  ops->Add(Vector("pre_rstd", stats.pre_rstd, s.rows * 4, 4, written));
  if (layer) ops->Add(Vector("pre_mean", stats.pre_mean, s.rows * 4, 4, written));
  if (!w.post_gamma) return;
  ops->Add(Vector("post_rstd", stats.post_rstd, s.rows * 4, 4, written));
  if (layer) ops->Add(Vector("post_mean", stats.post_mean, s.rows * 4, 4, written));
}

k::JoinArgs ArgsOf(const see_join_shape& s, const see_join_weights& w, const see_join_stats& stats) {
  k::JoinArgs a;
  a.w = w;
  a.stats = stats;
  a.rows = s.rows;
  a.x_stride = s.x_stride;
  a.y_stride = s.y_stride;
  a.cols = static_cast<uint32_t>(s.cols);
  a.x_type = s.x_type;
  a.y_type = s.y_type;
  a.rms = s.kind == SEE_NORM_RMS;
  a.eps = s.eps;
  a.scale = s.residual_scale;
  return a;
}

}  // namespace

uint64_t JoinBackwardWorkspace(uint64_t rows, uint64_t cols) {
  if (cols == 0 || cols > k::kNormMaxCols) return 0;
  return std::max<uint64_t>(16, k::NormPartialRows(rows) * cols * 4 * sizeof(float));
}

Status CheckJoinForward(see_join_shape* shape, const void* x, const void* block, const see_join_weights* weights, const void* x_out,
                        const void* y, const see_join_stats* stats) {
  const char* const what = "cuda: join forward";
  if (auto r = CheckJoin(what, shape, weights, stats); !r) return r;
  const see_join_shape& s = *shape;
  const see_join_weights& w = *weights;
  const bool layer = s.kind == SEE_NORM_LAYER;
  const uint64_t xs = SizeOfType(s.x_type), ys = SizeOfType(s.y_type), vector = s.cols * 4;
  Operands ops = {{"x", x, s.rows, s.cols * xs, s.x_stride * xs, xs, false},
                  {"block", block, s.rows, s.cols * ys, s.y_stride * ys, ys, false},
                  {"x_out", x_out, s.rows, s.cols * xs, s.x_stride * xs, xs, true},
                  {"y", y, s.rows, s.cols * ys, s.y_stride * ys, ys, true},
                  Vector("pre_gamma", w.pre_gamma, vector, 4, false)};
  if (layer) ops.Add(Vector("pre_beta", w.pre_beta, vector, 4, false));
  if (w.gate) ops.Add(Vector("gate", w.gate, vector, 4, false));
  if (w.post_gamma) ops.Add(Vector("post_gamma", w.post_gamma, vector, 4, false));
  if (w.post_gamma && layer) ops.Add(Vector("post_beta", w.post_beta, vector, 4, false));
  AddStats(&ops, s, w, *stats, true);
  return ops.Check(what);
}

Status CudaBackend::JoinForward(const see_join_shape& given, const void* x, const void* block, const see_join_weights* weights, void* x_out,
                                void* y, const see_join_stats* stats) {
  see_join_shape s = given;
  if (auto r = CheckJoinForward(&s, x, block, weights, x_out, y, stats); !r) return r;
  if (s.rows == 0) return {};
  k::JoinArgs a = ArgsOf(s, *weights, *stats);
  a.x = x;
  a.block = block;
  a.x_out = x_out;
  a.y = y;
  a.status = d_status_;
  OnDevice on(device_);
  if (!on.ok()) return Check(cudaGetLastError(), "join forward: device");
  int launches = 0;
  const cudaError_t e = k::Join(a, false, sms_, stream_, &launches);
  counters_.kernel_launches += static_cast<uint64_t>(launches);
  return Check(e, "join forward");
}

Status CheckJoinBackward(see_join_shape* shape, const void* dy, const void* dx_out, const void* x_out, const void* block,
                         const see_join_weights* weights, const see_join_stats* stats, const void* dx, const void* dblock,
                         const see_join_weights* gradients, const void* workspace, uint64_t workspace_bytes) {
  const char* const what = "cuda: join backward";
  if (auto r = CheckJoin(what, shape, weights, stats); !r) return r;
  if (!gradients) return Refuse(what, "gradients is null");
  const see_join_shape& s = *shape;
  const see_join_weights &w = *weights, &g = *gradients;
  const bool layer = s.kind == SEE_NORM_LAYER, post = w.post_gamma != nullptr;
  if ((!layer && (g.pre_beta || g.post_beta)) || (!post && (g.post_gamma || g.post_beta)) || (!w.gate && g.gate))
    return Refuse(what, "a gradient of a weight that is not there");
  if (workspace_bytes < JoinBackwardWorkspace(s.rows, s.cols)) return Refuse(what, "the workspace is too small");
  const uint64_t xs = SizeOfType(s.x_type), ys = SizeOfType(s.y_type), vector = s.cols * 4;
  Operands ops = {{"dy", dy, s.rows, s.cols * ys, s.y_stride * ys, ys, false},
                  {"x_out", x_out, s.rows, s.cols * xs, s.x_stride * xs, xs, false},
                  {"block", block, s.rows, s.cols * ys, s.y_stride * ys, ys, false},
                  {"dx", dx, s.rows, s.cols * xs, s.x_stride * xs, xs, true},
                  {"dblock", dblock, s.rows, s.cols * ys, s.y_stride * ys, ys, true},
                  Vector("pre_gamma", w.pre_gamma, vector, 4, false),
                  Vector("pre_gamma's gradient", g.pre_gamma, vector, 4, true),
                  Vector("workspace", workspace, workspace_bytes, 16, true)};
  if (dx_out) ops.Add({"dx_out", dx_out, s.rows, s.cols * xs, s.x_stride * xs, xs, false});
  if (layer) ops.Add(Vector("pre_beta's gradient", g.pre_beta, vector, 4, true));
  if (w.gate) {
    ops.Add(Vector("gate", w.gate, vector, 4, false));
    ops.Add(Vector("gate's gradient", g.gate, vector, 4, true));
  }
  if (post) {
    ops.Add(Vector("post_gamma", w.post_gamma, vector, 4, false));
    ops.Add(Vector("post_gamma's gradient", g.post_gamma, vector, 4, true));
    if (layer) {
      ops.Add(Vector("post_beta", w.post_beta, vector, 4, false));
      ops.Add(Vector("post_beta's gradient", g.post_beta, vector, 4, true));
    }
  }
  AddStats(&ops, s, w, *stats, false);
  return ops.Check(what);
}

Status CudaBackend::JoinBackward(const see_join_shape& given, const void* dy, const void* dx_out, const void* x_out, const void* block,
                                 const see_join_weights* weights, const see_join_stats* stats, void* dx, void* dblock,
                                 const see_join_weights* gradients, void* workspace, uint64_t workspace_bytes) {
  see_join_shape s = given;
  if (auto r = CheckJoinBackward(&s, dy, dx_out, x_out, block, weights, stats, dx, dblock, gradients, workspace, workspace_bytes); !r) return r;
  OnDevice on(device_);
  if (!on.ok()) return Check(cudaGetLastError(), "join backward: device");
  if (s.rows == 0) {
    for (float* g : {gradients->post_gamma, gradients->post_beta, gradients->gate, gradients->pre_gamma, gradients->pre_beta})
      if (g)
        if (auto r = Check(cudaMemsetAsync(g, 0, s.cols * 4, stream_), "join backward"); !r) return r;
    return {};
  }
  k::JoinArgs a = ArgsOf(s, *weights, *stats);
  a.dy = dy;
  a.dx_out = dx_out;
  a.x = x_out;
  a.block = block;
  a.dx = dx;
  a.dblock = dblock;
  a.grads = *gradients;
  a.partials = static_cast<float*>(workspace);
  a.status = d_status_;
  int launches = 0;
  const cudaError_t e = k::Join(a, true, sms_, stream_, &launches);
  counters_.kernel_launches += static_cast<uint64_t>(launches);
  return Check(e, "join backward");
}

}  // namespace see
