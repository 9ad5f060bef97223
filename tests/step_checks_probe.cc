// Calls the checks of the operators around a block's own weights (block_checks.h) with made-up addresses: nothing is read, no device is
// needed.  One line a call: its name, a tab, the refusal or "ok".  Built and read by test_step_op_refusals.py.
#include <cstdio>
#include <functional>
#include <limits>
#include <string>

#include "../include/see_cuda.h"
#include "../see_ai_b200/csrc/block_checks.h"

namespace {

template <typename T = void>
T* At(uint64_t mebibyte, uint64_t offset = 0) { return reinterpret_cast<T*>((mebibyte << 20) + offset); }
const float kNan = std::numeric_limits<float>::quiet_NaN(), kInf = std::numeric_limits<float>::infinity();

void Say(const char* name, const see::Status& s) { std::printf("%s\t%s\n", name, s ? "ok" : s.error().c_str()); }

struct Join {
  see_join_shape shape{SEE_NORM_LAYER, SEE_F32, SEE_BF16, 1e-5f, 1.0f, 0, 100, 64, 0, 0};
  const void *x = At(1), *block = At(2), *dy = At(3), *dx_out = At(4);
  void *x_out = At(5), *y = At(6), *dx = At(7), *dblock = At(8), *work = At(9);
  see_join_weights w{At<float>(20), At<float>(21), At<float>(22), At<float>(23), At<float>(24)};
  see_join_weights g{At<float>(30), At<float>(31), At<float>(32), At<float>(33), At<float>(34)};
  see_join_stats stats{At<float>(40), At<float>(41), At<float>(42), At<float>(43)};
  const see_join_weights *weights = &w, *gradients = &g;
  const see_join_stats* kept = &stats;
  uint64_t bytes = 1 << 20;
  void Rms() {
    shape.kind = SEE_NORM_RMS;
    w.post_beta = w.pre_beta = g.post_beta = g.pre_beta = nullptr;
    stats.post_mean = stats.pre_mean = nullptr;
  }
  void NoPost() {
    w.post_gamma = w.post_beta = g.post_gamma = g.post_beta = nullptr;
    stats.post_mean = stats.post_rstd = nullptr;
  }
};
void Forward(const char* name, std::function<void(Join&)> change) {
  Join j;
  change(j);
  Say(name, see::CheckJoinForward(&j.shape, j.x, j.block, j.weights, j.x_out, j.y, j.kept));
}
void Backward(const char* name, std::function<void(Join&)> change) {
  Join j;
  change(j);
  Say(name, see::CheckJoinBackward(&j.shape, j.dy, j.dx_out, j.x_out, j.block, j.weights, j.kept, j.dx, j.dblock, j.gradients, j.work, j.bytes));
}

struct Preference {
  see_preference_shape shape{SEE_BF16, SEE_PREFERENCE_SIGMOID, 0.1f, 0.0f, 0.0f, 1.0f, 0, 0, 100, 250, 0, 3};
  const void* logits = At(1);
  const int32_t *labels = At<int32_t>(2), *starts = At<int32_t>(3);
  const float *ref = At<float>(4), *grad = At<float>(5);
  float *loss = At<float>(6), *margins = At<float>(7), *sums = At<float>(8);
  void *d = At(9), *work = At(10);
  uint64_t bytes = 1 << 20;
};
void Pairs(const char* name, std::function<void(Preference&)> change) {
  Preference p;
  change(p);
  Say(name, see::CheckPreference(&p.shape, p.logits, p.labels, p.starts, p.ref, p.grad, p.loss, p.margins, p.sums, p.d, p.work, p.bytes));
}

struct Policy {
  see_policy_shape shape{SEE_F32, 1.0f, 0.2f, 0.2f, 0.1f, 0, 100, 250, 0};
  const void* logits = At(1);
  const int32_t* labels = At<int32_t>(2);
  const float *old = At<float>(3), *ref = At<float>(4), *a = At<float>(5), *w = At<float>(6), *grad = At<float>(7);
  float *loss = At<float>(8), *logp = At<float>(9);
  void *d = At(10), *work = At(11);
  uint64_t bytes = 1 << 20;
};
void Clipped(const char* name, std::function<void(Policy&)> change) {
  Policy p;
  change(p);
  Say(name, see::CheckPolicy(&p.shape, p.logits, p.labels, p.old, p.ref, p.a, p.w, p.grad, p.loss, p.logp, p.d, p.work, p.bytes));
}

struct Grad {
  see_grad_tensor t[3] = {};
  uint64_t count = 3;
  float most = 1.0f;
  const float* scale = nullptr;
  float *norm = At<float>(10), *factor = At<float>(10, 4);
  void* work = At(11);
  uint64_t bytes = see::GradWorkspace();
  Grad() {
    for (uint64_t i = 0; i < 3; ++i) t[i] = {At(1, i * 2000), At(2, i * 2000), 1000, SEE_BF16, 0};
  }
};
void Norm(const char* name, bool clip, std::function<void(Grad&)> change) {
  Grad g;
  change(g);
  Say(name, see::CheckGrad(g.t, g.count, clip, g.most, g.scale, g.norm, g.factor, g.work, g.bytes));
}

}  // namespace

int main() {
  Forward("join", [](Join&) {});
  Forward("join rms", [](Join& j) { j.Rms(); });
  Forward("join no post", [](Join& j) { j.NoPost(); });
  Forward("join no gate", [](Join& j) { j.w.gate = nullptr; });
  Forward("join kind", [](Join& j) { j.shape.kind = 2; });
  Forward("join types", [](Join& j) { j.shape.x_type = SEE_F16; });
  Forward("join y_type", [](Join& j) { j.shape.y_type = 5; });
  Forward("join eps", [](Join& j) { j.shape.eps = kNan; });
  Forward("join scale", [](Join& j) { j.shape.residual_scale = kInf; });
  Forward("join no columns", [](Join& j) { j.shape.cols = 0; });
  Forward("join columns", [](Join& j) { j.shape.cols = 16385; });
  Forward("join rows", [](Join& j) { j.shape.rows = 1ull << 31; });
  Forward("join stride", [](Join& j) { j.shape.y_stride = 63; });
  Forward("join stride wide", [](Join& j) { j.shape.x_stride = 1ull << 41; });
  Forward("join no weights", [](Join& j) { j.weights = nullptr; });
  Forward("join no stats", [](Join& j) { j.kept = nullptr; });
  Forward("join rms beta", [](Join& j) { j.Rms(); j.w.pre_beta = At<float>(24); });
  Forward("join rms mean", [](Join& j) { j.Rms(); j.stats.post_mean = At<float>(40); });
  Forward("join layer beta", [](Join& j) { j.w.post_beta = nullptr; });
  Forward("join stray beta", [](Join& j) { j.NoPost(); j.w.post_beta = At<float>(21); });
  Forward("join stray rstd", [](Join& j) { j.NoPost(); j.stats.post_rstd = At<float>(41); });
  Forward("join pre_gamma", [](Join& j) { j.w.pre_gamma = nullptr; });
  Forward("join post_rstd", [](Join& j) { j.stats.post_rstd = nullptr; });
  Forward("join null", [](Join& j) { j.block = nullptr; });
  Forward("join aligned", [](Join& j) { j.y = At(6, 1); });
  Forward("join gate aligned", [](Join& j) { j.w.gate = At<float>(22, 2); });
  Forward("join in place", [](Join& j) { j.x_out = const_cast<void*>(j.x); });
  Forward("join y over block", [](Join& j) { j.y = const_cast<void*>(j.block); });
  Forward("join side by side", [](Join& j) { j.shape.y_stride = 128; j.y = At(2, 128); });
  Forward("join empty", [](Join& j) { j.shape.rows = 0; j.x = j.block = nullptr; j.x_out = j.y = nullptr; j.stats = {}; });
  Backward("join back", [](Join&) {});
  Backward("join back rms", [](Join& j) { j.Rms(); });
  Backward("join back no post", [](Join& j) { j.NoPost(); });
  Backward("join back no gate", [](Join& j) { j.w.gate = j.g.gate = nullptr; });
  Backward("join back no dx_out", [](Join& j) { j.dx_out = nullptr; });
  Backward("join back no gradients", [](Join& j) { j.gradients = nullptr; });
  Backward("join back stray gate", [](Join& j) { j.w.gate = nullptr; });
  Backward("join back stray post", [](Join& j) { j.NoPost(); j.g.post_gamma = At<float>(30); });
  Backward("join back rms beta", [](Join& j) { j.Rms(); j.g.pre_beta = At<float>(34); });
  Backward("join back gate null", [](Join& j) { j.g.gate = nullptr; });
  Backward("join back dbeta null", [](Join& j) { j.g.post_beta = nullptr; });
  Backward("join back pre_beta unread", [](Join& j) { j.w.pre_beta = nullptr; });
  Backward("join back work", [](Join& j) { j.bytes = see::JoinBackwardWorkspace(100, 64) - 1; });
  Backward("join back work aligned", [](Join& j) { j.work = At(9, 8); });
  Backward("join back dx over dx_out", [](Join& j) { j.dx = const_cast<void*>(j.dx_out); });
  Backward("join back dblock over dy", [](Join& j) { j.dblock = const_cast<void*>(j.dy); });
  Backward("join back gradient over weight", [](Join& j) { j.g.post_gamma = j.w.post_gamma; });
  Backward("join back empty", [](Join& j) { j.shape.rows = 0; j.dy = j.dx_out = j.block = nullptr; j.x_out = j.dx = j.dblock = nullptr; j.stats = {}; });

  Pairs("preference", [](Preference&) {});
  Pairs("preference bare", [](Preference& p) { p.ref = p.grad = nullptr; p.d = nullptr; });
  Pairs("preference in place", [](Preference& p) { p.d = const_cast<void*>(p.logits); });
  Pairs("preference into logits", [](Preference& p) { p.d = At(1, 2); });
  Pairs("preference type", [](Preference& p) { p.shape.type = 3; });
  Pairs("preference kind", [](Preference& p) { p.shape.kind = 3; });
  Pairs("preference scale", [](Preference& p) { p.shape.logit_scale = 0.0f; });
  Pairs("preference scale nan", [](Preference& p) { p.shape.logit_scale = kNan; });
  Pairs("preference no classes", [](Preference& p) { p.shape.classes = 0; });
  Pairs("preference classes", [](Preference& p) { p.shape.classes = (1 << 20) + 1; });
  Pairs("preference rows", [](Preference& p) { p.shape.rows = 1ull << 31; });
  Pairs("preference stride", [](Preference& p) { p.shape.stride = 249; });
  Pairs("preference no pairs", [](Preference& p) { p.shape.pairs = 0; });
  Pairs("preference pairs", [](Preference& p) { p.shape.pairs = (1 << 24) + 1; });
  Pairs("preference beta", [](Preference& p) { p.shape.beta = 0.0f; });
  Pairs("preference smoothing", [](Preference& p) { p.shape.smoothing = 0.5f; });
  Pairs("preference smoothed hinge", [](Preference& p) { p.shape.kind = SEE_PREFERENCE_HINGE; p.shape.smoothing = 0.1f; });
  Pairs("preference margin", [](Preference& p) { p.shape.margin = kInf; });
  Pairs("preference square margin", [](Preference& p) { p.shape.kind = SEE_PREFERENCE_SQUARE; p.shape.margin = 0.1f; });
  Pairs("preference work", [](Preference& p) { p.bytes = see::PreferenceWorkspace(100, 3) - 1; });
  Pairs("preference work aligned", [](Preference& p) { p.work = At(10, 8); });
  Pairs("preference starts", [](Preference& p) { p.starts = nullptr; });
  Pairs("preference labels aligned", [](Preference& p) { p.labels = At<int32_t>(2, 2); });
  Pairs("preference loss into margins", [](Preference& p) { p.loss = p.margins + 2; });
  Pairs("preference empty", [](Preference& p) { p.shape.rows = 0; p.logits = nullptr; p.labels = nullptr; p.d = nullptr; });

  Clipped("policy", [](Policy&) {});
  Clipped("policy bare", [](Policy& p) { p.ref = p.w = p.grad = nullptr; p.shape.kl_coef = 0.0f; p.d = nullptr; });
  Clipped("policy in place", [](Policy& p) { p.d = const_cast<void*>(p.logits); });
  Clipped("policy into logits", [](Policy& p) { p.d = At(1, 4); });
  Clipped("policy type", [](Policy& p) { p.shape.type = -1; });
  Clipped("policy scale", [](Policy& p) { p.shape.logit_scale = -1.0f; });
  Clipped("policy classes", [](Policy& p) { p.shape.classes = (1 << 20) + 1; });
  Clipped("policy stride", [](Policy& p) { p.shape.stride = 1ull << 41; });
  Clipped("policy low", [](Policy& p) { p.shape.clip_low = 1.5f; });
  Clipped("policy low nan", [](Policy& p) { p.shape.clip_low = kNan; });
  Clipped("policy high", [](Policy& p) { p.shape.clip_high = kInf; });
  Clipped("policy kl", [](Policy& p) { p.shape.kl_coef = -0.1f; });
  Clipped("policy kl without", [](Policy& p) { p.ref = nullptr; });
  Clipped("policy old", [](Policy& p) { p.old = nullptr; });
  Clipped("policy work", [](Policy& p) { p.bytes = see::PolicyWorkspace(100) - 1; });
  Clipped("policy logp over old", [](Policy& p) { p.logp = const_cast<float*>(p.old); });
  Clipped("policy empty", [](Policy& p) { p.shape.rows = 0; p.logits = nullptr; p.labels = nullptr; p.old = p.ref = p.a = p.w = nullptr; p.logp = nullptr; p.d = nullptr; });

  for (bool clip : {false, true}) {
    const std::string kind = clip ? "clip" : "grad";
    auto norm = [&](const char* what, std::function<void(Grad&)> change) { Norm((kind + what).c_str(), clip, change); };
    norm("", [](Grad&) {});
    norm(" infinite", [](Grad& g) { g.most = kInf; });
    norm(" max", [](Grad& g) { g.most = 0.0f; });
    norm(" max nan", [](Grad& g) { g.most = kNan; });
    norm(" type", [](Grad& g) { g.t[1].type = 4; });
    norm(" null", [](Grad& g) { g.t[2].g = nullptr; });
    norm(" aligned", [](Grad& g) { g.t[0].g = At(1, 1); });
    norm(" large", [](Grad& g) { g.t[0].n = (1ull << 38) + 1; });
    norm(" work", [](Grad& g) { g.bytes -= 1; });
    norm(" work aligned", [](Grad& g) { g.work = At(11, 8); });
    norm(" factor null", [](Grad& g) { g.factor = nullptr; });
    norm(" norm is factor", [](Grad& g) { g.norm = g.factor; });
    norm(" scale", [](Grad& g) { g.scale = At<float>(12); });
    norm(" scale is factor", [](Grad& g) { g.scale = g.factor; });
    norm(" descending", [](Grad& g) { std::swap(g.t[0], g.t[2]); });
    norm(" twice", [](Grad& g) { g.t[2] = g.t[1]; });
    norm(" in place", [](Grad& g) { for (auto& t : g.t) t.out = t.g; });
    norm(" in place unsaid", [](Grad& g) { for (auto& t : g.t) t.out = nullptr; });
    norm(" in place twice", [](Grad& g) { for (auto& t : g.t) t.out = nullptr; g.t[2] = g.t[1]; });
    norm(" out over another", [](Grad& g) { g.t[0].out = g.t[1].g; });
    norm(" norm in a tensor", [](Grad& g) { g.norm = At<float>(1, 100); });
    norm(" empty tensor", [](Grad& g) { g.t[1] = {}; });
    norm(" none", [](Grad& g) { g.count = 0; });
  }
  Say("grad no table", see::CheckGrad(nullptr, 3, false, 1.0f, nullptr, At<float>(10), At<float>(10, 4), At(11), see::GradWorkspace()));

  auto handle = [](const char* name, int rc) { Say(name, rc == SEE_ERROR ? see::Status{} : std::unexpected("taken")); };
  handle("handle join", see_cuda_join_forward(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr));
  handle("handle join back", see_cuda_join_backward(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 0));
  handle("handle preference", see_cuda_preference_loss(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 0));
  handle("handle policy", see_cuda_policy_loss(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 0));
  handle("handle grad", see_cuda_grad_norm(nullptr, nullptr, 0, 1.0f, nullptr, nullptr, nullptr, nullptr, 0));
  handle("handle clip", see_cuda_grad_clip(nullptr, nullptr, 0, 1.0f, nullptr, nullptr, nullptr, nullptr, 0));
  return 0;
}
