// Calls the checks of the operators on caller memory (block_checks.h) with made-up addresses: nothing is read, no device is
// needed.  One line a call: its name, a tab, the refusal or "ok".  Built and read by test_block_op_refusals.py.
#include <cstdio>
#include <functional>
#include <limits>
#include <string>

#include "../include/see_cuda.h"
#include "../see_ai_b200/csrc/block_checks.h"

namespace {

template <typename T = void>
T* At(uint64_t mebibyte, uint64_t offset = 0) { return reinterpret_cast<T*>((mebibyte << 20) + offset); }

void Say(const char* name, const see::Status& s) { std::printf("%s\t%s\n", name, s ? "ok" : s.error().c_str()); }

struct Norm {
  see_norm_shape shape{SEE_NORM_LAYER, SEE_F32, SEE_F32, 1e-5f, 100, 64, 0, 0};
  const void *x = At(1), *dy = At(2), *addend = nullptr;
  const float *gamma = At<float>(3), *beta = At<float>(4);
  void *y = At(5), *dx = At(6), *work = At(7);
  float *mean = At<float>(8), *rstd = At<float>(9), *dgamma = At<float>(10), *dbeta = At<float>(11);
  uint64_t bytes = 1 << 20;
};
void Forward(const char* name, std::function<void(Norm&)> change) {
  Norm n;
  change(n);
  Say(name, see::CheckNormForward(&n.shape, n.x, n.gamma, n.beta, n.y, n.mean, n.rstd));
}
void Backward(const char* name, std::function<void(Norm&)> change) {
  Norm n;
  change(n);
  Say(name, see::CheckNormBackward(&n.shape, n.dy, n.x, n.gamma, n.mean, n.rstd, n.addend, n.dx, n.dgamma, n.dbeta, n.work, n.bytes));
}

struct Gated {
  see_gated_shape shape{SEE_BF16, SEE_ACT_SILU, 100, 64, 128, 0, 0};
  const void *x = At(1), *wg = At(2), *wu = At(3), *dh = At(4);
  void *hidden = At(5), *gate = At(6), *up = At(7), *dx = At(8), *dwg = At(9), *dwu = At(10), *work = At(64);
  uint64_t bytes = 64 << 20;
};
void GatedFwd(const char* name, std::function<void(Gated&)> change) {
  Gated g;
  change(g);
  Say(name, see::CheckGatedForward(&g.shape, g.x, g.wg, g.wu, g.hidden, g.gate, g.up));
}
void GatedBwd(const char* name, std::function<void(Gated&)> change) {
  Gated g;
  change(g);
  Say(name, see::CheckGatedBackward(&g.shape, g.dh, g.x, g.wg, g.wu, g.gate, g.up, g.dx, g.dwg, g.dwu, g.work, g.bytes));
}

struct Adam {
  see_adamw_tensor t[3] = {};
  uint64_t count = 3;
  int bits = 8;
  see::StepParams params;
  const float* scale = nullptr;
  Adam() {
    params.step = 1;
    for (uint64_t i = 0; i < 3; ++i)   // side by side in common buffers
      t[i] = {At<float>(1, i * 4000), At(2, i * 2000), At(3, i * 1000), At(4, i * 1000), At<float>(5, i * 16), At<float>(6, i * 16), At(7, i * 2000), 1000, SEE_BF16, SEE_F16, 0, 0};
  }
};
void AdamW(const char* name, std::function<void(Adam&)> change) {
  Adam a;
  change(a);
  Say(name, see::CheckAdamW(a.t, a.count, a.bits, a.params, a.scale));
}

}  // namespace

int main() {
  Forward("norm", [](Norm&) {});
  Forward("norm kind", [](Norm& n) { n.shape.kind = 2; });
  Forward("norm x_type", [](Norm& n) { n.shape.x_type = 3; });
  Forward("norm types", [](Norm& n) { n.shape.x_type = SEE_BF16; });
  Forward("norm eps", [](Norm& n) { n.shape.eps = -1.0f; });
  Forward("norm eps nan", [](Norm& n) { n.shape.eps = std::numeric_limits<float>::quiet_NaN(); });
  Forward("norm no columns", [](Norm& n) { n.shape.cols = 0; });
  Forward("norm columns", [](Norm& n) { n.shape.cols = 16385; });
  Forward("norm rows", [](Norm& n) { n.shape.rows = 1ull << 31; });
  Forward("norm stride", [](Norm& n) { n.shape.x_stride = 63; });
  Forward("norm stride wide", [](Norm& n) { n.shape.y_stride = 1ull << 41; });
  Forward("norm null", [](Norm& n) { n.gamma = nullptr; });
  Forward("norm null mean", [](Norm& n) { n.mean = nullptr; });
  Forward("norm aligned", [](Norm& n) { n.x = At(1, 2); });
  Forward("norm in place", [](Norm& n) { n.y = const_cast<void*>(n.x); });
  Forward("norm behind", [](Norm& n) { n.y = At(1, 100 * 64 * 4); });
  Forward("norm into", [](Norm& n) { n.y = At(1, 100 * 64 * 4 - 4); });
  Forward("norm side by side", [](Norm& n) { n.shape.x_stride = n.shape.y_stride = 128; n.y = At(1, 64 * 4); });
  Forward("norm side into", [](Norm& n) { n.shape.x_stride = n.shape.y_stride = 128; n.y = At(1, 63 * 4); });
  Forward("norm rms beta", [](Norm& n) { n.shape.kind = SEE_NORM_RMS; });
  Forward("norm rms", [](Norm& n) { n.shape.kind = SEE_NORM_RMS; n.beta = nullptr; n.mean = nullptr; });
  Forward("norm empty", [](Norm& n) { n.shape.rows = 0; });
  Backward("norm back", [](Norm&) {});
  Backward("norm back addend", [](Norm& n) { n.addend = At(12); });
  Backward("norm back addend into", [](Norm& n) { n.addend = n.dx; });
  Backward("norm back work", [](Norm& n) { n.bytes = see::NormBackwardWorkspace(100, 64) - 1; });
  Backward("norm back work null", [](Norm& n) { n.work = nullptr; });
  Backward("norm back work aligned", [](Norm& n) { n.work = At(7, 8); });
  Backward("norm back work into", [](Norm& n) { n.work = At(8); });
  Backward("norm back dbeta", [](Norm& n) { n.dbeta = nullptr; });
  Backward("norm back rms dbeta", [](Norm& n) { n.shape.kind = SEE_NORM_RMS; n.mean = nullptr; });

  GatedFwd("gated", [](Gated&) {});
  GatedFwd("gated not kept", [](Gated& g) { g.gate = g.up = nullptr; });
  GatedFwd("gated half kept", [](Gated& g) { g.up = nullptr; });
  GatedFwd("gated type", [](Gated& g) { g.shape.type = SEE_F32; });
  GatedFwd("gated act", [](Gated& g) { g.shape.act = 0; });
  GatedFwd("gated d_in", [](Gated& g) { g.shape.d_in = 60; });
  GatedFwd("gated d_hidden", [](Gated& g) { g.shape.d_hidden = (1 << 20) + 8; });
  GatedFwd("gated no d_in", [](Gated& g) { g.shape.d_in = 0; });
  GatedFwd("gated rows", [](Gated& g) { g.shape.rows = 0x7FFFFF01ull; });
  GatedFwd("gated rows by widths", [](Gated& g) { g.shape.rows = 0x7FFFFF00ull; g.shape.d_hidden = 1 << 20; });
  GatedFwd("gated stride", [](Gated& g) { g.shape.x_stride = 68; });
  GatedFwd("gated aligned", [](Gated& g) { g.wg = At(2, 8); });
  GatedFwd("gated null", [](Gated& g) { g.x = nullptr; });
  GatedFwd("gated into", [](Gated& g) { g.gate = g.hidden; });
  GatedFwd("gated side by side", [](Gated& g) { g.shape.hidden_stride = 256; g.up = At(6, 256); });
  GatedBwd("gated back", [](Gated&) {});
  GatedBwd("gated back dx", [](Gated& g) { g.dwg = g.dwu = nullptr; });
  GatedBwd("gated back dw", [](Gated& g) { g.dx = nullptr; });
  GatedBwd("gated back half dw", [](Gated& g) { g.dwu = nullptr; });
  GatedBwd("gated back nothing", [](Gated& g) { g.dx = g.dwg = g.dwu = nullptr; });
  GatedBwd("gated back work", [](Gated& g) { g.bytes = 2 * 100 * 128 * 2 - 1; });
  GatedBwd("gated back work aligned", [](Gated& g) { g.work = At(64, 64); });
  GatedBwd("gated back into", [](Gated& g) { g.dx = const_cast<void*>(g.x); });
  GatedBwd("gated back weights", [](Gated& g) { g.dwg = const_cast<void*>(g.wg); });

  AdamW("adamw", [](Adam&) {});
  AdamW("adamw 32", [](Adam& a) {
    a.bits = 32;
    for (auto& t : a.t) t.m = At(8, reinterpret_cast<uint64_t>(t.p) & 0xFFFFF), t.v = At(9, reinterpret_cast<uint64_t>(t.p) & 0xFFFFF), t.m_scale = t.v_scale = nullptr;
  });
  AdamW("adamw bits", [](Adam& a) { a.bits = 16; });
  AdamW("adamw step", [](Adam& a) { a.params.step = 0; });
  AdamW("adamw beta", [](Adam& a) { a.params.beta2 = 1.0f; });
  AdamW("adamw g_type", [](Adam& a) { a.t[1].g_type = 7; });
  AdamW("adamw copy", [](Adam& a) { a.t[1].copy = nullptr; });
  AdamW("adamw no copy", [](Adam& a) { a.t[1].copy = nullptr; a.t[1].copy_type = SEE_F32; });
  AdamW("adamw flag", [](Adam& a) { a.t[2].flags = 2; });
  AdamW("adamw null", [](Adam& a) { a.t[2].v = nullptr; });
  AdamW("adamw scale null", [](Adam& a) { a.t[0].m_scale = nullptr; });
  AdamW("adamw aligned", [](Adam& a) { a.t[0].p = At<float>(1, 1); });
  AdamW("adamw large", [](Adam& a) { a.t[0].n = (1ull << 38) + 1; });
  AdamW("adamw twice", [](Adam& a) { a.t[2] = a.t[1]; });
  AdamW("adamw into", [](Adam& a) { a.t[1].p = At<float>(1, 3996); });
  AdamW("adamw p over g", [](Adam& a) { a.t[1].p = At<float>(2, 4000); });
  AdamW("adamw same g", [](Adam& a) { a.t[1].g = a.t[0].g; });
  AdamW("adamw descending", [](Adam& a) { std::swap(a.t[0], a.t[2]); });
  AdamW("adamw interleaved", [](Adam& a) {   // each tensor's operands together, in one buffer
    for (uint64_t i = 0; i < 3; ++i) a.t[i].p = At<float>(1, i * 16384), a.t[i].g = At(1, i * 16384 + 4096), a.t[i].m = At(1, i * 16384 + 8192);
  });
  AdamW("adamw scale in p", [](Adam& a) { a.scale = At<float>(1, 4); });
  AdamW("adamw scale", [](Adam& a) { a.scale = At<float>(12); });
  AdamW("adamw scale aligned", [](Adam& a) { a.scale = At<float>(12, 2); });
  AdamW("adamw empty tensor", [](Adam& a) { a.t[1] = {}; });
  AdamW("adamw none", [](Adam& a) { a.count = 0; });
  Say("adamw no table", see::CheckAdamW(nullptr, 3, 8, Adam().params, nullptr));

  Say("handle", see_cuda_norm_forward(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr) == SEE_ERROR ? see::Status{} : std::unexpected("taken"));
  Say("handle gated", see_cuda_gated_forward(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr) == SEE_ERROR ? see::Status{} : std::unexpected("taken"));
  Say("handle adamw", see_cuda_adamw_step(nullptr, nullptr, 0, 8, nullptr, nullptr) == SEE_ERROR ? see::Status{} : std::unexpected("taken"));
  return 0;
}
