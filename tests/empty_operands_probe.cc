// Calls of the operators on caller memory in which some operands cover no bytes and, as empty allocations do, have no address:
// the checks alone, without a device.  One line a call: its name, a tab, the refusal or "ok".  Built and read by
// test_empty_operands.py.
#include <cstdio>

#include "../include/see_cuda.h"
#include "../see_ai_b200/csrc/block_checks.h"

namespace {

template <typename T = void>
T* At(uint64_t mebibyte, uint64_t offset = 0) { return reinterpret_cast<T*>((mebibyte << 20) + offset); }

void Say(const char* name, const see::Status& s) { std::printf("%s\t%s\n", name, s ? "ok" : s.error().c_str()); }

}  // namespace

int main() {
  const float *gamma = At<float>(3), *beta = At<float>(4);
  float *dgamma = At<float>(10), *dbeta = At<float>(11);
  void* work = At(64);
  auto norm = [](int kind, uint64_t rows) { return see_norm_shape{kind, SEE_F32, SEE_F32, 1e-5f, rows, 64, 0, 0}; };
  see_norm_shape s = norm(SEE_NORM_LAYER, 0);
  Say("norm", see::CheckNormForward(&s, nullptr, gamma, beta, nullptr, nullptr, nullptr));
  Say("norm gamma", see::CheckNormForward(&s, nullptr, nullptr, beta, nullptr, nullptr, nullptr));
  Say("norm beta", see::CheckNormForward(&s, nullptr, gamma, nullptr, nullptr, nullptr, nullptr));
  Say("norm addresses", see::CheckNormForward(&s, At(1, 1), gamma, beta, At(1, 1), At<float>(1, 1), At<float>(1, 1)));
  Say("norm back", see::CheckNormBackward(&s, nullptr, nullptr, gamma, nullptr, nullptr, nullptr, nullptr, dgamma, dbeta, work, 16));
  Say("norm back dgamma", see::CheckNormBackward(&s, nullptr, nullptr, gamma, nullptr, nullptr, nullptr, nullptr, nullptr, dbeta, work, 16));
  Say("norm back dbeta", see::CheckNormBackward(&s, nullptr, nullptr, gamma, nullptr, nullptr, nullptr, nullptr, dgamma, nullptr, work, 16));
  Say("norm back work", see::CheckNormBackward(&s, nullptr, nullptr, gamma, nullptr, nullptr, nullptr, nullptr, dgamma, dbeta, nullptr, 16));
  Say("norm back no bytes", see::CheckNormBackward(&s, nullptr, nullptr, gamma, nullptr, nullptr, nullptr, nullptr, dgamma, dbeta, nullptr, 0));
  s = norm(SEE_NORM_RMS, 0);
  Say("rms", see::CheckNormForward(&s, nullptr, gamma, nullptr, nullptr, nullptr, nullptr));
  Say("rms back", see::CheckNormBackward(&s, nullptr, nullptr, gamma, nullptr, nullptr, nullptr, nullptr, dgamma, nullptr, work, 16));
  s = norm(SEE_NORM_LAYER, 1);
  Say("norm one row", see::CheckNormForward(&s, nullptr, gamma, beta, At(5), At<float>(8), At<float>(9)));

  see_gated_shape g{SEE_BF16, SEE_ACT_SILU, 0, 64, 128, 0, 0};
  const void *wg = At(1), *wu = At(2);
  void *dwg = At(5), *dwu = At(6);
  Say("gated", see::CheckGatedForward(&g, nullptr, wg, wu, nullptr, nullptr, nullptr));
  Say("gated weights", see::CheckGatedForward(&g, nullptr, wg, nullptr, nullptr, nullptr, nullptr));
  Say("gated back", see::CheckGatedBackward(&g, nullptr, nullptr, wg, wu, nullptr, nullptr, nullptr, dwg, dwu, work, 128));
  Say("gated back half", see::CheckGatedBackward(&g, nullptr, nullptr, wg, wu, nullptr, nullptr, nullptr, dwg, nullptr, work, 128));
  Say("gated back nothing", see::CheckGatedBackward(&g, nullptr, nullptr, wg, wu, nullptr, nullptr, nullptr, nullptr, nullptr, work, 128));
  Say("gated back dx", see::CheckGatedBackward(&g, nullptr, nullptr, wg, wu, nullptr, nullptr, At(7), nullptr, nullptr, work, 128));
  Say("gated back weights", see::CheckGatedBackward(&g, nullptr, nullptr, nullptr, wu, nullptr, nullptr, nullptr, dwg, dwu, work, 128));
  g.rows = 1;
  Say("gated one row", see::CheckGatedForward(&g, At(7), wg, wu, nullptr, nullptr, nullptr));

  see::StepParams params;
  params.step = 1;
  see_adamw_tensor t{nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 0, SEE_BF16, SEE_BF16, 0, 0};
  Say("adamw", see::CheckAdamW(&t, 1, 8, params, nullptr));
  t.copy = At(1, 1);
  t.copy_type = SEE_F32;
  Say("adamw copy", see::CheckAdamW(&t, 1, 8, params, nullptr));
  t.copy_type = 3;
  Say("adamw type", see::CheckAdamW(&t, 1, 8, params, nullptr));
  t = {At<float>(1), At(2), At(3), At(4), At<float>(5), At<float>(6), nullptr, 1, SEE_BF16, SEE_BF16, 0, 0};
  Say("adamw one element", see::CheckAdamW(&t, 1, 8, params, nullptr));
  return 0;
}
