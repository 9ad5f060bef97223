// Calls the checks of the losses over rows of logits with many values of logit_scale and made-up addresses: nothing is read, no device is
// needed.  One line a call: "policy" or "preference", the scale, "ok" or the refusal, tabs between.  Built and read by test_logit_scale.py.
#include <cstdint>
#include <cstdio>
#include <limits>

#include "../include/see_cuda.h"
#include "../see_ai_b200/csrc/block_checks.h"

int main() {
  auto at = [](uint64_t mebibyte) { return reinterpret_cast<void*>(mebibyte << 20); };
  auto floats = [&](uint64_t mebibyte) { return static_cast<float*>(at(mebibyte)); };
  auto labels = [&](uint64_t mebibyte) { return static_cast<int32_t*>(at(mebibyte)); };
  const float inf = std::numeric_limits<float>::infinity();
  for (float scale : {0.0f, -1.0f, -0.0f, 1e-45f, 1e-38f, 0x1p-101f, 0x1.fffffep-101f, 0x1p-100f, 1e-3f, 1.0f, 1e3f, 0x1p100f, 0x1.000002p100f,
                      0x1p127f, std::numeric_limits<float>::max(), inf, -inf, std::numeric_limits<float>::quiet_NaN()}) {
    see_policy_shape policy{SEE_F32, scale, 0.2f, 0.2f, 0.0f, 0, 100, 250, 0};
    const see::Status a = see::CheckPolicy(&policy, at(1), labels(2), floats(3), nullptr, floats(4), nullptr, nullptr, floats(5), floats(6), at(7), at(8), 1 << 20);
    std::printf("policy\t%a\t%s\n", static_cast<double>(scale), a ? "ok" : a.error().c_str());
    see_preference_shape pairs{SEE_F32, SEE_PREFERENCE_SIGMOID, 0.1f, 0.0f, 0.0f, scale, 0, 0, 100, 250, 0, 3};
    const see::Status b = see::CheckPreference(&pairs, at(1), labels(2), labels(3), nullptr, nullptr, floats(4), floats(5), floats(6), at(7), at(8), 1 << 20);
    std::printf("preference\t%a\t%s\n", static_cast<double>(scale), b ? "ok" : b.error().c_str());
  }
}
