// What the gated backward pass uses of its workspace, against what the query promises to suffice, on devices of several sizes:
// host code alone.  One line for each number of SMs: it, a tab, the shapes tried, a tab, those that would want more.  Built and
// read by test_gated_workspace.py.
#include <cstdint>
#include <cstdio>

#include "../see_ai_b200/csrc/block_checks.h"

int main() {
  const uint64_t rows[] = {1, 16, 200, 600, 1000, 1500, 2048, 4096, 5000, 8191, 20000, 65536, 300000};
  const uint64_t widths[] = {8, 64, 200, 512, 768, 1000, 1376, 2048, 4096, 5632, 11264};
  for (uint32_t sms : {2u, 40u, 78u, 108u, 114u, 120u, 132u, 142u, 144u, 146u, 148u, 160u}) {
    uint64_t tried = 0, short_of = 0;
    for (uint64_t r : rows)
      for (uint64_t d : widths)
        for (uint64_t f : widths) {
          const uint64_t promised = see::GatedBackwardWorkspace(r, d, f);
          for (int want = 1; want < 4; ++want) {
            ++tried;
            short_of += see::GatedBackwardUses(r, d, f, want & 1, want & 2, sms) > promised;
          }
        }
    std::printf("%u\t%llu\t%llu\n", sms, static_cast<unsigned long long>(tried), static_cast<unsigned long long>(short_of));
  }
  return 0;
}
