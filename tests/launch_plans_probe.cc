// Walks through what the host decides before it launches, over many sizes: nothing is read, no device is needed.  One line a family: its
// name, a tab, "ok" or what is wrong first.  Built and read by test_launch_plans.py.
#include <cstdio>
#include <string>
#include <utility>
#include <vector>

#include "../see_ai_b200/csrc/grad_table.h"
#include "../see_ai_b200/csrc/join_ring.h"

namespace {

void Say(const std::string& name, const std::string& wrong) { std::printf("%s\t%s\n", name.c_str(), wrong.empty() ? "ok" : wrong.c_str()); }

// Tensors of 5 to 40000 elements, `empty` of none at each of some places; every launch as GradNorm makes it, and the table that is in hand
// when there was one.
std::string GradLists(uint64_t count, uint64_t empty, bool front, bool between, bool behind) {
  using namespace see::k;
  std::vector<see_grad_tensor> list;
  auto gap = [&](bool here) {
    for (uint64_t i = 0; here && i < empty; ++i) list.push_back({nullptr, nullptr, 0, SEE_BF16, 0});
  };
  gap(front);
  uint64_t at = 1 << 20;
  for (uint64_t i = 0; i < count; ++i) {
    if (i == count / 2) gap(between);
    list.push_back({reinterpret_cast<void*>(at), nullptr, 5 + i * 7919 % 40000, i % 3 ? SEE_BF16 : SEE_F32, 0});
    at += 1 << 20;
  }
  gap(behind);
  std::vector<uint64_t> seen;
  std::string wrong;
  GradTable table;
  unsigned tables = 0, blocks = 0;
  auto look = [&](const GradTable& t, unsigned grid) {
    if (t.count == 0 || t.count > kGradEntries) wrong = "a table of " + std::to_string(t.count);
    for (uint32_t i = 0; i < t.count && i < kGradEntries; ++i) seen.push_back(reinterpret_cast<uint64_t>(t.entry[i].g));
    const uint64_t units = t.count ? t.entry[t.count - 1].unit_end : 0;
    if (grid == 0 || grid > kGradPartials || t.each * grid + t.rest != units || t.rest >= grid) wrong = "ranges that are not the table's";
    return 0;
  };
  EachGradTable(&table, list.data(), list.size(), 148, 0, &tables, &blocks, look);
  if (tables != (count + kGradEntries - 1) / kGradEntries) wrong = std::to_string(tables) + " tables";
  if (seen.size() != count) wrong = std::to_string(seen.size()) + " tensors of " + std::to_string(count);
  for (uint64_t i = 0; i < seen.size() && wrong.empty(); ++i)
    if (seen[i] != (i + 1) << 20) wrong = "tensor " + std::to_string(i) + " is another";
  if (tables == 1) {   // launched again as it is
    seen.clear();
    look(table, blocks);
    if (seen.size() != count && wrong.empty()) wrong = "the table in hand has " + std::to_string(seen.size());
  }
  return wrong;
}

void GradTables() {
  for (uint64_t count : {0, 1, 2, 159, 160, 161, 319, 320, 321, 500})
    for (uint64_t empty : {1, 160, 333})
      for (int places = 0; places < 8; ++places) {
        const std::string wrong = GradLists(count, empty, places & 1, places & 2, places & 4);
        if (!wrong.empty()) return Say("grad tables", std::to_string(count) + " tensors, " + std::to_string(empty) + " empty at " + std::to_string(places) + ": " + wrong);
      }
  Say("grad tables", "");
}

// Rings of both passes of the join, of every width, of each pair of types and kind of norm, for groups of all sizes that hold such a row.
void JoinRings() {
  using namespace see::k;
  auto slot = [](size_t cols, size_t size) { return (cols * size + 45) / 16 * 16; };
  for (size_t cols = 1; cols <= kJoinRingCols; ++cols)
    for (auto [x, y] : {std::pair<size_t, size_t>{4, 4}, {4, 2}, {2, 2}})
      for (int pass = 0; pass < 4; ++pass) {   // forward, rms and layer; backward, without and with dx_out
        const size_t slot_bytes = pass < 2 ? slot(cols, x) + slot(cols, y) : (pass - 1) * slot(cols, x) + 2 * slot(cols, y);
        const size_t weights = (cols + 3) / 4 * 16 * (pass == 1 ? 4 : 2);
        for (uint32_t threads : {384, 512, 768})
          for (uint32_t T = 32; T <= threads; T += 32) {
            if (T * 32 < cols) continue;
            for (uint64_t rows : {1ull, 149ull, 1000ull, 5000ull, 22000ull, 0x7FFFFFFFull}) {
              const JoinRing r = RingOf(rows, threads, T, slot_bytes, weights, 148);
              if (r.bytes <= kMostShared && r.slots > 0 && r.slots <= kJoinMostSlots && r.groups > 0 && r.groups * T <= threads && r.grid > 0 &&
                  r.bytes == r.groups * r.slots * (slot_bytes + kJoinBarrier) + weights)
                continue;
              return Say("join rings", std::to_string(rows) + " x " + std::to_string(cols) + ", pass " + std::to_string(pass) + ", " +
                                           std::to_string(threads) + " threads, " + std::to_string(T) + " to a row: " + std::to_string(r.groups) + " groups of " +
                                           std::to_string(r.slots) + " slots, " + std::to_string(r.bytes) + " bytes");
            }
          }
      }
  Say("join rings", "");
}

}  // namespace

int main() {
  GradTables();
  JoinRings();
  return 0;
}
