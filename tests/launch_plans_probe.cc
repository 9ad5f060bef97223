// Walks through what the host decides before it launches, over many sizes: nothing is read, no device is needed.  One line a family: its
// name, a tab, "ok" or what is wrong first.  Built and read by test_launch_plans.py.
#include <cstdio>
#include <string>
#include <vector>

#include "../see_ai_b200/csrc/grad_table.h"

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

}  // namespace

int main() {
  GradTables();
  return 0;
}
