// The table of one launch over many gradients, and how its units are cut among thread blocks.
#ifndef SEE_CUDA_GRAD_TABLE_H_
#define SEE_CUDA_GRAD_TABLE_H_

#include <cstdint>

#include "../../include/see_cuda.h"

namespace see::k {

constexpr uint32_t kGradThreads = 256;
constexpr uint32_t kGradEntries = 160;       // tensors a launch
constexpr uint32_t kGradBlocks = 4;          // to an SM
constexpr uint32_t kGradPartials = 1024;     // most thread blocks' sums

struct GradEntry {
  const uint8_t* g;
  uint8_t* out;
  uint64_t n, unit_end;   // elements; units, counted over the launch's tensors
  uint8_t type, wide;     // wide: out is aligned to 16 bytes as g is
};
struct GradTable {
  GradEntry entry[kGradEntries];
  uint64_t each;          // units to a block,
  uint32_t rest, count;   // and one more to the first `rest`; tensors
};

// The table of the next tensors from *next on.  *next is left at a tensor that has elements, or at `count`: a call before that always
// finds one, so that a table is never emptied in the search for more.
inline void FillGradTable(GradTable* table, const see_grad_tensor* tensors, uint64_t count, uint64_t* next) {
  table->count = 0;
  uint64_t units = 0;
  for (; *next < count; ++*next) {
    const see_grad_tensor& t = tensors[*next];
    if (t.n == 0) continue;
    if (table->count == kGradEntries) return;
    const uint64_t at = reinterpret_cast<uint64_t>(t.g) & 15;
    units += (at + t.n * (t.type == SEE_F32 ? 4 : 2) + 15) / 16;
    void* out = t.out ? t.out : t.g;
    table->entry[table->count++] = {static_cast<const uint8_t*>(t.g), static_cast<uint8_t*>(out), t.n, units, static_cast<uint8_t>(t.type),
                                    static_cast<uint8_t>(at == (reinterpret_cast<uint64_t>(out) & 15))};
  }
}

// Blocks, of a table that is not empty: four units to a thread at least.  Cuts the table's units into their ranges.
inline unsigned CutGradTable(GradTable& table, uint32_t sms) {
  const uint64_t units = table.entry[table.count - 1].unit_end, blocks = (units + 4 * kGradThreads - 1) / (4 * kGradThreads);
  const uint64_t most = sms * kGradBlocks < kGradPartials ? sms * kGradBlocks : kGradPartials, grid = blocks < most ? blocks : most;
  table.each = units / grid;
  table.rest = static_cast<uint32_t>(units % grid);
  return static_cast<unsigned>(grid);
}

// For each table in turn, its ranges cut: launch(table, blocks), until one of them returns something else than `ok`, which is returned.
// *tables: how many there were; of one, *table and *blocks are what was launched.
template <typename Error, typename F>
Error EachGradTable(GradTable* table, const see_grad_tensor* tensors, uint64_t count, uint32_t sms, Error ok, unsigned* tables, unsigned* blocks, F launch) {
  *tables = 0;
  for (uint64_t next = 0; next < count;) {
    FillGradTable(table, tensors, count, &next);
    if (table->count == 0) break;   // (no tensor has elements)
    *blocks = CutGradTable(*table, sms);
    ++*tables;
    if (Error e = launch(*table, *blocks); e != ok) return e;
  }
  return ok;
}

}  // namespace see::k

#endif  // SEE_CUDA_GRAD_TABLE_H_
