// How the rows of a block's join reach the groups of a thread block: the sizes of its ring in shared memory.
#ifndef SEE_CUDA_JOIN_RING_H_
#define SEE_CUDA_JOIN_RING_H_

#include <cstddef>
#include <cstdint>

#include "block_ops.h"

namespace see::k {

constexpr uint32_t kJoinRingCols = 8192;   // of wider rows a block holds none
constexpr uint32_t kJoinMostSlots = 8;     // to a group
constexpr size_t kJoinBarrier = 8;         // bytes, beside each slot

// Groups of T threads with `slots` slots each, of what a block's shared memory holds beside the weights; every SM gets rows before one
// gets two.
struct JoinRing {
  uint32_t groups, slots, grid;
  size_t bytes;
};
inline JoinRing RingOf(uint64_t rows, uint32_t threads, uint32_t T, size_t slot_bytes, size_t weights, uint32_t sms) {
  const size_t budget = kMostShared - 1024 - weights;
  const uint64_t most = sms < kNormPartials ? sms : kNormPartials, each = (rows + most - 1) / most;
  uint32_t groups = threads / T;
  if (groups > each) groups = static_cast<uint32_t>(each);
  while (groups > 1 && 2 * groups * slot_bytes > budget) --groups;   // two slots to a group, unless it is alone
  uint32_t slots = static_cast<uint32_t>(budget / (groups * slot_bytes));
  const uint64_t turns = (rows + most * groups - 1) / (most * groups);
  slots = slots < 1 ? 1 : slots > kJoinMostSlots ? kJoinMostSlots : slots;
  if (slots > turns) slots = static_cast<uint32_t>(turns);
  // (the 1024 bytes hold 128 barriers: all that 16 groups can have, not all of 24)
  while (slots > 1 && groups * slots * (slot_bytes + kJoinBarrier) + weights > kMostShared) --slots;
  const uint64_t grid = (rows + groups - 1) / groups;
  return {groups, slots, static_cast<uint32_t>(grid < most ? grid : most), groups * slots * (slot_bytes + kJoinBarrier) + weights};
}

}  // namespace see::k

#endif  // SEE_CUDA_JOIN_RING_H_
