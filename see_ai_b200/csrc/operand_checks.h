// Checks of device operands before anything is enqueued, shared by the operators that take the caller's own memory.
#ifndef SEE_CUDA_OPERAND_CHECKS_H_
#define SEE_CUDA_OPERAND_CHECKS_H_

#include <cuda_runtime.h>

#include <cstdint>
#include <expected>
#include <initializer_list>
#include <string>

#include "../../include/see_cuda.h"

namespace see {

using Status = std::expected<void, std::string>;

// The handle's device for the calls of a scope; the caller's current device is left as it was.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    ok_ = cudaGetDevice(&before_) == cudaSuccess && (before_ == device || cudaSetDevice(device) == cudaSuccess);
    moved_ = ok_ && before_ != device;
  }
  ~OnDevice() {
    if (moved_) cudaSetDevice(before_);
  }
  bool ok() const { return ok_; }

 private:
  int before_ = 0;
  bool ok_ = false, moved_ = false;
};

inline uint64_t SizeOfType(int type) { return type == SEE_F32 ? 4 : 2; }
inline bool IsType(int type) { return type == SEE_F32 || type == SEE_BF16 || type == SEE_F16; }

// `rows` runs of `width` bytes, `pitch` bytes apart.
struct Operand {
  const char* name;
  const void* p;
  uint64_t rows, width, pitch, align;
  bool written;
  uint64_t begin() const { return reinterpret_cast<uint64_t>(p); }
  uint64_t end() const { return rows ? begin() + (rows - 1) * pitch + width : begin(); }
};
inline Operand Vector(const char* name, const void* p, uint64_t bytes, uint64_t align, bool written) {
  return {name, p, bytes ? 1u : 0u, bytes, 0, align, written};
}

inline bool Overlap(const Operand& a, const Operand& b) {
  if (a.rows == 0 || b.rows == 0 || a.end() <= b.begin() || b.end() <= a.begin()) return false;
  if (a.rows > 1 && b.rows > 1 && a.pitch == b.pitch) {   // side by side in the rows of one buffer
    const uint64_t shift =
        b.begin() >= a.begin() ? (b.begin() - a.begin()) % a.pitch : (a.pitch - (a.begin() - b.begin()) % a.pitch) % a.pitch;
    if (shift >= a.width && shift + b.width <= a.pitch) return false;
  }
  return true;
}

// A call's operands, without allocation: these checks are part of calls of a few microseconds.
class Operands {
 public:
  Operands(std::initializer_list<Operand> list) {
    for (const Operand& o : list) Add(o);
  }
  void Add(const Operand& o) { ops_[count_++] = o; }
  // Null, misaligned, too large, or overlapping something that is written.
  Status Check(const char* what) const {
    auto refuse = [what](const std::string& why) { return std::unexpected(std::string(what) + ": " + why); };
    for (size_t i = 0; i < count_; ++i) {
      const Operand& o = ops_[i];
      if (o.rows == 0) continue;   // (no bytes: an empty allocation has no address)
      if (!o.p) return refuse(std::string(o.name) + " is null");
      if (o.begin() % o.align) return refuse(std::string(o.name) + " is not aligned");
      uint64_t span;
      if (__builtin_mul_overflow(o.rows, o.pitch, &span) || span > (1ull << 56) || o.width > (1ull << 56) || o.begin() > (1ull << 57))
        return refuse(std::string(o.name) + " is too large");
    }
    for (size_t i = 0; i < count_; ++i)
      for (size_t j = i + 1; j < count_; ++j)
        if ((ops_[i].written || ops_[j].written) && Overlap(ops_[i], ops_[j]))
          return refuse(std::string(ops_[i].name) + " and " + ops_[j].name + " overlap");
    return {};
  }

 private:
  Operand ops_[12];
  size_t count_ = 0;
};

}  // namespace see

#endif  // SEE_CUDA_OPERAND_CHECKS_H_
