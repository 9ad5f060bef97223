// A handle without a plan: its status word for a wait that ran out is set from the host, as a kernel would set it, and flushes
// follow.  One line each: the flush's message, or "ok".  Built and read by test_gpu_unbound_flush.py.
#include <cstdio>

#include "../see_ai_b200/csrc/cuda_backend.h"

namespace see {
struct DeviceStatusAccess {
  static void RaiseWaitTimeout(CudaBackend& b) {
    uint32_t* one = b.h_published_ + 512;   // pinned, behind what a flush publishes
    *one = 1;
    k::StageFromHost({&b.d_status_->wait_timeout, one, 4}, {}, b.stream());
  }
};
}  // namespace see

int main() {
  auto made = see::CudaBackend::Create(0);
  if (!made) return std::printf("%s\n", made.error().c_str()), 1;
  see::CudaBackend& b = **made;
  auto flush = [&] {
    const see::Status s = b.Flush();
    std::printf("%s\n", s ? "ok" : s.error().c_str());
  };
  flush();
  see::DeviceStatusAccess::RaiseWaitTimeout(b);
  flush();
  flush();
  return 0;
}
