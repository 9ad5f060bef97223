// Rows that belong to groups of a block's threads: sums over a group, and rows that reach it through a ring in shared memory.
#ifndef SEE_CUDA_ROW_GROUPS_CUH_
#define SEE_CUDA_ROW_GROUPS_CUH_

#include <atomic>
#include <cstddef>
#include <cstdint>

#include "block_ops.h"
#include "kernels.h"
#include "umma_device.cuh"
#include "vec_types.cuh"

namespace see::k {

constexpr uint32_t kWideThreads = 768;                                // most threads of a block
constexpr size_t kRingBytes = 200 * 1024;                              // of a block

template <bool kBoth>
__device__ __forceinline__ float2 WarpSum(float2 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xFFFFFFFFu, v.x, o);
    if (kBoth) v.y += __shfl_xor_sync(0xFFFFFFFFu, v.y, o);
  }
  return v;
}

// The sums of a group's T threads, in all of them.  `slots`: two sets of 16 per block, used in turn, so that one barrier
// a sum is enough: who writes a set again has passed the barrier that the readers of its last use arrived at after it.
template <bool kBoth>   // or v.x alone
__device__ __forceinline__ float2 GroupSum(float2 v, uint32_t T, uint32_t group, float2 (*slots)[kWideThreads / 32], uint32_t& turn) {
  v = WarpSum<kBoth>(v);
  if (T == 32) return v;
  float2* set = slots[turn] + group * (T / 32);
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) set[(threadIdx.x - group * T) >> 5] = v;
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(T) : "memory");
  float2 sum = set[0];
  for (uint32_t w = 1; w < T / 32; ++w) {
    sum.x += set[w].x;
    if (kBoth) sum.y += set[w].y;
  }
  return sum;
}

// The same of one double.
__device__ __forceinline__ double GroupSum(double v, uint32_t T, uint32_t group, float2 (*slots)[kWideThreads / 32], uint32_t& turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  if (T == 32) return v;
  double* set = reinterpret_cast<double*>(slots[turn]) + group * (T / 32);
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) set[(threadIdx.x - group * T) >> 5] = v;
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(T) : "memory");
  double sum = set[0];
  for (uint32_t w = 1; w < T / 32; ++w) sum += set[w];
  return sum;
}

// The variance, from the average square of deviations from a mean that is off by `off`, their own average.  (What is not finite stays.)
__device__ __forceinline__ float Variance(float square, float off) {
  const float less = square - off * off;
  return !isfinite(off * off) ? square : less < 0.0f ? 0.0f : less;
}

// 8, 4 or 1 consecutive columns.
template <typename T, int VEC>
__device__ __forceinline__ void LoadCols(const T* p, float* v) {
  if constexpr (VEC == 8) {
    Load8<T>(p, v);
  } else if constexpr (VEC == 4 && sizeof(T) == 4) {
    const float4 r = *reinterpret_cast<const float4*>(p);
    v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
  } else if constexpr (VEC == 4) {
    const uint2 r = *reinterpret_cast<const uint2*>(p);
    Unpack2<T>(r.x, v[0], v[1]);
    Unpack2<T>(r.y, v[2], v[3]);
  } else {
    v[0] = ToF32(*p);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void StoreCols(T* p, const float* v) {
  if constexpr (VEC == 8) Store8<T>(p, v);
  else if constexpr (VEC == 4 && sizeof(T) == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  else if constexpr (VEC == 4) *reinterpret_cast<uint2*>(p) = make_uint2(Pack2<T>(v[0], v[1]), Pack2<T>(v[2], v[3]));
  else *p = FromF32<T>(v[0]);
}

__device__ __forceinline__ void GroupBarrier(uint32_t T, uint32_t group) {
  if (T == 32) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(T) : "memory");
}
// A bulk copy of this device's memory always lands; that nothing can wait for good even so, the wait is bounded, and a thread
// that ran out raises the flag and goes on (the others of its group count on it at their barriers).
__device__ __forceinline__ void AwaitRow(uint64_t* bar, uint32_t parity, DeviceStatus* status) {
  if (umma_dev::MbarWait(bar, parity)) return;
  status->wait_timeout = 1;
  umma_dev::DrainDelay();
}

// A bulk copy begins and ends on 16 bytes: a row of any alignment is copied with what lies beside it up to there.
template <typename T>
struct OddRow {
  const uint8_t* from;   // 16-byte aligned, at most 15 bytes before the row
  uint32_t skip, bytes;  // ... in front of it; to copy, a multiple of 16
  __device__ __forceinline__ OddRow(const void* base, uint64_t row, uint64_t stride, uint32_t cols) {
    const uint64_t at = reinterpret_cast<uint64_t>(static_cast<const T*>(base) + row * stride);
    skip = static_cast<uint32_t>(at & 15);
    from = reinterpret_cast<const uint8_t*>(at - skip);
    bytes = (skip + cols * static_cast<uint32_t>(sizeof(T)) + 15) & ~15u;
  }
};
template <typename T> __host__ __device__ constexpr uint32_t OddSlot(uint32_t cols) { return (cols * sizeof(T) + 45) / 16 * 16; }

// Element-wise, by the whole group; the caller synchronises.
template <typename T>
__device__ __forceinline__ void CopyRow(uint8_t* slot, const void* base, uint64_t row, uint64_t stride, uint32_t cols, uint32_t t, uint32_t threads) {
  const T* from = static_cast<const T*>(base) + row * stride;
  T* to = reinterpret_cast<T*>(slot + (reinterpret_cast<uint64_t>(from) & 15));
  for (uint32_t c = t; c < cols; c += threads) to[c] = from[c];
}

// A kernel's limit of shared memory is a device's: what has been granted is remembered for each (the call takes the driver a
// microsecond or two).
template <auto kKernel>
cudaError_t AllowShared(size_t bytes) {
  if (bytes > kMostShared) return cudaErrorInvalidValue;
  if (bytes <= 32 * 1024) return cudaSuccess;   // (the static part counts too)
  static std::atomic<size_t> granted[64] = {};
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
  if (dev >= 0 && dev < 64 && granted[dev].load(std::memory_order_acquire) >= bytes) return cudaSuccess;
  // (grants only grow: the most that any call asks for)
  if (cudaError_t e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMostShared)); e != cudaSuccess)
    return e;
  if (dev >= 0 && dev < 64) granted[dev].store(kMostShared, std::memory_order_release);
  return cudaSuccess;
}
}  // namespace see::k

#endif  // SEE_CUDA_ROW_GROUPS_CUH_
