// What the two passes of a block's join to the residual stream share.
#ifndef SEE_CUDA_JOIN_CUH_
#define SEE_CUDA_JOIN_CUH_

#include <initializer_list>

#include <type_traits>

#include "act_expr.cuh"
#include "block_ops.h"
#include "launch.cuh"
#include "row_groups.cuh"

namespace see::k {

// A thread's columns of one access: four as two pairs for the packed f32 instructions, or one as it is.
template <int VEC> using Lane = std::conditional_t<VEC == 1, float, f32x2>;
template <int VEC> constexpr int kLanes = VEC == 1 ? 1 : VEC / 2;
template <typename P> __device__ __forceinline__ P SplatOf(float v);
template <> __device__ __forceinline__ float SplatOf<float>(float v) { return v; }
template <> __device__ __forceinline__ f32x2 SplatOf<f32x2>(float v) { return Splat2(v); }
__device__ __forceinline__ float Add(float a, float b) { return a + b; }
__device__ __forceinline__ f32x2 Add(f32x2 a, f32x2 b) { return AddF2(a, b); }
__device__ __forceinline__ float Mul(float a, float b) { return a * b; }
__device__ __forceinline__ f32x2 Mul(f32x2 a, f32x2 b) { return Mul2(a, b); }
__device__ __forceinline__ float Fma(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ f32x2 Fma(f32x2 a, f32x2 b, f32x2 c) { return Fma2(a, b, c); }
__device__ __forceinline__ float Total(float a) { return a; }
__device__ __forceinline__ float Total(f32x2 a) {
  float lo, hi;
  UnpackF2(a, &lo, &hi);
  return lo + hi;
}
template <typename T, int VEC>
__device__ __forceinline__ void LoadLanes(const T* p, Lane<VEC> (&v)[kLanes<VEC>]) {
  float f[VEC];
  LoadCols<T, VEC>(p, f);
  if constexpr (VEC == 1) {
    v[0] = f[0];
  } else {
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) v[j] = PackF2(f[2 * j], f[2 * j + 1]);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void StoreLanes(T* p, const Lane<VEC> (&v)[kLanes<VEC>]) {
  float f[VEC];
  if constexpr (VEC == 1) {
    f[0] = v[0];
  } else {
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) UnpackF2(v[j], &f[2 * j], &f[2 * j + 1]);
  }
  StoreCols<T, VEC>(p, f);
}

// How many rows at either end of the matrices are not copied in bulk: rows whose 16-byte surroundings may lie outside.
inline uint32_t JoinEdge(const JoinArgs& a, std::initializer_list<const void*> x_like, std::initializer_list<const void*> y_like) {
  const uint64_t xs = a.x_type == SEE_F32 ? 4 : 2, ys = a.y_type == SEE_F32 ? 4 : 2;
  auto exact = [&](std::initializer_list<const void*> list, uint64_t size, uint64_t stride) {
    for (const void* p : list)
      if (p && (reinterpret_cast<uintptr_t>(p) & 15)) return false;
    return (a.cols * size & 15) == 0 && (stride * size & 15) == 0;
  };
  if (exact(x_like, xs, a.x_stride) && exact(y_like, ys, a.y_stride)) return 0;
  const uint64_t narrow = a.x_stride * xs < a.y_stride * ys ? a.x_stride * xs : a.y_stride * ys;
  return static_cast<uint32_t>((15 + narrow) / narrow);
}
// Four columns at a time: addresses and strides allow it everywhere.
inline bool JoinFours(const JoinArgs& a, std::initializer_list<const void*> x_like, std::initializer_list<const void*> y_like) {
  auto aligned = [](std::initializer_list<const void*> list, uintptr_t by) {
    for (const void* p : list)
      if (reinterpret_cast<uintptr_t>(p) & (by - 1)) return false;
    return true;
  };
  return a.cols % 4 == 0 && a.x_stride % 4 == 0 && a.y_stride % 4 == 0 && aligned(x_like, a.x_type == SEE_F32 ? 16 : 8) &&
         aligned(y_like, a.y_type == SEE_F32 ? 16 : 8);
}
inline uint32_t Warps(uint32_t n) { return (n + 31) / 32 * 32; }

// Groups of T threads with `slots` slots each, of what `budget` bytes hold; every SM gets rows before one gets two.
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
  slots = slots < 1 ? 1 : slots > 8 ? 8 : slots;
  if (slots > turns) slots = static_cast<uint32_t>(turns);
  const uint64_t grid = (rows + groups - 1) / groups;
  return {groups, slots, static_cast<uint32_t>(grid < most ? grid : most), groups * slots * (slot_bytes + 8) + weights};
}

// Up to kJoinRingCols columns, one launch; grid: the rows of partial sums that the backward pass leaves.
constexpr uint32_t kJoinRingCols = 8192;
cudaError_t JoinForwardRing(const JoinArgs& a, uint32_t sms, cudaStream_t s);
cudaError_t JoinBackwardRing(const JoinArgs& a, uint32_t sms, cudaStream_t s, uint32_t* grid);

}  // namespace see::k

#endif  // SEE_CUDA_JOIN_CUH_
