// What the two passes of a block's join to the residual stream share.
#ifndef SEE_CUDA_JOIN_CUH_
#define SEE_CUDA_JOIN_CUH_

#include <initializer_list>
#include <type_traits>

#include "act_expr.cuh"
#include "block_ops.h"
#include "join_ring.h"
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

// A row at an end of the matrix for the ring, without anything beside it: its 16-byte units are copied in bulk, the elements before and
// behind them (fewer than 16 bytes each) by the group's threads.  The row begins `skip` bytes into its slot.
template <typename T>
struct EndRow {
  const uint8_t* from;         // the units
  uint32_t skip, to, bytes;    // bytes into the slot; ... of the units
  uint32_t head, tail;         // elements before the units; the first one behind them
  __device__ __forceinline__ EndRow(const void* base, uint64_t row, uint64_t stride, uint32_t cols) {
    const uint64_t at = reinterpret_cast<uint64_t>(static_cast<const T*>(base) + row * stride), end = at + cols * sizeof(T);
    const uint64_t first = (at + 15) & ~15ull, last = end & ~15ull;
    skip = static_cast<uint32_t>(at & 15);
    from = reinterpret_cast<const uint8_t*>(first);
    to = skip == 0 ? 0 : 16;
    bytes = last > first ? static_cast<uint32_t>(last - first) : 0;
    head = bytes ? static_cast<uint32_t>(first - at) / sizeof(T) : cols;
    tail = bytes ? static_cast<uint32_t>(last - at) / sizeof(T) : cols;
  }
};
// The elements beside the units; the caller synchronises.
template <typename T>
__device__ __forceinline__ void CopyEnds(uint8_t* slot, const void* base, uint64_t row, uint64_t stride, uint32_t cols, uint32_t t, uint32_t threads) {
  const EndRow<T> r(base, row, stride, cols);
  const T* from = static_cast<const T*>(base) + row * stride;
  T* to = reinterpret_cast<T*>(slot + r.skip);
  for (uint32_t c = t; c < r.head; c += threads) to[c] = from[c];
  for (uint32_t c = r.tail + t; c < cols; c += threads) to[c] = from[c];
}

// Rows that begin and end on 16 bytes in every matrix: four columns at a time, and nothing beside them.
inline bool JoinFours(const JoinArgs& a, std::initializer_list<const void*> x_like, std::initializer_list<const void*> y_like) {
  auto exact = [&](std::initializer_list<const void*> list, uint64_t size, uint64_t stride) {
    for (const void* p : list)
      if (reinterpret_cast<uintptr_t>(p) & 15) return false;
    return (a.cols * size & 15) == 0 && (stride * size & 15) == 0;
  };
  return exact(x_like, a.x_type == SEE_F32 ? 4 : 2, a.x_stride) && exact(y_like, a.y_type == SEE_F32 ? 4 : 2, a.y_stride);
}
// Of others: how many rows at either end of the matrices are not copied with what lies beside them, for that may lie outside.
inline uint32_t JoinEdge(const JoinArgs& a) {
  const uint64_t x = a.x_stride * (a.x_type == SEE_F32 ? 4 : 2), y = a.y_stride * (a.y_type == SEE_F32 ? 4 : 2), narrow = x < y ? x : y;
  return static_cast<uint32_t>((15 + narrow) / narrow);
}
inline uint32_t Warps(uint32_t n) { return (n + 31) / 32 * 32; }

// Up to kJoinRingCols columns, one launch; grid: the rows of partial sums that the backward pass leaves.
cudaError_t JoinForwardRing(const JoinArgs& a, uint32_t sms, cudaStream_t s);
cudaError_t JoinBackwardRing(const JoinArgs& a, uint32_t sms, cudaStream_t s, uint32_t* grid);

}  // namespace see::k

#endif  // SEE_CUDA_JOIN_CUH_
