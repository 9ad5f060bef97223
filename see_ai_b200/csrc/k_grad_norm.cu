// The norm over all elements of many tensors, the factor that clips them, and the clipped tensors.
//   norm = |grad_scale| (sum g^2)^1/2,   factor = grad_scale min(1, max_norm / norm),   out = g factor
// Bound by HBM: each gradient is read once, and once more (from L2, as far as it holds them) and written where it is clipped.
//
// All tensors' units of 16 bytes, one tensor behind the other, are cut into equal ranges, one to a thread block, which walks its own
// eight accesses to a thread at a time.  (Chunks of 32 KB taken in turn: 43 us for 87 million elements of bf16, for a last round of few
// chunks.)  Units that are no whole 16 bytes of their tensor are taken element by element.  A thread's squares of one step are summed in
// f32, 32 to 64 of them; where that sum is not finite or so small that squares may have been lost, they are summed again in double.
// What is beyond is double: the blocks' sums meet in the workspace and are added in a fixed order.
#include "block_ops.h"
#include "grad_table.h"
#include "launch.cuh"
#include "vec_types.cuh"

namespace see::k {

namespace {

constexpr uint32_t kThreads = kGradThreads, kUnits = 8, kStep = kThreads * kUnits;   // units to a thread, and to a block, at a time

// Calls step(entry, first unit, units) for all of a block's range, or, of kBack, from its end on.
template <bool kBack, typename F>
__device__ __forceinline__ void Walk(const GradTable& t, F step) {
  const uint64_t each = t.each, rest = t.rest, b = kBack ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
  const uint64_t begin = b * each + min(b, rest), end = begin + each + (b < rest);
  if (begin == end) return;
  uint32_t lo = 0, hi = t.count - 1;   // the tensor of the first unit, or the last
  const uint64_t at = kBack ? end - 1 : begin;
  while (lo < hi) {
    const uint32_t mid = (lo + hi) / 2;
    if (at < t.entry[mid].unit_end) hi = mid;
    else lo = mid + 1;
  }
  if constexpr (!kBack) {
    for (uint64_t from = begin; from < end; ++lo) {
      const GradEntry& e = t.entry[lo];
      const uint64_t base = lo ? t.entry[lo - 1].unit_end : 0, to = min(end, e.unit_end);
      for (; from < to; from += kStep) step(e, from - base, static_cast<uint32_t>(min(static_cast<uint64_t>(kStep), to - from)));
      from = to;
    }
  } else {
    for (uint64_t to = end; to > begin; --lo) {
      const GradEntry& e = t.entry[lo];
      const uint64_t base = lo ? t.entry[lo - 1].unit_end : 0, from = max(begin, base);
      while (to > from) {
        const uint32_t units = static_cast<uint32_t>(min(static_cast<uint64_t>(kStep), to - from));
        to -= units;
        step(e, to - base, units);
      }
    }
  }
}

template <typename T> constexpr int kPerUnit = 16 / sizeof(T);

// The values of 16 bytes.
template <typename T>
__device__ __forceinline__ void Elements(uint4 r, float* v) {
  if constexpr (sizeof(T) == 4) {
    v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
  } else {
    Unpack2<T>(r.x, v[0], v[1]);
    Unpack2<T>(r.y, v[2], v[3]);
    Unpack2<T>(r.z, v[4], v[5]);
    Unpack2<T>(r.w, v[6], v[7]);
  }
}
template <typename T>
struct Tensor {
  const T* g;          // element 0
  uint32_t skip;       // elements of its first unit in front of it
  uint64_t n;
  __device__ __forceinline__ explicit Tensor(const GradEntry& e)
      : g(reinterpret_cast<const T*>(e.g)), skip(static_cast<uint32_t>((reinterpret_cast<uint64_t>(e.g) & 15) / sizeof(T))), n(e.n) {}
  __device__ __forceinline__ int64_t At(uint64_t unit) const { return static_cast<int64_t>(unit * kPerUnit<T>) - skip; }
  // Whether these units lie wholly in the tensor.
  __device__ __forceinline__ bool Whole(uint64_t unit, uint64_t units) const {
    return (unit != 0 || skip == 0) && At(unit + units) <= static_cast<int64_t>(n);
  }
  __device__ __forceinline__ const uint4* Units(uint64_t unit) const { return reinterpret_cast<const uint4*>(g + At(unit)); }
  template <typename F>
  __device__ __forceinline__ void EachOf(uint64_t unit, F f) const {   // f(element) for a unit's elements in the tensor
    const int64_t at = At(unit), end = min(at + kPerUnit<T>, static_cast<int64_t>(n));
    for (int64_t i = max(at, static_cast<int64_t>(0)); i < end; ++i) f(i);
  }
};

// Below this a sum of f32 squares may have lost a part of itself (their own rounding ends at 2^-149).
constexpr float kSmallSum = 1e-28f;

template <typename T>
__device__ __forceinline__ double Squares(const GradEntry& e, uint64_t first, uint32_t units) {
  const Tensor<T> t(e);
  double wide = 0.0;
  if (!t.Whole(first, units)) {   // a tensor's first or last step, where it begins or ends within 16 bytes
#pragma unroll 1
    for (uint32_t u = threadIdx.x; u < units; u += kThreads)
      t.EachOf(first + u, [&](int64_t i) {
        const double v = static_cast<double>(ToF32(t.g[i]));
        wide = fma(v, v, wide);
      });
    return wide;
  }
  const uint4* from = t.Units(first) + threadIdx.x;
  uint4 r[kUnits];
#pragma unroll
  for (uint32_t i = 0; i < kUnits; ++i) r[i] = threadIdx.x + i * kThreads < units ? from[i * kThreads] : make_uint4(0, 0, 0, 0);
  float sum = 0.0f, v[kPerUnit<T>];
#pragma unroll
  for (uint32_t i = 0; i < kUnits; ++i) {
    Elements<T>(r[i], v);
    float part = 0.0f;
#pragma unroll
    for (int j = 0; j < kPerUnit<T>; ++j) part = fmaf(v[j], v[j], part);
    sum += part;
  }
  if (sum >= kSmallSum && sum < __int_as_float(0x7F800000)) return static_cast<double>(sum);
#pragma unroll 1
  for (uint32_t u = threadIdx.x; u < units; u += kThreads) {   // (asked for again: rare, and the registers stay few)
    Elements<T>(t.Units(first)[u], v);
#pragma unroll
    for (int j = 0; j < kPerUnit<T>; ++j) wide = fma(static_cast<double>(v[j]), static_cast<double>(v[j]), wide);
  }
  return wide;
}

__device__ __forceinline__ double WarpSum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
// The sum of all threads' v, in every one; `slots` is free again after the caller's next barrier.
__device__ __forceinline__ double BlockSum(double v, double (&slots)[kThreads / 32]) {
  v = WarpSum(v);
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
  __syncthreads();
  double sum = slots[0];
#pragma unroll
  for (uint32_t w = 1; w < kThreads / 32; ++w) sum += slots[w];
  return sum;
}

// partials[block] = the squares of the block's range, added to what is there unless `first`.
__global__ void __launch_bounds__(kThreads, kGradBlocks)
GradSquaresKernel(const __grid_constant__ GradTable table, double* __restrict__ partials, int first) {
  AwaitPrevious();
  __shared__ double slots[kThreads / 32];
  double sum = 0.0;
  Walk<false>(table, [&](const GradEntry& e, uint64_t from, uint32_t units) {
    sum += e.type == SEE_F32 ? Squares<float>(e, from, units) : e.type == SEE_BF16 ? Squares<Bf16>(e, from, units) : Squares<F16>(e, from, units);
  });
  sum = BlockSum(sum, slots);
  if (threadIdx.x == 0) partials[blockIdx.x] = first ? sum : partials[blockIdx.x] + sum;
}

// The blocks' sums to norm and factor, by a block's threads; all of them get the factor.
__device__ __forceinline__ float Factor(const double* __restrict__ partials, uint32_t count, float max_norm, const float* __restrict__ grad_scale,
                                        double (&slots)[kThreads / 32], float* norm_out) {
  double sum = 0.0;
  for (uint32_t i = threadIdx.x; i < count; i += kThreads) sum += partials[i];
  const double scale = grad_scale ? static_cast<double>(*grad_scale) : 1.0;
  const double norm = sqrt(BlockSum(sum, slots)) * fabs(scale), most = static_cast<double>(max_norm);
  *norm_out = static_cast<float>(norm);
  return static_cast<float>(scale * (norm <= most || norm == 0.0 ? 1.0 : most / norm));
}

__global__ void __launch_bounds__(kThreads)
GradFactorKernel(const double* __restrict__ partials, uint32_t count, float max_norm, const float* __restrict__ grad_scale,
                 float* __restrict__ norm, float* __restrict__ factor) {
  AwaitPrevious();
  __shared__ double slots[kThreads / 32];
  float n;
  const float f = Factor(partials, count, max_norm, grad_scale, slots, &n);
  if (threadIdx.x == 0) {
    *norm = n;
    *factor = f;
  }
}

template <typename T>
__device__ __forceinline__ void Scale(const GradEntry& e, uint64_t first, uint32_t units, float by) {
  const Tensor<T> t(e);
  T* out = reinterpret_cast<T*>(e.out);
  if (!e.wide || !t.Whole(first, units)) {
#pragma unroll 1
    for (uint32_t u = threadIdx.x; u < units; u += kThreads) t.EachOf(first + u, [&](int64_t i) { out[i] = FromF32<T>(ToF32(t.g[i]) * by); });
    return;
  }
  const uint4* from = t.Units(first) + threadIdx.x;
  uint4* to = reinterpret_cast<uint4*>(out + t.At(first)) + threadIdx.x;
  uint4 r[kUnits];
#pragma unroll
  for (uint32_t i = 0; i < kUnits; ++i) r[i] = threadIdx.x + i * kThreads < units ? from[i * kThreads] : make_uint4(0, 0, 0, 0);
#pragma unroll
  for (uint32_t i = 0; i < kUnits; ++i) {
    float v[kPerUnit<T>];
    Elements<T>(r[i], v);
#pragma unroll
    for (int j = 0; j < kPerUnit<T>; ++j) v[j] *= by;
    if constexpr (sizeof(T) == 4) r[i] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    else r[i] = make_uint4(Pack2<T>(v[0], v[1]), Pack2<T>(v[2], v[3]), Pack2<T>(v[4], v[5]), Pack2<T>(v[6], v[7]));
    if (threadIdx.x + i * kThreads < units) to[i * kThreads] = r[i];
  }
}

// Every block makes the factor itself, from the same sums in the same order; then from the end on, for what was read last is in L2.
__global__ void __launch_bounds__(kThreads, kGradBlocks)
GradScaleKernel(const __grid_constant__ GradTable table, const double* __restrict__ partials, uint32_t count, float max_norm,
                const float* __restrict__ grad_scale, float* __restrict__ norm, float* __restrict__ factor) {
  AwaitPrevious();
  __shared__ double slots[kThreads / 32];
  float n;
  const float by = Factor(partials, count, max_norm, grad_scale, slots, &n);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    *norm = n;
    *factor = by;
  }
  Walk<true>(table, [&](const GradEntry& e, uint64_t from, uint32_t units) {
    if (e.out == e.g && by == 1.0f) return;
    if (e.type == SEE_F32) Scale<float>(e, from, units, by);
    else if (e.type == SEE_BF16) Scale<Bf16>(e, from, units, by);
    else Scale<F16>(e, from, units, by);
  });
}

}  // namespace

cudaError_t GradNorm(const see_grad_tensor* tensors, uint64_t count, bool clip, float max_norm, const float* grad_scale, float* norm,
                     float* factor, double* partials, uint32_t sms, cudaStream_t s, int* launches) {
  GradTable table;
  unsigned used = 0, blocks = 0, tables = 0;   // used: partial sums
  cudaError_t e = EachGradTable(&table, tensors, count, sms, cudaSuccess, &tables, &blocks, [&](const GradTable& t, unsigned grid) {
    // (blocks that an earlier launch had are added to; those that it had not are new)
    if (used != 0 && grid > used) {
      if (cudaError_t e = cudaMemsetAsync(partials + used, 0, (grid - used) * sizeof(double), s); e != cudaSuccess) return e;
    }
    ++*launches;
    const int first = used == 0 ? 1 : 0;
    used = used > grid ? used : grid;
    return Next(GradSquaresKernel, grid, kThreads, 0, s)(t, partials, first);
  });
  if (e != cudaSuccess) return e;
  if (!clip || used == 0) {
    ++*launches;
    return Next(GradFactorKernel, 1, kThreads, 0, s)(static_cast<const double*>(partials), used, max_norm, grad_scale, norm, factor);
  }
  auto scale = [&](const GradTable& t, unsigned grid) {
    ++*launches;
    return Next(GradScaleKernel, grid, kThreads, 0, s)(t, static_cast<const double*>(partials), used, max_norm, grad_scale, norm, factor);
  };
  if (tables == 1) return scale(table, blocks);   // (the table is there)
  return EachGradTable(&table, tensors, count, sms, cudaSuccess, &tables, &blocks, scale);
}

}  // namespace see::k
