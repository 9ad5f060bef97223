// The norm over all elements of many tensors, the factor that clips them, and the clipped tensors.
//   norm = |grad_scale| (sum g^2)^1/2,   factor = grad_scale min(1, max_norm / norm),   out = g factor
// Bound by HBM: each gradient is read once, and once more (from L2, as far as it holds them) and written where it is clipped.
//
// The tensors are cut into chunks of 256 threads' 8 accesses of 16 bytes; a thread block takes every gridDim-th chunk.  A chunk's
// ends that are no whole 16 bytes are taken element by element.  A thread's squares of one chunk are summed in f32, 32 to 64 of them; where that sum is not
// finite or so small that squares may have been lost, they are summed again in double.  What is beyond is double: the blocks' sums
// meet in the workspace and are added in a fixed order.
#include <type_traits>

#include "block_ops.h"
#include "launch.cuh"
#include "vec_types.cuh"

namespace see::k {

namespace {

constexpr uint32_t kThreads = 256, kUnits = 8;                       // accesses of 16 bytes to a thread and chunk
constexpr uint32_t kChunkUnits = kThreads * kUnits;                  // 32 KB
constexpr uint32_t kEntries = 160;                                   // tensors a launch

struct GradEntry {
  const uint8_t* g;
  uint8_t* out;
  uint64_t n;
  uint32_t chunk_end;   // of the chunks of the launch, counted over its tensors
  uint8_t type, wide;   // wide: out is aligned to 16 bytes as g is
};
struct GradTable {
  GradEntry entry[kEntries];
  uint32_t count;
};

// One chunk's place: units of 16 bytes by address, of which the tensor's first and last may stick out of it.
struct Chunk {
  const GradEntry* e;
  uint64_t first;       // its first unit
  uint32_t units;       // at most kChunkUnits
};
__device__ __forceinline__ Chunk Find(const GradTable& t, uint32_t chunk) {
  uint32_t lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const uint32_t mid = (lo + hi) / 2;
    if (chunk < t.entry[mid].chunk_end) hi = mid;
    else lo = mid + 1;
  }
  const GradEntry& e = t.entry[lo];
  const uint32_t begin = lo ? t.entry[lo - 1].chunk_end : 0;
  const uint32_t size = e.type == SEE_F32 ? 4 : 2;
  const uint64_t units = ((reinterpret_cast<uint64_t>(e.g) & 15) + e.n * size + 15) / 16, first = static_cast<uint64_t>(chunk - begin) * kChunkUnits;
  return {&e, first, static_cast<uint32_t>(min(static_cast<uint64_t>(kChunkUnits), units - first))};
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
  __device__ __forceinline__ bool Whole(int64_t at) const { return at >= 0 && at + kPerUnit<T> <= static_cast<int64_t>(n); }
  // The unit's 16 bytes, zeros where it sticks out.
  __device__ __forceinline__ uint4 Load(uint64_t unit) const {
    const int64_t at = At(unit);
    if (Whole(at)) return *reinterpret_cast<const uint4*>(g + at);
    using Bits = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;
    const Bits* bits = reinterpret_cast<const Bits*>(g);
    uint32_t r[4] = {};
#pragma unroll
    for (int j = 0; j < kPerUnit<T>; ++j)
      if (at + j >= 0 && at + j < static_cast<int64_t>(n)) r[j * sizeof(T) / 4] |= static_cast<uint32_t>(bits[at + j]) << (j * sizeof(T) % 4 * 8);
    return make_uint4(r[0], r[1], r[2], r[3]);
  }
};

// Below this a sum of f32 squares may have lost a part of itself (their own rounding ends at 2^-149).
constexpr float kSmallSum = 1e-28f;

template <typename T>
__device__ __forceinline__ double ChunkSquares(const Chunk& c) {
  const Tensor<T> t(*c.e);
  uint4 r[kUnits];
#pragma unroll
  for (uint32_t i = 0; i < kUnits; ++i) {
    const uint32_t u = threadIdx.x + i * kThreads;
    r[i] = u < c.units ? t.Load(c.first + u) : make_uint4(0, 0, 0, 0);
  }
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
  double wide = 0.0;
#pragma unroll 1
  for (uint32_t i = 0; i < kUnits; ++i) {   // (asked for again: rare, and the registers stay few)
    const uint32_t u = threadIdx.x + i * kThreads;
    if (u >= c.units) break;
    Elements<T>(t.Load(c.first + u), v);
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

// partials[block] = the squares of the block's chunks, added to what is there unless `first`.
__global__ void __launch_bounds__(kThreads)
GradSquaresKernel(const __grid_constant__ GradTable table, double* __restrict__ partials, int first) {
  AwaitPrevious();
  __shared__ double slots[kThreads / 32];
  const uint32_t chunks = table.entry[table.count - 1].chunk_end;
  double sum = 0.0;
  for (uint32_t i = blockIdx.x; i < chunks; i += gridDim.x) {
    const Chunk c = Find(table, i);
    sum += c.e->type == SEE_F32 ? ChunkSquares<float>(c) : c.e->type == SEE_BF16 ? ChunkSquares<Bf16>(c) : ChunkSquares<F16>(c);
  }
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
__device__ __forceinline__ void ScaleChunk(const Chunk& c, float by) {
  const Tensor<T> t(*c.e);
  T* out = reinterpret_cast<T*>(c.e->out);
  uint4 r[kUnits];
#pragma unroll
  for (uint32_t i = 0; i < kUnits; ++i)
    if (threadIdx.x + i * kThreads < c.units) r[i] = t.Load(c.first + threadIdx.x + i * kThreads);
#pragma unroll
  for (uint32_t i = 0; i < kUnits; ++i) {
    const uint32_t u = threadIdx.x + i * kThreads;
    if (u >= c.units) continue;
    const int64_t at = t.At(c.first + u);
    float v[kPerUnit<T>];
    Elements<T>(r[i], v);
#pragma unroll
    for (int j = 0; j < kPerUnit<T>; ++j) v[j] *= by;
    if (c.e->wide && t.Whole(at)) {
      if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(out + at) = make_float4(v[0], v[1], v[2], v[3]);
      else Store8<T>(out + at, v);
    } else {
#pragma unroll
      for (int j = 0; j < kPerUnit<T>; ++j)
        if (at + j >= 0 && at + j < static_cast<int64_t>(t.n)) out[at + j] = FromF32<T>(v[j]);
    }
  }
}

// Every block makes the factor itself, from the same sums in the same order.
__global__ void __launch_bounds__(kThreads)
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
  const uint32_t chunks = table.entry[table.count - 1].chunk_end;
  for (uint32_t i = blockIdx.x; i < chunks; i += gridDim.x) {
    const Chunk c = Find(table, chunks - 1 - i);   // what was read last is in L2
    if (c.e->out == c.e->g && by == 1.0f) continue;
    if (c.e->type == SEE_F32) ScaleChunk<float>(c, by);
    else if (c.e->type == SEE_BF16) ScaleChunk<Bf16>(c, by);
    else ScaleChunk<F16>(c, by);
  }
}

// The table of the next tensors from `next` on; false: none are left.
bool Fill(GradTable* table, const see_grad_tensor* tensors, uint64_t count, uint64_t* next) {
  table->count = 0;
  uint64_t chunks = 0;
  for (; *next < count && table->count < kEntries; ++*next) {
    const see_grad_tensor& t = tensors[*next];
    if (t.n == 0) continue;
    const uint64_t at = reinterpret_cast<uint64_t>(t.g) & 15, units = (at + t.n * (t.type == SEE_F32 ? 4 : 2) + 15) / 16;
    const uint64_t more = (units + kChunkUnits - 1) / kChunkUnits;
    if (chunks + more > 0x7FFFFFFFull) break;   // (one tensor alone has at most 2^25)
    chunks += more;
    void* out = t.out ? t.out : t.g;
    table->entry[table->count++] = {static_cast<const uint8_t*>(t.g), static_cast<uint8_t*>(out), t.n, static_cast<uint32_t>(chunks),
                                    static_cast<uint8_t>(t.type), static_cast<uint8_t>(at == (reinterpret_cast<uint64_t>(out) & 15))};
  }
  return table->count != 0;
}
unsigned Grid(const GradTable& table, uint32_t sms) {
  const uint32_t chunks = table.entry[table.count - 1].chunk_end, most = sms * 6 < kGradPartials ? sms * 6 : kGradPartials;
  return chunks < most ? chunks : most;
}

}  // namespace

cudaError_t GradNorm(const see_grad_tensor* tensors, uint64_t count, bool clip, float max_norm, const float* grad_scale, float* norm,
                     float* factor, double* partials, uint32_t sms, cudaStream_t s, int* launches) {
  GradTable table;
  uint64_t next = 0;
  unsigned used = 0;   // partial sums
  while (Fill(&table, tensors, count, &next)) {
    const unsigned grid = Grid(table, sms);
    // (blocks that an earlier launch had are added to; those that it had not are new)
    if (used != 0 && grid > used) {
      if (cudaError_t e = cudaMemsetAsync(partials + used, 0, (grid - used) * sizeof(double), s); e != cudaSuccess) return e;
    }
    if (cudaError_t e = Next(GradSquaresKernel, grid, kThreads, 0, s)(table, partials, used == 0 ? 1 : 0); e != cudaSuccess) return e;
    ++*launches;
    used = used > grid ? used : grid;
  }
  if (!clip || used == 0) {
    ++*launches;
    return Next(GradFactorKernel, 1, kThreads, 0, s)(static_cast<const double*>(partials), used, max_norm, grad_scale, norm, factor);
  }
  next = 0;
  while (Fill(&table, tensors, count, &next)) {
    if (cudaError_t e = Next(GradScaleKernel, Grid(table, sms), kThreads, 0, s)(table, static_cast<const double*>(partials), used, max_norm, grad_scale,
                                                                                 norm, factor);
        e != cudaSuccess)
      return e;
    ++*launches;
  }
  return cudaSuccess;
}

}  // namespace see::k
