// Layer norm and root-mean-square norm of rows in f32, bf16 or f16, and their backward pass with the gradients of the
// weights.  With u = (x - mean) rstd (rms: mean = 0), q = dy gamma and <.> a row's average:
//   y = u gamma + beta,   dx = rstd (q - <q> - u <q u>) (+ addend),   dgamma = sum over rows of dy u,   dbeta = of dy
// (rms: neither beta nor <q>).  Bound by HBM: each matrix is read or written once.
//
// A row belongs to a group of T threads (a multiple of 32), which hold it in registers, eight consecutive columns at a
// time where widths, strides and addresses allow 16-byte accesses and single columns T apart otherwise; a block has as
// many groups as fit into 512 threads.  A thread has the same columns in every row, so that the backward pass sums dgamma
// and dbeta over a block's rows in registers; the groups meet in shared memory, the blocks (at most two to an SM) in
// NormFoldKernel, both in an order that the sizes alone fix.
//
// All sums are f32.  The forward pass takes the mean twice: the second pass over the registers sums the deviations from
// the first result, which corrects it, beside their squares, so rows far from zero lose nothing to cancellation.
#include "block_ops.h"
#include "launch.cuh"
#include "vec_types.cuh"

namespace see::k {

namespace {

constexpr uint32_t kNormThreads = 512;

__device__ __forceinline__ float2 WarpSum2(float2 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xFFFFFFFFu, v.x, o);
    v.y += __shfl_xor_sync(0xFFFFFFFFu, v.y, o);
  }
  return v;
}

// The sums of a group's T threads, in all of them.  `slots`: two sets of 16 per block, used in turn, so that one barrier
// a sum is enough: who writes a set again has passed the barrier that the readers of its last use arrived at after it.
__device__ __forceinline__ float2 GroupSum(float2 v, uint32_t T, uint32_t group, float2 (*slots)[kNormThreads / 32], uint32_t& turn) {
  v = WarpSum2(v);
  if (T == 32) return v;
  float2* set = slots[turn] + group * (T / 32);
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) set[(threadIdx.x - group * T) >> 5] = v;
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(T) : "memory");
  float2 sum = set[0];
  for (uint32_t w = 1; w < T / 32; ++w) {
    sum.x += set[w].x;
    sum.y += set[w].y;
  }
  return sum;
}

template <typename T, int VEC>
__device__ __forceinline__ void LoadCols(const T* p, float* v) {
  if constexpr (VEC == 8) Load8<T>(p, v);
  else v[0] = ToF32(*p);
}
template <typename T, int VEC>
__device__ __forceinline__ void StoreCols(T* p, const float* v) {
  if constexpr (VEC == 8) Store8<T>(p, v);
  else *p = FromF32<T>(v[0]);
}

template <typename XT, typename YT, bool kRms, int VEC, int NV>
__global__ void __launch_bounds__(kNormThreads)
NormFwdKernel(const __grid_constant__ NormArgs a, uint32_t T) {
  __shared__ float2 slots[2][kNormThreads / 32];
  AwaitPrevious();
  const uint32_t group = threadIdx.x / T, t = threadIdx.x - group * T;
  const uint64_t row = static_cast<uint64_t>(blockIdx.x) * (blockDim.x / T) + group;
  if (row >= a.rows) return;
  const XT* x = static_cast<const XT*>(a.x) + row * a.x_stride;
  uint32_t turn = 0;
  float v[NV][VEC];
  float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t c = (t + i * T) * VEC;
    if (c < a.cols) {
      LoadCols<XT, VEC>(x + c, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum.x += kRms ? v[i][j] * v[i][j] : v[i][j];
  }
  sum = GroupSum(sum, T, group, slots, turn);
  const float per_col = 1.0f / static_cast<float>(a.cols);
  float mean = 0.0f, var;
  if constexpr (kRms) {
    var = sum.x * per_col;
  } else {
    mean = sum.x * per_col;
    sum = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((t + i * T) * VEC < a.cols) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float d = v[i][j] - mean;
          sum.x += d;
          sum.y += d * d;
        }
      }
    sum = GroupSum(sum, T, group, slots, turn);
    const float shift = sum.x * per_col;
    if (isfinite(shift)) mean += shift;
    var = fmaxf(sum.y * per_col - shift * shift, 0.0f);
    if (!isfinite(sum.y)) var = sum.y;   // (fmaxf drops a NaN)
  }
  const float rstd = 1.0f / sqrtf(var + a.eps);
  if (t == 0) {
    a.rstd[row] = rstd;
    if (!kRms) a.mean[row] = mean;
  }
  YT* y = static_cast<YT*>(a.y) + row * a.y_stride;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t c = (t + i * T) * VEC;
    if (c < a.cols) {
      float g[VEC], b[VEC];
      LoadCols<float, VEC>(a.gamma + c, g);
      if (!kRms) LoadCols<float, VEC>(a.beta + c, b);
#pragma unroll
      for (int j = 0; j < VEC; ++j) g[j] = kRms ? v[i][j] * rstd * g[j] : (v[i][j] - mean) * rstd * g[j] + b[j];
      StoreCols<YT, VEC>(y + c, g);
    }
  }
}

// One row of partial sums a block; a lone block writes the gradients themselves.
template <typename XT, typename YT, bool kRms, int VEC, int NV>
__global__ void __launch_bounds__(kNormThreads, 1)
NormBwdKernel(const __grid_constant__ NormArgs a, uint32_t T) {
  extern __shared__ float meet[];   // [groups][cols]
  __shared__ float2 slots[2][kNormThreads / 32];
  AwaitPrevious();
  const uint32_t groups = blockDim.x / T, group = threadIdx.x / T, t = threadIdx.x - group * T;
  const float per_col = 1.0f / static_cast<float>(a.cols);
  uint32_t turn = 0;
  float sum_g[NV][VEC], sum_b[kRms ? 1 : NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      sum_g[i][j] = 0.0f;
      if (!kRms) sum_b[i][j] = 0.0f;
    }
  for (uint64_t row = static_cast<uint64_t>(blockIdx.x) * groups + group; row < a.rows; row += static_cast<uint64_t>(gridDim.x) * groups) {
    const XT* x = static_cast<const XT*>(a.x) + row * a.x_stride;
    const YT* dy = static_cast<const YT*>(a.dy) + row * a.y_stride;
    float u[NV][VEC], d[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (t + i * T) * VEC;
      if (c < a.cols) {
        LoadCols<XT, VEC>(x + c, u[i]);
        LoadCols<YT, VEC>(dy + c, d[i]);
      }
    }
    const float rstd = a.rstd[row], mean = kRms ? 0.0f : a.mean[row];
    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (t + i * T) * VEC;
      if (c < a.cols) {
        float g[VEC];
        LoadCols<float, VEC>(a.gamma + c, g);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          u[i][j] = (u[i][j] - mean) * rstd;
          sum_g[i][j] += d[i][j] * u[i][j];
          if (!kRms) sum_b[i][j] += d[i][j];
          d[i][j] *= g[j];
          sum.x += d[i][j] * u[i][j];
          if (!kRms) sum.y += d[i][j];
        }
      }
    }
    sum = GroupSum(sum, T, group, slots, turn);
    sum.x *= per_col;
    sum.y *= per_col;
    XT* dx = static_cast<XT*>(a.dx) + row * a.x_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (t + i * T) * VEC;
      if (c < a.cols) {
        float v[VEC];
        if (a.addend) LoadCols<XT, VEC>(static_cast<const XT*>(a.addend) + row * a.x_stride + c, v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float r = rstd * (kRms ? d[i][j] - u[i][j] * sum.x : d[i][j] - sum.y - u[i][j] * sum.x);
          v[j] = a.addend ? r + v[j] : r;
        }
        StoreCols<XT, VEC>(dx + c, v);
      }
    }
  }
  float* out_g = gridDim.x == 1 ? a.dgamma : a.partials + static_cast<size_t>(blockIdx.x) * a.cols;
  float* out_b = gridDim.x == 1 ? a.dbeta : a.partials + static_cast<size_t>(gridDim.x + blockIdx.x) * a.cols;
#pragma unroll
  for (int which = 0; which < (kRms ? 1 : 2); ++which) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (t + i * T) * VEC;
      if (c < a.cols) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) meet[group * a.cols + c + j] = which ? sum_b[kRms ? 0 : i][j] : sum_g[i][j];
      }
    }
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
      float s = meet[c];
      for (uint32_t r = 1; r < groups; ++r) s += meet[r * a.cols + c];
      (which ? out_b : out_g)[c] = s;
    }
  }
}

// The blocks' partial sums of 32 columns: warp w of a block adds rows w, w + 32, ...; then the warps' sums in order.
__global__ void __launch_bounds__(1024)
NormFoldKernel(const float* __restrict__ partials, float* __restrict__ dgamma, float* __restrict__ dbeta, uint32_t blocks, uint32_t cols) {
  __shared__ float meet[32][33];
  AwaitPrevious();
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  const float* p = partials + static_cast<size_t>(blockIdx.y) * blocks * cols;
  float s = 0.0f;
  if (c < cols)
#pragma unroll 4
    for (uint32_t r = warp; r < blocks; r += 32) s += p[static_cast<size_t>(r) * cols + c];
  meet[warp][lane] = s;
  __syncthreads();
  s = meet[lane][warp];   // column `warp` of the block's 32, one warp's sum a lane
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  const uint32_t col = blockIdx.x * 32 + warp;
  if (lane == 0 && col < cols) (blockIdx.y ? dbeta : dgamma)[col] = s;
}

bool Vec8Able(const NormArgs& a, bool backward) {
  auto ok = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  return a.cols % 8 == 0 && a.x_stride % 8 == 0 && a.y_stride % 8 == 0 && ok(a.x) && ok(a.gamma) &&
         (backward ? ok(a.dy) && ok(a.dx) && ok(a.addend) : ok(a.y) && ok(a.beta));
}

// Threads of a row and registers of a thread.  A row of up to 1024 columns is a warp's, so its sums need no barrier;
// wider ones have 16 columns a thread (8 where single), as much as leaves room for two such rows and their sums.
struct NormShape { uint32_t T; int nv; };
NormShape ShapeOf(uint32_t cols, bool vec) {
  const uint32_t n = vec ? cols / 8 : cols;
  auto up = [](uint32_t v) { return (v + 31) / 32 * 32; };
  if (vec) {
    if (n <= 128) return {32, static_cast<int>((n + 31) / 32)};
    return n <= 1024 ? NormShape{up((n + 1) / 2), 2} : NormShape{up((n + 3) / 4), 4};
  }
  if (n <= 4096) return {up((n + 7) / 8), 8};
  return n <= 8192 ? NormShape{up((n + 15) / 16), 16} : NormShape{up((n + 31) / 32), 32};
}

template <typename XT, typename YT, bool kRms, int VEC, int NV>
cudaError_t Run(const NormArgs& a, uint32_t T, bool backward, uint32_t sms, cudaStream_t s, int* launches) {
  const uint32_t groups = kNormThreads / T;
  const uint64_t blocks = (a.rows + groups - 1) / groups;
  if (!backward) return Next(NormFwdKernel<XT, YT, kRms, VEC, NV>, static_cast<unsigned>(blocks), groups * T, 0, s)(a, T);
  auto* kernel = NormBwdKernel<XT, YT, kRms, VEC, NV>;
  const size_t smem = static_cast<size_t>(groups) * a.cols * 4;
  if (smem > 32 * 1024)   // (the static part counts too)
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)); e != cudaSuccess) return e;
  uint64_t grid = sms < kNormPartials ? sms : kNormPartials;
  if (grid > blocks) grid = blocks;
  if (cudaError_t e = Next(kernel, static_cast<unsigned>(grid), groups * T, smem, s)(a, T); e != cudaSuccess) return e;
  ++*launches;
  if (grid == 1) return cudaSuccess;
  ++*launches;
  return Next(NormFoldKernel, dim3((a.cols + 31) / 32, kRms ? 1 : 2), 1024, 0, s)(a.partials, a.dgamma, a.dbeta, static_cast<uint32_t>(grid), a.cols);
}

template <typename XT, typename YT, bool kRms>
cudaError_t Pick(const NormArgs& a, bool backward, uint32_t sms, cudaStream_t s, int* launches) {
  const bool vec = Vec8Able(a, backward);
  const NormShape shape = ShapeOf(a.cols, vec);
  if (vec) {
    switch (shape.nv) {
      case 1: return Run<XT, YT, kRms, 8, 1>(a, shape.T, backward, sms, s, launches);
      case 2: return Run<XT, YT, kRms, 8, 2>(a, shape.T, backward, sms, s, launches);
      case 3: return Run<XT, YT, kRms, 8, 3>(a, shape.T, backward, sms, s, launches);
      default: return Run<XT, YT, kRms, 8, 4>(a, shape.T, backward, sms, s, launches);
    }
  }
  switch (shape.nv) {
    case 8: return Run<XT, YT, kRms, 1, 8>(a, shape.T, backward, sms, s, launches);
    case 16: return Run<XT, YT, kRms, 1, 16>(a, shape.T, backward, sms, s, launches);
    default: return Run<XT, YT, kRms, 1, 32>(a, shape.T, backward, sms, s, launches);
  }
}

template <typename XT, typename YT>
cudaError_t Pick(const NormArgs& a, bool backward, uint32_t sms, cudaStream_t s, int* launches) {
  return a.rms ? Pick<XT, YT, true>(a, backward, sms, s, launches) : Pick<XT, YT, false>(a, backward, sms, s, launches);
}
cudaError_t Pick(const NormArgs& a, bool backward, uint32_t sms, cudaStream_t s, int* launches) {
  if (a.x_type == SEE_BF16) return Pick<Bf16, Bf16>(a, backward, sms, s, launches);
  if (a.x_type == SEE_F16) return Pick<F16, F16>(a, backward, sms, s, launches);
  if (a.y_type == SEE_BF16) return Pick<float, Bf16>(a, backward, sms, s, launches);
  if (a.y_type == SEE_F16) return Pick<float, F16>(a, backward, sms, s, launches);
  return Pick<float, float>(a, backward, sms, s, launches);
}

}  // namespace

cudaError_t NormForward(const NormArgs& a, uint32_t sms, cudaStream_t s) { return Pick(a, false, sms, s, nullptr); }

cudaError_t NormBackward(const NormArgs& a, uint32_t sms, cudaStream_t s, int* launches) { return Pick(a, true, sms, s, launches); }

}  // namespace see::k
