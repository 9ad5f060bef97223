// Layer norm and root-mean-square norm of rows in f32, bf16 or f16, and their backward pass with the gradients of the
// weights.  With u = (x - mean) rstd (rms: mean = 0), q = dy gamma and <.> a row's average:
//   y = u gamma + beta,   dx = rstd (q - <q> - u <q u>) (+ addend),   dgamma = sum over rows of dy u,   dbeta = of dy
// (rms: neither beta nor <q>).  Bound by HBM: each matrix is read or written once.  Layer norm of 32768 x 768, f32 and bf16,
// backward with an addend: 61 us, 5.8 TB/s (loads straight into registers: 84); forward 27 us, 5.6 TB/s.  16384 x 4096 in bf16
// backward: rms 72 us, 5.6 TB/s; layer 90 us, 4.5, short of issue slots beside a row's three barriers.
//
// A row belongs to a group of T threads (a multiple of 32), which hold it in registers, four or eight consecutive columns at a
// time where widths, strides and addresses allow 16-byte accesses and single columns T apart otherwise; a block has several
// groups.  Rows reach them through a ring in shared memory, or, single columns and few rows, directly.  A thread has the same
// columns in every row, so that the backward pass sums dgamma and dbeta over a block's rows in registers; the groups meet in
// shared memory, the blocks (one to an SM) in NormFoldKernel, both in a fixed order, which goes by the sizes and by what chooses
// the kernel and its groups: types, strides, alignment, and whether there is an addend.
//
// Sums are f32, but for the mean: the threads' sums are added in double.  A thread's share is summed plainly where it has 16 bits
// (a few dozen values of 8 or 11 fit); in f32, with what each addition rounds away in NormFwdKernel, where it costs nothing
// beside the latency, and corrected by the average deviation from the first result in NormFwdRingKernel, where it would (26.6 us
// to 31.5 at 32768 x 768).  The variance is the average square of the deviations, a second pass over the registers, less the
// square of what that mean is off (its rounding; in the ring kernels the average deviation): beside a small eps that would show in
// rows far from zero, whose squares a sum of x^2 would lose altogether.
#include "act_expr.cuh"
#include "block_ops.h"
#include "launch.cuh"
#include "row_groups.cuh"
#include "umma_device.cuh"
#include "vec_types.cuh"

namespace see::k {

namespace {

constexpr uint32_t kNormThreads = 512;

// sum + x into sum, what that rounds away into rest (Knuth's TwoSum: no order of magnitudes asked for).
__device__ __forceinline__ void AddExactly(float& sum, float& rest, float x) {
  const float s = sum + x, z = s - sum;
  rest += (sum - (s - z)) + (x - z);
  sum = s;
}

template <typename XT, typename YT, bool kRms, int VEC, int NV>
__global__ void __launch_bounds__(kNormThreads)
NormFwdKernel(const __grid_constant__ NormArgs a, uint32_t T) {
  AwaitPrevious();
  __shared__ __align__(8) float2 slots[2][kWideThreads / 32];
  const uint32_t group = threadIdx.x / T, t = threadIdx.x - group * T;
  const uint64_t row = static_cast<uint64_t>(blockIdx.x) * (blockDim.x / T) + group;
  if (row >= a.rows) return;
  const XT* x = static_cast<const XT*>(a.x) + row * a.x_stride;
  uint32_t turn = 0;
  float v[NV][VEC], total = 0.0f;
  [[maybe_unused]] float rest = 0.0f;
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
    for (int j = 0; j < VEC; ++j) {
      if (kRms) total += v[i][j] * v[i][j];
      else if (sizeof(XT) == 4) AddExactly(total, rest, v[i][j]);
      else total += v[i][j];
    }
  }
  const float per_col = 1.0f / static_cast<float>(a.cols);
  float mean = 0.0f;
  [[maybe_unused]] float off = 0.0f;
  if constexpr (!kRms) {
    const double share = isfinite(rest) ? static_cast<double>(total) + static_cast<double>(rest) : static_cast<double>(total);
    const double wide = GroupSum(share, T, group, slots, turn) / static_cast<double>(a.cols);
    mean = static_cast<float>(wide);
    off = static_cast<float>(wide - static_cast<double>(mean));
    total = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((t + i * T) * VEC < a.cols) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float d = v[i][j] - mean;
          total += d * d;
        }
      }
  }
  const float square = GroupSum<false>(make_float2(total, 0.0f), T, group, slots, turn).x * per_col, var = kRms ? square : Variance(square, off);
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

// Eight columns as four pairs for the packed f32 instructions (the kernel below is short of issue slots, not of memory's).
template <typename T> __device__ __forceinline__ void LoadPairs(const T* p, f32x2 (&v)[4]) {
  float f[8];
  Load8<T>(p, f);
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = PackF2(f[2 * j], f[2 * j + 1]);
}
template <typename T> __device__ __forceinline__ void StorePairs(T* p, const f32x2 (&v)[4]) {
  float f[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) UnpackF2(v[j], &f[2 * j], &f[2 * j + 1]);
  Store8<T>(p, f);
}

// Four columns as two pairs: where gamma and beta lie in shared memory beside the rows, a warp's accesses are then whole runs.
template <typename T> __device__ __forceinline__ void LoadFour(const T* p, f32x2 (&v)[2]) {
  float f[4];
  if constexpr (sizeof(T) == 4) {
    const float4 r = *reinterpret_cast<const float4*>(p);
    f[0] = r.x; f[1] = r.y; f[2] = r.z; f[3] = r.w;
  } else {
    const uint2 r = *reinterpret_cast<const uint2*>(p);
    Unpack2<T>(r.x, f[0], f[1]);
    Unpack2<T>(r.y, f[2], f[3]);
  }
  v[0] = PackF2(f[0], f[1]);
  v[1] = PackF2(f[2], f[3]);
}
template <typename T> __device__ __forceinline__ void StoreFour(T* p, const f32x2 (&v)[2]) {
  float f[4];
  UnpackF2(v[0], &f[0], &f[1]);
  UnpackF2(v[1], &f[2], &f[3]);
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  else *reinterpret_cast<uint2*>(p) = make_uint2(Pack2<T>(f[0], f[1]), Pack2<T>(f[2], f[3]));
}

// ---- rows through a ring in shared memory -----------------------------------------------
// Each group has `slots` of its own, filled by one thread's bulk copies (a whole row each, counted on the slot's mbarrier)
// and emptied into registers; a slot is asked to be filled again as soon as the group has read it, so that between 60 and
// 200 KB are on their way to an SM at any time.
// The forward pass of more than two rows to a group.  NV: times four columns to a thread.  Up to 768 columns a row is a warp's
// and gamma and beta stay in registers (kHold); of wider ones they lie in shared memory, which leaves registers for half as many
// threads again.  Read from global memory for every row, as NormFwdKernel does, they are twice an f32 row's bytes.  NormFwdKernel
// / this, us: 32768 x 768 f32 to bf16 32 / 26.6, 32768 x 1024 40 / 36, 16384 x 4096 bf16 101 / 66, rms 58 / 48.
template <typename XT, typename YT, bool kRms, int NV, bool kHold>
__global__ void __launch_bounds__(kHold ? kNormThreads : kWideThreads, 1)
NormFwdRingKernel(const __grid_constant__ NormArgs a, uint32_t T, uint32_t slots) {
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ float2 sums[2][kWideThreads / 32];
  const uint32_t groups = blockDim.x / T, group = threadIdx.x / T, t = threadIdx.x - group * T, row_bytes = a.cols * sizeof(XT);
  uint8_t* ring = dyn + static_cast<size_t>(group) * slots * row_bytes;
  float* weights = reinterpret_cast<float*>(dyn + static_cast<size_t>(groups) * slots * row_bytes);   // gamma, beta
  uint64_t* bars = reinterpret_cast<uint64_t*>(weights + (kHold ? 0 : (kRms ? 1 : 2) * a.cols)) + group * slots;
  const uint64_t first = static_cast<uint64_t>(blockIdx.x) * groups + group, step = static_cast<uint64_t>(gridDim.x) * groups;
  if (t == 0) {
    for (uint32_t i = 0; i < slots; ++i) umma_dev::MbarInit(&bars[i], 1);
    umma_dev::MbarInitFence();
  }
  auto fill = [&](uint64_t row, uint32_t slot) {   // the group's thread 0
    umma_dev::MbarExpectTx(&bars[slot], row_bytes);
    umma_dev::BulkLoad(ring + static_cast<size_t>(slot) * row_bytes, static_cast<const XT*>(a.x) + row * a.x_stride, row_bytes, &bars[slot]);
  };
  AwaitPrevious();
  if (t == 0)
    for (uint32_t i = 0; i < slots && first + i * step < a.rows; ++i) fill(first + i * step, i);
  f32x2 gamma[kHold ? NV : 1][2], beta[kHold && !kRms ? NV : 1][2];
  if constexpr (kHold) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((t + i * T) * 4 < a.cols) {
        LoadFour(a.gamma + (t + i * T) * 4, gamma[i]);
        if (!kRms) LoadFour(a.beta + (t + i * T) * 4, beta[kRms ? 0 : i]);
      }
  } else {
    for (uint32_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
      weights[c] = a.gamma[c];
      if (!kRms) weights[a.cols + c] = a.beta[c];
    }
  }
  __syncthreads();
  const float per_col = 1.0f / static_cast<float>(a.cols);
  [[maybe_unused]] const double per_col_wide = 1.0 / static_cast<double>(a.cols);
  uint32_t turn = 0, slot = 0, parity = 0;
  for (uint64_t row = first; row < a.rows; row += step) {
    AwaitRow(&bars[slot], parity, a.status);
    const XT* x = reinterpret_cast<const XT*>(ring + static_cast<size_t>(slot) * row_bytes);
    f32x2 v[NV][2], total = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (t + i * T) * 4;
      if (c < a.cols) {
        LoadFour(x + c, v[i]);
#pragma unroll
        for (int j = 0; j < 2; ++j) total = kRms ? Fma2(v[i][j], v[i][j], total) : AddF2(total, v[i][j]);
      }
    }
    float one, other;
    UnpackF2(total, &one, &other);
    float mean = 0.0f, var;
    if constexpr (kRms) {
      var = GroupSum<false>(make_float2(one + other, 0.0f), T, group, sums, turn).x * per_col;
    } else {
      mean = static_cast<float>(GroupSum(static_cast<double>(one) + static_cast<double>(other), T, group, sums, turn) * per_col_wide);
    }
    if (T == 32) __syncwarp();   // (a wider group has met at the sum's barrier: the slot is read)
    if (t == 0 && row + slots * step < a.rows) fill(row + slots * step, slot);
    if (++slot == slots) {
      slot = 0;
      parity ^= 1;
    }
    if constexpr (!kRms) {
      constexpr bool kCorrect = sizeof(XT) == 4;
      const f32x2 away = Splat2(-mean);
      f32x2 linear = 0;
      total = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if ((t + i * T) * 4 < a.cols) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const f32x2 d = AddF2(v[i][j], away);
            if (kCorrect) linear = AddF2(linear, d);
            total = Fma2(d, d, total);
          }
        }
      float2 sum = make_float2(0.0f, 0.0f);
      if (kCorrect) {
        UnpackF2(linear, &one, &other);
        sum.x = one + other;
      }
      UnpackF2(total, &one, &other);
      sum.y = one + other;
      if (!kCorrect) sum.x = sum.y;
      sum = GroupSum<kCorrect>(sum, T, group, sums, turn);
      if (kCorrect) {
        sum.x *= per_col;
        var = Variance(sum.y * per_col, sum.x);
        if (isfinite(sum.x)) mean += sum.x;
      } else {
        var = sum.x * per_col;   // (a few dozen values of 8 or 11 bits: the mean has its own rounding alone)
      }
    }
    const float rstd = 1.0f / sqrtf(var + a.eps);
    if (t == 0) {
      a.rstd[row] = rstd;
      if (!kRms) a.mean[row] = mean;
    }
    const f32x2 away = Splat2(-mean), rstd2 = Splat2(rstd);
    YT* y = static_cast<YT*>(a.y) + row * a.y_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (t + i * T) * 4;
      if (c < a.cols) {
        f32x2 g[2], b[2];
        if (!kHold) {
          LoadFour(weights + c, g);
          if (!kRms) LoadFour(weights + a.cols + c, b);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const f32x2 unit = Mul2(kRms ? v[i][j] : AddF2(v[i][j], away), rstd2), by = kHold ? gamma[kHold ? i : 0][j] : g[j];
          v[i][j] = kRms ? Mul2(unit, by) : Fma2(unit, by, kHold ? beta[kHold && !kRms ? i : 0][j] : b[j]);
        }
        StoreFour(y + c, v[i]);
      }
    }
  }
}

template <typename XT, typename YT, bool kRms, int NV, uint32_t kThreads>
__global__ void __launch_bounds__(kThreads, 1)
NormBwdRingKernel(const __grid_constant__ NormArgs a, uint32_t T, uint32_t slots) {
  constexpr bool kHoldGamma = kThreads < 512 || NV <= 2;   // in registers, as far as they go
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ float2 sums[2][kWideThreads / 32];
  const uint32_t groups = blockDim.x / T, group = threadIdx.x / T, t = threadIdx.x - group * T;
  const uint32_t x_bytes = a.cols * sizeof(XT), y_bytes = a.cols * sizeof(YT);
  const uint32_t slot_bytes = x_bytes + y_bytes + (a.addend ? x_bytes : 0);
  uint8_t* ring = dyn + static_cast<size_t>(group) * slots * slot_bytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(dyn + static_cast<size_t>(groups) * slots * slot_bytes) + group * slots;
  const uint64_t first = static_cast<uint64_t>(blockIdx.x) * groups + group, step = static_cast<uint64_t>(gridDim.x) * groups;
  if (t == 0) {
    for (uint32_t i = 0; i < slots; ++i) umma_dev::MbarInit(&bars[i], 1);
    umma_dev::MbarInitFence();
  }
  auto fill = [&](uint64_t row, uint32_t slot) {   // the group's thread 0
    uint8_t* dst = ring + static_cast<size_t>(slot) * slot_bytes;
    umma_dev::MbarExpectTx(&bars[slot], slot_bytes);
    umma_dev::BulkLoad(dst, static_cast<const XT*>(a.x) + row * a.x_stride, x_bytes, &bars[slot]);
    umma_dev::BulkLoad(dst + x_bytes, static_cast<const YT*>(a.dy) + row * a.y_stride, y_bytes, &bars[slot]);
    if (a.addend) umma_dev::BulkLoad(dst + x_bytes + y_bytes, static_cast<const XT*>(a.addend) + row * a.x_stride, x_bytes, &bars[slot]);
  };
  AwaitPrevious();
  if (t == 0)
    for (uint32_t i = 0; i < slots && first + i * step < a.rows; ++i) fill(first + i * step, i);
  const float per_col = 1.0f / static_cast<float>(a.cols);
  uint32_t turn = 0;
  f32x2 gamma[kHoldGamma ? NV : 1][4], sum_g[NV][4], sum_b[kRms ? 1 : NV][4];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (kHoldGamma && (t + i * T) * 8 < a.cols) LoadPairs<float>(a.gamma + (t + i * T) * 8, gamma[kHoldGamma ? i : 0]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sum_g[i][j] = 0;
      if (!kRms) sum_b[i][j] = 0;
    }
  }
  GroupBarrier(T, group);   // the barriers are there
  uint32_t slot = 0, parity = 0;
  float next_rstd = 0.0f, next_mean = 0.0f;   // asked for a row ahead, like the row itself
  if (first < a.rows) {
    next_rstd = a.rstd[first];
    if (!kRms) next_mean = a.mean[first];
  }
  for (uint64_t row = first; row < a.rows; row += step) {
    const float rstd = next_rstd, mean = next_mean;
    if (row + step < a.rows) {
      next_rstd = a.rstd[row + step];
      if (!kRms) next_mean = a.mean[row + step];
    }
    const f32x2 rstd2 = Splat2(rstd), mean2 = Splat2(-mean);
    AwaitRow(&bars[slot], parity, a.status);
    const XT* x = reinterpret_cast<const XT*>(ring + static_cast<size_t>(slot) * slot_bytes);
    const YT* dy = reinterpret_cast<const YT*>(x + a.cols);
    f32x2 u[NV][4], d[NV][4], with_u = 0, plain = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (t + i * T) * 8;
      if (c < a.cols) {
        LoadPairs<XT>(x + c, u[i]);
        LoadPairs<YT>(dy + c, d[i]);
        f32x2 g[4];
        if (!kHoldGamma) LoadPairs<float>(a.gamma + c, g);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          u[i][j] = Mul2(kRms ? u[i][j] : AddF2(u[i][j], mean2), rstd2);
          sum_g[i][j] = Fma2(d[i][j], u[i][j], sum_g[i][j]);
          if (!kRms) sum_b[i][j] = AddF2(sum_b[i][j], d[i][j]);
          d[i][j] = Mul2(d[i][j], kHoldGamma ? gamma[kHoldGamma ? i : 0][j] : g[j]);
          with_u = Fma2(d[i][j], u[i][j], with_u);
          if (!kRms) plain = AddF2(plain, d[i][j]);
        }
      }
    }
    float2 sum, other;
    UnpackF2(with_u, &sum.x, &other.x);
    UnpackF2(plain, &sum.y, &other.y);
    sum = GroupSum<!kRms>(make_float2(sum.x + other.x, sum.y + other.y), T, group, sums, turn);
    const f32x2 pull = Splat2(-sum.x * per_col), shift = Splat2(-sum.y * per_col);
    const XT* add = reinterpret_cast<const XT*>(dy + a.cols);
    XT* dx = static_cast<XT*>(a.dx) + row * a.x_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (t + i * T) * 8;
      if (c < a.cols) {
        f32x2 v[4];
        if (a.addend) LoadPairs<XT>(add + c, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f32x2 r = Fma2(u[i][j], pull, kRms ? d[i][j] : AddF2(d[i][j], shift));
          v[j] = a.addend ? Fma2(r, rstd2, v[j]) : Mul2(r, rstd2);
        }
        StorePairs<XT>(dx + c, v);
      }
    }
    GroupBarrier(T, group);   // the slot is read
    if (t == 0 && row + slots * step < a.rows) fill(row + slots * step, slot);
    if (++slot == slots) {
      slot = 0;
      parity ^= 1;
    }
  }
  float* meet = reinterpret_cast<float*>(dyn);   // [groups][cols]; every copy has been read
  float* out_g = gridDim.x == 1 ? a.dgamma : a.partials + static_cast<size_t>(blockIdx.x) * a.cols;
  float* out_b = gridDim.x == 1 ? a.dbeta : a.partials + static_cast<size_t>(gridDim.x + blockIdx.x) * a.cols;
#pragma unroll
  for (int which = 0; which < (kRms ? 1 : 2); ++which) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (t + i * T) * 8;
      if (c < a.cols) StorePairs<float>(meet + group * a.cols + c, which ? sum_b[kRms ? 0 : i] : sum_g[i]);
    }
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
      float s = meet[c];
      for (uint32_t r = 1; r < groups; ++r) s += meet[r * a.cols + c];
      (which ? out_b : out_g)[c] = s;
    }
  }
}

// ---- rows of any width and alignment through the ring ----------------------------------------
// A bulk copy begins and ends on 16 bytes: a row is copied with what lies beside it up to there, which for all but the first and
// the last row (or rows, where they are shorter than that) lies within the matrix, its neighbours' ends or what is between them,
// and is used from where it begins.  The others are copied element by element.  Threads then take single columns, T apart.
// Straight into registers / so, us: 30000 x 1029 f32 155 / 144, bf16 295 / 127; 8000 x 5003 f32 and bf16 566 / 215;
// 40373 x 55 f32 and f16 with an addend 34 / 23.
// NV single columns a thread.
template <typename XT, typename YT, bool kRms, int NV>
__global__ void __launch_bounds__(kNormThreads, 1)
NormBwdOddKernel(const __grid_constant__ NormArgs a, uint32_t T, uint32_t slots) {
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ float2 sums[2][kWideThreads / 32];
  const uint32_t groups = blockDim.x / T, group = threadIdx.x / T, t = threadIdx.x - group * T;
  const uint32_t x_slot = OddSlot<XT>(a.cols), y_slot = OddSlot<YT>(a.cols), slot_bytes = x_slot + y_slot + (a.addend ? x_slot : 0);
  uint8_t* ring = dyn + static_cast<size_t>(group) * slots * slot_bytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(dyn + static_cast<size_t>(groups) * slots * slot_bytes) + group * slots;
  const uint64_t first = static_cast<uint64_t>(blockIdx.x) * groups + group, step = static_cast<uint64_t>(gridDim.x) * groups;
  if (t == 0) {
    for (uint32_t i = 0; i < slots; ++i) umma_dev::MbarInit(&bars[i], 1);
    umma_dev::MbarInitFence();
  }
  // Rows with 16 bytes of the matrix on either side.
  const uint64_t narrow = min(a.x_stride * sizeof(XT), a.y_stride * sizeof(YT)), edge = (15 + narrow) / narrow;
  auto inner = [&](uint64_t row) { return row >= edge && row + edge < a.rows; };
  auto fill = [&](uint64_t row, uint32_t slot) {   // the group's thread 0
    if (!inner(row)) return;
    umma_dev::FenceProxyAsync();   // (an edge row's elements may have been written there)
    uint8_t* dst = ring + static_cast<size_t>(slot) * slot_bytes;
    const OddRow<XT> x(a.x, row, a.x_stride, a.cols);
    const OddRow<YT> dy(a.dy, row, a.y_stride, a.cols);
    const OddRow<XT> add(a.addend, row, a.x_stride, a.cols);
    umma_dev::MbarExpectTx(&bars[slot], x.bytes + dy.bytes + (a.addend ? add.bytes : 0));
    umma_dev::BulkLoad(dst, x.from, x.bytes, &bars[slot]);
    umma_dev::BulkLoad(dst + x_slot, dy.from, dy.bytes, &bars[slot]);
    if (a.addend) umma_dev::BulkLoad(dst + x_slot + y_slot, add.from, add.bytes, &bars[slot]);
  };
  AwaitPrevious();
  if (t == 0)
    for (uint32_t i = 0; i < slots && first + i * step < a.rows; ++i) fill(first + i * step, i);
  float gamma[NV], sum_g[NV], sum_b[kRms ? 1 : NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    gamma[i] = t + i * T < a.cols ? a.gamma[t + i * T] : 0.0f;
    sum_g[i] = 0.0f;
    if (!kRms) sum_b[i] = 0.0f;
  }
  GroupBarrier(T, group);   // the barriers are there
  const float per_col = 1.0f / static_cast<float>(a.cols);
  uint32_t turn = 0, slot = 0, parities = 0;   // a bit for each slot, of the copies that went through it
  float next_rstd = 0.0f, next_mean = 0.0f;
  if (first < a.rows) {
    next_rstd = a.rstd[first];
    if (!kRms) next_mean = a.mean[first];
  }
  for (uint64_t row = first; row < a.rows; row += step) {
    const float rstd = next_rstd, mean = next_mean;
    if (row + step < a.rows) {
      next_rstd = a.rstd[row + step];
      if (!kRms) next_mean = a.mean[row + step];
    }
    uint8_t* at = ring + static_cast<size_t>(slot) * slot_bytes;
    if (inner(row)) {
      AwaitRow(&bars[slot], parities >> slot & 1u, a.status);
      parities ^= 1u << slot;
    } else {
      CopyRow<XT>(at, a.x, row, a.x_stride, a.cols, t, T);
      CopyRow<YT>(at + x_slot, a.dy, row, a.y_stride, a.cols, t, T);
      if (a.addend) CopyRow<XT>(at + x_slot + y_slot, a.addend, row, a.x_stride, a.cols, t, T);
      GroupBarrier(T, group);
    }
    const XT* x = reinterpret_cast<const XT*>(at + OddRow<XT>(a.x, row, a.x_stride, a.cols).skip);
    const YT* dy = reinterpret_cast<const YT*>(at + x_slot + OddRow<YT>(a.dy, row, a.y_stride, a.cols).skip);
    const XT* add = reinterpret_cast<const XT*>(at + x_slot + y_slot + OddRow<XT>(a.addend, row, a.x_stride, a.cols).skip);
    float u[NV], d[NV];
    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = t + i * T;
      if (c < a.cols) {
        u[i] = (ToF32(x[c]) - mean) * rstd;
        const float dv = ToF32(dy[c]);
        sum_g[i] += dv * u[i];
        if (!kRms) sum_b[i] += dv;
        d[i] = dv * gamma[i];
        sum.x += d[i] * u[i];
        if (!kRms) sum.y += d[i];
      }
    }
    sum = GroupSum<!kRms>(sum, T, group, sums, turn);
    sum.x *= per_col;
    sum.y *= per_col;
    XT* dx = static_cast<XT*>(a.dx) + row * a.x_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = t + i * T;
      if (c < a.cols) {
        const float r = rstd * (kRms ? d[i] - u[i] * sum.x : d[i] - sum.y - u[i] * sum.x);
        dx[c] = FromF32<XT>(a.addend ? r + ToF32(add[c]) : r);
      }
    }
    GroupBarrier(T, group);   // the slot is read
    if (t == 0 && row + slots * step < a.rows) fill(row + slots * step, slot);
    if (++slot == slots) slot = 0;
  }
  float* meet = reinterpret_cast<float*>(dyn);   // [groups][cols]; every copy has been read
  float* out_g = gridDim.x == 1 ? a.dgamma : a.partials + static_cast<size_t>(blockIdx.x) * a.cols;
  float* out_b = gridDim.x == 1 ? a.dbeta : a.partials + static_cast<size_t>(gridDim.x + blockIdx.x) * a.cols;
#pragma unroll
  for (int which = 0; which < (kRms ? 1 : 2); ++which) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + i * T < a.cols) meet[group * a.cols + t + i * T] = which ? sum_b[kRms ? 0 : i] : sum_g[i];
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
      float s = meet[c];
      for (uint32_t r = 1; r < groups; ++r) s += meet[r * a.cols + c];
      (which ? out_b : out_g)[c] = s;
    }
  }
}

// The forward pass of such rows, as NormFwdRingKernel takes its own.  NormFwdKernel / this, us: 30000 x 1029 f32 114 / 88, rms in
// bf16 99 / 67, 30000 x 333 f32 to bf16 44 / 32.
template <typename XT, typename YT, bool kRms, int NV>
__global__ void __launch_bounds__(kNormThreads, 1)
NormFwdOddKernel(const __grid_constant__ NormArgs a, uint32_t T, uint32_t slots) {
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ float2 sums[2][kWideThreads / 32];
  const uint32_t groups = blockDim.x / T, group = threadIdx.x / T, t = threadIdx.x - group * T, slot_bytes = OddSlot<XT>(a.cols);
  uint8_t* ring = dyn + static_cast<size_t>(group) * slots * slot_bytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(dyn + static_cast<size_t>(groups) * slots * slot_bytes) + group * slots;
  const uint64_t first = static_cast<uint64_t>(blockIdx.x) * groups + group, step = static_cast<uint64_t>(gridDim.x) * groups;
  if (t == 0) {
    for (uint32_t i = 0; i < slots; ++i) umma_dev::MbarInit(&bars[i], 1);
    umma_dev::MbarInitFence();
  }
  const uint64_t narrow = a.x_stride * sizeof(XT), edge = (15 + narrow) / narrow;
  auto inner = [&](uint64_t row) { return row >= edge && row + edge < a.rows; };
  auto fill = [&](uint64_t row, uint32_t slot) {   // the group's thread 0
    if (!inner(row)) return;
    umma_dev::FenceProxyAsync();   // (an edge row's elements may have been written there)
    const OddRow<XT> x(a.x, row, a.x_stride, a.cols);
    umma_dev::MbarExpectTx(&bars[slot], x.bytes);
    umma_dev::BulkLoad(ring + static_cast<size_t>(slot) * slot_bytes, x.from, x.bytes, &bars[slot]);
  };
  AwaitPrevious();
  if (t == 0)
    for (uint32_t i = 0; i < slots && first + i * step < a.rows; ++i) fill(first + i * step, i);
  float gamma[NV], beta[kRms ? 1 : NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const bool there = t + i * T < a.cols;
    gamma[i] = there ? a.gamma[t + i * T] : 0.0f;
    if (!kRms) beta[kRms ? 0 : i] = there ? a.beta[t + i * T] : 0.0f;
  }
  GroupBarrier(T, group);   // the barriers are there
  const float per_col = 1.0f / static_cast<float>(a.cols);
  [[maybe_unused]] const double per_col_wide = 1.0 / static_cast<double>(a.cols);
  uint32_t turn = 0, slot = 0, parities = 0;   // a bit for each slot, of the copies that went through it
  for (uint64_t row = first; row < a.rows; row += step) {
    uint8_t* at = ring + static_cast<size_t>(slot) * slot_bytes;
    if (inner(row)) {
      AwaitRow(&bars[slot], parities >> slot & 1u, a.status);
      parities ^= 1u << slot;
    } else {
      CopyRow<XT>(at, a.x, row, a.x_stride, a.cols, t, T);
      GroupBarrier(T, group);
    }
    const XT* x = reinterpret_cast<const XT*>(at + OddRow<XT>(a.x, row, a.x_stride, a.cols).skip);
    float v[NV], total = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      v[i] = t + i * T < a.cols ? ToF32(x[t + i * T]) : 0.0f;
      total += kRms ? v[i] * v[i] : v[i];
    }
    float mean = 0.0f, var;
    if constexpr (kRms) var = GroupSum<false>(make_float2(total, 0.0f), T, group, sums, turn).x * per_col;
    else mean = static_cast<float>(GroupSum(static_cast<double>(total), T, group, sums, turn) * per_col_wide);
    if (T == 32) __syncwarp();   // (a wider group has met at the sum's barrier: the slot is read)
    if (t == 0 && row + slots * step < a.rows) fill(row + slots * step, slot);
    if (++slot == slots) slot = 0;
    if constexpr (!kRms) {
      float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (t + i * T < a.cols) {
          const float d = v[i] - mean;
          sum.x += d;
          sum.y += d * d;
        }
      sum = GroupSum<true>(sum, T, group, sums, turn);
      sum.x *= per_col;
      var = Variance(sum.y * per_col, sum.x);
      if (isfinite(sum.x)) mean += sum.x;
    }
    const float rstd = 1.0f / sqrtf(var + a.eps);
    if (t == 0) {
      a.rstd[row] = rstd;
      if (!kRms) a.mean[row] = mean;
    }
    YT* y = static_cast<YT*>(a.y) + row * a.y_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + i * T < a.cols)
        y[t + i * T] = FromF32<YT>(kRms ? v[i] * rstd * gamma[i] : (v[i] - mean) * rstd * gamma[i] + beta[kRms ? 0 : i]);
  }
}

// Single columns, T apart, straight into registers.  One row of partial sums a block; a lone block writes the gradients themselves.
template <typename XT, typename YT, bool kRms, int NV>
__global__ void __launch_bounds__(kNormThreads, 1)
NormBwdKernel(const __grid_constant__ NormArgs a, uint32_t T) {
  AwaitPrevious();
  extern __shared__ float meet[];   // [groups][cols]
  __shared__ float2 slots[2][kWideThreads / 32];
  const uint32_t groups = blockDim.x / T, group = threadIdx.x / T, t = threadIdx.x - group * T;
  const float per_col = 1.0f / static_cast<float>(a.cols);
  uint32_t turn = 0;
  float sum_g[NV], sum_b[kRms ? 1 : NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    sum_g[i] = 0.0f;
    if (!kRms) sum_b[i] = 0.0f;
  }
  for (uint64_t row = static_cast<uint64_t>(blockIdx.x) * groups + group; row < a.rows; row += static_cast<uint64_t>(gridDim.x) * groups) {
    const XT* x = static_cast<const XT*>(a.x) + row * a.x_stride;
    const YT* dy = static_cast<const YT*>(a.dy) + row * a.y_stride;
    float u[NV], d[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = t + i * T;
      if (c < a.cols) {
        u[i] = ToF32(x[c]);
        d[i] = ToF32(dy[c]);
      }
    }
    const float rstd = a.rstd[row], mean = kRms ? 0.0f : a.mean[row];
    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = t + i * T;
      if (c < a.cols) {
        u[i] = (u[i] - mean) * rstd;
        sum_g[i] += d[i] * u[i];
        if (!kRms) sum_b[i] += d[i];
        d[i] *= a.gamma[c];
        sum.x += d[i] * u[i];
        if (!kRms) sum.y += d[i];
      }
    }
    sum = GroupSum<!kRms>(sum, T, group, slots, turn);
    sum.x *= per_col;
    sum.y *= per_col;
    XT* dx = static_cast<XT*>(a.dx) + row * a.x_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = t + i * T;
      if (c < a.cols) {
        float v;
        if (a.addend) v = ToF32(static_cast<const XT*>(a.addend)[row * a.x_stride + c]);
        const float r = rstd * (kRms ? d[i] - u[i] * sum.x : d[i] - sum.y - u[i] * sum.x);
        dx[c] = FromF32<XT>(a.addend ? r + v : r);
      }
    }
  }
  float* out_g = gridDim.x == 1 ? a.dgamma : a.partials + static_cast<size_t>(blockIdx.x) * a.cols;
  float* out_b = gridDim.x == 1 ? a.dbeta : a.partials + static_cast<size_t>(gridDim.x + blockIdx.x) * a.cols;
#pragma unroll
  for (int which = 0; which < (kRms ? 1 : 2); ++which) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + i * T < a.cols) meet[group * a.cols + t + i * T] = which ? sum_b[kRms ? 0 : i] : sum_g[i];
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
  AwaitPrevious();
  __shared__ float meet[32][33];
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

template <bool kRms>
cudaError_t Fold(const NormArgs& a, uint64_t grid, cudaStream_t s, int* launches) {
  ++*launches;
  if (grid == 1) return cudaSuccess;
  ++*launches;
  return Next(NormFoldKernel, dim3((a.cols + 31) / 32, kRms ? 1 : 2), 1024, 0, s)(a.partials, a.dgamma, a.dbeta, static_cast<uint32_t>(grid), a.cols);
}
uint64_t Blocks(uint64_t rows, uint32_t groups, uint32_t sms) {
  const uint64_t blocks = (rows + groups - 1) / groups, most = sms < kNormPartials ? sms : kNormPartials;
  return blocks < most ? blocks : most;
}

template <typename XT, typename YT, bool kRms, int NV, uint32_t kThreads>
cudaError_t RunRing(const NormArgs& a, uint32_t T, uint32_t sms, cudaStream_t s, int* launches) {
  const size_t row_bytes = static_cast<size_t>(a.cols) * (sizeof(XT) * (a.addend ? 2 : 1) + sizeof(YT));
  uint32_t groups = kThreads / T;
  while (groups > 1 && 2 * groups * row_bytes > kRingBytes) --groups;   // two slots to a group, unless it is alone
  uint32_t slots = static_cast<uint32_t>(kRingBytes / (groups * row_bytes));
  slots = slots < 1 ? 1 : slots > 8 ? 8 : slots;
  const size_t smem = groups * slots * (row_bytes + 8);
  constexpr auto* kernel = NormBwdRingKernel<XT, YT, kRms, NV, kThreads>;
  if (cudaError_t e = AllowShared<kernel>(smem); e != cudaSuccess) return e;
  const uint64_t grid = Blocks(a.rows, groups, sms);
  if (cudaError_t e = Next(kernel, static_cast<unsigned>(grid), groups * T, smem, s)(a, T, slots); e != cudaSuccess) return e;
  return Fold<kRms>(a, grid, s, launches);
}

template <typename XT, typename YT, bool kRms, int NV, bool kHold>
cudaError_t RunFwdRing(const NormArgs& a, uint32_t T, uint32_t sms, cudaStream_t s) {
  const size_t row_bytes = static_cast<size_t>(a.cols) * sizeof(XT), weights = kHold ? 0 : a.cols * (kRms ? 4 : 8);
  uint32_t groups = (kHold ? kNormThreads : kWideThreads) / T;
  while (groups > 1 && groups * row_bytes > kRingBytes - weights) --groups;
  uint32_t slots = static_cast<uint32_t>((kRingBytes - weights) / (groups * row_bytes));   // (one at least, up to 8192 columns)
  slots = slots > 8 ? 8 : slots;
  const size_t smem = groups * slots * (row_bytes + 8) + weights;
  constexpr auto* kernel = NormFwdRingKernel<XT, YT, kRms, NV, kHold>;
  if (cudaError_t e = AllowShared<kernel>(smem); e != cudaSuccess) return e;
  return Next(kernel, static_cast<unsigned>(Blocks(a.rows, groups, sms)), groups * T, smem, s)(a, T, slots);
}

template <typename XT, typename YT, bool kRms, int VEC, int NV>
cudaError_t Run(const NormArgs& a, uint32_t T, cudaStream_t s) {
  const uint32_t groups = kNormThreads / T;
  return Next(NormFwdKernel<XT, YT, kRms, VEC, NV>, static_cast<unsigned>((a.rows + groups - 1) / groups), groups * T, 0, s)(a, T);
}
template <typename XT, typename YT, bool kRms, int NV>
cudaError_t RunFwdOdd(const NormArgs& a, uint32_t T, uint32_t sms, cudaStream_t s) {
  const size_t slot_bytes = OddSlot<XT>(a.cols);
  uint32_t groups = kNormThreads / T;
  while (groups > 1 && 2 * groups * slot_bytes > kRingBytes) --groups;
  uint32_t slots = static_cast<uint32_t>(kRingBytes / (groups * slot_bytes));
  slots = slots > 8 ? 8 : slots;   // (two at least: 8192 columns are 32 KB)
  const size_t smem = groups * slots * (slot_bytes + 8);
  constexpr auto* kernel = NormFwdOddKernel<XT, YT, kRms, NV>;
  if (cudaError_t e = AllowShared<kernel>(smem); e != cudaSuccess) return e;
  return Next(kernel, static_cast<unsigned>(Blocks(a.rows, groups, sms)), groups * T, smem, s)(a, T, slots);
}

template <typename XT, typename YT, bool kRms, int NV>
cudaError_t RunOdd(const NormArgs& a, uint32_t T, uint32_t sms, cudaStream_t s, int* launches) {
  const size_t slot_bytes = OddSlot<XT>(a.cols) * (a.addend ? 2 : 1) + OddSlot<YT>(a.cols);
  uint32_t groups = kNormThreads / T;
  while (groups > 1 && 2 * groups * slot_bytes > kRingBytes) --groups;   // two slots to a group, unless it is alone
  uint32_t slots = static_cast<uint32_t>(kRingBytes / (groups * slot_bytes));
  slots = slots < 1 ? 1 : slots > 8 ? 8 : slots;
  const size_t smem = groups * slots * (slot_bytes + 8);
  constexpr auto* kernel = NormBwdOddKernel<XT, YT, kRms, NV>;
  if (cudaError_t e = AllowShared<kernel>(smem); e != cudaSuccess) return e;
  const uint64_t grid = Blocks(a.rows, groups, sms);
  if (cudaError_t e = Next(kernel, static_cast<unsigned>(grid), groups * T, smem, s)(a, T, slots); e != cudaSuccess) return e;
  return Fold<kRms>(a, grid, s, launches);
}

template <typename XT, typename YT, bool kRms, int NV>
cudaError_t RunSingles(const NormArgs& a, uint32_t T, uint32_t sms, cudaStream_t s, int* launches) {
  const uint32_t groups = kNormThreads / T;
  constexpr auto* kernel = NormBwdKernel<XT, YT, kRms, NV>;
  const size_t smem = static_cast<size_t>(groups) * a.cols * 4;
  if (cudaError_t e = AllowShared<kernel>(smem); e != cudaSuccess) return e;
  const uint64_t grid = Blocks(a.rows, groups, sms);
  if (cudaError_t e = Next(kernel, static_cast<unsigned>(grid), groups * T, smem, s)(a, T); e != cudaSuccess) return e;
  return Fold<kRms>(a, grid, s, launches);
}

template <typename XT, typename YT, bool kRms>
cudaError_t Pick(const NormArgs& a, bool backward, uint32_t sms, cudaStream_t s, int* launches) {
  const bool vec = Vec8Able(a, backward);
  const NormShape f = ShapeOf(a.cols, vec);
  if (vec && backward) {
    // A warp's row of up to 768 columns, or threads with 16 of wider ones: a row's u and q, the sums and gamma are then in
    // registers; rms, with one sum, has room for 32, which spreads a row's fixed cost further.  (16384 x 4096 bf16: layer
    // norm with 32 columns a thread 117 us, spilling, 16 90; rms 16 columns 80, 32 73.)
    const uint32_t n = a.cols / 8;
    auto up = [](uint32_t v) { return (v + 31) / 32 * 32; };
    if (n <= 96) {   // a warp's row
      if (n <= 32) return RunRing<XT, YT, kRms, 1, 384>(a, 32, sms, s, launches);
      return n <= 64 ? RunRing<XT, YT, kRms, 2, 384>(a, 32, sms, s, launches) : RunRing<XT, YT, kRms, 3, 384>(a, 32, sms, s, launches);
    }
    if (kRms && n <= 1536) return RunRing<XT, YT, kRms, 4, 384>(a, up((n + 3) / 4), sms, s, launches);
    if (n <= 1024) return RunRing<XT, YT, kRms, 2, 512>(a, up((n + 1) / 2), sms, s, launches);
    return RunRing<XT, YT, kRms, 4, 512>(a, up((n + 3) / 4), sms, s, launches);
  }
  if (vec && a.cols <= 8192) {   // (two slots to a group of the widest)
    const uint32_t n = a.cols / 4, T = n <= 256 ? 32 : (n + 255) / 256 * 32;
    // Two rows to a group of NormFwdKernel.  About there, us, it / the ring: 768 columns f32 to bf16, 4736 rows 7.2 / 7.2, 5920
    // 11.2 / 8.9; 2048 f32, 2368 rows 12.8 / 13.0, 2960 16.3 / 13.4; 4096 bf16, 1184 rows 10.3 / 12.8, 1480 13.5 / 13.5.  Rows of few
    // bytes, and rms ones of 16 bits, would want some more: 64 columns bf16, 14208 rows 4.6 / 5.7; 1024, 9472 rows 10.4 / 12.4; 8192,
    // 1776 rows 17.7 / 19.9.
    if (a.rows > 2ull * (kNormThreads / T) * sms) {
      if (n <= 64) return RunFwdRing<XT, YT, kRms, 2, true>(a, T, sms, s);
      if (n <= 128) return RunFwdRing<XT, YT, kRms, 4, true>(a, T, sms, s);
      if (n <= 192) return RunFwdRing<XT, YT, kRms, 6, true>(a, T, sms, s);
      return RunFwdRing<XT, YT, kRms, 8, false>(a, T, sms, s);
    }
  }
  if (vec) {
    switch (f.nv) {
      case 1: return Run<XT, YT, kRms, 8, 1>(a, f.T, s);
      case 2: return Run<XT, YT, kRms, 8, 2>(a, f.T, s);
      case 3: return Run<XT, YT, kRms, 8, 3>(a, f.T, s);
      default: return Run<XT, YT, kRms, 8, 4>(a, f.T, s);
    }
  }
  if (backward) {
    // Few rows are over before a ring pays, and the widest have no room for one.  About four rows to a group, us, straight into
    // registers / ring: 9472 x 55 bf16 11.0 / 8.6; 4736 x 333 f32 and bf16 19.5 / 21.1, 7104 26.3 / 24.6; 1776 x 1029 bf16 22.3 / 21.0; 592 x
    // 4095 bf16 28.4 / 28.7.  Wide f32 rows would want some more: 2664 x 1029 18.9 / 30.0, 1184 x 8001 50.8 / 65.6 (30000 x 1029 155 / 144).
    if (a.cols > 8192 || a.rows <= 4ull * sms * (kNormThreads / f.T)) {
      switch (f.nv) {
        case 8: return RunSingles<XT, YT, kRms, 8>(a, f.T, sms, s, launches);
        case 16: return RunSingles<XT, YT, kRms, 16>(a, f.T, sms, s, launches);
        default: return RunSingles<XT, YT, kRms, 32>(a, f.T, sms, s, launches);
      }
    }
    const uint32_t T = a.cols <= 512 ? 32 : (a.cols + 511) / 512 * 32, each = (a.cols + T - 1) / T;
    if (each <= 2) return RunOdd<XT, YT, kRms, 2>(a, T, sms, s, launches);
    if (each <= 4) return RunOdd<XT, YT, kRms, 4>(a, T, sms, s, launches);
    return each <= 8 ? RunOdd<XT, YT, kRms, 8>(a, T, sms, s, launches) : RunOdd<XT, YT, kRms, 16>(a, T, sms, s, launches);
  }
  // (With two groups at least: 5003 columns 122 us, so 129.  About four rows to a group, us, NormFwdKernel / so: 9472 x 55 bf16 5.0 /
  // 4.9, 4736 x 333 f32 to bf16 8.9 / 10.4, 7104 12.4 / 12.4, 2220 x 1029 f32 12.8 / 14.0, rms bf16 11.1 / 10.8, 1184 x 4095 18.0 / 18.0.)
  if (a.cols <= 4096 && a.rows > 4ull * sms * (kNormThreads / f.T)) {
    const uint32_t T = a.cols <= 512 ? 32 : (a.cols + 511) / 512 * 32, each = (a.cols + T - 1) / T;
    if (each <= 2) return RunFwdOdd<XT, YT, kRms, 2>(a, T, sms, s);
    if (each <= 4) return RunFwdOdd<XT, YT, kRms, 4>(a, T, sms, s);
    return each <= 8 ? RunFwdOdd<XT, YT, kRms, 8>(a, T, sms, s) : RunFwdOdd<XT, YT, kRms, 16>(a, T, sms, s);
  }
  switch (f.nv) {
    case 8: return Run<XT, YT, kRms, 1, 8>(a, f.T, s);
    case 16: return Run<XT, YT, kRms, 1, 16>(a, f.T, s);
    default: return Run<XT, YT, kRms, 1, 32>(a, f.T, s);
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
