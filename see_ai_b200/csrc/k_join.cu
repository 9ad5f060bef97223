// A block joins the residual stream: x' = a x + g N1(b), y = N2(x'), with the norm after the block, its gate, the scaled residual and
// the norm before the next block in one pass over the rows, and its backward pass.  With u = (b - mean1) rstd1, v = (x' - mean2) rstd2,
// A = g gamma1 (what is absent: 1; without a norm after the block u = b), q = dy gamma2 and <.> a row's average:
//   d = rstd2 (q - <q> - v <q v>) + dx',   dx = a d,   db = rstd1 (A d - <A d> - u <A d u>)  (without that norm: A d),
//   P1 = sum over rows of dy v,  P2 = of dy,  S1 = of d u,  S2 = of d:
//   dgamma2 = P1,  dbeta2 = P2,  dgamma1 = g S1,  dbeta1 = g S2,  dg = gamma1 S1 + beta1 S2:
// the gate's gradient needs no sums of its own.  (Rms: no means, no <q>, no P2, S2.)  Bound by HBM: each matrix is read or written once.
//
// A mean is that of the threads' f32 sums, added in double here and in f32 in the ring kernels, corrected by the average deviation from
// it; the variance is the average square of the deviations less the square of that correction.  y comes of x' before it is rounded to the stream's type.
#include "join.cuh"

namespace see::k {

namespace {

constexpr uint32_t kThreads = 512;

template <int N>
struct Sums {
  float v[N];
};
// Sums of a block's threads, in all of them.  Two sets of slots, used in turn, need one barrier a sum.
template <int N>
__device__ __forceinline__ Sums<N> BlockSum(Sums<N> s, float (*slots)[kThreads / 32][2], uint32_t& turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) s.v[i] += __shfl_xor_sync(0xFFFFFFFFu, s.v[i], o);
  auto* set = slots[turn];
  turn ^= 1;
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) set[threadIdx.x >> 5][i] = s.v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) s.v[i] = set[0][i];
  for (uint32_t w = 1; w < kThreads / 32; ++w)
#pragma unroll
    for (int i = 0; i < N; ++i) s.v[i] += set[w][i];
  return s;
}
__device__ __forceinline__ float BlockMean(float sum, float (*slots)[kThreads / 32][2], uint32_t& turn, uint32_t cols) {
  double wide = sum;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) wide += __shfl_xor_sync(0xFFFFFFFFu, wide, o);
  auto* set = reinterpret_cast<double*>(slots[turn]);
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) set[threadIdx.x >> 5] = wide;
  __syncthreads();
  wide = set[0];
  for (uint32_t w = 1; w < kThreads / 32; ++w) wide += set[w];
  return static_cast<float>(wide / static_cast<double>(cols));
}

struct Stats {
  float mean, rstd;
};
// Of the row in buf, of which a thread has the columns t, t + kThreads, ...; total: the thread's sum (rms: of squares).
template <bool kRms>
__device__ __forceinline__ Stats StatsOf(const float* buf, uint32_t cols, float total, float eps, float (*slots)[kThreads / 32][2], uint32_t& turn) {
  const float per_col = 1.0f / static_cast<float>(cols);
  if (kRms) return {0.0f, 1.0f / sqrtf(BlockSum<1>({{total}}, slots, turn).v[0] * per_col + eps)};
  float mean = BlockMean(total, slots, turn, cols);
  Sums<2> s = {{0.0f, 0.0f}};
  for (uint32_t c = threadIdx.x; c < cols; c += kThreads) {
    const float d = buf[c] - mean;
    s.v[0] += d;
    s.v[1] += d * d;
  }
  s = BlockSum<2>(s, slots, turn);
  const float off = s.v[0] * per_col, var = Variance(s.v[1] * per_col, off);
  if (isfinite(off)) mean += off;
  return {mean, 1.0f / sqrtf(var + eps)};
}

// A row to a block, its values in shared memory, single columns to a thread.
template <typename XT, typename YT, bool kRms>
__global__ void __launch_bounds__(kThreads)
JoinFwdKernel(const __grid_constant__ JoinArgs a) {
  AwaitPrevious();
  extern __shared__ float buf[];   // [cols]
  __shared__ __align__(8) float slots[2][kThreads / 32][2];
  const uint64_t row = blockIdx.x;
  const XT* x = static_cast<const XT*>(a.x) + row * a.x_stride;
  const YT* b = static_cast<const YT*>(a.block) + row * a.y_stride;
  XT* x_out = static_cast<XT*>(a.x_out) + row * a.x_stride;
  YT* y = static_cast<YT*>(a.y) + row * a.y_stride;
  const bool post = a.w.post_gamma != nullptr;
  uint32_t turn = 0;
  Stats one = {0.0f, 1.0f};
  float total = 0.0f;
  for (uint32_t c = threadIdx.x; c < a.cols; c += kThreads) {
    const float v = ToF32(b[c]);
    buf[c] = v;
    total += kRms ? v * v : v;
  }
  if (post) one = StatsOf<kRms>(buf, a.cols, total, a.eps, slots, turn);
  total = 0.0f;
  for (uint32_t c = threadIdx.x; c < a.cols; c += kThreads) {
    float u = buf[c];
    if (post) u = (u - one.mean) * one.rstd * a.w.post_gamma[c] + (kRms ? 0.0f : a.w.post_beta[c]);
    const float v = fmaf(a.scale, ToF32(x[c]), a.w.gate ? a.w.gate[c] * u : u);
    buf[c] = v;
    x_out[c] = FromF32<XT>(v);
    total += kRms ? v * v : v;
  }
  const Stats two = StatsOf<kRms>(buf, a.cols, total, a.eps, slots, turn);
  for (uint32_t c = threadIdx.x; c < a.cols; c += kThreads)
    y[c] = FromF32<YT>((buf[c] - two.mean) * two.rstd * a.w.pre_gamma[c] + (kRms ? 0.0f : a.w.pre_beta[c]));
  if (threadIdx.x == 0) {
    if (post) a.stats.post_rstd[row] = one.rstd;
    a.stats.pre_rstd[row] = two.rstd;
    if (!kRms) {
      if (post) a.stats.post_mean[row] = one.mean;
      a.stats.pre_mean[row] = two.mean;
    }
  }
}

// The four sums' rows of partials are [4][blocks][cols]: P1, P2, S1, S2.
template <typename XT, typename YT, bool kRms>
__global__ void __launch_bounds__(kThreads)
JoinBwdKernel(const __grid_constant__ JoinArgs a) {
  AwaitPrevious();
  extern __shared__ float buf[];   // [cols]
  __shared__ __align__(8) float slots[2][kThreads / 32][2];
  const bool post = a.w.post_gamma != nullptr;
  const float per_col = 1.0f / static_cast<float>(a.cols);
  const size_t each = static_cast<size_t>(gridDim.x) * a.cols;
  float* sums = a.partials + static_cast<size_t>(blockIdx.x) * a.cols;
  uint32_t turn = 0;
  for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const bool first = row == blockIdx.x;
    const YT* dy = static_cast<const YT*>(a.dy) + row * a.y_stride;
    const YT* b = static_cast<const YT*>(a.block) + row * a.y_stride;
    const XT* x = static_cast<const XT*>(a.x) + row * a.x_stride;
    const XT* dx_out = a.dx_out ? static_cast<const XT*>(a.dx_out) + row * a.x_stride : nullptr;
    XT* dx = static_cast<XT*>(a.dx) + row * a.x_stride;
    YT* db = static_cast<YT*>(a.dblock) + row * a.y_stride;
    const float rstd2 = a.stats.pre_rstd[row], mean2 = kRms ? 0.0f : a.stats.pre_mean[row];
    const float rstd1 = post ? a.stats.post_rstd[row] : 1.0f, mean1 = post && !kRms ? a.stats.post_mean[row] : 0.0f;
    auto add = [&](uint32_t which, uint32_t c, float v) {
      float& at = sums[which * each + c];
      at = first ? v : at + v;
    };
    Sums<2> s = {{0.0f, 0.0f}};
    for (uint32_t c = threadIdx.x; c < a.cols; c += kThreads) {
      const float d = ToF32(dy[c]), v = (ToF32(x[c]) - mean2) * rstd2, q = d * a.w.pre_gamma[c];
      add(0, c, d * v);
      if (!kRms) add(1, c, d);
      s.v[0] += q * v;
      s.v[1] += q;
    }
    s = BlockSum<2>(s, slots, turn);
    const float pull = s.v[0] * per_col, shift = kRms ? 0.0f : s.v[1] * per_col;
    s = {{0.0f, 0.0f}};
    for (uint32_t c = threadIdx.x; c < a.cols; c += kThreads) {
      const float v = (ToF32(x[c]) - mean2) * rstd2, q = ToF32(dy[c]) * a.w.pre_gamma[c];
      float d = rstd2 * (q - shift - v * pull);
      if (dx_out) d += ToF32(dx_out[c]);
      buf[c] = d;
      dx[c] = FromF32<XT>(a.scale * d);
      const float u = (ToF32(b[c]) - mean1) * rstd1;
      add(2, c, d * u);
      if (!kRms) add(3, c, d);
      if (a.w.gate) d *= a.w.gate[c];
      if (post) d *= a.w.post_gamma[c];
      s.v[0] += d * u;
      s.v[1] += d;
    }
    float pull1 = 0.0f, shift1 = 0.0f;
    if (post) {
      s = BlockSum<2>(s, slots, turn);
      pull1 = s.v[0] * per_col;
      shift1 = kRms ? 0.0f : s.v[1] * per_col;
    }
    for (uint32_t c = threadIdx.x; c < a.cols; c += kThreads) {
      float d = buf[c];
      if (a.w.gate) d *= a.w.gate[c];
      if (post) {
        const float u = (ToF32(b[c]) - mean1) * rstd1;
        d = rstd1 * (d * a.w.post_gamma[c] - shift1 - u * pull1);
      }
      db[c] = FromF32<YT>(d);
    }
  }
}

// The blocks' partial sums of 32 columns, blockIdx.y 0: P1 and P2, 1: S1 and S2.  Half of the warps add a sum's rows w, w + 16, ...
// (rms: all of them, w + 32); then the warps' sums in order; then the weights' gradients.
__global__ void __launch_bounds__(1024)
JoinFoldKernel(const __grid_constant__ JoinArgs a, uint32_t blocks, int rms) {
  AwaitPrevious();
  __shared__ float meet[32][33];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane, col = blockIdx.x * 32 + warp;
  const uint32_t second = rms ? 0 : warp >> 4, way = rms ? warp : warp & 15, ways = rms ? 32 : 16;
  const float* p = a.partials + static_cast<size_t>(2 * blockIdx.y + second) * blocks * a.cols;
  float s = 0.0f;
  if (c < a.cols)
#pragma unroll 8
    for (uint32_t r = way; r < blocks; r += ways) s += p[static_cast<size_t>(r) * a.cols + c];
  meet[warp][lane] = s;
  __syncthreads();
  // Column `warp` of the block's 32, one warp's sum a lane: the first sum's in the lower lanes, the second's in the upper ones.
  s = meet[lane][warp];
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  const float upper = __shfl_sync(0xFFFFFFFFu, s, 16), first = rms ? s + upper : s;
  if (lane != 0 || col >= a.cols) return;
  if (blockIdx.y == 0) {
    a.grads.pre_gamma[col] = first;
    if (!rms) a.grads.pre_beta[col] = upper;
    return;
  }
  const bool post = a.w.post_gamma != nullptr;
  const float gate = a.w.gate ? a.w.gate[col] : 1.0f;
  if (post) {
    a.grads.post_gamma[col] = gate * first;
    if (!rms) a.grads.post_beta[col] = gate * upper;
  }
  if (a.w.gate) a.grads.gate[col] = !post ? first : a.w.post_gamma[col] * first + (rms ? 0.0f : a.w.post_beta[col] * upper);
}

// Rows of more columns than the ring kernels take.  (us, floors: forward 4096 x 12288 bf16 rms 160, 61, layer 232, 61; 4096 x 16384 f32 and
// bf16 rms 319, 123; backward 1243, 92, 1490, 92 and 1674, 184: it adds each row to four sums in global memory.)
template <typename XT, typename YT, bool kRms>
cudaError_t Pick(const JoinArgs& a, bool backward, cudaStream_t s, uint32_t* grid) {
  const size_t smem = a.cols * sizeof(float);
  if (!backward) {
    constexpr auto* kernel = JoinFwdKernel<XT, YT, kRms>;
    if (cudaError_t e = AllowShared<kernel>(smem); e != cudaSuccess) return e;
    return Next(kernel, static_cast<unsigned>(a.rows), kThreads, smem, s)(a);
  }
  constexpr auto* kernel = JoinBwdKernel<XT, YT, kRms>;
  if (cudaError_t e = AllowShared<kernel>(smem); e != cudaSuccess) return e;
  *grid = static_cast<uint32_t>(NormPartialRows(a.rows));
  return Next(kernel, *grid, kThreads, smem, s)(a);
}
template <typename XT, typename YT>
cudaError_t Pick(const JoinArgs& a, bool backward, cudaStream_t s, uint32_t* grid) {
  return a.rms ? Pick<XT, YT, true>(a, backward, s, grid) : Pick<XT, YT, false>(a, backward, s, grid);
}
cudaError_t Pick(const JoinArgs& a, bool backward, uint32_t sms, cudaStream_t s, uint32_t* grid) {
  if (a.cols <= kJoinRingCols) return backward ? JoinBackwardRing(a, sms, s, grid) : JoinForwardRing(a, sms, s);
  if (a.x_type == SEE_BF16) return Pick<Bf16, Bf16>(a, backward, s, grid);
  if (a.x_type == SEE_F16) return Pick<F16, F16>(a, backward, s, grid);
  if (a.y_type == SEE_BF16) return Pick<float, Bf16>(a, backward, s, grid);
  return a.y_type == SEE_F16 ? Pick<float, F16>(a, backward, s, grid) : Pick<float, float>(a, backward, s, grid);
}

}  // namespace

cudaError_t Join(const JoinArgs& a, bool backward, uint32_t sms, cudaStream_t s, int* launches) {
  uint32_t grid = 0;
  if (cudaError_t e = Pick(a, backward, sms, s, &grid); e != cudaSuccess) return e;
  ++*launches;
  if (!backward) return cudaSuccess;
  ++*launches;
  return Next(JoinFoldKernel, dim3((a.cols + 31) / 32, a.w.post_gamma || a.w.gate ? 2 : 1), 1024, 0, s)(a, grid, a.rms ? 1 : 0);
}

}  // namespace see::k
