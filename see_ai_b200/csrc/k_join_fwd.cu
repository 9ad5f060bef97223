// The forward pass of a block's join to the residual stream for rows of up to 8192 columns (k_join.cu has the formulas).
//
// A row belongs to a group of T threads, which hold it in registers, four consecutive columns at a time or, where addresses or widths do
// not allow that, single ones T apart.  x and block reach the groups through rings in shared memory, filled by bulk copies; the weights,
// the gate already times the first norm's, lie there beside them.
#include "join.cuh"

namespace see::k {

namespace {

// The statistics of a group's row in v, of which a thread has the columns (t + i T) VEC below cols, and zeros beyond.
template <bool kRms, int VEC, int NV>
__device__ __forceinline__ float2 StatsOf(const Lane<VEC> (&v)[NV][kLanes<VEC>], uint32_t t, uint32_t T, uint32_t group, uint32_t cols, float eps,
                                          float per_col, float2 (*sums)[kWideThreads / 32], uint32_t& turn) {
  using P = Lane<VEC>;
  P total = SplatOf<P>(0.0f);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < kLanes<VEC>; ++j) total = kRms ? Fma(v[i][j], v[i][j], total) : Add(total, v[i][j]);
  const float sum = GroupSum<false>(make_float2(Total(total), 0.0f), T, group, sums, turn).x * per_col;
  if constexpr (kRms) {
    return make_float2(0.0f, 1.0f / sqrtf(sum + eps));
  } else {
    const P away = SplatOf<P>(-sum);
    P first = SplatOf<P>(0.0f), second = first;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((t + i * T) * VEC < cols) {
#pragma unroll
        for (int j = 0; j < kLanes<VEC>; ++j) {
          const P d = Add(v[i][j], away);
          first = Add(first, d);
          second = Fma(d, d, second);
        }
      }
    const float2 s = GroupSum<true>(make_float2(Total(first), Total(second)), T, group, sums, turn);
    const float off = s.x * per_col, var = Variance(s.y * per_col, off);
    return make_float2(isfinite(off) ? sum + off : sum, 1.0f / sqrtf(var + eps));
  }
}

template <typename XT, typename YT, bool kRms, int VEC, int NV, uint32_t kThreads>
__global__ void __launch_bounds__(kThreads, 1)
JoinFwdRingKernel(const __grid_constant__ JoinArgs a, uint32_t T, uint32_t slots, uint32_t edge) {
  using P = Lane<VEC>;
  constexpr int L = kLanes<VEC>;
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ __align__(8) float2 sums[2][kWideThreads / 32];
  const uint32_t groups = blockDim.x / T, group = threadIdx.x / T, t = threadIdx.x - group * T;
  const uint32_t x_slot = OddSlot<XT>(a.cols), y_slot = OddSlot<YT>(a.cols), slot_bytes = x_slot + y_slot, pitch = (a.cols + 3) & ~3u;
  uint8_t* ring = dyn + static_cast<size_t>(group) * slots * slot_bytes;
  float* weights = reinterpret_cast<float*>(dyn + static_cast<size_t>(groups) * slots * slot_bytes);   // A, gamma2 and, layer, g beta1, beta2
  uint64_t* bars = reinterpret_cast<uint64_t*>(weights + (kRms ? 2 : 4) * pitch) + group * slots;
  const uint64_t first = static_cast<uint64_t>(blockIdx.x) * groups + group, step = static_cast<uint64_t>(gridDim.x) * groups;
  if (t == 0) {
    for (uint32_t i = 0; i < slots; ++i) umma_dev::MbarInit(&bars[i], 1);
    umma_dev::MbarInitFence();
  }
  auto inner = [&](uint64_t row) { return VEC == 4 || (row >= edge && row + edge < a.rows); };
  auto fill = [&](uint64_t row, uint32_t slot) {   // the group's thread 0
    uint8_t* dst = ring + static_cast<size_t>(slot) * slot_bytes;
    if (inner(row)) {
      const OddRow<XT> x(a.x, row, a.x_stride, a.cols);
      const OddRow<YT> b(a.block, row, a.y_stride, a.cols);
      umma_dev::MbarExpectTx(&bars[slot], x.bytes + b.bytes);
      umma_dev::BulkLoad(dst + x_slot, b.from, b.bytes, &bars[slot]);
      umma_dev::BulkLoad(dst, x.from, x.bytes, &bars[slot]);
    } else {
      const EndRow<XT> x(a.x, row, a.x_stride, a.cols);
      const EndRow<YT> b(a.block, row, a.y_stride, a.cols);
      umma_dev::MbarExpectTx(&bars[slot], x.bytes + b.bytes);
      if (b.bytes) umma_dev::BulkLoad(dst + x_slot + b.to, b.from, b.bytes, &bars[slot]);
      if (x.bytes) umma_dev::BulkLoad(dst + x.to, x.from, x.bytes, &bars[slot]);
    }
  };
  AwaitPrevious();
  if (t == 0)
    for (uint32_t i = 0; i < slots && first + i * step < a.rows; ++i) fill(first + i * step, i);
  const bool post = a.w.post_gamma != nullptr;
  for (uint32_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
    const float gate = a.w.gate ? a.w.gate[c] : 1.0f;
    weights[c] = post ? gate * a.w.post_gamma[c] : gate;
    weights[pitch + c] = a.w.pre_gamma[c];
    if constexpr (!kRms) {
      weights[2 * pitch + c] = post ? gate * a.w.post_beta[c] : 0.0f;
      weights[3 * pitch + c] = a.w.pre_beta[c];
    }
  }
  __syncthreads();
  const float per_col = 1.0f / static_cast<float>(a.cols);
  uint32_t turn = 0, slot = 0, parities = 0;   // a bit for each slot, of the copies that went through it
  for (uint64_t row = first; row < a.rows; row += step) {
    uint8_t* at = ring + static_cast<size_t>(slot) * slot_bytes;
    if (!inner(row)) {
      CopyEnds<XT>(at, a.x, row, a.x_stride, a.cols, t, T);
      CopyEnds<YT>(at + x_slot, a.block, row, a.y_stride, a.cols, t, T);
      umma_dev::FenceProxyAsync();   // (the slot is filled in bulk again)
      GroupBarrier(T, group);
    }
    AwaitRow(&bars[slot], parities >> slot & 1u, a.status);
    parities ^= 1u << slot;
    const XT* x = reinterpret_cast<const XT*>(at + (VEC == 4 ? 0 : reinterpret_cast<uint64_t>(static_cast<const XT*>(a.x) + row * a.x_stride) & 15));
    const YT* b = reinterpret_cast<const YT*>(at + x_slot + (VEC == 4 ? 0 : reinterpret_cast<uint64_t>(static_cast<const YT*>(a.block) + row * a.y_stride) & 15));
    P v[NV][L];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (t + i * T) * VEC;
      if (c < a.cols) {
        LoadLanes<YT, VEC>(b + c, v[i]);
      } else {
#pragma unroll
        for (int j = 0; j < L; ++j) v[i][j] = SplatOf<P>(0.0f);
      }
    }
    float2 one = make_float2(0.0f, 1.0f);
    if (post) one = StatsOf<kRms, VEC, NV>(v, t, T, group, a.cols, a.eps, per_col, sums, turn);
    XT* x_out = static_cast<XT*>(a.x_out) + row * a.x_stride;
    const P scale = SplatOf<P>(a.scale), rstd1 = SplatOf<P>(one.y), away1 = SplatOf<P>(-one.x);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (t + i * T) * VEC;
      if (c < a.cols) {
        P w[L], beta[L], r[L];
        LoadLanes<float, VEC>(weights + c, w);
        if (!kRms) LoadLanes<float, VEC>(weights + 2 * pitch + c, beta);
        LoadLanes<XT, VEC>(x + c, r);
#pragma unroll
        for (int j = 0; j < L; ++j) {
          const P unit = Mul(kRms ? v[i][j] : Add(v[i][j], away1), rstd1);
          v[i][j] = Fma(scale, r[j], kRms ? Mul(unit, w[j]) : Fma(unit, w[j], beta[j]));
        }
        StoreLanes<XT, VEC>(x_out + c, v[i]);
      }
    }
    GroupBarrier(T, group);   // the slot is read
    if (t == 0 && row + slots * step < a.rows) fill(row + slots * step, slot);
    if (++slot == slots) slot = 0;
    const float2 two = StatsOf<kRms, VEC, NV>(v, t, T, group, a.cols, a.eps, per_col, sums, turn);
    const P rstd2 = SplatOf<P>(two.y), away2 = SplatOf<P>(-two.x);
    YT* y = static_cast<YT*>(a.y) + row * a.y_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (t + i * T) * VEC;
      if (c < a.cols) {
        P w[L], beta[L];
        LoadLanes<float, VEC>(weights + pitch + c, w);
        if (!kRms) LoadLanes<float, VEC>(weights + 3 * pitch + c, beta);
#pragma unroll
        for (int j = 0; j < L; ++j) {
          const P unit = Mul(kRms ? v[i][j] : Add(v[i][j], away2), rstd2);
          w[j] = kRms ? Mul(unit, w[j]) : Fma(unit, w[j], beta[j]);
        }
        StoreLanes<YT, VEC>(y + c, w);
      }
    }
    if (t == 0) {
      if (post) a.stats.post_rstd[row] = one.y;
      a.stats.pre_rstd[row] = two.y;
      if constexpr (!kRms) {
        if (post) a.stats.post_mean[row] = one.x;
        a.stats.pre_mean[row] = two.x;
      }
    }
  }
}

template <typename XT, typename YT, bool kRms, int VEC, int NV, uint32_t kThreads>
cudaError_t Run(const JoinArgs& a, uint32_t T, uint32_t sms, cudaStream_t s) {
  const size_t weights = static_cast<size_t>((a.cols + 3) & ~3u) * 4 * (kRms ? 2 : 4);
  const JoinRing r = RingOf(a.rows, kThreads, T, OddSlot<XT>(a.cols) + OddSlot<YT>(a.cols), weights, sms);
  constexpr auto* kernel = JoinFwdRingKernel<XT, YT, kRms, VEC, NV, kThreads>;
  if (cudaError_t e = AllowShared<kernel>(r.bytes); e != cudaSuccess) return e;
  return Next(kernel, r.grid, r.groups * T, r.bytes, s)(a, T, r.slots, JoinEdge(a));
}

template <typename XT, typename YT, bool kRms>
cudaError_t Pick(const JoinArgs& a, uint32_t sms, cudaStream_t s) {
  if (JoinFours(a, {a.x, a.x_out}, {a.block, a.y})) {
    const uint32_t n = a.cols / 4;
    if (a.rows <= sms) {   // a row to an SM: over as many threads as it has work for
      const uint32_t T = n < 512 ? Warps(n) : 512;
      if (n <= T) return Run<XT, YT, kRms, 4, 1, 512>(a, T, sms, s);
      return n <= 2 * T ? Run<XT, YT, kRms, 4, 2, 512>(a, T, sms, s) : Run<XT, YT, kRms, 4, 4, 512>(a, T, sms, s);
    }
    const uint32_t T = Warps((n + 7) / 8), each = (n + T - 1) / T;
    if (each <= 2) return Run<XT, YT, kRms, 4, 2, 512>(a, T, sms, s);
    if (each <= 4) return Run<XT, YT, kRms, 4, 4, 512>(a, T, sms, s);
    return each <= 6 ? Run<XT, YT, kRms, 4, 6, 512>(a, T, sms, s) : Run<XT, YT, kRms, 4, 8, 512>(a, T, sms, s);
  }
  const uint32_t T = Warps((a.cols + 15) / 16), each = (a.cols + T - 1) / T;
  if (each <= 4) return Run<XT, YT, kRms, 1, 4, 512>(a, T, sms, s);
  if (each <= 8) return Run<XT, YT, kRms, 1, 8, 512>(a, T, sms, s);
  return each <= 12 ? Run<XT, YT, kRms, 1, 12, 768>(a, T, sms, s) : Run<XT, YT, kRms, 1, 16, 768>(a, T, sms, s);
}
template <typename XT, typename YT>
cudaError_t Pick(const JoinArgs& a, uint32_t sms, cudaStream_t s) {
  return a.rms ? Pick<XT, YT, true>(a, sms, s) : Pick<XT, YT, false>(a, sms, s);
}

}  // namespace

cudaError_t JoinForwardRing(const JoinArgs& a, uint32_t sms, cudaStream_t s) {
  if (a.x_type == SEE_BF16) return Pick<Bf16, Bf16>(a, sms, s);
  if (a.x_type == SEE_F16) return Pick<F16, F16>(a, sms, s);
  if (a.y_type == SEE_BF16) return Pick<float, Bf16>(a, sms, s);
  return a.y_type == SEE_F16 ? Pick<float, F16>(a, sms, s) : Pick<float, float>(a, sms, s);
}

}  // namespace see::k
