// The backward pass of a block's join to the residual stream for rows of up to 8192 columns (k_join.cu has the formulas).
//
// As in the forward pass a row belongs to a group of T threads and reaches it through a ring, here all four of its matrices at once.  A
// thread has the same columns in every row, so that the four sums over rows stay in its registers; a block's groups meet in shared
// memory, the blocks in JoinFoldKernel, in a fixed order.
#include "join.cuh"

namespace see::k {

namespace {

template <typename XT, typename YT, bool kRms, int VEC, int NV, uint32_t kThreads>
__global__ void __launch_bounds__(kThreads, 1)
JoinBwdRingKernel(const __grid_constant__ JoinArgs a, uint32_t T, uint32_t slots, uint32_t edge) {
  using P = Lane<VEC>;
  constexpr int L = kLanes<VEC>;
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ __align__(8) float2 sums[2][kWideThreads / 32];
  const uint32_t groups = blockDim.x / T, group = threadIdx.x / T, t = threadIdx.x - group * T;
  const uint32_t x_slot = OddSlot<XT>(a.cols), y_slot = OddSlot<YT>(a.cols), pitch = (a.cols + 3) & ~3u;
  const uint32_t slot_bytes = (a.dx_out ? 2 : 1) * x_slot + 2 * y_slot;
  uint8_t* ring = dyn + static_cast<size_t>(group) * slots * slot_bytes;
  float* weights = reinterpret_cast<float*>(dyn + static_cast<size_t>(groups) * slots * slot_bytes);   // gamma2, A
  uint64_t* bars = reinterpret_cast<uint64_t*>(weights + 2 * pitch) + group * slots;
  const uint64_t first = static_cast<uint64_t>(blockIdx.x) * groups + group, step = static_cast<uint64_t>(gridDim.x) * groups;
  if (t == 0) {
    for (uint32_t i = 0; i < slots; ++i) umma_dev::MbarInit(&bars[i], 1);
    umma_dev::MbarInitFence();
  }
  auto inner = [&](uint64_t row) { return VEC == 4 || (row >= edge && row + edge < a.rows); };
  auto copy = [&](auto x, auto more, auto dy, auto b, uint8_t* dst, uint64_t* bar, uint32_t x_to, uint32_t more_to, uint32_t dy_to, uint32_t b_to) {
    umma_dev::MbarExpectTx(bar, x.bytes + dy.bytes + b.bytes + (a.dx_out ? more.bytes : 0));
    if (dy.bytes) umma_dev::BulkLoad(dst + dy_to, dy.from, dy.bytes, bar);
    if (x.bytes) umma_dev::BulkLoad(dst + 2 * y_slot + x_to, x.from, x.bytes, bar);
    if (b.bytes) umma_dev::BulkLoad(dst + y_slot + b_to, b.from, b.bytes, bar);
    if (a.dx_out && more.bytes) umma_dev::BulkLoad(dst + 2 * y_slot + x_slot + more_to, more.from, more.bytes, bar);
  };
  auto fill = [&](uint64_t row, uint32_t slot) {   // the group's thread 0
    uint8_t* dst = ring + static_cast<size_t>(slot) * slot_bytes;
    if (inner(row)) {
      copy(OddRow<XT>(a.x, row, a.x_stride, a.cols), OddRow<XT>(a.dx_out, row, a.x_stride, a.cols), OddRow<YT>(a.dy, row, a.y_stride, a.cols),
           OddRow<YT>(a.block, row, a.y_stride, a.cols), dst, &bars[slot], 0, 0, 0, 0);
    } else {
      const EndRow<XT> x(a.x, row, a.x_stride, a.cols), more(a.dx_out, row, a.x_stride, a.cols);
      const EndRow<YT> dy(a.dy, row, a.y_stride, a.cols), b(a.block, row, a.y_stride, a.cols);
      copy(x, more, dy, b, dst, &bars[slot], x.to, more.to, dy.to, b.to);
    }
  };
  AwaitPrevious();
  if (t == 0)
    for (uint32_t i = 0; i < slots && first + i * step < a.rows; ++i) fill(first + i * step, i);
  const bool post = a.w.post_gamma != nullptr;
  for (uint32_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
    const float gate = a.w.gate ? a.w.gate[c] : 1.0f;
    weights[c] = a.w.pre_gamma[c];
    weights[pitch + c] = post ? gate * a.w.post_gamma[c] : gate;
  }
  __syncthreads();
  const float per_col = 1.0f / static_cast<float>(a.cols);
  // (sums: P1, S1 and, layer, P2, S2)
  P p1[NV][L], s1[NV][L], p2[kRms ? 1 : NV][L], s2[kRms ? 1 : NV][L];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < L; ++j) {
      p1[i][j] = s1[i][j] = SplatOf<P>(0.0f);
      if (!kRms) p2[i][j] = s2[i][j] = SplatOf<P>(0.0f);
    }
  uint32_t turn = 0, slot = 0, parities = 0;   // a bit for each slot, of the copies that went through it
  float2 next2 = make_float2(0.0f, 0.0f), next1 = make_float2(0.0f, 1.0f);   // statistics, asked for a row ahead
  auto ask = [&](uint64_t row) {
    next2.y = a.stats.pre_rstd[row];
    if (!kRms) next2.x = a.stats.pre_mean[row];
    if (!post) return;
    next1.y = a.stats.post_rstd[row];
    if (!kRms) next1.x = a.stats.post_mean[row];
  };
  if (first < a.rows) ask(first);
  for (uint64_t row = first; row < a.rows; row += step) {
    const float2 two = next2, one = next1;
    if (row + step < a.rows) ask(row + step);
    uint8_t* at = ring + static_cast<size_t>(slot) * slot_bytes;
    if (!inner(row)) {
      CopyEnds<YT>(at, a.dy, row, a.y_stride, a.cols, t, T);
      CopyEnds<YT>(at + y_slot, a.block, row, a.y_stride, a.cols, t, T);
      CopyEnds<XT>(at + 2 * y_slot, a.x, row, a.x_stride, a.cols, t, T);
      if (a.dx_out) CopyEnds<XT>(at + 2 * y_slot + x_slot, a.dx_out, row, a.x_stride, a.cols, t, T);
      umma_dev::FenceProxyAsync();   // (the slot is filled in bulk again)
      GroupBarrier(T, group);
    }
    AwaitRow(&bars[slot], parities >> slot & 1u, a.status);
    parities ^= 1u << slot;
    auto x_skip = [&](const void* p) { return VEC == 4 ? 0 : reinterpret_cast<uint64_t>(static_cast<const XT*>(p) + row * a.x_stride) & 15; };
    auto y_skip = [&](const void* p) { return VEC == 4 ? 0 : reinterpret_cast<uint64_t>(static_cast<const YT*>(p) + row * a.y_stride) & 15; };
    const YT* dy = reinterpret_cast<const YT*>(at + y_skip(a.dy));
    const YT* b = reinterpret_cast<const YT*>(at + y_slot + y_skip(a.block));
    const XT* x = reinterpret_cast<const XT*>(at + 2 * y_slot + x_skip(a.x));
    const XT* more = reinterpret_cast<const XT*>(at + 2 * y_slot + x_slot + x_skip(a.dx_out));
    P d[NV][L], u[NV][L], with_u = SplatOf<P>(0.0f), plain = with_u;
    const P rstd2 = SplatOf<P>(two.y), away2 = SplatOf<P>(-two.x), rstd1 = SplatOf<P>(one.y), away1 = SplatOf<P>(-one.x), scale = SplatOf<P>(a.scale);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (t + i * T) * VEC;
      if (c < a.cols) {
        P g[L];
        LoadLanes<float, VEC>(weights + c, g);
        LoadLanes<YT, VEC>(dy + c, d[i]);
        LoadLanes<XT, VEC>(x + c, u[i]);
#pragma unroll
        for (int j = 0; j < L; ++j) {
          u[i][j] = Mul(kRms ? u[i][j] : Add(u[i][j], away2), rstd2);
          p1[i][j] = Fma(d[i][j], u[i][j], p1[i][j]);
          if (!kRms) p2[i][j] = Add(p2[i][j], d[i][j]);
          d[i][j] = Mul(d[i][j], g[j]);
          with_u = Fma(d[i][j], u[i][j], with_u);
          if (!kRms) plain = Add(plain, d[i][j]);
        }
      }
    }
    float2 sum = GroupSum<!kRms>(make_float2(Total(with_u), kRms ? 0.0f : Total(plain)), T, group, sums, turn);
    P pull = SplatOf<P>(-sum.x * per_col), shift = SplatOf<P>(-sum.y * per_col);
    with_u = plain = SplatOf<P>(0.0f);
    XT* dx = static_cast<XT*>(a.dx) + row * a.x_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (t + i * T) * VEC;
      if (c < a.cols) {
        P w[L], r[L];
        if (a.dx_out) {
          LoadLanes<XT, VEC>(more + c, r);
        } else {
#pragma unroll
          for (int j = 0; j < L; ++j) r[j] = SplatOf<P>(0.0f);
        }
#pragma unroll
        for (int j = 0; j < L; ++j) d[i][j] = Fma(Fma(u[i][j], pull, kRms ? d[i][j] : Add(d[i][j], shift)), rstd2, r[j]);
        LoadLanes<YT, VEC>(b + c, u[i]);
        LoadLanes<float, VEC>(weights + pitch + c, w);
#pragma unroll
        for (int j = 0; j < L; ++j) {
          r[j] = Mul(scale, d[i][j]);
          u[i][j] = Mul(kRms ? u[i][j] : Add(u[i][j], away1), rstd1);
          s1[i][j] = Fma(d[i][j], u[i][j], s1[i][j]);
          if (!kRms) s2[i][j] = Add(s2[i][j], d[i][j]);
          d[i][j] = Mul(d[i][j], w[j]);
          with_u = Fma(d[i][j], u[i][j], with_u);
          if (!kRms) plain = Add(plain, d[i][j]);
        }
        StoreLanes<XT, VEC>(dx + c, r);
      }
    }
    pull = shift = SplatOf<P>(0.0f);
    if (post) {
      sum = GroupSum<!kRms>(make_float2(Total(with_u), kRms ? 0.0f : Total(plain)), T, group, sums, turn);
      pull = SplatOf<P>(-sum.x * per_col);
      shift = SplatOf<P>(-sum.y * per_col);
    }
    if (!post || T == 32) GroupBarrier(T, group);   // the slot is read (a wider group has met at the sum's barrier)
    if (t == 0 && row + slots * step < a.rows) fill(row + slots * step, slot);
    if (++slot == slots) slot = 0;
    YT* db = static_cast<YT*>(a.dblock) + row * a.y_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (t + i * T) * VEC;
      if (c < a.cols) {
#pragma unroll
        for (int j = 0; j < L; ++j) d[i][j] = Mul(Fma(u[i][j], pull, kRms ? d[i][j] : Add(d[i][j], shift)), rstd1);
        StoreLanes<YT, VEC>(db + c, d[i]);
      }
    }
  }
  float* meet = reinterpret_cast<float*>(dyn);   // [groups][pitch]; every copy has been read
#pragma unroll
  for (int which = 0; which < 4; ++which) {
    if (kRms && (which & 1)) continue;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (t + i * T) * VEC;
      if (c < a.cols)
        StoreLanes<float, VEC>(meet + group * pitch + c, which == 0 ? p1[i] : which == 1 ? p2[kRms ? 0 : i] : which == 2 ? s1[i] : s2[kRms ? 0 : i]);
    }
    __syncthreads();
    float* out = a.partials + (static_cast<size_t>(which) * gridDim.x + blockIdx.x) * a.cols;
    for (uint32_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
      float s = meet[c];
      for (uint32_t r = 1; r < groups; ++r) s += meet[r * pitch + c];
      out[c] = s;
    }
  }
}

template <typename XT, typename YT, bool kRms, int VEC, int NV, uint32_t kThreads>
cudaError_t Run(const JoinArgs& a, uint32_t T, uint32_t sms, cudaStream_t s, uint32_t* grid) {
  const uint32_t pitch = (a.cols + 3) & ~3u;
  const size_t slot_bytes = OddSlot<XT>(a.cols) * (a.dx_out ? 2 : 1) + OddSlot<YT>(a.cols) * 2;
  const JoinRing r = RingOf(a.rows, kThreads, T, slot_bytes, static_cast<size_t>(pitch) * 8, sms);   // (a slot holds a row of floats)
  constexpr auto* kernel = JoinBwdRingKernel<XT, YT, kRms, VEC, NV, kThreads>;
  if (cudaError_t e = AllowShared<kernel>(r.bytes); e != cudaSuccess) return e;
  *grid = r.grid;
  return Next(kernel, r.grid, r.groups * T, r.bytes, s)(a, T, r.slots, JoinEdge(a));
}

template <typename XT, typename YT, bool kRms>
cudaError_t Pick(const JoinArgs& a, uint32_t sms, cudaStream_t s, uint32_t* grid) {
  // Sixteen columns to a thread at most: the four sums of layer norms take 64 registers, and a row's values 32.
  constexpr uint32_t kThreads = kRms ? 512 : 384;
  if (JoinFours(a, {a.x, a.dx_out, a.dx}, {a.dy, a.block, a.dblock})) {
    const uint32_t n = a.cols / 4;
    // Layer norms of wide rows: eight or twelve columns a thread (16384 x 4096 bf16 253 us, with sixteen, which spill, 304).
    if (!kRms && n > 768) {
      if (n <= 1024) return Run<XT, YT, kRms, 4, 2, 512>(a, Warps((n + 1) / 2), sms, s, grid);
      if (n <= 1536) return Run<XT, YT, kRms, 4, 3, 512>(a, Warps((n + 2) / 3), sms, s, grid);
    }
    if (a.rows <= sms) {   // a row to an SM: over as many threads as it has work for
      const uint32_t T = n < kThreads ? Warps(n) : kThreads;
      if (n <= T) return Run<XT, YT, kRms, 4, 1, kThreads>(a, T, sms, s, grid);
      if (n <= 2 * T) return Run<XT, YT, kRms, 4, 2, kThreads>(a, T, sms, s, grid);
    }
    // Rms norms: a warp's row, which needs no barriers, of up to 768 columns of 16 bits (32768 rows 58 us, on 64 threads 72; an f32
    // stream's rows leave the ring too few of them: 88, 83).
    if constexpr (kRms && sizeof(XT) == 2)
      if (n > 128 && n <= 192) return Run<XT, YT, kRms, 4, 6, 384>(a, 32, sms, s, grid);
    const uint32_t T = Warps((n + 3) / 4), each = (n + T - 1) / T;
    if (each <= 1) return Run<XT, YT, kRms, 4, 1, kThreads>(a, T, sms, s, grid);
    if (each <= 2) return Run<XT, YT, kRms, 4, 2, kThreads>(a, T, sms, s, grid);
    if (each <= 3) return Run<XT, YT, kRms, 4, 3, kThreads>(a, T, sms, s, grid);
    return T <= 192 ? Run<XT, YT, kRms, 4, 4, kThreads>(a, T, sms, s, grid) : Run<XT, YT, kRms, 4, 4, 512>(a, T, sms, s, grid);
  }
  const uint32_t T = Warps((a.cols + 15) / 16), each = (a.cols + T - 1) / T;
  if (each <= 4) return Run<XT, YT, kRms, 1, 4, kThreads>(a, T, sms, s, grid);
  if (each <= 8) return Run<XT, YT, kRms, 1, 8, kThreads>(a, T, sms, s, grid);
  if (each <= 12 && T <= 384) return Run<XT, YT, kRms, 1, 12, kThreads>(a, T, sms, s, grid);
  return T <= 192 ? Run<XT, YT, kRms, 1, 16, kThreads>(a, T, sms, s, grid) : Run<XT, YT, kRms, 1, 16, 512>(a, T, sms, s, grid);
}
template <typename XT, typename YT>
cudaError_t Pick(const JoinArgs& a, uint32_t sms, cudaStream_t s, uint32_t* grid) {
  return a.rms ? Pick<XT, YT, true>(a, sms, s, grid) : Pick<XT, YT, false>(a, sms, s, grid);
}

}  // namespace

cudaError_t JoinBackwardRing(const JoinArgs& a, uint32_t sms, cudaStream_t s, uint32_t* grid) {
  if (a.x_type == SEE_BF16) return Pick<Bf16, Bf16>(a, sms, s, grid);
  if (a.x_type == SEE_F16) return Pick<F16, F16>(a, sms, s, grid);
  if (a.y_type == SEE_BF16) return Pick<float, Bf16>(a, sms, s, grid);
  return a.y_type == SEE_F16 ? Pick<float, F16>(a, sms, s, grid) : Pick<float, float>(a, sms, s, grid);
}

}  // namespace see::k
