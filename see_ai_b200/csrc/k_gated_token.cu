// The gated block's forward pass for one row (a token): bound by HBM, or by latency where the weights are small, for each
// weight is read and used once; the tensor cores' 256-row tiles would be empty.
//
// A thread holds eight consecutive columns of gate and up in f32 registers and walks down its share of d_in: sixteen 16-byte
// loads in flight, the first of them asked for before x is there, and packed multiply-adds with x from shared memory.  A block
// covers `columns` of d_hidden and an eighth of d_in, the eight blocks of a cluster all of it: the groups of a block meet in
// its shared memory, the blocks in distributed shared memory, where each finishes an eighth of the columns (sum in block order,
// activation, product), so nothing passes through global memory between.  Weights from HBM, this kernel / the tensor cores', us:
// 768 x 2048 5.3 / 7.0, 2048 x 5632 17 / 18, 4096 x 12288 44 / 55, 8192 x 28672 161 / 194.  (Two rows: 6.8 / 7.0, 19.7 / 18, 61 / 55.)
#include "act_expr.cuh"
#include "gated_act.cuh"
#include "gated_umma.h"
#include "launch.cuh"
#include "umma_device.cuh"
#include "vec_types.cuh"

namespace see::k {

namespace {

constexpr uint32_t kThreads = 256, kCluster = 8, kUnroll = 8;
constexpr uint32_t kMostDepth = 7680;   // of a block: x beside the sums in 48 KB

template <typename T> __device__ __forceinline__ void Pairs(const uint4& r, f32x2 (&v)[4]) {
  float f[8];
  Unpack2<T>(r.x, f[0], f[1]);
  Unpack2<T>(r.y, f[2], f[3]);
  Unpack2<T>(r.z, f[4], f[5]);
  Unpack2<T>(r.w, f[6], f[7]);
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = PackF2(f[2 * j], f[2 * j + 1]);
}
__device__ __forceinline__ float PeerFloat(const float* p, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(umma_dev::MapToCta(umma_dev::SmemAddr(p), rank)));
  return v;
}

// Shared memory: x of this block's share of d_in, then the groups' sums [groups][2][columns], whose first becomes the block's.
template <typename T>
__global__ void __launch_bounds__(kThreads)
GatedTokenKernel(const GatedTokenArgs a, uint32_t columns) {
  AwaitPrevious();
  extern __shared__ __align__(16) float token[];
  const uint32_t rank = umma_dev::ClusterCtaRank(), first_col = (blockIdx.x / kCluster) * columns;
  const uint32_t lanes = columns / 8, groups = kThreads / lanes, group = threadIdx.x / lanes, col = (threadIdx.x - group * lanes) * 8;
  const uint32_t share = (a.d_in + kCluster - 1) / kCluster, from = min(rank * share, a.d_in), depth = min(share, a.d_in - from);
  float* sums = token + share;
  const bool inside = first_col + col < a.d_hidden;
  const size_t at = static_cast<size_t>(from) * a.d_hidden + first_col + col;
  const T *wg = static_cast<const T*>(a.w_gate) + at, *wu = static_cast<const T*>(a.w_up) + at;
  uint4 g[kUnroll], u[kUnroll];
  auto ask = [&](uint32_t k, uint32_t d) {   // (weights are read once)
    if (!inside || d >= depth) return;
    g[k] = __ldcs(reinterpret_cast<const uint4*>(wg + static_cast<size_t>(d) * a.d_hidden));
    u[k] = __ldcs(reinterpret_cast<const uint4*>(wu + static_cast<size_t>(d) * a.d_hidden));
  };
#pragma unroll
  for (uint32_t k = 0; k < kUnroll; ++k) ask(k, group + k * groups);
  for (uint32_t i = threadIdx.x; i < depth; i += kThreads) token[i] = ToF32(static_cast<const T*>(a.x)[from + i]);
  __syncthreads();
  f32x2 gate[4] = {0, 0, 0, 0}, up[4] = {0, 0, 0, 0};
  for (uint32_t d = group; d < depth; d += kUnroll * groups) {
#pragma unroll
    for (uint32_t k = 0; k < kUnroll; ++k) {
      if (d + k * groups < depth) {
        f32x2 pg[4], pu[4];
        Pairs<T>(g[k], pg);
        Pairs<T>(u[k], pu);
        const f32x2 x = Splat2(token[d + k * groups]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          gate[j] = Fma2(x, pg[j], gate[j]);
          up[j] = Fma2(x, pu[j], up[j]);
        }
      }
    }
    // (The next batch behind the whole of this one: each load behind its own use kept fewer of them in flight, 84 us for 44.)
#pragma unroll
    for (uint32_t k = 0; k < kUnroll; ++k) ask(k, d + (kUnroll + k) * groups);
  }
  const uint32_t outputs = 2 * columns;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float* to = sums + group * outputs + col + 2 * j;
    UnpackF2(gate[j], &to[0], &to[1]);
    UnpackF2(up[j], &to[columns], &to[columns + 1]);
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < outputs; i += kThreads) {
    float s = sums[i];
    for (uint32_t k = 1; k < groups; ++k) s += sums[k * outputs + i];
    sums[i] = s;
  }
  umma_dev::ClusterSync();
  const uint32_t mine = columns / kCluster;   // columns that this block finishes
  if (threadIdx.x < mine) {
    const uint32_t c = rank * mine + threadIdx.x;
    if (first_col + c < a.d_hidden) {
      float gs = 0.0f, us = 0.0f;
#pragma unroll
      for (uint32_t k = 0; k < kCluster; ++k) {
        gs += PeerFloat(sums + c, k);
        us += PeerFloat(sums + columns + c, k);
      }
      const uint32_t to = first_col + c;
      const float value = a.act == kActSilu ? GatedAct<kActSilu>(gs) : a.act == kActGelu ? GatedAct<kActGelu>(gs) : GatedAct<kActRelu>(gs);
      static_cast<T*>(a.hidden)[to] = FromF32<T>(value * us);
      if (a.gate) {
        static_cast<T*>(a.gate)[to] = FromF32<T>(gs);
        static_cast<T*>(a.up)[to] = FromF32<T>(us);
      }
    }
  }
  umma_dev::ClusterSync();   // no block leaves while another may still read its sums
}

template <typename T>
cudaError_t Run(const GatedTokenArgs& a, uint32_t sms, cudaStream_t s) {
  // Rows of 512 bytes of the weights to a group, or shorter ones where that leaves fewer than two blocks to an SM (four were
  // slower: 4096 x 12288 44 us, 53).
  uint32_t columns = 256;
  while (columns > 64 && (a.d_hidden + columns - 1) / columns * kCluster < 2 * sms) columns /= 2;
  const uint32_t share = (a.d_in + kCluster - 1) / kCluster;
  const size_t smem = (share + static_cast<size_t>(kThreads) * 16) * 4;
  return Next(GatedTokenKernel<T>, (a.d_hidden + columns - 1) / columns * kCluster, kThreads, smem, s, kCluster)(a, columns);
}

}  // namespace

bool GatedTokenTakes(uint64_t rows, uint64_t d_in) { return rows == 1 && d_in <= kMostDepth * kCluster; }

cudaError_t GatedToken(const GatedTokenArgs& a, bool f16, uint32_t sms, cudaStream_t s) { return f16 ? Run<F16>(a, sms, s) : Run<Bf16>(a, sms, s); }

}  // namespace see::k
