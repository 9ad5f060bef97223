// The gated feed-forward block on the tensor cores: hidden = act(x Wg) * (x Wu) in one kernel, and the products of its
// backward pass, dx = dg Wg^T + du Wu^T, dWg = x^T dg, dWu = x^T du, in one launch behind the element-wise dg and du.
//
// A persistent kernel of CTA pairs (cta_group::2): a pair owns a tile of 256 rows by kTN accumulator columns, each CTA loads
// its own 128 rows of A and its own half of the columns' B, the even CTA issues the 256-row MMAs, and each CTA's tensor memory
// receives its 128 rows.  Forward: the even CTA's half of B is the gate's columns and the odd one's the up projection's, so
// one MMA makes both, and column j's two factors lie kTN / 2 columns apart in one thread's lane: the activation and the
// product need no exchange.  The accumulator is double-buffered: a tile's epilogue (eight warps) runs under the next one's
// products.  (Sixteen warps with slabs of 32 columns: 32768 x 768 x 2048 177 us / 219, for rows of 64 bytes leave worse.)
//
// No operand is ever transposed or copied: x, the weights [d_in, d_hidden] and dg, du lie as the caller has them, and a box of
// 64 x 64 elements under the 128-byte swizzle is a K-major operand where the reduction runs along its rows and an MN-major one
// where it runs down its columns (one descriptor bit).  x is K-major forward and MN-major for dW; the weights are MN-major
// forward and K-major for dx.
//
// Bound by the tensor pipe: 256 x 256 x 64 of a pair are 512 cycles.  4096 x 4096 x 4096 forward, gate and up kept: 191 us,
// 1440 TFLOP/s, where the library's product did one of the two at 1230 on the same board; busy 66 to 75 % of a launch's cycles under the
// profiler.  With d_in = 768 a tile's products (6100 cycles) are shorter than its three stores: 32768 x 768 x 2048 177 us, 152
// without gate and up.  dg and du are rounded to the operands' 16 bits between the passes, as the products take them: half a step
// of each term, which leaves dx and dW 1.4 times one rounding's error.
#include <atomic>

#include "gated_act.cuh"
#include "gated_umma.h"
#include "launch.cuh"
#include "umma_device.cuh"
#include "vec_types.cuh"

namespace see::k {

namespace {

using namespace umma_dev;

constexpr uint32_t kRows = 128;            // a CTA's rows of a tile
constexpr uint32_t kBlockK = 64;
constexpr uint32_t kBoxBytes = 64 * 64 * 2;
constexpr uint32_t kEpiWarps = 8;
constexpr uint32_t kThreads = 64 + 32 * kEpiWarps;   // warp 0 TMA, warp 1 MMA, then the epilogue warps
constexpr uint32_t kSlabBytes = 32 * 128;  // 32 rows of 64 16-bit columns
constexpr uint32_t kBand = 8;              // row tiles that share a column tile's B before the next column tile

template <uint32_t kTN>
struct Tile {
  static constexpr uint32_t kHalf = kTN / 2;                             // columns of B a CTA loads
  static constexpr uint32_t kABytes = kRows * kBlockK * 2, kBBytes = kHalf * kBlockK * 2;
  static constexpr uint32_t kStageBytes = kABytes + kBBytes;
  static constexpr uint32_t kStages = kTN == 256 ? 6 : 8;
  static constexpr uint32_t kSmem = kStages * kStageBytes + kEpiWarps * kSlabBytes + 256 + 1024;
};

struct __align__(8) Barriers {
  uint64_t full[8], empty[8];
  uint64_t tmem_full[2], tmem_empty[2];
  uint32_t tmem_base;
  volatile uint32_t abort;
};

// A tile may take as long as its reduction: longer waits than a ring's, as bounded.
__device__ __forceinline__ bool Wait(uint64_t* bar, uint32_t parity) {
  for (int i = 0; i < 16; ++i)
    if (MbarWait(bar, parity)) return true;
  return false;
}

// A work item: a tile, or part `part` of `parts` of its reduction (blocks from, to).  Whole tiles come first.
struct At { uint32_t p, m_tile, n_tile, part, parts, from, to; };
__device__ __forceinline__ void TileAt(const GatedProblem& p, uint32_t t, uint32_t& m_tile, uint32_t& n_tile) {
  const uint32_t per_band = kBand * p.tiles_n, band = t / per_band, within = t - band * per_band, first = band * kBand;
  const uint32_t height = p.tiles_m - first < kBand ? p.tiles_m - first : kBand;
  n_tile = within / height;
  m_tile = first + within - n_tile * height;
}
__device__ __forceinline__ At Locate(const GatedLaunch& l, uint32_t t) {
  At at;
  at.part = 0;
  at.parts = 1;
  at.p = 0;
  while (at.p < l.count && t >= l.p[at.p].whole) t -= l.p[at.p++].whole;
  if (at.p == l.count) {   // among the parts
    at.p = 0;
    while (true) {
      const GatedProblem& p = l.p[at.p];
      const uint32_t items = (p.tiles_m * p.tiles_n - p.whole) * p.parts;
      if (at.p + 1 == l.count || t < items) break;
      t -= items;
      ++at.p;
    }
    at.parts = l.p[at.p].parts;
    at.part = t % at.parts;
    t = l.p[at.p].whole + t / at.parts;
  }
  const GatedProblem& p = l.p[at.p];
  TileAt(p, t, at.m_tile, at.n_tile);
  const uint32_t blocks = p.blocks[0] + p.blocks[1];
  at.from = static_cast<uint32_t>(static_cast<uint64_t>(blocks) * at.part / at.parts);
  at.to = static_cast<uint32_t>(static_cast<uint64_t>(blocks) * (at.part + 1) / at.parts);
  if (at.parts > 1) at.part += p.first_part + (t - p.whole) * at.parts;   // from here on its place among all parts
  return at;
}
__host__ __device__ inline uint32_t Items(const GatedLaunch& l) {
  uint32_t n = 0;
  for (uint32_t p = 0; p < l.count; ++p) n += l.p[p].whole + (l.p[p].tiles_m * l.p[p].tiles_n - l.p[p].whole) * l.p[p].parts;
  return n;
}

// 64 columns of this lane's row: the slab's row by 16-byte chunks, as the 128-byte swizzle places them.
template <typename T>
__device__ __forceinline__ void PutHalfSlab(uint8_t* slab, uint32_t lane, uint32_t half, const float (&v)[32]) {
#pragma unroll
  for (uint32_t c = 0; c < 4; ++c) {
    const float* q = v + 8 * c;
    *reinterpret_cast<uint4*>(slab + Sw128Offset(lane, half * 4 + c)) =
        make_uint4(Pack2<T>(q[0], q[1]), Pack2<T>(q[2], q[3]), Pack2<T>(q[4], q[5]), Pack2<T>(q[6], q[7]));
  }
}

// An epilogue warp's slab, written again once the store before has read it (a second slab each took the ring's sixth stage:
// 32768 x 768 x 2048 185 us, 177 with the stage).
struct Slab {
  uint8_t* base;
  __device__ __forceinline__ uint8_t* Await() {
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");   // (of the lane that commits; none for the others)
    __syncwarp();
    return base;
  }
  __device__ __forceinline__ void Store(const CUtensorMap* map, uint32_t col, uint32_t row, bool inside) {
    FenceProxyAsync();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) {
      if (inside) TmaStore2D(map, base, static_cast<int32_t>(col), static_cast<int32_t>(row));
      TmaStoreCommit();
    }
  }
};

__device__ __forceinline__ void LoadAcc(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  TmemLoad32(taddr, r);
  TmemWaitLd();
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

template <typename T>
__device__ __forceinline__ void PlainSlab(Slab& out, const CUtensorMap* map, uint32_t taddr, uint32_t col, uint32_t row, bool inside) {
  const uint32_t lane = threadIdx.x & 31;
  uint8_t* slab = out.Await();
#pragma unroll
  for (uint32_t h = 0; h < 2; ++h) {
    float v[32];
    LoadAcc(taddr + 32 * h, v);
    PutHalfSlab<T>(slab, lane, h, v);
  }
  out.Store(map, col, row, inside);
}

// hidden = act(gate) up of 64 columns, from accumulators `apart` columns apart.
template <typename T, int kAct>
__device__ __forceinline__ void HiddenSlab(Slab& out, const CUtensorMap* map, uint32_t taddr, uint32_t apart, uint32_t col, uint32_t row,
                                           bool inside) {
  const uint32_t lane = threadIdx.x & 31;
  uint8_t* slab = out.Await();
#pragma unroll
  for (uint32_t h = 0; h < 2; ++h) {
    float g[32], u[32];
    LoadAcc(taddr + 32 * h, g);
    LoadAcc(taddr + apart + 32 * h, u);
#pragma unroll
    for (int i = 0; i < 32; ++i) g[i] = GatedAct<kAct>(g[i]) * u[i];
    PutHalfSlab<T>(slab, lane, h, g);
  }
  out.Store(map, col, row, inside);
}

template <typename T>
__device__ __forceinline__ void GatedColumns(Slab& out, const GatedLaunch& l, uint32_t taddr, uint32_t apart, uint32_t col, uint32_t row,
                                             bool inside) {
  if (l.act == kActSilu) HiddenSlab<T, kActSilu>(out, &l.p[0].c, taddr, apart, col, row, inside);
  else if (l.act == kActGelu) HiddenSlab<T, kActGelu>(out, &l.p[0].c, taddr, apart, col, row, inside);
  else HiddenSlab<T, kActRelu>(out, &l.p[0].c, taddr, apart, col, row, inside);
  if (l.keep) {
    PlainSlab<T>(out, &l.gate, taddr, col, row, inside);
    PlainSlab<T>(out, &l.up, taddr + apart, col, row, inside);
  }
}

template <uint32_t kTN, bool kGated>
__global__ void __launch_bounds__(kThreads, 1)
GatedProductsKernel(const __grid_constant__ GatedLaunch l) {
  using C = Tile<kTN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (SmemAddr(smem_raw) & 1023u)) & 1023u);
  uint8_t* slabs = smem + C::kStages * C::kStageBytes;
  Barriers* bars = reinterpret_cast<Barriers*>(slabs + kEpiWarps * kSlabBytes);
  static_assert(sizeof(Barriers) <= 256);

  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = ClusterCtaRank(), unit = blockIdx.x >> 1, units = gridDim.x >> 1;
  const uint32_t total = Items(l);

  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < C::kStages; ++s) {
      MbarInit(&bars->full[s], 1);
      MbarInit(&bars->empty[s], 1);
    }
    for (uint32_t b = 0; b < 2; ++b) {
      MbarInit(&bars->tmem_full[b], 1);
      MbarInit(&bars->tmem_empty[b], 2 * kEpiWarps);   // the even CTA's counts the epilogue warps of both
    }
    bars->abort = 0;
    MbarInitFence();
  }
  if (warp == 1) TmemAllocPair(&bars->tmem_base, 2 * kTN);
  TcFenceBefore();
  __syncthreads();
  ClusterSync();   // the peer's barriers exist before anything signals them
  TcFenceAfter();
  AwaitPrevious();
  const uint32_t tmem_base = bars->tmem_base;
  auto give_up = [&] {
    l.status->wait_timeout = 1;
    bars->abort = 1;
  };

  if (warp == 0) {
    if (lane == 0) {   // ---- TMA
      uint32_t it = 0;
      bool ok = true;
      for (uint32_t t = unit; t < total && ok; t += units) {
        const At at = Locate(l, t);
        const GatedProblem& p = l.p[at.p];
        const uint32_t m0 = at.m_tile * 2 * kRows + rank * kRows;
        const uint32_t n0 = kGated ? at.n_tile * C::kHalf : at.n_tile * kTN + rank * C::kHalf;
        for (uint32_t kb = at.from; kb < at.to; ++kb, ++it) {
          const uint32_t pair = kb < p.blocks[0] ? 0 : 1;
          const CUtensorMap *ma = &p.a[pair], *mb = kGated ? &p.b[rank] : &p.b[pair];
          const uint32_t s = it % C::kStages, round = it / C::kStages;
          if (round > 0 && !Wait(&bars->empty[s], (round - 1) & 1)) {
            give_up();
            ok = false;
            break;
          }
          if (rank == 0) MbarExpectTx(&bars->full[s], 2 * C::kStageBytes);   // both CTAs' bytes
          const uint32_t full = MapToCta(SmemAddr(&bars->full[s]), 0);
          uint8_t* dst = smem + s * C::kStageBytes;
          const int32_t k0 = static_cast<int32_t>((kb - (pair ? p.blocks[0] : 0)) * kBlockK);
#pragma unroll
          for (uint32_t i = 0; i < kRows / 64; ++i) {
            const int32_t r = static_cast<int32_t>(m0 + 64 * i);
            TmaLoad2DPair(dst + i * kBoxBytes, ma, full, p.a_mn ? r : k0, p.a_mn ? k0 : r);
          }
#pragma unroll
          for (uint32_t i = 0; i < C::kHalf / 64; ++i) {
            const int32_t r = static_cast<int32_t>(n0 + 64 * i);
            TmaLoad2DPair(dst + C::kABytes + i * kBoxBytes, mb, full, p.b_mn ? r : k0, p.b_mn ? k0 : r);
          }
        }
      }
    }
  } else if (warp == 1) {
    if (ElectOne() && rank == 0) {   // ---- MMA
      uint32_t it = 0, lt = 0;
      bool ok = true;
      for (uint32_t t = unit; t < total && ok; t += units, ++lt) {
        const At at = Locate(l, t);
        const GatedProblem& p = l.p[at.p];
        const uint32_t idesc = ((1u << 4) | ((kTN >> 3) << 17) | ((2 * kRows >> 4) << 24)) | (l.f16 ? 0u : (1u << 7) | (1u << 10)) |
                               (p.a_mn << 15) | (p.b_mn << 16);
        const uint32_t step_a = p.a_mn ? 2048 / 16 : 2, step_b = p.b_mn ? 2048 / 16 : 2;   // 16 along K, in a descriptor
        const uint32_t buf = lt & 1, use = lt >> 1;
        if (use > 0 && !Wait(&bars->tmem_empty[buf], (use - 1) & 1)) {
          give_up();
          break;
        }
        TcFenceAfter();
        const uint32_t acc = tmem_base + buf * kTN;
        for (uint32_t kb = at.from; kb < at.to; ++kb, ++it) {
          const uint32_t s = it % C::kStages, round = it / C::kStages;
          if (!Wait(&bars->full[s], round & 1)) {
            give_up();
            ok = false;
            break;
          }
          TcFenceAfter();
          const uint32_t a_addr = SmemAddr(smem + s * C::kStageBytes), b_addr = a_addr + C::kABytes;
          // (of an operand whose 64-element groups are not MN-major, the group stride is ignored)
          const uint64_t desc_a = MakeSmemDescMn(a_addr, p.a_mn ? kBoxBytes : 16), desc_b = MakeSmemDescMn(b_addr, p.b_mn ? kBoxBytes : 16);
#pragma unroll
          for (uint32_t k = 0; k < kBlockK / 16; ++k)
            UmmaBf16Pair(acc, desc_a + step_a * k, desc_b + step_b * k, idesc, kb != at.from || k != 0 ? 1u : 0u);
          UmmaCommitPair(&bars->empty[s], 0);
        }
        UmmaCommitPair(&bars->tmem_full[buf], 0);
      }
    }
  } else {   // ---- epilogue: TMEM lane quarter = warp % 4; the two warps of a quarter share the columns
    const uint32_t quarter = warp & 3, which = (warp - 2) >> 2;
    Slab slab{slabs + (warp - 2) * kSlabBytes};
    uint32_t lt = 0;
    for (uint32_t t = unit; t < total; t += units, ++lt) {
      const uint32_t buf = lt & 1, use = lt >> 1;
      const At at = Locate(l, t);
      const GatedProblem& p = l.p[at.p];
      bool there = Wait(&bars->tmem_full[buf], use & 1);
      if (!there && lane == 0) give_up();
      if (bars->abort) there = false;
      if (!__all_sync(0xFFFFFFFFu, there)) break;
      TcFenceAfter();
      const uint32_t row = at.m_tile * 2 * kRows + rank * kRows + quarter * 32;
      const uint32_t lanes = tmem_base + buf * kTN + ((quarter * 32) << 16);
      constexpr uint32_t kCols = kGated ? C::kHalf : kTN;   // output columns of the tile, 64 to a slab
      for (uint32_t c = which * 64; c < kCols; c += 128) {
        const uint32_t col = at.n_tile * kCols + c;
        if (!kGated && at.parts > 1) {
          // [4 columns][256 rows][4]: a warp's store is 512 bytes in a row
          float4* to = reinterpret_cast<float4*>(l.partials + static_cast<size_t>(at.part) * 2 * kRows * kTN) + (c / 4) * 2 * kRows + rank * kRows +
                       quarter * 32 + lane;
#pragma unroll
          for (uint32_t h = 0; h < 2; ++h) {
            float v[32];
            LoadAcc(lanes + c + 32 * h, v);
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) to[(8 * h + i) * 2 * kRows] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
          }
        } else if (kGated) {
          if (l.f16) GatedColumns<F16>(slab, l, lanes + c, C::kHalf, col, row, row < p.M && col < p.N);
          else GatedColumns<Bf16>(slab, l, lanes + c, C::kHalf, col, row, row < p.M && col < p.N);
        } else {
          if (l.f16) PlainSlab<F16>(slab, &p.c, lanes + c, col, row, row < p.M && col < p.N);
          else PlainSlab<Bf16>(slab, &p.c, lanes + c, col, row, row < p.M && col < p.N);
        }
      }
      TcFenceBefore();
      __syncwarp();
      if (lane == 0) MbarArriveCluster(MapToCta(SmemAddr(&bars->tmem_empty[buf]), 0));
    }
    TmaStoreWaitAll();
  }

  TcFenceBefore();
  __syncthreads();
  if (bars->abort) DrainDelay();
  ClusterSync();   // neither CTA leaves while the other may still read its memories
  if (warp == 1) {
    TcFenceAfter();
    TmemFreePair(tmem_base, 2 * kTN);
  }
}

constexpr uint32_t kFoldTN = 256;   // (cuts are the backward pass's, whose tiles have no other width)
// 32 rows x 64 columns of a cut tile a block: its parts added in order, turned to rows in shared memory, stored.
template <typename T>
__global__ void __launch_bounds__(256)
GatedFoldKernel(const __grid_constant__ GatedLaunch l) {
  AwaitPrevious();
  __shared__ float turn[32][65];
  constexpr uint32_t across = kFoldTN / 64, per_tile = 8 * across;   // blocks
  uint32_t t = blockIdx.x / per_tile, q = 0;
  const uint32_t within = blockIdx.x - t * per_tile;
  while (q + 1 < l.count && t >= l.p[q].tiles_m * l.p[q].tiles_n - l.p[q].whole) {
    t -= l.p[q].tiles_m * l.p[q].tiles_n - l.p[q].whole;
    ++q;
  }
  const GatedProblem& p = l.p[q];
  uint32_t m_tile, n_tile;
  TileAt(p, p.whole + t, m_tile, n_tile);
  const uint32_t r0 = (within / across) * 32, c0 = (within % across) * 64;   // in the tile
  if (m_tile * 256 + r0 >= p.M || n_tile * kFoldTN + c0 >= p.N) return;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr size_t part_floats = 256ull * kFoldTN;
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i) {
    const uint32_t c4 = warp + 8 * i;   // four columns of the block's 64
    const float4* from = reinterpret_cast<const float4*>(l.partials + (p.first_part + static_cast<size_t>(t) * p.parts) * part_floats) +
                         (c0 / 4 + c4) * 256 + r0 + lane;
    float4 sum = from[0];
    for (uint32_t k = 1; k < p.parts; ++k) {
      const float4 v = from[k * (part_floats / 4)];
      sum = make_float4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
    }
    float* to = &turn[lane][c4 * 4];
    to[0] = sum.x;
    to[1] = sum.y;
    to[2] = sum.z;
    to[3] = sum.w;
  }
  __syncthreads();
  const uint32_t row = threadIdx.x >> 3, c = (threadIdx.x & 7) * 8;   // eight columns a thread
  const uint32_t m = m_tile * 256 + r0 + row, n = n_tile * kFoldTN + c0 + c;
  if (m < p.M && n < p.N) Store8<T>(static_cast<T*>(p.out) + m * p.out_stride + n, &turn[row][c]);
}

template <typename T, int kAct>
__global__ void __launch_bounds__(256)
GatedSlopesKernel(const T* __restrict__ dh, const T* __restrict__ g, const T* __restrict__ u, T* __restrict__ dg, T* __restrict__ du,
                  uint64_t vectors, uint32_t row_vectors, uint64_t stride) {
  AwaitPrevious();
  for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < vectors; i += gridDim.x * 256ull) {
    const uint64_t row = i / row_vectors, at = row * stride + (i - row * row_vectors) * 8;
    float d[8], a[8], b[8];
    Load8<T>(dh + at, d);
    Load8<T>(g + at, a);
    Load8<T>(u + at, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float value, slope;
      GatedActAndSlope<kAct>(a[j], value, slope);
      a[j] = d[j] * b[j] * slope;
      b[j] = d[j] * value;
    }
    Store8<T>(dg + i * 8, a);
    Store8<T>(du + i * 8, b);
  }
}

template <typename T>
cudaError_t Slopes(const void* dh, const void* g, const void* u, void* dg, void* du, uint64_t rows, uint32_t cols, uint64_t stride, int act,
                   uint32_t sms, cudaStream_t s) {
  auto* kernel = act == kActSilu ? GatedSlopesKernel<T, kActSilu> : act == kActGelu ? GatedSlopesKernel<T, kActGelu> : GatedSlopesKernel<T, kActRelu>;
  const uint64_t vectors = rows * (cols / 8), blocks = (vectors + 255) / 256, most = sms * 8ull;
  return Next(kernel, static_cast<unsigned>(blocks < most ? blocks : most), 256, 0, s)(
      static_cast<const T*>(dh), static_cast<const T*>(g), static_cast<const T*>(u), static_cast<T*>(dg), static_cast<T*>(du), vectors,
      cols / 8, stride);
}

template <uint32_t kTN, bool kGated>
cudaError_t Run(const GatedLaunch& l, uint32_t sms, cudaStream_t s) {
  auto* kernel = GatedProductsKernel<kTN, kGated>;
  // The shared-memory limit is a device's: one flag for each.
  static std::atomic<bool> configured[64] = {};
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<kTN>::kSmem); e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
  }
  const uint64_t tiles = Items(l), pairs = sms / 2;
  return Next(kernel, static_cast<unsigned>(2 * (tiles < pairs ? tiles : pairs)), kThreads, Tile<kTN>::kSmem, s, 2)(l);
}

}  // namespace

cudaError_t GatedProducts(const GatedLaunch& l, bool gated, uint32_t tn, uint32_t sms, cudaStream_t s) {
  if (!gated) return Run<256, false>(l, sms, s);
  return tn == 256 ? Run<256, true>(l, sms, s) : Run<128, true>(l, sms, s);
}

cudaError_t GatedFold(const GatedLaunch& l, cudaStream_t s) {
  uint32_t tiles = 0;
  for (uint32_t p = 0; p < l.count; ++p) tiles += l.p[p].tiles_m * l.p[p].tiles_n - l.p[p].whole;
  const unsigned grid = tiles * 8 * (kFoldTN / 64);
  return l.f16 ? Next(GatedFoldKernel<F16>, grid, 256, 0, s)(l) : Next(GatedFoldKernel<Bf16>, grid, 256, 0, s)(l);
}

cudaError_t GatedSlopes(const void* dh, const void* g, const void* u, void* dg, void* du, uint64_t rows, uint32_t cols, uint64_t stride,
                        int act, bool f16, uint32_t sms, cudaStream_t s) {
  return f16 ? Slopes<F16>(dh, g, u, dg, du, rows, cols, stride, act, sms, s) : Slopes<Bf16>(dh, g, u, dg, du, rows, cols, stride, act, sms, s);
}

}  // namespace see::k
