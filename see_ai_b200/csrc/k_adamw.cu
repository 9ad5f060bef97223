// AdamW over many tensors in one launch, with moments in f32 or in 8 bits.
//
//   m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g g,
//   p -= lr (m inv_bc1 / (sqrt(v inv_bc2) + eps) + weight_decay p)
//
// in the expression of the kAdamWStep instruction, compiled without fused multiply-adds: with f32 moments and gradients the
// bits are that instruction's.  Moments in 8 bits: m and sqrt(v) as e4m3, each block of 256 elements with an f32 scale that
// puts its largest on 448.  sqrt(v) because its exponents span half of v's, which e4m3's 2^18 between the largest and the
// smallest then cover.  The arithmetic between reading and writing them is f32 (sqrt(v inv_bc2) as sqrt(v) sqrt(inv_bc2):
// one root, not two).
//
// Their rounding: e4m3 keeps three bits after the leading one, and a second moment moves by a thousandth a step, so to
// nearest it would never move.  The cut instead adds a 20-bit number to the 20 bits that go, which takes the upper
// neighbour in proportion to the distance: element i of a tensor at step t adds the top bits of
// (i phi + t sqrt(2)) mod 1 (phi the golden section), spread evenly over elements and over steps.  A root that is not zero
// is held as at least the smallest e4m3: a zero would let a later step divide by eps alone.
//
// Bound by HBM: 14 bytes an element with 16-bit gradients and moments in 8 bits (16 with a 16-bit copy), 28 in f32.  A warp
// takes blocks of 256 elements, eight a lane, through a ring of two in shared memory that bulk copies fill: the loads of a step
// straight into registers left half of the bandwidth unused (587 us of 110 million weights, 304 to 339 so, by the board: 5.2 to 5.8 TB/s).  Of the
// instructions, which came next, the roots, quotients and conversions went to the hardware's approximations with a Newton step,
// and to two elements at once.  The launch carries the table of tensors as a parameter: nothing is uploaded, and a captured
// launch owns its copy.
#include <atomic>
#include <type_traits>

#include "act_expr.cuh"
#include "block_ops.h"
#include "launch.cuh"
#include "umma_device.cuh"
#include "vec_types.cuh"

namespace see::k {

namespace {

constexpr uint32_t kGolden = 0x9E3779B9u;       // 2^32 times the golden section
constexpr uint32_t kHalfTurn = 0x80000000u;     // between the words of m and of sqrt(v)

struct AdamEntry {
  float* p;
  const void* g;
  void *m, *v;
  float *m_scale, *v_scale;
  void* copy;
  uint64_t n;
  uint8_t g_type, copy_type, decays, wide;   // copy_type SEE_F32: no copy; wide: every address is a multiple of 16
};
template <uint32_t kEntries>
struct AdamTable {
  uint32_t count;
  uint32_t block_end[kEntries];   // blocks of 256 of entries 0 .. i
  AdamEntry entry[kEntries];
};

// A warp's ring: p, m, v and g of a block, gradients as wide as they come.
template <int kBits>
struct AdamRing {
  static constexpr uint32_t kStateBytes = kAdamBlock * kBits / 8;
  static constexpr uint32_t kM = kAdamBlock * 4, kV = kM + kStateBytes, kG = kV + kStateBytes;   // offsets in a slot
  static constexpr uint32_t kSlotBytes = kG + kAdamBlock * 4;
  // 110 million weights with moments in 8 bits, us: 20 warps 343, 22 341, 23 330, 24 343, 28 351.
  static constexpr uint32_t kWarps = kBits == 8 ? 23 : 24, kSlots = 2;
  static constexpr uint32_t kBytes = kWarps * kSlots * (kSlotBytes + 8);
};

// Where a block of the table's list lies.
template <uint32_t kEntries>
struct AdamCursor {
  uint32_t entry, begin, end;
  __device__ __forceinline__ void Find(const AdamTable<kEntries>& t, uint32_t block) {
    uint32_t lo = 0, hi = t.count - 1;   // the first entry that ends behind the block
    while (lo < hi) {
      const uint32_t mid = (lo + hi) / 2;
      if (t.block_end[mid] > block) hi = mid;
      else lo = mid + 1;
    }
    entry = lo;
    begin = lo ? t.block_end[lo - 1] : 0u;
    end = t.block_end[lo];
  }
  __device__ __forceinline__ void MoveTo(const AdamTable<kEntries>& t, uint32_t block) {   // not before the last one
    if (block < end) return;
    if (block >= t.block_end[entry + 1]) return Find(t, block);
    begin = end;
    end = t.block_end[++entry];
  }
};

__device__ __forceinline__ void Load4(const void* p, int type, uint64_t i, float* v) {   // i % 4 == 0, aligned
  if (type == SEE_F32) {
    const float4 r = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
  } else {
    const uint2 r = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
    if (type == SEE_BF16) {
      Unpack2<Bf16>(r.x, v[0], v[1]);
      Unpack2<Bf16>(r.y, v[2], v[3]);
    } else {
      Unpack2<F16>(r.x, v[0], v[1]);
      Unpack2<F16>(r.y, v[2], v[3]);
    }
  }
}
__device__ __forceinline__ float Load1(const void* p, int type, uint64_t i) {
  if (type == SEE_F32) return static_cast<const float*>(p)[i];
  return type == SEE_BF16 ? ToF32(static_cast<const Bf16*>(p)[i]) : ToF32(static_cast<const F16*>(p)[i]);
}

__device__ __forceinline__ void FromE4m3x2(uint16_t codes, float& lo, float& hi) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(codes));
  Unpack2<F16>(h, lo, hi);
}
// Two values times their block's factor as e4m3, cut as above: the sum's upper 12 bits are the value where e4m3 is normal
// (whose neighbours are a step of those apart), so that the conversion finds nothing left to round.  kLow: some value may lie
// below 2^-6, where the distance of codes stays 2^-9 and the sum is taken 2^-6 further out.
template <bool kLow>
__device__ __forceinline__ uint32_t ToE4m3x2(f32x2 pair, uint32_t word_a, uint32_t word_b) {
  auto cut = [](float x, uint32_t word) {
    const float out = kLow && fabsf(x) < 0.015625f ? copysignf(0.015625f, x) : 0.0f;
    const float y = kLow ? x + out : x;
    const float c = __uint_as_float((__float_as_uint(y) + (word >> 12)) & 0xFFF00000u);
    return kLow ? c - out : c;
  };
  float a, b;
  UnpackF2(pair, &a, &b);
  uint16_t codes;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(codes) : "f"(cut(b, word_b)), "f"(cut(a, word_a)));
  return codes;
}
// The largest and the smallest magnitude of three; a NaN stays in the largest.
__device__ __forceinline__ float MaxMagnitude(float a, f32x2 pair) {
  float x, y, r;
  UnpackF2(pair, &x, &y);
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float MinMagnitude(float a, f32x2 pair) {
  float x, y, r;
  UnpackF2(pair, &x, &y);
  asm("min.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(x), "f"(y));
  return r;
}
// sqrt(v) by one Newton step on the hardware's reciprocal root: s = v y, s + (v - s s) y / 2, the remainder exact in an FMA.
// (A call of sqrtf costs three times as much here.)  Zero stays zero; what is not finite becomes NaN.  kTiny: some value may be
// zero or lie below the smallest normal, whose reciprocal root takes three instructions more; the remainder, a multiple of 2^-149, is then
// off by at most half of that, 2^-23 of the root from 2^-128 on, and nothing below, where the first s is as good.
constexpr float kSmallestNormal = 1.17549435e-38f;
template <bool kTiny>
__device__ __forceinline__ f32x2 Root2(f32x2 v) {
  float a, b;
  UnpackF2(v, &a, &b);
  auto reciprocal = [](float x) {
    float y;
    if constexpr (kTiny) asm("rsqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(fmaxf(x, 1.4e-45f)));
    else asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
  };
  const f32x2 y = PackF2(reciprocal(a), reciprocal(b)), s = Mul2(v, y);
  return Fma2(Fma2(Mul2(s, Splat2(-1.0f)), s, v), Mul2(y, Splat2(0.5f)), s);
}

// The largest magnitude's block scale: 0 where it is below 2^-100, NaN from 2^126 on (a moment that is not finite makes its
// block's NaN: eight bits hold none).
struct BlockScale { float factor, scale; };
__device__ __forceinline__ BlockScale ScaleOf(uint32_t largest_bits) {
  const float largest = __uint_as_float(largest_bits);
  if (largest_bits >= 0x7E800000u) return {0.0f, __uint_as_float(0x7FC00000u)};
  if (largest < 7.888609052210118e-31f) return {0.0f, 0.0f};
  const float r = RcpApprox(largest);   // a Newton step makes 1 / largest of it
  return {__fmaf_rn(__fmaf_rn(-largest, r, 1.0f), r, r) * 448.0f, largest * (1.0f / 448.0f)};
}

// One block: a whole one that lies in `src`, or the elements that there are, where they lie.  `read` is called once nothing
// more is read.
template <int kBits, bool kWhole, typename Read>
__device__ __forceinline__ void StepBlock(const AdamEntry& e, uint64_t block, const uint8_t* src, const AdamStepScalars& a, float gs,
                                          uint32_t lane, [[maybe_unused]] float m_scale, [[maybe_unused]] float v_scale, Read read) {
  using R = AdamRing<kBits>;
  const uint64_t base = block * kAdamBlock;
  // Element j of a lane: four consecutive ones in each half of the block, or single ones 32 apart.
  auto at = [&](int j) -> uint64_t { return kWhole ? base + (j >> 2) * 128 + lane * 4 + (j & 3) : base + j * 32 + lane; };
  float p[8], g[8], m[8], v[8];
  if constexpr (kWhole) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t i = h * 128 + lane * 4;
      Load4(src, SEE_F32, i, p + 4 * h);
      Load4(src + R::kG, e.g_type, i, g + 4 * h);
      if constexpr (kBits == 32) {
        Load4(src + R::kM, SEE_F32, i, m + 4 * h);
        Load4(src + R::kV, SEE_F32, i, v + 4 * h);
      } else {
        const uint32_t mc = *reinterpret_cast<const uint32_t*>(src + R::kM + i), vc = *reinterpret_cast<const uint32_t*>(src + R::kV + i);
        FromE4m3x2(static_cast<uint16_t>(mc), m[4 * h], m[4 * h + 1]);
        FromE4m3x2(static_cast<uint16_t>(mc >> 16), m[4 * h + 2], m[4 * h + 3]);
        FromE4m3x2(static_cast<uint16_t>(vc), v[4 * h], v[4 * h + 1]);
        FromE4m3x2(static_cast<uint16_t>(vc >> 16), v[4 * h + 2], v[4 * h + 3]);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint64_t i = at(j);
      p[j] = g[j] = m[j] = v[j] = 0.0f;
      if (i < e.n) {
        p[j] = e.p[i];
        g[j] = Load1(e.g, e.g_type, i);
        if constexpr (kBits == 32) {
          m[j] = static_cast<const float*>(e.m)[i];
          v[j] = static_cast<const float*>(e.v)[i];
        } else {
          float none;
          FromE4m3x2(static_cast<const uint8_t*>(e.m)[i], m[j], none);
          FromE4m3x2(static_cast<const uint8_t*>(e.v)[i], v[j], none);
        }
      }
    }
  }
  read();
  const float decay = e.decays ? a.weight_decay : 0.0f;
  [[maybe_unused]] uint32_t mc[4], vc[4];   // two codes each
  if (gs != 1.0f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] *= gs;
  }
  if constexpr (kBits == 32) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m[j] = a.beta1 * m[j] + a.om_beta1 * g[j];
      v[j] = a.beta2 * v[j] + a.om_beta2 * g[j] * g[j];
      p[j] -= a.lr * (m[j] * a.inv_bc1 / (sqrtf(v[j] * a.inv_bc2) + a.eps) + decay * p[j]);
    }
  } else {
    float m_top = 0.0f, v_top = 0.0f, v_least = 1.0f;
    f32x2 m2[4], v2[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      // (One by one: a packed product and the packed sum behind it come out as one operation, and these have two roundings.)
      float m1[2], v1[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float grad = g[2 * k + j], root = v[2 * k + j] * v_scale;
        m1[j] = m[2 * k + j] * m_scale * a.beta1 + grad * a.om_beta1;
        v1[j] = root * root * a.beta2 + grad * a.om_beta2 * grad;
      }
      m2[k] = PackF2(m1[0], m1[1]);
      v2[k] = PackF2(v1[0], v1[1]);
      v_least = MinMagnitude(v_least, v2[k]);
    }
    auto roots = [&](auto tiny) {
#pragma unroll
      for (int k = 0; k < 4; ++k) v2[k] = Root2<tiny.value>(v2[k]);
    };
    if (v_least >= kSmallestNormal) roots(std::false_type{});
    else roots(std::true_type{});
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const f32x2 weight = PackF2(p[2 * k], p[2 * k + 1]);
      float size0, size1;
      UnpackF2(Fma2(v2[k], Splat2(a.root_inv_bc2), Splat2(a.eps)), &size0, &size1);
      const f32x2 move = Mul2(Mul2(m2[k], Splat2(a.inv_bc1)), PackF2(RcpApprox(size0), RcpApprox(size1)));
      UnpackF2(Fma2(Fma2(weight, Splat2(decay), move), Splat2(-a.lr), weight), &p[2 * k], &p[2 * k + 1]);
      m_top = MaxMagnitude(m_top, m2[k]);
      v_top = MaxMagnitude(v_top, v2[k]);
    }
    const uint32_t m_bits = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(m_top)), v_bits = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(v_top));
    const BlockScale mine = ScaleOf(lane & 1 ? v_bits : m_bits);   // (one division for both)
    const float m_factor = __shfl_sync(0xFFFFFFFFu, mine.factor, 0), v_factor = __shfl_sync(0xFFFFFFFFu, mine.factor, 1);
    if (lane < 2) (lane ? e.v_scale : e.m_scale)[block] = mine.scale;
    float lowest = 1.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      m2[k] = Mul2(m2[k], Splat2(m_factor));
      v2[k] = Mul2(v2[k], Splat2(v_factor));
      lowest = MinMagnitude(MinMagnitude(lowest, m2[k]), v2[k]);
    }
    const uint32_t word = static_cast<uint32_t>(at(0)) * kGolden + a.phase;
    auto codes = [&](auto low) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        // (how far element j lies behind the lane's first)
        const uint32_t w0 = word + (kWhole ? (k >> 1) * 128 + (k & 1) * 2 : 64 * k) * kGolden, w1 = w0 + (kWhole ? 1 : 32) * kGolden;
        mc[k] = ToE4m3x2<low.value>(m2[k], w0, w1);
        vc[k] = ToE4m3x2<low.value>(v2[k], w0 + kHalfTurn, w1 + kHalfTurn);
      }
    };
    if (lowest >= 0.015625f) {
      codes(std::false_type{});
    } else {   // a few blocks in a hundred
      codes(std::true_type{});
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float x, y;
        UnpackF2(v2[k], &x, &y);
        if (x > 0.0f && (vc[k] & 0xFFu) == 0) vc[k] |= 1u;
        if (y > 0.0f && (vc[k] & 0xFF00u) == 0) vc[k] |= 0x100u;
      }
    }
    if (m_factor == 0.0f) mc[0] = mc[1] = mc[2] = mc[3] = 0;   // (what is not finite times 0)
    if (v_factor == 0.0f) vc[0] = vc[1] = vc[2] = vc[3] = 0;
  }
  if constexpr (kWhole) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint64_t i = at(4 * h);
      const float* q = p + 4 * h;
      *reinterpret_cast<float4*>(e.p + i) = make_float4(q[0], q[1], q[2], q[3]);
      if constexpr (kBits == 32) {
        *reinterpret_cast<float4*>(static_cast<float*>(e.m) + i) = make_float4(m[4 * h], m[4 * h + 1], m[4 * h + 2], m[4 * h + 3]);
        *reinterpret_cast<float4*>(static_cast<float*>(e.v) + i) = make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
      } else {
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(e.m) + i) = mc[2 * h] | mc[2 * h + 1] << 16;
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(e.v) + i) = vc[2 * h] | vc[2 * h + 1] << 16;
      }
      if (e.copy_type != SEE_F32) {
        uint2* to = reinterpret_cast<uint2*>(static_cast<uint16_t*>(e.copy) + i);
        if (e.copy_type == SEE_BF16) *to = make_uint2(Pack2<Bf16>(q[0], q[1]), Pack2<Bf16>(q[2], q[3]));
        else *to = make_uint2(Pack2<F16>(q[0], q[1]), Pack2<F16>(q[2], q[3]));
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint64_t i = at(j);
      if (i >= e.n) continue;
      e.p[i] = p[j];
      if constexpr (kBits == 32) {
        static_cast<float*>(e.m)[i] = m[j];
        static_cast<float*>(e.v)[i] = v[j];
      } else {
        static_cast<uint8_t*>(e.m)[i] = static_cast<uint8_t>(mc[j / 2] >> 8 * (j & 1));
        static_cast<uint8_t*>(e.v)[i] = static_cast<uint8_t>(vc[j / 2] >> 8 * (j & 1));
      }
      if (e.copy_type == SEE_BF16) static_cast<Bf16*>(e.copy)[i] = FromF32<Bf16>(p[j]);
      else if (e.copy_type == SEE_F16) static_cast<F16*>(e.copy)[i] = FromF32<F16>(p[j]);
    }
  }
}

template <int kBits, uint32_t kEntries>
__global__ void __launch_bounds__(32 * AdamRing<kBits>::kWarps, 1)
AdamWTensorsKernel(const __grid_constant__ AdamTable<kEntries> table, const AdamStepScalars a, const float* __restrict__ grad_scale,
                   DeviceStatus* status) {
  using R = AdamRing<kBits>;
  extern __shared__ __align__(128) uint8_t dyn[];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint8_t* ring = dyn + warp * R::kSlots * R::kSlotBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(dyn + R::kWarps * R::kSlots * R::kSlotBytes) + warp * R::kSlots;
  if (lane == 0) {
    for (uint32_t i = 0; i < R::kSlots; ++i) umma_dev::MbarInit(&bars[i], 1);
    umma_dev::MbarInitFence();
  }
  __syncwarp();
  AwaitPrevious();
  // A thread block's warps sweep its range of the list side by side (304 us; a range to each warp, or one sweep of all, 330 to 350 on that board); a
  // list that one sweep of all covers is spread over the SMs instead.
  const uint32_t blocks = table.block_end[table.count - 1], all = gridDim.x * R::kWarps;
  const uint32_t each = blocks / gridDim.x, rest = blocks % gridDim.x, begin = blockIdx.x * each + min(blockIdx.x, rest);
  const uint32_t end = blocks > all ? begin + each + (blockIdx.x < rest) : blocks, warps = blocks > all ? R::kWarps : all;
  const uint32_t first = blocks > all ? begin + warp : warp * gridDim.x + blockIdx.x;
  if (first >= end) return;
  AdamCursor<kEntries> now, ahead;
  now.Find(table, first);
  ahead = now;
  // Lanes 0 to 3 fill a slot with p, m, v and g, lanes 4 and 5 ask for the block's two scales: each keeps where its operand of the
  // current tensor lies, so that a fill is a handful of instructions of the warp.  A block that the copies cannot take is read
  // where it lies.
  const uint8_t* source = nullptr;
  uint32_t bytes = 0, total = 0, offset = 0, fillable = 0;   // of a block of mine, of the first four; in the slot; whole blocks
  auto look_up = [&] {
    const AdamEntry& e = table.entry[ahead.entry];
    const uint32_t g_bytes = kAdamBlock * (e.g_type == SEE_F32 ? 4 : 2);
    const void* const operands[6] = {e.p, e.m, e.v, e.g, e.m_scale, e.v_scale};
    const uint32_t sizes[6] = {kAdamBlock * 4, R::kStateBytes, R::kStateBytes, g_bytes, 4, 4}, offsets[6] = {0, R::kM, R::kV, R::kG, 0, 0};
#pragma unroll
    for (uint32_t i = 0; i < 6; ++i)
      if (lane == i) {
        source = static_cast<const uint8_t*>(operands[i]);
        bytes = sizes[i];
        offset = offsets[i];
      }
    total = R::kG + g_bytes;
    fillable = e.wide ? static_cast<uint32_t>(e.n / kAdamBlock) : 0;
  };
  look_up();
  static_assert(R::kSlots == 2);
  [[maybe_unused]] float scale0 = 0.0f, scale1 = 0.0f;   // of the block in either slot: m's in lane 4, v's in lane 5
  auto fill = [&](uint32_t f, uint32_t slot) {
    if (f >= ahead.end) {
      ahead.MoveTo(table, f);
      look_up();
    }
    const uint32_t block = f - ahead.begin;
    if (kBits == 8 && (lane == 4 || lane == 5)) (slot ? scale1 : scale0) = *reinterpret_cast<const float*>(source + static_cast<uint64_t>(block) * 4);
    if (block >= fillable) return;
    if (lane == 0) umma_dev::MbarExpectTx(&bars[slot], total);
    if (lane < 4) umma_dev::BulkLoad(ring + slot * R::kSlotBytes + offset, source + static_cast<uint64_t>(block) * bytes, bytes, &bars[slot]);
  };
  const uint32_t count = (end - first + warps - 1) / warps;   // mine
  for (uint32_t i = 0; i < R::kSlots && i < count; ++i) fill(first + i * warps, i);
  const float gs = grad_scale ? *grad_scale : 1.0f;
  uint32_t slot = 0, parities = 0;   // a bit for each slot
  for (uint32_t i = 0; i < count; ++i) {
    const uint32_t f = first + i * warps;
    now.MoveTo(table, f);
    const AdamEntry& e = table.entry[now.entry];
    const uint64_t block = f - now.begin, base = block * kAdamBlock;
    const bool whole = e.wide && base + kAdamBlock <= e.n;
    if (whole) {
      if (!umma_dev::MbarWait(&bars[slot], parities >> slot & 1u)) {   // (the copies always land; but no wait is without end)
        status->wait_timeout = 1;
        umma_dev::DrainDelay();
      }
      parities ^= 1u << slot;
    }
    auto read = [&] {   // the slot may be filled again
      __syncwarp();
      if (i + R::kSlots < count) fill(f + R::kSlots * warps, slot);
    };
    const float scale = slot ? scale1 : scale0, m_scale = __shfl_sync(0xFFFFFFFFu, scale, 4), v_scale = __shfl_sync(0xFFFFFFFFu, scale, 5);
    if (whole) StepBlock<kBits, true>(e, block, ring + slot * R::kSlotBytes, a, gs, lane, m_scale, v_scale, read);
    else StepBlock<kBits, false>(e, block, nullptr, a, gs, lane, m_scale, v_scale, read);
    slot = slot + 1 < R::kSlots ? slot + 1 : 0;
  }
}

template <int kBits, uint32_t kEntries>
cudaError_t Launch(const see_adamw_tensor* tensors, uint64_t count, const AdamStepScalars& a, const float* grad_scale, uint32_t sms,
                   DeviceStatus* status, cudaStream_t s, int* launches) {
  using R = AdamRing<kBits>;
  auto* kernel = AdamWTensorsKernel<kBits, kEntries>;
  // The shared-memory limit is a device's: one flag for each.
  static std::atomic<bool> configured[64] = {};
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, R::kBytes); e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
  }
  AdamTable<kEntries> table;
  uint64_t next = 0;
  while (next < count) {
    table.count = 0;
    uint64_t blocks = 0;
    for (; next < count && table.count < kEntries; ++next) {
      const see_adamw_tensor& t = tensors[next];
      if (t.n == 0) continue;
      const uint64_t more = (t.n + kAdamBlock - 1) / kAdamBlock;
      if (blocks + more > 0x7FFFFFFFull) break;   // (one tensor alone has at most half as many)
      auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
      AdamEntry& e = table.entry[table.count];
      e = {t.p, t.g, t.m, t.v, t.m_scale, t.v_scale, t.copy, t.n, static_cast<uint8_t>(t.g_type), static_cast<uint8_t>(t.copy_type),
           static_cast<uint8_t>((t.flags & SEE_ADAMW_NO_DECAY) == 0), 0};
      e.wide = aligned(t.p) && aligned(t.g) && aligned(t.m) && aligned(t.v) && aligned(t.copy);
      blocks += more;
      table.block_end[table.count++] = static_cast<uint32_t>(blocks);
    }
    if (!table.count) break;
    if (cudaError_t e = Next(kernel, static_cast<unsigned>(blocks < sms ? blocks : sms), 32 * R::kWarps, R::kBytes, s)(table, a, grad_scale, status);
        e != cudaSuccess)
      return e;
    ++*launches;
  }
  return cudaSuccess;
}

}  // namespace

cudaError_t AdamWTensors(const see_adamw_tensor* tensors, uint64_t count, int state_bits, const AdamStepScalars& a,
                         const float* grad_scale, uint32_t sms, DeviceStatus* status, cudaStream_t s, int* launches) {
  return state_bits == 8 ? Launch<8, 192>(tensors, count, a, grad_scale, sms, status, s, launches)
                         : Launch<32, 192>(tensors, count, a, grad_scale, sms, status, s, launches);
}

}  // namespace see::k
