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
// Bound by HBM: 14 bytes an element with 16-bit gradients and moments in 8 bits, 28 in f32.  A warp takes a block of 256
// elements, eight a lane; a thread block takes eight of them, and finds its tensor by bisection over the table, which the
// launch carries as a parameter: nothing is uploaded, and a captured launch owns its copy.
#include "block_ops.h"
#include "launch.cuh"
#include "vec_types.cuh"

namespace see::k {

namespace {

constexpr uint32_t kAdamWarps = 8;
constexpr uint32_t kGolden = 0x9E3779B9u;       // 2^32 times the golden section
constexpr uint32_t kHalfTurn = 0x80000000u;     // between the words of m and of sqrt(v)

struct AdamEntry {
  float* p;
  const void* g;
  void *m, *v;
  float *m_scale, *v_scale;
  void* copy;
  uint64_t n;
  uint8_t g_type, copy_type, decays, wide;   // copy_type SEE_F32: no copy; wide: every address is aligned to its four elements
};
template <uint32_t kEntries>
struct AdamTable {
  uint32_t count;
  uint32_t chunk_end[kEntries];   // chunks (eight blocks of 256) of entries 0 .. i
  AdamEntry entry[kEntries];
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
// |x| times `factor` as e4m3 without its sign (see above); `word` is the element's.
__device__ __forceinline__ uint32_t ToE4m3(float magnitude, float factor, uint32_t word) {
  const float a = magnitude * factor;
  const bool low = a < 0.015625f;   // below the smallest normal: the distance of codes stays 2^-9
  const uint32_t bits = __float_as_uint(low ? a + 0.015625f : a) + (word >> 12);
  const uint32_t code = (bits >> 20) - (low ? 968u : 960u);
  return code < 126u ? code : 126u;
}

// The largest magnitude's block scale: 0 where it is below 2^-100, NaN where it is not finite (one such element makes the
// block's moments NaN: eight bits hold none).
struct BlockScale { float factor, scale; };
__device__ __forceinline__ BlockScale ScaleOf(uint32_t largest_bits) {
  const float largest = __uint_as_float(largest_bits);
  if (largest_bits >= 0x7F800000u) return {0.0f, __uint_as_float(0x7FC00000u)};
  if (largest < 7.888609052210118e-31f) return {0.0f, 0.0f};
  return {1.0f / largest * 448.0f, largest * (1.0f / 448.0f)};
}

template <int kBits, uint32_t kEntries>
__global__ void __launch_bounds__(32 * kAdamWarps)
AdamWTensorsKernel(const __grid_constant__ AdamTable<kEntries> table, const AdamStepScalars a, const float* __restrict__ grad_scale) {
  AwaitPrevious();
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float gs = grad_scale ? *grad_scale : 1.0f;
  const uint32_t chunks = table.chunk_end[table.count - 1];
  for (uint32_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    uint32_t lo = 0, hi = table.count - 1;   // the first entry that ends behind the chunk
    while (lo < hi) {
      const uint32_t mid = (lo + hi) / 2;
      if (table.chunk_end[mid] > chunk) hi = mid;
      else lo = mid + 1;
    }
    const AdamEntry& e = table.entry[lo];
    const uint64_t block = static_cast<uint64_t>(chunk - (lo ? table.chunk_end[lo - 1] : 0u)) * kAdamWarps + warp;
    const uint64_t base = block * kAdamBlock;
    if (base >= e.n) continue;
    const bool whole = e.wide && base + kAdamBlock <= e.n;
    // Element j of a lane: four consecutive ones in each half of the block, or single ones 32 apart.
    auto at = [&](int j) -> uint64_t { return whole ? base + (j >> 2) * 128 + lane * 4 + (j & 3) : base + j * 32 + lane; };
    float p[8], g[8], m[8], v[8];
    if (whole) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint64_t i = at(4 * h);
        Load4(e.p, SEE_F32, i, p + 4 * h);
        Load4(e.g, e.g_type, i, g + 4 * h);
        if constexpr (kBits == 32) {
          Load4(e.m, SEE_F32, i, m + 4 * h);
          Load4(e.v, SEE_F32, i, v + 4 * h);
        } else {
          const uint32_t mc = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(e.m) + i);
          const uint32_t vc = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(e.v) + i);
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
    [[maybe_unused]] const float m_scale = kBits == 8 ? e.m_scale[block] : 0.0f, v_scale = kBits == 8 ? e.v_scale[block] : 0.0f;
    const float decay = e.decays ? a.weight_decay : 0.0f;
    [[maybe_unused]] uint32_t m_top = 0, v_top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (grad_scale) g[j] *= gs;
      float size;
      if constexpr (kBits == 8) {
        const float root = v[j] * v_scale;
        m[j] = m[j] * m_scale * a.beta1 + g[j] * a.om_beta1;
        v[j] = sqrtf(root * root * a.beta2 + g[j] * a.om_beta2 * g[j]);   // from here on the root
        size = v[j] * a.root_inv_bc2;
        m_top = max(m_top, __float_as_uint(m[j]) & 0x7FFFFFFFu);
        v_top = max(v_top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
      } else {
        m[j] = a.beta1 * m[j] + a.om_beta1 * g[j];
        v[j] = a.beta2 * v[j] + a.om_beta2 * g[j] * g[j];
        size = sqrtf(v[j] * a.inv_bc2);
      }
      p[j] -= a.lr * (m[j] * a.inv_bc1 / (size + a.eps) + decay * p[j]);
    }
    uint32_t mc[8], vc[8];
    if constexpr (kBits == 8) {
      m_top = __reduce_max_sync(0xFFFFFFFFu, m_top);
      v_top = __reduce_max_sync(0xFFFFFFFFu, v_top);
      const BlockScale ms = ScaleOf(m_top), vs = ScaleOf(v_top);
      if (lane == 0) {
        e.m_scale[block] = ms.scale;
        e.v_scale[block] = vs.scale;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t word = static_cast<uint32_t>(at(j)) * kGolden + a.phase;
        const uint32_t sign = (__float_as_uint(m[j]) >> 31) << 7;
        mc[j] = ms.factor != 0.0f ? ToE4m3(fabsf(m[j]), ms.factor, word) | (m[j] < 0.0f ? sign : 0u) : 0u;
        vc[j] = vs.factor != 0.0f ? ToE4m3(v[j], vs.factor, word + kHalfTurn) : 0u;
        if (vc[j] == 0 && v[j] * vs.factor > 0.0f) vc[j] = 1;
      }
    }
    if (whole) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint64_t i = at(4 * h);
        const float* q = p + 4 * h;
        *reinterpret_cast<float4*>(e.p + i) = make_float4(q[0], q[1], q[2], q[3]);
        if constexpr (kBits == 32) {
          *reinterpret_cast<float4*>(static_cast<float*>(e.m) + i) = make_float4(m[4 * h], m[4 * h + 1], m[4 * h + 2], m[4 * h + 3]);
          *reinterpret_cast<float4*>(static_cast<float*>(e.v) + i) = make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
        } else {
          const uint32_t* c = mc + 4 * h;
          *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(e.m) + i) = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
          c = vc + 4 * h;
          *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(e.v) + i) = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
        }
        if (e.copy_type != SEE_F32) {
          const bool bf = e.copy_type == SEE_BF16;
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(e.copy) + i) =
              make_uint2(bf ? Pack2<Bf16>(q[0], q[1]) : Pack2<F16>(q[0], q[1]), bf ? Pack2<Bf16>(q[2], q[3]) : Pack2<F16>(q[2], q[3]));
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
          static_cast<uint8_t*>(e.m)[i] = static_cast<uint8_t>(mc[j]);
          static_cast<uint8_t*>(e.v)[i] = static_cast<uint8_t>(vc[j]);
        }
        if (e.copy_type == SEE_BF16) static_cast<Bf16*>(e.copy)[i] = FromF32<Bf16>(p[j]);
        else if (e.copy_type == SEE_F16) static_cast<F16*>(e.copy)[i] = FromF32<F16>(p[j]);
      }
    }
  }
}

template <int kBits, uint32_t kEntries>
cudaError_t Launch(const see_adamw_tensor* tensors, uint64_t count, const AdamStepScalars& a, const float* grad_scale, uint32_t sms,
                   cudaStream_t s, int* launches) {
  constexpr uint64_t kChunk = static_cast<uint64_t>(kAdamBlock) * kAdamWarps;
  AdamTable<kEntries> table;
  uint64_t next = 0;
  while (next < count) {
    table.count = 0;
    uint64_t chunks = 0;
    for (; next < count && table.count < kEntries; ++next) {
      const see_adamw_tensor& t = tensors[next];
      if (t.n == 0) continue;
      const uint64_t more = (t.n + kChunk - 1) / kChunk;
      if (table.count && chunks + more > 0xFFFFFFFFull) break;
      auto aligned = [](const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; };
      AdamEntry& e = table.entry[table.count];
      e = {t.p, t.g, t.m, t.v, t.m_scale, t.v_scale, t.copy, t.n, static_cast<uint8_t>(t.g_type), static_cast<uint8_t>(t.copy_type),
           static_cast<uint8_t>((t.flags & SEE_ADAMW_NO_DECAY) == 0), 0};
      e.wide = aligned(t.p, 16) && aligned(t.g, t.g_type == SEE_F32 ? 16 : 8) && aligned(t.m, kBits == 32 ? 16 : 4) &&
               aligned(t.v, kBits == 32 ? 16 : 4) && (t.copy_type == SEE_F32 || aligned(t.copy, 8));
      chunks += more;
      table.chunk_end[table.count++] = static_cast<uint32_t>(chunks);
    }
    if (!table.count) break;
    const uint64_t most = static_cast<uint64_t>(sms) * 8;
    if (cudaError_t e = Next(AdamWTensorsKernel<kBits, kEntries>, static_cast<unsigned>(chunks < most ? chunks : most), 32 * kAdamWarps, 0,
                             s)(table, a, grad_scale);
        e != cudaSuccess)
      return e;
    ++*launches;
  }
  return cudaSuccess;
}

}  // namespace

cudaError_t AdamWTensors(const see_adamw_tensor* tensors, uint64_t count, int state_bits, const AdamStepScalars& a,
                         const float* grad_scale, uint32_t sms, cudaStream_t s, int* launches) {
  return state_bits == 8 ? Launch<8, 48>(tensors, count, a, grad_scale, sms, s, launches)
                         : Launch<32, 48>(tensors, count, a, grad_scale, sms, s, launches);
}

}  // namespace see::k
