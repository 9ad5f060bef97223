// Losses over rows of logits: the labels' log-probabilities, a clipped policy loss or a preference loss of them, and the
// gradient of the logits.  With z = logit_scale logits, M its maximum and l the label, a row is
//   e_c = 2^(k logit_c - k M),  k = logit_scale / ln 2,   others = sum of e_c over c != l,   s = others + e_l,
//   logp = (z_l - M) - log s, or -log1p(others / e_l) where the label holds three quarters (no digits are lost next to 0),
//   dlogit_c = -slope logit_scale e_c / s,  of the label  slope logit_scale others / s   (not 1 - p, which would lose them),
// slope being the loss's derivative by logp.  The product k M is rounded once and the same in every exponent of a row, so that its
// rounding cancels between e_c and s.  Bound by HBM: logits are read once, dlogits written once.
//
// Far from 0 the rounding of k M becomes more than 2^x can make good.  A row whose maximum is far either way, |k M| from 2^26 on (all
// classes masked, say), is left to the kernel that comes next, whose warps make its sums from memory with exponents k (z - M) (FarRow).
// Parts of another row that lie below -2^30 count as nothing beside it.
//
// A row is walked in units of 16 bytes by address, of which the first and the last may stick out of it, whatever its alignment.  Rows
// reach registers through a ring in shared memory (LogitRowsKernel); wide rows, and few ones, are shared by the blocks of a cluster.
// A policy loss's rows that are wider still are walked twice (LogitStreamKernel), a preference loss's that are many and wide go through
// rings of single warps (LogitSumsKernel).
//
// logp is made in double.  A preference loss holds sums of hundreds of them against a reference's, where what is off the same way in each
// row adds up, so it does more: k M is rounded up to an integer, so that sums are carried over to a larger maximum without rounding; its
// exponents have what k's rounding leaves too (k rounded downwards, the rest above 0: -inf stays); and log s has kLow on top, by which
// ex2.approx falls short on average (measured over 2^24 arguments from each of several ranges from -60 on).  Margins of 8 pairs of 512
// rows are 2e-7 off so, 1e-6 without.  The policy loss, whose rows are rounded to f32 each, does without.
#include <type_traits>

#include "act_expr.cuh"
#include "block_ops.h"
#include "launch.cuh"
#include "row_groups.cuh"
#include "umma_device.cuh"
#include "vec_types.cuh"

namespace see::k {

namespace {

constexpr uint32_t kThreads = 512;
__device__ __forceinline__ float MinusInf() { return __int_as_float(0xFF800000); }

template <typename T> constexpr int kPerUnit = 16 / sizeof(T);
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

// -inf, and 16 bytes of it.
template <typename T>
__device__ __forceinline__ constexpr uint32_t NoElement() {
  return sizeof(T) == 4 ? 0xFF800000u : std::is_same_v<T, Bf16> ? 0xFF80u : 0xFC00u;
}
template <typename T>
__device__ __forceinline__ uint4 Nothing() {
  const uint32_t w = sizeof(T) == 4 ? NoElement<T>() : NoElement<T>() * 0x10001u;
  return make_uint4(w, w, w, w);
}

// The elements from `from` on and before `to` (and not `but`), -inf in place of the others.
template <typename T>
__device__ __forceinline__ uint4 Only(const uint4& r, int32_t from, int32_t to, int32_t but) {
  uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      w[i] = i >= from && i < to && i != but ? w[i] : NoElement<T>();
    } else {
      const uint32_t lo = 2 * i >= from && 2 * i < to && 2 * i != but ? w[i] & 0xFFFFu : NoElement<T>();
      const uint32_t hi = 2 * i + 1 >= from && 2 * i + 1 < to && 2 * i + 1 != but ? w[i] >> 16 : NoElement<T>();
      w[i] = lo | hi << 16;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// A row of logits and of dlogits.
template <typename T>
struct Row {
  const T* z;
  T* d;
  uint32_t skip, classes, units;   // elements of the first unit in front of the row; ... ; units
  bool alike;                      // d lies in its units as z does
  __device__ __forceinline__ Row(const LogitArgs& a, uint64_t row) {
    z = static_cast<const T*>(a.logits) + row * a.stride;
    d = static_cast<T*>(a.dlogits) + row * a.stride;
    classes = a.classes;
    skip = static_cast<uint32_t>(reinterpret_cast<uint64_t>(z) & 15) / sizeof(T);
    units = (skip + classes + kPerUnit<T> - 1) / kPerUnit<T>;
    alike = ((reinterpret_cast<uint64_t>(z) ^ reinterpret_cast<uint64_t>(d)) & 15) == 0;
  }
  __device__ __forceinline__ int32_t At(uint32_t unit) const { return static_cast<int32_t>(unit * kPerUnit<T>) - static_cast<int32_t>(skip); }
  __device__ __forceinline__ bool Whole(int32_t at) const { return at >= 0 && at + kPerUnit<T> <= static_cast<int32_t>(classes); }
  // A unit's 16 bytes, -inf where it sticks out.
  __device__ __forceinline__ uint4 Raw(uint32_t unit) const {
    const int32_t at = At(unit);
    if (Whole(at)) return *reinterpret_cast<const uint4*>(z + at);
    using Bits = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;
    const Bits* bits = reinterpret_cast<const Bits*>(z);
    uint32_t r[4] = {};
#pragma unroll
    for (int j = 0; j < kPerUnit<T>; ++j)
      r[j * sizeof(T) / 4] |= (at + j >= 0 && at + j < static_cast<int32_t>(classes) ? static_cast<uint32_t>(bits[at + j]) : NoElement<T>()) << (j * sizeof(T) % 4 * 8);
    return make_uint4(r[0], r[1], r[2], r[3]);
  }
  // The same of what nobody reads again, so that it does not stay in L2.
  __device__ __forceinline__ uint4 RawOnce(uint32_t unit) const {
    const int32_t at = At(unit);
    return Whole(at) ? __ldcs(reinterpret_cast<const uint4*>(z + at)) : Raw(unit);
  }
  __device__ __forceinline__ void Load(uint32_t unit, float* v) const { Elements<T>(Raw(unit), v); }
  __device__ __forceinline__ void Store(uint32_t unit, const float* v) const {
    const int32_t at = At(unit);
    if (alike && Whole(at)) {
      if constexpr (sizeof(T) == 4) __stcs(reinterpret_cast<float4*>(d + at), make_float4(v[0], v[1], v[2], v[3]));
      else __stcs(reinterpret_cast<uint4*>(d + at), make_uint4(Pack2<T>(v[0], v[1]), Pack2<T>(v[2], v[3]), Pack2<T>(v[4], v[5]), Pack2<T>(v[6], v[7])));
      return;
    }
#pragma unroll
    for (int j = 0; j < kPerUnit<T>; ++j)
      if (at + j >= 0 && at + j < static_cast<int32_t>(classes)) d[at + j] = FromF32<T>(v[j]);
  }
};

// log((1 + t) / (1 - t)) for |t| up to 0.18, from the series of atanh; what is left out is below 3e-12 of it.
__device__ __forceinline__ double LogRatio(double t) {
  const double q = t * t;
  double sum = 1.0 / 13.0;
  sum = fma(sum, q, 1.0 / 11.0);
  sum = fma(sum, q, 1.0 / 9.0);
  sum = fma(sum, q, 1.0 / 7.0);
  sum = fma(sum, q, 1.0 / 5.0);
  sum = fma(sum, q, 1.0 / 3.0);
  return fma(t * q, 2.0 * sum, 2.0 * t);
}
// n / d, in two steps of Newton's iteration from an approximation in f32.
__device__ __forceinline__ double Quotient(double n, double d) {
  double r = static_cast<double>(RcpApprox(static_cast<float>(d)));
  r = fma(r, fma(-d, r, 1.0), r);
  r = fma(r, fma(-d, r, 1.0), r);
  return __dmul_rn(n, r);
}
// log s of a sum of f32 terms: s = 2^e m with m next to 1, and (m - 1) / (m + 1) into the series.
__device__ __forceinline__ double LogOf(float s) {
  if (!(s > 1e-30f && s < __int_as_float(0x7F800000))) return static_cast<double>(logf(s));
  const int32_t bits = __float_as_int(s) - 0x3F3504F3;   // (of 2^-1/2)
  const int32_t e = bits >> 23;
  const double m = static_cast<double>(__int_as_float((bits & 0x007FFFFF) + 0x3F3504F3));
  return fma(static_cast<double>(e), 0.6931471805599453, LogRatio(Quotient(m - 1.0, m + 1.0)));
}

constexpr double kLow = 5.1e-8;
constexpr float kFar = 0x1p26f, kNothing = -0x1p30f;
__device__ __forceinline__ bool IsFar(float mk) { return fabsf(mk) >= kFar; }
// k M as it is used; -inf: nothing here, or nothing that shows beside a row that is not far.  (Above -2^30 a part's terms are 2^96 at
// most, and its factor beside a row that is not far is 0.)
template <bool kPolicy>
__device__ __forceinline__ float TopOf(const LogitArgs& a, float z) {
  const float km = __fmul_rn(z, a.k), top = kPolicy ? km : ceilf(km);
  return top > kNothing ? top : MinusInf();
}

// Of a row: the label's logit, k M (of a far row: what FarOf makes of M), the sum over the others, the sum over all.
struct RowSums {
  float z_label, mk, others, s;
};
// A far row's M is kept times a power of two, which is exact, and above k, so that what was far is 2^26 at least.  (What that takes beyond
// f32, where a mask's lowest value may lie, is as good as f32's largest number.)
__device__ __forceinline__ float FarOf(const LogitArgs& a, float z) {
  const float m = z * a.k_up;
  return isinf(m) && !isinf(z) ? copysignf(0x1.fffffep127f, m) : m;
}
// z - M of such a row, and 2^(k (z - M)).
__device__ __forceinline__ float FarOff(const LogitArgs& a, float z, float mk) { return (FarOf(a, z) - mk) / a.k_up; }
__device__ __forceinline__ float FarPower(const LogitArgs& a, float z, float mk) { return Ex2Approx(FarOff(a, z, mk) * a.k); }
__device__ __forceinline__ float LabelTerm(const LogitArgs& a, float z_label, float mk) {
  return Ex2Approx(fmaf(z_label, a.k_rest, fmaf(z_label, a.k, -mk)));
}
// (Every product and sum is written as the instruction it is, so that the compiler contracts it alike wherever it stands: what a kernel
// decides by a logp agrees with what another one reports.)
template <bool kPolicy>
__device__ __forceinline__ double LogpOf(const LogitArgs& a, const RowSums& q) {
  const bool far = IsFar(q.mk);
  const float e = far ? FarPower(a, q.z_label, q.mk) : LabelTerm(a, q.z_label, q.mk);
  if (3.0f * q.others < e) {   // -log1p(others / e)
    const double ratio = Quotient(static_cast<double>(q.others), static_cast<double>(e));
    return -LogRatio(Quotient(ratio, 2.0 + ratio));
  }
  if (far)
    return fma(static_cast<double>(a.scale), (static_cast<double>(FarOf(a, q.z_label)) - static_cast<double>(q.mk)) / static_cast<double>(a.k_up), -LogOf(q.s));
  const double above = fma(static_cast<double>(a.scale), fma(-static_cast<double>(q.mk), a.inv_k, static_cast<double>(q.z_label)), -LogOf(q.s));
  return kPolicy ? above : above - kLow;
}

__device__ __forceinline__ bool Counts(int32_t label, uint32_t classes) { return label >= 0 && static_cast<uint32_t>(label) < classes; }

// ---- the policy loss ------------------------------------------------------------------------------------
// What a row brings besides its logits.
struct PolicyRow {
  float old, ref, advantage, weight;
};
__device__ __forceinline__ PolicyRow PolicyRowOf(const PolicyArgs& p, uint64_t row) {
  return {p.old_logp[row], p.ref_logp ? p.ref_logp[row] : 0.0f, p.advantages[row], p.weights ? p.weights[row] : 1.0f};
}
// x y, and 0 where y is 0 beside an x that has grown beyond its type: a ratio of probabilities.  (NaN stays.)
template <typename F>
__device__ __forceinline__ F Times(F x, F y) {
  return y == 0 && x == x ? F(0) : x * y;
}
struct PolicyTerms {
  float slope, loss;   // slope: of the loss by logp, with its KL term; loss: without; none of them weighted
  bool clipped;
};
__device__ __forceinline__ PolicyTerms PolicyOf(const PolicyArgs& p, const PolicyRow& row, double logp) {
  const float off = static_cast<float>(logp - static_cast<double>(row.old)), above = static_cast<float>(static_cast<double>(row.ref) - logp);
  const float a = row.advantage, r = expf(off), cut = r < 1.0f - p.clip_low ? 1.0f - p.clip_low : r > 1.0f + p.clip_high ? 1.0f + p.clip_high : r;
  const float by = Times(r, a);
  PolicyTerms t;
  t.clipped = by > cut * a;
  t.loss = t.clipped ? -(cut * a) : -by;
  t.slope = t.clipped ? 0.0f : -by;
  if (p.ref_logp) t.slope -= Times(expm1f(above), p.kl_coef);
  return t;
}
// exp(x) - x - 1, some x^2 / 2: in double, and next to 0 by its series, since the difference would leave none of an f32's digits.
__device__ __forceinline__ double KlOf(double x) {
  return fabs(x) < 0x1p-10 ? x * x * fma(x, fma(x, 1.0 / 24.0, 1.0 / 6.0), 0.5) : expm1(x) - x;
}
// The loss's weighted derivative by a row's logp, as it goes into dlogits.  Of 16-bit logits, 8 or 11 bits: mostly a logp in f32 is enough,
// and takes each warp a third of the instructions.  It is not next to a corner, where the row is on the side that
// PolicyFinishKernel counts it on, nor where the slope is what is left of two terms, or little because the policy is next to its
// reference.  `off` bounds how far logp, less what it is compared with, and the exponential of that, relative, are from those of the double
// one, in 2^-22: lg2.approx 0.7 of 1 or of its result, ex2.approx 1 for the label's term and 1 for the exponential, whose double has 1/2;
// roundings of 2^-24 or 2^-25, 3.5 of logp, 2.5 of the difference, 0.7 of the logarithm.
// (Rows of 250 in bf16, 16384 18.7 us, 65536 52.0, as with the f32 logp alone; each in double: f32 logits, 52.6.)
template <typename T>
__device__ __forceinline__ float SlopeOf(const LogitArgs& a, const PolicyArgs& p, const PolicyRow& row, const RowSums& q) {
  if constexpr (sizeof(T) == 2) {
    constexpr float kLn2 = 0.6931471805599453f, kLog2E = 1.4426950408889634f;
    float log2s;
    asm("lg2.approx.f32 %0, %1;" : "=f"(log2s) : "f"(q.s));
    const float logp = kLn2 * (fmaf(q.z_label, a.k, -q.mk) - log2s);
    const float d = logp - row.old, x = p.ref_logp ? row.ref - logp : 0.0f;
    const float off = 0x1p-22f * (4.0f + fabsf(log2s) + fabsf(logp) + fabsf(d) + fabsf(x));
    const float r = Ex2Approx(d * kLog2E);   // beyond: the corner that the advantage's sign chooses
    const float beyond = row.advantage > 0.0f ? r - (1.0f + p.clip_high) : row.advantage < 0.0f ? (1.0f - p.clip_low) - r : -r;
    float slope = beyond > 0.0f ? 0.0f : -(r * row.advantage), most = fabsf(slope);   // most: what the slope is off by, divided by `off`
    if (p.ref_logp) {
      const float by = p.kl_coef * (Ex2Approx(x * kLog2E) - 1.0f);
      slope -= by;
      most += p.kl_coef + fabsf(by);
    }
    // (what is beyond f32, and NaN, does not pass either)
    if (fabsf(beyond) > 2.0f * off * r && most * off < fmaf(0x1p-15f, fabsf(slope), 0x1p-126f)) return row.weight * slope;
  }
  return Times(PolicyOf(p, row, LogpOf<true>(a, q)).slope, row.weight);
}

__device__ __forceinline__ double WarpSum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
__device__ __forceinline__ float WarpMax(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xFFFFFFFF;" : "=f"(r) : "f"(v));
  return r;
}

// The sums of a far row, by a warp, from memory.  (Of -inf alone: NaN.)
template <typename T>
__device__ __noinline__ RowSums FarRow(const LogitArgs& a, uint64_t r, int32_t label) {
  const Row<T> row(a, r);
  const uint32_t lane = threadIdx.x & 31;
  float top = MinusInf(), v[kPerUnit<T>];
  for (uint32_t u = lane; u < row.units; u += 32) {
    row.Load(u, v);
#pragma unroll
    for (int j = 0; j < kPerUnit<T>; ++j) top = fmaxf(top, v[j]);
  }
  const float z_label = ToF32(row.z[label]), mk = FarOf(a, WarpMax(top));
  double sum = 0.0;   // (a lane has thousands of terms)
  for (uint32_t u = lane; u < row.units; u += 32) {
    row.Load(u, v);
    float part = 0.0f;
#pragma unroll
    for (int j = 0; j < kPerUnit<T>; ++j)
      if (row.At(u) + j != label) part += FarPower(a, v[j], mk);
    sum += static_cast<double>(part);
  }
  const float others = static_cast<float>(WarpSum(sum));
  return {z_label, mk, others, others + FarPower(a, z_label, mk)};
}
// Its dlogits, by a warp.
template <typename T>
__device__ __noinline__ void FarGradient(const LogitArgs& a, uint64_t r, int32_t label, const RowSums q, float slope) {
  const Row<T> row(a, r);
  const float by = -slope / q.s;
  const uint32_t label_unit = (static_cast<uint32_t>(label) + row.skip) / kPerUnit<T>;
  for (uint32_t u = threadIdx.x & 31; u < row.units; u += 32) {
    float v[kPerUnit<T>];
    row.Load(u, v);
#pragma unroll
    for (int j = 0; j < kPerUnit<T>; ++j) v[j] = slope == 0.0f ? 0.0f : by * FarPower(a, v[j], q.mk);
    row.Store(u, v);
    if (u == label_unit) row.d[label] = FromF32<T>(slope == 0.0f ? 0.0f : slope * (q.others / q.s));
  }
}
// Calls far(lane) for each lane of a warp whose row is far; all lanes are here.
template <typename F>
__device__ __forceinline__ void EachFar(bool is, F far) {
  for (uint32_t left = __ballot_sync(0xFFFFFFFFu, is); left != 0; left &= left - 1) far(static_cast<uint32_t>(__ffs(static_cast<int>(left)) - 1));
}

constexpr uint32_t kFinishThreads = 256;

// From what is kept of the rows: logp and the loss's three sums, a block's rows in its partials; the block that comes last (*arrived,
// which the rows' kernel has set to 0) adds them up, in the blocks' order.  A far row's dlogits are made here.
template <typename T>
__global__ void __launch_bounds__(kFinishThreads)
PolicyFinishKernel(const __grid_constant__ LogitArgs a, const __grid_constant__ PolicyArgs p, const float4* __restrict__ kept,
                   double* __restrict__ partials, uint32_t* __restrict__ arrived) {
  AwaitPrevious();
  __shared__ double meet[kFinishThreads / 32][3];
  __shared__ bool last;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double sums[3] = {};
  for (uint64_t r0 = static_cast<uint64_t>(blockIdx.x) * kFinishThreads + warp * 32; r0 < a.rows; r0 += static_cast<uint64_t>(gridDim.x) * kFinishThreads) {
    double logp = 0.0;
    const bool here = r0 + lane < a.rows;
    const uint64_t r = here ? r0 + lane : r0;
    const float4 k = kept[r];   // (all at once; of a row that does not count, whatever is there)
    const PolicyRow row = PolicyRowOf(p, r);
    const int32_t label = a.labels[r];
    const bool counts = here && Counts(label, a.classes);
    RowSums q = {k.x, k.y, k.z, k.w};
    EachFar(counts && IsFar(q.mk), [&](uint32_t which) {
      const RowSums sums = FarRow<T>(a, r0 + which, __shfl_sync(0xFFFFFFFFu, label, which));
      if (which == lane) q = sums;
    });
    if (counts) {
      logp = LogpOf<true>(a, q);
      const PolicyTerms t = PolicyOf(p, row, logp);
      const double kl = p.ref_logp ? KlOf(static_cast<double>(row.ref) - logp) : 0.0, weight = static_cast<double>(row.weight);
      sums[0] += Times(static_cast<double>(t.loss) + Times(kl, static_cast<double>(p.kl_coef)), weight);
      sums[1] += Times(kl, weight);
      sums[2] += t.clipped ? static_cast<double>(row.weight) : 0.0;
    }
    if (here) p.logp[r] = static_cast<float>(logp);
    if (a.dlogits == nullptr) continue;
    EachFar(counts && IsFar(q.mk), [&](uint32_t which) {
      auto of = [which](float v) { return __shfl_sync(0xFFFFFFFFu, v, which); };
      const float slope = Times(PolicyOf(p, row, logp).slope, row.weight) * ((p.loss_grad ? *p.loss_grad : 1.0f) * a.scale);
      FarGradient<T>(a, r0 + which, __shfl_sync(0xFFFFFFFFu, label, which), {of(q.z_label), of(q.mk), of(q.others), of(q.s)}, of(slope));
    });
  }
  auto block_sum = [&] {   // in warp 0's lanes, the three sums
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      sums[i] = WarpSum(sums[i]);
      if (lane == 0) meet[warp][i] = sums[i];
    }
    __syncthreads();
    if (warp == 0)
#pragma unroll
      for (int i = 0; i < 3; ++i) sums[i] = WarpSum(lane < kFinishThreads / 32 ? meet[lane][i] : 0.0);
  };
  block_sum();
  if (gridDim.x == 1) {
    if (threadIdx.x == 0)
#pragma unroll
      for (int i = 0; i < 3; ++i) p.loss[i] = static_cast<float>(sums[i]);
    return;
  }
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 0; i < 3; ++i) partials[blockIdx.x * 3 + i] = sums[i];
    __threadfence();
    last = atomicAdd(arrived, 1u) == gridDim.x - 1;
    __threadfence();
  }
  __syncthreads();
  if (!last) return;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    sums[i] = 0.0;
    for (uint32_t b = threadIdx.x; b < gridDim.x; b += kFinishThreads) sums[i] += __ldcg(&partials[b * 3 + i]);
  }
  block_sum();
  if (threadIdx.x == 0)
#pragma unroll
    for (int i = 0; i < 3; ++i) p.loss[i] = static_cast<float>(sums[i]);
}

// Rows of a preference loss that are a sequence's.
struct Sequences {
  const int32_t* starts;   // null: all are (the policy loss)
  uint32_t count;
};

// ---- rows in registers --------------------------------------------------------------------------------------
// A group of threads holds a row in registers as it lies in memory, NU units to a thread, or, where the blocks of a cluster share it, its
// part.  Exponentials are made twice, for the sums and for dlogits: 64 elements of 16 bits take 32 registers so, and two rows are at work
// on an SM at a time, one while the other's sums meet (8192 rows of 32000 in bf16 172 us; with the first exponentials kept, one row to an
// SM, 198).  Two exponentials an element take 4000 cycles of an SM's units a row, of the 5500 that HBM takes.  The rows that a group comes
// to next are on their way into its slots meanwhile.
template <typename T> constexpr int kPairs = kPerUnit<T> / 2;
template <typename T>
__device__ __forceinline__ void Pairs(const uint4& r, f32x2 (&v)[kPairs<T>]) {
  float f[kPerUnit<T>];
  Elements<T>(r, f);
#pragma unroll
  for (int j = 0; j < kPairs<T>; ++j) v[j] = PackF2(f[2 * j], f[2 * j + 1]);
}
__device__ __forceinline__ uint32_t Max2(uint32_t a, uint32_t b, Bf16) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t Max2(uint32_t a, uint32_t b, F16) {
  uint32_t r;
  asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// 2^x of both.
__device__ __forceinline__ f32x2 Powers(f32x2 x) {
  float lo, hi;
  UnpackF2(x, &lo, &hi);
  return PackF2(Ex2Approx(lo), Ex2Approx(hi));
}
// The largest of a thread's elements that is a number.
template <typename T, int NU>
__device__ __forceinline__ float Largest(const uint4 (&raw)[NU]) {
  if constexpr (sizeof(T) == 4) {
    float top = MinusInf();
#pragma unroll
    for (int i = 0; i < NU; ++i)
      top = fmaxf(top, fmaxf(fmaxf(__uint_as_float(raw[i].x), __uint_as_float(raw[i].y)), fmaxf(__uint_as_float(raw[i].z), __uint_as_float(raw[i].w))));
    return top;
  } else {
    uint32_t top = Nothing<T>().x;
#pragma unroll
    for (int i = 0; i < NU; ++i) top = Max2(top, Max2(Max2(raw[i].x, raw[i].y, T{}), Max2(raw[i].z, raw[i].w, T{}), T{}), T{});
    float a, b;
    Unpack2<T>(top, a, b);
    return fmaxf(a, b);
  }
}

// What a block shows the others of its cluster, and a barrier that counts them; two of each, used in turn.
struct Exchange {
  float2 parts[2][8];   // k M and the sum, of a block
  uint64_t bars[2];
};
__device__ __forceinline__ bool AwaitCluster(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = umma_dev::SmemAddr(bar);
  for (uint32_t it = 0; it < umma_dev::kWaitLimit; ++it) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(addr), "r"(parity)
        : "memory");
    if (done) return true;
  }
  return false;
}

// How a launch shares its rows: `threads` threads and `blocks` blocks of a cluster to a row, `part` units to a block.  Rows from `edge`
// on to `edge` before the last are copied in bulk: what sticks out of theirs is the matrix's too.
struct RowsPlan {
  uint32_t threads, over_threads, slots, blocks, part, edge;   // over_threads: 2^32 / threads, rounded up
};

// Blocks to an SM: of short rows, whose time is a row's chain, two.
constexpr uint32_t BlocksOf(uint32_t units) { return units <= 2 ? 2 : 1; }

template <typename T, int NU, bool kPolicy, bool kCluster>
__global__ void __launch_bounds__(kThreads, BlocksOf(NU))
LogitRowsKernel(const __grid_constant__ LogitArgs a, const __grid_constant__ PolicyArgs p, const Sequences seq, float4* __restrict__ kept,
                uint32_t* __restrict__ arrived, const RowsPlan plan) {
  constexpr uint32_t E = kPerUnit<T>;
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ float2 sums[2][kThreads / 32];            // k M and the sum, of a warp
  __shared__ uint32_t brought[2][kThreads / 32][8];    // of a group: the label's logit, and a PolicyRow
  __shared__ Exchange exchange[2];                     // of a group
  const uint32_t threads = plan.threads, group = threadIdx.x / threads, t = threadIdx.x - group * threads, lane = threadIdx.x & 31;
  const uint32_t groups = blockDim.x / threads, rank = kCluster ? blockIdx.x % plan.blocks : 0;
  const uint32_t slot_bytes = plan.part * 16, begin = rank * plan.part;   // begin: of this block's units of a row
  uint8_t* ring = dyn + static_cast<size_t>(group) * plan.slots * slot_bytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(dyn + static_cast<size_t>(groups) * plan.slots * slot_bytes) + group * plan.slots;
  const uint32_t rows = static_cast<uint32_t>(a.rows), step = (kCluster ? gridDim.x / plan.blocks : gridDim.x) * groups;
  const uint32_t first = (kCluster ? blockIdx.x / plan.blocks : blockIdx.x) * groups + group;
  if (t == 0) {
    for (uint32_t i = 0; i < plan.slots; ++i) umma_dev::MbarInit(&bars[i], 1);
    if constexpr (kCluster)
      for (uint32_t i = 0; i < 2; ++i) umma_dev::MbarInit(&exchange[group].bars[i], plan.blocks);
    umma_dev::MbarInitFence();
  }
  AwaitPrevious();
  auto logit_row = [&](uint32_t r) { return static_cast<const T*>(a.logits) + static_cast<uint64_t>(r) * a.stride; };
  auto skip_of = [](const T* z) { return static_cast<uint32_t>(reinterpret_cast<uint64_t>(z) & 15) / static_cast<uint32_t>(sizeof(T)); };
  auto units_of = [&](uint32_t skip) {   // of this block
    const uint32_t all = (skip + a.classes + E - 1) / E;
    return kCluster ? (all > begin ? min(plan.part, all - begin) : 0u) : all;
  };
  auto counts = [&](uint32_t r, int32_t label) {
    if (!Counts(label, a.classes)) return false;
    return kPolicy || (static_cast<int64_t>(r) >= seq.starts[0] && static_cast<int64_t>(r) < seq.starts[seq.count]);
  };
  auto bulk = [&](uint32_t r) { return r >= plan.edge && r < rows - plan.edge; };   // (edge is rows at most)
  auto fill = [&](uint32_t r, int32_t label, uint32_t slot) {   // the group's thread 0
    if (!counts(r, label) || !bulk(r)) return;
    const T* z = logit_row(r);
    const uint32_t skip = skip_of(z), bytes = units_of(skip) * 16;
    if (bytes == 0) return;
    umma_dev::MbarExpectTx(&bars[slot], bytes);
    umma_dev::BulkLoad(ring + static_cast<size_t>(slot) * slot_bytes, reinterpret_cast<const uint4*>(z - skip) + begin, bytes, &bars[slot]);
  };
  // What a row brings besides its logits is asked for while the one before it is at work: each item by one of the group's first threads,
  // as it is read.
  uint32_t ahead = 0;
  auto ask = [&](uint32_t r, int32_t label) {
    if (r >= rows || t > (kPolicy ? 4u : 0u) || !counts(r, label)) return;
    if (t == 0) ahead = reinterpret_cast<const std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>*>(logit_row(r))[label];
    else if (t == 1) ahead = __float_as_uint(p.old_logp[r]);
    else if (t == 2) ahead = p.ref_logp ? __float_as_uint(p.ref_logp[r]) : 0u;
    else if (t == 3) ahead = __float_as_uint(p.advantages[r]);
    else ahead = p.weights ? __float_as_uint(p.weights[r]) : 0x3F800000u;
  };
  int32_t fill_label = -1;   // of the row that goes into the slot that the next one leaves
  if (t == 0) {
    int32_t labels[9];
#pragma unroll
    for (uint32_t i = 0; i < 9; ++i) labels[i] = i <= plan.slots && first + i * step < rows ? a.labels[first + i * step] : -1;
#pragma unroll 1
    for (uint32_t i = 0; i < plan.slots && first + i * step < rows; ++i) {
      fill(first + i * step, labels[0], i);
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) labels[j] = labels[j + 1];
    }
    fill_label = labels[0];
  }
  const float grad = (kPolicy && p.loss_grad ? *p.loss_grad : 1.0f) * a.scale;
  if (kPolicy && blockIdx.x == 0 && threadIdx.x == 0) *arrived = 0;
  int32_t next_label = first < rows ? a.labels[first] : -1, label_behind = first + step < rows ? a.labels[first + step] : -1;
  ask(first, next_label);
  __syncwarp();
  if constexpr (kCluster) umma_dev::ClusterSync();   // (every block of it has begun: its shared memory may be written)
  else GroupBarrier(threads, group);                 // the barriers are there
  uint32_t turn = 0, slot = 0, parities = 0, exchanged = 0;   // a bit for each slot, of the copies that went through it; rows exchanged
  for (uint32_t r = first; r < rows; r += step) {
    const int32_t label = next_label;
    next_label = label_behind;
    label_behind = r + 2 * step < rows ? a.labels[r + 2 * step] : -1;
    const uint32_t item = ahead, now = slot;
    ask(r + step, next_label);
    if (++slot == plan.slots) slot = 0;
    auto refill = [&] {
      if (t != 0) return;
      const uint32_t next = r + plan.slots * step;
      if (next < rows) fill(next, fill_label, now);
      if (next + step < rows) fill_label = a.labels[next + step];
    };
    auto zeros = [&] {
      const Row<T> row(a, r);
      const float none[E] = {};
      const uint32_t end = units_of(row.skip);
      for (uint32_t u = t; u < end; u += threads) row.Store(begin + u, none);
    };
    if (!counts(r, label)) {
      if (kPolicy && a.dlogits) zeros();
      refill();
      continue;
    }
    uint4 raw[NU];
    bool owner;   // of the label
    {
      // This block's part in the slot, each thread's own units; -inf in place of the label and of what sticks out of the row.
      const uint32_t skip = skip_of(logit_row(r)), count = units_of(skip);
      uint4* mine = reinterpret_cast<uint4*>(ring + static_cast<size_t>(now) * slot_bytes);
      auto owns = [&](uint32_t u) { return u < count && u - __umulhi(u, plan.over_threads) * threads == t; };
      const int32_t at = label + static_cast<int32_t>(skip - begin * E), end = static_cast<int32_t>(skip + a.classes - begin * E);
      auto patch = [&](uint32_t u) {   // (the label of another unit: beyond the unit's elements)
        const int32_t from = static_cast<int32_t>(u * E);
        mine[u] = Only<T>(mine[u], static_cast<int32_t>(skip - begin * E) - from, end - from, at - from);
        umma_dev::FenceProxyAsync();   // (the next row's copy comes there)
      };
      owner = at >= 0 && owns(static_cast<uint32_t>(at) / E);
      if (bulk(r)) {
        if (count != 0) {
          AwaitRow(&bars[now], parities >> now & 1u, a.status);
          parities ^= 1u << now;
        }
        if (t == 0 && begin == 0 && skip != 0) patch(0);
        if (end < static_cast<int32_t>(count * E) && owns(count - 1)) patch(count - 1);
      } else {
        const Row<T> row(a, r);
        for (uint32_t u = t; u < count; u += threads) mine[u] = row.Raw(begin + u);
        umma_dev::FenceProxyAsync();   // (other rows' copies come there)
      }
      if (owner) patch(static_cast<uint32_t>(at) / E);
#pragma unroll
      for (int i = 0; i < NU; ++i) raw[i] = t + i * threads < count ? mine[t + i * threads] : Nothing<T>();
    }
    float mk = TopOf<kPolicy>(a, Largest<T, NU>(raw)), sum;
    // A lone slot is filled while the exponentials are made, unless dlogits will be stored meanwhile: loads and stores in turn are
    // faster then (8192 rows of 32000 in bf16: 172 us, early 184; a preference loss of 16 x 512 x 16001 in f32 357, early 344).
    const bool early = plan.slots == 1 && !(kPolicy && a.dlogits);
    if (early) {
      GroupBarrier(threads, group);
      refill();
    }
    {
      const f32x2 k2 = Splat2(a.k), rest2 = Splat2(a.k_rest), away = Splat2(mk == MinusInf() ? 0.0f : -mk);
      f32x2 sum2[kPairs<T>] = {};
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        f32x2 v[kPairs<T>];
        Pairs<T>(raw[i], v);
#pragma unroll
        for (int j = 0; j < kPairs<T>; ++j) sum2[j] = AddF2(sum2[j], Powers(kPolicy ? Fma2(v[j], k2, away) : Fma2(v[j], rest2, Fma2(v[j], k2, away))));
      }
#pragma unroll
      for (int j = 1; j < kPairs<T>; ++j) sum2[0] = AddF2(sum2[0], sum2[j]);
      float lo;
      UnpackF2(sum2[0], &lo, &sum);
      sum += lo;
    }
    // Warps, groups, blocks: the largest k M, and sums relative to it.  (A part without numbers has factor 0; NaN stays NaN.)
    auto factor = [](float own, float all) { return own == MinusInf() ? 0.0f : Ex2Approx(own - all); };
    auto join = [&](uint32_t most) {
      const float top = WarpMax(mk);   // (beyond `most` the lanes repeat themselves)
      sum *= factor(mk, top);
      mk = top;
#pragma unroll
      for (uint32_t o = 16; o > 0; o >>= 1)
        if (o <= most) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    };
    join(16);
    uint32_t* items = brought[turn][group];
    if (t < 5) items[t] = item;
    if (threads > 32) {
      float2* set = sums[turn] + group * (threads / 32);
      if (lane == 0) set[t >> 5] = make_float2(mk, sum);
      GroupBarrier(threads, group);
      const float2 warp_part = (lane & 15) < threads / 32 ? set[lane & 15] : make_float2(MinusInf(), 0.0f);
      mk = warp_part.x;
      sum = warp_part.y;
      join(8);
    } else {
      __syncwarp();
    }
    if constexpr (kCluster) {
      Exchange& x = exchange[group];
      if (t < plan.blocks) {
        const uint32_t to = umma_dev::MapToCta(umma_dev::SmemAddr(&x.parts[turn][rank]), t);
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(mk), "f"(sum) : "memory");
        umma_dev::MbarArriveCluster(umma_dev::MapToCta(umma_dev::SmemAddr(&x.bars[turn]), t));
      }
      if (!early) refill();   // (the slot is read)
      __syncwarp();
      if (!AwaitCluster(&x.bars[turn], exchanged >> 1 & 1u)) {
        a.status->wait_timeout = 1;
        umma_dev::DrainDelay();
      }
      ++exchanged;
      const float2 block_part = (lane & 7) < plan.blocks ? x.parts[turn][lane & 7] : make_float2(MinusInf(), 0.0f);
      mk = block_part.x;
      sum = block_part.y;
      join(4);
    } else if (!early) {
      refill();
    }
    turn ^= 1;
    // The label joins the maximum, so that its term is 1 at most.
    T raw_label;
    if constexpr (sizeof(T) == 4) raw_label = __uint_as_float(items[0]);
    else raw_label.bits = static_cast<uint16_t>(items[0]);
    const float z_label = ToF32(raw_label), mk_label = TopOf<kPolicy>(a, z_label), all = fmaxf(mk, mk_label);
    RowSums q = {z_label, all, sum * factor(mk, all), 0.0f};
    q.s = q.others + LabelTerm(a, z_label, q.mk);
    if (t == 0 && rank == 0) kept[r] = make_float4(q.z_label, q.mk, q.others, q.s);
    if constexpr (kPolicy) {
      if (!a.dlogits || IsFar(q.mk)) continue;
      const PolicyRow brings = {__uint_as_float(items[1]), __uint_as_float(items[2]), __uint_as_float(items[3]), __uint_as_float(items[4])};
      const float slope = SlopeOf<T>(a, p, brings, q) * grad;
      if (slope == 0.0f) {
        zeros();
        continue;
      }
      const float each = -slope / q.s;
      uint32_t again = r;
      asm volatile("" : "+r"(again));   // (the row's addresses anew: kept across the sums they cost registers that the units need)
      const Row<T> row(a, again);
      const uint32_t count = units_of(row.skip);
      // Units that lie wholly in the row, then, by their owners, the two that may not.
      const uint32_t whole_first = begin == 0 && row.skip != 0 ? 1 : 0, whole_end = min(count, (row.skip + a.classes) / E - begin);   // (without units: 0)
      const uint32_t whole = whole_end > whole_first ? whole_end - whole_first : 0;
      const f32x2 k2 = Splat2(a.k), away = Splat2(-q.mk), by = Splat2(each);
      auto unit = [&](const uint4& r, float (&v)[E]) {
        f32x2 pair[kPairs<T>];
        Pairs<T>(r, pair);
#pragma unroll
        for (int j = 0; j < kPairs<T>; ++j) UnpackF2(Mul2(Powers(Fma2(pair[j], k2, away)), by), &v[2 * j], &v[2 * j + 1]);
      };
      auto store_whole = [&] {
        uint4* to = reinterpret_cast<uint4*>(row.d - row.skip) + begin + t;
#pragma unroll
        for (int i = 0; i < NU; ++i) {
          if (t + i * threads - whole_first < whole) {
            // (unpacked anew: values of the first time, kept, would be spilled)
            asm volatile("" : "+r"(raw[i].x), "+r"(raw[i].y), "+r"(raw[i].z), "+r"(raw[i].w));
            float v[E];
            unit(raw[i], v);
            if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
            else Store8<T>(reinterpret_cast<T*>(to), v);
          }
          to += threads;
        }
      };
      if (row.alike && whole == count) {
        store_whole();
      } else if (row.alike) {
        float v[E];
        if (whole_first && t == 0) {
          unit(raw[0], v);
          row.Store(begin, v);
        }
        if (whole + whole_first != count) {   // the last one sticks out too
          uint4 last = raw[0];
#pragma unroll
          for (int i = 1; i < NU; ++i)
            if (t + i * threads == count - 1) last = raw[i];
          if (count - 1 - __umulhi(count - 1, plan.over_threads) * threads == t) {
            unit(last, v);
            row.Store(begin + count - 1, v);
          }
        }
        store_whole();
      } else {   // (from memory, element by element)
        for (uint32_t u = t; u < count; u += threads) {
          float v[E];
          row.Load(begin + u, v);
#pragma unroll
          for (uint32_t j = 0; j < E; ++j) v[j] = each * Ex2Approx(fmaf(v[j], a.k, -q.mk));
          row.Store(begin + u, v);
        }
      }
      if (owner) row.d[label] = FromF32<T>(slope * (q.others / q.s));
    }
  }
}

// ---- short rows ------------------------------------------------------------------------------------------------
// Rows of up to 128 units, more than a few: a warp to a row, straight into registers, the next row asked for while this one is at work.
// Their time is instructions: 16384 rows of 250 in bf16 with the ring's bookkeeping 29 us, so 18.5; 65536 in f32 64, so 52.
constexpr uint32_t kShortThreads = 256;
template <typename T, int NU, bool kPolicy>
__global__ void __launch_bounds__(kShortThreads)
LogitShortKernel(const __grid_constant__ LogitArgs a, const __grid_constant__ PolicyArgs p, const Sequences seq, float4* __restrict__ kept,
                 uint32_t* __restrict__ arrived) {
  AwaitPrevious();
  constexpr uint32_t E = kPerUnit<T>;
  const uint32_t lane = threadIdx.x & 31, rows = static_cast<uint32_t>(a.rows), step = gridDim.x * (kShortThreads / 32);
  const uint32_t first = (threadIdx.x >> 5) * gridDim.x + blockIdx.x;   // (every block gets rows before one gets two)
  if (kPolicy && blockIdx.x == 0 && threadIdx.x == 0) *arrived = 0;
  const uint64_t begin = reinterpret_cast<uint64_t>(a.logits), end = begin + (static_cast<uint64_t>(rows - 1) * a.stride + a.classes) * sizeof(T);
  const float grad = (kPolicy && p.loss_grad ? *p.loss_grad : 1.0f) * a.scale;
  auto counts = [&](uint32_t r, int32_t label) {
    if (!Counts(label, a.classes)) return false;
    return kPolicy || (static_cast<int64_t>(r) >= seq.starts[0] && static_cast<int64_t>(r) < seq.starts[seq.count]);
  };
  // Units as they lie, what is beside the row with them where it is the matrix's too; and, a lane each, what the row brings besides.
  uint4 next_raw[NU];
  uint32_t next_item = 0;
  auto ask = [&](uint32_t r, int32_t label) {
    if (r >= rows || !counts(r, label)) return;
    const Row<T> row(a, r);
    const uint64_t from = reinterpret_cast<uint64_t>(row.z) - row.skip * sizeof(T);
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const uint32_t u = lane + i * 32;
      const uint64_t at = from + static_cast<uint64_t>(u) * 16;
      if (u >= row.units) next_raw[i] = Nothing<T>();
      else if (at >= begin && at + 16 <= end) next_raw[i] = *reinterpret_cast<const uint4*>(at);
      else next_raw[i] = row.Raw(u);
    }
    if (lane == 0) next_item = reinterpret_cast<const std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>*>(row.z)[label];
    if (!kPolicy) return;
    const float* from_item = lane == 1 ? p.old_logp : lane == 2 ? p.ref_logp : lane == 3 ? p.advantages : lane == 4 ? p.weights : nullptr;
    if (from_item) next_item = __float_as_uint(from_item[r]);
    else if (lane == 4) next_item = 0x3F800000u;
  };
  int32_t next_label = first < rows ? a.labels[first] : -1, label_behind = first + step < rows ? a.labels[first + step] : -1;
  ask(first, next_label);
  const f32x2 k2 = Splat2(a.k), rest2 = Splat2(a.k_rest);
  for (uint32_t r = first; r < rows; r += step) {
    const int32_t label = next_label;
    next_label = label_behind;
    label_behind = r + 2 * step < rows ? a.labels[r + 2 * step] : -1;
    uint4 raw[NU];
#pragma unroll
    for (int i = 0; i < NU; ++i) raw[i] = next_raw[i];
    const uint32_t item = next_item;
    ask(r + step, next_label);
    const Row<T> row(a, r);
    if (!counts(r, label)) {
      if (kPolicy && a.dlogits) {
        const float none[E] = {};
        for (uint32_t u = lane; u < row.units; u += 32) row.Store(u, none);
      }
      continue;
    }
    const uint32_t label_unit = (static_cast<uint32_t>(label) + row.skip) / E, whole_end = (row.skip + a.classes) / E;
#pragma unroll
    for (int i = 0; i < NU; ++i) {   // -inf in place of the label and of what sticks out
      const uint32_t u = lane + i * 32;
      const int32_t e0 = static_cast<int32_t>(u * E) - static_cast<int32_t>(row.skip);
      if ((e0 < 0 || u >= whole_end || u == label_unit) && u < row.units) raw[i] = Only<T>(raw[i], -e0, static_cast<int32_t>(a.classes) - e0, label - e0);
    }
    const float mk = WarpMax(TopOf<kPolicy>(a, Largest<T, NU>(raw)));
    const f32x2 away = Splat2(mk == MinusInf() ? 0.0f : -mk);
    f32x2 sum2 = 0;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      f32x2 v[kPairs<T>];
      Pairs<T>(raw[i], v);
#pragma unroll
      for (int j = 0; j < kPairs<T>; ++j) sum2 = AddF2(sum2, Powers(kPolicy ? Fma2(v[j], k2, away) : Fma2(v[j], rest2, Fma2(v[j], k2, away))));
    }
    float lo, sum;
    UnpackF2(sum2, &lo, &sum);
    sum += lo;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    const uint32_t label_bits = __shfl_sync(0xFFFFFFFFu, item, 0);
    T raw_label;
    if constexpr (sizeof(T) == 4) raw_label = __uint_as_float(label_bits);
    else raw_label.bits = static_cast<uint16_t>(label_bits);
    const float z_label = ToF32(raw_label), mk_label = TopOf<kPolicy>(a, z_label), all = fmaxf(mk, mk_label);
    RowSums q = {z_label, all, mk == MinusInf() ? 0.0f * sum : sum * Ex2Approx(mk - all), 0.0f};
    q.s = q.others + LabelTerm(a, z_label, q.mk);
    if (lane == 0) kept[r] = make_float4(q.z_label, q.mk, q.others, q.s);
    if constexpr (kPolicy) {
      if (!a.dlogits || IsFar(q.mk)) continue;
      const PolicyRow brings = {__uint_as_float(__shfl_sync(0xFFFFFFFFu, item, 1)), __uint_as_float(__shfl_sync(0xFFFFFFFFu, item, 2)),
                                __uint_as_float(__shfl_sync(0xFFFFFFFFu, item, 3)), __uint_as_float(__shfl_sync(0xFFFFFFFFu, item, 4))};
      const float slope = SlopeOf<T>(a, p, brings, q) * grad;   // (0: zeros come out)
      const f32x2 by = Splat2(-slope / q.s), away_all = Splat2(-q.mk);
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        const uint32_t u = lane + i * 32;
        if (u >= row.units) continue;
        f32x2 pair[kPairs<T>];
        float v[E];
        Pairs<T>(raw[i], pair);
#pragma unroll
        for (int j = 0; j < kPairs<T>; ++j) UnpackF2(Mul2(Powers(Fma2(pair[j], k2, away_all)), by), &v[2 * j], &v[2 * j + 1]);
        row.Store(u, v);
        if (u == label_unit) row.d[label] = FromF32<T>(slope * (q.others / q.s));
      }
    }
  }
}

// ---- rows for their sums alone ----------------------------------------------------------------------------------
// A preference loss's rows, whose pairs decide on dlogits first, many of them and wide: `warps` warps of a block to a row, each with a ring
// of its own that runs ahead over its chunks of the block's rows.  (A group's ring costs a barrier a chunk.)  A policy loss that wants no
// dlogits would gain from it too (8192 rows of 32000 in bf16 109 us, so 93), but would not have the bits of the one that does.
//
// Only rows that count cost anything, and where they lie is known to the device alone.  So every block counts over the labels of a window
// of rows and lists each gridDim.x-th that counts for itself.  Each gridDim.x-th of all rows left an SM with 13 % more than its share of
// 8 pairs' answers: their sums took 88 us, so 78.
constexpr uint32_t kSumThreads = 768, kSumWarps = 8;   // kSumWarps: to a row, at most
constexpr uint32_t kSumUnits = 8, kSumChunk = kSumUnits * 32, kSumSlots = 2;   // units to a lane, and to a warp, at a time; chunks on their way to a warp
constexpr uint32_t kListed = 512, kCounted = 32768;   // rows of a block, and of a window, at most
template <typename T>
__global__ void __launch_bounds__(kSumThreads, 1)
LogitSumsKernel(const __grid_constant__ LogitArgs a, const Sequences seq, float4* __restrict__ kept, uint32_t warps, uint32_t window) {
  constexpr uint32_t E = kPerUnit<T>;
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ float2 sums[2][kSumThreads / 32];   // k M and the sum, of a warp
  __shared__ uint32_t before[kSumThreads / 32];
  __shared__ uint64_t all_bars[kSumThreads / 32][kSumSlots];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = warp / warps, part = warp - group * warps, groups = kSumThreads / 32 / warps;
  uint4* ring = reinterpret_cast<uint4*>(dyn) + warp * kSumSlots * kSumChunk;
  int2* list = reinterpret_cast<int2*>(dyn + kSumThreads / 32 * kSumSlots * kSumChunk * 16);   // [kListed] row and label
  uint32_t* masks = reinterpret_cast<uint32_t*>(list + kListed);                               // [kCounted / 32]
  uint64_t* bars = all_bars[warp];
  if (lane == 0) {
    for (uint32_t i = 0; i < kSumSlots; ++i) umma_dev::MbarInit(&bars[i], 1);
    umma_dev::MbarInitFence();
  }
  AwaitPrevious();
  const uint32_t rows_begin = static_cast<uint32_t>(max(seq.starts[0], 0));
  const uint32_t rows_end = min(static_cast<uint32_t>(a.rows), static_cast<uint32_t>(max(seq.starts[seq.count], 0)));
  const uint64_t begin = reinterpret_cast<uint64_t>(a.logits), end = begin + ((a.rows - 1) * a.stride + a.classes) * sizeof(T);
  // Whether these units of a row can be copied whole: the matrix's first and last may begin before it or end behind it.
  auto bulk = [&](const uint4* from, uint32_t units) {
    return reinterpret_cast<uint64_t>(from) >= begin && reinterpret_cast<uint64_t>(from + units) <= end;
  };
  const uint32_t stride_units = warps * kSumChunk;   // of a warp's chunks in a row
  uint32_t slot = 0, parities = 0;                   // a bit for each slot, of the copies that went through it
  const f32x2 k2 = Splat2(a.k), rest2 = Splat2(a.k_rest);
  auto factor = [](float own, float all) { return own == MinusInf() ? 0.0f : Ex2Approx(own - all); };
  uint32_t turn = 0;
  for (uint32_t base = rows_begin; base < rows_end; base += window) {
    const uint32_t count = min(window, rows_end - base), words = (count + 31) / 32;   // a bit for each row, set if it counts
#pragma unroll 8
    for (uint32_t w = warp; w < words; w += kSumThreads / 32) {
      const uint32_t i = w * 32 + lane;
      const uint32_t mask = __ballot_sync(0xFFFFFFFFu, i < count && Counts(a.labels[base + min(i, count - 1)], a.classes));
      if (lane == 0) masks[w] = mask;
    }
    __syncthreads();
    const uint32_t m0 = 2 * threadIdx.x < words ? masks[2 * threadIdx.x] : 0, m1 = 2 * threadIdx.x + 1 < words ? masks[2 * threadIdx.x + 1] : 0;
    const uint32_t own = __popc(m0) + __popc(m1);
    uint32_t at = own;
#pragma unroll
    for (uint32_t o = 1; o < 32; o *= 2) {
      const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, at, o);
      if (lane >= o) at += v;
    }
    if (lane == 31) before[warp] = at;
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (uint32_t w = 0; w < kSumThreads / 32; ++w) {
      if (w < warp) at += before[w];
      all += before[w];
    }
    at -= own;   // rows that count, before this thread's
    const uint32_t apart = gridDim.x, which = blockIdx.x;
    for (uint32_t n = at + (which + apart - at % apart) % apart; n < at + own; n += apart) {   // this block's among this thread's
      uint32_t i = n - at, m = m0, word = 2 * threadIdx.x;
      if (i >= __popc(m0)) {
        i -= __popc(m0);
        m = m1;
        ++word;
      }
      for (; i != 0; --i) m &= m - 1;
      const uint32_t r = base + word * 32 + __ffs(static_cast<int>(m)) - 1;
      list[n / apart] = make_int2(static_cast<int>(r), a.labels[r]);
    }
    const uint32_t listed = all > which ? (all - which - 1) / apart + 1 : 0;
    __syncthreads();
    // The chunk that is asked for next (by lane 0), ahead of the one at work.
    uint32_t f_row = group, f_unit = 0, f_units = 0, f_slot = slot;
    const uint4* f_from = nullptr;
    auto fill = [&] {
      if (lane != 0) return;
      while (f_unit >= f_units) {   // the next row (one may be too narrow for this warp)
        if (f_row >= listed) return;
        const Row<T> row(a, static_cast<uint32_t>(list[f_row].x));
        f_row += groups;
        f_from = reinterpret_cast<const uint4*>(row.z - row.skip);
        f_units = row.units;
        f_unit = part * kSumChunk;
      }
      const uint32_t units = min(kSumChunk, f_units - f_unit);
      if (bulk(f_from + f_unit, units)) {
        umma_dev::MbarExpectTx(&bars[f_slot], units * 16);
        umma_dev::BulkLoad(ring + f_slot * kSumChunk, f_from + f_unit, units * 16, &bars[f_slot]);
      }
      if (++f_slot == kSumSlots) f_slot = 0;
      f_unit += stride_units;
    };
#pragma unroll 1
    for (uint32_t i = 0; i < kSumSlots; ++i) fill();
    for (uint32_t i = group; i < listed; i += groups) {
      const uint32_t r = static_cast<uint32_t>(list[i].x);
      const int32_t label = list[i].y;
      const Row<T> row(a, r);
      uint32_t label_bits = 0;
      if (part == 0 && lane == 0) label_bits = reinterpret_cast<const std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>*>(row.z)[label];
      const uint32_t label_unit = (static_cast<uint32_t>(label) + row.skip) / E, ends_at = row.skip + a.classes;
      const uint4* from = reinterpret_cast<const uint4*>(row.z - row.skip);
      float mk = MinusInf(), sum = 0.0f;   // k M and the sum relative to it, of the others
      for (uint32_t u0 = part * kSumChunk; u0 < row.units; u0 += stride_units) {
        uint4 raw[kSumUnits];
        const uint32_t u1 = u0 + kSumChunk, units = min(kSumChunk, row.units - u0);
        if (bulk(from + u0, units)) {
          AwaitRow(&bars[slot], parities >> slot & 1u, a.status);
          parities ^= 1u << slot;
          const uint4* in = ring + slot * kSumChunk + lane;
#pragma unroll
          for (uint32_t j = 0; j < kSumUnits; ++j) raw[j] = lane + j * 32 < units ? in[j * 32] : Nothing<T>();
        } else {
#pragma unroll
          for (uint32_t j = 0; j < kSumUnits; ++j) raw[j] = lane + j * 32 < units ? row.Raw(u0 + lane + j * 32) : Nothing<T>();
        }
        if (++slot == kSumSlots) slot = 0;
        if ((u0 == 0 && row.skip != 0) || u1 * E > ends_at || (label_unit >= u0 && label_unit < u1)) {   // -inf in place of the label and of what sticks out
#pragma unroll
          for (uint32_t j = 0; j < kSumUnits; ++j) {
            const uint32_t u = u0 + lane + j * 32;
            const int32_t e0 = static_cast<int32_t>(u * E);
            if ((u == 0 && row.skip != 0) || u == row.units - 1 || u == label_unit)
              raw[j] = Only<T>(raw[j], static_cast<int32_t>(row.skip) - e0, static_cast<int32_t>(ends_at) - e0, label + static_cast<int32_t>(row.skip) - e0);
          }
        }
        const float top = fmaxf(mk, TopOf<false>(a, Largest<T, kSumUnits>(raw)));
        __syncwarp();   // the slot is read
        fill();
        const f32x2 away = Splat2(top == MinusInf() ? 0.0f : -top);
        f32x2 sum2[2] = {};
#pragma unroll
        for (uint32_t j = 0; j < kSumUnits; ++j) {
          f32x2 v[kPairs<T>];
          Pairs<T>(raw[j], v);
#pragma unroll
          for (int l = 0; l < kPairs<T>; ++l) sum2[l & 1] = AddF2(sum2[l & 1], Powers(Fma2(v[l], rest2, Fma2(v[l], k2, away))));
        }
        float lo, hi;
        UnpackF2(AddF2(sum2[0], sum2[1]), &lo, &hi);
        sum = fmaf(sum, factor(mk, top), lo + hi);
        mk = top;
      }
      // Lanes, warps: the largest k M, and sums relative to it.
      auto join = [&](uint32_t most) {
        const float top = WarpMax(mk);   // (beyond `most` the lanes repeat themselves)
        sum *= factor(mk, top);
        mk = top;
#pragma unroll
        for (uint32_t o = 16; o > 0; o >>= 1)
          if (o <= most) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
      };
      join(16);
      if (warps > 1) {
        float2* set = sums[turn] + group * warps;
        if (lane == 0) set[part] = make_float2(mk, sum);
        GroupBarrier(warps * 32, group);
        turn ^= 1;
        if (part != 0) continue;
        const float2 warp_part = (lane & (kSumWarps - 1)) < warps ? set[lane & (kSumWarps - 1)] : make_float2(MinusInf(), 0.0f);
        mk = warp_part.x;
        sum = warp_part.y;
        join(kSumWarps / 2);
      }
      if (lane != 0) continue;
      T raw_label;
      if constexpr (sizeof(T) == 4) raw_label = __uint_as_float(label_bits);
      else raw_label.bits = static_cast<uint16_t>(label_bits);
      const float z_label = ToF32(raw_label), mk_label = TopOf<false>(a, z_label), top = fmaxf(mk, mk_label);
      RowSums q = {z_label, top, sum * factor(mk, top), 0.0f};
      q.s = q.others + LabelTerm(a, z_label, q.mk);
      kept[r] = make_float4(q.z_label, q.mk, q.others, q.s);
    }
    __syncthreads();   // the list is read
  }
}

// ---- rows as streams ----------------------------------------------------------------------------------------
// A policy loss's rows wider than a cluster's registers: a group of 256 threads walks a row 16 KB at a time (four units a thread) through
// its ring, first for the sums, then, from L2, for dlogits.  The ring runs ahead over both walks and into the next row, so that loads
// never pause while sums meet; the other groups of the SM compute meanwhile.
constexpr uint32_t kWalkers = 256, kWalkUnits = 4, kChunk = kWalkers * kWalkUnits;   // threads of a group; units to a thread, and in a chunk
constexpr uint32_t kStreams = 3, kStreamSlots = (kMostShared - 8192) / (kStreams * kChunk * 16);   // groups to an SM, and chunks on their way to each

template <typename T>
__global__ void __launch_bounds__(kStreams * kWalkers, 1)
LogitStreamKernel(const __grid_constant__ LogitArgs a, const __grid_constant__ PolicyArgs p, float4* __restrict__ kept,
                  uint32_t* __restrict__ arrived) {
  constexpr uint32_t E = kPerUnit<T>;
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ float2 sums[2][kStreams * kWalkers / 32];   // k M and the sum, of a warp
  __shared__ uint32_t brought[2][kStreams][8];           // of a group: the label's logit, and a PolicyRow
  __shared__ uint64_t all_bars[kStreams][kStreamSlots];
  const uint32_t group = threadIdx.x / kWalkers, t = threadIdx.x % kWalkers, lane = threadIdx.x & 31;
  uint4* ring = reinterpret_cast<uint4*>(dyn) + group * kStreamSlots * kChunk;
  uint64_t* bars = all_bars[group];
  const uint32_t rows = static_cast<uint32_t>(a.rows), step = gridDim.x * kStreams, first = group * gridDim.x + blockIdx.x;   // (every SM gets rows before one gets two)
  const bool twice = a.dlogits != nullptr;
  if (t == 0) {
    for (uint32_t i = 0; i < kStreamSlots; ++i) umma_dev::MbarInit(&bars[i], 1);
    umma_dev::MbarInitFence();
  }
  AwaitPrevious();
  auto logit_row = [&](uint32_t r) { return static_cast<const T*>(a.logits) + static_cast<uint64_t>(r) * a.stride; };
  // A row's units and chunks, and whether a chunk can be copied whole: the matrix's first and last may begin before it or end behind it.
  struct Walk {
    const uint4* from;
    uint32_t skip, units, chunks;
  };
  auto walk_of = [&](uint32_t r) {
    Walk w;
    const T* z = logit_row(r);
    w.skip = static_cast<uint32_t>(reinterpret_cast<uint64_t>(z) & 15) / static_cast<uint32_t>(sizeof(T));
    w.from = reinterpret_cast<const uint4*>(z - w.skip);
    w.units = (w.skip + a.classes + E - 1) / E;
    w.chunks = (w.units + kChunk - 1) / kChunk;
    return w;
  };
  auto bulk = [&](const Walk& w, uint32_t chunk) {
    const T* begin = static_cast<const T*>(a.logits);
    const uint4* last = w.from + min((chunk + 1) * kChunk, w.units);
    return reinterpret_cast<const T*>(w.from + chunk * kChunk) >= begin &&
           reinterpret_cast<const T*>(last) <= begin + static_cast<uint64_t>(rows - 1) * a.stride + a.classes;
  };
  // The chunk that is asked for next (by the group's thread 0), ahead of the one at work.
  uint32_t f_row = first, f_chunk = 0, f_slot = 0;
  int32_t f_label = -1, f_next = -1;
  if (t == 0) {
    if (first < rows) f_label = a.labels[first];
    if (first + step < rows) f_next = a.labels[first + step];
  }
  auto fill = [&] {
    if (t != 0) return;
    auto next_row = [&] {
      f_row += step;
      f_label = f_next;
      f_next = f_row + step < rows ? a.labels[f_row + step] : -1;
      f_chunk = 0;
    };
    while (f_row < rows && f_chunk == 0 && !Counts(f_label, a.classes)) next_row();
    if (f_row >= rows) return;
    const Walk w = walk_of(f_row);
    const uint32_t chunk = f_chunk < w.chunks ? f_chunk : f_chunk - w.chunks, units = min(kChunk, w.units - chunk * kChunk);
    if (bulk(w, chunk)) {
      umma_dev::MbarExpectTx(&bars[f_slot], units * 16);
      umma_dev::BulkLoad(ring + f_slot * kChunk, w.from + chunk * kChunk, units * 16, &bars[f_slot]);
    }
    if (++f_slot == kStreamSlots) f_slot = 0;
    if (++f_chunk == w.chunks * (twice ? 2 : 1)) next_row();
  };
  // What a row brings besides its logits is asked for while the one before it is at work: each item by one of the group's first threads,
  // as it is read.
  uint32_t ahead = 0;
  auto ask = [&](uint32_t r, int32_t label) {
    if (r >= rows || t > 4 || !Counts(label, a.classes)) return;
    if (t == 0) ahead = reinterpret_cast<const std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>*>(logit_row(r))[label];
    else if (t == 1) ahead = __float_as_uint(p.old_logp[r]);
    else if (t == 2) ahead = p.ref_logp ? __float_as_uint(p.ref_logp[r]) : 0u;
    else if (t == 3) ahead = __float_as_uint(p.advantages[r]);
    else ahead = p.weights ? __float_as_uint(p.weights[r]) : 0x3F800000u;
  };
#pragma unroll 1
  for (uint32_t i = 0; i < kStreamSlots; ++i) fill();
  const float grad = (p.loss_grad ? *p.loss_grad : 1.0f) * a.scale;
  if (blockIdx.x == 0 && threadIdx.x == 0) *arrived = 0;
  int32_t next_label = first < rows ? a.labels[first] : -1, label_behind = first + step < rows ? a.labels[first + step] : -1;
  ask(first, next_label);
  __syncwarp();
  GroupBarrier(kWalkers, group);   // the barriers are there
  uint32_t turn = 0, slot = 0, parities = 0;   // a bit for each slot, of the copies that went through it
  for (uint32_t r = first; r < rows; r += step) {
    const int32_t label = next_label;
    next_label = label_behind;
    label_behind = r + 2 * step < rows ? a.labels[r + 2 * step] : -1;
    const uint32_t item = ahead;
    ask(r + step, next_label);
    const Row<T> row(a, r);
    if (!Counts(label, a.classes)) {
      const float none[E] = {};
      for (uint32_t u = t; twice && u < row.units; u += kWalkers) row.Store(u, none);
      continue;
    }
    const Walk w = walk_of(r);
    const uint32_t label_unit = (static_cast<uint32_t>(label) + w.skip) / E, ends_at = w.skip + a.classes;
    // A chunk's units of this thread, asked for by their number in the row; beyond it: nothing.
    uint4 raw[kWalkUnits];
    auto read = [&](uint32_t chunk) {
      const uint32_t u0 = chunk * kChunk + t;
      if (bulk(w, chunk)) {
        AwaitRow(&bars[slot], parities >> slot & 1u, a.status);
        parities ^= 1u << slot;
        const uint4* from = ring + slot * kChunk + t;
#pragma unroll
        for (uint32_t i = 0; i < kWalkUnits; ++i) raw[i] = u0 + i * kWalkers < w.units ? from[i * kWalkers] : Nothing<T>();
      } else {
#pragma unroll
        for (uint32_t i = 0; i < kWalkUnits; ++i) raw[i] = u0 + i * kWalkers < w.units ? row.Raw(u0 + i * kWalkers) : Nothing<T>();
      }
      if (++slot == kStreamSlots) slot = 0;
    };
    const f32x2 k2 = Splat2(a.k);
    float mk = MinusInf(), sum = 0.0f;   // k M and the sum relative to it, of the others
    auto factor = [](float own, float all) { return own == MinusInf() ? 0.0f : Ex2Approx(own - all); };
    for (uint32_t chunk = 0; chunk < w.chunks; ++chunk) {
      read(chunk);
      const uint32_t u0 = chunk * kChunk, u1 = u0 + kChunk;
      if ((chunk == 0 && w.skip != 0) || u1 * E > ends_at || (label_unit >= u0 && label_unit < u1)) {   // -inf in place of the label and of what sticks out
#pragma unroll
        for (uint32_t i = 0; i < kWalkUnits; ++i) {
          const uint32_t u = u0 + t + i * kWalkers;
          const int32_t e0 = static_cast<int32_t>(u * E);
          if ((u == 0 && w.skip != 0) || u == w.units - 1 || u == label_unit)
            raw[i] = Only<T>(raw[i], static_cast<int32_t>(w.skip) - e0, static_cast<int32_t>(ends_at) - e0, label + static_cast<int32_t>(w.skip) - e0);
        }
      }
      const float top = fmaxf(mk, TopOf<true>(a, Largest<T, kWalkUnits>(raw)));
      GroupBarrier(kWalkers, group);   // the slot is read
      fill();
      const f32x2 away = Splat2(top == MinusInf() ? 0.0f : -top);
      f32x2 sum2[kPairs<T>] = {};
#pragma unroll
      for (uint32_t i = 0; i < kWalkUnits; ++i) {
        f32x2 v[kPairs<T>];
        Pairs<T>(raw[i], v);
#pragma unroll
        for (int j = 0; j < kPairs<T>; ++j) sum2[j] = AddF2(sum2[j], Powers(Fma2(v[j], k2, away)));
      }
#pragma unroll
      for (int j = 1; j < kPairs<T>; ++j) sum2[0] = AddF2(sum2[0], sum2[j]);
      float lo, hi;
      UnpackF2(sum2[0], &lo, &hi);
      sum = fmaf(sum, factor(mk, top), lo + hi);
      mk = top;
    }
    // Warps and the group: the largest k M, and sums relative to it.
    auto join = [&](uint32_t most) {
      const float top = WarpMax(mk);
      sum *= factor(mk, top);
      mk = top;
#pragma unroll
      for (uint32_t o = 16; o > 0; o >>= 1)
        if (o <= most) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    };
    join(16);
    uint32_t* items = brought[turn][group];
    float2* set = sums[turn] + group * (kWalkers / 32);
    if (t < 5) items[t] = item;
    if (lane == 0) set[t >> 5] = make_float2(mk, sum);
    GroupBarrier(kWalkers, group);
    const float2 warp_part = set[lane & 7];
    mk = warp_part.x;
    sum = warp_part.y;
    join(4);
    turn ^= 1;
    T raw_label;
    if constexpr (sizeof(T) == 4) raw_label = __uint_as_float(items[0]);
    else raw_label.bits = static_cast<uint16_t>(items[0]);
    const float z_label = ToF32(raw_label), mk_label = TopOf<true>(a, z_label), all = fmaxf(mk, mk_label);
    RowSums q = {z_label, all, sum * factor(mk, all), 0.0f};
    q.s = q.others + LabelTerm(a, z_label, q.mk);
    if (t == 0) kept[r] = make_float4(q.z_label, q.mk, q.others, q.s);
    if (!twice) continue;   // (a far row is walked again all the same, as its chunks are on their way)
    const bool far = IsFar(q.mk);
    const PolicyRow brings = {__uint_as_float(items[1]), __uint_as_float(items[2]), __uint_as_float(items[3]), __uint_as_float(items[4])};
    const float slope = SlopeOf<T>(a, p, brings, q) * grad;   // (0: zeros come out)
    const f32x2 by = Splat2(-slope / q.s), away = Splat2(-q.mk);
    for (uint32_t chunk = 0; chunk < w.chunks; ++chunk) {
      read(chunk);
      uint4 out[kWalkUnits];
#pragma unroll
      for (uint32_t i = 0; i < kWalkUnits; ++i) {
        f32x2 pair[kPairs<T>];
        float v[E];
        Pairs<T>(raw[i], pair);
#pragma unroll
        for (int j = 0; j < kPairs<T>; ++j) UnpackF2(Mul2(Powers(Fma2(pair[j], k2, away)), by), &v[2 * j], &v[2 * j + 1]);
        if constexpr (sizeof(T) == 4) out[i] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        else out[i] = make_uint4(Pack2<T>(v[0], v[1]), Pack2<T>(v[2], v[3]), Pack2<T>(v[4], v[5]), Pack2<T>(v[6], v[7]));
      }
      GroupBarrier(kWalkers, group);   // the slot is read
      fill();
      const uint32_t u0 = chunk * kChunk + t;
      if (far) continue;
      if (row.alike && (chunk != 0 || w.skip == 0) && (chunk + 1) * kChunk * E <= ends_at) {
        uint4* to = reinterpret_cast<uint4*>(row.d - w.skip) + u0;
#pragma unroll
        for (uint32_t i = 0; i < kWalkUnits; ++i) to[i * kWalkers] = out[i];
      } else {
#pragma unroll
        for (uint32_t i = 0; i < kWalkUnits; ++i) {
          if (u0 + i * kWalkers >= w.units) continue;
          float v[E];
          Elements<T>(out[i], v);
          row.Store(u0 + i * kWalkers, v);
        }
      }
      if (label_unit / kChunk == chunk && label_unit % kWalkers == t) row.d[label] = FromF32<T>(slope * (q.others / q.s));
    }
  }
}

// ---- the preference loss ----------------------------------------------------------------------------------
// log(1 + e^x), in its tails too.
__device__ __forceinline__ double Softplus(double x) { return (x > 0.0 ? x : 0.0) + log1p(exp(-fabs(x))); }

constexpr uint32_t kPairThreads = 512;

// The logp of the far ones among a warp's rows first .. first + 31, and those kPairThreads / 2 further on, ... before `end`, whose sums are
// kept anew.
template <typename T>
__device__ __noinline__ double FarRows(const LogitArgs& a, float4* __restrict__ kept, int64_t first, int64_t end) {
  const uint32_t lane = threadIdx.x & 31;
  double sum = 0.0;
  for (int64_t r0 = first; r0 < end; r0 += kPairThreads / 2) {
    const int64_t r = r0 + lane;
    const int32_t label = r < end ? a.labels[r] : -1;
    EachFar(Counts(label, a.classes) && IsFar(kept[r].y), [&](uint32_t which) {
      const RowSums q = FarRow<T>(a, static_cast<uint64_t>(r0) + which, __shfl_sync(0xFFFFFFFFu, label, which));
      if (which != lane) return;
      kept[r] = make_float4(q.z_label, q.mk, q.others, q.s);
      sum += LogpOf<false>(a, q);
    });
  }
  return sum;
}

// Their dlogits; slope: the loss's derivative by the logp of each.
template <typename T>
__device__ __noinline__ void FarGradients(const LogitArgs& a, const float4* kept, int64_t first, int64_t end, float slope) {
  for (int64_t r0 = first; r0 < end; r0 += kPairThreads / 2) {
    const int64_t r = r0 + (threadIdx.x & 31);
    const int32_t label = r < end ? a.labels[r] : -1;
    EachFar(Counts(label, a.classes) && IsFar(kept[r].y), [&](uint32_t which) {
      const float4 q = kept[r0 + which];   // (the block has met since that was written)
      FarGradient<T>(a, static_cast<uint64_t>(r0) + which, __shfl_sync(0xFFFFFFFFu, label, which), {q.x, q.y, q.z, q.w}, slope);
    });
  }
}

// A pair to a block: the first eight warps sum the chosen rows, the others the rejected ones.  Then each row's kept.x becomes the loss's
// derivative by its logp, logit_scale and loss_grad included, 0 where it does not count; far rows get their dlogits.  losses [pairs]:
// added up by PreferenceFoldKernel.
template <typename T>
__global__ void __launch_bounds__(kPairThreads)
PreferencePairsKernel(const __grid_constant__ LogitArgs a, const __grid_constant__ PreferenceArgs p, float4* __restrict__ kept) {
  AwaitPrevious();
  __shared__ double sums[kPairThreads / 32][2];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, side = threadIdx.x / (kPairThreads / 2), t = threadIdx.x % (kPairThreads / 2);
  const float grad = (p.loss_grad ? *p.loss_grad : 1.0f) * a.scale;
  for (uint32_t pair = blockIdx.x; pair < p.pairs; pair += gridDim.x) {
    const uint32_t s = 2 * pair + side;
    const int64_t most = static_cast<int64_t>(a.rows);
    const int64_t begin = min(max(static_cast<int64_t>(p.starts[s]), static_cast<int64_t>(0)), most);
    const int64_t end = min(static_cast<int64_t>(p.starts[s + 1]), most);
    double sum = 0.0, counted = 0.0;
    bool far = false;
    for (int64_t r = begin + t; r < end; r += kPairThreads / 2) {
      const float4 q = kept[r];   // (asked for beside the label; of a row that does not count, whatever is there)
      if (Counts(a.labels[r], a.classes)) {
        counted += 1.0;
        if (IsFar(q.y)) far = true;
        else sum += LogpOf<false>(a, {q.x, q.y, q.z, q.w});
      }
    }
    far = __any_sync(0xFFFFFFFFu, far);
    if (far) sum += FarRows<T>(a, kept, begin + (t - lane), end);
    sum = WarpSum(sum);
    counted = WarpSum(counted);
    __syncthreads();   // (the last pair's are read)
    if (lane == 0) {
      sums[warp][0] = sum;
      sums[warp][1] = counted;
    }
    __syncthreads();
    double ratio[2], per_row[2];
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      sum = counted = 0.0;
#pragma unroll
      for (uint32_t w = i * (kPairThreads / 64); w < (i + 1) * (kPairThreads / 64); ++w) {
        sum += sums[w][0];
        counted += sums[w][1];
      }
      per_row[i] = p.average && counted > 0.0 ? 1.0 / counted : 1.0;
      sum *= per_row[i];
      if (threadIdx.x == 0) p.sequence_logp[2 * pair + i] = static_cast<float>(sum);
      ratio[i] = sum - (p.ref_logp ? static_cast<double>(p.ref_logp[2 * pair + i]) : 0.0);
    }
    const double beta = p.beta, h = beta * (ratio[0] - ratio[1]) - static_cast<double>(p.margin), smoothing = p.smoothing;
    double slope;
    if (p.kind == SEE_PREFERENCE_SIGMOID) slope = smoothing - 1.0 / (1.0 + exp(h));   // (a difference: f32 would leave no digits of it)
    else if (p.kind == SEE_PREFERENCE_HINGE) slope = h >= 1.0 ? 0.0 : h < 1.0 ? -1.0 : h;   // (NaN stays)
    else slope = 2.0 * (h - 0.5) / (beta * beta);
    if (a.dlogits) {
      const double each = slope * beta / static_cast<double>(p.pairs);
      const float of_row = static_cast<float>((side ? -each * per_row[1] : each * per_row[0]) * static_cast<double>(grad));
      for (int64_t r = begin + t; r < end; r += kPairThreads / 2) kept[r].x = Counts(a.labels[r], a.classes) ? of_row : 0.0f;
      if (far) FarGradients<T>(a, kept, begin + (t - lane), end, of_row);
    }
    if (threadIdx.x != 0) continue;   // (its functions take a microsecond: after the rows)
    const double off = (h - 0.5) / beta;
    p.margins[pair] = static_cast<float>(h);
    p.losses[pair] = p.kind == SEE_PREFERENCE_SIGMOID ? (1.0 - smoothing) * Softplus(-h) + smoothing * Softplus(h)
                     : p.kind == SEE_PREFERENCE_HINGE ? (h >= 1.0 ? 0.0 : 1.0 - h)
                                                      : off * off;
  }
}

// The pairs' average loss.
__device__ __forceinline__ void FoldLosses(const PreferenceArgs& p, double (&slots)[32]) {
  double loss = 0.0;
  for (uint32_t i = threadIdx.x; i < p.pairs; i += blockDim.x) loss += p.losses[i];
  loss = WarpSum(loss);
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = loss;
  __syncthreads();
  if (threadIdx.x != 0) return;
  loss = 0.0;
  for (uint32_t w = 0; w < blockDim.x / 32; ++w) loss += slots[w];
  *p.loss = static_cast<float>(loss / static_cast<double>(p.pairs));
}
__global__ void __launch_bounds__(256)
PreferenceFoldKernel(const __grid_constant__ PreferenceArgs p) {
  AwaitPrevious();
  __shared__ double slots[32];
  FoldLosses(p, slots);
}

constexpr uint32_t kGradThreads = 256;
constexpr int kGradUnits = 4;   // asked for at a time

// `warps` warps to a row, side by side; rows from the last one on, for what was read last is in L2.  Block 0 folds the losses first.
template <typename T>
__global__ void __launch_bounds__(kGradThreads)
PreferenceGradientKernel(const __grid_constant__ LogitArgs a, const __grid_constant__ PreferenceArgs p, const float4* __restrict__ kept, uint32_t warps) {
  AwaitPrevious();
  __shared__ double slots[32];
  if (blockIdx.x == 0) FoldLosses(p, slots);
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, side_by_side = kGradThreads / 32 / warps;
  const int64_t begin = max(static_cast<int64_t>(p.starts[0]), static_cast<int64_t>(0));
  const int64_t end = min(static_cast<int64_t>(p.starts[2 * p.pairs]), static_cast<int64_t>(a.rows));
  const float k = a.k, rest = a.k_rest;
  for (int64_t r = end - 1 - (static_cast<int64_t>(blockIdx.x) * side_by_side + warp / warps); r >= begin;
       r -= static_cast<int64_t>(gridDim.x) * side_by_side) {
    const float4 q = kept[r];
    const int32_t label = a.labels[r];
    const Row<T> row(a, r);
    const bool counts = Counts(label, a.classes);   // (what is kept of other rows is not set)
    const float slope = counts ? q.x : 0.0f, by = -slope / q.w, mk = q.y;
    const uint32_t label_unit = counts ? (static_cast<uint32_t>(label) + row.skip) / kPerUnit<T> : ~0u;
    const uint32_t units = counts && IsFar(mk) ? 0 : row.units;   // (a far row's dlogits are there)
    for (uint32_t u0 = (warp % warps) * 32 * kGradUnits + lane; u0 < units; u0 += warps * 32 * kGradUnits) {
      uint4 raw[kGradUnits];
      if (slope != 0.0f) {
#pragma unroll
        for (int i = 0; i < kGradUnits; ++i)
          if (u0 + i * 32 < units) raw[i] = row.RawOnce(u0 + i * 32);
      }
#pragma unroll
      for (int i = 0; i < kGradUnits; ++i) {
        const uint32_t u = u0 + i * 32;
        if (u >= units) break;
        float v[kPerUnit<T>];
        if (slope == 0.0f) {
#pragma unroll
          for (int j = 0; j < kPerUnit<T>; ++j) v[j] = 0.0f;
        } else {
          Elements<T>(raw[i], v);
#pragma unroll
          for (int j = 0; j < kPerUnit<T>; ++j) v[j] = by * Ex2Approx(fmaf(v[j], rest, fmaf(v[j], k, -mk)));
        }
        row.Store(u, v);
        if (u == label_unit) row.d[label] = FromF32<T>(slope == 0.0f ? 0.0f : slope * (q.z / q.w));
      }
    }
  }
}

// ---- launches ------------------------------------------------------------------------------------------------
// How rows are shared: `threads` threads and `blocks` blocks of a cluster to a row, `part` units to a block, `units` of them to a thread.
struct Sharing {
  uint32_t threads, units, blocks, part, groups, slots, clusters, edge;
  size_t bytes;
};
constexpr uint32_t kMostUnits = 16;   // to a thread, 64 registers
template <typename T>
bool ShareRows(const LogitArgs& a, uint32_t sms, Sharing* out) {
  const uint32_t all = (a.classes + 2 * (kPerUnit<T> - 1)) / kPerUnit<T>;   // units, wherever a row begins
  auto of = [all](uint32_t blocks) { return (all + blocks - 1) / blocks; };
  uint32_t blocks = 1;
  while (blocks < 8 && of(blocks) > kThreads * kMostUnits) blocks *= 2;
  // Few rows are shared by more blocks, down to two kilobytes each.
  while (blocks < 8 && a.rows * blocks * 2 <= sms && all / blocks > 256) blocks *= 2;
  Sharing s;
  s.blocks = blocks;
  s.part = of(blocks);
  if (s.part > kThreads * kMostUnits) return false;
  s.units = kMostUnits;
  if (a.rows * blocks <= sms) {   // a row to an SM: spread it over its threads
    s.units = 1;
    while (s.part > kThreads * s.units) s.units *= 2;
  }
  while (s.units > 1 && s.part <= 32 * (s.units / 2)) s.units /= 2;   // (a warp's row)
  s.threads = (((s.part + s.units - 1) / s.units) + 31) / 32 * 32;
  s.groups = kThreads / s.threads;
  if (blocks > 1 && s.groups > 2) s.groups = 2;
  const uint32_t resident = BlocksOf(s.units);
  const uint64_t most = resident * sms / blocks, each = (a.rows + most - 1) / most;
  if (s.groups > each) s.groups = static_cast<uint32_t>(each);
  const size_t slot = static_cast<size_t>(s.part) * 16, budget = (kMostShared - 4096) / resident;
  while (s.groups * (slot + 8) > budget) --s.groups;   // (a group's part is 128 KB at most)
  s.slots = static_cast<uint32_t>(budget / (s.groups * (slot + 8)));
  s.slots = s.slots > 8 ? 8 : s.slots;
  const uint64_t wanted = (a.rows + s.groups - 1) / s.groups;
  s.clusters = static_cast<uint32_t>(wanted < most ? wanted : most);
  const uint64_t turns = (wanted + s.clusters - 1) / s.clusters;
  if (s.slots > turns) s.slots = static_cast<uint32_t>(turns);
  s.bytes = s.groups * s.slots * (slot + 8);
  const uint64_t pitch = a.stride * sizeof(T);
  const bool exact = ((reinterpret_cast<uintptr_t>(a.logits) | pitch | a.classes * sizeof(T)) & 15) == 0;
  s.edge = exact ? 0 : static_cast<uint32_t>((15 + pitch) / pitch);
  if (2ull * s.edge > a.rows) s.edge = static_cast<uint32_t>(a.rows);   // (none in bulk)
  *out = s;
  return true;
}

// How many clusters of `blocks` blocks of a kernel the device holds at a time: fewer than its SMs would make, for a cluster lies within
// one of their groups.  A grid beyond that would leave whole rows to a second round (132 SMs of 148 in clusters of four, 120 of eight).
// Asked for once for each device and size, of blocks at their largest.
template <auto kKernel>
cudaError_t MostClusters(uint32_t blocks, uint32_t threads, size_t bytes, uint32_t* most) {
  static std::atomic<int> known[64][4] = {};   // by device, and blocks 2, 4, 8
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
  const uint32_t which = blocks == 2 ? 0 : blocks == 4 ? 1 : 2;
  int n = dev >= 0 && dev < 64 ? known[dev][which].load(std::memory_order_acquire) : 0;
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = blocks;
    cfg.blockDim = threads;
    cfg.dynamicSmemBytes = bytes;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = blocks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaError_t e = cudaOccupancyMaxActiveClusters(&n, kKernel, &cfg); e != cudaSuccess) return e;
    if (n < 1) n = 1;
    if (dev >= 0 && dev < 64) known[dev][which].store(n, std::memory_order_release);
  }
  *most = static_cast<uint32_t>(n);
  return cudaSuccess;
}

template <typename T, int NU, bool kPolicy, bool kCluster>
cudaError_t RunRows(const LogitArgs& a, const PolicyArgs& p, const Sequences& seq, float4* kept, uint32_t* arrived, Sharing& w, cudaStream_t s) {
  constexpr auto* kernel = LogitRowsKernel<T, NU, kPolicy, kCluster>;
  if (cudaError_t e = AllowShared<kernel>(kCluster ? kMostShared - 4096 : w.bytes); e != cudaSuccess) return e;
  if constexpr (kCluster) {
    uint32_t most;
    if (cudaError_t e = MostClusters<kernel>(w.blocks, kThreads, (kMostShared - 4096) / BlocksOf(NU), &most); e != cudaSuccess) return e;
    if (w.clusters > most) w.clusters = most;
  }
  return Next(kernel, w.clusters * w.blocks, w.groups * w.threads, w.bytes, s, w.blocks)(
      a, p, seq, kept, arrived, RowsPlan{w.threads, static_cast<uint32_t>(0xFFFFFFFFu / w.threads) + 1, w.slots, w.blocks, w.part, w.edge});
}
template <typename T, bool kPolicy, bool kCluster>
cudaError_t RunRows(const LogitArgs& a, const PolicyArgs& p, const Sequences& seq, float4* kept, uint32_t* arrived, Sharing& w, cudaStream_t s) {
  switch (w.units) {
    case 1: return RunRows<T, 1, kPolicy, kCluster>(a, p, seq, kept, arrived, w, s);
    case 2: return RunRows<T, 2, kPolicy, kCluster>(a, p, seq, kept, arrived, w, s);
    case 4: return RunRows<T, 4, kPolicy, kCluster>(a, p, seq, kept, arrived, w, s);
    case 8: return RunRows<T, 8, kPolicy, kCluster>(a, p, seq, kept, arrived, w, s);
    default: return RunRows<T, kMostUnits, kPolicy, kCluster>(a, p, seq, kept, arrived, w, s);
  }
}
template <typename T, bool kPolicy>
cudaError_t RunRows(const LogitArgs& a, const PolicyArgs& p, const Sequences& seq, float4* kept, uint32_t* arrived, uint32_t sms, cudaStream_t s) {
  // Short rows, from a few to a warp on.
  const uint32_t all = (a.classes + 2 * (kPerUnit<T> - 1)) / kPerUnit<T>;
  if (all <= 128 && a.rows > 8 * sms) {
    const uint64_t blocks = (a.rows + kShortThreads / 32 - 1) / (kShortThreads / 32), most = 4ull * sms;
    const unsigned grid = static_cast<unsigned>(blocks < most ? blocks : most);
    if (all <= 32) return Next(LogitShortKernel<T, 1, kPolicy>, grid, kShortThreads, 0, s)(a, p, seq, kept, arrived);
    if (all <= 64) return Next(LogitShortKernel<T, 2, kPolicy>, grid, kShortThreads, 0, s)(a, p, seq, kept, arrived);
    return Next(LogitShortKernel<T, 4, kPolicy>, grid, kShortThreads, 0, s)(a, p, seq, kept, arrived);
  }
  Sharing w;
  const bool shared = ShareRows<T>(a, sms, &w);
  if constexpr (kPolicy) {
    if (!shared) {   // (for 8192 rows of 32000 in bf16 227 us, in registers 172; for 2048 of 128256 254, in clusters 204)
      constexpr auto* kernel = LogitStreamKernel<T>;
      constexpr size_t bytes = kStreams * kStreamSlots * kChunk * 16;
      if (cudaError_t e = AllowShared<kernel>(bytes); e != cudaSuccess) return e;
      return Next(kernel, static_cast<unsigned>(a.rows < sms ? a.rows : sms), kStreams * kWalkers, bytes, s)(a, p, kept, arrived);
    }
  } else if (!shared || (a.rows > 2 * sms && (w.threads > kThreads / 2 || a.classes >= 20000))) {
    // Many rows wider than two groups of an SM hold, or of 20000 classes on: with pairs and gradient, 8 x 512 x 32000 in bf16 take 190 us,
    // in groups' registers 195; 16 x 100 x 50001 117 and 128; 16 x 512 x 20001 in f16 244 and 251.  But 16 x 512 x 16000 191 and 182, in
    // f32 356 and 344.  (The 20000 are for 16 bits: f32 rows have more than half a block's threads from 16384 classes on.)
    const uint32_t chunks = (all + kSumChunk - 1) / kSumChunk, window = sms * kListed;
    uint32_t warps = kSumWarps;   // to a row: as many as its chunks keep busy
    while (warps > 1 && (chunks + warps - 1) / warps * warps * 15 > chunks * 16) warps /= 2;
    constexpr auto* kernel = LogitSumsKernel<T>;
    constexpr size_t bytes = kSumThreads / 32 * kSumSlots * kSumChunk * 16 + kListed * sizeof(int2) + kCounted / 8;
    if (cudaError_t e = AllowShared<kernel>(bytes); e != cudaSuccess) return e;
    return Next(kernel, sms, kSumThreads, bytes, s)(a, seq, kept, warps, window < kCounted ? window : kCounted);
  }
  return w.blocks > 1 ? RunRows<T, kPolicy, true>(a, p, seq, kept, arrived, w, s) : RunRows<T, kPolicy, false>(a, p, seq, kept, arrived, w, s);
}

template <typename T>
cudaError_t Policy(const LogitArgs& a, const PolicyArgs& p, float4* kept, uint32_t sms, cudaStream_t s, int* launches) {
  if (a.rows == 0) return cudaMemsetAsync(p.loss, 0, 3 * sizeof(float), s);
  double* partials = reinterpret_cast<double*>(kept + a.rows);
  uint32_t* arrived = reinterpret_cast<uint32_t*>(partials + 3 * kPolicyPartials);
  if (cudaError_t e = RunRows<T, true>(a, p, {}, kept, arrived, sms, s); e != cudaSuccess) return e;
  *launches += 2;
  const uint64_t blocks = (a.rows + kFinishThreads - 1) / kFinishThreads;
  return Next(PolicyFinishKernel<T>, static_cast<unsigned>(blocks < kPolicyPartials ? blocks : kPolicyPartials), kFinishThreads, 0, s)(
      a, p, static_cast<const float4*>(kept), partials, arrived);
}

template <typename T>
cudaError_t Preference(const LogitArgs& a, const PreferenceArgs& p, float4* kept, uint32_t sms, cudaStream_t s, int* launches) {
  if (a.rows) {
    if (cudaError_t e = RunRows<T, false>(a, {}, {p.starts, 2 * p.pairs}, kept, nullptr, sms, s); e != cudaSuccess) return e;
    ++*launches;
  }
  if (cudaError_t e = Next(PreferencePairsKernel<T>, p.pairs < 4 * sms ? p.pairs : 4 * sms, kPairThreads, 0, s)(a, p, kept); e != cudaSuccess) return e;
  *launches += 2;
  if (!a.dlogits) return Next(PreferenceFoldKernel, 1, 256, 0, s)(p);
  // Warps to a row: as many as its pieces of 128 units keep busy, or, of few rows, as many as there are pieces for.
  const uint32_t pieces = (a.classes / kPerUnit<T> + 32 * kGradUnits) / (32 * kGradUnits);
  uint32_t warps = kGradThreads / 32;
  while (warps > 1 && (a.rows < 8 * sms ? warps > pieces : (pieces + warps - 1) / warps * warps * 15 > pieces * 16)) warps /= 2;
  const uint32_t rows_a_block = kGradThreads / 32 / warps;
  const uint64_t blocks = (a.rows + rows_a_block - 1) / rows_a_block, most = 6ull * sms;
  return Next(PreferenceGradientKernel<T>, static_cast<unsigned>(blocks < most ? blocks : most), kGradThreads, 0, s)(
      a, p, static_cast<const float4*>(kept), warps);
}

}  // namespace

cudaError_t PolicyLoss(const LogitArgs& a, int type, const PolicyArgs& p, float4* kept, uint32_t sms, cudaStream_t s, int* launches) {
  if (type == SEE_F32) return Policy<float>(a, p, kept, sms, s, launches);
  return type == SEE_BF16 ? Policy<Bf16>(a, p, kept, sms, s, launches) : Policy<F16>(a, p, kept, sms, s, launches);
}
cudaError_t PreferenceLoss(const LogitArgs& a, int type, const PreferenceArgs& p, float4* kept, uint32_t sms, cudaStream_t s, int* launches) {
  if (type == SEE_F32) return Preference<float>(a, p, kept, sms, s, launches);
  return type == SEE_BF16 ? Preference<Bf16>(a, p, kept, sms, s, launches) : Preference<F16>(a, p, kept, sms, s, launches);
}

}  // namespace see::k
