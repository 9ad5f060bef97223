// Losses over rows of logits: the labels' log-probabilities, a clipped policy loss or a preference loss of them, and the
// gradient of the logits.  With z = logit_scale logits, M its maximum and l the label, a row is
//   e_c = 2^(k logit_c - k M),  k = logit_scale / ln 2,   others = sum of e_c over c != l,   s = others + e_l,
//   logp = (z_l - M) - log s, or -log1p(others / e_l) where the label holds three quarters (no digits are lost next to 0),
//   dlogit_c = -slope logit_scale e_c / s,  of the label  slope logit_scale others / s   (not 1 - p, which would lose them),
// slope being the loss's derivative by logp.  The product k M is rounded once and the same in every exponent of a row, so that its
// rounding cancels between e_c and s.  Bound by HBM: logits are read once, dlogits written once.
//
// A row is walked in units of 16 bytes by address, of which the first and the last may stick out of it, whatever its alignment.  Rows reach
// registers through a ring in shared memory (LogitRowsKernel); wide rows, and few ones, are shared by the blocks of a cluster.  What
// is wider still is read from memory twice (LogitWideKernel).
//
// logp is made in double: a sequence's sum of hundreds of them is held against a reference's.
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
    constexpr uint32_t kNone = sizeof(T) == 4 ? 0xFF800000u : std::is_same_v<T, Bf16> ? 0xFF80u : 0xFC00u;
    uint32_t r[4] = {};
#pragma unroll
    for (int j = 0; j < kPerUnit<T>; ++j)
      r[j * sizeof(T) / 4] |= (at + j >= 0 && at + j < static_cast<int32_t>(classes) ? static_cast<uint32_t>(bits[at + j]) : kNone) << (j * sizeof(T) % 4 * 8);
    return make_uint4(r[0], r[1], r[2], r[3]);
  }
  __device__ __forceinline__ void Load(uint32_t unit, float* v) const { Elements<T>(Raw(unit), v); }
  __device__ __forceinline__ void Store(uint32_t unit, const float* v) const {
    const int32_t at = At(unit);
    if (alike && Whole(at)) {
      if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(d + at) = make_float4(v[0], v[1], v[2], v[3]);
      else Store8<T>(d + at, v);
      return;
    }
#pragma unroll
    for (int j = 0; j < kPerUnit<T>; ++j)
      if (at + j >= 0 && at + j < static_cast<int32_t>(classes)) d[at + j] = FromF32<T>(v[j]);
  }
};

// A maximum m, its product mk = k m (0 where m is -inf), and sum = the sum of e relative to it.
struct Part {
  float m, mk, sum;
};
__device__ __forceinline__ Part NoPart() { return {MinusInf(), 0.0f, 0.0f}; }
// (sums of nothing are 0, or NaN if what they are of is: neither is scaled)
__device__ __forceinline__ float Rescaled(const Part& p, float mk) { return p.m == MinusInf() ? p.sum : p.sum * Ex2Approx(p.mk - mk); }
__device__ __forceinline__ Part Joined(const Part& a, const Part& b) {
  const Part& top = a.m >= b.m ? a : b;
  return {top.m, top.mk, Rescaled(a, top.mk) + Rescaled(b, top.mk)};
}
__device__ __forceinline__ Part WarpJoin(Part p) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Part other = {__shfl_xor_sync(0xFFFFFFFFu, p.m, o), __shfl_xor_sync(0xFFFFFFFFu, p.mk, o), __shfl_xor_sync(0xFFFFFFFFu, p.sum, o)};
    p = threadIdx.x & o ? Joined(other, p) : Joined(p, other);   // (one order in both)
  }
  return p;
}

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
  return n * r;
}
// log s of a sum of f32 terms: s = 2^e m with m next to 1, and (m - 1) / (m + 1) into the series.
__device__ __forceinline__ double LogOf(float s) {
  if (!(s > 1e-30f && s < __int_as_float(0x7F800000))) return static_cast<double>(logf(s));
  const int32_t bits = __float_as_int(s) - 0x3F3504F3;   // (of 2^-1/2)
  const int32_t e = bits >> 23;
  const double m = static_cast<double>(__int_as_float((bits & 0x007FFFFF) + 0x3F3504F3));
  return fma(static_cast<double>(e), 0.6931471805599453, LogRatio(Quotient(m - 1.0, m + 1.0)));
}

// Of a row: the label's logit, k M, the sum over the others, the sum over all.
struct RowSums {
  float z_label, mk, others, s;
};
__device__ __forceinline__ float LabelTerm(const LogitArgs& a, float z_label, float mk) { return Ex2Approx(fmaf(z_label, a.k, -mk)); }
__device__ __forceinline__ double LogpOf(const LogitArgs& a, const RowSums& q) {
  const float e = LabelTerm(a, q.z_label, q.mk);
  if (3.0f * q.others < e) {   // -log1p(others / e)
    const double ratio = Quotient(static_cast<double>(q.others), static_cast<double>(e));
    return -LogRatio(Quotient(ratio, 2.0 + ratio));
  }
  return static_cast<double>(a.scale) * (static_cast<double>(q.z_label) - static_cast<double>(q.mk) * a.inv_k) - LogOf(q.s);
}

// By a block's threads; `slots` is free after the caller's next barrier.
template <typename T>
__device__ __forceinline__ RowSums SumsOf(const Row<T>& row, uint32_t label, float k, Part (&slots)[kThreads / 32]) {
  const uint32_t label_unit = (label + row.skip) / kPerUnit<T>, label_slot = (label + row.skip) % kPerUnit<T>;
  const float z_label = ToF32(row.z[label]);
  Part p = NoPart();
  for (uint32_t u = threadIdx.x; u < row.units; u += kThreads) {
    float v[kPerUnit<T>], top = MinusInf();
    row.Load(u, v);
#pragma unroll
    for (int j = 0; j < kPerUnit<T>; ++j) top = fmaxf(top, v[j]);
    if (top > p.m) {
      const float mk = __fmul_rn(top, k);
      p = {top, mk, Rescaled(p, mk)};
    }
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kPerUnit<T>; ++j) {
      const float e = Ex2Approx(fmaf(v[j], k, -p.mk));
      sum += u == label_unit && static_cast<uint32_t>(j) == label_slot ? 0.0f : e;
    }
    p.sum += sum;
  }
  p = WarpJoin(p);
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = p;
  __syncthreads();
  p = (threadIdx.x & 31) < kThreads / 32 ? slots[threadIdx.x & 31] : NoPart();
  p = WarpJoin(p);
  return {z_label, p.mk, p.sum, p.sum + Ex2Approx(fmaf(z_label, k, -p.mk))};
}

// dlogits of a row; slope includes logit_scale.
template <typename T>
__device__ __forceinline__ void Gradient(const Row<T>& row, uint32_t label, float k, float mk, float others, float s, float slope) {
  const uint32_t label_unit = (label + row.skip) / kPerUnit<T>, label_slot = (label + row.skip) % kPerUnit<T>;
  const float by = -slope / s, of_label = slope * (others / s);
  for (uint32_t u = threadIdx.x; u < row.units; u += kThreads) {
    float v[kPerUnit<T>];
    row.Load(u, v);
#pragma unroll
    for (int j = 0; j < kPerUnit<T>; ++j) {
      v[j] = by * Ex2Approx(fmaf(v[j], k, -mk));
      if (u == label_unit && static_cast<uint32_t>(j) == label_slot) v[j] = of_label;
    }
    row.Store(u, v);
  }
}
template <typename T>
__device__ __forceinline__ void Zeros(const Row<T>& row) {
  const float v[kPerUnit<T>] = {};
  for (uint32_t u = threadIdx.x; u < row.units; u += kThreads) row.Store(u, v);
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
struct PolicyTerms {
  float slope, loss, kl, clipped;   // slope: of the weighted loss by logp
};
__device__ __forceinline__ PolicyTerms PolicyOf(const PolicyArgs& p, const PolicyRow& row, double logp) {
  const float a = row.advantage, w = row.weight;
  const float r = expf(static_cast<float>(logp - static_cast<double>(row.old)));
  const float cut = r < 1.0f - p.clip_low ? 1.0f - p.clip_low : r > 1.0f + p.clip_high ? 1.0f + p.clip_high : r;
  const bool clipped = r * a > cut * a;
  float loss = clipped ? -(cut * a) : -(r * a), slope = clipped ? 0.0f : -(r * a), kl = 0.0f;
  if (p.ref_logp) {
    const float x = static_cast<float>(static_cast<double>(row.ref) - logp), grown = expm1f(x);
    kl = grown - x;
    loss += p.kl_coef * kl;
    slope -= p.kl_coef * grown;
  }
  return {w * slope, w * loss, w * kl, clipped ? w : 0.0f};
}

__device__ __forceinline__ double WarpSum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// A warp to each of the three sums.
__global__ void __launch_bounds__(96)
PolicyFoldKernel(const double* __restrict__ partials, uint32_t count, float* __restrict__ loss) {
  AwaitPrevious();
  const uint32_t which = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double sum = 0.0;
  for (uint32_t i = lane; i < count; i += 32) sum += partials[i * 3 + which];
  sum = WarpSum(sum);
  if (lane == 0) loss[which] = static_cast<float>(sum);
}

// Rows of a preference loss that are a sequence's.
struct Sequences {
  const int32_t* starts;   // null: all are (the policy loss)
  uint32_t count;
};

// ---- rows in registers --------------------------------------------------------------------------------------
// A group of T threads holds a row, or where C blocks of a cluster share it, its part of `part` units: NU units to a thread, first as they lie in memory, then
// as e relative to the thread's own maximum.  One exponential an element and no second reading: 8192 rows of 32000 in bf16 would take 4000 cycles of an
// SM's exponential units a row with two, of the 5500 that HBM takes.  The rows that a group comes to next are on their way into its slots meanwhile.
template <typename T> constexpr int kPairs = kPerUnit<T> / 2;
template <typename T>
__device__ __forceinline__ void Pairs(const uint4& r, f32x2 (&v)[kPairs<T>]) {
  float f[kPerUnit<T>];
  Elements<T>(r, f);
#pragma unroll
  for (int j = 0; j < kPairs<T>; ++j) v[j] = PackF2(f[2 * j], f[2 * j + 1]);
}
// -inf in every element.
template <typename T>
__device__ __forceinline__ uint4 Nothing() {
  const uint32_t w = sizeof(T) == 4 ? 0xFF800000u : std::is_same_v<T, Bf16> ? 0xFF80FF80u : 0xFC00FC00u;
  return make_uint4(w, w, w, w);
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

// kC > 1: the blocks of a cluster share each row.
template <typename T, int NU, bool kPolicy, bool kCluster>
__global__ void __launch_bounds__(kThreads, 1)
LogitRowsKernel(const __grid_constant__ LogitArgs a, const __grid_constant__ PolicyArgs p, const Sequences seq, float4* __restrict__ kept,
                double* __restrict__ partials, uint32_t threads, uint32_t slots, uint32_t blocks, uint32_t part) {
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ float2 sums[2][kThreads / 32];        // k M and the sum, of a warp
  __shared__ float2 parts[2][8];                   // of a block
  const uint32_t groups = blockDim.x / threads, group = threadIdx.x / threads, t = threadIdx.x - group * threads, lane = threadIdx.x & 31;
  const uint32_t rank = kCluster ? blockIdx.x % blocks : 0, cluster = kCluster ? blockIdx.x / blocks : blockIdx.x;
  const uint32_t clusters = kCluster ? gridDim.x / blocks : gridDim.x;
  const uint32_t slot_bytes = part * 16;
  uint8_t* ring = dyn + static_cast<size_t>(group) * slots * slot_bytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(dyn + static_cast<size_t>(groups) * slots * slot_bytes) + group * slots;
  const uint64_t first = static_cast<uint64_t>(cluster) * groups + group, step = static_cast<uint64_t>(clusters) * groups;
  if (t == 0) {
    for (uint32_t i = 0; i < slots; ++i) umma_dev::MbarInit(&bars[i], 1);
    umma_dev::MbarInitFence();
  }
  AwaitPrevious();
  const uint64_t begin = reinterpret_cast<uint64_t>(a.logits), end = begin + ((a.rows - 1) * a.stride + a.classes) * sizeof(T);
  // The units of this block's part of a row, and whether they can be copied whole.
  struct Share {
    uint64_t from;
    uint32_t first, count;
    bool bulk;
  };
  auto share_of = [&](const Row<T>& row) {
    Share w;
    w.first = rank * part;
    w.count = row.units > w.first ? min(part, row.units - w.first) : 0;
    w.from = reinterpret_cast<uint64_t>(row.z) - row.skip * sizeof(T) + static_cast<uint64_t>(w.first) * 16;
    w.bulk = w.count != 0 && w.from >= begin && w.from + static_cast<uint64_t>(w.count) * 16 <= end;
    return w;
  };
  int64_t seq_first = 0, seq_end = 0;
  if (!kPolicy) {
    seq_first = seq.starts[0];
    seq_end = seq.starts[seq.count];
  }
  auto counts = [&](uint64_t r, int32_t label) {
    return Counts(label, a.classes) && (kPolicy || (static_cast<int64_t>(r) >= seq_first && static_cast<int64_t>(r) < seq_end));
  };
  auto fill = [&](uint64_t r, int32_t label, uint32_t slot) {   // the group's thread 0
    if (!counts(r, label)) return;
    const Share w = share_of(Row<T>(a, r));
    if (!w.bulk) return;
    umma_dev::MbarExpectTx(&bars[slot], w.count * 16);
    umma_dev::BulkLoad(ring + static_cast<size_t>(slot) * slot_bytes, reinterpret_cast<const void*>(w.from), w.count * 16, &bars[slot]);
  };
  int32_t fill_label = -1;   // of the row that goes into the slot that the next one leaves
  if (t == 0) {
    int32_t labels[9];
#pragma unroll
    for (uint32_t i = 0; i < 9; ++i) labels[i] = i <= slots && first + i * step < a.rows ? a.labels[first + i * step] : -1;
#pragma unroll
    for (uint32_t i = 0; i < 9; ++i) {
      if (i < slots && first + i * step < a.rows) fill(first + i * step, labels[i], i);
      if (i == slots) fill_label = labels[i];
    }
  }
  const float grad = (kPolicy && p.loss_grad ? *p.loss_grad : 1.0f) * a.scale;
  if constexpr (kCluster) umma_dev::ClusterSync();   // (every block of it has begun: its shared memory may be written)
  else GroupBarrier(threads, group);                  // the barriers are there
  double total[3] = {};
  uint32_t turn = 0, slot = 0, parities = 0;   // a bit for each slot, of the copies that went through it
  int32_t next_label = first < a.rows ? a.labels[first] : -1;
  for (uint64_t r = first; r < a.rows; r += step) {
    const int32_t label = next_label;
    if (r + step < a.rows) next_label = a.labels[r + step];
    const Row<T> row(a, r);
    const Share w = share_of(row);
    const uint32_t now = slot;
    if (++slot == slots) slot = 0;
    auto refill = [&] {
      if (t != 0) return;
      const uint64_t next = r + slots * step;
      if (next < a.rows) fill(next, fill_label, now);
      if (next + step < a.rows) fill_label = a.labels[next + step];
    };
    auto zeros = [&] {
      const float none[kPerUnit<T>] = {};
      for (uint32_t u = t; u < w.count; u += threads) row.Store(w.first + u, none);
    };
    if (!counts(r, label)) {
      if (kPolicy) {
        if (t == 0 && rank == 0) p.logp[r] = 0.0f;
        if (a.dlogits) zeros();
      }
      refill();
      continue;
    }
    const float z_label = ToF32(row.z[label]);
    PolicyRow brings = {};
    if (kPolicy) brings = PolicyRowOf(p, r);
    uint4 raw[NU];
    if (w.bulk) {
      AwaitRow(&bars[now], parities >> now & 1u, a.status);
      parities ^= 1u << now;
      const uint4* from = reinterpret_cast<const uint4*>(ring + static_cast<size_t>(now) * slot_bytes);
#pragma unroll
      for (int i = 0; i < NU; ++i) raw[i] = t + i * threads < w.count ? from[t + i * threads] : Nothing<T>();
    }
    // What sticks out of the row, and the rows at the matrix's ends.
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const uint32_t u = w.first + t + i * threads;
      if (!w.bulk || u == 0 || u == row.units - 1) raw[i] = t + i * threads < w.count ? row.Raw(u) : Nothing<T>();
    }
    float mk = __fmul_rn(Largest<T, NU>(raw), a.k);   // -inf: nothing here
    const f32x2 k2 = Splat2(a.k), away = Splat2(mk == MinusInf() ? 0.0f : -mk);
    const uint32_t label_unit = (static_cast<uint32_t>(label) + row.skip) / kPerUnit<T>, label_at = (static_cast<uint32_t>(label) + row.skip) % kPerUnit<T>;
    f32x2 e[NU][kPairs<T>], sum2 = 0;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      f32x2 v[kPairs<T>];
      Pairs<T>(raw[i], v);
#pragma unroll
      for (int j = 0; j < kPairs<T>; ++j) {
        float lo, hi;
        UnpackF2(Fma2(v[j], k2, away), &lo, &hi);
        e[i][j] = PackF2(Ex2Approx(lo), Ex2Approx(hi));
      }
      if (w.first + t + i * threads == label_unit) {   // the label is not among the others
#pragma unroll
        for (int j = 0; j < kPairs<T>; ++j) {
          float lo, hi;
          UnpackF2(e[i][j], &lo, &hi);
          e[i][j] = PackF2(label_at == 2 * j ? 0.0f : lo, label_at == 2 * j + 1 ? 0.0f : hi);
        }
      }
#pragma unroll
      for (int j = 0; j < kPairs<T>; ++j) sum2 = AddF2(sum2, e[i][j]);
    }
    float lo, sum;
    UnpackF2(sum2, &lo, &sum);
    sum += lo;
    // Warps, groups, blocks: the largest k M, and sums relative to it.  (A part without numbers has factor 0; NaN stays NaN.)
    auto factor = [](float own, float all) { return own == MinusInf() ? 0.0f : Ex2Approx(own - all); };
    const float own = mk;
    auto join = [&](uint32_t most) {
      float top = mk;
      for (uint32_t o = most; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
      sum *= factor(mk, top);
      mk = top;
      for (uint32_t o = most; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    };
    join(16);
    if (threads > 32) {
      float2* set = sums[turn] + group * (threads / 32);
      if (lane == 0) set[t >> 5] = make_float2(mk, sum);
      GroupBarrier(threads, group);
      const float2 mine = lane < threads / 32 ? set[lane] : make_float2(MinusInf(), 0.0f);
      mk = mine.x;
      sum = mine.y;
      join(16);
    } else {
      __syncwarp();
    }
    refill();   // (the slot is read)
    if constexpr (kCluster) {
      if (t < blocks) {
        const uint32_t to = umma_dev::MapToCta(umma_dev::SmemAddr(&parts[turn][rank]), t);
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(mk), "f"(sum) : "memory");
      }
      __syncwarp();
      umma_dev::ClusterSync();
      const float2 mine = lane < blocks ? parts[turn][lane] : make_float2(MinusInf(), 0.0f);
      mk = mine.x;
      sum = mine.y;
      join(4);
      mk = __shfl_sync(0xFFFFFFFFu, mk, 0);
      sum = __shfl_sync(0xFFFFFFFFu, sum, 0);
    }
    turn ^= 1;
    RowSums q = {z_label, mk == MinusInf() ? 0.0f : mk, sum, 0.0f};
    q.s = q.others + LabelTerm(a, z_label, q.mk);
    if constexpr (!kPolicy) {
      if (t == 0 && rank == 0) kept[r] = make_float4(q.z_label, q.mk, q.others, q.s);
    } else {
      const double logp = LogpOf(a, q);
      const PolicyTerms terms = PolicyOf(p, brings, logp);
      if (t == 0 && rank == 0) {
        p.logp[r] = static_cast<float>(logp);
        total[0] += terms.loss;
        total[1] += terms.kl;
        total[2] += terms.clipped;
      }
      if (!a.dlogits) continue;
      const float slope = terms.slope * grad;
      if (slope == 0.0f) {
        zeros();
        continue;
      }
      const f32x2 by = Splat2(factor(own, q.mk) * (-slope / q.s));
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        const uint32_t u = t + i * threads;
        if (u >= w.count) continue;
        float v[kPerUnit<T>];
#pragma unroll
        for (int j = 0; j < kPairs<T>; ++j) UnpackF2(Mul2(e[i][j], by), &v[2 * j], &v[2 * j + 1]);
        row.Store(w.first + u, v);
        if (w.first + u == label_unit) row.d[label] = FromF32<T>(slope * (q.others / q.s));
      }
    }
  }
  if (kPolicy && t == 0 && rank == 0)
#pragma unroll
    for (int i = 0; i < 3; ++i) partials[(static_cast<size_t>(cluster) * groups + group) * 3 + i] = total[i];
}

// Rows that no cluster holds in its registers, read twice: a block to a row.
template <typename T, bool kPolicy>
__global__ void __launch_bounds__(kThreads)
LogitWideKernel(const __grid_constant__ LogitArgs a, const __grid_constant__ PolicyArgs p, const Sequences seq, float4* __restrict__ kept,
                double* __restrict__ partials) {
  AwaitPrevious();
  __shared__ Part slots[2][kThreads / 32];
  const float grad = (kPolicy && p.loss_grad ? *p.loss_grad : 1.0f) * a.scale;
  double sums[3] = {};
  uint32_t turn = 0;
  for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const Row<T> row(a, r);
    const int32_t label = a.labels[r];
    if (!kPolicy && (static_cast<int64_t>(r) < seq.starts[0] || static_cast<int64_t>(r) >= seq.starts[seq.count])) continue;
    if (!Counts(label, a.classes)) {
      if (!kPolicy) continue;
      if (threadIdx.x == 0) p.logp[r] = 0.0f;
      if (a.dlogits) Zeros(row);
      continue;
    }
    const RowSums q = SumsOf(row, label, a.k, slots[turn]);
    turn ^= 1;
    if (!kPolicy) {
      if (threadIdx.x == 0) kept[r] = make_float4(q.z_label, q.mk, q.others, q.s);
      continue;
    }
    const double logp = LogpOf(a, q);
    const PolicyTerms t = PolicyOf(p, PolicyRowOf(p, r), logp);
    if (threadIdx.x == 0) {
      p.logp[r] = static_cast<float>(logp);
      sums[0] += t.loss;
      sums[1] += t.kl;
      sums[2] += t.clipped;
    }
    if (!a.dlogits) continue;
    const float slope = t.slope * grad;
    if (slope == 0.0f) Zeros(row);
    else Gradient(row, label, a.k, q.mk, q.others, q.s, slope);
  }
  if (kPolicy && threadIdx.x == 0)
    for (int i = 0; i < 3; ++i) partials[blockIdx.x * 3 + i] = sums[i];
}

// ---- the preference loss ----------------------------------------------------------------------------------
// log(1 + e^x), exact in its tails.
__device__ __forceinline__ double Softplus(double x) { return x > 0.0 ? x + log1p(exp(-x)) : log1p(exp(x)); }

constexpr uint32_t kPairThreads = 256;

// A pair to a block: the first four warps sum the chosen rows, the others the rejected ones.  Then each row's kept.x becomes the
// loss's derivative by its logp, logit_scale and loss_grad included, 0 where it does not count.  losses [pairs]: added up by PreferenceFoldKernel.
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
    for (int64_t r = begin + t; r < end; r += kPairThreads / 2)
      if (Counts(a.labels[r], a.classes)) {
        const float4 q = kept[r];
        sum += LogpOf(a, {q.x, q.y, q.z, q.w});
        counted += 1.0;
      }
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
      const uint32_t w = i * (kPairThreads / 64);
      sum = (sums[w][0] + sums[w + 1][0]) + (sums[w + 2][0] + sums[w + 3][0]);
      counted = (sums[w][1] + sums[w + 1][1]) + (sums[w + 2][1] + sums[w + 3][1]);
      per_row[i] = p.average && counted > 0.0 ? 1.0 / counted : 1.0;
      sum *= per_row[i];
      if (threadIdx.x == 0) p.sequence_logp[2 * pair + i] = static_cast<float>(sum);
      ratio[i] = sum - (p.ref_logp ? static_cast<double>(p.ref_logp[2 * pair + i]) : 0.0);
    }
    const double beta = p.beta, h = beta * (ratio[0] - ratio[1]) - static_cast<double>(p.margin), smoothing = p.smoothing;
    double slope, loss;
    if (p.kind == SEE_PREFERENCE_SIGMOID) {
      loss = (1.0 - smoothing) * Softplus(-h) + smoothing * Softplus(h);
      slope = smoothing - 1.0 / (1.0 + exp(h));
    } else if (p.kind == SEE_PREFERENCE_HINGE) {
      loss = h >= 1.0 ? 0.0 : 1.0 - h;
      slope = h >= 1.0 ? 0.0 : h < 1.0 ? -1.0 : h;   // (NaN stays)
    } else {
      const double off = (h - 0.5) / beta;
      loss = off * off;
      slope = 2.0 * off / beta;
    }
    if (threadIdx.x == 0) {
      p.margins[pair] = static_cast<float>(h);
      p.losses[pair] = loss;
    }
    if (!a.dlogits) continue;
    const double each = slope * beta / static_cast<double>(p.pairs);
    const float of_row = static_cast<float>((side ? -each * per_row[1] : each * per_row[0]) * static_cast<double>(grad));
    for (int64_t r = begin + t; r < end; r += kPairThreads / 2) kept[r].x = Counts(a.labels[r], a.classes) ? of_row : 0.0f;
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
  const float k = a.k;
  for (int64_t r = end - 1 - (static_cast<int64_t>(blockIdx.x) * side_by_side + warp / warps); r >= begin;
       r -= static_cast<int64_t>(gridDim.x) * side_by_side) {
    const float4 q = kept[r];
    const int32_t label = a.labels[r];
    const Row<T> row(a, r);
    const bool counts = Counts(label, a.classes);   // (what is kept of other rows is not set)
    const float slope = counts ? q.x : 0.0f, by = -slope / q.w, mk = q.y;
    const uint32_t label_unit = counts ? (static_cast<uint32_t>(label) + row.skip) / kPerUnit<T> : ~0u;
    for (uint32_t u0 = (warp % warps) * 32 * kGradUnits + lane; u0 < row.units; u0 += warps * 32 * kGradUnits) {
      uint4 raw[kGradUnits];
      if (slope != 0.0f) {
#pragma unroll
        for (int i = 0; i < kGradUnits; ++i)
          if (u0 + i * 32 < row.units) raw[i] = row.Raw(u0 + i * 32);
      }
#pragma unroll
      for (int i = 0; i < kGradUnits; ++i) {
        const uint32_t u = u0 + i * 32;
        if (u >= row.units) break;
        float v[kPerUnit<T>];
        if (slope == 0.0f) {
#pragma unroll
          for (int j = 0; j < kPerUnit<T>; ++j) v[j] = 0.0f;
        } else {
          Elements<T>(raw[i], v);
#pragma unroll
          for (int j = 0; j < kPerUnit<T>; ++j) v[j] = by * Ex2Approx(fmaf(v[j], k, -mk));
        }
        row.Store(u, v);
        if (u == label_unit) row.d[label] = FromF32<T>(slope == 0.0f ? 0.0f : slope * (q.z / q.w));
      }
    }
  }
}

// ---- launches ------------------------------------------------------------------------------------------------
// How rows are shared: T threads and `blocks` blocks of a cluster to a row, `part` units to a block, `units` of them to a thread.
struct Sharing {
  uint32_t T, units, blocks, part, groups, slots, clusters;
  size_t bytes;
};
template <typename T>
bool ShareRows(const LogitArgs& a, uint32_t sms, Sharing* out) {
  constexpr uint32_t kMostUnits = 64 / kPerUnit<T>;   // to a thread: 64 elements
  const uint32_t all = (a.classes + 2 * (kPerUnit<T> - 1)) / kPerUnit<T>;   // units, wherever a row begins
  uint32_t blocks = 1;
  while (blocks < 8 && ((all + blocks - 1) / blocks > kThreads * kMostUnits || (all + blocks - 1) / blocks * 32 > kMostShared - 2048)) blocks *= 2;
  // Few rows are shared by more blocks, down to a kilobyte each.
  while (blocks < 8 && a.rows * blocks * 2 <= sms && all / blocks > 128) blocks *= 2;
  const uint32_t part = (all + blocks - 1) / blocks;
  if (part > kThreads * kMostUnits) return false;
  uint32_t units = kMostUnits;
  if (a.rows * blocks <= sms) {   // a row to an SM: spread it over its threads
    units = 1;
    while (part > kThreads * units) units *= 2;
  }
  while (units > 1 && part <= 32 * (units / 2)) units /= 2;   // (a warp's row)
  Sharing s;
  s.T = (((part + units - 1) / units) + 31) / 32 * 32;
  s.units = units;
  s.blocks = blocks;
  s.part = part;
  s.groups = blocks > 1 ? 1 : kThreads / s.T;
  const uint64_t each = (a.rows + sms - 1) / sms;
  if (s.groups > each) s.groups = static_cast<uint32_t>(each);
  const size_t slot = static_cast<size_t>(part) * 16, budget = kMostShared - 2048;
  while (s.groups > 1 && 2 * s.groups * slot > budget) --s.groups;
  s.slots = static_cast<uint32_t>(budget / (s.groups * (slot + 8)));
  s.slots = s.slots < 1 ? 1 : s.slots > 8 ? 8 : s.slots;
  const uint64_t wanted = (a.rows + s.groups - 1) / s.groups, most = sms / blocks;
  s.clusters = static_cast<uint32_t>(wanted < most ? wanted : most);
  const uint64_t turns = (wanted + s.clusters - 1) / s.clusters;
  if (s.slots > turns) s.slots = static_cast<uint32_t>(turns);
  s.bytes = s.groups * s.slots * (slot + 8);
  *out = s;
  return true;
}

template <typename T, int NU, bool kPolicy, bool kCluster>
cudaError_t RunRows(const LogitArgs& a, const PolicyArgs& p, const Sequences& seq, float4* kept, double* partials, const Sharing& w, cudaStream_t s) {
  constexpr auto* kernel = LogitRowsKernel<T, NU, kPolicy, kCluster>;
  if (cudaError_t e = AllowShared<kernel>(w.bytes); e != cudaSuccess) return e;
  return Next(kernel, w.clusters * w.blocks, w.groups * w.T, w.bytes, s, w.blocks)(a, p, seq, kept, partials, w.T, w.slots, w.blocks, w.part);
}
template <typename T, bool kPolicy, bool kCluster>
cudaError_t RunRows(const LogitArgs& a, const PolicyArgs& p, const Sequences& seq, float4* kept, double* partials, const Sharing& w, cudaStream_t s) {
  switch (w.units) {
    case 1: return RunRows<T, 1, kPolicy, kCluster>(a, p, seq, kept, partials, w, s);
    case 2: return RunRows<T, 2, kPolicy, kCluster>(a, p, seq, kept, partials, w, s);
    case 4: return RunRows<T, 4, kPolicy, kCluster>(a, p, seq, kept, partials, w, s);
    case 8: return RunRows<T, 8, kPolicy, kCluster>(a, p, seq, kept, partials, w, s);
    default:
      if constexpr (sizeof(T) == 4) return RunRows<T, 16, kPolicy, kCluster>(a, p, seq, kept, partials, w, s);
      return cudaErrorInvalidValue;
  }
}
// The rows' pass; *count: partial sums of the policy loss.
template <typename T, bool kPolicy>
cudaError_t RunRows(const LogitArgs& a, const PolicyArgs& p, const Sequences& seq, float4* kept, double* partials, uint32_t sms, cudaStream_t s,
                    uint32_t* count) {
  Sharing w;
  if (ShareRows<T>(a, sms, &w)) {
    *count = w.clusters * w.groups;
    return w.blocks > 1 ? RunRows<T, kPolicy, true>(a, p, seq, kept, partials, w, s) : RunRows<T, kPolicy, false>(a, p, seq, kept, partials, w, s);
  }
  *count = static_cast<uint32_t>(a.rows < 4 * sms ? a.rows : 4 * sms);
  return Next(LogitWideKernel<T, kPolicy>, *count, kThreads, 0, s)(a, p, seq, kept, partials);
}

template <typename T>
cudaError_t Policy(const LogitArgs& a, const PolicyArgs& p, double* partials, uint32_t sms, cudaStream_t s, int* launches) {
  uint32_t count = 0;
  if (a.rows) {
    if (cudaError_t e = RunRows<T, true>(a, p, {}, nullptr, partials, sms, s, &count); e != cudaSuccess) return e;
    ++*launches;
  }
  ++*launches;
  return Next(PolicyFoldKernel, 1, 96, 0, s)(static_cast<const double*>(partials), count, p.loss);
}

template <typename T>
cudaError_t Preference(const LogitArgs& a, const PreferenceArgs& p, float4* kept, uint32_t sms, cudaStream_t s, int* launches) {
  if (a.rows) {
    uint32_t count;
    if (cudaError_t e = RunRows<T, false>(a, {}, {p.starts, 2 * p.pairs}, kept, nullptr, sms, s, &count); e != cudaSuccess) return e;
    ++*launches;
  }
  if (cudaError_t e = Next(PreferencePairsKernel, p.pairs < 4 * sms ? p.pairs : 4 * sms, kPairThreads, 0, s)(a, p, kept); e != cudaSuccess) return e;
  *launches += 2;
  if (!a.dlogits) return Next(PreferenceFoldKernel, 1, 256, 0, s)(p);
  const uint32_t pieces = (a.classes / kPerUnit<T> + 32 * kGradUnits) / (32 * kGradUnits);
  const uint32_t warps = pieces >= 8 ? 8 : pieces >= 4 ? 4 : pieces >= 2 ? 2 : 1, rows_a_block = kGradThreads / 32 / warps;
  const uint64_t blocks = (a.rows + rows_a_block - 1) / rows_a_block, most = 6ull * sms;
  return Next(PreferenceGradientKernel<T>, static_cast<unsigned>(blocks < most ? blocks : most), kGradThreads, 0, s)(
      a, p, static_cast<const float4*>(kept), warps);
}

}  // namespace

cudaError_t PolicyLoss(const LogitArgs& a, int type, const PolicyArgs& p, double* partials, uint32_t sms, cudaStream_t s, int* launches) {
  if (type == SEE_F32) return Policy<float>(a, p, partials, sms, s, launches);
  return type == SEE_BF16 ? Policy<Bf16>(a, p, partials, sms, s, launches) : Policy<F16>(a, p, partials, sms, s, launches);
}
cudaError_t PreferenceLoss(const LogitArgs& a, int type, const PreferenceArgs& p, float4* kept, uint32_t sms, cudaStream_t s, int* launches) {
  if (type == SEE_F32) return Preference<float>(a, p, kept, sms, s, launches);
  return type == SEE_BF16 ? Preference<Bf16>(a, p, kept, sms, s, launches) : Preference<F16>(a, p, kept, sms, s, launches);
}

}  // namespace see::k
