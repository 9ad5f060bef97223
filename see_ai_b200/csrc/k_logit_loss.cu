// Losses over rows of logits: the labels' log-probabilities, a clipped policy loss or a preference loss of them, and the
// gradient of the logits.  With z = logit_scale logits, M its maximum and l the label, a row is
//   e_c = 2^(k logit_c - k M),  k = logit_scale / ln 2,   others = sum of e_c over c != l,   s = others + e_l,
//   logp = (z_l - M) - log s, or -log1p(others / e_l) where the label holds more than half (no digits are lost next to 0),
//   dlogit_c = -slope logit_scale e_c / s,  of the label  slope logit_scale others / s   (not 1 - p, which would lose them),
// slope being the loss's derivative by logp.  The product k M is rounded once and the same in every exponent of a row, so that its
// rounding cancels between e_c and s.  Bound by HBM: logits are read once, dlogits written once.
//
// A row is walked in units of 16 bytes by address, of which the first and the last may stick out of it, whatever its alignment.
#include <type_traits>

#include "act_expr.cuh"
#include "block_ops.h"
#include "launch.cuh"
#include "vec_types.cuh"

namespace see::k {

namespace {

constexpr uint32_t kThreads = 512;
constexpr float kLn2 = 0.6931471805599453f;
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
  __device__ __forceinline__ void Load(uint32_t unit, float* v) const {   // -inf where it sticks out
    const int32_t at = At(unit);
    if (Whole(at)) {
      Elements<T>(*reinterpret_cast<const uint4*>(z + at), v);
      return;
    }
#pragma unroll
    for (int j = 0; j < kPerUnit<T>; ++j) v[j] = at + j >= 0 && at + j < static_cast<int32_t>(classes) ? ToF32(z[at + j]) : MinusInf();
  }
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

// Of a row: k M, the sum over the others, the sum over all and logp.
struct RowSums {
  float mk, others, s, logp;
};
__device__ __forceinline__ RowSums Finish(const Part& p, float z_label, float k) {
  const float x = fmaf(z_label, k, -p.mk), e = Ex2Approx(x), s = p.sum + e;
  return {p.mk, p.sum, s, p.sum < e ? -log1pf(p.sum / e) : x * kLn2 - logf(s)};
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
  return Finish(WarpJoin(p), z_label, k);
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
struct PolicyTerms {
  float slope, loss, kl, clipped;   // slope: of the weighted loss by logp
};
__device__ __forceinline__ PolicyTerms PolicyOf(const PolicyArgs& p, uint64_t row, float logp) {
  const float a = p.advantages[row], w = p.weights ? p.weights[row] : 1.0f;
  const float r = expf(logp - p.old_logp[row]), cut = r < 1.0f - p.clip_low ? 1.0f - p.clip_low : r > 1.0f + p.clip_high ? 1.0f + p.clip_high : r;
  const bool clipped = r * a > cut * a;
  float loss = clipped ? -(cut * a) : -(r * a), slope = clipped ? 0.0f : -(r * a), kl = 0.0f;
  if (p.ref_logp) {
    const float x = p.ref_logp[row] - logp, grown = expm1f(x);
    kl = grown - x;
    loss += p.kl_coef * kl;
    slope -= p.kl_coef * grown;
  }
  return {w * slope, w * loss, w * kl, clipped ? w : 0.0f};
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
PolicyKernel(const __grid_constant__ LogitArgs a, const __grid_constant__ PolicyArgs p, double* __restrict__ partials) {
  AwaitPrevious();
  __shared__ Part slots[2][kThreads / 32];
  const float grad = (p.loss_grad ? *p.loss_grad : 1.0f) * a.scale;
  double sums[3] = {};
  uint32_t turn = 0;
  for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const Row<T> row(a, r);
    const int32_t label = a.labels[r];
    if (!Counts(label, a.classes)) {
      if (threadIdx.x == 0) p.logp[r] = 0.0f;
      if (a.dlogits) Zeros(row);
      continue;
    }
    const RowSums q = SumsOf(row, label, a.k, slots[turn]);
    turn ^= 1;
    const PolicyTerms t = PolicyOf(p, r, q.logp);
    if (threadIdx.x == 0) {
      p.logp[r] = q.logp;
      sums[0] += t.loss;
      sums[1] += t.kl;
      sums[2] += t.clipped;
    }
    if (!a.dlogits) continue;
    const float slope = t.slope * grad;
    if (slope == 0.0f) Zeros(row);
    else Gradient(row, label, a.k, q.mk, q.others, q.s, slope);
  }
  if (threadIdx.x == 0)
    for (int i = 0; i < 3; ++i) partials[blockIdx.x * 3 + i] = sums[i];
}

__device__ __forceinline__ double WarpSum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// A warp to each of the three sums.
__global__ void __launch_bounds__(96)
PolicyFoldKernel(const double* __restrict__ partials, uint32_t blocks, float* __restrict__ loss) {
  AwaitPrevious();
  const uint32_t which = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double sum = 0.0;
  for (uint32_t i = lane; i < blocks; i += 32) sum += partials[i * 3 + which];
  sum = WarpSum(sum);
  if (lane == 0) loss[which] = static_cast<float>(sum);
}

// ---- the preference loss ----------------------------------------------------------------------------------
// The sequence of a row: the last one that does not begin behind it.  `count`: none has it.
__device__ __forceinline__ uint32_t SequenceOf(const int32_t* __restrict__ starts, uint32_t count, uint64_t row) {
  const int64_t r = static_cast<int64_t>(row);
  if (r < starts[0] || r >= starts[count]) return count;
  uint32_t lo = 0, hi = count - 1;   // (empty sequences begin where the next one does)
  while (lo < hi) {
    const uint32_t mid = (lo + hi + 1) / 2;
    if (starts[mid] <= r) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
PreferenceRowsKernel(const __grid_constant__ LogitArgs a, const int32_t* __restrict__ starts, uint32_t sequences, float4* __restrict__ kept) {
  AwaitPrevious();
  __shared__ Part slots[2][kThreads / 32];
  uint32_t turn = 0;
  for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const int32_t label = a.labels[r];
    if (!Counts(label, a.classes) || SequenceOf(starts, sequences, r) == sequences) continue;
    const RowSums q = SumsOf(Row<T>(a, r), label, a.k, slots[turn]);
    turn ^= 1;
    if (threadIdx.x == 0) kept[r] = make_float4(q.logp, q.mk, q.others, q.s);
  }
}

// log(1 + e^x), exact in its tails.
__device__ __forceinline__ double Softplus(double x) { return x > 0.0 ? x + log1p(exp(-x)) : log1p(exp(x)); }

// One block: each pair is a warp's.  slopes [2 pairs]: of the loss by the rows' logp of a sequence.
__global__ void __launch_bounds__(1024)
PreferencePairsKernel(const __grid_constant__ PreferenceArgs p, const int32_t* __restrict__ labels, uint64_t rows, uint32_t classes,
                      const float4* __restrict__ kept) {
  AwaitPrevious();
  __shared__ double losses[32];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double loss = 0.0;
  for (uint32_t pair = warp; pair < p.pairs; pair += 32) {
    double ratio[2], per_row[2];
    for (uint32_t side = 0; side < 2; ++side) {
      const uint32_t s = 2 * pair + side;
      const int64_t most = static_cast<int64_t>(rows);
      const int64_t begin = min(max(static_cast<int64_t>(p.starts[s]), static_cast<int64_t>(0)), most);
      const int64_t end = min(static_cast<int64_t>(p.starts[s + 1]), most);
      double sum = 0.0, counted = 0.0;
      for (int64_t r = begin + lane; r < end; r += 32)
        if (Counts(labels[r], classes)) {
          sum += static_cast<double>(kept[r].x);
          counted += 1.0;
        }
      sum = WarpSum(sum);
      counted = WarpSum(counted);
      per_row[side] = p.average && counted > 0.0 ? 1.0 / counted : 1.0;
      sum *= per_row[side];
      if (lane == 0) p.sequence_logp[s] = static_cast<float>(sum);
      ratio[side] = sum - (p.ref_logp ? static_cast<double>(p.ref_logp[s]) : 0.0);
    }
    const double beta = p.beta, h = beta * (ratio[0] - ratio[1]) - static_cast<double>(p.margin), smoothing = p.smoothing;
    double slope;
    if (p.kind == SEE_PREFERENCE_SIGMOID) {
      loss += (1.0 - smoothing) * Softplus(-h) + smoothing * Softplus(h);
      slope = smoothing - 1.0 / (1.0 + exp(h));
    } else if (p.kind == SEE_PREFERENCE_HINGE) {
      loss += h >= 1.0 ? 0.0 : 1.0 - h;
      slope = h >= 1.0 ? 0.0 : h < 1.0 ? -1.0 : h;   // (NaN stays)
    } else {
      const double off = (h - 0.5) / beta;
      loss += off * off;
      slope = 2.0 * off / beta;
    }
    if (lane == 0) {
      p.margins[pair] = static_cast<float>(h);
      const double each = slope * beta / static_cast<double>(p.pairs);
      p.slopes[2 * pair] = static_cast<float>(each * per_row[0]);
      p.slopes[2 * pair + 1] = static_cast<float>(-each * per_row[1]);
    }
  }
  if (lane == 0) losses[warp] = loss;
  __syncthreads();
  if (warp == 0) {
    loss = WarpSum(losses[lane]);
    if (lane == 0) *p.loss = static_cast<float>(loss / static_cast<double>(p.pairs));
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
PreferenceGradientKernel(const __grid_constant__ LogitArgs a, const __grid_constant__ PreferenceArgs p, const float4* __restrict__ kept) {
  AwaitPrevious();
  const float grad = (p.loss_grad ? *p.loss_grad : 1.0f) * a.scale;
  for (uint64_t i = blockIdx.x; i < a.rows; i += gridDim.x) {
    const uint64_t r = a.rows - 1 - i;   // what was read last is in L2
    const uint32_t s = SequenceOf(p.starts, 2 * p.pairs, r);
    if (s == 2 * p.pairs) continue;
    const Row<T> row(a, r);
    const int32_t label = a.labels[r];
    const bool counts = Counts(label, a.classes);
    const float slope = counts ? p.slopes[s] * grad : 0.0f;
    if (slope == 0.0f) {
      Zeros(row);
    } else {
      const float4 q = kept[r];
      Gradient(row, label, a.k, q.y, q.z, q.w, slope);
    }
  }
}

uint32_t Grid(uint64_t rows, uint32_t sms) {
  const uint64_t most = sms * 4 < kLogitPartials ? sms * 4 : kLogitPartials;
  return static_cast<uint32_t>(rows < most ? rows : most);
}

template <typename T>
cudaError_t Policy(const LogitArgs& a, const PolicyArgs& p, double* partials, uint32_t sms, cudaStream_t s, int* launches) {
  const uint32_t grid = Grid(a.rows, sms);
  if (grid) {
    if (cudaError_t e = Next(PolicyKernel<T>, grid, kThreads, 0, s)(a, p, partials); e != cudaSuccess) return e;
    ++*launches;
  }
  ++*launches;
  return Next(PolicyFoldKernel, 1, 96, 0, s)(static_cast<const double*>(partials), grid, p.loss);
}

template <typename T>
cudaError_t Preference(const LogitArgs& a, const PreferenceArgs& p, float4* kept, uint32_t sms, cudaStream_t s, int* launches) {
  const uint32_t grid = Grid(a.rows, sms);
  if (grid) {
    if (cudaError_t e = Next(PreferenceRowsKernel<T>, grid, kThreads, 0, s)(a, p.starts, 2 * p.pairs, kept); e != cudaSuccess) return e;
    ++*launches;
  }
  if (cudaError_t e = Next(PreferencePairsKernel, 1, 1024, 0, s)(p, a.labels, a.rows, a.classes, static_cast<const float4*>(kept)); e != cudaSuccess)
    return e;
  ++*launches;
  if (!grid || !a.dlogits) return cudaSuccess;
  ++*launches;
  return Next(PreferenceGradientKernel<T>, grid, kThreads, 0, s)(a, p, static_cast<const float4*>(kept));
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
