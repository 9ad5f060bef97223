// Host side of the gated feed-forward block: what a call refuses, the tensor maps of its operands, and the choice of tiles.
#include <algorithm>
#include <atomic>

#include "block_checks.h"
#include "cuda_backend.h"
#include "gated_umma.h"

namespace see {
namespace {

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                              CUtensorMapFloatOOBfill);

EncodeFn Encoder() {
  static const EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found{};
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found);
    return e == cudaSuccess && found == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeFn>(p) : nullptr;
  }();
  return fn;
}

// A row-major 16-bit matrix in boxes of box_rows x 64 elements under the 128-byte swizzle.
bool MapOf(CUtensorMap* map, bool f16, const void* base, uint64_t rows, uint64_t cols, uint64_t stride, uint32_t box_rows) {
  const cuuint64_t dims[2] = {cols, rows}, strides[1] = {stride * 2};
  const cuuint32_t box[2] = {64, box_rows}, elem[2] = {1, 1};
  return Encoder()(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides,
                   box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

uint32_t Up(uint64_t n, uint64_t by) { return static_cast<uint32_t>((n + by - 1) / by); }

Status CheckGated(const char* what, see_gated_shape* s) {
  if (s->type != SEE_BF16 && s->type != SEE_F16) return std::unexpected(std::string(what) + ": the type is bf16 or f16");
  if (s->act != SEE_ACT_RELU && s->act != SEE_ACT_GELU && s->act != SEE_ACT_SILU) return std::unexpected(std::string(what) + ": unknown activation");
  if (s->d_in == 0 || s->d_hidden == 0 || s->d_in % 8 || s->d_hidden % 8 || s->d_in > (1u << 20) || s->d_hidden > (1u << 20))
    return std::unexpected(std::string(what) + ": d_in and d_hidden are multiples of 8 from 8 to 2^20");
  if (s->rows > 0x7FFFFF00ull) return std::unexpected(std::string(what) + ": more than 2^31 - 256 rows");
  if (s->x_stride == 0) s->x_stride = s->d_in;
  if (s->hidden_stride == 0) s->hidden_stride = s->d_hidden;
  if (s->x_stride < s->d_in || s->hidden_stride < s->d_hidden || s->x_stride % 8 || s->hidden_stride % 8 || s->x_stride > (1ull << 36) ||
      s->hidden_stride > (1ull << 36))
    return std::unexpected(std::string(what) + ": a stride is smaller than a row, not a multiple of 8, or over 2^36");
  // (the tiles of any product are numbered in 32 bits)
  if ((s->rows / 256 + 1) * (s->d_hidden / 64 + 1) > 0x7FFFFFFFull || (s->rows / 256 + 1) * (s->d_in / 128 + 1) > 0x7FFFFFFFull)
    return std::unexpected(std::string(what) + ": too many rows for these widths");
  return {};
}

uint64_t SlopeBytes(uint64_t rows, uint64_t d_hidden) { return (rows * d_hidden * 2 + 127) / 128 * 128; }

// The backward pass's problems on `pairs` CTA pairs, which take the tiles, then the parts of cut ones, in turn.  A tile's
// reduction is cut into parts of up to `length` blocks where that ends the launch sooner: the tiles of the last, unfull round;
// or all of dx's (few rows leave it few tiles with the longest reduction); or all.  By estimate, in blocks (about 0.28 us): a
// tile costs two besides its own, a part five, for its sums' way to memory, the fold eight and a third for each part.
// 4096 x 768 x 2048 59 us / 54 in a graph (63 to 65 called one by one); 16 rows of it 25 / 15; 600 x 512 x 1376 21 / 16.
constexpr uint32_t kMostPairs = 74, kMostParts = 2 * kMostPairs;
struct Cut { uint32_t whole, parts, first_part; };
struct BackwardPlan {
  Cut cut[k::kGatedProblems] = {};
  uint32_t parts = 0;   // in all
};
struct Run { uint64_t count; double cost; };
// The time of the pair that ends last: it changes from pair to pair only where a run of equal items begins or ends.
double Longest(const Run* runs, uint32_t count, uint32_t pairs) {
  uint32_t begin[2 * k::kGatedProblems], rest[2 * k::kGatedProblems];   // of a run: its first pair, items behind full rounds
  double full = 0.0, longest = 0.0;
  uint64_t first = 0;
  for (uint32_t r = 0; r < count; first += runs[r++].count) {
    const uint64_t rounds = runs[r].count / pairs;
    begin[r] = static_cast<uint32_t>(first % pairs);
    rest[r] = static_cast<uint32_t>(runs[r].count - rounds * pairs);
    full += static_cast<double>(rounds) * runs[r].cost;
  }
  for (uint32_t i = 0; i < 2 * count; ++i) {
    uint32_t pair = begin[i / 2] + (i & 1 ? rest[i / 2] + pairs - 1 : 0);
    while (pair >= pairs) pair -= pairs;
    double time = full;
    for (uint32_t r = 0; r < count; ++r) {
      const uint32_t behind = pair >= begin[r] ? pair - begin[r] : pair + pairs - begin[r];
      if (behind < rest[r]) time += runs[r].cost;
    }
    longest = std::max(longest, time);
  }
  return longest;
}
BackwardPlan PlanCuts(const uint64_t* tiles, const uint64_t* blocks, uint32_t count, uint32_t pairs, uint32_t most_parts) {
  uint64_t total = 0, longest = 0;
  for (uint32_t i = 0; i < count; ++i) {
    total += tiles[i];
    longest = std::max(longest, blocks[i]);
  }
  BackwardPlan best;
  double best_time = 1e300;
  enum { kLastRound, kFirst, kAll };
  for (int which : {kLastRound, kFirst, kAll})
    for (uint64_t cuts : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
      const uint64_t length = (longest + cuts - 1) / cuts;
      if (cuts > 1 && length < 6) break;
      BackwardPlan plan;
      Run runs[2 * k::kGatedProblems];
      uint64_t full = which == kLastRound ? total / pairs * pairs : 0, parts = 0;
      for (uint32_t i = 0; i < count; ++i) {
        uint64_t whole = which == kLastRound ? std::min(tiles[i], full) : which == kFirst && i > 0 ? tiles[i] : 0;
        full -= std::min(full, whole);
        const uint64_t each = (blocks[i] + length - 1) / length;
        if (each <= 1) whole = tiles[i];
        plan.cut[i] = {static_cast<uint32_t>(whole), static_cast<uint32_t>(std::max<uint64_t>(1, each)), static_cast<uint32_t>(std::min<uint64_t>(parts, kMostParts))};
        runs[i] = {whole, static_cast<double>(blocks[i]) + 2.0};
        runs[count + i] = {(tiles[i] - whole) * each, static_cast<double>(blocks[i]) / static_cast<double>(std::max<uint64_t>(1, each)) + 5.0};
        parts += runs[count + i].count;
      }
      if (parts > most_parts) continue;
      plan.parts = static_cast<uint32_t>(parts);
      const double time = Longest(runs, 2 * count, pairs) + (parts ? 8.0 + 0.3 * static_cast<double>(parts) : 0.0);
      if (time < best_time) {
        best_time = time;
        best = plan;
      }
    }
  return best;
}
BackwardPlan PlanOn(uint32_t pairs, uint32_t most_parts, uint64_t rows, uint64_t d_in, uint64_t d_hidden, bool dx, bool dw) {
  uint64_t tiles[3], blocks[3];
  uint32_t count = 0;
  if (dx) {
    tiles[count] = static_cast<uint64_t>(Up(rows, 256)) * Up(d_in, 256);
    blocks[count++] = 2ull * Up(d_hidden, 64);
  }
  for (int which = 0; which < 2 && dw; ++which) {
    tiles[count] = static_cast<uint64_t>(Up(d_in, 256)) * Up(d_hidden, 256);
    blocks[count++] = Up(rows, 64);
  }
  return PlanCuts(tiles, blocks, count, pairs, most_parts);
}
// The parts that a workspace has room for, whichever gradients are wanted: what 148 SMs take.  (Another number of pairs ends its
// rounds elsewhere, and might do with more.)
uint32_t PartsReserved(uint64_t rows, uint64_t d_in, uint64_t d_hidden) {
  uint32_t parts = 0;
  for (int want = 1; want < 4; ++want) parts = std::max(parts, PlanOn(kMostPairs, kMostParts, rows, d_in, d_hidden, want & 1, want & 2).parts);
  return parts;
}
BackwardPlan PlanBackward(uint64_t rows, uint64_t d_in, uint64_t d_hidden, bool dx, bool dw, uint32_t pairs) {
  const uint32_t most = pairs == kMostPairs ? kMostParts : PartsReserved(rows, d_in, d_hidden);
  return PlanOn(pairs, most, rows, d_in, d_hidden, dx, dw);
}
uint64_t PartialBytes(uint32_t parts) { return parts * 256ull * 256 * 4; }
uint32_t PairsOf(uint32_t sms) { return std::min(sms / 2, kMostPairs); }

}  // namespace

uint64_t GatedBackwardWorkspace(uint64_t rows, uint64_t d_in, uint64_t d_hidden) {
  if (d_in == 0 || d_hidden == 0 || d_in % 8 || d_hidden % 8 || d_in > (1u << 20) || d_hidden > (1u << 20) || rows > 0x7FFFFF00ull) return 0;
  if (rows == 0) return 128;
  return 2 * SlopeBytes(rows, d_hidden) + PartialBytes(PartsReserved(rows, d_in, d_hidden));
}

uint64_t GatedBackwardUses(uint64_t rows, uint64_t d_in, uint64_t d_hidden, bool dx, bool dw, uint32_t sms) {
  return 2 * SlopeBytes(rows, d_hidden) + PartialBytes(PlanBackward(rows, d_in, d_hidden, dx, dw, PairsOf(sms)).parts);
}

Status CheckGatedForward(see_gated_shape* shape, const void* x, const void* w_gate, const void* w_up, const void* hidden, const void* gate,
                         const void* up) {
  const char* const what = "cuda: gated forward";
  if (auto r = CheckGated(what, shape); !r) return r;
  const see_gated_shape& s = *shape;
  if (!gate != !up) return std::unexpected(std::string(what) + ": gate and up are kept together or not at all");
  const uint64_t weights = s.d_in * s.d_hidden * 2, width = s.d_hidden * 2, pitch = s.hidden_stride * 2;
  Operands ops = {{"x", x, s.rows, s.d_in * 2, s.x_stride * 2, 16, false},
                              Vector("w_gate", w_gate, weights, 16, false),
                              Vector("w_up", w_up, weights, 16, false),
                              {"hidden", hidden, s.rows, width, pitch, 16, true}};
  if (gate) {
    ops.Add({"gate", gate, s.rows, width, pitch, 16, true});
    ops.Add({"up", up, s.rows, width, pitch, 16, true});
  }
  return ops.Check(what);
}

Status CheckGatedBackward(see_gated_shape* shape, const void* dhidden, const void* x, const void* w_gate, const void* w_up,
                          const void* gate, const void* up, const void* dx, const void* dw_gate, const void* dw_up, const void* workspace,
                          uint64_t workspace_bytes) {
  const char* const what = "cuda: gated backward";
  if (auto r = CheckGated(what, shape); !r) return r;
  const see_gated_shape& s = *shape;
  if (!dw_gate != !dw_up) return std::unexpected(std::string(what) + ": dw_gate and dw_up are wanted together or not at all");
  if (!dx && !dw_gate) return std::unexpected(std::string(what) + ": no output is wanted");
  if (workspace_bytes < std::max<uint64_t>(128, 2 * SlopeBytes(s.rows, s.d_hidden))) return std::unexpected(std::string(what) + ": the workspace is too small");
  const uint64_t weights = s.d_in * s.d_hidden * 2, width = s.d_hidden * 2, pitch = s.hidden_stride * 2;
  Operands ops = {{"dhidden", dhidden, s.rows, width, pitch, 16, false},
                              {"x", x, s.rows, s.d_in * 2, s.x_stride * 2, 16, false},
                              Vector("w_gate", w_gate, weights, 16, false),
                              Vector("w_up", w_up, weights, 16, false),
                              {"gate", gate, s.rows, width, pitch, 16, false},
                              {"up", up, s.rows, width, pitch, 16, false},
                              Vector("workspace", workspace, workspace_bytes, 128, true)};
  if (dx) ops.Add({"dx", dx, s.rows, s.d_in * 2, s.x_stride * 2, 16, true});
  if (dw_gate) {
    ops.Add(Vector("dw_gate", dw_gate, weights, 16, true));
    ops.Add(Vector("dw_up", dw_up, weights, 16, true));
  }
  return ops.Check(what);
}

Status CudaBackend::GatedForward(const see_gated_shape& given, const void* x, const void* w_gate, const void* w_up, void* hidden, void* gate,
                                 void* up) {
  see_gated_shape s = given;
  if (auto r = CheckGatedForward(&s, x, w_gate, w_up, hidden, gate, up); !r) return r;
  if (s.rows == 0) return {};
  OnDevice on(device_);
  if (!on.ok()) return Check(cudaGetLastError(), "gated forward: device");
  if (k::GatedTokenTakes(s.rows, s.d_in)) {
    const k::GatedTokenArgs a = {x, w_gate, w_up, hidden, gate, up, static_cast<uint32_t>(s.d_in), static_cast<uint32_t>(s.d_hidden), s.act};
    if (auto r = Check(k::GatedToken(a, s.type == SEE_F16, sms_, stream_), "gated forward"); !r) return r;
    ++counters_.kernel_launches;
    return {};
  }
  if (!Encoder()) return std::unexpected("cuda: gated forward: the driver does not provide cuTensorMapEncodeTiled");
  const bool f16 = s.type == SEE_F16;
  k::GatedLaunch l = {};
  k::GatedProblem& p = l.p[0];
  // A pair's accumulator of 128 columns instead of 256 costs nearly as much a block of the reduction (A is read as often), so
  // it pays only where one round takes the twice as many tiles.  In a graph, us, 256 columns / 128: 600 x 512 x 1376 (66 such
  // tiles) 9.8 / 9.6, 1024 x 2048 x 1152 (72) 16.9 / 16.4, 600 x 768 x 2048 (96) 13.0 / 14.4, 1024 x 512 x 1376 (88) 11.8 / 12.8;
  // where 256 columns begin a second round that 128 do not make longer, the rule errs: 1024 x 2048 x 2368 (148) 30.4 / 26.7.
  const uint32_t tn = static_cast<uint64_t>(Up(s.rows, 256)) * Up(s.d_hidden, 64) <= sms_ / 2 ? 128 : 256;
  bool ok = MapOf(&p.a[0], f16, x, s.rows, s.d_in, s.x_stride, 64) && MapOf(&p.b[0], f16, w_gate, s.d_in, s.d_hidden, s.d_hidden, 64) &&
            MapOf(&p.b[1], f16, w_up, s.d_in, s.d_hidden, s.d_hidden, 64) && MapOf(&p.c, f16, hidden, s.rows, s.d_hidden, s.hidden_stride, 32);
  if (gate)
    ok = ok && MapOf(&l.gate, f16, gate, s.rows, s.d_hidden, s.hidden_stride, 32) && MapOf(&l.up, f16, up, s.rows, s.d_hidden, s.hidden_stride, 32);
  if (!ok) return std::unexpected("cuda: gated forward: cuTensorMapEncodeTiled refused an operand layout");
  p.M = static_cast<uint32_t>(s.rows);
  p.N = static_cast<uint32_t>(s.d_hidden);
  p.blocks[0] = Up(s.d_in, 64);
  p.b_mn = 1;
  p.tiles_m = Up(s.rows, 256);
  p.tiles_n = Up(s.d_hidden, tn / 2);
  p.whole = p.tiles_m * p.tiles_n;
  p.parts = 1;
  l.count = 1;
  l.f16 = f16;
  l.act = s.act;
  l.keep = gate != nullptr;
  l.status = d_status_;
  if (auto r = Check(k::GatedProducts(l, true, tn, sms_, stream_), "gated forward"); !r) return r;
  ++counters_.kernel_launches;
  return {};
}

Status CudaBackend::GatedBackward(const see_gated_shape& given, const void* dhidden, const void* x, const void* w_gate, const void* w_up,
                                  const void* gate, const void* up, void* dx, void* dw_gate, void* dw_up, void* workspace,
                                  uint64_t workspace_bytes) {
  see_gated_shape s = given;
  if (auto r = CheckGatedBackward(&s, dhidden, x, w_gate, w_up, gate, up, dx, dw_gate, dw_up, workspace, workspace_bytes); !r) return r;
  OnDevice on(device_);
  if (!on.ok()) return Check(cudaGetLastError(), "gated backward: device");
  const uint64_t weights = s.d_in * s.d_hidden * 2;
  if (s.rows == 0) {
    for (void* w : {dw_gate, dw_up})
      if (w)
        if (auto r = Check(cudaMemsetAsync(w, 0, weights, stream_), "gated backward"); !r) return r;
    return {};
  }
  if (!Encoder()) return std::unexpected("cuda: gated backward: the driver does not provide cuTensorMapEncodeTiled");
  const bool f16 = s.type == SEE_F16;
  void* dg = workspace;
  void* du = static_cast<uint8_t*>(workspace) + SlopeBytes(s.rows, s.d_hidden);
  k::GatedLaunch l = {};
  l.f16 = f16;
  l.status = d_status_;
  const uint32_t rows = static_cast<uint32_t>(s.rows), d_in = static_cast<uint32_t>(s.d_in), d_hidden = static_cast<uint32_t>(s.d_hidden);
  const uint32_t pairs = PairsOf(sms_);
  const BackwardPlan plan = PlanBackward(s.rows, s.d_in, s.d_hidden, dx != nullptr, dw_gate != nullptr, pairs);
  if (2 * SlopeBytes(s.rows, s.d_hidden) + PartialBytes(plan.parts) > workspace_bytes)
    return std::unexpected("cuda: gated backward: the workspace is too small");
  l.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + 2 * SlopeBytes(s.rows, s.d_hidden));
  auto problem = [&](uint32_t M, uint32_t N, void* out, uint64_t out_stride) -> k::GatedProblem& {
    const Cut& cut = plan.cut[l.count];
    k::GatedProblem& p = l.p[l.count++];
    p.M = M;
    p.N = N;
    p.tiles_m = Up(M, 256);
    p.tiles_n = Up(N, 256);
    p.whole = cut.whole;
    p.parts = cut.parts;
    p.first_part = cut.first_part;
    p.out = out;
    p.out_stride = out_stride;
    return p;
  };
  bool ok = true;
  if (dx) {   // A: dg, then du, along their rows; B: the weights' rows are dx's columns
    k::GatedProblem& p = problem(rows, d_in, dx, s.x_stride);
    p.blocks[0] = p.blocks[1] = Up(d_hidden, 64);
    ok = MapOf(&p.a[0], f16, dg, rows, d_hidden, d_hidden, 64) && MapOf(&p.a[1], f16, du, rows, d_hidden, d_hidden, 64) &&
         MapOf(&p.b[0], f16, w_gate, d_in, d_hidden, d_hidden, 64) && MapOf(&p.b[1], f16, w_up, d_in, d_hidden, d_hidden, 64) &&
         MapOf(&p.c, f16, dx, rows, d_in, s.x_stride, 32);
  }
  for (int which = 0; which < 2 && dw_gate && ok; ++which) {   // both operands down their columns
    k::GatedProblem& p = problem(d_in, d_hidden, which ? dw_up : dw_gate, d_hidden);
    p.a_mn = p.b_mn = 1;
    p.blocks[0] = Up(rows, 64);
    ok = MapOf(&p.a[0], f16, x, rows, d_in, s.x_stride, 64) && MapOf(&p.b[0], f16, which ? du : dg, rows, d_hidden, d_hidden, 64) &&
         MapOf(&p.c, f16, which ? dw_up : dw_gate, d_in, d_hidden, d_hidden, 32);
  }
  if (!ok) return std::unexpected("cuda: gated backward: cuTensorMapEncodeTiled refused an operand layout");
  if (auto r = Check(k::GatedSlopes(dhidden, gate, up, dg, du, s.rows, d_hidden, s.hidden_stride, s.act, f16, sms_, stream_), "gated backward"); !r)
    return r;
  ++counters_.kernel_launches;
  if (auto r = Check(k::GatedProducts(l, false, 256, 2 * pairs, stream_), "gated backward"); !r) return r;
  ++counters_.kernel_launches;
  if (plan.parts) {
    if (auto r = Check(k::GatedFold(l, stream_), "gated backward"); !r) return r;
    ++counters_.kernel_launches;
  }
  return {};
}

}  // namespace see
