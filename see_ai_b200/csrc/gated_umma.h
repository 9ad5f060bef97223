// Interface between the kernels of the gated feed-forward block (k_gated_umma.cu, k_gated_token.cu) and their host side (gated.cc).
#ifndef SEE_CUDA_GATED_UMMA_H_
#define SEE_CUDA_GATED_UMMA_H_

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "kernels.h"

namespace see::k {

// One output matrix [M, N] = A B, worked in tiles of 256 rows by a CTA pair.  The reduction runs over one or two operand
// pairs one after the other.  Every operand is loaded in boxes of 64 x 64 elements (128-byte rows): K-major, 64 of the
// reduction to a row, or MN-major, 64 of M or N to a row.
struct GatedProblem {
  CUtensorMap a[2], b[2];    // gated: b[0] the gate's weights, b[1] the up projection's, one operand pair
  CUtensorMap c;             // boxes of 32 rows x 64 columns
  uint32_t M, N;             // gated: N hidden columns
  uint32_t blocks[2];        // of 64 along the reduction, for each operand pair (the second may have none)
  uint32_t a_mn, b_mn;       // 1: MN-major
  uint32_t tiles_m, tiles_n;
  // Tiles from `whole` on (in the kernel's order) have their reduction cut into `parts`, each its own work: its f32 sums go to
  // partials, part by part from `first_part` on, and GatedFold adds them.  whole = all tiles: none.
  uint32_t whole, parts, first_part;
  void* out;                 // what c maps, for the fold
  uint64_t out_stride;
};
constexpr uint32_t kGatedProblems = 3;
struct GatedLaunch {
  GatedProblem p[kGatedProblems];
  CUtensorMap gate, up;      // gated, when kept: boxes like c
  uint32_t count;
  uint32_t f16;              // operands and outputs: 1 f16, 0 bf16
  int act;
  uint32_t keep;             // gated: gate and up leave too
  float* partials;           // [part][256 x 256]
  DeviceStatus* status;
};
// tn: columns of a pair's accumulator, 256, or gated also 128 (half of them the gate's, half the up projection's).
cudaError_t GatedProducts(const GatedLaunch& l, bool gated, uint32_t tn, uint32_t sms, cudaStream_t s);

// The cut tiles' parts added in order, rounded and stored.
cudaError_t GatedFold(const GatedLaunch& l, cudaStream_t s);

// dg = dh u act'(g), du = dh act(g): rows of `cols` elements (a multiple of 8); dh, g, u `stride` apart, dg, du dense.
cudaError_t GatedSlopes(const void* dh, const void* g, const void* u, void* dg, void* du, uint64_t rows, uint32_t cols, uint64_t stride,
                        int act, bool f16, uint32_t sms, cudaStream_t s);

// The forward pass of one row (k_gated_token.cu).
struct GatedTokenArgs {
  const void *x, *w_gate, *w_up;
  void *hidden, *gate, *up;   // gate and up null: not kept
  uint32_t d_in, d_hidden;
  int act;
};
bool GatedTokenTakes(uint64_t rows, uint64_t d_in);
cudaError_t GatedToken(const GatedTokenArgs& a, bool f16, uint32_t sms, cudaStream_t s);

}  // namespace see::k

#endif  // SEE_CUDA_GATED_UMMA_H_
