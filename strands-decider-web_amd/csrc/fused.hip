// Products of f16 rows with quantised weights (formats: mnb.hip) whose sums are never stored as they are, gfx950:
//   products  out = residual + act(a W^T + bias), or gated out = residual + act(z_j) z_(half + j)      (launch_fused)
//   logits    z = scale a W^T over a vocabulary, of which each row's 64-column blocks leave a record   (launch_logit_records)
// No counterpart in the reference, which stores the product in f16 and runs SILU_MUL, ADD_BIAS and ADD_NORM on it
// (web/public/engine/wgsl.js:55-121), and has no product with its embedding table.
#include <hip/hip_runtime.h>

#include "fused.h"
#include "fused_common.h"
#include "fused_plan.h"

namespace ha {
namespace {

// Any operands (K a multiple of 32, a 16-byte and codes 4-byte aligned). A wave makes 16 rows x 4 tiles of 16 columns (gated:
// two of the gate and the two of the up projection 32 columns on): v_mfma_f32_16x16x32_f16, lane (g = l / 16, c = l % 16) row c
// of a and column c of a tile, k 8 g .. + 7 of a 32-k block; D: rows 4 g + e, column c. Operands come straight from memory.
template <int BITS, bool ASYM, int EPI>
__global__ __launch_bounds__(256) void fused_any_kernel(FusedArgs p) {
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int cols = EPI == kEpiAct && p.half ? p.half : p.N, wide = EPI == kEpiAct && p.half ? 32 : 64;
  const int ntn = (cols + wide - 1) / wide, groups = (ntn + 3) / 4;
  const int tn = 4 * (blockIdx.x % groups) + (threadIdx.x >> 6), m0 = 16 * (blockIdx.x / groups), n0 = wide * tn;
  if (tn >= ntn) return;
  const int nblk = p.K / 32, ng = p.K / p.group, gl = p.group == 64 ? 1 : 0;
  gptr<h8> ap = (gptr<h8>)(gp<_Float16>(p.a) + (size_t)min(m0 + c, p.M - 1) * p.K + 8 * g);
  gptr<unsigned> wp[4];
  gptr<unsigned short> sp[4], bp[4];
#pragma unroll
  for (int t = 0; t < 4; t++) {
    int n = wide == 32 ? min(n0 + 16 * (t & 1) + c, cols - 1) + (t >> 1) * p.half : min(n0 + 16 * t + c, cols - 1);
    wp[t] = gp<unsigned>(p.q) + (size_t)n * nblk * BITS;
    sp[t] = gp<unsigned short>(p.s) + (size_t)n * ng;
    bp[t] = ASYM ? gp<unsigned short>(p.b) + (size_t)n * ng : sp[t];
  }
  f4 acc[4];
#pragma unroll
  for (int t = 0; t < 4; t++) acc[t] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 2
  for (int k = 0; k < nblk; k++) {
    const h8 av = ap[4 * k];
    f4 sum{0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (ASYM) sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, ones8(), sum, 0, 0, 0);
#pragma unroll
    for (int t = 0; t < 4; t++) {
      unsigned lo, hi = 0;
      if constexpr (BITS == 4) lo = wp[t][4 * k + g];
      else lo = wp[t][BITS * k + (g >> 1)] >> (16 * (g & 1)) & 0xFFFFu;
      if constexpr (BITS == 3) hi = wp[t][BITS * k + 2] >> (8 * g) & 0xFFu;
      const float s = f16_bits(sp[t][k >> gl]);
      const f4 d = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, codes8<BITS>(lo, hi), f4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
      for (int e = 0; e < 4; e++) acc[t][e] = fmaf(s, d[e], acc[t][e]);
      if constexpr (ASYM) {
        const float b = centred<BITS>(s, f16_bits(bp[t][k >> gl]));
#pragma unroll
        for (int e = 0; e < 4; e++) acc[t][e] = fmaf(b, sum[e], acc[t][e]);
      }
    }
  }
  const int m = m0 + 4 * g;
  if constexpr (EPI == kEpiLogits) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float z[4] = {p.scale * acc[0][e], p.scale * acc[1][e], p.scale * acc[2][e], p.scale * acc[3][e]};
      const LpRecord r = record16(z, c, cols - n0);
      if (c == 0 && m + e < p.M) p.rec[(size_t)(m + e) * ntn + tn] = r;
    }
  } else {
    if (m >= p.M) return;
#pragma unroll
    for (int t = 0; t < 4; t++) {
      if (wide == 32 && t >= 2) break;
      results<4>(p, m, n0 + 16 * t + c, cols, [](int v) { return v; }, (const float*)&acc[t], wide == 32 ? (const float*)&acc[t ^ 2] : nullptr);
    }
  }
}

template <int BITS, bool ASYM, int EPI>
hipError_t launch_any_as(const FusedArgs& p, hipStream_t s) {
  const int cols = EPI == kEpiAct && p.half ? p.half : p.N, wide = EPI == kEpiAct && p.half ? 32 : 64;
  const long groups = ((cols + wide - 1) / wide + 3) / 4, rows = (p.M + 15) / 16;
  if (groups * rows > 0x7FFFFFFFl) return hipErrorInvalidValue;
  hipLaunchKernelGGL((fused_any_kernel<BITS, ASYM, EPI>), dim3((unsigned)(groups * rows)), dim3(256), 0, s, p);
  return hipGetLastError();
}

template <int EPI>
hipError_t launch_any(const FusedArgs& p, hipStream_t s) {
  switch (2 * p.bits + (p.asym ? 1 : 0)) {
    case 4: return launch_any_as<2, false, EPI>(p, s);
    case 5: return launch_any_as<2, true, EPI>(p, s);
    case 6: return launch_any_as<3, false, EPI>(p, s);
    case 7: return launch_any_as<3, true, EPI>(p, s);
    case 8: return launch_any_as<4, false, EPI>(p, s);
    case 9: return launch_any_as<4, true, EPI>(p, s);
  }
  return hipErrorInvalidValue;
}

// Whether the kernels that move whole 64-k tiles can run the operands: codes in whole words of a block's half, two scales at once.
bool whole(const FusedArgs& p) {
  const uintptr_t sb = (uintptr_t)p.s | (p.asym ? (uintptr_t)p.b : 0);
  return p.K % 64 == 0 && (p.group == 32 || p.K % 128 == 0) && (uintptr_t)p.q % (p.bits == 4 ? 16 : 4) == 0 && sb % 4 == 0;
}

}  // namespace

hipError_t launch_fused(const FusedArgs& p, hipStream_t s) {
  const fused::Plan plan = fused::plan({p.M, p.half ? p.half : p.N, p.K, p.half != 0, p.asym != 0, whole(p)});
  if (plan.path == fused::kRows) return launch_fused_rows(p, plan.a, plan.b, s);
  if (plan.path == fused::kTiles) return launch_fused_tiles(p, plan.a, plan.b, s);
  return launch_any<kEpiAct>(p, s);
}

hipError_t launch_logit_records(const FusedArgs& p, hipStream_t s) {
  return whole(p) ? launch_logit_tiles(p, s) : launch_any<kEpiLogits>(p, s);
}

}  // namespace ha
