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

// Any operands (K a multiple of 32, a 16-byte and codes 4-byte aligned). A workgroup makes 16 rows x 4 tiles of 16 columns (gated:
// two of the gate and the two of the up projection 32 columns on), its waves taking every kAnyWaves-th 32-k group:
// v_mfma_f32_16x16x32_f16, lane (g = l / 16, c = l % 16) row c of a and column c of a tile, k 8 g .. + 7 of the group; D: rows
// 4 g + e, column c. Operands come straight from memory, four groups a wave at a time (7 x 36 x 4000, 3 bits: 115 us with one
// wave for all of K).
constexpr int kAnyWaves = fused::kAnyThreads / 64;
template <int BITS, bool ASYM, int EPI>
__global__ __launch_bounds__(64 * kAnyWaves) void fused_any_kernel(FusedArgs p) {
  __shared__ f4 red[kAnyWaves][4][64];
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int cols = EPI == kEpiAct && p.half ? p.half : p.N, wide = EPI == kEpiAct && p.half ? 32 : 64;
  const int ntn = (cols + wide - 1) / wide, tn = blockIdx.x % ntn, m0 = 16 * (blockIdx.x / ntn), n0 = wide * tn;
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
#pragma unroll 4
  for (int k = w; k < nblk; k += kAnyWaves) {
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
#pragma unroll
  for (int t = 0; t < 4; t++) red[w][t][lane] = acc[t];
  __syncthreads();
  auto total = [&](int t) {
    f4 s = red[0][t][lane];
#pragma unroll
    for (int v = 1; v < kAnyWaves; v++) s += red[v][t][lane];
    return s;
  };
  const int m = m0 + 4 * g;
  if constexpr (EPI == kEpiLogits) {
    if (w) return;
#pragma unroll
    for (int t = 0; t < 4; t++) acc[t] = total(t);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float z[4] = {p.scale * acc[0][e], p.scale * acc[1][e], p.scale * acc[2][e], p.scale * acc[3][e]};
      const LpRecord r = record16(z, c, cols - n0);
      if (c == 0 && m + e < p.M) p.rec[(size_t)(m + e) * ntn + tn] = r;
    }
  } else {
    if (m >= p.M || w >= wide / 16) return;
    const f4 z = total(w), up = wide == 32 ? total(w ^ 2) : f4{};
    results<4>(p, m, n0 + 16 * w + c, cols, [](int v) { return v; }, (const float*)&z, wide == 32 ? (const float*)&up : nullptr);
  }
}

template <int BITS, bool ASYM, int EPI>
hipError_t launch_any_as(const FusedArgs& p, hipStream_t s) {
  const int cols = EPI == kEpiAct && p.half ? p.half : p.N, wide = EPI == kEpiAct && p.half ? 32 : 64;
  const long tiles = (long)((cols + wide - 1) / wide) * ((p.M + 15) / 16);
  if (!fused::fits(tiles, 64 * kAnyWaves)) return hipErrorInvalidValue;
  hipLaunchKernelGGL((fused_any_kernel<BITS, ASYM, EPI>), dim3((unsigned)tiles), dim3(64 * kAnyWaves), 0, s, p);
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

// Rows from .. from + M - 1 of a call.
FusedArgs part_of(const FusedArgs& p, int from, int M) {
  FusedArgs x = p;
  x.M = M;
  x.a = (const char*)p.a + (size_t)from * p.K * 2;
  if (p.res) x.res = (const char*)p.res + (size_t)from * p.res_stride * (p.res_f32 ? 4 : 2);
  if (p.out) x.out = (char*)p.out + (size_t)from * p.out_stride * (p.out_f32 ? 4 : 2);
  if (p.rec) x.rec = p.rec + (size_t)from * ((p.N + kLpBlock - 1) / kLpBlock);
  return x;
}
// A call that one launch cannot hold, in two parts of its rows.
template <class Launch>
hipError_t in_parts(const FusedArgs& p, hipStream_t s, Launch launch) {
  const int first = fused::first_part(p.M);
  if (!first) return hipErrorInvalidValue;
  const hipError_t e = launch(part_of(p, 0, first), s);
  return e == hipSuccess ? launch(part_of(p, first, p.M - first), s) : e;
}

}  // namespace

hipError_t launch_fused(const FusedArgs& p, hipStream_t s) {
  const fused::Shape shape{p.M, p.half ? p.half : p.N, p.K, p.half != 0, p.asym != 0, whole(p), p.K % (32 * p.group) == 0, p.bits};
  const fused::Plan plan = fused::plan(shape);
  if (plan.path == fused::kLanes) return launch_fused_lanes(p, s);
  if (plan.path == fused::kRows) return launch_fused_rows(p, plan.a, plan.b, s);
  if (plan.path == fused::kTiles) return launch_fused_tiles(p, plan.a, plan.b, plan.halves, s);
  if (!fused::launchable(shape, plan)) return in_parts(p, s, launch_fused);
  return launch_any<kEpiAct>(p, s);
}

hipError_t launch_logit_records(const FusedArgs& p, hipStream_t s) {
  if (!fused::logits_fit(p.M, p.N, whole(p), p.asym != 0)) return in_parts(p, s, launch_logit_records);
  return whole(p) ? launch_logit_tiles(p, s) : launch_any<kEpiLogits>(p, s);
}

}  // namespace ha
