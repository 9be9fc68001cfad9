// Products of few rows for fused.hip, gfx950: a workgroup's waves split K and meet once, at the end.
//
// A workgroup makes 16 MT rows x 16 NT columns (gated: 8 NT of the gate and the 8 NT of the up projection that they multiply). Its
// waves take the 128-k pieces w, w + SW, ... of K in 64-k halves: each copies rows of a, codes and scales of a half into LDS of its own
// by DMA and waits for its own copies only, so there is no barrier in the loop; it reads a half into registers, starts the next half's
// copies into the same place and multiplies. Rows of a go through LDS because lanes hold different rows: a 16-byte load straight into
// the operands is a cache line a lane. The order of a row's sums depends on K and SW alone.
//
// v_mfma_f32_16x16x32_f16: lane (g = l / 16, c = l % 16) holds row c (A operand) or column c (B operand), k 8 g .. + 7 of a 32-k
// group; D: rows 4 g + e, column c. One product is a group, and four fma add s times it.
//
// Bound: round trips. A call of a few us reads each weight once (0.56 bytes) and M rows of a for every workgroup.
#pragma once
#include <hip/hip_runtime.h>

#include "fused.h"
#include "fused_common.h"
#include "fused_plan.h"
#include "lds_dma.h"

namespace ha {
namespace {

template <int BITS, bool ASYM, int MT, int NT, int SW>
struct RowsLds {
  static constexpr int kA = MT * 16 * 128, kW = NT * 16 * 8 * BITS, kS = NT * 64;
  static constexpr int kStage = kA + kW + kS * (ASYM ? 2 : 1);
  static constexpr int kSums = SW / 2 * MT * NT * 1024;
  static constexpr int kBytes = SW * kStage > kSums ? SW * kStage : kSums;
};

template <int BITS, bool ASYM, int MT, int NT, int SW, bool G64>
__global__ __launch_bounds__(64 * SW) void fused_rows_kernel(FusedArgs p) {
  using L = RowsLds<BITS, ASYM, MT, NT, SW>;
  constexpr int kUnit = BITS == 4 ? 16 : 4, kLanes = L::kW / kUnit, kUnits = (kLanes + 63) / 64;
  extern __shared__ __attribute__((aligned(16))) unsigned char sm[];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool gated = p.half != 0;
  const int cols = gated ? p.half : p.N, wide = gated ? 8 * NT : 16 * NT;
  const int ntn = (cols + wide - 1) / wide, j0 = wide * (blockIdx.x % ntn), m0 = 16 * MT * (blockIdx.x / ntn);
  const int nh = p.K / 64, nblk = p.K / 32, ng = p.K / p.group;
  // this wave's halves, two for each 128-k piece (one where the last piece has no second)
  const int np = (nh + 1) / 2, mine = w < np ? (np - 1 - w) / SW + 1 : 0;
  const int T = 2 * mine - ((nh & 1) && mine > 0 && (np - 1) % SW == w ? 1 : 0);
  auto half_of = [&](int t) { return 2 * (w + SW * (t >> 1)) + (t & 1); };
  // the weight row of column `col` of the workgroup's tiles (past the last: that one again, not stored)
  auto row_of = [&](int col) {
    if (!gated) return min(j0 + col, cols - 1);
    const int up = col >= wide ? 1 : 0;
    return min(j0 + col - up * wide, cols - 1) + up * p.half;
  };
  unsigned char* const st = sm + w * L::kStage;
  const unsigned lds = __builtin_amdgcn_readfirstlane(lds_addr(sm) + w * L::kStage);
  // lanes' byte offsets. a: copy i takes rows 8 i .. + 7, 16-byte chunk j of row r into slot j ^ (r & 7), so that operand reads of
  // 16 rows at one chunk fall in distinct banks; rows past M repeat the last one and are not stored
  unsigned ao[2 * MT];
  size_t wo[kUnits];
#pragma unroll
  for (int i = 0; i < 2 * MT; i++)
    ao[i] = (unsigned)min(8 * i + (lane >> 3), p.M - 1 - m0) * (unsigned)p.K * 2u + 16u * ((lane & 7) ^ (lane >> 3));
#pragma unroll
  for (int i = 0; i < kUnits; i++) {
    const int u = min(64 * i + lane, kLanes - 1), per = 8 * BITS / kUnit;
    wo[i] = (size_t)row_of(u / per) * nblk * (4 * BITS) + kUnit * (u % per);
  }
  const size_t so = (size_t)row_of(min(lane, 16 * NT - 1)) * ng * 2;
  const char* ap = (const char*)p.a + (size_t)m0 * p.K * 2;
  auto issue = [&](int t) {
    const int h = half_of(t);
#pragma unroll
    for (int i = 0; i < 2 * MT; i++)
      if (m0 + 8 * i < p.M) dma16(lds + 1024 * i, ao[i], ap + (size_t)h * 128);  // (rows that are not there may be anything)
#pragma unroll
    for (int i = 0; i < kUnits; i++) {
      if (64 * i + lane < kLanes) {
        const char* from = (const char*)p.q + wo[i] + (size_t)h * (8 * BITS);
        if constexpr (BITS == 4) dma16_at(lds + L::kA + 1024 * i, from);
        else dma4_at(lds + L::kA + 256 * i, from);
      }
    }
    const size_t sb = G64 ? (size_t)(h >> 1) * 4 : (size_t)h * 4;  // the half's two scales, or those of its piece's two halves
    if (lane < 16 * NT) {
      dma4_at(lds + L::kA + L::kW, (const char*)p.s + so + sb);
      if constexpr (ASYM) dma4_at(lds + L::kA + L::kW + L::kS, (const char*)p.b + so + sb);
    }
  };
  f4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int n = 0; n < NT; n++) acc[i][n] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  if (T > 0) issue(0);
  // Where a wave finishes one 16-column piece at most, what goes into it besides the sums is on its way from here on (at the end it is
  // a round trip of its own)
  const int per = (wide + 15) / 16;  // 16-column pieces of the result
  auto next = [](int v) { return v; };
  constexpr bool kEarly = MT * NT <= SW;
  Given<4> early{};
  if constexpr (kEarly) {
    const int col = 16 * (w % per) + c, m = m0 + 16 * (w / per) + 4 * g;
    if (w < MT * per && col < wide && m < p.M && j0 + col < cols) early = given<4>(p, m, j0 + col, next);
  }
  for (int t = 0; t < T; t++) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    h8 af[MT][2];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int j = 0; j < 2; j++) af[i][j] = *(const h8*)(st + (16 * i + c) * 128 + 16 * ((4 * j + g) ^ (c & 7)));
    unsigned lo[NT][2], hi[NT][2], sw[NT], bw[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const unsigned char* wc = st + L::kA + (16 * n + c) * (8 * BITS);
#pragma unroll
      for (int j = 0; j < 2; j++) {
        lo[n][j] = *(const unsigned*)(wc + 4 * BITS * j + 4 * (BITS == 4 ? g : g >> 1));
        hi[n][j] = BITS == 3 ? *(const unsigned*)(wc + 12 * j + 8) : 0u;
      }
      sw[n] = *(const unsigned*)(st + L::kA + L::kW + 4 * (16 * n + c));
      bw[n] = ASYM ? *(const unsigned*)(st + L::kA + L::kW + L::kS + 4 * (16 * n + c)) : 0u;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage has been read: refill it
    if (t + 1 < T) issue(t + 1);
    const f4 zero = f4{0.0f, 0.0f, 0.0f, 0.0f};
    auto codes = [&](int n, int j) {
      if constexpr (BITS == 4) return codes8<BITS>(lo[n][j], 0);
      else return codes8<BITS>(lo[n][j] >> (16 * (g & 1)) & 0xFFFFu, hi[n][j] >> (8 * g) & 0xFFu);
    };
    auto add = [&](int n, int shift, const f4* d, const f4* sum) __attribute__((always_inline)) {
      const float s = f16_bits(sw[n] >> shift);
      float bias = 0.0f;
      if constexpr (ASYM) bias = centred<BITS>(s, f16_bits(bw[n] >> shift));
#pragma unroll
      for (int i = 0; i < MT; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          acc[i][n][e] = fmaf(s, d[i][e], acc[i][n][e]);
          if constexpr (ASYM) acc[i][n][e] = fmaf(bias, sum[i][e], acc[i][n][e]);
        }
    };
    f4 sum[MT], d[MT];
    if constexpr (G64) {  // the half is one group: both 32 k one sum, scaled once
      if constexpr (ASYM) {
#pragma unroll
        for (int i = 0; i < MT; i++) {
          sum[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(af[i][0], ones8(), zero, 0, 0, 0);
          sum[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(af[i][1], ones8(), sum[i], 0, 0, 0);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const h8 b = codes(n, j);
#pragma unroll
          for (int i = 0; i < MT; i++) d[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(af[i][j], b, j ? d[i] : zero, 0, 0, 0);
        }
        add(n, 16 * (half_of(t) & 1), d, sum);  // (which of the piece's two scales)
      }
    } else {
#pragma unroll
      for (int j = 0; j < 2; j++) {
        if constexpr (ASYM) {
#pragma unroll
          for (int i = 0; i < MT; i++) sum[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(af[i][j], ones8(), zero, 0, 0, 0);
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
          const h8 b = codes(n, j);
#pragma unroll
          for (int i = 0; i < MT; i++) d[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(af[i][j], b, zero, 0, 0, 0);
          add(n, 16 * j, d, sum);
        }
      }
    }
  }
  // the waves' sums: w + (w + SW / 2), then those SW / 2 in order
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (none is in flight: the last half issues none)
  __syncthreads();  // every wave has drained and read its stage
  f4* red = (f4*)sm;
  if (w >= SW / 2) {
#pragma unroll
    for (int q = 0; q < MT * NT; q++) red[((w - SW / 2) * MT * NT + q) * 64 + lane] = acc[q / NT][q % NT];
  }
  __syncthreads();
  if (w < SW / 2) {
#pragma unroll
    for (int q = 0; q < MT * NT; q++) red[(w * MT * NT + q) * 64 + lane] += acc[q / NT][q % NT];
  }
  __syncthreads();
  // a row tile's sums of the workgroup's column `col`, rows 4 g ..
  auto total = [&](int i, int col) {
    const f4* from = red + (i * NT + col / 16) * 64 + 16 * g + col % 16;
    f4 s = from[0];
#pragma unroll
    for (int v = 1; v < SW / 2; v++) s += from[v * MT * NT * 64];
    return s;
  };
  for (int q = w; q < MT * per; q += SW) {
    const int i = q / per, col = 16 * (q % per) + c, m = m0 + 16 * i + 4 * g;
    if (col >= wide || m >= p.M || j0 + col >= cols) continue;
    const f4 z = total(i, col), up = gated ? total(i, wide + col) : f4{};
    if constexpr (kEarly) finish<4>(p, m, j0 + col, next, (const float*)&z, (const float*)&up, early);
    else results<4>(p, m, j0 + col, cols, next, (const float*)&z, (const float*)&up);
  }
}

template <int BITS, bool ASYM, int MT, int NT, int SW>
hipError_t launch_rows_as(const FusedArgs& p, hipStream_t s) {
  constexpr int lds = RowsLds<BITS, ASYM, MT, NT, SW>::kBytes;
  static_assert(lds <= 160 * 1024, "LDS of one CU");
  auto k = p.group == 64 ? fused_rows_kernel<BITS, ASYM, MT, NT, SW, true> : fused_rows_kernel<BITS, ASYM, MT, NT, SW, false>;
  if (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
  }
  const int cols = p.half ? p.half : p.N, wide = p.half ? 8 * NT : 16 * NT;
  const long tiles = (long)((cols + wide - 1) / wide) * ((p.M + 16 * MT - 1) / (16 * MT));
  if (!fused::fits(tiles, 64 * SW)) return hipErrorInvalidValue;
  hipLaunchKernelGGL(k, dim3((unsigned)tiles), dim3(64 * SW), lds, s, p);
  return hipGetLastError();
}

}  // namespace
}  // namespace ha
