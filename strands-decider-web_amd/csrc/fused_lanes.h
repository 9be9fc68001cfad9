// Products of one or two rows for fused.hip, gfx950: lanes along K.
//
// A wave owns two columns (gated: one of the gate and the one of the up projection that it multiplies), its lanes take blocks l,
// l + 64, ... of each: one load of a whole packed block a column, 1 KiB of its row for a wave. A lane multiplies a block's codes into
// each row of a by v_dot2_f32_f16 from zero, then one fma adds s times that sum (asymmetric: and b' times the sum of the block's a,
// by dot2 with ones). The rows of a come through LDS, copied once in whole lines while the first blocks are on their way; blocks of
// the next two steps are loaded before a step's are used, so up to K = 6144 all are in flight at once. The lanes' sums are added by
// DPP and permlane, in an order that K alone decides.
//
// Bound: round trips, and with many columns the vector unit. us, against the waves that split K (fused_rows.h): 1 row, 2048 x 2048 2.9
// (4.1), 2048 x 6144 4.4 (6.3), gated 12288 x 2048 5.7 (6.9), 12288 x 512 5.1 (4.4); 2 rows 3.2 (4.1), 5.3 (6.3), 7.5 (6.8). Four
// columns a wave or one are no faster (5.9 and 6.6 at 12288 x 2048; 3.2 and 3.0 at 2048 x 2048), four rows no faster than those waves.
#pragma once
#include <hip/hip_runtime.h>

#include <type_traits>

#include "fused.h"
#include "fused_common.h"
#include "fused_plan.h"

namespace ha {
namespace {

constexpr int kLanesWaves = fused::kLanesThreads / 64;

// V values of each lane (1, 2 or 4), summed over the lanes: row r = l / 16 of lanes gets that of value r % V. Pairs meet in one
// register, so four values cost hardly more than one.
template <int V>
__device__ __forceinline__ float lanes_sums(const float* v) {
  auto swap = [](float a, float b, auto halves) {  // a's even rows of 16 plus its odd ones, and b's likewise in turn; or halves of 32
    const unsigned x = __builtin_bit_cast(unsigned, a), y = __builtin_bit_cast(unsigned, b);
    const auto r = decltype(halves)::value ? __builtin_amdgcn_permlane32_swap(x, y, false, false) : __builtin_amdgcn_permlane16_swap(x, y, false, false);
    return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
  };
  auto ror = [](float x, auto ctrl) {
    return x + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), decltype(ctrl)::value, 0xf, 0xf, false));
  };
  const float a = swap(v[0], v[V > 1 ? 1 : 0], std::false_type{}), b = V > 2 ? swap(v[V > 2 ? 2 : 0], v[V > 2 ? 3 : 0], std::false_type{}) : a;
  float x = swap(a, b, std::true_type{});
  x = ror(x, std::integral_constant<int, 0x128>{});  // row_ror:8, 4, 2, 1
  x = ror(x, std::integral_constant<int, 0x124>{});
  x = ror(x, std::integral_constant<int, 0x122>{});
  return ror(x, std::integral_constant<int, 0x121>{});
}

template <int BITS, bool ASYM, int MR>
__global__ __launch_bounds__(64 * kLanesWaves) void fused_lanes_kernel(FusedArgs p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char sm[];  // [row][16-byte chunks], chunk q at q ^ (q / 16 % 4)
  constexpr int LW = 2;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool gated = p.half != 0;
  const int cols = gated ? p.half : p.N, mine = gated ? 1 : LW, j0 = mine * (kLanesWaves * blockIdx.x + w);
  const int nblk = p.K / 32, ng = p.K / p.group, g64 = p.group == 64;
  typedef unsigned wv __attribute__((ext_vector_type(BITS), aligned(4)));
  const char *wp[LW], *sp[LW], *bp[LW];
#pragma unroll
  for (int c = 0; c < LW; c++) {  // (columns past the last: that one again, not stored)
    const int n = gated ? min(j0, cols - 1) + c * p.half : min(j0 + c, cols - 1);
    wp[c] = (const char*)p.q + (size_t)n * nblk * (4 * BITS);
    sp[c] = (const char*)p.s + (size_t)n * ng * 2;
    bp[c] = ASYM ? (const char*)p.b + (size_t)n * ng * 2 : sp[c];
  }
  struct Blocks {
    wv wd[LW];
    unsigned s[LW], b[LW];  // f16 bits
  };
  auto load = [&](int at, Blocks& x) {
    const unsigned k = min(at, nblk - 1);
#pragma unroll
    for (int c = 0; c < LW; c++) {
      x.wd[c] = *(gptr<wv>)(gp<char>(wp[c]) + k * (4 * BITS));
      x.s[c] = *(gptr<unsigned short>)(gp<char>(sp[c]) + 2 * (k >> g64));
      if constexpr (ASYM) x.b[c] = *(gptr<unsigned short>)(gp<char>(bp[c]) + 2 * (k >> g64));
    }
  };
  Blocks x, x1;
  load(lane, x);
  load(lane + 64, x1);
  // the first lane of row i (lanes_sums) finishes column i / MR, row i % MR
  const int ic = (lane >> 4) / MR, im = (lane >> 4) % MR;
  const bool store = lane % 16 == 0 && ic < mine && im < p.M && j0 + ic < cols;
  auto one = [](int) { return 0; };
  Given<1> early{};
  if (store) early = given<1>(p, im, j0 + ic, one);
  const int per = p.K / 8;  // 16-byte chunks of a row
#pragma unroll
  for (int m = 0; m < MR; m++)
    for (int q = tid; q < per; q += 64 * kLanesWaves)
      *(h8*)(sm + 16 * ((size_t)m * per + (q ^ ((q >> 4) & 3)))) = *(gptr<h8>)(gp<_Float16>(p.a) + (size_t)min(m, p.M - 1) * p.K + 8 * q);
  __syncthreads();
  float acc[LW][MR];
#pragma unroll
  for (int c = 0; c < LW; c++)
#pragma unroll
    for (int m = 0; m < MR; m++) acc[c][m] = 0.0f;
  for (int at = lane; at < nblk; at += 64) {
    Blocks x2;
    load(at + 128, x2);
    h8 av[MR][4];
    float sum[MR];
#pragma unroll
    for (int m = 0; m < MR; m++) {
      sum[m] = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int q = 4 * at + j;
        av[m][j] = *(const h8*)(sm + 16 * ((size_t)m * per + (q ^ ((q >> 4) & 3))));
        if constexpr (ASYM) {
#pragma unroll
          for (int e = 0; e < 4; e++)
            sum[m] = __builtin_amdgcn_fdot2(h2{av[m][j][2 * e], av[m][j][2 * e + 1]}, h2{(_Float16)1.0f, (_Float16)1.0f}, sum[m], false);
        }
      }
    }
#pragma unroll
    for (int c = 0; c < LW; c++) {
      float d[MR];
#pragma unroll
      for (int m = 0; m < MR; m++) d[m] = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        h8 v;
        if constexpr (BITS == 4) v = codes8<BITS>(x.wd[c][j], 0);
        else v = codes8<BITS>(x.wd[c][j >> 1] >> (16 * (j & 1)) & 0xFFFFu, BITS == 3 ? x.wd[c][BITS - 1] >> (8 * j) & 0xFFu : 0u);
#pragma unroll
        for (int m = 0; m < MR; m++)
#pragma unroll
          for (int e = 0; e < 4; e++)
            d[m] = __builtin_amdgcn_fdot2(h2{av[m][j][2 * e], av[m][j][2 * e + 1]}, h2{v[2 * e], v[2 * e + 1]}, d[m], false);
      }
      const float s = f16_bits(x.s[c]);
#pragma unroll
      for (int m = 0; m < MR; m++) {
        acc[c][m] = fmaf(s, d[m], acc[c][m]);
        if constexpr (ASYM) acc[c][m] = fmaf(centred<BITS>(s, f16_bits(x.b[c])), sum[m], acc[c][m]);
      }
    }
    x = x1;
    x1 = x2;
  }
  float z, up = 0.0f;
  if (gated) {
    z = lanes_sums<MR>(acc[0]);
    up = lanes_sums<MR>(acc[1]);
  } else {
    z = lanes_sums<LW * MR>(acc[0]);
  }
  if (store) finish<1>(p, im, j0 + ic, one, &z, &up, early);
}

template <int BITS, bool ASYM, int MR>
hipError_t launch_lanes_as(const FusedArgs& p, hipStream_t s) {
  const int cols = p.half ? p.half : p.N, wide = kLanesWaves * (p.half ? 1 : 2);
  if (!fused::fits((cols + wide - 1) / wide, 64 * kLanesWaves)) return hipErrorInvalidValue;
  hipLaunchKernelGGL((fused_lanes_kernel<BITS, ASYM, MR>), dim3((unsigned)((cols + wide - 1) / wide)), dim3(64 * kLanesWaves), (size_t)MR * p.K * 2, s, p);
  return hipGetLastError();
}
template <int BITS, bool ASYM>
hipError_t launch_lanes(const FusedArgs& p, hipStream_t s) {
  return p.M == 1 ? launch_lanes_as<BITS, ASYM, 1>(p, s) : launch_lanes_as<BITS, ASYM, 2>(p, s);
}

}  // namespace
}  // namespace ha
