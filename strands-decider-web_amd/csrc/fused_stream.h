// Records of the logits of up to 16 rows for fused.hip, gfx950: the table passes once, straight into the registers of waves that
// share nothing but the rows of a.
//
// A wave makes a 64-column block, 16 columns at a time, all of K in parts of 256 k: lane (g = l / 16, c = l % 16) loads the packed
// blocks 2 g and 2 g + 1 of column c, so that four lanes read whole 128-byte lines, and swaps of lane groups turn them into the operands
// of v_mfma_f32_16x16x32_f16, of which lane (g, c) holds k 8 g .. + 7 of one 32-k group of column c: a 4 x 4 transposition of (lane
// group, word). Four parts are on their way at any time. Along K first: the eight parts that share a column's line of scales follow
// each other (16 columns after another for each 256 k, which shares the operands of a, fetched those lines again: a sixth slower).
//
// a stands in LDS, 16-byte chunk j of row r in slot j ^ (r & 15) of its 16.
//
// Bound: the table's bytes: 67 us (65 at best) for one row over 248320 tokens of 2048 (4 bits, groups of 32), 4.3 TB/s, 57 with groups of
// 64; with 3 and 2 bits (83 and 54) the vector unit: decoding, a swap a word, four fma a group. Products of up to 16 rows, with K split over the
// waves of a workgroup, gained nothing on the rows kernel this way (1 x 12288 x 2048 7.5 : 7.4 us, 8 rows 8.3 : 7.2).
#pragma once
#include <hip/hip_runtime.h>

#include "fused.h"
#include "fused_common.h"

namespace ha {
namespace {

constexpr int kStreamWaves = 8, kStreamK = 256, kStreamRows = 16, kStreamLds = 128 * 1024;

// r[w] at lane group b to r[b] at lane group w
__device__ __forceinline__ void transpose4(unsigned* r) {
  const auto p = __builtin_amdgcn_permlane32_swap(r[0], r[2], false, false);
  const auto q = __builtin_amdgcn_permlane32_swap(r[1], r[3], false, false);
  const auto x = __builtin_amdgcn_permlane16_swap((unsigned)p[0], (unsigned)q[0], false, false);
  const auto y = __builtin_amdgcn_permlane16_swap((unsigned)p[1], (unsigned)q[1], false, false);
  r[0] = (unsigned)x[0];
  r[1] = (unsigned)x[1];
  r[2] = (unsigned)y[0];
  r[3] = (unsigned)y[1];
}

// A lane's share of 256 k of a column.
template <int BITS, bool ASYM>
struct Part {
  unsigned wd[2 * BITS];           // two packed blocks
  unsigned s[4], b[ASYM ? 4 : 1];  // eight groups' f16, with groups of 64 four
};

// q, s and b: where 256-k piece 0 of the lane's column starts (q: at the lane's blocks)
template <int BITS, bool ASYM, bool G64>
__device__ __forceinline__ void load_part(const char* q, unsigned qo, const char* s, const char* b, unsigned so, int u, Part<BITS, ASYM>& x) {
  typedef unsigned u4 __attribute__((ext_vector_type(4), aligned(4)));
  typedef unsigned u2 __attribute__((ext_vector_type(2), aligned(4)));
  const gptr<char> from = gp<char>(q + (size_t)u * (32 * BITS)) + qo;
#pragma unroll
  for (int i = 0; i < 2 * BITS; i += 4) {
    if (2 * BITS - i >= 4) {
      const u4 v = *(gptr<u4>)(from + 4 * i);
      x.wd[i] = v[0], x.wd[i + 1] = v[1], x.wd[i + 2] = v[2], x.wd[i + 3] = v[3];
    } else {
      const u2 v = *(gptr<u2>)(from + 4 * i);
      x.wd[i] = v[0], x.wd[i + 1] = v[1];
    }
  }
  auto eight = [&](const char* table, unsigned* to) {
    if constexpr (G64) {
      const u2 v = *(gptr<u2>)(gp<char>(table + (size_t)u * 8) + so);
      to[0] = v[0], to[1] = v[1], to[2] = to[3] = 0;
    } else {
      const u4 v = *(gptr<u4>)(gp<char>(table + (size_t)u * 16) + so);
      to[0] = v[0], to[1] = v[1], to[2] = v[2], to[3] = v[3];
    }
  };
  eight(s, x.s);
  if constexpr (ASYM) eight(b, x.b);
}

// acc += the part's products. operand(b): the lane's k of group b of the 256 k.
template <int BITS, bool ASYM, bool G64, class Operand>
__device__ __forceinline__ void add_part(const Part<BITS, ASYM>& y, int g, Operand operand, f4& acc) {
  const f4 zero = f4{0.0f, 0.0f, 0.0f, 0.0f};
  f4 d[4], sum[ASYM ? 4 : 1];  // of groups of 64 both halves together
#pragma unroll
  for (int e = 0; e < 2; e++) {  // groups 2 b + e
    // (operands of a are read again for each column tile: kept, they would cost a wave of four on a SIMD)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    unsigned r[4], hi[4] = {0, 0, 0, 0};
    const unsigned* wd = y.wd + e * BITS;
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = BITS == 4 ? wd[i] : wd[i >> 1];
    transpose4(r);
    if constexpr (BITS == 3) {
#pragma unroll
      for (int i = 0; i < 4; i++) hi[i] = wd[2];
      transpose4(hi);
    }
#pragma unroll
    for (int b = 0; b < 4; b++) {
      const unsigned lo = BITS == 4 ? r[b] : r[b] >> (16 * (g & 1)) & 0xFFFFu;
      const h8 av = operand(2 * b + e);
      const bool fresh = !G64 || e == 0;
      d[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, codes8<BITS>(lo, hi[b] >> (8 * g) & 0xFFu), fresh ? zero : d[b], 0, 0, 0);
      if constexpr (ASYM) sum[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, ones8(), fresh ? zero : sum[b], 0, 0, 0);
      if (G64 && e == 0) continue;
      const float s = f16_bits(G64 ? y.s[b >> 1] >> (16 * (b & 1)) : y.s[b] >> (16 * e));
#pragma unroll
      for (int i = 0; i < 4; i++) acc[i] = fmaf(s, d[b][i], acc[i]);
      if constexpr (ASYM) {
        const float bias = centred<BITS>(s, f16_bits(G64 ? y.b[b >> 1] >> (16 * (b & 1)) : y.b[b] >> (16 * e)));
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] = fmaf(bias, sum[b][i], acc[i]);
      }
    }
  }
}

template <int BITS, bool ASYM, bool G64>
__global__ __launch_bounds__(64 * kStreamWaves, 4) void fused_stream_kernel(FusedArgs p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char sm[];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), nb = (p.N + kLpBlock - 1) / kLpBlock;
  const int block = blockIdx.x * kStreamWaves + w, n0 = kLpBlock * min(block, nb - 1);
  const int nblk = p.K / 32, ng = p.K / p.group, chunks = p.K / kStreamK;
  const char* wp = (const char*)p.q + (size_t)n0 * nblk * (4 * BITS);
  const char* sp = (const char*)p.s + (size_t)n0 * ng * 2;
  const char* bp = ASYM ? (const char*)p.b + (size_t)n0 * ng * 2 : sp;
  const int left = p.N - 1 - n0;  // (columns past the last repeat it and do not count)
  // part i is 256-k piece i % chunks of column tile i / chunks: 32 bits of lane offset from a scalar address on
  Part<BITS, ASYM> x[4];
  int lt = 0, lu = 0;  // of the next part to load
  auto load = [&](int slot) {
    const unsigned n = min(16 * min(lt, 3) + c, left);
    load_part<BITS, ASYM, G64>(wp, (n * nblk + 2 * g) * (4 * BITS), sp, bp, n * ng * 2, lu, x[slot]);
    if (++lu == chunks) lu = 0, lt++;
  };
#pragma unroll
  for (int t = 0; t < 4; t++) load(t);
  const int per = p.K / 8;  // 16-byte chunks of a row
  for (int i = tid; i < p.M * per; i += 64 * kStreamWaves) {
    const int r = i / per, j = i - r * per;
    *(h8*)(sm + 16 * ((size_t)r * per + ((j & ~15) | ((j ^ r) & 15)))) = ((gptr<h8>)gp<_Float16>(p.a))[i];
  }
  __syncthreads();
  if (block >= nb) return;
  const int row = min(c, p.M - 1);
  const unsigned char* ar = sm + (size_t)row * per * 16;
  f4 acc = f4{0.0f, 0.0f, 0.0f, 0.0f}, done[4];
#pragma unroll
  for (int t = 0; t < 4; t++) done[t] = acc;
  int t = 0, u = 0;
#pragma unroll 1
  for (int i = 0; i < chunks; i++) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
      auto operand = [&](int b) {
        const int j = 32 * u + 4 * b + g;
        return *(const h8*)(ar + 16 * ((j & ~15) | ((j ^ row) & 15)));
      };
      const Part<BITS, ASYM> y = x[k];  // (and the part after the next three on its way into its place)
      load(k);
      add_part<BITS, ASYM, G64>(y, g, operand, acc);
      if (++u == chunks) {
#pragma unroll
        for (int n = 0; n < 4; n++)
          if (n == t) done[n] = acc;
        acc = f4{0.0f, 0.0f, 0.0f, 0.0f};
        u = 0, t++;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 4; e++) {
    if (e >= p.M) break;
    const float z[4] = {p.scale * done[0][e], p.scale * done[1][e], p.scale * done[2][e], p.scale * done[3][e]};
    const LpRecord r = record16(z, c, p.N - n0);
    const int m = 4 * g + e;
    if (c == 0 && m < p.M) p.rec[(size_t)m * nb + block] = r;
  }
}

// Whether it can run a call: whole 256 k, rows that fit LDS.
inline bool stream_takes(const FusedArgs& p) {
  return p.M <= kStreamRows && p.K % kStreamK == 0 && (size_t)p.M * p.K * 2 <= kStreamLds;
}

template <int BITS, bool ASYM, bool G64>
hipError_t launch_stream_as(const FusedArgs& p, hipStream_t s) {
  const int lds = p.M * p.K * 2, nb = (p.N + kLpBlock - 1) / kLpBlock;
  auto k = fused_stream_kernel<BITS, ASYM, G64>;
  if (lds > 48 * 1024) {  // (the same limit for every call: it is the function's, not the launch's, and calls may overlap)
    const hipError_t e = hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, kStreamLds);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(k, dim3((nb + kStreamWaves - 1) / kStreamWaves), dim3(64 * kStreamWaves), lds, s, p);
  return hipGetLastError();
}
template <int BITS, bool ASYM>
hipError_t launch_stream(const FusedArgs& p, hipStream_t s) {
  return p.group == 64 ? launch_stream_as<BITS, ASYM, true>(p, s) : launch_stream_as<BITS, ASYM, false>(p, s);
}

}  // namespace
}  // namespace ha
