// Products of many rows for fused.hip, gfx950: matrix-core tiles whose group sums are scaled in f32.
//
// v_mfma_f32_32x32x16_f16: lane (h = l / 32, f = l % 32) holds row f of a (A operand) or column f (B operand), k 16 h + 8 j .. + 7
// of a 32-k group for product j = 0, 1; D: column f, rows 8 (v / 4) + 4 h + v % 4. The two products of a group start from zero,
// and one fma a value adds s times their sum: 16 fma beside 64 cycles of the matrix unit, so the vector unit (fma, decoding:
// some 46 instructions a tile and group with RT = 4) is the busier of the two and what bounds the loop.
//
// A workgroup makes 32 RT rows x 256 columns, a wave all of the rows and 64 columns (gated: 32 of the gate and the 32 of the up
// projection that they multiply). Rows of a come through LDS by DMA, three stages of 64 k; a wave's weights go straight into its
// registers, a lane half h loading whole blocks 2 kt + h of its column, which a swap of lane halves turns into the operands.
// Two workgroups a CU: one multiplies while the other decodes, or makes its results.
#pragma once
#include <hip/hip_runtime.h>

#include "fused.h"
#include "fused_common.h"
#include "lds_dma.h"

namespace ha {
namespace {

typedef float f16v __attribute__((ext_vector_type(16)));
constexpr int kTileCols = 256, kTileWaves = 4, kTileStages = 3;

// x.low, y.low in x and x.high, y.high in y (halves of the wave)
__device__ __forceinline__ void swap_halves(unsigned& x, unsigned& y) {
  const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
  x = (unsigned)r[0];
  y = (unsigned)r[1];
}

template <int BITS, bool ASYM, int EPI, int RT>
__global__ __launch_bounds__(64 * kTileWaves, 2) void fused_tiles_kernel(FusedArgs p) {
  constexpr int kRows = 32 * RT, kStage = kRows * 128, CT = 2;
  constexpr int kCopies = kRows / 8 / kTileWaves;  // DMA instructions of a wave for a stage, 8 rows each
  constexpr int kPitch = 68;                       // of a wave's 32 x 64 results in LDS
  constexpr int kLds = kTileStages * kStage > kTileWaves * 32 * kPitch * 4 ? kTileStages * kStage : kTileWaves * 32 * kPitch * 4;
  __shared__ __attribute__((aligned(16))) unsigned char sm[kLds];
  const int tid = threadIdx.x, lane = tid & 63, f = lane & 31, h = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool gated = EPI == kEpiAct && p.half;
  const int cols = gated ? p.half : p.N, wide = gated ? kTileCols / 2 : kTileCols;
  const int ntn = (cols + wide - 1) / wide, ntm = (p.M + kRows - 1) / kRows, ntiles = ntn * ntm;
  // workgroups go to the 8 XCDs in turn: XCD x takes a contiguous range of tiles, in bands of 8 tile rows, rows fastest, so that
  // neighbours share rows of a and columns of W in its L2
  int id = blockIdx.x;
  {
    const int q = ntiles / 8, r = ntiles % 8, x = id % 8;
    id = x * q + min(x, r) + id / 8;
  }
  constexpr int kBand = 8;
  const int band = id / (kBand * ntn), in_band = id - band * kBand * ntn, rows = min(kBand, ntm - band * kBand);
  const int tm = band * kBand + in_band % rows, tn = in_band / rows;
  const int m0 = tm * kRows, j0 = tn * wide + (gated ? 32 : 64) * w;  // the wave's first column (of the result)
  const int nblk = p.K / 32, nkt = p.K / 64, ng = p.K / p.group;
  // rows past M repeat the last one, columns past the last likewise; neither is stored
  const unsigned last = (unsigned)(p.M - 1 - m0), k2 = 2u * (unsigned)p.K;
  const unsigned chunk = 16u * ((lane & 7) ^ (lane >> 3));  // chunk j of row r in slot j ^ (r & 7)
  const char* ap = (const char*)p.a + (size_t)m0 * p.K * 2;
  const unsigned lds = __builtin_amdgcn_readfirstlane(lds_addr(sm) + 1024u * kCopies * w);
  auto copy_a = [&](int kt, int stage) {
    kt = min(kt, nkt - 1);  // (past the last tile: that one again, not read)
#pragma unroll
    for (int i = 0; i < kCopies; i++)
      dma16(lds + (unsigned)(stage * kStage + 1024 * i), min(8u * (kCopies * w + i) + (lane >> 3), last) * k2 + chunk, ap + (size_t)kt * 128);
  };
  // a wave's columns: from a scalar address for each column tile, 32 bits of lane offset on
  const char *wp[CT], *sp[CT], *bp[CT];
  unsigned wo[CT], so[CT];
#pragma unroll
  for (int c = 0; c < CT; c++) {
    const int first = gated ? min(j0, cols - 1) + c * p.half : min(j0 + 32 * c, cols - 1), left = (gated ? c * p.half : 0) + cols - 1 - first;
    wp[c] = (const char*)p.q + (size_t)first * nblk * (4 * BITS);
    sp[c] = (const char*)p.s + (size_t)first * ng * 2;
    bp[c] = ASYM ? (const char*)p.b + (size_t)first * ng * 2 : sp[c];
    wo[c] = ((unsigned)min(f, left) * (unsigned)nblk + h) * (4u * BITS);
    so[c] = (unsigned)min(f, left) * (unsigned)ng * 2u;
  }
  typedef unsigned uw __attribute__((ext_vector_type(BITS)));
  uw wr[2][CT];
  unsigned sr[2][CT], br[2][CT];  // two groups' f16, or with groups of 64 two tiles'
  const bool g64 = p.group == 64;
  constexpr int kLoads = (ASYM ? 3 : 2) * CT;  // loads of a wave for a tile's weights
  auto load_w = [&](int kt, int q) {
    kt = min(kt, nkt - 1);
    const size_t st = g64 ? 2 * (size_t)(kt & ~1) : 4 * (size_t)kt;
#pragma unroll
    for (int c = 0; c < CT; c++) {
      wr[q][c] = *(gptr<uw>)(gp<char>(wp[c] + (size_t)kt * (8 * BITS)) + wo[c]);
      sr[q][c] = *(gptr<unsigned>)(gp<char>(sp[c] + st) + so[c]);
      if constexpr (ASYM) br[q][c] = *(gptr<unsigned>)(gp<char>(bp[c] + st) + so[c]);
    }
  };
  f16v acc[RT][CT];
#pragma unroll
  for (int i = 0; i < RT; i++)
#pragma unroll
    for (int c = 0; c < CT; c++) acc[i][c] = f16v{};
  const unsigned arow = (unsigned)f * 128u;
  // Tile kt, in stage kt % 3, its weights in registers kt % 2. Loads complete in order: in flight at the top are the weights of
  // tile kt, this wave's part of the copy of tile kt + 1 and the weights of tile kt + 1, so waiting for all but the last kLoads
  // lands the first two; the barrier at the end then makes tile kt + 1 everybody's. The copy of tile kt + 2 goes into the stage
  // that tile kt - 1 left before the last barrier.
  auto step = [&](int kt, int stage, int q) {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLoads) : "memory");
#pragma unroll
    for (int c = 0; c < CT; c++) {
      asm volatile("" : "+v"(wr[q][c]), "+v"(sr[q][c])::"memory");
      if constexpr (ASYM) asm volatile("" : "+v"(br[q][c])::"memory");
    }
    copy_a(kt + 2, stage == 0 ? 2 : stage - 1);
    // the words of group G for this lane: lo[G][c][j] as codes8 takes them
    unsigned lo[2][CT][2], hi[2][CT][2];
    float s[2][CT], b[2][CT];
#pragma unroll
    for (int c = 0; c < CT; c++) {
      unsigned x[BITS];
#pragma unroll
      for (int i = 0; i < BITS; i++) x[i] = wr[q][c][i];
      if constexpr (BITS == 4) {
        swap_halves(x[0], x[2]);
        swap_halves(x[1], x[3]);
#pragma unroll
        for (int g = 0; g < 2; g++)
#pragma unroll
          for (int j = 0; j < 2; j++) lo[g][c][j] = x[2 * g + j], hi[g][c][j] = 0;
      } else {
        swap_halves(x[0], x[1]);
        unsigned t[2] = {BITS == 3 ? x[BITS - 1] : 0u, BITS == 3 ? x[BITS - 1] : 0u};
        if constexpr (BITS == 3) swap_halves(t[0], t[1]);
#pragma unroll
        for (int g = 0; g < 2; g++)
#pragma unroll
          for (int j = 0; j < 2; j++) lo[g][c][j] = x[g] >> (16 * j) & 0xFFFFu, hi[g][c][j] = t[g] >> (16 * h + 8 * j) & 0xFFu;
      }
      const unsigned sv = g64 ? sr[q][c] >> (16 * (kt & 1)) : sr[q][c], bv = ASYM ? (g64 ? br[q][c] >> (16 * (kt & 1)) : br[q][c]) : 0u;
#pragma unroll
      for (int g = 0; g < 2; g++) {
        s[g][c] = f16_bits(g64 ? sv : sv >> (16 * g));
        if constexpr (ASYM) b[g][c] = centred<BITS>(s[g][c], f16_bits(g64 ? bv : bv >> (16 * g)));
      }
    }
    const unsigned char* as = sm + stage * kStage + arow;
    // The (row tile, column tile) pairs of both groups in turn: a pair's two products go with the fma of the pair before.
    f16v d[2], sum[ASYM ? 2 : 1];
    h8 bf[CT][2], af[2];
    auto operand = [&](int g, int i, int j) { return *(const h8*)(as + 32 * 128 * i + 16 * ((4 * g + 2 * h + j) ^ (f & 7))); };
    auto add = [&](int t, int from) {  // eight values of pair t
      const int g = t / (RT * CT), i = t / CT % RT, c = t % CT;
#pragma unroll
      for (int v = from; v < from + 8; v++) {
        acc[i][c][v] = fmaf(s[g][c], d[t & 1][v], acc[i][c][v]);
        if constexpr (ASYM) acc[i][c][v] = fmaf(b[g][c], sum[(t / CT) & 1][v], acc[i][c][v]);
      }
    };
    af[0] = operand(0, 0, 0);
    af[1] = operand(0, 0, 1);
#pragma unroll
    for (int t = 0; t < 2 * RT * CT; t++) {
      const int g = t / (RT * CT), c = t % CT, next = t / CT + 1;
      const bool load = c == CT - 1 && t + 1 < 2 * RT * CT;  // the next row tile's operands, into the registers that are done with
      if (t % (RT * CT) == 0) {
#pragma unroll
        for (int n = 0; n < CT; n++)
#pragma unroll
          for (int j = 0; j < 2; j++) bf[n][j] = codes8<BITS>(lo[g][n][j], hi[g][n][j]);
      }
      if constexpr (ASYM) {
        if (c == 0) {
          sum[(t / CT) & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[0], ones8(), f16v{}, 0, 0, 0);
          sum[(t / CT) & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[1], ones8(), sum[(t / CT) & 1], 0, 0, 0);
        }
      }
      d[t & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[0], bf[c][0], f16v{}, 0, 0, 0);
      if (load) af[0] = operand(next / RT, next % RT, 0);
      __builtin_amdgcn_sched_barrier(0);
      if (t > 0) add(t - 1, 0);
      __builtin_amdgcn_sched_barrier(0);
      d[t & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[1], bf[c][1], d[t & 1], 0, 0, 0);
      if (load) af[1] = operand(next / RT, next % RT, 1);
      __builtin_amdgcn_sched_barrier(0);
      if (t > 0) add(t - 1, 8);
      __builtin_amdgcn_sched_barrier(0);
    }
    add(2 * RT * CT - 1, 0);
    add(2 * RT * CT - 1, 8);
    load_w(kt + 2, q);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this wave's reads of the stage are done
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  copy_a(0, 0);
  load_w(0, 0);
  copy_a(1, 1);
  load_w(1, 1);
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kCopies + 2 * kLoads) : "memory");  // tile 0 has landed
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  int stage = 0;
  auto next = [&]() { stage = stage == kTileStages - 1 ? 0 : stage + 1; };
  int kt = 0;
  for (; kt + 2 <= nkt; kt += 2) {
    step(kt, stage, 0);
    next();
    step(kt + 1, stage, 1);
    next();
  }
  if (kt < nkt) step(kt, stage, 0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // copies past the end land before the LDS is given up
  if constexpr (EPI == kEpiLogits) {
    __syncthreads();  // the stages become the waves' own
    float* own = (float*)sm + w * 32 * kPitch;
    const int nb = (p.N + kLpBlock - 1) / kLpBlock, valid = min(p.N - j0, 64);
#pragma unroll
    for (int i = 0; i < RT; i++) {
#pragma unroll
      for (int c = 0; c < CT; c++)
#pragma unroll
        for (int v = 0; v < 16; v++) own[(8 * (v >> 2) + 4 * h + (v & 3)) * kPitch + 32 * c + f] = p.scale * acc[i][c][v];
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_wave_barrier();
      // lane (h, f): columns 32 h .. + 31 of row f
      float z[32];
#pragma unroll
      for (int t = 0; t < 8; t++) {
        const f4 v = *(const f4*)(own + f * kPitch + 32 * h + 4 * t);
#pragma unroll
        for (int e = 0; e < 4; e++) z[4 * t + e] = v[e];
      }
      __builtin_amdgcn_wave_barrier();
      if (valid > 0) {
        const LpRecord r = record32(z, h, valid);
        const int m = m0 + 32 * i + f;
        if (h == 0 && m < p.M) p.rec[(size_t)m * nb + (j0 >> 6)] = r;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
      for (int v = 0; v < 16; v++) {
        const int m = m0 + 32 * i + 8 * (v >> 2) + 4 * h + (v & 3);
        if (m >= p.M) continue;
        if (gated) {
          const int j = j0 + f;
          if (j < cols) store_result(p, m, j, result_of(p, j, acc[i][0][v], acc[i][1][v]));
        } else {
#pragma unroll
          for (int c = 0; c < CT; c++) {
            const int j = j0 + 32 * c + f;
            if (j < cols) store_result(p, m, j, result_of(p, j, acc[i][c][v]));
          }
        }
      }
  }
}

template <int BITS, bool ASYM, int EPI, int RT>
hipError_t launch_tiles(const FusedArgs& p, hipStream_t s) {
  const bool gated = EPI == kEpiAct && p.half;
  const int cols = gated ? p.half : p.N, wide = gated ? kTileCols / 2 : kTileCols;
  const long tiles = (long)((cols + wide - 1) / wide) * ((p.M + 32 * RT - 1) / (32 * RT));
  if (tiles > 0x7FFFFFFFl) return hipErrorInvalidValue;
  hipLaunchKernelGGL((fused_tiles_kernel<BITS, ASYM, EPI, RT>), dim3((unsigned)tiles), dim3(64 * kTileWaves), 0, s, p);
  return hipGetLastError();
}

}  // namespace
}  // namespace ha
