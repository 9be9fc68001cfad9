// Products of many rows for fused.hip, gfx950: matrix-core tiles whose group sums are scaled in f32.
//
// v_mfma_f32_32x32x16_f16: lane (h = l / 32, f = l % 32) holds row f of a (A operand) or column f (B operand), k 16 h + 8 j .. + 7
// of a 32-k group for product j = 0, 1; D: column f, rows 8 (v / 4) + 4 h + v % 4. The two products of a group start from zero,
// and one fma a value adds s times their sum: 16 fma beside 64 cycles of the matrix unit, so the vector unit (fma, decoding:
// some 46 instructions a tile and group with RT = 4) is the busier of the two and what bounds the loop.
//
// A workgroup makes 32 RT rows x 256 columns, a wave all of the rows and 64 columns (gated: 32 of the gate and the 32 of the up
// projection that they multiply). Rows of a and packed weights come through LDS by DMA, three stages of 64 k; a wave copies and
// reads weights and scales of its own columns, so only a needs the barrier. Two workgroups a CU.
#pragma once
#include <hip/hip_runtime.h>

#include "fused.h"
#include "fused_common.h"
#include "lds_dma.h"

namespace ha {
namespace {

typedef float f16v __attribute__((ext_vector_type(16)));
constexpr int kTileWaves = 4, kTileStages = 3;

template <int BITS, bool ASYM, int EPI, int RT, int CT>
__global__ __launch_bounds__(64 * kTileWaves, RT * CT <= 2 ? 4 : RT * CT <= 4 && !ASYM ? 3 : 2) void fused_tiles_kernel(FusedArgs p) {
  constexpr int kRows = 32 * RT, kA = kRows * 128, kCols = 32 * CT;  // kCols: of a wave
  constexpr int kW = CT * 64 * 4 * BITS, kS = ASYM ? 512 : 256;    // a wave's packed words and scales (, biases) of a stage
  constexpr int kStage = kA + kTileWaves * (kW + kS);
  constexpr int kCopiesA = kRows / 8 / kTileWaves, kCopiesW = (BITS == 4 ? CT : CT * BITS) + (ASYM ? 2 : 1);  // DMA instructions of a wave
  constexpr int kPitch = 68;                                       // of a wave's 32 x 64 results in LDS
  constexpr int kLds = kTileStages * kStage > kTileWaves * 32 * kPitch * 4 ? kTileStages * kStage : kTileWaves * 32 * kPitch * 4;
  __shared__ __attribute__((aligned(16))) unsigned char sm[kLds];
  const int tid = threadIdx.x, lane = tid & 63, f = lane & 31, h = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool gated = EPI == kEpiAct && p.half;
  const int cols = gated ? p.half : p.N, wide = kTileWaves * (gated ? 32 : kCols);
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
  const int m0 = tm * kRows, j0 = tn * wide + (gated ? 32 : kCols) * w;  // the wave's first column (of the result)
  const int nblk = p.K / 32, nkt = p.K / 64, ng = p.K / p.group;
  // rows past M repeat the last one, columns past the last likewise; neither is stored
  const unsigned last = (unsigned)(p.M - 1 - m0), k2 = 2u * (unsigned)p.K;
  const unsigned chunk = 16u * ((lane & 7) ^ (lane >> 3));  // chunk j of row r in slot j ^ (r & 7)
  const char* ap = (const char*)p.a + (size_t)m0 * p.K * 2;
  // a wave's columns: from a scalar address for each column tile, 32 bits of lane offset on. Copies of packed words: lane (h, f)
  // takes block h of column f, 16 bytes or a word at a time; of scales: lane l the pair of column l
  const char *wp[CT], *sp[CT], *bp[CT];
  unsigned wo[CT], so = 0;
#pragma unroll
  for (int c = 0; c < CT; c++) {
    const int first = gated ? min(j0, cols - 1) + c * p.half : min(j0 + 32 * c, cols - 1), left = (gated ? c * p.half : 0) + cols - 1 - first;
    wp[c] = (const char*)p.q + (size_t)first * nblk * (4 * BITS);
    sp[c] = (const char*)p.s + (size_t)first * ng * 2;
    bp[c] = ASYM ? (const char*)p.b + (size_t)first * ng * 2 : sp[c];
    wo[c] = ((unsigned)min(f, left) * (unsigned)nblk + h) * (4u * BITS);
    if (c == h) so = (unsigned)min(f, left) * (unsigned)ng * 2u;
  }
  const char *sl = (h ? sp[CT - 1] : sp[0]) + so, *bl = (h ? bp[CT - 1] : bp[0]) + so;
  const bool g64 = p.group == 64;
  const unsigned lds_a = __builtin_amdgcn_readfirstlane(lds_addr(sm) + 1024u * kCopiesA * w);
  const unsigned lds_w = __builtin_amdgcn_readfirstlane(lds_addr(sm) + kA + (kW + kS) * w);
  auto copy = [&](int kt, int stage) {
    kt = min(kt, nkt - 1);  // (past the last tile: that one again, not read)
    const unsigned to = lds_w + (unsigned)(stage * kStage);
#pragma unroll
    for (int c = 0; c < CT; c++) {
      if constexpr (BITS == 4) {
        dma16(to + 1024 * c, wo[c], wp[c] + (size_t)kt * (8 * BITS));
      } else {
#pragma unroll
        for (int i = 0; i < BITS; i++) dma4(to + 256 * (c * BITS + i), wo[c] + 4 * i, wp[c] + (size_t)kt * (8 * BITS));
      }
    }
    const size_t st = g64 ? 2 * (size_t)(kt & ~1) : 4 * (size_t)kt;  // the tile's two scales, or two tiles'
    dma4_at(to + kW, sl + st);
    if constexpr (ASYM) dma4_at(to + kW + 256, bl + st);
#pragma unroll
    for (int i = 0; i < kCopiesA; i++)
      dma16(lds_a + (unsigned)(stage * kStage + 1024 * i), min(8u * (kCopiesA * w + i) + (lane >> 3), last) * k2 + chunk, ap + (size_t)kt * 128);
  };
  // the words of group g of the tile in a stage as codes8 takes them, and the scales
  struct Words {
    unsigned lo[CT][2], hi[CT][2];
  };
  const unsigned char* const own = sm + kA + (kW + kS) * w;
  auto words = [&](int stage, int g) {
    const unsigned char* from = own + stage * kStage;
    Words x;
#pragma unroll
    for (int c = 0; c < CT; c++) {
      if constexpr (BITS == 4) {
        const uint2 v = *(const uint2*)(from + 1024 * c + 16 * (32 * g + f) + 8 * h);  // k 16 h .. + 15 of the group
        x.lo[c][0] = v.x, x.lo[c][1] = v.y, x.hi[c][0] = x.hi[c][1] = 0;
      } else {
        const unsigned v = *(const unsigned*)(from + 256 * (c * BITS + h) + 4 * (32 * g + f));
        const unsigned t = BITS == 3 ? *(const unsigned*)(from + 256 * (c * BITS + 2) + 4 * (32 * g + f)) >> (16 * h) : 0u;
#pragma unroll
        for (int j = 0; j < 2; j++) x.lo[c][j] = v >> (16 * j) & 0xFFFFu, x.hi[c][j] = t >> (8 * j) & 0xFFu;
      }
    }
    return x;
  };
  f16v acc[RT][CT];
#pragma unroll
  for (int i = 0; i < RT; i++)
#pragma unroll
    for (int c = 0; c < CT; c++) acc[i][c] = f16v{};
  const unsigned arow = (unsigned)f * 128u;
  constexpr int kPairs = RT * CT;  // (row tile, column tile) pairs of a group
  f16v d[2] = {f16v{}, f16v{}}, sum[ASYM ? 2 : 1] = {};
  h8 bf[CT][2], af[2][2];
  float s[2][CT] = {}, b[2][CT] = {};
  auto add = [&](int t, int from) {  // eight values of pair t of a tile
    const int g = t / kPairs, i = t / CT % RT, c = t % CT;
#pragma unroll
    for (int v = from; v < from + 8; v++) {
      acc[i][c][v] = fmaf(s[g][c], d[t & 1][v], acc[i][c][v]);
      if constexpr (ASYM) acc[i][c][v] = fmaf(b[g][c], sum[(t / CT) & 1][v], acc[i][c][v]);
    }
  };
  auto decode = [&](const Words& x, int c) {
#pragma unroll
    for (int j = 0; j < 2; j++) bf[c][j] = codes8<BITS>(x.lo[c][j], x.hi[c][j]);
  };
  // Copies complete in order. At the top of tile kt this wave's copies of tile kt + 1 may still be in flight, those of tile kt have
  // landed; behind the barrier everybody's have, and everybody has read tile kt - 1, whose stage takes tile kt + 2.
  copy(0, 0);
  copy(1, 1);
  int stage = 0;
  Words x0;
  for (int kt = 0; kt < nkt; kt++) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kCopiesA + kCopiesW) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    copy(kt + 2, stage == 0 ? 2 : stage - 1);
    const int next_stage = stage == kTileStages - 1 ? 0 : stage + 1;
    const unsigned char* as = sm + stage * kStage + arow;
    auto operand = [&](int g, int i, int j) { return *(const h8*)(as + 32 * 128 * i + 16 * ((4 * g + 2 * h + j) ^ (f & 7))); };
    af[0][0] = operand(0, 0, 0);
    af[0][1] = operand(0, 0, 1);
    if (kt == 0) {
      x0 = words(0, 0);
      decode(x0, 0);
    }
    unsigned sw[CT], bw[CT];
#pragma unroll
    for (int c = 0; c < CT; c++) {
      sw[c] = *(const unsigned*)(own + stage * kStage + kW + 4 * (32 * c + f));
      bw[c] = ASYM ? *(const unsigned*)(own + stage * kStage + kW + 256 + 4 * (32 * c + f)) : 0u;
    }
    Words x1;
    // The pairs of both groups in turn: a pair's two products go with the fma of the pair before (of a tile's first, with those of
    // the last tile's last), with the next row tile's reads and the next group's decoding
#pragma unroll
    for (int t = 0; t < 2 * kPairs; t++) {
      const int g = t / kPairs, i = t / CT % RT, c = t % CT, u = (t / CT) & 1;
      if constexpr (ASYM) {
        if (c == 0) {
          sum[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[u][0], ones8(), f16v{}, 0, 0, 0);
          sum[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[u][1], ones8(), sum[u], 0, 0, 0);
        }
      }
      d[t & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[u][0], bf[c][0], f16v{}, 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      if (c == 0 && t + CT < 2 * kPairs) {
        af[u ^ 1][0] = operand((t + CT) / kPairs, (t + CT) / CT % RT, 0);
        af[u ^ 1][1] = operand((t + CT) / kPairs, (t + CT) / CT % RT, 1);
      }
      if (t == CT - 1) x1 = words(stage, 1);
      add(t == 0 ? 2 * kPairs - 1 : t - 1, 0);
      __builtin_amdgcn_sched_barrier(0);
      d[t & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[u][1], bf[c][1], d[t & 1], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      add(t == 0 ? 2 * kPairs - 1 : t - 1, 8);
      if (t == 0) {  // (the last tile's scales are done with)
        if constexpr (CT == 2) decode(x0, 1);
#pragma unroll
        for (int n = 0; n < CT; n++) {
          const unsigned sv = g64 ? sw[n] >> (16 * (kt & 1)) : sw[n], bv = g64 ? bw[n] >> (16 * (kt & 1)) : bw[n];
#pragma unroll
          for (int q = 0; q < 2; q++) {
            s[q][n] = f16_bits(g64 ? sv : sv >> (16 * q));
            if constexpr (ASYM) b[q][n] = centred<BITS>(s[q][n], f16_bits(g64 ? bv : bv >> (16 * q)));
          }
        }
      }
      if (t == kPairs - 1) decode(x1, 0);
      if constexpr (CT == 2) {
        if (t == kPairs) decode(x1, 1);
      }
      if (t == 2 * kPairs - CT - 1) {  // the next tile's first words (its copies into this wave's part have landed)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * kCopiesA + kCopiesW) : "memory");
        x0 = words(next_stage, 0);
      }
      if (t == 2 * kPairs - 1) decode(x0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    stage = next_stage;
  }
  add(2 * kPairs - 1, 0);
  add(2 * kPairs - 1, 8);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // copies past the end land before the LDS is given up
  if constexpr (EPI == kEpiLogits) {
    __syncthreads();  // the stages become the waves' own
    float* mine = (float*)sm + w * 32 * kPitch;
    const int nb = (p.N + kLpBlock - 1) / kLpBlock, valid = min(p.N - j0, 64);
#pragma unroll
    for (int i = 0; i < RT; i++) {
#pragma unroll
      for (int c = 0; c < CT; c++)
#pragma unroll
        for (int v = 0; v < 16; v++) mine[(8 * (v >> 2) + 4 * h + (v & 3)) * kPitch + 32 * c + f] = p.scale * acc[i][c][v];
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_wave_barrier();
      // lane (h, f): columns 32 h .. + 31 of row f
      float z[32];
#pragma unroll
      for (int t = 0; t < 8; t++) {
        const f4 v = *(const f4*)(mine + f * kPitch + 32 * h + 4 * t);
#pragma unroll
        for (int e = 0; e < 4; e++) z[4 * t + e] = v[e];
      }
      __builtin_amdgcn_wave_barrier();
      if (valid > 0) {
        if (valid < 64) {
#pragma unroll
          for (int t = 0; t < 32; t++) z[t] = 32 * h + t < valid ? z[t] : kNoLogit;
        }
        const LpRecord r = record_of<32, 32, 64>(z, [h](int t) { return 32 * h + t; });
        const int m = m0 + 32 * i + f;
        if (h == 0 && m < p.M) p.rec[(size_t)m * nb + (j0 >> 6)] = r;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < RT; i++) {
      const int m = m0 + 32 * i + 4 * h;  // the lane's first row; its 16 are m + 8 (v / 4) + v % 4
      if (m0 + 32 * i >= p.M) break;
      auto row_of = [](int v) { return 8 * (v >> 2) + (v & 3); };
      if (gated) {
        if constexpr (CT == 2) results<16>(p, m, j0 + f, cols, row_of, (const float*)&acc[i][0], (const float*)&acc[i][1]);
      } else {
#pragma unroll
        for (int c = 0; c < CT; c++) results<16>(p, m, j0 + 32 * c + f, cols, row_of, (const float*)&acc[i][c], nullptr);
      }
    }
  }
}

template <int BITS, bool ASYM, int EPI, int RT, int CT>
hipError_t launch_tiles(const FusedArgs& p, hipStream_t s) {
  const bool gated = EPI == kEpiAct && p.half;
  const int cols = gated ? p.half : p.N, wide = kTileWaves * (gated ? 32 : 32 * CT);
  if (CT == 1 && (gated || EPI == kEpiLogits)) return hipErrorInvalidValue;  // (a pair of column tiles a wave)
  const long tiles = (long)((cols + wide - 1) / wide) * ((p.M + 32 * RT - 1) / (32 * RT));
  if (tiles > 0x7FFFFFFFl) return hipErrorInvalidValue;
  hipLaunchKernelGGL((fused_tiles_kernel<BITS, ASYM, EPI, RT, CT>), dim3((unsigned)tiles), dim3(64 * kTileWaves), 0, s, p);
  return hipGetLastError();
}

}  // namespace
}  // namespace ha
