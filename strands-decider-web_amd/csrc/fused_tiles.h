// Products of many rows for fused.hip, gfx950: matrix-core tiles whose group sums are scaled in f32.
//
// v_mfma_f32_32x32x16_f16: lane (h = l / 32, f = l % 32) holds row f of a (A operand) or column f (B operand), k 16 h + 8 j .. + 7
// of a 32-k group for product j = 0, 1; D: column f, rows 8 (v / 4) + 4 h + v % 4. The two products of a group start from zero,
// and one fma a value adds s times their sum: 16 fma beside 64 cycles of the matrix unit, so the vector unit is the busier of the two.
// Compiled (4 bits, groups of 32), a tile and group take 24 vector instructions of 4 cycles with 4 x 2 tiles a wave, 32 with 2 x 1.
// Counted in 4 x 2 tiles: 2048 rows over 248320 tokens, the vector unit 0.84 of the time and the matrix unit 0.45 (two waves a SIMD, each
// in order, leave the rest); gated 2048 x 12288 x 2048, of which 768 workgroups at two a CU are one and a half rounds, 0.68 and 0.38.
//
// A workgroup makes 32 RT rows x 128 CT columns, a wave all of the rows and 32 CT columns (gated: 32 of the gate and the 32 of the
// up projection that they multiply). Everything comes through LDS by DMA: rows of a by 64 k, two stages, shared; packed words by
// 128 k and scales by 128 U k, two stages each, of a wave's own columns, so only a needs the barrier. The L2 hands out whole lines
// of 128 bytes, and a line of a column that is asked for in four parts, 64 k at a time, has left the L1 in between: four times
// the words' bytes and, scales 4 bytes at a time, 32 times theirs were most of what a CU fetched (2048 x 248320 x 2048: 80 KB a
// tile and workgroup, 1480 us without any arithmetic, 2415 with it; now 2330).
//
// KS = 2: twice the waves, of which half take each half of K, with stages of their own; each half then finishes half of the row tiles.
#pragma once
#include <hip/hip_runtime.h>

#include <type_traits>

#include "fused.h"
#include "fused_common.h"
#include "fused_plan.h"
#include "lds_dma.h"

namespace ha {
namespace {

typedef float f16v __attribute__((ext_vector_type(16)));
constexpr int kTileWaves = fused::kTileThreads / 64;

// A workgroup's LDS and waves a SIMD. U: 128-k pieces whose scales come together.
template <int BITS, bool ASYM, int RT, int CT, int KS>
struct TileShape {
  static constexpr int U = 4;
  static constexpr int kRows = 32 * RT, kCols = 32 * CT;
  static constexpr int kA = kRows * 128, kW = kCols * 16 * BITS, kS = kCols * 8 * U;  // stages: rows of a; a wave's words, scales
  static constexpr int kOwn = 2 * (kW + kS * (ASYM ? 2 : 1));
  static constexpr int kPitch = 68;  // of a wave's 32 x 64 results
  static constexpr int kStaged = 2 * kA + kTileWaves * kOwn, kResults = kTileWaves * 32 * kPitch * 4;
  static constexpr int kSums = KS == 1 ? 0 : kTileWaves * RT * CT * 4096;  // what two halves of K give each other
  static constexpr int kMost = kSums > kResults ? kSums : kResults, kLds = KS * kStaged > kMost ? KS * kStaged : kMost;
  static constexpr int kWaves = RT * CT > 2 || ASYM ? 2 : BITS == 4 ? 4 : 3;  // that the registers fit
};

template <int BITS, bool ASYM, int EPI, int RT, int CT, int KS, bool WHOLE>
__global__ __launch_bounds__(64 * kTileWaves * KS, (TileShape<BITS, ASYM, RT, CT, KS>::kWaves)) void fused_tiles_kernel(FusedArgs p) {
  using L = TileShape<BITS, ASYM, RT, CT, KS>;
  constexpr int kRows = L::kRows, kCols = L::kCols, kA = L::kA, kW = L::kW, kS = L::kS, U = L::U, kPitch = L::kPitch;
  constexpr int kCopiesA = kRows / 8 / kTileWaves, kCopiesW = BITS == 4 ? kCols / 16 : kCols * 4 * BITS / 64, kCopiesS = ASYM ? 4 : 2;
  __shared__ __attribute__((aligned(16))) unsigned char sm[L::kLds];
  const int tid = threadIdx.x, lane = tid & 63, f = lane & 31, h = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane((tid >> 6) % kTileWaves), ks = KS == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid / (64 * kTileWaves));
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
  // a column's blocks and scales; those of this wave's part of K
  const int nblk = p.K / 32, ng = p.K / p.group, kblk = nblk / KS, kg = ng / KS, nkt = kblk / 2;
  // rows past M repeat the last one, columns past the last likewise; neither is stored
  const unsigned last = (unsigned)(p.M - 1 - m0), k2 = 2u * (unsigned)p.K;
  const unsigned chunk = 16u * ((lane & 7) ^ (lane >> 3));  // chunk j of row r in slot j ^ (r & 7)
  const char* ap = (const char*)p.a + (size_t)m0 * p.K * 2 + (size_t)ks * kblk * 64;
  // a wave's columns: from a scalar address for each column tile, 32 bits of lane offset on
  const char *wp[CT], *sp[CT], *bp[CT];
  int left[CT];  // the last of the wave's columns of a tile
#pragma unroll
  for (int c = 0; c < CT; c++) {
    const int first = gated ? min(j0, cols - 1) + c * p.half : min(j0 + 32 * c, cols - 1);
    left[c] = (gated ? c * p.half : 0) + cols - 1 - first;
    wp[c] = (const char*)p.q + ((size_t)first * nblk + ks * kblk) * (4 * BITS);
    sp[c] = (const char*)p.s + ((size_t)first * ng + ks * kg) * 2;
    bp[c] = ASYM ? (const char*)p.b + ((size_t)first * ng + ks * kg) * 2 : sp[c];
  }
  const bool g64 = WHOLE || p.group == 64;
  unsigned char* const stage0 = sm + ks * L::kStaged;
  const unsigned lds_a = __builtin_amdgcn_readfirstlane(lds_addr(stage0) + 1024u * kCopiesA * w);
  const unsigned lds_w = __builtin_amdgcn_readfirstlane(lds_addr(stage0) + 2 * kA + L::kOwn * w), lds_s = lds_w + 2 * kW;
  auto copy_a = [&](int kt, int stage) {
    kt = min(kt, nkt - 1);  // (past the last tile: that one again, not read)
#pragma unroll
    for (int i = 0; i < kCopiesA; i++)
      dma16(lds_a + (unsigned)(stage * kA + 1024 * i), min(8u * (kCopiesA * w + i) + (lane >> 3), last) * k2 + chunk, ap + (size_t)kt * 128);
  };
  // Packed words of piece u (blocks 4 u .. + 3). 4 bits: four lanes a column, block b of column f in slot b ^ (f / 4 % 4) of the
  // column's four, so that reads of 32 columns fall in distinct banks; else word by word
  auto copy_w = [&](int u, int stage) {
    u = min(u, (nkt - 1) / 2);
    const unsigned to = lds_w + (unsigned)(stage * kW);
    const int blocks = min(4, kblk - 4 * u);  // (the last piece may have two)
#pragma unroll
    for (int i = 0; i < kCopiesW; i++) {
      if constexpr (BITS == 4) {
        const int f0 = 16 * (i & 1) + (lane >> 2), c = i >> 1;
        const unsigned blk = min((lane & 3) ^ ((f0 >> 2) & 3), blocks - 1);
        dma16(to + 1024 * i, (unsigned)min(f0, left[c]) * (unsigned)nblk * 16u + 16u * blk, wp[c] + (size_t)u * 64);
      } else {
        constexpr int kWords = 4 * BITS, kEach = 32 * kWords / 64;  // a column's words; instructions of a column tile
        const int x = 64 * (i % kEach) + lane, f0 = x / kWords, c = i / kEach;
        dma4(to + 256 * i, ((unsigned)min(f0, left[c]) * (unsigned)nblk * BITS + min(x % kWords, blocks * BITS - 1)) * 4u, wp[c] + (size_t)u * (16 * BITS));
      }
    }
  };
  // Two of the 2 U instructions that bring U pieces' scales (groups of 64: 2 U pieces'), pairs of f16, column by column
  auto copy_s = [&](int part, int piece, int stage) {
    constexpr int kPairs = 2 * U;
    part = min(part, (kg / 2 - 1) / kPairs);
    const unsigned to = lds_s + (unsigned)(stage * kS * (ASYM ? 2 : 1)) + 256u * piece;
    const int x = 64 * piece + lane, f0 = x / kPairs % 32;
    const unsigned pair = min(x % kPairs, kg / 2 - 1 - part * kPairs);
    const bool second = CT == 2 && x >= 32 * kPairs;
    const unsigned at = (unsigned)min(f0, second ? left[CT - 1] : left[0]) * (unsigned)ng * 2u + 4u * pair;
    const char* from = (second ? sp[CT - 1] : sp[0]) + (size_t)part * (4 * kPairs);
    dma4_at(to, from + at);
    if constexpr (ASYM) dma4_at(to + kS, (second ? bp[CT - 1] : bp[0]) + (size_t)part * (4 * kPairs) + at);
  };
  constexpr int kPieces = kCols * 2 * U / 64;  // instructions for U pieces' scales
  const int per_part = g64 ? 2 * U : U;        // pieces u of a part
  // the words of group g of tile kt = 2 u + q as codes8 takes them
  struct Words {
    unsigned lo[CT][2], hi[CT][2];
  };
  const unsigned char* const own = stage0 + 2 * kA + L::kOwn * w;
  auto words = [&](int stage, int block) {
    const unsigned char* from = own + stage * kW;
    Words x;
#pragma unroll
    for (int c = 0; c < CT; c++) {
      if constexpr (BITS == 4) {
        const uint2 v = *(const uint2*)(from + 64 * (32 * c + f) + 16 * (block ^ ((f >> 2) & 3)) + 8 * h);  // k 16 h .. + 15 of the group
        x.lo[c][0] = v.x, x.lo[c][1] = v.y, x.hi[c][0] = x.hi[c][1] = 0;
      } else {
        const unsigned char* at = from + 4 * (4 * BITS * (32 * c + f) + BITS * block);
        const unsigned v = *(const unsigned*)(at + 4 * h), t = BITS == 3 ? *(const unsigned*)(at + 8) >> (16 * h) : 0u;
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
  static_assert(!WHOLE || (RT == 2 && CT == 1), "a group's sums wait in d and sum");
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
  // Copies complete in order. At the top of tile 2 u those of a(2 u), words and scales of piece u have landed (nothing newer is in
  // flight); at the top of 2 u + 1 those of a(2 u + 1), issued at the top of 2 u before the next piece's words and scales. Behind
  // the barrier everybody's have, and everybody has read the tile before, whose stage takes the next one.
  Words x0;
  auto tile = [&](auto parity, int kt, int ws, int ss) {
    constexpr int q = decltype(parity)::value;
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(q ? kCopiesW + kCopiesS : 0) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    copy_a(kt + 1, q ^ 1);
    if (q == 0) {
      const int u = kt >> 1, in_part = u % per_part, part = u / per_part + 1;
      copy_w(u + 1, ws ^ 1);
      // (groups of 64 have twice the time: a piece of them twice; one column tile has half the pieces: each twice)
      const int piece = g64 ? in_part : 2 * in_part;
      copy_s(part, piece % kPieces, ss ^ 1);
      copy_s(part, (g64 ? piece : piece + 1) % kPieces, ss ^ 1);
    }
    const unsigned char* as = stage0 + q * kA + arow;
    auto operand = [&](int g, int i, int j) { return *(const h8*)(as + 32 * 128 * i + 16 * ((4 * g + 2 * h + j) ^ (f & 7))); };
    af[0][0] = operand(0, 0, 0);
    af[0][1] = operand(0, 0, 1);
    if (q == 0 && kt == 0) {
      x0 = words(0, 0);
      decode(x0, 0);
    }
    unsigned sw[CT], bw[CT];
    const int pair = g64 ? (kt >> 1) % (2 * U) : kt % (2 * U);
#pragma unroll
    for (int c = 0; c < CT; c++) {
      const unsigned char* at = own + 2 * kW + ss * kS * (ASYM ? 2 : 1) + 8 * U * (32 * c + f) + 4 * pair;
      sw[c] = *(const unsigned*)at;
      bw[c] = ASYM ? *(const unsigned*)(at + kS) : 0u;
    }
    Words x1;
    // The pairs of both groups in turn: a pair's two products go with the fma of the pair before (of a tile's first, with those of
    // the last tile's last), with the next row tile's reads and the next group's decoding
#pragma unroll
    for (int t = 0; t < 2 * kPairs; t++) {
      const int c = t % CT, v = (t / CT) & 1, before = t == 0 ? 2 * kPairs - 1 : t - 1;
      const bool on = WHOLE && t >= kPairs, due = !WHOLE || before >= kPairs;  // (a tile is a group: its second 32 k go onto the first's sums)
      if constexpr (ASYM) {
        if (c == 0) {
          sum[v] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[v][0], ones8(), on ? sum[v] : f16v{}, 0, 0, 0);
          sum[v] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[v][1], ones8(), sum[v], 0, 0, 0);
        }
      }
      d[t & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[v][0], bf[c][0], on ? d[t & 1] : f16v{}, 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      if (c == 0 && t + CT < 2 * kPairs) {
        af[v ^ 1][0] = operand((t + CT) / kPairs, (t + CT) / CT % RT, 0);
        af[v ^ 1][1] = operand((t + CT) / kPairs, (t + CT) / CT % RT, 1);
      }
      if (t == CT - 1) x1 = words(ws, 2 * q + 1);
      if (due) add(before, 0);
      __builtin_amdgcn_sched_barrier(0);
      d[t & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[v][1], bf[c][1], d[t & 1], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      if (due) add(before, 8);
      if (t == 0) {  // (the last tile's scales are done with)
        if constexpr (CT == 2) decode(x0, 1);
#pragma unroll
        for (int n = 0; n < CT; n++) {
          const unsigned sv = g64 ? sw[n] >> (16 * q) : sw[n], bv = g64 ? bw[n] >> (16 * q) : bw[n];
#pragma unroll
          for (int e = 0; e < 2; e++) {
            s[e][n] = f16_bits(g64 ? sv : sv >> (16 * e));
            if constexpr (ASYM) b[e][n] = centred<BITS>(s[e][n], f16_bits(g64 ? bv : bv >> (16 * e)));
          }
        }
      }
      if (t == kPairs - 1) decode(x1, 0);
      if constexpr (CT == 2) {
        if (t == kPairs) decode(x1, 1);
      }
      if (t == 2 * kPairs - CT - 1) {  // the next tile's first words: of this piece, or of the next, whose copies have landed
        if (q) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kCopiesA) : "memory");
        x0 = words(q ? ws ^ 1 : ws, q ? 0 : 2);
      }
      if (t == 2 * kPairs - 1) decode(x0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  for (int i = 0; i < kPieces; i++) copy_s(0, i, 0);
  copy_w(0, 0);
  copy_a(0, 0);
  int ws = 0, ss = 0;
  int kt = 0;
  for (; kt + 2 <= nkt; kt += 2) {
    tile(std::integral_constant<int, 0>{}, kt, ws, ss);
    tile(std::integral_constant<int, 1>{}, kt + 1, ws, ss);
    ws ^= 1;
    if ((kt / 2 + 1) % per_part == 0) ss ^= 1;
  }
  if (kt < nkt) tile(std::integral_constant<int, 0>{}, kt, ws, ss);
  add(2 * kPairs - 1, 0);
  add(2 * kPairs - 1, 8);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // copies past the end land before the LDS is given up
  if constexpr (EPI == kEpiLogits) {
    __syncthreads();  // the stages become the waves' own, or those of two waves that share blocks of 64 columns
    const int nb = (p.N + kLpBlock - 1) / kLpBlock, part = CT == 2 ? 0 : w & 1, first = j0 - 32 * part, valid = min(p.N - first, 64);
    float* mine = (float*)sm + (CT == 2 ? w : w & ~1) * 32 * kPitch;
    // row tile i, columns 32 n + f of the block
    auto put = [&](float* to, int i, int c, int n) {
#pragma unroll
      for (int v = 0; v < 16; v++) to[(8 * (v >> 2) + 4 * h + (v & 3)) * kPitch + 32 * n + f] = p.scale * acc[i][c][v];
    };
    auto record = [&](const float* from, int i) {  // lane (h, f): columns 32 h .. + 31 of row f
      float z[32];
#pragma unroll
      for (int t = 0; t < 8; t++) {
        const f4 v = *(const f4*)(from + f * kPitch + 32 * h + 4 * t);
#pragma unroll
        for (int e = 0; e < 4; e++) z[4 * t + e] = v[e];
      }
      if (valid < 64) {
#pragma unroll
        for (int t = 0; t < 32; t++) z[t] = 32 * h + t < valid ? z[t] : kNoLogit;
      }
      const LpRecord r = record_of<32, 32, 64>(z, [h](int t) { return 32 * h + t; });
      const int m = m0 + 32 * i + f;
      if (h == 0 && m < p.M) p.rec[(size_t)m * nb + (first >> 6)] = r;
    };
    if constexpr (CT == 2) {
#pragma unroll
      for (int i = 0; i < RT; i++) {
        put(mine, i, 0, 0);
        put(mine, i, 1, 1);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        if (valid > 0) record(mine, i);
        __builtin_amdgcn_wave_barrier();
      }
    } else {  // two row tiles at a time, one for each wave of a pair
#pragma unroll
      for (int i = 0; i < RT; i += 2) {
        put(mine, i, 0, part);
        if constexpr (RT > 1) {
          if (i + 1 < RT) put(mine + 32 * kPitch, i + 1 < RT ? i + 1 : i, 0, part);
        }
        __syncthreads();
        if (valid > 0 && i + part < RT) record(mine + 32 * kPitch * part, i + part);
        if (i + 2 < RT) __syncthreads();
      }
    }
  } else {
    auto row_of = [](int v) { return 8 * (v >> 2) + (v & 3); };
    auto store = [&](int i) __attribute__((always_inline)) {
      const int m = m0 + 32 * i + 4 * h;  // the lane's first row; its 16 are m + 8 (v / 4) + v % 4
      if (m0 + 32 * i >= p.M) return;
      if (gated) {
        if constexpr (CT == 2) results<16>(p, m, j0 + f, cols, row_of, (const float*)&acc[i][0], (const float*)&acc[i][1]);
      } else {
#pragma unroll
        for (int c = 0; c < CT; c++) results<16>(p, m, j0 + 32 * c + f, cols, row_of, (const float*)&acc[i][c], nullptr);
      }
    };
    if constexpr (KS == 1) {
#pragma unroll
      for (int i = 0; i < RT; i++) store(i);
    } else {  // each half of K finishes half of the row tiles: it takes the other's sums of those and gives its own of the rest
      f16v* const give = (f16v*)sm + (size_t)w * RT * CT * 64 + lane;
      __syncthreads();  // the stages have been read
      auto meet = [&](auto half) __attribute__((always_inline)) {
        constexpr int H = decltype(half)::value, R = RT / 2;
#pragma unroll
        for (int i = 0; i < R; i++)
#pragma unroll
          for (int c = 0; c < CT; c++) give[((R * (1 - H) + i) * CT + c) * 64] = acc[R * (1 - H) + i][c];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < R; i++) {
#pragma unroll
          for (int c = 0; c < CT; c++) acc[R * H + i][c] += give[((R * H + i) * CT + c) * 64];
          store(R * H + i);
        }
      };
      if (ks == 0) meet(std::integral_constant<int, 0>{});
      else meet(std::integral_constant<int, 1>{});
    }
  }
}

// KS = 2 takes K of whole parts of scales for each half (512 k, with groups of 64 1024).
template <int BITS, bool ASYM, int EPI, int RT, int CT, int KS = 1>
hipError_t launch_tiles(const FusedArgs& p, hipStream_t s) {
  if (KS == 2 && p.K % (32 * p.group) != 0) return hipErrorInvalidValue;
  const bool gated = EPI == kEpiAct && p.half;
  const int cols = gated ? p.half : p.N, wide = kTileWaves * (gated ? 32 : 32 * CT);
  if (CT == 1 && gated) return hipErrorInvalidValue;  // (a pair of column tiles a wave)
  const long tiles = (long)((cols + wide - 1) / wide) * ((p.M + 32 * RT - 1) / (32 * RT));
  if (!fused::fits(tiles, 64 * kTileWaves * KS)) return hipErrorInvalidValue;
  // Groups of 64 are a tile's 64 k: where the pairs' sums have registers, both halves are one sum, scaled once
  auto k = fused_tiles_kernel<BITS, ASYM, EPI, RT, CT, KS, false>;
  if constexpr (RT == 2 && CT == 1) {
    if (p.group == 64) k = fused_tiles_kernel<BITS, ASYM, EPI, RT, CT, KS, true>;
  }
  hipLaunchKernelGGL(k, dim3((unsigned)tiles), dim3(64 * kTileWaves * KS), 0, s, p);
  return hipGetLastError();
}

}  // namespace
}  // namespace ha
