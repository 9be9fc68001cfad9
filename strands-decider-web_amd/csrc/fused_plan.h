// Which kernel serves a product whose results are not stored as they are (fused.hip), with which tiles: host code from sizes and
// formats alone (no HIP, so that a test can compile it by itself).
#pragma once
#include <algorithm>
#include <cstddef>

namespace ha {
namespace fused {

enum Path { kAny, kRows, kTiles, kLanes };
struct Shape {
  int M, cols, K;  // cols: of the result
  bool gated, asym;
  bool whole;      // K and alignment as the kernels that move whole 64-k tiles need them
  bool halves;     // K / 2 is whole pieces of the tile kernel's scales
  int bits = 4;
};
// Rows: 16 a x 16 b columns of weights a workgroup. Tiles: 32 a rows, 128 b columns of weights, `halves` of K. us: the time this is
// expected to take.
struct Plan {
  Path path;
  int a, b;
  float us;
  int halves = 1;
};

constexpr int kLanesRows = 2, kLanesValues = 32768;  // rows and values of a that the lanes kernel takes

// Workgroups of a product with tiles of `rows` x `weights` columns of weights.
inline long groups(const Shape& p, int rows, int weights) {
  const int wide = p.gated ? weights / 2 : weights;
  return (long)((p.cols + wide - 1) / wide) * ((p.M + rows - 1) / rows);
}

// A launch has fewer than 2^32 threads (HIP's limit).
inline bool fits(long workgroups, int threads) { return workgroups <= ((1l << 32) - 1) / threads; }
// Threads of a workgroup. The rows kernel splits a long K of few rows over 16 waves where its workgroups are the fewest (1 x 1 tiles of
// 2048 x 6144: 1 row 7.0 -> 6.1 us, 16 rows 7.4 -> 7.2; 2048 x 2048, 4.1 -> 4.3).
constexpr int kAnyThreads = 512, kLanesThreads = 256, kTileThreads = 256;
inline int rows_waves(int M, int K, int a, int b) { return a == 1 && b == 1 && K >= 4096 && M <= 16 ? 16 : 8; }
inline long any_groups(const Shape& p) { return groups(p, 16, 64); }
inline long lanes_groups(const Shape& p) { return groups(p, kLanesRows, 8); }
inline bool launchable(const Shape& p, const Plan& x) {
  switch (x.path) {
    case kAny: return fits(any_groups(p), kAnyThreads);
    case kLanes: return fits(lanes_groups(p), kLanesThreads);
    case kRows: return fits(groups(p, 16 * x.a, 16 * x.b), 64 * rows_waves(p.M, p.K, x.a, x.b));
    case kTiles: return fits(groups(p, 32 * x.a, 128 * x.b), x.halves * kTileThreads);
  }
  return false;
}
// Rows of the first of two launches for a call that no kernel takes in one (0: it cannot be parted).
inline int first_part(int M) { return M > 16 ? (M / 2 + 15) / 16 * 16 : 0; }

// What asymmetric weights and 3 bits cost where arithmetic counts: 1744 x 2560 x 2560, us, rows 4 x 2 and tiles 2 x 1, 4 bits 56 and 49,
// asymmetric 75 and 74, 3 bits 74 and 58, both 84 and 88 (2 bits as 4).
inline float rows_cost(const Shape& p) { return 1.0f + (p.asym ? 0.35f : 0.0f) + (p.bits == 3 ? 0.3f : 0.0f); }
inline float tiles_cost(const Shape& p) { return 1.0f + (p.asym ? 0.45f : 0.0f) + (p.bits == 3 ? 0.25f : 0.0f); }

// Both fitted to 1 to 2048 rows of 2048 to 12288 columns at K = 192 to 6144 (4 bits, groups of 32; r.m.s. error 12 and 9 %); what
// they choose is 3 % slower than the best of all shapes in the mean. n: workgroups on the busiest of 256 CUs.
// The rows kernel: a workgroup's time grows with the rows of a and columns of W that it reads and the results that it writes. Shapes
// of 12 tiles and more run one to a CU. us, a x b: 1 row, gated 12288 x 2048 1 x 3 6.9, 1 x 4 7.5; 61 rows 4 x 3 10.6, 4 x 4 11.1,
// 2 x 4 12.6; 256 rows, 2048 x 2048 4 x 2 7.8, 2 x 4 8.6; 512 rows, 2048 x 6144 4 x 4 26, 4 x 2 29.
inline float rows_us(const Shape& p, int a, int b) {
  const float x = p.K / 2048.0f, n = (float)((groups(p, 16 * a, 16 * b) + 255) / 256);
  const float each = x * (0.51f * a + 0.73f * b - 0.2f) + 0.26f + 0.09f * a + 0.145f * a * b;
  return 2.85f + 0.18f * x + (1.0f + (n - 1.0f) * (a * b >= 12 ? 1.34f : 0.87f)) * each * rows_cost(p);
}
// The tile kernel. us: 512 rows, gated 12288 x 2048 2 x 2 43.5, 4 x 2 43.7 (rows kernel 54); 2048 rows 119, 100; 1024 rows, 2048 x
// 2048 2 x 1 21, 4 x 1 31, 2 x 2 32 (rows kernel 22); 2048 rows, 2048 x 6144 2 x 1 76, 4 x 1 76, 2 x 2 82, 4 x 2 121; 512 rows,
// 12288 x 192 2 x 1 12, 4 x 1 16 (rows kernel 26).
inline float tiles_us(const Shape& p, int a, int b) {
  const float n = (float)((groups(p, 32 * a, 128 * b) + 255) / 256), x = p.K / 2048.0f * tiles_cost(p);
  const float k = a == 4 ? (b == 2 ? 21.8f + 12.5f * n : 10.3f + 11.4f * n) : a == 3 ? (b == 2 ? 5.4f + 17.5f * n : 8.0f + 8.7f * n)
                         : (b == 2 ? 11.5f + 11.3f * n : 8.2f + 6.35f * n);
  return 2.6f + x * k + 1.46f * a * b * n;
}

// Tiles of 64 x 128 by twice the waves, half of them for each half of K: for products of few workgroups, which leave the vector unit
// waiting. us, against whole K: 1024 rows, 2048 x 2048 17.8 (22.1), 2048 x 6144 43.4 (51.9); 2048 rows 28.8 (32.5), 65 (75); 512 rows,
// 4096 x 4096 31 (36); 2048 rows, 12288 x 1024 86 (77). 128 x 128 by halves has 29.2, 64 and 43 where this has 28.8, 65 and 31.
inline float halves_us(const Shape& p) {
  const float n = (float)((groups(p, 64, 128) + 255) / 256), x = p.K / 2048.0f * tiles_cost(p);
  return 2.6f + x * (3.1f + 8.0f * n) + 2.4f * n;
}
// The lanes kernel (one or two rows that fit 64 KiB of LDS; any alignment). Times in fused_lanes.h; each 2048 k are a step, each 2048
// columns a wave on every SIMD.
inline float lanes_us(const Shape& p) {
  const float x = std::max(1.0f, p.K / 2048.0f), n = std::max(1.0f, p.cols * (p.gated ? 2.0f : 1.0f) / 2048.0f);
  return p.M == 1 ? 2.1f + 0.75f * x + 0.6f * (n - 1.0f) * x : 2.2f + x + 0.85f * (n - 1.0f) * x;
}

// The fastest kernel, or the fastest of those that one launch suffices for.
inline Plan fastest(const Shape& p, bool one_launch) {
  const bool lanes = p.M <= kLanesRows && p.M * p.K <= kLanesValues;
  Plan best{kAny, 0, 0, 1e30f};
  auto look = [&](Path path, int a, int b, float us, int halves = 1) {
    const Plan x{path, a, b, us, halves};
    if (us < best.us && (!one_launch || launchable(p, x))) best = x;
  };
  if (!p.whole) {
    if (lanes) look(kLanes, 0, 0, 0.0f);
    else best.us = 0.0f;
    return best;
  }
  if (lanes) look(kLanes, 0, 0, lanes_us(p));
  for (int a : {1, 2, 4})
    for (int b : {1, 2, 3, 4}) look(kRows, a, b, rows_us(p, a, b));
  for (int a : {2, 3, 4})
    for (int b : {1, 2})
      if ((!p.gated || b == 2) && !(p.asym && a * b > 4)) look(kTiles, a, b, tiles_us(p, a, b));  // (asymmetric 3 x 2, 4 x 2: too many registers)
  // (asymmetric: one such workgroup fits a CU)
  if (p.halves && !p.gated && (!p.asym || groups(p, 64, 128) <= 256)) look(kTiles, 2, 1, halves_us(p), 2);
  return best;
}
inline Plan plan(const Shape& p) {
  const Plan best = fastest(p, false);
  return launchable(p, best) ? best : fastest(p, true);
}

// The tile kernel's shape for logits, of so many columns that rounds of workgroups count for little: base + each for every 32 a rows.
// Fitted to 98304 x 2048, us (4 bits; symmetric, then asymmetric), 61 rows 2 x 1 38, 2 x 2 46, 1 x 1 50; 58, 63, 66; 128 rows 4 x 1
// 60, 2 x 1 65, 4 x 2 70; 92, 103, -; 192 rows 3 x 1 89, 2 x 1 91, 4 x 2 101; 138, 149, -; 512 rows 4 x 2 188, 4 x 1 213, 2 x 1 226;
// -, 333, 391. One column tile leaves room for twice the waves.
inline Plan logit_tiles(int M, bool asym) {
  const struct { int a, b; float base, each; } shapes[] = {{1, 1, 10.0f, 20.3f}, {2, 1, 11.5f, 26.8f}, {3, 1, 10.0f, 39.4f}, {4, 1, 10.0f, 51.0f}, {4, 2, 25.0f, 42.0f}};
  Plan best{kTiles, 0, 0, 1e30f};
  for (const auto& x : shapes) {
    const float us = x.base + x.each * (float)((M + 32 * x.a - 1) / (32 * x.a));
    if (us < best.us && !(asym && x.b == 2)) best = {kTiles, x.a, x.b, us};
  }
  return best;
}

// Whether one launch makes a call's records. Vocabularies are up to 2^20: 16 rows always fit.
inline bool logits_fit(int M, int n_vocab, bool whole, bool asym) {
  const Shape p{M, n_vocab, 64, false, asym, whole, false};
  if (!whole) return fits(any_groups(p), kAnyThreads);
  const Plan x = logit_tiles(M, asym);
  return fits(groups(p, 32 * x.a, 128 * x.b), kTileThreads);
}

// Whether log probabilities store the logits (f32) and read them back rather than leave records of 64 columns: in vocabularies up
// to 32768 for few rows, where the records' kernels are few workgroups, and where more than one block in two rows would hold two
// of the top_k largest, which costs 62 products in 64 bits each. Measured, us, records : stored: 1431 x 1383 x 256 top 20 1125 :
// 51, 1 x 4284 x 640 (3 bits) top 32 178 : 25, 187 x 2507 x 4096 (3 bits) 114 : 35, 605 x 20658 x 192 top 20 108 : 106; the other
// way, 2048 x 32768 x 2048 top 5 372, stored (top 30) 616; 1024 x 8192 x 2048 top 5 98, stored (top 12) 97.
constexpr int kStoredVocab = 32768;
// The rows of a call up to which that is (0: none).
inline int stored_rows(int n_vocab, int top_k) {
  if (n_vocab > kStoredVocab) return 0;
  if (top_k * top_k > (n_vocab + 63) / 64) return 0x7FFFFFFF;
  return 255 / ((n_vocab + 255) / 256) * 128;  // fewer than 256 tiles of 128 x 256
}
inline bool store_logits(int M, int n_vocab, int top_k) { return M <= stored_rows(n_vocab, top_k); }
// Rows whose logits are stored at a time: 1 GiB of them, whole tiles.
inline int stored_part(int n_vocab) { return (1 << 28) / n_vocab / 128 * 128; }

// Bytes that a call's logits or records take.
inline size_t logits_bytes(int M, int n_vocab, int top_k) {
  if (store_logits(M, n_vocab, top_k)) return (size_t)std::min(M, stored_part(n_vocab)) * n_vocab * 4;
  return (size_t)M * ((n_vocab + 63) / 64) * 16;
}
// The most that a call of up to M rows takes: logits are 16 times the records' bytes, so fewer rows, where they are stored, may take more.
inline size_t most_logits_bytes(int M, int n_vocab, int top_k) {
  const int stored = std::min(M, stored_rows(n_vocab, top_k));
  return std::max(logits_bytes(M, n_vocab, top_k), stored > 0 ? logits_bytes(stored, n_vocab, top_k) : 0);
}

}  // namespace fused
}  // namespace ha
