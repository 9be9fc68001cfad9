// Which kernel serves a product whose results are not stored as they are (fused.hip), with which tiles: host code from sizes and
// formats alone (no HIP, so that a test can compile it by itself).
#pragma once
#include <algorithm>

namespace ha {
namespace fused {

enum Path { kAny, kRows, kTiles };
struct Shape {
  int M, cols, K;  // cols: of the result
  bool gated, asym;
  bool whole;      // K and alignment as the kernels that move whole 64-k tiles need them
};
// Rows: 16 a x 16 b columns of weights a workgroup. Tiles: 32 a rows, 128 b columns of weights. us: the time this is expected to take.
struct Plan {
  Path path;
  int a, b;
  float us;
};

// Workgroups of a product with tiles of `rows` x `weights` columns of weights.
inline long groups(const Shape& p, int rows, int weights) {
  const int wide = p.gated ? weights / 2 : weights;
  return (long)((p.cols + wide - 1) / wide) * ((p.M + rows - 1) / rows);
}

// The rows kernel: rounds of 256 workgroups, each of which takes as long as the rows of a and columns of W that it reads. Measured,
// us, 4 bits, K = 2048 unless said (cost: rounds x (a + b + 2)): 61 x 5120 4 x 2 7.6 (8), 512 x 5120 4 x 2 27 (40), 2048 x 2048
// 4 x 2 41 (64), 512 x 2048 x 6144 4 x 4 27 (10), 2048 x 2048 x 6144 4 x 4 97 (40), 61 x 2048 x 6144 1 x 2 9.0 (5).
inline float rows_us(const Shape& p, int a, int b) {
  const float x = p.K / 2048.0f;
  return 2.0f + (float)((groups(p, 16 * a, 16 * b) + 255) / 256) * (a + b + 2) * (0.1f + 0.5f * x + 0.08f * x * x);
}
// The tile kernel: a workgroup takes b_us of a CU's time, and one alone a_us more. Measured, us, 4 bits, K = 2048, for n workgroups
// on the busiest CU: 4 x 2 n = 1 50, 2 71, 3 106; 2 x 2 31, 45, 70, n = 6 128; 4 x 1 30, 45, 67; 2 x 1 19, 33, 43, n = 5 67.
inline float tiles_us(const Shape& p, int a, int b) {
  const float alone = a * b == 8 ? 15.0f : a * b == 2 ? 6.0f : 9.0f, each = a * b == 8 ? 32.0f : a * b == 2 ? 12.5f : 20.5f;
  return p.K / 2048.0f * (alone + each * (float)((groups(p, 32 * a, 128 * b) + 255) / 256)) * (p.asym ? 1.5f : 1.0f);
}

inline Plan plan(const Shape& p) {
  if (!p.whole) return {kAny, 0, 0, 0.0f};
  Plan best{kAny, 0, 0, 1e30f};
  auto look = [&](Path path, int a, int b, float us) {
    if (us < best.us) best = {path, a, b, us};
  };
  for (int a : {1, 2, 4})
    for (int b : {1, 2, 4})
      if (!p.gated || b > 1) look(kRows, a, b, rows_us(p, a, b));  // (gated: tiles of both halves)
  for (int a : {2, 4})
    for (int b : {1, 2})
      if ((!p.gated || b == 2) && !(p.asym && a * b == 8)) look(kTiles, a, b, tiles_us(p, a, b));  // (asymmetric 4 x 2: too many registers)
  return best;
}

}  // namespace fused
}  // namespace ha
