// The paged cache of 4-bit keys and values of the full-attention layers, gfx950: appending a batch's rows to it, with q's
// and k's norms and rotation on the way (kv_attn.hip reads it).
//
// A row (one token and KV head) is 4 groups of G = HD / 4 consecutive channels, each with a scale s and a zero z in f16:
//   channel value = s (c - 8) + z, code c in 0..15
//   z = f16(lo + (hi - lo) 8/15), s = f16(max((hi - z) / 7, (z - lo) / 8)), c = clamp(rint((x - z) / s) + 8, 0, 15)
// for the group's least and largest values lo, hi: the nearest code is at most s / 2 off (but for the rounding of s).
// Codes stand in nibbles, channel (group g, 4 i + e) of the row in nibble 16 i + 4 g + e: a 16-bit half-word holds four
// channels of one group, so a lane that reads 8 bytes of a row has 4 channels of each group.
#include <cmath>
#include <type_traits>

#include "kv_common.h"

namespace ha {
namespace {

__global__ void kv_rope_kernel(float* rope, const double* theta_pow, int n, int half) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long)n * half) return;
  const double ang = (double)(i / half) / theta_pow[i % half];
  rope[2 * i] = (float)cos(ang);
  rope[2 * i + 1] = (float)sin(ang);
}

// ---- append ----
//
// A lane has 8 consecutive channels of a row, HD / 8 lanes a row, a wave 64 / (HD / 8) rows of one head at a time; a group's
// channels are in HD / 32 neighbouring lanes. All sums and extremes are DPP steps, and a rotated channel's partner is loaded
// once more instead of exchanged, so that only the norms' factors go through LDS. It is bound by memory where there are many rows
// (16384 of the model's heads, 211 MB: 53.8 us, 3.9 TB/s, on new buffers, 46.6 on the same ones again, where a copy reaches 4.8)
// and by a chain of loads where there are few (one row each of 8 sequences: 3.3 us, in a graph of such calls).

typedef unsigned u2v __attribute__((ext_vector_type(2)));
template <int kCtrl>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), kCtrl, 0xf, 0xf, false));
}
template <int kCtrl>
__device__ __forceinline__ double dpp(double v) {
  u2v u = __builtin_bit_cast(u2v, v);
  u[0] = (unsigned)__builtin_amdgcn_mov_dpp((int)u[0], kCtrl, 0xf, 0xf, false);
  u[1] = (unsigned)__builtin_amdgcn_mov_dpp((int)u[1], kCtrl, 0xf, 0xf, false);
  return __builtin_bit_cast(double, u);
}
__device__ __forceinline__ float other_row(float v, float& w) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
  w = __builtin_bit_cast(float, (unsigned)r[1]);
  return __builtin_bit_cast(float, (unsigned)r[0]);
}
__device__ __forceinline__ double other_row(double v, double& w) {
  const u2v u = __builtin_bit_cast(u2v, v);
  const auto lo = __builtin_amdgcn_permlane16_swap(u[0], u[0], false, false), hi = __builtin_amdgcn_permlane16_swap(u[1], u[1], false, false);
  w = __builtin_bit_cast(double, u2v{(unsigned)lo[1], (unsigned)hi[1]});
  return __builtin_bit_cast(double, u2v{(unsigned)lo[0], (unsigned)hi[0]});
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kHalfMirror = 0x141, kMirror = 0x140;  // quad_perm 1 0 3 2, 2 3 0 1; lanes 7 - i, 15 - i of 8, 16
// sum over the LANES (16 or 32) lanes of a row
template <int LANES, typename F>
__device__ __forceinline__ F row_sum(F v) {
  v += dpp<kXor1>(v);
  v += dpp<kXor2>(v);
  v += dpp<kHalfMirror>(v);
  v += dpp<kMirror>(v);
  if constexpr (LANES == 32) {
    F w;
    v = other_row(v, w);
    v += w;
  }
  return v;
}

template <typename T>
struct Eight;  // 8 consecutive channels of a row in memory
template <>
struct Eight<_Float16> {
  h8 v;
  __device__ __forceinline__ void load(const _Float16* p) { v = *gp<h8>(p); }
  __device__ __forceinline__ float operator[](int e) const { return (float)v[e]; }
  __device__ __forceinline__ float squares() const {
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e += 2) s = __builtin_amdgcn_fdot2(h2{v[e], v[e + 1]}, h2{v[e], v[e + 1]}, s, false);
    return s;
  }
};
template <>
struct Eight<float> {
  f4 a, b;
  __device__ __forceinline__ void load(const float* p) { a = ld4(p); b = ld4(p + 4); }
  __device__ __forceinline__ float operator[](int e) const { return e < 4 ? a[e] : b[e - 4]; }
  __device__ __forceinline__ float squares() const {
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) s = fmaf((*this)[e], (*this)[e], s);
    return s;
  }
};

// What rotation needs of a lane's two quads of channels (c .. c + 3): whether they are rotated and in the first half, where the
// partner channels are, and their gains.
struct Turn {
  bool in[2], first[2];
  int other[2], angle[2];
  __device__ __forceinline__ Turn(int c, int rot) {
#pragma unroll
    for (int n = 0; n < 2; n++) {
      const int x = c + 4 * n;
      in[n] = x < rot;
      first[n] = x < rot / 2;
      other[n] = !in[n] ? x : first[n] ? x + rot / 2 : x - rot / 2;
      angle[n] = !in[n] ? 0 : 2 * (first[n] ? x : x - rot / 2);
    }
  }
};

// x inv w, rotated; py: the partner channels' values, wp their gains, cs the four channels' (cos, sin). F is float for q, which is
// rounded to f16, and double for k: a key next to the border between two codes then falls on the same side whatever the order of
// the sum.
template <typename F, typename X>
__device__ __forceinline__ void scale_rotate(const X& x, F inv, const f4* w, const Turn& tn, const f4* py, const f4* wp, const f4* cs, F* y) {
#pragma unroll
  for (int e = 0; e < 8; e++) y[e] = (F)x[e] * (inv * (F)w[e >> 2][e & 3]);
#pragma unroll
  for (int n = 0; n < 2; n++)
    if (tn.in[n]) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const f4 c = cs[2 * n + (e >> 1)];
        const F other = (F)py[n][e] * (inv * (F)wp[n][e]), sn = (F)c[2 * (e & 1) + 1];
        y[4 * n + e] = y[4 * n + e] * (F)c[2 * (e & 1)] + (tn.first[n] ? -other : other) * sn;
      }
    }
}

// The group's scale, zero and this lane's eight codes (see the top). Every operation is rounded by itself (no contraction): the
// codes are a function of the values alone. The quotient by s is a product with 1 / s and one correction by the exact remainder,
// which gives the rounded quotient (Markstein: the reciprocal is correctly rounded, s has few bits).
// c: code - 8.
template <int HD>
__device__ __forceinline__ void quantise(const float* x, _Float16& s16, _Float16& z16, float* c) {
#pragma clang fp contract(off)
  float lo = x[0], hi = x[0], bad = x[0] * 0.0f;  // bad: NaN where a value is not finite
#pragma unroll
  for (int e = 1; e < 8; e++) {
    lo = fminf(lo, x[e]);
    hi = fmaxf(hi, x[e]);
    bad = fmaf(x[e], 0.0f, bad);
  }
  auto step = [&](auto ctrl) {
    constexpr int k = decltype(ctrl)::value;
    lo = fminf(lo, dpp<k>(lo));
    hi = fmaxf(hi, dpp<k>(hi));
    bad += dpp<k>(bad);
  };
  step(std::integral_constant<int, kXor1>{});
  step(std::integral_constant<int, kXor2>{});
  if constexpr (HD == 256) step(std::integral_constant<int, kHalfMirror>{});
  const float range = hi - lo;
  z16 = (_Float16)(lo + range * (float)(8.0 / 15.0));
  const float z = (float)z16;
  s16 = (_Float16)fmaxf((hi - z) * (float)(1.0 / 7.0), (z - lo) * 0.125f);
  const float s = (float)s16, r = 1.0f / s;
  const bool fine = bad == 0.0f && fabsf(s) < INFINITY && fabsf(z) < INFINITY, some = fine && s > 0.0f;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const float d = x[e] - z, q = d * r, t = fmaf(fmaf(-q, s, d), r, q);
    c[e] = some ? __builtin_amdgcn_fmed3f(rintf(t), -8.0f, 7.0f) : 0.0f;
  }
  if (!fine) {
    s16 = (_Float16)__builtin_nanf("");
    z16 = (_Float16)0.0f;
  }
}
// four codes - 8 as the half-word of their nibbles: an exact sum below 2^16
__device__ __forceinline__ unsigned short nibbles(const float* c) {
  return (unsigned short)(unsigned)fmaf(fmaf(fmaf(c[3], 16.0f, c[2]), 16.0f, c[1]), 16.0f, c[0] + (float)0x8888);
}

// Block x of `rows` rows among those of all sequences, or false where there is none. A sequence that does not fit its batch is
// one block, from row 0.
__device__ __forceinline__ bool find_rows(const KvArgs& a, int rows, int x, int& b, int& b0, Seq& sq) {
  const int lane = threadIdx.x & 63;
  int top = 0;
  for (int s0 = 0; s0 < a.n_seqs; s0 += 64) {
    const Seq l = seq_in_order(a, s0 + lane, top);
    const int n = l.n == 0 ? 0 : l.ok ? (l.n + rows - 1) / rows : 1, sum = scan64(n);
    const unsigned long long past = __ballot(sum > x);
    if (past) {
      const int at = __builtin_ctzll(past);
      b = s0 + at;
      b0 = (x - lane_value(sum, at) + lane_value(n, at)) * rows;
      sq = lane_value(l, at);
      return true;
    }
    x -= lane_value(sum, 63);
  }
  return false;
}

// q and values of the largest calls (NR 4) do not stay in the caches, which leaves those to the rows: 16384 rows 46.6 us instead of
// 52.8 (on new buffers 53.8 and 57.7), and the attention after them takes as long as before.
template <int NR>
__device__ __forceinline__ void put8(_Float16* p, h8 v) {
  if constexpr (NR == 4) __builtin_nontemporal_store(v, gpw<h8>(p));
  else *gpw<h8>(p) = v;
}

// A wave has one head slot (the query heads, then the keys', then the values') of NR x 64 / (HD / 8) rows of a sequence. A query
// head's rotated channels, which are in few of a row's lanes, are done for all its rows at once, by lanes of their own.
template <int HD, typename T, int NR>
__global__ __launch_bounds__(256) void kv_append_kernel(KvArgs a, int listed) {
  constexpr int kLanes = HD / 8, kRows = 64 / kLanes, kBlock = NR * kRows;
  __shared__ float invs[4][kBlock];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, l = lane % kLanes, c = 8 * l, lr = lane / kLanes;
  const int slot = blockIdx.y * 4 + wave;
  if (slot >= a.HQ + 2 * a.HK || (slot < a.HQ && !a.q)) return;
  int b = blockIdx.z, b0 = blockIdx.x * kBlock;  // rows b0 + lr, b0 + lr + kRows, ... of sequence b
  Seq sq;
  if (listed) {
    if (!find_rows(a, kBlock, blockIdx.x, b, b0, sq)) return;
  } else {
    sq = seq_alone(a, b);
    if (b0 >= sq.n) return;
  }
  const h8 nan8 = h8{} + (_Float16)__builtin_nanf("");
  if (!sq.ok) {
    for (int i = b0 + lr; i < (listed ? sq.n : min(b0 + kBlock, sq.n)); i += kRows) {
      if (slot < a.HQ) *gpw<h8>(a.q + ((size_t)(sq.r0 + i) * a.HQ + slot) * HD + c) = nan8;
      else if (a.values) *gpw<h8>(a.values + ((size_t)(sq.r0 + i) * 2 * a.HK + slot - a.HQ) * HD + c) = nan8;
    }
    return;
  }
  const int per = a.gated ? 2 * HD : HD, which = slot >= a.HQ + a.HK, kh = slot - a.HQ - which * a.HK;
  const size_t col = slot < a.HQ ? (size_t)slot * per : (size_t)a.HQ * per + (size_t)(slot - a.HQ) * HD;
  const T* base = static_cast<const T*>(a.rows) + col + (size_t)sq.r0 * a.stride;
  const int first_pos = sq.len - sq.n;
  auto row_of = [&](int n) { return min(b0 + lr + n * kRows, sq.n - 1); };
  Eight<T> x[NR];
#pragma unroll
  for (int n = 0; n < NR; n++) x[n].load(base + (size_t)row_of(n) * a.stride + c);

  if (slot < a.HQ) {
    _Float16* q = a.q + ((size_t)sq.r0 * a.HQ + slot) * HD;
    const f4 w[2] = {ld4(a.qw + c), ld4(a.qw + c + 4)};
#pragma unroll
    for (int n = 0; n < NR; n++) {
      const float inv = rsqrtf(row_sum<kLanes>(x[n].squares()) * (1.0f / HD) + a.eps);
      if (l == 0) invs[wave][lr + n * kRows] = inv;
      const int i = b0 + lr + n * kRows;
      h8 o;
#pragma unroll
      for (int e = 0; e < 8; e++) o[e] = (_Float16)(x[n][e] * (inv * w[e >> 2][e & 3]));
      if (c >= a.rot && i < sq.n) put8<NR>(q + (size_t)i * a.HQ * HD + c, o);
    }
    wave_sync();
    const int chunks = a.rot / 8, share = min(kBlock, sq.n - b0) * chunks;  // 8 channels of a row a lane
    const unsigned by_chunks = chunks ? (65536u + chunks - 1) / chunks : 0;  // (exact for k chunks < 2^16)
    for (int k = lane; k < share; k += 64) {
      const int r = (int)((unsigned)k * by_chunks >> 16), c = 8 * (k - r * chunks), i = b0 + r;
      const Turn tn(c, a.rot);
      const T* row = base + (size_t)i * a.stride;
      const float* rope = a.rope + (size_t)(first_pos + i) * a.rot;
      Eight<T> x;
      x.load(row + c);
      f4 w[2], py[2], wp[2], cs[4];
#pragma unroll
      for (int n = 0; n < 2; n++) {
        w[n] = ld4(a.qw + c + 4 * n);
        py[n] = ld4(row + tn.other[n]);
        wp[n] = ld4(a.qw + tn.other[n]);
        cs[2 * n] = ld4(rope + tn.angle[n]);
        cs[2 * n + 1] = ld4(rope + tn.angle[n] + 4);
      }
      float y[8];
      scale_rotate<float>(x, invs[wave][r], w, tn, py, wp, cs, y);
      h8 o;
#pragma unroll
      for (int e = 0; e < 8; e++) o[e] = (_Float16)y[e];
      put8<NR>(q + (size_t)i * a.HQ * HD + c, o);
    }
    return;
  }

  int page[NR];
#pragma unroll
  for (int n = 0; n < NR; n++) page[n] = gp<int>(a.table)[(size_t)b * a.table_stride + ((first_pos + row_of(n)) >> a.page_log2)];
  // the values of a row (channels c .. + 7 of the lane) into their page
  auto put = [&](int n, const float* v) {
    _Float16 s, z;
    float code[8];
    quantise<HD>(v, s, z, code);
    const int i = b0 + lr + n * kRows;
    if (i >= sq.n) return;
    const int ps = (first_pos + i) & (a.page - 1);
    const bool in_pool = (unsigned)page[n] < (unsigned)a.n_pages;
    const int g = l / (HD / 32), gl = l % (HD / 32);  // the group; nibbles 16 (2 gl) + 4 g and 16 (2 gl + 1) + 4 g on
    if (in_pool) {
      unsigned char* blk = a.pool + (((size_t)page[n] * a.HK + kh) * 2 + which) * kv_block_bytes(a.page, HD);
      __attribute__((address_space(1))) unsigned short* row = gpw<unsigned short>(blk + (size_t)ps * (HD / 2)) + 8 * gl + g;
      row[0] = nibbles(code);
      row[4] = nibbles(code + 4);
      if (gl < 2) gpw<_Float16>(blk + (size_t)a.page * (HD / 2))[param_at(ps, g, gl)] = gl ? z : s;
    }
    if (a.values) {
      h8 o;
#pragma unroll
      for (int e = 0; e < 8; e++) o[e] = (_Float16)fmaf((float)s, code[e], (float)z);
      put8<NR>(a.values + (((size_t)(sq.r0 + i) * 2 + which) * a.HK + kh) * HD + c, in_pool ? o : nan8);
    }
  };
  if (which) {
#pragma unroll
    for (int n = 0; n < NR; n++) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = x[n][e];
      put(n, v);
    }
    return;
  }
  const Turn tn(c, a.rot);
  const f4 w[2] = {ld4(a.kw + c), ld4(a.kw + c + 4)};
#pragma unroll
  for (int n = 0; n < NR; n++) {
    const T* row = base + (size_t)row_of(n) * a.stride;
    const float* rope = a.rope + (size_t)(first_pos + row_of(n)) * a.rot;
    f4 py[2], wp[2], cs[4];
#pragma unroll
    for (int k = 0; k < 2; k++)
      if (tn.in[k]) {
        py[k] = ld4(row + tn.other[k]);
        wp[k] = ld4(a.kw + tn.other[k]);
        cs[2 * k] = ld4(rope + tn.angle[k]);
        cs[2 * k + 1] = ld4(rope + tn.angle[k] + 4);
      }
    double ss = 0.0, y[8];
#pragma unroll
    for (int e = 0; e < 8; e++) ss = fma((double)x[n][e], (double)x[n][e], ss);
    scale_rotate<double>(x[n], rsqrt(row_sum<kLanes>(ss) * (1.0 / HD) + (double)a.eps), w, tn, py, wp, cs, y);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = (float)y[e];
    put(n, v);
  }
}

}  // namespace

hipError_t launch_kv_rope(float* rope, const double* theta_pow, int max_ctx, int rot, hipStream_t s) {
  const long n = (long)max_ctx * (rot / 2);
  hipLaunchKernelGGL(kv_rope_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, rope, theta_pow, max_ctx, rot / 2);
  return hipGetLastError();
}

// A workgroup's place is in a grid of (rows, sequences), or, where most of that would be empty, in a list that the wave goes through.
// Measured, us, grid / list, the model's heads, in a graph of 40 calls: one new row each of 8 sequences 3.3 / 3.6, 2048 rows each
// 46.5 / 48.0; 2048 rows and 47 single ones 46.2 / 11.4, 400 rows and 200 single ones 58.5 / 7.9; 20 rows and 500 single ones
// 13.8 / 12.0, 8 rows and 1000 single ones (the list is 16 loads deep, the grid a quarter full) 20.9 / 29.1.
constexpr int kListFrom = 2;
template <int HD, typename T, int NR>
hipError_t append_rows(const KvArgs& a, hipStream_t s) {
  constexpr int kBlock = NR * 64 / (HD / 8);
  const long grid = (long)a.n_seqs * ((a.max_rows + kBlock - 1) / kBlock), list = a.n_rows / kBlock + a.n_seqs;
  const bool listed = grid > kListFrom * list;
  const dim3 blocks((unsigned)(listed ? list : (a.max_rows + kBlock - 1) / kBlock), (a.HQ + 2 * a.HK + 3) / 4, listed ? 1 : a.n_seqs);
  hipLaunchKernelGGL((kv_append_kernel<HD, T, NR>), blocks, dim3(256), 0, s, a, (int)listed);
  return hipGetLastError();
}
// More rows a wave where there are enough waves. Measured, us, 1 / 2 / 4 times 64 / (HD / 8) rows a wave, the model's heads: 256 rows
// 5.0 / 4.7 / 7.0, 1024 rows 7.1 / 6.2 / 8.1, 4096 rows 18.5 / 17.6 / 18.4, 16384 rows 66.5 / 58.4 / 52.5 (without streaming stores).
template <int HD, typename T>
hipError_t append(const KvArgs& a, hipStream_t s) {
  constexpr int kRows = 64 / (HD / 8);
  const long passes = (long)a.n_rows * (a.HQ + 2 * a.HK) / kRows;
  if (a.max_rows <= kRows || passes < 4096) return append_rows<HD, T, 1>(a, s);
  return passes < 32768 ? append_rows<HD, T, 2>(a, s) : append_rows<HD, T, 4>(a, s);
}

hipError_t launch_kv_append(const KvArgs& a, hipStream_t s) {
  if (a.HD == 256) return a.dtype == 0 ? append<256, float>(a, s) : append<256, _Float16>(a, s);
  return a.dtype == 0 ? append<128, float>(a, s) : append<128, _Float16>(a, s);
}

}  // namespace ha
