// The paged cache of 4-bit keys and values of the full-attention layers, gfx950: appending a batch's rows to it, with q's
// and k's norms and rotation on the way, and the attention that reads it.
//
// A row (one token and KV head) is 4 groups of G = HD / 4 consecutive channels, each with a scale s and a zero z in f16:
//   channel value = s (c - 8) + z, code c in 0..15
//   z = f16(lo + (hi - lo) 8/15), s = f16(max((hi - z) / 7, (z - lo) / 8)), c = clamp(rint((x - z) / s) + 8, 0, 15)
// for the group's least and largest values lo, hi: the nearest code is at most s / 2 off (but for the rounding of s).
// Codes stand in nibbles, channel (group g, 4 i + e) of the row in nibble 16 i + 4 g + e: a 16-bit half-word holds four
// channels of one group, so a lane that reads 8 bytes of a row has 4 channels of each group.
#include <cmath>

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

template <int W, typename F>
__device__ __forceinline__ F xor_sum(F v) {
#pragma unroll
  for (int d = W / 2; d >= 1; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// x normed (mean square over the row's lanes), with gain w, and rotated: channel c < rot / 2 pairs with c + rot / 2, which
// a lane at a distance of rot / 8 holds. F is float for q, which is rounded to f16, and double for k: a key next to
// the border between two codes then falls on the same side whatever the order of the sums.
template <int HD, typename F>
__device__ __forceinline__ void norm_rotate(F* x, const f4& w, const float* rope, int rot, float eps, int l) {
  F ss = 0;
#pragma unroll
  for (int e = 0; e < 4; e++) ss += x[e] * x[e];
  ss = xor_sum<HD / 4>(ss);
  const F inv = (F)1 / sqrt(ss / (F)HD + (F)eps);
#pragma unroll
  for (int e = 0; e < 4; e++) x[e] = x[e] * inv * (F)w[e];
  const int span = rot / 8;  // lanes of one half of the rotated channels
  const bool first = l < span, in = l < 2 * span;
  const int lane = threadIdx.x & 63, other = in ? (first ? lane + span : lane - span) : lane;
  F y[4];
#pragma unroll
  for (int e = 0; e < 4; e++) y[e] = __shfl(x[e], other);
  if (in) {
    const float* r = rope + 8 * (first ? l : l - span);
    const f4 r0 = ld4(r), r1 = ld4(r + 4);
    const float cs[4] = {r0[0], r0[2], r1[0], r1[2]}, sn[4] = {r0[1], r0[3], r1[1], r1[3]};
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = first ? x[e] * (F)cs[e] - y[e] * (F)sn[e] : x[e] * (F)cs[e] + y[e] * (F)sn[e];
  }
}

// The group's scale, zero and this lane's four codes (see the top). Every operation is rounded by itself (no contraction):
// the codes are a function of the values alone.
template <int HD>
__device__ __forceinline__ void quantise(const float* x, _Float16& s16, _Float16& z16, int* c) {
#pragma clang fp contract(off)
  float lo = fminf(fminf(x[0], x[1]), fminf(x[2], x[3])), hi = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
  float bad = x[0] * 0.0f + x[1] * 0.0f + x[2] * 0.0f + x[3] * 0.0f;  // NaN where a value is not finite
#pragma unroll
  for (int d = 1; d < HD / 16; d <<= 1) {
    lo = fminf(lo, __shfl_xor(lo, d));
    hi = fmaxf(hi, __shfl_xor(hi, d));
    bad += __shfl_xor(bad, d);
  }
  const float range = hi - lo;
  z16 = (_Float16)(lo + range * (float)(8.0 / 15.0));
  const float z = (float)z16;
  s16 = (_Float16)fmaxf((hi - z) * (float)(1.0 / 7.0), (z - lo) * 0.125f);
  const float s = (float)s16;
  const bool fine = bad == 0.0f && fabsf(s) < INFINITY && fabsf(z) < INFINITY;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const float r = rintf((x[e] - z) / s) + 8.0f;
    c[e] = fine && s > 0.0f ? (int)fminf(fmaxf(r, 0.0f), 15.0f) : 8;
  }
  if (!fine) {
    s16 = (_Float16)__builtin_nanf("");
    z16 = (_Float16)0.0f;
  }
}

// One wave per (head slot, 64 / (HD / 4) rows of a sequence); slots are the query heads, then the keys', then the values'. A
// lane has 4 channels of a row.
template <int HD, typename T>
__global__ __launch_bounds__(256) void kv_append_kernel(KvArgs a) {
  constexpr int kLanes = HD / 4, kRows = 64 / kLanes;
  const int lane = threadIdx.x & 63, l = lane % kLanes;
  const int slot = blockIdx.y * 4 + (threadIdx.x >> 6), b = blockIdx.z;
  if (slot >= a.HQ + 2 * a.HK) return;
  const Seq sq = seq_of(a, b);
  const int i = blockIdx.x * kRows + lane / kLanes;
  const bool live = i < sq.n;
  if (!__any(live)) return;
  const int t = sq.r0 + min(i, sq.n - 1), pos = sq.ok ? sq.len - sq.n + min(i, sq.n - 1) : 0;
  const float* rope = a.rope + (size_t)pos * a.rot;
  const int per = a.gated ? 2 * HD : HD;
  const T* row = static_cast<const T*>(a.rows) + (size_t)t * a.stride;
  const _Float16 nan16 = (_Float16)__builtin_nanf("");
  if (slot < a.HQ) {
    if (!a.q) return;
    const f4 v = ld4(row + (size_t)slot * per + 4 * l);
    float x[4] = {v[0], v[1], v[2], v[3]};
    norm_rotate<HD, float>(x, ld4(a.qw + 4 * l), rope, a.rot, a.eps, l);
    if (live)
      *reinterpret_cast<h4*>(a.q + ((size_t)t * a.HQ + slot) * HD + 4 * l) = sq.ok ? to_h4(f4{x[0], x[1], x[2], x[3]}) : h4{nan16, nan16, nan16, nan16};
    return;
  }
  const int which = slot >= a.HQ + a.HK, kh = slot - a.HQ - which * a.HK;
  const f4 v = ld4(row + (size_t)a.HQ * per + (size_t)(which * a.HK + kh) * HD + 4 * l);
  float x[4] = {v[0], v[1], v[2], v[3]};
  if (!which) {
    double y[4] = {v[0], v[1], v[2], v[3]};
    norm_rotate<HD, double>(y, ld4(a.kw + 4 * l), rope, a.rot, a.eps, l);
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = (float)y[e];
  }
  _Float16 s, z;
  int c[4];
  quantise<HD>(x, s, z, c);
  if (!live) return;
  unsigned char* blk = sq.ok ? block_of(a, b, pos, kh, which) : nullptr;
  const int g = l / (HD / 16), gi = l % (HD / 16), ps = pos & (a.page - 1);
  if (blk) {
    reinterpret_cast<unsigned short*>(blk + (size_t)ps * (HD / 2))[4 * gi + g] = (unsigned short)(c[0] | c[1] << 4 | c[2] << 8 | c[3] << 12);
    if (gi == 0) {
      _Float16* par = reinterpret_cast<_Float16*>(blk + (size_t)a.page * (HD / 2));
      par[param_at(ps, g, 0)] = s;
      par[param_at(ps, g, 1)] = z;
    }
  }
  if (a.values) {
    f4 w;
#pragma unroll
    for (int e = 0; e < 4; e++) w[e] = fmaf((float)s, (float)(c[e] - 8), (float)z);
    *reinterpret_cast<h4*>(a.values + (((size_t)t * 2 + which) * a.HK + kh) * HD + 4 * l) = blk ? to_h4(w) : h4{nan16, nan16, nan16, nan16};
  }
}

}  // namespace

hipError_t launch_kv_rope(float* rope, const double* theta_pow, int max_ctx, int rot, hipStream_t s) {
  const long n = (long)max_ctx * (rot / 2);
  hipLaunchKernelGGL(kv_rope_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, rope, theta_pow, max_ctx, rot / 2);
  return hipGetLastError();
}

hipError_t launch_kv_append(const KvArgs& a, hipStream_t s) {
  const int rows = 64 / (a.HD / 4);
  const dim3 grid((a.max_rows + rows - 1) / rows, (a.HQ + 2 * a.HK + 3) / 4, a.n_seqs), block(256);
  if (a.HD == 256) {
    if (a.dtype == 0) hipLaunchKernelGGL((kv_append_kernel<256, float>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((kv_append_kernel<256, _Float16>), grid, block, 0, s, a);
  } else {
    if (a.dtype == 0) hipLaunchKernelGGL((kv_append_kernel<128, float>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((kv_append_kernel<128, _Float16>), grid, block, 0, s, a);
  }
  return hipGetLastError();
}

}  // namespace ha
