// Shared by the kernels of fused.hip: decoding without rounding, and what is done with a finished tile.
//
// Weights stay exact. A code less 2^(bits-1) is a small integer, which f16 holds; the matrix unit sums its products with the 32
// f16 values of a in f32, and the group's f16 scale multiplies that sum in f32 (one fma a sum). Against weights rounded to f16
// before the product (mnb_common.h: up to 2^-11 of each weight) the sums are some 500 times nearer to 64 bits (3e-7 against 1.4e-4 of
// their size at K = 2048), which results in f32 show, and the decoding has no multiplications. Asymmetric weights s c + b are
// s (c - 2^(bits-1)) + b', b' = b + 2^(bits-1) s: b' times the group's sum of a, which a product with ones gives.
#pragma once
#include <hip/hip_runtime.h>

#include "fused.h"
#include "mnb_common.h"

namespace ha {
namespace {

template <typename T>
using gptr = const __attribute__((address_space(1))) T*;
template <typename T>
__device__ __forceinline__ gptr<T> gp(const void* p) { return (gptr<T>)(p); }

constexpr int kEpiAct = 0, kEpiLogits = 1;

// Eight consecutive codes less 2^(BITS-1), in element order. 4 bits: lo is their word; else lo holds their low two bits
// (element e at bits 2 e) and, for 3, hi their third (element e at bit e), with nothing above them. In the mantissa of 1024.0 bit 0
// is worth 1, in that of 64.0 bit 4: two elements 2 i (low half) and 2 i + 1 (high half) where they stand, two pairs a word, and one
// subtraction leaves the code less its middle exactly. 12, 20 and 10 instructions for 4, 3 and 2 bits.
template <int BITS>
__device__ __forceinline__ h8 codes8(unsigned lo, unsigned hi) {
  h8 r;
  if constexpr (BITS == 4) {
    unsigned mask = 0x00F0000Fu, one = 0x54006400u;
    asm("" : "+s"(mask), "+v"(one));  // (in registers: one v_and_or_b32 takes one scalar and no literal)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      // a byte (two codes) in both halves
      const unsigned p = __builtin_amdgcn_perm(lo, lo, 0x01010101u * i);
      const h2 q = __builtin_bit_cast(h2, (p & mask) | one) - h2{(_Float16)1032.0f, (_Float16)72.0f};
      r[2 * i] = q[0];
      r[2 * i + 1] = q[1];
    }
  } else {
    constexpr unsigned kField = BITS == 3 ? 0x00070007u : 0x00030003u;
    unsigned m0 = kField, m1 = kField << 4, one0 = 0x64006400u, one1 = 0x54005400u;
    asm("" : "+s"(m0), "+s"(m1), "+v"(one0), "+v"(one1));
    const unsigned u = lo | lo << 14;  // elements 2 i at bits 4 i of the low half, 2 i + 1 at bits 4 i of the high one
    unsigned w[2] = {u, u >> 8};       // pairs 0 and 1 at bits 0 and 4 of each half; 2 and 3
    if constexpr (BITS == 3) {
      const unsigned v = hi | hi << 15;  // third bits at 2 i of the halves
      w[0] = (w[0] & 0x00330033u) | (v << 2 & 0x00040004u) | (v << 4 & 0x00400040u);
      w[1] = (w[1] & 0x00330033u) | (v >> 2 & 0x00040004u) | (v & 0x00400040u);
    }
    constexpr float kMid = 1 << (BITS - 1);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const unsigned p = i & 1 ? (w[i >> 1] & m1) | one1 : (w[i >> 1] & m0) | one0;
      const _Float16 off = (_Float16)((i & 1 ? 64 : 1024) + kMid);
      const h2 q = __builtin_bit_cast(h2, p) - h2{off, off};
      r[2 * i] = q[0];
      r[2 * i + 1] = q[1];
    }
  }
  return r;
}

// The f16 of u's low half as an f32 in a register of its own: the compiler would otherwise put the conversion into each fma that
// takes it (v_fma_mix_f32, twice as long and not bound to its accumulator's register, which made the tile kernel spill).
__device__ __forceinline__ float f16_bits(unsigned u) {
  float v = (float)__builtin_bit_cast(_Float16, (unsigned short)u);
  asm("" : "+v"(v));
  return v;
}
// b + 2^(BITS-1) s
template <int BITS>
__device__ __forceinline__ float centred(float s, float b) { return fmaf((float)(1 << (BITS - 1)), s, b); }

__device__ __forceinline__ h8 ones8() {
  const _Float16 o = (_Float16)1.0f;
  return h8{o, o, o, o, o, o, o, o};
}

// ---- results ----

// 1 / (1 + e^-t), 0 where e^-t is infinite. silu(z) = z sigmoid(z), gelu(z) = z sigmoid(2 sqrt(2/pi) (z + 0.044715 z^3)) (the
// tanh form).
__device__ __forceinline__ float sigmoid(float t) { return __builtin_amdgcn_rcpf(1.0f + __expf(-t)); }
// What goes into N values of a column of the result besides their sums, rows m + row_of(v): residual and biases. Loaded together:
// asked for one by one, a tile's results took longer than its products (2048 x 2048 x 6144: 172 us).
template <int N>
struct Given {
  float res[N], bias, up_bias;
};
template <int N, class Row>
__device__ __forceinline__ Given<N> given(const FusedArgs& p, int m, int j, Row row_of) {
  Given<N> x;
#pragma unroll
  for (int v = 0; v < N; v++) x.res[v] = 0.0f;
  if (p.res) {
    const size_t from = (size_t)m * p.res_stride + j;
    const int last = p.M - 1 - m;
    if (p.res_f32) {
#pragma unroll
      for (int v = 0; v < N; v++) x.res[v] = row_of(v) <= last ? gp<float>(p.res)[from + (size_t)row_of(v) * p.res_stride] : 0.0f;
    } else {
#pragma unroll
      for (int v = 0; v < N; v++) x.res[v] = row_of(v) <= last ? (float)gp<_Float16>(p.res)[from + (size_t)row_of(v) * p.res_stride] : 0.0f;
    }
  }
  x.bias = p.bias ? p.bias[j] : 0.0f;
  x.up_bias = p.bias && p.half ? p.bias[p.half + j] : 0.0f;
  return x;
}
// The N values from their sums z (gated: of the gate, with the up projection's) and what is given; type and activation are asked for
// once for all N.
template <int N, class Row>
__device__ __forceinline__ void finish(const FusedArgs& p, int m, int j, Row row_of, const float* z, const float* up, const Given<N>& x) {
  float r[N];
#pragma unroll
  for (int v = 0; v < N; v++) r[v] = z[v];
  if (p.bias) {
#pragma unroll
    for (int v = 0; v < N; v++) r[v] += x.bias;
  }
  if (p.act == 1) {
#pragma unroll
    for (int v = 0; v < N; v++) r[v] = r[v] * sigmoid(r[v]);
  } else if (p.act == 2) {
#pragma unroll
    for (int v = 0; v < N; v++) r[v] = r[v] * sigmoid(1.5957691216057308f * fmaf(0.044715f * r[v] * r[v], r[v], r[v]));
  }
  if (p.half) {
#pragma unroll
    for (int v = 0; v < N; v++) r[v] *= up[v] + x.up_bias;
  }
  if (p.res) {
#pragma unroll
    for (int v = 0; v < N; v++) r[v] += x.res[v];
  }
  const size_t to = (size_t)m * p.out_stride + j;
  const int last = p.M - 1 - m;
  if (p.out_f32) {
#pragma unroll
    for (int v = 0; v < N; v++)
      if (row_of(v) <= last) ((float*)p.out)[to + (size_t)row_of(v) * p.out_stride] = r[v];
  } else {
#pragma unroll
    for (int v = 0; v < N; v++)
      if (row_of(v) <= last) ((_Float16*)p.out)[to + (size_t)row_of(v) * p.out_stride] = (_Float16)r[v];
  }
}
template <int N, class Row>
__device__ __forceinline__ void results(const FusedArgs& p, int m, int j, int cols, Row row_of, const float* z, const float* up) {
  if (j >= cols) return;
  finish<N>(p, m, j, row_of, z, up, given<N>(p, m, j, row_of));
}

// ---- records of logits ----

__device__ __forceinline__ unsigned ordered(float f) {
  const unsigned u = __builtin_bit_cast(unsigned, f);
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(unsigned o) {
  return __builtin_bit_cast(float, o >> 31 ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ unsigned pack_second(float second, int arg) {
  return (min(ordered(second) >> 6, (1u << 26) - 2) + 1) << 6 | (unsigned)arg;
}

// What stands for a column that is none: below every logit (|z| < 2 10^24: f16 rows, scales and biases, K up to 2^24 and the factor up
// to 10^6, which fused_host.cpp sees to).
constexpr float kNoLogit = -3e38f;

// The record of a row's block of which this lane has the N columns col(0) < col(1) < ..., and the lanes at distance D, 2 D, ...
// < L of it the others (z: scaled, kNoLogit where there is no column). All of them get it. About ten instructions a value and an
// exponential: columns that equal the largest are taken out of the sums, counted, and put back but for one.
template <int N, int D, int L, class Col>
__device__ __forceinline__ LpRecord record_of(const float* z, Col col) {
  float top = z[0];
#pragma unroll
  for (int i = 1; i < N; i++) top = fmaxf(top, z[i]);
#pragma unroll
  for (int d = D; d < L; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
  float second = kNoLogit, rest = 0.0f, rest_z = 0.0f;
  int arg = kLpBlock - 1, equal = 0;
#pragma unroll
  for (int i = N - 1; i >= 0; i--) {
    const bool is = z[i] == top;
    const float other = is ? kNoLogit : z[i];
    equal += is;
    arg = is ? col(i) : arg;
    second = fmaxf(second, other);
    const float x = other - top, e = __expf(x);  // (0 of kNoLogit)
    rest += e;
    rest_z = fmaf(e, x, rest_z);
  }
  if (!equal) arg = kLpBlock - 1;
#pragma unroll
  for (int d = D; d < L; d *= 2) {
    second = fmaxf(second, __shfl_xor(second, d));
    rest += __shfl_xor(rest, d);
    rest_z += __shfl_xor(rest_z, d);
    arg = min(arg, __shfl_xor(arg, d));
    equal += __shfl_xor(equal, d);
  }
  if (equal > 1) second = top, rest += (float)(equal - 1);
  return LpRecord{top, rest, rest_z, pack_second(second, arg)};
}
// Lane c of 16 has columns 16 t + c, t < 4, `valid` of the block's columns exist.
__device__ __forceinline__ LpRecord record16(const float* z, int c, int valid) {
  float y[4];
#pragma unroll
  for (int t = 0; t < 4; t++) y[t] = 16 * t + c < valid ? z[t] : kNoLogit;
  return record_of<4, 1, 16>(y, [c](int t) { return 16 * t + c; });
}

}  // namespace
}  // namespace ha
