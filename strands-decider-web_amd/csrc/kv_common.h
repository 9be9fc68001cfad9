// Shared by the kernels of the paged 4-bit K/V cache (kv.hip, kv_attn.hip), gfx950.
#pragma once
#include "kv.h"

namespace ha {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));

// ---- a batch's sequences ----

// Sequence b's rows [r0, r0 + n) and its context, positions [len - n, len) of which are the rows'. A sequence whose
// numbers do not fit the call's (ok false) stores nothing; the rows of it that lie in the call come out as NaN.
// `top`: the greatest of row_start[0 .. b] (and 0). A sequence that starts below it does not fit, and keeps clear of the rows before
// it: those of the sequences that fit are then disjoint, whatever row_start holds, and lists of them end within their grids.
struct Seq {
  int r0, n, len;
  bool ok;
};
__device__ __forceinline__ Seq seq_of(const KvArgs& a, int r0, int r1, int len, int top) {
  Seq s;
  s.ok = r0 >= top && r1 >= r0 && r1 <= a.n_rows && r1 - r0 <= a.max_rows && len >= r1 - r0 && len <= a.max_len;
  s.r0 = min(top, a.n_rows);
  s.n = min(min(max(r1, s.r0), a.n_rows) - s.r0, a.max_rows);
  s.len = s.ok ? len : 0;
  return s;
}
__device__ __forceinline__ Seq seq_of(const KvArgs& a, int b, int top) { return seq_of(a, a.row_start[b], a.row_start[b + 1], a.len[b], top); }

// ---- over a wave, with a sequence a lane ----

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }  // (for the compiler)
template <int kCtrl, int kRows>
__device__ __forceinline__ int dpp_add(int v) { return v + __builtin_amdgcn_update_dpp(0, v, kCtrl, kRows, 0xf, true); }
template <int kCtrl, int kRows>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), kCtrl, kRows, 0xf, true));
}
// inclusive prefix sum over the wave
template <typename F>
__device__ __forceinline__ F scan64(F v) {
  v = dpp_add<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  v = dpp_add<0x118, 0xf>(v);
  v = dpp_add<0x142, 0xa>(v);  // row_bcast 15, 31
  return dpp_add<0x143, 0xc>(v);
}
// inclusive running maximum over the wave, of values >= 0
template <int kCtrl, int kRows>
__device__ __forceinline__ int dpp_max(int v) { return max(v, __builtin_amdgcn_update_dpp(0, v, kCtrl, kRows, 0xf, true)); }
__device__ __forceinline__ int max64(int v) {
  v = dpp_max<0x111, 0xf>(v);
  v = dpp_max<0x112, 0xf>(v);
  v = dpp_max<0x114, 0xf>(v);
  v = dpp_max<0x118, 0xf>(v);
  v = dpp_max<0x142, 0xa>(v);
  return dpp_max<0x143, 0xc>(v);
}
__device__ __forceinline__ int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ Seq lane_value(const Seq& s, int lane) {
  return Seq{lane_value(s.r0, lane), lane_value(s.n, lane), lane_value(s.len, lane), lane_value((int)s.ok, lane) != 0};
}

// A sequence that has a place of its own in the grid, whatever those before it hold.
__device__ __forceinline__ Seq seq_alone(const KvArgs& a, int b) { return seq_of(a, b, max(a.row_start[b], 0)); }
// A lane's sequence s = s0 + lane, s0 = 0, 64, ... in this order: `top` is 0 at first, and handed on.
__device__ __forceinline__ Seq seq_in_order(const KvArgs& a, int s, int& top) {
  const bool in = s < a.n_seqs;
  const int at = min(s, a.n_seqs - 1), r0 = a.row_start[at], r1 = a.row_start[at + 1], len = a.len[at];  // (all loads at once)
  const int mine = max(top, max64(max(r0, 0)));
  top = lane_value(mine, 63);
  Seq q = seq_of(a, r0, r1, len, mine);
  if (!in) q = Seq{};
  return q;
}

// f16 index of (token slot, group, 0: scale, 1: zero) among a block's parameters
__device__ __forceinline__ int param_at(int slot, int g, int which) { return ((slot >> 2) * kKvGroups + g) * 8 + which * 4 + (slot & 3); }

template <typename T>
using gptr = const __attribute__((address_space(1))) T*;
template <typename T>
__device__ __forceinline__ gptr<T> gp(const void* p) { return (gptr<T>)(p); }
template <typename T>
__device__ __forceinline__ __attribute__((address_space(1))) T* gpw(void* p) { return (__attribute__((address_space(1))) T*)(p); }

__device__ __forceinline__ f4 ld4(const float* p) { return *gp<f4>(p); }
__device__ __forceinline__ f4 ld4(const _Float16* p) {
  const h4 x = *gp<h4>(p);
  return f4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
}
__device__ __forceinline__ h4 to_h4(const f4& x) { return h4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]}; }

// Orders a wave's LDS accesses before its later ones to other lanes' entries (no workgroup barrier).
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

}  // namespace
}  // namespace ha
