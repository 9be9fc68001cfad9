// Causal grouped-query attention over the paged 4-bit K/V cache, gfx950.
//
//   out[t][h] = sum_j softmax_j(scale q[t][h] . k_j) v_j * sigmoid(gate[t][h]),  j <= position of row t
//
// The rows of a sequence that share a KV head are its columns: row i, head hh of the group is column i ratio + hh, so the
// matrix products have as many columns as the group has heads, also where a sequence has a single new token.
//
// kv_few_kernel: a workgroup has 16 columns and a piece of the keys, its four waves 32 keys each in turn, with nothing shared
// until the end. It computes S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_f16, straight from the codes:
//   - a code c in bits 6..9 of an f16 whose exponent is 2^4 is the number 16 + c: with one v_perm for eight codes, a shift and
//     an and-or for two, the operands need no arithmetic. The dot product starts at -24 sum(q) (C operand), which leaves
//     sum(q (c - 8)) with f32 roundings only; the scale and zero of a group come in afterwards, on its 16 x 16 sums:
//     S = sum_g s_g (q . (c - 8))_g + z_g sum(q_g).
//   - K's operand is 16 bytes of a token's row a lane, V's 8 bytes of 8 tokens' rows, two tokens' half-words joined by
//     v_perm; S^T's layout (a column a lane) is that of P^T as an operand, so P goes from registers to registers.
//   - V's scales go onto P (P s_g, f16), and its zeros and the -24 into one more sum for each group: Z_g = sum P z_g - 24 sum P s_g.
//   - a column's maximum is the wave's own; it is raised only when a score exceeds it by 2^8.
// Pieces leave their O, maximum and sum in the workspace, and kv_merge_kernel joins them.
#include <algorithm>
#include <cmath>

#include "kv_common.h"

namespace ha {
namespace {

typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
constexpr float kRaise = 8.0f;  // log2 headroom before a column's maximum is raised
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kCols = 16, kWaves = 4, kStep = 32;

// x combined over the four lanes l, l ^ 16, l ^ 32, l ^ 48
template <typename F>
__device__ __forceinline__ float over_quads(float x, F f) {
  auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  x = f(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
  r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  return f(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}
__device__ __forceinline__ float max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  return fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
}
__device__ __forceinline__ float max_quads(float x) { return over_quads(x, [](float u, float v) { return fmaxf(u, v); }); }
__device__ __forceinline__ float sum_quads(float x) { return over_quads(x, [](float u, float v) { return u + v; }); }

// the low (high) half-words of u and v, u's first
__device__ __forceinline__ unsigned halves(unsigned u, unsigned v, bool high) {
  return __builtin_amdgcn_perm(v, u, high ? 0x07060302u : 0x05040100u);
}
// Masks in scalar, exponents in vector registers (an instruction reads one scalar): an and-or takes both at once.
struct Magic {
  unsigned lo = 0x000F000Fu, hi = 0x00F000F0u, top = 0x03C003C0u;         // of nibbles 0, 1, and of one in bits 6..9
  unsigned m1024 = 0x64006400u, m64 = 0x54005400u, m16 = 0x4C004C00u;
  __device__ __forceinline__ Magic() {
    asm volatile("" : "+s"(lo), "+s"(hi), "+s"(top));
    asm volatile("" : "+v"(m1024), "+v"(m64), "+v"(m16));
  }
};
// nibbles 0 .. 3 of each half-word as the f16 1024 + c, 64 + c, 1024 + c, 64 + c
__device__ __forceinline__ u4 codes_k(const Magic& k, unsigned x) {
  const unsigned y = x >> 8;
  return u4{(x & k.lo) | k.m1024, (x & k.hi) | k.m64, (y & k.lo) | k.m1024, (y & k.hi) | k.m64};
}
// nibble e of each half-word as the f16 16 + c
__device__ __forceinline__ unsigned code_v(const Magic& k, unsigned x, int e) {
  return ((e == 0 ? x << 6 : e == 1 ? x << 2 : e == 2 ? x >> 2 : x >> 6) & k.top) | k.m16;
}
__device__ __forceinline__ h2 as_h2(unsigned u) { return __builtin_bit_cast(h2, u); }
__device__ __forceinline__ unsigned as_u(h2 h) { return __builtin_bit_cast(unsigned, h); }

// f16 (a0 s0, a1 s1), one rounding each
__device__ __forceinline__ unsigned scale2(float a0, float a1, unsigned s) {
  unsigned r;
  asm("v_fma_mixlo_f16 %0, %1, %3, 0 op_sel_hi:[0,1,0]\n\t"
      "v_fma_mixhi_f16 %0, %2, %3, 0 op_sel:[0,1,0] op_sel_hi:[0,1,0]" : "=&v"(r) : "v"(a0), "v"(a1), "v"(s));
  return r;
}

__device__ __forceinline__ f4 gate4(const KvArgs& a, int t, int h, int ch) {
  const size_t at = (size_t)t * a.stride + (size_t)h * 2 * a.HD + a.HD + ch;
  return a.dtype == 0 ? ld4(static_cast<const float*>(a.rows) + at) : ld4(static_cast<const _Float16*>(a.rows) + at);
}
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }

// Partial results: for each (sequence, KV head, column block, piece, column) O (unnormalised) [HD], maximum, sum.
struct Parts {
  float* p;
  int cols, ns;  // columns a block has, pieces
  __device__ __forceinline__ float* column(const KvArgs& a, int ncb, int b, int kh, int cb, int piece, int c) const {
    return p + ((((((size_t)b * a.HK + kh) * ncb + cb) * ns + piece) * cols) + c) * (a.HD + 4);
  }
};

// The rows of a sequence that does not fit its batch.
template <int HD>
__device__ __forceinline__ void nan_rows(const KvArgs& a, const Seq& sq, int kh, int c0, int cols, int threads) {
  const int ratio = a.HQ / a.HK;
  for (int k = threadIdx.x; k < cols * HD; k += threads) {
    const int r = c0 + k / HD;
    a.out[((size_t)(sq.r0 + r / ratio) * a.HQ + kh * ratio + r % ratio) * HD + k % HD] = (_Float16)__builtin_nanf("");
  }
}
// Channels ch .. + 3 of column r: O / l, the gate, f16.
template <int HD>
__device__ __forceinline__ void finish(const KvArgs& a, const Seq& sq, int kh, int r, int ch, f4 v, float inv) {
  const int ratio = a.HQ / a.HK, t = sq.r0 + r / ratio, h = kh * ratio + r % ratio;
  v *= inv;
  if (a.gated) {
    const f4 gt = gate4(a, t, h, ch);
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] *= sigmoid(gt[e]);
  }
  *gpw<h4>(a.out + ((size_t)t * a.HQ + h) * HD + ch) = to_h4(v);
}

template <int HD>
__global__ __launch_bounds__(64 * kWaves, 2) void kv_few_kernel(KvArgs a, int chunk, int ncb, Parts parts) {
  constexpr int G = HD / 4, kH = HD / 128, kE = HD / 64, kRow = HD / 2;
  constexpr int kPitch = HD + 4;
  __shared__ float ol[kWaves * kCols * kPitch];
  __shared__ float ml[kWaves][kCols][2];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, j = lane & 15, kg = lane >> 4;
  const int ratio = a.HQ / a.HK;
  // the last column blocks first: they have the most keys; (sequence, KV head) pairs cycle fastest, so that the workgroups of
  // a pair share an XCD and its cache
  int id = blockIdx.x;
  const int pairs = a.n_seqs * a.HK, pair = id % pairs;
  id /= pairs;
  const int piece = id % parts.ns, cb = ncb - 1 - id / parts.ns, b = pair / a.HK, kh = pair % a.HK;
  const int k0 = piece * chunk;
  const int* table = a.table + (size_t)b * a.table_stride;
  const int page_log2 = a.page_log2, top_page = a.table_stride - 1;
  // lane k: the page of tokens k0 + 1024 seg + 16 k .. + 15
  int ids = gp<int>(table)[min((k0 + 16 * lane) >> page_log2, top_page)], seg = 0;
  const Seq sq = seq_of(a, b);
  const int c0 = cb * kCols, cols = min(kCols, sq.n * ratio - c0);
  if (cols <= 0) return;
  if (!sq.ok) {
    if (piece == 0) nan_rows<HD>(a, sq, kh, c0, cols, 64 * kWaves);
    return;
  }
  const int before = sq.len - sq.n;
  const int keys = before + (c0 + cols - 1) / ratio + 1, ns = (keys + chunk - 1) / chunk;
  if (piece >= ns) return;
  const int k1 = min(k0 + chunk, keys);
  const int all = before + c0 / ratio + 1;  // keys below this are seen by every column
  const int r = c0 + min(j, cols - 1), last = before + r / ratio;  // columns behind the last one repeat it
  h8 q[kH][4];
  float qs[4], qc[4];  // over each group: sum of the column's q, and what the codes' offsets add to its products
  const Magic mg;
  {
    const _Float16* qp = a.q + ((size_t)(sq.r0 + r / ratio) * a.HQ + kh * ratio + r % ratio) * HD + 8 * kg;
#pragma unroll
    for (int h = 0; h < kH; h++)
#pragma unroll
      for (int g = 0; g < 4; g++) q[h][g] = *gp<h8>(qp + G * g + 32 * h);
  }
#pragma unroll
  for (int g = 0; g < 4; g++) {
    float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
    for (int h = 0; h < kH; h++) {
      const h8 x = q[h][g];
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        s0 += (float)x[e];
        s1 += (float)x[e + 1];
      }
      q[h][g] = h8{x[0], x[4], x[1], x[5], x[2], x[6], x[3], x[7]};
    }
    s0 = sum_quads(s0);
    s1 = sum_quads(s1);
    qs[g] = s0 + s1;
    qc[g] = -1032.0f * s0 - 72.0f * s1;
  }
  const float scale = a.scale * kLog2e;
  f4 o[4][kE], zs[4];
  float m = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int g = 0; g < 4; g++) {
    zs[g] = f4{};
#pragma unroll
    for (int e = 0; e < kE; e++) o[g][e] = f4{};
  }
  const size_t blk_bytes = kv_block_bytes(a.page, HD);
  const unsigned par_off = (unsigned)a.page * kRow;

  for (int t0 = k0 + kStep * wave; t0 < k1; t0 += kStep * kWaves) {
    if ((t0 - k0) >> 10 != seg) {
      seg = (t0 - k0) >> 10;
      ids = gp<int>(table)[min((k0 + 1024 * seg + 16 * lane) >> page_log2, top_page)];
    }
    // this step's 32 keys: two tiles of 16, each in one page (any page for a tile behind the last key)
    const unsigned char* blk[2];
    int slot[2];
    bool gone[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      int page = __builtin_amdgcn_readlane(ids, ((t0 - k0) & 1023) / 16 + i);
      if (t0 + 16 * i >= k1) page = 0;
      gone[i] = (unsigned)page >= (unsigned)a.n_pages;
      blk[i] = a.pool + ((size_t)(gone[i] ? 0 : page) * a.HK + kh) * 2 * blk_bytes;
      slot[i] = (t0 + 16 * i) & (a.page - 1);
    }
    u4 kc[2][kH], kp[2][4], vp[2][4];
    u2 vc[2][4];
#pragma unroll
    for (int i = 0; i < 2; i++) {
#pragma unroll
      for (int h = 0; h < kH; h++) kc[i][h] = *gp<u4>(blk[i] + (unsigned)((slot[i] + j) * kRow + 64 * h + 16 * kg));
#pragma unroll
      for (int g = 0; g < 4; g++) kp[i][g] = *gp<u4>(blk[i] + par_off + (unsigned)((slot[i] + 4 * kg) * kKvParamBytes + 16 * g));
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
#pragma unroll
      for (int k = 0; k < 4; k++)
        vc[i][k] = *gp<u2>(blk[i] + blk_bytes + (unsigned)((slot[i] + 4 * kg + k) * kRow + 8 * (HD == 256 ? j : j & 7)));
#pragma unroll
      for (int g = 0; g < 4; g++) vp[i][g] = *gp<u4>(blk[i] + blk_bytes + par_off + (unsigned)((slot[i] + 4 * kg) * kKvParamBytes + 16 * g));
    }
    // scores of tokens t0 + 16 i + 4 kg + k
    float sc[2][4];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int g = 0; g < 4; g++) {
        f4 acc = f4{} + qc[g];
#pragma unroll
        for (int h = 0; h < kH; h++) {
          const u4 op = codes_k(mg, halves(kc[i][h][g >> 1], kc[i][h][(g >> 1) + 2], g & 1));
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, op), q[h][g], acc, 0, 0, 0);
        }
        const h8 p = __builtin_bit_cast(h8, kp[i][g]);
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const float z = g ? fmaf((float)p[4 + k], qs[g], sc[i][k]) : (float)p[4 + k] * qs[g];
          sc[i][k] = fmaf((float)p[k], acc[k], z);
        }
      }
    const bool edge = t0 + kStep > all || gone[0] || gone[1];
    if (edge) {
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int tok = t0 + 16 * i + 4 * kg + k;
          if (gone[i]) sc[i][k] = __builtin_nanf("");
          if (tok > last) sc[i][k] = -INFINITY;
          // beyond the sequence, and in no page: scales and zeros of any bits
          if (tok >= keys || gone[i]) {
            const unsigned clear = k & 1 ? 0x0000FFFFu : 0xFFFF0000u;
#pragma unroll
            for (int g = 0; g < 4; g++) {
              vp[i][g][k >> 1] &= clear;
              vp[i][g][2 + (k >> 1)] &= clear;
            }
          }
        }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int k = 0; k < 4; k++) mx = fmaxf(mx, sc[i][k]);
    mx = max_quads(mx) * scale;
    const float mn = mx > m + kRaise ? mx : m;
    if (__any(mn != m)) {
      const float al = mn == m ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
      sum *= al;
#pragma unroll
      for (int g = 0; g < 4; g++) {
        zs[g] *= al;
#pragma unroll
        for (int e = 0; e < kE; e++) o[g][e] *= al;
      }
      m = mn;
    }
    const float base = m == -INFINITY ? 0.0f : m;
    u4 p;  // P of tokens (t0 + 4 kg + 0, 1), (2, 3), then those of the second tile: f16
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int k = 0; k < 4; k += 2) {
        float &p0 = sc[i][k], &p1 = sc[i][k + 1];
        p0 = __builtin_amdgcn_exp2f(fmaf(p0, scale, -base));
        p1 = __builtin_amdgcn_exp2f(fmaf(p1, scale, -base));
        sum += p0 + p1;
        p[2 * i + k / 2] = as_u(h2{(_Float16)p0, (_Float16)p1});
      }
    const _Float16 off = (_Float16)-24.0f;
#pragma unroll
    for (int g = 0; g < 4; g++) {
      u4 w;  // P s_g
#pragma unroll
      for (int k = 0; k < 4; k++) w[k] = scale2(sc[k >> 1][2 * (k & 1)], sc[k >> 1][2 * (k & 1) + 1], vp[k >> 1][g][k & 1]);
      if (edge) {  // a masked token's scale may be NaN
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int tok = t0 + 16 * (k >> 1) + 4 * kg + 2 * (k & 1);
          w[k] = tok + 1 <= last ? w[k] : tok <= last ? w[k] & 0xFFFFu : 0u;
        }
      }
      const h8 wh = __builtin_bit_cast(h8, w);
      const u4 z = {vp[0][g][2], vp[0][g][3], vp[1][g][2], vp[1][g][3]};
      zs[g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, z), __builtin_bit_cast(h8, p), zs[g], 0, 0, 0);
      zs[g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h8{off, off, off, off, off, off, off, off}, wh, zs[g], 0, 0, 0);
      unsigned x[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        x[k] = halves(vc[k >> 1][2 * (k & 1)][g >> 1], vc[k >> 1][2 * (k & 1) + 1][g >> 1], g & 1);
        if constexpr (HD == 128) x[k] >>= 8 * (j >> 3);
      }
#pragma unroll
      for (int e = 0; e < kE; e++) {
        const u4 op = {code_v(mg, x[0], e), code_v(mg, x[1], e), code_v(mg, x[2], e), code_v(mg, x[3], e)};
        o[g][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, op), wh, o[g][e], 0, 0, 0);
      }
    }
  }
  // the four waves' sums: O^T row 4 kg + k of (g, e) is channel G g + 16 kg + 4 k + e (HD 256), G g + 4 (row & 7) + 2 (row >> 3) + e
  // (HD 128)
  sum = sum_quads(sum);
  if (kg == 0) {
    ml[wave][j][0] = m;
    ml[wave][j][1] = sum;
  }
  if (j < cols) {
    float* d = ol + (wave * kCols + j) * kPitch;
#pragma unroll
    for (int g = 0; g < 4; g++)
#pragma unroll
      for (int k = 0; k < 4; k++) {
        if constexpr (HD == 256) {
          *reinterpret_cast<f4*>(d + G * g + 16 * kg + 4 * k) = f4{o[g][0][k], o[g][1][k], o[g][2][k], o[g][3][k]} + zs[g][k];
        } else {
          const int ii = 4 * kg + k;
          *reinterpret_cast<float2*>(d + G * g + 4 * (ii & 7) + 2 * (ii >> 3)) = float2{o[g][0][k] + zs[g][k], o[g][1][k] + zs[g][k]};
        }
      }
  }
  __syncthreads();
  for (int k = tid; k < cols * (HD / 4); k += 64 * kWaves) {
    const int c = k / (HD / 4), ch = 4 * (k % (HD / 4));
    float mm = -INFINITY, l = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; w++) mm = fmaxf(mm, ml[w][c][0]);
    f4 v = {};
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
      const float f = ml[w][c][0] == mm ? 1.0f : __builtin_amdgcn_exp2f(ml[w][c][0] - mm);
      l += f * ml[w][c][1];
      v += f * *reinterpret_cast<const f4*>(ol + (w * kCols + c) * kPitch + ch);
    }
    if (ns > 1) {
      float* s = parts.column(a, ncb, b, kh, cb, piece, c);
      *gpw<f4>(s + ch) = v;
      if (ch == 0) {
        s[HD] = mm;
        s[HD + 1] = l;
      }
    } else {
      finish<HD>(a, sq, kh, c0 + c, ch, v, 1.0f / l);
    }
  }
}

// ---- many columns ----

constexpr int kBigCols = 128, kTile = 32;
typedef float f16v __attribute__((ext_vector_type(16)));

// LDS of kv_many_kernel, each part twice: K tile [32][HD] and V^T tile [HD][32] as f16 (rows 16 bytes longer, so that eight rows
// of an operand lie in different banks), K's scales [4][32] and zeros [32][4] twice each, V's scales and zeros [4][32], P f32 in
// the lanes' order, the columns' factors and the waves' flags.
template <int HD>
struct ManyLds {
  static constexpr int kKPitch = HD * 2 + 16, kVPitch = kTile * 2 + 16;
  static constexpr int kKs = kTile * kKPitch, kKz = kKs + 256, kV = kKz + 512, kVs = kV + HD * kVPitch, kVz = kVs + 256, kP = kVz + 256;
  static constexpr int kAl = kP + kBigCols * kTile * 4, kFlag = kAl + kBigCols * 4, kBuf = kFlag + 16;
};

// A workgroup has 128 columns and walks the keys in tiles of 32. Four of its eight waves compute P (32 columns each: S^T = K Q^T on
// v_mfma_f32_32x32x16_f16, scales and zeros, online softmax), the other four the outputs of the tile before (64 columns and half
// the channels each: O^T = V^T P^T) and unpack the next codes, as f16 numbers c - 8, into LDS; each SIMD has one of either
// kind, so the matrix products of the one run beside the vector instructions of the other. One barrier a tile. Scales and
// zeros stay apart from the codes, so that both operands are exact: S = sum_g s_g (q . (c - 8))_g + sum_g z_g sum(q_g), the last
// as one more product (with sum(q_g) / G as two f16), and O takes P s_g, rounded to f16 once, and sum P z_g.
template <int HD>
__global__ __launch_bounds__(512, 2) void kv_many_kernel(KvArgs a, int chunk, int ncb, Parts parts) {
  constexpr int G = HD / 4, U = HD / 16, kRow = HD / 2, kKs = G / 16, kDt = HD / 64;  // kKs: k-steps of a group; kDt: 32-row blocks of V^T a wave
  typedef ManyLds<HD> M;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, c32 = lane & 31, half = lane >> 5;
  const int ratio = a.HQ / a.HK;
  int id = blockIdx.x;  // (the order of kv_attend_kernel)
  const int pairs = a.n_seqs * a.HK, pair = id % pairs;
  id /= pairs;
  const int piece = id % parts.ns, cb = ncb - 1 - id / parts.ns, b = pair / a.HK, kh = pair % a.HK;
  const Seq sq = seq_of(a, b);
  const int c0 = cb * kBigCols, cols = min(kBigCols, sq.n * ratio - c0);
  if (cols <= 0) return;
  if (!sq.ok) {
    if (piece == 0) nan_rows<HD>(a, sq, kh, c0, cols, 512);
    return;
  }
  const int before = sq.len - sq.n, keys = before + (c0 + cols - 1) / ratio + 1, ns = (keys + chunk - 1) / chunk;
  if (piece >= ns) return;
  const int k0 = piece * chunk, k1 = min(k0 + chunk, keys), tiles = (k1 - k0 + kTile - 1) / kTile;
  const int all = before + c0 / ratio + 1;  // keys below this are seen by every column
  const float scale = a.scale * kLog2e;
  float* stats = reinterpret_cast<float*>(lds);  // after the last tile: [128] maxima, [128] sums

  if (wave < 4) {
    // ---- P of columns 32 wave .. + 31 ----
    const int w0 = 32 * wave, r = c0 + min(w0 + c32, cols - 1), last = before + r / ratio;
    const bool idle = w0 >= cols;
    // the B operand of k-step ks of group g is channels G g + 16 ks + 8 half .. + 7, in the order of K's chunks
    h8 q[4][kKs], qz;
    {
      const _Float16* qp = a.q + ((size_t)(sq.r0 + r / ratio) * a.HQ + kh * ratio + r % ratio) * HD + 8 * half;
#pragma unroll
      for (int g = 0; g < 4; g++)
#pragma unroll
        for (int ks = 0; ks < kKs; ks++) q[g][ks] = *gp<h8>(qp + G * g + 16 * ks);
#pragma unroll
      for (int g = 0; g < 4; g++) {
        float s = 0.0f;
#pragma unroll
        for (int ks = 0; ks < kKs; ks++) {
          const h8 x = q[g][ks];
#pragma unroll
          for (int e = 0; e < 8; e++) s += (float)x[e];
          q[g][ks] = h8{x[0], x[4], x[1], x[5], x[2], x[6], x[3], x[7]};
        }
        s = sum_halves(s) * (1.0f / G);
        const _Float16 hi = (_Float16)s;
        qz[2 * g] = half ? (_Float16)0.0f : hi;
        qz[2 * g + 1] = half ? (_Float16)0.0f : (_Float16)(s - (float)hi);
      }
    }
    float m = -INFINITY, sum = 0.0f;
    // S^T row i holds key pi(i) (bits 2 and 3 of i swapped): the lane's values 8 kb .. 8 kb + 7 are then keys 16 kb + 8 half .. + 7,
    // which is P^T's operand of k-step kb
    const int pr = (c32 & 19) | ((c32 & 4) << 1) | ((c32 & 8) >> 1);
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i <= tiles; i++) {
      if (i < tiles && !idle) {
        const int t0 = k0 + kTile * i;
        unsigned char* buf = lds + (i & 1) * M::kBuf;
        const unsigned char* kr = buf + pr * M::kKPitch + 16 * half;
        f16v st = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const h8*>(buf + M::kKz + pr * 16), qz, f16v{}, 0, 0, 0);
#pragma unroll
        for (int v = 0; v < 16; v++) st[v] *= (float)G;
#pragma unroll
        for (int g = 0; g < 4; g++) {
          f16v acc = f16v{};
#pragma unroll
          for (int ks = 0; ks < kKs; ks++)
            acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const h8*>(kr + 16 * ((G / 8) * g + 2 * ks)), q[g][ks], acc, 0, 0, 0);
#pragma unroll
          for (int kb = 0; kb < 2; kb++) {
            const h8 s = *reinterpret_cast<const h8*>(buf + M::kKs + g * 64 + 32 * kb + 16 * half);
#pragma unroll
            for (int e = 0; e < 8; e++) st[8 * kb + e] = fmaf((float)s[e], acc[8 * kb + e], st[8 * kb + e]);
          }
        }
        if (t0 + kTile > all || t0 + kTile > k1) {
          const int tok = t0 + 8 * half;
#pragma unroll
          for (int v = 0; v < 16; v++) st[v] = tok + 16 * (v >> 3) + (v & 7) <= last ? st[v] : -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int v = 0; v < 16; v++) mx = fmaxf(mx, st[v]);
        mx = max_halves(mx) * scale;
        const float mn = mx > m + kRaise ? mx : m;
        const bool raise = __any(mn != m);
        if (lane == 0) *reinterpret_cast<int*>(buf + M::kFlag + 4 * wave) = raise;
        if (raise) {
          const float al = mn == m ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
          sum *= al;
          m = mn;
          if (half == 0) *reinterpret_cast<float*>(buf + M::kAl + 4 * (w0 + c32)) = al;
        }
        const float base = m == -INFINITY ? 0.0f : m;
        f4* pl = reinterpret_cast<f4*>(buf + M::kP) + wave * 256 + lane;
#pragma unroll
        for (int k = 0; k < 4; k++) {
          f4 p;
#pragma unroll
          for (int e = 0; e < 4; e++) {
            p[e] = __builtin_amdgcn_exp2f(fmaf(st[4 * k + e], scale, -base));
            sum += p[e];
          }
          pl[64 * k] = p;
        }
      }
      __syncthreads();
    }
    sum = sum_halves(sum);
    if (half == 0) {
      stats[w0 + c32] = m;
      stats[kBigCols + w0 + c32] = sum;
    }
    __syncthreads();
    return;
  }

  // ---- outputs of columns 64 cp .. + 63 and groups 2 dh, 2 dh + 1 ----
  const int u = tid - 256, cp = wave & 1, dh = (wave >> 1) & 1;
  const bool idle = 64 * cp >= cols;
  const size_t blk_bytes = kv_block_bytes(a.page, HD);
  const int* table = a.table + (size_t)b * a.table_stride;
  const unsigned par_off = (unsigned)a.page * kRow;
  // what this thread unpacks: 16 bytes of a key, 4 bytes of four keys' values, two keys' parameters of K or of V
  const bool unpacks = HD == 256 || u < 128;
  const int kkey = HD == 256 ? u >> 3 : (u >> 2) & 31, kpos = HD == 256 ? u & 7 : u & 3;
  const int vquad = HD == 256 ? u >> 5 : (u >> 4) & 7, vpos = HD == 256 ? u & 31 : u & 15;
  const int pwhich = u >> 7, pquad = (u >> 4) & 7, pdw = u & 15;  // parameter word pdw of key quad pquad: (g, s or z, key pair)
  auto block_at = [&](int tok, bool& gone) {
    const int p = gp<int>(table)[min(tok, keys - 1) >> a.page_log2];
    gone = (unsigned)p >= (unsigned)a.n_pages;
    return a.pool + ((size_t)(gone ? 0 : p) * a.HK + kh) * 2 * blk_bytes;
  };
  u4 kraw = {}, vraw = {};
  unsigned praw = 0;
  bool pgone = false;
  // K of the tile at tk, V of the tile at tv
  auto fetch = [&](int tk, int tv) {
    bool gone;
    if (unpacks) {
      kraw = *gp<u4>(block_at(tk + kkey, gone) + (unsigned)(((tk + kkey) & (a.page - 1)) * kRow + 16 * kpos));
      const unsigned char* p = block_at(tv + 4 * vquad, gone) + blk_bytes + (unsigned)(((tv + 4 * vquad) & (a.page - 1)) * kRow + 4 * vpos);
#pragma unroll
      for (int k = 0; k < 4; k++) vraw[k] = *gp<unsigned>(p + k * kRow);
    }
    const int tok = (pwhich ? tv : tk) + 4 * pquad;
    praw = *gp<unsigned>(block_at(tok, pgone) + pwhich * blk_bytes + par_off + (unsigned)((tok & (a.page - 1)) * kKvParamBytes + 4 * pdw));
  };
  const Magic mg;
  const h2 m24 = {(_Float16)-24.0f, (_Float16)-24.0f};
  auto unpack = [&](int tk, int tv, unsigned char* kb, unsigned char* vb) {
    if (unpacks) {
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const unsigned x = halves(kraw[g >> 1], kraw[(g >> 1) + 2], g & 1);
        u4 w;
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = as_u(as_h2(code_v(mg, x, e)) + m24);
        *reinterpret_cast<u4*>(kb + kkey * M::kKPitch + 16 * ((G / 8) * g + kpos)) = w;
      }
#pragma unroll
      for (int gg = 0; gg < 2; gg++) {
        const unsigned x0 = halves(vraw[0], vraw[1], gg), x1 = halves(vraw[2], vraw[3], gg);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const u2 w = {as_u(as_h2(code_v(mg, x0, e)) + m24), as_u(as_h2(code_v(mg, x1, e)) + m24)};
          const int R = 4 * U * (2 * (vpos & 1) + gg) + U * e + (vpos >> 1);
          *reinterpret_cast<u2*>(vb + M::kV + R * M::kVPitch + 8 * vquad) = w;
        }
      }
    }
    const int g = pdw >> 2, part = (pdw >> 1) & 1, key = 4 * pquad + 2 * (pdw & 1), t0 = pwhich ? tv : tk;
    // behind the sequence, and in no page: parameters of any bits (a score of no page is NaN)
    unsigned w = pgone ? (pwhich == 0 && part == 0 ? 0x7E007E00u : 0u) : praw;
    if (t0 + key >= keys) w = 0;
    else if (t0 + key + 1 >= keys) w &= 0xFFFFu;
    if (pwhich) {
      *reinterpret_cast<unsigned*>(vb + (part ? M::kVz : M::kVs) + g * 64 + key * 2) = w;
    } else if (part) {
      *reinterpret_cast<unsigned*>(kb + M::kKz + key * 16 + 4 * g) = (w & 0xFFFFu) * 0x10001u;
      *reinterpret_cast<unsigned*>(kb + M::kKz + key * 16 + 16 + 4 * g) = (w >> 16) * 0x10001u;
    } else {
      *reinterpret_cast<unsigned*>(kb + M::kKs + g * 64 + key * 2) = w;
    }
  };
  f16v o[2][kDt], zacc[2];
  int last[2];
#pragma unroll
  for (int n = 0; n < 2; n++) {
    last[n] = before + (c0 + min(64 * cp + 32 * n + c32, cols - 1)) / ratio;
    zacc[n] = f16v{};
#pragma unroll
    for (int d = 0; d < kDt; d++) o[n][d] = f16v{};
  }
  fetch(k0, k0);
  unpack(k0, k0, lds, lds);
  fetch(k0 + kTile, k0);
  __syncthreads();
  // step i: P of tile i, outputs of tile i - 1; K of tile i + 1 and V of tile i go to LDS (while the other waves are busy with their
  // products), the next codes are fetched (K's behind the last tile: any)
#pragma unroll 1
  for (int i = 0; i <= tiles; i++) {
    if (i < tiles) {
      unpack(k0 + kTile * (i + 1), k0 + kTile * i, lds + ((i + 1) & 1) * M::kBuf, lds + (i & 1) * M::kBuf);
      if (i + 1 < tiles) fetch(k0 + kTile * (i + 2), k0 + kTile * (i + 1));
    }
    if (i > 0 && !idle) {
      const int t0 = k0 + kTile * (i - 1);
      const unsigned char* buf = lds + ((i - 1) & 1) * M::kBuf;
      const int* flag = reinterpret_cast<const int*>(buf + M::kFlag) + 2 * cp;
      const bool f0 = flag[0], f1 = flag[1] && 64 * cp + 32 < cols;
      if (f0 || f1) {
#pragma unroll
        for (int n = 0; n < 2; n++) {
          const float al = (n ? f1 : f0) ? *reinterpret_cast<const float*>(buf + M::kAl + 4 * (64 * cp + 32 * n + c32)) : 1.0f;
          zacc[n] *= al;
#pragma unroll
          for (int d = 0; d < kDt; d++) o[n][d] *= al;
        }
      }
      const bool edge = t0 + kTile > all || t0 + kTile > k1;
      const f4* pl = reinterpret_cast<const f4*>(buf + M::kP) + 2 * cp * 256 + lane;
      const unsigned char* vr = buf + M::kV + (2 * dh * G + c32) * M::kVPitch + 16 * half;
#pragma unroll
      for (int kb = 0; kb < 2; kb++) {
        f4 p[2][2];
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
          for (int k = 0; k < 2; k++) p[n][k] = pl[256 * n + 64 * (2 * kb + k)];
        const h8 z = *reinterpret_cast<const h8*>(buf + M::kVz + (2 * dh + (c32 & 1)) * 64 + 32 * kb + 16 * half);
#pragma unroll
        for (int n = 0; n < 2; n++) {
          const h8 ph = {(_Float16)p[n][0][0], (_Float16)p[n][0][1], (_Float16)p[n][0][2], (_Float16)p[n][0][3],
                         (_Float16)p[n][1][0], (_Float16)p[n][1][1], (_Float16)p[n][1][2], (_Float16)p[n][1][3]};
          zacc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(z, ph, zacc[n], 0, 0, 0);
        }
#pragma unroll
        for (int gg = 0; gg < 2; gg++) {
          const u4 s = *reinterpret_cast<const u4*>(buf + M::kVs + (2 * dh + gg) * 64 + 32 * kb + 16 * half);
          h8 wh[2];
#pragma unroll
          for (int n = 0; n < 2; n++) {
            u4 w;
#pragma unroll
            for (int k = 0; k < 4; k++) w[k] = scale2(p[n][k >> 1][2 * (k & 1)], p[n][k >> 1][2 * (k & 1) + 1], s[k]);
            if (edge) {  // a masked token's scale may be NaN
#pragma unroll
              for (int k = 0; k < 4; k++) {
                const int tok = t0 + 16 * kb + 8 * half + 2 * k;
                w[k] = tok + 1 <= last[n] ? w[k] : tok <= last[n] ? w[k] & 0xFFFFu : 0u;
              }
            }
            wh[n] = __builtin_bit_cast(h8, w);
          }
#pragma unroll
          for (int d = 0; d < G / 32; d++) {
            const int dt = (G / 32) * gg + d;
            const h8 vt = *reinterpret_cast<const h8*>(vr + 32 * dt * M::kVPitch + 32 * kb);
#pragma unroll
            for (int n = 0; n < 2; n++) o[n][dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vt, wh[n], o[n][dt], 0, 0, 0);
          }
        }
      }
    }
    __syncthreads();
  }
  __syncthreads();
  if (idle) return;
#pragma unroll
  for (int n = 0; n < 2; n++) {
    const int c = 64 * cp + 32 * n + c32;
    if (c >= cols) continue;
    const float mm = stats[c], l = stats[kBigCols + c], inv = 1.0f / l;
    // O^T row rho of dt is V^T row R = 32 dt + rho: channel G g + 4 i + e with R = 4 U g + U e + i
    float* pp = ns > 1 ? parts.column(a, ncb, b, kh, cb, piece, c) : nullptr;
#pragma unroll
    for (int gg = 0; gg < 2; gg++)
#pragma unroll
      for (int k = 0; k < U / 2; k++) {
        f4 v;
        int i;
        if constexpr (HD == 256) {
          i = 8 * (k >> 2) + 4 * half + (k & 3);
          v = f4{o[n][2 * gg][k], o[n][2 * gg][k + 8], o[n][2 * gg + 1][k], o[n][2 * gg + 1][k + 8]};
        } else {
          i = 4 * half + k;
          v = f4{o[n][gg][k], o[n][gg][k + 4], o[n][gg][k + 8], o[n][gg][k + 12]};
        }
        v += zacc[n][gg];
        const int ch = G * (2 * dh + gg) + 4 * i;
        if (ns > 1) {
          *gpw<f4>(pp + ch) = v;
        } else {
          finish<HD>(a, sq, kh, c0 + c, ch, v, inv);
        }
      }
    if (ns > 1 && half == 0 && dh == 0) {
      pp[HD] = mm;
      pp[HD + 1] = l;
    }
  }
}

// out of one (row, head) from its pieces: thread (k, c) adds pieces k, k + blockDim / (HD / 4), ... of channels 4 c .. + 3.
constexpr int kMergeMost = 2048;  // pieces
template <int HD>
__global__ __launch_bounds__(1024) void kv_merge_kernel(KvArgs a, int chunk, int ncb, int block_cols, Parts parts) {
  constexpr int C = HD / 4;
  __shared__ float wl[kMergeMost], red[2][16];
  __shared__ f4 vl[1024];
  const int tid = threadIdx.x, i = blockIdx.x, h = blockIdx.y, b = blockIdx.z, ratio = a.HQ / a.HK, kh = h / ratio;
  const Seq sq = seq_of(a, b);
  if (i >= sq.n || !sq.ok) return;
  const int col = i * ratio + h % ratio, cb = col / block_cols, c = col % block_cols;
  const int end = min(block_cols, sq.n * ratio - cb * block_cols);
  const int keys = sq.len - sq.n + (cb * block_cols + end - 1) / ratio + 1, ns = (keys + chunk - 1) / chunk;
  if (ns <= 1) return;
  const float* p = parts.column(a, ncb, b, kh, cb, 0, c);
  const size_t step = (size_t)parts.cols * (HD + 4);
  const int k = tid / C, n = blockDim.x / C, ch = 4 * (tid % C), wave = tid >> 6, waves = blockDim.x >> 6;
  // the first pieces' O and the gate go out before the maxima are waited for
  constexpr int kAhead = 4;
  f4 ahead[kAhead];
#pragma unroll
  for (int x = 0; x < kAhead; x++) ahead[x] = ld4(p + min(k + x * n, ns - 1) * step + ch);
  const int t = sq.r0 + i;
  const f4 gt = a.gated && k == 0 ? gate4(a, t, h, ch) : f4{};
  float mm = -INFINITY, l = 0.0f, mine[kMergeMost / 256], suml[kMergeMost / 256];
  const int per = (ns + (int)blockDim.x - 1) / (int)blockDim.x;
#pragma unroll
  for (int x = 0; x < kMergeMost / 256; x++)
    if (x < per) {
      const int s = tid + x * (int)blockDim.x;
      mine[x] = s < ns ? gp<float>(p)[s * step + HD] : -INFINITY;
      suml[x] = s < ns ? gp<float>(p)[s * step + HD + 1] : 0.0f;
      mm = fmaxf(mm, mine[x]);
    }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) mm = fmaxf(mm, __shfl_xor(mm, d));
  if ((tid & 63) == 0) red[0][wave] = mm;
  __syncthreads();
  mm = red[0][0];
  for (int w = 1; w < waves; w++) mm = fmaxf(mm, red[0][w]);
#pragma unroll
  for (int x = 0; x < kMergeMost / 256; x++)
    if (x < per) {
      const int s = tid + x * (int)blockDim.x;
      const float f = mine[x] == mm ? 1.0f : __builtin_amdgcn_exp2f(mine[x] - mm);
      if (s < ns) {
        wl[s] = f;
        l += f * suml[x];
      }
    }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) l += __shfl_xor(l, d);
  if ((tid & 63) == 0) red[1][wave] = l;
  __syncthreads();
  f4 v = {};
#pragma unroll
  for (int x = 0; x < kAhead; x++)
    if (k + x * n < ns) v += wl[k + x * n] * ahead[x];
#pragma unroll 4
  for (int s = k + kAhead * n; s < ns; s += n) v += wl[s] * ld4(p + s * step + ch);
  vl[tid] = v;
  __syncthreads();
  if (k) return;
  for (int s = 1; s < n; s++) v += vl[s * C + tid];
  l = red[1][0];
  for (int w = 1; w < waves; w++) l += red[1][w];
  v *= 1.0f / l;
  if (a.gated) {
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] *= sigmoid(gt[e]);
  }
  *gpw<h4>(a.out + ((size_t)t * a.HQ + h) * HD + ch) = to_h4(v);
}

// The pieces of a call of `units` (column block, KV head, sequence): `want` workgroups in all, of at least `unit` keys each, as
// long as the pieces' results fit the workspace.
int pieces(long units, int max_len, int want, int unit, size_t unit_bytes, size_t ws_bytes, int* chunk) {
  long c = std::max<long>((units * max_len / want + unit - 1) / unit * unit, unit);
  while ((max_len + c - 1) / c > 1 && ((size_t)units * ((max_len + c - 1) / c) * unit_bytes > ws_bytes || (max_len + c - 1) / c > kMergeMost)) c *= 2;
  *chunk = (int)std::min<long>(c, 1 << 30);
  return (int)((max_len + c - 1) / c);
}

template <int HD, bool MANY>
hipError_t launch(const KvArgs& a, float* ws, size_t ws_bytes, int want, hipStream_t s) {
  constexpr int block_cols = MANY ? kBigCols : kCols;
  const int most = a.max_rows * (a.HQ / a.HK), ncb = (most + block_cols - 1) / block_cols;
  Parts parts{ws, std::min(block_cols, most), 1};
  const long units = (long)a.n_seqs * a.HK * ncb;
  int chunk;
  parts.ns = pieces(units, a.max_len, want, MANY ? 2 * kTile : kStep * kWaves, (size_t)parts.cols * (HD + 4) * sizeof(float), ws_bytes, &chunk);
  if constexpr (MANY) {
    constexpr int lds = 2 * ManyLds<HD>::kBuf;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kv_many_kernel<HD>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((kv_many_kernel<HD>), dim3((unsigned)(units * parts.ns)), dim3(512), lds, s, a, chunk, ncb, parts);
  } else {
    hipLaunchKernelGGL((kv_few_kernel<HD>), dim3((unsigned)(units * parts.ns)), dim3(64 * kWaves), 0, s, a, chunk, ncb, parts);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || parts.ns == 1) return e;
  hipLaunchKernelGGL((kv_merge_kernel<HD>), dim3(a.max_rows, a.HQ, a.n_seqs), dim3(parts.ns > 16 ? 1024 : 256), 0, s, a, chunk, ncb, block_cols, parts);
  return hipGetLastError();
}

#ifndef KV_FEW_COLS
#define KV_FEW_COLS 16
#endif
template <int HD>
hipError_t attend(const KvArgs& a, float* ws, size_t ws_bytes, hipStream_t s) {
  const int most = a.max_rows * (a.HQ / a.HK);
  if (most > KV_FEW_COLS) return launch<HD, true>(a, ws, ws_bytes, 512, s);
  return launch<HD, false>(a, ws, ws_bytes, 1024, s);
}

}  // namespace

size_t kv_workspace_bytes() { return (size_t)64 << 20; }

hipError_t launch_kv_attention(const KvArgs& a, void* ws, size_t ws_bytes, hipStream_t s) {
  return a.HD == 256 ? attend<256>(a, static_cast<float*>(ws), ws_bytes, s) : attend<128>(a, static_cast<float*>(ws), ws_bytes, s);
}

}  // namespace ha
