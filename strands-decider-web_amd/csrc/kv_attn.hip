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
__device__ __forceinline__ float max_quads(float x) { return over_quads(x, [](float u, float v) { return fmaxf(u, v); }); }
__device__ __forceinline__ float sum_quads(float x) { return over_quads(x, [](float u, float v) { return u + v; }); }

// the low (high) half-words of u and v, u's first
__device__ __forceinline__ unsigned halves(unsigned u, unsigned v, bool high) {
  return __builtin_amdgcn_perm(v, u, high ? 0x07060302u : 0x05040100u);
}
// nibble e of each half-word as the f16 16 + c
__device__ __forceinline__ unsigned code2(unsigned x, int e) {
  const unsigned s = e == 0 ? x << 6 : e == 1 ? x << 2 : e == 2 ? x >> 2 : x >> 6;
  return (s & 0x03C003C0u) | 0x4C004C00u;
}
__device__ __forceinline__ h2 as_h2(unsigned u) { return __builtin_bit_cast(h2, u); }
__device__ __forceinline__ unsigned as_u(h2 h) { return __builtin_bit_cast(unsigned, h); }

__device__ __forceinline__ float gate_of(const KvArgs& a, int t, int h, int ch) {
  const size_t at = (size_t)t * a.stride + (size_t)h * 2 * a.HD + a.HD + ch;
  return a.dtype == 0 ? gp<float>(a.rows)[at] : (float)gp<_Float16>(a.rows)[at];
}
__device__ __forceinline__ f4 gate4(const KvArgs& a, int t, int h, int ch) {
  const size_t at = (size_t)t * a.stride + (size_t)h * 2 * a.HD + a.HD + ch;
  return a.dtype == 0 ? ld4(static_cast<const float*>(a.rows) + at) : ld4(static_cast<const _Float16*>(a.rows) + at);
}
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }

// Partial results of one column of one piece: O (unnormalised) [HD], then the columns' (maximum, sum).
struct Parts {
  float* p;
  int cols, ns;  // columns a slot, pieces a column block
  __device__ __forceinline__ size_t slot(const KvArgs& a, int ncb, int b, int kh, int cb, int piece) const {
    return (((size_t)b * a.HK + kh) * ncb + cb) * ns + piece;
  }
};

template <int HD>
__global__ __launch_bounds__(64 * kWaves, 2) void kv_few_kernel(KvArgs a, int chunk, int ncb, Parts parts) {
  constexpr int G = HD / 4, kH = HD / 128, kE = HD / 64, kRow = HD / 2;
  constexpr int kPitch = HD + 4;
  __shared__ float ol[kWaves * kCols * kPitch];
  __shared__ float ml[kWaves][kCols][2];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, j = lane & 15, kg = lane >> 4;
  const int piece = blockIdx.x, b = blockIdx.z, kh = blockIdx.y / ncb, cb = blockIdx.y % ncb;
  const int ratio = a.HQ / a.HK;
  const Seq sq = seq_of(a, b);
  const int cols = min(kCols, sq.n * ratio - cb * kCols);
  if (cols <= 0) return;
  const int r0 = cb * kCols;
  if (!sq.ok) {
    if (piece == 0)
      for (int k = tid; k < cols * HD; k += 64 * kWaves) {
        const int r = r0 + k / HD;
        a.out[((size_t)(sq.r0 + r / ratio) * a.HQ + kh * ratio + r % ratio) * HD + k % HD] = (_Float16)__builtin_nanf("");
      }
    return;
  }
  const int before = sq.len - sq.n;
  const int keys = before + (r0 + cols - 1) / ratio + 1, ns = (keys + chunk - 1) / chunk;
  if (piece >= ns) return;
  const int k0 = piece * chunk, k1 = min(k0 + chunk, keys);
  const int all = before + r0 / ratio + 1;  // keys below this are seen by every column
  const int r = r0 + min(j, cols - 1), last = before + r / ratio;

  h8 q[kH][4];
  float qs[4];  // sum of the column's q over each group
  {
    const _Float16* qp = a.q + ((size_t)(sq.r0 + r / ratio) * a.HQ + kh * ratio + r % ratio) * HD + 8 * kg;
#pragma unroll
    for (int h = 0; h < kH; h++)
#pragma unroll
      for (int g = 0; g < 4; g++) q[h][g] = *gp<h8>(qp + G * g + 32 * h);
#pragma unroll
    for (int g = 0; g < 4; g++) {
      float s = 0.0f;
#pragma unroll
      for (int h = 0; h < kH; h++) {
        const h8 x = q[h][g];
#pragma unroll
        for (int e = 0; e < 8; e++) s += (float)x[e];
        q[h][g] = h8{x[0], x[4], x[1], x[5], x[2], x[6], x[3], x[7]};
      }
      qs[g] = sum_quads(s);
    }
  }
  const float scale = a.scale * kLog2e;
  f4 o[4][kE], zs[4];
#pragma unroll
  for (int g = 0; g < 4; g++) {
    zs[g] = f4{};
#pragma unroll
    for (int e = 0; e < kE; e++) o[g][e] = f4{};
  }
  float m = -INFINITY, sum = 0.0f;
  const size_t blk_bytes = kv_block_bytes(a.page, HD);
  const unsigned par_off = (unsigned)a.page * kRow;
  const int* table = a.table + (size_t)b * a.table_stride;
  int ids = 0, seg = -1;  // lane k: the page of tokens 1024 seg + 16 k .. + 15 of the piece

  for (int t0 = k0 + kStep * wave; t0 < k1; t0 += kStep * kWaves) {
    if ((t0 - k0) >> 10 != seg) {
      seg = (t0 - k0) >> 10;
      const int tok = k0 + 1024 * seg + 16 * lane;
      ids = tok < keys ? gp<int>(table)[tok >> a.page_log2] : 0;
    }
    // this step's 32 keys: two tiles of 16, each in one page
    const unsigned char* blk[2];
    int slot[2];
    bool gone[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int id = __builtin_amdgcn_readlane(ids, ((t0 - k0) & 1023) / 16 + i);
      gone[i] = (unsigned)id >= (unsigned)a.n_pages;
      blk[i] = a.pool + ((size_t)(gone[i] ? 0 : id) * a.HK + kh) * 2 * blk_bytes;
      slot[i] = (t0 + 16 * i) & (a.page - 1);
    }
    u4 kc[2][kH], kp[2][4], vp[2][4];
    u2 vc[2][4];
#pragma unroll
    for (int i = 0; i < 2; i++) {
#pragma unroll
      for (int h = 0; h < kH; h++) kc[i][h] = *gp<u4>(blk[i] + (unsigned)((slot[i] + j) * kRow + 64 * h + 16 * kg));
#pragma unroll
      for (int g = 0; g < 4; g++) kp[i][g] = *gp<u4>(blk[i] + par_off + (unsigned)((slot[i] + 4 * kg) * 16 + 16 * g));
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
#pragma unroll
      for (int k = 0; k < 4; k++)
        vc[i][k] = *gp<u2>(blk[i] + blk_bytes + (unsigned)((slot[i] + 4 * kg + k) * kRow + 8 * (HD == 256 ? j : j & 7)));
#pragma unroll
      for (int g = 0; g < 4; g++) vp[i][g] = *gp<u4>(blk[i] + blk_bytes + par_off + (unsigned)((slot[i] + 4 * kg) * 16 + 16 * g));
    }
    // scores of tokens t0 + 16 i + 4 kg + k
    float sc[2][4];
#pragma unroll
    for (int i = 0; i < 2; i++) {
#pragma unroll
      for (int k = 0; k < 4; k++) sc[i][k] = 0.0f;
#pragma unroll
      for (int g = 0; g < 4; g++) {
        f4 acc = f4{} - 24.0f * qs[g];
#pragma unroll
        for (int h = 0; h < kH; h++) {
          const unsigned x = halves(kc[i][h][g >> 1], kc[i][h][(g >> 1) + 2], g & 1);
          const u4 op = {code2(x, 0), code2(x, 1), code2(x, 2), code2(x, 3)};
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, op), q[h][g], acc, 0, 0, 0);
        }
        const h8 p = __builtin_bit_cast(h8, kp[i][g]);
#pragma unroll
        for (int k = 0; k < 4; k++) sc[i][k] = fmaf((float)p[k], acc[k], fmaf((float)p[4 + k], qs[g], sc[i][k]));
      }
    }
    const bool edge = t0 + kStep > all || gone[0] || gone[1];
    u4 keep = {~0u, ~0u, ~0u, ~0u};  // the column's half-words of P that are not masked
    if (edge) {
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int tok = t0 + 16 * i + 4 * kg + k;
          if (gone[i]) sc[i][k] = __builtin_nanf("");
          if (tok > last) {
            sc[i][k] = -INFINITY;
            keep[2 * i + (k >> 1)] &= k & 1 ? 0x0000FFFFu : 0xFFFF0000u;
          }
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
        const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[i][k], scale, -base)), p1 = __builtin_amdgcn_exp2f(fmaf(sc[i][k + 1], scale, -base));
        sum += p0 + p1;
        p[2 * i + k / 2] = as_u(h2{(_Float16)p0, (_Float16)p1});
      }
    const h8 ph = __builtin_bit_cast(h8, p);
    const _Float16 off = (_Float16)-24.0f;
#pragma unroll
    for (int g = 0; g < 4; g++) {
      u4 w;  // P s_g
#pragma unroll
      for (int k = 0; k < 4; k++) w[k] = as_u(as_h2(p[k]) * as_h2(vp[k >> 1][g][k & 1]));
      if (edge) w &= keep;
      const h8 wh = __builtin_bit_cast(h8, w);
      const u4 z = {vp[0][g][2], vp[0][g][3], vp[1][g][2], vp[1][g][3]};
      zs[g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, z), ph, zs[g], 0, 0, 0);
      zs[g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h8{off, off, off, off, off, off, off, off}, wh, zs[g], 0, 0, 0);
      unsigned x[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        x[k] = halves(vc[k >> 1][2 * (k & 1)][g >> 1], vc[k >> 1][2 * (k & 1) + 1][g >> 1], g & 1);
        if constexpr (HD == 128) x[k] >>= 8 * (j >> 3);
      }
#pragma unroll
      for (int e = 0; e < kE; e++) {
        const u4 op = {code2(x[0], e), code2(x[1], e), code2(x[2], e), code2(x[3], e)};
        o[g][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, op), wh, o[g][e], 0, 0, 0);
      }
    }
  }
  // the four waves' sums: O^T row 4 kg + k of (g, e) is channel G g + 16 kg + 4 k + e (HD 256)
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
      const size_t s = (parts.slot(a, ncb, b, kh, cb, piece) * parts.cols + c) * (HD + 4);
      *reinterpret_cast<f4*>(parts.p + s + ch) = v;
      if (ch == 0) {
        parts.p[s + HD] = mm;
        parts.p[s + HD + 1] = l;
      }
    } else {
      const int rr = r0 + c, t = sq.r0 + rr / ratio, h = kh * ratio + rr % ratio;
      v *= 1.0f / l;
      if (a.gated) {
        const f4 gt = gate4(a, t, h, ch);
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] *= sigmoid(gt[e]);
      }
      *gpw<h4>(a.out + ((size_t)t * a.HQ + h) * HD + ch) = to_h4(v);
    }
  }
}

// out of one (row, head) from its pieces: thread (k, c) adds pieces k, k + blockDim / (HD / 4), ... of channels 4 c .. + 3.
template <int HD>
__global__ __launch_bounds__(1024) void kv_merge_kernel(KvArgs a, int chunk, int ncb, int block_cols, Parts parts) {
  constexpr int C = HD / 4;
  __shared__ float wl[1024];
  __shared__ f4 vl[1024];
  const int tid = threadIdx.x, i = blockIdx.x, h = blockIdx.y, b = blockIdx.z, ratio = a.HQ / a.HK, kh = h / ratio;
  const Seq sq = seq_of(a, b);
  if (i >= sq.n || !sq.ok) return;
  const int col = i * ratio + h % ratio, cb = col / block_cols, c = col % block_cols;
  const int end = min(block_cols, sq.n * ratio - cb * block_cols);
  const int keys = sq.len - sq.n + (cb * block_cols + end - 1) / ratio + 1, ns = (keys + chunk - 1) / chunk;
  if (ns <= 1) return;
  const float* p = parts.p + (parts.slot(a, ncb, b, kh, cb, 0) * parts.cols + c) * (HD + 4);
  const size_t step = (size_t)parts.cols * (HD + 4);
  const int k = tid / C, n = blockDim.x / C, ch = 4 * (tid % C);
  float mm = -INFINITY, l = 0.0f;
  for (int s = 0; s < ns; s++) mm = fmaxf(mm, p[s * step + HD]);
  f4 v = {};
  for (int s = k; s < ns; s += n) {
    const float f = p[s * step + HD] == mm ? 1.0f : __builtin_amdgcn_exp2f(p[s * step + HD] - mm);
    l += f * p[s * step + HD + 1];
    v += f * ld4(p + s * step + ch);
  }
  vl[tid] = v;
  if (tid % C == 0) wl[k] = l;
  __syncthreads();
  if (k) return;
  for (int s = 1; s < n; s++) {
    v += vl[s * C + tid];
    l += wl[s];
  }
  const int t = sq.r0 + i;
  v *= 1.0f / l;
  if (a.gated) {
    const f4 gt = gate4(a, t, h, ch);
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] *= sigmoid(gt[e]);
  }
  *gpw<h4>(a.out + ((size_t)t * a.HQ + h) * HD + ch) = to_h4(v);
}

template <int HD>
hipError_t launch(const KvArgs& a, float* ws, size_t ws_bytes, hipStream_t s) {
  const int ratio = a.HQ / a.HK, most = a.max_rows * ratio, ncb = (most + kCols - 1) / kCols;
  Parts parts{ws, std::min(kCols, most), 1};
  // pieces: enough workgroups for the chip, as long as their results fit the workspace
  const long units = (long)a.n_seqs * a.HK * ncb;
  constexpr int kUnit = kStep * kWaves;
  long chunk = (units * a.max_len / 1024 + kUnit - 1) / kUnit * kUnit;
  chunk = std::max<long>(chunk, kUnit);
  const size_t col_bytes = (size_t)parts.cols * (HD + 4) * sizeof(float);
  while ((parts.ns = (int)((a.max_len + chunk - 1) / chunk)) > 1 && (size_t)units * parts.ns * col_bytes > ws_bytes) chunk *= 2;
  hipLaunchKernelGGL((kv_few_kernel<HD>), dim3(parts.ns, a.HK * ncb, a.n_seqs), dim3(64 * kWaves), 0, s, a, (int)chunk, ncb, parts);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || parts.ns == 1) return e;
  hipLaunchKernelGGL((kv_merge_kernel<HD>), dim3(a.max_rows, a.HQ, a.n_seqs), dim3(parts.ns > 32 ? 1024 : 256), 0, s, a, (int)chunk, ncb, kCols, parts);
  return hipGetLastError();
}

}  // namespace

size_t kv_workspace_bytes() { return (size_t)64 << 20; }

hipError_t launch_kv_attention(const KvArgs& a, void* ws, size_t ws_bytes, hipStream_t s) {
  return a.HD == 256 ? launch<256>(a, static_cast<float*>(ws), ws_bytes, s) : launch<128>(a, static_cast<float*>(ws), ws_bytes, s);
}

}  // namespace ha
