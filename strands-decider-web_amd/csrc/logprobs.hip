// What the records of a row's logits (fused.hip) come to, gfx950: log probabilities of given tokens, the entropy, the largest
// tokens in order. No counterpart in the reference.
//
// With M the row's largest logit and Z = sum e^(z - M): lse = M + log Z, log p(t) = z_t - lse, entropy = log Z - sum e^(z - M)
// (z - M) / Z. Each block's record has its largest value apart from the sums over the others, so that a row with one near
// certain token keeps the digits of what is left. Sums over blocks are in 64 bits.
//
// The top_k largest logits stand in the top_k blocks of the largest maxima: a block further down has nothing that top_k others
// do not exceed (with fewer blocks than that, all are looked at). Their largest columns, and every column of such a block whose second largest comes near the last of them, are
// multiplied out again in 64 bits, and so are the given tokens: sums in f32 differ by 1e-6 of the logits, which is enough to
// change the order of two tokens. kLpMargin more blocks are looked at, and blocks are taken by (largest value, first block), so
// that equal logits come in order too. The 64-bit values of the blocks' largest columns also replace their f32 ones in Z.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "fused.h"
#include "fused_common.h"

namespace ha {
namespace {

constexpr int kT = 512, kWaves = kT / 64;
typedef unsigned long long u64;

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) v += __shfl_xor(v, d);
  return v;
}

// a[m] . W[n] in 64 bits, by one wave: lanes over the packed blocks.
template <int BITS, bool ASYM>
__device__ double dot64(const FusedArgs& p, int m, int n, int lane) {
  const int nblk = p.K / 32, ng = p.K / p.group, gl = p.group == 64 ? 1 : 0;
  gptr<unsigned> wp = gp<unsigned>(p.q) + (size_t)n * nblk * BITS;
  gptr<h8> ap = (gptr<h8>)(gp<_Float16>(p.a) + (size_t)m * p.K);
  double acc = 0.0;
  for (int k = lane; k < nblk; k += 64) {
    unsigned wd[BITS];
#pragma unroll
    for (int i = 0; i < BITS; i++) wd[i] = wp[(size_t)k * BITS + i];
    const double s = f16_bits(gp<unsigned short>(p.s)[(size_t)n * ng + (k >> gl)]);
    double d = 0.0, sum = 0.0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const h8 av = ap[4 * k + j];
      unsigned lo, hi = 0;
      if constexpr (BITS == 4) lo = wd[j];
      else lo = wd[j >> 1] >> (16 * (j & 1)) & 0xFFFFu;
      if constexpr (BITS == 3) hi = wd[BITS - 1] >> (8 * j) & 0xFFu;
      const h8 c = codes8<BITS>(lo, hi);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        d += (double)((float)av[e] * (float)c[e]);  // (15 bits: exact)
        if constexpr (ASYM) sum += (double)(float)av[e];
      }
    }
    acc += s * d;
    if constexpr (ASYM) acc += ((double)f16_bits(gp<unsigned short>(p.b)[(size_t)n * ng + (k >> gl)]) + (1 << (BITS - 1)) * s) * sum;
  }
  return wave_sum(acc);
}

// A workgroup for a row. Dynamic LDS: list_cap keys, then cand_cap values and their columns.
template <int BITS, bool ASYM>
__global__ __launch_bounds__(kT) void logprobs_kernel(LpArgs a, int nb, int list_cap, int cand_cap) {
  extern __shared__ __attribute__((aligned(16))) unsigned char sm[];
  __shared__ u64 best[kT];
  __shared__ u64 threshold;
  __shared__ double red[2][kWaves];
  __shared__ int chosen[kLpMaxTop + kLpMargin];
  __shared__ int n_list, n_cand;
  u64* list = (u64*)sm;
  double* val = (double*)(list + list_cap);
  int* ids = (int*)(val + cand_cap);
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), m = blockIdx.x;
  const int n_vocab = a.p.N, k = a.top_k, kk = min(k + kLpMargin, nb);
  const LpRecord* rec = a.p.rec + (size_t)m * nb;
  auto key_of = [](float max, int i) { return (u64)ordered(max) << 32 | (0xFFFFFFFFu - (unsigned)i); };
  // the thread's largest key (0: no block)
  u64 mine = 0;
  bool bad = false;
  for (int i = tid; i < nb; i += kT) {
    const LpRecord r = rec[i];
    bad |= !(fabsf(r.max) <= 3.4e38f && fabsf(r.rest) <= 3.4e38f && fabsf(r.rest_z) <= 3.4e38f);
    mine = max(mine, key_of(r.max, i));
  }
  best[tid] = mine;
  if (tid == 0) n_list = 0, n_cand = 0;
  if (__syncthreads_or(bad)) {  // a logit that is not finite
    const float nan = __builtin_nanf("");
    for (int t = tid; t < a.n_targets; t += kT) a.logp[(size_t)m * a.n_targets + t] = nan;
    for (int t = tid; t < k; t += kT) a.top_ids[(size_t)m * k + t] = -1, a.top_logp[(size_t)m * k + t] = nan;
    if (tid == 0 && a.entropy) a.entropy[m] = nan;
    if (tid == 0 && a.lse) a.lse[m] = nan;
    return;
  }
  // a key that at least kk blocks reach and few others: the kk-th largest of the threads' largest, found bit by bit
  if (w == 0) {
    u64 v[kWaves];
    u64 top = 0;
#pragma unroll
    for (int i = 0; i < kWaves; i++) v[i] = best[lane + 64 * i], top = max(top, v[i]);
#pragma unroll
    for (int d = 32; d >= 1; d /= 2) top = max(top, (u64)__shfl_xor((long long)top, d));
    u64 t = 0;
    for (int bit = 63; bit >= 0; bit--) {
      const u64 next = t | 1ull << bit;
      int n = 0;
#pragma unroll
      for (int i = 0; i < kWaves; i++) n += __popcll(__ballot(v[i] >= next));
      if (n >= kk) t = next;
      if (n == kk) break;
    }
    if (lane == 0) threshold = t, best[0] = top;
  }
  __syncthreads();
  const u64 cut = threshold, top_key = best[0];
  const float M = unordered((unsigned)(top_key >> 32));
  // sums over the blocks; the largest columns of those from the cut on wait
  double z = 0.0, zx = 0.0;
  for (int i = tid; i < nb; i += kT) {
    const LpRecord r = rec[i];
    const u64 key = key_of(r.max, i);
    const double x = (double)r.max - (double)M, e = (double)__expf((float)x);
    double rest = r.rest;
    if (key >= cut) list[atomicAdd(&n_list, 1)] = key;
    else rest += 1.0;
    z += e * rest;
    zx += e * ((double)r.rest_z + rest * x);
  }
  __syncthreads();
  const int nl = n_list;
  for (int i = tid; i < nl; i += kT) {
    const u64 key = list[i];
    int rank = 0;
    for (int j = 0; j < nl; j++) rank += list[j] > key;
    if (rank < kk) {
      chosen[rank] = (int)(0xFFFFFFFFu - (unsigned)key);
    } else {
      const double x = (double)unordered((unsigned)(key >> 32)) - (double)M, e = (double)__expf((float)x);
      z += e;
      zx += e * x;
    }
  }
  z = wave_sum(z);
  zx = wave_sum(zx);
  if (lane == 0) red[0][w] = z, red[1][w] = zx;
  __syncthreads();
  // candidates: the chosen blocks' largest columns, and blocks whose second largest may be among the top_k
  if (tid < kk) {
    const int i = chosen[tid];
    const LpRecord r = rec[i];
    const int arg = (int)(r.second & 63u);
    ids[tid] = kLpBlock * i + arg;
    if (k > 0) {
      const float last = rec[chosen[min(k, kk) - 1]].max;
      const float near = last - fmaxf(fabsf(M), fabsf(last)) * 0x1p-12f;
      if (kk < k || unordered(r.second & ~63u) >= near) {
        const int cols = min(kLpBlock, n_vocab - kLpBlock * i);
        int at = kk + atomicAdd(&n_cand, cols - 1);
        for (int c = 0; c < cols; c++)
          if (c != arg) ids[at++] = kLpBlock * i + c;
      }
    }
  }
  __syncthreads();
  const int nc = kk + n_cand, nt = a.n_targets;
  for (int i = w; i < nc + nt; i += kWaves) {
    int n = i < nc ? ids[i] : a.targets[(size_t)m * nt + i - nc];
    if ((unsigned)n >= (unsigned)n_vocab) {  // no token: its log probability is NaN
      if (lane == 0) val[i] = __builtin_nan("");
      continue;
    }
    const double d = (double)a.p.scale * dot64<BITS, ASYM>(a.p, m, n, lane);
    if (lane == 0) val[i] = d;
  }
  __syncthreads();
  z = zx = 0.0;
  for (int i = 0; i < kWaves; i++) z += red[0][i], zx += red[1][i];
  for (int i = 0; i < kk; i++) {
    const double x = val[i] - (double)M, e = exp(x);
    z += e;
    zx += e * x;
  }
  const double log_z = log(z);
  auto logp = [&](double v) { return (float)((v - (double)M) - log_z); };
  if (tid == 0 && a.entropy) a.entropy[m] = (float)(log_z - zx / z);
  if (tid == 0 && a.lse) a.lse[m] = (float)((double)M + log_z);
  for (int t = tid; t < nt; t += kT) a.logp[(size_t)m * nt + t] = logp(val[nc + t]);
  if (k > 0) {
    for (int i = tid; i < nc; i += kT) {
      const double v = val[i];
      const int id = ids[i];
      int rank = 0;
      for (int j = 0; j < nc; j++) rank += val[j] > v || (val[j] == v && ids[j] < id);
      if (rank < k) a.top_ids[(size_t)m * k + rank] = id, a.top_logp[(size_t)m * k + rank] = logp(v);
    }
  }
}

template <int BITS, bool ASYM>
hipError_t launch(const LpArgs& a, hipStream_t s) {
  const int nb = (a.p.N + kLpBlock - 1) / kLpBlock, kk = std::min(a.top_k + kLpMargin, nb);
  const int list_cap = kk * ((nb + kT - 1) / kT), cand_cap = (a.top_k > 0 ? kk * kLpBlock : kk) + a.n_targets;
  const size_t lds = 8 * (size_t)list_cap + 12 * (size_t)cand_cap;
  auto k = logprobs_kernel<BITS, ASYM>;
  if (lds > 48 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(k, dim3(a.p.M), dim3(kT), lds, s, a, nb, list_cap, cand_cap);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_logprobs(const LpArgs& a, hipStream_t s) {
  switch (2 * a.p.bits + (a.p.asym ? 1 : 0)) {
    case 4: return launch<2, false>(a, s);
    case 5: return launch<2, true>(a, s);
    case 6: return launch<3, false>(a, s);
    case 7: return launch<3, true>(a, s);
    case 8: return launch<4, false>(a, s);
    case 9: return launch<4, true>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace ha
