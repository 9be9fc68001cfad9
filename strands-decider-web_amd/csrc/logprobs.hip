// What the records of a row's logits (fused.hip) come to, gfx950: log probabilities of given tokens, the entropy, the largest
// tokens in order. No counterpart in the reference.
//
// With M the row's largest logit and Z = sum e^(z - M): lse = M + log Z, log p(t) = z_t - lse, entropy = log Z - sum e^(z - M)
// (z - M) / Z. Each block's record has its largest value apart from the sums over the others, so that a row with one near
// certain token keeps the digits of what is left. Sums over threads are in 64 bits.
//
// The top_k largest logits stand in the top_k blocks of the largest maxima: a block further down has nothing that top_k others
// do not exceed (with fewer blocks than that, all are looked at). Their largest columns, and every column of such a block whose second
// largest comes near the last of them, are multiplied out again in 64 bits, and so are the given tokens: sums in f32 differ by 1e-6 of
// the logits, which is enough to change the order of two tokens. Near: within what f32 sums may be off, which goes with sum |a| |w| and
// not with the logit (terms may cancel), so the chosen columns' own such sums are taken along. kLpMargin more blocks are looked at, and
// blocks are taken by (largest value, first block), so that equal logits come in order too. The 64-bit values of the blocks' largest
// columns also replace their f32 ones in Z.
// (The sizes cost 1 us of 78 to 90 for 8 rows x 248320, top 20, and 2 where a block is multiplied out, behind the other products; those that
// come within 2^-12 of the largest logits at once, beside the others, gains nothing.)
//
// Smaller vocabularies, where two of the top_k often share a block, or whose blocks are too few workgroups, have their logits
// stored in f32 by a product (fused.hip) and read here in the records' place (fused_plan.h says when).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "fused.h"
#include "fused_common.h"
#include "fused_plan.h"

namespace ha {
namespace {

constexpr int kLpSets = 256;  // sets of threads whose largest keys the cut is looked for in
static_assert(kLpSets >= kLpMaxTop + kLpMargin, "as many sets as blocks that are chosen");

typedef unsigned long long u64;

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) v += __shfl_xor(v, d);
  return v;
}

// 16 + code e of a packed block, its bits straight into the mantissa: two instructions for 2 and 4 bits (a conversion to f32 and one
// to f64 and a product took five: 2048 x 248320, top 5 75 us, now 69; 1744 x 2559 of 3 bits, top 32 114, now 104).
template <int BITS>
__device__ __forceinline__ double sixteen_and(const unsigned* wd, int e) {
  auto at16 = [](unsigned v, int from) { return from <= 16 ? v << (16 - from) : v >> (from - 16); };  // bit `from` to bit 16
  unsigned hi;
  if constexpr (BITS == 4) hi = at16(wd[e >> 3], 4 * (e & 7)) & 0x000F0000u;
  else hi = at16(wd[e >> 4], 2 * (e & 15)) & 0x00030000u;
  if constexpr (BITS == 3) hi |= (e <= 18 ? wd[2] << (18 - e) : wd[2] >> (e - 18)) & 0x00040000u;
  return __builtin_bit_cast(double, (u64)(hi | 0x40300000u) << 32);
}

// a[m] . W[n] of two rows n in 64 bits, by one wave: lanes over the packed blocks. SIZE: returns a bound on the larger sum |a| |w| (codes
// at their largest: within some four times), else 0.
template <int BITS, bool ASYM, bool SIZE>
__device__ float dot64(const FusedArgs& p, int m, const int* n, int lane, double* out) {
  const int nblk = p.K / 32, ng = p.K / p.group, gl = p.group == 64 ? 1 : 0;
  gptr<h8> ap = (gptr<h8>)(gp<_Float16>(p.a) + (size_t)m * p.K);
  out[0] = out[1] = 0.0;
  float most = 0.0f;
  for (int k = lane; k < nblk; k += 64) {
    unsigned wd[2][BITS];
    float s[2], b[2] = {0.0f, 0.0f};
    h8 av[4];
#pragma unroll
    for (int x = 0; x < 2; x++) {
      gptr<unsigned> wp = gp<unsigned>(p.q) + ((size_t)n[x] * nblk + k) * BITS;
#pragma unroll
      for (int i = 0; i < BITS; i++) wd[x][i] = wp[i];
      s[x] = f16_bits(gp<unsigned short>(p.s)[(size_t)n[x] * ng + (k >> gl)]);
      if constexpr (ASYM) b[x] = f16_bits(gp<unsigned short>(p.b)[(size_t)n[x] * ng + (k >> gl)]);
    }
#pragma unroll
    for (int j = 0; j < 4; j++) av[j] = ap[4 * k + j];
    double d[2] = {0.0, 0.0}, sum = 0.0;
    float abs_sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float af = (float)av[j][e];
        const double ad = (double)af;
        sum += ad;
        if constexpr (SIZE) abs_sum += fabsf(af);
#pragma unroll
        for (int x = 0; x < 2; x++) d[x] = fma(ad, sixteen_and<BITS>(wd[x], 8 * j + e), d[x]);
      }
    }
    constexpr double kMid = 1 << (BITS - 1);
#pragma unroll
    for (int x = 0; x < 2; x++) {
      out[x] += (double)s[x] * (d[x] - (16.0 + kMid) * sum);
      if constexpr (ASYM) out[x] += ((double)b[x] + kMid * (double)s[x]) * sum;
    }
    constexpr float kCodes = ASYM ? 2 * kMid : kMid;
    if constexpr (SIZE) most = fmaf(fmaxf(kCodes * fabsf(s[0]) + fabsf(b[0]), kCodes * fabsf(s[1]) + fabsf(b[1])), abs_sum, most);
  }
#pragma unroll
  for (int x = 0; x < 2; x++) out[x] = wave_sum(out[x]);
  if constexpr (SIZE) {
#pragma unroll
    for (int d = 32; d >= 1; d /= 2) most += __shfl_xor(most, d);
  }
  return most;
}

// A workgroup of T threads for a row. Dynamic LDS: list_cap keys, cand_cap values, their columns, the targets, list_cap maxima. STORED: the row's
// logits themselves (unscaled, f32), each a block of its own.
template <int BITS, bool ASYM, int T, bool STORED>
__global__ __launch_bounds__(T) void logprobs_kernel(LpArgs a, int nb, int list_cap, int cand_cap) {
  constexpr int kWaves = T / 64, kKeep = STORED ? (T < 512 ? 16 : 32) : T < 512 ? 0 : 4096 / T, kSets = kLpSets / 64;
  extern __shared__ __attribute__((aligned(16))) unsigned char sm[];
  __shared__ u64 best[kLpSets];
  __shared__ u64 threshold;
  __shared__ double red[2][kWaves];
  __shared__ int chosen[kLpMaxTop + kLpMargin];
  __shared__ int n_list, n_cand;
  __shared__ unsigned most;  // bits of the largest bound on a chosen column's sum |a| |w|
  u64* list = (u64*)sm;
  double* val = (double*)(list + list_cap);
  int* ids = (int*)(val + cand_cap);
  int* wanted = ids + cand_cap;
  unsigned* others = (unsigned*)(wanted + a.n_targets);
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), m = blockIdx.x;
  const int n_vocab = a.p.N, k = a.top_k, kk = min(k + kLpMargin, nb), nt = a.n_targets;
  const LpRecord* rec = STORED ? nullptr : a.p.rec + (size_t)m * nb;
  const float* logits = STORED ? a.logits + (size_t)m * nb : nullptr;
  auto key_of = [](float max, int i) { return (u64)ordered(max) << 32 | (0xFFFFFFFFu - (unsigned)i); };
  // records tid, tid + T, ...: the first kKeep stay in registers, loaded at once
  auto record = [&](int i) __attribute__((always_inline)) {
    if constexpr (STORED) return LpRecord{a.p.scale * logits[i], 0.0f, 0.0f, 0u};
    else return rec[i];
  };
  for (int t = tid; t < nt; t += T) wanted[t] = a.targets[(size_t)m * nt + t];
  LpRecord keep[kKeep + 1];
#pragma unroll
  for (int i = 0; i < kKeep; i++)
    if (i * T < nb) keep[i] = record(min(tid + i * T, nb - 1));
  auto each = [&](auto f) {
#pragma unroll
    for (int i = 0; i < kKeep; i++)
      if (tid + i * T < nb) f(keep[i], tid + i * T);
#pragma unroll 4
    for (int i = tid + kKeep * T; i < nb; i += T) f(record(i), i);
  };
  float top = kNoLogit;
  int at = -1;
  bool bad = false;
  each([&](const LpRecord& r, int i) {
    bad |= !(fabsf(r.max) <= 3.4e38f && fabsf(r.rest) <= 3.4e38f && fabsf(r.rest_z) <= 3.4e38f);
    if (r.max > top) top = r.max, at = i;
  });
  u64 mine = at < 0 ? 0 : key_of(top, at);
  // the largest key of every T / kLpSets threads (0: no block)
#pragma unroll
  for (int d = 1; d < T / kLpSets; d *= 2) mine = max(mine, (u64)__shfl_xor((long long)mine, d));
  if (tid % (T / kLpSets) == 0) best[tid / (T / kLpSets)] = mine;
  if (tid == 0) n_list = 0, n_cand = 0, most = 0;
  if (__syncthreads_or(bad)) {  // a logit that is not finite
    const float nan = __builtin_nanf("");
    for (int t = tid; t < nt; t += T) a.logp[(size_t)m * nt + t] = nan;
    for (int t = tid; t < k; t += T) a.top_ids[(size_t)m * k + t] = -1, a.top_logp[(size_t)m * k + t] = nan;
    if (tid == 0 && a.entropy) a.entropy[m] = nan;
    if (tid == 0 && a.lse) a.lse[m] = nan;
    return;
  }
  // a key that at least kk blocks reach and few others: the kk-th largest of those, found bit by bit (where there are fewer, 0)
  if (w == 0) {
    u64 v[kSets];
    u64 top = 0;
#pragma unroll
    for (int i = 0; i < kSets; i++) v[i] = best[lane + 64 * i], top = max(top, v[i]);
#pragma unroll
    for (int d = 32; d >= 1; d /= 2) top = max(top, (u64)__shfl_xor((long long)top, d));
    u64 t = 0;
    for (int bit = 63; bit >= 0; bit--) {
      const u64 next = t | 1ull << bit;
      int n = 0;
#pragma unroll
      for (int i = 0; i < kSets; i++) n += __popcll(__ballot(v[i] >= next));
      if (n >= kk) t = next;
      if (n == kk) break;
    }
    if (lane == 0) threshold = t, best[0] = top;
  }
  __syncthreads();
  const u64 cut = threshold, top_key = best[0];
  const float M = unordered((unsigned)(top_key >> 32));
  // sums over the blocks, a thread's in f32; the largest columns of those from the cut on wait
  const float cut_max = cut ? unordered((unsigned)(cut >> 32)) : kNoLogit;
  float z32 = 0.0f, zx32 = 0.0f;
  each([&](const LpRecord& r, int i) {
    const float x = r.max - M, e = __expf(x);
    float rest = r.rest + 1.0f;
    if (r.max >= cut_max && key_of(r.max, i) >= cut) list[atomicAdd(&n_list, 1)] = key_of(r.max, i), rest = r.rest;
    z32 = fmaf(e, rest, z32);
    zx32 = fmaf(e, fmaf(rest, x, r.rest_z), zx32);
  });
  double z = z32, zx = zx32;
  __syncthreads();
  // those in order, a wave for each (in the list they come in any order): the kk largest are chosen, the others go into the sums
  const int nl = n_list;
  for (int i = w; i < nl; i += kWaves) {
    const u64 key = list[i];
    int rank = 0;
    for (int j = 0; j < nl; j += 64) rank += __popcll(__ballot(j + lane < nl && list[min(j + lane, nl - 1)] > key));
    if (lane == 0 && rank < kk) chosen[rank] = (int)(0xFFFFFFFFu - (unsigned)key);
    if (lane == 0 && rank >= kk) others[rank - kk] = (unsigned)(key >> 32);
  }
  __syncthreads();
  for (int i = tid; i < nl - kk; i += T) {
    const double x = (double)unordered(others[i]) - (double)M, e = (double)__expf((float)x);
    z += e;
    zx += e * x;
  }
  z = wave_sum(z);
  zx = wave_sum(zx);
  if (lane == 0) red[0][w] = z, red[1][w] = zx;
  __syncthreads();
  // candidates: the chosen blocks' largest columns, then all others of blocks whose second largest may be among the top_k. Their values
  // stand behind those of the targets.
  unsigned second = 0;
  int arg = 0;
  float last = 0.0f;
  if (STORED && tid < kk) ids[tid] = chosen[tid];
  if (!STORED && tid < kk) {
    const LpRecord r = rec[chosen[tid]];
    arg = (int)(r.second & 63u);
    second = r.second & ~63u;
    ids[tid] = kLpBlock * chosen[tid] + arg;
    if (k > 0) last = rec[chosen[min(k, kk) - 1]].max;
  }
  __syncthreads();
  int from = 0, to = kk + nt;
#pragma unroll 1
  while (true) {
    for (int i = from + 2 * w; i < to; i += 2 * kWaves) {
      int n[2];
      bool token[2];
#pragma unroll
      for (int x = 0; x < 2; x++) {
        const int at = min(i + x, to - 1), id = at < kk ? ids[at] : at < kk + nt ? wanted[at - kk] : ids[at - nt];
        token[x] = (unsigned)id < (unsigned)n_vocab;  // (no token: its log probability is NaN)
        n[x] = token[x] ? id : 0;
      }
      double d[2];
      float size = 0.0f;
      if (!STORED && from == 0) size = dot64<BITS, ASYM, true>(a.p, m, n, lane, d);
      else dot64<BITS, ASYM, false>(a.p, m, n, lane, d);
#pragma unroll
      for (int x = 0; x < 2; x++)
        if (lane == 0 && i + x < to) val[i + x] = token[x] ? (double)a.p.scale * d[x] : __builtin_nan("");
      if (!STORED && lane == 0 && i < kk) atomicMax(&most, __builtin_bit_cast(unsigned, size));
    }
    __syncthreads();
    if (STORED || k == 0 || from > 0) break;
    // Two f32 sums of K / 32 groups: K / 32 additions and as many products, 40 within groups and reductions, each off by 2^-23 of
    // sum |a| |w| at most
    const float off = 2.0f * ((float)a.p.K / 16.0f + 40.0f) * 0x1p-23f * a.p.scale * __builtin_bit_cast(float, most);
    if (tid < kk && (kk < k || unordered(second) >= last - off)) {
      const int base = kLpBlock * chosen[tid], cols = min(kLpBlock, n_vocab - base);
      int at = kk + atomicAdd(&n_cand, cols - 1);
      for (int c = 0; c < cols; c++)
        if (c != arg) ids[at++] = base + c;
    }
    __syncthreads();
    if (n_cand == 0) break;
    from = to;
    to += n_cand;
  }
  const int nc = kk + n_cand;
  auto value = [&](int i) { return val[i < kk ? i : i + nt]; };  // of candidate i
  // every wave: the sums, with the chosen blocks' largest columns from 64 bits
  z = lane < kWaves ? red[0][lane] : 0.0;
  zx = lane < kWaves ? red[1][lane] : 0.0;
  for (int i = lane; i < kk; i += 64) {
    const double x = val[i] - (double)M, e = exp(x);
    z += e;
    zx += e * x;
  }
  z = wave_sum(z);
  zx = wave_sum(zx);
  const double log_z = log(z);
  auto logp = [&](double v) { return (float)((v - (double)M) - log_z); };
  if (tid == 0 && a.entropy) a.entropy[m] = (float)(log_z - zx / z);
  if (tid == 0 && a.lse) a.lse[m] = (float)((double)M + log_z);
  for (int t = tid; t < nt; t += T) a.logp[(size_t)m * nt + t] = logp(val[kk + t]);
  if (k > 0) {
    for (int i = w; i < nc; i += kWaves) {
      const double v = value(i);
      const int id = ids[i];
      int rank = 0;
      for (int j = 0; j < nc; j += 64) {
        const int at = min(j + lane, nc - 1);
        rank += __popcll(__ballot(j + lane < nc && (value(at) > v || (value(at) == v && ids[at] < id))));
      }
      if (lane == 0 && rank < k) a.top_ids[(size_t)m * k + rank] = id, a.top_logp[(size_t)m * k + rank] = logp(v);
    }
  }
}

// Dynamic LDS: keys and maxima of the list, values and columns of the candidates, targets. At most, over all vocabularies:
constexpr int kLpLds = 128 * 1024;
constexpr size_t lds_bytes(int list, int cand, int targets) { return 12 * (size_t)list + 12 * (size_t)cand + 4 * (size_t)targets; }
constexpr int list_most(int T, bool stored) {
  return (kLpMaxTop + kLpMargin) * (T / kLpSets) * (((stored ? fused::kStoredVocab : kLpMaxVocab / kLpBlock) + T - 1) / T);
}
constexpr int cand_most(bool stored) { return (kLpMaxTop + kLpMargin) * (stored ? 1 : kLpBlock) + kLpMaxTargets; }

template <int BITS, bool ASYM, int T, bool STORED>
hipError_t launch_as(const LpArgs& a, hipStream_t s) {
  const int nb = STORED ? a.p.N : (a.p.N + kLpBlock - 1) / kLpBlock, kk = std::min(a.top_k + kLpMargin, nb);
  // the kk sets of T / kLpSets threads that hold a key from the cut on (where there are fewer sets, all of them)
  const int list_cap = std::min(nb, kk * (T / kLpSets) * ((nb + T - 1) / T));
  const int cand_cap = (a.top_k > 0 && !STORED ? kk * kLpBlock : kk) + a.n_targets;
  const size_t lds = lds_bytes(list_cap, cand_cap, a.n_targets);
  static_assert(lds_bytes(list_most(T, STORED), cand_most(STORED), kLpMaxTargets) <= kLpLds, "what a call may need");
  auto k = logprobs_kernel<BITS, ASYM, T, STORED>;
  if (lds > 48 * 1024) {  // (the same limit for every call: it is the function's, not the launch's, and calls may overlap)
    const hipError_t e = hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, kLpLds);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(k, dim3(a.p.M), dim3(T), lds, s, a, nb, list_cap, cand_cap);
  return hipGetLastError();
}
// Few rows: 16 waves for each, more of its loads and products at once (one row over 248320 tokens, top 8: 19 -> 12 us, 13 with the columns'
// sizes). Many: as many rows on a CU as their blocks leave work for (2048 x 248320, 3880 blocks: 8 waves 71 us; before the ranks were
// counted by waves 8 waves 75, 4 waves 92, and 1431 rows of 1383 logits 53 and 41).
template <int BITS, bool ASYM, bool STORED>
hipError_t launch_for(const LpArgs& a, hipStream_t s) {
  if (a.p.M <= 256) return launch_as<BITS, ASYM, 1024, STORED>(a, s);
  return a.p.N > (STORED ? 4096 : 4096 * kLpBlock / 2) ? launch_as<BITS, ASYM, 512, STORED>(a, s) : launch_as<BITS, ASYM, 256, STORED>(a, s);
}
template <int BITS, bool ASYM>
hipError_t launch(const LpArgs& a, hipStream_t s) {
  return a.logits ? launch_for<BITS, ASYM, true>(a, s) : launch_for<BITS, ASYM, false>(a, s);
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
