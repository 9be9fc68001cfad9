// Causal grouped-query attention over the paged 4-bit K/V cache, gfx950.
//
//   out[t][h] = sum_j softmax_j(scale q[t][h] . k_j) v_j * sigmoid(gate[t][h]),  j <= position of row t
//
// The rows of a sequence that share a KV head are its columns: row i, head hh of the group is column i ratio + hh, so the
// matrix products have as many columns as the group has heads, also where a sequence has a single new token.
//
// kv_few_kernel: a workgroup has 16 columns and a piece of the keys, its four waves 32 keys each in turn, with nothing shared
// until the end. It computes S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_f16, straight from the codes:
//   - a code c in the low bits of an f16 whose exponent is 2^10 (2^6, 2^4) is the number 1024 + c (64 + c, 16 + c), as published for
//     4-bit weights (Kim et al. 2022, arXiv 2211.10017): with a v_perm and an and-or for two codes, the operands need no
//     arithmetic. K's products start at -1032 sum(q) (-72 sum(q) for the others), as the C operand, which leaves
//     sum(q (c - 8)) with f32 roundings only; the scale and zero of a group come in afterwards, on its 16 x 16 sums:
//     S = sum_g s_g (q . (c - 8))_g + z_g sum(q_g).
//   - K's operand is 16 bytes of a token's row a lane, V's 8 bytes of 8 tokens' rows, two tokens' half-words joined by
//     v_perm; S^T's layout (a column a lane) is that of P^T as an operand, so P goes from registers to registers.
//   - V's scales go onto P (P s_g), and its zeros into one more sum for each group, sum P z_g; that product's other rows give
//     sum P s_g, of which the codes' offset, -24 times it, is added after every segment of 1024 keys.
//   - a column's maximum is the wave's own; it is raised only when a score exceeds what P may be (Range).
// P and P s_g are sums of two f16 each (22 bits), whose products take two matrix instructions: the output's error is its own
// rounding, 2.07e-4 of its norm, where one f16 each gave 2.5 to 3.1e-4, the more the longer the context, and took 1 to 5 % less
// time (us: 61 rows after 1531 16.4 / 16.7, 2 x 1000 rows after 1000 97 / 101, 64 sequences of 8192 59.4 / 62.2). Sums are f32.
// Pieces leave their O, maximum and sum in the workspace; the last of a unit's pieces joins them, or kv_merge_kernel where
// they are many. Two workgroups a CU (242 registers for HD 256) and codes fetched a step ahead keep memory busy where there are
// few columns: 8 sequences of 32768 tokens, 2 x 4 heads of 256, 151 MB: 34.7 us, 4.4 TB/s (a copy 4.8). With 16 columns
// and more it is bound by the vector instructions that unpack codes (2048 rows of 8 sequences: 455 us), which kv_many_kernel shares
// among 128 columns (284 us, 485 TFLOP/s).
#include <algorithm>
#include <cmath>

#include "kv_common.h"

namespace ha {
namespace {

typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
// P = exp2(score - m) and P s are f16, whose steps end at 2^-24, so P is kept high: m is `lift` below a column's maximum when it is
// set, and set again when a score exceeds m by more than `room`, by the largest scale of the tile's values. P s stays below 2^16, and
// P is at least 1 for the column's heaviest key.
struct Range {
  float room, lift;
  __device__ __forceinline__ explicit Range(int cls) : room(cls == 0 ? 14.0f : cls == 1 ? 6.0f : 0.0f), lift(cls == 0 ? 8.0f : 0.0f) {}
};
// the class of two words of scales: 0 below 2, 1 below 512, 2 (and NaN)
__device__ __forceinline__ int scale_class(unsigned s, unsigned t) {
  return ((s & (s << 1)) | (t & (t << 1))) & 0x40004000u ? 2 : (s | t) & 0x40004000u ? 1 : 0;
}
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kCols = 16, kWaves = 4, kStep = 32;  // few columns: of a workgroup; waves; keys a wave's step
constexpr int kBigCols = 128, kTile = 32;          // many columns

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

// (Results of inline asm may go straight into a matrix instruction, before which the compiler waits for instructions it knows: they
// end with the two wait states that it would put there.)
// (a0, a1) as a sum of two f16 each, 22 bits: the first cut off, so that the rest has its sign
__device__ __forceinline__ u2 split2(float a0, float a1) {
  const unsigned hi = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(a0, a1));
  unsigned lo;
  asm("v_fma_mixlo_f16 %0, %1, 1.0, -%3 op_sel_hi:[0,0,1]\n\t"
      "v_fma_mixhi_f16 %0, %2, 1.0, -%3 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n\t"
      "s_nop 1" : "=&v"(lo) : "v"(a0), "v"(a1), "v"(hi));
  return u2{hi, lo};
}
// the products of such a pair of sums and the f16 s, again as two f16: h s rounded, and what that leaves (exact) with l s
__device__ __forceinline__ u2 scale2(unsigned h, unsigned l, unsigned s) {
  const h2 w = as_h2(h) * as_h2(s);
  return u2{as_u(w), as_u(__builtin_elementwise_fma(as_h2(l), as_h2(s), __builtin_elementwise_fma(as_h2(h), as_h2(s), -w)))};
}
// the larger of two f16 each, NaN the smaller
__device__ __forceinline__ u2 max2(u2 x, unsigned y) {
  unsigned a = x[0], b = x[1];
  asm("v_pk_max_f16 %0, %0, %2\n\tv_pk_max_f16 %1, %1, %2\n\ts_nop 1" : "+v"(a), "+v"(b) : "v"(y));
  return u2{a, b};
}

__device__ __forceinline__ f4 gate4(const KvArgs& a, int t, int h, int ch) {
  const size_t at = (size_t)t * a.stride + (size_t)h * 2 * a.HD + a.HD + ch;
  return a.dtype == 0 ? ld4(static_cast<const float*>(a.rows) + at) : ld4(static_cast<const _Float16*>(a.rows) + at);
}
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }

// ---- who does what ----
//
// The host knows neither how long the sequences are nor which of them have many rows, so the device shares the work out. A
// sequence is of one of two kinds (few or many columns); its (column block, KV head)s are units. Units of few columns
// are cut into pieces of `chunk` keys, chosen so that all of them make about `want` pieces; those of many columns, which are only
// used where they fill the chip, are not. A workgroup's index is its place in the list of all pieces of all sequences, which
// each wave finds by a prefix sum with a sequence a lane. Of more than kScanMost sequences the sums are taken once, by
// kv_plan_kernel, and searched. Short contexts of that many sequences, and equal sequences with many columns, are laid out in a
// grid instead (`direct`), with the host's bounds.
constexpr int kWant = 512;                // pieces: two workgroups a CU
constexpr size_t kSlots = 2 * kWant;      // (cut units have less than 2 kWant pieces)
constexpr size_t kSlotBytes = (size_t)kCols * (256 + 4) * sizeof(float);
constexpr int kFewCols = 256, kManyUnits = 160;  // (see attend())
struct Kind {
  float* p;  // results of the pieces of cut units: for each piece and column O (unnormalised) [HD], maximum, sum
  int* count;  // of a cut unit's pieces (a group's) that are done, at the first one's slot, then of its groups; zero between calls
  int* plan;   // or nullptr: keys a piece, limit_of(); then for each sequence the sums up to and with it of its pieces, of those of
               // them that are cut, and of its (row, head)s to be merged, and the greatest row_start up to its own
  int cols;  // columns a block has, at most
  int split;   // both kinds are in use
  int want, direct, ncb;
};
constexpr int kPlanHead = 2;
struct Item {
  int b, kh, cb, piece, size, slot;  // size: keys a piece; slot: of the piece, where there is more than one
  int row;                            // of the sequence (merge)
  Seq sq;
};
constexpr int kScanMost = 128, kPlanMost = 65536;

// a lane's sequence: its rows and units
struct Lane {
  Seq sq;
  int ncb;
};
// A unit of many columns is not cut: one that walks many more keys than the others would end long after them. So a sequence of more
// than kFewCols columns is only one of many where its context is at most `limit`: the keys of all such sequences' units over
// kManyUnits, w / kManyUnits: its units then end within 256 / kManyUnits of the time in which those of all would, spread evenly.
// (6 prompts of 1000 rows and 100 rows after 6000, 20000 and 131000 tokens, us: 124, 167 and 384; 326, 1010 and 6470 without a limit.)
// (No contraction: the kernels of a call have to agree on it.)
__device__ __forceinline__ float wide_keys(const KvArgs& a, const Seq& sq) {
#pragma clang fp contract(off)
  const int cols = sq.n * a.ratio;
  return cols > kFewCols ? (float)((cols + kBigCols - 1) / kBigCols) * (float)sq.len : 0.0f;
}
__device__ __forceinline__ int limit_of(const KvArgs& a, float w) { return uniform((int)fminf(w * (float)a.HK * (1.0f / kManyUnits), 1e9f)); }
__device__ __forceinline__ int limit_of(const KvArgs& a, const Kind& k, const Seq& first, int lane, int top) {
#pragma clang fp contract(off)
  if (!k.split) return 0;
  float w = wide_keys(a, first);
  for (int s0 = 64; s0 < a.n_seqs; s0 += 64) w += wide_keys(a, seq_in_order(a, s0 + lane, top));
  return limit_of(a, __builtin_bit_cast(float, lane_value(__builtin_bit_cast(int, scan64(w)), 63)));
}
template <int BC>
__device__ __forceinline__ Lane lane_of(const KvArgs& a, const Kind& k, const Seq& sq, int limit) {
  Lane l{sq, 0};
  const int cols = sq.n * a.ratio;
  const bool many = k.split && cols > kFewCols && sq.len <= limit;
  if (cols > 0 && many == (BC == kBigCols)) l.ncb = sq.ok ? (cols + BC - 1) / BC : 1;  // (one unit writes all rows of a sequence that does not fit)
  return l;
}
constexpr int kUnit = kStep * kWaves;  // keys that a piece has at least
constexpr int kEven = 4;               // times that, from which pieces are made even
// a / s of 0 <= a < 2^21, s > 0: (a + 1/2) / s is 1 / (2 s) away from the next integer, its error at most a 2^-22 / s
__device__ __forceinline__ int small_div(int a, int s) { return (int)(((float)a + 0.5f) * __builtin_amdgcn_rcpf((float)s)); }
// Keys a piece of a sequence, a multiple of kUnit: `chunk` where that is short, else as near to it as pieces of one size come.
// (240 sequences of 3001 tokens, us: 88 so, 135 with a short last piece.)
__device__ __forceinline__ int size_of(int len, int chunk) {
  const int c = chunk / kUnit, u = (len + kUnit - 1) / kUnit;
  if (c < kEven) return chunk;
  const int n = max(1, small_div(u + c / 2, c));
  return small_div(u + n - 1, n) * kUnit;
}
__device__ __forceinline__ int pieces_of(int len, int size) {
  const int s = size / kUnit;
  return len > size ? small_div((len + kUnit - 1) / kUnit + s - 1, s) : 1;
}
// keys a piece: the keys of one KV head's units, w, over `want`
__device__ __forceinline__ int chunk_of(const KvArgs& a, const Kind& k, float w) {
  return uniform(kUnit * max(1, (int)fminf(ceilf(w * (float)a.HK / (float)(k.want * kUnit)), 1e6f)));
}
__device__ __forceinline__ int chunk_of(const KvArgs& a, const Kind& k, const Lane& first, int lane, int top, int limit) {
  float w = (float)first.ncb * (float)first.sq.len;
  for (int s0 = 64; s0 < a.n_seqs; s0 += 64) {
    const Lane l = lane_of<kCols>(a, k, seq_in_order(a, s0 + lane, top), limit);
    w += (float)l.ncb * (float)l.sq.len;
  }
  return chunk_of(a, k, __builtin_bit_cast(float, lane_value(__builtin_bit_cast(int, scan64(w)), 63)));
}
// A unit's ns pieces are joined by the last of them, or by the last of each group of neighbours and then the last of the groups, or
// by kv_merge_kernel. The pieces of a group (ns: one group), or 0 for the merge: joining costs what a thread loads one after the other.
// Measured, us, joined / merged: one row (4 columns) after 8000 (63 pieces) 11.1 / 12.9, after 20000 (157) 15.9 / 16.7, after 131071
// (512) 25.1 / 27.2; 4 sequences of 8000 (63) 14.4 / 15.7; after 4000 (32) 11.0 in groups, 12.0 at once; 2 rows (8 columns) after
// 1000 (8) 10.6 / 11.6, after 8000 (63) 23.6 / 13.3; 61 rows (16 columns) after 1531 (13) 24.4 / 17.3, of heads of 128 after 1000 (9)
// 14.7 / 16.6. (61 rows after 500 (5), 14.9 / 13.6, are on the wrong side of this rule by 1.3 us: it does not tell heads of 256 apart.)
constexpr int kJoinMost = 32;
__host__ __device__ inline int group_of(const KvArgs& a, const Kind& k, int ns) {
  const int per = (k.cols * (a.HD / 4) + 64 * kWaves - 1) / (64 * kWaves);  // columns' channels a thread
  if (per > 1) return ns * per <= kJoinMost ? ns : 0;
  return ns <= 16 ? ns : ns <= 64 ? 8 : ns <= 256 ? 16 : 32;
}
// a sequence's pieces (with all its column blocks and KV heads), those of them that are cut, and its (row, head)s to be merged
struct Counts {
  int items, cut, rows;
  int size, ns;  // of a unit's pieces
};
__device__ __forceinline__ Counts counts_of(const KvArgs& a, const Kind& k, const Lane& l, int chunk) {
  const int size = size_of(l.sq.len, chunk), n = pieces_of(l.sq.len, size), items = l.ncb * n * a.HK;
  return Counts{items, n > 1 ? items : 0, l.ncb && !group_of(a, k, n) ? l.sq.n * a.HQ : 0, size, n};
}

// Kind::plan: a thread has neighbouring sequences.
__global__ __launch_bounds__(1024) void kv_plan_kernel(KvArgs a, Kind k) {
  __shared__ float ws[16];
  __shared__ int tot[16][3], tops[16];
  const int tid = threadIdx.x, wave = tid >> 6, per = (a.n_seqs + 1023) / 1024, s0 = tid * per, s1 = min(s0 + per, a.n_seqs);
  int* sums = k.plan + kPlanHead;
  int top = 0;  // of the thread's sequences, then of those before them
  for (int s = s0; s < s1; s++) top = max(top, a.row_start[s]);
  top = max64(top);
  if ((tid & 63) == 63) tops[wave] = top;
  top = __shfl_up(top, 1);
  if ((tid & 63) == 0) top = 0;
  __syncthreads();
  for (int x = 0; x < wave; x++) top = max(top, tops[x]);
  auto block_sum = [&](float w) {
    w = scan64(w);
    __syncthreads();
    if ((tid & 63) == 63) ws[wave] = w;
    __syncthreads();
    w = 0.0f;
    for (int x = 0; x < 16; x++) w += ws[x];
    return w;
  };
  float w = 0.0f;
  Seq first{};  // of the thread's sequences (there is one where n_seqs <= 1024)
  for (int s = s0; s < s1; s++) {
    top = max(top, a.row_start[s]);
    sums[3 * kPlanMost + s] = top;
    const Seq sq = seq_of(a, s, top);
    if (s == s0) first = sq;
    w += wide_keys(a, sq);
  }
  const int limit = k.split ? limit_of(a, block_sum(w)) : 0;
  auto lane = [&](int s) { return lane_of<kCols>(a, k, s == s0 ? first : seq_of(a, s, sums[3 * kPlanMost + s]), limit); };
  w = 0.0f;
  for (int s = s0; s < s1; s++) {
    const Lane l = lane(s);
    w += (float)l.ncb * (float)l.sq.len;
  }
  w = block_sum(w);
  const int chunk = chunk_of(a, k, w);
  Counts c{};
  for (int s = s0; s < s1; s++) {
    const Counts x = counts_of(a, k, lane(s), chunk);
    c = Counts{c.items + x.items, c.cut + x.cut, c.rows + x.rows, 0, 0};
  }
  const Counts in = {scan64(c.items), scan64(c.cut), scan64(c.rows), 0, 0};
  if ((tid & 63) == 63) {
    tot[wave][0] = in.items;
    tot[wave][1] = in.cut;
    tot[wave][2] = in.rows;
  }
  __syncthreads();
  Counts at = {in.items - c.items, in.cut - c.cut, in.rows - c.rows, 0, 0};
  for (int x = 0; x < wave; x++) at = Counts{at.items + tot[x][0], at.cut + tot[x][1], at.rows + tot[x][2], 0, 0};
  if (tid == 0) {
    k.plan[0] = chunk;
    k.plan[1] = limit;
  }
  for (int s = s0; s < s1; s++) {
    const Counts x = counts_of(a, k, lane(s), chunk);
    at = Counts{at.items + x.items, at.cut + x.cut, at.rows + x.rows, 0, 0};
    sums[s] = at.items;
    sums[kPlanMost + s] = at.cut;
    sums[2 * kPlanMost + s] = at.rows;
  }
}
// the first of n sums, in order, that is more than x, or n
__device__ __forceinline__ int search(const int* sums, int n, int x) {
  const int lane = threadIdx.x & 63;
  int lo = 0;
  for (int step = n > 4096 ? 4096 : n > 64 ? 64 : 1; step; step >>= 6) {
    const int last = lo + (lane + 1) * step - 1;  // of the lane's block
    const unsigned long long past = __ballot(gp<int>(sums)[min(last, n - 1)] > x);
    if (!past) return n;
    lo += __builtin_ctzll(past) * step;
  }
  return uniform(lo);
}

// Piece x of few columns, or false where there is none.
__device__ __forceinline__ bool find_piece(const KvArgs& a, const Kind& k, int x, Item& it) {
  const int lane = threadIdx.x & 63;
  if (k.direct) {
    it.b = x;
    it.kh = blockIdx.y;
    it.cb = it.piece = it.slot = 0;
    it.size = 0x7fffffff;
    it.sq = seq_alone(a, it.b);
    return it.sq.n > 0;
  }
  int rel, ns;  // rel: piece of the sequence; ns: pieces of a unit
  if (k.plan) {
    const int *sums = k.plan + kPlanHead, s = search(sums, a.n_seqs, x);
    if (s == a.n_seqs) return false;
    it.b = s;
    const Lane l = lane_of<kCols>(a, k, seq_of(a, s, gp<int>(sums)[3 * kPlanMost + s]), gp<int>(k.plan)[1]);
    const Counts c = counts_of(a, k, l, gp<int>(k.plan)[0]);
    it.size = uniform(c.size);
    ns = uniform(c.ns);
    rel = uniform(x - gp<int>(sums)[s] + c.items);
    it.slot = uniform(gp<int>(sums)[kPlanMost + s] - c.cut + rel);
    it.sq = l.sq;
  } else {
    int top = 0;
    const Seq first = seq_in_order(a, lane, top);
    const int limit = limit_of(a, k, first, lane, top);
    Lane l = lane_of<kCols>(a, k, first, limit);
    const int chunk = chunk_of(a, k, l, lane, top, limit);
    int base = 0, slots = 0;
    for (int s0 = 0;; s0 += 64) {
      if (s0) l = lane_of<kCols>(a, k, seq_in_order(a, s0 + lane, top), limit);
      const Counts c = counts_of(a, k, l, chunk);
      const int sum = scan64(c.items), csum = scan64(c.cut);
      const unsigned long long past = __ballot(base + sum > x);
      if (past) {
        const int at = __builtin_ctzll(past);
        rel = x - base - lane_value(sum, at) + lane_value(c.items, at);
        it.b = s0 + at;
        it.slot = slots + lane_value(csum, at) - lane_value(c.cut, at) + rel;
        it.sq = lane_value(l.sq, at);
        it.size = lane_value(c.size, at);
        ns = lane_value(c.ns, at);
        break;
      }
      base += lane_value(sum, 63);
      slots += lane_value(csum, 63);
      if (s0 + 64 >= a.n_seqs) return false;
    }
  }
  const int unit = uniform(rel / ns);
  it.cb = uniform(unit / a.HK);
  it.piece = rel - unit * ns;
  it.kh = unit - it.cb * a.HK;
  return true;
}
// Column block x of many columns, or false where there is none: those with the most keys first (each of 64 sequences, in
// kOrder steps of the longest; 3000, 1777, 2000 and 1000 rows of 4 sequences, us: 171 so, 246 by the blocks' numbers).
constexpr int kOrder = 16;
__device__ __forceinline__ bool find_block(const KvArgs& a, const Kind& k, int x, Item& it) {
  const int lane = threadIdx.x & 63;
  if (k.direct) {  // a pair's workgroups share an XCD
    const int pairs = a.n_seqs * a.HK, row = x / pairs, pair = x - row * pairs;
    it.b = pair / a.HK;
    it.kh = pair - it.b * a.HK;
    it.cb = k.ncb - 1 - row;
    it.sq = seq_alone(a, it.b);
    return it.cb * kBigCols < it.sq.n * a.ratio && (it.sq.ok || it.cb == 0);
  }
  int top = 0;
  Seq sq = seq_in_order(a, lane, top);
  const int limit = k.plan ? gp<int>(k.plan)[1] : limit_of(a, k, sq, lane, top);
  for (int s0 = 0; s0 < a.n_seqs; s0 += 64) {
    if (s0) sq = seq_in_order(a, s0 + lane, top);
    const Lane l = lane_of<kBigCols>(a, k, sq, limit);
    const int all = lane_value(scan64(l.ncb), 63) * a.HK;
    if (x >= all) {
      x -= all;
      continue;
    }
    const int before = l.sq.len - l.sq.n;
    int left = l.ncb;  // the lane's blocks that are not yet in the list
    for (int step = kOrder - 1;; step--) {
      // blocks whose first row sees more than step / kOrder of the longest context (all, at last)
      const int from = (int)((long)a.max_len * step / kOrder), low = step == 0 ? 0 : min(l.ncb, (max(from - before, 0) * a.ratio + kBigCols - 1) / kBigCols);
      const int here = max(left - low, 0), sum = scan64(here), n = lane_value(sum, 63) * a.HK;
      if (x >= n) {
        x -= n;
        left -= here;
        continue;
      }
      const int nth = uniform(x / a.HK), at = __builtin_ctzll(__ballot(sum > nth));
      it.b = s0 + at;
      it.kh = x - nth * a.HK;
      it.cb = lane_value(left, at) - 1 - (nth - lane_value(sum, at) + lane_value(here, at));
      it.sq = lane_value(l.sq, at);
      return true;
    }
  }
  return false;
}
// (row, head) x of those that kv_merge_kernel merges, or false where there is none; it.slot: of its unit's first piece.
__device__ __forceinline__ bool find_row(const KvArgs& a, const Kind& k, int x, int& h, Item& it) {
  const int lane = threadIdx.x & 63;
  int rel, ns, slot = 0;
  if (k.plan) {
    const int *sums = k.plan + kPlanHead, s = search(sums + 2 * kPlanMost, a.n_seqs, x);
    if (s == a.n_seqs) return false;
    it.b = s;
    const Lane l = lane_of<kCols>(a, k, seq_of(a, s, gp<int>(sums)[3 * kPlanMost + s]), gp<int>(k.plan)[1]);
    const Counts c = counts_of(a, k, l, gp<int>(k.plan)[0]);
    it.size = uniform(c.size);
    ns = uniform(c.ns);
    rel = uniform(x - gp<int>(sums)[2 * kPlanMost + s] + c.rows);
    slot = uniform(gp<int>(sums)[kPlanMost + s] - c.cut);
    it.sq = l.sq;
  } else {
    int top = 0;
    const Seq first = seq_in_order(a, lane, top);
    const int limit = limit_of(a, k, first, lane, top);
    Lane l = lane_of<kCols>(a, k, first, limit);
    const int chunk = chunk_of(a, k, l, lane, top, limit);
    int base = 0;
    for (int s0 = 0;; s0 += 64) {
      if (s0) l = lane_of<kCols>(a, k, seq_in_order(a, s0 + lane, top), limit);
      const Counts c = counts_of(a, k, l, chunk);
      const int sum = scan64(c.rows), csum = scan64(c.cut);
      const unsigned long long past = __ballot(base + sum > x);
      if (past) {
        const int at = __builtin_ctzll(past);
        it.b = s0 + at;
        rel = x - base - lane_value(sum, at) + lane_value(c.rows, at);
        slot += lane_value(csum, at) - lane_value(c.cut, at);
        it.sq = lane_value(l.sq, at);
        it.size = lane_value(c.size, at);
        ns = lane_value(c.ns, at);
        break;
      }
      base += lane_value(sum, 63);
      slot += lane_value(csum, 63);
      if (s0 + 64 >= a.n_seqs) return false;
    }
  }
  it.row = uniform(rel / a.HQ);
  h = rel - it.row * a.HQ;
  it.kh = a.by_ratio(h);
  it.cb = (it.row * a.ratio + h - it.kh * a.ratio) / kCols;
  it.slot = slot + (it.cb * a.HK + it.kh) * ns;
  return true;
}
// byte offset of a piece's column among the results: O [HD], maximum, sum, padding
template <int HD>
__device__ __forceinline__ unsigned column_at(const Kind& k, int slot, int c) { return (unsigned)(slot * k.cols + c) * (HD + 4) * 4; }
constexpr int kCacheSc1 = 16;  // cache-policy operand of buffer instructions: device-coherent (sc1)
typedef int i4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void put4(__amdgpu_buffer_rsrc_t rs, unsigned at, f4 v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(i4, v), rs, at, 0, kCacheSc1);
}
__device__ __forceinline__ f4 get4(__amdgpu_buffer_rsrc_t rs, unsigned at) {
  return __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(rs, at, 0, kCacheSc1));
}
// The rows of a sequence that does not fit its batch.
template <int HD>
__device__ __forceinline__ void nan_rows(const KvArgs& a, const Seq& sq, int kh, int threads) {
  const _Float16 x = (_Float16)__builtin_nanf("");
  for (int r = threadIdx.x / (HD / 4); r < sq.n * a.ratio; r += threads / (HD / 4)) {
    const int i = a.by_ratio(r);
    *gpw<h4>(a.out + ((size_t)(sq.r0 + i) * a.HQ + kh * a.ratio + r - i * a.ratio) * HD + 4 * (threadIdx.x % (HD / 4))) = h4{x, x, x, x};
  }
}
// Channels ch .. + 3 of column r: the gate, and with it O / l as f16.
__device__ __forceinline__ f4 gate_of(const KvArgs& a, const Seq& sq, int kh, int r, int ch) {
  const int i = a.by_ratio(r);
  return a.gated ? gate4(a, sq.r0 + i, kh * a.ratio + r - i * a.ratio, ch) : f4{};
}
template <int HD>
__device__ __forceinline__ void finish(const KvArgs& a, const Seq& sq, int kh, int r, int ch, f4 v, float inv, const f4& gt) {
  const int i = a.by_ratio(r), t = sq.r0 + i, h = kh * a.ratio + r - i * a.ratio;
  v *= inv;
  if (a.gated) {
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] *= sigmoid(gt[e]);
  }
  *gpw<h4>(a.out + ((size_t)t * a.HQ + h) * HD + ch) = to_h4(v);
}

template <int HD>
__global__ __launch_bounds__(64 * kWaves, 2) void kv_few_kernel(KvArgs a, Kind kind) {
  constexpr int G = HD / 4, kH = HD / 128, kE = HD / 64, kRow = HD / 2;
  constexpr int kPitch = HD + 4;
  __shared__ __attribute__((aligned(16))) float ol[kWaves * (kCols / 2) * kPitch];
  __shared__ float ml[kWaves][kCols][2];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, j = lane & 15, kg = lane >> 4;
  const int ratio = a.ratio;
  Item it;
  if (!find_piece(a, kind, blockIdx.x, it)) return;
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(kind.p, 0, (int)(kSlots * kSlotBytes), 0x00020000);
  const Seq sq = it.sq;
  const int kh = it.kh, b = it.b, k0 = it.piece * it.size, c0 = it.cb * kCols, cols = min(kCols, sq.n * ratio - c0);
  if (!sq.ok) {
    if (it.piece == 0) nan_rows<HD>(a, sq, kh, 64 * kWaves);
    return;
  }
  const int* table = a.table + (size_t)b * a.table_stride;
  const int page_log2 = a.page_log2, top_page = a.table_stride - 1;
  int ids = gp<int>(table)[min((k0 + 16 * lane) >> page_log2, top_page)];  // lane k: the page of tokens seg + 16 k .. + 15
  const int before = sq.len - sq.n;
  const int keys = before + a.by_ratio(c0 + cols - 1) + 1;
  if (k0 >= keys) return;
  const int k1 = min(k0 + it.size, keys);
  const int all = before + a.by_ratio(c0) + 1;  // keys below this are seen by every column
  const int r = c0 + min(j, cols - 1), ri = a.by_ratio(r), last = before + ri;  // columns behind the last one repeat it
  h8 q[kH][4];
  {
    const _Float16* qp = a.q + ((size_t)(sq.r0 + ri) * a.HQ + kh * ratio + r - ri * ratio) * HD + 8 * kg;
#pragma unroll
    for (int h = 0; h < kH; h++)
#pragma unroll
      for (int g = 0; g < 4; g++) q[h][g] = *gp<h8>(qp + G * g + 32 * h);
  }
  // A step's 32 keys are two tiles of 16, each in one page. Its codes wait in registers: K's of the next step are fetched when
  // the scores are done, V's when the outputs are. The parameters (16 bytes a lane: tile and K or V, key quad, group) go through
  // the wave's part of LDS, where each lane finds those of its keys.
  const size_t blk_bytes = kv_block_bytes(a.page, HD);
  const unsigned par_off = (unsigned)a.page * kRow;
  u4 kc[2][kH], pr;
  u2 vc[2][4];
  bool gone[2];
  const unsigned char* blk[2];
  int slot[2];
  auto locate = [&](int seg, int t0) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      int page = __builtin_amdgcn_readlane(ids, ((t0 - seg) / 16 + i) & 63);
      if (t0 + 16 * i >= k1) page = 0;  // (behind the last key: any page)
      gone[i] = (unsigned)page >= (unsigned)a.n_pages;
      blk[i] = a.pool + ((size_t)(gone[i] ? 0 : page) * a.HK + kh) * 2 * blk_bytes;
      slot[i] = (t0 + 16 * i) & (a.page - 1);
    }
  };
  auto fetch_k = [&]() {
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int h = 0; h < kH; h++) kc[i][h] = *gp<u4>(blk[i] + (unsigned)((slot[i] + j) * kRow + 64 * h + 16 * kg));
    const bool second = lane & 16;
    pr = *gp<u4>((second ? blk[1] : blk[0]) + (lane & 32 ? blk_bytes : 0) + par_off + (unsigned)((second ? slot[1] : slot[0]) * kKvParamBytes + 16 * (lane & 15)));
  };
  auto fetch_v = [&]() {
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int k = 0; k < 4; k++)
        vc[i][k] = *gp<u2>(blk[i] + blk_bytes + (unsigned)((slot[i] + 4 * kg + k) * kRow + 8 * (HD == 256 ? j : j & 7)));
  };
  unsigned char* params = reinterpret_cast<unsigned char*>(ol + wave * (kCols / 2) * kPitch);
  Range range(0);
  auto put_params = [&](int t0) {
    const bool lost = lane & 16 ? gone[1] : gone[0];
    // beyond the sequence, and in no page: parameters of any bits (a score of no page is NaN)
    if (lost) pr = lane & 32 ? u4{} : u4{0x7E007E00u, 0x7E007E00u, 0u, 0u};
    if (t0 + kStep > keys) {
      const int t = t0 + (lane & 16) + (lane & 12);
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (t + e >= keys) {
          pr[e >> 1] &= e & 1 ? 0x0000FFFFu : 0xFFFF0000u;
          pr[2 + (e >> 1)] &= e & 1 ? 0x0000FFFFu : 0xFFFF0000u;
        }
    }
    *reinterpret_cast<u4*>(params + 16 * lane) = pr;
    const int cls = lane & 32 ? scale_class(pr[0], pr[1]) : 0;
    range = Range(!__any(cls) ? 0 : !__any(cls == 2) ? 1 : 2);
    wave_sync();
  };
  locate(k0, k0 + kStep * wave);  // (a wave without keys: any page)
  fetch_k();
  fetch_v();
  const Magic mg;
  float qs[4], qc[4];  // over each group: sum of the column's q, and what the codes' offsets add to its products
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
  const unsigned least = j & 4 ? 0u : 0xFC00FC00u;  // NaN scales are 0 in zs, where columns share them (O has them where they are seen)
  f4 o[4][kE], zs = {};  // zs[g]: sum P z_g where kg is even, sum P s_g where it is odd (A's row 4 i + g has group g's zeros or scales)
  float m = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int g = 0; g < 4; g++)
#pragma unroll
    for (int e = 0; e < kE; e++) o[g][e] = f4{};

  // The keys t0 .. t0 + 31. `more`: the wave's next step is one of the segment's (a template argument: with a branch the compiler
  // would not know how many loads are in flight, and wait for all of them).
  auto step = [&](int seg, int t0, auto more_c) {
    constexpr bool more = decltype(more_c)::value;
    put_params(t0);
    const u4* par = reinterpret_cast<const u4*>(params) + 4 * kg;  // [tile and K or V: 16][group]
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
        const h8 p = __builtin_bit_cast(h8, par[16 * i + g]);
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const float z = g ? fmaf((float)p[4 + k], qs[g], sc[i][k]) : (float)p[4 + k] * qs[g];
          sc[i][k] = fmaf((float)p[k], acc[k], z);
        }
      }
    if constexpr (more) {
      locate(seg, t0 + kStep * kWaves);
      fetch_k();
    }
    const bool edge = t0 + kStep > all;
    if (edge) {
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (t0 + 16 * i + 4 * kg + k > last) sc[i][k] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int k = 0; k < 4; k++) mx = fmaxf(mx, sc[i][k]);
    mx = max_quads(mx) * scale;
    const float mn = mx > m + range.room ? mx - range.lift : m;
    if (__any(mn != m)) {
      if (__any(m != -INFINITY)) {  // (else O is zero)
        const float al = mn == m ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
        sum *= al;
        zs *= al;
#pragma unroll
        for (int g = 0; g < 4; g++) {
#pragma unroll
          for (int e = 0; e < kE; e++) o[g][e] *= al;
        }
      }
      m = mn;
    }
    const float base = m == -INFINITY ? 0.0f : m;
    u4 p, p2;  // P of tokens (t0 + 4 kg + 0, 1), (2, 3), then those of the second tile
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int k = 0; k < 4; k += 2) {
        float &p0 = sc[i][k], &p1 = sc[i][k + 1];
        p0 = __builtin_amdgcn_exp2f(fmaf(p0, scale, -base));
        p1 = __builtin_amdgcn_exp2f(fmaf(p1, scale, -base));
        sum += p0 + p1;
        const u2 x = split2(p0, p1);
        p[2 * i + k / 2] = x[0];
        p2[2 * i + k / 2] = x[1];
      }
    {
      u2 z[2];
#pragma unroll
      for (int i = 0; i < 2; i++) {
        z[i] = max2(reinterpret_cast<const u2*>(par + 32 + 16 * i + (j & 3))[j & 4 ? 0 : 1], least);
      }
      const h8 zh = __builtin_bit_cast(h8, u4{z[0][0], z[0][1], z[1][0], z[1][1]});
      zs = __builtin_amdgcn_mfma_f32_16x16x32_f16(zh, __builtin_bit_cast(h8, p), zs, 0, 0, 0);
      zs = __builtin_amdgcn_mfma_f32_16x16x32_f16(zh, __builtin_bit_cast(h8, p2), zs, 0, 0, 0);
    }
#pragma unroll
    for (int g = 0; g < 4; g++) {
      u2 vs[2] = {*reinterpret_cast<const u2*>(par + 32 + g), *reinterpret_cast<const u2*>(par + 48 + g)};
      if (edge) {
#pragma unroll
        for (int k = 0; k < 4; k++) {  // a masked token's scale may be NaN
          const int tok = t0 + 16 * (k >> 1) + 4 * kg + 2 * (k & 1);
          vs[k >> 1][k & 1] &= tok + 1 <= last ? 0xFFFFFFFFu : tok <= last ? 0xFFFFu : 0u;
        }
      }
      u4 w, w2;  // P s_g
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const u2 x = scale2(p[k], p2[k], vs[k >> 1][k & 1]);
        w[k] = x[0];
        w2[k] = x[1];
      }
      const h8 wh = __builtin_bit_cast(h8, w), wh2 = __builtin_bit_cast(h8, w2);
      unsigned x[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        x[k] = halves(vc[k >> 1][2 * (k & 1)][g >> 1], vc[k >> 1][2 * (k & 1) + 1][g >> 1], g & 1);
        if constexpr (HD == 128) x[k] >>= 8 * (j >> 3);
      }
      h8 op[kE];
#pragma unroll
      for (int e = 0; e < kE; e++)
        op[e] = __builtin_bit_cast(h8, u4{code_v(mg, x[0], e), code_v(mg, x[1], e), code_v(mg, x[2], e), code_v(mg, x[3], e)});
      // (not one sum's two products in succession: the second waits for the first)
#pragma unroll
      for (int e = 0; e < kE; e++) o[g][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(op[e], wh, o[g][e], 0, 0, 0);
#pragma unroll
      for (int e = 0; e < kE; e++) o[g][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(op[e], wh2, o[g][e], 0, 0, 0);
    }
    if constexpr (more) fetch_v();
    wave_sync();  // (the parameters' place is used again)
  };
  for (int seg = k0;;) {  // segments of 1024 keys, whose pages the lanes hold
    const int end = min(seg + 1024, k1);
    if (seg > k0) {
      // The offsets of the segment before: sums of 16 + c that ran on would lose what remains of c - 8 (131072 values of equal weight
      // whose mean is zero came out as up to 5.2e-5; now below 2.7e-7).
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const float t = sum_quads(kg & 1 ? -12.0f * zs[g] : 0.0f);  // (two of the four lanes have it)
        if (kg & 1) zs[g] = 0.0f;
#pragma unroll
        for (int e = 0; e < kE; e++) o[g][e] += t;
      }
    }
    int t0 = seg + kStep * wave;
#pragma clang loop unroll(disable)
    for (; t0 + kStep * kWaves < end; t0 += kStep * kWaves) step(seg, t0, std::true_type{});
    if (t0 < end) step(seg, t0, std::false_type{});
    seg += 1024;
    if (seg >= k1) break;
    ids = gp<int>(table)[min((seg + 16 * lane) >> page_log2, top_page)];
    locate(seg, seg + kStep * wave);
    fetch_k();
    fetch_v();
  }
  // the four waves' sums: O^T row 4 kg + k of (g, e) is channel G g + 16 kg + 4 k + e (HD 256), G g + 4 (row & 7) + 2 (row >> 3) + e
  // (HD 128)
  sum = sum_quads(sum);
#pragma unroll
  for (int g = 0; g < 4; g++) zs[g] = sum_quads((kg & 1 ? -12.0f : 0.5f) * zs[g]);
  if (kg == 0) {
    ml[wave][j][0] = m;
    ml[wave][j][1] = sum;
  }
  for (int h0 = 0; h0 < cols; h0 += kCols / 2) {  // half of the columns at a time (LDS)
    if (h0) __syncthreads();
    constexpr int kEach = (kCols / 2) * (HD / 4) / (64 * kWaves);
    const int left = min(kCols / 2, cols - h0) * (HD / 4);
    f4 gt[kEach];
    if (keys <= it.size) {  // (loaded before the others are waited for)
#pragma unroll
      for (int n = 0; n < kEach; n++) {
        const int k = min(tid + n * 64 * kWaves, left - 1);
        gt[n] = gate_of(a, sq, kh, c0 + h0 + k / (HD / 4), 4 * (k % (HD / 4)));
      }
    }
    if (j >= h0 && j < min(h0 + kCols / 2, cols)) {
      float* d = ol + (wave * (kCols / 2) + j - h0) * kPitch;
#pragma unroll
      for (int g = 0; g < 4; g++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
          if constexpr (HD == 256) {
            *reinterpret_cast<f4*>(d + G * g + 16 * kg + 4 * k) = f4{o[g][0][k], o[g][1][k], o[g][2][k], o[g][3][k]} + zs[g];
          } else {
            const int ii = 4 * kg + k;
            *reinterpret_cast<float2*>(d + G * g + 4 * (ii & 7) + 2 * (ii >> 3)) = float2{o[g][0][k] + zs[g], o[g][1][k] + zs[g]};
          }
        }
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < kEach; n++) {
      const int k = tid + n * 64 * kWaves;
      if (k >= left) break;
      const int c = h0 + k / (HD / 4), ch = 4 * (k % (HD / 4));
      float mm = -INFINITY, l = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; w++) mm = fmaxf(mm, ml[w][c][0]);
      f4 v = {};
#pragma unroll
      for (int w = 0; w < kWaves; w++) {
        const float f = ml[w][c][0] == mm ? 1.0f : __builtin_amdgcn_exp2f(ml[w][c][0] - mm);
        l += f * ml[w][c][1];
        v += f * *reinterpret_cast<const f4*>(ol + (w * (kCols / 2) + c - h0) * kPitch + ch);
      }
      if (keys > it.size) {
        const unsigned at = column_at<HD>(kind, it.slot, c);
        put4(rs, at + 4 * ch, v);
        if (ch == 0) put4(rs, at + 4 * HD, f4{mm, l, 0.0f, 0.0f});
      } else {
        finish<HD>(a, sq, kh, c0 + c, ch, v, 1.0f / l, gt[n]);
      }
    }
  }
  const int ns = pieces_of(keys, it.size), group = group_of(a, kind, ns);
  if (ns <= 1 || !group) return;

  // The last of a group's pieces to get here joins them, and the last of the groups those. What they write goes past the XCDs' caches
  // (sc1), and is counted when it is there; the last one clears the count for the next call. Nobody waits.
  const int first = it.slot - it.piece;
  __shared__ int is_last;
  auto last_of = [&](int* count, int n) {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) {
      const bool x = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n - 1;
      if (x) __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      is_last = x;
    }
    __syncthreads();
    return is_last != 0;
  };
  // channels ch .. + 3 of column c over the results s0, s0 + stride, ... (n of them): O, maximum, sum
  auto join = [&](int s0, int stride, int n, int c, int ch, float& mm, float& l) {
    f4 v = {};
    mm = -INFINITY;
    l = 0.0f;
    constexpr int kAt = 8;  // loaded at once
    for (int x0 = 0; x0 < n; x0 += kAt) {
      f4 w[kAt], x[kAt];
#pragma unroll
      for (int e = 0; e < kAt; e++) {
        const unsigned at = column_at<HD>(kind, s0 + min(x0 + e, n - 1) * stride, c);
        w[e] = get4(rs, at + 4 * HD);
        x[e] = get4(rs, at + 4 * ch);
      }
      float mx = mm;
#pragma unroll
      for (int e = 0; e < kAt; e++) mx = fmaxf(mx, w[e][0]);
      const float al = mm == mx ? 1.0f : __builtin_amdgcn_exp2f(mm - mx);
      mm = mx;
      l *= al;
      v *= al;
#pragma unroll
      for (int e = 0; e < kAt; e++) {
        const float f = x0 + e >= n ? 0.0f : w[e][0] == mm ? 1.0f : __builtin_amdgcn_exp2f(w[e][0] - mm);
        l += f * w[e][1];
        v += f * x[e];
      }
    }
    return v;
  };
  int s0 = first, stride = 1, n = ns;
  if (group < ns) {
    s0 = first + it.piece / group * group;
    n = min(group, first + ns - s0);
    if (!last_of(kind.count + s0, n)) return;
    for (int k0 = 0; k0 < cols * (HD / 4); k0 += 64 * kWaves) {
      const int k = k0 + tid, c = min(k / (HD / 4), cols - 1), ch = 4 * (k % (HD / 4));
      float mm, l;
      const f4 v = join(s0, 1, n, c, ch, mm, l);
      __syncthreads();  // (the sum is written over one of those that were read)
      if (k < cols * (HD / 4)) {
        const unsigned at = column_at<HD>(kind, s0, c);
        put4(rs, at + 4 * ch, v);
        if (ch == 0) put4(rs, at + 4 * HD, f4{mm, l, 0.0f, 0.0f});
      }
    }
    s0 = first;
    stride = group;
    n = (ns + group - 1) / group;
  }
  if (!last_of(kind.count + (group < ns ? (int)kSlots : 0) + first, n)) return;
  for (int k = tid; k < cols * (HD / 4); k += 64 * kWaves) {
    const int c = k / (HD / 4), ch = 4 * (k % (HD / 4));
    const f4 gt = gate_of(a, sq, kh, c0 + c, ch);
    float mm, l;
    const f4 v = join(s0, stride, n, c, ch, mm, l);
    finish<HD>(a, sq, kh, c0 + c, ch, v, 1.0f / l, gt);
  }
}

// ---- many columns ----

typedef float f16v __attribute__((ext_vector_type(16)));

// LDS of kv_many_kernel, each part twice: K tile [32][HD] and V^T tile [HD][32] as f16 (rows 16 bytes longer, so that eight rows
// of an operand lie in different banks), K's scales [4][32] and zeros [32][4] twice each, P as two f16 in the lanes' order, the columns'
// factors, the waves' flags and the class of V's scales; V's scales and zeros [4][32] each of four tiles.
template <int HD>
struct ManyLds {
  static constexpr int kKPitch = HD * 2 + 16, kVPitch = kTile * 2 + 16;
  static constexpr int kKs = kTile * kKPitch, kKz = kKs + 256, kV = kKz + 512, kP = kV + HD * kVPitch;
  static constexpr int kAl = kP + kBigCols * kTile * 4, kFlag = kAl + kBigCols * 4, kClass = kFlag + 16, kBuf = kClass + 16;
  static constexpr int kParam = 2 * kBuf, kAll = kParam + 4 * 512;
};

// A workgroup has 128 columns and walks the keys in tiles of 32. Four of its eight waves compute P (32 columns each: S^T = K Q^T on
// v_mfma_f32_32x32x16_f16, scales and zeros, online softmax) and unpack the next tile's keys into LDS, the other four the outputs
// of the tile before (64 columns and half the channels each: O^T = V^T P^T) and this tile's values; each SIMD has one of either
// kind, so the matrix products of the one run beside the vector instructions of the other. One barrier a tile, which takes about
// 3700 cycles (HD 256): matrix products 1060 of them a SIMD, vector instructions about 2150, LDS about 2000 (250 KB read and
// written), each waiting for the others at times; with 64 columns a wave that compute P, or the values unpacked by both kinds,
// it took longer (spills; 311 us where this took 296 for 2048 rows of 8 sequences). Scales and zeros
// stay apart from the codes, so that both operands are exact: S = sum_g s_g (q . (c - 8))_g + sum_g z_g sum(q_g), the last
// as one more product (with sum(q_g) / G as two f16), and O takes P s_g and sum P z_g. P goes through LDS as two f16 each; P s_g is
// rounded to f16 once here (2.75e-4 of the output's norm, 2.07e-4 of it the output's own rounding; the framework's attention on f16
// rows rounds its P as well): two f16 each, as above, would be 16 more matrix instructions and as many vector ones a tile in the
// waves that bound it, 346 us instead of 284.
template <int HD>
__global__ __launch_bounds__(512, 2) void kv_many_kernel(KvArgs a, Kind kind) {
  constexpr int G = HD / 4, U = HD / 16, kRow = HD / 2, kKs = G / 16, kDt = HD / 64;  // kKs: k-steps of a group; kDt: 32-row blocks of V^T a wave
  typedef ManyLds<HD> M;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, c32 = lane & 31, half = lane >> 5;
  const int ratio = a.ratio;
  Item it;
  if (!find_block(a, kind, blockIdx.x, it)) return;
  const Seq sq = it.sq;
  const int kh = it.kh, b = it.b, c0 = it.cb * kBigCols, cols = min(kBigCols, sq.n * ratio - c0);
  if (!sq.ok) {
    nan_rows<HD>(a, sq, kh, 512);
    return;
  }
  const int before = sq.len - sq.n, keys = before + a.by_ratio(c0 + cols - 1) + 1;
  const int tiles = (keys + kTile - 1) / kTile;
  const int all = before + a.by_ratio(c0) + 1;  // keys below this are seen by every column
  const float scale = a.scale * kLog2e;
  float* stats = reinterpret_cast<float*>(lds);  // after the last tile: the columns' sums

  // the codes: a wave of either kind takes its quarter of a tile's keys (values)
  const int u = tid & 255;
  const size_t blk_bytes = kv_block_bytes(a.page, HD);
  const int* table = a.table + (size_t)b * a.table_stride;
  const unsigned par_off = (unsigned)a.page * kRow;
  const int page_log2 = a.page_log2, top_page = a.table_stride - 1;
  int ids = 0;  // lane k: the page of tokens 1024 seg + 16 k .. + 15, seg that of the tile fetched last
  // the block (K: 0, V: 1) of the half of the tile at t0 that `second` says, and whether its page is none; a half behind the last
  // key lies in any page
  auto block_at = [&](int t0, bool second, int which, bool& gone) {
    const int n = (t0 & 1023) / 16;
    int p0 = __builtin_amdgcn_readlane(ids, n), p1 = __builtin_amdgcn_readlane(ids, n + 1);
    p0 = t0 < keys ? p0 : 0;
    p1 = t0 + 16 < keys ? p1 : 0;
    const int p = second ? p1 : p0;
    gone = (unsigned)p >= (unsigned)a.n_pages;
    return a.pool + ((size_t)(gone ? 0 : p) * a.HK + kh) * 2 * blk_bytes + which * blk_bytes;
  };
  auto load_ids = [&](int t0) {
    if ((t0 & 1023) == 0) ids = gp<int>(table)[min((t0 + 16 * lane) >> page_log2, top_page)];
  };
  const Magic mg;

  if (wave < 4) {
    // ---- P of columns 32 wave .. + 31 ----
    const int kkey = HD == 256 ? u >> 3 : (u >> 2) & 31, kpos = HD == 256 ? u & 7 : u & 3;
    const bool unpacks = HD == 256 || u < 128;
    // two keys' parameters of K or of V: word pdw of key quad pquad: (g, s or z, key pair)
    const int pwhich = u >> 7, pquad = (u >> 4) & 7, pdw = u & 15, pg = pdw >> 2, ppart = (pdw >> 1) & 1, pkey = 4 * pquad + 2 * (pdw & 1);
    u4 raw = {};
    unsigned praw = 0;
    bool pgone = false;
    auto fetch = [&](int t0) {
      load_ids(t0);
      bool gone;
      const unsigned char* p = block_at(t0, kkey >= 16, 0, gone);
      if (unpacks) raw = *gp<u4>(p + (unsigned)(((t0 + kkey) & (a.page - 1)) * kRow + 16 * kpos));
      p = block_at(t0, pquad >= 4, pwhich, pgone) + par_off;
      praw = *gp<unsigned>(p + (unsigned)(((t0 + 4 * pquad) & (a.page - 1)) * kKvParamBytes + 4 * pdw));
    };
    auto unpack = [&](int t0, unsigned char* buf) {
      if (unpacks) {
#pragma unroll
        for (int g = 0; g < 4; g++)
          *reinterpret_cast<u4*>(buf + kkey * M::kKPitch + 16 * ((G / 8) * g + kpos)) = codes_k(mg, halves(raw[g >> 1], raw[(g >> 1) + 2], g & 1));
      }
      // behind the sequence, and in no page: parameters of any bits (a score of no page is NaN)
      unsigned w = pgone ? (pwhich || ppart ? 0u : 0x7E007E00u) : praw;
      if (t0 + pkey >= keys) w = 0;
      else if (t0 + pkey + 1 >= keys) w &= 0xFFFFu;
      const int cls = ppart ? 0 : scale_class(w, w);
      const int most = !__any(cls) ? 0 : !__any(cls == 2) ? 1 : 2;
      if (wave >= 2 && lane == 0) *reinterpret_cast<int*>(buf + M::kClass + 4 * (wave - 2)) = most;  // (waves 2, 3: V's)
      if (pwhich) {
        *reinterpret_cast<unsigned*>(lds + M::kParam + ((t0 / kTile) & 3) * 512 + ppart * 256 + pg * 64 + pkey * 2) = w;
      } else {
        if (ppart) {
          *reinterpret_cast<unsigned*>(buf + M::kKz + pkey * 16 + 4 * pg) = (w & 0xFFFFu) * 0x10001u;
          *reinterpret_cast<unsigned*>(buf + M::kKz + pkey * 16 + 16 + 4 * pg) = (w >> 16) * 0x10001u;
        } else {
          *reinterpret_cast<unsigned*>(buf + M::kKs + pg * 64 + pkey * 2) = w;
        }
      }
    };
    const int w0 = 32 * wave, r = c0 + min(w0 + c32, cols - 1), ri = a.by_ratio(r), last = before + ri;
    const bool idle = w0 >= cols;
    fetch(0);
    // the B operand of k-step ks of group g is channels G g + 16 ks + 8 half .. + 7, in the order of K's chunks
    h8 q[4][kKs], qz;
    f16v qc[4];  // what the codes' offsets add to a column's products, in every row
    {
      const _Float16* qp = a.q + ((size_t)(sq.r0 + ri) * a.HQ + kh * ratio + r - ri * ratio) * HD + 8 * half;
#pragma unroll
      for (int g = 0; g < 4; g++)
#pragma unroll
        for (int ks = 0; ks < kKs; ks++) q[g][ks] = *gp<h8>(qp + G * g + 16 * ks);
#pragma unroll
      for (int g = 0; g < 4; g++) {
        float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
        for (int ks = 0; ks < kKs; ks++) {
          const h8 x = q[g][ks];
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            s0 += (float)x[e];
            s1 += (float)x[e + 1];
          }
          q[g][ks] = h8{x[0], x[4], x[1], x[5], x[2], x[6], x[3], x[7]};
        }
        s0 = sum_halves(s0);
        s1 = sum_halves(s1);
        qc[g] = f16v{} + (-1032.0f * s0 - 72.0f * s1);
        const float s = (s0 + s1) * (1.0f / G);
        const _Float16 hi = (_Float16)s;
        qz[2 * g] = half ? (_Float16)0.0f : hi;
        qz[2 * g + 1] = half ? (_Float16)0.0f : (_Float16)(s - (float)hi);
      }
    }
    unpack(0, lds);
    if (tiles > 1) fetch(kTile);
    float m = -INFINITY, sum = 0.0f;
    // S^T row i holds key pi(i) (bits 2 and 3 of i swapped): the lane's values 8 kb .. 8 kb + 7 are then keys 16 kb + 8 half .. + 7,
    // which is P^T's operand of k-step kb
    const int pr = (c32 & 19) | ((c32 & 4) << 1) | ((c32 & 8) >> 1);
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i <= tiles; i++) {
      const int t0 = kTile * i;
      unsigned char* buf = lds + (i & 1) * M::kBuf;
      if (i < tiles && !idle) {
        const unsigned char* kr = buf + pr * M::kKPitch + 16 * half;
        f16v st = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const h8*>(buf + M::kKz + pr * 16), qz, f16v{}, 0, 0, 0);
#pragma unroll
        for (int v = 0; v < 16; v++) st[v] *= (float)G;
#pragma unroll
        for (int g = 0; g < 4; g++) {
          f16v acc = qc[g];
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
        if (t0 + kTile > all) {
          const int tok = t0 + 8 * half;
#pragma unroll
          for (int v = 0; v < 16; v++) st[v] = tok + 16 * (v >> 3) + (v & 7) <= last ? st[v] : -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int v = 0; v < 16; v++) mx = fmaxf(mx, st[v]);
        mx = max_halves(mx) * scale;
        const int* cls = reinterpret_cast<const int*>(buf + M::kClass);
        const Range range(max(cls[0], cls[1]));
        const float mn = mx > m + range.room ? mx - range.lift : m;
        const bool raise = __any(mn != m);
        if (lane == 0) *reinterpret_cast<int*>(buf + M::kFlag + 4 * wave) = raise;
        if (raise) {
          const float al = mn == m ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
          sum *= al;
          m = mn;
          if (half == 0) *reinterpret_cast<float*>(buf + M::kAl + 4 * (w0 + c32)) = al;
        }
        const float base = m == -INFINITY ? 0.0f : m;
        u4* pl = reinterpret_cast<u4*>(buf + M::kP) + wave * 256 + lane;
#pragma unroll
        for (int k = 0; k < 4; k++) {
          f4 p;
#pragma unroll
          for (int e = 0; e < 4; e++) {
            p[e] = __builtin_amdgcn_exp2f(fmaf(st[4 * k + e], scale, -base));
            sum += p[e];
          }
          const u2 x = split2(p[0], p[1]), y = split2(p[2], p[3]);
          pl[64 * k] = u4{x[0], y[0], x[1], y[1]};
        }
      }
      if (i + 1 < tiles) {
        unpack(t0 + kTile, lds + ((i + 1) & 1) * M::kBuf);
        if (i + 2 < tiles) fetch(t0 + 2 * kTile);
      }
      __syncthreads();
    }
    sum = sum_halves(sum);
    if (half == 0) stats[w0 + c32] = sum;
    __syncthreads();
    return;
  }

  // ---- outputs of columns 64 cp .. + 63 and groups 2 dh, 2 dh + 1 ----
  const int cp = wave & 1, dh = (wave >> 1) & 1;
  const bool idle = 64 * cp >= cols;
  const int vquad = HD == 256 ? u >> 5 : (u >> 4) & 7, vpos = HD == 256 ? u & 31 : u & 15;  // 4 bytes of four keys' values
  const bool unpacks = HD == 256 || u < 128;
  u4 raw = {};
  auto fetch = [&](int t0) {
    load_ids(t0);
    bool gone;
    const unsigned char* p = block_at(t0, vquad >= 4, 1, gone) + (unsigned)(((t0 + 4 * vquad) & (a.page - 1)) * kRow + 4 * vpos);
    if (unpacks) {
#pragma unroll
      for (int k = 0; k < 4; k++) raw[k] = *gp<unsigned>(p + k * kRow);
    }
  };
  const h2 m24 = {(_Float16)-24.0f, (_Float16)-24.0f};
  auto unpack = [&](unsigned char* buf) {
    if (unpacks) {
#pragma unroll
      for (int gg = 0; gg < 2; gg++) {
        const unsigned x0 = halves(raw[0], raw[1], gg), x1 = halves(raw[2], raw[3], gg);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const u2 w = {as_u(as_h2(code_v(mg, x0, e)) + m24), as_u(as_h2(code_v(mg, x1, e)) + m24)};
          const int R = 4 * U * (2 * (vpos & 1) + gg) + U * e + (vpos >> 1);
          *reinterpret_cast<u2*>(buf + M::kV + R * M::kVPitch + 8 * vquad) = w;
        }
      }
    }
  };
  f16v o[2][kDt];
  float zs[2][2] = {};  // the lane's part of sum P z_g
  int last[2];
#pragma unroll
  for (int n = 0; n < 2; n++) {
    last[n] = before + a.by_ratio(c0 + min(64 * cp + 32 * n + c32, cols - 1));
#pragma unroll
    for (int d = 0; d < kDt; d++) o[n][d] = f16v{};
  }
  fetch(0);
  __syncthreads();
  // step i: the values of tile i are unpacked (while the other waves compute its P), the outputs take tile i - 1
#pragma unroll 1
  for (int i = 0; i <= tiles; i++) {
    const bool takes = i > 0 && !idle;
    const int t0 = kTile * (i - 1);
    const unsigned char* buf = lds + ((i & 1) ^ 1) * M::kBuf;
    // what the outputs need first is on its way while the codes are unpacked
    u4 p[2][4], ps[2][2], pz[2][2];  // p: of two pairs of keys, and what their f16 leave
    bool f0 = false, f1 = false;
    const unsigned char* par = lds + M::kParam + ((i - 1) & 3) * 512 + 16 * half;
    if (takes) {
      const int* flag = reinterpret_cast<const int*>(buf + M::kFlag) + 2 * cp;
      f0 = flag[0];
      f1 = flag[1] && 64 * cp + 32 < cols;
      const u4* pl = reinterpret_cast<const u4*>(buf + M::kP) + 2 * cp * 256 + lane;
#pragma unroll
      for (int k = 0; k < 4; k++)
#pragma unroll
        for (int n = 0; n < 2; n++) p[n][k] = pl[256 * n + 64 * k];
#pragma unroll
      for (int kb = 0; kb < 2; kb++)
#pragma unroll
        for (int gg = 0; gg < 2; gg++) {
          ps[kb][gg] = *reinterpret_cast<const u4*>(par + (2 * dh + gg) * 64 + 32 * kb);
          pz[kb][gg] = *reinterpret_cast<const u4*>(par + 256 + (2 * dh + gg) * 64 + 32 * kb);
        }
    }
    if (i < tiles) {
      unpack(lds + (i & 1) * M::kBuf);
      if (i + 1 < tiles) fetch(kTile * (i + 1));
    }
    if (takes) {
      if (f0 || f1) {
#pragma unroll
        for (int n = 0; n < 2; n++) {
          const float al = (n ? f1 : f0) ? *reinterpret_cast<const float*>(buf + M::kAl + 4 * (64 * cp + 32 * n + c32)) : 1.0f;
          zs[n][0] *= al;
          zs[n][1] *= al;
#pragma unroll
          for (int d = 0; d < kDt; d++) o[n][d] *= al;
        }
      }
      const bool edge = t0 + kTile > all;
      const unsigned char* vr = buf + M::kV + (2 * dh * G + c32) * M::kVPitch + 16 * half;
#pragma unroll
      for (int kb = 0; kb < 2; kb++) {
#pragma unroll
        for (int gg = 0; gg < 2; gg++) {
          h8 wh[2];
#pragma unroll
          for (int n = 0; n < 2; n++) {
            u4 w;
#pragma unroll
            for (int k = 0; k < 4; k++) {
              const u4& pk = p[n][2 * kb + (k >> 1)];
              const h2 hi = as_h2(pk[k & 1]), lo = as_h2(pk[2 + (k & 1)]), z = as_h2(pz[kb][gg][k]), s = as_h2(ps[kb][gg][k]);
              zs[n][gg] = __builtin_amdgcn_fdot2(lo, z, __builtin_amdgcn_fdot2(hi, z, zs[n][gg], false), false);
              w[k] = as_u(__builtin_elementwise_fma(hi, s, lo * s));
            }
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
    const float zz[2] = {sum_halves(zs[n][0]), sum_halves(zs[n][1])};
    if (c >= cols) continue;
    const float inv = 1.0f / stats[c];
    // O^T row rho of dt is V^T row R = 32 dt + rho: channel G g + 4 i + e with R = 4 U g + U e + i
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
        v += zz[gg];
        const int ch = G * (2 * dh + gg) + 4 * i;
        finish<HD>(a, sq, kh, c0 + c, ch, v, inv, gate_of(a, sq, kh, c0 + c, ch));
      }
  }
}

// out of one (row, head) from its pieces: thread (k, c) adds pieces k, k + blockDim / (HD / 4), ... of channels 4 c .. + 3.
constexpr int kMergeMost = kSlots;  // pieces
template <int HD>
__global__ __launch_bounds__(1024) void kv_merge_kernel(KvArgs a, Kind kind) {
  constexpr int C = HD / 4;
  __shared__ float wl[kMergeMost], red[2][16];
  __shared__ f4 vl[1024];
  const int tid = threadIdx.x;
  Item it;
  int h;
  if (!find_row(a, kind, blockIdx.x, h, it)) return;
  const Seq sq = it.sq;
  const int t = sq.r0 + it.row, c = it.row * a.ratio + h - it.kh * a.ratio - it.cb * kCols, end = min((it.cb + 1) * kCols, sq.n * a.ratio);
  const int keys = sq.len - sq.n + a.by_ratio(end - 1) + 1, ns = pieces_of(keys, it.size);
  if (group_of(a, kind, ns)) return;
  const float* p = kind.p + column_at<HD>(kind, it.slot, c) / 4;
  const size_t step = (size_t)kind.cols * (HD + 4);
  const int k = tid / C, n = blockDim.x / C, ch = 4 * (tid % C), wave = tid >> 6, waves = blockDim.x >> 6;
  // the first pieces' O and the gate go out before the maxima are waited for
  constexpr int kAhead = 4;
  f4 ahead[kAhead];
#pragma unroll
  for (int x = 0; x < kAhead; x++) ahead[x] = ld4(p + min(k + x * n, ns - 1) * step + ch);
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

// Which kernel serves a sequence. A unit of many columns is one workgroup that walks all its keys, so they pay where there are
// enough units for the longest of them, about 1.5 us for 32 keys, to end with the others: units x (mean keys / most keys) is at
// least kManyUnits, with the mean as in a batch of equal sequences, or half of the most where they are not. Measured, us, few
// columns' kernel / many columns', with that product: the model's heads, rows of n sequences without a prefix, 4096 of 1 (128)
// 215 / 218, 2048 of 2 (128) 132 / 117, of 3 (192) 184 / 120, of 8 (512) 455 / 277; 300, 500 rows after 1000 of 8 (133, 208)
// 89 / 91, 141 / 105; 3000, 1777, 2000, 1000 rows (243) 232 / 171; 2 or 4 of 1500 rows after 500, 2 of 600, 30 single ones (132,
// 226) 124 / 130, 213 / 162; 32 heads of 128 on 8: 1000, 1200, 1500 rows of one (125, 150, 187) 55 / 55, 74 / 65, 102 / 79; 777
// rows, 130 after 2000, 300 after 64, 8 single ones (152) 81 / 123; 100 rows after 500 of 16 (366) 90 / 86. Up to kFewCols columns
// a sequence stays with the first also beside others that do not, and so does one whose context is over limit_of(). Only equal
// numbers of rows on contexts of at most twice as many are laid out in a grid, as other contexts may be of any lengths (8 sequences of
// 500 rows after 1000, us: 100 in a grid, 106 so; 7 prompts of 800 rows and 800 rows after 60000: 5970 in a grid, 1280 so).
// Contexts up to which more than kScanMost sequences are neither cut nor planned. Measured, us, in a grid / planned: single rows of
// 140 sequences of 100, 1000, 3000 tokens 9.1 / 13.9, 27.4 / 34.0, 71.3 / 68.7, of 1000 sequences of 10 tokens 24 / 34, of 200 of
// 300 and one of 20000 269 / 23.
constexpr int kDirectKeys = 1024;
template <int HD>
hipError_t attend(const KvArgs& a, float* ws, hipStream_t s) {
  const int most = a.max_rows * a.ratio;  // columns a sequence has, at most
  const bool equal = (long)a.n_rows == (long)a.n_seqs * a.max_rows;
  const double units_of_many = (double)a.n_rows * a.ratio / kBigCols * a.HK;
  const bool use_many = most > kFewCols && units_of_many * (equal ? 1.0 - 0.5 * a.max_rows / a.max_len : 0.5) >= kManyUnits;
  const bool direct = use_many && equal && a.max_len <= 2 * a.max_rows;  // (else the contexts may be of any lengths)
  Kind few{}, many{};
  few.p = ws;
  few.count = reinterpret_cast<int*>(ws + kSlots * kSlotBytes / sizeof(float));
  few.split = many.split = use_many;
  few.cols = std::min(kCols, most);
  few.want = kWant;
  few.ncb = (std::min(most, use_many ? kFewCols : most) + kCols - 1) / kCols;
  const bool rows_in_grid = a.n_seqs > kScanMost && few.ncb == 1 && a.max_len <= kDirectKeys;
  hipError_t e = hipSuccess;
  if (a.n_seqs > kScanMost && !direct && !rows_in_grid) {
    few.plan = many.plan = few.count + 2 * kSlots;
    hipLaunchKernelGGL(kv_plan_kernel, dim3(1), dim3(1024), 0, s, a, few);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  if (use_many) {
    many.direct = direct;
    many.ncb = (most + kBigCols - 1) / kBigCols;
    const long grid = direct ? (long)a.n_seqs * a.HK * many.ncb : ((long)a.n_rows * a.ratio / kBigCols + a.n_seqs) * a.HK;
    constexpr int lds = ManyLds<HD>::kAll;
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(kv_many_kernel<HD>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((kv_many_kernel<HD>), dim3((unsigned)grid), dim3(512), lds, s, a, many);
    if ((e = hipGetLastError()) != hipSuccess || direct) return e;
  }
  // units of few columns; those of sequences whose contexts are over the limit are less than kManyUnits of 128 columns
  const long units = std::min<long>((long)a.n_seqs * few.ncb, (long)a.n_rows * a.ratio / kCols + a.n_seqs) * a.HK +
                     (use_many ? kManyUnits * (kBigCols / kCols) : 0);
  dim3 grid((unsigned)(units + (a.max_len > kUnit ? kSlots : 0)));
  if (rows_in_grid) {
    few.direct = 1;
    grid = dim3((unsigned)a.n_seqs, (unsigned)a.HK);
  }
  hipLaunchKernelGGL((kv_few_kernel<HD>), grid, dim3(64 * kWaves), 0, s, a, few);
  if ((e = hipGetLastError()) != hipSuccess || a.max_len <= kUnit || few.direct) return e;
  if (group_of(a, few, (int)std::min<size_t>((a.max_len + kUnit - 1) / kUnit, kSlots))) return e;  // whatever the chunk: more pieces, more loads
  // units of c columns that are not joined have more than 128 / c pieces, of at most kSlots in all: 8 c^2 (row, head)s
  const long rows = std::min<long>((long)a.n_rows * a.HQ, 8 * kCols * kCols);
  hipLaunchKernelGGL((kv_merge_kernel<HD>), dim3((unsigned)rows), dim3(a.max_len > 16 * kUnit && rows <= 512 ? 1024 : 256), 0, s, a, few);
  return hipGetLastError();
}

}  // namespace

size_t kv_workspace_bytes() { return kSlots * (kSlotBytes + 2 * sizeof(int)) + sizeof(int) * (kPlanHead + 4 * (size_t)kPlanMost); }

hipError_t launch_kv_attention(const KvArgs& a, void* ws, hipStream_t s) {
  return a.HD == 256 ? attend<256>(a, static_cast<float*>(ws), s) : attend<128>(a, static_cast<float*>(ws), s);
}

}  // namespace ha
