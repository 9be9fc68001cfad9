// Products with quantised weights whose results go straight into what follows (fused_*.h, fused.hip, logprobs.hip): argument
// blocks shared with their host side (fused_host.cpp).
#pragma once
#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>
#include <string>

#include "ha_kernels.h"

namespace ha {

constexpr int kLpBlock = 64;     // columns of a block of logits (a record of its own)
constexpr int kLpMargin = 8;     // blocks looked at beyond the top_k largest
constexpr int kLpMaxTop = 64;    // top_k, at most
constexpr int kLpMaxTargets = 1024;
constexpr int kLpMaxVocab = 1 << 20;

// What a 64-column block of a row's scaled logits comes to: its largest value, over the other columns the sums of e^(z - max)
// and e^(z - max) (z - max), and a word whose upper 26 bits are a bound from above of the second largest value (as an unsigned
// number in the same order) and whose lower 6 say which column is the largest (the first of equals).
struct LpRecord {
  float max, rest, rest_z;
  unsigned second;
};

struct FusedArgs {
  int M, N, K, group;  // N: rows of the weight that count
  const void* a;       // [M][K] f16, 16-byte aligned
  const void* q;       // [N][K/32][bits] u32
  const void* s;       // [N][K/group] f16
  const void* b;       // the same, asymmetric only
  int bits, asym;
  // products
  int half;            // gated: N / 2, the columns of the result; 0: not gated
  int act, out_f32, res_f32;
  const float* bias;   // [N] or nullptr
  const void* res;     // or nullptr
  long res_stride;
  void* out;
  long out_stride;
  // logits
  float scale;
  LpRecord* rec;       // [M][ceil(N / 64)]
};

// Whether the kernels that move whole 64-k tiles can run the operands: codes in whole words of a block's half, two scales at once.
inline bool whole(const FusedArgs& p) {
  const uintptr_t sb = (uintptr_t)p.s | (p.asym ? (uintptr_t)p.b : 0);
  return p.K % 64 == 0 && (p.group == 32 || p.K % 128 == 0) && (uintptr_t)p.q % (p.bits == 4 ? 16 : 4) == 0 && sb % 4 == 0;
}

struct LpArgs {
  FusedArgs p;         // the product that the records are of
  const float* logits; // [M][N] in the records' place, or nullptr
  int n_targets, top_k;
  const int* targets;  // [M][n_targets]
  float* logp;         // [M][n_targets]
  float* entropy;      // [M] or nullptr
  float* lse;          // [M] or nullptr
  int* top_ids;        // [M][top_k]
  float* top_logp;     // [M][top_k]
};

hipError_t launch_fused(const FusedArgs& a, hipStream_t s);         // product with its activation, bias and residual
hipError_t launch_logit_records(const FusedArgs& a, hipStream_t s);  // records of the scaled logits
hipError_t launch_fused_lanes(const FusedArgs& a, hipStream_t s);  // one or two rows, up to 64 KiB of them
hipError_t launch_fused_rows(const FusedArgs& a, int mt, int nt, hipStream_t s);   // with the tiles that fused_plan.h gives
hipError_t launch_fused_tiles(const FusedArgs& a, int rt, int ct, int halves, hipStream_t s);
hipError_t launch_logit_tiles(const FusedArgs& a, hipStream_t s);
hipError_t launch_logprobs(const LpArgs& a, hipStream_t s);          // what the records come to

int set_error(int code, const std::string& msg);  // the calling thread's ha_last_error(); returns the code

}  // namespace ha
