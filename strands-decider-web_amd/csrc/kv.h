// Argument blocks of the paged 4-bit K/V cache's kernels (kv.hip), shared with their host side (kv_host.cpp).
#pragma once
#include <hip/hip_runtime.h>
#include <cstddef>
#include <string>

namespace ha {

constexpr int kKvGroups = 4;       // groups of a row: HD / 4 consecutive channels share a scale and a zero
constexpr int kKvParamBytes = 16;  // (scale, zero) f16 of a row's groups
constexpr int kKvMaxRatio = 16;    // query heads per KV head, at most

// One (page, KV head, K or V) block: page x HD / 2 bytes of codes, then page x 16 bytes of parameters.
__host__ __device__ inline size_t kv_block_bytes(int page, int HD) { return (size_t)page * (HD / 2 + kKvParamBytes); }

// A ragged batch (ha_kv_batch) and the shape of the cache it works on.
struct KvArgs {
  int n_seqs, n_rows, max_rows, max_len, table_stride;
  const int* row_start;  // [n_seqs + 1]
  const int* len;        // [n_seqs]
  const int* table;      // [n_seqs][table_stride]
  int n_pages, page, page_log2, HQ, HK, HD, rot, gated, dtype;
  int ratio;             // HQ / HK
  unsigned ratio_inv;    // ceil(2^32 / ratio), 0 for 1
  float eps, scale;
  unsigned char* pool;   // the layer's pages
  const float* rope;     // [max_ctx][rot / 2] (cos, sin)
  const float* qw;       // [HD]
  const float* kw;       // [HD]
  const void* rows;      // [n_rows][stride] fused rows, f32 (dtype 0) or f16
  long stride;
  _Float16* q;           // [n_rows][HQ][HD]: written by append, read by attention
  _Float16* values;      // [n_rows][2][HK][HD] or nullptr
  _Float16* out;         // [n_rows][HQ][HD]
  // x / ratio of 0 <= x < 2^28 (with ratio <= 16, x ratio_inv is less than 2^32 too large)
  __host__ __device__ int by_ratio(int x) const { return ratio_inv ? (int)(((unsigned long long)(unsigned)x * ratio_inv) >> 32) : x; }
};

hipError_t launch_kv_rope(float* rope, const double* theta_pow, int max_ctx, int rot, hipStream_t s);
hipError_t launch_kv_append(const KvArgs& a, hipStream_t s);
size_t kv_workspace_bytes();  // of partial results, whatever the call; zero at first
hipError_t launch_kv_attention(const KvArgs& a, void* ws, hipStream_t s);

// Sets the calling thread's ha_last_error() message; returns the code.
int set_error(int code, const std::string& msg);

}  // namespace ha
