// The cache's host code (csrc/kv_host.cpp) against a HIP runtime of two devices that runs nothing: what its calls refuse before
// they launch, what the launches get, which device is current afterwards, and creations that run out of memory.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <string>

#include "ha.h"
#include "kv.h"

#define CHECK(x) \
  do { if (!(x)) { fprintf(stderr, "%s:%d: %s (%s)\n", __FILE__, __LINE__, #x, last.c_str()); exit(1); } } while (0)

static std::string last;
static int current = 0, blocks = 0, allowed = 1 << 30, launches = 0, launched_on = -1;
static ha::KvArgs got;
static hipError_t launch_result = hipSuccess;

namespace ha {
int set_error(int code, const std::string& msg) { last = msg; return code; }
hipError_t launch_kv_rope(float* rope, const double* p, int max_ctx, int rot, hipStream_t) {
  for (long i = 0; i < (long)max_ctx * rot; i++) rope[i] = (float)p[(i % rot) / 2];
  return hipSuccess;
}
static hipError_t note(const KvArgs& a) { got = a; launches++; launched_on = current; return launch_result; }
hipError_t launch_kv_append(const KvArgs& a, hipStream_t) { return note(a); }
size_t kv_workspace_bytes() { return 4096; }
hipError_t launch_kv_attention(const KvArgs& a, void* ws, hipStream_t) { CHECK(ws); return note(a); }
}  // namespace ha

extern "C" {
hipError_t hipGetDeviceCount(int* n) { *n = 2; return hipSuccess; }
hipError_t hipGetDevice(int* d) { *d = current; return hipSuccess; }
hipError_t hipSetDevice(int d) { current = d; return hipSuccess; }
hipError_t hipMalloc(void** p, size_t n) {
  if (allowed-- <= 0) return hipErrorOutOfMemory;
  blocks++;
  *p = malloc(n);
  return hipSuccess;
}
hipError_t hipFree(void* p) { blocks--; free(p); return hipSuccess; }
hipError_t hipMemset(void* p, int v, size_t n) { memset(p, v, n); return hipSuccess; }
hipError_t hipMemcpy(void* d, const void* s, size_t n, hipMemcpyKind) { memcpy(d, s, n); return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipDeviceSynchronize() { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "an error"; }
}

int main() {
  alignas(16) static unsigned char pages[64], rows[64], q[64], out[64];
  static int ints[4];
  const ha_kv_config c = {3, 5, 16, 100, 6, 2, 128, 32, 1, HA_F16, 1e4f, 1e-6f, 0.0f};
  ha_kv* k = nullptr;
  // every allocation that can fail: nothing is kept
  for (allowed = 0; allowed < 4; ) {
    const int n = allowed;
    CHECK(ha_kv_create(&c, pages, 1, &k) == HA_ERR_NOMEM && !k && blocks == 0 && current == 0);
    allowed = n + 1;
  }
  allowed = 1 << 30;
  CHECK(ha_kv_create(&c, pages, 2, &k) == HA_ERR_ARG && ha_kv_create(&c, pages, -1, &k) == HA_ERR_ARG && !k);
  CHECK(ha_kv_create(&c, pages, 1, &k) == HA_OK && k && current == 0);
  const int kept = blocks;

  const ha_kv_batch ok = {2, 9, 5, 40, ints, ints, ints, 3};
  const long width = 6 * 2 * 128 + 2 * 2 * 128;
  CHECK(ha_kv_append(k, 2, &ok, rows, width, q, out, nullptr) == HA_OK && launches == 1 && launched_on == 1 && current == 0);
  size_t page = 0;
  CHECK(ha_kv_page_bytes(&c, &page) == HA_OK && page == 2 * 2 * 16 * (64 + 16));
  CHECK(got.pool == pages + 2 * 5 * page && got.n_seqs == 2 && got.n_rows == 9 && got.max_rows == 5 && got.max_len == 40 && got.table_stride == 3);
  CHECK(got.page == 16 && got.page_log2 == 4 && got.ratio == 3 && got.gated == 1 && got.rot == 32 && got.dtype == HA_F16);
  CHECK(got.scale == (float)(1.0 / 11.313708498984761) && got.kw == got.qw + 128 && got.qw[0] == 1.0f && got.kw[127] == 1.0f);
  for (int ratio = 1; ratio <= 16; ratio++) {  // the division by the ratio, at its far end too
    ha::KvArgs a{};
    a.ratio = ratio; a.ratio_inv = ratio > 1 ? (unsigned)((0x100000000ull + ratio - 1) / ratio) : 0u;
    for (long x = 0; x < 1l << 28; x += x < 4096 || x > (1l << 28) - 4096 ? 1 : 4093) CHECK(a.by_ratio((int)x) == x / ratio);
  }
  float w[128];
  for (int i = 0; i < 128; i++) w[i] = 2.0f;
  CHECK(ha_kv_set_param(k, 2, "k_norm", w, 128) == HA_OK && got.kw[5] == 2.0f && got.qw[5] == 1.0f && current == 0);
  CHECK(ha_kv_attention(k, 0, &ok, q, rows, width, out, nullptr) == HA_OK && launches == 2 && got.pool == pages && got.out == (_Float16*)out);

  auto refused = [&](int code, int layer, const ha_kv_batch* b, void* r, long stride, void* qq, void* o) {
    const int n = launches;
    CHECK(ha_kv_append(k, layer, b, r, stride, qq, o, nullptr) == code);
    if (qq && o) CHECK(ha_kv_attention(k, layer, b, qq, r, stride, o, nullptr) == code);
    CHECK(launches == n && current == 0);
  };
  refused(HA_ERR_ARG, 3, &ok, rows, width, q, out);
  refused(HA_ERR_ARG, -1, &ok, rows, width, q, out);
  refused(HA_ERR_ARG, 0, nullptr, rows, width, q, out);
  refused(HA_ERR_ARG, 0, &ok, nullptr, width, q, out);
  refused(HA_ERR_ARG, 0, &ok, rows + 8, width, q, out);
  refused(HA_ERR_ARG, 0, &ok, rows, width - 8, q, out);
  refused(HA_ERR_ARG, 0, &ok, rows, width + 4, q, out);
  refused(HA_ERR_ARG, 0, &ok, rows, -width, q, out);
  refused(HA_ERR_ARG, 0, &ok, rows, width, q + 2, out);
  refused(HA_ERR_ARG, 0, &ok, rows, width, q, out + 8);
  CHECK(ha_kv_attention(k, 0, &ok, nullptr, rows, width, out, nullptr) == HA_ERR_ARG);
  CHECK(ha_kv_attention(k, 0, &ok, q, rows, width, nullptr, nullptr) == HA_ERR_ARG);
  struct { int field, value, code; } bad[] = {
      {0, 0, HA_ERR_ARG}, {0, 65536, HA_ERR_ARG}, {0, -1, HA_ERR_ARG}, {1, -1, HA_ERR_ARG}, {1, 4, HA_ERR_ARG}, {2, 10, HA_ERR_ARG},
      {2, -1, HA_ERR_ARG}, {3, 4, HA_ERR_ARG}, {3, 49, HA_ERR_ARG}, {3, 101, HA_ERR_CONTEXT}, {3, 0x7fffffff, HA_ERR_CONTEXT}, {4, 0, HA_ERR_ARG},
      {4, 2, HA_ERR_ARG}, {1, 0x7fffffff, HA_ERR_ARG}, {1, (1 << 27) / 6 + 1, HA_ERR_ARG}};
  for (auto& x : bad) {
    ha_kv_batch b = ok;
    int* f[] = {&b.n_seqs, &b.n_rows, &b.max_rows, &b.max_len, &b.table_stride};
    *f[x.field] = x.value;
    refused(x.code, 0, &b, rows, width, q, out);
  }
  for (int i = 0; i < 3; i++) {
    ha_kv_batch b = ok;
    const int** f[] = {&b.row_start, &b.len, &b.pages};
    *f[i] = nullptr;
    refused(HA_ERR_ARG, 0, &b, rows, width, q, out);
  }
  ha_kv_batch none = ok;
  none.max_rows = 0;  // nothing to do
  int n = launches;
  CHECK(ha_kv_append(k, 0, &none, rows, width, q, out, nullptr) == HA_OK && ha_kv_attention(k, 0, &none, q, rows, width, out, nullptr) == HA_OK);
  CHECK(launches == n);
  CHECK(ha_kv_set_param(k, 3, "q_norm", w, 128) == HA_ERR_ARG && ha_kv_set_param(k, 0, "q_norm", w, 127) == HA_ERR_PARAM);
  CHECK(ha_kv_set_param(k, 0, "gnorm", w, 128) == HA_ERR_PARAM && ha_kv_set_param(k, 0, nullptr, w, 128) == HA_ERR_ARG);
  launch_result = hipErrorInvalidValue;
  CHECK(ha_kv_append(k, 0, &ok, rows, width, q, out, nullptr) == HA_ERR_DEVICE && ha_kv_attention(k, 0, &ok, q, rows, width, out, nullptr) == HA_ERR_DEVICE);

  // no gates, no rotation: rows are q | k | v, and attention reads none
  ha_kv_config u = c;
  u.gated = 0; u.rot_dim = 0; u.scale = 0.5f;
  ha_kv* k2 = nullptr;
  launch_result = hipSuccess;
  CHECK(ha_kv_create(&u, pages, 0, &k2) == HA_OK && blocks == 2 * kept - 1);
  CHECK(ha_kv_append(k2, 0, &ok, rows, 6 * 128 + 4 * 128, nullptr, nullptr, nullptr) == HA_OK && !got.rope && got.scale == 0.5f);
  CHECK(ha_kv_attention(k2, 0, &ok, q, nullptr, 0, out, nullptr) == HA_OK);
  CHECK(ha_kv_destroy(k) == HA_OK && ha_kv_destroy(k) == HA_ERR_HANDLE && ha_kv_destroy(k2) == HA_OK && blocks == 0);
  CHECK(ha_kv_append(k2, 0, &ok, rows, width, q, out, nullptr) == HA_ERR_HANDLE);
  return 0;
}
