// Host side of the paged 4-bit K/V cache (ha_kv_*, include/ha.h): handles, checks of arguments, launches of kv.hip. No
// counterpart in the reference, whose K/V are one f16 block of a single sequence (web/public/engine/engine.js:95-104).
#include <cmath>
#include <cstdint>
#include <mutex>
#include <new>
#include <string>
#include <unordered_set>
#include <vector>

#include "ha.h"
#include "kv.h"

namespace {

using ha::set_error;

constexpr uint32_t kKvMagic = 0x48414b56u;
std::mutex g_kv_mu;
std::unordered_set<const ha_kv*> g_live_kvs;  // handles that exist: a destroyed or forged one is refused before it is read

// The calling thread's current device is the caller's again after a call.
struct OnDevice {
  int before = -1;
  hipError_t rc;
  explicit OnDevice(int device) {
    rc = hipGetDevice(&before);
    if (rc == hipSuccess && before != device) rc = hipSetDevice(device);
    else before = -1;
  }
  ~OnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

int hip_error(const char* what, hipError_t e) { return set_error(HA_ERR_DEVICE, std::string(what) + ": " + hipGetErrorString(e)); }

int check_config(const ha_kv_config* c) {
  auto bad = [](const char* m) { return set_error(HA_ERR_ARG, m); };
  if (!c) return bad("config is NULL");
  if (c->n_layers < 1 || c->n_pages < 1) return bad("n_layers and n_pages must be > 0");
  if (c->max_ctx < 1 || c->max_ctx > 1 << 24) return bad("max_ctx must be in [1, 2^24]");
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1))) return bad("page_size must be 16, 32, 64, 128 or 256");
  if (c->HD != 128 && c->HD != 256) return bad("head_dim must be 128 or 256");
  if (c->HK < 1 || c->HQ < 1 || c->HQ % c->HK || c->HQ / c->HK > ha::kKvMaxRatio || c->HQ > 1024)
    return bad("HQ must be a multiple of HK, at most 16 times HK and at most 1024");
  if (c->rot_dim < 0 || c->rot_dim % 8 || c->rot_dim > c->HD) return bad("rotary_dim must be a multiple of 8, at most head_dim");
  if (c->dtype != HA_F32 && c->dtype != HA_F16) return bad("dtype must be HA_F32 or HA_F16");
  if (!(c->rope_theta > 0.0f) || !std::isfinite(c->rope_theta)) return bad("rope_theta must be > 0");
  if (!(c->eps > 0.0f) || !std::isfinite(c->eps)) return bad("eps must be > 0");
  if (!(c->scale >= 0.0f) || !std::isfinite(c->scale)) return bad("scale must be >= 0");
  return HA_OK;
}

}  // namespace

struct ha_kv {
  uint32_t magic = kKvMagic;
  ha_kv_config cfg{};
  int device = 0;
  unsigned char* pages = nullptr;  // the caller's
  size_t layer_bytes = 0;
  float* rope = nullptr;
  float* norms = nullptr;          // [n_layers][2][HD]: q_norm, k_norm
  void* ws = nullptr;              // partial results of attention calls
};

namespace {

bool kv_ok(const ha_kv* k) {
  std::lock_guard<std::mutex> lock(g_kv_mu);
  return k && g_live_kvs.count(k) && k->magic == kKvMagic;
}

void free_kv(ha_kv* k) {
  for (void* p : {(void*)k->rope, (void*)k->norms, k->ws})
    if (p) (void)hipFree(p);
  k->magic = 0xdeadbeefu;
  delete k;
}

// The kernels' arguments of a call, or the reason why there are none.
int call_args(ha_kv* k, int layer, const ha_kv_batch* b, ha::KvArgs* a) {
  const ha_kv_config& c = k->cfg;
  if (layer < 0 || layer >= c.n_layers) return set_error(HA_ERR_ARG, "layer index out of range");
  if (!b || !b->row_start || !b->len || !b->pages) return set_error(HA_ERR_ARG, "batch, row_start, len and pages must be non-NULL");
  if (b->n_seqs < 1 || b->n_seqs > 65535 || (long)b->n_seqs * c.HK > 1l << 22)
    return set_error(HA_ERR_ARG, "n_seqs must be in [1, 65535] and n_seqs * HK at most 2^22");
  if (b->n_rows < 0 || b->max_rows < 0 || b->max_rows > b->n_rows) return set_error(HA_ERR_ARG, "max_rows must be in [0, n_rows]");
  if ((long)b->n_rows * c.HQ > 1l << 27) return set_error(HA_ERR_ARG, "too many rows: n_rows * HQ must be at most 2^27");
  if (b->max_len < b->max_rows || b->table_stride < 1) return set_error(HA_ERR_ARG, "max_len must be >= max_rows and table_stride > 0");
  if (b->max_len > c.max_ctx)
    return set_error(HA_ERR_CONTEXT, "context " + std::to_string(b->max_len) + " exceeds " + std::to_string(c.max_ctx));
  if ((b->max_len + (long)c.page_size - 1) / c.page_size > b->table_stride)
    return set_error(HA_ERR_ARG, "a context of " + std::to_string(b->max_len) + " does not fit a page table of " + std::to_string(b->table_stride));
  *a = ha::KvArgs{};
  a->n_seqs = b->n_seqs; a->n_rows = b->n_rows; a->max_rows = b->max_rows; a->max_len = b->max_len; a->table_stride = b->table_stride;
  a->row_start = b->row_start; a->len = b->len; a->table = b->pages;
  a->n_pages = c.n_pages; a->page = c.page_size; a->page_log2 = __builtin_ctz((unsigned)c.page_size);
  a->HQ = c.HQ; a->HK = c.HK; a->HD = c.HD; a->rot = c.rot_dim; a->gated = c.gated ? 1 : 0; a->dtype = c.dtype;
  a->ratio = c.HQ / c.HK; a->ratio_inv = a->ratio > 1 ? (unsigned)((0x100000000ull + a->ratio - 1) / a->ratio) : 0u;
  a->eps = c.eps; a->scale = c.scale > 0.0f ? c.scale : (float)(1.0 / std::sqrt((double)c.HD));
  a->pool = k->pages + (size_t)layer * k->layer_bytes;
  a->rope = k->rope;
  a->qw = k->norms + (size_t)layer * 2 * c.HD; a->kw = a->qw + c.HD;
  return HA_OK;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check_rows(const ha_kv_config& c, const void* rows, long stride) {
  const long width = (long)c.HQ * c.HD * (c.gated ? 2 : 1) + 2L * c.HK * c.HD;
  if (!rows || !aligned16(rows)) return set_error(HA_ERR_ARG, "rows must be non-NULL and 16-byte aligned");
  if (stride < width || stride % 8) return set_error(HA_ERR_ARG, "row_stride must be a multiple of 8 and at least " + std::to_string(width));
  return HA_OK;
}

}  // namespace

extern "C" {

int ha_kv_page_bytes(const ha_kv_config* cfg, size_t* bytes) {
  if (!bytes) return set_error(HA_ERR_ARG, "bytes is NULL");
  *bytes = 0;
  if (int rc = check_config(cfg)) return rc;
  *bytes = ha::kv_block_bytes(cfg->page_size, cfg->HD) * 2 * cfg->HK;
  return HA_OK;
}

int ha_kv_create(const ha_kv_config* cfg, void* pages, int device, ha_kv** out) {
  if (!out) return set_error(HA_ERR_ARG, "out is NULL");
  *out = nullptr;
  if (int rc = check_config(cfg)) return rc;
  if (!pages || !aligned16(pages)) return set_error(HA_ERR_ARG, "pages must be non-NULL and 16-byte aligned");
  int ndev = 0;
  if (hipGetDeviceCount(&ndev) != hipSuccess || ndev <= 0) return set_error(HA_ERR_DEVICE, "no HIP device is visible");
  if (device < 0 || device >= ndev) return set_error(HA_ERR_ARG, "device index out of range");
  OnDevice on(device);
  if (on.rc != hipSuccess) return hip_error("hipSetDevice", on.rc);
  ha_kv* k = nullptr;
  double* pow_dev = nullptr;
  auto bail = [&](int rc) {
    if (pow_dev) (void)hipFree(pow_dev);
    if (k) free_kv(k);
    return rc;
  };
  try {
    k = new ha_kv();
    k->cfg = *cfg;
    k->device = device;
    k->pages = static_cast<unsigned char*>(pages);
    k->layer_bytes = ha::kv_block_bytes(cfg->page_size, cfg->HD) * 2 * cfg->HK * (size_t)cfg->n_pages;
    const size_t nn = (size_t)cfg->n_layers * 2 * cfg->HD;
    const std::vector<float> ones(nn, 1.0f);
    if (hipMalloc(reinterpret_cast<void**>(&k->norms), nn * sizeof(float)) != hipSuccess) return bail(set_error(HA_ERR_NOMEM, "hipMalloc of the norms failed"));
    if (hipMalloc(&k->ws, ha::kv_workspace_bytes()) != hipSuccess) return bail(set_error(HA_ERR_NOMEM, "hipMalloc of the workspace failed"));
    hipError_t he = hipMemset(k->ws, 0, ha::kv_workspace_bytes());
    if (he != hipSuccess) return bail(hip_error("workspace", he));
    he = hipMemcpy(k->norms, ones.data(), nn * sizeof(float), hipMemcpyHostToDevice);
    if (he != hipSuccess) return bail(hip_error("norms", he));
    if (cfg->rot_dim) {
      // angle t / theta^(2 i / rot) in f64, its cosine and sine stored as f32, as the engine's table
      std::vector<double> pw(cfg->rot_dim / 2);
      for (int i = 0; i < cfg->rot_dim / 2; i++) pw[i] = std::pow((double)cfg->rope_theta, 2.0 * i / cfg->rot_dim);
      if (hipMalloc(reinterpret_cast<void**>(&k->rope), sizeof(float) * cfg->rot_dim * (size_t)cfg->max_ctx) != hipSuccess ||
          hipMalloc(reinterpret_cast<void**>(&pow_dev), sizeof(double) * pw.size()) != hipSuccess)
        return bail(set_error(HA_ERR_NOMEM, "hipMalloc of the RoPE table failed"));
      he = hipMemcpy(pow_dev, pw.data(), sizeof(double) * pw.size(), hipMemcpyHostToDevice);
      if (he == hipSuccess) he = ha::launch_kv_rope(k->rope, pow_dev, cfg->max_ctx, cfg->rot_dim, nullptr);
      if (he != hipSuccess) return bail(hip_error("RoPE table", he));
    }
    he = hipStreamSynchronize(nullptr);  // the calls may come on streams that do not wait for the null stream
    if (he != hipSuccess) return bail(hip_error("tables", he));
    if (pow_dev) (void)hipFree(pow_dev);
    pow_dev = nullptr;
    std::lock_guard<std::mutex> lock(g_kv_mu);
    g_live_kvs.insert(k);
  } catch (const std::bad_alloc&) {
    return bail(set_error(HA_ERR_NOMEM, "out of host memory"));
  }
  *out = k;
  return HA_OK;
}

int ha_kv_set_param(ha_kv* k, int layer, const char* name, const float* host, size_t count) {
  if (!kv_ok(k)) return set_error(HA_ERR_HANDLE, "invalid K/V cache handle");
  if (!name || !host) return set_error(HA_ERR_ARG, "name and data must be non-NULL");
  if (layer < 0 || layer >= k->cfg.n_layers) return set_error(HA_ERR_ARG, "layer index out of range");
  const std::string n(name);
  if (n != "q_norm" && n != "k_norm") return set_error(HA_ERR_PARAM, "no tensor " + n + " of a K/V cache");
  if (count != (size_t)k->cfg.HD)
    return set_error(HA_ERR_PARAM, n + ": expected " + std::to_string(k->cfg.HD) + " floats, got " + std::to_string(count));
  OnDevice on(k->device);
  if (on.rc != hipSuccess) return hip_error("hipSetDevice", on.rc);
  const hipError_t he = hipMemcpy(k->norms + ((size_t)layer * 2 + (n == "k_norm")) * k->cfg.HD, host, count * sizeof(float), hipMemcpyHostToDevice);
  return he == hipSuccess ? HA_OK : hip_error("hipMemcpy", he);
}

int ha_kv_append(ha_kv* k, int layer, const ha_kv_batch* batch, const void* rows, long row_stride, void* q, void* values, void* stream) {
  if (!kv_ok(k)) return set_error(HA_ERR_HANDLE, "invalid K/V cache handle");
  ha::KvArgs a;
  if (int rc = call_args(k, layer, batch, &a)) return rc;
  if (int rc = check_rows(k->cfg, rows, row_stride)) return rc;
  if (!aligned16(q) || !aligned16(values)) return set_error(HA_ERR_ARG, "q and values must be 16-byte aligned");
  if (a.max_rows == 0) return HA_OK;
  a.rows = rows; a.stride = row_stride; a.q = static_cast<_Float16*>(q); a.values = static_cast<_Float16*>(values);
  OnDevice on(k->device);
  if (on.rc != hipSuccess) return hip_error("hipSetDevice", on.rc);
  const hipError_t he = ha::launch_kv_append(a, static_cast<hipStream_t>(stream));
  return he == hipSuccess ? HA_OK : hip_error("append launch", he);
}

int ha_kv_attention(ha_kv* k, int layer, const ha_kv_batch* batch, const void* q, const void* rows, long row_stride, void* out, void* stream) {
  if (!kv_ok(k)) return set_error(HA_ERR_HANDLE, "invalid K/V cache handle");
  ha::KvArgs a;
  if (int rc = call_args(k, layer, batch, &a)) return rc;
  if (k->cfg.gated)
    if (int rc = check_rows(k->cfg, rows, row_stride)) return rc;
  if (!q || !out || !aligned16(q) || !aligned16(out)) return set_error(HA_ERR_ARG, "q and out must be non-NULL and 16-byte aligned");
  if (a.max_rows == 0) return HA_OK;
  a.rows = rows; a.stride = row_stride; a.q = static_cast<_Float16*>(const_cast<void*>(q)); a.out = static_cast<_Float16*>(out);
  OnDevice on(k->device);
  if (on.rc != hipSuccess) return hip_error("hipSetDevice", on.rc);
  const hipError_t he = ha::launch_kv_attention(a, k->ws, static_cast<hipStream_t>(stream));
  return he == hipSuccess ? HA_OK : hip_error("attention launch", he);
}

int ha_kv_destroy(ha_kv* k) {
  if (!k) return HA_OK;
  {
    std::lock_guard<std::mutex> lock(g_kv_mu);
    if (!g_live_kvs.count(k) || k->magic != kKvMagic) return set_error(HA_ERR_HANDLE, "invalid K/V cache handle");
    g_live_kvs.erase(k);
  }
  OnDevice on(k->device);
  (void)hipDeviceSynchronize();  // queued calls may still read the tables
  free_kv(k);
  return HA_OK;
}

}  // extern "C"
