// The host code of the products whose results are not stored as they are (csrc/fused_host.cpp) against a HIP runtime of two
// devices that runs nothing: what its calls refuse before they launch, what the launches get, which device is current afterwards.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <string>

#include "fused.h"
#include "ha.h"

#define CHECK(x) \
  do { if (!(x)) { fprintf(stderr, "%s:%d: %s (%s)\n", __FILE__, __LINE__, #x, last.c_str()); exit(1); } } while (0)
// a refusal with this in its message, and no launch
#define BAD(call, text) \
  do { last = ""; const int n = launches; CHECK((call) == HA_ERR_ARG && last.find(text) != std::string::npos && launches == n && current == 0); } while (0)

static std::string last;
static int current = 0, launches = 0, launched_on = -1;
static ha::FusedArgs got;
static ha::LpArgs got_lp;
static hipError_t launch_result = hipSuccess;
struct ha_mnb { ha::MnbArgs args; int device; };
static ha_mnb good;

namespace ha {
int set_error(int code, const std::string& msg) { last = msg; return code; }
bool mnb_weight(const ha_mnb* w, MnbArgs* args, int* device) {
  if (w != &good) return false;
  *args = w->args;
  *device = w->device;
  return true;
}
static hipError_t note(const FusedArgs& a) { got = a; launches++; launched_on = current; return launch_result; }
hipError_t launch_fused(const FusedArgs& a, hipStream_t) { return note(a); }
hipError_t launch_logit_records(const FusedArgs& a, hipStream_t) { return note(a); }
hipError_t launch_logprobs(const LpArgs& a, hipStream_t) { got_lp = a; launches++; return launch_result; }
}  // namespace ha

extern "C" {
hipError_t hipGetDevice(int* d) { *d = current; return hipSuccess; }
hipError_t hipSetDevice(int d) { current = d; return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "an error"; }
}

int main() {
  char* const base = (char*)0x100000;  // (addresses only: nothing is read)
  char *q = base, *s = base + 0x10000, *a = base + 0x20000, *out = base + 0x40000, *res = base + 0x80000, *bias = base + 0xC0000;
  good.args.N = 100; good.args.K = 128; good.args.bits = 4; good.args.group = 32;
  good.args.q = q; good.args.s = s;
  good.device = 1;

  // ---- products ----
  ha_epilogue e = {};
  e.out_dtype = HA_F16;
  CHECK(ha_mnb_fused(nullptr, 3, a, &e, out, nullptr) == HA_ERR_HANDLE);
  CHECK(ha_mnb_fused((ha_mnb*)a, 3, a, &e, out, nullptr) == HA_ERR_HANDLE && launches == 0);
  CHECK(ha_mnb_fused(&good, 3, a, &e, out, nullptr) == HA_OK && launches == 1 && launched_on == 1 && current == 0);
  CHECK(got.M == 3 && got.N == 100 && got.K == 128 && got.half == 0 && got.out_stride == 100 && !got.out_f32 && !got.res && !got.bias);
  BAD(ha_mnb_fused(&good, 0, a, &e, out, nullptr), "M must");
  BAD(ha_mnb_fused(&good, (1 << 20) + 1, a, &e, out, nullptr), "M must");
  BAD(ha_mnb_fused(&good, 3, nullptr, &e, out, nullptr), "a must");
  BAD(ha_mnb_fused(&good, 3, a + 8, &e, out, nullptr), "a must");
  BAD(ha_mnb_fused(&good, 3, a, nullptr, out, nullptr), "epilogue");
  BAD(ha_mnb_fused(&good, 3, a, &e, nullptr, nullptr), "out must");
  BAD(ha_mnb_fused(&good, 3, a, &e, out + 1, nullptr), "out must");
  for (int act : {-1, 3}) { ha_epilogue b = e; b.act = act; BAD(ha_mnb_fused(&good, 3, a, &b, out, nullptr), "act must"); }
  for (int t : {-1, 2}) { ha_epilogue b = e; b.out_dtype = t; BAD(ha_mnb_fused(&good, 3, a, &b, out, nullptr), "dtypes"); }
  { ha_epilogue b = e; b.out_dtype = HA_F32; BAD(ha_mnb_fused(&good, 3, a, &b, out + 2, nullptr), "out must"); }
  for (long t : {99l, -1l}) { ha_epilogue b = e; b.out_stride = t; BAD(ha_mnb_fused(&good, 3, a, &b, out, nullptr), "out_stride"); }
  { ha_epilogue b = e; b.bias = (float*)(bias + 2); BAD(ha_mnb_fused(&good, 3, a, &b, out, nullptr), "bias"); }
  { ha_epilogue b = e; b.bias = (float*)(out + 3 * 200 - 4); BAD(ha_mnb_fused(&good, 3, a, &b, out, nullptr), "bias"); }
  // the rows of a and out: next to each other, and one byte into each other
  CHECK(ha_mnb_fused(&good, 3, a, &e, a + 3 * 256, nullptr) == HA_OK);
  BAD(ha_mnb_fused(&good, 3, a, &e, a + 3 * 256 - 2, nullptr), "overlap a");
  CHECK(ha_mnb_fused(&good, 3, a, &e, a - 600, nullptr) == HA_OK);
  BAD(ha_mnb_fused(&good, 3, a, &e, a - 598, nullptr), "overlap a");
  {  // residuals: apart, the result itself, or refused
    ha_epilogue b = e;
    b.residual = res; b.residual_dtype = HA_F32; b.residual_stride = 104;
    CHECK(ha_mnb_fused(&good, 3, a, &b, out, nullptr) == HA_OK && got.res == res && got.res_f32 == 1 && got.res_stride == 104);
    b.residual_dtype = 7; BAD(ha_mnb_fused(&good, 3, a, &b, out, nullptr), "dtypes");
    b.residual_dtype = HA_F32;
    b.residual_stride = 99; BAD(ha_mnb_fused(&good, 3, a, &b, out, nullptr), "residual_stride");
    b.residual_stride = 0; b.residual = res + 2; BAD(ha_mnb_fused(&good, 3, a, &b, out, nullptr), "residual");
    b.residual = out; BAD(ha_mnb_fused(&good, 3, a, &b, out, nullptr), "residual itself");  // (another type)
    b.residual_dtype = HA_F16; CHECK(ha_mnb_fused(&good, 3, a, &b, out, nullptr) == HA_OK);
    b.residual_stride = 101; BAD(ha_mnb_fused(&good, 3, a, &b, out, nullptr), "residual itself");
    b.residual_stride = 100; CHECK(ha_mnb_fused(&good, 3, a, &b, out, nullptr) == HA_OK);
    b.residual = out + 2; BAD(ha_mnb_fused(&good, 3, a, &b, out, nullptr), "residual itself");
  }
  {  // gated: half of the columns
    ha_epilogue b = e;
    b.gated = 1; b.act = HA_ACT_SILU; b.out_stride = 50;
    CHECK(ha_mnb_fused(&good, 3, a, &b, out, nullptr) == HA_OK && got.half == 50 && got.N == 100 && got.act == HA_ACT_SILU && got.out_stride == 50);
    good.args.N = 101;
    BAD(ha_mnb_fused(&good, 3, a, &b, out, nullptr), "even N");
    good.args.N = 100;
  }
  good.args.q = q + 2; BAD(ha_mnb_fused(&good, 3, a, &e, out, nullptr), "codes"); good.args.q = q;
  good.args.s = s + 1; BAD(ha_mnb_fused(&good, 3, a, &e, out, nullptr), "codes"); good.args.s = s;
  { ha_epilogue b = e; b.out_stride = (1l << 40) + 1; BAD(ha_mnb_fused(&good, 3, a, &b, out, nullptr), "2^40"); }
  { ha_epilogue b = e; b.residual = res; b.residual_dtype = HA_F32; b.residual_stride = 1l << 62; BAD(ha_mnb_fused(&good, 3, a, &b, out, nullptr), "2^40"); }
  good.args.N = (1 << 30) + 2; BAD(ha_mnb_fused(&good, 1, a, &e, out, nullptr), "2^30"); good.args.N = 100;
  good.args.K = (1 << 24) + 32; BAD(ha_mnb_fused(&good, 1, a, &e, out, nullptr), "2^24"); good.args.K = 128;
  launch_result = hipErrorInvalidValue;
  CHECK(ha_mnb_fused(&good, 3, a, &e, out, nullptr) == HA_ERR_DEVICE && current == 0);
  launch_result = hipSuccess;

  // ---- log probabilities ----
  ha_logprobs p = {};
  p.n_vocab = 90; p.n_targets = 2; p.targets = (int*)base; p.logp = (float*)out; p.entropy = (float*)(out + 64);
  p.top_k = 5; p.top_ids = (int*)(out + 128); p.top_logp = (float*)(out + 256);
  size_t bytes = 1;
  CHECK(ha_mnb_logprobs_bytes(&good, 7, &p, &bytes) == HA_OK && bytes == 7 * 90 * 4);
  CHECK(ha_mnb_logprobs_bytes(nullptr, 7, &p, &bytes) == HA_ERR_HANDLE && bytes == 0);
  BAD(ha_mnb_logprobs_bytes(&good, 7, &p, nullptr), "bytes");
  BAD(ha_mnb_logprobs_bytes(&good, 0, &p, &bytes), "M must");
  BAD(ha_mnb_logprobs_bytes(&good, 7, nullptr, &bytes), "NULL");
  launches = 0;
  CHECK(ha_mnb_logprobs(&good, 7, a, &p, res, 2520, nullptr) == HA_OK && launches == 2 && launched_on == 1 && current == 0);
  CHECK(got.N == 90 && got.scale == 1.0f && got.out == res && got.out_f32 && got.out_stride == 90 && (char*)got_lp.logits == res && got_lp.n_targets == 2 && got_lp.top_k == 5 && got_lp.p.N == 90 && !got_lp.lse);
  CHECK(ha_mnb_logprobs(nullptr, 7, a, &p, res, 2520, nullptr) == HA_ERR_HANDLE);
  BAD(ha_mnb_logprobs(&good, 7, a, &p, res, 2519, nullptr), "2520 bytes");
  BAD(ha_mnb_logprobs(&good, 7, a, &p, res + 8, 3000, nullptr), "workspace");
  BAD(ha_mnb_logprobs(&good, 7, a, &p, nullptr, 3000, nullptr), "workspace");
  BAD(ha_mnb_logprobs(&good, 7, a, nullptr, res, 3000, nullptr), "NULL");
  BAD(ha_mnb_logprobs(&good, 7, a + 2, &p, res, 3000, nullptr), "a must");
  // a workspace that ends where a or an output begins, and one byte into each
  CHECK(ha_mnb_logprobs(&good, 7, res + 2528, &p, res, 2520, nullptr) == HA_OK);
  BAD(ha_mnb_logprobs(&good, 7, res + 2512, &p, res, 2520, nullptr), "overlap");
  for (int i = 0; i < 6; i++) {
    ha_logprobs b = p;
    b.lse = (float*)(out + 512);
    char* const at = res + 2516;
    switch (i) {
      case 0: b.targets = (int*)at; break;
      case 1: b.logp = (float*)at; break;
      case 2: b.entropy = (float*)at; break;
      case 3: b.lse = (float*)at; break;
      case 4: b.top_ids = (int*)at; break;
      case 5: b.top_logp = (float*)at; break;
    }
    BAD(ha_mnb_logprobs(&good, 7, a, &b, res, 2520, nullptr), "overlap");
  }
#define WITH(field, value, text) do { ha_logprobs b = p; b.field = value; BAD(ha_mnb_logprobs(&good, 7, a, &b, res, 1 << 20, nullptr), text); } while (0)
  WITH(n_vocab, 101, "n_vocab"); WITH(n_vocab, -1, "n_vocab");
  WITH(n_targets, -1, "n_targets"); WITH(n_targets, 1025, "n_targets");
  WITH(top_k, -1, "top_k"); WITH(top_k, 65, "top_k");
  WITH(scale, -1.0f, "scale"); WITH(scale, 1.1e6f, "scale"); WITH(scale, INFINITY, "scale"); WITH(scale, NAN, "scale");
  WITH(targets, nullptr, "targets"); WITH(logp, nullptr, "targets"); WITH(top_ids, nullptr, "top_ids"); WITH(top_logp, nullptr, "top_ids");
  WITH(targets, (int*)(base + 2), "aligned"); WITH(entropy, (float*)(base + 1), "aligned"); WITH(lse, (float*)(base + 3), "aligned");
  { ha_logprobs b = p; b.n_vocab = 3; b.top_k = 4; BAD(ha_mnb_logprobs(&good, 7, a, &b, res, 1 << 20, nullptr), "top_k"); }
  { ha_logprobs b = {}; BAD(ha_mnb_logprobs(&good, 7, a, &b, res, 1 << 20, nullptr), "nothing"); }
  { ha_logprobs b = {}; b.lse = (float*)out; b.scale = 2.5f;
    CHECK(ha_mnb_logprobs(&good, 7, a, &b, res, 1 << 20, nullptr) == HA_OK && got.scale == 2.5f && got.N == 100); }
  good.args.N = 40000;  // (a larger vocabulary: records)
  { ha_logprobs b = p; b.n_vocab = 0;
    CHECK(ha_mnb_logprobs_bytes(&good, 7, &b, &bytes) == HA_OK && bytes == 7 * 625 * 16);
    CHECK(ha_mnb_logprobs(&good, 7, a, &b, res, bytes, nullptr) == HA_OK && (char*)got.rec == res && !got.out && !got_lp.logits); }
  good.args.N = (1 << 20) + 64;
  { ha_logprobs b = p; b.n_vocab = 0; BAD(ha_mnb_logprobs(&good, 7, a, &b, res, 1 << 30, nullptr), "2^20");
    b.n_vocab = 1 << 20; CHECK(ha_mnb_logprobs(&good, 7, a, &b, res, 1 << 30, nullptr) == HA_OK); }
  launch_result = hipErrorInvalidValue;
  CHECK(ha_mnb_logprobs(&good, 7, a, &p, res, 2520, nullptr) == HA_ERR_DEVICE && current == 0);
  return 0;
}
