// What the products whose results are not stored as they are launch (csrc/fused_host.cpp and the host side of fused*.hip and
// logprobs.hip, compiled for the host alone) against a HIP runtime that runs nothing. Lines of stdin:
//   fused M N K bits group asym gated q_at s_at               (q_at, s_at: bytes past an aligned address)
//   logprobs M V K bits group asym n_vocab targets top_k q_at bytes   (bytes: of the workspace; -1: as many as the call asks for)
//   bytes M V K n_vocab targets top_k
//   put <output> <a | targets> <bytes>           (the next call's output of that name stands there)
//   kernels                                      (lines "kernel <name>" of all there are)
// For each, the launches ("launch <kernel> <workgroups> <threads> <lds> <rows> <bytes from a, out, residual, records, logp, lse,
// top_ids of the first row's>"), the functions' LDS limits that were set ("limit <kernel> <bytes>"), and "done <status> <bytes>".
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstring>
#include <map>
#include <string>

#include "fused.h"
#include "ha.h"

struct ha_mnb { ha::MnbArgs args; };
static ha_mnb weight;
static std::map<const void*, std::string>& names() {  // (filled before main)
  static std::map<const void*, std::string> m;
  return m;
}
static dim3 grid, block;
static size_t shared;
static char *const kA = (char*)(1l << 53), *const kQ = (char*)(2l << 53), *const kS = (char*)(3l << 53), *const kB = (char*)(4l << 53),
                  *const kWork = (char*)(5l << 53), *const kRes = (char*)(6l << 53), *const kOut = (char*)(7l << 53), *const kLogp = (char*)(8l << 53),
                  *const kLse = (char*)(9l << 53), *const kIds = (char*)(10l << 53), *const kTop = (char*)(11l << 53), *const kTargets = (char*)(12l << 53);

namespace ha {
int set_error(int code, const std::string& msg) { printf("refused %s\n", msg.c_str()); return code; }
bool mnb_weight(const ha_mnb* w, MnbArgs* args, int* device) { *args = w->args; *device = 0; return true; }
}  // namespace ha

extern "C" {
hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "an error"; }
hipError_t hipFuncSetAttribute(const void* f, hipFuncAttribute, int value) { printf("limit %s %d\n", names()[f].c_str(), value); return hipSuccess; }
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t n, hipStream_t) { grid = g; block = b; shared = n; return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3* g, dim3* b, size_t* n, hipStream_t* s) { *g = grid; *b = block; *n = shared; *s = nullptr; return hipSuccess; }
void** __hipRegisterFatBinary(const void*) { static void* h; return &h; }
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void* host, char*, const char* name, unsigned, void*, void*, void*, void*, int*) { names()[host] = name; }
hipError_t hipLaunchKernel(const void* f, dim3 g, dim3 b, void** args, size_t lds, hipStream_t) {
  const std::string& n = names()[f];
  const bool join = n.find("logprobs_kernel") != std::string::npos;
  const ha::LpArgs* l = join ? (const ha::LpArgs*)args[0] : nullptr;
  const ha::FusedArgs& p = join ? l->p : *(const ha::FusedArgs*)args[0];
  auto from = [](const void* x, const char* base) { return x ? (long)((const char*)x - base) : -1l; };
  printf("launch %s %u %u %zu %d %ld %ld %ld %ld %ld %ld %ld\n", n.c_str(), g.x, b.x, lds, p.M, from(p.a, kA), p.out && p.out < kRes ? from(p.out, kWork) : from(p.out, kOut),
         from(p.res, kRes), from(p.rec, kWork), from(l ? l->logp : nullptr, kLogp), from(l ? l->lse : nullptr, kLse), from(l ? l->top_ids : nullptr, kIds));
  return hipSuccess;
}
}

int main() {
  char line[256], what[16], name[16], base[16];
  std::map<std::string, void*> put;
  while (fgets(line, sizeof line, stdin)) {
    long v[11] = {};
    if (!strncmp(line, "kernels", 7)) {
      for (const auto& x : names()) printf("kernel %s\n", x.second.c_str());
      continue;
    }
    if (sscanf(line, "put %15s %15s %ld", name, base, v) == 3) {
      put[name] = (strcmp(base, "a") ? kTargets : kA) + v[0];
      continue;
    }
    if (sscanf(line, "%15s %ld %ld %ld %ld %ld %ld %ld %ld %ld %ld %ld", what, v, v + 1, v + 2, v + 3, v + 4, v + 5, v + 6, v + 7, v + 8, v + 9, v + 10) < 2) continue;
    ha::MnbArgs& w = weight.args;
    w = {};
    w.N = (int)v[1]; w.K = (int)v[2];
    size_t bytes = 0;
    int rc = 0;
    auto asked = [&](int n_vocab, int targets, int top_k) {
      ha_logprobs p = {};
      p.n_vocab = n_vocab; p.n_targets = targets; p.top_k = top_k;
      p.targets = (int*)kTargets; p.logp = (float*)kLogp; p.lse = (float*)kLse; p.top_ids = (int*)kIds; p.top_logp = (float*)kTop;
      if (put.count("logp")) p.logp = (float*)put["logp"];
      if (put.count("entropy")) p.entropy = (float*)put["entropy"];
      if (put.count("lse")) p.lse = (float*)put["lse"];
      if (put.count("top_ids")) p.top_ids = (int*)put["top_ids"];
      if (put.count("top_logp")) p.top_logp = (float*)put["top_logp"];
      put.clear();
      return p;
    };
    if (!strcmp(what, "bytes")) {
      w.bits = 4; w.group = 32;
      const ha_logprobs p = asked((int)v[3], (int)v[4], (int)v[5]);
      rc = ha_mnb_logprobs_bytes(&weight, (int)v[0], &p, &bytes);
    } else {
      w.bits = (int)v[3]; w.group = (int)v[4]; w.asym = (int)v[5];
      w.s = kS; w.b = w.asym ? kB : nullptr;
      if (!strcmp(what, "fused")) {
        w.q = kQ + v[7]; w.s = kS + v[8];
        ha_epilogue e = {};
        e.gated = (int)v[6]; e.out_dtype = HA_F32; e.residual = kRes; e.residual_dtype = HA_F16;
        rc = ha_mnb_fused(&weight, (int)v[0], kA, &e, kOut, nullptr);
      } else {
        w.q = kQ + v[9];
        const ha_logprobs p = asked((int)v[6], (int)v[7], (int)v[8]);
        rc = ha_mnb_logprobs_bytes(&weight, (int)v[0], &p, &bytes);
        if (v[10] >= 0) bytes = (size_t)v[10];
        if (rc == 0) rc = ha_mnb_logprobs(&weight, (int)v[0], kA, &p, kWork, bytes, nullptr);
      }
    }
    printf("done %d %zu\n", rc, bytes);
    fflush(stdout);
  }
  return 0;
}
