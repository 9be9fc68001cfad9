// Host side of the products whose results are not stored as they are (ha_mnb_fused, ha_mnb_logprobs, include/ha.h): checks of
// arguments, launches of fused.hip and logprobs.hip. No counterpart in the reference.
#include <algorithm>
#include <cstdint>
#include <iterator>
#include <string>

#include "fused.h"
#include "fused_plan.h"
#include "ha.h"
#include "on_device.h"

namespace {

using ha::set_error;

int bad(const std::string& m) { return set_error(HA_ERR_ARG, m); }
int hip_error(const char* what, hipError_t e) { return set_error(HA_ERR_DEVICE, std::string(what) + ": " + hipGetErrorString(e)); }

bool off(const void* p, size_t align) { return (uintptr_t)p % align != 0; }
bool overlap(const void* p, size_t np, const void* q, size_t nq) {
  const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
  return a < b + nq && b < a + np;
}
constexpr int kMaxN = 1 << 30, kMaxK = 1 << 24;  // (the kernels' 32-bit column numbers and offsets within a tile)
constexpr long kMaxStride = 1l << 40;
// Bytes from the first value to the end of the last row.
size_t span(int M, long stride, int cols, size_t size) { return ((size_t)(M - 1) * stride + cols) * size; }

// The weight and rows of a call.
int operands(const ha_mnb* w, int M, const void* a, ha::FusedArgs* f, int* device) {
  ha::MnbArgs g{};
  if (!ha::mnb_weight(w, &g, device)) return set_error(HA_ERR_HANDLE, "invalid MatMulNBits handle");
  if (M < 1 || M > 1 << 20) return bad("M must be in [1, 2^20]");
  if (!a || off(a, 16)) return bad("a must be non-NULL and 16-byte aligned");
  if (off(g.q, 4) || off(g.s, 2) || (g.asym && off(g.b, 2))) return bad("the weight's codes must be 4-byte and its scales and biases 2-byte aligned");
  if (g.N > kMaxN || g.K > kMaxK) return bad("the weight must have N up to 2^30 and K up to 2^24");
  *f = ha::FusedArgs{};
  f->M = M; f->N = g.N; f->K = g.K; f->group = g.group; f->bits = g.bits; f->asym = g.asym;
  f->a = a; f->q = g.q; f->s = g.s; f->b = g.b;
  f->scale = 1.0f;
  return HA_OK;
}

int check_logprobs(const ha_logprobs* p, int N, int* n_vocab) {
  if (!p) return bad("the description is NULL");
  *n_vocab = p->n_vocab ? p->n_vocab : N;
  if (*n_vocab < 1 || *n_vocab > N) return bad("n_vocab must be in [1, " + std::to_string(N) + "], the table's rows");
  if (*n_vocab > ha::kLpMaxVocab) return bad("n_vocab must be at most 2^20");
  if (p->n_targets < 0 || p->n_targets > ha::kLpMaxTargets) return bad("n_targets must be in [0, 1024]");
  if (p->top_k < 0 || p->top_k > ha::kLpMaxTop || p->top_k > *n_vocab) return bad("top_k must be in [0, 64] and at most n_vocab");
  if (!(p->scale >= 0.0f && p->scale <= 1e6f)) return bad("scale must be in [0, 1e6] (0: 1)");
  return HA_OK;
}

}  // namespace

extern "C" {

int ha_mnb_fused(ha_mnb* w, int M, const void* a, const ha_epilogue* e, void* out, void* stream) {
  ha::FusedArgs f{};
  int device = 0;
  if (int rc = operands(w, M, a, &f, &device)) return rc;
  if (!e) return bad("the epilogue is NULL");
  if (e->act != HA_ACT_NONE && e->act != HA_ACT_SILU && e->act != HA_ACT_GELU) return bad("act must be HA_ACT_NONE, HA_ACT_SILU or HA_ACT_GELU");
  if (e->gated && f.N % 2) return bad("a gated weight needs an even N");
  const int cols = e->gated ? f.N / 2 : f.N;
  if ((e->out_dtype != HA_F32 && e->out_dtype != HA_F16) || (e->residual && e->residual_dtype != HA_F32 && e->residual_dtype != HA_F16))
    return bad("dtypes must be HA_F32 or HA_F16");
  const size_t size = e->out_dtype == HA_F32 ? 4 : 2, rsize = e->residual_dtype == HA_F32 ? 4 : 2;
  const long stride = e->out_stride ? e->out_stride : cols, rstride = e->residual_stride ? e->residual_stride : cols;
  if (!out || off(out, size) || stride < cols || stride > kMaxStride)
    return bad("out must be non-NULL and aligned, out_stride at least " + std::to_string(cols) + " and at most 2^40");
  if (e->bias && off(e->bias, 4)) return bad("bias must be 4-byte aligned");
  const size_t bytes = span(M, stride, cols, size);
  if (overlap(out, bytes, a, (size_t)M * f.K * 2)) return bad("out must not overlap a");
  if (e->residual) {
    if (off(e->residual, rsize) || rstride < cols || rstride > kMaxStride)
      return bad("residual must be aligned, residual_stride at least " + std::to_string(cols) + " and at most 2^40");
    const bool same = e->residual == out && rsize == size && rstride == stride;
    if (!same && overlap(out, bytes, e->residual, span(M, rstride, cols, rsize)))
      return bad("out must be the residual itself (with its type and stride) or not overlap it");
  }
  if (e->bias && overlap(out, bytes, e->bias, (size_t)f.N * 4)) return bad("out must not overlap bias");
  f.half = e->gated ? cols : 0;
  f.act = e->act; f.bias = e->bias; f.out = out; f.out_f32 = e->out_dtype == HA_F32; f.out_stride = stride;
  f.res = e->residual; f.res_f32 = e->residual_dtype == HA_F32; f.res_stride = rstride;
  if (!ha::whole(f) && !ha::fused::fits(ha::fused::any_groups({16, cols, f.K, f.half != 0, f.asym != 0, false, false}), ha::fused::kAnyThreads))
    return bad("a weight of more than 2^29 - 64 rows needs K and an alignment that the fast kernels take");
  ha::OnDevice on(device);
  if (on.rc != hipSuccess) return hip_error("hipSetDevice", on.rc);
  const hipError_t he = ha::launch_fused(f, (hipStream_t)stream);
  return he == hipSuccess ? HA_OK : hip_error("fused product", he);
}

int ha_mnb_logprobs_bytes(const ha_mnb* w, int M, const ha_logprobs* p, size_t* bytes) {
  if (!bytes) return bad("bytes is NULL");
  *bytes = 0;
  ha::MnbArgs g{};
  int device = 0, n_vocab = 0;
  if (!ha::mnb_weight(w, &g, &device)) return set_error(HA_ERR_HANDLE, "invalid MatMulNBits handle");
  if (M < 1 || M > 1 << 20) return bad("M must be in [1, 2^20]");
  if (int rc = check_logprobs(p, g.N, &n_vocab)) return rc;
  *bytes = ha::fused::most_logits_bytes(M, n_vocab, p->top_k);
  return HA_OK;
}

int ha_mnb_logprobs(ha_mnb* w, int M, const void* a, const ha_logprobs* p, void* workspace, size_t bytes, void* stream) {
  ha::LpArgs l{};
  int device = 0, n_vocab = 0;
  if (int rc = operands(w, M, a, &l.p, &device)) return rc;
  if (int rc = check_logprobs(p, l.p.N, &n_vocab)) return rc;
  if (p->n_targets && (!p->targets || !p->logp)) return bad("targets and logp must be non-NULL where n_targets > 0");
  if (p->top_k && (!p->top_ids || !p->top_logp)) return bad("top_ids and top_logp must be non-NULL where top_k > 0");
  if (!p->n_targets && !p->top_k && !p->entropy && !p->lse) return bad("nothing is asked for");
  for (const void* q : {(const void*)p->targets, (const void*)p->logp, (const void*)p->entropy, (const void*)p->lse, (const void*)p->top_ids,
                        (const void*)p->top_logp})
    if (off(q, 4)) return bad("targets and outputs must be 4-byte aligned");
  const size_t need = ha::fused::logits_bytes(M, n_vocab, p->top_k);
  if (!workspace || off(workspace, 16) || bytes < need) return bad("the workspace must be 16-byte aligned and have " + std::to_string(need) + " bytes");
  // A row's results are written while other rows still read a and the targets
  const struct Span { const void* p; size_t n; } others[] = {{a, (size_t)M * l.p.K * 2}, {p->targets, 4 * (size_t)M * p->n_targets}, {p->logp, 4 * (size_t)M * p->n_targets},
                                                        {p->entropy, 4 * (size_t)M}, {p->lse, 4 * (size_t)M}, {p->top_ids, 4 * (size_t)M * p->top_k},
                                                        {p->top_logp, 4 * (size_t)M * p->top_k}};
  for (const auto& x : others)
    if (x.p && x.n && overlap(workspace, need, x.p, x.n)) return bad("the workspace must not overlap a, the targets or an output");
  const Span &rows = others[0], &targets = others[1];
  for (const Span* x = others + 2; x != std::end(others); x++) {
    if (!x->p || !x->n) continue;
    if (overlap(x->p, x->n, rows.p, rows.n)) return bad("an output must not overlap a");
    const bool in_place = x == others + 2 && x->p == targets.p;  // (a row's targets are read before its logp is written)
    if (targets.p && targets.n && !in_place && overlap(x->p, x->n, targets.p, targets.n)) return bad("an output must not overlap the targets (logp may be them)");
  }
  l.p.N = n_vocab;
  l.p.scale = p->scale > 0.0f ? p->scale : 1.0f;
  const bool stored = ha::fused::store_logits(M, n_vocab, p->top_k);
  if (stored) {  // a product in f32
    l.logits = (const float*)workspace;
    l.p.out = workspace; l.p.out_f32 = 1; l.p.out_stride = n_vocab;
  } else {
    l.p.rec = (ha::LpRecord*)workspace;
  }
  l.n_targets = p->n_targets; l.targets = p->targets; l.logp = p->logp;
  l.entropy = p->entropy; l.lse = p->lse;
  l.top_k = p->top_k; l.top_ids = p->top_ids; l.top_logp = p->top_logp;
  ha::OnDevice on(device);
  if (on.rc != hipSuccess) return hip_error("hipSetDevice", on.rc);
  hipError_t he = hipSuccess;
  for (int left = M; left > 0 && he == hipSuccess;) {  // (parts of stored logits stand in the same place)
    const int part = l.p.M = stored ? std::min(left, ha::fused::stored_part(n_vocab)) : left;
    he = stored ? ha::launch_fused(l.p, (hipStream_t)stream) : ha::launch_logit_records(l.p, (hipStream_t)stream);
    if (he == hipSuccess) he = ha::launch_logprobs(l, (hipStream_t)stream);
    l.p.a = (const char*)l.p.a + (size_t)part * l.p.K * 2;
    if (l.n_targets) l.targets += (size_t)part * l.n_targets, l.logp += (size_t)part * l.n_targets;
    if (l.entropy) l.entropy += part;
    if (l.lse) l.lse += part;
    if (l.top_k) l.top_ids += (size_t)part * l.top_k, l.top_logp += (size_t)part * l.top_k;
    left -= part;
  }
  return he == hipSuccess ? HA_OK : hip_error("log probabilities", he);
}

}  // extern "C"
