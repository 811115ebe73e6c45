// Gradients of attention with terms beside scale q k (attention_terms.h; the kernels:
// attention_backward.h).
#include "attention_backward.h"

namespace hi3d {

int term_args(const hi3d_attention_desc* d, const hi3d_attention_terms* t, TermArgs& a);

namespace {

// Parts of the bias's gradient: one a workgroup of the dq kernel, then one a run of them.
constexpr int kRun = 64;
int64_t bias_length(const TermArgs& a) { return sum_length(a.far); }
int64_t bias_runs(const TermArgs& a) { return a.dq_slots <= kRun ? 0 : ceil_div(a.dq_slots, kRun); }
int64_t dbias_bytes(const TermArgs& a) {
  return align_up((a.dq_slots + bias_runs(a)) * a.hq * bias_length(a) * 4, 256);
}

int launch_dbias(const TermArgs& a, void* out, hipStream_t stream) {
  const int length = static_cast<int>(bias_length(a));
  const float* parts = a.dbias;
  int64_t count = a.total_q > 0 ? a.dq_slots : 0;
  if (count > kRun) {
    const int64_t runs = bias_runs(a);
    HI3D_REQUIRE(runs < 65536 && a.hq < 65536, "too many rows for one launch");
    float* to = a.dbias + a.dq_slots * a.hq * bias_length(a);
    hipLaunchKernelGGL(attend_dbias_sum_kernel,
                       dim3(static_cast<unsigned>(ceil_div(length, 64)), static_cast<unsigned>(runs), static_cast<unsigned>(a.hq)),
                       dim3(256), 0, stream, parts, to, length, count, kRun);
    HI3D_LAUNCH_CHECK();
    parts = to, count = runs;
  }
  hipLaunchKernelGGL(attend_dbias_kernel, dim3(static_cast<unsigned>(a.hq)), dim3(256), length * 8, stream, a, parts, count, out);
  HI3D_LAUNCH_CHECK();
  return HI3D_OK;
}

}  // namespace
}  // namespace hi3d

using namespace hi3d;

extern "C" {

int hi3d_attention_terms_backward_workspace(const hi3d_attention_desc* d, const hi3d_attention_terms* t, int64_t* bytes) {
  TermArgs a;
  const int rc = term_args(d, t, a);
  if (rc != HI3D_OK) return rc;
  HI3D_REQUIRE(bytes != nullptr, "null pointer argument");
  *bytes = 0;
  if (a.batch == 0) return HI3D_OK;
  int cus = compute_units();
  if (cus <= 0) cus = 256;  // without a device: the MI355X's
  const int splits = a.total_k > 0 ? dkv_splits(a, cus) : 1;
  dq_tiles(a, 1);
  *bytes = 2 * stats_bytes(a) + bound_bytes(a, a.hq) + (a.bias != nullptr ? dbias_bytes(a) : 0) +
           (splits > 1 ? splits * 2 * a.total_k * a.hk * a.dim * 4 : 0);
  return HI3D_OK;
}

int hi3d_attention_terms_backward(const hi3d_attention_desc* d, const hi3d_attention_terms* t, const void* out,
                                  const void* rest, const float* lse, const void* dout, const float* dlse, void* dq,
                                  void* dk, void* dv, void* dbias, void* workspace, int64_t workspace_bytes, void* stream_) {
  TermArgs a;
  int64_t need = 0;
  int rc = term_args(d, t, a);
  if (rc == HI3D_OK) rc = hi3d_attention_terms_backward_workspace(d, t, &need);
  if (rc != HI3D_OK) return rc;
  HI3D_REQUIRE((dk == nullptr) == (dv == nullptr), "dk and dv are formed together");
  HI3D_REQUIRE(dbias == nullptr || a.bias != nullptr, "no bias to form a gradient of");
  HI3D_REQUIRE(a.hq <= 65536 && (a.group - 1) * a.q_h < (1ll << 29) && a.q_h >= 0,
               "the query heads of one key head must lie within 2^29 elements");
  if (dq == nullptr && dk == nullptr && dbias == nullptr) return HI3D_OK;
  const bool rows = a.total_q > 0 || a.total_k > 0;
  if (!rows && dbias == nullptr) return HI3D_OK;
  HI3D_REQUIRE(a.batch > 0 || !rows, "rows without a segment");
  if (a.total_q > 0) HI3D_REQUIRE(out != nullptr && lse != nullptr && dout != nullptr, "null pointer argument");
  const uintptr_t at = reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(dq) |
                       reinterpret_cast<uintptr_t>(dk) | reinterpret_cast<uintptr_t>(dv) |
                       reinterpret_cast<uintptr_t>(workspace) | reinterpret_cast<uintptr_t>(rest);
  HI3D_REQUIRE(at % 16 == 0, "out, dout, the gradients and the workspace must be 16-byte aligned");
  HI3D_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), "workspace too small (%lld bytes, need %lld)",
               static_cast<long long>(workspace_bytes), static_cast<long long>(need));
  hipStream_t stream = as_stream(stream_);
  if (!rows) return launch_dbias(a, dbias, stream);
  const int cus = compute_units();
  HI3D_REQUIRE(cus > 0, "cannot query the compute unit count");
  a.o = out, a.lse = const_cast<float*>(lse), a.dout = dout, a.dlse = dlse, a.rest = const_cast<void*>(rest);
  a.out = dq, a.dk = dk, a.dv = dv;
  dq_tiles(a, 1);
  char* at_ws = static_cast<char*>(workspace);
  auto take = [&](int64_t bytes) {
    char* p = at_ws;
    at_ws += bytes;
    return reinterpret_cast<float*>(p);
  };
  a.lse2 = take(stats_bytes(a)), a.delta = take(stats_bytes(a)), a.bound = take(bound_bytes(a, a.hq));
  if (a.bias != nullptr) {
    float* parts = take(dbias_bytes(a));
    if (dbias != nullptr) a.dbias = parts;
  }
  a.part = reinterpret_cast<float*>(at_ws);
  a.splits = a.total_k > 0 ? dkv_splits(a, cus) : 1;
  const int kind = one_term(a);
  if (kind != kAll && a.dq_waves == 4 && ceil_div(a.total_k, a.batch) > 32) rc = launch_grad_of_one(a, d->dtype, kind, stream);
  else rc = d->dtype == HI3D_F16 ? launch_grad_type<_Float16, kAll>(a, stream) : launch_grad_type<__bf16, kAll>(a, stream);
  if (rc != HI3D_OK || dbias == nullptr) return rc;
  return launch_dbias(a, dbias, stream);
}

}  // extern "C"
