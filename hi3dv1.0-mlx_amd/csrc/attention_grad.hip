// Gradients of attention over packed segments (the kernels: attention_backward.h).
#include "attention_backward.h"

using namespace hi3d;

extern "C" {

int hi3d_attention_backward_workspace(const hi3d_attention_desc* d, int64_t* bytes) {
  AttnArgs a;
  const int rc = attention_args(d, a);
  if (rc != HI3D_OK) return rc;
  HI3D_REQUIRE(bytes != nullptr, "null pointer argument");
  *bytes = 0;
  if (a.batch == 0) return HI3D_OK;
  int cus = compute_units();
  if (cus <= 0) cus = 256;  // without a device: the MI355X's
  const int splits = a.total_k > 0 ? dkv_splits(a, cus) : 1;
  dq_tiles(a, a.group);
  *bytes = 2 * stats_bytes(a) + bound_bytes(a, a.hk) + (splits > 1 ? splits * 2 * a.total_k * a.hk * a.dim * 4 : 0);
  return HI3D_OK;
}

int hi3d_attention_backward(const hi3d_attention_desc* d, const void* out, const float* lse, const void* dout,
                            const float* dlse, void* dq, void* dk, void* dv, void* workspace, int64_t workspace_bytes,
                            void* stream_) {
  AttnArgs a;
  int64_t need = 0;
  int rc = attention_args(d, a);
  if (rc == HI3D_OK) rc = hi3d_attention_backward_workspace(d, &need);
  if (rc != HI3D_OK) return rc;
  HI3D_REQUIRE((dk == nullptr) == (dv == nullptr), "dk and dv are formed together");
  HI3D_REQUIRE(a.hq <= 65536 && (a.group - 1) * a.q_h < (1ll << 29) && a.q_h >= 0,
               "the query heads of one key head must lie within 2^29 elements");
  if ((a.total_q == 0 && a.total_k == 0) || (dq == nullptr && dk == nullptr)) return HI3D_OK;
  HI3D_REQUIRE(a.batch > 0, "rows without a segment");
  if (a.total_q > 0) HI3D_REQUIRE(out != nullptr && lse != nullptr && dout != nullptr, "null pointer argument");
  const uintptr_t at = reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(dq) |
                       reinterpret_cast<uintptr_t>(dk) | reinterpret_cast<uintptr_t>(dv) |
                       reinterpret_cast<uintptr_t>(workspace);
  HI3D_REQUIRE(at % 16 == 0, "out, dout, the gradients and the workspace must be 16-byte aligned");
  HI3D_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), "workspace too small (%lld bytes, need %lld)",
               static_cast<long long>(workspace_bytes), static_cast<long long>(need));
  const int cus = compute_units();
  HI3D_REQUIRE(cus > 0, "cannot query the compute unit count");
  a.o = out, a.lse = const_cast<float*>(lse), a.dout = dout, a.dlse = dlse;
  a.out = dq, a.dk = dk, a.dv = dv;
  a.lse2 = static_cast<float*>(workspace);
  a.delta = reinterpret_cast<float*>(static_cast<char*>(workspace) + stats_bytes(a));
  dq_tiles(a, a.group);
  a.bound = reinterpret_cast<float*>(static_cast<char*>(workspace) + 2 * stats_bytes(a));
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + 2 * stats_bytes(a) + bound_bytes(a, a.hk));
  a.splits = a.total_k > 0 ? dkv_splits(a, cus) : 1;
  hipStream_t stream = as_stream(stream_);
  return d->dtype == HI3D_F16 ? launch_grad_type<_Float16, 0>(a, stream) : launch_grad_type<__bf16, 0>(a, stream);
}

}  // extern "C"
