// Attention over packed segments: out = softmax(scale q k^T) v, with grouped heads, a
// causal limit aligned to the last query and key, and a mask of keys.
#include "attention_forward.h"

namespace hi3d {

int attention_args(const hi3d_attention_desc* d, AttnArgs& a) {
  HI3D_REQUIRE(d != nullptr, "null descriptor");
  HI3D_REQUIRE(d->dtype == HI3D_F16 || d->dtype == HI3D_BF16, "attention takes fp16 or bf16 (got type %d)", d->dtype);
  HI3D_REQUIRE(d->dim >= 8 && d->dim <= 128 && d->dim % 8 == 0, "head size must be a multiple of 8 up to 128 (got %d)",
               d->dim);
  HI3D_REQUIRE(d->heads_k > 0 && d->heads_q > 0 && d->heads_q % d->heads_k == 0,
               "%d query heads are no multiple of %d key heads", d->heads_q, d->heads_k);
  HI3D_REQUIRE(d->batch >= 0 && d->total_q >= 0 && d->total_k >= 0, "bad sizes");
  HI3D_REQUIRE(d->total_q < (1ll << 31) && d->total_k < (1ll << 31), "at most 2^31 - 1 rows");
  HI3D_REQUIRE(d->scale > 0.0f && d->scale < INFINITY, "scale must be positive and finite");
  const int group = d->heads_q / d->heads_k;
  HI3D_REQUIRE(group <= 4096 && d->total_q * group < (1ll << 31) / group, "too many rows for this many heads to a key head");
  HI3D_REQUIRE(d->cu_q != nullptr || (d->len_q >= 0 && d->total_q == static_cast<int64_t>(d->batch) * d->len_q),
               "queries: %lld rows are not %d segments of %d", static_cast<long long>(d->total_q), d->batch, d->len_q);
  HI3D_REQUIRE(d->cu_k != nullptr || (d->len_k >= 0 && d->total_k == static_cast<int64_t>(d->batch) * d->len_k),
               "keys: %lld rows are not %d segments of %d", static_cast<long long>(d->total_k), d->batch, d->len_k);
  HI3D_REQUIRE(d->lens_k == nullptr || d->cu_k == nullptr, "lens_k belongs to segments of equal room, not to offsets");
  if (d->total_q > 0) HI3D_REQUIRE(d->q != nullptr, "null pointer argument");
  if (d->total_k > 0) HI3D_REQUIRE(d->k != nullptr && d->v != nullptr, "null pointer argument");
  const uintptr_t at = reinterpret_cast<uintptr_t>(d->q) | reinterpret_cast<uintptr_t>(d->k) | reinterpret_cast<uintptr_t>(d->v);
  HI3D_REQUIRE(at % 16 == 0, "q, k and v must be 16-byte aligned");
  for (int i = 0; i < 9; ++i) HI3D_REQUIRE(d->strides[i] % 8 == 0, "strides must be multiples of 8 elements");
  // 64 rows of a tile are addressed with 32-bit byte offsets
  for (int i : {1, 4, 7})
    HI3D_REQUIRE(d->strides[i] >= 0 && d->strides[i] < (1ll << 23), "row strides must be below 2^23 elements");
  a = AttnArgs{};
  a.q = d->q, a.k = d->k, a.v = d->v;
  a.q_b = d->strides[0], a.q_n = d->strides[1], a.q_h = d->strides[2];
  a.k_b = d->strides[3], a.k_n = d->strides[4], a.k_h = d->strides[5];
  a.v_b = d->strides[6], a.v_n = d->strides[7], a.v_h = d->strides[8];
  if (d->cu_q != nullptr) a.q_b = 0;
  if (d->cu_k != nullptr) a.k_b = a.v_b = 0;
  a.cu_q = d->cu_q, a.cu_k = d->cu_k, a.lens_k = d->lens_k, a.mask = d->key_mask;
  a.batch = d->batch, a.len_q = d->len_q, a.len_k = d->len_k, a.total_q = d->total_q, a.total_k = d->total_k;
  a.hq = d->heads_q, a.hk = d->heads_k, a.group = group, a.dim = d->dim;
  a.group_magic = group > 1 ? static_cast<uint32_t>(((1ull << 32) + group - 1) / group) : 0;
  a.scale = d->scale, a.scale2 = d->scale * kLog2e;
  a.causal = d->causal != 0, a.splits = 1;
  // short segments: the heads of a row share its cache lines, so they run side by side
  a.head_minor = d->batch > 0 && d->total_k / d->batch <= 512;
  a.reverse = a.causal;
  a.once = d->total_k * d->heads_k * d->dim * 4 > (256ll << 20);
  return HI3D_OK;
}

}  // namespace hi3d

using namespace hi3d;

extern "C" {

int hi3d_attention_workspace(const hi3d_attention_desc* d, int64_t* bytes) {
  AttnArgs a;
  const int rc = attention_args(d, a);
  if (rc != HI3D_OK) return rc;
  HI3D_REQUIRE(bytes != nullptr, "null pointer argument");
  *bytes = 0;
  if (a.total_q == 0 || a.batch == 0) return HI3D_OK;
  // without a device (a size query on a build host) the MI355X's 256 compute units
  int cus = compute_units();
  if (cus <= 0) cus = 256;
  const bool few = few_rows(a.total_q, a.total_k, a.batch, a.hq, a.hk, a.dim, cus);
  const int splits = attend_splits(a.total_q, a.total_k, a.batch, a.hq, a.hk, a.dim, cus, few);
  if (splits > 1) *bytes = static_cast<int64_t>(splits) * a.total_q * a.hq * (a.dim + 2) * 4 + 256;
  return HI3D_OK;
}

int hi3d_attention_forward(const hi3d_attention_desc* d, void* out, float* lse, void* workspace,
                           int64_t workspace_bytes, void* stream_) {
  AttnArgs a;
  const int rc = attention_args(d, a);
  if (rc != HI3D_OK) return rc;
  if (a.total_q == 0) return HI3D_OK;
  HI3D_REQUIRE(a.batch > 0, "rows without a segment");
  HI3D_REQUIRE(out != nullptr && reinterpret_cast<uintptr_t>(out) % 16 == 0, "out must be 16-byte aligned");
  const int cus = compute_units();
  HI3D_REQUIRE(cus > 0, "cannot query the compute unit count");
  a.out = out, a.lse = lse;
  a.few = few_rows(a.total_q, a.total_k, a.batch, a.hq, a.hk, a.dim, cus);
  const int splits = attend_splits(a.total_q, a.total_k, a.batch, a.hq, a.hk, a.dim, cus, a.few);
  a.rows = attend_rows(a.total_q, a.batch, a.hq, a.hk, a.dim, cus);
  if (splits > 1) {
    const int64_t row_bytes = a.total_q * a.hq * 4;
    HI3D_REQUIRE(workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 &&
                     workspace_bytes >= splits * row_bytes * (a.dim + 2),
                 "workspace too small (%lld bytes)", static_cast<long long>(workspace_bytes));
    a.splits = splits;
    a.part = static_cast<float*>(workspace);
    a.part_ml = a.part + static_cast<int64_t>(splits) * a.total_q * a.hq * a.dim;
  }
  hipStream_t stream = as_stream(stream_);
  return d->dtype == HI3D_F16 ? launch_attend_type<_Float16, 0>(a, stream) : launch_attend_type<__bf16, 0>(a, stream);
}

}  // extern "C"
