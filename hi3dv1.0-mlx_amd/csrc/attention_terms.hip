// Attention with terms beside scale q k (attention_terms.h), and attention over keys that many
// sequences share in front of their own.
#include <algorithm>

#include "attention_forward.h"

namespace hi3d {

int term_args(const hi3d_attention_desc* d, const hi3d_attention_terms* t, TermArgs& a) {
  a = TermArgs{};
  const int rc = attention_args(d, a);
  if (rc != HI3D_OK) return rc;
  HI3D_REQUIRE(t != nullptr, "null terms");
  HI3D_REQUIRE(t->cap == 0.0f || (t->cap >= 1e-6f && t->cap <= 1024.0f), "a cap must be at most 1024 (got %g)", t->cap);
  HI3D_REQUIRE(t->slopes == nullptr || d->scale >= 1e-30f, "scores with slopes need a scale of 1e-30 or more");
  HI3D_REQUIRE(t->prefix == nullptr || d->causal, "keys that all queries see belong to causal segments");
  if (t->bias != nullptr) {
    HI3D_REQUIRE(t->bias_dtype == HI3D_F32 || t->bias_dtype == HI3D_F16 || t->bias_dtype == HI3D_BF16,
                 "the bias must be fp32, fp16 or bf16 (got type %d)", t->bias_dtype);
    HI3D_REQUIRE(t->bucket_map != nullptr, "null pointer argument");
    HI3D_REQUIRE(t->buckets >= 1 && static_cast<int64_t>(t->buckets) * d->heads_q < (1 << 30), "bad number of buckets (%d)",
                 t->buckets);
    HI3D_REQUIRE(t->far >= 0 && t->far <= 1024, "a bias reaches at most 1024 keys (got %d)", t->far);
    a.bias = t->bias, a.map = t->bucket_map, a.bias_type = t->bias_dtype, a.buckets = t->buckets, a.far = t->far;
    a.stride = bias_stride(a.far, kPad, a.group), a.stride_keys = bias_stride(a.far, kPadKeys, a.group);
    HI3D_REQUIRE(static_cast<int64_t>(a.group) * a.stride_keys * 4 <= kMostTermBytes,
                 "a bias that reaches %d keys takes at most %d query heads to a key head (got %d)", a.far,
                 kMostTermBytes / 4 / a.stride_keys, a.group);
  }
  if (t->cap > 0.0f) {
    a.cap2 = t->cap * kLog2e, a.cap_in = 2.0f * kLog2e * d->scale / t->cap;
    HI3D_REQUIRE(a.cap_in < INFINITY, "scale / cap must be a number of fp32 (scale %g, cap %g)", d->scale, t->cap);
  }
  a.per_mul = 1.0f / (t->cap > 0.0f ? 2.0f * a.cap2 : a.scale2);
  a.slopes = t->slopes, a.prefix = t->prefix, a.share = 1;
  return HI3D_OK;
}

namespace {

// Kernel, tile and splits of the key axis. 33 to 64 rows take workgroups of four waves too: two blocks of 32 rows
// a wave spill 30 to 300 registers with terms.
void choose(TermArgs& a, int cus) {
  a.few = few_rows(a.total_q, a.total_k, a.batch, a.hq, a.hk, a.dim, cus, term_bytes<kAll>(a));
  a.splits = attend_splits(a.total_q, a.total_k, a.batch, a.hq, a.hk, a.dim, cus, a.few);
  a.rows = attend_rows(a.total_q, a.batch, a.hq, a.hk, a.dim, cus);
  if (a.rows == 64) a.rows = 128;
}

// Rows whose gradients take what rounding leaves of the output: those of attend_kernel's own rows. Short and
// few rows, and those of which parts are joined, have the backward's walk for it.
bool keeps_rest(const TermArgs& a) { return a.splits == 1 && !a.few && !short_segments<kAll>(a); }

int64_t part_bytes(const TermArgs& a, int splits) { return static_cast<int64_t>(splits) * a.total_q * a.hq * (a.dim + 2) * 4; }

// Attention over shared keys in one launch: all rows over the keys that they share, as one segment, and each
// sequence's rows over its own. Both leave parts of the rows, which are joined. Workgroups of four
// waves in both: where a sequence has few rows three of them only help to load.
struct Halves {
  TermArgs of[2];
  int64_t blocks[2];
};

template <typename T, int DP, bool Z>
__global__ __launch_bounds__(256, DP <= 64 ? 3 : 2) void attend_shared_kernel(Halves p) {
  const int which = blockIdx.x >= p.blocks[0];
  attend_rows_of<T, DP, 4, 1, Z, true, kAll>(p.of[which], blockIdx.x - (which ? p.blocks[0] : 0), p.blocks[which]);
}

// Splits of the keys so that all workgroups, two to a compute unit, walk over about as many keys, and at least
// four tiles.
void choose_halves(const TermArgs& a, const hi3d_attention_shared* s, Halves& p, int cus) {
  TermArgs &shared = p.of[0], &own = p.of[1];
  own = shared = a;
  shared.k = s->k, shared.v = s->v, shared.mask = s->key_mask;
  shared.k_b = shared.v_b = 0, shared.k_n = s->strides[0], shared.k_h = s->strides[1];
  shared.v_n = s->strides[2], shared.v_h = s->strides[3];
  shared.batch = 1, shared.len_q = static_cast<int32_t>(a.total_q), shared.len_k = s->len, shared.total_k = s->len;
  shared.lens_k = nullptr, shared.causal = shared.reverse = 0;
  shared.own_lens = a.lens_k, shared.own_len = a.len_k, shared.per = a.len_q;
  shared.head_minor = s->len <= 512;
  int64_t keys = 0;
  for (TermArgs* x : {&shared, &own}) {
    x->slots = static_cast<int>(ceil_div(static_cast<int64_t>(x->len_q) * x->group, 128) * x->batch);
    keys += static_cast<int64_t>(x->slots) * x->hk * x->len_k;
  }
  const int64_t each = std::max<int64_t>(4 * kKT, ceil_div(keys, 2 * cus));
  for (TermArgs* x : {&shared, &own}) {
    x->splits = static_cast<int>(std::min<int64_t>(128, std::max<int64_t>(1, (x->len_k + each / 2) / each)));
    p.blocks[x == &own] = static_cast<int64_t>(x->slots) * x->hk * x->splits;
  }
}

template <typename T, int DP>
int launch_halves(const Halves& p, hipStream_t stream) {
  const bool z = p.of[0].mask != nullptr || p.of[1].mask != nullptr || p.of[0].dim < DP;
  const int64_t blocks = p.blocks[0] + p.blocks[1];
  HI3D_REQUIRE(blocks < (1ll << 31), "too many rows for one launch");
  const size_t lds = 4 * kTile<DP> + (z ? kBiasBytes : 0) + term_bytes<kAll>(p.of[0]);
  const int rc = z ? launch_tiles<&attend_shared_kernel<T, DP, true>>(p, blocks, 256, lds, stream)
                   : launch_tiles<&attend_shared_kernel<T, DP, false>>(p, blocks, 256, lds, stream);
  if (rc != HI3D_OK) return rc;
  TermArgs all = p.of[0];
  all.splits = p.of[0].splits + p.of[1].splits;
  return launch_join<T>(all, stream);
}

template <typename T>
int launch_shared(const Halves& p, hipStream_t stream) {
  switch ((p.of[0].dim + 31) / 32) {
    case 1: return launch_halves<T, 32>(p, stream);
    case 2: return launch_halves<T, 64>(p, stream);
    case 3: return launch_halves<T, 96>(p, stream);
    default: return launch_halves<T, 128>(p, stream);
  }
}

int shared_args(const hi3d_attention_desc* d, const hi3d_attention_terms* t, const hi3d_attention_shared* s, TermArgs& a) {
  const int rc = term_args(d, t, a);
  if (rc != HI3D_OK) return rc;
  HI3D_REQUIRE(s != nullptr, "null shared keys");
  HI3D_REQUIRE(d->cu_q == nullptr && d->cu_k == nullptr, "shared keys stand in front of sequences of equal room, not of offsets");
  HI3D_REQUIRE(t->prefix == nullptr, "shared keys are seen by all queries as they are");
  HI3D_REQUIRE(s->len >= 0, "bad sizes");
  HI3D_REQUIRE(static_cast<int64_t>(s->len) + d->len_k < (1ll << 31) - kKT,  // places count through both, and to a tile's end
               "shared and own keys of a sequence must be fewer than 2^31 - %d", kKT);
  HI3D_REQUIRE(s->len == 0 || (s->k != nullptr && s->v != nullptr), "null pointer argument");
  HI3D_REQUIRE((reinterpret_cast<uintptr_t>(s->k) | reinterpret_cast<uintptr_t>(s->v)) % 16 == 0,
               "the shared keys and values must be 16-byte aligned");
  for (int i = 0; i < 4; ++i) HI3D_REQUIRE(s->strides[i] % 8 == 0, "strides must be multiples of 8 elements");
  for (int i : {0, 2})
    HI3D_REQUIRE(s->strides[i] >= 0 && s->strides[i] < (1ll << 23), "row strides must be below 2^23 elements");
  return HI3D_OK;
}

}  // namespace
}  // namespace hi3d

using namespace hi3d;

extern "C" {

int hi3d_attention_terms_workspace(const hi3d_attention_desc* d, const hi3d_attention_terms* t, int32_t* rest, int64_t* bytes) {
  TermArgs a;
  const int rc = term_args(d, t, a);
  if (rc != HI3D_OK) return rc;
  HI3D_REQUIRE(bytes != nullptr, "null pointer argument");
  *bytes = 0;
  if (rest != nullptr) *rest = 0;
  if (a.total_q == 0 || a.batch == 0) return HI3D_OK;
  const int cus = compute_units();
  choose(a, cus > 0 ? cus : 256);  // without a device (a size query on a build host): the MI355X's
  if (rest != nullptr) *rest = keeps_rest(a);
  if (a.splits > 1) *bytes = part_bytes(a, a.splits) + 256;
  return HI3D_OK;
}

int hi3d_attention_terms_forward(const hi3d_attention_desc* d, const hi3d_attention_terms* t, void* out, void* rest, float* lse,
                                 void* workspace, int64_t workspace_bytes, void* stream_) {
  TermArgs a;
  const int rc = term_args(d, t, a);
  if (rc != HI3D_OK) return rc;
  if (a.total_q == 0) return HI3D_OK;
  HI3D_REQUIRE(a.batch > 0, "rows without a segment");
  HI3D_REQUIRE(out != nullptr && reinterpret_cast<uintptr_t>(out) % 16 == 0, "out must be 16-byte aligned");
  const int cus = compute_units();
  HI3D_REQUIRE(cus > 0, "cannot query the compute unit count");
  a.out = out, a.rest = rest, a.lse = lse;
  choose(a, cus);
  HI3D_REQUIRE(rest == nullptr || (keeps_rest(a) && reinterpret_cast<uintptr_t>(rest) % 16 == 0),
               "no rest of the output is kept of these rows, or it is not 16-byte aligned");
  if (a.splits > 1) {
    HI3D_REQUIRE(workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 &&
                     workspace_bytes >= part_bytes(a, a.splits),
                 "workspace too small (%lld bytes)", static_cast<long long>(workspace_bytes));
    a.part = static_cast<float*>(workspace);
    a.part_ml = a.part + static_cast<int64_t>(a.splits) * a.total_q * a.hq * a.dim;
  }
  hipStream_t stream = as_stream(stream_);
  if (!a.few && !short_segments<kAll>(a) && a.rows > 32 && a.splits == 1 && one_term(a) != kAll)
    return launch_rows_of_one(a, d->dtype, one_term(a), stream);
  return d->dtype == HI3D_F16 ? launch_attend_type<_Float16, kAll>(a, stream) : launch_attend_type<__bf16, kAll>(a, stream);
}

int hi3d_attention_shared_workspace(const hi3d_attention_desc* d, const hi3d_attention_terms* t,
                                    const hi3d_attention_shared* s, int64_t* bytes) {
  TermArgs a;
  Halves p;
  const int rc = shared_args(d, t, s, a);
  if (rc != HI3D_OK) return rc;
  HI3D_REQUIRE(bytes != nullptr, "null pointer argument");
  *bytes = 0;
  if (a.total_q == 0 || a.batch == 0) return HI3D_OK;
  const int cus = compute_units();
  choose_halves(a, s, p, cus > 0 ? cus : 256);
  *bytes = part_bytes(a, p.of[0].splits + p.of[1].splits) + 256;
  return HI3D_OK;
}

int hi3d_attention_shared_forward(const hi3d_attention_desc* d, const hi3d_attention_terms* t, const hi3d_attention_shared* s,
                                  void* out, float* lse, void* workspace, int64_t workspace_bytes, void* stream_) {
  TermArgs a;
  Halves p;
  const int rc = shared_args(d, t, s, a);
  if (rc != HI3D_OK) return rc;
  if (a.total_q == 0) return HI3D_OK;
  HI3D_REQUIRE(out != nullptr && reinterpret_cast<uintptr_t>(out) % 16 == 0, "out must be 16-byte aligned");
  const int cus = compute_units();
  HI3D_REQUIRE(cus > 0, "cannot query the compute unit count");
  a.out = out, a.lse = lse;
  choose_halves(a, s, p, cus);
  TermArgs &shared = p.of[0], &own = p.of[1];
  const int splits = shared.splits + own.splits;
  HI3D_REQUIRE(workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 &&
                   workspace_bytes >= part_bytes(a, splits),
               "workspace too small (%lld bytes)", static_cast<long long>(workspace_bytes));
  const int64_t rows = a.total_q * a.hq;
  shared.part = static_cast<float*>(workspace);
  shared.part_ml = shared.part + splits * rows * a.dim;
  own.part = shared.part + shared.splits * rows * a.dim;
  own.part_ml = shared.part_ml + shared.splits * rows * 2;
  hipStream_t stream = as_stream(stream_);
  return d->dtype == HI3D_F16 ? launch_shared<_Float16>(p, stream) : launch_shared<__bf16>(p, stream);
}

}  // extern "C"
