// Gradients of attention (attention.hip). With D_i = sum_d dout_id out_id - dlse_i and
// p_ij = exp(scale q_i k_j - lse_i), recomputed from q, k and the forward's lse:
//   dv_j = sum_i p_ij dout_i          dp_ij = dout_i v_j       ds_ij = p_ij (dp_ij - D_i)
//   dq_i = scale sum_j ds_ij k_j      dk_j = scale sum_i ds_ij q_i
// Two kernels, each of which owns what it sums, so nothing is added by atomics and the bits
// are the same every time: dq by query rows (it also forms D), then dk and dv by key rows.
// Scores and dp are formed in both: 7 products for 5, against fp32 atomics on dq.
//
// p and ds are rounded once to the inputs' type for their products. fp16 holds 2^-24 to
// 2^16, and a loss's gradients over long rows (p near 1 / keys) would sink below that, so in
// fp16 both are scaled by powers of two that come out again in fp32 at the end: p by 2^10,
// ds so that 8 to 16 stands for the largest sum_d |dout_d| of the rows that are summed
// (|ds| <= p (1 - p) 2 sum |dout| max |v|: it cannot overflow below |v| = 8190). bf16 has
// fp32's range and takes no scale.
#include <type_traits>

#include "attention.h"

namespace hi3d {

int attention_args(const hi3d_attention_desc* d, AttnArgs& a);

namespace {

// 32 owned rows of a wave as second operands (lane l: row l % 32, chunks 2 k + l / 32).
template <int DP>
__device__ __forceinline__ void load_owned(const char* src, int dim, int h, bool on, u32x4 (&x)[DP / 16]) {
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) {
    const int c = 16 * k + 8 * h;
    u32x4 v = {0, 0, 0, 0};
    if (on && c < dim) v = *reinterpret_cast<const u32x4*>(src + c * 2);
    x[k] = v;
  }
}

template <typename T, int DP>
__device__ __forceinline__ void store_owned(T* to, int dim, int h, const f32x16 (&acc)[DP / 32], float by, bool zero) {
  typedef T t4 __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = 32 * d + 8 * e + 4 * h;
      t4 x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = static_cast<T>(zero ? 0.0f : acc[d][4 * e + j] * by);
      if (c < dim) *reinterpret_cast<t4*>(to + c) = x;
    }
}

template <typename T>
constexpr float kPLog2 = std::is_same_v<T, _Float16> ? 10.0f : 0.0f;

// Exponent of the scale of ds for rows whose sum |dout| is at most `bound`.
template <typename T>
__device__ __forceinline__ int ds_exponent(float bound) {
  if constexpr (!std::is_same_v<T, _Float16>) return 0;
  if (!(bound > 0.0f && bound < INFINITY)) return 0;
  const int e = 4 - __builtin_amdgcn_frexp_expf(bound);
  return e < -64 ? -64 : (e > 64 ? 64 : e);
}
__device__ __forceinline__ float power_of_two(int e) { return __builtin_amdgcn_ldexpf(1.0f, e); }

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}

// D from the forward's output carries that output's rounding (p's and its own), which for a
// row of few keys is as large as the rounding of ds: sum_j ds_ij, which is zero, misses by
// just that. Rows that see at most 4 tiles of keys take one walk more to find and mend it:
// gradients of 16 to 128 causal keys come from 1.7-1.55 times the error of a single rounding
// down to 1.42 (sqrt 2); above that many keys the miss is below a tenth of ds's rounding.
constexpr int kExactTiles = 4;

// dq and D. A workgroup owns NW * 32 packed query rows of one key head (queries and
// dout in registers) and walks the keys in tiles of 64 held twice in LDS, as the forward
// does. Per 32 keys a wave forms S^T = K Q^T and dP^T = V dO^T, then dq += K^T dS^T with
// the same K tile read transposed.
//
// One block of 32 rows a wave: two (half the LDS reads) leave fewer waves a SIMD and ran at
// lower speed (64 values a head: 294 us for 271). Bound by each wave's chain of products
// and vector operations, which 2 or 3 waves a SIMD overlap in part: 8,191 rows x 33 heads x 64
// fp16 in four segments 264 us (805 TFLOP/s of its 3 products), 8,192 causal x 32/8 heads x 128
// bf16 414 us (995).
template <typename T, int DP, int NW, bool Z>
__global__ __launch_bounds__(64 * NW, 2) void attend_dq_kernel(AttnArgs a) {
  constexpr int ROWS = NW * 32, KS = DP / 16, DB = DP / 32, PAIR = 2 * kTile<DP>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c32 = lane & 31, h = lane >> 5;
  const TileLane place_of = tile_lane<DP>(lane);
  float* bias = reinterpret_cast<float*>(smem + 2 * PAIR);
  const int64_t id = xcd_remap(blockIdx.x, gridDim.x);
  int head, slot;
  if (a.head_minor) head = static_cast<int>(id % a.hk), slot = static_cast<int>(id / a.hk);
  else slot = static_cast<int>(id % a.slots), head = static_cast<int>(id / a.slots);
  if (a.causal) slot = a.slots - 1 - slot;  // the longest rows first
  Segment s;
  find_segment(a.cu_q, a.len_q, a.batch, a.total_q, a.group, ROWS, slot, s);
  segment_rows(a, s);
  const int rows = s.lq * a.group, row0 = s.tile * ROWS;
  const int wrow = row0 + wave * 32;
  float* bound = a.bound + (static_cast<int64_t>(head) * a.slots + slot) * NW + wave;
  if (s.tile < 0 || row0 >= rows) return;

  const int off = s.lk - s.lq;
  // place of this lane's row among [total_q, hq]
  auto row_at = [&]() -> int64_t {
    int i, g;
    split_row(a, min(wrow + (fresh_lane() & 31), rows - 1), i, g);
    return (s.q0 + i) * a.hq + head * a.group + g;
  };
  u32x4 qf[KS], df[KS];
  int qi, qg;
  split_row(a, min(wrow + c32, rows - 1), qi, qg);
  const int64_t at = (s.q0 + qi) * a.hq + head * a.group + qg;
  const T* src = static_cast<const T*>(a.q) + s.b * a.q_b + (a.cu_q != nullptr ? s.q0 + qi : qi) * a.q_n +
                 static_cast<int64_t>(head * a.group + qg) * a.q_h;
  load_owned<DP>(reinterpret_cast<const char*>(src), a.dim, h, true, qf);
  load_owned<DP>(reinterpret_cast<const char*>(static_cast<const T*>(a.dout) + at * a.dim), a.dim, h, true, df);
  u32x4 of[KS];
  load_owned<DP>(reinterpret_cast<const char*>(static_cast<const T*>(a.o) + at * a.dim), a.dim, h, true, of);
  float x = 0.0f, y = 0.0f;
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    const auto u = __builtin_bit_cast(typename Vec8<T>::type, df[k]), v = __builtin_bit_cast(typename Vec8<T>::type, of[k]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x = __builtin_fmaf(static_cast<float>(u[e]), static_cast<float>(v[e]), x);
      y += __builtin_fabsf(static_cast<float>(u[e]));
    }
  }
  float delta = half_sum(x), size = half_sum(y);  // D, sum |dout|
  if (a.dlse != nullptr) {
    const float z = a.dlse[at];
    delta -= z, size = fmaxf(size, __builtin_fabsf(z));
  }
  const float lse = a.lse[at];
  const bool none = lse == -INFINITY;  // a row that sees no key: all its scores are hidden
  const float ref = (none ? 0.0f : lse * kLog2e) - kPLog2<T>;  // log2 of the scaled p's divisor
  if constexpr (std::is_same_v<T, _Float16>) {  // (a row repeated past the end changes no maximum)
    const float x = wave_max(size);
    if (lane == 0) *bound = wrow < rows ? x : 0.0f;
  }
  const int exponent = ds_exponent<T>(size);
  const float by = power_of_two(exponent - static_cast<int>(kPLog2<T>));  // of dp - D: the scale of ds without that of p
  delta *= by;
  const float dq_by = a.scale * power_of_two(-exponent);  // takes the scale out of dq
  auto store_stats = [&]() {  // for the rows' part in dk and dv: lse in powers of two, and D
    const int r = wrow + c32;
    const int64_t at = (head * a.total_q + s.q0) * a.group + r;
    if (h == 0 && r < rows) a.lse2[at] = none ? INFINITY : ref, a.delta[at] = none ? 0.0f : delta / by;
  };
  int kend = s.lk, wkend = wrow < rows ? s.lk : 0, wfull = s.lk;  // keys of the workgroup; of the wave; of all its rows
  if (a.causal) {
    int i, g;
    split_row(a, min(rows, row0 + ROWS) - 1, i, g);
    kend = min(kend, i + off + 1);
    if (wrow < rows) {
      split_row(a, min(rows, wrow + 32) - 1, i, g);
      wkend = min(wkend, i + off + 1);
      split_row(a, wrow, i, g);
      wfull = min(wfull, i + off + 1);
    }
  }
  const int tiles = kend > 0 ? (kend + kKT - 1) / kKT : 0;

  const char* kp = reinterpret_cast<const char*>(static_cast<const T*>(a.k) + s.b * a.k_b + head * a.k_h +
                                                 (a.cu_k != nullptr ? s.k0 * a.k_n : 0));
  const char* vp = reinterpret_cast<const char*>(static_cast<const T*>(a.v) + s.b * a.v_b + head * a.v_h +
                                                 (a.cu_k != nullptr ? s.k0 * a.v_n : 0));
  auto key_bits = [&](int t) -> uint64_t {
    const int key = t * kKT + lane;
    bool on = key < s.lk;
    if (Z && a.mask != nullptr) on = on && a.mask[s.k0 + (key < s.lk ? key : 0)] != 0;
    return __ballot(on);
  };
  // rows past the segment repeat the last key, hidden ones the tile's first visible key: their
  // probabilities are zero, and what a hidden key holds cannot reach a product
  auto load = [&](int t, uint64_t bits, int buf) {
    if (Z && bits == 0) return;
    if (Z && wave == 0) store_bias(bias + buf * kKT, bits, fresh_lane());
    const int64_t at = static_cast<int64_t>(t) * kKT;
    const int lane = fresh_lane(), last = s.lk - t * kKT - 1, shown = Z ? __builtin_ctzll(bits) : 0;
    load_pair<DP, NW, Z, false>(kp + at * a.k_n * 2, a.k_n, vp + at * a.v_n * 2, a.v_n, a.dim, smem + buf * PAIR, wave, lane,
                         [&](int row) { return Z ? ((bits >> row) & 1 ? row : shown) : (row < last ? row : last); });
  };

  f32x16 acc[DB];
  float miss;
  // one tile; hide: some keys are hidden from some rows; EXACT: only sums ds
  auto walk = [&](const char* kt, const float* tile_bias, int t, uint64_t bits, bool hide, auto EXACT) {
    const char* vt = kt + kTile<DP>;
#pragma unroll 2
    for (int n = 0; n < 2; ++n) {
      f32x16 sc = {}, dp = {};
      if constexpr (Z) sc = read_bias(tile_bias, n, h);
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const u32x4 x = read_rows<DP>(kt, 32 * n, k, place_of), y = read_rows<DP>(vt, 32 * n, k, place_of);
        Mfma<T>::run(x, qf[k], sc), Mfma<T>::run(y, df[k], dp);
      }
      if (hide) {
        asm volatile("");  // a branch, not 16 selects for every tile
        uint64_t on = bits;
        if (a.causal) {
          int i, g;
          split_row(a, min(wrow + (fresh_lane() & 31), rows - 1), i, g);
          const int seen = i + off + 1 - t * kKT;  // keys of this tile that the row sees
          on &= seen >= 64 ? ~0ull : (seen <= 0 ? 0ull : (1ull << seen) - 1);
        }
        const uint32_t w = static_cast<uint32_t>(on >> (32 * n)) >> (4 * h);
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] = (w >> (8 * (e >> 2) + (e & 3))) & 1 ? sc[e] : -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], a.scale2, -ref));
        dp[e] = p * __builtin_fmaf(dp[e], by, -delta);
      }
      if constexpr (EXACT) {
#pragma unroll
        for (int e = 0; e < 16; ++e) miss += dp[e];
      } else {
        u32x4 pk[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          f32x8 x;
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = dp[8 * k + e];
          pk[k] = pack8<T>(x);
        }
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
          for (int d = 0; d < DB; ++d) {
            const u32x4 x = read_columns<DP>(kt, 32 * n + 16 * k, d, place_of);
            Mfma<T>::run(x, pk[k], acc[d]);
          }
        }
        __builtin_amdgcn_s_setprio(0);
      }
    }
  };
  // one pass over the tiles
  auto pass = [&](auto EXACT) {
    uint64_t bits = key_bits(0), next = 0;
    load(0, bits, 0);
    if (tiles > 1) next = key_bits(1);
    tile_barrier();
    for (int t = 0, buf = 0; t < tiles; ++t, buf ^= 1) {
      if (t + 1 < tiles) load(t + 1, next, buf ^ 1);
      uint64_t after = 0;
      if (t + 2 < tiles) after = key_bits(t + 2);
      if (t * kKT < wkend && (!Z || bits != 0))
        walk(smem + buf * PAIR, bias + buf * kKT, t, bits, (!Z && bits != ~0ull) || (t + 1) * kKT > wfull, EXACT);
      bits = next, next = after;
      tile_barrier();
    }
  };
  if (Z && a.dim < DP) clear_tiles(smem, 2 * PAIR);
  if (tiles > 0 && tiles <= kExactTiles) {
    miss = 0.0f;
    pass(std::true_type{});
    // sum ds was to be dlse
    delta += half_sum(miss) * power_of_two(-static_cast<int>(kPLog2<T>));
    if (a.dlse != nullptr) delta -= a.dlse[row_at()] * by;
  }
  store_stats();
  if (a.out == nullptr) return;  // only D and the bounds are wanted
#pragma unroll
  for (int d = 0; d < DB; ++d) acc[d] = f32x16{};
  if (tiles > 0) pass(std::false_type{});
  if (wrow + c32 >= rows) return;
  store_owned<T, DP>(static_cast<T*>(a.out) + row_at() * a.dim, a.dim, h, acc, dq_by, false);
}

__device__ const float kPastRows[2] = {INFINITY, 0.0f};

// dk and dv. A workgroup owns NW * 32 keys of one key head (keys and values in
// registers) and walks the packed query rows that read the head in tiles of 64 (queries and
// dout, with lse and D of each row) held twice in LDS, so the query heads of a shared key
// head sum in registers. Rows past the segment and rows that saw no key have lse = +infinity:
// their probabilities are zero.
//
// Registers decide: keys, values and both sums take 192 of 256 at 128 values a head, and a
// register spilled into the loop waits, when it is read again, for the tile loads in flight
// (48 of them: 1628 us for 1000; one: 545 for 532). So lse and D go straight to LDS, places are
// formed anew from the lane, at 128 values those in LDS too, for every tile, and masked and
// plain tiles share one path (two paths copied the sums): no register is spilled. The
// same figures as above: 355 us (795 TFLOP/s of its 4 products) and 532 us (1035).
//
// Causal: early keys see the most rows, so their blocks start first, and each block is split
// at least in two, which levels the ends (1008 us to 623, with 25 for the join).
template <typename T, int DP, int NW, bool Z, bool SPLIT>
__global__ __launch_bounds__(64 * NW, DP <= 64 ? 3 : 2) void attend_dkv_kernel(AttnArgs a) {
  constexpr int KEYS = NW * 32, KS = DP / 16, DB = DP / 32, PAIR = 2 * kTile<DP>, CH = DP / 8;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* stats = reinterpret_cast<float*>(smem + 2 * PAIR);  // [2][lse, D][64]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c32 = lane & 31, h = lane >> 5;
  int head, split = 0, slot;
  if (a.causal) {  // slot by slot, so that the first keys, which see the most rows, come first
    const int of = a.hk * a.splits;
    head = blockIdx.x % of, slot = blockIdx.x / of;
    if constexpr (SPLIT) split = head / a.hk, head -= split * a.hk;
  } else {
    const int64_t id = xcd_remap(blockIdx.x, gridDim.x);
    if (a.head_minor) {
      head = static_cast<int>(id % a.hk), slot = static_cast<int>(id / a.hk);
      if constexpr (SPLIT) split = slot % a.splits, slot /= a.splits;
    } else {
      slot = static_cast<int>(id % a.slots), head = static_cast<int>(id / a.slots);
      if constexpr (SPLIT) split = head % a.splits, head /= a.splits;
    }
  }
  Segment s;
  find_segment(a.cu_k, a.len_k, a.batch, a.total_k, 1, KEYS, slot, s);
  segment_rows(a, s);
  const int key0 = s.tile * KEYS;
  if (s.tile < 0 || key0 >= s.room) return;  // keys past those in use get zeros

  const int wkey = key0 + wave * 32;
  const int off = s.lk - s.lq, rows = s.lk > 0 ? s.lq * a.group : 0;
  u32x4 kf[KS], vf[KS];
  const int key = wkey + c32;
  bool on = key < s.lk;
  const int64_t row = (a.cu_k != nullptr ? s.k0 : 0) + (on ? key : 0);
  if (Z && a.mask != nullptr) on = on && a.mask[s.k0 + (on ? key : 0)] != 0;
  load_owned<DP>(reinterpret_cast<const char*>(static_cast<const T*>(a.k) + s.b * a.k_b + row * a.k_n + head * a.k_h),
                 a.dim, h, on, kf);
  load_owned<DP>(reinterpret_cast<const char*>(static_cast<const T*>(a.v) + s.b * a.v_b + row * a.v_n + head * a.v_h),
                 a.dim, h, on, vf);
  // packed rows that see a key of the workgroup, of the wave, and all keys of the wave: i >= key - off
  int first = 0, wfirst = wkey < s.lk ? 0 : rows, wfull = 0;
  if (a.causal) {
    first = min(s.lq, max(0, key0 - off)) * a.group;
    if (wkey < s.lk) wfirst = min(s.lq, max(0, wkey - off)) * a.group;
    wfull = min(s.lq, max(0, wkey + 31 - off)) * a.group;
  }
  const int tiles = key0 < s.lk ? (rows + kKT - 1) / kKT : 0;
  int t0 = first / kKT, t1 = tiles;
  if constexpr (SPLIT) {
    const int per = max(1, (tiles - t0 + a.splits - 1) / a.splits);
    t0 = min(tiles, t0 + split * per), t1 = min(tiles, t0 + per);
  }

  const char* qp = reinterpret_cast<const char*>(static_cast<const T*>(a.q) + s.b * a.q_b +
                                                 (a.cu_q != nullptr ? s.q0 * a.q_n : 0) +
                                                 static_cast<int64_t>(head) * a.group * a.q_h);
  const int64_t row_at = s.q0 * a.hq + head * a.group;  // of lse, D and dout
  const char* dp_ = reinterpret_cast<const char*>(static_cast<const T*>(a.dout) + row_at * a.dim);
  const uint32_t q_row = static_cast<uint32_t>(a.q_n) * 2, q_head = static_cast<uint32_t>(a.q_h) * 2, d_head = a.dim * 2;
  auto load = [&](int t, int buf) {
    int i0, g0;
    split_row(a, t * kKT, i0, g0);  // the tile's first query: offsets from it fit 32 bits
    const int lane = fresh_lane();
    const char *x = qp + i0 * a.q_n * 2, *y = dp_ + static_cast<int64_t>(i0) * a.hq * a.dim * 2;
#pragma unroll
    for (int i = 0; i < CH / NW; ++i) {
      int row, c, qi, qg;
      tile_chunk<DP, NW>(i, wave, lane, row, c);
      if (Z && c * 8 >= a.dim) continue;
      split_row(a, min(t * kKT + row, rows - 1), qi, qg);
      const uint32_t from = qi - i0;
      char* to = smem + buf * PAIR + (wave + i * NW) * kBlock<DP>;
      lds_dma16(x + (from * q_row + qg * q_head + c * 16), to);
      lds_dma16(y + ((from * a.hq + qg) * d_head + c * 16), to + kTile<DP>);
    }
  };
  // the scale of ds of this segment and head, from the bounds that the dq kernel's waves left
  float by = 1.0f, dk_by = a.scale, dv_by = 1.0f;
  if constexpr (std::is_same_v<T, _Float16>) {
    const int64_t slot0 = a.cu_q != nullptr
                              ? s.q0 * a.group / a.dq_rows + s.b + 1
                              : s.b * ((static_cast<int64_t>(a.len_q) * a.group + a.dq_rows - 1) / a.dq_rows);
    const float* bounds = a.bound + (static_cast<int64_t>(head) * a.dq_slots + slot0) * a.dq_waves;
    const int count = (rows + a.dq_rows - 1) / a.dq_rows * a.dq_waves;
    float x = 0.0f;
    for (int j = lane; j < count; j += 64) x = fmaxf(x, bounds[j]);
    const int e = ds_exponent<T>(wave_max(x));
    by = power_of_two(e - static_cast<int>(kPLog2<T>)), dk_by *= power_of_two(-e);
    dv_by = power_of_two(-static_cast<int>(kPLog2<T>));
  }
  // lse and D of a tile's rows, by the first wave; rows past the segment: +infinity and 0
  const int64_t stats_at = (head * a.total_q + s.q0) * a.group;
  auto load_stats = [&](int t, int buf) {
    const int r = t * kKT + fresh_lane();
    float* to = stats + buf * 128;
    lds_dma4(r < rows ? a.lse2 + stats_at + r : &kPastRows[0], reinterpret_cast<char*>(to));
    lds_dma4(r < rows ? a.delta + stats_at + r : &kPastRows[1], reinterpret_cast<char*>(to + 64));
  };
  f32x16 dk[DB] = {}, dv[DB] = {};
  // one tile; hide: some rows do not see some keys
  auto walk = [&](const char* qt, const float* st, int t, bool hide) {
    const TileLane place_of = tile_lane<DP>(DP == 128 ? fresh_lane() : lane);
    const char* dt = qt + kTile<DP>;
#pragma unroll 2
    for (int n = 0; n < 2; ++n) {
      f32x16 sc = {}, dp = {};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const u32x4 x = read_rows<DP>(qt, 32 * n, k, place_of), y = read_rows<DP>(dt, 32 * n, k, place_of);
        Mfma<T>::run(x, kf[k], sc), Mfma<T>::run(y, vf[k], dp);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (hide) {
        asm volatile("");  // a branch, not 16 selects for every tile
        const int l = fresh_lane();  // first packed row that sees the lane's key, from the lane's first on
        const int seen = max(0, wkey + (l & 31) - off) * a.group - t * kKT - 32 * n - 4 * (l >> 5);
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] = seen <= 8 * (e >> 2) + (e & 3) ? sc[e] : -INFINITY;
      }
      u32x4 p[2], ds[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        f32x8 ps, dss;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const f32x4 l4 = *reinterpret_cast<const f32x4*>(st + 32 * n + 16 * k + 8 * g + 4 * h);
          const f32x4 d4 = *reinterpret_cast<const f32x4*>(st + 64 + 32 * n + 16 * k + 8 * g + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at = 8 * k + 4 * g + e;
            const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[at], a.scale2, -l4[e]));
            ps[4 * g + e] = x, dss[4 * g + e] = (x * by) * (dp[at] - d4[e]);
          }
        }
        p[k] = pack8<T>(ps), ds[k] = pack8<T>(dss);
      }
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const u32x4 x = read_columns<DP>(dt, 32 * n + 16 * k, d, place_of), y = read_columns<DP>(qt, 32 * n + 16 * k, d, place_of);
          Mfma<T>::run(x, p[k], dv[d]), Mfma<T>::run(y, ds[k], dk[d]);
        }
      }
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  if (Z && a.dim < DP) clear_tiles(smem, 2 * PAIR);
  if (t0 < t1) {
    load(t0, 0);
    if (wave == 0) load_stats(t0, 0);
  }
  tile_barrier();
  for (int t = t0, buf = 0; t < t1; ++t, buf ^= 1) {
    if (t + 1 < t1) {
      load(t + 1, buf ^ 1);
      if (wave == 0) load_stats(t + 1, buf ^ 1);
    }
    if ((t + 1) * kKT > wfirst) walk(smem + buf * PAIR, stats + buf * 128, t, t * kKT < wfull);
    tile_barrier();
  }
  if (key >= s.room) return;
  const int64_t to = ((s.k0 + key) * a.hk + head) * a.dim;
  if constexpr (SPLIT) {
    const int64_t all = a.total_k * a.hk * a.dim;
    store_owned<float, DP>(a.part + split * 2 * all + to, a.dim, h, dk, dk_by, !on);
    store_owned<float, DP>(a.part + (split * 2 + 1) * all + to, a.dim, h, dv, dv_by, !on);
  } else {
    store_owned<T, DP>(static_cast<T*>(a.dk) + to, a.dim, h, dk, dk_by, !on);
    store_owned<T, DP>(static_cast<T*>(a.dv) + to, a.dim, h, dv, dv_by, !on);
  }
}

// Sums the splits of dk and dv in order; 4 values a thread. 2 splits of 8,192 x 8 x 128: 25 us,
// 5.3 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void attend_dkv_join_kernel(AttnArgs a, int64_t all) {
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (i >= 2 * all) return;
  f32x4 x = {0, 0, 0, 0};
  for (int s = 0; s < a.splits; ++s) x += *reinterpret_cast<const f32x4*>(a.part + s * 2 * all + i);
  typedef T t4 __attribute__((ext_vector_type(4)));
  T* to = i < all ? static_cast<T*>(a.dk) + i : static_cast<T*>(a.dv) + (i - all);
  *reinterpret_cast<t4*>(to) = t4{static_cast<T>(x[0]), static_cast<T>(x[1]), static_cast<T>(x[2]), static_cast<T>(x[3])};
}

template <typename T, int DP, int NW>
int launch_dq(AttnArgs a, hipStream_t stream) {
  constexpr int rows = NW * 32;
  HI3D_REQUIRE(static_cast<int64_t>(a.dq_slots) * a.hk < (1ll << 31), "too many rows for one launch");
  if (rows != a.dq_rows || NW != a.dq_waves) return fail(HI3D_ERR_INVALID, "the tile differs from the workspace's");
  a.slots = a.dq_slots;
  const int64_t blocks = static_cast<int64_t>(a.slots) * a.hk;
  constexpr size_t lds = 4 * kTile<DP>;
  return a.mask != nullptr || a.dim < DP ? launch_tiles<&attend_dq_kernel<T, DP, NW, true>>(a, blocks, 64 * NW, lds + kBiasBytes, stream)
                                         : launch_tiles<&attend_dq_kernel<T, DP, NW, false>>(a, blocks, 64 * NW, lds, stream);
}

template <typename T, int DP, int NW>
int launch_dkv(AttnArgs a, hipStream_t stream) {
  constexpr int keys = NW * 32, threads = 64 * NW;
  constexpr size_t lds = 4 * kTile<DP> + 1024;
  const int64_t per = a.cu_k != nullptr ? packed_slots(a.total_k, 1, keys, a.batch) : ceil_div(a.len_k, keys) * a.batch;
  const int64_t blocks = per * a.hk * a.splits;
  HI3D_REQUIRE(blocks < (1ll << 31), "too many rows for one launch");
  a.slots = static_cast<int>(per);
  const bool z = a.mask != nullptr || a.dim < DP;
  if (a.splits == 1)
    return z ? launch_tiles<&attend_dkv_kernel<T, DP, NW, true, false>>(a, blocks, threads, lds, stream)
             : launch_tiles<&attend_dkv_kernel<T, DP, NW, false, false>>(a, blocks, threads, lds, stream);
  const int rc = z ? launch_tiles<&attend_dkv_kernel<T, DP, NW, true, true>>(a, blocks, threads, lds, stream)
                   : launch_tiles<&attend_dkv_kernel<T, DP, NW, false, true>>(a, blocks, threads, lds, stream);
  if (rc != HI3D_OK) return rc;
  const int64_t all = a.total_k * a.hk * a.dim;
  hipLaunchKernelGGL(attend_dkv_join_kernel<T>, dim3(static_cast<unsigned>(ceil_div(2 * all, 1024))), dim3(256), 0, stream, a,
                     all);
  HI3D_LAUNCH_CHECK();
  return HI3D_OK;
}

template <typename T, int DP>
int launch_grad_dim(const AttnArgs& a, hipStream_t stream) {
  if (a.total_q > 0) {
    int rc = HI3D_OK;
    if (a.dq_waves == 1) rc = launch_dq<T, DP, 1>(a, stream);
    else rc = launch_dq<T, DP, 4>(a, stream);
    if (rc != HI3D_OK) return rc;
  }
  if (a.total_k == 0 || a.dk == nullptr) return HI3D_OK;
  if (ceil_div(a.total_k, a.batch) <= 32) return launch_dkv<T, DP, 1>(a, stream);
  return launch_dkv<T, DP, 4>(a, stream);
}

template <typename T>
int launch_grad_type(const AttnArgs& a, hipStream_t stream) {
  switch ((a.dim + 31) / 32) {
    case 1: return launch_grad_dim<T, 32>(a, stream);
    case 2: return launch_grad_dim<T, 64>(a, stream);
    case 3: return launch_grad_dim<T, 96>(a, stream);
    default: return launch_grad_dim<T, 128>(a, stream);
  }
}

// Splits of the query rows for dk and dv: as many as give every compute unit two workgroups
// (four where causal blocks differ in length), each of at least 4 tiles of the average segment.
int dkv_splits(const AttnArgs& a, int cus) {
  const int64_t average = ceil_div(a.total_k, a.batch), tile = average <= 32 ? 32 : 128;
  const int64_t blocks = a.batch * ceil_div(average, tile) * a.hk;
  const int64_t tiles = ceil_div(ceil_div(a.total_q * a.group, a.batch), kKT);
  int64_t splits = (a.causal ? 4 : 2) * static_cast<int64_t>(cus) * (tile == 32 ? 4 : 1) / (blocks > 0 ? blocks : 1);
  if (splits > tiles / 4) splits = tiles / 4;
  if (splits > 64) splits = 64;
  return splits < 1 ? 1 : static_cast<int>(splits);
}

// Query rows to a workgroup: segments of up to 32 rows on average get a wave each (a larger
// tile would be empty).
void dq_tiles(AttnArgs& a) {
  a.dq_waves = ceil_div(a.total_q * a.group, a.batch) <= 32 ? 1 : 4;
  a.dq_rows = 32 * a.dq_waves;
  a.dq_slots = static_cast<int>(a.cu_q != nullptr ? packed_slots(a.total_q, a.group, a.dq_rows, a.batch)
                                                  : ceil_div(static_cast<int64_t>(a.len_q) * a.group, a.dq_rows) * a.batch);
}

// Workspace: lse and D of the packed rows, the bounds of dout's rows, the parts of dk and dv.
int64_t stats_bytes(const AttnArgs& a) { return align_up(a.total_q * a.hq * 4, 256); }
int64_t bound_bytes(const AttnArgs& a) { return align_up(static_cast<int64_t>(a.hk) * a.dq_slots * a.dq_waves * 4, 256); }

}  // namespace
}  // namespace hi3d

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
  dq_tiles(a);
  *bytes = 2 * stats_bytes(a) + bound_bytes(a) + (splits > 1 ? splits * 2 * a.total_k * a.hk * a.dim * 4 : 0);
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
  dq_tiles(a);
  a.bound = reinterpret_cast<float*>(static_cast<char*>(workspace) + 2 * stats_bytes(a));
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + 2 * stats_bytes(a) + bound_bytes(a));
  a.splits = a.total_k > 0 ? dkv_splits(a, cus) : 1;
  hipStream_t stream = as_stream(stream_);
  return d->dtype == HI3D_F16 ? launch_grad_type<_Float16>(a, stream) : launch_grad_type<__bf16>(a, stream);
}

}  // extern "C"
