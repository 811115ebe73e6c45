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
#pragma once

#include <type_traits>

#include "attention_terms.h"

namespace hi3d {

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

// D from the forward's output carries that output's rounding (p's and its own), which for a
// row of few keys is as large as the rounding of ds: sum_j ds_ij, which is zero, misses by
// just that. Rows that see at most 4 tiles of keys take one walk more to find and mend it:
// gradients of 16 to 128 causal keys come from 1.7-1.55 times the error of a single rounding
// down to 1.42 (sqrt 2); above that many keys the miss is below a tenth of ds's rounding.
// Scores with terms are sharp in rows of many keys too (a cap lets them be, slopes leave few keys). There
// the forward also keeps what its rounding took from the output (TermArgs::rest), which gives D its
// digits, and where it did not the walk is taken for every row: dq and dk of capped scores of
// standard deviation 4 come from 2.0 times the error of a single rounding down to 1.4 (sqrt 2).
constexpr int kExactTiles = 4;

// The bias's gradient, one query head of a wave's 32 rows at consecutive places. ds of 8 keys at a time
// (without the cap's derivative; `unscale` takes its scale out and is 0 for rows that are not there)
// goes to LDS row by row, and each lane sums one relative position down its 8 keys (rows of zeros
// stand in for those outside): rows of 9, so that neither side's accesses share banks. LDS float
// atomics took 175 cycles each here (dq of 8,191 rows x 33 heads x 64: 838 us for 339). Of the 63
// positions that 32 keys give the lower half is complete, and each is written once in a wave's life; the
// upper half waits in `carry` for the next 32 keys. Keys of tiles past `far` only count by their side.
struct BiasSums {
  float carry = 0.0f, far[2] = {0.0f, 0.0f};
  int next = 0;      // place (of sums) of lane 0 in the next 32 keys
  bool open = false;  // carry holds something
};

__device__ __forceinline__ void close_sums(BiasSums& b, float* sums, int lane) {
  if (b.open && lane >= 32 && lane < 63) sums[b.next + lane - 32] = b.carry;
  b.carry = 0.0f, b.open = false;
}

__device__ __forceinline__ void sum_bias(const TermArgs& a, const RowTerms<1>& w, const f32x16& ds, int k0, int n, float unscale,
                                         float* skew, float* sums, BiasSums& b) {
  const bool before = k0 + kKT - 1 - w.first <= -a.far, after = k0 - w.last >= a.far;
  if (before || after) {
    float x = 0.0f;
#pragma unroll
    for (int e = 0; e < 16; ++e) x += ds[e];
    if (before) b.far[0] += x;
    else b.far[1] += x;
    return;
  }
  const int lane = fresh_lane(), c32 = lane & 31, h = lane >> 5;
  const int at = k0 + 32 * n - w.first - 31 + a.far + kPadSums;  // of lane 0's position
  if (b.open && b.next != at) close_sums(b, sums, lane);
  float* to = skew + (7 + c32) * kSkewRow + 4 * h;
  float x = 0.0f;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    asm volatile("" ::: "memory");  // a wave's LDS operations run in order
#pragma unroll
    for (int e = 0; e < 4; ++e) to[e] = ds[4 * g + e] * unscale;
    asm volatile("" ::: "memory");
    const int row = 38 + 8 * g - lane;  // of the lane's first key
    const float* from = skew + min(max(row, 0), 38) * kSkewRow;
    float y = 0.0f, z = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j += 2) y += from[j * (kSkewRow + 1)], z += from[(j + 1) * (kSkewRow + 1)];
    x += row >= 0 && row <= 38 ? y + z : 0.0f;
  }
  asm volatile("" ::: "memory");
  float lo, hi;
  both_halves(b.carry, lo, hi);
  if (lane < 32) sums[at + lane] = x + hi;
  b.carry = x, b.next = at + 32, b.open = true;
}

// A workgroup's sums by relative position for attend_dbias_kernel: those of its waves in order, or zeros.
template <int NW>
__device__ __forceinline__ void write_part(const TermArgs& a, int head, int slot, const float* sums) {
  const int length = sum_length(a.far);
  float* to = a.dbias + (static_cast<int64_t>(head) * a.slots + slot) * length;
  for (int x = threadIdx.x; x < length; x += 64 * NW) {
    float v = 0.0f;
    if (sums != nullptr) {
#pragma unroll
      for (int c = 0; c < NW; ++c) v += sums[c * sum_stride(a.far) + x];
    }
    to[x] = v;
  }
}

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
template <typename T, int DP, int NW, bool Z, int TERMS>
__global__ __launch_bounds__(64 * NW, 2) void attend_dq_kernel(ArgsOf<TERMS> a) {
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
  int key_head = head;
  bool sums = false;  // the bias's gradient is formed too
  if constexpr (TERMS != 0) key_head = head / a.share, sums = has_bias<TERMS>(a) && a.dbias != nullptr;  // rows of one query head (group is 1)
  if (s.tile < 0 || row0 >= rows) {
    if constexpr (TERMS != 0)
      if (sums) write_part<NW>(a, head, slot, nullptr);
    return;
  }

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
  u32x4 of[KS], rest[KS];
  load_owned<DP>(reinterpret_cast<const char*>(static_cast<const T*>(a.o) + at * a.dim), a.dim, h, true, of);
  bool with_rest = false;
  if constexpr (TERMS != 0) {
    with_rest = a.rest != nullptr;
    load_owned<DP>(reinterpret_cast<const char*>(static_cast<const T*>(a.rest) + at * a.dim), a.dim, h, with_rest, rest);
  }
  float x = 0.0f, y = 0.0f, z = 0.0f;
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    const auto u = __builtin_bit_cast(typename Vec8<T>::type, df[k]), v = __builtin_bit_cast(typename Vec8<T>::type, of[k]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x = __builtin_fmaf(static_cast<float>(u[e]), static_cast<float>(v[e]), x);
      y += __builtin_fabsf(static_cast<float>(u[e]));
    }
    if constexpr (TERMS != 0) {
      const auto r = __builtin_bit_cast(typename Vec8<T>::type, rest[k]);
#pragma unroll
      for (int e = 0; e < 8; ++e) z = __builtin_fmaf(static_cast<float>(u[e]), static_cast<float>(r[e]), z);
    }
  }
  if constexpr (TERMS != 0) x = __builtin_fmaf(z, 1.0f / kRest<T>, x);
  float delta = half_sum(x), size = half_sum(y);  // D, sum |dout|
  if (a.dlse != nullptr) {
    const float dlse = a.dlse[at];
    delta -= dlse, size = fmaxf(size, __builtin_fabsf(dlse));
  }
  const float lse = a.lse[at];
  const bool none = lse == -INFINITY;  // a row that sees no key: all its scores are hidden
  const float ref = (none ? 0.0f : lse * kLog2e) - kPLog2<T>;  // log2 of the scaled p's divisor
  if constexpr (std::is_same_v<T, _Float16>) {  // (a row repeated past the end changes no maximum)
    const float x = wave_max(size);
    if (lane == 0) *bound = wrow < rows ? x : 0.0f;
  }
  const int exponent = ds_exponent<T>(size);
  float by = power_of_two(exponent - static_cast<int>(kPLog2<T>));  // of dp - D: the scale of ds without that of p
  if constexpr (TERMS != 0) by *= has_cap<TERMS>(a) ? -4.0f : 1.0f;  // add_terms keeps the cap's derivative times -1/4
  delta *= by;
  const float dq_by = a.scale * power_of_two(-exponent);  // takes the scale out of dq
  auto store_stats = [&]() {  // for the rows' part in dk and dv: lse in powers of two, and D
    const int r = wrow + c32;
    int64_t at = (head * a.total_q + s.q0) * a.group + r;
    if constexpr (TERMS != 0) at = (key_head * a.total_q + s.q0 + r) * a.share + (head - key_head * a.share);
    if (h == 0 && r < rows) a.lse2[at] = none ? INFINITY : ref, a.delta[at] = none ? 0.0f : delta / by;
  };
  const int seen_by_all = first_keys<TERMS>(a, s);
  auto seen_by = [&](int i) { return TERMS ? max(i + off + 1, seen_by_all) : i + off + 1; };
  int kend = s.lk, wkend = wrow < rows ? s.lk : 0, wfull = s.lk;  // keys of the workgroup; of the wave; of all its rows
  if (a.causal) {
    int i, g;
    split_row(a, min(rows, row0 + ROWS) - 1, i, g);
    kend = min(kend, seen_by(i));
    if (wrow < rows) {
      split_row(a, min(rows, wrow + 32) - 1, i, g);
      wkend = min(wkend, seen_by(i));
      split_row(a, wrow, i, g);
      wfull = min(wfull, seen_by(i));
    }
  }
  const int tiles = kend > 0 ? (kend + kKT - 1) / kKT : 0;

  const char* kp = reinterpret_cast<const char*>(static_cast<const T*>(a.k) + s.b * a.k_b + key_head * a.k_h +
                                                 (a.cu_k != nullptr ? s.k0 * a.k_n : 0));
  const char* vp = reinterpret_cast<const char*>(static_cast<const T*>(a.v) + s.b * a.v_b + key_head * a.v_h +
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

  // TERMS: the head's bias in LDS, and behind it each wave's sums of its gradient and room for a tile's part
  RowTerms<1> terms;
  bool capped = false;
  float *table = nullptr, *bias_sums = nullptr, *skew = nullptr;
  BiasSums part;
  if constexpr (TERMS != 0) {
    capped = has_cap<TERMS>(a);
    table = reinterpret_cast<float*>(smem + 2 * PAIR + (Z ? kBiasBytes : 0));
    const int is[1] = {qi}, gs[1] = {0};
    row_terms<1>(a, s, terms, table, head, wrow, rows, is, gs);
    if (has_bias<TERMS>(a)) {  // the barrier in front of the first tile is this loop's too
      stage_bias<kPad>(a, table, a.stride, head, 1, 0, 2 * (a.far + kPad) + 1, threadIdx.x, 64 * NW);
      if (sums) {
        bias_sums = table + a.stride + wave * sum_stride(a.far);
        skew = table + a.stride + NW * sum_stride(a.far) + wave * kSkew;
        for (int x = threadIdx.x; x < NW * (sum_stride(a.far) + kSkew); x += 64 * NW) table[a.stride + x] = 0.0f;
        __syncthreads();  // a wave adds to its sums and writes them also where there is no tile, and others zeroed them
      }
    }
  }
  constexpr bool FOLD = TERMS == kSlopes;
  std::conditional_t<FOLD, SideProduct<T>, char> side;
  if constexpr (FOLD) side.set(terms.slope[0] * a.per_mul, h);
  const float unscale = wrow + c32 < rows ? power_of_two(-exponent) * (capped ? -0.25f : 1.0f) : 0.0f;  // of ds
  f32x16 acc[DB];
  float miss;
  // one tile; hide: some keys are hidden from some rows; EXACT: only sums ds
  auto walk = [&](const char* kt, const float* tile_bias, int t, uint64_t bits, bool hide, auto EXACT) {
    const char* vt = kt + kTile<DP>;
#pragma unroll 2
    for (int n = 0; n < 2; ++n) {
      f32x16 scs[1][1] = {}, dp = {}, bend;
      f32x16& sc = scs[0][0];
      if (Z && !capped) sc = read_bias(tile_bias, n, h);
      bool folded = false;
      if constexpr (FOLD) {
        const bool after = t * kKT >= terms.last;
        folded = side.on && (after || (t + 1) * kKT - 1 <= terms.first);
        // a product with zeros where it does not hold: a branch would copy the scores
        const u32x4 slope = (side.slope ^ (after ? 0x80008000u : 0u)) & (folded ? ~0u : 0u);
        Mfma<T>::run(SideProduct<T>::keys(n, c32, side.down), slope, sc);
      }
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const u32x4 x = read_rows<DP>(kt, 32 * n, k, place_of), y = read_rows<DP>(vt, 32 * n, k, place_of);
        Mfma<T>::run(x, qf[k], sc), Mfma<T>::run(y, df[k], dp);
      }
      float mul = a.scale2, add[1];
      if constexpr (TERMS != 0) mul = add_terms<TERMS, 1, 1, true>(a, terms, scs, t * kKT, n, h, folded, add, &bend);
      const float less = TERMS ? add[0] - ref : -ref;
      if (hide) {
        asm volatile("");  // a branch, not 16 selects for every tile
        uint64_t on = bits;
        if (a.causal) {
          int i, g;
          split_row(a, min(wrow + (fresh_lane() & 31), rows - 1), i, g);
          const int seen = seen_by(i) - t * kKT;  // keys of this tile that the row sees
          on &= seen >= 64 ? ~0ull : (seen <= 0 ? 0ull : (1ull << seen) - 1);
        }
        const uint32_t w = static_cast<uint32_t>(on >> (32 * n)) >> (4 * h);
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] = (w >> (8 * (e >> 2) + (e & 3))) & 1 ? sc[e] : -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], mul, less));
        dp[e] = p * __builtin_fmaf(dp[e], by, -delta);
      }
      if constexpr (EXACT) {
#pragma unroll
        for (int e = 0; e < 16; ++e) miss += dp[e];
      } else {
        if constexpr (TERMS != 0) {
          if (sums) sum_bias(a, terms, dp, t * kKT, n, unscale, skew, bias_sums, part);
          if (capped) {
#pragma unroll
            for (int e = 0; e < 16; ++e) dp[e] *= bend[e];
          }
        }
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
        walk(smem + buf * PAIR, bias + buf * kKT, t, bits, ((!Z || capped) && bits != ~0ull) || (t + 1) * kKT > wfull, EXACT);
      bits = next, next = after;
      tile_barrier();
    }
  };
  if (Z && a.dim < DP) clear_tiles(smem, 2 * PAIR);
  if (tiles > 0 && (tiles <= kExactTiles || (TERMS && !with_rest))) {
    miss = 0.0f;
    pass(std::true_type{});
    // sum ds was to be dlse
    delta += half_sum(miss) * power_of_two(-static_cast<int>(kPLog2<T>));
    if (a.dlse != nullptr) delta -= a.dlse[row_at()] * by;
  }
  store_stats();
  if (a.out == nullptr && !sums) return;  // only D and the bounds are wanted
#pragma unroll
  for (int d = 0; d < DB; ++d) acc[d] = f32x16{};
  if (tiles > 0) pass(std::false_type{});
  if constexpr (TERMS != 0)
    if (sums) {
      close_sums(part, bias_sums, lane);
      asm volatile("" ::: "memory");
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        float x = half_sum(part.far[side] * unscale);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) x += __shfl_xor(x, d);
        if (lane == 0) bias_sums[side * (sum_length(a.far) - 1)] += x;
      }
      __syncthreads();
      write_part<NW>(a, head, slot, table + a.stride);
      if (a.out == nullptr) return;
    }
  if (wrow + c32 >= rows) return;
  store_owned<T, DP>(static_cast<T*>(a.out) + row_at() * a.dim, a.dim, h, acc, dq_by, false);
}

__device__ const float kPastRows[2] = {INFINITY, 0.0f};

// Numbers of a row in LDS beside its queries and dout: lse and D; a constant; its slope and place; where its
// bias stands.
template <int TERMS>
constexpr int kStats = TERMS == 0 || TERMS == kCap ? 2 : (TERMS == kSlopes ? 5 : (TERMS == kBias ? 4 : 6));
template <int TERMS>
constexpr int kBiasAt = kStats<TERMS> - 1;

// What the terms of a score take in the kernel whose lanes own keys, for row r of a tile's 64 (a lane
// each, one wave): a constant; the slope that multiplies the key's number in the workgroup, with
// the side's sign; and for tiles between, the row's place from the workgroup's first key on and where
// its bias stands for that key.
struct TileSides {
  bool before, after, near;  // all keys of the workgroup before / behind all rows of the tile; bias is looked up
  bool left;                 // the bias is that of keys before the row
};
template <int KEYS>
__device__ __forceinline__ TileSides tile_sides(const TermArgs& a, const Segment& s, int key0, int t, int rows) {
  const int off = s.lk - s.lq;
  int i, g;
  split_row(a, t * kKT, i, g);
  const int first = i + off;
  split_row(a, min(t * kKT + kKT, rows) - 1, i, g);
  const int last = i + off;
  const bool left = key0 + KEYS - 1 - first <= -a.far, right = key0 - last >= a.far;
  return {key0 + KEYS - 1 <= first, key0 >= last, !left && !right, left};
}

template <int TERMS, int KEYS>
__device__ __forceinline__ void stage_key_terms(const TermArgs& a, const Segment& s, int key0, int head, int r, int t, int rows,
                                                const float* table, float* to) {
  if (!has_slopes<TERMS>(a) && !has_bias<TERMS>(a)) return;
  const TileSides side = tile_sides<KEYS>(a, s, key0, t, rows);
  int i, g;
  split_row(a, min(r, rows - 1), i, g);
  const int lane = r - t * kKT, place = i + s.lk - s.lq - key0;
  float constant = 0.0f;
  if (has_slopes<TERMS>(a)) {
    const float slope = a.slopes[head * a.group + g] * kLog2e, by = side.before ? slope : -slope;
    if (side.before || side.after) constant = -by * static_cast<float>(place);
    to[kKT + lane] = by;
    to[2 * kKT + lane] = static_cast<float>(place);
  }
  if (has_bias<TERMS>(a)) {
    const float* of = table + g * a.stride_keys;
    if (!side.near) constant += of[side.left ? 0 : 2 * (a.far + kPadKeys)];
    reinterpret_cast<int*>(to)[(kBiasAt<TERMS> - 2) * kKT + lane] = g * a.stride_keys + a.far + kPadKeys - min(max(place, -a.far), a.far + kPadKeys);
  }
  to[lane] = constant;
}

// Adds to scores sc of rows 32 n + 8 (e / 4) + 4 h + e % 4 of the tile and the lane's key `key` of the
// workgroup what the loop over probabilities does not add by itself. Scores in powers of two are then sc *
// mul + base (and, with one bias alone, the row's constant). folded: distances are in the scores
// already. kAll: also takes D from dp, which takes the cap's derivative, times -1/4.
template <int TERMS, int KEYS>
__device__ __forceinline__ void add_key_terms(const TermArgs& a, f32x16& sc, f32x16& dp, const float* st, int key, int n,
                                              const float* table, const TileSides& side, bool folded, float& mul, float& base) {
  typedef int i32x4 __attribute__((ext_vector_type(4)));
  const int from = 32 * n + 4 * (fresh_lane() >> 5);
  mul = a.scale2, base = 0.0f;
  if constexpr (TERMS == kAll) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 d4 = *reinterpret_cast<const f32x4*>(st + kKT + from + 8 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e) dp[4 * g + e] -= d4[e];
      __builtin_amdgcn_sched_barrier(0);  // four numbers in flight: more would cost registers that are not there
    }
    if (a.cap2 > 0.0f) {
      mul = 2.0f * a.cap2, base = a.cap2;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float u = minus_u(a, sc[e]);
        sc[e] = u;
        dp[e] *= __builtin_fmaf(u, u, u);
      }
    }
  }
  const bool slopes = has_slopes<TERMS>(a) && !folded, look_up = has_bias<TERMS>(a) && side.near;
  const bool constants = slopes || (TERMS == kAll && has_bias<TERMS>(a));
  if (!constants && !look_up) return;
  if (constants) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 c4 = *reinterpret_cast<const f32x4*>(st + 2 * kKT + from + 8 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[4 * g + e] = __builtin_fmaf(sc[4 * g + e], mul, c4[e]);
      __builtin_amdgcn_sched_barrier(0);
    }
    mul = 1.0f;
  }
  if (slopes) {
    const float x = static_cast<float>(key);
    if (side.before || side.after) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 s4 = *reinterpret_cast<const f32x4*>(st + 3 * kKT + from + 8 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[4 * g + e] = __builtin_fmaf(s4[e], x, sc[4 * g + e]);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 s4 = *reinterpret_cast<const f32x4*>(st + 3 * kKT + from + 8 * g);
        const f32x4 p4 = *reinterpret_cast<const f32x4*>(st + 4 * kKT + from + 8 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[4 * g + e] = __builtin_fmaf(s4[e], __builtin_fabsf(x - p4[e]), sc[4 * g + e]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  if (look_up) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const i32x4 x4 = *reinterpret_cast<const i32x4*>(st + kBiasAt<TERMS> * kKT + from + 8 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[4 * g + e] = __builtin_fmaf(sc[4 * g + e], mul, table[x4[e] + key]);
    }
    mul = 1.0f;
  }
  __builtin_amdgcn_sched_barrier(0);
}

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
// plain tiles share one path (two paths copied the sums): without terms no register is spilled
// (with them: attention_terms.h). The same figures as above: 355 us (795 TFLOP/s of its 4 products)
// and 532 us (1035).
//
// Causal: early keys see the most rows, so their blocks start first, and where blocks are few enough
// that twice as many are still at most four to a compute unit, their rows are split, which levels the
// ends (8,192 x 32/8 heads x 128, in two: 1008 us to 623, with 25 for the join).
template <typename T, int DP, int NW, bool Z, bool SPLIT, int TERMS>
__global__ __launch_bounds__(64 * NW, DP <= 64 ? 3 : 2) void attend_dkv_kernel(ArgsOf<TERMS> a) {
  constexpr int KEYS = NW * 32, KS = DP / 16, DB = DP / 32, PAIR = 2 * kTile<DP>, CH = DP / 8;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int STATS = kStats<TERMS> * kKT;
  float* stats = reinterpret_cast<float*>(smem + 2 * PAIR);  // [2][lse, D, and what the terms take][64]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c32 = lane & 31, h = lane >> 5;
  // with terms the last of the values' operands is in LDS: 256 registers do not hold it at 128 values a head, and
  // a spilled operand waits for the tile loads in flight when it is read again
  constexpr bool LAST = TERMS != 0 && DP == 128;
  u32x4* last_of = reinterpret_cast<u32x4*>(stats + 2 * STATS) + wave * 64;
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
  if constexpr (LAST) last_of[lane] = vf[KS - 1];
  const int seen_by_all = first_keys<TERMS>(a, s);
  if (a.causal) {
    auto sees = [&](int key) { return TERMS && key < seen_by_all ? 0 : min(s.lq, max(0, key - off)) * a.group; };
    first = sees(key0);
    if (wkey < s.lk) wfirst = sees(wkey);
    wfull = sees(wkey + 31);
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
    const int group = TERMS ? 1 : a.group, heads = TERMS ? a.group : 1;  // rows to a query in the dq kernel, and its heads
    const int64_t slot0 = a.cu_q != nullptr
                              ? s.q0 * group / a.dq_rows + s.b + 1
                              : s.b * ((static_cast<int64_t>(a.len_q) * group + a.dq_rows - 1) / a.dq_rows);
    const int count = (rows / heads + a.dq_rows - 1) / a.dq_rows * a.dq_waves;
    float x = 0.0f;
    for (int of = 0; of < heads; ++of) {
      const float* bounds = a.bound + (static_cast<int64_t>(head * heads + of) * a.dq_slots + slot0) * a.dq_waves;
      for (int j = lane; j < count; j += 64) x = fmaxf(x, bounds[j]);
    }
    const int e = ds_exponent<T>(wave_max(x));
    by = power_of_two(e - static_cast<int>(kPLog2<T>)), dk_by *= power_of_two(-e);
    dv_by = power_of_two(-static_cast<int>(kPLog2<T>));
  }
  float* table = stats + 2 * STATS + (LAST ? NW * 256 : 0);
  if constexpr (TERMS != 0)
    if (has_bias<TERMS>(a)) {
      stage_bias<kPadKeys>(a, table, a.stride_keys, head * a.group, a.group, 0, 2 * (a.far + kPadKeys) + 1, threadIdx.x,
                           64 * NW);
      __syncthreads();
    }
  // lse and D of a tile's rows, by the first wave; rows past the segment: +infinity and 0
  const int64_t stats_at = (head * a.total_q + s.q0) * a.group;
  auto load_stats = [&](int t, int buf) {
    const int r = t * kKT + fresh_lane();
    float* to = stats + buf * STATS;
    if constexpr (TERMS != 0) stage_key_terms<TERMS, KEYS>(a, s, key0, head, r, t, rows, table, to + 2 * kKT);
    lds_dma4(r < rows ? a.lse2 + stats_at + r : &kPastRows[0], reinterpret_cast<char*>(to));
    lds_dma4(r < rows ? a.delta + stats_at + r : &kPastRows[1], reinterpret_cast<char*>(to + 64));
  };
  constexpr bool FOLD = TERMS == kSlopes;
  bool folds = false;
  float down = 1.0f;
  u32x4* side_at = reinterpret_cast<u32x4*>(table);  // [2][64], no bias then
  if constexpr (FOLD) {
    float t[2];
    int i[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {  // every wave the same
      const int r = 32 * n + c32;
      i[n] = r / a.group;
      t[n] = a.slopes[head * a.group + r - i[n] * a.group] * kLog2e * a.per_mul;
    }
    const float most = wave_max(fmaxf(__builtin_fabsf(t[0]), __builtin_fabsf(t[1])));
    folds = 64 % a.group == 0 && !(most > 1000.0f);
    const float up = SideProduct<T>::upwards(most);
    down = 1.0f / up;
#pragma unroll
    for (int n = 0; n < 2; ++n)  // zeros: infinity times zero is not
      side_at[n * 64 + lane] = folds ? SideProduct<T>::of_row(t[n] * up, i[n], h) : u32x4{0, 0, 0, 0};
  }
  if constexpr (TERMS != 0) by *= has_cap<TERMS>(a) ? -4.0f : 1.0f;  // the cap's derivative comes times -1/4
  f32x16 dk[DB] = {}, dv[DB] = {};
  // a hidden score; with a cap a finite one, of which a derivative can be formed, whose exponential is zero all the same
  // (1e-6 * 1e9 are far more powers of two than there are)
  constexpr float hidden = TERMS == kCap ? -1e9f : -INFINITY;
  // one tile; hide: some rows do not see some keys
  auto walk = [&](const char* qt, const float* st, int t, bool hide) {
    const TileLane place_of = tile_lane<DP>(DP == 128 || TERMS ? fresh_lane() : lane);
    const char* dt = qt + kTile<DP>;
    TileSides side = {};
    bool folded = false;
    int distance = 0;  // of the segment's first key to the tile's first row
    if constexpr (TERMS != 0) {
      if (has_slopes<TERMS>(a) || has_bias<TERMS>(a)) side = tile_sides<KEYS>(a, s, key0, t, rows);
      if constexpr (FOLD) {
        distance = -(t * kKT / a.group + off);
        folded = folds && (side.before || side.after) && max(abs(distance + key0), abs(distance + key0 + KEYS)) <= SideProduct<T>::kFarthest;
      }
    }
#pragma unroll 2
    for (int n = 0; n < 2; ++n) {
      f32x16 sc = {}, dp = {};
      if constexpr (FOLD) {  // a product with zeros where it does not hold: a branch would copy the scores
        const int l = fresh_lane();
        const u32x4 far = SideProduct<T>::of_key(distance + wkey + (l & 31), l >> 5, down) ^ (side.after ? 0x80008000u : 0u);
        Mfma<T>::run(side_at[n * 64 + l], far & (folded ? ~0u : 0u), sc);
      }
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const u32x4 x = read_rows<DP>(qt, 32 * n, k, place_of), y = read_rows<DP>(dt, 32 * n, k, place_of);
        Mfma<T>::run(x, kf[k], sc), Mfma<T>::run(y, LAST && k == KS - 1 ? last_of[fresh_lane()] : vf[k], dp);
      }
      __builtin_amdgcn_sched_barrier(0);
      float mul = a.scale2, base = 0.0f;  // scores in powers of two are sc * mul + base
      if constexpr (TERMS == kCap) {
        mul = 2.0f * a.cap2, base = a.cap2;
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] = minus_u(a, sc[e]);
      } else if constexpr (TERMS != 0)
        add_key_terms<TERMS, KEYS>(a, sc, dp, st, wkey - key0 + (fresh_lane() & 31), n, table, side, folded, mul, base);
      if (hide) {
        asm volatile("");  // a branch, not 16 selects for every tile
        const int l = fresh_lane();  // first packed row that sees the lane's key, from the lane's first on
        const int key = wkey + (l & 31), row = TERMS && key < seen_by_all ? 0 : max(0, key - off) * a.group;
        const int seen = row - t * kKT - 32 * n - 4 * (l >> 5);
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] = seen <= 8 * (e >> 2) + (e & 3) ? sc[e] : hidden;
        if constexpr (TERMS == kCap) {  // and dp is D there: (1e9)^2 times a difference can pass fp32's range
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f32x4 d4 = *reinterpret_cast<const f32x4*>(st + kKT + 32 * n + 4 * (l >> 5) + 8 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) dp[4 * g + e] = seen <= 8 * g + e ? dp[4 * g + e] : d4[e];
          }
        }
      }
      u32x4 p[2], ds[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        f32x8 ps, dss;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const f32x4 l4 = *reinterpret_cast<const f32x4*>(st + 32 * n + 16 * k + 8 * g + 4 * h);
          f32x4 d4 = {0, 0, 0, 0}, c4 = {0, 0, 0, 0};
          if constexpr (TERMS != kAll) d4 = *reinterpret_cast<const f32x4*>(st + 64 + 32 * n + 16 * k + 8 * g + 4 * h);
          if constexpr (TERMS == kBias) c4 = *reinterpret_cast<const f32x4*>(st + 128 + 32 * n + 16 * k + 8 * g + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at = 8 * k + 4 * g + e;
            const float score = sc[at];
            float less = -l4[e], by_ds = dp[at];
            if constexpr (TERMS == kBias) less = c4[e] - l4[e];
            else if constexpr (TERMS != 0 && TERMS != kSlopes) less = base - l4[e];
            if constexpr (TERMS != kAll) by_ds -= d4[e];
            if constexpr (TERMS == kCap) by_ds *= __builtin_fmaf(score, score, score);  // -1/4 of the cap's derivative
            const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(score, mul, less));
            ps[4 * g + e] = x, dss[4 * g + e] = (x * by) * by_ds;
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
    if ((t + 1) * kKT > wfirst) walk(smem + buf * PAIR, stats + buf * STATS, t, t * kKT < wfull);
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

// Sums `count` parts of the bias's gradient in runs of `run`, [heads, count, length] to [heads, runs,
// length]: four threads take every fourth part of a run each, and are summed in order.
__global__ __launch_bounds__(256) void attend_dbias_sum_kernel(const float* from, float* to, int length, int64_t count, int run) {
  __shared__ float quarter[4][64];
  const int x = blockIdx.x * 64 + (threadIdx.x & 63), of = threadIdx.x >> 6;
  const int64_t head = blockIdx.z, first = static_cast<int64_t>(blockIdx.y) * run;
  const int64_t end = first + run < count ? first + run : count;
  float v = 0.0f;
  if (x < length)
#pragma unroll 8
    for (int64_t i = first + of; i < end; i += 4) v += from[(head * count + i) * length + x];
  quarter[of][threadIdx.x & 63] = v;
  __syncthreads();
  if (of == 0 && x < length) {
    const int l = threadIdx.x;
    to[(head * gridDim.y + blockIdx.y) * length + x] = (quarter[0][l] + quarter[1][l]) + (quarter[2][l] + quarter[3][l]);
  }
}

// A workgroup a head sums what is left by relative position, then each wave eight buckets at a time: a
// lane takes every 64th place, and the lanes' sums are joined in a fixed order.
__global__ __launch_bounds__(256) void attend_dbias_kernel(TermArgs a, const float* parts, int64_t count, void* out) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* total = reinterpret_cast<float*>(smem);
  const int length = sum_length(a.far), head = blockIdx.x;
  int* bucket = reinterpret_cast<int*>(total + length);
  for (int x = threadIdx.x; x < length; x += 256) {
    float v = 0.0f;
#pragma unroll 16
    for (int64_t i = 0; i < count; ++i) v += parts[(head * count + i) * length + x];
    total[x] = v, bucket[x] = bucket_at(a, x, kPadSums);
  }
  __syncthreads();
  const int lane = threadIdx.x & 63;
  for (int first = (threadIdx.x >> 6) * 8; first < a.buckets; first += 32) {  // a wave's eight buckets
    float v[8] = {};
    for (int x = lane; x < length; x += 64) {
      const int b = bucket[x] - first;
      const float add = total[x];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += b == j ? add : 0.0f;
    }
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float x = half_sum(v[j]);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) x += __shfl_xor(x, d);
      sum = lane == j ? x : sum;
    }
    if (lane >= 8 || first + lane >= a.buckets) continue;
    const int64_t at = static_cast<int64_t>(first + lane) * a.hq + head;
    if (a.bias_type == HI3D_F32) static_cast<float*>(out)[at] = sum;
    else if (a.bias_type == HI3D_F16) static_cast<_Float16*>(out)[at] = static_cast<_Float16>(sum);
    else static_cast<__bf16*>(out)[at] = static_cast<__bf16>(sum);
  }
}

template <typename T, int DP, int NW, int TERMS>
int launch_dq(ArgsOf<TERMS> a, hipStream_t stream) {
  constexpr int rows = NW * 32;
  HI3D_REQUIRE(static_cast<int64_t>(a.dq_slots) * a.hk < (1ll << 31), "too many rows for one launch");
  if (rows != a.dq_rows || NW != a.dq_waves) return fail(HI3D_ERR_INVALID, "the tile differs from the workspace's");
  a.slots = a.dq_slots;
  const int64_t blocks = static_cast<int64_t>(a.slots) * a.hk;
  size_t lds = 4 * kTile<DP>;
  if constexpr (TERMS != 0) lds += term_bytes<kAll>(a) + (a.dbias != nullptr ? NW * (sum_stride(a.far) + kSkew) * 4 : 0);
  return a.mask != nullptr || a.dim < DP
             ? launch_tiles<&attend_dq_kernel<T, DP, NW, true, TERMS>>(a, blocks, 64 * NW, lds + kBiasBytes, stream)
             : launch_tiles<&attend_dq_kernel<T, DP, NW, false, TERMS>>(a, blocks, 64 * NW, lds, stream);
}

template <typename T, int DP, int NW, int TERMS>
int launch_dkv(ArgsOf<TERMS> a, hipStream_t stream) {
  constexpr int keys = NW * 32, threads = 64 * NW;
  size_t lds = 4 * kTile<DP> + kStats<TERMS> * kKT * 8 + (TERMS != 0 && DP == 128 ? threads * 16 : 0);
  if constexpr (TERMS == kSlopes) lds += 2048;
  else if constexpr (TERMS != 0) lds += a.bias != nullptr ? a.group * a.stride_keys * 4 : 0;
  const int64_t per = a.cu_k != nullptr ? packed_slots(a.total_k, 1, keys, a.batch) : ceil_div(a.len_k, keys) * a.batch;
  const int64_t blocks = per * a.hk * a.splits;
  HI3D_REQUIRE(blocks < (1ll << 31), "too many rows for one launch");
  a.slots = static_cast<int>(per);
  const bool z = a.mask != nullptr || a.dim < DP;
  if (a.splits == 1)
    return z ? launch_tiles<&attend_dkv_kernel<T, DP, NW, true, false, TERMS>>(a, blocks, threads, lds, stream)
             : launch_tiles<&attend_dkv_kernel<T, DP, NW, false, false, TERMS>>(a, blocks, threads, lds, stream);
  const int rc = z ? launch_tiles<&attend_dkv_kernel<T, DP, NW, true, true, TERMS>>(a, blocks, threads, lds, stream)
                   : launch_tiles<&attend_dkv_kernel<T, DP, NW, false, true, TERMS>>(a, blocks, threads, lds, stream);
  if (rc != HI3D_OK) return rc;
  const int64_t all = a.total_k * a.hk * a.dim;
  hipLaunchKernelGGL(attend_dkv_join_kernel<T>, dim3(static_cast<unsigned>(ceil_div(2 * all, 1024))), dim3(256), 0, stream, a,
                     all);
  HI3D_LAUNCH_CHECK();
  return HI3D_OK;
}

// WIDE: workgroups of four waves only.
template <typename T, int DP, int TERMS, bool WIDE>
int launch_dq_dim(const ArgsOf<TERMS>& a, hipStream_t stream) {
  if constexpr (!WIDE)
    if (a.dq_waves == 1) return launch_dq<T, DP, 1, TERMS>(a, stream);
  return launch_dq<T, DP, 4, TERMS>(a, stream);
}

template <typename T, int DP, int TERMS, bool WIDE>
int launch_grad_dim(const ArgsOf<TERMS>& a, hipStream_t stream) {
  if (a.total_q > 0) {
    int rc = HI3D_OK;
    if constexpr (TERMS != 0) {  // rows of one query head to a workgroup: one bias in LDS, with its sums
      TermArgs b = a;
      b.share = a.group, b.hk = a.hq, b.group = 1, b.stride = 2 * (a.far + kPad) + 4;
      rc = launch_dq_dim<T, DP, TERMS, WIDE>(b, stream);
    } else {
      rc = launch_dq_dim<T, DP, 0, WIDE>(a, stream);
    }
    if (rc != HI3D_OK) return rc;
  }
  if (a.total_k == 0 || a.dk == nullptr) return HI3D_OK;
  if constexpr (!WIDE)
    if (ceil_div(a.total_k, a.batch) <= 32) return launch_dkv<T, DP, 1, TERMS>(a, stream);
  return launch_dkv<T, DP, 4, TERMS>(a, stream);
}

template <typename T, int TERMS, bool WIDE = false>
int launch_grad_type(const ArgsOf<TERMS>& a, hipStream_t stream) {
  switch ((a.dim + 31) / 32) {
    case 1: return launch_grad_dim<T, 32, TERMS, WIDE>(a, stream);
    case 2: return launch_grad_dim<T, 64, TERMS, WIDE>(a, stream);
    case 3: return launch_grad_dim<T, 96, TERMS, WIDE>(a, stream);
    default: return launch_grad_dim<T, 128, TERMS, WIDE>(a, stream);
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
// `group`: rows to a query.
void dq_tiles(AttnArgs& a, int group) {
  a.dq_waves = ceil_div(a.total_q * group, a.batch) <= 32 ? 1 : 4;
  a.dq_rows = 32 * a.dq_waves;
  a.dq_slots = static_cast<int>(a.cu_q != nullptr ? packed_slots(a.total_q, group, a.dq_rows, a.batch)
                                                  : ceil_div(static_cast<int64_t>(a.len_q) * group, a.dq_rows) * a.batch);
}

// Workspace: lse and D of the packed rows, the bounds of dout's rows, the parts of dk and dv.
int64_t stats_bytes(const AttnArgs& a) { return align_up(a.total_q * a.hq * 4, 256); }
int64_t bound_bytes(const AttnArgs& a, int heads) {
  return align_up(static_cast<int64_t>(heads) * a.dq_slots * a.dq_waves * 4, 256);
}

}  // namespace
}  // namespace hi3d
