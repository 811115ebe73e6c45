// Forward kernels of attention over packed segments and how their tiles are chosen.
//   out = softmax(s) v with grouped heads, a causal limit aligned to the last query and key, and
//   a mask of keys; s = scale q k^T, or that with the terms of attention_terms.h.
#pragma once

#include <type_traits>

#include "attention_terms.h"

namespace hi3d {
namespace {

// How far below a row's maximum its reference is kept, in powers of two. fp16 holds 2^-24 to
// 2^16: with probabilities of up to 2^7 beside a reference at the maximum, 10^5 keys whose
// scores lie 25 powers of two below it still count (they hold 0.3 % of the row; from a
// reference at the maximum all of it was lost). The quotient and lse take it out again. bf16
// has fp32's range.
template <typename T>
constexpr float kBelow = std::is_same_v<T, _Float16> ? 7.0f : 0.0f;

// Scores of the keys that `bits` leaves out become -infinity.
template <int QW>
__device__ __forceinline__ void hide_keys(f32x16 (&sc)[2][QW], uint64_t bits) {
  if (bits == ~0ull) return;
  asm volatile("");  // a branch, not a select a score in every tile
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const bool on = sees_key(bits, 32 * n + 8 * (e >> 2) + (e & 3));
#pragma unroll
      for (int b = 0; b < QW; ++b) sc[n][b][e] = on ? sc[n][b][e] : -INFINITY;
    }
}

// A workgroup owns NW * QW * 32 packed rows of one key head (QW blocks of 32 per wave,
// their queries in registers) and walks the keys in tiles of 64 held twice in LDS: the
// next tile's loads go straight to LDS while the present one is computed, one barrier per
// tile. Per 64 keys a wave forms S^T = K Q^T, keeps the running reference m and sum of
// exp2(s - m) of its rows in fp32, and adds V^T P^T to the output it holds.
//
// m is kBelow under the row's maximum and only moves when that has grown by more than 2^8 (the
// first tile included): any reference gives the same quotient, and between moves the
// probabilities stay below 2^15, inside fp16's and fp32's range, so the output is rescaled
// rarely. In fp16 a tile's probabilities are summed before they join the row's sum, which
// would round away keys 24 powers of two below the first one by one.
//
// Bound by the two waves of a SIMD sharing its matrix and vector units: per 64 keys and 32
// rows 32 * DP / 128 matrix instructions of 32 cycles, and about 140 vector operations for
// the softmax (32 exponentials of 8 cycles), which at 64 values a head take longer. Matrix
// products run at a higher wave priority, so that the other wave's softmax fills in behind
// them (1.5 % at 64). 20,011 tokens x 33 heads x 64 fp16 in two objects: 1880 us, 900
// TFLOP/s; 16,384 causal x 32/8 heads x 128 bf16: 2045 us, 1075 TFLOP/s.
//
// SPLIT, few rows over many keys: parts of the keys go to workgroups of their own, and their
// outputs and (m, sum) to attend_join_kernel in fp32. One-wave workgroups then read keys and
// values that no other one does; more of them than the chip's 256 MiB of cache go past it, as
// the next token's call would not find them there. Single tokens of 8 sequences over caches of
// up to 65,536 x 8 x 128 bf16 (1.9 GB): 308 us, 6.1 TB/s (326 for 358 through the caches, in
// turn on a slower card); below that size the cache helps (8 x 4,096 keys, 134 MB: 30.8 us for 32.3).
template <typename T, int DP, int NW, int QW, bool Z, bool SPLIT, int TERMS>
__device__ __forceinline__ void attend_rows_of(const ArgsOf<TERMS>& a, int64_t block, int64_t blocks) {
  constexpr int ROWS = NW * QW * 32, KS = DP / 16, DB = DP / 32, PAIR = 2 * kTile<DP>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c32 = lane & 31, h = lane >> 5;
  const TileLane at = tile_lane<DP>(lane);
  float* bias = reinterpret_cast<float*>(smem + 2 * PAIR);

  // task: (head, split, slot), neighbours on one XCD so that they share its L2
  const int64_t id = xcd_remap(block, blocks);
  int head, split = 0, slot;
  if (a.head_minor) {
    head = static_cast<int>(id % a.hk), slot = static_cast<int>(id / a.hk);
    if constexpr (SPLIT) split = slot % a.splits, slot /= a.splits;
  } else {
    slot = static_cast<int>(id % a.slots), head = static_cast<int>(id / a.slots);
    if constexpr (SPLIT) split = head % a.splits, head /= a.splits;
  }
  if (a.reverse) slot = a.slots - 1 - slot;  // causal: the longest rows first
  Segment s;
  find_segment(a.cu_q, a.len_q, a.batch, a.total_q, a.group, ROWS, slot, s);
  segment_rows(a, s);
  const int rows = s.lq * a.group, row0 = s.tile * ROWS;
  if (s.tile < 0 || row0 >= rows) return;

  // this wave's rows and the keys they see
  const int wrow = row0 + wave * (QW * 32);
  const int off = s.lk - s.lq;
  int qi[QW], qg[QW];
  u32x4 qf[QW][KS];
#pragma unroll
  for (int b = 0; b < QW; ++b) {
    const int r = wrow + b * 32 + c32;
    split_row(a, r < rows ? r : rows - 1, qi[b], qg[b]);
    const T* src = static_cast<const T*>(a.q) + s.b * a.q_b + (a.cu_q != nullptr ? s.q0 + qi[b] : qi[b]) * a.q_n +
                   static_cast<int64_t>(head * a.group + qg[b]) * a.q_h;
    if constexpr (TERMS != 0)
      if (a.per > 0) {  // rows of many sequences over what they share
        const int of = qi[b] / a.per;
        src += of * a.q_b - static_cast<int64_t>(of) * a.per * a.q_n;
      }
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int c = 16 * k + 8 * h;
      u32x4 x = {0, 0, 0, 0};
      if (c < a.dim) x = *reinterpret_cast<const u32x4*>(src + c);
      qf[b][k] = x;
    }
  }
  const int seen_by_all = first_keys<TERMS>(a, s);
  auto seen_by = [&](int i) { return TERMS ? max(i + off + 1, seen_by_all) : i + off + 1; };
  int kend = s.lk, wkend = wrow < rows ? s.lk : 0, wfull = s.lk;  // keys of the workgroup; of the wave; of all its rows
  if (a.causal) {
    int i, g;
    split_row(a, min(rows, row0 + ROWS) - 1, i, g);
    kend = min(kend, seen_by(i));
    if (wrow < rows) {
      split_row(a, min(rows, wrow + QW * 32) - 1, i, g);
      wkend = min(wkend, seen_by(i));
      split_row(a, wrow, i, g);
      wfull = min(wfull, seen_by(i));
    }
  }
  const int tiles = kend > 0 ? (kend + kKT - 1) / kKT : 0;
  int t0 = 0, t1 = tiles;
  if constexpr (SPLIT) {
    const int per = (tiles + a.splits - 1) / a.splits;
    t0 = min(tiles, split * per), t1 = min(tiles, t0 + per);
  }

  const char* kp = reinterpret_cast<const char*>(static_cast<const T*>(a.k) + s.b * a.k_b + head * a.k_h +
                                                 (a.cu_k != nullptr ? s.k0 * a.k_n : 0));
  const char* vp = reinterpret_cast<const char*>(static_cast<const T*>(a.v) + s.b * a.v_b + head * a.v_h +
                                                 (a.cu_k != nullptr ? s.k0 * a.v_n : 0));
  // bit j: key 64 t + j is in the segment and not hidden
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
    if (Z && wave == 0) store_bias(bias + buf * kKT, bits, lane);
    const int64_t from = static_cast<int64_t>(t) * kKT;
    const int last = s.lk - t * kKT - 1, shown = Z ? __builtin_ctzll(bits) : 0;
    auto of = [&](int row) { return Z ? ((bits >> row) & 1 ? row : shown) : (row < last ? row : last); };
    const char *x = kp + from * a.k_n * 2, *y = vp + from * a.v_n * 2;
    char* to = smem + buf * PAIR;
    if (SPLIT && NW == 1 && a.once) load_pair<DP, NW, Z, true>(x, a.k_n, y, a.v_n, a.dim, to, wave, lane, of);
    else load_pair<DP, NW, Z, false>(x, a.k_n, y, a.v_n, a.dim, to, wave, lane, of);
  };

  RowTerms<QW> terms;
  bool capped = false;
  if constexpr (TERMS != 0) {
    capped = has_cap<TERMS>(a);
    float* table = reinterpret_cast<float*>(smem + 2 * PAIR + (Z ? kBiasBytes : 0));
    row_terms<QW>(a, s, terms, table, head, wrow, rows, qi, qg);
    if (has_bias<TERMS>(a)) {  // the barrier in front of the first tile is this one's too
      int x0 = 0, x1 = 2 * (a.far + kPad) + 1;
      if (a.per == 0) {  // what the workgroup's rows and keys reach (add_terms reads 64 places from a clamped one on)
        int i, g;
        split_row(a, min(rows, row0 + ROWS) - 1, i, g);
        x0 = min(max(t0 * kKT - (i + off) + a.far + kPad, 0), 2 * a.far + kPad);
        split_row(a, row0, i, g);
        x1 = min(x1, max(t1 * kKT - (i + off) + a.far + kPad, kKT));
      }
      stage_bias<kPad>(a, table, a.stride, head * a.group, a.group, x0, max(x1, x0 + 1), threadIdx.x, 64 * NW);
    }
  }
  f32x16 acc[DB][QW] = {};
  float m[QW], l[QW];
#pragma unroll
  for (int b = 0; b < QW; ++b) m[b] = -INFINITY, l[b] = 0.0f;
  float lr[QW] = {};  // TERMS: sums of the rounded probabilities
  // For gradients the reference stays within a factor of 4 of the maximum: a key that a row hangs on becomes the
  // reference itself, so that its probability rounds without an error and D keeps its digits (dq of capped scores
  // of standard deviation 4: 1.4 times the error of a single rounding, 1.5 with the forward's own factor of 256).
  float slack = 8.0f;
  if constexpr (TERMS != 0) slack = a.rest != nullptr ? 2.0f : 8.0f;
  constexpr bool FOLD = TERMS == kSlopes;
  std::conditional_t<FOLD, SideProduct<T>, char> side;
  bool folds = false;
  if constexpr (FOLD) {  // one for all blocks of a lane's rows, where these have the same head
    side.set(terms.slope[0] * a.per_mul, h);
    folds = side.on && (QW == 1 || 32 % a.group == 0);
  }

  if (Z && a.dim < DP) clear_tiles(smem, 2 * PAIR);
  uint64_t bits = 0, next = 0;
  if (t0 < t1) {
    bits = key_bits(t0);
    load(t0, bits, 0);
    if (t0 + 1 < t1) next = key_bits(t0 + 1);
  }
  tile_barrier();
  for (int t = t0, buf = 0; t < t1; ++t, buf ^= 1) {
    if (t + 1 < t1) load(t + 1, next, buf ^ 1);
    uint64_t after = 0;
    if (t + 2 < t1) after = key_bits(t + 2);
    if (t * kKT < wkend && (!Z || bits != 0)) {
      const char* kt = smem + buf * PAIR;
      const char* vt = kt + kTile<DP>;
      f32x16 sc[2][QW] = {};
      if (Z && !capped) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const f32x16 x = read_bias(bias + buf * kKT, n, h);
#pragma unroll
          for (int b = 0; b < QW; ++b) sc[n][b] = x;
        }
      }
      bool folded = false;
      if constexpr (FOLD) {
        const bool after = t * kKT >= terms.last;
        folded = folds && (after || (t + 1) * kKT - 1 <= terms.first);
        // a product with zeros where it does not hold: a branch would copy the scores
        const uint32_t turn = after ? 0x80008000u : 0u, keep = folded ? ~0u : 0u;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          f32x16 from = sc[n][0];  // zeros, or the masked keys' -infinity, the same in all blocks
          Mfma<T>::run(SideProduct<T>::keys(n, c32, side.down), (side.slope ^ turn) & keep, from);
#pragma unroll
          for (int b = 0; b < QW; ++b) sc[n][b] = from;
        }
      }
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const u32x4 x = read_rows<DP>(kt, 32 * n, k, at);
#pragma unroll
          for (int b = 0; b < QW; ++b) Mfma<T>::run(x, qf[b][k], sc[n][b]);
        }
      float mul = a.scale2, add[QW];  // scores in powers of two are sc * mul (+ add)
      if constexpr (TERMS != 0) mul = add_terms<TERMS, 2, QW, false>(a, terms, sc, t * kKT, 0, h, folded, add, nullptr);
      // keys that are hidden from a row
      if (((!Z || capped) && bits != ~0ull) || (t + 1) * kKT > wfull) {
        if (!Z || capped) hide_keys<QW>(sc, bits);
        if (a.causal) {
          asm volatile("");
#pragma unroll
          for (int b = 0; b < QW; ++b) {
            const int seen = seen_by(qi[b]) - t * kKT - 4 * h;  // keys of this tile that the row sees, from its half's first
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int e = 0; e < 16; ++e)
                sc[n][b][e] = 32 * n + 8 * (e >> 2) + (e & 3) < seen ? sc[n][b][e] : -INFINITY;
          }
        }
      }
      float top[QW];
      bool grow = false;
#pragma unroll
      for (int b = 0; b < QW; ++b) {
        float x = larger(sc[0][b][0], sc[1][b][0]);
#pragma unroll
        for (int e = 1; e < 16; ++e) x = larger(larger(x, sc[0][b][e]), sc[1][b][e]);
        if constexpr (TERMS != 0) top[b] = kept_max(__builtin_fmaf(x, mul, add[b])) - kBelow<T>;
        else top[b] = half_max(x) * a.scale2 - kBelow<T>;
        grow = grow || top[b] > m[b] + slack;
      }
      if (__any(grow)) {
#pragma unroll
        for (int b = 0; b < QW; ++b) {
          const float to = fmaxf(m[b], top[b]);
          const float by = m[b] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[b] - to);
          m[b] = to;
          l[b] *= by;
          if constexpr (TERMS != 0) lr[b] *= by;
#pragma unroll
          for (int d = 0; d < DB; ++d) acc[d][b] *= by;
        }
      }
#pragma unroll
      for (int b = 0; b < QW; ++b) {
        const float ref = m[b] == -INFINITY ? 0.0f : m[b];
        constexpr bool APART = kBelow<T> > 0;  // bf16's own rounding is far coarser than the sum's
        float sum = APART ? 0.0f : l[b];
        const float less = TERMS ? add[b] - ref : -ref;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            sc[n][b][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[n][b][e], mul, less));
            sum += sc[n][b][e];
          }
        l[b] = APART ? l[b] + sum : sum;
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        u32x4 p[QW];
#pragma unroll
        for (int b = 0; b < QW; ++b) {
          f32x8 x;
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = sc[k >> 1][b][8 * (k & 1) + e];
          p[b] = pack8<T>(x);
          if constexpr (TERMS && !SPLIT)
            if (a.rest != nullptr) {
              float pair = 0.0f;
#pragma unroll
              for (int e = 0; e < 4; ++e) pair = add_pair<T>(p[b][e], pair);
              lr[b] += pair;
            }
        }
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const u32x4 x = read_columns<DP>(vt, 16 * k, d, at);
#pragma unroll
          for (int b = 0; b < QW; ++b) Mfma<T>::run(x, p[b], acc[d][b]);
        }
      }
    }
    __builtin_amdgcn_s_setprio(0);
    bits = next, next = after;
    tile_barrier();
  }

#pragma unroll
  for (int b = 0; b < QW; ++b) {
    if (wrow + b * 32 + c32 >= rows) continue;
    const float sum = half_sum(l[b]);
    const int64_t place = (s.q0 + qi[b]) * a.hq + head * a.group + qg[b];
    if constexpr (SPLIT) {
      float* to = a.part + (static_cast<int64_t>(split) * a.total_q * a.hq + place) * a.dim;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = 32 * d + 8 * e + 4 * h;
          if (c < a.dim)
            *reinterpret_cast<f32x4*>(to + c) = f32x4{acc[d][b][4 * e], acc[d][b][4 * e + 1], acc[d][b][4 * e + 2],
                                                       acc[d][b][4 * e + 3]};
        }
      if (h == 0) {
        float* ml = a.part_ml + (static_cast<int64_t>(split) * a.total_q * a.hq + place) * 2;
        ml[0] = m[b], ml[1] = sum;
      }
    } else {
      float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // no key seen: zeros
      if constexpr (TERMS != 0)
        if (a.rest != nullptr) {
          const float rounded = half_sum(lr[b]);
          inv = rounded == 0.0f ? 0.0f : 1.0f / rounded;
        }
      store_row<T, DP>(static_cast<T*>(a.out) + place * a.dim, a.dim, h, &acc[0][b], QW, inv);
      if constexpr (TERMS != 0)
        if (a.rest != nullptr) store_row<T, DP, true>(static_cast<T*>(a.rest) + place * a.dim, a.dim, h, &acc[0][b], QW, inv);
      if (a.lse != nullptr && h == 0) a.lse[place] = sum == 0.0f ? -INFINITY : (m[b] + __builtin_amdgcn_logf(sum)) * kLn2;
    }
  }
}

template <typename T, int DP, int NW, int QW, bool Z, bool SPLIT, int TERMS>
__global__ __launch_bounds__(64 * NW, DP <= 64 && NW * QW == 4 ? 3 : 2) void attend_kernel(ArgsOf<TERMS> a) {
  attend_rows_of<T, DP, NW, QW, Z, SPLIT, TERMS>(a, blockIdx.x, gridDim.x);
}

// Short segments and small problems: waves that work on their own, on blocks of 32 packed
// rows of one key head. Keys go from memory straight to matrix operands, values through a tile
// of 64 rows in LDS for the transposed read; there is little to prefetch for, so one tile is
// held and more waves are resident. Groups of 16 keys that are all hidden or past the segment
// are skipped.
//
// KW = 1, segments of tens of rows and keys (windows of a serialized level): four tasks to a
// workgroup, the heads of a segment side by side since they share its cache lines, no
// barriers. A task is up to 256 rows of a segment, block after block, the next block's
// queries on their way; keys and values that fit one tile are loaded once. KW > 1, too few
// rows to fill the chip: KW waves share a block and take every KW-th tile of the keys; their
// parts meet in LDS, weighed by exp2(m - max m) in fp32.
//
// Bound by memory latency and the waves that fit: 327,581 rows in windows of 48, 8 heads of 32
// (671 MB) in 166 us, 4.05 TB/s; a fifth more as 64-row workgroups of attend_kernel.
constexpr int kShortSpan = 256;

template <typename T, int DP, int KW, bool Z, int TERMS>
__global__ __launch_bounds__(KW == 1 ? 256 : 64 * KW,
                             KW > 1 ? KW / 4 : (DP <= 32 ? (TERMS ? 3 : 4) : (DP <= 64 ? 2 : 1))) void
attend_short_kernel(ArgsOf<TERMS> a) {
  constexpr int SPAN = KW == 1 ? kShortSpan : 32, KS = DP / 16, DB = DP / 32;
  constexpr int TILE = KW > 1 && DP * 132 > kTile<DP> ? DP * 132 : kTile<DP>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c32 = lane & 31, h = lane >> 5;
  const TileLane at = tile_lane<DP>(lane);
  char* vt = smem + wave * TILE;
  const int64_t id = KW > 1 ? blockIdx.x : xcd_remap(blockIdx.x, gridDim.x) * 4 + wave;
  const int head = static_cast<int>(id % a.hk), slot = static_cast<int>(id / a.hk);
  if (slot >= a.slots) return;
  Segment s;
  find_segment<KW == 1>(a.cu_q, a.len_q, a.batch, a.total_q, a.group, SPAN, slot, s);
  segment_rows(a, s);
  const int rows = s.lq * a.group, off = s.lk - s.lq, first = s.tile * SPAN, last = min(rows, first + SPAN);
  if (s.tile < 0 || first >= last) return;

  const T* qp = static_cast<const T*>(a.q) + s.b * a.q_b + (a.cu_q != nullptr ? s.q0 * a.q_n : 0) +
                static_cast<int64_t>(head) * a.group * a.q_h;
  const T* kp = static_cast<const T*>(a.k) + s.b * a.k_b + head * a.k_h + (a.cu_k != nullptr ? s.k0 * a.k_n : 0);
  const char* vp = reinterpret_cast<const char*>(static_cast<const T*>(a.v) + s.b * a.v_b + head * a.v_h +
                                                 (a.cu_k != nullptr ? s.k0 * a.v_n : 0));
  auto load_rows = [&](const T* src, u32x4 (&x)[KS]) {
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int c = 16 * k + 8 * h;
      u32x4 v = {0, 0, 0, 0};
      if (!Z || c < a.dim) v = *reinterpret_cast<const u32x4*>(src + c);
      x[k] = v;
    }
  };
  auto load_queries = [&](int row0, u32x4 (&x)[KS]) {
    int i, g;
    split_row(a, min(row0 + c32, rows - 1), i, g);
    load_rows(qp + i * a.q_n + g * a.q_h, x);
  };
  // a tile of keys, in registers, and of values, on their way to LDS; the keys that are there
  u32x4 kf[2][KS];
  auto load_keys = [&](int k0) -> uint64_t {
    bool shown = k0 + lane < s.lk;
    if (Z && a.mask != nullptr) shown = shown && a.mask[s.k0 + (shown ? k0 + lane : 0)] != 0;
    const uint64_t bits = __ballot(shown);
    if (bits == 0) return bits;
    const int one = __builtin_ctzll(bits);  // stands in for the keys that are hidden or not there
    asm volatile("" ::: "memory");  // the reads of the tile before are done: their products have waited for them
#pragma unroll
    for (int n = 0; n < 2; ++n)
      if ((bits >> (32 * n) & 0xffffffffull) != 0)
        load_rows(kp + k0 * a.k_n + ((bits >> (32 * n + c32)) & 1 ? 32 * n + c32 : one) * a.k_n, kf[n]);
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) {
      int row, c;
      tile_chunk<DP, 1>(i, 0, lane, row, c);
      if (Z && c * 8 >= a.dim) continue;
      const uint32_t from = (bits >> row) & 1 ? row : one;
      lds_dma16(vp + k0 * a.v_n * 2 + (from * (static_cast<uint32_t>(a.v_n) * 2) + c * 16), vt + i * kBlock<DP>);
    }
    return bits;
  };

  if (Z && a.dim < DP) {
    for (int i = lane * 16; i < kTile<DP>; i += 1024) *reinterpret_cast<u32x4*>(vt + i) = u32x4{0, 0, 0, 0};
    wait_lgkm0();
  }
  const int seen_by_all = first_keys<TERMS>(a, s);
  auto seen_by = [&](int i) { return TERMS ? max(i + off + 1, seen_by_all) : i + off + 1; };
  u32x4 qf[KS], qn[KS];
  load_queries(first, qn);
  const bool once = KW == 1 && s.lk <= kKT;
  bool landed = false;  // once: the value tile has been waited for (a block that sees no key does not)
  uint64_t bits = 0;
  if (once) bits = load_keys(0);
  RowTerms<1> terms;
  float* table = nullptr;
  if constexpr (TERMS != 0) {
    if (has_bias<TERMS>(a)) {
      table = reinterpret_cast<float*>(smem + (KW == 1 ? 4 * kTile<DP> : KW * (TILE + 256)));
      int x0 = 0, x1 = 2 * (a.far + kPad) + 1;
      if constexpr (KW == 1) {  // a wave's own copy, of the places that its rows and keys reach
        table += wave * a.group * a.stride;
        int i, g;
        split_row(a, last - 1, i, g);
        x0 = min(max(a.far + kPad - (i + off), 0), 2 * a.far + kPad);
        split_row(a, first, i, g);
        x1 = min(x1, max(s.lk - (i + off) + a.far + kPad, x0 + 1));
        stage_bias<kPad>(a, table, a.stride, head * a.group, a.group, x0, x1, lane, 64);
        wait_lgkm0();
        asm volatile("" ::: "memory");
      } else {
        stage_bias<kPad>(a, table, a.stride, head * a.group, a.group, x0, x1, threadIdx.x, 64 * KW);
        __syncthreads();
      }
    }
  }
  for (int row0 = first; row0 < last; row0 += 32) {
#pragma unroll
    for (int k = 0; k < KS; ++k) qf[k] = qn[k];
    if (row0 + 32 < last) load_queries(row0 + 32, qn);
    int qi, qg;
    split_row(a, min(row0 + c32, rows - 1), qi, qg);
    int kend = s.lk, full = s.lk;  // keys that some row sees, that every row sees
    if (a.causal) {
      int i, g;
      split_row(a, min(rows, row0 + 32) - 1, i, g);
      kend = min(kend, seen_by(i));
      split_row(a, row0, i, g);
      full = min(full, seen_by(i));
    }
    if constexpr (TERMS != 0) {
      const int is[1] = {qi}, gs[1] = {qg};
      row_terms<1>(a, s, terms, table, head, row0, rows, is, gs);
    }
    f32x16 acc[DB] = {};
    float m = -INFINITY, l = 0.0f;
    const int start = KW > 1 ? wave * kKT : 0;
    for (int k0 = start; k0 < kend; k0 += KW * kKT) {
      if (!once) bits = load_keys(k0);
      if (bits == 0) continue;
      f32x16 sc[2][1] = {};
#pragma unroll
      for (int n = 0; n < 2; ++n)
        if ((bits >> (32 * n) & 0xffffffffull) != 0)
#pragma unroll
          for (int k = 0; k < KS; ++k) Mfma<T>::run(kf[n][k], qf[k], sc[n][0]);
      float mul = a.scale2, add[1];
      if constexpr (TERMS != 0) mul = add_terms<TERMS, 2, 1, false>(a, terms, sc, k0, 0, h, false, add, nullptr);
      float top = -INFINITY;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint64_t some = bits >> (16 * k) & 0xffff;
        if (some == 0) continue;
        if (some != 0xffff) {
#pragma unroll
          for (int e = 8 * (k & 1); e < 8 * (k & 1) + 8; ++e)
            sc[k >> 1][0][e] = sees_key(bits, 32 * (k >> 1) + 8 * (e >> 2) + (e & 3)) ? sc[k >> 1][0][e] : -INFINITY;
        }
        if (k0 + 16 * k + 16 > full && a.causal) {
          const int seen = seen_by(qi) - k0 - 4 * h;
#pragma unroll
          for (int e = 8 * (k & 1); e < 8 * (k & 1) + 8; ++e)
            sc[k >> 1][0][e] = 32 * (k >> 1) + 8 * (e >> 2) + (e & 3) < seen ? sc[k >> 1][0][e] : -INFINITY;
        }
#pragma unroll
        for (int e = 8 * (k & 1); e < 8 * (k & 1) + 8; ++e) top = larger(top, sc[k >> 1][0][e]);
      }
      if constexpr (TERMS != 0) top = kept_max(__builtin_fmaf(top, mul, add[0]));
      else top = half_max(top) * a.scale2;
      const float to = fmaxf(m, top - kBelow<T>);
      if (k0 > start) {
        const float by = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - to);
        l *= by;
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[d] *= by;
      }
      m = to;
      const float ref = m == -INFINITY ? 0.0f : m, less = TERMS ? add[0] - ref : -ref;
      if (!once || !landed) wait_vmcnt<0>();  // the value tile
      landed = true;
      asm volatile("" ::: "memory");
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if ((bits >> (16 * k) & 0xffff) == 0) continue;
        f32x8 x;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[k >> 1][0][8 * (k & 1) + e], mul, less));
          l += x[e];
        }
        const u32x4 p = pack8<T>(x);
#pragma unroll
        for (int d = 0; d < DB; ++d) Mfma<T>::run(read_columns<DP>(vt, 16 * k, d, at), p, acc[d]);
      }
    }
    if constexpr (KW > 1) {
      // parts in LDS as [column / 4][33 rows][4], so that neither side's accesses share banks
      float* ml = reinterpret_cast<float*>(smem + KW * TILE);
      l = half_sum(l);
      if (h == 0) ml[wave * 32 + c32] = m, ml[(KW + wave) * 32 + c32] = l;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<f32x4*>(vt + ((8 * d + 2 * e + h) * 33 + c32) * 16) =
              f32x4{acc[d][4 * e], acc[d][4 * e + 1], acc[d][4 * e + 2], acc[d][4 * e + 3]};
      __syncthreads();
      const int quads = a.dim / 4;
      for (int i = threadIdx.x; i < 32 * quads; i += 64 * KW) {
        const int row = i / quads, q = i - row * quads;
        if (row0 + row >= rows) break;
        float high = -INFINITY;
#pragma unroll
        for (int w = 0; w < KW; ++w) high = fmaxf(high, ml[w * 32 + row]);
        const float from = high == -INFINITY ? 0.0f : high;
        f32x4 x = {0, 0, 0, 0};
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          const float by = __builtin_amdgcn_exp2f(ml[w * 32 + row] - from);
          sum += ml[(KW + w) * 32 + row] * by;
          x += *reinterpret_cast<const f32x4*>(smem + w * TILE + (q * 33 + row) * 16) * by;
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // no key seen: zeros
        int r, g;
        split_row(a, row0 + row, r, g);
        const int64_t place = (s.q0 + r) * a.hq + head * a.group + g;
        typedef T t4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<t4*>(static_cast<T*>(a.out) + place * a.dim + 4 * q) =
            t4{static_cast<T>(x[0] * inv), static_cast<T>(x[1] * inv), static_cast<T>(x[2] * inv), static_cast<T>(x[3] * inv)};
        if (a.lse != nullptr && q == 0)
          a.lse[place] = sum == 0.0f ? -INFINITY : (high + __builtin_amdgcn_logf(sum)) * kLn2;
      }
    } else {
      const float sum = half_sum(l), inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      if (row0 + c32 < rows) {
        const int64_t place = (s.q0 + qi) * a.hq + head * a.group + qg;
        store_row<T, DP>(static_cast<T*>(a.out) + place * a.dim, a.dim, h, acc, 1, inv);
        if (a.lse != nullptr && h == 0) a.lse[place] = sum == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(sum)) * kLn2;
      }
    }
  }
  if (once && !landed) wait_vmcnt<0>();  // no block saw a key: the wave must not leave loads to LDS behind
}

// Joins the splits of a row: a workgroup per row. Every wave weighs the parts by exp2(m -
// max m) (lane s: split s) and sums a quarter of them, two columns a lane, all loads in
// flight together; the quarters meet in LDS in a fixed order. Reads splits * (dim + 2) * 4
// bytes a row: 32 splits of 256 rows of 128 in 4.6 us.
template <typename T>
__global__ __launch_bounds__(256) void attend_join_kernel(AttnArgs a, int64_t rows) {
  __shared__ float parts[4][128];
  __shared__ float weights[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t r = blockIdx.x;
  float m[4], l[4], top = -INFINITY;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int s = j * 64 + lane;
    const bool on = s < a.splits;
    const float* ml = a.part_ml + ((on ? s : 0) * rows + r) * 2;
    m[j] = on ? ml[0] : -INFINITY, l[j] = on ? ml[1] : 0.0f;
    top = fmaxf(top, m[j]);
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  const float ref = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < 4; ++j) m[j] = __builtin_amdgcn_exp2f(m[j] - ref), sum += m[j] * l[j];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  // this wave's splits: wave, wave + 4, ...; at most 64
  if ((lane & 3) == wave)
#pragma unroll
    for (int j = 0; j < 4; ++j) weights[wave][j * 16 + (lane >> 2)] = m[j];
  __syncthreads();
  const int c = 2 * lane;
  float x = 0.0f, y = 0.0f;
  if (c < a.dim) {
#pragma unroll 8
    for (int s = wave; s < a.splits; s += 4) {
      const float2 v = *reinterpret_cast<const float2*>(a.part + (s * rows + r) * a.dim + c);
      const float w = weights[wave][s >> 2];
      x = __builtin_fmaf(v.x, w, x), y = __builtin_fmaf(v.y, w, y);
    }
  }
  parts[wave][c] = x, parts[wave][c + 1] = y;
  __syncthreads();
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  if (threadIdx.x < a.dim) {
    const int d = threadIdx.x;
    static_cast<T*>(a.out)[r * a.dim + d] =
        static_cast<T>(((parts[0][d] + parts[1][d]) + (parts[2][d] + parts[3][d])) * inv);
  }
  if (a.lse != nullptr && threadIdx.x == 0)
    a.lse[r] = sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

template <typename T>
int launch_join(const AttnArgs& a, hipStream_t stream) {
  const int64_t n = a.total_q * a.hq;
  HI3D_REQUIRE(n < (1ll << 31), "too many rows for one launch");
  hipLaunchKernelGGL(attend_join_kernel<T>, dim3(static_cast<unsigned>(n)), dim3(256), 0, stream, a, n);
  HI3D_LAUNCH_CHECK();
  return HI3D_OK;
}

template <typename T, int DP, int NW, int QW, int TERMS>
int launch_attend(ArgsOf<TERMS> a, hipStream_t stream) {
  constexpr int rows = NW * QW * 32;
  const bool z = a.mask != nullptr || a.dim < DP;
  const int64_t per = a.cu_q != nullptr ? packed_slots(a.total_q, a.group, rows, a.batch)
                                        : ceil_div(static_cast<int64_t>(a.len_q) * a.group, rows) * a.batch;
  const int64_t blocks = per * a.hk * a.splits;
  HI3D_REQUIRE(blocks < (1ll << 31), "too many rows for one launch");
  a.slots = static_cast<int>(per);
  const size_t lds = 4 * kTile<DP> + (z ? kBiasBytes : 0) + term_bytes<TERMS>(a);
  if (a.splits == 1)
    return z ? launch_tiles<&attend_kernel<T, DP, NW, QW, true, false, TERMS>>(a, blocks, 64 * NW, lds, stream)
             : launch_tiles<&attend_kernel<T, DP, NW, QW, false, false, TERMS>>(a, blocks, 64 * NW, lds, stream);
  if constexpr (NW * QW == 8) {  // rows that fill the chip four times over are not split
    return fail(HI3D_ERR_INVALID, "256 rows to a workgroup are not split");
  } else {
    const int rc = z ? launch_tiles<&attend_kernel<T, DP, NW, QW, true, true, TERMS>>(a, blocks, 64 * NW, lds, stream)
                     : launch_tiles<&attend_kernel<T, DP, NW, QW, false, true, TERMS>>(a, blocks, 64 * NW, lds, stream);
    return rc != HI3D_OK ? rc : launch_join<T>(a, stream);
  }
}

template <typename T, int DP, int KW, int TERMS>
int launch_short(ArgsOf<TERMS> a, hipStream_t stream) {
  constexpr int rows = KW == 1 ? kShortSpan : 32;
  constexpr int part = DP * 132 > kTile<DP> ? DP * 132 : kTile<DP>;  // a wave's tile, or its 32 rows of the output
  const size_t lds = KW == 1 ? 4 * (kTile<DP> + term_bytes<TERMS>(a)) : KW * (part + 256) + term_bytes<TERMS>(a);
  const int64_t per = a.cu_q != nullptr ? packed_slots(a.total_q, a.group, rows, a.batch)
                                        : ceil_div(static_cast<int64_t>(a.len_q) * a.group, rows) * a.batch;
  HI3D_REQUIRE(per * a.hk < (1ll << 31), "too many rows for one launch");
  a.slots = static_cast<int>(per);
  const int64_t blocks = KW == 1 ? ceil_div(per * a.hk, 4) : per * a.hk;
  constexpr int threads = KW == 1 ? 256 : 64 * KW;
  return a.mask != nullptr || a.dim < DP
             ? launch_tiles<&attend_short_kernel<T, DP, KW, true, TERMS>>(a, blocks, threads, lds, stream)
             : launch_tiles<&attend_short_kernel<T, DP, KW, false, TERMS>>(a, blocks, threads, lds, stream);
}

// Few rows: 32-row blocks that leave compute units without a workgroup, over keys that 8
// waves get through sooner than parts of them and a join: 517 x 517 x 8 heads x 64 takes
// 8.1 us for 18.8, 1000 x 1000 10.9 for 22.9, 517 x 4000 26.5 for 29.1. Single tokens fill
// little of a block and need more workgroups on their keys: 1030 keys x 33 heads x 64 in 9.7
// us for 10.8, but 2048 keys x 8 heads x 128 in 23.7 for 12.4.
// `more`: bytes of LDS besides the tiles of 8 waves.
bool few_rows(int64_t total_q, int64_t total_k, int batch, int hq, int hk, int dim, int cus, int more = 0) {
  const int64_t average = ceil_div(total_q * (hq / hk), batch), keys = ceil_div(total_k, batch);
  if (8 * (ceil_div(dim, 32) * 32 * 132 + 256) + more > 160 * 1024) return false;
  return batch * ceil_div(average, 32) * hk <= cus && keys * dim <= (average <= 32 ? 98304 : 262144);
}

int64_t segment_average(const AttnArgs& a) { return ceil_div(a.total_q * a.group, a.batch); }

// Rows of a workgroup: one wave where segments are short (a larger tile would be empty), else
// four waves of one block of 32 rows, or of two where heads are small and that still leaves
// four workgroups to each place on the chip: two blocks share their reads of LDS (20,011 x 33
// heads x 64: 1865 us for 1926), one fills the chip more evenly (8,191 x 33 x 64 in four
// segments: 193 us for 210).
int attend_rows(int64_t total_q, int batch, int hq, int hk, int dim, int cus) {
  const int64_t rows = total_q * (hq / hk), average = ceil_div(rows, batch);
  if (average <= 64) return average <= 32 ? 32 : 64;
  return dim <= 64 && ceil_div(rows, 256) * hk >= 8 * cus ? 256 : 128;
}

// Segments of tens of rows and keys: a wave each.
template <int TERMS>
bool short_segments(const ArgsOf<TERMS>& a) {
  const int tile = a.dim > 96 ? kTile<128> : static_cast<int>(ceil_div(a.dim, 32)) * kTile<32>;
  return segment_average(a) <= 64 && ceil_div(a.total_k, a.batch) <= 128 && 4 * (tile + term_bytes<TERMS>(a)) <= 160 * 1024;
}

// Rows of four waves each, not split: the kernels that are built for one term.
template <typename T, int DP, int TERMS>
int launch_wide(const ArgsOf<TERMS>& a, hipStream_t stream) {
  if constexpr (DP <= 64)
    if (a.rows == 256) return launch_attend<T, DP, 4, 2, TERMS>(a, stream);
  return launch_attend<T, DP, 4, 1, TERMS>(a, stream);
}

template <typename T, int TERMS>
int launch_wide_type(const ArgsOf<TERMS>& a, hipStream_t stream) {
  switch ((a.dim + 31) / 32) {
    case 1: return launch_wide<T, 32, TERMS>(a, stream);
    case 2: return launch_wide<T, 64, TERMS>(a, stream);
    case 3: return launch_wide<T, 96, TERMS>(a, stream);
    default: return launch_wide<T, 128, TERMS>(a, stream);
  }
}

template <typename T, int DP, int TERMS>
int launch_attend_dim(const ArgsOf<TERMS>& a, hipStream_t stream) {
  if (short_segments<TERMS>(a))
    return launch_short<T, DP, 1, TERMS>(a, stream);
  if (a.few) return launch_short<T, DP, 8, TERMS>(a, stream);
  if (a.rows == 32) return launch_attend<T, DP, 1, 1, TERMS>(a, stream);
  if constexpr (TERMS == 0)
    if (a.rows == 64) return launch_attend<T, DP, 1, 2, TERMS>(a, stream);
  return launch_wide<T, DP, TERMS>(a, stream);
}

template <typename T, int TERMS>
int launch_attend_type(const ArgsOf<TERMS>& a, hipStream_t stream) {
  switch ((a.dim + 31) / 32) {
    case 1: return launch_attend_dim<T, 32, TERMS>(a, stream);
    case 2: return launch_attend_dim<T, 64, TERMS>(a, stream);
    case 3: return launch_attend_dim<T, 96, TERMS>(a, stream);
    default: return launch_attend_dim<T, 128, TERMS>(a, stream);
  }
}

// Splits of the key axis: as many as fill the chip twice over, each of at least 4 tiles.
int attend_splits(int64_t total_q, int64_t total_k, int batch, int hq, int hk, int dim, int cus, bool few) {
  if (few) return 1;
  const int64_t average = ceil_div(total_q * (hq / hk), batch);
  const int tile = attend_rows(total_q, batch, hq, hk, dim, cus);
  const int64_t blocks = (batch * ceil_div(average, tile)) * hk;
  const int64_t tiles = ceil_div(ceil_div(total_k, batch), kKT);
  const int64_t fill = static_cast<int64_t>(cus) * (tile <= 64 ? 8 : 2);
  int64_t splits = fill / (blocks > 0 ? blocks : 1);
  if (splits > tiles / 4) splits = tiles / 4;
  if (splits > 256) splits = 256;
  return splits < 1 ? 1 : static_cast<int>(splits);
}

}  // namespace
}  // namespace hi3d
