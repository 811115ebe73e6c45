// Terms of attention scores beside scale q k: a cap, a cost that grows with the distance, a
// learned bias by relative position, and keys that every query of a causal segment sees.
//
// Row i of a segment with lq queries and lk keys stands at place i + lk - lq among the keys; r =
// j - place is the relative position of key j. With x = scale q k:
//   s = cap tanh(x / cap)      (or x)
//     - slope[head] |r|
//     + bias[map[clamp(r, -far, far) + far], head]
// and a causal row sees the keys with r <= 0 or j < prefix.
//
// All in powers of two (times log2 e). cap tanh(x / cap) = cap (1 - 2 u), u = 1 / (1 + exp(2 x /
// cap)): an exponential and a reciprocal, 1 ulp each, so a capped score is off by at most 10 e
// cap (e = 2^-24; caps end at 1024, where that is 6e-4); its derivative is 4 u (1 - u). What is
// left is kept as a sum mul * score + add that goes into the softmax's own multiply-add: a capped
// score stays -u with mul = 2 cap, a distance costs one step of the score product where a tile lies
// on one side of the rows (its constant part is in add), and a bias costs nothing where a tile lies
// past `far`: there it is one number. Tiles between look it up in LDS, where every query head of
// the workgroup has its bias by relative position, extended on both sides by what a tile can reach
// past `far`, so that a lane's places are one address with constant offsets.
//
// 20,011 rows x 33 heads x 64 fp16 in two objects: 1841 us without terms, 2000 with a bias of 128
// keys to each side, 2121 with slopes, 2690 with a cap (its 24 cycles a score and wave are vector
// operations in a loop that these bound); causal 8,192 x 32/8 heads x 128 bf16 in two: 273, 283, 307
// and 323.
#pragma once

#include <type_traits>

#include "attention.h"

namespace hi3d {

// A bias below hides its key: -infinity, the lowest numbers of fp32 and bf16, and the -1e9 that stands for "not seen".
// Beside any other key such a one has no part of a row in fp32; a row that sees nothing else would be left with
// the rounding of its scores (1.4e9 in steps of 128), and lse with less. fp16's lowest, -65504, is a number:
// scores keep steps of 2^-7 there.
constexpr float kHideBelow = -1e5f;
// Keys of a tile whose scores are all below, in powers of two, are as good as hidden (from a reference of zero their
// probabilities are), and so a row that sees no others counts as one that sees none: steep slopes and distant
// keys alone get there. fp32 keeps half a power of two at that size, which fp16 probabilities of up to 2^15
// have room for; where it keeps less, neither a reference nor lse says which power a row's probabilities have.
constexpr float kLost = -4194304.0f;
__device__ __forceinline__ float kept_max(float x) {
  x = half_max(x);
  return x < kLost ? -INFINITY : x;
}
constexpr int kPad = kKT, kPadKeys = 128;  // what the rows' and the keys' kernels look up past `far`
constexpr int kPadSums = 93;               // what a wave's 32 rows and a tile's 64 keys reach past it together
constexpr int kMostTermBytes = 72 * 1024;

struct TermArgs : AttnArgs {
  float cap2, cap_in;           // log2(e) cap, and 2 log2(e) scale / cap; 0 without a cap
  float per_mul;                // 1 / mul of a score without a bias
  const float* slopes;          // [hq], or null
  const void* bias;             // [buckets, hq], or null
  const int32_t* map;           // [2 far + 1]
  int32_t bias_type, buckets, far;
  int32_t stride, stride_keys;  // floats of a head's bias in LDS, in the kernels over rows and over keys
  const int32_t* prefix;        // [batch], or null
  // the keys are the common beginning of `per`-row sequences (rows of segment 0 one after another):
  const int32_t* own_lens;      // keys in use of each sequence behind it, or null: own_len
  int32_t per, own_len;
  int32_t share;                // backward: query heads of a key head, where hk counts query heads
  float* dbias;                 // backward: [hq, slots, sum_length(far)] parts, or null
  void* rest;                   // [total_q, hq, d] what rounding took from out, times kRest; or null
};

// Which terms a kernel is built for: none, one of them, or any (each asked for when it runs).
constexpr int kCap = 1, kSlopes = 2, kBias = 4, kAll = 7;
template <int TERMS>
using ArgsOf = std::conditional_t<TERMS != 0, TermArgs, AttnArgs>;
template <int TERMS>
__device__ __forceinline__ bool has_cap(const TermArgs& a) { return TERMS == kAll ? a.cap2 > 0.0f : (TERMS & kCap) != 0; }
template <int TERMS>
__device__ __forceinline__ bool has_slopes(const TermArgs& a) { return TERMS == kAll ? a.slopes != nullptr : (TERMS & kSlopes) != 0; }
template <int TERMS>
__device__ __forceinline__ bool has_bias(const TermArgs& a) { return TERMS == kAll ? a.bias != nullptr : (TERMS & kBias) != 0; }

// Floats of a head's bias in LDS: its length, up to the next number after which the lanes' heads
// (32 / group rows of each) start at banks of their own.
inline int bias_stride(int far, int pad, int group) {
  const int want = group >= 32 ? 1 : 32 / group, length = 2 * far + 2 * pad + 1;
  return length + ((want - length) % 64 + 64) % 64;
}
__host__ __device__ constexpr int sum_length(int far) { return 2 * (far + kPadSums) + 1; }
__host__ __device__ constexpr int sum_stride(int far) { return (sum_length(far) + 3) / 4 * 4; }
// A wave's score gradients of 32 rows and 8 keys in LDS, between 7 rows of zeros on either side.
constexpr int kSkewRow = 9, kSkew = (7 + 32 + 7) * kSkewRow + 2;

template <int TERMS>
int term_bytes(const ArgsOf<TERMS>& a) {
  if constexpr (TERMS != 0) return a.bias != nullptr ? a.group * a.stride * 4 : 0;
  else return 0;
}

__device__ __forceinline__ float load_bias(const TermArgs& a, int at) {
  if (a.bias_type == HI3D_F32) return static_cast<const float*>(a.bias)[at];
  if (a.bias_type == HI3D_F16) return static_cast<float>(static_cast<const _Float16*>(a.bias)[at]);
  return static_cast<float>(static_cast<const __bf16*>(a.bias)[at]);
}

// Which bucket place x of a padded bias belongs to. (Numbers outside the table count as the nearest.)
__device__ __forceinline__ int bucket_at(const TermArgs& a, int x, int pad) {
  const int b = a.map[min(max(x - pad, 0), 2 * a.far)];
  return min(max(b, 0), a.buckets - 1);
}

// Places x0 to x1 of the bias of `count` query heads from `head0` on into LDS, in powers of two.
template <int PAD>
__device__ __forceinline__ void stage_bias(const TermArgs& a, float* to, int stride, int head0, int count, int x0, int x1,
                                           int thread, int threads) {
  // and the two ends, which stand for all places past `far`
  const int end = 2 * (a.far + PAD), places = x1 - x0 + (x0 > 0) + (x1 <= end);
  for (int i = thread; i < places; i += threads) {
    const int x = i < x1 - x0 ? x0 + i : (i == x1 - x0 && x0 > 0 ? 0 : end);
    const int at = bucket_at(a, x, PAD) * a.hq + head0;
    for (int g = 0; g < count; ++g) {
      const float v = load_bias(a, at + g);
      to[g * stride + x] = v < kHideBelow ? -INFINITY : v * kLog2e;
    }
  }
}

__device__ __forceinline__ float minus_u(const TermArgs& a, float score) {
  return __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(score * a.cap_in));
}

// x + the two values in a word of T.
template <typename T>
__device__ __forceinline__ float add_pair(uint32_t word, float x) {
  typedef T t2 __attribute__((ext_vector_type(2)));
  const t2 one = {static_cast<T>(1.0f), static_cast<T>(1.0f)};
  if constexpr (std::is_same_v<T, _Float16>) return __builtin_amdgcn_fdot2(__builtin_bit_cast(t2, word), one, x, false);
  else return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(t2, word), one, x, false);
}

// A lane's rows (QW blocks of 32 of a wave) in the kernels whose lanes own query rows.
template <int QW>
struct RowTerms {
  float slope[QW];       // log2(e) slope
  int place[QW];         // among the keys
  const float* bias[QW]; // of the row's head, in LDS
  int first, last;       // least and largest place of the wave's rows
};

// Keys of a segment that all of its rows see.
template <int TERMS>
__device__ __forceinline__ int first_keys(const ArgsOf<TERMS>& a, const Segment& s) {
  if constexpr (TERMS != 0)
    if (a.prefix != nullptr && s.b >= 0 && s.b < a.batch) return min(max(a.prefix[s.b], 0), s.lk);
  return 0;
}

// What the terms of a lane's rows depend on: rows r = wrow + 32 b + lane % 32 of queries i and heads g.
template <int QW>
__device__ __forceinline__ void row_terms(const TermArgs& a, const Segment& s, RowTerms<QW>& w, const float* table, int head,
                                          int wrow, int rows, const int (&i)[QW], const int (&g)[QW]) {
  const int off = s.lk - s.lq;
  int least = 0x7fffffff, most = -0x7fffffff - 1;
#pragma unroll
  for (int b = 0; b < QW; ++b) {
    w.slope[b] = a.slopes != nullptr ? a.slopes[head * a.group + g[b]] * kLog2e : 0.0f;
    w.bias[b] = table + g[b] * a.stride;
    w.place[b] = i[b] + off;
    if (a.per > 0) {
      const int of = i[b] / a.per;
      int own = a.own_len;
      if (a.own_lens != nullptr) own = min(max(a.own_lens[of], 0), own);
      w.place[b] = s.lk + own - a.per + i[b] - of * a.per;
      least = min(least, w.place[b]), most = max(most, w.place[b]);
    }
  }
  if (a.per > 0) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) least = min(least, __shfl_xor(least, d)), most = max(most, __shfl_xor(most, d));
    w.first = __builtin_amdgcn_readfirstlane(least), w.last = __builtin_amdgcn_readfirstlane(most);
    return;
  }
  int x, y;
  split_row(a, min(wrow, rows - 1), x, y);
  w.first = x + off;
  split_row(a, min(wrow + QW * 32, rows) - 1, x, y);
  w.last = x + off;
}

// Distances to the keys of one side, as one more step of the score product: slope * (number of the key in
// its tile), with the slope in three numbers of the inputs' type and the key's number, which has one. It
// takes a matrix instruction a 32 x 32 block where a multiply-add a score takes 16 vector ones, in loops that
// vector operations bound: slopes cost 20,011 rows x 33 heads x 64 15 % (20 % as multiply-adds).
//
// Three numbers of bf16 hold fp32's 24 bits. Those of fp16 end at 2^-24, which the second one of a slope
// below 1/8 is already past: slopes are multiplied by a power of two, 1 to 2^14, that brings the wave's largest
// up to 2^9, and the numbers of keys divided by it (2^-14 times a whole number of up to 11 bits is
// exact). A slope is then off by at most 2^-34 of the largest, or 2^-39: over 65,504 keys, the
// farthest that are taken this way, by 4e-6 of the largest slope, or 1.2e-7 scale, in a score.
template <typename T>
struct SideProduct {
  u32x4 slope;  // second operand: the lane's row (with the signs turned: keys behind it)
  float down;   // of the keys' numbers
  bool on;      // within the type's range in all lanes

  __device__ __forceinline__ static float upwards(float most) {
    if constexpr (!std::is_same_v<T, _Float16>) return 1.0f;
    const int e = min(max(10 - __builtin_amdgcn_frexp_expf(most), 0), 14);
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane((127 + e) << 23));
  }
  __device__ __forceinline__ static void split(float t, T (&x)[3]) {
    x[0] = static_cast<T>(t);
    const float r = t - static_cast<float>(x[0]);
    x[1] = static_cast<T>(r), x[2] = static_cast<T>(r - static_cast<float>(x[1]));
  }
  __device__ __forceinline__ void set(float t, int h) {
    const float most = wave_max(__builtin_fabsf(t)), up = upwards(most);
    on = !(most > 16384.0f), down = 1.0f / up;
    T x[3];
    split(t * up, x);
    const T zero = static_cast<T>(0.0f);
    const typename Vec8<T>::type v = {x[0], x[1], x[2], zero, zero, zero, zero, zero};
    slope = h == 0 ? __builtin_bit_cast(u32x4, v) : u32x4{0, 0, 0, 0};
  }
  // Lanes that own keys: t * (key - place of the row) where the heads of a tile's 64 rows are the same in
  // every tile (the group divides 64). A row's slope in three numbers meets the key's distance to
  // the tile's first row in numbers of 8 (11) bits, and its own distance from there, slope times row /
  // group in three numbers, meets -1: 12 of the 16 products of a step. (t of up to 1024: 63 t is in fp16's range.)
  __device__ __forceinline__ static u32x4 of_row(float t, int row, int h) {
    T x[3], y[3];
    split(t, x), split(-t * static_cast<float>(row), y);
    const T zero = static_cast<T>(0.0f);
    const typename Vec8<T>::type a = {x[0], x[1], x[2], x[0], x[1], x[2], x[0], x[1]}, b = {x[2], y[0], y[1], y[2], zero, zero, zero, zero};
    return h == 0 ? __builtin_bit_cast(u32x4, a) : __builtin_bit_cast(u32x4, b);
  }
  static constexpr int kBits = std::is_same_v<T, _Float16> ? 11 : 8;
  static constexpr int kFarthest = std::is_same_v<T, _Float16> ? 65504 : (1 << 24) - 1;
  __device__ __forceinline__ static u32x4 of_key(int distance, int h, float down) {
    const int far = distance < 0 ? -distance : distance, low = (1 << kBits) - 1;
    auto number = [&](int x) { return static_cast<T>(static_cast<float>(distance < 0 ? -x : x) * down); };
    const T b0 = number(far & low), b1 = number(far & low << kBits), b2 = number(far & ~(low << kBits | low));
    const T one = static_cast<T>(down), zero = static_cast<T>(0.0f);
    const typename Vec8<T>::type a = {b0, b0, b0, b1, b1, b1, b2, b2}, b = {b2, one, one, one, zero, zero, zero, zero};
    return h == 0 ? __builtin_bit_cast(u32x4, a) : __builtin_bit_cast(u32x4, b);
  }
  // first operand: keys 32 n + l % 32
  __device__ __forceinline__ static u32x4 keys(int n, int c32, float down) {
    const T j = static_cast<T>(static_cast<float>(32 * n + c32) * down), zero = static_cast<T>(0.0f);
    const typename Vec8<T>::type v = {j, j, j, zero, zero, zero, zero, zero};
    return __builtin_bit_cast(u32x4, v);
  }
};

// Adds a tile's terms to its scores sc[n][b] (keys k0 + 32 (n0 + n) + 8 (e / 4) + 4 h + e % 4). Scores
// in powers of two are then sc * (returned factor) + add[b]. KEEP: derivative of the cap, times -1/4. folded:
// the distances within a tile on one side are in the scores already.
template <int TERMS, int N, int QW, bool KEEP>
__device__ __forceinline__ float add_terms(const TermArgs& a, const RowTerms<QW>& w, f32x16 (&sc)[N][QW], int k0, int n0,
                                           int h, bool folded, float (&add)[QW], f32x16* bend) {
  float mul = a.scale2;
#pragma unroll
  for (int b = 0; b < QW; ++b) add[b] = 0.0f;
  if (has_cap<TERMS>(a)) {
    mul = 2.0f * a.cap2;
#pragma unroll
    for (int b = 0; b < QW; ++b) {
      add[b] = a.cap2;
#pragma unroll
      for (int n = 0; n < N; ++n) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float u = minus_u(a, sc[n][b][e]);
          sc[n][b][e] = u;
          if constexpr (KEEP) (*bend)[e] = __builtin_fmaf(u, u, u);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  if (has_slopes<TERMS>(a)) {
    const bool before = k0 + kKT - 1 <= w.first, after = k0 >= w.last;
#pragma unroll
    for (int b = 0; b < QW; ++b) {
      const float from = static_cast<float>(k0 + 4 * h - w.place[b]);
      if (before || after) {
        const float s = after ? -w.slope[b] : w.slope[b], t = s * a.per_mul;
        add[b] = __builtin_fmaf(s, folded ? static_cast<float>(k0 - w.place[b]) : from, add[b]);
        if (!folded) {
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              sc[n][b][e] = __builtin_fmaf(t, static_cast<float>(32 * (n0 + n) + 8 * (e >> 2) + (e & 3)), sc[n][b][e]);
        }
      } else {
        const float t = -w.slope[b] * a.per_mul;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            sc[n][b][e] = __builtin_fmaf(
                t, __builtin_fabsf(from + static_cast<float>(32 * (n0 + n) + 8 * (e >> 2) + (e & 3))), sc[n][b][e]);
      }
    }
  }
  if (has_bias<TERMS>(a)) {
    if (k0 + kKT - 1 - w.first <= -a.far) {
#pragma unroll
      for (int b = 0; b < QW; ++b) add[b] += w.bias[b][0];
    } else if (k0 - w.last >= a.far) {
#pragma unroll
      for (int b = 0; b < QW; ++b) add[b] += w.bias[b][2 * (a.far + kPad)];
    } else {
#pragma unroll
      for (int b = 0; b < QW; ++b) {
        const float* at = w.bias[b] + min(max(k0 + 4 * h - w.place[b] + a.far + kPad, 0), 2 * a.far + kPad);
#pragma unroll
        for (int n = 0; n < N; ++n) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            sc[n][b][e] = __builtin_fmaf(sc[n][b][e], mul, at[32 * (n0 + n) + 8 * (e >> 2) + (e & 3)]);
          __builtin_amdgcn_sched_barrier(0);  // 16 numbers in flight: more of them spill
        }
      }
      mul = 1.0f;
    }
  }
  return mul;
}

// The one term of a problem, or kAll.
inline int one_term(const TermArgs& a) {
  const int kind = (a.cap2 > 0.0f ? kCap : 0) | (a.slopes != nullptr ? kSlopes : 0) | (a.bias != nullptr ? kBias : 0);
  return kind == kCap || kind == kSlopes || kind == kBias ? kind : kAll;
}

// Workgroups of four waves whose rows are not parts (attention_terms_one.hip), and the gradients over them
// (attention_terms_grad_one.hip), built for one term each: with the others' registers gone most need
// no spills. (Left: dk and dv at 128 values a head, 8 registers in fp16 and 2 in bf16 with slopes, 4 and 8 with a
// bias, and 4 at 64 values in fp16 with a bias; 3 of masked rows of two blocks a wave with a bias.)
int launch_rows_of_one(const TermArgs& a, int dtype, int kind, hipStream_t stream);
int launch_grad_of_one(const TermArgs& a, int dtype, int kind, hipStream_t stream);

}  // namespace hi3d
