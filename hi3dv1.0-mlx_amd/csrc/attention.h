// Shared parts of the attention kernels (attention.hip, attention_grad.hip): arguments,
// the packed rows and their segments, LDS tiles and the two matrix products on them.
//
// Definitions. A segment is one sequence: lq queries and lk keys, hq query heads over hk
// key heads, G = hq / hk query heads to each. All rows of a segment that read the same key
// head, (query i, head hk * G + g), are packed rows r = i * G + g: one packed row is one
// row of the score matrix of that key head, so shared key heads cost no second read of K
// and V and their gradients sum inside one workgroup.
//
// Matrix layout. v_mfma_f32_32x32x16 with the streamed operand (a tile of 64 rows in LDS)
// first and the owned operand (32 rows a wave keeps in registers) second: lane l then
// holds, for owned row l % 32, the 16 streamed rows 8 g + 4 (l / 32) + e. That layout is
// also the second operand of the product that follows (streamed^T times P), when the
// streamed rows of a 16-row step are taken in the order 4 h + {0..3}, 8 + 4 h + {0..3}
// for lane half h: the probabilities never leave the registers, and the first operand
// comes from the same LDS tile through the transposing read ds_read_b64_tr_b16.
//
// LDS tiles are rows of DP values (DP = head size rounded up to 32).
#pragma once

#include "common.h"
#include "conv_tile.h"

namespace hi3d {

typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kKT = 64;  // streamed rows of an LDS tile
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct AttnArgs {
  const void *q, *k, *v;        // rows of heads: element (b, i, h, d) at b*_b + i*_n + h*_h + d
  const void *o, *dout;         // backward: output and its gradient, [total_q, hq, d]
  const float* dlse;            // gradient of lse [total_q, hq], or null
  void *out, *dk, *dv;          // out: output, or dq; all [total, heads, d]
  float* lse;                   // [total_q, hq]
  float *lse2, *delta;          // backward: log2(e) lse and D of the packed rows, [hk, total_q * group]
  float* bound;                 // backward: [hk, dq_slots, dq_waves] bounds of dout's rows (fp16)
  int32_t dq_rows, dq_waves, dq_slots;
  float *part, *part_ml;        // split forward: [split, total_q, hq, d], [split, total_q, hq, 2]
  int64_t q_b, q_n, q_h, k_b, k_n, k_h, v_b, v_n, v_h;
  const int32_t *cu_q, *cu_k;   // [batch + 1] offsets of packed segments, or null: b * len
  const int32_t* lens_k;        // [batch] keys in use of each segment of len_k rows, or null
  const uint8_t* mask;          // [total_k], 0 where a key is hidden, or null
  int32_t batch, len_q, len_k;
  int64_t total_q, total_k;
  int32_t hq, hk, group, dim;
  uint32_t group_magic;         // ceil(2^32 / group) for group > 1
  float scale, scale2;          // scale, scale * log2(e)
  int32_t causal, splits, slots, head_minor, reverse, few, rows;
  int32_t once;                 // keys and values that no cache holds until they are read again
};

template <typename T>
struct Vec8;
template <>
struct Vec8<_Float16> {
  typedef f16x8 type;
};
template <>
struct Vec8<__bf16> {
  typedef bf16x8 type;
};

// 8 fp32 values rounded to nearest into one 16-byte operand. Probabilities and score
// gradients take this one rounding before their product; sums stay in fp32.
template <typename T>
__device__ __forceinline__ u32x4 pack8(f32x8 v) {
  return __builtin_bit_cast(u32x4, __builtin_convertvector(v, typename Vec8<T>::type));
}

// An LDS tile is DP / 8 blocks of 1024 bytes, each filled by one load of a wave, rows one after
// another; with 128 values a row, 16 bytes lie between blocks. Chunk c of a row is kept at c ^
// f(row). LDS serves 16 lanes' 16 bytes (row reads) or 32 lanes' 8 (transposing reads) a cycle
// from 64 banks. Row reads take one chunk of 16 consecutive rows: f (and the gaps) spread those
// that start at the same bank over all chunk places. Transposing reads take an aligned group
// of 4 chunks of 4 consecutive rows: f moves rows of the same bank into different groups.
// Counted: no bank conflicts (a third to a half of the LDS cycles with f of 8 rows alone).
template <int DP>
constexpr int kBlock = 1024 + (DP == 128 ? 16 : 0);
template <int DP>
constexpr int kTile = DP / 8 * kBlock<DP>;

template <int DP>
__device__ __forceinline__ int row_xor(int row) {
  if constexpr (DP == 128) return (row & 3) << 2;
  else if constexpr (DP == 64) return ((row & 2) << 1) | ((row >> 2) & 3);
  else return (row >> 2) & 3;
}
template <int DP>
__device__ __forceinline__ constexpr int row_place(int row) {
  return row * 2 * DP + (DP == 128 ? (row >> 2) * 16 : 0);
}

// Where a lane reads in a tile: base + (x ^ number of the chunk), bytes.
struct TileLane {
  int row, row_x;  // row reads: row l % 32, chunk l / 32
  int col, col_x;  // transposing reads: row 4 h + i / 4, columns 16 (l / 16 % 2) + 4 (i % 4), i = l % 16
};

template <int DP>
__device__ __forceinline__ TileLane tile_lane(int lane) {
  const int r = lane & 31, h = lane >> 5, i = lane & 15, q = 4 * h + (i >> 2);
  const int c = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
  if constexpr (DP == 128)  // f leaves the low bits of a chunk's number alone
    return {row_place<DP>(r) + h * 16, row_xor<DP>(r) * 16, row_place<DP>(q) + c * 16 + (i & 1) * 8, row_xor<DP>(q) * 16};
  return {row_place<DP>(r), (h ^ row_xor<DP>(r)) * 16, row_place<DP>(q) + (i & 1) * 8, (c ^ row_xor<DP>(q)) * 16};
}

// First operand of a score product: chunk 2 s + h of rows row0 + l % 32 (row0 a multiple of 32).
template <int DP>
__device__ __forceinline__ u32x4 read_rows(const char* tile, int row0, int s, const TileLane& at) {
  const char* p = tile + row_place<DP>(row0) + at.row;
  if constexpr (DP == 128) return *reinterpret_cast<const u32x4*>(p + (s & 1) * 32 + (at.row_x ^ (s >> 1) << 6));
  else return *reinterpret_cast<const u32x4*>(p + (at.row_x ^ s << 5));
}

// First operand of a product over streamed rows: columns 32 db + l % 32 of rows
// row0 + {4 h + 0..3, 8 + 4 h + 0..3} (row0 a multiple of 16). A 16-lane group reads 4 rows x
// 16 columns and gets them transposed (lane i: column i).
template <int DP>
__device__ __forceinline__ u32x4 read_columns(const char* tile, int row0, int db, const TileLane& at) {
  const char* p = tile + row_place<DP>(row0) + at.col;
  const int x = at.col_x ^ db << 6, y = DP == 128 ? x : x ^ 32;  // f(row + 8) = f(row), or f(row) ^ 2
  typedef __attribute__((address_space(3))) s16x4* lds4;
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + x));
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + row_place<DP>(8) + y));
  const u32x2 u = __builtin_bit_cast(u32x2, a), v = __builtin_bit_cast(u32x2, b);
  return u32x4{u[0], u[1], v[0], v[1]};
}

// v_maximum3_f32 by pairs. (fmaxf first quiets both operands, a vector operation each.) NaN
// if one is: such a row's output is NaN whatever its reference.
__device__ __forceinline__ float larger(float x, float y) { return __builtin_elementwise_maximum(x, y); }

// The values of the two lanes (l, l ^ 32) that hold one owned row.
__device__ __forceinline__ void both_halves(float x, float& lo, float& hi) {
  const uint32_t a = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  const uint32_t r0 = r[0], r1 = r[1];  // a bit cast of r[1] itself would read r[0]
  lo = __builtin_bit_cast(float, r0), hi = __builtin_bit_cast(float, r1);
}
__device__ __forceinline__ float half_max(float x) {
  float lo, hi;
  both_halves(x, lo, hi);
  return fmaxf(lo, hi);
}
__device__ __forceinline__ float half_sum(float x) {
  float lo, hi;
  both_halves(x, lo, hi);
  return lo + hi;
}

struct Segment {
  int b, tile;          // segment and the workgroup's tile of it
  int lq, lk, room;     // queries, keys in use, keys there are
  int64_t q0, k0;       // first row of the segment among all queries / keys
};

__device__ __forceinline__ int clamp_offset(int v, int64_t total) {
  return v < 0 ? 0 : (v > total ? static_cast<int>(total) : v);
}

// Lengths and first rows of segment b. Offsets are clamped to the rows there are, so no
// offset can lead outside the tensors. Rows outside the offsets are segments too, -1 in front
// and `batch` behind, whose keys are not in use: their outputs and gradients are zeros.
__device__ __forceinline__ void segment_rows(const AttnArgs& a, Segment& s) {
  const bool front = s.b < 0, back = s.b >= a.batch;
  const int from = front ? 0 : s.b, to = back ? a.batch : s.b + 1;
  if (a.cu_q != nullptr) {
    const int q0 = front ? 0 : clamp_offset(a.cu_q[from], a.total_q);
    const int q1 = back ? static_cast<int>(a.total_q) : clamp_offset(a.cu_q[to], a.total_q);
    s.q0 = q0, s.lq = q1 > q0 ? q1 - q0 : 0;
  } else {
    s.q0 = static_cast<int64_t>(s.b) * a.len_q, s.lq = a.len_q;
  }
  if (a.cu_k != nullptr) {
    const int k0 = front ? 0 : clamp_offset(a.cu_k[from], a.total_k);
    const int k1 = back ? static_cast<int>(a.total_k) : clamp_offset(a.cu_k[to], a.total_k);
    s.k0 = k0, s.room = k1 > k0 ? k1 - k0 : 0, s.lk = front || back ? 0 : s.room;
  } else {
    s.k0 = static_cast<int64_t>(s.b) * a.len_k, s.room = a.len_k, s.lk = front || back ? 0 : a.len_k;
    if (a.lens_k != nullptr && s.lk > 0) {
      const int n = a.lens_k[s.b];
      s.lk = n < 0 ? 0 : (n < s.lk ? n : s.lk);
    }
  }
}

// Slots of a launch over packed rows: see find_segment.
inline int64_t packed_slots(int64_t total, int64_t rows, int tile, int batch) { return total * rows / tile + batch + 2; }

// Which segment and tile slot `slot` is. Segment b, from -1 (the rows in front of the offsets)
// to batch (those behind), owns the slots from floor(cu[b] * rows / T) + b + 1 to those of b + 1
// (cu[-1] = 0): at least ceil(length * rows / T) of them and at most one more, so the launch
// needs only the total, and nothing is built beforehand. The segment is found by 64-way search,
// first around the place an even split gives.
// FIRST: every segment's first tile has a slot of its own, slot b + 1, which needs no search; the
// others follow from batch + 2 on, segment b's from floor(cu[b] * rows / T).
template <bool FIRST = false>
__device__ __forceinline__ void find_segment(const int32_t* cu, int len, int batch, int64_t total, int rows, int tile,
                                             int slot, Segment& s) {
  if (cu == nullptr) {
    const int per = static_cast<int>((static_cast<int64_t>(len) * rows + tile - 1) / tile);
    s.b = slot / per, s.tile = slot - s.b * per;
    return;
  }
  if constexpr (FIRST) {
    if (slot < batch + 2) {
      s.b = slot - 1, s.tile = 0;
      return;
    }
    slot -= batch + 2;
  }
  const int lane = threadIdx.x & 63;
  auto first = [&](int b) {
    return static_cast<int>(static_cast<int64_t>(clamp_offset(cu[b], total)) * rows / tile) + (FIRST ? 0 : b + 1);
  };
  int lo = 0, hi = batch + 1;  // lo is 0 or first(lo) <= slot; the answer is below hi
  if (batch > 64) {
    const int64_t all = total * rows / tile + (FIRST ? 0 : batch + 2);
    int at = static_cast<int>(static_cast<int64_t>(slot) * batch / (all > 0 ? all : 1)) - 32;
    at = at < 0 ? 0 : (at > batch - 64 ? batch - 64 : at);
    const uint64_t le = __ballot(first(at + lane) <= slot);
    if (le == ~0ull) lo = at + 63;
    else if (le == 0) hi = at;
    else lo = at + 63 - __builtin_clzll(le), hi = lo + 1;
  }
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64;
    const int at = lo + lane * step;
    const uint64_t le = __ballot(at < hi && first(at < hi ? at : lo) <= slot);  // bit 0 is set unless lo is 0
    lo += (63 - __builtin_clzll(le | 1)) * step;
    hi = lo + step < hi ? lo + step : hi;
  }
  s.b = __builtin_amdgcn_readfirstlane(lo);
  s.tile = slot - first(s.b) + (FIRST ? 1 : 0);
  if (s.tile < (FIRST ? 1 : 0)) s.b = -1, s.tile = slot + (FIRST ? 1 : 0);  // in front of all offsets
}

__device__ __forceinline__ void split_row(const AttnArgs& a, int r, int& i, int& g) {
  i = a.group == 1 ? r : static_cast<int>(__umulhi(static_cast<uint32_t>(r), a.group_magic));
  g = r - i * a.group;
}

// The lane, formed anew: what follows from it is not kept in registers across the tile loop,
// where a spilled register's reload would also wait for the tile loads in flight.
__device__ __forceinline__ int fresh_lane() {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  return lane;
}

// Chunk of an LDS tile that a lane loads in step i: row and (unswizzled) chunk. A wave's 64
// lanes fill 1024 bytes of the tile in order.
template <int DP, int NW>
__device__ __forceinline__ void tile_chunk(int i, int wave, int lane, int& row, int& c) {
  constexpr int CH = DP / 8, STEP = 64 * NW / CH;
  if constexpr (64 * NW % CH == 0 && STEP % 16 == 0) {  // the same chunk of rows STEP apart
    const int u = wave * 64 + lane;
    row = u / CH, c = (u % CH) ^ row_xor<DP>(row);
    row += i * STEP;
  } else {
    const int u = (wave + i * NW) * 64 + lane;
    row = u / CH, c = (u % CH) ^ row_xor<DP>(row);
  }
}

// 16 bytes a lane straight to LDS; ONCE: past the caches.
template <bool ONCE>
__device__ __forceinline__ void load_chunk(const void* src, char* to) {
  __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)(to), 16, 0, ONCE ? 2 : 0);
}

// Copies a tile of 64 keys and their values from x and y on straight to LDS; row r comes from
// row of(r). Chunks past the head size are left out (Z): they were zeroed once.
template <int DP, int NW, bool Z, bool ONCE, typename F>
__device__ __forceinline__ void load_pair(const char* x, int64_t x_n, const char* y, int64_t y_n, int dim, char* tile,
                                          int wave, int lane, F of) {
  static_assert(DP / 8 % NW == 0, "the waves share a tile's loads evenly");
  const uint32_t xs = static_cast<uint32_t>(x_n) * 2, ys = static_cast<uint32_t>(y_n) * 2;
#pragma unroll
  for (int i = 0; i < DP / 8 / NW; ++i) {
    int row, c;
    tile_chunk<DP, NW>(i, wave, lane, row, c);
    if (Z && c * 8 >= dim) continue;
    const uint32_t from = of(row);
    char* to = tile + (wave + i * NW) * kBlock<DP>;
    load_chunk<ONCE>(x + (from * xs + c * 16), to);
    load_chunk<ONCE>(y + (from * ys + c * 16), to + kTile<DP>);
  }
}

// Lanes that see key j (lane half 0) or j + 4 (half 1) of a tile whose visible keys are `bits`:
// a mask in scalar registers, so that a hidden key costs one vector select an element.
__device__ __forceinline__ bool sees_key(uint64_t bits, int j) {
  const uint64_t lo = (bits >> j) & 1 ? 0xffffffffull : 0, hi = (bits >> (j + 4)) & 1 ? 0xffffffffull << 32 : 0;
  return __builtin_amdgcn_inverse_ballot_w64(lo | hi);
}

// Writes 32 accumulated rows (lane l: row l % 32, columns 32 d + 8 e + 4 (l / 32) ..) times
// `by` as T. The lane halves exchange every second group of 4 columns, so that each stores 8
// adjacent ones.
template <typename T, int DP>
__device__ __forceinline__ void store_row(T* to, int dim, int h, const f32x16* acc, int step, float by) {
  typedef T t4 __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      t4 x, y;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = static_cast<T>(acc[d * step][4 * e + j] * by);
        y[j] = static_cast<T>(acc[d * step][4 * e + 4 + j] * by);
      }
      const u32x2 a = __builtin_bit_cast(u32x2, x), b = __builtin_bit_cast(u32x2, y);
      const uint32_t a0 = a[0], a1 = a[1], b0 = b[0], b1 = b[1];
      const auto p = __builtin_amdgcn_permlane32_swap(a0, b0, false, false);
      const auto q = __builtin_amdgcn_permlane32_swap(a1, b1, false, false);
      const uint32_t p0 = p[0], p1 = p[1], q0 = q[0], q1 = q[1];
      const int c = 32 * d + 8 * (e + h);
      if (c < dim) *reinterpret_cast<u32x4*>(to + c) = u32x4{p0, q0, p1, q1};
    }
}

// Launches kKernel, which may take more than 64 KB of LDS (asked for once a device).
template <auto kKernel>
int launch_tiles(const AttnArgs& a, int64_t blocks, int threads, size_t lds, hipStream_t stream) {
  static uint64_t asked = 0;
  if (lds > 65536) {
    int dev = 0;
    HI3D_HIP_CHECK(hipGetDevice(&dev));
    if (dev >= 64 || !(__atomic_load_n(&asked, __ATOMIC_RELAXED) >> dev & 1)) {
      HI3D_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kKernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(lds)));
      if (dev < 64) __atomic_fetch_or(&asked, 1ull << dev, __ATOMIC_RELAXED);
    }
  }
  hipLaunchKernelGGL(kKernel, dim3(static_cast<unsigned>(blocks)), dim3(threads), lds, stream, a);
  HI3D_LAUNCH_CHECK();
  return HI3D_OK;
}

// Masked keys: each tile has 64 numbers beside it in LDS, 0 for a key that is seen and
// -infinity for one that is not, from which the score products start. Costs 8 reads of LDS a
// tile, where selects cost 3 vector operations a score (or 8 scalar ones).
__device__ __forceinline__ void store_bias(float* bias, uint64_t bits, int lane) {
  bias[lane] = (bits >> lane) & 1 ? 0.0f : -INFINITY;
}
__device__ __forceinline__ f32x16 read_bias(const float* bias, int n, int h) {
  f32x16 x;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(bias + 32 * n + 8 * g + 4 * h);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[4 * g + e] = v[e];
  }
  return x;
}
constexpr int kBiasBytes = 2 * kKT * 4;

// Zeroes LDS tiles, for heads that do not fill their rows. Ends with a barrier.
__device__ __forceinline__ void clear_tiles(char* smem, int bytes) {
  for (int i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16) *reinterpret_cast<u32x4*>(smem + i) = u32x4{0, 0, 0, 0};
  __syncthreads();
}

// Every wave's tile loads have landed and its reads of the other tile are done. The wait is
// explicit: a wave that skips a tile runs none of the reads that the compiler waits before,
// and a workgroup of one wave has no barrier at all.
__device__ __forceinline__ void tile_barrier() {
  wait_vmcnt<0>();
  __syncthreads();
}

}  // namespace hi3d
