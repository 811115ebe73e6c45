// Rotary positions of token heads: pairs of a head's values turned by angles that grow with
// the token's positions, forward (t) and gradient (-t), for queries and keys in one launch.
#include <type_traits>

#include "common.h"

namespace hi3d {
namespace {

struct RotaryArgs {
  const void* x[2];
  void* y[2];
  int64_t row[2], head[2];  // strides of x in elements
  int heads[2];
  int64_t n;
  int dim, rot, axes;
  const void* positions;
  int64_t p_row, p_axis;
  const double* freqs;
  float scale, turn;  // turn = 1, or -1 for the gradient
  int units;          // units of a head (see below)
  uint32_t units_magic;
  int tokens;         // tokens of a workgroup
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Chunk {
  T v[V];
};

// A chunk that is read once: past the caches, which keep what is written for its reader.
template <typename C, typename T>
__device__ __forceinline__ C load_once(const T* p) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  if constexpr (sizeof(C) == 16) return __builtin_bit_cast(C, __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p)));
  else return *reinterpret_cast<const C*>(p);
}

// A workgroup takes `tokens` tokens. It first forms cos and sin of their rot / 2 angles,
// once for all heads: the angle in fp64, reduced to half a turn before it is rounded (an
// angle of 10^5 radians would keep 2 digits in fp32), then sine and cosine in fp32 in LDS.
// The heads then move as units of one 16-byte chunk (interleaved; or a copied chunk past
// rot) or two (a half-layout unit is chunk c of the first half and of the second), so each
// value is read and written once. V is 1 where sizes, strides or pointers do not allow
// 16-byte chunks. Bound by HBM: 20,011 tokens x 66 heads x 64 fp16 by three axes in 76 us (4.5
// TB/s; 82 with loads through the caches), 65,536 x 40 x 128 bf16 in 278 us (4.8); one token
// in 3 us.
template <typename T, typename P, int V, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  extern __shared__ float2 turns[];  // [tokens][rot / 2]
  const int pairs = a.rot / 2;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * a.tokens;
  const int count = static_cast<int>(a.n - first < a.tokens ? a.n - first : a.tokens);
  for (int j = threadIdx.x; j < count * pairs; j += 256) {
    const int t = j / pairs, p = j - t * pairs;
    const P* pos = static_cast<const P*>(a.positions) + (first + t) * a.p_row;
    double angle = 0.0;
    for (int x = 0; x < a.axes; ++x) angle += static_cast<double>(pos[x * a.p_axis]) * a.freqs[x * pairs + p];
    angle *= 0.15915494309189533577;  // 1 / (2 pi)
    const float f = static_cast<float>(angle - rint(angle));
    float sn, cs;
    sincospif(2.0f * f, &sn, &cs);
    turns[j] = float2{cs * a.scale, sn * a.scale * a.turn};
  }
  __syncthreads();
  // Units of a head: [0, turned) turn, the rest copies. A scalar interleaved unit is a pair.
  const int half = a.rot / 2;
  const int turned = INTERLEAVED ? (V > 1 ? a.rot / V : half) : half / V;
  const int heads = a.heads[0] + a.heads[1], all = heads * a.units;
  typedef Chunk<T, V> C;
  for (int t = 0; t < count; ++t) {
    const float2* w = turns + t * pairs;
    for (int u = threadIdx.x; u < all; u += 256) {
      int h = a.units == 1 ? u : static_cast<int>(__umulhi(static_cast<uint32_t>(u), a.units_magic));
      const int c = u - h * a.units;
      const int which = h >= a.heads[0];
      h -= which ? a.heads[0] : 0;
      const T* x = static_cast<const T*>(a.x[which]) + (first + t) * a.row[which] + h * a.head[which];
      T* y = static_cast<T*>(a.y[which]) + ((first + t) * a.heads[which] + h) * a.dim;
      if (c >= turned) {
        const int d = a.rot + (c - turned) * V;
        *reinterpret_cast<C*>(y + d) = load_once<C>(x + d);
      } else if constexpr (!INTERLEAVED || V == 1) {
        const int d0 = INTERLEAVED ? 2 * c : c * V, d1 = INTERLEAVED ? d0 + 1 : d0 + half;
        C p = load_once<C>(x + d0), q = load_once<C>(x + d1);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float2 r = w[c * V + e];
          const float f = static_cast<float>(p.v[e]), g = static_cast<float>(q.v[e]);
          p.v[e] = static_cast<T>(f * r.x - g * r.y);
          q.v[e] = static_cast<T>(f * r.y + g * r.x);
        }
        *reinterpret_cast<C*>(y + d0) = p;
        *reinterpret_cast<C*>(y + d1) = q;
      } else {
        C p = load_once<C>(x + c * V);
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
          const float2 r = w[c * (V / 2) + e];
          const float f = static_cast<float>(p.v[2 * e]), g = static_cast<float>(p.v[2 * e + 1]);
          p.v[2 * e] = static_cast<T>(f * r.x - g * r.y);
          p.v[2 * e + 1] = static_cast<T>(f * r.y + g * r.x);
        }
        *reinterpret_cast<C*>(y + c * V) = p;
      }
    }
  }
}

template <typename T, typename P, int V, bool INTERLEAVED>
int launch_rotary(RotaryArgs a, hipStream_t stream) {
  const int half = a.rot / 2;
  a.units = (INTERLEAVED ? (V > 1 ? a.rot / V : half) : half / V) + (a.dim - a.rot) / V;
  a.units_magic = a.units > 1 ? static_cast<uint32_t>(((1ull << 32) + a.units - 1) / a.units) : 0;
  // about 8 units a thread, so that the angles' latency is paid once for several tokens
  const int all = (a.heads[0] + a.heads[1]) * a.units;
  int tokens = 2048 / (all > 0 ? all : 1);
  tokens = tokens < 1 ? 1 : (tokens > 16 ? 16 : tokens);
  a.tokens = tokens;
  const size_t lds = static_cast<size_t>(tokens) * half * sizeof(float2);
  const int64_t blocks = ceil_div(a.n, tokens);
  HI3D_REQUIRE(blocks < (1ll << 31), "too many tokens for one launch");
  hipLaunchKernelGGL((rotary_kernel<T, P, V, INTERLEAVED>), dim3(static_cast<unsigned>(blocks)), dim3(256), lds,
                     stream, a);
  HI3D_LAUNCH_CHECK();
  return HI3D_OK;
}

template <typename T, typename P>
int launch_rotary_type(const RotaryArgs& a, bool interleaved, hipStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const int grain = interleaved ? a.rot : a.rot / 2;
  bool wide = a.dim % V == 0 && a.rot % V == 0 && grain % V == 0;
  for (int i = 0; i < 2; ++i) {
    if (a.heads[i] == 0) continue;
    wide = wide && a.row[i] % V == 0 && a.head[i] % V == 0 &&
           (reinterpret_cast<uintptr_t>(a.x[i]) | reinterpret_cast<uintptr_t>(a.y[i])) % 16 == 0;
  }
  if (wide) return interleaved ? launch_rotary<T, P, V, true>(a, stream) : launch_rotary<T, P, V, false>(a, stream);
  return interleaved ? launch_rotary<T, P, 1, true>(a, stream) : launch_rotary<T, P, 1, false>(a, stream);
}

template <typename T>
int launch_rotary_positions(const RotaryArgs& a, int position_dtype, bool interleaved, hipStream_t stream) {
  return position_dtype == HI3D_I64 ? launch_rotary_type<T, int64_t>(a, interleaved, stream)
                                    : launch_rotary_type<T, int32_t>(a, interleaved, stream);
}

}  // namespace
}  // namespace hi3d

using namespace hi3d;

extern "C" {

int hi3d_rotary(const void* const x[2], void* const y[2], const int32_t heads[2], const int64_t x_strides[4],
                int32_t dtype, int64_t n, int32_t dim, int32_t rot, const void* positions, int32_t position_dtype,
                int64_t position_row, int64_t position_axis, int32_t axes, const double* freqs, int32_t interleaved,
                int32_t inverse, float scale, void* stream_) {
  HI3D_REQUIRE(x && y && heads && x_strides, "null pointer argument");
  HI3D_REQUIRE(dtype == HI3D_F32 || dtype == HI3D_F16 || dtype == HI3D_BF16, "rotary takes fp32, fp16 or bf16 (got type %d)",
               dtype);
  HI3D_REQUIRE(position_dtype == HI3D_I32 || position_dtype == HI3D_I64, "positions must be int32 or int64");
  HI3D_REQUIRE(n >= 0 && heads[0] >= 0 && heads[1] >= 0 && heads[0] <= 2048 && heads[1] <= 2048, "bad sizes");
  HI3D_REQUIRE(dim > 0 && dim <= 1024, "head size must be 1 to 1024 (got %d)", dim);
  HI3D_REQUIRE(rot >= 0 && rot % 2 == 0 && rot <= dim, "%d turned values of %d: must be even and at most the head size",
               rot, dim);
  HI3D_REQUIRE(axes >= 1 && axes <= 4, "1 to 4 position axes (got %d)", axes);
  if (n == 0 || heads[0] + heads[1] == 0) return HI3D_OK;
  HI3D_REQUIRE((positions && freqs) || rot == 0, "null pointer argument");
  RotaryArgs a{};
  for (int i = 0; i < 2; ++i) {
    if (heads[i] == 0) continue;
    HI3D_REQUIRE(x[i] && y[i], "null pointer argument");
    a.x[i] = x[i], a.y[i] = y[i], a.heads[i] = heads[i];
    a.row[i] = x_strides[2 * i], a.head[i] = x_strides[2 * i + 1];
  }
  a.n = n, a.dim = dim, a.rot = rot, a.axes = axes, a.positions = positions, a.p_row = position_row;
  a.p_axis = position_axis, a.freqs = freqs, a.scale = scale, a.turn = inverse ? -1.0f : 1.0f;
  hipStream_t stream = as_stream(stream_);
  switch (dtype) {
    case HI3D_F32: return launch_rotary_positions<float>(a, position_dtype, interleaved != 0, stream);
    case HI3D_F16: return launch_rotary_positions<_Float16>(a, position_dtype, interleaved != 0, stream);
    default: return launch_rotary_positions<__bf16>(a, position_dtype, interleaved != 0, stream);
  }
}

}  // extern "C"
