// rope.h - rotary positions: the frequencies a soc_rope keeps on the device, and the rotation of one row's heads that
// soc_rope_apply and soc_paged_append share.
#pragma once

#include "device_common.h"
#include "soc_hip.h"

struct soc_rope {
  soc_ctx* ctx = nullptr;
  int head_dim = 0, rotary_dim = 0;
  bool interleaved = false;
  float gain = 1.0f;         // of cosines and sines (YaRN's attention factor)
  double* turns = nullptr;   // device, [rotary_dim / 2]: turns a position (radians / 2 pi)
};

namespace soc {

constexpr int kRopeMaxDim = 1024;

// What the kernels need of a soc_rope. turns == nullptr: nothing is rotated (rotary_dim 0).
struct RopeView {
  const double* turns;
  int head_dim, rotary_dim;
  bool interleaved;
  float gain;
};

// cs[i] = {cos, sin} of pair i at `position`, for i < rotary_dim / 2, by all threads of the block (a barrier follows).
// The angle is formed in turns and in 64 bits: at position 1e6 a 32-bit product would be off by a tenth of a radian.
// Its fraction of a turn, at most a half, is exact to 2^-25 in 32 bits, 1e-7 of a radian.
__device__ __forceinline__ void rope_angles(const RopeView& v, int position, f32x2* cs) {
  for (int i = threadIdx.x; i < v.rotary_dim / 2; i += blockDim.x) {
    const double t = static_cast<double>(position) * v.turns[i];
    float s, c;
    sincospif(2.0f * static_cast<float>(t - rint(t)), &s, &c);
    cs[i] = f32x2{c * v.gain, s * v.gain};
  }
}

template <typename T, int W>
struct VecOf {
  typedef T type __attribute__((ext_vector_type(W)));
};
template <typename T>
struct VecOf<T, 1> {
  typedef T type;
};

template <typename T, int W>
__device__ __forceinline__ void load_vec(const T* p, float* x) {
  const auto v = *reinterpret_cast<const typename VecOf<T, W>::type*>(p);
  if constexpr (W == 1) {
    x[0] = static_cast<float>(v);
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) x[i] = static_cast<float>(v[i]);
  }
}

template <typename T, int W>
__device__ __forceinline__ void store_vec(T* p, const float* x) {
  typename VecOf<T, W>::type v;
  if constexpr (W == 1) {
    v = static_cast<T>(x[0]);
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = static_cast<T>(x[i]);
  }
  *reinterpret_cast<typename VecOf<T, W>::type*>(p) = v;
}

// Units a head is worked in: W pairs together (2 W values), then the values behind the rotated ones, W a unit.
__device__ __forceinline__ int rope_units(const RopeView& v, int w) {
  return v.rotary_dim / (2 * w) + (v.head_dim - v.rotary_dim) / w;
}

// Unit u of one head: x -> y (another type where y is the cache's). y may be x: a unit's values are read before any of
// them is written, and no other unit touches them.
template <typename T, typename O, int W>
__device__ __forceinline__ void rope_unit(const RopeView& v, const f32x2* cs, const T* x, O* y, int u) {
  const int pair_units = v.rotary_dim / (2 * W);
  if (u >= pair_units) {
    const int at = v.rotary_dim + (u - pair_units) * W;
    float a[W];
    load_vec<T, W>(x + at, a);
    store_vec<O, W>(y + at, a);
    return;
  }
  float a[W], b[W], p[W], q[W];
  if (v.interleaved) {
    float m[2 * W];
    load_vec<T, W>(x + 2 * W * u, m);
    load_vec<T, W>(x + 2 * W * u + W, m + W);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      a[i] = m[2 * i];
      b[i] = m[2 * i + 1];
    }
  } else {
    load_vec<T, W>(x + W * u, a);
    load_vec<T, W>(x + v.rotary_dim / 2 + W * u, b);
  }
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const f32x2 t = cs[W * u + i];
    p[i] = a[i] * t[0] - b[i] * t[1];
    q[i] = b[i] * t[0] + a[i] * t[1];
  }
  if (v.interleaved) {
    float m[2 * W];
#pragma unroll
    for (int i = 0; i < W; ++i) {
      m[2 * i] = p[i];
      m[2 * i + 1] = q[i];
    }
    store_vec<O, W>(y + 2 * W * u, m);
    store_vec<O, W>(y + 2 * W * u + W, m + W);
  } else {
    store_vec<O, W>(y + W * u, p);
    store_vec<O, W>(y + v.rotary_dim / 2 + W * u, q);
  }
}

inline RopeView view_of(const soc_rope* r, int head_dim) {
  if (r == nullptr) return RopeView{nullptr, head_dim, 0, false, 1.0f};
  return RopeView{r->turns, r->head_dim, r->rotary_dim, r->interleaved, r->gain};
}

// Whether rows of heads that start at p, `stride` elements apart, can be read and written four elements at a time.
inline bool four_wide(const void* p, int64_t stride, int size) {
  return reinterpret_cast<uintptr_t>(p) % (4 * size) == 0 && stride % 4 == 0;
}
// Whether a head's units can be four wide: pairs and the values behind them come in fours.
inline bool four_wide(const RopeView& v) { return v.rotary_dim % 8 == 0 && v.head_dim % 4 == 0; }

}  // namespace soc
