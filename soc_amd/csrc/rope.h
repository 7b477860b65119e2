// rope.h - rotary positions: the frequencies a soc_rope keeps on the device, and the rotation of one row's heads that
// soc_rope_apply and soc_paged_append share.
#pragma once

#include <algorithm>

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
__device__ __forceinline__ typename VecOf<T, W>::type load_vec(const T* p) {
  return *reinterpret_cast<const typename VecOf<T, W>::type*>(p);
}
template <typename T, int W>
__device__ __forceinline__ float element(typename VecOf<T, W>::type v, int i) {
  if constexpr (W == 1) return static_cast<float>(v);
  else return static_cast<float>(v[i]);
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

// Units a head is worked in: W pairs together (2 W values), then the values behind the rotated ones, W a unit. A unit's
// values are all read before any of them is written, and no other unit touches them: in place is fine.
__device__ __forceinline__ int rope_units(const RopeView& v, int w) {
  return v.rotary_dim / (2 * w) + (v.head_dim - v.rotary_dim) / w;
}
template <typename T, int W>
struct RopeUnit {
  typename VecOf<T, W>::type a, b;  // the pairs' first and second values (interleaved: as they lie); or a to copy
};

template <typename T, int W>
__device__ __forceinline__ RopeUnit<T, W> load_unit(const RopeView& v, const T* x, int u) {
  const int pair_units = v.rotary_dim / (2 * W);
  const bool pairs = u < pair_units;
  const int at = !pairs ? v.rotary_dim + (u - pair_units) * W : v.interleaved ? 2 * W * u : W * u;
  RopeUnit<T, W> r;
  r.a = load_vec<T, W>(x + at);
  r.b = load_vec<T, W>(x + at + (!pairs ? 0 : v.interleaved ? W : v.rotary_dim / 2));
  return r;
}

// W values of a unit as they are.
template <typename T, typename O, int W>
__device__ __forceinline__ void store_copy(const RopeUnit<T, W>& r, O* y) {
  float x[W];
#pragma unroll
  for (int i = 0; i < W; ++i) x[i] = element<T, W>(r.a, i);
  store_vec<O, W>(y, x);
}

// Unit u, rotated, to y (O: another type where y is the cache's). Every width computes the same bits: the rotation is
// written as explicit fmaf, and its fp32 results are materialised, since the compiler would otherwise fold the conversion
// of some of a unit's values into their fma (v_fma_mixlo_f16, one rounding straight to fp16) and round the others twice.
template <typename T, typename O, int W>
__device__ __forceinline__ void store_unit(const RopeView& v, const f32x2* cs, const RopeUnit<T, W>& r, O* y, int u) {
  const int pair_units = v.rotary_dim / (2 * W);
  if (u >= pair_units) {
    store_copy<T, O, W>(r, y + v.rotary_dim + (u - pair_units) * W);
    return;
  }
  float p[W], q[W];
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const f32x2 t = cs[W * u + i];
    float a = element<T, W>(r.a, i), b = element<T, W>(r.b, i);
    if (v.interleaved) {  // pair i of the 2 W values a, b
      if constexpr (W > 1) {
        a = 2 * i < W ? element<T, W>(r.a, (2 * i) % W) : element<T, W>(r.b, (2 * i) % W);
        b = 2 * i + 1 < W ? element<T, W>(r.a, (2 * i + 1) % W) : element<T, W>(r.b, (2 * i + 1) % W);
      }
    }
    p[i] = fmaf(a, t[0], -(b * t[1]));
    q[i] = fmaf(a, t[1], b * t[0]);
    if constexpr (sizeof(O) == 2) __asm__ volatile("" : "+v"(p[i]), "+v"(q[i]));
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

// Values that one load or store takes: 16 bytes where rows that start at p, `stride` elements apart, allow it.
inline bool aligned_rows(const void* p, int64_t stride, int size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * size % 16 == 0;
}
// Whether a head's units can be w wide: pairs, and the values behind them, come in w.
inline bool wide_units(const RopeView& v, int w) { return v.rotary_dim % (2 * w) == 0 && v.head_dim % w == 0; }

// Blocks a row of `units` is given: one for 256 of them while the card has CUs to spare, else one for all.
inline int row_blocks(int64_t rows, int64_t units) {
  return static_cast<int>(rows < 512 ? std::min<int64_t>((units + 255) / 256, (1024 + rows - 1) / rows) : 1);
}
constexpr int64_t kRowsALaunch = 1 << 20;  // rows of one launch: its work-items stay below 2^32

}  // namespace soc
