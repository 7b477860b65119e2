// top_keys.h - the first n tokens of logit rows in order, by thresholds found with ballots (soc_logprobs, soc_beam_select).
#pragma once

#include "device_common.h"

namespace soc {
namespace {

constexpr int kMaxTop = 64;
constexpr int kThreads = 256;  // of a block

// Order of logits as unsigned words: NaNs first, then by value, both zeros alike; never 0 nor all ones. A 16-bit logit's
// order is in the upper half.
constexpr uint32_t kOrderNan = 0xffff0000u;  // above +inf's 0xff800000 (16 bits: 0xfc000000)
template <typename T>
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return kOrderNan;
  uint32_t b = __float_as_uint(x + 0.0f);
  if constexpr (sizeof(T) == 2) b = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<f16>(x + 0.0f))) << 16;
  const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
  return sizeof(T) == 2 ? o & 0xffff0000u : o;
}
template <typename T>
__device__ __forceinline__ float value_of(uint32_t o) {
  if (o == kOrderNan) return __builtin_nanf("");
  const uint32_t b = o & 0x80000000u ? o & 0x7fffffffu : ~o;
  if constexpr (sizeof(T) == 2) return static_cast<float>(__builtin_bit_cast(f16, static_cast<uint16_t>(b >> 16)));
  return __uint_as_float(b);
}
// Order of tokens: by logit, then by lowest id. Distinct for every token of a row; 0 is below all of them.
constexpr int kMaxVocab = 1 << 20;
__device__ __forceinline__ uint32_t low_of(int id) { return static_cast<uint32_t>(kMaxVocab - id); }  // 1 .. 2^20
template <typename T>
__device__ __forceinline__ uint64_t key_of(float x, int id) {
  return static_cast<uint64_t>(order_of<T>(x)) << 32 | low_of(id);
}

// How many of the wave's words, K a lane, are not below x.
template <int K>
__device__ __forceinline__ int reaching(const uint32_t (&w)[K], uint32_t x) {
  int c = 0;
#pragma unroll
  for (int j = 0; j < K; ++j) c += __popcll(__ballot(w[j] >= x));
  return c;
}
// Largest and smallest word of the wave (DPP within rows of 16, then the four rows).
template <typename F>
__device__ __forceinline__ uint32_t wave_fold(uint32_t v, F f) {
  v = f(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0xB1, 0xF, 0xF, true)));
  v = f(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x4E, 0xF, 0xF, true)));
  v = f(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x141, 0xF, 0xF, true)));
  v = f(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x140, 0xF, 0xF, true)));
  const auto row = [&](int lane) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane)); };
  return __builtin_amdgcn_readfirstlane(f(f(row(0), row(16)), f(row(32), row(48))));
}
// The largest x with bits from `low` up that at least n <= 64 K of the wave's words reach (0 where fewer are above 0), by
// bisection with ballots from the first bit in which the words differ. Ends as soon as exactly n reach it: *exact. That
// is after about ten bits of the orders of ordinary logits.
template <int K>
__device__ __forceinline__ uint32_t nth_word(const uint32_t (&w)[K], int n, int low, bool* exact) {
  uint32_t most = w[0], least = w[0];
#pragma unroll
  for (int j = 1; j < K; ++j) {
    most = max(most, w[j]);
    least = min(least, w[j]);
  }
  most = wave_fold(most, [](uint32_t x, uint32_t y) { return max(x, y); });
  least = wave_fold(least, [](uint32_t x, uint32_t y) { return min(x, y); });
  const uint32_t differ = most ^ least;
  const int top = differ == 0 ? -1 : 31 - __builtin_clz(differ);
  // the bits that all words share: 64 bits, so that the shift by 32 is one
  uint32_t t = most & static_cast<uint32_t>(~0ull << (top + 1));
  *exact = false;
  for (int bit = top; bit >= low; --bit) {
    const uint32_t x = t | 1u << bit;
    const int c = reaching(w, x);
    if (c >= n) t = x;
    if (c == n) {
      *exact = true;
      break;
    }
  }
  return t;
}
// The n-th largest of `count` <= 64 K keys (distinct, or 0 for none), by the calling wave: at least 1; where there are
// fewer than n keys, none is below it. First the orders, then the ids among equal orders.
template <typename T, int K, typename Key>
__device__ __forceinline__ uint64_t nth_largest(Key key, int count, int n) {
  constexpr int kLow = sizeof(T) == 2 ? 16 : 0;
  const int lane = threadIdx.x & (kWave - 1);
  uint32_t w[K];
#pragma unroll
  for (int j = 0; j < K; ++j)
    w[j] = j * kWave + lane < count ? static_cast<uint32_t>(key(j * kWave + lane) >> 32) : 0;
  bool exact;
  const uint32_t t = nth_word(w, n, kLow, &exact);
  if (exact) return static_cast<uint64_t>(t) << 32;
  if (t == 0) return 1;
  const int ties = n - reaching(w, t + 1);  // wanted of those of order t
#pragma unroll
  for (int j = 0; j < K; ++j) w[j] = w[j] == t ? static_cast<uint32_t>(key(j * kWave + lane)) : 0;
  return static_cast<uint64_t>(t) << 32 | nth_word(w, ties, 0, &exact);
}

// The n largest of `count` distinct keys in LDS, in order, to `first`, by all threads: each key counts the larger ones.
__device__ __forceinline__ void rank_first(const uint64_t* keys, int count, int n, uint64_t* first) {
  for (int i = threadIdx.x; i < count; i += kThreads) {
    const uint64_t key = keys[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < count; ++j) rank += keys[j] > key;
    if (rank < n) first[rank] = key;
  }
}

}  // namespace
}  // namespace soc
