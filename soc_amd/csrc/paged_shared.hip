// paged_shared.hip - attention of one token of each sequence over a paged cache, where groups of sequences begin with the same
// positions (soc_paged_attention_shared): beams, samples of one prompt, users behind one system prompt. The reference has one
// sequence (Mac/gpu/src/module/qwen_attention.mm).
//
// A column is a query head of one sequence. The keys of a group's prefix are read once for the columns of all its sequences, a
// sequence's own keys behind it for its own. What a block leaves of a column is a part: a reference m, the sum l of the weights
// 2^(t - m) (t: scores in base 2) and the sum of the weighted values; a second launch joins the parts of each (sequence, KV
// head). (Joined by the last block to add one, a prefix's blocks have up to 16 of them to join one after the other: 16 groups
// of 4 rows, 2000 common keys, took 100 us for 34.) Two ways to a part:
//   a row's own keys, and up to 16 columns of a prefix: four waves take the 32-key tiles of a chunk in turn, all with the same
//   columns, and add up their sums in LDS (16 groups of 4 rows with 4 heads each behind 2000 common keys 36.5 us, all in blocks of
//   64 columns 45.7; 24 groups of 1 to 8 rows in fp16 67 and 66);
//   up to 64 columns of a prefix: four waves with 16 columns each, whose key tiles go through LDS (256 rows behind 4096 common keys
//   133 us, with the first way alone 194).
// Keys and values are matrix operands as they come from memory:
//   scores  S [16 keys][16 columns] = K . Q^T, v_mfma_f32_16x16x32_f16: lane l holds 8 dims of key l % 16, and of column
//           l % 16. An fp32 query is an fp16 high part and what fp32 has beyond it, both added into one sum.
//   output  O^T [16 dims][16 columns] += V^T . P^T: S leaves 4 keys of each half of a 32-key tile in a lane, which are the 8
//           keys of the operand P^T. A weight's fp16 high part is cut off, the low part is the rest.
// The reference follows a score only where that gives a weight above 2^14, and then makes it 2^10: the sums are seldom
// rescaled, and no maximum is sought otherwise. l is another row of O^T, of values 1.
//
// Bound: reading keys and values once. 256 rows behind 4096 common keys with 512 of their own, 32 query and 8 KV heads of 128,
// fp32: 133 us, of which 123 reading 588 MB (4.8 TB/s; a large copy reaches 4.7); read row by row they would be 4.8 GB.
// 24 groups of ragged rows in fp16, 260 MB: 67 us, 4.4 TB/s and 7 us of joining. The products of a prefix take 8.8 us per 1000
// keys of those 256 rows, 0.96 PFLOP/s with both parts (a large fp16 product reaches 1.2): more than its reading beyond 64 rows.
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <string>

#include "device_common.h"
#include "paged_host.h"
#include "paged_math.h"

namespace soc {
namespace {

constexpr int kTile = 32;  // keys of a step
constexpr int kFew = 16, kMany = 64;  // columns of a block that takes a prefix
constexpr int kMaxParts = 64;  // of a prefix, and of a row's own keys
// A prefix worth a part of its own: 64 groups of 8 rows, 130 keys of their own, take 96 us for 106 row by row where 256 are common,
// with 128 common ones 92 for 84; 128 groups of 2 rows, 300 of their own, 96 for 87 with 256 and 82 for 72 with 128, 64 of them
// with 512 and 100 49 for 46.
constexpr int kShortest = 8 * kTile;

struct SharedArgs {
  const f16 *keys, *values;
  int64_t page_stride;
  int num_pages, page_shift, nkv, group, max_pages, n;
  const void* q;
  int64_t q_stride;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
  const int32_t *starts, *prefix;  // [groups + 1], [groups]
  int groups, max_group, max_prefix;
  float scale;
  void* out;
  int64_t out_stride;
  float* lse;
  bool wide_q;  // query rows are 32-byte aligned (16 in fp16): eight values a load
  int columns, tiles;  // of a block; blocks for the columns of a group
  Chunks prefix_chunks, own_chunks;
  int prefix_blocks;
  int most;        // parts of a (sequence, KV head): prefix_chunks.grid + own_chunks.grid
  float* part;     // [n][nkv][most][stride]: outputs, then references, then sums
  int stride;      // group * HD and 2 * group more, an even number
  int32_t* counts; // [n][nkv]: parts to join
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kMostWeight = 16384.0f, kStartBits = 10.0f;

// Reduces over the four lanes l % 16 + {0, 16, 32, 48}; every lane gets the result.
template <typename F>
__device__ __forceinline__ float across_rows(float x, F f) {
  const uint32_t u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t v = __float_as_uint(f(__uint_as_float(a[0]), __uint_as_float(a[1])));
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// The columns of a wave or block and the keys they attend to.
template <typename T>
struct Columns {
  const T* q;  // of the first row's first head of the KV head
  int64_t q_stride;
  int group;
  int first, count;      // columns first .. first + count - 1 of rows * group
  const int32_t* table;  // of the row whose pages are read
  uint32_t begin, end;   // keys; begin a multiple of 16
};

// One column tile: lane l holds column l % 16.
template <typename T, int HD>
struct Query {
  static constexpr bool kLow = sizeof(T) == 4;  // fp16 queries are their high part
  f16x8 high[HD / 32], low[kLow ? HD / 32 : 1];
  float to_log2;  // sum of products -> score in base 2; not negative
};
template <int HD>
struct Sums {
  f32x4 o[HD / 16], l;
  float m;
};

// Column `c` of the columns, times a power of two so that its fp16 parts are normal numbers, with the scale's sign.
template <typename T, int HD>
__device__ __forceinline__ void load_query(const SharedArgs& a, const Columns<T>& cols, int c, Query<T, HD>& q) {
  constexpr int KC = HD / 32;
  const int at = cols.first + min(c, cols.count - 1), r = at / cols.group;
  const T* p = cols.q + r * cols.q_stride + (at - r * cols.group) * HD + ((threadIdx.x & 63) >> 4) * 8;
  T x[KC][8];
#pragma unroll
  for (int k = 0; k < KC; ++k) {
    if (a.wide_q) {
      typedef T Q8 __attribute__((ext_vector_type(8)));
      const Q8 v = *reinterpret_cast<const Q8*>(p + k * 32);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[k][i] = v[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[k][i] = p[k * 32 + i];
    }
  }
  float big = 0.0f;
#pragma unroll
  for (int k = 0; k < KC; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) big = fmaxf(big, fabsf(static_cast<float>(x[k][i])));
  big = across_rows(big, [](float u, float v) { return fmaxf(u, v); });
  // times 2^e, by which the largest becomes 2^13 .. 2^14 (subnormal ones less, by 2^126); not where it is 0 or no number
  const int exponent = static_cast<int>(__float_as_uint(big) >> 23);
  const int e = big > 0.0f && exponent < 255 ? min(140 - exponent, 126) : 0;
  const float up = copysignf(__uint_as_float(static_cast<uint32_t>(127 + e) << 23), a.scale);
  // the power of two first: scale times log2(e) alone may pass fp32
  q.to_log2 = fabsf(a.scale) * __uint_as_float(static_cast<uint32_t>(127 - e) << 23) * kLog2e;
#pragma unroll
  for (int k = 0; k < KC; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float v = static_cast<float>(x[k][i]) * up;
      q.high[k][i] = static_cast<f16>(v);
      if constexpr (Query<T, HD>::kLow) q.low[k][i] = static_cast<f16>(v - static_cast<float>(q.high[k][i]));
    }
}

template <int HD>
__device__ __forceinline__ void clear(Sums<HD>& s) {
  s.m = -INFINITY;
  s.l = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int d = 0; d < HD / 16; ++d) s.o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
}

// The weights of a tile's scores as P^T operands, high and low parts; the reference moved and the sums rescaled where need
// be. Of a tile that `left` < 32 keys are in, the others (which repeat the last key) get weight 0.
// Scores are rounded before the reference is taken from them, as it was rounded itself: it then lies within a rounding of the
// scores' greatest, however large they are. (The exact product less the reference leaves what the reference was rounded by,
// which passes the range of a weight for scores from 2^28 on.)
template <int HD>
__device__ __forceinline__ void weigh(const f32x4 (&sc)[2], float to_log2, uint32_t left, Sums<HD>& s, f16x8& high,
                                      f16x8& low) {
#pragma clang fp contract(off)
  float t[8], p[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) t[j] = sc[j >> 2][j & 3] * to_log2;
  auto weights = [&] {
    float largest = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      p[j] = __builtin_amdgcn_exp2f(t[j] - s.m);
      largest = fmaxf(largest, p[j]);
    }
    return largest;
  };
  const float most = weights();
  if (__ballot(!(most <= kMostWeight)) != 0) {
    // a column moves by its own weights, whichever other column (of another row, as a rule) brought the wave here
    const auto larger = [](float x, float y) { return fmaxf(x, y); };
    float top = t[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) top = fmaxf(top, t[j]);
    top = across_rows(top, larger);
    const bool moves = across_rows(most, larger) > kMostWeight && top > -INFINITY;
    const float to = moves ? top - kStartBits : s.m, f = moves ? __builtin_amdgcn_exp2f(s.m - to) : 1.0f;
    s.m = to;
#pragma unroll
    for (int r = 0; r < 4; ++r) s.l[r] *= f;
#pragma unroll
    for (int d = 0; d < HD / 16; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) s.o[d][r] *= f;
    weights();
  }
  if (left < kTile) {
    const uint32_t row = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = (j >> 2) * 16 + row * 4 + (j & 3) < left ? p[j] : 0.0f;
  }
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const auto hv = __builtin_amdgcn_cvt_pkrtz(p[j], p[j + 1]);
    const auto lv = __builtin_amdgcn_cvt_pkrtz(p[j] - static_cast<float>(hv[0]), p[j + 1] - static_cast<float>(hv[1]));
    high[j] = hv[0];
    high[j + 1] = hv[1];
    low[j] = lv[0];
    low[j + 1] = lv[1];
  }
}
__device__ __forceinline__ f16x8 all_ones() {
  f16x8 v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = static_cast<f16>(1.0f);
  return v;
}

// One wave of four, 16 columns, every fourth tile; kOnce: keys that nobody else reads, past the caches (256 rows behind 4096
// common keys 133 us, else 143). Keys and values go from memory to registers, 16 bytes a lane, the next tile's on their way; of
// the 8 dims x 8 keys of values that a lane reads, v_perm_b32 makes the operand V^T, in whose rows dim d * 16 + i stands for
// dim i * (HD / 16) + d. Whether a page was none of the cache.
template <typename T, int HD, bool kOnce>
__device__ __forceinline__ bool attend_wave(const SharedArgs& a, int g, const Columns<T>& cols, Sums<HD>& s) {
  constexpr int KC = HD / 32, VD = HD / 16;
  typedef uint32_t VReg __attribute__((ext_vector_type(VD / 2)));
  const int lane = threadIdx.x & 63, col = lane & 15, row = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = static_cast<int>(cols.end - cols.begin - 1) / kTile + 1, mine = (tiles - wid + 3) / 4;
  const uint32_t mask = (1u << a.page_shift) - 1;
  const f16* keys = a.keys + (static_cast<int64_t>(g) << a.page_shift) * HD;
  const f16* values = a.values + (static_cast<int64_t>(g) << a.page_shift) * HD;
  auto within = [&](uint32_t key) { return min(key, cols.end - 1); };
  // lane l holds the page of half l % 2 of this wave's tile l / 2 (32 tiles ahead)
  bool lost = false;
  auto pages_from = [&](int first) {
    const uint32_t key = within(cols.begin + (wid + 4 * (first + (lane >> 1))) * kTile + (lane & 1) * 16);
    const int page = checked_page(cols.table[key >> a.page_shift], a.num_pages);
    lost |= page < 0;
    return max(page, 0);
  };
  int pages = pages_from(0);
  u32x4 kr[2][KC];
  VReg vr[2][4];
  // keys and values of a half tile are in one page
  auto load_keys = [&](int i) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t page = __builtin_amdgcn_readlane(pages, 2 * (i & 31) + h);
      const uint32_t key = within(cols.begin + (wid + 4 * i) * kTile + h * 16 + col);
      const f16* p = keys + page * a.page_stride + ((key & mask) * HD + row * 8);
#pragma unroll
      for (int c = 0; c < KC; ++c) kr[h][c] = kOnce ? load_stream16(p + c * 32) : load16(p + c * 32);
    }
  };
  auto load_values = [&](int i) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t page = __builtin_amdgcn_readlane(pages, 2 * (i & 31) + h);
      const f16* base = values + page * a.page_stride;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t key = within(cols.begin + (wid + 4 * i) * kTile + h * 16 + row * 4 + j);
        const auto* p = (const __attribute__((address_space(1))) VReg*)(base + ((key & mask) * HD + col * VD));
        vr[h][j] = kOnce ? __builtin_nontemporal_load(p) : *p;
      }
    }
  };
  Query<T, HD> q;
  load_query(a, cols, col, q);
  if (mine > 0) {
    load_keys(0);
    load_values(0);
  }
  clear(s);
  const f16x8 ones = all_ones();
  for (int i = 0; i < mine; ++i) {
    f32x4 sc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      if constexpr (Query<T, HD>::kLow) {
#pragma unroll
        for (int h = 0; h < 2; ++h) sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_f16x8(kr[h][c]), q.low[c], sc[h], 0, 0, 0);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_f16x8(kr[h][c]), q.high[c], sc[h], 0, 0, 0);
    }
    const bool more = i + 1 < mine;
    // pages of the next 32 tiles, before they are needed; the values of tile i are already on their way
    if (more && ((i + 1) & 31) == 0) pages = pages_from(i + 1);
    if (more) load_keys(i + 1);
    f16x8 ph, pl;
    weigh(sc, q.to_log2, cols.end - (cols.begin + (wid + 4 * i) * kTile), s, ph, pl);
#pragma unroll
    for (int d = 0; d < VD; ++d) {
      u32x4 av;
#pragma unroll
      for (int w = 0; w < 4; ++w)  // keys 2 w and 2 w + 1 of the lane's 8, dim d of its VD
        av[w] = __builtin_amdgcn_perm(vr[w >> 1][2 * (w & 1) + 1][d >> 1], vr[w >> 1][2 * (w & 1)][d >> 1],
                                      d & 1 ? 0x07060302u : 0x05040100u);
      s.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_f16x8(av), pl, s.o[d], 0, 0, 0);
      s.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_f16x8(av), ph, s.o[d], 0, 0, 0);
    }
    s.l = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pl, s.l, 0, 0, 0);
    s.l = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, ph, s.l, 0, 0, 0);
    if (more) load_values(i + 1);
  }
  return __ballot(lost) != 0;
}

// A block's four waves, 16 columns each: the keys' tiles, which are whole, go through a ring in LDS, the next two on their way
// while one's scores are formed. (Before a tile's transposing reads the compiler waits for all of them: it cannot tell the places
// that they go to from those that are read.) A tile row's 16-byte chunk c lies at slot c ^ swizzle(row), so that 16 rows read at one chunk
// reach all banks; ds_read_b64_tr_b16 gives V^T (in each 16-lane group, lane j names 4 dims of one key, and lane i receives
// dim i of 4 keys).
constexpr int kRing = 3;  // tiles in LDS
template <int HD>
struct Ring {
  f16 keys[kRing][kTile * HD], values[kRing][kTile * HD];
};
typedef __fp16 hv4 __attribute__((__vector_size__(4 * sizeof(__fp16))));  // what the transposing read gives
template <int HD>
__device__ __forceinline__ constexpr int swizzle(int row) {
  return HD == 128 ? row & 15 : (row >> 1) & 7;
}
// 16 bytes a lane from memory to LDS, lane after lane from `to` on.
__device__ __forceinline__ void load_to_lds(const f16* from, f16* to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                   (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}
// Waits until at most N of this wave's loads are on their way.
template <int N>
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | (0x7 << 4) | (0xF << 8));
}
// A barrier with no fence: loads into LDS stay on their way across it. This wave's reads of LDS are over before it (nothing else
// makes them: their results may be used behind the barrier, when other waves' loads already take the place).
__device__ __forceinline__ void block_barrier() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0) alone
  __builtin_amdgcn_s_barrier();
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}
template <typename T, int HD>
__device__ __forceinline__ bool attend_block(const SharedArgs& a, int g, const Columns<T>& cols, char* lds,
                                             Sums<HD>& s) {
  Ring<HD>& ring = *reinterpret_cast<Ring<HD>*>(lds);
  constexpr int KC = HD / 32, ND = HD / 16;
  constexpr int kChunks = HD / 8, kRows = 64 / kChunks;  // 16-byte chunks of a row; rows of a wave's load
  constexpr int kLoads = 8 / kRows;                      // of a wave's 8 rows of a tile
  const int lane = threadIdx.x & 63, col = lane & 15, row = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = static_cast<int>(cols.end - cols.begin) / kTile;
  const uint32_t mask = (1u << a.page_shift) - 1;
  // a wave loads rows 8 wid .. 8 wid + 7 of a tile, which lie in its half wid / 2; lane l holds the page of that half of
  // tile l (64 tiles ahead)
  bool lost = false;
  auto pages_from = [&](int first) {
    const uint32_t key = min(cols.begin + (first + lane) * kTile + (wid >> 1) * 16, cols.end - 1);
    const int page = checked_page(cols.table[key >> a.page_shift], a.num_pages);
    lost |= page < 0;
    return max(page, 0);
  };
  int pages = pages_from(0);
  const f16* keys = a.keys + (static_cast<int64_t>(g) << a.page_shift) * HD;
  const f16* values = a.values + (static_cast<int64_t>(g) << a.page_shift) * HD;
  auto load_tile = [&](int i, int slot) {
    if ((i & 63) == 0 && i > 0) pages = pages_from(i);
    const int64_t page = __builtin_amdgcn_readlane(pages, i & 63);
    const uint32_t place = (cols.begin + i * kTile + (wid >> 1) * 16) & mask;
    const int64_t at = page * a.page_stride + place * HD;
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      const int first = 8 * wid + n * kRows, r = first + lane / kChunks;  // of the tile
      const int off = (r & 15) * HD + ((lane % kChunks) ^ swizzle<HD>(r)) * 8;
      load_to_lds(keys + at + off, ring.keys[slot] + first * HD);
      load_to_lds(values + at + off, ring.values[slot] + first * HD);
    }
  };
  load_tile(0, 0);
  if (tiles > 1) load_tile(1, 1);
  // tile i is there, and nobody needs tile i - 1, whose place tile i + 2 takes
  auto next_tile = [&](int i, int slot) {
    if (i + 1 < tiles) wait_loads<2 * kLoads>();
    else wait_loads<0>();
    block_barrier();
    if (i + 2 < tiles) load_tile(i + 2, slot == 0 ? kRing - 1 : slot - 1);
  };
  const int mine = cols.count - wid * 16;  // columns of this wave
  if (mine <= 0) {
    for (int i = 0, slot = 0; i < tiles; ++i, slot = slot == kRing - 1 ? 0 : slot + 1) next_tile(i, slot);
    return __ballot(lost) != 0;
  }
  Query<T, HD> q;
  load_query(a, cols, wid * 16 + col, q);
  clear(s);
  const f16x8 ones = all_ones();
  // where this lane reads keys and values of a tile's first 16 rows; the next 16 have the same swizzles
  int key_at[KC], value_at[ND];
#pragma unroll
  for (int c = 0; c < KC; ++c) key_at[c] = col * HD + ((c * 4 + row) ^ swizzle<HD>(col)) * 8;
  const int vrow = row * 4 + (col >> 2);
#pragma unroll
  for (int d = 0; d < ND; ++d)
    value_at[d] = vrow * HD + ((2 * d + ((col & 3) >> 1)) ^ swizzle<HD>(vrow)) * 8 + (col & 1) * 4;
  for (int i = 0, slot = 0; i < tiles; ++i, slot = slot == kRing - 1 ? 0 : slot + 1) {
    next_tile(i, slot);
    const f16* kt = ring.keys[slot];
    const f16* vt = ring.values[slot];
    f32x4 sc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      f16x8 k[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) k[h] = *reinterpret_cast<const f16x8*>(kt + key_at[c] + h * 16 * HD);
      if constexpr (Query<T, HD>::kLow) {
#pragma unroll
        for (int h = 0; h < 2; ++h) sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[h], q.low[c], sc[h], 0, 0, 0);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[h], q.high[c], sc[h], 0, 0, 0);
    }
    f16x8 ph, pl;
    weigh(sc, q.to_log2, kTile, s, ph, pl);
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      f16x8 v;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f16* at = vt + value_at[d] + h * 16 * HD;
        const f16x4 u = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16(
                                                      (__attribute__((address_space(3))) hv4*)at));
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * h + j] = u[j];
      }
      s.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl, s.o[d], 0, 0, 0);
      s.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph, s.o[d], 0, 0, 0);
    }
    s.l = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pl, s.l, 0, 0, 0);
    s.l = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, ph, s.l, 0, 0, 0);
  }
  return __ballot(lost) != 0;
}

// A group's rows and what of its prefix is read once for them.
struct GroupOf {
  int first, count;  // rows; count 0: none
  int prefix;        // keys read once for the group: whole tiles; 0: none
};
// The group of row `row` (>= 0), or group `want`; by each wave for itself, 256 groups a trip to memory. All starts are looked at:
// where they do not ascend within the rows there are no groups, for every wave alike.
__device__ __forceinline__ GroupOf group_of(const SharedArgs& a, int row, int want) {
  const int lane = threadIdx.x & 63;
  GroupOf g{0, 0, 0};
  bool bad = false;
  for (int base = 0; base < a.groups; base += 256) {
    int32_t s[4], e[4], p[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = min(base + k * 64 + lane, a.groups - 1);
      s[k] = a.starts[i];
      e[k] = a.starts[i + 1];
      p[k] = a.prefix[i];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = base + k * 64 + lane;
      bad |= s[k] < 0 || e[k] < s[k] || e[k] > a.n;
      const uint64_t here = __ballot(i < a.groups && (row >= 0 ? s[k] <= row && row < e[k] : i == want));
      if (here != 0) {
        const int l = __builtin_ctzll(here);
        g.first = __builtin_amdgcn_readlane(s[k], l);
        g.count = min(__builtin_amdgcn_readlane(e[k], l) - g.first, a.max_group);
        g.prefix = min(__builtin_amdgcn_readlane(p[k], l), a.max_prefix) & ~(kTile - 1);
      }
    }
  }
  // a short prefix, and rows beyond max_group: all keys are the row's own. (A group of one shares nothing, but its prefix has
  // blocks, where a row's own keys have few)
  if (__ballot(bad) != 0 || g.count < 1 || g.prefix < kShortest || (row >= 0 && row >= g.first + g.count))
    return GroupOf{0, 0, 0};
  return g;
}

// Four waves' sums of the same columns over other keys, made one in LDS.
template <int HD>
struct Merge {
  float o[4][16][HD + 4];  // 4 floats behind a column's: 16-byte stores of 8 columns reach 8 bank groups
  float m[4][16], l[4][16];
};
template <int HD>
__device__ __forceinline__ void merge(const Sums<HD>& s, Merge<HD>& sh) {
  constexpr int ND = HD / 16;
  const int lane = threadIdx.x & 63, col = lane & 15, row = lane >> 4, wid = threadIdx.x >> 6;
  if (row == 0) sh.m[wid][col] = s.m;
  __syncthreads();
  const float top = fmaxf(fmaxf(sh.m[0][col], sh.m[1][col]), fmaxf(sh.m[2][col], sh.m[3][col]));
  const float f = __builtin_amdgcn_exp2f(s.m - top);  // a wave without keys has m = -inf and adds 0
  if (row == 0) sh.l[wid][col] = s.l[0] * f;
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int d = 0; d < ND; d += 4)
      *reinterpret_cast<f32x4*>(&sh.o[wid][col][(row * 4 + r) * ND + d]) =
          f32x4{s.o[d][r] * f, s.o[d + 1][r] * f, s.o[d + 2][r] * f, s.o[d + 3][r] * f};
  __syncthreads();
}
// dims d and d + 1 of a column after it; its reference and sum
template <int HD>
__device__ __forceinline__ f32x2 merged(const Merge<HD>& sh, int c, int d) {
  f32x2 x = *reinterpret_cast<const f32x2*>(&sh.o[0][c][d]);
#pragma unroll
  for (int w = 1; w < 4; ++w) {
    const f32x2 y = *reinterpret_cast<const f32x2*>(&sh.o[w][c][d]);
    x[0] += y[0];
    x[1] += y[1];
  }
  return x;
}
template <int HD>
__device__ __forceinline__ f32x2 merged_sum(const Merge<HD>& sh, int c) {
  return f32x2{fmaxf(fmaxf(sh.m[0][c], sh.m[1][c]), fmaxf(sh.m[2][c], sh.m[3][c])),
               (sh.l[0][c] + sh.l[1][c]) + (sh.l[2][c] + sh.l[3][c])};
}

// A part of a group's prefix: chunk s of it, columns from tile * kColumns on.
template <typename T, int HD, int kColumns>
__device__ __forceinline__ void prefix_part(const SharedArgs& a, int unit, char* lds) {
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.group, g = unit % a.nkv;
  int rest = unit / a.nkv;
  const int tile = rest % a.tiles;
  rest /= a.tiles;
  const int s = rest % a.prefix_chunks.grid, want = rest / a.prefix_chunks.grid;
  const GroupOf of = group_of(a, -1, want);
  if (of.prefix <= 0) return;
  const int chunk = chunk_of(of.prefix, a.prefix_chunks), c0 = s * chunk;
  Columns<T> cols;
  cols.first = tile * kColumns;
  cols.count = min(of.count * G - cols.first, kColumns);
  if (c0 >= of.prefix || cols.count <= 0) return;
  // pages are those of the first row that holds the whole prefix
  const auto holds = [&](int r) { return checked_length(a.lens[of.first + r], a.max_pages, a.page_shift) >= of.prefix; };
  int leader = -1;
  for (int base = 0; base < of.count && leader < 0; base += 64) {
    const uint64_t some = __ballot(base + lane < of.count && holds(min(base + lane, of.count - 1)));
    if (some != 0) leader = base + __builtin_ctzll(some);
  }
  if (leader < 0) return;
  cols.q = static_cast<const T*>(a.q) + of.first * a.q_stride + static_cast<int64_t>(g) * G * HD;
  cols.q_stride = a.q_stride;
  cols.group = G;
  cols.table = a.table + (of.first + leader) * a.table_stride;
  cols.begin = c0;
  cols.end = min(of.prefix, c0 + chunk);
  Sums<HD> sums;
  bool lost;
  const bool many = kColumns == kMany && cols.count > kFew;
  if constexpr (kColumns == kMany) {
    if (many) lost = attend_block<T, HD>(a, g, cols, lds, sums);
  }
  if (!many) lost = attend_wave<T, HD, false>(a, g, cols, sums);
  lost = __syncthreads_or(lost) != 0;
  const float nan = __builtin_nanf("");
  const auto part_of = [&](int r) {
    return a.part + (((of.first + r) * static_cast<int64_t>(a.nkv) + g) * a.most + s) * a.stride;
  };
  // not for a row that does not hold the prefix: it reads all its keys by itself
  if (many) {
    typedef float Four __attribute__((ext_vector_type(4), aligned(8)));
    const int c = wid * 16 + (lane & 15), at = cols.first + c, r = at / G, h = at - r * G, row = lane >> 4;
    if (c >= cols.count || !holds(r)) return;
    float* part = part_of(r);
    // past the caches, where the many parts of a block would push out what others read (256 rows behind 4096 common keys 133 us,
    // with plain stores 140, with no keys of their own 66 and 64; the parts of the other way, fewer, gain nothing so)
#pragma unroll
    for (int d = 0; d < HD / 16; ++d)
      __builtin_nontemporal_store(static_cast<Four>(sums.o[d]), reinterpret_cast<Four*>(part + h * HD + d * 16 + row * 4));
    if (row == 0) {
      part[G * HD + h] = sums.m;
      part[G * HD + G + h] = lost ? nan : sums.l[0];
    }
  } else {
    auto& sh = *reinterpret_cast<Merge<HD>*>(lds);
    merge(sums, sh);
    for (int i = threadIdx.x; i < cols.count * (HD / 2); i += 256) {
      const int c = i / (HD / 2), d = (i - c * (HD / 2)) * 2, at = cols.first + c, r = at / G, h = at - r * G;
      if (!holds(r)) continue;
      float* part = part_of(r);
      *reinterpret_cast<f32x2*>(part + h * HD + d) = merged(sh, c, d);
      if (d == 0) {
        const f32x2 y = merged_sum(sh, c);
        part[G * HD + h] = y[0];
        part[G * HD + G + h] = lost ? nan : y[1];
      }
    }
  }
}

// A part of a row's own keys, or all there is.
template <typename T, int HD>
__device__ __forceinline__ void own_part(const SharedArgs& a, int64_t unit, char* lds) {
  const int tid = threadIdx.x;
  const int G = a.group, g = unit % a.nkv;
  const int64_t rest = unit / a.nkv;
  const int b = rest % a.n, s = rest / a.n;
  const int len = checked_length(a.lens[b], a.max_pages, a.page_shift);
  if (s > 0 && s * a.own_chunks.least >= len) return;
  const GroupOf of = group_of(a, b, 0);
  const int begin = of.prefix > 0 && len >= of.prefix ? of.prefix : 0;
  const int keys = len - begin;
  const int64_t pair = static_cast<int64_t>(b) * a.nkv + g;
  const int before = begin > 0 ? chunks_of(begin, chunk_of(begin, a.prefix_chunks)) : 0;
  const int chunk = chunk_of(keys, a.own_chunks), c0 = s * chunk;
  const int count = before + chunks_of(keys, chunk);
  const bool alone = before == 0 && count <= 1;
  if (s == 0 && tid == 0) a.counts[pair] = alone ? 0 : count;
  const float nan = __builtin_nanf("");
  T* out = static_cast<T*>(a.out) + b * a.out_stride + static_cast<int64_t>(g) * G * HD;
  float* lse = a.lse != nullptr ? a.lse + pair * G : nullptr;
  if (len <= 0) {
    if (s > 0) return;
    for (int i = tid; i < G * HD; i += 256) out[i] = static_cast<T>(len < 0 ? nan : 0.0f);
    if (lse != nullptr && tid < G) lse[tid] = len < 0 ? nan : -INFINITY;
    return;
  }
  if (c0 >= keys) return;
  Columns<T> cols;
  cols.q = static_cast<const T*>(a.q) + b * a.q_stride + static_cast<int64_t>(g) * G * HD;
  cols.q_stride = 0;
  cols.group = G;
  cols.first = 0;
  cols.count = G;
  cols.table = a.table + b * a.table_stride;
  cols.begin = begin + c0;
  cols.end = min(len, begin + c0 + chunk);
  float* part = a.part + (pair * a.most + before + s) * a.stride;
  Sums<HD> sums;
  const bool lost = __syncthreads_or(attend_wave<T, HD, true>(a, g, cols, sums)) != 0;
  auto& sh = *reinterpret_cast<Merge<HD>*>(lds);
  merge(sums, sh);
  for (int i = tid; i < G * (HD / 2); i += 256) {
    const int h = i / (HD / 2), d = (i - h * (HD / 2)) * 2;
    const f32x2 x = merged(sh, h, d), y = merged_sum(sh, h);
    const float sum = lost ? nan : y[1];
    if (alone) {
      out[h * HD + d] = static_cast<T>(x[0] / sum);
      out[h * HD + d + 1] = static_cast<T>(x[1] / sum);
      if (d == 0 && lse != nullptr) lse[h] = (y[0] + __builtin_amdgcn_logf(sum)) * kLn2;
    } else {
      *reinterpret_cast<f32x2*>(part + h * HD + d) = x;
      if (d == 0) {
        part[G * HD + h] = y[0];
        part[G * HD + G + h] = sum;
      }
    }
  }
}

template <typename T, int HD, int kColumns>
__global__ __launch_bounds__(256, 3) void k_shared(SharedArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];  // Merge, or Ring if that is larger and used
  if (static_cast<int>(blockIdx.x) < a.prefix_blocks) prefix_part<T, HD, kColumns>(a, blockIdx.x, lds);
  else own_part<T, HD>(a, blockIdx.x - a.prefix_blocks, lds);
}

// A block for each (sequence, KV head) joins its parts, in order.
template <typename T, int HD>
__global__ __launch_bounds__(256) void k_shared_join(SharedArgs a) {
  extern __shared__ float weight[];  // [most][group]
  __shared__ float total[16];
  const int t = threadIdx.x, lane = t & 63, G = a.group;
  const int64_t pair = blockIdx.x, b = pair / a.nkv;
  const int count = a.counts[pair];
  if (count == 0) return;
  T* out = static_cast<T*>(a.out) + b * a.out_stride + (pair - b * a.nkv) * G * HD;
  const float* all = a.part + pair * a.most * a.stride;
  for (int i = t; i < count * G; i += 256) {
    const int u = i / G;
    weight[i] = all[static_cast<int64_t>(u) * a.stride + G * HD + (i - u * G)];
  }
  __syncthreads();
  for (int h = t >> 6; h < G; h += 4) {
    float top = -INFINITY, sum = 0.0f;
    for (int u = lane; u < count; u += 64) top = fmaxf(top, weight[u * G + h]);
    top = wave_max(top);
    for (int u = lane; u < count; u += 64) {
      const float f = __builtin_amdgcn_exp2f(weight[u * G + h] - top);
      weight[u * G + h] = f;
      sum += f * all[static_cast<int64_t>(u) * a.stride + G * HD + G + h];
    }
    sum = wave_sum(sum);
    if (lane == 0) {
      total[h] = sum;
      if (a.lse != nullptr) a.lse[pair * G + h] = (top + __builtin_amdgcn_logf(sum)) * kLn2;
    }
  }
  __syncthreads();
  typedef T T2 __attribute__((ext_vector_type(2), aligned(sizeof(T))));
  for (int i = t * 2; i < G * HD; i += 512) {
    const int h = i / HD;
    float x0 = 0.0f, x1 = 0.0f;
    for (int u0 = 0; u0 < count; u0 += 16) {  // sixteen parts on their way at a time
      f32x2 v[16];
#pragma unroll
      for (int j = 0; j < 16; ++j)
        v[j] = *reinterpret_cast<const f32x2*>(all + static_cast<int64_t>(min(u0 + j, count - 1)) * a.stride + i);
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (u0 + j < count) {
          const float f = weight[(u0 + j) * G + h];
          x0 += f * v[j][0];
          x1 += f * v[j][1];
        }
    }
    *reinterpret_cast<T2*>(out + i) = T2{static_cast<T>(x0 / total[h]), static_cast<T>(x1 / total[h])};
  }
}

template <typename T, int HD>
hipError_t launch_shared(const SharedArgs& a, hipStream_t s) {
  const uint32_t pairs = static_cast<uint32_t>(a.n) * a.nkv;
  const dim3 blocks(a.prefix_blocks + pairs * a.own_chunks.grid);
  const size_t lds = sizeof(Merge<HD>);
  if (a.columns == kFew) hipLaunchKernelGGL((k_shared<T, HD, kFew>), blocks, dim3(256), lds, s, a);
  else hipLaunchKernelGGL((k_shared<T, HD, kMany>), blocks, dim3(256), std::max(lds, sizeof(Ring<HD>)), s, a);
  const size_t weights = static_cast<size_t>(a.most) * a.group * sizeof(float);  // at most 8 KiB
  hipLaunchKernelGGL((k_shared_join<T, HD>), dim3(pairs), dim3(256), weights, s, a);
  return hipGetLastError();
}
hipError_t launch_shared(const SharedArgs& a, bool f32, int hd, hipStream_t s) {
  if (hd == 128) return f32 ? launch_shared<float, 128>(a, s) : launch_shared<f16, 128>(a, s);
  return f32 ? launch_shared<float, 64>(a, s) : launch_shared<f16, 64>(a, s);
}

}  // namespace
}  // namespace soc

extern "C" {

int soc_paged_attention_shared(soc_ctx* ctx, const soc_paged_cache* cache, const void* q, int64_t q_stride, int32_t dtype,
                               const int32_t* block_table, int64_t table_stride, int32_t max_pages,
                               const int32_t* seq_lens, int32_t n, const int32_t* group_starts,
                               const int32_t* prefix_lens, int32_t groups, int32_t max_group, int32_t max_prefix,
                               int32_t q_heads, float scale, void* out, int64_t out_stride, float* lse) {
  SOC_API_BEGIN
  SOC_TRY(soc::check_cache_shape(cache));
  if (dtype != SOC_DTYPE_F32 && dtype != SOC_DTYPE_F16)
    return soc::fail(SOC_ERR_INVALID, "shared attention: dtype must be F32 or F16");
  if (n <= 0 || n > 65535) return soc::fail(SOC_ERR_INVALID, "shared attention: 1 to 65535 sequences");
  if (max_pages <= 0 || static_cast<int64_t>(max_pages) * cache->page_size > (1 << 30))
    return soc::fail(SOC_ERR_INVALID, "shared attention: need max_pages > 0 and max_pages * page_size up to 2^30");
  if (groups <= 0 || groups > n || groups > 4096)
    return soc::fail(SOC_ERR_INVALID, "shared attention: 1 to 4096 groups, no more than sequences");
  if (max_group <= 0 || max_prefix < 0)
    return soc::fail(SOC_ERR_INVALID, "shared attention: need max_group > 0 and max_prefix >= 0");
  max_group = std::min(max_group, n);
  max_prefix = std::min(max_prefix, max_pages * cache->page_size);
  if (q_heads <= 0 || q_heads % cache->kv_heads != 0 || q_heads / cache->kv_heads > 16)
    return soc::fail(SOC_ERR_INVALID, "shared attention: query heads per KV head must be 1 to 16");
  if (!std::isfinite(scale)) return soc::fail(SOC_ERR_INVALID, "shared attention: scale must be finite");
  if (q == out && q_stride != out_stride)
    return soc::fail(SOC_ERR_INVALID, "shared attention: in place needs equal strides");
  const int64_t pairs = static_cast<int64_t>(n) * cache->kv_heads;
  if (pairs > (1 << 20)) return soc::fail(SOC_ERR_INVALID, "shared attention: sequences times KV heads beyond 2^20");
  if (ctx == nullptr) return soc::fail(SOC_ERR_INVALID, "null context");
  soc::DeviceScope device(ctx);
  soc::Operands operands(ctx);
  const int size = dtype == SOC_DTYPE_F32 ? 4 : 2, hd = cache->head_dim;
  const int64_t width = static_cast<int64_t>(q_heads) * hd;
  SOC_TRY(soc::check_cache_memory(operands, cache));
  SOC_TRY(operands.rows("shared attention queries", q, n, q_stride, width, size));
  if (out != q) SOC_TRY(operands.rows("shared attention output", out, n, out_stride, width, size));
  SOC_TRY(operands.rows("shared attention block_table", block_table, n, table_stride, max_pages, 4));
  SOC_TRY(operands.array("shared attention seq_lens", seq_lens, n, 4));
  SOC_TRY(operands.array("shared attention group_starts", group_starts, groups + 1, 4));
  SOC_TRY(operands.array("shared attention prefix_lens", prefix_lens, groups, 4));
  if (lse != nullptr) SOC_TRY(operands.rows("shared attention lse", lse, n, q_heads, q_heads, 4));
  soc::SharedArgs a{};
  a.keys = static_cast<const soc::f16*>(cache->keys);
  a.values = static_cast<const soc::f16*>(cache->values);
  a.page_stride = soc::page_stride(cache);
  a.num_pages = cache->num_pages;
  a.page_shift = soc::shift_of(cache->page_size);
  a.nkv = cache->kv_heads;
  a.group = q_heads / cache->kv_heads;
  a.max_pages = max_pages;
  a.n = n;
  a.q = q;
  a.q_stride = q_stride;
  a.table = block_table;
  a.table_stride = table_stride;
  a.lens = seq_lens;
  a.starts = group_starts;
  a.prefix = prefix_lens;
  a.groups = groups;
  a.max_group = max_group;
  a.max_prefix = max_prefix;
  a.scale = scale != 0.0f ? scale : 1.0f / std::sqrt(static_cast<float>(hd));
  a.out = out;
  a.out_stride = out_stride;
  a.lse = lse;
  a.wide_q = reinterpret_cast<uintptr_t>(q) % (8 * size) == 0 && q_stride % 8 == 0;
  const int64_t longest = static_cast<int64_t>(max_pages) * cache->page_size;
  // Where there is nothing to share, or little to read, each row's keys are read for it alone, in one launch: 4 rows of 1100
  // keys, 16 query and 8 KV heads (18 MB), 9.9 us so and 11.8 shared; 4 of 4100, 32 and 8 heads (67 MB) 15.7 and 16.2; 8 of 4160
  // (136 MB) 22.7 and 16.7. The table's width stands for the rows' lengths, which the host does not know.
  const int64_t bytes = pairs * longest * hd * 4;
  const char* always = std::getenv("SOC_PAGED_SHARED");  // =always: the tests' small sizes too
  const bool little = bytes < (int64_t{64} << 20) && !(always != nullptr && std::strcmp(always, "always") == 0);
  if (max_group < 2 || max_prefix < soc::kShortest || little)
    return soc_paged_attention_decode(ctx, cache, q, q_stride, dtype, block_table, table_stride, max_pages, seq_lens, n, q_heads,
                                      scale, out, out_stride, lse);
  a.stride = a.group * hd + 2 * a.group;
  const size_t part = static_cast<size_t>(a.stride) * sizeof(float);
  const int room = static_cast<int>(std::min<int64_t>(
      soc::kMaxParts, std::max<int64_t>(1, (int64_t{256} << 20) / static_cast<int64_t>(pairs * part))));
  const int64_t columns = static_cast<int64_t>(max_group) * a.group;
  a.columns = columns <= soc::kFew ? soc::kFew : soc::kMany;
  a.tiles = static_cast<int>((columns + a.columns - 1) / a.columns);
  const int64_t units = static_cast<int64_t>(groups) * a.nkv * a.tiles;
  // a block for each CU where there are few (parts cost: 64 rows behind 4096 common keys 26.0 us, with twice as many blocks 27.7; 16
  // groups of 4 rows behind 2000 36.5 and 38.6), and 1024 keys a block where there are many
  a.prefix_chunks = soc::chunks_for(units, max_prefix, 256, 128, 1024, room);
  if (units * a.prefix_chunks.grid > (1 << 23))
    return soc::fail(SOC_ERR_INVALID, "shared attention: too many groups of this size");
  a.prefix_blocks = static_cast<int>(units * a.prefix_chunks.grid);
  a.own_chunks = soc::chunks_for(pairs, longest, 256, 128, 1024, room);
  // what a row has behind the longest prefix: no more blocks are launched for a row than twice that takes, or 1024 for all rows
  // (256 rows behind 12000 common keys, 10 of their own: 135 us, with eight blocks a row 172). A row that shares nothing has
  // few blocks then
  const int64_t own = std::max<int64_t>(1, longest - max_prefix);
  const int64_t few = std::max<int64_t>(2 * soc::chunks_for(pairs, own, 256, 128, 1024, room).grid, 1024 / pairs);
  a.own_chunks.grid = static_cast<int32_t>(std::min<int64_t>(a.own_chunks.grid, few));
  a.most = a.prefix_chunks.grid + a.own_chunks.grid;
  const size_t parts = static_cast<size_t>(pairs) * a.most * part;
  SOC_TRY(soc::ensure_serve_ws(ctx, parts + static_cast<size_t>(pairs) * sizeof(int32_t), 0));
  a.part = reinterpret_cast<float*>(ctx->serve_ws);
  a.counts = reinterpret_cast<int32_t*>(ctx->serve_ws + parts);
  const hipError_t e = soc::launch_shared(a, size == 4, hd, ctx->stream);
  return soc::hip_status(e, "shared attention");
  SOC_API_END
}

}  // extern "C"
