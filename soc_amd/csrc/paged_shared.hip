// paged_shared.hip - attention of one token of each sequence over a paged cache, where groups of sequences begin with the same
// positions (soc_paged_attention_shared): beams, samples of one prompt, users behind one system prompt. The reference has one
// sequence (Mac/gpu/src/module/qwen_attention.mm).
//
// The keys of a group's prefix are read once for all of its sequences: a block takes 16 or 32 query columns, each a
// (sequence, head) of one KV head's group, over a chunk of the prefix. A sequence's own keys behind it are taken by blocks of
// their own, whose columns are its heads. Every block leaves for each column its maximum m, its sum l = sum 2^(t - m) and its
// output sum 2^(t - m) v (t: scores in base 2); a second launch joins a sequence's parts.
#include <algorithm>
#include <cmath>
#include <string>

#include "device_common.h"
#include "paged_host.h"
#include "paged_math.h"

namespace soc {
namespace {

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
  int columns, tiles;  // columns of a block; blocks for the columns of a group
  int prefix_splits, prefix_grid, prefix_blocks;
  int splits, grid, most;
  float* part;   // [n][nkv][prefix_grid + grid][group * (HD + 2)]: outputs, then maxima, then sums
  int32_t* parts;  // [n][nkv]: how many of them there are; -1: NaN
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kWeightBits = 14.0f;  // weights are held times 2^14
constexpr int kPrefixMost = 1024;     // keys of a prefix a block takes, where there are blocks enough
constexpr int kTile = 32;             // keys a wave takes at a time
constexpr int kNarrow = 16, kWide = 64;  // columns of a block
constexpr float kWideBits = 10.0f, kLazy = 4.0f;  // weights of a reference that may be 2^4 too low

// Reduces over the four lanes l % 16 + {0, 16, 32, 48}; every lane gets the result.
template <typename F>
__device__ __forceinline__ float across_rows(float x, F f) {
  const uint32_t u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t v = __float_as_uint(f(__uint_as_float(a[0]), __uint_as_float(a[1])));
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// The query columns of a block, or of a wave, and the keys they attend to.
template <typename T>
struct Columns {
  const T* q;       // of the first row's first head of the KV head
  int64_t q_stride;
  int group;
  int first, count;  // columns first .. first + count - 1 of rows * group
  const int32_t* table;  // of the row whose pages are read
  uint32_t begin, end;   // keys; begin a multiple of the tile
};

// Four waves take the 32-key tiles of [begin, end) in turn, each with all NT * 16 columns; they join in LDS. The keys and
// values are read once, 16 bytes a lane, and are matrix operands as they come from memory:
//   scores  S [16 keys][16 columns] = K . Q^T, v_mfma_f32_16x16x32_f16: lane l holds 8 dims of key l % 16, and of query
//           column l % 16. An fp32 query is an fp16 high part and what fp32 has beyond it, both added into one sum.
//   output  O^T [16 dims][16 columns] += V^T . P^T: S leaves 4 keys of each half tile in a lane, which are the 8 keys of
//           the operand P^T; v_perm_b32 turns the 8 x 8 block of values that a lane reads. Weights are an fp16 high and low
//           part, times 2^14 so that small ones stay normal fp16 numbers.
template <typename T, int HD, int NT>
struct AttendShared {
  float o[4][16 * NT][HD + 4];
  float m[4][16 * NT], l[4][16 * NT];
};
template <typename T, int HD, int NT>
__device__ __forceinline__ bool attend(const SharedArgs& a, int g, const Columns<T>& cols, AttendShared<T, HD, NT>& sh) {
  constexpr int KC = HD / 32, VD = HD / 16;
  constexpr bool kLow = sizeof(T) == 4;  // fp16 queries are their high part
  typedef uint32_t VReg __attribute__((ext_vector_type(VD / 2)));
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, row = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t c0 = cols.begin, len = cols.end;
  const int tiles = static_cast<int>(len - c0 - 1) / kTile + 1;
  const int mine = (tiles - wid + 3) / 4;
  const uint32_t mask = (1u << a.page_shift) - 1;
  const f16* keys = a.keys + (static_cast<int64_t>(g) << a.page_shift) * HD;
  const f16* values = a.values + (static_cast<int64_t>(g) << a.page_shift) * HD;
  auto within = [&](uint32_t key) { return min(key, len - 1); };
  // lane l holds the page of half tile l % 2 of this wave's tile l / 2 (32 tiles ahead)
  bool lost = false;
  auto pages_from = [&](int first) {
    const uint32_t key = within(c0 + (wid + 4 * (first + (lane >> 1))) * kTile + (lane & 1) * 16);
    const int page = checked_page(cols.table[key >> a.page_shift], a.num_pages);
    lost |= page < 0;
    return max(page, 0);
  };
  int pages = pages_from(0);
  u32x4 kr[2][KC];
  VReg vr[2][4];
  auto load_keys = [&](int i) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t page = __builtin_amdgcn_readlane(pages, 2 * (i & 31) + h);
      const uint32_t key = within(c0 + (wid + 4 * i) * kTile + h * 16 + col);
      const f16* p = keys + page * a.page_stride + ((key & mask) * HD + row * 8);
#pragma unroll
      for (int c = 0; c < KC; ++c) kr[h][c] = load16(p + c * 32);
    }
  };
  auto load_values = [&](int i) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t page = __builtin_amdgcn_readlane(pages, 2 * (i & 31) + h);
      const f16* base = values + page * a.page_stride;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t key = within(c0 + (wid + 4 * i) * kTile + h * 16 + row * 4 + j);
        vr[h][j] = *(const __attribute__((address_space(1))) VReg*)(base + ((key & mask) * HD + col * VD));
      }
    }
  };
  // the query columns, scaled by a power of two so that their fp16 parts are normal numbers
  f16x8 qh[NT][KC], ql[NT][kLow ? KC : 1];
  float to_log2[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int c = t * 16 + col;
    const int at = cols.first + min(c, cols.count - 1), r = at / cols.group;
    const T* p = cols.q + r * cols.q_stride + (at - r * cols.group) * HD + row * 8;
    T qr[KC][8];
#pragma unroll
    for (int k = 0; k < KC; ++k) {
      if (a.wide_q) {
        typedef T Q8 __attribute__((ext_vector_type(8)));
        const Q8 v = *reinterpret_cast<const Q8*>(p + k * 32);
#pragma unroll
        for (int i = 0; i < 8; ++i) qr[k][i] = v[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) qr[k][i] = p[k * 32 + i];
      }
    }
    float big = 0.0f;
#pragma unroll
    for (int k = 0; k < KC; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (c >= cols.count) qr[k][i] = static_cast<T>(0.0f);
        big = fmaxf(big, fabsf(static_cast<float>(qr[k][i])));
      }
    big = across_rows(big, [](float u, float v) { return fmaxf(u, v); });
    // times 2^e, by which the largest becomes 2^13 .. 2^14 (subnormal ones less, by 2^126); not where it is 0 or no number
    const int exponent = static_cast<int>(__float_as_uint(big) >> 23);
    const int e = big > 0.0f && exponent < 255 ? min(140 - exponent, 126) : 0;
    const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
    // the power of two first: scale times log2(e) alone may pass fp32
    to_log2[t] = a.scale * __uint_as_float(static_cast<uint32_t>(127 - e) << 23) * kLog2e;
#pragma unroll
    for (int k = 0; k < KC; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = static_cast<float>(qr[k][i]) * up;
        qh[t][k][i] = static_cast<f16>(v);
        if constexpr (kLow) ql[t][k][i] = static_cast<f16>(v - static_cast<float>(qh[t][k][i]));
      }
  }
  if (mine > 0) {
    load_keys(0);
    load_values(0);
  }
  float m[NT], l[NT];
  f32x4 o[NT][VD];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t] = -INFINITY;
    l[t] = 0.0f;
#pragma unroll
    for (int d = 0; d < VD; ++d) o[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  for (int i = 0; i < mine; ++i) {
    const uint32_t key0 = c0 + (wid + 4 * i) * kTile;
    f32x4 sc[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sc[t][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          if constexpr (kLow)
            sc[t][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_f16x8(kr[h][c]), ql[t][c], sc[t][h], 0, 0, 0);
          sc[t][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_f16x8(kr[h][c]), qh[t][c], sc[t][h], 0, 0, 0);
        }
      }
    const bool more = i + 1 < mine;
    if (more && ((i + 1) & 31) == 0) pages = pages_from(i + 1);
    if (more) load_keys(i + 1);
    f16x8 ph[NT], pl[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float x[8];
      float top = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float v = sc[t][h][r] * to_log2[t];
          x[4 * h + r] = key0 + h * 16 + row * 4 + r < len ? v : -INFINITY;
          top = fmaxf(top, x[4 * h + r]);
        }
      top = fmaxf(m[t], across_rows(top, [](float u, float v) { return fmaxf(u, v); }));
      const float f = __builtin_amdgcn_exp2f(m[t] - top);
      if (__ballot(top != m[t]) != 0) {
#pragma unroll
        for (int d = 0; d < VD; ++d)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[t][d][r] *= f;
      }
      m[t] = top;
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float p = __builtin_amdgcn_exp2f((x[j] - top) + kWeightBits);  // the difference first: scores may be large
        sum += p;
        ph[t][j] = static_cast<f16>(p);
        pl[t][j] = static_cast<f16>(p - static_cast<float>(ph[t][j]));
      }
      l[t] = l[t] * f + sum;
    }
#pragma unroll
    for (int d = 0; d < VD; ++d) {
      u32x4 av;
#pragma unroll
      for (int w = 0; w < 4; ++w)  // keys 2 w and 2 w + 1 of the lane's 8, dim d of its VD
        av[w] = __builtin_amdgcn_perm(vr[w >> 1][2 * (w & 1) + 1][d >> 1], vr[w >> 1][2 * (w & 1)][d >> 1],
                                      d & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_f16x8(av), pl[t], o[t][d], 0, 0, 0);
        o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_f16x8(av), ph[t], o[t][d], 0, 0, 0);
      }
    }
    if (more) load_values(i + 1);
  }
  // the four waves: brought to their common maximum, then added. A wave without a tile has m = -inf and adds 0
  if (row == 0)
#pragma unroll
    for (int t = 0; t < NT; ++t) sh.m[wid][t * 16 + col] = m[t];
  lost = __syncthreads_or(lost);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int c = t * 16 + col;
    const float top = fmaxf(fmaxf(sh.m[0][c], sh.m[1][c]), fmaxf(sh.m[2][c], sh.m[3][c]));
    const float f = __builtin_amdgcn_exp2f(m[t] - top);
    const float sum = across_rows(l[t], [](float u, float v) { return u + v; }) * f;
    if (row == 0) sh.l[wid][c] = sum;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int d = 0; d < VD; d += 4)
        *reinterpret_cast<f32x4*>(&sh.o[wid][c][(row * 4 + r) * VD + d]) =
            f32x4{o[t][d][r] * f, o[t][d + 1][r] * f, o[t][d + 2][r] * f, o[t][d + 3][r] * f};
  }
  __syncthreads();
  return lost;
}

// A group's prefix for 64 columns, 16 for each of the four waves: the keys' 32-key tiles go through LDS, the next one on its
// way while one is in use. A tile row's 16-byte chunk c lies at slot c ^ swizzle(row), so that 16 rows read at one chunk reach
// all banks; ds_read_b64_tr_b16 gives V^T (in each 16-lane group, lane j names 4 dims of one key, and lane i receives dim i of
// 4 keys). Tiles are whole. The running reference, weights 2^(t - m), follows a score only where that gives a weight above 2^14,
// and then makes it 2^10, so that the sums are seldom rescaled. A weight's fp16 high part is cut off, the low part is the rest.
template <int HD>
struct WideShared {
  f16 keys[2][kTile * HD], values[2][kTile * HD];
};
typedef __fp16 hv4 __attribute__((__vector_size__(4 * sizeof(__fp16))));  // what the transposing read gives
template <int HD>
__device__ __forceinline__ constexpr int swizzle(int row) {
  return HD == 128 ? row & 15 : (row >> 1) & 7;
}
template <typename T, int HD>
struct WideResult {
  f32x4 o[HD / 16];  // dims 16 d + 4 (lane / 16) + r of column lane % 16
  float m, l;
  bool lost;
};
template <typename T, int HD>
__device__ __forceinline__ WideResult<T, HD> attend_wide(const SharedArgs& a, int g, const Columns<T>& cols,
                                                         WideShared<HD>& sh) {
  constexpr int KC = HD / 32, ND = HD / 16;
  constexpr int kChunks = HD / 8, kRows = 64 / kChunks;  // 16-byte chunks of a row; rows of a wave's load
  constexpr int kLoads = 8 / kRows;                      // of a wave's 8 rows of a tile
  constexpr bool kLow = sizeof(T) == 4;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, row = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tiles = static_cast<int>(cols.end - cols.begin) / kTile;
  const uint32_t mask = (1u << a.page_shift) - 1;
  WideResult<T, HD> out;
  out.lost = false;
  // a wave loads rows 8 wid .. 8 wid + 7 of a tile, which lie in its half wid / 2; lane l holds the page of that half of
  // tile l (64 tiles ahead)
  auto pages_from = [&](int first) {
    const uint32_t key = min(cols.begin + (first + lane) * kTile + (wid >> 1) * 16, cols.end - 1);
    const int page = checked_page(cols.table[key >> a.page_shift], a.num_pages);
    out.lost |= page < 0;
    return max(page, 0);
  };
  int pages = pages_from(0);
  const f16* keys = a.keys + (static_cast<int64_t>(g) << a.page_shift) * HD;
  const f16* values = a.values + (static_cast<int64_t>(g) << a.page_shift) * HD;
  auto load_tile = [&](int i) {
    const int64_t page = __builtin_amdgcn_readlane(pages, i & 63);
    const uint32_t place = (cols.begin + i * kTile + (wid >> 1) * 16) & mask;
    const int64_t at = page * a.page_stride + place * HD;
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      const int first = 8 * wid + n * kRows, r = first + lane / kChunks;  // of the tile
      const int off = (r & 15) * HD + ((lane % kChunks) ^ swizzle<HD>(r)) * 8;
      __builtin_amdgcn_global_load_lds(keys + at + off, sh.keys[i & 1] + first * HD, 16, 0, 0);
      __builtin_amdgcn_global_load_lds(values + at + off, sh.values[i & 1] + first * HD, 16, 0, 0);
    }
  };
  load_tile(0);
  const int mine = cols.count - wid * 16;  // columns of this wave
  f16x8 qh[KC], ql[kLow ? KC : 1];
  float to_log2;
  {
    const int at = cols.first + min(wid * 16 + col, cols.count - 1), r = at / cols.group;
    const T* p = cols.q + r * cols.q_stride + (at - r * cols.group) * HD + row * 8;
    float v[KC][8];
    float big = 0.0f;
#pragma unroll
    for (int k = 0; k < KC; ++k) {
      if (a.wide_q) {
        typedef T Q8 __attribute__((ext_vector_type(8)));
        const Q8 x = *reinterpret_cast<const Q8*>(p + k * 32);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[k][i] = static_cast<float>(x[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[k][i] = static_cast<float>(p[k * 32 + i]);
      }
    }
#pragma unroll
    for (int k = 0; k < KC; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) big = fmaxf(big, fabsf(v[k][i]));
    big = across_rows(big, [](float x, float y) { return fmaxf(x, y); });
    const int exponent = static_cast<int>(__float_as_uint(big) >> 23);
    const int e = big > 0.0f && exponent < 255 ? min(140 - exponent, 126) : 0;
    const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
    to_log2 = fabsf(a.scale) * __uint_as_float(static_cast<uint32_t>(127 - e) << 23) * kLog2e;
    const float signed_up = copysignf(up, a.scale);  // so that larger sums are larger scores
#pragma unroll
    for (int k = 0; k < KC; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = v[k][i] * signed_up;
        qh[k][i] = static_cast<f16>(x);
        if constexpr (kLow) ql[k][i] = static_cast<f16>(x - static_cast<float>(qh[k][i]));
      }
  }
  float m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int d = 0; d < ND; ++d) out.o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  __syncthreads();  // tile 0 is there
  for (int i = 0; i < tiles; ++i) {
    if (i + 1 < tiles) {
      if (((i + 1) & 63) == 0) pages = pages_from(i + 1);
      load_tile(i + 1);
    }
    if (mine > 0) {
      const f16* kt = sh.keys[i & 1];
      const f16* vt = sh.values[i & 1];
      f32x4 sc[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sc[h] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int r = h * 16 + col;
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          const f16x8 k = *reinterpret_cast<const f16x8*>(kt + r * HD + ((c * 4 + row) ^ swizzle<HD>(r)) * 8);
          if constexpr (kLow) sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql[c], sc[h], 0, 0, 0);
          sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh[c], sc[h], 0, 0, 0);
        }
      }
      float top = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                        fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
      top = across_rows(top, [](float u, float v) { return fmaxf(u, v); }) * to_log2;
      const bool moves = top - (kWideBits + kLazy) > m;
      if (__ballot(moves) != 0) {
        const float to = moves ? top - kWideBits : m, f = moves ? __builtin_amdgcn_exp2f(m - to) : 1.0f;
        m = to;
        l *= f;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int r = 0; r < 4; ++r) out.o[d][r] *= f;
      }
      f16x8 ph, pl;
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[j >> 2][j & 3], to_log2, -m));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[j >> 2][(j & 3) + 1], to_log2, -m));
        l += p0 + p1;
        const auto hv = __builtin_amdgcn_cvt_pkrtz(p0, p1);
        const auto lv = __builtin_amdgcn_cvt_pkrtz(fmaf(static_cast<float>(hv[0]), -1.0f, p0),
                                                   fmaf(static_cast<float>(hv[1]), -1.0f, p1));
        ph[j] = hv[0];
        ph[j + 1] = hv[1];
        pl[j] = lv[0];
        pl[j + 1] = lv[1];
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        f16x8 v;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = h * 16 + row * 4 + (col >> 2), c = 2 * d + ((col & 3) >> 1);
          const f16* at = vt + r * HD + (c ^ swizzle<HD>(r)) * 8 + (col & 1) * 4;
          const hv4 w = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) hv4*)at);
          const f16x4 u = __builtin_bit_cast(f16x4, w);
#pragma unroll
          for (int j = 0; j < 4; ++j) v[4 * h + j] = u[j];
        }
        out.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl, out.o[d], 0, 0, 0);
        out.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph, out.o[d], 0, 0, 0);
      }
    }
    __syncthreads();  // tile i + 1 is there, and nobody needs tile i
  }
  out.m = m + kWeightBits;  // of weights held times 2^14, as the other parts' are
  out.l = across_rows(l, [](float u, float v) { return u + v; });
  return out;
}

// What a block finds out about the groups, in one trip: whether their starts ascend within the rows, and a group's bounds and
// prefix. `row` >= 0: the group of that row (-1 if none), else group `want`.
struct GroupOf {
  int first, count;  // rows; count 0: none
  int prefix;        // keys read once for the group: whole tiles; 0: none
};
__device__ __forceinline__ GroupOf group_of(const SharedArgs& a, int row, int want, int32_t* lds) {
  // lds [4]: the group, its bounds and prefix
  const int tid = threadIdx.x;
  if (tid == 0) lds[0] = -1;
  __syncthreads();
  bool bad = false;
  for (int i = tid; i < a.groups; i += 256) {
    const int32_t s = a.starts[i], e = a.starts[i + 1], p = a.prefix[i];
    bad |= s < 0 || e < s || e > a.n;
    if (row >= 0 ? s <= row && row < e : i == want) {
      lds[0] = i;
      lds[1] = s;
      lds[2] = e;
      lds[3] = p;
    }
  }
  if (__syncthreads_or(bad) != 0 || lds[0] < 0) return GroupOf{0, 0, 0};
  GroupOf g;
  g.first = lds[1];
  g.count = min(lds[2] - lds[1], a.max_group);
  g.prefix = min(lds[3], a.max_prefix) & ~(kTile - 1);
  // a group of one, a short prefix, and rows beyond max_group: all keys are the row's own
  if (g.count < 2 || g.prefix < 4 * kTile || (row >= 0 && row >= g.first + g.count)) return GroupOf{0, 0, 0};
  return g;
}
__device__ __forceinline__ int chunks_of(int keys, int chunk) { return keys <= 0 ? 0 : (keys - 1) / chunk + 1; }

template <typename T, int HD>
__global__ __launch_bounds__(256, 3) void k_shared(SharedArgs a) {
  union Shared {
    AttendShared<T, HD, 1> narrow;
    WideShared<HD> wide;
  };
  __shared__ alignas(16) Shared lds;
  __shared__ int32_t found[4];
  __shared__ int leader;
  __shared__ bool whole[kWide];  // whether a column's row holds the whole prefix
  __shared__ bool bad_page;
  AttendShared<T, HD, 1>& sh = lds.narrow;
  const int tid = threadIdx.x, G = a.group;
  const int stride = G * (HD + 2), all = a.prefix_grid + a.grid;
  if (static_cast<int>(blockIdx.x) < a.prefix_blocks) {
    // a group's prefix
    const int g = blockIdx.x % a.nkv;
    int rest = blockIdx.x / a.nkv;
    const int tile = rest % a.tiles;
    rest /= a.tiles;
    const int s = rest % a.prefix_grid, want = rest / a.prefix_grid;
    const GroupOf of = group_of(a, -1, want, found);
    if (of.prefix <= 0) return;
    const int chunk = attention_chunk(of.prefix, a.prefix_splits, a.prefix_grid, kPrefixMost);
    const int c0 = s * chunk;
    Columns<T> cols;
    cols.first = tile * a.columns;
    cols.count = min(of.count * G - cols.first, a.columns);
    if (c0 >= of.prefix || cols.count <= 0) return;
    // pages are those of the first row that holds the whole prefix
    if (tid == 0) {
      leader = of.count;
      bad_page = false;
    }
    if (tid < cols.count)
      whole[tid] = checked_length(a.lens[of.first + (cols.first + tid) / G], a.max_pages, a.page_shift) >= of.prefix;
    __syncthreads();
    for (int i = tid; i < of.count; i += 256)
      if (checked_length(a.lens[of.first + i], a.max_pages, a.page_shift) >= of.prefix) {
        atomicMin(&leader, i);
        break;
      }
    __syncthreads();
    if (leader == of.count) return;
    cols.q = static_cast<const T*>(a.q) + of.first * a.q_stride + static_cast<int64_t>(g) * G * HD;
    cols.q_stride = a.q_stride;
    cols.group = G;
    cols.table = a.table + (of.first + leader) * a.table_stride;
    cols.begin = c0;
    cols.end = min(of.prefix, c0 + chunk);
    if (a.columns == kWide) {
      const WideResult<T, HD> x = attend_wide<T, HD>(a, g, cols, lds.wide);
      if (x.lost) bad_page = true;
      __syncthreads();
      const int lane = tid & 63, row = lane >> 4, c = tid / 64 * 16 + (lane & 15);
      if (c >= cols.count || !whole[c]) return;
      const int at = cols.first + c, r = at / G, h = at - r * G;
      float* part = a.part + (((of.first + r) * static_cast<int64_t>(a.nkv) + g) * all + s) * stride;
#pragma unroll
      for (int d = 0; d < HD / 16; ++d)
#pragma unroll
        for (int j = 0; j < 4; j += 2)
          *reinterpret_cast<f32x2*>(part + h * HD + d * 16 + row * 4 + j) = f32x2{x.o[d][j], x.o[d][j + 1]};
      if (row == 0) {
        part[G * HD + h] = x.m;
        part[G * HD + G + h] = bad_page ? __builtin_nanf("") : x.l;
      }
      return;
    }
    const bool lost = attend<T, HD, 1>(a, g, cols, sh);
    for (int i = tid; i < cols.count * (HD / 2); i += 256) {
      const int c = i / (HD / 2), d = (i - c * (HD / 2)) * 2, at = cols.first + c, r = at / G, h = at - r * G;
      if (!whole[c]) continue;  // reads all its keys by itself
      const int64_t b = of.first + r;
      float* part = a.part + ((b * a.nkv + g) * all + s) * stride;
      f32x2 x{0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        x[0] += sh.o[w][c][d];
        x[1] += sh.o[w][c][d + 1];
      }
      *reinterpret_cast<f32x2*>(part + h * HD + d) = x;
      if (d == 0) {
        part[G * HD + h] = fmaxf(fmaxf(sh.m[0][c], sh.m[1][c]), fmaxf(sh.m[2][c], sh.m[3][c]));
        const float sum = (sh.l[0][c] + sh.l[1][c]) + (sh.l[2][c] + sh.l[3][c]);
        part[G * HD + G + h] = lost ? __builtin_nanf("") : sum;
      }
    }
    return;
  }
  // a row's own keys
  const int at = blockIdx.x - a.prefix_blocks;
  const int g = at % a.nkv, rest = at / a.nkv, b = rest % a.n, s = rest / a.n;
  const int len = checked_length(a.lens[b], a.max_pages, a.page_shift);
  const GroupOf of = group_of(a, b, 0, found);
  const int begin = of.prefix > 0 && len >= of.prefix ? of.prefix : 0;
  const int keys = len - begin;
  const int before = begin > 0 ? chunks_of(begin, attention_chunk(begin, a.prefix_splits, a.prefix_grid, kPrefixMost)) : 0;
  const int chunk = keys > 0 ? attention_chunk(keys, a.splits, a.grid, a.most) : 128;
  const int64_t pair = static_cast<int64_t>(b) * a.nkv + g;
  if (s == 0 && tid == 0) a.parts[pair] = len < 0 ? -1 : before + chunks_of(keys, chunk);
  const int c0 = s * chunk;
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
  const bool lost = attend<T, HD, 1>(a, g, cols, sh);
  float* part = a.part + (pair * all + before + s) * stride;
  for (int i = tid; i < G * (HD / 2); i += 256) {
    const int c = i / (HD / 2), d = (i - c * (HD / 2)) * 2;
    f32x2 x{0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      x[0] += sh.o[w][c][d];
      x[1] += sh.o[w][c][d + 1];
    }
    *reinterpret_cast<f32x2*>(part + c * HD + d) = x;
    if (d == 0) {
      part[G * HD + c] = fmaxf(fmaxf(sh.m[0][c], sh.m[1][c]), fmaxf(sh.m[2][c], sh.m[3][c]));
      const float sum = (sh.l[0][c] + sh.l[1][c]) + (sh.l[2][c] + sh.l[3][c]);
      part[G * HD + G + c] = lost ? __builtin_nanf("") : sum;
    }
  }
}

// One block joins the parts of a (sequence, KV head), in order.
template <typename T>
__global__ __launch_bounds__(256) void k_shared_join(SharedArgs a, int hd) {
  __shared__ float weight[256][16], sums[256][16], total[16], tops[16];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int g = blockIdx.x % a.nkv, b = blockIdx.x / a.nkv, G = a.group;
  const int64_t pair = static_cast<int64_t>(b) * a.nkv + g;
  const int count = a.parts[pair], stride = G * (hd + 2);
  T* out = static_cast<T*>(a.out) + b * a.out_stride + static_cast<int64_t>(g) * G * hd;
  float* lse = a.lse != nullptr ? a.lse + pair * G : nullptr;
  if (count <= 0) {
    const float nan = __builtin_nanf("");
    for (int i = tid; i < G * hd; i += 256) out[i] = static_cast<T>(count < 0 ? nan : 0.0f);
    if (lse != nullptr && tid < G) lse[tid] = count < 0 ? nan : -INFINITY;
    return;
  }
  const float* all = a.part + pair * (a.prefix_grid + a.grid) * stride;
  for (int i = tid; i < count * G; i += 256) {
    const int u = i / G, h = i - u * G;
    const float* p = all + static_cast<int64_t>(u) * stride + G * hd + h;
    weight[u][h] = p[0];
    sums[u][h] = p[G];
  }
  __syncthreads();
  for (int h = wid; h < G; h += 4) {
    float top = -INFINITY, sum = 0.0f;
    for (int u = lane; u < count; u += 64) top = fmaxf(top, weight[u][h]);
    top = wave_max(top);
    for (int u = lane; u < count; u += 64) {
      const float w = __builtin_amdgcn_exp2f(weight[u][h] - top);
      weight[u][h] = w;
      sum += w * sums[u][h];
    }
    sum = wave_sum(sum);
    if (lane == 0) {
      total[h] = sum;
      if (lse != nullptr) lse[h] = (top + __builtin_amdgcn_logf(sum) - kWeightBits) * kLn2;
    }
  }
  __syncthreads();
  for (int i = tid; i < G * hd / 2; i += 256) {
    const int h = 2 * i / hd;
    float x0 = 0.0f, x1 = 0.0f;
#pragma unroll 8
    for (int u = 0; u < count; ++u) {
      const f32x2 v = *reinterpret_cast<const f32x2*>(all + static_cast<int64_t>(u) * stride + 2 * i);
      x0 += weight[u][h] * v[0];
      x1 += weight[u][h] * v[1];
    }
    out[2 * i] = static_cast<T>(x0 / total[h]);
    out[2 * i + 1] = static_cast<T>(x1 / total[h]);
  }
}

template <typename T, int HD>
hipError_t launch_shared(const SharedArgs& a, hipStream_t s) {
  const uint32_t blocks = a.prefix_blocks + static_cast<uint32_t>(a.n) * a.nkv * a.grid;
  hipLaunchKernelGGL((k_shared<T, HD>), dim3(blocks), dim3(256), 0, s, a);
  hipLaunchKernelGGL((k_shared_join<T>), dim3(static_cast<uint32_t>(a.n) * a.nkv), dim3(256), 0, s, a, HD);
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
  const size_t part = static_cast<size_t>(a.group) * (hd + 2) * sizeof(float);
  const int64_t room = std::max<int64_t>(2, (int64_t{512} << 20) / static_cast<int64_t>(pairs * part));
  const bool share = max_group > 1 && max_prefix >= 4 * soc::kTile;
  if (share) {
    a.columns = max_group * a.group > soc::kNarrow ? soc::kWide : soc::kNarrow;
    a.tiles = (max_group * a.group + a.columns - 1) / a.columns;
    const int64_t units = static_cast<int64_t>(groups) * a.nkv * a.tiles;
    a.prefix_splits = static_cast<int>(std::min<int64_t>(32, (256 + units - 1) / units));
    a.prefix_grid = static_cast<int>(
        std::min({((max_prefix - int64_t{1}) / soc::kPrefixMost / a.prefix_splits + 1) * a.prefix_splits,
                  std::max<int64_t>(8, 4096 / units), (max_prefix + int64_t{127}) / 128, room / 2, int64_t{128}}));
    if (units * a.prefix_grid > (1 << 23)) return soc::fail(SOC_ERR_INVALID, "shared attention: too many groups of this size");
    a.prefix_blocks = static_cast<int>(units * a.prefix_grid);
  }
  a.splits = static_cast<int>(std::min<int64_t>(32, (256 + pairs - 1) / pairs));
  a.most = pairs >= 2 * 768 && a.group >= 4 ? 2048 : soc::kAttentionMost;
  a.grid = static_cast<int>(std::min({((longest - 1) / a.most / a.splits + 1) * a.splits,
                                      std::max<int64_t>(8, 4096 / pairs), (longest + 127) / 128, room / 2, int64_t{128}}));
  const size_t bytes = static_cast<size_t>(pairs) * (a.prefix_grid + a.grid) * part;
  SOC_TRY(soc::ensure_serve_ws(ctx, bytes + static_cast<size_t>(pairs) * 4, 0));
  a.part = reinterpret_cast<float*>(ctx->serve_ws);
  a.parts = reinterpret_cast<int32_t*>(ctx->serve_ws + bytes);
  const hipError_t e = soc::launch_shared(a, size == 4, hd, ctx->stream);
  return soc::hip_status(e, "shared attention");
  SOC_API_END
}

}  // extern "C"
