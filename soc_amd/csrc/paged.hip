// paged.hip - serving from a paged key-value cache (soc_paged_*): the pages, positions and slots of a step from the
// requests' lengths, the append of new keys and values with their rotary positions, and attention of one token of each
// sequence over its pages. The reference has one contiguous cache per sequence (Mac/gpu/src/runtime/kv_cache.mm:32-204).
#include <algorithm>
#include <cmath>
#include <string>

#include "capi_internal.h"
#include "paged_math.h"
#include "rope.h"

namespace soc {
namespace {

// ---- plan ------------------------------------------------------------------------------------------------------------
// One launch. Every block forms the same exclusive sums over the requests (rows, pages taken, pages given back) in LDS,
// so that no block waits for another, and then finds the request of each of its rows and pages by bisection. The sums
// are over at most 4096 lengths, read from L2; a second launch for them alone would cost more than repeating them. Bound
// by latency (lengths, scan, bisection, table, store): 64 requests of one row 5.8 us a call, 4.3 of them the kernel's;
// 1000 requests with 32768 rows 7.0. Beyond 1024 requests a thread holds sixteen, in 452 registers: 2000 with a row each
// take 15.1 us, 4096 with 32000 rows 19.
constexpr int kPlanThreads = 256;

struct PlanArgs {
  int n;
  const int32_t *before, *after;
  int32_t* table;
  int max_pages;
  int64_t table_stride;
  int32_t* ring;
  int num_pages, page_shift;
  const int64_t* cursors_in;
  int64_t* cursors_out;
  int32_t *row_starts, *positions, *slots;
  int max_rows;
  int32_t* status;
  int32_t* step_lens;  // nullptr: not asked for
  int* arrived;
};

// The request whose share [starts[i], starts[i + 1]) of the sums holds x, 0 <= x < starts[n].
__device__ __forceinline__ int request_of(const int32_t* starts, int n, int32_t x) {
  int lo = 0, hi = n;  // starts[lo] <= x < starts[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// kEach: requests a thread holds in registers, so that all lengths are requested at once.
template <int kEach>
__global__ __launch_bounds__(kPlanThreads) void k_paged_plan(PlanArgs a) {
  constexpr int kRoom = kEach * kPlanThreads;
  __shared__ int32_t rows[kRoom + 1], take[kRoom + 1], give[kRoom + 1];
  __shared__ int32_t had[kRoom];  // positions before the step
  __shared__ int32_t wave_total[3][kPlanThreads / kWave];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
  const int64_t head = a.cursors_in[0], tail = a.cursors_in[1];
  const int32_t head0 = ring_place(head, a.num_pages), tail0 = ring_place(tail, a.num_pages);
  // thread t holds requests [t * kEach, (t + 1) * kEach); the block scans the threads' sums
  const int first = tid * kEach;
  PlanItem item[kEach];
  {
    int32_t before[kEach], after[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      before[j] = after[j] = 0;
      if (first + j < a.n) {
        before[j] = a.before[first + j];
        after[j] = a.after[first + j];
      }
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      item[j] = plan_item(before[j], after[j], a.max_pages, a.page_shift);
      if (first + j < a.n) had[first + j] = before[j];
    }
  }
  int32_t sum[3] = {0, 0, 0};
  bool bad = false;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    bad |= item[j].bad;
    sum[0] = min(sum[0] + item[j].rows, kPlanMaxRows + 1);
    sum[1] += item[j].take;
    sum[2] += item[j].give;
  }
  int32_t incl[3] = {sum[0], sum[1], sum[2]};
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const int32_t o = __shfl_up(incl[j], d, kWave);
      if (lane >= d) incl[j] += o;
    }
  }
  if (lane == kWave - 1)
#pragma unroll
    for (int j = 0; j < 3; ++j) wave_total[j][wid] = incl[j];
  const bool any_bad = __syncthreads_or(bad) != 0;
  int32_t at[3], total[3];
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    at[j] = incl[j] - sum[j];
    total[j] = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / kWave; ++w) {
      if (w < wid) at[j] += wave_total[j][w];
      total[j] += wave_total[j][w];
    }
  }
#pragma unroll
  for (int j = 0; j < kEach; ++j)
    if (first + j < a.n) {
      rows[first + j] = at[0];
      take[first + j] = at[1];
      give[first + j] = at[2];
      at[0] += item[j].rows;
      at[1] += item[j].take;
      at[2] += item[j].give;
    }
  if (tid == 0) {
    rows[a.n] = total[0];
    take[a.n] = total[1];
    give[a.n] = total[2];
  }
  __syncthreads();
  // any words may stand there: the difference wraps, and is looked at only where both are counts
  const int64_t free_pages = static_cast<int64_t>(static_cast<uint64_t>(tail) - static_cast<uint64_t>(head));
  int status = any_bad ? SOC_PLAN_LENGTHS : 0;
  if (head < 0 || tail < 0 || free_pages < 0 || free_pages > a.num_pages) status |= SOC_PLAN_CURSORS;
  else if (free_pages + total[2] > a.num_pages) status |= SOC_PLAN_CURSORS;
  else if (total[1] > free_pages) status |= SOC_PLAN_PAGES;
  if (total[0] > a.max_rows) status |= SOC_PLAN_ROWS;

  const int64_t gid = blockIdx.x * static_cast<int64_t>(kPlanThreads) + tid;
  const int64_t stride = gridDim.x * static_cast<int64_t>(kPlanThreads);
  const int live_rows = status == 0 ? total[0] : 0;
  for (int64_t r = gid; r < a.max_rows; r += stride) {
    int position = 0, slot = -1;
    if (r < live_rows) {
      const int i = request_of(rows, a.n, static_cast<int32_t>(r));
      const int before = had[i], held = pages_of(before, a.page_shift);
      position = before + (static_cast<int>(r) - rows[i]);
      const int index = position >> a.page_shift;
      const int page = index < held ? a.table[i * a.table_stride + index]
                                    : a.ring[ring_place(head0, take[i] + (index - held), a.num_pages)];
      slot = slot_of(page, position & ((1 << a.page_shift) - 1), a.num_pages, a.page_shift);
    }
    a.positions[r] = position;
    a.slots[r] = slot;
  }
  for (int64_t i = gid; i <= a.n; i += stride) a.row_starts[i] = status == 0 ? rows[i] : 0;
  if (a.step_lens != nullptr)
    for (int64_t i = gid; i < a.n; i += stride) a.step_lens[i] = status == 0 ? a.after[i] : had[i];
  if (status == 0) {
    // entries at or behind the pages a request had are written, entries before them read: no thread reads what another
    // writes, and the ring's places from the tail on are not among those taken from the head (at most num_pages free)
    for (int64_t j = gid; j < total[1]; j += stride) {
      const int i = request_of(take, a.n, static_cast<int32_t>(j));
      const int held = pages_of(had[i], a.page_shift);
      a.table[i * a.table_stride + held + (j - take[i])] =
          a.ring[ring_place(head0, static_cast<int32_t>(j), a.num_pages)];
    }
    for (int64_t j = gid; j < total[2]; j += stride) {
      const int i = request_of(give, a.n, static_cast<int32_t>(j));
      const int keep = pages_of(had[i], a.page_shift) - (give[i + 1] - give[i]);
      a.ring[ring_place(tail0, static_cast<int32_t>(j), a.num_pages)] =
          a.table[i * a.table_stride + keep + (j - give[i])];
    }
  }
  // where cursors_out is cursors_in, the last block to have read them writes them
  if (tid == 0) {
    bool write = blockIdx.x == 0;
    if (a.arrived != nullptr) {
      write = atomicAdd(a.arrived, 1) == static_cast<int>(gridDim.x) - 1;
      if (write) st_dev(a.arrived, 0);
    }
    if (write) {
      a.cursors_out[0] = status == 0 ? head + total[1] : head;
      a.cursors_out[1] = status == 0 ? tail + total[2] : tail;
      *a.status = status;
    }
  }
}

// ---- append ----------------------------------------------------------------------------------------------------------
struct AppendArgs {
  RopeView rope;
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride, q_out_stride;
  void* q_out;
  f16 *keys, *values;
  int64_t page_stride;
  int num_pages, page_shift, nkv, nq, hd, parts;
  const int32_t *positions, *slots;
};

// One row a block, or `parts` blocks where there are few rows: the units (rope.h) of the query heads, of the key heads,
// then the value heads' W values each. The first unit is requested before slot and angles are known; a row without a
// slot ends there. Bound by memory: 2531 rows of 16 query and 8 KV heads fp32 (72.6 MB) 13.1 us, 5.5 TB/s; 48 rows
// of 32 and 8 by the launch: 5.7 us a call, 3.4 of them the kernel's (4.5 with one block a row). In fp16 8.9 and 5.6 us.
template <typename T, int W>
__global__ __launch_bounds__(256) void k_paged_append(AppendArgs a) {
  __shared__ f32x2 cs[64];  // head_dim <= 128
  const int64_t r = blockIdx.x / a.parts;
  const int units = rope_units(a.rope, W), copies = a.hd / W;
  const int rotated = (a.nq + a.nkv) * units, all = rotated + a.nkv * copies;
  const T* q = static_cast<const T*>(a.q) + r * a.q_stride;
  const T* k = static_cast<const T*>(a.k) + r * a.k_stride;
  const T* v = static_cast<const T*>(a.v) + r * a.v_stride;
  T* q_out = static_cast<T*>(a.q_out) + r * a.q_out_stride;
  const int first = (blockIdx.x % a.parts) * 256 + threadIdx.x, step = a.parts * 256;
  auto load = [&](int u) {
    RopeUnit<T, W> unit;
    if (u >= rotated) {
      unit.a = unit.b = load_vec<T, W>(v + (u - rotated) * W);
    } else {
      const int h = u / units;
      unit = load_unit<T, W>(a.rope, h < a.nq ? q + h * a.hd : k + (h - a.nq) * a.hd, u - h * units);
    }
    return unit;
  };
  RopeUnit<T, W> unit = load(min(first, all - 1));
  const int slot = checked_slot(a.slots[r], a.num_pages, a.page_shift);
  if (slot < 0) return;
  if (a.rope.turns != nullptr) rope_angles(a.rope, a.positions[r], cs);
  __syncthreads();
  const int place = slot & ((1 << a.page_shift) - 1);
  const int64_t page = static_cast<int64_t>(slot >> a.page_shift) * a.page_stride;
  auto cached = [&](f16* pool, int g) { return pool + page + ((static_cast<int64_t>(g) << a.page_shift) + place) * a.hd; };
  for (int u = first; u < all; u += step) {
    if (u != first) unit = load(u);
    const int h = u / units, w = u - h * units;
    if (u >= rotated) {
      const int c = u - rotated, g = c / copies;
      store_copy<T, f16, W>(unit, cached(a.values, g) + (c - g * copies) * W);
    } else if (h < a.nq) {
      store_unit<T, T, W>(a.rope, cs, unit, q_out + h * a.hd, w);
    } else {
      store_unit<T, f16, W>(a.rope, cs, unit, cached(a.keys, h - a.nq), w);
    }
  }
}

template <typename T>
hipError_t launch_paged_append(AppendArgs a, int64_t rows, hipStream_t s) {
  constexpr int W = 16 / sizeof(T);
  const bool aligned = aligned_rows(a.k, a.k_stride, sizeof(T)) && aligned_rows(a.v, a.v_stride, sizeof(T)) &&
                       (a.nq == 0 || (aligned_rows(a.q, a.q_stride, sizeof(T)) &&
                                      aligned_rows(a.q_out, a.q_out_stride, sizeof(T))));
  const int w = aligned && wide_units(a.rope, W) ? W : aligned && wide_units(a.rope, 4) ? 4 : 1;
  auto* kernel = w == W ? k_paged_append<T, W> : w == 4 ? k_paged_append<T, 4> : k_paged_append<T, 1>;
  const int64_t units = (a.nq + a.nkv) * (a.rope.rotary_dim / (2 * w) + (a.hd - a.rope.rotary_dim) / w) +
                        a.nkv * (a.hd / w);
  a.parts = row_blocks(rows, units);
  for (int64_t r = 0; r < rows; r += kRowsALaunch) {
    AppendArgs b = a;
    if (a.nq > 0) b.q = static_cast<const T*>(a.q) + r * a.q_stride;
    b.k = static_cast<const T*>(a.k) + r * a.k_stride;
    b.v = static_cast<const T*>(a.v) + r * a.v_stride;
    if (a.nq > 0) b.q_out = static_cast<T*>(a.q_out) + r * a.q_out_stride;
    if (a.rope.turns != nullptr) b.positions = a.positions + r;
    b.slots = a.slots + r;
    const int n = static_cast<int>(std::min<int64_t>(kRowsALaunch, rows - r));
    hipLaunchKernelGGL(kernel, dim3(n * a.parts), dim3(256), 0, s, b);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// ---- decode attention ------------------------------------------------------------------------------------------------
// One block per (sequence, KV head, chunk of keys); four waves take the chunk's 32-key tiles in turn, each with the
// group's query heads, a running maximum m and sum l and the output so far (in base 2: p = 2^(t - m)). The waves join in
// LDS; of several chunks the last block to finish joins them all, in chunk order.
//
// The keys and values are read once, 16 bytes a lane, and are matrix operands as they come from memory:
//   scores  S [16 keys][16 columns] = K . Q^T, v_mfma_f32_16x16x32_f16: lane l holds 8 dims of key l % 16, and of the
//           query column l % 16. A column is a query head's fp16 high part or (8 columns on) what fp32 has beyond it, so
//           high + low gives the score with about 22 bits of the query, at no further matrix work: a group has at most 8
//           heads (NT = 1), or 16 in two tiles. Queries are scaled by a power of two first, so that high and low are
//           normal fp16 numbers whatever the queries' magnitude.
//   output  O^T [16 dims][16 columns] += V^T . P^T: S leaves 4 keys of each half tile in a lane, which are the 8 keys of
//           the operand P^T; a lane reads 8 dims of those 8 keys (rows of 256 bytes across 16 lanes) and v_perm_b32
//           turns its 8 x 8 block, one instruction for 4 bytes: no LDS, no lane exchange. P is split high and low over
//           the columns as the queries are, and scaled by 2^14 so that small weights stay normal fp16 numbers.
// Keys behind the sequence's end are read as its last key and get weight 0: what memory holds there is never used.
//
// Bound by memory: 200 sequences up to 8192 keys, 32 query and 8 KV heads (3.4 GB), 550 us, 6.2 TB/s (head_dim 64 285 us,
// 6.0); 48 up to 1500 (147 MB) 38 us; one of 4071 keys 11.5 us, where launch, length, pages, keys, hand-over and join
// follow one another. Groups of 9 to 16 heads take two tiles of columns in up to 221 registers, two blocks a CU: 48 query
// and 4 KV heads, 200 sequences up to 8192 keys (1.7 GB) 358 us, 4.8 TB/s (32 and 4: 338, 5.0); one of 4071 keys 15.4
// (32 and 4: 12.6).
struct PagedAttnArgs {
  const f16 *keys, *values;
  int64_t page_stride;
  int num_pages, page_shift, nkv, group, max_pages, n;
  const void* q;
  int64_t q_stride;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
  float scale;
  void* out;
  int64_t out_stride;
  float* lse;
  bool wide_q;             // query rows are 32-byte aligned (16 in fp16): eight values a load
  int splits, grid, most;  // attention_chunk
  float* part;             // [n][nkv][grid][group * (HD + 2)]: outputs, then maxima, then sums
  int* arrived;            // [n][nkv], zero between launches
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kWeightBits = 14.0f;  // weights are held times 2^14

// Reduces over the four lanes l % 16 + {0, 16, 32, 48}; every lane gets the result.
template <typename F>
__device__ __forceinline__ float across_rows(float x, F f) {
  const uint32_t u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t v = __float_as_uint(f(__uint_as_float(a[0]), __uint_as_float(a[1])));
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// x of this lane + x of the lane 8 columns on (mod 16): high and low part.
__device__ __forceinline__ float both_parts(float x) { return x + dpp_mov<0x128>(x); }

template <typename T, int HD, int NT>
__global__ __launch_bounds__(256, 2) void k_paged_attention(PagedAttnArgs a) {
  constexpr int KC = HD / 32;  // 32-dim steps of a score
  constexpr int VD = HD / 16;  // dims of a value row a lane reads: 8 (16 bytes) or 4
  constexpr int HEADS = 8 * NT;
  typedef uint32_t VReg __attribute__((ext_vector_type(VD / 2)));
  // 4 floats behind a head's: 16-byte stores of 8 heads reach 8 bank groups
  __shared__ alignas(16) float so[4][HEADS][HD + 4];
  __shared__ float sm[4][HEADS], sl[4][HEADS];
  __shared__ float weight[256][HEADS], sums[256][HEADS];  // of up to 256 chunks
  __shared__ int last;

  const int g = blockIdx.x % a.nkv, rest = blockIdx.x / a.nkv;
  const int b = rest % a.n, s = rest / a.n;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, row = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = a.group;
  const float nan = __builtin_nanf("");
  T* out = static_cast<T*>(a.out) + b * a.out_stride + static_cast<int64_t>(g) * G * HD;
  // a row's first block requests its queries before it knows the length; others may have no keys
  T qr[NT][KC][8];
  auto load_queries = [&] {
    const T* q = static_cast<const T*>(a.q) + b * a.q_stride + static_cast<int64_t>(g) * G * HD + row * 8;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const T* p = q + min(t * 8 + (col & 7), G - 1) * HD;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        if (a.wide_q) {
          typedef T Q8 __attribute__((ext_vector_type(8)));
          const Q8 v = *reinterpret_cast<const Q8*>(p + c * 32);
#pragma unroll
          for (int i = 0; i < 8; ++i) qr[t][c][i] = v[i];
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) qr[t][c][i] = p[c * 32 + i];
        }
      }
    }
  };
  if (s == 0) load_queries();
  float* lse = a.lse != nullptr ? a.lse + (static_cast<int64_t>(b) * a.nkv + g) * G : nullptr;
  const int len = checked_length(a.lens[b], a.max_pages, a.page_shift);
  if (len <= 0) {
    if (s != 0) return;
    for (int i = tid; i < G * HD; i += 256) out[i] = static_cast<T>(len < 0 ? nan : 0.0f);
    if (lse != nullptr && tid < G) lse[tid] = len < 0 ? nan : -INFINITY;
    return;
  }
  const int chunk = attention_chunk(len, a.splits, a.grid, a.most);
  const uint32_t c0 = static_cast<uint32_t>(s) * chunk;
  if (c0 >= static_cast<uint32_t>(len)) return;
  if (s != 0) load_queries();
  const int tiles = (min(chunk, len - static_cast<int>(c0)) - 1) / 32 + 1;
  const int mine = (tiles - wid + 3) / 4;  // this wave's: wid, wid + 4, ..
  const int32_t* table = a.table + b * a.table_stride;
  const uint32_t mask = (1u << a.page_shift) - 1;
  const f16* keys = a.keys + (static_cast<int64_t>(g) << a.page_shift) * HD;
  const f16* values = a.values + (static_cast<int64_t>(g) << a.page_shift) * HD;

  // (key numbers are unsigned words: at most 2^30 keys and 2^14 behind them)
  auto within = [&](uint32_t key) { return min(key, static_cast<uint32_t>(len) - 1); };
  // lane l holds the page of half tile l % 2 of this wave's tile l / 2 (32 tiles ahead)
  bool lost = false;
  auto pages_from = [&](int first) {
    const uint32_t key = within(c0 + (wid + 4 * (first + (lane >> 1))) * 32 + (lane & 1) * 16);
    const int page = checked_page(table[key >> a.page_shift], a.num_pages);
    lost |= page < 0;
    return max(page, 0);
  };
  int pages = pages_from(0);

  u32x4 kr[2][KC];
  VReg vr[2][4];
  // tile i of this wave; key and value rows of a half tile are in one page
  auto load_keys = [&](int i) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t page = __builtin_amdgcn_readlane(pages, 2 * (i & 31) + h);
      const uint32_t key = within(c0 + (wid + 4 * i) * 32 + h * 16 + col);
      const f16* p = keys + page * a.page_stride + ((key & mask) * HD + row * 8);
#pragma unroll
      for (int c = 0; c < KC; ++c) kr[h][c] = load_stream16(p + c * 32);
    }
  };
  auto load_values = [&](int i) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t page = __builtin_amdgcn_readlane(pages, 2 * (i & 31) + h);
      const f16* base = values + page * a.page_stride;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t key = within(c0 + (wid + 4 * i) * 32 + h * 16 + row * 4 + j);
        vr[h][j] = __builtin_nontemporal_load(
            (const __attribute__((address_space(1))) VReg*)(base + ((key & mask) * HD + col * VD)));
      }
    }
  };
  // the query columns, while the pages are looked up
  f16x8 qb[NT][KC];
  float to_log2[NT];  // score of the scaled query -> base-2 exponent
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const bool there = t * 8 + (col & 7) < G;
    float big = 0.0f;
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (!there) qr[t][c][i] = static_cast<T>(0.0f);
        big = fmaxf(big, fabsf(static_cast<float>(qr[t][c][i])));
      }
    big = across_rows(big, [](float u, float v) { return fmaxf(u, v); });
    // times 2^e, by which the largest becomes 2^13 .. 2^14 (subnormal ones less, by 2^126); not where it is 0 or no number
    const int exponent = static_cast<int>(__float_as_uint(big) >> 23);
    const int e = big > 0.0f && exponent < 255 ? min(140 - exponent, 126) : 0;
    const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
    // the power of two first: scale times log2(e) alone may pass fp32
    to_log2[t] = a.scale * __uint_as_float(static_cast<uint32_t>(127 - e) << 23) * kLog2e;
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = static_cast<float>(qr[t][c][i]) * up;
        const f16 high = static_cast<f16>(v);
        qb[t][c][i] = col < 8 ? high : static_cast<f16>(v - static_cast<float>(high));
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
    const uint32_t key0 = c0 + (wid + 4 * i) * 32;
    f32x4 sc[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sc[t][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < KC; ++c)
          sc[t][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_f16x8(kr[h][c]), qb[t][c], sc[t][h], 0, 0, 0);
      }
    const bool more = i + 1 < mine;
    // pages of the next 32 tiles, before they are needed; the values of tile i are already on their way
    if (more && ((i + 1) & 31) == 0) pages = pages_from(i + 1);
    if (more) load_keys(i + 1);
    f16x8 pb[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float x[8];
      float top = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float v = both_parts(sc[t][h][r]) * to_log2[t];
          x[4 * h + r] = key0 + h * 16 + row * 4 + r < static_cast<uint32_t>(len) ? v : -INFINITY;
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
        const f16 high = static_cast<f16>(p);
        pb[t][j] = col < 8 ? high : static_cast<f16>(p - static_cast<float>(high));
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
      for (int t = 0; t < NT; ++t)
        o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_f16x8(av), pb[t], o[t][d], 0, 0, 0);
    }
    if (more) load_values(i + 1);
  }

  // the four waves: brought to their common maximum, then added. A wave without a tile has m = -inf and adds 0; a score
  // of NaN leaves NaN in the sums
  if (row == 0 && col < 8)
#pragma unroll
    for (int t = 0; t < NT; ++t) sm[wid][t * 8 + col] = m[t];
  lost = __syncthreads_or(lost);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int h = t * 8 + (col & 7);
    const float top = fmaxf(fmaxf(sm[0][h], sm[1][h]), fmaxf(sm[2][h], sm[3][h]));
    const float f = __builtin_amdgcn_exp2f(m[t] - top);
    const float sum = across_rows(l[t], [](float u, float v) { return u + v; }) * f;
    if (row == 0 && col < 8) sl[wid][h] = sum;
    // both columns of a head hold its sums: the high one stores rows 0 and 1 of the lane's four, the low one 2 and 3
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int d = 0; d < VD; d += 4) {
        f32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a0 = both_parts(o[t][d + i][r]), a1 = both_parts(o[t][d + i][r + 2]);
          x[i] = (col < 8 ? a0 : a1) * f;
        }
        *reinterpret_cast<f32x4*>(&so[wid][h][(row * 4 + r + (col < 8 ? 0 : 2)) * VD + d]) = x;
      }
  }
  __syncthreads();
  const int blocks = (len - 1) / chunk + 1;
  const int64_t pair = static_cast<int64_t>(b) * a.nkv + g;
  const int stride = G * (HD + 2);
  float* part = a.part + (pair * a.grid + s) * stride;
  for (int i = tid; i < G * HD / 2; i += 256) {
    const int h = 2 * i / HD, d = 2 * i % HD;
    f32x2 x = *reinterpret_cast<const f32x2*>(&so[0][h][d]);
    float sum = sl[0][h];
#pragma unroll
    for (int u = 1; u < 4; ++u) {
      const f32x2 y = *reinterpret_cast<const f32x2*>(&so[u][h][d]);
      x[0] += y[0];
      x[1] += y[1];
      sum += sl[u][h];
    }
    if (blocks == 1) {
      out[2 * i] = static_cast<T>(lost ? nan : x[0] / sum);
      out[2 * i + 1] = static_cast<T>(lost ? nan : x[1] / sum);
    } else {
      __hip_atomic_store(reinterpret_cast<uint64_t*>(part) + i, __builtin_bit_cast(uint64_t, x), __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  if (tid < G) {
    const float top = fmaxf(fmaxf(sm[0][tid], sm[1][tid]), fmaxf(sm[2][tid], sm[3][tid]));
    float sum = (sl[0][tid] + sl[1][tid]) + (sl[2][tid] + sl[3][tid]);
    if (lost) sum = nan;
    if (blocks > 1) {
      st_dev(part + G * HD + tid, top);
      st_dev(part + G * HD + G + tid, sum);
    } else if (lse != nullptr) {
      lse[tid] = (top + __builtin_amdgcn_logf(sum) - kWeightBits) * kLn2;
    }
  }
  if (blocks == 1) return;

  // the chunks: this block's part is out before its arrival is counted
  wait_mem();
  __syncthreads();
  if (tid == 0) last = atomicAdd(a.arrived + pair, 1) == blocks - 1;
  __syncthreads();
  if (!last) return;
  float* all = a.part + pair * a.grid * stride;
  for (int i = tid; i < blocks * G; i += 256) {
    const int u = i / G, h = i - u * G;
    const float* p = all + static_cast<int64_t>(u) * stride + G * HD + h;
    weight[u][h] = ld_dev(p);
    sums[u][h] = ld_dev(p + G);
  }
  __syncthreads();
  for (int h = wid; h < G; h += 4) {
    float top = -INFINITY, sum = 0.0f;
    for (int u = lane; u < blocks; u += 64) top = fmaxf(top, weight[u][h]);
    top = wave_max(top);
    for (int u = lane; u < blocks; u += 64) {
      const float w = __builtin_amdgcn_exp2f(weight[u][h] - top);
      weight[u][h] = w;
      sum += w * sums[u][h];
    }
    sum = wave_sum(sum);
    if (lane == 0) {
      sl[0][h] = sum;
      if (lse != nullptr) lse[h] = (top + __builtin_amdgcn_logf(sum) - kWeightBits) * kLn2;
    }
  }
  __syncthreads();
  for (int i = tid; i < G * HD / 2; i += 256) {
    const int h = 2 * i / HD;
    float x0 = 0.0f, x1 = 0.0f;
    for (int u0 = 0; u0 < blocks; u0 += 16) {  // sixteen parts on their way at a time, added in order
      uint64_t v[16];
#pragma unroll
      for (int j = 0; j < 16; ++j)
        v[j] = __hip_atomic_load(reinterpret_cast<uint64_t*>(all + static_cast<int64_t>(min(u0 + j, blocks - 1)) * stride) + i,
                                 __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (u0 + j < blocks) {
          const float w = weight[u0 + j][h];
          x0 += w * __uint_as_float(static_cast<uint32_t>(v[j]));
          x1 += w * __uint_as_float(static_cast<uint32_t>(v[j] >> 32));
        }
    }
    out[2 * i] = static_cast<T>(x0 / sl[0][h]);
    out[2 * i + 1] = static_cast<T>(x1 / sl[0][h]);
  }
  if (tid == 0) st_dev(a.arrived + pair, 0);
}

template <typename T, int HD>
hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t s) {
  auto* kernel = a.group <= 8 ? k_paged_attention<T, HD, 1> : k_paged_attention<T, HD, 2>;
  hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(a.n) * a.nkv * a.grid), dim3(256), 0, s, a);
  return hipGetLastError();
}
hipError_t launch_paged_attention(const PagedAttnArgs& a, bool f32, int hd, hipStream_t s) {
  if (hd == 128) return f32 ? launch_paged_attention<float, 128>(a, s) : launch_paged_attention<f16, 128>(a, s);
  return f32 ? launch_paged_attention<float, 64>(a, s) : launch_paged_attention<f16, 64>(a, s);
}

int shift_of(int page_size) {
  int s = 0;
  while ((1 << s) < page_size) ++s;
  return s;
}

int check_page_size(int32_t page_size) {
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128 && page_size != 256)
    return fail(SOC_ERR_INVALID, "paged cache: page_size must be 16, 32, 64, 128 or 256");
  return SOC_OK;
}

int check_cache_shape(const soc_paged_cache* c) {
  if (c == nullptr) return fail(SOC_ERR_INVALID, "null paged cache");
  SOC_TRY(check_page_size(c->page_size));
  if (c->head_dim != 64 && c->head_dim != 128) return fail(SOC_ERR_INVALID, "paged cache: head_dim must be 64 or 128");
  if (c->kv_heads <= 0 || c->kv_heads > 1024 || c->num_pages <= 0)
    return fail(SOC_ERR_INVALID, "paged cache: need num_pages > 0 and 1 to 1024 kv_heads");
  if (static_cast<int64_t>(c->num_pages) * c->page_size > INT32_MAX)
    return fail(SOC_ERR_INVALID, "paged cache: num_pages * page_size must be below 2^31");
  const int64_t page = static_cast<int64_t>(c->kv_heads) * c->page_size * c->head_dim;
  if (c->page_stride != 0 && (c->page_stride < page || c->page_stride % 8 != 0))
    return fail(SOC_ERR_INVALID, "paged cache: page_stride must be 0 or a multiple of 8 that holds a page");
  if (reinterpret_cast<uintptr_t>(c->keys) % 16 != 0 || reinterpret_cast<uintptr_t>(c->values) % 16 != 0)
    return fail(SOC_ERR_INVALID, "paged cache: keys and values must be 16-byte aligned");
  return SOC_OK;
}

int64_t page_stride(const soc_paged_cache* c) {
  return c->page_stride != 0 ? c->page_stride : static_cast<int64_t>(c->kv_heads) * c->page_size * c->head_dim;
}

int check_cache_memory(Operands& operands, const soc_paged_cache* c) {
  const int64_t page = static_cast<int64_t>(c->kv_heads) * c->page_size * c->head_dim;
  SOC_TRY(operands.rows("paged cache keys", c->keys, c->num_pages, page_stride(c), page, 2));
  return operands.rows("paged cache values", c->values, c->num_pages, page_stride(c), page, 2);
}

int hip_status(hipError_t e, const char* what) {
  return e == hipSuccess ? SOC_OK : fail(SOC_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}

// soc_paged_plan (step_lens: nullptr) and soc_paged_plan_step.
int plan_step(soc_ctx* ctx, int32_t n, const int32_t* old_lens, const int32_t* new_lens, int32_t page_size,
              int32_t* block_table, int32_t max_pages, int64_t table_stride, int32_t* free_ring, int32_t num_pages,
              const int64_t* cursors_in, int64_t* cursors_out, int32_t* row_starts, int32_t* positions, int32_t* slots,
              int32_t max_rows, int32_t* status, int32_t* step_lens) {
  if (n <= 0 || n > kPlanMaxRequests) return fail(SOC_ERR_INVALID, "paged plan: 1 to 4096 requests");
  SOC_TRY(check_page_size(page_size));
  if (max_pages <= 0 || max_pages > kPlanMaxPages)
    return fail(SOC_ERR_INVALID, "paged plan: max_pages must be 1 to 2^18");
  if (max_rows <= 0 || max_rows > kPlanMaxRows)
    return fail(SOC_ERR_INVALID, "paged plan: max_rows must be 1 to 2^22");
  if (num_pages <= 0 || static_cast<int64_t>(num_pages) * page_size > INT32_MAX)
    return fail(SOC_ERR_INVALID, "paged plan: need num_pages > 0 and num_pages * page_size below 2^31");
  if (step_lens != nullptr)  // another block may still read what one writes
    for (const int32_t* lens : {old_lens, new_lens})
      if (step_lens < lens + n && lens < step_lens + n)
        return fail(SOC_ERR_INVALID, "paged plan: step_lens must not overlap old_lens or new_lens");
  if (ctx == nullptr) return fail(SOC_ERR_INVALID, "null context");
  DeviceScope device(ctx);
  Operands operands(ctx);
  SOC_TRY(operands.array("paged plan old_lens", old_lens, n, 4));
  SOC_TRY(operands.array("paged plan new_lens", new_lens, n, 4));
  SOC_TRY(operands.rows("paged plan block_table", block_table, n, table_stride, max_pages, 4));
  SOC_TRY(operands.array("paged plan free_ring", free_ring, num_pages, 4));
  SOC_TRY(operands.array("paged plan cursors_in", cursors_in, 2, 8));
  SOC_TRY(operands.array("paged plan cursors_out", cursors_out, 2, 8));
  SOC_TRY(operands.array("paged plan row_starts", row_starts, n + 1, 4));
  SOC_TRY(operands.array("paged plan positions", positions, max_rows, 4));
  SOC_TRY(operands.array("paged plan slots", slots, max_rows, 4));
  SOC_TRY(operands.array("paged plan status", status, 1, 4));
  if (step_lens != nullptr) SOC_TRY(operands.array("paged plan step_lens", step_lens, n, 4));
  // a row a thread
  const int blocks = std::min(256, std::max(1, (max_rows + kPlanThreads - 1) / kPlanThreads));
  int* arrived = nullptr;
  if (blocks > 1 && cursors_out < cursors_in + 2 && cursors_in < cursors_out + 2) {
    SOC_TRY(ensure_serve_ws(ctx, 0, 1));
    arrived = ctx->serve_counters;
  }
  PlanArgs a{n, old_lens, new_lens, block_table, max_pages, table_stride, free_ring, num_pages, shift_of(page_size),
             cursors_in, cursors_out, row_starts, positions, slots, max_rows, status, step_lens, arrived};
  auto* kernel = n <= kPlanThreads       ? k_paged_plan<1>
                 : n <= 4 * kPlanThreads ? k_paged_plan<4>
                                         : k_paged_plan<kPlanMaxRequests / kPlanThreads>;
  hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kPlanThreads), 0, ctx->stream, a);
  return hip_status(hipGetLastError(), "paged plan");
}

}  // namespace
}  // namespace soc

extern "C" {

int soc_paged_plan(soc_ctx* ctx, int32_t n, const int32_t* old_lens, const int32_t* new_lens, int32_t page_size,
                   int32_t* block_table, int32_t max_pages, int64_t table_stride, int32_t* free_ring, int32_t num_pages,
                   const int64_t* cursors_in, int64_t* cursors_out, int32_t* row_starts, int32_t* positions,
                   int32_t* slots, int32_t max_rows, int32_t* status) {
  SOC_API_BEGIN
  return soc::plan_step(ctx, n, old_lens, new_lens, page_size, block_table, max_pages, table_stride, free_ring, num_pages,
                        cursors_in, cursors_out, row_starts, positions, slots, max_rows, status, nullptr);
  SOC_API_END
}

int soc_paged_plan_step(soc_ctx* ctx, int32_t n, const int32_t* old_lens, const int32_t* new_lens, int32_t page_size,
                        int32_t* block_table, int32_t max_pages, int64_t table_stride, int32_t* free_ring,
                        int32_t num_pages, const int64_t* cursors_in, int64_t* cursors_out, int32_t* row_starts,
                        int32_t* positions, int32_t* slots, int32_t max_rows, int32_t* status, int32_t* step_lens) {
  SOC_API_BEGIN
  return soc::plan_step(ctx, n, old_lens, new_lens, page_size, block_table, max_pages, table_stride, free_ring, num_pages,
                        cursors_in, cursors_out, row_starts, positions, slots, max_rows, status, step_lens);
  SOC_API_END
}

int soc_paged_append(soc_ctx* ctx, const soc_paged_cache* cache, const soc_rope* rope, const void* q, int64_t q_stride,
                     const void* k, int64_t k_stride, const void* v, int64_t v_stride, int32_t dtype, void* q_out,
                     int64_t q_out_stride, int32_t rows, int32_t q_heads, const int32_t* positions,
                     const int32_t* slots) {
  SOC_API_BEGIN
  SOC_TRY(soc::check_cache_shape(cache));
  if (dtype != SOC_DTYPE_F32 && dtype != SOC_DTYPE_F16)
    return soc::fail(SOC_ERR_INVALID, "paged append: dtype must be F32 or F16");
  if (rows <= 0 || q_heads < 0 || q_heads > (1 << 16))
    return soc::fail(SOC_ERR_INVALID, "paged append: need rows > 0 and 0 to 65536 q_heads");
  if (rope == nullptr && q_heads != 0) return soc::fail(SOC_ERR_INVALID, "paged append: queries need a rope");
  if (q_heads > 0 && q == q_out && q_stride != q_out_stride)
    return soc::fail(SOC_ERR_INVALID, "paged append: in place needs equal strides");
  if (ctx == nullptr) return soc::fail(SOC_ERR_INVALID, "null context");
  if (rope != nullptr && (rope->ctx != ctx || rope->head_dim != cache->head_dim))
    return soc::fail(SOC_ERR_INVALID, "paged append: the rope is of another context or head_dim");
  soc::DeviceScope device(ctx);
  soc::Operands operands(ctx);
  const int size = dtype == SOC_DTYPE_F32 ? 4 : 2, hd = cache->head_dim;
  const int64_t kv = static_cast<int64_t>(cache->kv_heads) * hd, qw = static_cast<int64_t>(q_heads) * hd;
  SOC_TRY(soc::check_cache_memory(operands, cache));
  SOC_TRY(operands.rows("paged append keys", k, rows, k_stride, kv, size));
  SOC_TRY(operands.rows("paged append values", v, rows, v_stride, kv, size));
  if (q_heads > 0) {
    SOC_TRY(operands.rows("paged append queries", q, rows, q_stride, qw, size));
    if (q_out != q) SOC_TRY(operands.rows("paged append q_out", q_out, rows, q_out_stride, qw, size));
  }
  if (rope != nullptr) SOC_TRY(operands.array("paged append positions", positions, rows, 4));
  SOC_TRY(operands.array("paged append slots", slots, rows, 4));
  soc::AppendArgs a{};
  a.rope = soc::view_of(rope, hd);
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.q_out = q_out;
  a.q_out_stride = q_out_stride;
  a.keys = static_cast<soc::f16*>(cache->keys);
  a.values = static_cast<soc::f16*>(cache->values);
  a.page_stride = soc::page_stride(cache);
  a.num_pages = cache->num_pages;
  a.page_shift = soc::shift_of(cache->page_size);
  a.nkv = cache->kv_heads;
  a.nq = q_heads;
  a.hd = hd;
  a.positions = positions;
  a.slots = slots;
  const hipError_t e = size == 4 ? soc::launch_paged_append<float>(a, rows, ctx->stream)
                                 : soc::launch_paged_append<soc::f16>(a, rows, ctx->stream);
  return soc::hip_status(e, "paged append");
  SOC_API_END
}

int soc_paged_attention_decode(soc_ctx* ctx, const soc_paged_cache* cache, const void* q, int64_t q_stride,
                               int32_t dtype, const int32_t* block_table, int64_t table_stride, int32_t max_pages,
                               const int32_t* seq_lens, int32_t n, int32_t q_heads, float scale, void* out,
                               int64_t out_stride, float* lse) {
  SOC_API_BEGIN
  SOC_TRY(soc::check_cache_shape(cache));
  if (dtype != SOC_DTYPE_F32 && dtype != SOC_DTYPE_F16)
    return soc::fail(SOC_ERR_INVALID, "paged attention: dtype must be F32 or F16");
  if (n <= 0 || n > 65535) return soc::fail(SOC_ERR_INVALID, "paged attention: 1 to 65535 sequences");
  if (max_pages <= 0 || static_cast<int64_t>(max_pages) * cache->page_size > (1 << 30))
    return soc::fail(SOC_ERR_INVALID, "paged attention: need max_pages > 0 and max_pages * page_size up to 2^30");
  if (q_heads <= 0 || q_heads % cache->kv_heads != 0 || q_heads / cache->kv_heads > 16)
    return soc::fail(SOC_ERR_INVALID, "paged attention: query heads per KV head must be 1 to 16");
  if (!std::isfinite(scale)) return soc::fail(SOC_ERR_INVALID, "paged attention: scale must be finite");
  if (q == out && q_stride != out_stride)
    return soc::fail(SOC_ERR_INVALID, "paged attention: in place needs equal strides");
  if (ctx == nullptr) return soc::fail(SOC_ERR_INVALID, "null context");
  soc::DeviceScope device(ctx);
  soc::Operands operands(ctx);
  const int size = dtype == SOC_DTYPE_F32 ? 4 : 2, hd = cache->head_dim;
  const int64_t width = static_cast<int64_t>(q_heads) * hd;
  SOC_TRY(soc::check_cache_memory(operands, cache));
  SOC_TRY(operands.rows("paged attention queries", q, n, q_stride, width, size));
  if (out != q) SOC_TRY(operands.rows("paged attention output", out, n, out_stride, width, size));
  SOC_TRY(operands.rows("paged attention block_table", block_table, n, table_stride, max_pages, 4));
  SOC_TRY(operands.array("paged attention seq_lens", seq_lens, n, 4));
  if (lse != nullptr) SOC_TRY(operands.rows("paged attention lse", lse, n, q_heads, q_heads, 4));
  soc::PagedAttnArgs a{};
  a.keys = static_cast<const soc::f16*>(cache->keys);
  a.values = static_cast<const soc::f16*>(cache->values);
  a.page_stride = soc::page_stride(cache);
  a.num_pages = cache->num_pages;
  a.page_shift = soc::shift_of(cache->page_size);
  a.nkv = cache->kv_heads;
  a.group = q_heads / cache->kv_heads;
  a.max_pages = max_pages;
  a.q = q;
  a.q_stride = q_stride;
  a.table = block_table;
  a.table_stride = table_stride;
  a.lens = seq_lens;
  a.scale = scale != 0.0f ? scale : 1.0f / std::sqrt(static_cast<float>(hd));
  a.out = out;
  a.out_stride = out_stride;
  a.lse = lse;
  a.wide_q = reinterpret_cast<uintptr_t>(q) % (8 * size) == 0 && q_stride % 8 == 0;
  a.n = n;
  const int64_t pairs = static_cast<int64_t>(n) * cache->kv_heads;
  if (pairs > (1 << 20)) return soc::fail(SOC_ERR_INVALID, "paged attention: sequences times KV heads beyond 2^20");
  const int64_t longest = static_cast<int64_t>(max_pages) * cache->page_size;
  const size_t part = static_cast<size_t>(a.group) * (hd + 2) * sizeof(float);
  const int64_t room = std::max<int64_t>(1, (int64_t{512} << 20) / static_cast<int64_t>(pairs * part));
  // Blocks of a sequence. `splits`: one for each CU where there are few sequences (8 x 1000 keys, 16 query and 8 KV
  // heads: 11.8 us so, 14.6 with half of them; 8 x 4000, 32 and 8: 26.7 us, 28.1 with twice as many), but 32 at most (one
  // of 16000 keys, 14 and 2 heads: 17.9 us with 32 parts a head, 19.4 with 63).
  // `most`: keys a block, so that ragged lengths even out: 1024 (512: 256 sequences up to 1500 keys, 32 and 8 heads,
  // 162 us for 148); 2048 where whole sequences fill 768 places for blocks twice over (three a CU: head_dim 128 and up to
  // 8 heads a group; the other kernels have two to four a CU, not measured apart) and a part is of four query heads or
  // more, which cost most to prepare and join (256 up to 6000: 535 us for 551, all of 1500 248 for 272; but 128 up to 1500
  // 89 for 81, and 256 up to 1500 with 16 and 8 heads of 64 81 for 75).
  // `grid`: what is launched for each row of the table, by its width alone; a large batch has 8 (64 rows of 200 keys in a
  // table 32768 wide: 11 us, 20 with 32, most of them empty). The price: one long sequence among many short ones has 8
  // blocks too, of whatever length (one of 131072 keys among 64 of 200, 32 and 8 heads: 448 us; alone 95).
  a.splits = static_cast<int>(std::min<int64_t>(32, (256 + pairs - 1) / pairs));
  a.most = pairs >= 2 * 768 && a.group >= 4 ? 2048 : soc::kAttentionMost;
  a.grid = static_cast<int>(std::min({((longest - 1) / a.most / a.splits + 1) * a.splits,
                                      std::max<int64_t>(8, 4096 / pairs), (longest + 127) / 128, room, int64_t{256}}));
  if (a.grid > 1) {
    SOC_TRY(soc::ensure_serve_ws(ctx, static_cast<size_t>(pairs) * a.grid * part, static_cast<size_t>(pairs)));
    a.part = reinterpret_cast<float*>(ctx->serve_ws);
    a.arrived = ctx->serve_counters;
  }
  const hipError_t e = soc::launch_paged_attention(a, size == 4, hd, ctx->stream);
  return soc::hip_status(e, "paged attention");
  SOC_API_END
}

}  // extern "C"
