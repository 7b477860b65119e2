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
// are over at most 4096 lengths, read from L2; a second launch for them alone would cost more than repeating them.
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

__global__ __launch_bounds__(kPlanThreads) void k_paged_plan(PlanArgs a) {
  __shared__ int32_t rows[kPlanMaxRequests + 1], take[kPlanMaxRequests + 1], give[kPlanMaxRequests + 1];
  __shared__ int32_t wave_total[3][kPlanThreads / kWave];
  __shared__ int any_bad;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
  if (tid == 0) any_bad = 0;
  const int64_t head = a.cursors_in[0], tail = a.cursors_in[1];
  // thread t sums requests [t * per, (t + 1) * per) one after the other, then the block scans the threads' sums
  const int per = (a.n + kPlanThreads - 1) / kPlanThreads;
  const int first = min(tid * per, a.n), last = min(first + per, a.n);
  int32_t sum[3] = {0, 0, 0};
  bool bad = false;
  for (int i = first; i < last; ++i) {
    const PlanItem p = plan_item(a.before[i], a.after[i], a.max_pages, a.page_shift);
    bad |= p.bad;
    sum[0] = min(sum[0] + p.rows, kPlanMaxRows + 1);
    sum[1] += p.take;
    sum[2] += p.give;
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
  __syncthreads();  // any_bad is cleared
  if (bad) any_bad = 1;
  if (lane == kWave - 1)
#pragma unroll
    for (int j = 0; j < 3; ++j) wave_total[j][wid] = incl[j];
  __syncthreads();
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
  for (int i = first; i < last; ++i) {
    const PlanItem p = plan_item(a.before[i], a.after[i], a.max_pages, a.page_shift);
    rows[i] = at[0];
    take[i] = at[1];
    give[i] = at[2];
    at[0] += p.rows;
    at[1] += p.take;
    at[2] += p.give;
  }
  if (tid == 0) {
    rows[a.n] = total[0];
    take[a.n] = total[1];
    give[a.n] = total[2];
  }
  __syncthreads();
  const int64_t free_pages = tail - head;
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
      const int before = a.before[i], had = pages_of(before, a.page_shift);
      position = before + (static_cast<int>(r) - rows[i]);
      const int index = position >> a.page_shift;
      const int page = index < had ? a.table[i * a.table_stride + index]
                                   : a.ring[ring_place(head, take[i] + (index - had), a.num_pages)];
      slot = slot_of(page, position & ((1 << a.page_shift) - 1), a.num_pages, a.page_shift);
    }
    a.positions[r] = position;
    a.slots[r] = slot;
  }
  for (int64_t i = gid; i <= a.n; i += stride) a.row_starts[i] = status == 0 ? rows[i] : 0;
  if (status == 0) {
    // entries at or behind the pages a request had are written, entries before them read: no thread reads what another
    // writes, and the ring's places from the tail on are not among those taken from the head (at most num_pages free)
    for (int64_t j = gid; j < total[1]; j += stride) {
      const int i = request_of(take, a.n, static_cast<int32_t>(j));
      const int had = pages_of(a.before[i], a.page_shift);
      a.table[i * a.table_stride + had + (j - take[i])] =
          a.ring[ring_place(head, static_cast<int32_t>(j), a.num_pages)];
    }
    for (int64_t j = gid; j < total[2]; j += stride) {
      const int i = request_of(give, a.n, static_cast<int32_t>(j));
      const int keep = pages_of(a.after[i], a.page_shift);
      a.ring[ring_place(tail, static_cast<int32_t>(j), a.num_pages)] =
          a.table[i * a.table_stride + keep + (j - give[i])];
    }
  }
  // cursors_out may be cursors_in: the last block to have read them writes them
  if (tid == 0) {
    bool write = gridDim.x == 1;
    if (!write) write = atomicAdd(a.arrived, 1) == static_cast<int>(gridDim.x) - 1;
    if (write) {
      if (gridDim.x > 1) st_dev(a.arrived, 0);
      a.cursors_out[0] = head + (status == 0 ? total[1] : 0);
      a.cursors_out[1] = tail + (status == 0 ? total[2] : 0);
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
  int num_pages, page_shift, nkv, nq, hd;
  const int32_t *positions, *slots;
};

template <typename T, int W>
__global__ __launch_bounds__(256) void k_paged_append(AppendArgs a) {
  __shared__ f32x2 cs[64];  // head_dim <= 128
  const int64_t r = blockIdx.x;
  const int slot = checked_slot(a.slots[r], a.num_pages, a.page_shift);
  if (slot < 0) return;
  if (a.rope.turns != nullptr) rope_angles(a.rope, a.positions[r], cs);
  __syncthreads();
  const int units = rope_units(a.rope, W);
  const int place = slot & ((1 << a.page_shift) - 1);
  const int64_t page = static_cast<int64_t>(slot >> a.page_shift) * a.page_stride;
  const T* q = static_cast<const T*>(a.q) + r * a.q_stride;
  const T* k = static_cast<const T*>(a.k) + r * a.k_stride;
  const T* v = static_cast<const T*>(a.v) + r * a.v_stride;
  T* q_out = static_cast<T*>(a.q_out) + r * a.q_out_stride;
  const int rotated = (a.nq + a.nkv) * units, copied = a.nkv * (a.hd / W);
  for (int u = threadIdx.x; u < rotated + copied; u += blockDim.x) {
    if (u < rotated) {
      const int h = u / units, w = u - h * units;
      if (h < a.nq) {
        rope_unit<T, T, W>(a.rope, cs, q + h * a.hd, q_out + h * a.hd, w);
      } else {
        const int g = h - a.nq;
        f16* dst = a.keys + page + ((static_cast<int64_t>(g) << a.page_shift) + place) * a.hd;
        rope_unit<T, f16, W>(a.rope, cs, k + g * a.hd, dst, w);
      }
    } else {
      const int w = u - rotated, g = w / (a.hd / W), d = (w - g * (a.hd / W)) * W;
      float x[W];
      load_vec<T, W>(v + g * a.hd + d, x);
      store_vec<f16, W>(a.values + page + ((static_cast<int64_t>(g) << a.page_shift) + place) * a.hd + d, x);
    }
  }
}

// ---- decode attention ------------------------------------------------------------------------------------------------
struct PagedAttnArgs {
  const f16 *keys, *values;
  int64_t page_stride;
  int num_pages, page_shift, nkv, group, max_pages;
  const void* q;
  int64_t q_stride;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
  float scale;
  void* out;
  int64_t out_stride;
  float* lse;
};

template <typename T, int HD>
__global__ __launch_bounds__(256) void k_paged_attention(PagedAttnArgs a) {
  constexpr int E = HD / kWave;
  __shared__ float ms[4], ls[4], os[4][HD];
  const int nq = a.nkv * a.group;
  const int b = blockIdx.x / nq, h = blockIdx.x % nq, g = h / a.group;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int len = checked_length(a.lens[b], a.max_pages, a.page_shift);
  const T* q = static_cast<const T*>(a.q) + b * a.q_stride + h * HD + lane * E;
  float qv[E], o[E];
  for (int i = 0; i < E; ++i) {
    qv[i] = static_cast<float>(q[i]) * a.scale;
    o[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  bool lost = len < 0;
  for (int j = wid; j < len; j += 4) {
    const int page = checked_page(a.table[b * a.table_stride + (j >> a.page_shift)], a.num_pages);
    if (page < 0) {
      lost = true;
      break;
    }
    const int64_t at = page * a.page_stride +
                       ((static_cast<int64_t>(g) << a.page_shift) + (j & ((1 << a.page_shift) - 1))) * HD + lane * E;
    float s = 0.0f;
    for (int i = 0; i < E; ++i) s += qv[i] * static_cast<float>(a.keys[at + i]);
    s = wave_sum(s);
    const float m1 = fmaxf(m, s), f = m1 == -INFINITY ? 0.0f : expf(m - m1), p = m1 == -INFINITY ? 0.0f : expf(s - m1);
    l = l * f + p;
    for (int i = 0; i < E; ++i) o[i] = o[i] * f + p * static_cast<float>(a.values[at + i]);
    m = m1;
  }
  if (lost) l = __builtin_nanf("");
  if (lane == 0) {
    ms[wid] = m;
    ls[wid] = l;
  }
  for (int i = 0; i < E; ++i) os[wid][lane * E + i] = o[i];
  __syncthreads();
  const float top = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3]));
  float total = 0.0f;
  for (int w = 0; w < 4; ++w) total += ls[w] != ls[w] || top != -INFINITY ? ls[w] * expf(ms[w] - top) : 0.0f;
  const bool nan = total != total || ls[0] != ls[0] || ls[1] != ls[1] || ls[2] != ls[2] || ls[3] != ls[3];
  const int d = threadIdx.x;
  if (d < HD) {
    float x = 0.0f;
    for (int w = 0; w < 4; ++w)
      if (ls[w] > 0.0f) x += os[w][d] * expf(ms[w] - top);
    x = nan ? __builtin_nanf("") : total > 0.0f ? x / total : 0.0f;
    static_cast<T*>(a.out)[b * a.out_stride + h * HD + d] = static_cast<T>(x);
  }
  if (d == 0 && a.lse != nullptr)
    a.lse[static_cast<int64_t>(b) * nq + h] = nan ? __builtin_nanf("") : total > 0.0f ? top + logf(total) : -INFINITY;
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

int check_cache_memory(const soc_ctx* ctx, const soc_paged_cache* c) {
  const int64_t page = static_cast<int64_t>(c->kv_heads) * c->page_size * c->head_dim;
  SOC_TRY(check_device_rows(ctx, "paged cache keys", c->keys, c->num_pages, page_stride(c), page, 2));
  return check_device_rows(ctx, "paged cache values", c->values, c->num_pages, page_stride(c), page, 2);
}

int hip_status(hipError_t e, const char* what) {
  return e == hipSuccess ? SOC_OK : fail(SOC_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}

}  // namespace
}  // namespace soc

extern "C" {

int soc_paged_plan(soc_ctx* ctx, int32_t n, const int32_t* old_lens, const int32_t* new_lens, int32_t page_size,
                   int32_t* block_table, int32_t max_pages, int64_t table_stride, int32_t* free_ring, int32_t num_pages,
                   const int64_t* cursors_in, int64_t* cursors_out, int32_t* row_starts, int32_t* positions,
                   int32_t* slots, int32_t max_rows, int32_t* status) {
  SOC_API_BEGIN
  using soc::check_device_rows;
  if (n <= 0 || n > soc::kPlanMaxRequests) return soc::fail(SOC_ERR_INVALID, "paged plan: 1 to 4096 requests");
  SOC_TRY(soc::check_page_size(page_size));
  if (max_pages <= 0 || max_pages > soc::kPlanMaxPages)
    return soc::fail(SOC_ERR_INVALID, "paged plan: max_pages must be 1 to 2^18");
  if (max_rows <= 0 || max_rows > soc::kPlanMaxRows)
    return soc::fail(SOC_ERR_INVALID, "paged plan: max_rows must be 1 to 2^22");
  if (num_pages <= 0 || static_cast<int64_t>(num_pages) * page_size > INT32_MAX)
    return soc::fail(SOC_ERR_INVALID, "paged plan: need num_pages > 0 and num_pages * page_size below 2^31");
  if (ctx == nullptr) return soc::fail(SOC_ERR_INVALID, "null context");
  soc::DeviceScope device(ctx);
  SOC_TRY(check_device_rows(ctx, "paged plan old_lens", old_lens, n, 1, 1, 4));
  SOC_TRY(check_device_rows(ctx, "paged plan new_lens", new_lens, n, 1, 1, 4));
  SOC_TRY(check_device_rows(ctx, "paged plan block_table", block_table, n, table_stride, max_pages, 4));
  SOC_TRY(check_device_rows(ctx, "paged plan free_ring", free_ring, num_pages, 1, 1, 4));
  SOC_TRY(check_device_rows(ctx, "paged plan cursors_in", cursors_in, 2, 1, 1, 8));
  SOC_TRY(check_device_rows(ctx, "paged plan cursors_out", cursors_out, 2, 1, 1, 8));
  SOC_TRY(check_device_rows(ctx, "paged plan row_starts", row_starts, n + 1, 1, 1, 4));
  SOC_TRY(check_device_rows(ctx, "paged plan positions", positions, max_rows, 1, 1, 4));
  SOC_TRY(check_device_rows(ctx, "paged plan slots", slots, max_rows, 1, 1, 4));
  SOC_TRY(check_device_rows(ctx, "paged plan status", status, 1, 1, 1, 4));
  SOC_TRY(soc::ensure_serve_ws(ctx, 0, 64));
  soc::PlanArgs a{n,          old_lens,  new_lens,  block_table, max_pages, table_stride, free_ring,
                  num_pages,  soc::shift_of(page_size), cursors_in, cursors_out, row_starts, positions, slots,
                  max_rows,   status,    ctx->serve_counters};
  const int blocks = std::min(256, std::max(1, (max_rows + soc::kPlanThreads - 1) / soc::kPlanThreads));
  hipLaunchKernelGGL(soc::k_paged_plan, dim3(blocks), dim3(soc::kPlanThreads), 0, ctx->stream, a);
  return soc::hip_status(hipGetLastError(), "paged plan");
  SOC_API_END
}

int soc_paged_append(soc_ctx* ctx, const soc_paged_cache* cache, const soc_rope* rope, const void* q, int64_t q_stride,
                     const void* k, int64_t k_stride, const void* v, int64_t v_stride, int32_t dtype, void* q_out,
                     int64_t q_out_stride, int32_t rows, int32_t q_heads, const int32_t* positions,
                     const int32_t* slots) {
  SOC_API_BEGIN
  using soc::check_device_rows;
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
  const int size = dtype == SOC_DTYPE_F32 ? 4 : 2, hd = cache->head_dim;
  const int64_t kv = static_cast<int64_t>(cache->kv_heads) * hd, qw = static_cast<int64_t>(q_heads) * hd;
  SOC_TRY(soc::check_cache_memory(ctx, cache));
  SOC_TRY(check_device_rows(ctx, "paged append keys", k, rows, k_stride, kv, size));
  SOC_TRY(check_device_rows(ctx, "paged append values", v, rows, v_stride, kv, size));
  if (q_heads > 0) {
    SOC_TRY(check_device_rows(ctx, "paged append queries", q, rows, q_stride, qw, size));
    if (q_out != q) SOC_TRY(check_device_rows(ctx, "paged append q_out", q_out, rows, q_out_stride, qw, size));
  }
  if (rope != nullptr) SOC_TRY(check_device_rows(ctx, "paged append positions", positions, rows, 1, 1, 4));
  SOC_TRY(check_device_rows(ctx, "paged append slots", slots, rows, 1, 1, 4));
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
  const bool wide = soc::four_wide(a.rope) && soc::four_wide(k, k_stride, size) && soc::four_wide(v, v_stride, size) &&
                    (q_heads == 0 ||
                     (soc::four_wide(q, q_stride, size) && soc::four_wide(q_out, q_out_stride, size)));
  auto* kernel = size == 4 ? (wide ? soc::k_paged_append<float, 4> : soc::k_paged_append<float, 1>)
                           : (wide ? soc::k_paged_append<soc::f16, 4> : soc::k_paged_append<soc::f16, 1>);
  hipLaunchKernelGGL(kernel, dim3(rows), dim3(256), 0, ctx->stream, a);
  return soc::hip_status(hipGetLastError(), "paged append");
  SOC_API_END
}

int soc_paged_attention_decode(soc_ctx* ctx, const soc_paged_cache* cache, const void* q, int64_t q_stride,
                               int32_t dtype, const int32_t* block_table, int64_t table_stride, int32_t max_pages,
                               const int32_t* seq_lens, int32_t n, int32_t q_heads, float scale, void* out,
                               int64_t out_stride, float* lse) {
  SOC_API_BEGIN
  using soc::check_device_rows;
  SOC_TRY(soc::check_cache_shape(cache));
  if (dtype != SOC_DTYPE_F32 && dtype != SOC_DTYPE_F16)
    return soc::fail(SOC_ERR_INVALID, "paged attention: dtype must be F32 or F16");
  if (n <= 0 || n > 65535) return soc::fail(SOC_ERR_INVALID, "paged attention: 1 to 65535 sequences");
  if (max_pages <= 0 || static_cast<int64_t>(max_pages) * cache->page_size > INT32_MAX)
    return soc::fail(SOC_ERR_INVALID, "paged attention: need max_pages > 0 and max_pages * page_size below 2^31");
  if (q_heads <= 0 || q_heads % cache->kv_heads != 0 || q_heads / cache->kv_heads > 16)
    return soc::fail(SOC_ERR_INVALID, "paged attention: query heads per KV head must be 1 to 16");
  if (!std::isfinite(scale)) return soc::fail(SOC_ERR_INVALID, "paged attention: scale must be finite");
  if (q == out && q_stride != out_stride)
    return soc::fail(SOC_ERR_INVALID, "paged attention: in place needs equal strides");
  if (ctx == nullptr) return soc::fail(SOC_ERR_INVALID, "null context");
  soc::DeviceScope device(ctx);
  const int size = dtype == SOC_DTYPE_F32 ? 4 : 2, hd = cache->head_dim;
  const int64_t width = static_cast<int64_t>(q_heads) * hd;
  SOC_TRY(soc::check_cache_memory(ctx, cache));
  SOC_TRY(check_device_rows(ctx, "paged attention queries", q, n, q_stride, width, size));
  if (out != q) SOC_TRY(check_device_rows(ctx, "paged attention output", out, n, out_stride, width, size));
  SOC_TRY(check_device_rows(ctx, "paged attention block_table", block_table, n, table_stride, max_pages, 4));
  SOC_TRY(check_device_rows(ctx, "paged attention seq_lens", seq_lens, n, 1, 1, 4));
  if (lse != nullptr) SOC_TRY(check_device_rows(ctx, "paged attention lse", lse, n, q_heads, q_heads, 4));
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
  auto* kernel = size == 4 ? (hd == 128 ? soc::k_paged_attention<float, 128> : soc::k_paged_attention<float, 64>)
                           : (hd == 128 ? soc::k_paged_attention<soc::f16, 128> : soc::k_paged_attention<soc::f16, 64>);
  hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(n) * q_heads), dim3(256), 0, ctx->stream, a);
  return soc::hip_status(hipGetLastError(), "paged attention");
  SOC_API_END
}

}  // extern "C"
