// paged_fork.hip - rows of a paged cache that go on from other rows (soc_paged_fork), the copies of pages that this asks for
// (soc_paged_copy), and the pages in use brought to the front of the pool (soc_paged_compact). The reference has one
// contiguous cache per sequence and one sequence (Mac/gpu/src/runtime/kv_cache.mm:32-204).
#include <algorithm>
#include <string>

#include "paged_host.h"
#include "device_common.h"
#include "paged_math.h"

namespace soc {
namespace {

// ---- fork ------------------------------------------------------------------------------------------------------------
// Whether a page is still named is found from the tables alone: no counts are kept that could go wrong. Each page has a
// 64-bit word that outlives the call; its upper 48 bits are the call that wrote it last, so that nothing is cleared. Every
// entry of the new table (but where the row before has the same page, which is then marked already) raises its page's word to
// (call, all ones); every entry that a row loses (its old page at a place where its new one is another, or none) raises it to
// its own mark, later rows' above earlier ones'. Afterwards the mark of the last entry that lost it stands exactly at a page that no
// row names any more; that entry puts the page into the ring. Maxima do not depend on order. One block's tables have so few entries
// that a mark is (call, the entry's number + 1). In larger ones it is (call, row + 1, 0); an entry that finds its own mark there
// already, as only in a table that names a page twice in a row, sets the lowest bit, and the entries of such a page look in their row
// for a later one.
struct ForkArgs {
  int n;
  const int32_t *parents, *keep, *old_lens;
  const int32_t* table;
  int32_t* new_table;
  int max_pages;
  int64_t table_stride;
  int32_t* ring;
  int num_pages, page_shift;
  const int64_t* cursors_in;
  int64_t* cursors_out;
  int32_t *new_lens, *next_lens, *copies, *copy_count, *status;
  uint64_t* call;    // number of this call
  uint64_t* marks;   // [num_pages]
  // large tables
  int64_t* found;    // head, tail, copies, status
  int chunks;        // of kForkThreads columns
  int32_t* lost;     // [n * chunks][kForkThreads]: pages for the ring
  int32_t* lost_count;
};
constexpr int kForkThreads = 256;   // of a block where the table takes several
constexpr int kSmallThreads = 1024;

// What the rows ask for, in LDS; the same in every block.
template <int kRows, int kWaves>
struct ForkRows {
  int32_t held[kRows];    // pages before
  int32_t parent[kRows];  // -1: none
  int32_t pages[kRows];   // after
  int32_t take[kRows];    // first: the parent's heir; then: which of the pages taken becomes the row's last, or -1
  int32_t wave_total[kWaves];
  int32_t wide;           // the most pages that a row has before or after
};

template <int kEach, int kThreads, typename Rows>
__device__ __forceinline__ int fork_rows(const ForkArgs& a, Rows& s, int64_t head, int64_t tail, bool first_block,
                                         int* copies) {
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
  const int first = tid * kEach, all = (1 << 30);
  int32_t parent[kEach], keep[kEach], old[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    parent[j] = -1;
    keep[j] = old[j] = 0;
    if (first + j < a.n) {
      parent[j] = a.parents[first + j];
      if (a.keep != nullptr) keep[j] = a.keep[first + j];
      old[j] = a.old_lens[first + j];
    }
  }
  if (tid == 0) s.wide = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j)
    if (first + j < a.n) {
      s.held[first + j] = old[j];
      s.take[first + j] = all;
    }
  __syncthreads();
  ForkItem item[kEach];
  bool bad = false;
  int wide = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const bool of_table = parent[j] >= 0 && parent[j] < a.n;
    const int32_t held = of_table ? s.held[parent[j]] : 0;
    item[j] = fork_item(parent[j], a.n, held, a.keep != nullptr ? keep[j] : held, a.max_pages, a.page_shift);
    if (item[j].heir) atomicMin(&s.take[parent[j]], first + j);
    const bool lost = old[j] < 0 || pages_of(old[j], a.page_shift) > a.max_pages;
    bad |= item[j].bad || lost;
    if (lost) old[j] = 0;
    wide = max(wide, max(item[j].pages, pages_of(old[j], a.page_shift)));
  }
  const bool any_bad = __syncthreads_or(bad) != 0;
  bool copied[kEach];
  int sum = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    copied[j] = item[j].partial && !(item[j].heir && s.take[parent[j]] == first + j);
    sum += copied[j];
  }
  int incl = sum;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int o = __shfl_up(incl, d, kWave);
    if (lane >= d) incl += o;
    wide = max(wide, __shfl_xor(wide, d, kWave));
  }
  if (lane == kWave - 1) s.wave_total[wid] = incl;
  if (lane == 0) atomicMax(&s.wide, wide);
  __syncthreads();
  int at = incl - sum, total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / kWave; ++w) {
    if (w < wid) at += s.wave_total[w];
    total += s.wave_total[w];
  }
  const int64_t free_pages = static_cast<int64_t>(static_cast<uint64_t>(tail) - static_cast<uint64_t>(head));
  int status = any_bad ? SOC_PLAN_LENGTHS : 0;
  if (head < 0 || tail < 0 || free_pages < 0 || free_pages > a.num_pages) status |= SOC_PLAN_CURSORS;
  else if (total > free_pages) status |= SOC_PLAN_PAGES;
  *copies = total;
  const int32_t head0 = ring_place(head, a.num_pages);
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int i = first + j;
    if (i >= a.n) continue;
    s.held[i] = pages_of(old[j], a.page_shift);
    // a refused step leaves every row where it was
    s.parent[i] = status == 0 ? parent[j] : i;
    s.pages[i] = status == 0 ? item[j].pages : s.held[i];
    s.take[i] = status == 0 && copied[j] ? at : -1;
    if (first_block) {
      const int32_t len = status == 0 ? item[j].keep : a.old_lens[i];
      a.new_lens[i] = len;
      if (a.next_lens != nullptr) a.next_lens[i] = status != 0 ? len : parent[j] >= 0 ? len + 1 : 0;
      if (status == 0 && copied[j]) {
        int32_t* c = a.copies + 3 * static_cast<int64_t>(at);
        c[0] = a.table[parent[j] * a.table_stride + item[j].pages - 1];
        c[1] = a.ring[ring_place(head0, at, a.num_pages)];
        c[2] = item[j].keep & ((1 << a.page_shift) - 1);
      }
    }
    at += copied[j];
  }
  if (first_block && tid == 0) *a.copy_count = status == 0 ? total : 0;
  __syncthreads();
  return status;
}

// Row i's page at place j before and after; -1 where it has none there. `marked`: the row before has the same page after.
struct ForkEntry {
  int32_t was, is;
  bool marked;
};
template <typename Rows>
__device__ __forceinline__ ForkEntry fork_entry(const ForkArgs& a, const Rows& s, int i, int j, int32_t head0) {
  ForkEntry e{-1, -1, false};
  const bool had = j < s.held[i], has = j < s.pages[i];
  const int p = s.parent[i];
  if (had) e.was = a.table[i * a.table_stride + j];
  if (has) {
    const int t = s.take[i];
    if (t >= 0 && j == s.pages[i] - 1) e.is = a.ring[ring_place(head0, t, a.num_pages)];
    else e.is = p == i ? e.was : a.table[p * a.table_stride + j];
    if (i > 0 && j < s.pages[i - 1] - (s.take[i - 1] >= 0)) e.marked = a.table[s.parent[i - 1] * a.table_stride + j] == e.is;
  }
  return e;
}

// Writes the entry and marks its pages, a lost one with `mark`; whether the row lost one, whose word was *before.
template <typename Rows>
__device__ __forceinline__ bool fork_mark(const ForkArgs& a, const Rows& s, int i, int j, const ForkEntry& e, uint64_t call,
                                          uint64_t mark, uint64_t* before) {
  if (j < s.pages[i]) {
    a.new_table[i * a.table_stride + j] = e.is;
    if (call != 0 && !e.marked && checked_page(e.is, a.num_pages) >= 0)
      atomicMax(reinterpret_cast<unsigned long long*>(a.marks + e.is),
                static_cast<unsigned long long>(call << 16 | 0xffffu));
  }
  const bool lost = call != 0 && j < s.held[i] && (j >= s.pages[i] || e.was != e.is) &&
                    checked_page(e.was, a.num_pages) >= 0;
  if (lost)
    *before = atomicMax(reinterpret_cast<unsigned long long*>(a.marks + e.was), static_cast<unsigned long long>(mark));
  return lost;
}
// Whether row i's entry, of mark `mark`, is the last to have lost its page, which no row names now. After all marks.
template <typename Rows>
__device__ __forceinline__ bool fork_frees(const ForkArgs& a, const Rows& s, int i, int j, const ForkEntry& e,
                                           uint64_t mark) {
  if (j >= s.held[i] || (j < s.pages[i] && e.was == e.is) || checked_page(e.was, a.num_pages) < 0) return false;
  return __hip_atomic_load(a.marks + e.was, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == mark;
}
__device__ __forceinline__ uint64_t row_mark(uint64_t call, int row) { return call << 16 | static_cast<uint32_t>(row + 1) << 1; }

// Small tables: one block does everything, a chain of reads and barriers. (4 rows of 70 pages 7 us, 16 of 64 8.5, 64 of 64 19.4; the
// three launches below 11.4, 11.7 and 12.6 of kernel time: each 1024 entries take the block two turns, 3.6 us.)
__global__ __launch_bounds__(kSmallThreads) void k_fork_small(ForkArgs a) {
  __shared__ ForkRows<kSmallThreads, kSmallThreads / kWave> s;
  __shared__ int32_t freed[2][kSmallThreads / kWave];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
  const int64_t head = a.cursors_in[0], tail = a.cursors_in[1];
  const int32_t head0 = ring_place(head, a.num_pages), tail0 = ring_place(tail, a.num_pages);
  const uint64_t number = *a.call;
  int copies;
  const int status = fork_rows<1, kSmallThreads>(a, s, head, tail, true, &copies);
  const int wide = s.wide, entries = a.n * wide;
  const uint64_t call = status == 0 ? number : 0;
  bool any = false;
  uint64_t before;
  for (int e = tid; e < entries; e += kSmallThreads) {
    const int i = e / wide, j = e - i * wide;
    any |= fork_mark(a, s, i, j, fork_entry(a, s, i, j, head0), call, call << 16 | static_cast<uint32_t>(e + 1), &before);
  }
  int64_t back = 0;  // pages given back so far
  if (__syncthreads_or(any)) {
    const int64_t room = a.num_pages - (tail - head - copies);
    for (int e0 = 0, turn = 0; e0 < entries; e0 += kSmallThreads, turn ^= 1) {
      const int e = e0 + tid, i = min(e, entries - 1) / wide, j = min(e, entries - 1) - i * wide;
      const ForkEntry entry = fork_entry(a, s, i, j, head0);
      const bool free = e < entries && fork_frees(a, s, i, j, entry, call << 16 | static_cast<uint32_t>(e + 1));
      const uint64_t wave = __ballot(free);
      if (lane == 0) freed[turn][wid] = __popcll(wave);
      __syncthreads();
      int64_t at = back + __popcll(wave & ((uint64_t{1} << lane) - 1));
#pragma unroll
      for (int w = 0; w < kSmallThreads / kWave; ++w) {
        if (w < wid) at += freed[turn][w];
        back += freed[turn][w];
      }
      if (free && at < room) a.ring[ring_place(tail0, static_cast<int32_t>(at), a.num_pages)] = entry.was;
    }
    back = min(back, room);
  }
  if (tid == 0) {
    a.cursors_out[0] = status == 0 ? head + copies : head;
    a.cursors_out[1] = status == 0 ? tail + back : tail;
    *a.status = status;
    *a.call = number + 1;
  }
}

// Large tables in three launches: marks; the pages for the ring, by row and chunk of columns; their places in the ring.
template <int kEach>
__global__ __launch_bounds__(kSmallThreads) void k_fork_mark(ForkArgs a) {
  __shared__ ForkRows<kEach * kSmallThreads, kSmallThreads / kWave> s;
  const int64_t head = a.cursors_in[0], tail = a.cursors_in[1];
  const int32_t head0 = ring_place(head, a.num_pages);
  const uint64_t number = *a.call;
  int copies;
  const int status = fork_rows<kEach, kSmallThreads>(a, s, head, tail, blockIdx.x == 0, &copies);
  const uint64_t call = status == 0 ? number : 0;
  constexpr int kUnits = kSmallThreads / kForkThreads;  // of a block at a time
  for (int u = blockIdx.x * kUnits + threadIdx.x / kForkThreads; u < a.n * a.chunks; u += gridDim.x * kUnits) {
    const int i = u / a.chunks, j = (u - i * a.chunks) * kForkThreads + threadIdx.x % kForkThreads;
    if (j >= max(s.held[i], s.pages[i])) continue;
    const ForkEntry e = fork_entry(a, s, i, j, head0);
    const uint64_t mark = row_mark(call, i);
    uint64_t before;
    if (fork_mark(a, s, i, j, e, call, mark, &before) && (before | 1) == (mark | 1))
      atomicMax(reinterpret_cast<unsigned long long*>(a.marks + e.was), static_cast<unsigned long long>(mark | 1));
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.found[0] = head;
    a.found[1] = tail;
    a.found[2] = status == 0 ? copies : 0;
    a.found[3] = status;
  }
}
// After the marks the new table says what each row has: no row needs to be decided again.
__global__ __launch_bounds__(kForkThreads) void k_fork_find(ForkArgs a) {
  __shared__ int32_t freed[2][kForkThreads / kWave];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
  const uint64_t call = *a.call;
  if (a.found[3] != 0) return;
  int turn = 0;
  for (int u = blockIdx.x; u < a.n * a.chunks; u += gridDim.x, turn ^= 1) {
    const int i = u / a.chunks, j = (u - i * a.chunks) * kForkThreads + tid;
    const int held = pages_of(a.old_lens[i], a.page_shift), pages = pages_of(a.new_lens[i], a.page_shift);
    bool free = false;
    int32_t was = -1;
    if (j < held) {
      was = a.table[i * a.table_stride + j];
      if (checked_page(was, a.num_pages) >= 0 && (j >= pages || a.new_table[i * a.table_stride + j] != was)) {
        const uint64_t word = a.marks[was], mark = row_mark(call, i);
        free = (word | 1) == (mark | 1);
        if (free && word != mark)
          for (int k = j + 1; k < held && free; ++k) free = a.table[i * a.table_stride + k] != was;
      }
    }
    const uint64_t wave = __ballot(free);
    if (lane == 0) freed[turn][wid] = __popcll(wave);
    __syncthreads();
    int at = __popcll(wave & ((uint64_t{1} << lane) - 1)), all = 0;
#pragma unroll
    for (int w = 0; w < kForkThreads / kWave; ++w) {
      if (w < wid) at += freed[turn][w];
      all += freed[turn][w];
    }
    if (free) a.lost[static_cast<int64_t>(u) * kForkThreads + at] = was;
    if (tid == 0) a.lost_count[u] = all;
  }
}
__global__ __launch_bounds__(kForkThreads) void k_fork_give(ForkArgs a) {
  __shared__ int32_t part[2][kForkThreads / kWave];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
  const int64_t head = a.found[0], tail = a.found[1];
  const int copies = static_cast<int>(a.found[2]), status = static_cast<int>(a.found[3]);
  const int units = status == 0 ? a.n * a.chunks : 0;
  const int each = (units + gridDim.x - 1) / gridDim.x;
  const int lo = min(units, static_cast<int>(blockIdx.x) * each), hi = min(units, lo + each);
  int before = 0, all = 0;
  for (int u = tid; u < (blockIdx.x == 0 ? units : lo); u += kForkThreads) {
    const int c = a.lost_count[u];
    if (u < lo) before += c;
    all += c;
  }
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    before += __shfl_xor(before, d, kWave);
    all += __shfl_xor(all, d, kWave);
  }
  if (lane == 0) {
    part[0][wid] = before;
    part[1][wid] = all;
  }
  __syncthreads();
  before = all = 0;
#pragma unroll
  for (int w = 0; w < kForkThreads / kWave; ++w) {
    before += part[0][w];
    all += part[1][w];
  }
  const int64_t room = status == 0 ? a.num_pages - (tail - head - copies) : 0;
  const int32_t tail0 = ring_place(tail, a.num_pages);
  for (int u = lo; u < hi; ++u) {
    const int count = a.lost_count[u];
    if (tid < count && before + tid < room)
      a.ring[ring_place(tail0, before + tid, a.num_pages)] = a.lost[static_cast<int64_t>(u) * kForkThreads + tid];
    before += count;
  }
  if (blockIdx.x == 0 && tid == 0) {
    a.cursors_out[0] = head + copies;
    a.cursors_out[1] = tail + min(static_cast<int64_t>(all), room);
    *a.status = status;
    *a.call += 1;
  }
}

// ---- copy ------------------------------------------------------------------------------------------------------------
constexpr int kCopyLayers = 64;  // of a launch
struct CopyArgs {
  f16* planes[2 * kCopyLayers];  // keys and values of each layer
  int64_t stride[kCopyLayers];
  int layers, parts, room;
  const int32_t* moves;
  const int32_t* count;
  int num_pages, page_shift, nkv, vectors;  // vectors: 16 bytes each, of one position of a head
};
constexpr int kCopyEach = 8;  // vectors a thread has on their way

// A unit is 2048 vectors of one page of one plane. Of a partly filled page the places in use are copied, head by head. Bound by
// memory: 90 pages of 64 positions in 4 layers, 8 heads of 128, 189 MB in all, 41 us, 4.6 TB/s, the rate of a large copy. Up to 64
// layers a launch, whose planes are kernel arguments: 3 partly filled pages of 28 layers take 4.3 us of the call's 8.
__global__ __launch_bounds__(256) void k_paged_copy(CopyArgs a) {
  const int count = min(max(a.count != nullptr ? *a.count : a.room, 0), a.room);
  const int per_move = 2 * a.layers * a.parts;
  for (int64_t u = blockIdx.x; u < static_cast<int64_t>(count) * per_move; u += gridDim.x) {
    const int m = static_cast<int>(u / per_move), rest = static_cast<int>(u - static_cast<int64_t>(m) * per_move);
    const int plane = rest / a.parts, part = rest - plane * a.parts;
    const int32_t from = checked_page(a.moves[3 * m], a.num_pages), to = checked_page(a.moves[3 * m + 1], a.num_pages);
    const int places = min(max(a.moves[3 * m + 2], 0), 1 << a.page_shift);
    if (from < 0 || to < 0 || from == to) continue;
    const int run = places * a.vectors, gap = a.vectors << a.page_shift, all = a.nkv * run;  // of a head
    const int first = part * 256 * kCopyEach + threadIdx.x;
    if (part * 256 * kCopyEach >= all) continue;
    const u32x4* x = reinterpret_cast<const u32x4*>(a.planes[plane] + from * a.stride[plane >> 1]);
    u32x4* y = reinterpret_cast<u32x4*>(a.planes[plane] + to * a.stride[plane >> 1]);
    u32x4 v[kCopyEach];
    int at[kCopyEach];
#pragma unroll
    for (int k = 0; k < kCopyEach; ++k) {
      const int i = min(first + k * 256, all - 1), h = i / run;
      at[k] = h * gap + (i - h * run);
      v[k] = load16(x + at[k]);
    }
#pragma unroll
    for (int k = 0; k < kCopyEach; ++k)
      if (first + k * 256 < all) y[at[k]] = v[k];
  }
}

// ---- compact ---------------------------------------------------------------------------------------------------------
constexpr int kCompactThreads = 1024, kCompactPages = 1 << 20, kAlonePages = 1 << 17;
struct CompactArgs {
  int n;
  const int32_t* lens;
  const int32_t* table;
  int32_t* new_table;
  int max_pages;
  int64_t table_stride;
  const int32_t* ring;
  int32_t* new_ring;
  int num_pages, page_shift;
  const int64_t* cursors;
  int32_t* moves;
  int max_moves;
  int32_t *move_count, *status;
  uint32_t* words;  // the bitmap of free pages, zero between calls
  int words_count;
  int* arrived;
};
__device__ __forceinline__ bool good_cursors(int64_t head, int64_t tail, int num_pages) {
  const int64_t free_pages = static_cast<int64_t>(static_cast<uint64_t>(tail) - static_cast<uint64_t>(head));
  return head >= 0 && tail >= 0 && free_pages >= 0 && free_pages <= num_pages;
}

__global__ __launch_bounds__(256) void k_compact_mark(CompactArgs a) {
  const int64_t head = a.cursors[0], tail = a.cursors[1];
  if (!good_cursors(head, tail, a.num_pages)) return;
  const int free_pages = static_cast<int>(tail - head);
  const int32_t head0 = ring_place(head, a.num_pages);
  for (int i = blockIdx.x * 256 + threadIdx.x; i < free_pages; i += gridDim.x * 256) {
    const int32_t page = checked_page(a.ring[ring_place(head0, i, a.num_pages)], a.num_pages);
    if (page >= 0) atomicOr(a.words + (page >> 5), 1u << (page & 31));
  }
}

// Every block holds the whole bitmap and the counts of its groups of words in LDS, and answers for its share of the pages and
// of the table's entries where each goes. kAlone: it forms the bitmap itself, else k_compact_mark has. (2000 pages
// 8.5 us a call so, 11.7 in two launches; 131072 pages 15.6 both ways, each block reading 43000 entries of the ring.)
template <bool kAlone>
__global__ __launch_bounds__(kCompactThreads) void k_compact_apply(CompactArgs a) {
  extern __shared__ uint32_t words[];
  __shared__ int32_t counts[kCompactThreads + 1];
  __shared__ int32_t wave_total[kCompactThreads / kWave];
  __shared__ int last;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
  const int64_t head = a.cursors[0], tail = a.cursors[1];
  const int32_t head0 = ring_place(head, a.num_pages);
  // groups of a power of two words, one a thread
  int shift = 0;
  while ((kCompactThreads << shift) < a.words_count) ++shift;
  const int room = kCompactThreads << shift;
  bool bad = false;
  if constexpr (kAlone) {
    for (int w = tid; w < room; w += kCompactThreads) words[w] = 0;
    __syncthreads();
    const int entries = good_cursors(head, tail, a.num_pages) ? static_cast<int>(tail - head) : 0;
    for (int i0 = tid; i0 < entries; i0 += 8 * kCompactThreads) {
      int32_t page[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) page[k] = a.ring[ring_place(head0, min(i0 + k * kCompactThreads, entries - 1), a.num_pages)];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i0 + k * kCompactThreads < entries && checked_page(page[k], a.num_pages) >= 0)
          atomicOr(words + (page[k] >> 5), 1u << (page[k] & 31));
    }
  } else {
    for (int w = tid; w < room; w += kCompactThreads) words[w] = w < a.words_count ? a.words[w] : 0;
  }
  for (int i = tid; i < a.n; i += kCompactThreads) bad |= a.lens[i] < 0 || pages_of(a.lens[i], a.page_shift) > a.max_pages;
  const bool bad_lens = __syncthreads_or(bad) != 0;
  int sum = 0;
  for (int i = 0; i < 1 << shift; ++i) sum += __popc(words[(tid << shift) + i]);
  int incl = sum;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int o = __shfl_up(incl, d, kWave);
    if (lane >= d) incl += o;
  }
  if (lane == kWave - 1) wave_total[wid] = incl;
  __syncthreads();
  int at = incl - sum;
  for (int w = 0; w < wid; ++w) at += wave_total[w];
  counts[tid] = at;
  if (tid == kCompactThreads - 1) counts[kCompactThreads] = at + sum;
  __syncthreads();
  const FreePages f{words, counts, shift, kCompactThreads};
  const int free_pages = counts[kCompactThreads];
  int status = bad_lens ? SOC_PLAN_LENGTHS : 0;
  // entries of the ring that are no page, or the same one twice
  if (!good_cursors(head, tail, a.num_pages) || free_pages != tail - head) status |= SOC_PLAN_CURSORS;
  const int moved = status == 0 ? min(free_below(f, a.num_pages - free_pages), a.max_moves) : 0;

  const int gid = blockIdx.x * kCompactThreads + tid, stride = gridDim.x * kCompactThreads;
  if (status == 0) {
    for (int p = gid; p < a.num_pages; p += stride) {
      const bool free = words[p >> 5] >> (p & 31) & 1;
      const int above = used_above(f, p, a.num_pages);
      int place = -1;
      if (free) {
        const int rank = free_below(f, p);
        if (rank >= moved) place = rank - moved + (moved - min(moved, above));
      } else if (above < moved) {
        place = moved - 1 - above + max(0, free_below(f, p) - moved);
        int32_t* m = a.moves + 3 * static_cast<int64_t>(above);
        m[0] = p;
        m[1] = free_page(f, above);
        m[2] = 1 << a.page_shift;
      }
      if (place >= 0) a.new_ring[ring_place(head0, place, a.num_pages)] = p;
    }
  } else if (a.new_ring != a.ring && good_cursors(head, tail, a.num_pages)) {
    for (int i = gid; i < tail - head; i += stride) {
      const int32_t place = ring_place(head0, i, a.num_pages);
      a.new_ring[place] = a.ring[place];
    }
  }
  for (int64_t e = gid; e < static_cast<int64_t>(a.n) * a.max_pages; e += stride) {
    const int i = static_cast<int>(e / a.max_pages), j = static_cast<int>(e - static_cast<int64_t>(i) * a.max_pages);
    const int len = a.lens[i];
    if (len < 0 || j >= pages_of(len, a.page_shift)) continue;
    int32_t page = a.table[i * a.table_stride + j];
    if (status == 0 && checked_page(page, a.num_pages) >= 0 && !(words[page >> 5] >> (page & 31) & 1)) {
      const int above = used_above(f, page, a.num_pages);
      if (above < moved) page = free_page(f, above);
    }
    a.new_table[i * a.table_stride + j] = page;
  }
  if (gid == 0) {
    *a.move_count = moved;
    *a.status = status;
  }
  if constexpr (kAlone) return;
  // the last block clears the bitmap: all others have read it
  __syncthreads();
  if (tid == 0) last = atomicAdd(a.arrived, 1) == static_cast<int>(gridDim.x) - 1;
  __syncthreads();
  if (!last) return;
  for (int w = tid; w < a.words_count; w += kCompactThreads) a.words[w] = 0;
  if (tid == 0) st_dev(a.arrived, 0);
}

// The context's words of pages: 64 words of which the first two are the number of the next fork, a bitmap, and the marks. All
// zero when new, the number 1.
__global__ void k_first_call(uint64_t* call) { *call = 1; }
struct PageWords {
  uint64_t* call;
  uint32_t* bits;
  uint64_t* marks;
};
int ensure_page_words(soc_ctx* ctx, int32_t num_pages, PageWords* out) {
  if (ctx->page_words_pages < num_pages) {
    const size_t pages = (static_cast<size_t>(num_pages) + 4095) / 4096 * 4096;
    const size_t bytes = 256 + pages / 8 + pages * 8;
    SOC_HIP_TRY(hipStreamSynchronize(ctx->stream));
    (void)hipFree(ctx->page_words);
    ctx->page_words = nullptr;
    ctx->page_words_pages = 0;
    if (hipMalloc(&ctx->page_words, bytes) != hipSuccess) {
      (void)hipGetLastError();
      ctx->page_words = nullptr;
      return fail(SOC_ERR_NOMEM, "allocation of " + std::to_string(bytes) + " bytes of page words failed");
    }
    hipError_t e = hipMemsetAsync(ctx->page_words, 0, bytes, ctx->stream);
    if (e == hipSuccess) {
      hipLaunchKernelGGL(k_first_call, dim3(1), dim3(1), 0, ctx->stream,
                         reinterpret_cast<uint64_t*>(ctx->page_words));
      e = hipGetLastError();
    }
    if (e != hipSuccess) {
      (void)hipFree(ctx->page_words);
      ctx->page_words = nullptr;
      return fail(SOC_ERR_HIP, std::string("page words: ") + hipGetErrorString(e));
    }
    ctx->page_words_pages = static_cast<int64_t>(pages);
  }
  out->call = reinterpret_cast<uint64_t*>(ctx->page_words);
  out->bits = ctx->page_words + 64;
  out->marks = reinterpret_cast<uint64_t*>(out->bits + ctx->page_words_pages / 32);
  return SOC_OK;
}

int check_pool(const char* what, int32_t n, int32_t page_size, int32_t max_pages, int32_t num_pages) {
  const std::string name(what);
  if (n <= 0 || n > kPlanMaxRequests) return fail(SOC_ERR_INVALID, name + ": 1 to 4096 rows");
  SOC_TRY(check_page_size(page_size));
  if (max_pages <= 0 || max_pages > kPlanMaxPages)
    return fail(SOC_ERR_INVALID, name + ": max_pages must be 1 to 2^18");
  if (num_pages <= 0 || static_cast<int64_t>(num_pages) * page_size > INT32_MAX)
    return fail(SOC_ERR_INVALID, name + ": need num_pages > 0 and num_pages * page_size below 2^31");
  return SOC_OK;
}

// Whether `rows` rows of `width` elements, `stride` apart, at a and at b have a byte in common (as ranges).
bool overlap(const void* a, int64_t a_count, const void* b, int64_t b_count, int size) {
  const char *x = static_cast<const char*>(a), *y = static_cast<const char*>(b);
  return x < y + b_count * size && y < x + a_count * size;
}

}  // namespace
}  // namespace soc

extern "C" {

int soc_paged_fork(soc_ctx* ctx, int32_t n, const int32_t* parents, const int32_t* keep, const int32_t* old_lens,
                   int32_t page_size, const int32_t* block_table, int32_t* new_table, int32_t max_pages,
                   int64_t table_stride, int32_t* free_ring, int32_t num_pages, const int64_t* cursors_in,
                   int64_t* cursors_out, int32_t* new_lens, int32_t* next_lens, int32_t* copies, int32_t* copy_count,
                   int32_t* status) {
  SOC_API_BEGIN
  SOC_TRY(soc::check_pool("paged fork", n, page_size, max_pages, num_pages));
  if (ctx == nullptr) return soc::fail(SOC_ERR_INVALID, "null context");
  soc::DeviceScope device(ctx);
  soc::Operands operands(ctx);
  SOC_TRY(operands.array("paged fork parents", parents, n, 4));
  if (keep != nullptr) SOC_TRY(operands.array("paged fork keep", keep, n, 4));
  SOC_TRY(operands.array("paged fork old_lens", old_lens, n, 4));
  SOC_TRY(operands.rows("paged fork block_table", block_table, n, table_stride, max_pages, 4));
  SOC_TRY(operands.rows("paged fork new_table", new_table, n, table_stride, max_pages, 4));
  SOC_TRY(operands.array("paged fork free_ring", free_ring, num_pages, 4));
  SOC_TRY(operands.array("paged fork cursors_in", cursors_in, 2, 8));
  SOC_TRY(operands.array("paged fork cursors_out", cursors_out, 2, 8));
  SOC_TRY(operands.array("paged fork new_lens", new_lens, n, 4));
  if (next_lens != nullptr) SOC_TRY(operands.array("paged fork next_lens", next_lens, n, 4));
  SOC_TRY(operands.rows("paged fork copies", copies, n, 3, 3, 4));
  SOC_TRY(operands.array("paged fork copy_count", copy_count, 1, 4));
  SOC_TRY(operands.array("paged fork status", status, 1, 4));
  const int64_t span = (n - 1) * table_stride + max_pages;
  if (soc::overlap(block_table, span, new_table, span, 4))
    return soc::fail(SOC_ERR_INVALID, "paged fork: new_table must not overlap block_table");
  for (const int32_t* out : {static_cast<const int32_t*>(new_lens), static_cast<const int32_t*>(next_lens)})
    for (const int32_t* in : {parents, keep, old_lens})
      if (out != nullptr && in != nullptr && soc::overlap(out, n, in, n, 4))
        return soc::fail(SOC_ERR_INVALID, "paged fork: new_lens and next_lens must not overlap parents, keep or old_lens");
  soc::PageWords words;
  SOC_TRY(soc::ensure_page_words(ctx, num_pages, &words));
  soc::ForkArgs a{};
  a.n = n;
  a.parents = parents;
  a.keep = keep;
  a.old_lens = old_lens;
  a.table = block_table;
  a.new_table = new_table;
  a.max_pages = max_pages;
  a.table_stride = table_stride;
  a.ring = free_ring;
  a.num_pages = num_pages;
  a.page_shift = soc::shift_of(page_size);
  a.cursors_in = cursors_in;
  a.cursors_out = cursors_out;
  a.new_lens = new_lens;
  a.next_lens = next_lens;
  a.copies = copies;
  a.copy_count = copy_count;
  a.status = status;
  a.call = words.call;
  a.marks = words.marks;
  if (n <= soc::kSmallThreads && static_cast<int64_t>(n) * max_pages <= 2048) {
    hipLaunchKernelGGL(soc::k_fork_small, dim3(1), dim3(soc::kSmallThreads), 0, ctx->stream, a);
    return soc::hip_status(hipGetLastError(), "paged fork");
  }
  a.chunks = (max_pages + soc::kForkThreads - 1) / soc::kForkThreads;
  const int units = n * a.chunks;  // at most 2^22
  const size_t lists = static_cast<size_t>(units) * soc::kForkThreads * 4, counts = static_cast<size_t>(units) * 4;
  SOC_TRY(soc::ensure_serve_ws(ctx, 64 + lists + counts, 0));
  a.found = reinterpret_cast<int64_t*>(ctx->serve_ws);
  a.lost = reinterpret_cast<int32_t*>(ctx->serve_ws + 64);
  a.lost_count = reinterpret_cast<int32_t*>(ctx->serve_ws + 64 + lists);
  const int blocks = std::min((units + 3) / 4, 256);
  auto* mark = n <= soc::kSmallThreads ? soc::k_fork_mark<1> : soc::k_fork_mark<4>;
  hipLaunchKernelGGL(mark, dim3(blocks), dim3(soc::kSmallThreads), 0, ctx->stream, a);
  hipLaunchKernelGGL(soc::k_fork_find, dim3(std::min(units, 2048)), dim3(soc::kForkThreads), 0, ctx->stream, a);
  hipLaunchKernelGGL(soc::k_fork_give, dim3(std::min(units, 1024)), dim3(soc::kForkThreads), 0, ctx->stream, a);
  return soc::hip_status(hipGetLastError(), "paged fork");
  SOC_API_END
}

int soc_paged_copy(soc_ctx* ctx, const soc_paged_cache* caches, int32_t layers, const int32_t* moves,
                   const int32_t* move_count, int32_t max_moves) {
  SOC_API_BEGIN
  if (layers <= 0 || layers > 4096) return soc::fail(SOC_ERR_INVALID, "paged copy: 1 to 4096 layers");
  if (max_moves <= 0 || max_moves > (1 << 22)) return soc::fail(SOC_ERR_INVALID, "paged copy: 1 to 2^22 moves");
  if (caches == nullptr) return soc::fail(SOC_ERR_INVALID, "null paged cache");
  for (int32_t l = 0; l < layers; ++l) {
    SOC_TRY(soc::check_cache_shape(caches + l));
    if (caches[l].num_pages != caches[0].num_pages || caches[l].page_size != caches[0].page_size ||
        caches[l].kv_heads != caches[0].kv_heads || caches[l].head_dim != caches[0].head_dim)
      return soc::fail(SOC_ERR_INVALID, "paged copy: the layers must have one shape");
  }
  if (ctx == nullptr) return soc::fail(SOC_ERR_INVALID, "null context");
  soc::DeviceScope device(ctx);
  soc::Operands operands(ctx);
  SOC_TRY(operands.rows("paged copy moves", moves, max_moves, 3, 3, 4));
  if (move_count != nullptr) SOC_TRY(operands.array("paged copy move_count", move_count, 1, 4));
  for (int32_t l = 0; l < layers; ++l) SOC_TRY(soc::check_cache_memory(operands, caches + l));
  soc::CopyArgs a{};
  a.room = max_moves;
  a.moves = moves;
  a.count = move_count;
  a.num_pages = caches[0].num_pages;
  a.page_shift = soc::shift_of(caches[0].page_size);
  a.nkv = caches[0].kv_heads;
  a.vectors = caches[0].head_dim / 8;
  const int64_t page = (static_cast<int64_t>(a.nkv) * a.vectors) << a.page_shift;
  a.parts = static_cast<int>((page + 256 * soc::kCopyEach - 1) / (256 * soc::kCopyEach));
  for (int32_t first = 0; first < layers; first += soc::kCopyLayers) {
    a.layers = std::min(soc::kCopyLayers, layers - first);
    for (int l = 0; l < a.layers; ++l) {
      a.planes[2 * l] = static_cast<soc::f16*>(caches[first + l].keys);
      a.planes[2 * l + 1] = static_cast<soc::f16*>(caches[first + l].values);
      a.stride[l] = soc::page_stride(caches + first + l);
    }
    const int64_t units = static_cast<int64_t>(max_moves) * 2 * a.layers * a.parts;
    hipLaunchKernelGGL(soc::k_paged_copy, dim3(static_cast<uint32_t>(std::min<int64_t>(units, 2048))), dim3(256), 0,
                       ctx->stream, a);
    SOC_TRY(soc::hip_status(hipGetLastError(), "paged copy"));
  }
  return SOC_OK;
  SOC_API_END
}

int soc_paged_compact(soc_ctx* ctx, int32_t n, const int32_t* lens, int32_t page_size, const int32_t* block_table,
                      int32_t* new_table, int32_t max_pages, int64_t table_stride, const int32_t* free_ring,
                      int32_t* new_ring, int32_t num_pages, const int64_t* cursors, int32_t* moves, int32_t max_moves,
                      int32_t* move_count, int32_t* status) {
  SOC_API_BEGIN
  SOC_TRY(soc::check_pool("paged compact", n, page_size, max_pages, num_pages));
  if (num_pages > soc::kCompactPages) return soc::fail(SOC_ERR_INVALID, "paged compact: at most 2^20 pages");
  if (max_moves <= 0 || max_moves > (1 << 22)) return soc::fail(SOC_ERR_INVALID, "paged compact: 1 to 2^22 moves");
  if (ctx == nullptr) return soc::fail(SOC_ERR_INVALID, "null context");
  soc::DeviceScope device(ctx);
  soc::Operands operands(ctx);
  SOC_TRY(operands.array("paged compact lens", lens, n, 4));
  SOC_TRY(operands.rows("paged compact block_table", block_table, n, table_stride, max_pages, 4));
  SOC_TRY(operands.rows("paged compact new_table", new_table, n, table_stride, max_pages, 4));
  SOC_TRY(operands.array("paged compact free_ring", free_ring, num_pages, 4));
  SOC_TRY(operands.array("paged compact new_ring", new_ring, num_pages, 4));
  SOC_TRY(operands.array("paged compact cursors", cursors, 2, 8));
  SOC_TRY(operands.rows("paged compact moves", moves, max_moves, 3, 3, 4));
  SOC_TRY(operands.array("paged compact move_count", move_count, 1, 4));
  SOC_TRY(operands.array("paged compact status", status, 1, 4));
  const int64_t span = (n - 1) * table_stride + max_pages;
  if ((new_table != block_table && soc::overlap(block_table, span, new_table, span, 4)) ||
      (new_ring != free_ring && soc::overlap(free_ring, num_pages, new_ring, num_pages, 4)))
    return soc::fail(SOC_ERR_INVALID, "paged compact: table and ring are updated in place or have no byte in common");
  soc::CompactArgs a{};
  a.n = n;
  a.lens = lens;
  a.table = block_table;
  a.new_table = new_table;
  a.max_pages = max_pages;
  a.table_stride = table_stride;
  a.ring = free_ring;
  a.new_ring = new_ring;
  a.num_pages = num_pages;
  a.page_shift = soc::shift_of(page_size);
  a.cursors = cursors;
  a.moves = moves;
  a.max_moves = max_moves;
  a.move_count = move_count;
  a.status = status;
  a.words_count = (num_pages + 31) / 32;
  int room = soc::kCompactThreads;
  while (room < a.words_count) room *= 2;
  const size_t lds = static_cast<size_t>(room) * 4;  // at most 128 KiB
  const int64_t most = std::max<int64_t>(num_pages, static_cast<int64_t>(n) * max_pages);
  dim3 blocks(static_cast<uint32_t>(std::min<int64_t>(256, (most + soc::kCompactThreads - 1) / soc::kCompactThreads)));
  // in place, a block could write the ring while another still reads it: there one block does a small pool (4096 pages 12.7 us, 8192
  // 21.5; the two launches 13.6)
  const bool one = new_ring == free_ring && most <= 4 * soc::kCompactThreads;
  if (one) blocks.x = 1;
  if (num_pages <= soc::kAlonePages && (one || new_ring != free_ring)) {
    hipLaunchKernelGGL(soc::k_compact_apply<true>, blocks, dim3(soc::kCompactThreads), lds, ctx->stream, a);
    return soc::hip_status(hipGetLastError(), "paged compact");
  }
  soc::PageWords words;
  SOC_TRY(soc::ensure_page_words(ctx, num_pages, &words));
  SOC_TRY(soc::ensure_serve_ws(ctx, 0, 1));
  a.words = words.bits;
  a.arrived = ctx->serve_counters;
  if (lds > (size_t{48} << 10))
    SOC_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(soc::k_compact_apply<false>),
                                    hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
  hipLaunchKernelGGL(soc::k_compact_mark, dim3(std::min(256, (num_pages + 255) / 256)), dim3(256), 0, ctx->stream, a);
  hipLaunchKernelGGL(soc::k_compact_apply<false>, blocks, dim3(soc::kCompactThreads), lds, ctx->stream, a);
  return soc::hip_status(hipGetLastError(), "paged compact");
  SOC_API_END
}

}  // extern "C"
