// paged_math.h - index arithmetic of the paged key-value cache and of its page planner: every index that comes out of
// caller memory on the device (page ids, slots, ring cursors, lengths) passes one of these before it becomes an address.
// Plain functions, so that a host program can check them with hostile values.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define SOC_HD __host__ __device__ __forceinline__
#else
#define SOC_HD inline
#endif

namespace soc {

// Pages that hold `len` positions (len >= 0; 0 pages for 0).
SOC_HD int32_t pages_of(int32_t len, int page_shift) { return len <= 0 ? 0 : ((len - 1) >> page_shift) + 1; }

// A page id as it may be used: itself, or -1 where it names no page of the cache.
SOC_HD int32_t checked_page(int32_t page, int32_t num_pages) { return page >= 0 && page < num_pages ? page : -1; }

// A slot (page * page_size + place) as it may be used: itself, or -1 where it lies outside the cache.
SOC_HD int32_t checked_slot(int32_t slot, int32_t num_pages, int page_shift) {
  return slot >= 0 && (slot >> page_shift) < num_pages ? slot : -1;
}

// The slot of place `offset` of page `page`; -1 where the page is none of the cache (num_pages << page_shift fits 31
// bits).
SOC_HD int32_t slot_of(int32_t page, int32_t offset, int32_t num_pages, int page_shift) {
  return checked_page(page, num_pages) < 0 ? -1 : (page << page_shift) + offset;
}

// The keys of a sequence that may be read: its length; 0 for a negative one; -1 for one beyond its table's pages.
SOC_HD int32_t checked_length(int32_t len, int32_t max_pages, int page_shift) {
  return len < 0 ? 0 : pages_of(len, page_shift) > max_pages ? -1 : len;
}

// Keys a block of the decode attention takes of a sequence of `len` > 0 keys: whole tiles of 128 (32 for each of its four
// waves). The sequence gets `splits` blocks, while it has tiles for them and none would take more than 1024 keys; a longer
// one the multiple of `splits` with which no block takes more than `most` (a multiple of 128) keys. Never more than `grid`
// blocks. The multiple, because `splits` fills the card once: 16 sequences of 3000 keys, 32 query and 8 KV heads, take
// 38 us with four blocks each, 43 with three. More than 16 blocks take 256 keys at least: joining parts costs more than
// shorter chunks save (one sequence of 4071 keys, 32 and 8 heads: 11.6 us with 16 blocks, 12.4 with 32).
// Where `grid` is the least of these bounds (8 in a large batch), a long sequence's blocks take as many keys as that
// leaves them, beyond `most`.
constexpr int32_t kAttentionMost = 1024;
SOC_HD int32_t attention_chunk(int32_t len, int32_t splits, int32_t grid, int32_t most) {
  int32_t want = splits;
  if ((len - 1) / kAttentionMost >= splits) want = ((len - 1) / most / splits + 1) * splits;
  want = want < grid ? want : grid;
  const int32_t each = want == 1 ? len - 1 : (len - 1) / want;
  const int32_t chunk = (each / 128 + 1) * 128;
  return chunk == 128 && len > 16 * 128 ? 256 : chunk;
}

// How keys are split over waves or blocks: `splits` chunks where none would be longer than `most` keys, multiples of that
// where there are more keys, at most `grid` chunks; chunks of whole `least` keys (a multiple of 32).
struct Chunks {
  int32_t splits, grid, least, most;
};
SOC_HD int32_t chunk_of(int32_t keys, const Chunks& c) {
  if (keys <= 0) return c.least;
  int32_t want = ((keys - 1) / c.most / c.splits + 1) * c.splits;
  want = want < c.grid ? want : c.grid;
  return ((keys - 1) / want / c.least + 1) * c.least;
}
SOC_HD int32_t chunks_of(int32_t keys, int32_t chunk) { return keys <= 0 ? 0 : (keys - 1) / chunk + 1; }
// For `units` times up to `longest` keys (>= 1): enough chunks for `waves` of them at a time, no more than `room` a unit.
SOC_HD Chunks chunks_for(int64_t units, int64_t longest, int32_t waves, int32_t least, int32_t most, int32_t room) {
  Chunks c{1, 1, least, most};
  const int64_t splits = (waves + units - 1) / units;
  c.splits = static_cast<int32_t>(splits < room ? splits : room);
  const int64_t grid = ((longest - 1) / most / c.splits + 1) * c.splits, fit = (longest + least - 1) / least;
  const int64_t several = 8 * static_cast<int64_t>(waves) / units;  // of large batches' long rows
  int64_t g = grid < fit ? grid : fit;
  g = g < (several > 8 ? several : 8) ? g : (several > 8 ? several : 8);
  c.grid = static_cast<int32_t>(g < room ? g : room);
  return c;
}

// Place of a cursor in a ring of `size` entries, for any cursor.
SOC_HD int32_t ring_place(int64_t cursor, int32_t size) {
  return static_cast<int32_t>(static_cast<uint64_t>(cursor) % static_cast<uint64_t>(size));
}
// Place of the entry i <= size (< 2^30) places on from `place`.
SOC_HD int32_t ring_place(int32_t place, int32_t i, int32_t size) {
  const int32_t at = place + i;
  return at < size ? at : at - size < size ? at - size : 0;
}

// What a step asks for that brings a request from `before` to `after` positions: new rows, pages to take and to give
// back. The sums over kPlanMaxRequests requests stay within 32 bits: rows and pages saturate beyond kPlanMaxRows, which
// the plan refuses, and a table row has at most kPlanMaxPages pages.
constexpr int32_t kPlanMaxRequests = 4096, kPlanMaxRows = 1 << 22, kPlanMaxPages = 1 << 18;
struct PlanItem {
  int32_t rows, take, give;
  bool bad;  // a length that is negative or longer than the table's pages
};
SOC_HD PlanItem plan_item(int32_t before, int32_t after, int32_t max_pages, int page_shift) {
  PlanItem p{0, 0, 0, false};
  if (before < 0 || after < 0 || pages_of(before, page_shift) > max_pages || pages_of(after, page_shift) > max_pages) {
    p.bad = true;
    return p;
  }
  const int32_t had = pages_of(before, page_shift), want = pages_of(after, page_shift);
  const int32_t most = kPlanMaxRows + 1;
  if (after > before) p.rows = after - before < most ? after - before : most;
  if (want > had) p.take = want - had;
  if (had > want) p.give = had - want;
  return p;
}

// What a row of a forked table asks for: the first `keep` positions of its parent, which holds `held` positions. `heir`: its
// last page is partly filled by it and is the parent's own partly filled last page, which one such child may keep. A page
// that the parent has filled counts as shared, whoever else holds it.
struct ForkItem {
  int32_t keep, pages;
  bool partial, heir;
  bool bad;  // a parent or a length out of range
};
SOC_HD ForkItem fork_item(int32_t parent, int32_t n, int32_t held, int32_t keep, int32_t max_pages, int page_shift) {
  ForkItem f{0, 0, false, false, false};
  if (parent == -1) return f;
  if (parent < 0 || parent >= n || held < 0 || pages_of(held, page_shift) > max_pages || keep < 0 || keep > held) {
    f.bad = true;
    return f;
  }
  const int32_t inside = (1 << page_shift) - 1;
  f.keep = keep;
  f.pages = pages_of(keep, page_shift);
  f.partial = (keep & inside) != 0;
  f.heir = f.partial && (held & inside) != 0 && f.pages == pages_of(held, page_shift);
  return f;
}

// A pool's pages as a bitmap, one bit a free page, with the free pages before each group of 2^group_shift words of 32:
// counts[g], g <= the number of groups, the last of them all. Words hold no bit beyond the pool's pages.
struct FreePages {
  const uint32_t* words;
  const int32_t* counts;
  int group_shift, groups;
};
// Free pages below page p, 0 <= p <= the pool's pages.
SOC_HD int32_t free_below(const FreePages& f, int32_t p) {
  const int32_t w = p >> 5, g = w >> f.group_shift;
  int32_t c = f.counts[g];
  for (int32_t i = g << f.group_shift; i < w; ++i) c += __builtin_popcount(f.words[i]);
  if ((p & 31) != 0) c += __builtin_popcount(f.words[w] & ((1u << (p & 31)) - 1u));
  return c;
}
// The free page that `rank` free pages lie below, 0 <= rank < all of them.
SOC_HD int32_t free_page(const FreePages& f, int32_t rank) {
  int32_t lo = 0, hi = f.groups;  // counts[lo] <= rank < counts[hi]
  while (hi - lo > 1) {
    const int32_t mid = (lo + hi) >> 1;
    if (f.counts[mid] <= rank) lo = mid;
    else hi = mid;
  }
  int32_t left = rank - f.counts[lo], w = lo << f.group_shift;
  const int32_t end = (lo + 1) << f.group_shift;
  uint32_t word = f.words[w];
  for (int32_t c = __builtin_popcount(word); left >= c && w + 1 < end; c = __builtin_popcount(word)) {
    left -= c;
    word = f.words[++w];
  }
  for (; left > 0; --left) word &= word - 1;
  return (w << 5) + (word != 0 ? __builtin_ctz(word) : 0);
}
// Pages in use above page p.
SOC_HD int32_t used_above(const FreePages& f, int32_t p, int32_t num_pages) {
  return num_pages - 1 - p - (f.counts[f.groups] - free_below(f, p + 1));
}

}  // namespace soc
