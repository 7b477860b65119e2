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

}  // namespace soc
