// The index arithmetic of the paged cache (soc_amd/csrc/paged_math.h) on hostile values: whatever lengths, page ids,
// slots and cursors device memory may hold, what comes out is in bounds or -1. Host only.
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <random>
#include <vector>

#include "../../soc_amd/csrc/paged_math.h"

namespace {
int failures = 0;
void expect(bool ok, const char* what) {
  if (!ok && ++failures <= 20) std::printf("FAILED: %s\n", what);
}
}  // namespace

int main() {
  const std::vector<int32_t> words = {INT32_MIN, INT32_MIN + 1, -65536, -2, -1, 0, 1, 2, 15, 16, 17, 255, 256, 257, 65535,
                                      1 << 20, (1 << 20) + 1, 1 << 22, (1 << 22) + 1, 1 << 30, INT32_MAX - 1, INT32_MAX};
  for (int shift = 4; shift <= 8; ++shift) {
    for (int32_t len : words) {
      const int32_t p = soc::pages_of(len, shift);
      expect(p >= 0, "pages_of is not negative");
      if (len > 0) {
        expect((int64_t{p} << shift) >= len && (int64_t{p - 1} << shift) < len, "pages_of is the least that holds len");
      } else {
        expect(p == 0, "no pages for no positions");
      }
      for (int32_t max_pages : {1, 2, 300, 1 << 18, INT32_MAX >> shift}) {
        const int32_t c = soc::checked_length(len, max_pages, shift);
        expect(c >= -1, "checked_length");
        if (c > 0) expect(((c - 1) >> shift) < max_pages && c == len, "the last key's table entry is in the row");
        if (len >= 0 && len <= (int64_t{max_pages} << shift)) expect(c == len, "a fitting length is itself");
        for (int32_t after : words) {
          const soc::PlanItem i = soc::plan_item(len, after, max_pages, shift);
          expect(i.rows >= 0 && i.take >= 0 && i.give >= 0, "a plan's parts are not negative");
          expect(i.rows <= soc::kPlanMaxRows + 1, "rows saturate");
          if (i.bad) expect(i.rows == 0 && i.take == 0 && i.give == 0, "a bad request asks for nothing");
          if (max_pages <= soc::kPlanMaxPages)
            expect(int64_t{16} * i.take + (int64_t{16} << 18) <= INT32_MAX, "sums of 16 requests fit");
          if (!i.bad) {
            expect(soc::pages_of(len, shift) + i.take <= max_pages, "taken pages have entries");
            expect(soc::pages_of(after, shift) + i.give <= max_pages, "given pages have entries");
            expect(i.take == 0 || i.give == 0, "a request takes or gives");
          }
        }
      }
    }
    for (int32_t pages : {1, 2, 1000, INT32_MAX >> shift}) {
      for (int32_t w : words) {
        const int32_t p = soc::checked_page(w, pages);
        expect(p == -1 || (p >= 0 && p < pages), "checked_page");
        expect((w >= 0 && w < pages) ? p == w : p == -1, "a page of the cache is itself");
        const int32_t s = soc::checked_slot(w, pages, shift);
        expect(s == -1 || (s >= 0 && s < (int64_t{pages} << shift)), "checked_slot");
        const int32_t t = soc::slot_of(w, (1 << shift) - 1, pages, shift);
        expect(t == -1 || (t >= 0 && t < (int64_t{pages} << shift)), "slot_of");
        expect((p >= 0) == (t >= 0), "slot_of of a page of the cache");
      }
    }
  }
  std::mt19937_64 rng(5);
  for (int i = 0; i < 200000; ++i) {
    const int32_t len = 1 + static_cast<int32_t>((rng() >> 33) >> (rng() % 31)) % (1 << 30);
    const int32_t splits = 1 + rng() % 200, grid = 1 + rng() % 300, most = 256 * (1 + rng() % 8);
    const int64_t chunk = soc::attention_chunk(len, splits, grid, most), blocks = (len - 1) / chunk + 1;
    expect(chunk > 0 && chunk % 128 == 0, "a chunk is whole tiles");
    expect(blocks <= grid, "the grid holds a sequence's blocks");
    expect((blocks - 1) * chunk < len, "no block is empty");
    if ((int64_t{len} - 1) / most + splits <= grid) expect(chunk <= std::max(most, soc::kAttentionMost), "no block takes more than it may");
    if (len > 128 * splits && splits <= grid) expect(blocks * 2 >= splits, "a long sequence gets its blocks");
  }
  for (int i = 0; i < 200000; ++i) {
    const int64_t cursor = static_cast<int64_t>(rng() >> (rng() % 64)) * (i % 2 ? 1 : -1);
    const int32_t size = 1 + static_cast<int32_t>((rng() >> 33) >> (rng() % 31)) % ((1 << 27) - 1);
    const int32_t at = static_cast<int32_t>(rng() >> 33) % (size + 1);
    const int32_t base = soc::ring_place(cursor, size), place = soc::ring_place(base, at, size);
    expect(base >= 0 && base < size && place >= 0 && place < size, "ring_place is in the ring");
    if (cursor >= 0 && cursor < (int64_t{1} << 62))
      expect(place == static_cast<int32_t>((cursor + at) % size), "ring_place is the sum modulo the size");
  }
  if (failures) {
    std::printf("%d checks failed\n", failures);
    return 1;
  }
  std::printf("paged math ok\n");
  return 0;
}
