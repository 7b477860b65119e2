// Index arithmetic of forked rows, of a pool's bitmap and of keys split into chunks (soc_amd/csrc/paged_math.h) against loops
// that say what it means, with hostile lengths and parents.
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../soc_amd/csrc/paged_math.h"

#define CHECK(x)                                            \
  do {                                                      \
    if (!(x)) {                                             \
      std::printf("line %d: %s\n", __LINE__, #x);           \
      return 1;                                             \
    }                                                       \
  } while (0)

int main() {
  using namespace soc;
  const int32_t odd[] = {INT32_MIN, INT32_MIN + 1, -2, -1, 0, 1, 15, 16, 17, 31, 32, 33, 159, 160, 161, INT32_MAX - 1, INT32_MAX};
  for (int32_t parent : odd)
    for (int32_t held : odd)
      for (int32_t keep : odd)
        for (int n : {1, 2, 16, 4096}) {
          const ForkItem f = fork_item(parent, n, held, keep, 10, 4);
          if (parent == -1) {
            CHECK(!f.bad && f.keep == 0 && f.pages == 0 && !f.partial && !f.heir);
            continue;
          }
          const bool good = parent >= 0 && parent < n && held >= 0 && held <= 160 && keep >= 0 && keep <= held;
          CHECK(f.bad == !good);
          if (!good) {
            CHECK(f.keep == 0 && f.pages == 0 && !f.partial && !f.heir);
            continue;
          }
          CHECK(f.keep == keep && f.pages == (keep + 15) / 16 && f.pages <= 10);
          CHECK(f.partial == (keep % 16 != 0));
          CHECK(f.heir == (keep % 16 != 0 && held % 16 != 0 && (keep + 15) / 16 == (held + 15) / 16));
        }
  // a pool of any size, any density, groups of 1 to 8 words
  std::srand(1);
  for (int pages : {1, 2, 31, 32, 33, 63, 64, 65, 100, 511, 1000, 4096})
    for (int density : {0, 1, 50, 99, 100})
      for (int shift : {0, 1, 3}) {
        const int count = (pages + 31) / 32, groups = ((count + (1 << shift) - 1) >> shift) + 2;
        std::vector<uint32_t> words(static_cast<size_t>(groups) << shift, 0u);
        std::vector<int> free;
        for (int p = 0; p < pages; ++p)
          if (std::rand() % 100 < density) {
            words[p / 32] |= 1u << (p % 32);
            free.push_back(p);
          }
        std::vector<int32_t> counts(groups + 1, 0);
        for (int g = 0; g < groups; ++g) {
          counts[g + 1] = counts[g];
          for (int i = 0; i < 1 << shift; ++i) counts[g + 1] += __builtin_popcount(words[(g << shift) + i]);
        }
        const FreePages f{words.data(), counts.data(), shift, groups};
        int below = 0;
        for (int p = 0; p <= pages; ++p) {
          CHECK(free_below(f, p) == below);
          if (p == pages) break;
          const bool is = words[p / 32] >> (p % 32) & 1;
          const int above_free = static_cast<int>(free.size()) - below - is;
          CHECK(used_above(f, p, pages) == pages - 1 - p - above_free);
          below += is;
        }
        for (size_t r = 0; r < free.size(); ++r) CHECK(free_page(f, static_cast<int32_t>(r)) == free[r]);
      }
  // chunks of any number of keys, also of more than they were laid out for: whole multiples of `least`, all keys in them, none
  // empty, no more of them than the grid has blocks or a unit has room
  constexpr int64_t kMostKeys = int64_t{1} << 26;  // of 2^18 pages of 256
  for (int64_t units : {int64_t{1}, int64_t{3}, int64_t{64}, int64_t{1000}, int64_t{32768}, int64_t{1} << 24})
    for (int64_t longest : {int64_t{1}, int64_t{31}, int64_t{128}, int64_t{4097}, int64_t{131072}, kMostKeys})
      for (int32_t waves : {256, 512, 2048})
        for (int32_t least : {32, 128})
          for (int32_t most : {128, 256, 1024})
            for (int32_t room : {1, 16, 64}) {
              const Chunks c = chunks_for(units, longest, waves, least, most, room);
              CHECK(c.splits >= 1 && c.splits <= room && c.grid >= 1 && c.grid <= room && c.least == least && c.most == most);
              for (int64_t keys : {int64_t{0}, int64_t{1}, int64_t{32}, int64_t{33}, int64_t{127}, int64_t{129}, longest - 1, longest,
                                   4 * longest, kMostKeys}) {
                if (keys > kMostKeys) continue;
                const int32_t k = static_cast<int32_t>(keys), chunk = chunk_of(k, c), many = chunks_of(k, chunk);
                CHECK(chunk > 0 && chunk % least == 0);
                CHECK(many >= 0 && many <= c.grid && (many == 0) == (k == 0));
                CHECK(static_cast<int64_t>(many) * chunk >= k && (many == 0 || static_cast<int64_t>(many - 1) * chunk < k));
                if (k > 0 && c.grid >= ((k - 1) / most / c.splits + 1) * static_cast<int64_t>(c.splits)) CHECK(chunk <= std::max(most, least));
              }
            }
  std::printf("fork math ok\n");
  return 0;
}
