// The index arithmetic of the paged kernels (csrc/kernels/paged_index.hpp) against whatever the
// device arrays may hold: every row, position and page that comes out is in range.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "kernels/paged_index.hpp"

#define CHECK(x)                                              \
  do {                                                        \
    if (!(x)) {                                               \
      std::printf("%s:%d: %s\n", __FILE__, __LINE__, #x);     \
      std::exit(1);                                           \
    }                                                         \
  } while (0)

int main() {
  using namespace th;
  std::mt19937 rng(7);
  const int32_t odd[] = {0, 1, -1, 15, 16, 17, 99, 100, 101, -100, 2147483647, -2147483647 - 1};
  auto any = [&]() -> int32_t {
    return rng() % 3 ? odd[rng() % (sizeof(odd) / sizeof(odd[0]))] : static_cast<int32_t>(rng());
  };
  for (int round = 0; round < 20000; ++round) {
    const uint32_t batch = 1 + rng() % 4, max_pages = rng() % 5, shift = 4 + rng() % 3;
    const uint32_t num_pages = 1 + rng() % 7, total_q = rng() % 101;
    std::vector<int32_t> table(batch * max_pages), start(batch + 1), len(batch);
    for (auto* v : {&table, &start, &len})
      for (auto& x : *v) x = any();
    for (auto& x : table)
      if (rng() % 2) x = static_cast<int32_t>(rng() % num_pages);
    const PagedSeqs s{table.data(), start.data(), len.data(), batch,    max_pages,
                      total_q,      num_pages,    shift,      max_pages << shift};
    for (uint32_t b = 0; b < batch; ++b) {
      const PagedChunk c = paged_chunk(s, b);
      CHECK(c.first <= total_q && c.n <= total_q - c.first);
      CHECK(c.held <= s.cap);
      for (uint32_t i = 0; i < c.n; ++i) {
        const uint32_t vis = paged_visible(c, i);
        CHECK(vis <= c.held);
        CHECK(i == 0 || vis >= paged_visible(c, i - 1));
        const int32_t pos = c.base + static_cast<int32_t>(i);
        CHECK(vis == (pos < 0 ? 0u : static_cast<uint32_t>(pos) + 1 < c.held
                                         ? static_cast<uint32_t>(pos) + 1 : c.held));
      }
      for (int j = 0; j < 40; ++j) {
        const uint32_t pos = j < 20 ? rng() % (s.cap + 40) : rng();
        const int32_t page = paged_page(s, b, pos);   // reads inside `table` (checked by -fsanitize)
        CHECK(page >= -1 && page < static_cast<int32_t>(num_pages));
        CHECK(page < 0 || (pos < s.cap && table[b * max_pages + (pos >> shift)] == page));
        CHECK(paged_row(s, pos) == pos % (1u << shift));
      }
    }
  }
  // a chunk of a plain batch
  const int32_t table[] = {2, 0}, start[] = {0, 3}, len[] = {20};
  const PagedSeqs s{table, start, len, 1, 2, 3, 3, 4, 32};
  const PagedChunk c = paged_chunk(s, 0);
  CHECK(c.first == 0 && c.n == 3 && c.base == 17 && c.held == 20);
  CHECK(paged_visible(c, 0) == 18 && paged_visible(c, 2) == 20);
  CHECK(paged_page(s, 0, 15) == 2 && paged_page(s, 0, 16) == 0 && paged_page(s, 0, 32) == -1);
  std::printf("ok\n");
}
