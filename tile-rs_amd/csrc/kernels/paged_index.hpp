// Where a sequence's tokens and cached positions lie in a paged cache: the index arithmetic of
// the paged kernels (kv_cache.hpp, attention_paged.hpp), also compiled for the CPU by its test.
//
// The lengths and tables are device data that no host check sees, so every value read from them
// is brought into range here before an address is made of it.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define TH_HD __host__ __device__ __forceinline__
#else
#define TH_HD inline
#endif

namespace th {

// The batch as the kernels see it.
struct PagedSeqs {
  const int32_t* table;     // [batch][max_pages]
  const int32_t* q_start;   // [batch + 1]
  const int32_t* kv_len;    // [batch]
  uint32_t batch, max_pages, total_q;
  uint32_t num_pages, shift;   // pages of the pool, log2 of the positions in a page
  uint32_t cap;                // positions a table row reaches: max_pages << shift, below 2^31
};

// New tokens of one sequence: rows [first, first + n) of Q, K and V.  q_start is clamped to
// [0, total_q] and a falling one is an empty chunk, so no row lies past total_q.
struct PagedChunk {
  uint32_t first, n;
  int32_t base;    // position of the first new token (negative where kv_len < n)
  uint32_t held;   // positions that exist in the cache: kv_len, at most cap
};

TH_HD uint32_t paged_clamp(int32_t x, uint32_t hi) {
  return x < 0 ? 0u : static_cast<uint32_t>(x) < hi ? static_cast<uint32_t>(x) : hi;
}

TH_HD PagedChunk paged_chunk(const PagedSeqs& s, uint32_t b) {
  const uint32_t first = paged_clamp(s.q_start[b], s.total_q);
  const uint32_t last = paged_clamp(s.q_start[b + 1], s.total_q);
  const uint32_t len = paged_clamp(s.kv_len[b], 0x7fffffffu);
  PagedChunk c;
  c.first = first;
  c.n = last > first ? last - first : 0u;   // total_q < 2^31, so base does not overflow
  c.base = static_cast<int32_t>(len) - static_cast<int32_t>(c.n);
  c.held = len < s.cap ? len : s.cap;
  return c;
}

// Positions that new token i sees: those up to its own that are in the cache.
TH_HD uint32_t paged_visible(const PagedChunk& c, uint32_t i) {
  const int32_t own = c.base + static_cast<int32_t>(i) + 1;   // at most kv_len
  return paged_clamp(own, c.held);
}

// The page that holds position `pos` of sequence b, or -1 where there is none: past the table,
// or an entry outside the pool (a page that was given back, say).
TH_HD int32_t paged_page(const PagedSeqs& s, uint32_t b, uint32_t pos) {
  if (pos >= s.cap) return -1;
  const int32_t id = s.table[static_cast<uint64_t>(b) * s.max_pages + (pos >> s.shift)];
  return id >= 0 && static_cast<uint32_t>(id) < s.num_pages ? id : -1;
}

TH_HD uint32_t paged_row(const PagedSeqs& s, uint32_t pos) { return pos & ((1u << s.shift) - 1u); }

}  // namespace th
