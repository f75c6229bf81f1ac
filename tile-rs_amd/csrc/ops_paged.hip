// Paged cache entry points of the C ABI (include/tilers_hip.h, section 2): th_kv_cache_write,
// th_kv_cache_read and th_attention_paged.  The host checks what it can see (sizes, types,
// pointers); lengths and tables are device data that the kernels bring into range.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>
#include <type_traits>

#include "kernels/attention_paged.hpp"
#include "kernels/kv_cache.hpp"
#include "ops_common.hpp"
#include "runtime.hpp"

using th::fail;
using namespace th::ops;

namespace {

template <int N> using Int = std::integral_constant<int, N>;

// Lanes that one launch can have.
constexpr uint64_t kMostLanes = 0xffffffffu;

bool codes(th_dtype d) { return d == TH_E4M3 || d == TH_I8; }

// The structs' sizes and pointers; `need_rows`: the call has new tokens.
int check_paged(const char* op, const th_kv_pages* p, const th_kv_batch* s, bool need_rows,
                th::PagedPool* pool, th::PagedSeqs* seqs) {
  const std::string at = std::string(op) + ": ";
  if (!p || !s) return fail(TH_KERNEL_ERROR, at + "null pages or batch");
  if (p->dtype != TH_F16 && p->dtype != TH_BF16 && !codes(p->dtype))
    return fail(TH_KERNEL_ERROR, at + "the cache's dtype must be F16, BF16, E4M3 or I8");
  if (p->num_kv_heads == 0) return fail(TH_KERNEL_ERROR, at + "num_kv_heads == 0");
  if (p->head_dim == 0 || p->head_dim % 16 != 0 || p->head_dim > 256)
    return fail(TH_KERNEL_ERROR, at + "head_dim must be a multiple of 16 up to 256");
  if (p->page_size < 16 || p->page_size > 65536 || (p->page_size & (p->page_size - 1)) != 0)
    return fail(TH_KERNEL_ERROR, at + "page_size must be a power of two of 16 to 65536");
  if (p->num_pages == 0 || p->num_pages > 0x7fffffffu)
    return fail(TH_KERNEL_ERROR, at + "num_pages must be of 1 to 2^31 - 1");
  const uint64_t dense = static_cast<uint64_t>(p->page_size) * p->head_dim;   // below 2^24
  if (p->num_kv_heads > 0xffffffffu / dense)
    return fail(TH_KERNEL_ERROR, at + "a page has 2^32 elements or more");
  const uint64_t page = dense * p->num_kv_heads;
  if (p->page_stride != 0 && (p->page_stride < page || p->page_stride % 16 != 0))
    return fail(TH_KERNEL_ERROR, at + "page_stride must be a multiple of 16 elements and hold a page");
  if (p->page_stride > (uint64_t{1} << 61) / p->num_pages)
    return fail(TH_KERNEL_ERROR, at + "page_stride is too large");
  if (!p->k || !p->v) return fail(TH_KERNEL_ERROR, at + "null pages");
  if (!aligned16(p->k) || !aligned16(p->v))
    return fail(TH_KERNEL_ERROR, at + "pages must be 16-byte aligned");
  if (codes(p->dtype)) {
    if (!p->k_scale || !p->v_scale)
      return fail(TH_KERNEL_ERROR, at + "an 8-bit cache needs k_scale and v_scale");
    if (!aligned16(p->k_scale) || !aligned16(p->v_scale))
      return fail(TH_KERNEL_ERROR, at + "scales must be 16-byte aligned");
  }
  if (s->batch > 0x7ffffffeu || s->total_q > 0x7fffffffu)
    return fail(TH_KERNEL_ERROR, at + "batch and total_q must be below 2^31");
  if (s->batch != 0) {
    if (!s->kv_len || (need_rows && !s->q_start) || (s->max_pages != 0 && !s->page_table))
      return fail(TH_KERNEL_ERROR, at + "null page_table, q_start or kv_len");
    for (const void* x : {static_cast<const void*>(s->kv_len), static_cast<const void*>(s->q_start),
                          static_cast<const void*>(s->page_table)})
      if ((reinterpret_cast<uintptr_t>(x) & 3u) != 0)
        return fail(TH_KERNEL_ERROR, at + "page_table, q_start and kv_len must be 4-byte aligned");
  }
  uint32_t shift = 4;
  while ((1u << shift) < p->page_size) ++shift;
  *pool = {p->k, p->v, p->k_scale, p->v_scale, p->page_stride ? p->page_stride : page,
           p->num_kv_heads, p->head_dim};
  *seqs = {s->page_table, s->q_start, s->kv_len, s->batch, s->max_pages, s->total_q, p->num_pages,
           shift, static_cast<uint32_t>(std::min<uint64_t>(
                      static_cast<uint64_t>(s->max_pages) << shift, 0x7fffffffu))};
  return TH_OK;
}

// f(cache type, lanes of a row of eight-value pieces)
template <class F>
void by_cache(th_dtype cache, uint32_t head_dim, F&& f) {
  auto lanes = [&](auto ct) {
    if (head_dim <= 64) f(ct, Int<8>{});
    else if (head_dim <= 128) f(ct, Int<16>{});
    else f(ct, Int<32>{});
  };
  switch (cache) {
    case TH_F16: lanes(Int<th::kF16>{}); break;
    case TH_BF16: lanes(Int<th::kBF16>{}); break;
    case TH_E4M3: lanes(Int<th::kE4M3>{}); break;
    default: lanes(Int<th::kI8>{}); break;
  }
}
template <class F>
void by_float(th_dtype d, F&& f) {
  switch (d) {
    case TH_F32: f(Int<th::kF32>{}); break;
    case TH_F16: f(Int<th::kF16>{}); break;
    default: f(Int<th::kBF16>{}); break;
  }
}

// ---- attention ---------------------------------------------------------------------------

uint32_t head_width(uint32_t head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

// How a call is split over its kernels, from what the host knows: the structs' sizes.
struct AttnPlan {
  uint32_t runs = 0;         // workgroups of the rows' kernel (0: not launched)
  uint32_t tile_rows = 16;
  bool rows_merge = false;
  uint32_t split_rows = 0;   // sequences of more rows go to the chunks' kernel
  uint64_t items = 0;        // (tile, head) items of the chunks' kernel, at most (0: not launched)
  uint32_t parts = 1;
  size_t rows_bytes = 0, chunk_bytes = 0;
};

// CUs of a whole MI355X, not of the current device, so that the workspace's size does not
// depend on it.
constexpr uint32_t kCus = 256;

AttnPlan attn_plan(const th::PagedSeqs& s, const th_kv_pages& pages, uint32_t group) {
  const uint32_t nkv = pages.num_kv_heads, head_dim = pages.head_dim;
  // Rows up to which a sequence stays with the rows' kernel, which widens codes once for a tile
  // of 32 rows where the chunks' kernel does it for 256.  16 sequences of 2000 positions, 8 heads
  // of 128, with 32, 64 and 96 rows for each head: bf16 44, 57, 90 us there, 43 at each size on
  // the chunks' kernel; e4m3 38, 45, 66 there, 51 to 53 on the chunks' kernel.
  const uint32_t split = codes(pages.dtype) ? 64 : 32;
  AttnPlan p;
  const uint32_t hd = head_width(head_dim);
  const uint64_t rows = static_cast<uint64_t>(s.total_q) * group;
  // a token per sequence: all of them steps, most likely
  const bool chunks = hd <= 128 && rows > split && s.total_q > s.batch;
  p.split_rows = !chunks ? 0xffffffffu : s.batch == 1 ? 0u : split;
  if (p.split_rows != 0) {
    // more than 16 rows each, on average: 32 at a time, so that the cache is read once for them
    // (16 sequences of 2000, 32 rows: bf16 50 -> 44 us, e4m3 36 -> 38; 64 of 500, 24 rows: 49 ->
    // 31, 36 -> 25).  256 columns leave no registers for that.
    if (hd <= 128 && rows > 16ull * s.batch) p.tile_rows = 32;
    // at least the units of any lengths that the structs allow
    const uint64_t tiles = rows / p.tile_rows + s.batch;
    const uint64_t cap = uint64_t{1} << 40;
    const uint64_t blocks = s.cap / th::pgd::rows::UNIT + (s.cap % th::pgd::rows::UNIT != 0);
    const uint64_t units = std::min(cap, std::min(cap, tiles * nkv) * std::max<uint64_t>(1, blocks));
    const uint32_t per_cu = hd == 256 ? 1 : 2;   // (rows_waves)
    p.runs = static_cast<uint32_t>(std::min<uint64_t>(per_cu * kCus, units));
    p.rows_merge = p.runs > 1 && blocks > 1;
    if (p.rows_merge)
      p.rows_bytes = static_cast<size_t>(p.runs) * 2 *
                     th::pgd::rows::rec(static_cast<int>(hd), static_cast<int>(p.tile_rows)) *
                     sizeof(float);
  }
  if (chunks) {
    const uint64_t some = rows / (p.split_rows + 1);   // sequences of more than split_rows rows
    const uint64_t tiles = rows / th::pgd::chunk::TR + std::min<uint64_t>(s.batch, some);
    p.items = std::max<uint64_t>(1, tiles) * nkv;
    const uint32_t most = std::max(1u, s.cap / th::pgd::chunk::KB / th::pgd::chunk::kLeast);
    // as many parts as leave no CU idle; from a round of items on, none (in two
    // parts: 2048 tokens after 5952 290 -> 309 us, five prompts 104 -> 141, three chunks of 700
    // 185 -> 182), up to 16 (128 tokens after 7872: 46 us; at most 8 parts: 52; none: 263)
    if (p.items < kCus)
      p.parts = static_cast<uint32_t>(
          std::min<uint64_t>(std::min(16u, most), (kCus + p.items - 1) / p.items));
    if (p.parts > 1)
      p.chunk_bytes = static_cast<size_t>(p.parts) * s.total_q * nkv * group *
                      th::pgd::chunk::rec(static_cast<int>(hd)) * sizeof(float);
  }
  return p;
}

template <int DT, int CT, int HD>
void attn_paged_go(const th::pgd::AttnArgs& a, const AttnPlan& p, hipStream_t s) {
  constexpr uint32_t NT = th::pgd::rows::NT;
  if (p.runs && p.tile_rows == 16)
    hipLaunchKernelGGL((th::pgd::attn_paged_rows<DT, CT, HD, 1>), dim3(p.runs), dim3(NT), 0, s, a);
  if constexpr (HD <= 128) {
    if (p.runs && p.tile_rows == 32)
      hipLaunchKernelGGL((th::pgd::attn_paged_rows<DT, CT, HD, 2>), dim3(p.runs), dim3(NT), 0, s,
                         a);
    if (p.items)
      hipLaunchKernelGGL((th::pgd::attn_paged_chunk<DT, CT, HD>),
                         dim3(static_cast<uint32_t>(p.items * p.parts)), dim3(th::pgd::chunk::NT),
                         0, s, a);
  }
  const uint32_t first = p.rows_merge ? p.runs - 1 : 0;
  constexpr uint32_t MNT = th::pgd::merge_nt, RPB = MNT / (HD / 4);   // (chunk_merge)
  const uint32_t tokens =
      p.items && p.parts > 1 ? a.seqs.total_q * ((a.nh + RPB - 1) / RPB) : 0;   // parts: some 10^4 rows
  if (first + tokens)
    hipLaunchKernelGGL((th::pgd::attn_paged_merge<DT, HD>), dim3(first + tokens), dim3(MNT), 0, s,
                       a, first);
}

}  // namespace

extern "C" {

int th_kv_cache_write(const th_kv_pages* pages, const th_kv_batch* seqs, const void* k,
                      const void* v, uint64_t stride, th_dtype dtype, th_stream s) {
  th::PagedPool pool;
  th::PagedSeqs sq;
  if (!valid_dtype(dtype)) return fail(TH_KERNEL_ERROR, "kv_cache_write: unknown dtype");
  TH_TRY(check_paged("kv_cache_write", pages, seqs, true, &pool, &sq));
  const uint64_t dense = static_cast<uint64_t>(pool.nkv) * pool.head_dim;
  if (stride == 0) stride = dense;
  if (stride < dense || stride % (16 / dtype_size(dtype)) != 0)
    return fail(TH_KERNEL_ERROR,
                "kv_cache_write: stride must hold a token's heads in whole 16-byte blocks");
  if (sq.batch == 0 || sq.total_q == 0) return TH_OK;
  if (stride > (uint64_t{1} << 60) / sq.total_q)
    return fail(TH_KERNEL_ERROR, "kv_cache_write: stride is too large");
  if ((uint64_t{sq.total_q} + 3) / 4 * 256 > kMostLanes)
    return fail(TH_KERNEL_ERROR, "kv_cache_write: grid too large");
  if (!k || !v) return fail(TH_KERNEL_ERROR, "kv_cache_write: null pointer");
  if (!aligned16(k) || !aligned16(v))
    return fail(TH_KERNEL_ERROR, "kv_cache_write: K and V must be 16-byte aligned");
  by_float(dtype, [&](auto dt) {
    by_cache(pages->dtype, pool.head_dim, [&](auto ct, auto lg) {
      hipLaunchKernelGGL((th::kv_cache_write<dt.value, ct.value, lg.value, 4>),
                         dim3((sq.total_q + 3) / 4), dim3(256), 0, as_stream(s), pool, sq, k, v,
                         stride);
    });
  });
  return launch_status("kv_cache_write launch");
}

int th_kv_cache_read(const th_kv_pages* pages, const th_kv_batch* seqs, void* k, void* v,
                     uint32_t max_seq, th_dtype dtype, th_stream s) {
  th::PagedPool pool;
  th::PagedSeqs sq;
  if (!valid_dtype(dtype)) return fail(TH_KERNEL_ERROR, "kv_cache_read: unknown dtype");
  TH_TRY(check_paged("kv_cache_read", pages, seqs, false, &pool, &sq));
  if (sq.batch == 0 || max_seq == 0) return TH_OK;
  if (max_seq > 0x7fffffffu) return fail(TH_KERNEL_ERROR, "kv_cache_read: max_seq must be below 2^31");
  if (!k || !v) return fail(TH_KERNEL_ERROR, "kv_cache_read: null pointer");
  if (!aligned16(k) || !aligned16(v))
    return fail(TH_KERNEL_ERROR, "kv_cache_read: K and V must be 16-byte aligned");
  int rc = TH_OK;
  by_float(dtype, [&](auto dt) {
    by_cache(pages->dtype, pool.head_dim, [&](auto ct, auto lg) {
      constexpr uint32_t U = 2, per = U * 256 / lg.value;
      const uint32_t nchunks = (max_seq + per - 1) / per;
      const uint64_t rows = static_cast<uint64_t>(sq.batch) * pool.nkv;
      if (rows * 256 > kMostLanes / nchunks) {
        rc = fail(TH_KERNEL_ERROR, "kv_cache_read: grid too large");
        return;
      }
      hipLaunchKernelGGL((th::kv_cache_read<dt.value, ct.value, lg.value, U>),
                         dim3(static_cast<uint32_t>(rows * nchunks)), dim3(256), 0, as_stream(s),
                         pool, sq, k, v, max_seq, nchunks);
    });
  });
  TH_TRY(rc);
  return launch_status("kv_cache_read launch");
}

size_t th_attention_paged_workspace_size(const th_kv_pages* pages, const th_kv_batch* seqs,
                                         uint32_t num_heads) {
  th::PagedPool pool;
  th::PagedSeqs sq;
  if (check_paged("attention_paged_workspace_size", pages, seqs, false, &pool, &sq) != TH_OK ||
      num_heads == 0 || num_heads % pool.nkv != 0)
    return 0;   // (th_attention_paged refuses the same arguments)
  if (sq.batch == 0 || sq.total_q == 0) return 0;
  const AttnPlan p = attn_plan(sq, *pages, num_heads / pool.nkv);
  return p.rows_bytes + p.chunk_bytes;
}

int th_attention_paged(const void* q, const th_kv_pages* pages, const th_kv_batch* seqs, void* o,
                       uint32_t num_heads, uint64_t q_stride, th_dtype dtype, void* workspace,
                       size_t workspace_bytes, th_stream s) {
  th::pgd::AttnArgs a;
  if (dtype != TH_F16 && dtype != TH_BF16)
    return fail(TH_KERNEL_ERROR, "attention_paged: dtype must be F16 or BF16");
  TH_TRY(check_paged("attention_paged", pages, seqs, true, &a.pool, &a.seqs));
  if (!codes(pages->dtype) && pages->dtype != dtype)
    return fail(TH_KERNEL_ERROR, "attention_paged: a 16-bit cache must have the dtype of Q");
  const uint32_t nkv = a.pool.nkv, D = a.pool.head_dim;
  if (num_heads == 0 || num_heads % nkv != 0)
    return fail(TH_KERNEL_ERROR, "attention_paged: num_heads must be a multiple of num_kv_heads");
  const uint64_t dense = static_cast<uint64_t>(num_heads) * D;
  if (q_stride == 0) q_stride = dense;
  if (q_stride < dense || q_stride % 8 != 0)
    return fail(TH_KERNEL_ERROR,
                "attention_paged: q_stride must hold a token's heads and be a multiple of 8");
  if (a.seqs.batch == 0 || a.seqs.total_q == 0) return TH_OK;
  if (static_cast<uint64_t>(a.seqs.total_q) * num_heads > 0x7fffffffu)
    return fail(TH_KERNEL_ERROR, "attention_paged: total_q * num_heads must be below 2^31");
  if (q_stride > (uint64_t{1} << 60) / a.seqs.total_q)
    return fail(TH_KERNEL_ERROR, "attention_paged: q_stride is too large");
  if (!q || !o) return fail(TH_KERNEL_ERROR, "attention_paged: null pointer");
  if (!aligned16(q) || !aligned16(o))
    return fail(TH_KERNEL_ERROR, "attention_paged: Q and O must be 16-byte aligned");
  a.q = static_cast<const uint16_t*>(q);
  a.o = static_cast<uint16_t*>(o);
  a.q_stride = q_stride;
  a.nh = num_heads;
  a.group = num_heads / nkv;
  a.scale_log2 = th::kLog2e / std::sqrt(static_cast<float>(D));
  const AttnPlan plan = attn_plan(a.seqs, *pages, a.group);
  if (plan.items * plan.parts * th::pgd::chunk::NT > kMostLanes)
    return fail(TH_KERNEL_ERROR, "attention_paged: grid too large");
  const size_t need = plan.rows_bytes + plan.chunk_bytes;
  th::ScratchHold hold;
  if (workspace) {
    if (workspace_bytes < need)
      return fail(TH_MEMORY_ERROR, "attention_paged: workspace of " +
                                       std::to_string(workspace_bytes) + " bytes < required " +
                                       std::to_string(need));
    if (!aligned16(workspace))
      return fail(TH_KERNEL_ERROR, "attention_paged: workspace must be 16-byte aligned");
  } else {
    if (need && stream_capturing(as_stream(s)))
      return fail(TH_MEMORY_ERROR,
                  "attention_paged: a stream that is being captured needs a workspace");
    if (need) TH_TRY(th::stream_scratch(as_stream(s), need, &workspace, &hold));
  }
  a.ws = static_cast<float*>(workspace);
  a.chunk_ws = a.ws + plan.rows_bytes / sizeof(float);
  a.tile_rows = plan.tile_rows;
  a.split_rows = plan.split_rows;
  a.runs = plan.runs;
  a.parts = plan.parts;
  auto go = [&](auto dt, auto ct) {
    switch (head_width(D)) {
      case 64: attn_paged_go<dt.value, ct.value, 64>(a, plan, as_stream(s)); break;
      case 128: attn_paged_go<dt.value, ct.value, 128>(a, plan, as_stream(s)); break;
      default: attn_paged_go<dt.value, ct.value, 256>(a, plan, as_stream(s)); break;
    }
  };
  auto cache = [&](auto dt) {
    if (pages->dtype == TH_E4M3) go(dt, Int<th::kE4M3>{});
    else if (pages->dtype == TH_I8) go(dt, Int<th::kI8>{});
    else go(dt, dt);
  };
  if (dtype == TH_F16) cache(Int<th::kF16>{});
  else cache(Int<th::kBF16>{});
  return launch_status("attention_paged launch");
}

}  // extern "C"
