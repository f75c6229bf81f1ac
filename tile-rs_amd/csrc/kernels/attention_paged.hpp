// Causal GQA attention of ragged chunks of new tokens over a paged cache, 16-bit Q and O, the
// cache in the same type or in 8-bit codes with a scale per position and head.
//
// For one sequence and kv head the rows are the (new token i, query head g) pairs, r = i G + g,
// so that the G query heads of a kv head share each K/V read.  Row r sees visible(i) positions:
//     s_j = ks_j (q . k_j) log2(e) / sqrt(D)      ks_j, vs_j: the codes' scales (1 in 16 bits)
//     o   = sum_j 2^(s_j - m) vs_j v_j / sum_j 2^(s_j - m)
// The codes are exact in either 16-bit type, so the products run on them and the scales are
// applied in f32: ks to the score, vs to the weight, before it is rounded to 16 bits.  Without
// codes the weights' sum is that of the rounded ones.
//
// Two kernels share a call, which finds out on the device whose rows are whose: sequences of few
// rows are bound by the cache's bytes (attn_paged_rows), those of many by the products
// (attn_paged_chunk).
#pragma once

#include "common.hpp"
#include "kv_cache.hpp"

#include <type_traits>

namespace th {
namespace pgd {

// Two f32 -> packed 16-bit pair, to nearest even.
template <int DT>
__device__ __forceinline__ uint32_t pack2h(float lo, float hi) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  if constexpr (DT == kBF16) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{lo, hi}, b2));
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{lo, hi}, h2));
  }
}

// What pack2h's rounding left of a pair, rounded itself.
template <int DT>
__device__ __forceinline__ uint32_t pack2h_rest(float lo, float hi, uint32_t xy) {
  if constexpr (DT == kBF16) {
    lo -= __uint_as_float(xy << 16);
    hi -= __uint_as_float(xy & 0xffff0000u);
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 x = __builtin_bit_cast(h2, xy);
    lo -= static_cast<float>(x[0]);
    hi -= static_cast<float>(x[1]);
  }
  return pack2h<DT>(lo, hi);
}

// a + x + y of a pair as pack2h rounded it.  (Weights are summed as the product with V takes them,
// so that the mean is one of weights that sum to 1: a token that has all the weight gives its
// values exactly.)
template <int DT>
__device__ __forceinline__ float add_pair(uint32_t xy, float a) {
  if constexpr (DT == kBF16) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, xy),
                                           __builtin_bit_cast(b2, 0x3f803f80u), a, false);
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, xy), __builtin_bit_cast(h2, 0x3c003c00u),
                                  a, false);
  }
}

// Four codes -> four values of type DT, exactly.
template <int DT, int CT>
__device__ __forceinline__ u32x2 widen4(uint32_t w) {
  u32x2 out;
  if constexpr (CT == kE4M3) {
    const int d = static_cast<int>(w);
    if constexpr (DT == kBF16) {
      out[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d, 1.0f, false));
      out[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d, 1.0f, true));
    } else {
      out[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d, 1.0f, false));
      out[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d, 1.0f, true));
    }
  } else if constexpr (DT == kBF16) {
    // whole numbers below 2^8: their f32 patterns end in 16 zero bits
    uint32_t f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      f[j] = __float_as_uint(static_cast<float>(static_cast<int8_t>(w >> (8 * j))));
    out[0] = pack_halves<true>(f[0], f[1]);
    out[1] = pack_halves<true>(f[2], f[3]);
  } else {
    // 0x6400 + u is 1024 + u in f16 for u < 1024; u = code + 128
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const uint32_t u = w ^ 0x80808080u;
    const h2 off = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
    const uint32_t a = __builtin_amdgcn_perm(0x64646464u, u, 0x07010700u);
    const uint32_t b = __builtin_amdgcn_perm(0x64646464u, u, 0x07030702u);
    out[0] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, a) - off);
    out[1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, b) - off);
  }
  return out;
}

// paged_page with a scalar load, for a sequence and position that the whole wave shares.  (The
// table does not change while a call runs.)
__device__ __forceinline__ int32_t wave_page(const PagedSeqs& s, uint32_t b, uint32_t pos) {
  typedef __attribute__((address_space(4))) const int32_t* scalar_ptr;
  b = __builtin_amdgcn_readfirstlane(b);
  pos = __builtin_amdgcn_readfirstlane(pos);
  if (pos >= s.cap) return -1;
  const uint64_t at = static_cast<uint64_t>(b) * s.max_pages + (pos >> s.shift);
  const int32_t id = *(scalar_ptr)(reinterpret_cast<uintptr_t>(s.table + at));
  return id >= 0 && static_cast<uint32_t>(id) < s.num_pages ? id : -1;
}

// 16 bytes at `off` of the `bytes` bytes at p, zeros past them (the buffer's range check): p and
// bytes are the wave's, off is the lane's.
template <bool NT>
__device__ __forceinline__ u32x4 load_within(const void* p, uint32_t bytes, uint32_t off) {
  const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, static_cast<int>(bytes),
                                                   0x00020000);
  return __builtin_bit_cast(
      u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, static_cast<int>(off), 0, NT ? 2 : 0));
}
// An offset that is past every range.
constexpr uint32_t kPast = 0x7ffffff0u;

// The table's entry for min(pos, end - 1), 1 <= end <= cap, unchecked (paged_checked): whatever is
// done with it waits for the load.
__device__ __forceinline__ int32_t wave_entry(const PagedSeqs& s, uint32_t b, uint32_t pos,
                                              uint32_t end) {
  typedef __attribute__((address_space(4))) const int32_t* scalar_ptr;
  b = __builtin_amdgcn_readfirstlane(b);
  pos = __builtin_amdgcn_readfirstlane(pos);
  const uint64_t at = static_cast<uint64_t>(b) * s.max_pages + (min(pos, end - 1) >> s.shift);
  return *(scalar_ptr)(reinterpret_cast<uintptr_t>(s.table + at));
}
__device__ __forceinline__ int32_t paged_checked(const PagedSeqs& s, int32_t id) {
  return static_cast<uint32_t>(id) < s.num_pages ? id : -1;   // (num_pages is below 2^31)
}

// f16 probabilities times scales need not fit f16's five exponent bits.  So the scores of a row
// are taken relative to its maximum plus the exponent of the largest scale that it has seen (at
// least kLeastExp, so that f32 holds the rest): products are then at most 2^8 as without scales,
// and numerator and denominator share the factor.
// (Weights end at 2^-126 of f32: from exponents of kMostExp on they would lose what is 2^-36 of
// the largest and less, and a tile that sees such a scale is summed again by SlowRow.)
constexpr float kLeastExp = -100.0f, kMostExp = 90.0f;
__device__ __forceinline__ float scale_exp(float most) {
  const float e = most < INFINITY ? static_cast<float>(__builtin_amdgcn_frexp_expf(most)) : 128.0f;
  return most > 0.0f ? e : kLeastExp;
}

// Whether a NaN or an infinity is among the 16 bytes.
template <int CT>
__device__ __forceinline__ bool any_nonfinite(u32x4 v) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (CT == kE4M3) {
      bad |= (((v[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
    } else if constexpr (CT != kI8) {
      constexpr uint32_t E = CT == kBF16 ? 0x7f80u : 0x7c00u;
      bad |= ((v[i] & E) == E) | ((v[i] & (E << 16)) == (E << 16));
    }
  }
  return bad;
}

// ---- the rows' kernel: tiles of 16 or 32 rows, the positions split over the chip -----------
//
// For steps of one or a few tokens, which are bound by the cache's bytes.  The unit of work is
// UNIT positions of one (sequence, tile, kv head); the units of the whole batch, in that order,
// are dealt to the workgroups in equal contiguous runs, whatever the lengths.  A run that holds
// all units of a tile writes O; else the run's sums go to the workspace and rows_merge adds up
// the tile's parts.  A run has at most two such parts: one that ends its tile's or lies inside it
// (slot 2 w) and one that begins its tile (slot 2 w + 1).
//
// Within a workgroup each wave has 32 of the unit's positions to itself, with running maximum
// and sum of its own, so nothing waits for a barrier until the run's end.  Per 32 positions and
// 16 rows:
//   S^T (32 x 16) = K . Q^T     16x16x32 MFMA; K fragments come straight from global memory
//   O^T (D x 16) += V^T . P^T   P^T is S^T's accumulator layout, its 16 positions' tiles
//                               interleaved as the k index; V goes through the wave's own LDS,
//                               whose transposing read gives V^T in the same order
// The next 32 positions are loaded as soon as K is multiplied and V is in LDS.  The maximum is
// only moved where a score passes it by 8 (2^8 of headroom in the 16-bit weights).
//
// Bound by the cache's bytes where there are many: 64 sequences of up to 8192 positions, 32 heads
// over 8 of 128, bf16: 1.24 GB in 192 us, 6.5 TB/s (large reads reach 7.1), and 7.5 us for the
// merge.  Three of up to 32001 in e4m3: 26 us for 130 MB, bound by latency, a run having 4 or 5
// units.  Equal runs over two workgroups per CU: with four 199 and 36 us (more parts to merge and
// starts to wait for), with one 194 and 30.
namespace rows {
constexpr int NT = 256;
constexpr int UNIT = 128;    // positions of a unit: 32 for each wave
constexpr int rec(int hd, int tr) { return tr * (hd + 2); }   // floats of a part: O, then m, l
}  // namespace rows

struct AttnArgs {
  PagedPool pool;
  PagedSeqs seqs;
  const uint16_t* q;
  uint16_t* o;
  float* ws;
  uint64_t q_stride;
  float scale_log2;
  uint32_t nh, group;
  uint32_t tile_rows;    // of the rows' kernel: 16 or 32
  uint32_t split_rows;   // sequences of more rows are the chunk kernel's, the others the rows'
  uint32_t runs;         // workgroups of the rows' kernel
  uint32_t parts;        // parts that a chunk tile's positions are cut into, at most
  float* chunk_ws;       // the chunk kernel's sums: [parts][total_q * nh] records
};

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d) {
  const uint32_t lo = __shfl_up(static_cast<uint32_t>(v), d);
  const uint32_t hi = __shfl_up(static_cast<uint32_t>(v >> 32), d);
  return static_cast<uint64_t>(hi) << 32 | lo;
}
__device__ __forceinline__ uint32_t read_lane(uint32_t v, int l) {
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), l));
}
__device__ __forceinline__ uint64_t read_lane64(uint64_t v, int l) {
  return static_cast<uint64_t>(read_lane(static_cast<uint32_t>(v >> 32), l)) << 32 |
         read_lane(static_cast<uint32_t>(v), l);
}

// The rows' units of 64 sequences, one per lane.  A sequence has tiles x heads x (blocks of its
// positions, one at least, so that rows without any position are written too) units.  (All of a
// batch's stay far below 2^63: 2^31 rows, 2^25 blocks.)
struct SeqGroup {
  PagedChunk c;
  uint32_t tiles, blocks;
  uint64_t units, upto;   // of this lane's sequence, and of all up to it
};
__device__ __forceinline__ SeqGroup seq_group(const AttnArgs& a, uint32_t b0, uint64_t before) {
  const uint32_t lane = threadIdx.x & 63u;
  SeqGroup g{};
  if (b0 + lane < a.seqs.batch) {
    g.c = paged_chunk(a.seqs, b0 + lane);
    const uint32_t r = g.c.n * a.group;   // the host keeps total_q * num_heads below 2^31
    g.tiles = r <= a.split_rows ? (r + a.tile_rows - 1) / a.tile_rows : 0u;
    g.blocks = max(1u, g.c.held / rows::UNIT + (g.c.held % rows::UNIT != 0));
    g.units = static_cast<uint64_t>(g.tiles) * g.blocks * a.pool.nkv;
  }
  g.upto = g.units;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t x = shfl_up64(g.upto, d);
    if (lane >= static_cast<uint32_t>(d)) g.upto += x;
  }
  g.upto += before;
  return g;
}

// A place among the units: the sequence that holds unit u.  Every wave finds it on its own.
struct Place {
  SeqGroup g;      // of the 64 sequences from b0 on
  uint32_t b0;
  int l;           // the sequence's lane
  uint64_t units;  // of the whole batch

  __device__ __forceinline__ explicit Place(const AttnArgs& a) : g(seq_group(a, 0, 0)), b0(0), l(0) {
    units = read_lane64(g.upto, 63);
    if (a.seqs.batch > 64) {
      SeqGroup x = g;
      for (uint32_t i = 64; i < a.seqs.batch; i += 64) {
        x = seq_group(a, i, units);
        units = read_lane64(x.upto, 63);
      }
    }
  }
  // From the present group on; false if no sequence holds u (lengths that change under the call).
  __device__ __forceinline__ bool find(const AttnArgs& a, uint64_t u) {
    while (true) {
      const uint64_t in = __builtin_amdgcn_ballot_w64(g.upto - g.units <= u && u < g.upto);
      if (in != 0) {   // exactly one lane
        l = __builtin_ctzll(in);
        return true;
      }
      b0 += 64;
      if (b0 >= a.seqs.batch) return false;
      g = seq_group(a, b0, read_lane64(g.upto, 63));
    }
  }
  __device__ __forceinline__ PagedChunk chunk() const {
    PagedChunk c;
    c.first = read_lane(g.c.first, l);
    c.n = read_lane(g.c.n, l);
    c.base = static_cast<int32_t>(read_lane(static_cast<uint32_t>(g.c.base), l));
    c.held = read_lane(g.c.held, l);
    return c;
  }
};
// First unit of run w of n.
__device__ __forceinline__ uint64_t run_start(uint64_t units, uint32_t w, uint32_t n) {
  return units / n * w + min(static_cast<uint64_t>(w), units % n);
}

// Eight values of O from their weighted sum and the weights' sum.
template <int DT>
__device__ __forceinline__ void write_row(const AttnArgs& a, const PagedChunk& c, uint32_t h,
                                          uint32_t row, int c8, const float (&o)[8], float l) {
  const uint64_t tok = c.first + row / a.group;
  const uint32_t hq = h * a.group + row % a.group;
  float f[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = l == 0.0f ? 0.0f : o[j] / l;
  *reinterpret_cast<u32x4*>(a.o + (tok * a.nh + hq) * a.pool.head_dim + c8) =
      u32x4{pack2h<DT>(f[0], f[1]), pack2h<DT>(f[2], f[3]), pack2h<DT>(f[4], f[5]),
            pack2h<DT>(f[6], f[7])};
}

// One row by one wave on the vector ALUs, over its visible positions in [p0, p1): for tiles where
// V holds NaN or infinities that some rows do not see (in a matrix product 0 * NaN is NaN).  64
// positions at a time, one per lane; then the lanes hold columns lane, lane + 64, ...
template <int DT, int CT, int HD>
struct SlowRow {
  static constexpr int N = (HD + 63) / 64;
  float m, l, o[N];

  static __device__ float value(const void* p, uint64_t i) {
    if constexpr (CT == kE4M3) {
      return __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<const uint8_t*>(p)[i], false)[0];
    } else if constexpr (CT == kI8) {
      return static_cast<float>(static_cast<const int8_t*>(p)[i]);
    } else {
      return u16_to_f32<CT>(static_cast<const uint16_t*>(p)[i]);
    }
  }
  __device__ SlowRow(const AttnArgs& a, const PagedChunk& c, uint32_t b, uint32_t h, uint32_t row,
                     uint32_t p0, uint32_t p1)
      : m(-INFINITY), l(0.0f) {
    const uint32_t lane = threadIdx.x & 63u, D = a.pool.head_dim;
    const uint32_t end = min(p1, paged_visible(c, row / a.group));
    const uint16_t* const q = a.q + (c.first + row / a.group) * a.q_stride +
                              static_cast<uint64_t>(h * a.group + row % a.group) * D;
    for (int i = 0; i < N; ++i) o[i] = 0.0f;
    for (uint32_t base = p0; base < end; base += 64) {
      const uint32_t pos = base + lane;
      const int32_t page = pos < end ? paged_page(a.seqs, b, pos) : -1;
      const uint64_t at =
          page < 0 ? 0 : pool_row(a.pool, a.seqs, page, h, paged_row(a.seqs, pos));
      float s = -INFINITY, vs = 1.0f;
      if (page >= 0) {
        float dot = 0.0f;
        for (uint32_t d = 0; d < D; ++d)
          dot = __builtin_fmaf(u16_to_f32<DT>(q[d]), value(a.pool.k, at + d), dot);
        s = dot * a.scale_log2;
        if constexpr (cache_codes<CT>()) {
          const uint64_t sc = pool_scale(a.pool, a.seqs, page, h, paged_row(a.seqs, pos));
          s *= a.pool.k_scale[sc];
          vs = a.pool.v_scale[sc];
        }
      }
      const float mn = fmaxf(m, wave_max(s));
      if (__builtin_amdgcn_ballot_w64(page >= 0) == 0) continue;
      const float mu = mn == -INFINITY ? 0.0f : mn;
      const float alpha = m == -INFINITY ? 0.0f : exp2_fast(m - mu);
      const float p = page < 0 ? 0.0f : exp2_fast(s - mu);
      l = l * alpha + wave_sum(p);
      m = mn;
      for (int i = 0; i < N; ++i) o[i] *= alpha;
      for (int x = 0; x < 64; ++x) {
        const int32_t px = __builtin_amdgcn_readlane(page, x);
        if (px < 0) continue;
        const float w = __shfl(p * vs, x);
        const uint64_t ax = read_lane64(at, x);
        for (int i = 0; i < N; ++i) {
          const uint32_t d = lane + 64 * i;
          if (d < D) o[i] = __builtin_fmaf(w, value(a.pool.v, ax + d), o[i]);
        }
      }
    }
  }
  __device__ void keep(float* p) const {
    for (int i = 0; i < N; ++i) p[(threadIdx.x & 63u) + 64 * i] = o[i];
  }
  __device__ void write(uint16_t* p, uint32_t D) const {
    for (int i = 0; i < N; ++i) {
      const uint32_t d = (threadIdx.x & 63u) + 64 * i;
      if (d < D)
        p[d] = static_cast<uint16_t>(pack2h<DT>(l == 0.0f ? 0.0f : o[i] / l, 0.0f));
    }
  }
};

template <int DT, int CT, int HD, int MT>
struct RowsTile {
  static constexpr bool kCodes = cache_codes<CT>();
  // Weights times codes' scales, and the codes of V, which f16 holds exactly, go into the product
  // as f16 whatever Q is: 8 times less rounding than bf16, at 0 to 4% of the time.
  static constexpr int PT = kCodes ? static_cast<int>(kF16) : DT;
  // Tiles of 16 rows, whose time goes to the cache's bytes, take a weight in two parts of 16 bits,
  // with a product each, unless it has more bits than O as it is: O's own rounding is then all
  // that shows.
  static constexpr bool kTwo = MT == 1 && PT == DT;
  static constexpr int ESZ = cache_size<CT>();
  static constexpr int TR = 16 * MT;
  static constexpr int NS = HD / 32;             // K fragments (32 values deep) of a position
  static constexpr int NC = HD / 16;             // 16-wide column tiles of O
  static constexpr int KL = 2 * HD * ESZ / 64;   // 16-byte K loads per lane: 2 tiles x HD/4 values
  static constexpr int VL = 32 * HD * ESZ / 1024;   // 16-byte V loads per lane
  static constexpr int VROW = HD * ESZ / 16;     // lanes per V row
  static_assert(VL >= 2, "a V load lies in one half of the 32 rows");
  static constexpr int ORS = HD + 4;             // row stride of the merge arena (floats)
  static constexpr int VB = 32 * HD * 2;         // V in LDS, bytes per wave
  static constexpr int OB = TR * ORS * 4;        // O at the end, bytes per wave
  static constexpr int WB = VB > OB ? VB : OB;

  // 32 positions on their way.
  struct Stage {
    u32x4 k[KL], v[VL];
    f32x4 ks[2], vs[2];
    int32_t page[2];   // of positions 0-15 and 16-31, or -1
  };
  struct Sums {
    f32x4 acc[MT][NC];
    // m + ev: what the row's scores are taken relative to (all its lanes); l: this lane's positions
    float m[MT], l[MT], ev[MT];
  };

  // 16-byte chunk c of V row r (32 rows of HD 16-bit values) in LDS: the four rows of a
  // transposing read fall in distinct banks.
  static __device__ __forceinline__ uint32_t vaddr(uint32_t r, uint32_t c) {
    const uint32_t x = HD >= 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1);
    return r * (HD * 2) + ((c ^ x) << 4);
  }

  // Pages hold whole groups of 16 positions.
  static __device__ __forceinline__ void pages(const AttnArgs& a, uint32_t b, uint32_t base,
                                               uint32_t held, int32_t (&page)[2]) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
      page[t] = base + 16 * t < held ? wave_page(a.seqs, b, base + 16 * t) : -1;
  }

  // Rows of missing pages and from `end` on are loaded as zeros.
  static __device__ __forceinline__ void load(const AttnArgs& a, uint32_t h, uint32_t base,
                                              uint32_t end, const int32_t (&page)[2], Stage& st) {
    const PagedPool& p = a.pool;
    const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    const uint32_t rb = p.head_dim * ESZ;   // bytes of a row
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint32_t pos = base + 16 * t;
      const uint32_t n = page[t] >= 0 && pos < end ? min(16u, end - pos) : 0u;
      const int32_t id = max(page[t], 0);
      const uint32_t row = paged_row(a.seqs, pos);
      st.page[t] = page[t];
      const uint64_t at = pool_row(p, a.seqs, id, h, row) * ESZ;
      const char* const kp = static_cast<const char*>(p.k) + at;
      const char* const vp = static_cast<const char*>(p.v) + at;
#pragma unroll
      for (int i = 0; i < KL / 2; ++i) {
        const uint32_t c = 64 * i + 16 * g;
        st.k[t * (KL / 2) + i] = load_within<true>(kp, n * rb, c < rb ? l16 * rb + c : kPast);
      }
#pragma unroll
      for (int i = 0; i < VL / 2; ++i) {
        const uint32_t r = i * (32 / VL) + lane / VROW, c = 16u * (lane % VROW);
        st.v[t * (VL / 2) + i] = load_within<true>(vp, n * rb, c < rb ? r * rb + c : kPast);
      }
      if constexpr (kCodes) {
        const uint64_t sc = pool_scale(p, a.seqs, id, h, row);
        st.ks[t] = __builtin_bit_cast(f32x4, load_within<false>(p.k_scale + sc, n * 4, 16 * g));
        st.vs[t] = __builtin_bit_cast(f32x4, load_within<false>(p.v_scale + sc, n * 4, 16 * g));
      }
    }
  }

  // K fragment s of tile t, 8 values per lane.  16 bits: columns 32 s + 8 g; codes: a lane's 16
  // bytes are columns 64 (s / 2) + 16 g .. + 15, fragment s its half s % 2 (Q is read alike).
  static __device__ __forceinline__ uint32_t qcol(int s, int g) {
    return kCodes ? 64u * (s / 2) + 16u * g + 8u * (s % 2) : 32u * s + 8u * g;
  }
  static __device__ __forceinline__ u32x4 kfrag(const Stage& st, int t, int s) {
    if constexpr (kCodes) {
      const u32x4 w = st.k[t * (KL / 2) + s / 2];
      const u32x2 lo = widen4<DT, CT>(w[2 * (s % 2)]), hi = widen4<DT, CT>(w[2 * (s % 2) + 1]);
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    } else {
      return st.k[t * (KL / 2) + s];
    }
  }

  // V of the stage into LDS.
  static __device__ __forceinline__ void put_v(const Stage& st, char* lds) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      const uint32_t r = i * (32 / VL) + lane / VROW, c = lane % VROW;
      const u32x4 w = st.v[i];
      if constexpr (kCodes) {
        const u32x2 a = widen4<PT, CT>(w[0]), b = widen4<PT, CT>(w[1]);
        *reinterpret_cast<u32x4*>(lds + vaddr(r, 2 * c)) = u32x4{a[0], a[1], b[0], b[1]};
        const u32x2 d = widen4<PT, CT>(w[2]), e = widen4<PT, CT>(w[3]);
        *reinterpret_cast<u32x4*>(lds + vaddr(r, 2 * c + 1)) = u32x4{d[0], d[1], e[0], e[1]};
      } else {
        *reinterpret_cast<u32x4*>(lds + vaddr(r, c)) = w;
      }
    }
  }

  static __device__ __forceinline__ void lds_order() {
    // one wave's LDS operations run in order: only the compiler has to keep them so
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }

  // acc += V^T . P^T, V from LDS.
  static __device__ __forceinline__ void pv(const char* lds, const u32x4 (&pf)[MT],
                                            const u32x4& rest, Sums& y) {
    const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    const uint32_t r = 4 * g + (l16 >> 2);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      // column 16 c + 4 (l16 % 4): 8 bytes at chunk 2 c + (l16 % 4) / 2
      const uint32_t ch = 2 * c + ((l16 & 3) >> 1), in = 8 * (l16 & 1);
      const u32x2 lo = lds::read_tr16(lds + vaddr(r, ch) + in);
      const u32x2 hi = lds::read_tr16(lds + vaddr(16 + r, ch) + in);
#pragma unroll
      for (int i = 0; i < MT; ++i)
        y.acc[i][c] = mfma16x16x32<PT>(u32x4{lo[0], lo[1], hi[0], hi[1]}, pf[i], y.acc[i][c]);
      if constexpr (kTwo)
        y.acc[0][c] = mfma16x16x32<PT>(u32x4{lo[0], lo[1], hi[0], hi[1]}, rest, y.acc[0][c]);
    }
  }

  // Blocks [k0, k1) of tile `tile` of (b, h): the wave's share, then the workgroup's sum.
  // part: where the sums go, or null: O.
  static __device__ __forceinline__ void run(const AttnArgs& a, const PagedChunk& c, uint32_t b,
                                             uint32_t h, uint32_t tile, uint32_t k0, uint32_t k1,
                                             float* part, char* arena, u32x4* q_lds) {
    const int t = threadIdx.x, lane = t & 63, l16 = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const uint32_t D = a.pool.head_dim, G = a.group;
    const uint32_t nrows = c.n * G;
    // the tile's first and last rows bound what its rows see
    const uint32_t r0 = tile * TR, r1 = min(nrows, r0 + TR) - 1;
    const uint32_t vis_min = __builtin_amdgcn_readfirstlane(paged_visible(c, r0 / G));
    const uint32_t vis_max = __builtin_amdgcn_readfirstlane(paged_visible(c, r1 / G));
    uint32_t base = k0 * rows::UNIT + wave * 32;
    const uint32_t end = min(static_cast<uint64_t>(k1) * rows::UNIT, static_cast<uint64_t>(vis_max));
    Stage st;
    int32_t next[2];
    if (base < end) {
      pages(a, b, base, c.held, next);
      load(a, h, base, end, next, st);
      pages(a, b, base + rows::UNIT, c.held, next);
    }

    Sums y;
    u32x4 qf[MT == 1 ? NS : 1];
    uint32_t vis[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const uint32_t row = r0 + 16 * i + l16;
      const bool live = row < nrows;
      const uint32_t qi = live ? row / G : 0u, hq = h * G + (live ? row % G : 0u);
      vis[i] = live ? paged_visible(c, qi) : 0u;
      const uint16_t* const qp =
          a.q + (c.first + qi) * a.q_stride + static_cast<uint64_t>(hq) * D;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        if (MT > 1 && (i * NS + s) % 4 != static_cast<int>(wave)) continue;
        u32x4 x = {0, 0, 0, 0};
        if (live && qcol(s, g) < D) x = ldg128(qp + qcol(s, g));
        if constexpr (MT == 1) qf[s] = x;
        else q_lds[(i * NS + s) * 64 + lane] = x;
      }
#pragma unroll
      for (int x = 0; x < NC; ++x) y.acc[i][x] = f32x4{0, 0, 0, 0};
      y.m[i] = -INFINITY;
      y.l[i] = 0.0f;
      y.ev[i] = kCodes ? kLeastExp : 0.0f;
    }
    char* const vlds = arena + wave * WB;
    bool odd = false;   // NaN or infinities in V near the rows' ends
    if constexpr (MT > 1) __syncthreads();   // (Q of a pair of tiles leaves no registers for V)

    for (; base < end; base += rows::UNIT) {
      // scores: lane (row l16, g) has positions base + 16 t + 4 g + i
      f32x4 s[MT][2];
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
        for (int i = 0; i < MT; ++i) s[i][tt] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int f = 0; f < NS; ++f) {
          const u32x4 kf = kfrag(st, tt, f);
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            const u32x4 x = MT == 1 ? qf[MT == 1 ? f : 0] : q_lds[(i * NS + f) * 64 + lane];
            s[i][tt] = mfma16x16x32<DT>(kf, x, s[i][tt]);
          }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            s[i][tt][x] *= kCodes ? st.ks[tt][x] * a.scale_log2 : a.scale_log2;
      }
      const bool there[2] = {st.page[0] >= 0, st.page[1] >= 0};
      const bool hides = base + 32 > vis_min || !there[0] || !there[1];   // uniform
      if (hides) {
#pragma unroll
        for (int i = 0; i < VL; ++i) odd |= any_nonfinite<CT>(st.v[i]);
      }
      float vs[8];
      if constexpr (kCodes) {
#pragma unroll
        for (int i = 0; i < 8; ++i) vs[i] = st.vs[i >> 2][i & 3];
      }
      lds_order();
      put_v(st, vlds);
      lds_order();
      if (base + rows::UNIT < end) {
        load(a, h, base + rows::UNIT, end, next, st);
        pages(a, b, base + 2 * rows::UNIT, c.held, next);
      }

      u32x4 pf[MT], rest;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        // of positions base + 16 (x / 4) + 4 g + x % 4, the row sees those below lim[x / 4]
        int lim[2];
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
          lim[tt] = there[tt] ? static_cast<int>(vis[i] - base) - 16 * tt - 4 * g : 0;
        if (hides) {
#pragma unroll
          for (int x = 0; x < 8; ++x)
            s[i][x >> 2][x & 3] = (x & 3) < lim[x >> 2] ? s[i][x >> 2][x & 3] : -INFINITY;
        }
        float mx = s[i][0][0];
#pragma unroll
        for (int x = 1; x < 8; ++x) mx = fmaxf(mx, s[i][x >> 2][x & 3]);
        float w[8];
        float big = kLeastExp;
        if constexpr (kCodes) {
#pragma unroll
          for (int x = 0; x < 8; ++x) w[x] = vs[x];
          if (hides) {   // (a hidden token's scale may be NaN)
#pragma unroll
            for (int x = 0; x < 8; ++x) w[x] = (x & 3) < lim[x >> 2] ? vs[x] : 0.0f;
          }
          float most = w[0];
#pragma unroll
          for (int x = 1; x < 8; ++x) most = fmaxf(most, w[x]);
          big = scale_exp(most);
        }
        float alpha = 1.0f;
        bool moved = false;
        if (__builtin_amdgcn_ballot_w64(mx > y.m[i] + 8.0f || (kCodes && big > y.ev[i])) != 0) {
          mx = fmaxf(mx, __shfl_xor(mx, 16));
          mx = fmaxf(mx, __shfl_xor(mx, 32));
          const float old = y.m[i] + y.ev[i];
          y.m[i] = fmaxf(y.m[i], mx);
          if constexpr (kCodes) {
            big = fmaxf(big, __shfl_xor(big, 16));
            y.ev[i] = fmaxf(y.ev[i], fmaxf(big, __shfl_xor(big, 32)));
          }
          alpha = y.m[i] == -INFINITY ? 1.0f : exp2_fast(old - (y.m[i] + y.ev[i]));
          y.l[i] *= alpha;
          moved = true;
        }
        const float mu = y.m[i] == -INFINITY ? 0.0f : y.m[i] + y.ev[i];
        float p[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          p[x] = exp2_fast(s[i][x >> 2][x & 3] - mu);
          if constexpr (kCodes || kTwo) y.l[i] += p[x];
          if constexpr (kCodes) p[x] *= w[x];
        }
        if (moved) {
#pragma unroll
          for (int x = 0; x < NC; ++x)
#pragma unroll
            for (int j = 0; j < 4; ++j) y.acc[i][x][j] *= alpha;
        }
        pf[i] = u32x4{pack2h<PT>(p[0], p[1]), pack2h<PT>(p[2], p[3]), pack2h<PT>(p[4], p[5]),
                      pack2h<PT>(p[6], p[7])};
        if constexpr (kTwo) {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            rest[x] = pack2h_rest<PT>(p[2 * x], p[2 * x + 1], pf[i][x]);
        } else if constexpr (!kCodes) {
#pragma unroll
          for (int x = 0; x < 4; ++x) y.l[i] = add_pair<DT>(pf[i][x], y.l[i]);
        }
      }
      pv(vlds, pf, rest, y);
    }

    // the four waves' sums
    __shared__ float sm[4][TR], sl[4][TR];
    __shared__ uint32_t odds[4];
    lds_order();
    bool any_odd = __builtin_amdgcn_ballot_w64(odd) != 0 && vis_min < vis_max;
#pragma unroll
    for (int i = 0; i < MT; ++i)
      any_odd |= kCodes && __builtin_amdgcn_ballot_w64(y.ev[i] > kMostExp) != 0;
    if (lane == 0) odds[wave] = any_odd;
    float* wo = reinterpret_cast<float*>(vlds);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      float l = y.l[i];
      l += __shfl_xor(l, 16);
      l += __shfl_xor(l, 32);
#pragma unroll
      for (int x = 0; x < NC; ++x) {
        *reinterpret_cast<f32x4*>(wo + (16 * i + l16) * ORS + 16 * x + 4 * g) = y.acc[i][x];
      }
      if (g == 0) {
        sm[wave][16 * i + l16] = y.m[i] + y.ev[i];
        sl[wave][16 * i + l16] = l;
      }
    }
    __syncthreads();
    if ((odds[0] | odds[1] | odds[2] | odds[3]) != 0) {   // the whole workgroup
      for (uint32_t r = wave; r < TR && r0 + r < nrows; r += 4) {
        SlowRow<DT, CT, HD> x(a, c, b, h, r0 + r, k0 * rows::UNIT, k1 * rows::UNIT);
        if (part) {
          x.keep(part + r * HD);
          if (lane == 0) {
            part[TR * HD + r] = x.m;
            part[TR * HD + TR + r] = x.l;
          }
        } else {
          const uint64_t tok = c.first + (r0 + r) / G;
          x.write(a.o + (tok * a.nh + h * G + (r0 + r) % G) * D, D);
        }
      }
      __syncthreads();
      return;
    }
    constexpr int CPR = HD / 8;   // 8-value pieces of a row
    for (int x = t; x < TR * CPR; x += rows::NT) {
      const int r = x / CPR, c8 = 8 * (x % CPR);
      if (r0 + r >= nrows || c8 >= static_cast<int>(D)) continue;
      float M = sm[0][r], ls = 0.0f, o[8];
#pragma unroll
      for (int i = 1; i < 4; ++i) M = fmaxf(M, sm[i][r]);
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (sl[i][r] == 0.0f) continue;   // a wave that saw nothing
        const float w = sm[i][r] == -INFINITY ? 0.0f : exp2_fast(sm[i][r] - M);
        const float* src = reinterpret_cast<const float*>(arena + i * WB) + r * ORS + c8;
        ls = __builtin_fmaf(w, sl[i][r], ls);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = __builtin_fmaf(w, src[j], o[j]);
      }
      if (part) {
        *reinterpret_cast<f32x4*>(part + r * HD + c8) = f32x4{o[0], o[1], o[2], o[3]};
        *reinterpret_cast<f32x4*>(part + r * HD + c8 + 4) = f32x4{o[4], o[5], o[6], o[7]};
        if (c8 == 0) {
          part[TR * HD + r] = M;
          part[TR * HD + TR + r] = ls;
        }
      } else {
        write_row<DT>(a, c, h, r0 + r, c8, o, ls);
      }
    }
    __syncthreads();   // the arena and the statistics serve the run's next tile
  }
};

// Waves per SIMD that the registers of a tile's kernel are kept to.
template <int HD, int MT> constexpr int rows_waves() { return HD == 256 ? 1 : 2; }

template <int DT, int CT, int HD, int MT>
__global__ void __launch_bounds__(rows::NT, (rows_waves<HD, MT>()))
attn_paged_rows(AttnArgs a) {
  using T = RowsTile<DT, CT, HD, MT>;
  __shared__ __align__(16) char arena[4 * T::WB];
  __shared__ u32x4 q_lds[MT > 1 ? MT * T::NS * 64 : 1];
  Place at(a);
  const uint32_t w = blockIdx.x, nw = gridDim.x;
  const uint64_t u1 = run_start(at.units, w + 1, nw);
  uint64_t u = run_start(at.units, w, nw);
  while (u < u1) {
    if (!at.find(a, u)) return;
    const PagedChunk c = at.chunk();
    const uint32_t blocks = read_lane(at.g.blocks, at.l);
    const uint64_t upto = read_lane64(at.g.upto, at.l);
    const uint64_t before = upto - read_lane64(at.g.units, at.l);
    while (u < u1 && u < upto) {
      const uint64_t in = u - before;
      // (divisions leave what all lanes share in vector registers: back to scalar ones)
      const uint64_t item = in / blocks;
      const uint32_t k0 =
          __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(in - item * blocks));
      const uint32_t h = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(item % a.pool.nkv));
      const uint32_t tile =
          __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(item / a.pool.nkv));
      const uint32_t k1 = __builtin_amdgcn_readfirstlane(
          static_cast<uint32_t>(min(static_cast<uint64_t>(blocks), k0 + (u1 - u))));
      float* part = nullptr;
      if (k0 != 0 || k1 != blocks)
        part = a.ws + (2ull * w + (k0 == 0 ? 1 : 0)) * rows::rec(HD, T::TR);
      T::run(a, c, at.b0 + at.l, h, tile, k0, k1, part, arena, q_lds);
      u += k1 - k0;
    }
  }
}

constexpr int merge_nt = 512;

// Merge the parts of a tile that several runs share.  Workgroup w looks after the tile in which
// run w + 1 begins, if run w holds that tile's first unit: parts 2 w + 1, then 2 (w + 1), ...
// One wave per row, HD / 8 lanes per part of it.
template <int DT, int HD>
__device__ __forceinline__ void rows_merge(const AttnArgs& a, uint32_t w) {
  Place at(a);
  const uint32_t nw = a.runs, TR = a.tile_rows;
  const uint64_t u = run_start(at.units, w + 1, nw);
  if (u >= at.units || !at.find(a, u)) return;
  const PagedChunk c = at.chunk();
  const uint32_t blocks = read_lane(at.g.blocks, at.l);
  const uint64_t before = read_lane64(at.g.upto, at.l) - read_lane64(at.g.units, at.l);
  const uint64_t item = (u - before) / blocks;
  const uint64_t item0 = before + item * blocks, item1 = item0 + blocks;
  if (item0 == u || run_start(at.units, w, nw) > item0) return;
  // the last run with a unit of the tile
  const uint64_t each = at.units / nw, more = at.units % nw, lastu = item1 - 1;
  const uint32_t last = static_cast<uint32_t>(
      lastu < (each + 1) * more ? lastu / (each + 1) : more + (lastu - (each + 1) * more) / each);
  const uint32_t h = static_cast<uint32_t>(item % a.pool.nkv);
  const uint32_t r0 = static_cast<uint32_t>(item / a.pool.nkv) * TR, nrows = c.n * a.group;
  const uint32_t np = last - w + 1;
  const int size = rows::rec(HD, static_cast<int>(TR));
  auto rec = [&](uint32_t i) { return a.ws + (i == 0 ? 2ull * w + 1 : 2ull * (w + i)) * size; };
  const int lane = threadIdx.x & 63;
  constexpr int CPR = HD / 8, PG = 64 / CPR;   // parts that a wave reads at once
  const int c8 = 8 * (lane % CPR), pg = lane / CPR;
  for (uint32_t r = threadIdx.x >> 6; r < TR && r0 + r < nrows; r += merge_nt / 64) {
    float M = -INFINITY, o[8], ls = 0.0f;
    for (uint32_t i = lane; i < np; i += 64) M = fmaxf(M, rec(i)[TR * HD + r]);
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = 0.0f;
    M = wave_max(M);
#pragma unroll 4
    for (uint32_t i = pg; i < np; i += PG) {
      const float* p = rec(i);
      const float m = p[TR * HD + r], l = p[TR * HD + TR + r];
      const f32x4 x = *reinterpret_cast<const f32x4*>(p + r * HD + c8);
      const f32x4 y = *reinterpret_cast<const f32x4*>(p + r * HD + c8 + 4);
      const float wt = m == -INFINITY ? 0.0f : exp2_fast(m - M);
      if (l != 0.0f) {   // (else the part saw nothing)
        ls = __builtin_fmaf(wt, l, ls);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          o[j] = __builtin_fmaf(wt, x[j], o[j]);
          o[4 + j] = __builtin_fmaf(wt, y[j], o[4 + j]);
        }
      }
    }
#pragma unroll
    for (int d = CPR; d < 64; d <<= 1) {
      ls += __shfl_xor(ls, d);
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] += __shfl_xor(o[j], d);
    }
    if (pg == 0 && c8 < static_cast<int>(a.pool.head_dim))
      write_row<DT>(a, c, h, r0 + r, c8, o, ls);
  }
}

// ---- the chunks' kernel: tiles of 256 rows ------------------------------------------------
//
// For many new tokens, which are bound by the matrix cores.  One workgroup of 8 waves per (tile,
// kv head, part of the positions), 32 rows a wave; 64 positions at a time go through LDS, double-
// buffered, as 16-bit values (codes are widened on the way in, once for all eight waves).  Per
// wave and block:
//   S^T (64 x 32) = K . Q^T     2 x HD/16 32x32x16 MFMAs, Q^T in registers
//   O^T (HD x 32) += V^T . P^T  4 x HD/32 MFMAs; P^T is S^T's accumulator converted in place,
//                               the transposing read of V gives V^T in the same order
// Where there are fewer (tile, head) items than CUs the positions are cut into parts, which
// chunk_merge adds up.
//
// Bound by the vector ALUs and the matrix cores one after the other, of which two waves of a SIMD
// overlap little: 512 tokens after 7680, 32 heads over 8 of 128, bf16: 66.6 GFLOP in 95 us (0.70
// PFLOP/s; 86 us with the softmax left out, the MFMAs are busy 30 us), 8 us for the merge of 34
// MB of parts.  Tried, each the same time or up to 20% more: four waves a turn behind the other
// four, so that one's products meet the other's softmax; blocks of 32 positions; three or eight
// fragment reads ahead instead of five; a raised wave priority around the products.
namespace chunk {
constexpr int NT = 512;
constexpr int TR = 256;
constexpr int KB = 64;            // positions of a block
constexpr uint32_t RING = 2;      // blocks in LDS
constexpr uint32_t kLeast = 512 / KB;   // blocks of a part, at least
__host__ __device__ constexpr int rec(int hd) { return hd + 4; }   // O, then l, m

// Tiles of a sequence, and the blocks of each part of one whose last row sees `vis` positions.
__device__ __forceinline__ uint32_t tiles(const AttnArgs& a, const PagedChunk& c) {
  const uint32_t r = c.n * a.group;
  return r > a.split_rows ? (r + TR - 1) / TR : 0u;
}
__device__ __forceinline__ uint32_t part_blocks(uint32_t vis, uint32_t parts) {
  const uint32_t nb = (vis + KB - 1) / KB;
  return max(kLeast, (nb + parts - 1) / parts);
}
// Positions that the tile's last row sees.
__device__ __forceinline__ uint32_t tile_reach(const AttnArgs& a, const PagedChunk& c,
                                               uint32_t tile) {
  const uint32_t r1 = min(c.n * a.group, (tile + 1) * TR) - 1;
  return paged_visible(c, r1 / a.group);
}
}  // namespace chunk

// max (sum) of a lane's value and that of the lane 32 away
__device__ __forceinline__ float pair_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <int DT, int CT, int HD>
struct ChunkTile {
  static_assert(HD == 64 || HD == 128, "chunk kernel head dim");
  static constexpr bool kCodes = cache_codes<CT>();
  static constexpr int ESZ = cache_size<CT>();
  static constexpr int PT = kCodes ? static_cast<int>(kF16) : DT;   // (RowsTile)
  static constexpr int RB = HD * 2;                  // bytes of a row in LDS
  static constexpr int KBYTES = chunk::KB * RB;      // of a block's K (or V)
  static constexpr int CPR = HD * ESZ / 16;          // 16-byte pieces of a row in memory
  static constexpr int NX = chunk::KB * CPR;         // of a block
  static constexpr int XPT = (NX + chunk::NT - 1) / chunk::NT;   // per thread
  static constexpr int NDS = HD / 16, NDT = HD / 32;

  struct Lds {
    char kv[chunk::RING][2 * KBYTES];
    float ks[chunk::RING][chunk::KB], vs[chunk::RING][chunk::KB];   // 0 where nothing is held
    float big[chunk::RING];          // scale_exp of the largest of vs
    uint32_t there[chunk::RING][chunk::KB / 16];   // the pages of its groups of 16 exist
    uint32_t odd;                    // NaN or infinities among V that some rows do not see
  };
  struct Stage {
    u32x4 k[XPT], v[XPT];
    float scale;
  };

  // LDS layouts without bank conflicts: K in halves of 64 columns, chunk c of row r at
  // c ^ f(r), where a read of 32 rows' chunks meets every bank evenly; V as for the rows' kernel.
  static __device__ __forceinline__ uint32_t kswz(uint32_t r) {
    return ((r >> 1) & 3u) | ((r >> 2) & 4u);
  }
  static __device__ __forceinline__ uint32_t kaddr(uint32_t r, uint32_t c) {
    return (c >> 3) * (chunk::KB * 128) + r * 128 + (((c & 7) ^ kswz(r)) << 4);
  }
  static __device__ __forceinline__ uint32_t vswz(uint32_t r) {
    return HD == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1);
  }
  static __device__ __forceinline__ uint32_t vaddr(uint32_t r, uint32_t c) {
    return r * RB + ((c ^ vswz(r)) << 4);
  }
};

template <int DT, int CT, int HD>
__global__ void __launch_bounds__(chunk::NT)
attn_paged_chunk(AttnArgs a) {
  using T = ChunkTile<DT, CT, HD>;
  using namespace chunk;
  constexpr int XPT = T::XPT;
  __shared__ __align__(16) typename T::Lds sh;
  const int t = threadIdx.x, lane = t & 63, l32 = lane & 31, g = lane >> 5;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const uint32_t nkv = a.pool.nkv, D = a.pool.head_dim, G = a.group;

  // Item: heads fastest (workgroup w runs on XCD w % 8, so a head's tiles share an L2 where there
  // are eight), then parts, then tiles.  Of up to 64 sequences, those that have a tile t, t from
  // the largest down: about the longest first, which leaves the shortest for the end.  (Five
  // prompts of up to 2000 tokens, 64-wide e4m3: 113 -> 103 us; the longest CU had 47 blocks' work
  // sequence by sequence, 36 so, of 30 on average.)  Of more, whose items fill the CUs many times,
  // sequence by sequence, each from its last tile on, in one pass over the lengths.
  const uint32_t h = __builtin_amdgcn_readfirstlane(blockIdx.x % nkv);
  const uint32_t part = __builtin_amdgcn_readfirstlane(blockIdx.x / nkv % a.parts);
  uint32_t left = blockIdx.x / nkv / a.parts, b = 0;
  if (a.seqs.batch <= 64) {
    const uint32_t n = static_cast<uint32_t>(lane) < a.seqs.batch
                           ? tiles(a, paged_chunk(a.seqs, lane)) : 0u;
    auto from = [&](uint32_t t) {   // tiles t and later of all sequences
      uint32_t sum = n > t ? n - t : 0u;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
      return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(sum));
    };
    if (left >= from(0)) return;
    uint32_t lo = 0, hi = 1;   // from(lo) > left >= from(hi)
    while (from(hi) > left) {
      lo = hi;
      hi *= 2;
    }
    while (hi - lo > 1) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (from(mid) > left) lo = mid;
      else hi = mid;
    }
    uint64_t in = __builtin_amdgcn_ballot_w64(n > lo);
    for (left -= from(hi); left > 0; --left) in &= in - 1;
    b = __builtin_ctzll(in);
    left = lo;
  } else {
    bool found = false;
    for (uint32_t b0 = 0; b0 < a.seqs.batch && !found; b0 += 64) {
      const uint32_t n =
          b0 + lane < a.seqs.batch ? tiles(a, paged_chunk(a.seqs, b0 + lane)) : 0u;
      uint32_t inc = n;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const uint32_t x = __shfl_up(inc, d);
        if (lane >= d) inc += x;
      }
      const uint64_t in = __builtin_amdgcn_ballot_w64(left < inc);
      if (in != 0) {
        const int l = __builtin_ctzll(in);
        b = b0 + l;
        left = __builtin_amdgcn_readlane(static_cast<int>(inc), l) - 1 - left;
        found = true;
      } else {
        left -= __builtin_amdgcn_readlane(static_cast<int>(inc), 63);
      }
    }
    if (!found) return;
  }
  const uint32_t tile = __builtin_amdgcn_readfirstlane(left);
  const PagedChunk c = paged_chunk(a.seqs, b);
  const uint32_t nrows = c.n * G;
  const uint32_t reach = __builtin_amdgcn_readfirstlane(tile_reach(a, c, tile));
  const uint32_t per = __builtin_amdgcn_readfirstlane(part_blocks(reach, a.parts));
  const uint32_t nb_all = (reach + KB - 1) / KB;
  const uint32_t j0 = part * per, j1 = min(nb_all, j0 + per);
  if (part != 0 && j0 >= nb_all) return;
  const bool whole = per >= nb_all;

  // the wave's rows, and what they see
  const uint32_t wr0 = tile * TR + wave * 32;
  const uint32_t row = wr0 + l32;
  const bool live_wave = wr0 < nrows, live_row = row < nrows;
  const uint32_t qi = live_row ? row / G : 0u, hq = h * G + (live_row ? row % G : 0u);
  const uint32_t vis = live_row ? paged_visible(c, qi) : 0u;
  const uint32_t vis_min =
      live_wave ? __builtin_amdgcn_readfirstlane(paged_visible(c, wr0 / G)) : 0u;
  const uint32_t vis_max =
      live_wave ? __builtin_amdgcn_readfirstlane(paged_visible(c, (min(nrows, wr0 + 32) - 1) / G))
                : 0u;
  const uint32_t tile_min =
      __builtin_amdgcn_readfirstlane(paged_visible(c, tile * TR / G));

  u32x4 qf[T::NDS];
#pragma unroll
  for (int s = 0; s < T::NDS; ++s) {
    qf[s] = u32x4{0, 0, 0, 0};
    if (live_row && 16u * s + 8u * g < D)
      qf[s] = ldg128(a.q + (c.first + qi) * a.q_stride + static_cast<uint64_t>(hq) * D + 16 * s +
                     8 * g);
  }
  f32x16 acc[T::NDT];
#pragma unroll
  for (int i = 0; i < T::NDT; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[i][j] = 0.0f;
  float m = -INFINITY, l = 0.0f, ev = T::kCodes ? kLeastExp : 0.0f;
  if (t == 0) sh.odd = 0;

  // this thread's pieces of a block: rows xr, 16-byte pieces xc.  A wave's rows, from wr on, lie
  // in one group of 16, so in one page.
  static_assert(64 / T::CPR <= 16, "a wave's rows lie in one page");
  uint32_t xr[XPT], xc[XPT], wr[XPT];
#pragma unroll
  for (int i = 0; i < XPT; ++i) {
    const uint32_t x = min(static_cast<uint32_t>(t + NT * i), static_cast<uint32_t>(T::NX - 1));
    xr[i] = x / T::CPR;
    xc[i] = x % T::CPR;
    wr[i] = __builtin_amdgcn_readfirstlane(xr[i]) & ~(64u / T::CPR - 1);
  }
  const uint32_t rb = D * T::ESZ;
  typename T::Stage st;
  int32_t id[XPT], id_s = -1;       // pages of the next block to be loaded (id: unchecked)
  bool ok[XPT];                     // the stage's pages exist
  auto pages = [&](uint32_t j) {
    const uint32_t base = j * KB;
#pragma unroll
    for (int i = 0; i < XPT; ++i)
      id[i] = wave_entry(a.seqs, b, base + wr[i], reach);
    if constexpr (T::kCodes)
      id_s = t < 2 * KB && base + (t & (KB - 1)) < reach
                 ? paged_page(a.seqs, b, base + (t & (KB - 1)))
                 : -1;
  };
  // Rows of missing pages and from `reach` on come as zeros, scales too.
  auto load = [&](uint32_t j) {
    const uint32_t base = j * KB;
#pragma unroll
    for (int i = 0; i < XPT; ++i) {
      const uint32_t pos = base + wr[i];
      const int32_t page = paged_checked(a.seqs, id[i]);
      const uint32_t n = page >= 0 && pos < reach ? min(64u / T::CPR, reach - pos) : 0u;
      const uint64_t at = pool_row(a.pool, a.seqs, max(page, 0), h, paged_row(a.seqs, pos)) * T::ESZ;
      const uint32_t off = 16 * xc[i] < rb ? (xr[i] - wr[i]) * rb + 16 * xc[i] : kPast;
      st.k[i] = load_within<false>(static_cast<const char*>(a.pool.k) + at, n * rb, off);
      st.v[i] = load_within<false>(static_cast<const char*>(a.pool.v) + at, n * rb, off);
      ok[i] = page >= 0 || pos >= reach;   // (past reach nothing is seen anyway)
    }
    if constexpr (T::kCodes) {
      st.scale = 0.0f;
      if (id_s >= 0)
        st.scale = (t < KB ? a.pool.k_scale : a.pool.v_scale)[pool_scale(
            a.pool, a.seqs, id_s, h, paged_row(a.seqs, base + (t & (KB - 1))))];
    }
  };
  auto slot = [&](uint32_t j) { return j % RING; };
  auto store = [&](uint32_t j) {   // what load(j) brought
    char* const kl = sh.kv[slot(j)];
    char* const vl = kl + T::KBYTES;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < XPT; ++i) {
      if (T::NX < NT && t >= T::NX) break;
      const u32x4 k = st.k[i], v = st.v[i];
      const uint32_t r = xr[i], cc = xc[i];
      odd |= any_nonfinite<CT>(v);
      if constexpr (T::kCodes) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const u32x2 k0 = widen4<DT, CT>(k[2 * x]), k1 = widen4<DT, CT>(k[2 * x + 1]);
          *reinterpret_cast<u32x4*>(kl + T::kaddr(r, 2 * cc + x)) = u32x4{k0[0], k0[1], k1[0], k1[1]};
          const u32x2 v0 = widen4<T::PT, CT>(v[2 * x]), v1 = widen4<T::PT, CT>(v[2 * x + 1]);
          *reinterpret_cast<u32x4*>(vl + T::vaddr(r, 2 * cc + x)) = u32x4{v0[0], v0[1], v1[0], v1[1]};
        }
      } else {
        *reinterpret_cast<u32x4*>(kl + T::kaddr(r, cc)) = k;
        *reinterpret_cast<u32x4*>(vl + T::vaddr(r, cc)) = v;
      }
      if (cc == 0 && (r & 15) == 0) sh.there[slot(j)][r >> 4] = ok[i];
    }
    if constexpr (T::kCodes) {
      if (t < 2 * KB) (t < KB ? sh.ks : sh.vs)[slot(j)][t & (KB - 1)] = st.scale;
      if (wave == 1) {   // (its lanes hold all of vs)
        static_assert(KB == 64, "vs in one wave");
        const float most = wave_max(st.scale);
        if (lane == 0) sh.big[slot(j)] = scale_exp(most);
      }
    }
    if (odd && (j + 1) * KB > tile_min) sh.odd = 1;   // (from any thread: one value)
  };

  const uint32_t vlane = T::vaddr(4 * (lane >> 5) + ((lane & 15) >> 2),
                                  (16 * ((lane >> 4) & 1) + 4 * (lane & 3)) >> 3) +
                         2 * (4 * (lane & 3) & 7);
  const uint32_t klane = 128u * l32;
  constexpr int NKT = KB / 32, NSP = KB / 16;
  f32x16 s[NKT];        // a block's scores
  u32x4 pf[NSP];        // its probabilities, 16 positions a step
  // Products of block j: its scores (Q), or its probabilities with its V.  Fragments are read
  // AHEAD products early, and the order is kept as written: left to itself the compiler reads so
  // far ahead that registers spill.
  auto products = [&](uint32_t j, auto q_) {
    constexpr bool Q = decltype(q_)::value;
    constexpr int N = Q ? NKT * T::NDS : NSP * T::NDT, AHEAD = 5;
    const char* const kl = sh.kv[slot(j)];
    const char* const vl = kl + T::KBYTES;
    u32x4 frag[AHEAD + 1];
    auto read = [&](int i) {
      u32x4& f = frag[i % (AHEAD + 1)];
      if constexpr (Q) {
        const int ds = i / NKT, kt = i % NKT;
        f = *reinterpret_cast<const u32x4*>(kl + (ds >> 2) * (KB * 128) + kt * 4096 + klane +
                                            16 * ((2 * (ds & 3) + g) ^ T::kswz(l32)));
      } else {
        // columns 32 dt on: chunk bits 2 and up, which the swizzle's bit 2 meets by XOR
        const int sp = i / T::NDT, dt = i % T::NDT;
        const uint32_t va = vlane ^ (dt << 6);
        const u32x2 lo = lds::read_tr16(vl + va + 16 * T::RB * sp);
        const u32x2 hi = lds::read_tr16(vl + va + 16 * T::RB * sp + 8 * T::RB);
        f = u32x4{lo[0], lo[1], hi[0], hi[1]};
      }
    };
    if constexpr (Q) {
#pragma unroll
      for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kt][i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < AHEAD && i < N; ++i) read(i);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i + AHEAD < N) read(i + AHEAD);
      __builtin_amdgcn_sched_barrier(0);
      const u32x4 f = frag[i % (AHEAD + 1)];
      if constexpr (Q) s[i % NKT] = mfma32x32x16<DT>(f, qf[i / NKT], s[i % NKT]);
      else acc[i % T::NDT] = mfma32x32x16<T::PT>(f, pf[i / T::NDT], acc[i % T::NDT]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto softmax = [&](uint32_t j) {
    const uint32_t base = j * KB, at_ring = slot(j);
    // lane (row l32, g): accumulator r of s[kt] is position base + 32 kt + 8 (r / 4) + 4 g + r % 4
    if constexpr (T::kCodes) {
#pragma unroll
      for (int q = 0; q < 4 * NKT; ++q) {
        const f32x4 ks = *reinterpret_cast<const f32x4*>(&sh.ks[at_ring][8 * q + 4 * g]);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[q >> 2][4 * (q & 3) + i] *= ks[i];
      }
    }
    uint32_t there = 0;
#pragma unroll
    for (int i = 0; i < NSP; ++i) there |= sh.there[at_ring][i] << i;
    there = __builtin_amdgcn_readfirstlane(there);
    const bool hides = base + KB > vis_min || there != (1u << NSP) - 1;
    const int lim = static_cast<int>(vis) - static_cast<int>(base) - 4 * g;
    if (hides) {
#pragma unroll
      for (int i = 0; i < 16 * NKT; ++i) {
        const int at = 32 * (i >> 4) + 8 * ((i & 15) >> 2) + (i & 3);
        const int lim_g = there >> (at >> 4) & 1 ? lim : -64;   // (uniform)
        s[i >> 4][i & 15] = at < lim_g ? s[i >> 4][i & 15] : -INFINITY;
      }
    }
    float mx[NSP];
#pragma unroll
    for (int q = 0; q < NSP; ++q) {
      mx[q] = s[q >> 1][8 * (q & 1)];
#pragma unroll
      for (int i = 1; i < 8; ++i) mx[q] = fmaxf(mx[q], s[q >> 1][8 * (q & 1) + i]);
    }
#pragma unroll
    for (int q = 1; q < NSP; ++q) mx[0] = fmaxf(mx[0], mx[q]);
    const float top = pair_max(mx[0]) * a.scale_log2;
    float big = kLeastExp;
    if constexpr (T::kCodes) {
      if (hides) {
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < 16 * NKT; ++i) {
          const int at = 32 * (i >> 4) + 8 * ((i & 15) >> 2) + (i & 3);
          most = fmaxf(most, at < lim ? sh.vs[at_ring][at + 4 * g] : 0.0f);
        }
        big = scale_exp(pair_max(most));
      } else {
        big = sh.big[at_ring];
      }
    }
    if (__builtin_amdgcn_ballot_w64(top > m + 8.0f || (T::kCodes && big > ev)) != 0) {
      const float old = m + ev;
      m = fmaxf(m, top);
      ev = T::kCodes ? fmaxf(ev, big) : 0.0f;
      const float alpha = m == -INFINITY ? 1.0f : exp2_fast(old - (m + ev));
      l *= alpha;
#pragma unroll
      for (int i = 0; i < T::NDT; ++i)
#pragma unroll
        for (int x = 0; x < 16; ++x) acc[i][x] *= alpha;
    }
    const float mu = m == -INFINITY ? 0.0f : m + ev;
    float l0 = 0.0f, l1 = 0.0f;
#pragma unroll
    for (int sp = 0; sp < NSP; ++sp) {   // the product with V takes 16 positions a step
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = exp2_fast(__builtin_fmaf(s[sp >> 1][8 * (sp & 1) + i], a.scale_log2, -mu));
        if constexpr (T::kCodes) (i & 1 ? l1 : l0) += p[i];
      }
      if constexpr (T::kCodes) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int at = 16 * sp + 8 * q;
          const f32x4 vs = *reinterpret_cast<const f32x4*>(&sh.vs[at_ring][at + 4 * g]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            p[4 * q + i] *= vs[i];
            if (hides) p[4 * q + i] = at + i < lim ? p[4 * q + i] : 0.0f;   // (vs may be NaN)
          }
        }
      }
      pf[sp] = u32x4{pack2h<T::PT>(p[0], p[1]), pack2h<T::PT>(p[2], p[3]),
                     pack2h<T::PT>(p[4], p[5]), pack2h<T::PT>(p[6], p[7])};
      if constexpr (!T::kCodes) {
#pragma unroll
        for (int i = 0; i < 4; ++i) (i & 1 ? l1 : l0) = add_pair<DT>(pf[sp][i], i & 1 ? l1 : l0);
      }
    }
    l += l0 + l1;
  };
  // Block j, loaded a block ago, into LDS, and the next one on its way.  (Past the last block
  // these are zeros, and nothing is read.)
  auto bring = [&](uint32_t j) {
    store(j);
    load(j + 1);
    pages(j + 2);
  };
  auto turn = [&] {   // this wave's LDS writes are done, then everyone's
    lds::wait_lgkm0();
    lds::bar();
  };

  if (j0 < j1) {
    // Every wave takes part in bringing every block; those from jw on have nothing that its rows
    // see.  (The accumulators change in one straight line of code: with branches around the
    // products the compiler copies them back and forth.)
    const uint32_t jw = max(j0, min(j1, (vis_max + KB - 1) / KB));
    pages(j0);
    load(j0);
    pages(j0 + 1);
    turn();   // (sh.odd)
    bring(j0);
    turn();
    for (uint32_t j = j0; j < jw; ++j) {
      bring(j + 1);   // its place in the ring was last read before the last turn
      products(j, std::true_type{});
      softmax(j);
      products(j, std::false_type{});
      turn();
    }
    for (uint32_t j = jw; j < j1; ++j) {
      bring(j + 1);
      turn();
    }
  }
  if (!live_wave) return;
  auto record = [&](uint64_t at) {
    return a.chunk_ws + (static_cast<uint64_t>(part) * a.seqs.total_q * a.nh + at) * rec(HD);
  };
  if (j0 < j1 && (__builtin_amdgcn_readfirstlane(sh.odd) != 0 ||   // (set before the last turn)
                  (T::kCodes && __builtin_amdgcn_ballot_w64(ev > kMostExp) != 0))) {
    for (uint32_t r = wr0; r < min(nrows, wr0 + 32); ++r) {
      SlowRow<DT, CT, HD> y(a, c, b, h, r, j0 * KB, j1 * KB);
      const uint64_t at = (c.first + r / G) * static_cast<uint64_t>(a.nh) + h * G + r % G;
      if (whole) {
        y.write(a.o + at * D, D);
      } else {
        y.keep(record(at));
        if (lane == 0) {
          record(at)[HD] = y.l;
          record(at)[HD + 1] = y.m;
        }
      }
    }
    return;
  }
  l = pair_sum(l);
  if (!live_row) return;
  const uint64_t at = (c.first + qi) * static_cast<uint64_t>(a.nh) + hq;
  if (whole) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < T::NDT; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t d = 32 * i + 8 * q + 4 * g;
        float f[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) f[x] = l == 0.0f ? 0.0f : acc[i][4 * q + x] * inv;
        if (d < D)
          *reinterpret_cast<u32x2*>(a.o + at * D + d) =
              u32x2{pack2h<DT>(f[0], f[1]), pack2h<DT>(f[2], f[3])};
      }
  } else {
    float* const out = record(at);
#pragma unroll
    for (int i = 0; i < T::NDT; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(out + 32 * i + 8 * q + 4 * g) =
            f32x4{acc[i][4 * q], acc[i][4 * q + 1], acc[i][4 * q + 2], acc[i][4 * q + 3]};
    if (g == 0) {
      out[HD] = l;
      out[HD + 1] = m + ev;
    }
  }
}

// Merge a chunk tile's parts: rows of one token, HD / 4 lanes per row, four parts' loads at once.
template <int DT, int HD>
__device__ __forceinline__ void chunk_merge(const AttnArgs& a, uint32_t item) {
  using namespace chunk;
  constexpr uint32_t LPR = HD / 4, RPB = merge_nt / LPR;
  const uint32_t groups = (a.nh + RPB - 1) / RPB;
  const uint32_t lane = threadIdx.x & 63u, token = item / groups;
  const uint32_t hq = item % groups * RPB + threadIdx.x / LPR;
  uint32_t le = 0;
  for (uint32_t j0 = 0; j0 < a.seqs.batch; j0 += 64) {
    const uint32_t j = j0 + lane;
    le += __builtin_popcountll(__builtin_amdgcn_ballot_w64(
        j < a.seqs.batch && paged_clamp(a.seqs.q_start[j], a.seqs.total_q) <= token));
  }
  if (le == 0 || hq >= a.nh) return;
  const PagedChunk c = paged_chunk(a.seqs, le - 1);
  if (token < c.first || token - c.first >= c.n || c.n * a.group <= a.split_rows) return;
  const int d = 4 * (threadIdx.x % LPR);
  const uint32_t row = (token - c.first) * a.group + hq % a.group;
  const uint32_t reach = tile_reach(a, c, row / TR);
  const uint32_t per = part_blocks(reach, a.parts), nb = (reach + KB - 1) / KB;
  if (per >= nb) return;
  const uint32_t np = (nb + per - 1) / per;
  const uint64_t step = static_cast<uint64_t>(a.seqs.total_q) * a.nh * rec(HD);
  const float* r = a.chunk_ws + (static_cast<uint64_t>(token) * a.nh + hq) * rec(HD);
  float M = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (uint32_t p0 = 0; p0 < np; p0 += 4) {
    f32x4 x[4];
    float lp[4], mp[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const float* q = r + min(p0 + i, np - 1) * step;
      x[i] = *reinterpret_cast<const f32x4*>(q + d);
      lp[i] = p0 + i < np ? q[HD] : 0.0f;
      mp[i] = q[HD + 1];
    }
    float top = M;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = lp[i] == 0.0f ? top : fmaxf(top, mp[i]);
    const float keep = M == -INFINITY ? 0.0f : exp2_fast(M - top);
    M = top;
    l *= keep;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = M == -INFINITY ? o[j] : o[j] * keep;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (lp[i] == 0.0f) continue;   // a part that the row sees nothing of
      const float w = mp[i] == -INFINITY ? 0.0f : exp2_fast(mp[i] - M);
      l = __builtin_fmaf(w, lp[i], l);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = __builtin_fmaf(w, x[i][j], o[j]);
    }
  }
  if (d < static_cast<int>(a.pool.head_dim)) {
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = l == 0.0f ? 0.0f : o[i] / l;
    *reinterpret_cast<u32x2*>(a.o + (static_cast<uint64_t>(token) * a.nh + hq) * a.pool.head_dim +
                              d) = u32x2{pack2h<DT>(f[0], f[1]), pack2h<DT>(f[2], f[3])};
  }
}

// Both kernels' merges in one launch: `first` workgroups for the rows' runs, then those of the
// chunks' tokens.
template <int DT, int HD>
__global__ void __launch_bounds__(merge_nt)
attn_paged_merge(AttnArgs a, uint32_t first) {
  if (blockIdx.x < first) {
    rows_merge<DT, HD>(a, blockIdx.x);
  } else if constexpr (HD <= 128) {
    chunk_merge<DT, HD>(a, blockIdx.x - first);
  }
}

}  // namespace pgd
}  // namespace th
