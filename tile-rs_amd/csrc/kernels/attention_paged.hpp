// Causal GQA attention of ragged chunks of new tokens over a paged cache, 16-bit Q and O, the
// cache in the same type or in 8-bit codes with a scale per position and head.
//
// For one sequence and kv head the rows are the (new token i, query head g) pairs, r = i G + g,
// so that the G query heads of a kv head share each K/V read.  Row r sees visible(i) positions:
//     s_j = ks_j (q . k_j) log2(e) / sqrt(D)      ks_j, vs_j: the codes' scales (1 in 16 bits)
//     o   = sum_j 2^(s_j - m) vs_j v_j / sum_j 2^(s_j - m)
// The codes are exact in either 16-bit type, so the products run on them and the scales are
// applied in f32: ks to the score, vs to the probability, before it is rounded to 16 bits.
#pragma once

#include "common.hpp"
#include "kv_cache.hpp"

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

// ---- the rows' kernel: tiles of 16 rows, the positions split over the chip ---------------
//
// For steps of one or a few tokens, which are bound by the cache's bytes.  The unit of work is
// UNIT positions of one (sequence, tile, kv head); the units of the whole batch, in that order,
// are dealt to the workgroups in equal contiguous runs, whatever the lengths.  A run that holds
// all units of a tile writes O; else the run's sums go to the workspace and rows_merge adds up
// the tile's parts.  A run has at most two such parts: one that ends its tile's or lies inside it
// (slot 2 w) and one that begins its tile (slot 2 w + 1).
//
// Within a workgroup each wave has 32 of the unit's positions to itself, with running maximum
// and sum of its own, so nothing waits for a barrier until the run's end.  Per 32 positions:
//   S^T (32 x 16) = K . Q^T     16x16x32 MFMA; K fragments come straight from global memory
//   O^T (D x 16) += V^T . P^T   P^T is S^T's accumulator layout, its 16 positions' tiles
//                               interleaved as the k index; V goes through the wave's own LDS,
//                               whose transposing read gives V^T in the same order
// The next 32 positions' K and V are in flight meanwhile.  The maximum is only moved where a
// score passes it by 8 (2^8 of headroom in the 16-bit probabilities).
namespace rows {
constexpr int NT = 256;
constexpr int TR = 16;       // rows of a tile
constexpr int UNIT = 128;    // positions of a unit: 32 for each wave
constexpr int rec(int hd) { return TR * (hd + 2); }   // floats of a part: O, then m, then l
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
};

// Work of one sequence: tiles of `tr` rows, and units of `unit` positions (one at least, so that
// rows without any position are written too).
struct SeqWork {
  uint32_t tiles, units;
};
__device__ __forceinline__ SeqWork seq_work(const PagedChunk& c, uint32_t group, uint32_t tr,
                                            uint32_t unit) {
  SeqWork w;
  w.tiles = (c.n * group + tr - 1) / tr;
  const uint32_t u = c.held / unit + (c.held % unit != 0);
  w.units = u == 0 ? 1u : u;
  return w;
}

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d) {
  const uint32_t lo = __shfl_up(static_cast<uint32_t>(v), d);
  const uint32_t hi = __shfl_up(static_cast<uint32_t>(v >> 32), d);
  return static_cast<uint64_t>(hi) << 32 | lo;
}
__device__ __forceinline__ uint64_t read_lane64(uint64_t v, int l) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), l);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), l);
  return static_cast<uint64_t>(hi) << 32 | lo;
}

// Units of all sequences; and the sequence that holds unit u, with the units before it.  Each
// wave scans on its own, 64 sequences at a time.  (Units of a batch stay far below 2^63: under
// 2^31 rows of 2^25 units and 2^32 heads would not fit any memory.)
struct Where {
  uint32_t b;
  uint64_t before;
};
template <class F>
__device__ __forceinline__ uint64_t scan_units(const AttnArgs& a, F&& visit) {
  const uint32_t lane = threadIdx.x & 63u;
  uint64_t sum = 0;
  for (uint32_t b0 = 0; b0 < a.seqs.batch; b0 += 64) {
    uint64_t u = 0;
    if (b0 + lane < a.seqs.batch) {
      const SeqWork w = seq_work(paged_chunk(a.seqs, b0 + lane), a.group, rows::TR, rows::UNIT);
      u = static_cast<uint64_t>(w.tiles) * w.units * a.pool.nkv;
    }
    uint64_t inc = u;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint64_t x = shfl_up64(inc, d);
      if (lane >= static_cast<uint32_t>(d)) inc += x;
    }
    visit(b0, sum, u, inc);
    sum += read_lane64(inc, 63);
  }
  return sum;
}
__device__ __forceinline__ Where find_unit(const AttnArgs& a, uint64_t target) {
  Where w{a.seqs.batch, 0};
  scan_units(a, [&](uint32_t b0, uint64_t sum, uint64_t u, uint64_t inc) {
    const uint64_t in = __builtin_amdgcn_ballot_w64(sum + inc - u <= target && target < sum + inc);
    if (in != 0) {   // exactly one lane
      const int l = __builtin_ctzll(in);
      w.b = b0 + l;
      w.before = sum + read_lane64(inc, l) - read_lane64(u, l);
    }
  });
  return w;
}
// First unit of run w of n.
__device__ __forceinline__ uint64_t run_start(uint64_t units, uint32_t w, uint32_t n) {
  return units / n * w + min(static_cast<uint64_t>(w), units % n);
}

template <int DT, int CT, int HD>
struct RowsTile {
  static constexpr bool kCodes = cache_codes<CT>();
  static constexpr int ESZ = cache_size<CT>();
  static constexpr int NS = HD / 32;             // K fragments (32 values deep) of a position
  static constexpr int NC = HD / 16;             // 16-wide column tiles of O
  static constexpr int KL = 2 * HD * ESZ / 64;   // 16-byte K loads per lane: 2 tiles x HD/4 values
  static constexpr int VL = 32 * HD * ESZ / 1024;   // 16-byte V loads per lane
  static constexpr int VROW = HD * ESZ / 16;     // lanes per V row
  static_assert(VL >= 2, "a V load lies in one half of the 32 rows");
  static constexpr int ORS = HD + 4;             // row stride of the merge arena (floats)
  static constexpr int VB = 32 * HD * 2;         // V in LDS, bytes per wave
  static constexpr int OB = rows::TR * ORS * 4;  // O at the end, bytes per wave
  static constexpr int WB = VB > OB ? VB : OB;

  // What is in flight for 32 positions.
  struct Stage {
    u32x4 k[KL], v[VL];
    f32x4 ks[2], vs[2];
    bool there[2];   // the pages of positions 0-15 and 16-31 exist
  };

  // 16-byte chunk c of V row r (32 rows of HD 16-bit values) in LDS: the four rows of a
  // transposing read fall in distinct banks.
  static __device__ __forceinline__ uint32_t vaddr(uint32_t r, uint32_t c) {
    const uint32_t x = HD >= 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1);
    return r * (HD * 2) + ((c ^ x) << 4);
  }

  static __device__ __forceinline__ void load(const AttnArgs& a, uint32_t b, uint32_t h,
                                              uint32_t base, uint32_t held, Stage& st) {
    const PagedPool& p = a.pool;
    const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    uint64_t at[2], sc[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      // pages hold whole groups of 16 positions
      const uint32_t pos = base + 16 * t;
      const int32_t page = pos < held ? paged_page(a.seqs, b, pos) : -1;
      st.there[t] = page >= 0;
      const int32_t id = page >= 0 ? page : 0;   // num_pages >= 1; what is loaded is not used
      const uint32_t row = page >= 0 ? paged_row(a.seqs, pos) : 0u;
      at[t] = pool_row(p, a.seqs, id, h, row) * ESZ;
      sc[t] = pool_scale(p, a.seqs, id, h, row);
    }
    const uint32_t rb = p.head_dim * ESZ;   // bytes of a row
    const char* kp = static_cast<const char*>(p.k);
    const char* vp = static_cast<const char*>(p.v);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < KL / 2; ++i) {
        const uint32_t c = min(static_cast<uint32_t>(64 * i + 16 * g), rb - 16);
        st.k[t * (KL / 2) + i] = ldg128_nt(kp + at[t] + l16 * rb + c);
      }
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      const uint32_t r = i * (32 / VL) + lane / VROW;   // rows 0-15 in the first half of loads
      const uint32_t c = min(16u * (lane % VROW), rb - 16);
      st.v[i] = ldg128_nt(vp + at[2 * i / VL] + (r & 15) * rb + c);
    }
    if constexpr (kCodes) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        st.ks[t] = *reinterpret_cast<const f32x4*>(p.k_scale + sc[t] + 4 * g);
        st.vs[t] = *reinterpret_cast<const f32x4*>(p.v_scale + sc[t] + 4 * g);
      }
    }
  }

  // K fragment s of tile t, 8 values per lane.  16 bits: columns 32 s + 8 g; codes: a lane's 16
  // bytes are columns 64 (s / 2) + 16 g .. + 15, fragment s its half s % 2 (Q is read alike).
  static __device__ __forceinline__ u32x4 kfrag(const Stage& st, int t, int s) {
    if constexpr (kCodes) {
      const u32x4 w = st.k[t * (KL / 2) + s / 2];
      const u32x2 lo = widen4<DT, CT>(w[2 * (s % 2)]), hi = widen4<DT, CT>(w[2 * (s % 2) + 1]);
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    } else {
      return st.k[t * (KL / 2) + s];
    }
  }
  static __device__ __forceinline__ uint32_t qcol(int s, int g) {
    return kCodes ? 64u * (s / 2) + 16u * g + 8u * (s % 2) : 32u * s + 8u * g;
  }

  // V of the stage into LDS, rows from `live` on and rows of missing pages as zeros.
  static __device__ __forceinline__ void put_v(const Stage& st, char* lds, uint32_t live) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      const uint32_t r = i * (32 / VL) + lane / VROW, c = lane % VROW;
      u32x4 w = st.v[i];
      if (r >= live || !st.there[2 * i / VL]) w = u32x4{0, 0, 0, 0};
      if constexpr (kCodes) {
        const u32x2 a = widen4<DT, CT>(w[0]), b = widen4<DT, CT>(w[1]);
        const u32x2 d = widen4<DT, CT>(w[2]), e = widen4<DT, CT>(w[3]);
        *reinterpret_cast<u32x4*>(lds + vaddr(r, 2 * c)) = u32x4{a[0], a[1], b[0], b[1]};
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
  static __device__ __forceinline__ void pv(const char* lds, u32x4 pf, f32x4 (&acc)[NC]) {
    const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    const uint32_t r = 4 * g + (l16 >> 2);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      // column 16 c + 4 (l16 % 4): 8 bytes at chunk 2 c + (l16 % 4) / 2
      const uint32_t ch = 2 * c + ((l16 & 3) >> 1), in = 8 * (l16 & 1);
      const u32x2 lo = lds::read_tr16(lds + vaddr(r, ch) + in);
      const u32x2 hi = lds::read_tr16(lds + vaddr(16 + r, ch) + in);
      acc[c] = mfma16x16x32<DT>(u32x4{lo[0], lo[1], hi[0], hi[1]}, pf, acc[c]);
    }
  }

  // Units [k0, k1) of tile `tile` of (b, h): the wave's share, then the workgroup's sum.
  // part: where the sums go, or null: O.
  static __device__ __forceinline__ void run(const AttnArgs& a, const PagedChunk& c, uint32_t b,
                                             uint32_t h, uint32_t tile, uint32_t k0, uint32_t k1,
                                             float* part, char* arena) {
    const int t = threadIdx.x, lane = t & 63, l16 = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const uint32_t D = a.pool.head_dim, G = a.group;
    const uint32_t nrows = c.n * G;   // the host keeps total_q * num_heads below 2^31
    const uint32_t row = tile * rows::TR + l16;
    const bool live_row = row < nrows;
    const uint32_t qi = row / G, hq = h * G + row % G;
    const uint32_t vis = live_row ? paged_visible(c, qi) : 0u;
    // the tile's first and last rows bound what its rows see
    const uint32_t r0 = tile * rows::TR, r1 = min(nrows, r0 + rows::TR) - 1;
    const uint32_t vis_min = __builtin_amdgcn_readfirstlane(paged_visible(c, r0 / G));
    const uint32_t vis_max = __builtin_amdgcn_readfirstlane(paged_visible(c, r1 / G));

    u32x4 qf[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      qf[s] = u32x4{0, 0, 0, 0};
      if (live_row && qcol(s, g) < D)
        qf[s] = ldg128(a.q + (c.first + qi) * a.q_stride + static_cast<uint64_t>(hq) * D +
                       qcol(s, g));
    }
    f32x4 acc[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) acc[i] = f32x4{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;   // m: the row's (all its lanes); l: this lane's positions
    int ev = -1000;                  // f16 with codes: O is in units of 2^ev
    char* const vlds = arena + wave * WB;

    const uint32_t step = rows::UNIT;
    uint32_t base = k0 * rows::UNIT + wave * 32;
    const uint32_t end = min(static_cast<uint64_t>(k1) * rows::UNIT, static_cast<uint64_t>(vis_max));
    Stage cur, nxt;
    if (base < end) load(a, b, h, base, c.held, cur);
    for (; base < end; base += step) {
      if (base + step < end) load(a, b, h, base + step, c.held, nxt);
      // scores: lane (row l16, g) has positions base + 16 t + 4 g + i
      f32x4 s[2];
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        s[tt] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int f = 0; f < NS; ++f) s[tt] = mfma16x16x32<DT>(kfrag(cur, tt, f), qf[f], s[tt]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[tt][i] *= kCodes ? cur.ks[tt][i] * a.scale_log2 : a.scale_log2;
      }
      const bool hides = base + 32 > vis_min || !cur.there[0] || !cur.there[1];   // uniform
      bool hid[2][4];
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          hid[tt][i] = hides && (base + 16 * tt + 4 * g + i >= vis || !cur.there[tt]);
          if (hid[tt][i]) s[tt][i] = -INFINITY;
        }
      float mx = s[0][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[i >> 2][i & 3]);
      float alpha = 1.0f;
      bool moved = false;
      if (__builtin_amdgcn_ballot_w64(mx > m + 8.0f) != 0) {
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float mn = fmaxf(m, mx);
        alpha = mn == -INFINITY ? 1.0f : exp2_fast(m - mn);
        m = mn;
        l *= alpha;
        moved = true;
      }
      const float mu = m == -INFINITY ? 0.0f : m;
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = exp2_fast(s[i >> 2][i & 3] - mu);
        l += p[i];
      }
      if constexpr (kCodes) {
        float vs[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) vs[i] = hid[i >> 2][i & 3] ? 0.0f : cur.vs[i >> 2][i & 3];
        if constexpr (DT == kF16) {
          // f16 has five exponent bits: the scales enter relative to a power of two not far
          // below their largest so far
          float big = vs[0];
#pragma unroll
          for (int i = 1; i < 8; ++i) big = fmaxf(big, vs[i]);
          int e = big > 0.0f ? __builtin_amdgcn_frexp_expf(big) : -1000;
          if (__builtin_amdgcn_ballot_w64(e > ev) != 0) {
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) e = max(e, __shfl_xor(e, o));
            e = max(e, ev);
            alpha *= __builtin_ldexpf(1.0f, max(ev - e, -300));
            ev = e;
            moved = true;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) vs[i] = __builtin_ldexpf(vs[i], ev < -500 ? 0 : -ev);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] *= vs[i];
      }
      if (moved) {
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] *= alpha;
      }
      const u32x4 pf = {pack2h<DT>(p[0], p[1]), pack2h<DT>(p[2], p[3]), pack2h<DT>(p[4], p[5]),
                        pack2h<DT>(p[6], p[7])};
      bool odd = false;
      if (hides) {
#pragma unroll
        for (int i = 0; i < VL; ++i)
          odd |= base + i * (32 / VL) + lane / VROW < vis_max && any_nonfinite<CT>(cur.v[i]);
      }
      if (__builtin_amdgcn_ballot_w64(odd) != 0 && vis_min < vis_max) {
        // NaN or infinities among values that some rows do not see (0 * NaN is NaN): these 32
        // positions on the vector ALUs, each row over what it sees
        lds_order();
        put_v(cur, vlds, vis_max - base);
        lds_order();
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
#pragma unroll 1
          for (int gk = 0; gk < 4; ++gk) {
            const float pk = __shfl(p[0], l16 + 16 * gk);
            const uint32_t r = 16 * (i >> 2) + 4 * gk + (i & 3);
            if (base + r < vis) {
#pragma unroll
              for (int cc = 0; cc < NC; ++cc)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const uint32_t d = 16 * cc + 4 * g + j;
                  const uint16_t x = *reinterpret_cast<const uint16_t*>(
                      vlds + vaddr(r, d >> 3) + 2 * (d & 7));
                  acc[cc][j] = __builtin_fmaf(pk, u16_to_f32<DT>(x), acc[cc][j]);
                }
            }
          }
#pragma unroll
          for (int j = 0; j < 7; ++j) p[j] = p[j + 1];
        }
      } else {
        lds_order();
        put_v(cur, vlds, vis_max - base);
        lds_order();
        pv(vlds, pf, acc);
      }
      cur = nxt;
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if constexpr (kCodes && DT == kF16) {
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = ev < -500 ? 0.0f : __builtin_ldexpf(acc[i][j], ev);
    }

    // the four waves' sums
    __shared__ float sm[4][rows::TR], sl[4][rows::TR];
    lds_order();
    float* wo = reinterpret_cast<float*>(vlds);
#pragma unroll
    for (int i = 0; i < NC; ++i)
      *reinterpret_cast<f32x4*>(wo + l16 * ORS + 16 * i + 4 * g) = acc[i];
    if (g == 0) {
      sm[wave][l16] = m;
      sl[wave][l16] = l;
    }
    __syncthreads();
    constexpr int CPR = HD / 8;   // 8-value pieces of a row
    for (int x = t; x < rows::TR * CPR; x += rows::NT) {
      const int r = x / CPR, c8 = 8 * (x % CPR);
      if (r0 + r >= nrows || c8 >= static_cast<int>(D)) continue;
      float M = sm[0][r], w[4], ls = 0.0f, o[8];
#pragma unroll
      for (int i = 1; i < 4; ++i) M = fmaxf(M, sm[i][r]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = sm[i][r] == -INFINITY ? 0.0f : exp2_fast(sm[i][r] - M);
        ls = sl[i][r] != 0.0f ? __builtin_fmaf(w[i], sl[i][r], ls) : ls;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float* src = reinterpret_cast<const float*>(arena + i * WB) + r * ORS + c8;
        if (sl[i][r] == 0.0f) continue;   // a wave that saw nothing
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = __builtin_fmaf(w[i], src[j], o[j]);
      }
      if (part) {
        *reinterpret_cast<f32x4*>(part + r * HD + c8) = f32x4{o[0], o[1], o[2], o[3]};
        *reinterpret_cast<f32x4*>(part + r * HD + c8 + 4) = f32x4{o[4], o[5], o[6], o[7]};
        if (c8 == 0) {
          part[rows::TR * HD + r] = M;
          part[rows::TR * HD + rows::TR + r] = ls;
        }
      } else {
        write_row(a, c, h, r0 + r, c8, o, ls);
      }
    }
    __syncthreads();   // the arena and the statistics serve the run's next tile
  }

  static __device__ __forceinline__ void write_row(const AttnArgs& a, const PagedChunk& c,
                                                   uint32_t h, uint32_t row, int c8,
                                                   const float (&o)[8], float l) {
    const uint64_t tok = c.first + row / a.group;
    const uint32_t hq = h * a.group + row % a.group;
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = l == 0.0f ? 0.0f : o[j] / l;
    *reinterpret_cast<u32x4*>(a.o + (tok * a.nh + hq) * a.pool.head_dim + c8) =
        u32x4{pack2h<DT>(f[0], f[1]), pack2h<DT>(f[2], f[3]), pack2h<DT>(f[4], f[5]),
              pack2h<DT>(f[6], f[7])};
  }
};

template <int DT, int CT, int HD>
__global__ void __launch_bounds__(rows::NT, 2)
attn_paged_rows(AttnArgs a) {
  using T = RowsTile<DT, CT, HD>;
  __shared__ __align__(16) char arena[4 * T::WB];
  const uint64_t units = scan_units(a, [](uint32_t, uint64_t, uint64_t, uint64_t) {});
  const uint32_t w = blockIdx.x, nw = gridDim.x;
  const uint64_t u1 = run_start(units, w + 1, nw);
  uint64_t u = run_start(units, w, nw);
  if (u >= u1) return;
  Where at = find_unit(a, u);
  while (u < u1 && at.b < a.seqs.batch) {
    const PagedChunk c = paged_chunk(a.seqs, at.b);
    const SeqWork sw = seq_work(c, a.group, rows::TR, rows::UNIT);
    const uint64_t all = static_cast<uint64_t>(sw.tiles) * sw.units * a.pool.nkv;
    if (all == 0) {
      ++at.b;
      continue;
    }
    while (u < u1 && u < at.before + all) {
      const uint64_t in = u - at.before;
      const uint32_t k0 = static_cast<uint32_t>(in % sw.units);
      const uint64_t th_ = in / sw.units;
      const uint32_t h = static_cast<uint32_t>(th_ % a.pool.nkv);
      const uint32_t tile = static_cast<uint32_t>(th_ / a.pool.nkv);
      const uint32_t k1 =
          static_cast<uint32_t>(min(static_cast<uint64_t>(sw.units), k0 + (u1 - u)));
      float* part = nullptr;
      if (k0 != 0 || k1 != sw.units)
        part = a.ws + (2ull * w + (k0 == 0 ? 1 : 0)) * rows::rec(HD);
      T::run(a, c, at.b, h, tile, k0, k1, part, arena);
      u += k1 - k0;
    }
    at.before += all;
    ++at.b;
  }
}

// Merge the parts of tiles that several runs share.  Workgroup w looks after the tile in which
// run w + 1 begins, if run w holds that tile's first unit: parts 2 w + 1, then 2 (w + 1), ...
// One wave per row.
template <int DT, int CT, int HD>
__global__ void __launch_bounds__(256)
attn_paged_merge(AttnArgs a, uint32_t nw) {
  using T = RowsTile<DT, CT, HD>;
  const uint64_t units = scan_units(a, [](uint32_t, uint64_t, uint64_t, uint64_t) {});
  const uint32_t w = blockIdx.x;
  const uint64_t u = run_start(units, w + 1, nw);
  if (u >= units) return;
  const Where at = find_unit(a, u);
  if (at.b >= a.seqs.batch) return;
  const PagedChunk c = paged_chunk(a.seqs, at.b);
  const SeqWork sw = seq_work(c, a.group, rows::TR, rows::UNIT);
  const uint64_t in = u - at.before;
  const uint64_t item0 = u - in % sw.units, item1 = item0 + sw.units;
  if (item0 == u || run_start(units, w, nw) > item0) return;
  uint32_t last = w + 1;   // the last run with a unit of the tile
  while (last + 1 < nw && run_start(units, last + 1, nw) < item1) ++last;
  const uint64_t th_ = in / sw.units;
  const uint32_t h = static_cast<uint32_t>(th_ % a.pool.nkv);
  const uint32_t r0 = static_cast<uint32_t>(th_ / a.pool.nkv) * rows::TR, nrows = c.n * a.group;
  const uint32_t np = last - w + 1;
  auto rec = [&](uint32_t i) {
    return a.ws + (i == 0 ? 2ull * w + 1 : 2ull * (w + i)) * rows::rec(HD);
  };
  const int lane = threadIdx.x & 63;
  constexpr int CPR = HD / 8, PG = 64 / CPR;   // parts that a wave reads at once
  const int c8 = 8 * (lane % CPR), pg = lane / CPR;
  for (int r = threadIdx.x >> 6; r < rows::TR && r0 + r < nrows; r += 4) {
    float M = -INFINITY;
    for (uint32_t i = lane; i < np; i += 64) M = fmaxf(M, rec(i)[rows::TR * HD + r]);
    M = wave_max(M);
    float o[8], ls = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = 0.0f;
    for (uint32_t i = pg; i < np; i += PG) {
      const float* p = rec(i);
      const float m = p[rows::TR * HD + r], l = p[rows::TR * HD + rows::TR + r];
      if (l == 0.0f) continue;
      const float wt = m == -INFINITY ? 0.0f : exp2_fast(m - M);
      ls = __builtin_fmaf(wt, l, ls);
      const f32x4 x = *reinterpret_cast<const f32x4*>(p + r * HD + c8);
      const f32x4 y = *reinterpret_cast<const f32x4*>(p + r * HD + c8 + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        o[j] = __builtin_fmaf(wt, x[j], o[j]);
        o[4 + j] = __builtin_fmaf(wt, y[j], o[4 + j]);
      }
    }
#pragma unroll
    for (int d = CPR; d < 64; d <<= 1) {
      ls += __shfl_xor(ls, d);
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] += __shfl_xor(o[j], d);
    }
    if (pg == 0 && c8 < static_cast<int>(a.pool.head_dim))
      T::write_row(a, c, h, r0 + r, c8, o, ls);
  }
}

}  // namespace pgd
}  // namespace th
