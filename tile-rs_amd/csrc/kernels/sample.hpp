// Sampling of one token per row of logits: temperature, top-k, top-p, min-p, from a given
// random number.
//
//   w_i = exp((x_i - x_max) / T) in f32, held as a whole number of 2^-40, so that masses are
//   exact in 64 bits (up to 2^23 logits of weight 1) and no order of summation shows.
//
// The kept set is a prefix of the order (x falling, then index rising), so each limit is a cut:
// a (key, index) pair, the last one kept, with `key` the order-preserving whole number of x.  A
// cut is found from a histogram of counts and masses over bins of x, linear from x_max down to
// where weights vanish; then its bin's members, gathered into LDS, are ranked against each
// other.  A bin of more members than fit there is divided again, by the (key, index) pair as one
// 64-bit number, until they do.  No sort, and equal logits need no case of their own.
//
// The token is then the first index whose mass with the lower ones' exceeds u times the kept
// mass: the row is divided among the waves, and the share that holds the place is divided again.
//
// Bound by the vector ALUs and, with limits, the histogram's LDS atomics (42% of the LDS-active
// cycles are conflicts): 256 rows of 50257 f32 with all limits 46 us, 18 without (51 MB: 9 us at
// the rate of a copy); one launch's latency for few short rows (8 x 8000 bf16 8 us).
//
// One workgroup of 16 waves per row.  Rows of up to 16 vectors of 16 bytes per thread stay in
// registers between the passes, longer ones are read again (from the caches).
#pragma once

#include "common.hpp"

namespace th {
namespace smp {
constexpr int NT = 1024, NW = NT / 64;
constexpr int BINS = 2048;
constexpr int CAP = 2048;       // members that are ranked in LDS
constexpr float kLowest = 42.0f;   // 2^-42 rounds to no step of 2^-40
constexpr uint64_t kOne = 1ull << 40;

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int o) {
  return static_cast<uint64_t>(__shfl_xor(static_cast<uint32_t>(v >> 32), o)) << 32 |
         __shfl_xor(static_cast<uint32_t>(v), o);
}

struct Pair {   // a place in the order: larger key first, then lower index
  uint32_t key, idx;
};
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);   // (-0 is 0)
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

// A row of logits.  NaN counts as -infinity: no comparison below takes it for anything else.
template <int DT>
struct Row {
  static constexpr uint32_t E = Vec16<DT>::kElems;
  const void* p;
  uint32_t vocab;
};

// The row by aligned 16-byte blocks: block k holds elements k E - off + (0 .. E-1), those outside
// the row as -infinity.  Wave w has the blocks [w per, (w + 1) per).  NV: blocks of a thread that
// stay in registers; 0: every pass reads them.
template <int DT, int NV>
struct Blocks {
  static constexpr uint32_t E = Row<DT>::E;
  Row<DT> row;
  const char* base;          // of block 0
  uint32_t off, count, per;
  const u32x4* edge;
  u32x4 held[NV > 0 ? NV : 1];

  // edges: LDS for the row's first and last block, which may not be whole.
  __device__ __forceinline__ void init(const Row<DT>& r, u32x4* edges) {
    row = r;
    edge = edges;
    const uintptr_t at = reinterpret_cast<uintptr_t>(r.p);
    off = static_cast<uint32_t>(at & 15u) / (16 / E);
    base = reinterpret_cast<const char*>(at & ~uintptr_t{15});
    count = (off + r.vocab + E - 1) / E;
    per = NV > 0 ? 64u * NV : ((count + NW * 64 - 1) / (NW * 64)) * 64u;
    if (threadIdx.x < 2 * E) {
      const uint32_t k = threadIdx.x < E ? 0 : count - 1;
      const int32_t i = static_cast<int32_t>(k * E - off + threadIdx.x % E);
      const bool in = i >= 0 && i < static_cast<int32_t>(r.vocab);
      if constexpr (DT == kF32)
        reinterpret_cast<float*>(edges)[threadIdx.x] =
            in ? static_cast<const float*>(r.p)[i] : -INFINITY;
      else
        reinterpret_cast<uint16_t*>(edges)[threadIdx.x] =
            in ? static_cast<const uint16_t*>(r.p)[i] : static_cast<uint16_t>(kNone);
    }
    __syncthreads();
    if constexpr (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) held[j] = load(first() + 64 * j);
    }
  }
  __device__ __forceinline__ uint32_t index(uint32_t k) const { return k * E - off; }
  static __device__ __forceinline__ void unpack(u32x4 v, float (&x)[E]) { unpack16<DT>(v, x); }
  __device__ __forceinline__ uint32_t first() const {
    return (threadIdx.x >> 6) * per + (threadIdx.x & 63u);
  }
  static constexpr uint32_t kNone =   // -infinities
      DT == kF32 ? 0xff800000u : DT == kBF16 ? 0xff80ff80u : 0xfc00fc00u;
  __device__ __forceinline__ u32x4 load(uint32_t k) const {
    u32x4 v = {kNone, kNone, kNone, kNone};
    if (k > 0 && k + 1 < count) v = ldg128(base + 16ull * k);
    else if (k < count) v = edge[k == 0 ? 0 : 1];
    return v;
  }
  // f(index, logit) of every element of this thread (and -infinities outside the row).
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
    auto block = [&](u32x4 v, uint32_t k) {
      float x[E];
      unpack16<DT>(v, x);
#pragma unroll
      for (int e = 0; e < static_cast<int>(E); ++e) f(index(k) + e, x[e]);
    };
    if constexpr (NV > 0) {
      // What a pass makes of the row is not kept for the next one (there are no registers for
      // that): each works on copies that the compiler cannot tell from other values.
      uint32_t k = first();
      asm volatile("" : "+v"(k));
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        u32x4 v = held[j];
        asm volatile("" : "+v"(v));
        block(v, k + 64 * j);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      const uint32_t end = min(count, ((threadIdx.x >> 6) + 1) * per);
      for (uint32_t k = first(); k < end; k += 64 * 4) {
        u32x4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = load(k + 64 * j < end ? k + 64 * j : count);
#pragma unroll
        for (int j = 0; j < 4; ++j) block(v[j], k + 64 * j);
      }
    }
  }
};

struct Weigher {
  float top, c_hi, c_lo;   // log2(e) / T as the sum of two floats
  static __device__ __forceinline__ Weigher make(float top, float temp) {
    const double c = min(1.4426950408889634 / static_cast<double>(temp), 3.0e38);
    const float hi = static_cast<float>(c);
    return Weigher{top, hi, static_cast<float>(c - static_cast<double>(hi))};
  }
  __device__ __forceinline__ float weight(float x) const {
    const float d = x - top;
    const float y = d * c_hi;
    const float y_lo = __builtin_fmaf(d, c_lo, __builtin_fmaf(d, c_hi, -y));
    const float e = exp2_fast(y);
    const float w = __builtin_fmaf(e * y_lo, 0.69314718f, e);
    // (x = top = infinity; differences of -infinity and NaN)
    return x == top ? 1.0f : y > -kLowest ? w : 0.0f;
  }
  // In steps of 2^-40: the fraction bits of 2^12 + w, to nearest even.
  static __device__ __forceinline__ uint64_t steps(float w) {
    return __builtin_bit_cast(uint64_t, static_cast<double>(w) + 4096.0) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ uint64_t operator()(float x) const { return steps(weight(x)); }
};

__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v += shfl_xor64(v, o);
  return v;
}
__device__ __forceinline__ uint64_t wave_scan64(uint64_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t lo = __shfl_up(static_cast<uint32_t>(v), o);
    const uint32_t hi = __shfl_up(static_cast<uint32_t>(v >> 32), o);
    if (lane >= o) v += static_cast<uint64_t>(hi) << 32 | lo;
  }
  return v;
}

// What a limit asks of the order: a number of tokens, or a mass.
struct Goal {
  bool by_mass;
  uint64_t count;   // keep while fewer than this come before
  double mass;      // or while less mass than this comes before
  __device__ __forceinline__ bool wants(uint64_t n_before, uint64_t m_before) const {
    return by_mass ? static_cast<double>(m_before) < mass : n_before < count;
  }
};

struct Shared {
  uint32_t count[BINS];
  unsigned long long mass[BINS];
  uint64_t member[CAP];    // (key, ~index): larger comes first
  uint64_t weight[CAP];
  uint64_t wave_a[NW], wave_b[NW];
  float wave_f[NW];
  uint32_t members;
  uint32_t bin;
  uint64_t above_n, above_m, found, found_m;
  uint32_t in_bin, in_bin_first;
};

// The last bin that still holds a kept token: the first whose following bin the goal does not
// want.  Writes it to sh.bin with the count and mass of the bins before it (BINS if the goal
// takes everything).  `base_*`: what comes before the first bin.
__device__ __forceinline__ void find_bin(Shared& sh, const Goal& goal, uint64_t base_n,
                                         uint64_t base_m) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  if (t == 0) sh.bin = BINS;
  const uint32_t c0 = sh.count[2 * t], c1 = sh.count[2 * t + 1];
  const uint64_t m0 = sh.mass[2 * t], m1 = sh.mass[2 * t + 1];
  const uint64_t n = static_cast<uint64_t>(c0) + c1, m = m0 + m1;
  uint64_t ni = wave_scan64(n, lane), mi = wave_scan64(m, lane);
  if (lane == 63) {
    sh.wave_a[wave] = ni;
    sh.wave_b[wave] = mi;
  }
  __syncthreads();
  for (int i = 0; i < wave; ++i) {
    base_n += sh.wave_a[i];
    base_m += sh.wave_b[i];
  }
  uint64_t bn = base_n + ni - n, bm = base_m + mi - m;   // before bin 2 t
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint32_t c = j ? c1 : c0;
    const uint64_t w = j ? m1 : m0;
    if (c != 0 && goal.wants(bn, bm) && !goal.wants(bn + c, bm + w)) {
      sh.bin = 2 * t + j;
      sh.above_n = bn;
      sh.above_m = bm;
      sh.in_bin = c;
    }
    bn += c;
    bm += w;
  }
  __syncthreads();
}

template <int DT, int NV>
struct Sampler {
  const Blocks<DT, NV>& row;
  Weigher weigh;
  float bin_scale;
  Shared& sh;

  // BINS - 1: without weight (NaN and -infinity among them), which no pass counts
  __device__ __forceinline__ uint32_t bin_of(float x) const {
    const float d = (weigh.top - x) * bin_scale;   // (x = top = infinity: NaN)
    return x == weigh.top ? 0u : d < static_cast<float>(BINS - 1) ? static_cast<uint32_t>(d)
                                                                  : BINS - 1;
  }
  static __device__ __forceinline__ uint64_t place(float x, uint32_t i) {
    return static_cast<uint64_t>(order_key(x)) << 32 | (0xffffffffu - i);
  }
  __device__ __forceinline__ void clear() const {
    for (int i = threadIdx.x; i < BINS; i += NT) {
      sh.count[i] = 0;
      sh.mass[i] = 0;
    }
    __syncthreads();
  }

  // Counts and masses of all tokens with weight by bins of x.
  __device__ __forceinline__ void histogram() const {
    clear();
    row.each([&](uint32_t, float x) {
      const uint32_t b = bin_of(x);
      const uint64_t w = weigh(x);
      if (b < BINS - 1) {
        atomicAdd(&sh.count[b], 1u);
        atomicAdd(&sh.mass[b], static_cast<unsigned long long>(w));
      }
    });
    __syncthreads();
  }

  // The goal's cut; sum: the mass up to it.  The bins are those of histogram().
  __device__ __forceinline__ Pair select(const Goal& goal, uint64_t* sum) const {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    find_bin(sh, goal, 0, 0);
    // every token is wanted, or the cut is among those without weight
    if (sh.bin >= BINS) return Pair{0, 0xffffffffu};
    const uint32_t first_bin = sh.bin;
    uint64_t lo = 0, hi = ~0ull;   // the members' places
    auto members = [&](auto&& f) {
      row.each([&](uint32_t i, float x) {
        if (bin_of(x) != first_bin) return;
        const uint64_t v = place(x, i);
        if (v >= lo && v <= hi) f(v, x);
      });
    };
    if (t == 0) sh.in_bin_first = sh.in_bin;
    while (sh.in_bin > CAP) {
      // divide the members again, evenly between the least and the largest of them
      uint64_t a = ~0ull, b = 0;
      members([&](uint64_t v, float) {
        a = min(a, v);
        b = max(b, v);
      });
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        a = min(a, shfl_xor64(a, o));
        b = max(b, shfl_xor64(b, o));
      }
      if (lane == 0) {
        sh.wave_a[wave] = a;
        sh.wave_b[wave] = b;
      }
      const uint64_t base_n = sh.above_n, base_m = sh.above_m;
      __syncthreads();
      for (int i = 0; i < NW; ++i) {
        a = min(a, sh.wave_a[i]);
        b = max(b, sh.wave_b[i]);
      }
      lo = a;
      hi = b;
      int shift = 0;   // bin 0 has the largest
      while (((hi - lo) >> shift) >= BINS) ++shift;
      clear();
      members([&](uint64_t v, float x) {
        const uint32_t q = static_cast<uint32_t>((hi - v) >> shift);
        atomicAdd(&sh.count[q], 1u);
        atomicAdd(&sh.mass[q], static_cast<unsigned long long>(weigh(x)));
      });
      __syncthreads();
      find_bin(sh, goal, base_n, base_m);
      const uint64_t top = hi - (static_cast<uint64_t>(sh.bin) << shift);
      const uint64_t width = (1ull << shift) - 1;
      lo = top - lo > width ? top - width : lo;
      hi = top;
    }
    // the members, in any order; each is ranked by a walk over the others
    if (t == 0) sh.members = 0;
    __syncthreads();
    members([&](uint64_t v, float x) {
      const uint32_t at = atomicAdd(&sh.members, 1u);
      if (at < CAP) {
        sh.member[at] = v;
        sh.weight[at] = weigh(x);
      }
    });
    __syncthreads();
    const uint32_t n = min(sh.members, static_cast<uint32_t>(CAP));
    for (uint32_t i = t; i < n; i += NT) {
      const uint64_t v = sh.member[i];
      uint64_t bn = sh.above_n, bm = sh.above_m;
      for (uint32_t j = 0; j < n; ++j) {
        const bool before = sh.member[j] > v;
        bn += before;
        bm += before ? sh.weight[j] : 0ull;
      }
      if (goal.wants(bn, bm) && !goal.wants(bn + 1, bm + sh.weight[i])) {
        sh.found = v;
        sh.found_m = bm + sh.weight[i];
      }
    }
    __syncthreads();
    const Pair at{static_cast<uint32_t>(sh.found >> 32),
                  0xffffffffu - static_cast<uint32_t>(sh.found)};
    *sum = sh.found_m;
    return at;
  }
};

// A value that the f64 of a mass exceeds, for numbers of 1 and more: the last step of it, or past
// 2^53, where steps no longer show, a rounding.
__device__ __forceinline__ double short_of(uint64_t mass) {
  const double m = static_cast<double>(mass);
  return min(m - 1.0, m * (1.0 - 0x1p-52));
}

// The first element of blocks [k0, k1) at which the mass from `before` on exceeds `target`, which
// lies in them.  A long range is divided among the waves, and the share that holds the place
// divided again, down to a block per thread.  kept(index, logit): an element's mass.
template <class B, class F>
__device__ __forceinline__ void find_place(Shared& sh, const B& row, uint32_t k0, uint32_t k1,
                                           uint64_t before, double target, F&& kept,
                                           int32_t* token) {
  constexpr uint32_t E = B::E;
  const int t = threadIdx.x, lane = t & 63;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(t >> 6);
  float x[E];
  auto elements = [&](uint32_t k) { B::unpack(row.load(k), x); };
  while (k1 - k0 > NT) {
    const uint32_t share = (k1 - k0 + NW - 1) / NW;
    const uint32_t wa = min(k1, k0 + wave * share), wb = min(k1, wa + share);
    uint64_t m = 0;
#pragma unroll 2
    for (uint32_t k = wa + lane; k < wb; k += 64) {
      elements(k);
#pragma unroll
      for (int e = 0; e < static_cast<int>(E); ++e) m += kept(row.index(k) + e, x[e]);
    }
    m = wave_sum64(m);
    if (lane == 0) sh.wave_a[wave] = m;
    __syncthreads();
    uint32_t w = 0;
    while (w < NW - 1 && static_cast<double>(before + sh.wave_a[w]) <= target)
      before += sh.wave_a[w++];
    __syncthreads();
    k0 = min(k1, k0 + w * share);
    k1 = min(k1, k0 + share);
  }
  const uint32_t k = k0 + t;
  elements(k < k1 ? k : row.count);
  uint64_t m = 0;
#pragma unroll
  for (int e = 0; e < static_cast<int>(E); ++e) m += kept(row.index(k) + e, x[e]);
  const uint64_t upto = wave_scan64(m, lane);
  if (lane == 63) sh.wave_a[wave] = upto;
  __syncthreads();
  for (uint32_t w = 0; w < wave; ++w) before += sh.wave_a[w];
  before += upto - m;
  // one thread's block holds the place
  if (m != 0 && static_cast<double>(before) <= target &&
      static_cast<double>(before + m) > target) {
    uint32_t at = 0;
#pragma unroll
    for (int e = 0; e < static_cast<int>(E); ++e) {
      before += kept(row.index(k) + e, x[e]);
      at += static_cast<double>(before) <= target;
    }
    *token = static_cast<int32_t>(row.index(k) + at);
  }
}

// One workgroup per row.
template <int DT, int NV>
__global__ void __launch_bounds__(NT)
sample_rows(const void* __restrict__ logits, int32_t* __restrict__ tokens, uint32_t vocab,
            uint64_t stride, const float* __restrict__ uniform,
            const float* __restrict__ temperature, const int32_t* __restrict__ top_k,
            const float* __restrict__ top_p, const float* __restrict__ min_p) {
  __shared__ Shared sh;
  const uint32_t r = blockIdx.x;
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const float temp = temperature ? temperature[r] : 1.0f;
  const int32_t k = top_k ? top_k[r] : 0;
  const float p = top_p ? top_p[r] : 1.0f, mp = fmaxf(min_p ? min_p[r] : 0.0f, 0.0f);   // (no NaN)
  const float u = uniform[r];
  const Row<DT> row{static_cast<const char*>(logits) + r * stride * (DT == kF32 ? 4 : 2), vocab};
  Blocks<DT, NV> blocks;
  __shared__ u32x4 edges[2];
  blocks.init(row, edges);

  float top = -INFINITY;
  blocks.each([&](uint32_t, float x) { top = fmaxf(top, x); });
  top = wave_max(top);
  if (lane == 0) sh.wave_f[wave] = top;
  __syncthreads();
  for (int i = 0; i < NW; ++i) top = fmaxf(top, sh.wave_f[i]);
  if (top == -INFINITY) {
    if (t == 0) tokens[r] = -1;
    return;
  }
  // one token is kept (or asked for): the first of the largest
  if (!(temp > 0.0f) || k == 1 || p <= 0.0f || mp > 1.0f) {
    uint32_t at = 0xffffffffu;
    blocks.each([&](uint32_t i, float x) { at = x == top ? min(at, i) : at; });
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) at = min(at, __shfl_xor(at, o));
    if (lane == 0) sh.wave_a[wave] = at;
    __syncthreads();
    for (int i = 0; i < NW; ++i) at = min(at, static_cast<uint32_t>(sh.wave_a[i]));
    if (t == 0) tokens[r] = static_cast<int32_t>(at);
    return;
  }
  const Weigher weigh = Weigher::make(top, temp);
  const Sampler<DT, NV> s{blocks, weigh, weigh.c_hi * (static_cast<float>(BINS - 1) / kLowest), sh};

  Pair cut{0, 0xffffffffu};
  const bool cut_k = k > 0 && static_cast<uint32_t>(k) < vocab, cut_p = p < 1.0f;
  if (cut_k || cut_p) {
    s.histogram();
    uint64_t whole = 0;
    if (cut_p) {   // all the row's mass, unless top-k leaves less
      const uint64_t m = wave_sum64(sh.mass[2 * t] + sh.mass[2 * t + 1]);
      if (lane == 0) sh.wave_a[wave] = m;
      __syncthreads();
      for (int i = 0; i < NW; ++i) whole += sh.wave_a[i];
      __syncthreads();
    }
    bool fresh = true;   // the bins are the histogram's
    if (cut_k) {
      cut = s.select(Goal{false, static_cast<uint64_t>(k), 0.0}, &whole);
      fresh = sh.bin >= BINS || sh.in_bin_first <= CAP;
      __syncthreads();
    }
    if (cut_p) {
      if (!fresh) s.histogram();
      uint64_t sum;
      const Pair by_p =
          s.select(Goal{true, 0, static_cast<double>(p) * static_cast<double>(whole)}, &sum);
      // the stricter of the two
      if (by_p.key > cut.key || (by_p.key == cut.key && by_p.idx < cut.idx)) cut = by_p;
      __syncthreads();
    }
  }

  // kept mass by waves; then the place, in the share that holds it
  const bool all_kept = cut.key == 0 && mp == 0.0f;
  const float cut_x = cut.key == 0 ? -INFINITY : key_value(cut.key);
  auto kept = [&](uint32_t i, float x) -> uint64_t {
    const float w = weigh.weight(x);
    const bool in = (w >= mp) & ((x > cut_x) | ((x == cut_x) & (i <= cut.idx)));
    return Weigher::steps(in ? w : 0.0f);
  };
  uint64_t m = 0;
  if (all_kept)
    blocks.each([&](uint32_t, float x) { m += weigh(x); });
  else
    blocks.each([&](uint32_t i, float x) {
      // (a cut leaves few: most waves skip most weights)
      if (__builtin_amdgcn_ballot_w64(x >= cut_x) != 0) m += kept(i, x);
    });
  m = wave_sum64(m);
  if (lane == 0) sh.wave_a[wave] = m;
  __syncthreads();
  uint64_t all = 0, before = 0;
  for (int i = 0; i < NW; ++i) all += sh.wave_a[i];
  const double target =
      min(u > 0.0f ? static_cast<double>(u) * static_cast<double>(all) : 0.0, short_of(all));
  uint32_t w = 0;
  while (w < NW - 1 && static_cast<double>(before + sh.wave_a[w]) <= target)
    before += sh.wave_a[w++];
  __syncthreads();
  find_place(sh, blocks, min(blocks.count, w * blocks.per),
             min(blocks.count, (w + 1) * blocks.per), before, target, kept, tokens + r);
}

// ---- few long rows without limits: each over many workgroups -------------------------------
//
// A part is kPart blocks of a row; its weights are relative to its own largest logit, so that
// one pass gives part and mass, and sample_pick brings them together in f64.  8 rows of 128256
// bf16 take 22 us in one workgroup each (14 cycles of vector ALU per logit), the two launches 10.
constexpr uint32_t kPart = NT;
struct PartSum {
  float top;
  uint32_t pad;
  uint64_t mass;
};
template <int DT>
__global__ void __launch_bounds__(256)
sample_parts(const void* __restrict__ logits, PartSum* __restrict__ sums, uint32_t vocab,
             uint64_t stride, const float* __restrict__ temperature, uint32_t parts) {
  __shared__ u32x4 edges[2];
  __shared__ float tops[4];
  __shared__ uint64_t masses[4];
  const uint32_t r = blockIdx.x / parts, part = blockIdx.x % parts;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const float temp = temperature ? temperature[r] : 1.0f;
  Blocks<DT, 0> blocks;
  blocks.init(Row<DT>{static_cast<const char*>(logits) + r * stride * (DT == kF32 ? 4 : 2), vocab},
              edges);
  constexpr int N = kPart / 256, E = Row<DT>::E;
  u32x4 v[N];
  float x[N][E], top = -INFINITY;
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = blocks.load(part * kPart + 256 * j + t);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    unpack16<DT>(v[j], x[j]);
#pragma unroll
    for (int e = 0; e < E; ++e) top = fmaxf(top, x[j][e]);
  }
  top = wave_max(top);
  if (lane == 0) tops[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const Weigher weigh = Weigher::make(top, temp);
  uint64_t m = 0;
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int e = 0; e < E; ++e) m += weigh(x[j][e]);
  m = wave_sum64(m);
  if (lane == 0) masses[wave] = m;
  __syncthreads();
  if (t == 0)
    sums[static_cast<uint64_t>(r) * parts + part] =
        PartSum{top, 0, top == -INFINITY ? 0 : masses[0] + masses[1] + masses[2] + masses[3]};
}

template <int DT>
__global__ void __launch_bounds__(NT)
sample_pick(const void* __restrict__ logits, int32_t* __restrict__ tokens, uint32_t vocab,
            uint64_t stride, const float* __restrict__ uniform,
            const float* __restrict__ temperature, const PartSum* __restrict__ sums,
            uint32_t parts) {
  __shared__ Shared sh;
  const uint32_t r = blockIdx.x;
  const int t = threadIdx.x, lane = t & 63;
  const float temp = temperature ? temperature[r] : 1.0f, u = uniform[r];
  __shared__ u32x4 edges[2];
  Blocks<DT, 0> blocks;
  blocks.init(Row<DT>{static_cast<const char*>(logits) + r * stride * (DT == kF32 ? 4 : 2), vocab},
              edges);
  sums += static_cast<uint64_t>(r) * parts;
  float top = -INFINITY;
  for (uint32_t i = lane; i < parts; i += 64) top = fmaxf(top, sums[i].top);
  top = wave_max(top);
  if (top == -INFINITY) {
    if (t == 0) tokens[r] = -1;
    return;
  }
  // Masses relative to the row's largest logit, summed 64 parts at a time in a fixed order; then
  // the part that holds u.  Every wave does it on its own.
  const bool greedy = !(temp > 0.0f);
  const double c = greedy ? 0.0 : 1.4426950408889634 / static_cast<double>(temp);
  auto factor = [&](float x) {
    if (x == top) return 1.0;
    return greedy || !(x > -INFINITY) ? 0.0 : exp2(max(-2000.0, (static_cast<double>(x) - top) * c));
  };
  double mass = 0.0, upto = 0.0;   // of this lane's part, and of the 64's up to it
  auto sum64 = [&](uint32_t base) {
    const uint32_t i = base + lane;
    mass = i < parts ? static_cast<double>(sums[i].mass) * factor(sums[i].top) : 0.0;
    upto = mass;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double y = __shfl_up(upto, o);
      if (lane >= o) upto += y;
    }
  };
  double all = 0.0;
  uint32_t base = 0;
  for (; base < parts; base += 64) {
    sum64(base);
    all += __shfl(upto, 63);
  }
  const double target =
      greedy || !(u > 0.0f) ? 0.0 : min(static_cast<double>(u) * all, all * (1.0 - 0x1p-52));
  // (A lane's sum is of its own order: the last part's may round to below `all`, and is taken then
  // where none is above the target.)
  double before = 0.0, below = 0.0;
  uint32_t part = 0;
  for (base = 0; base < parts; base += 64) {
    if (parts > 64) sum64(base);
    const uint64_t some = __builtin_amdgcn_ballot_w64(mass > 0.0);
    const uint64_t in = __builtin_amdgcn_ballot_w64(mass > 0.0 && below + upto > target);
    if (some != 0) {
      const int l = in != 0 ? __builtin_ctzll(in) : 63 - __builtin_clzll(some);
      part = base + l;
      before = below + __shfl(upto - mass, l);
    }
    if (in != 0) break;
    below += __shfl(upto, 63);
  }
  const float part_top = sums[part].top;
  const double f = factor(part_top);
  const uint32_t k0 = part * kPart, k1 = min(blocks.count, k0 + kPart);
  if (greedy) {
    float x[Blocks<DT, 0>::E];
    Blocks<DT, 0>::unpack(blocks.load(k0 + t), x);
    uint32_t at = 0xffffffffu;
#pragma unroll
    for (int e = 0; e < static_cast<int>(Blocks<DT, 0>::E); ++e)
      at = x[e] == top ? min(at, blocks.index(k0 + t) + e) : at;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) at = min(at, __shfl_xor(at, o));
    if (lane == 0) sh.wave_a[t >> 6] = at;
    __syncthreads();
    for (int i = 0; i < NW; ++i) at = min(at, static_cast<uint32_t>(sh.wave_a[i]));
    if (t == 0) tokens[r] = static_cast<int32_t>(at);
    return;
  }
  const Weigher weigh = Weigher::make(part_top, temp);
  const double local =
      max(0.0, min((target - before) / f, short_of(sums[part].mass)));
  find_place(sh, blocks, k0, k1, 0, local, [&](uint32_t, float x) { return weigh(x); },
             tokens + r);
}

}  // namespace smp
}  // namespace th
