// Sampling of one token per row of logits: temperature, top-k, top-p, min-p, from a given
// random number.  Bound by the row's bytes; the passes after the first read the caches.
//
//   w_i = exp((x_i - x_max) / T), held as whole numbers of 2^-31, so that masses are exact in
//   64 bits and no order of summation shows.
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
#pragma once

#include "common.hpp"

namespace th {
namespace smp {
constexpr int NT = 1024, NW = NT / 64;
constexpr int BINS = 2048;
constexpr int CAP = 2048;       // members that are ranked in LDS
constexpr float kLowest = 33.0f;   // 2^-33 rounds to no step of 2^-31
constexpr uint32_t kOne = 1u << 31;

struct Pair {   // a place in the order: larger key first, then lower index
  uint32_t key, idx;
};
__device__ __forceinline__ bool upto(uint32_t key, uint32_t idx, Pair cut) {
  return key > cut.key || (key == cut.key && idx <= cut.idx);
}

__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

// Row of logits; NaN counts as -infinity, and -0 as 0.
template <int DT>
struct Row {
  const void* p;
  __device__ __forceinline__ float operator[](uint32_t i) const {
    float x;
    if constexpr (DT == kF32) x = static_cast<const float*>(p)[i];
    else x = u16_to_f32<DT>(static_cast<const uint16_t*>(p)[i]);
    return x != x ? -INFINITY : x + 0.0f;
  }
};

struct Weigher {
  float top, c_hi, c_lo;   // log2(e) / T as the sum of two floats
  __device__ __forceinline__ uint32_t operator()(float x) const {
    if (x == top) return kOne;   // (infinities too)
    const float d = x - top;
    if (!(d > -INFINITY)) return 0;
    const float y = d * c_hi;
    if (y < -kLowest) return 0;
    const float y_lo = __builtin_fmaf(d, c_hi, -y) + d * c_lo;
    const float e = exp2_fast(y);
    return static_cast<uint32_t>(
        __builtin_rintf(__builtin_fmaf(e * y_lo, 0.69314718f, e) * static_cast<float>(kOne)));
  }
};

__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t lo = __shfl_xor(static_cast<uint32_t>(v), o);
    const uint32_t hi = __shfl_xor(static_cast<uint32_t>(v >> 32), o);
    v += static_cast<uint64_t>(hi) << 32 | lo;
  }
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
  uint32_t weight[CAP];
  uint64_t wave_a[NW], wave_b[NW];
  float wave_f[NW];
  uint32_t members;
  uint32_t bin;
  uint64_t above_n, above_m, found, found_m;
  uint32_t in_bin;
  uint64_t lo, hi;
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

template <int DT>
struct Sampler {
  Row<DT> row;
  uint32_t vocab;
  Weigher weigh;
  float bin_scale;
  Shared& sh;

  __device__ __forceinline__ uint32_t bin_of(float x) const {
    const float d = (weigh.top - x) * bin_scale;
    return d < static_cast<float>(BINS - 1) ? static_cast<uint32_t>(d) : BINS - 1;
  }

  // Counts and masses of all tokens by bins of x.
  __device__ __forceinline__ void histogram() {
    const int t = threadIdx.x;
    for (int i = t; i < BINS; i += NT) {
      sh.count[i] = 0;
      sh.mass[i] = 0;
    }
    __syncthreads();
    for (uint32_t i = t; i < vocab; i += NT) {
      const float x = row[i];
      if (x == -INFINITY) continue;
      const uint32_t b = x == weigh.top ? 0u : bin_of(x);
      atomicAdd(&sh.count[b], 1u);
      const uint32_t w = weigh(x);
      if (w) atomicAdd(&sh.mass[b], static_cast<unsigned long long>(w));
    }
    __syncthreads();
  }

  // The goal's cut among the tokens up to `cut`; sum: the mass up to the new cut.  The bins are
  // those of histogram(), whole rows (a goal is met at or before `cut` if it was chosen so).
  __device__ __forceinline__ Pair select(const Goal& goal, Pair cut, uint64_t* sum) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    find_bin(sh, goal, 0, 0);
    // every token is wanted, or the cut is among those without weight
    if (sh.bin >= BINS - 1) return cut;
    const uint32_t first_bin = sh.bin;
    uint64_t lo = 0, hi = ~0ull;   // members' (key, ~index)
    while (sh.in_bin > CAP) {
      // divide the members again, evenly between the least and the largest of them
      uint64_t a = ~0ull, b = 0;
      for (uint32_t i = t; i < vocab; i += NT) {
        const float x = row[i];
        if (x == -INFINITY || (x == weigh.top ? 0u : bin_of(x)) != first_bin) continue;
        const uint64_t v = static_cast<uint64_t>(order_key(x)) << 32 | (0xffffffffu - i);
        if (v < lo || v > hi) continue;
        a = min(a, v);
        b = max(b, v);
      }
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint64_t a2 = static_cast<uint64_t>(__shfl_xor(static_cast<uint32_t>(a >> 32), o)) << 32 |
                            __shfl_xor(static_cast<uint32_t>(a), o);
        const uint64_t b2 = static_cast<uint64_t>(__shfl_xor(static_cast<uint32_t>(b >> 32), o)) << 32 |
                            __shfl_xor(static_cast<uint32_t>(b), o);
        a = min(a, a2);
        b = max(b, b2);
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
      for (int i = t; i < BINS; i += NT) {
        sh.count[i] = 0;
        sh.mass[i] = 0;
      }
      __syncthreads();
      for (uint32_t i = t; i < vocab; i += NT) {
        const float x = row[i];
        if (x == -INFINITY || (x == weigh.top ? 0u : bin_of(x)) != first_bin) continue;
        const uint64_t v = static_cast<uint64_t>(order_key(x)) << 32 | (0xffffffffu - i);
        if (v < lo || v > hi) continue;
        const uint32_t q = static_cast<uint32_t>((hi - v) >> shift);
        atomicAdd(&sh.count[q], 1u);
        atomicAdd(&sh.mass[q], static_cast<unsigned long long>(weigh(x)));
      }
      __syncthreads();
      find_bin(sh, goal, base_n, base_m);
      const uint64_t q = sh.bin;
      const uint64_t top = hi - (q << shift);
      const uint64_t width = (1ull << shift) - 1;
      lo = top - lo > width ? top - width : lo;
      hi = top;
    }
    // the members, in any order; each is ranked by a walk over the others
    if (t == 0) sh.members = 0;
    __syncthreads();
    for (uint32_t i = t; i < vocab; i += NT) {
      const float x = row[i];
      if (x == -INFINITY || (x == weigh.top ? 0u : bin_of(x)) != first_bin) continue;
      const uint64_t v = static_cast<uint64_t>(order_key(x)) << 32 | (0xffffffffu - i);
      if (v < lo || v > hi) continue;
      const uint32_t at = atomicAdd(&sh.members, 1u);
      if (at < CAP) {
        sh.member[at] = v;
        sh.weight[at] = weigh(x);
      }
    }
    __syncthreads();
    const uint32_t n = min(sh.members, static_cast<uint32_t>(CAP));
    for (uint32_t i = t; i < n; i += NT) {
      const uint64_t v = sh.member[i];
      uint64_t bn = sh.above_n, bm = sh.above_m;
      for (uint32_t j = 0; j < n; ++j) {
        const bool before = sh.member[j] > v;
        bn += before;
        bm += before ? sh.weight[j] : 0u;
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

// One workgroup per row.
template <int DT>
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
  const float p = top_p ? top_p[r] : 1.0f, mp = min_p ? min_p[r] : 0.0f;
  const Row<DT> row{static_cast<const char*>(logits) + r * stride * (DT == kF32 ? 4 : 2)};

  // the largest logit and its lowest index
  float top = -INFINITY;
  uint32_t at = 0xffffffffu;
  for (uint32_t i = t; i < vocab; i += NT) {
    const float x = row[i];
    if (x > top) {
      top = x;
      at = i;
    }
  }
  {
    uint64_t v = static_cast<uint64_t>(order_key(top)) << 32 | (0xffffffffu - at);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint64_t v2 = static_cast<uint64_t>(__shfl_xor(static_cast<uint32_t>(v >> 32), o)) << 32 |
                          __shfl_xor(static_cast<uint32_t>(v), o);
      v = max(v, v2);
    }
    if (lane == 0) sh.wave_a[wave] = v;
    __syncthreads();
    for (int i = 0; i < NW; ++i) v = max(v, sh.wave_a[i]);
    const uint32_t key = static_cast<uint32_t>(v >> 32);
    top = __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
    at = 0xffffffffu - static_cast<uint32_t>(v);
    __syncthreads();
  }
  if (top == -INFINITY) {
    if (t == 0) tokens[r] = -1;
    return;
  }
  // one token is kept (or asked for): the first
  if (!(temp > 0.0f) || k == 1 || p <= 0.0f || mp > 1.0f) {
    if (t == 0) tokens[r] = static_cast<int32_t>(at);
    return;
  }
  const double c = 1.4426950408889634 / static_cast<double>(temp);
  Weigher weigh;
  weigh.top = top;
  weigh.c_hi = static_cast<float>(min(c, 3.0e38));
  weigh.c_lo = static_cast<float>(min(c, 3.0e38) - static_cast<double>(weigh.c_hi));
  Sampler<DT> s{row, vocab, weigh, weigh.c_hi * (static_cast<float>(BINS - 1) / kLowest), sh};

  Pair cut{0, 0xffffffffu};
  const bool cut_k = k > 0 && static_cast<uint32_t>(k) < vocab, cut_p = p < 1.0f;
  if (cut_k || cut_p) {
    s.histogram();
    uint64_t whole = 0;
    if (cut_p) {   // all the row's mass, unless top-k leaves less
      uint64_t m = wave_sum64(sh.mass[2 * t] + sh.mass[2 * t + 1]);
      if (lane == 0) sh.wave_a[wave] = m;
      __syncthreads();
      for (int i = 0; i < NW; ++i) whole += sh.wave_a[i];
      __syncthreads();
    }
    if (cut_k) {
      cut = s.select(Goal{false, static_cast<uint64_t>(k), 0.0}, cut, &whole);
      __syncthreads();
    }
    if (cut_p) {
      if (cut_k) s.histogram();   // (a division may have used the bins)
      uint64_t sum;
      const Pair by_p =
          s.select(Goal{true, 0, static_cast<double>(p) * static_cast<double>(whole)}, cut, &sum);
      if (!upto(by_p.key, by_p.idx, cut)) {
        // rounding put the mass cut behind the other: the other holds
      } else {
        cut = by_p;
      }
      __syncthreads();
    }
  }

  // kept mass of [a, b) by waves; then the place, in the share that holds it
  auto kept = [&](uint32_t i) -> uint32_t {
    const float x = row[i];
    if (x == -INFINITY || !upto(order_key(x), i, cut)) return 0;
    const uint32_t w = weigh(x);
    return static_cast<float>(w) * (1.0f / static_cast<float>(kOne)) >= mp || !(mp > 0.0f) ? w : 0u;
  };
  uint32_t a = 0, b = vocab;
  uint64_t before = 0;   // mass below a
  double target = 0.0;
  bool first = true;
  while (true) {
    const uint32_t share = (b - a + NW - 1) / NW;
    const uint32_t wa = min(b, a + wave * share), wb = min(b, wa + share);
    uint64_t m = 0;
    for (uint32_t i = wa + lane; i < wb; i += 64) m += kept(i);
    m = wave_sum64(m);
    if (lane == 0) sh.wave_a[wave] = m;
    __syncthreads();
    if (first) {
      uint64_t all = 0;
      for (int i = 0; i < NW; ++i) all += sh.wave_a[i];
      const float u = uniform[r];
      target = min(u > 0.0f ? static_cast<double>(u) * static_cast<double>(all) : 0.0,
                   static_cast<double>(all) - 0.5);
      first = false;
    }
    int w = 0;
    while (w < NW - 1 && static_cast<double>(before + sh.wave_a[w]) <= target) {
      before += sh.wave_a[w];
      ++w;
    }
    __syncthreads();
    const uint32_t na = min(b, a + w * share);
    b = min(b, na + share);
    a = na;
    if (b - a <= 64) break;
  }
  if (wave == 0) {
    const uint32_t i = a + lane;
    const uint64_t m = wave_scan64(i < b ? kept(i) : 0u, lane);
    const uint64_t over =
        __builtin_amdgcn_ballot_w64(i < b && static_cast<double>(before + m) > target);
    if (lane == 0)
      tokens[r] = static_cast<int32_t>(over ? a + __builtin_ctzll(over) : at);
  }
}

}  // namespace smp
}  // namespace th
