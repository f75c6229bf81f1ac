// Paged K/V cache: writing new tokens (16 bits, or 8 bits with a scale per token and head) and
// reading sequences back into the contiguous layout.  Both are bound by their bytes.
//
//   write  a = max |x| over the head's values, scale = a / M, code = rn(x * (M / a)), with
//          M = 448 (e4m3) or 127 (i8); every quotient and product is rounded to f32 once, so the
//          codes are the same on any machine that does that.
//   read   code * scale rounded to f32, then to the output's type.
//
// A row (one token and head of K or V) is `LG` lanes of eight values: 16 bytes of a 16-bit
// tensor per lane, and the row's maximum takes log2(LG) lane exchanges.
//
// Measured, 8 heads of 128: writing 25663 tokens of bf16 as i8 30 us (159 MB, 5.3 TB/s; 34 with
// the loads behind the lookup of the page and the codes gathered by shifts), 56 tokens 4.6;
// reading 8 sequences of up to 8192 positions from e4m3 into bf16 46 us (311 MB, 6.7 TB/s, a
// third of it found in the last-level cache; 65 where nothing is), 77 with stores that go through
// the caches and four rows in flight per lane instead of two, 118 with eight.
#pragma once

#include "common.hpp"
#include "paged_index.hpp"

namespace th {

// The pool as the kernels see it; strides in elements.
struct PagedPool {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  uint64_t page_stride;
  uint32_t nkv, head_dim;
};

template <int CT> constexpr int cache_size() { return CT == kE4M3 || CT == kI8 ? 1 : 2; }
template <int CT> constexpr float cache_most() { return CT == kE4M3 ? 448.0f : 127.0f; }
template <int CT> constexpr bool cache_codes() { return CT == kE4M3 || CT == kI8; }

// Element offset of a row of the pool, and index of its scale.
__device__ __forceinline__ uint64_t pool_row(const PagedPool& p, const PagedSeqs& s, int32_t page,
                                             uint32_t head, uint32_t row) {
  return static_cast<uint64_t>(page) * p.page_stride +
         ((static_cast<uint64_t>(head) << s.shift) + row) * p.head_dim;
}
__device__ __forceinline__ uint64_t pool_scale(const PagedPool& p, const PagedSeqs& s, int32_t page,
                                               uint32_t head, uint32_t row) {
  return ((static_cast<uint64_t>(page) * p.nkv + head) << s.shift) + row;
}

// Eight values of a tensor of type DT as they lie in memory; their values in f32, and back (one
// rounding).
template <int DT> struct Raw8 {
  u32x4 w[DT == kF32 ? 2 : 1];
};
template <int DT>
__device__ __forceinline__ Raw8<DT> load8(const void* p) {
  Raw8<DT> r;
  r.w[0] = ldg128(p);
  if constexpr (DT == kF32) r.w[1] = ldg128(static_cast<const float*>(p) + 4);
  return r;
}
template <int DT>
__device__ __forceinline__ void widen8(const Raw8<DT>& r, float (&f)[8]) {
  if constexpr (DT == kF32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(r.w[i / 4][i % 4]);
  } else {
    unpack16<DT>(r.w[0], f);
  }
}
// (Past: around the caches.)
template <int DT, bool Past>
__device__ __forceinline__ void store8(void* p, const float (&f)[8]) {
  auto put = [](u32x4 x, u32x4* to) {
    if constexpr (Past) __builtin_nontemporal_store(x, to);
    else *to = x;
  };
  if constexpr (DT == kF32) {
    u32x4 a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = __float_as_uint(f[i]);
      b[i] = __float_as_uint(f[4 + i]);
    }
    put(a, static_cast<u32x4*>(p));
    put(b, static_cast<u32x4*>(p) + 1);
  } else {
    put(pack16<DT>(f), static_cast<u32x4*>(p));
  }
}

// Eight codes in two dwords from values already multiplied by M / a, and their values.
template <int CT>
__device__ __forceinline__ u32x2 encode8(const float (&f)[8]) {
  u32x2 w;
  if constexpr (CT == kE4M3) {
    // at most 448 (1 + 2^-22), which rounds to 448: nothing overflows
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int d = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i], f[4 * i + 1], 0, false);
      d = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2], f[4 * i + 3], d, true);
      w[i] = static_cast<uint32_t>(d);
    }
  } else {
    // f + 3 * 2^22 has the integer nearest to f (ties to even) in its low bits: at most 127
    // (1 + 2^-22), so in its low byte
    uint32_t d[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] = __float_as_uint(f[i] + 12582912.0f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t lo = __builtin_amdgcn_perm(d[4 * i + 1], d[4 * i], 0x0c0c0400u);
      const uint32_t hi = __builtin_amdgcn_perm(d[4 * i + 3], d[4 * i + 2], 0x04000c0cu);
      w[i] = lo | hi;
    }
  }
  return w;
}
template <int CT>
__device__ __forceinline__ void decode8(u32x2 w, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (CT == kE4M3) {
      const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[i]), false);
      const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[i]), true);
      f[4 * i] = a[0];
      f[4 * i + 1] = a[1];
      f[4 * i + 2] = b[0];
      f[4 * i + 3] = b[1];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        f[4 * i + j] = static_cast<float>(static_cast<int8_t>(w[i] >> (8 * j)));
    }
  }
}

// One wave per new token: which sequence it belongs to is a count of the q_start values at or
// below it (64 at a time), and its rows of all K heads, then V heads, go through the wave
// 64 / LG at a time, U steps in flight.
template <int DT, int CT, int LG, int U>
__global__ void __launch_bounds__(256)
kv_cache_write(PagedPool p, PagedSeqs s, const void* __restrict__ k, const void* __restrict__ v,
               uint64_t stride) {
  constexpr int RPW = 64 / LG;
  constexpr int SZ = DT == kF32 ? 4 : 2;
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t token =
      __builtin_amdgcn_readfirstlane(blockIdx.x * 4u + (threadIdx.x >> 6));
  if (token >= s.total_q) return;
  const uint32_t col = 8u * (lane % LG), rows = 2u * p.nkv;
  Raw8<DT> x[U];
  auto bring = [&](uint32_t r0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t r = r0 + u * RPW, h = r < p.nkv ? r : r - p.nkv;
      x[u] = {};
      if (r < rows && col < p.head_dim)
        x[u] = load8<DT>(static_cast<const char*>(r < p.nkv ? k : v) +
                         SZ * (token * stride + static_cast<uint64_t>(h) * p.head_dim + col));
    }
  };
  bring(lane / LG);   // in flight while the sequence is looked up
  uint32_t le = 0;
  for (uint32_t j0 = 0; j0 < s.batch; j0 += 64) {
    const uint32_t j = j0 + lane;
    const bool at = j < s.batch && paged_clamp(s.q_start[j], s.total_q) <= token;
    le += __builtin_popcountll(__builtin_amdgcn_ballot_w64(at));
  }
  if (le == 0) return;
  const uint32_t b = __builtin_amdgcn_readfirstlane(le - 1);
  const PagedChunk c = paged_chunk(s, b);
  if (token < c.first || token - c.first >= c.n) return;
  const int32_t pos = c.base + static_cast<int32_t>(token - c.first);
  if (pos < 0) return;
  const int32_t page = paged_page(s, b, static_cast<uint32_t>(pos));
  if (page < 0) return;
  const uint32_t row = paged_row(s, static_cast<uint32_t>(pos));
  for (uint32_t r0 = lane / LG; r0 < rows; r0 += RPW * U) {
    if (r0 >= RPW * U) bring(r0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t r = r0 + u * RPW, h = r < p.nkv ? r : r - p.nkv;
      float f[8];
      widen8<DT>(x[u], f);
      float scale = 0.0f;
      if constexpr (cache_codes<CT>()) {
        float a = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) a = maximumf(a, __builtin_fabsf(f[i]));
#pragma unroll
        for (int o = 1; o < LG; o <<= 1) a = maximumf(a, __shfl_xor(a, o));
        const bool some = a >= 1e-30f, fine = a < INFINITY;   // neither where a is NaN
        const float inv = some && fine ? cache_most<CT>() / a : 0.0f;
        if (inv == 0.0f) {   // (codes of zero, not of minus zero)
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = 0.0f;
        }
        scale = fine ? (some ? a / cache_most<CT>() : 0.0f) : NAN;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          f[i] *= inv;
          asm("" : "+v"(f[i]));   // (rounded before the code is)
        }
      }
      if (r < rows && col < p.head_dim) {
        void* pool = r < p.nkv ? p.k : p.v;
        const uint64_t at = pool_row(p, s, page, h, row) + col;
        if constexpr (cache_codes<CT>()) {
          *reinterpret_cast<u32x2*>(static_cast<uint8_t*>(pool) + at) = encode8<CT>(f);
          if (col == 0)
            (r < p.nkv ? p.k_scale : p.v_scale)[pool_scale(p, s, page, h, row)] = scale;
        } else {
          store8<CT, false>(static_cast<uint16_t*>(pool) + at, f);
        }
      }
    }
  }
}

// One workgroup per (sequence, head, U * 256 / LG positions), K and V; those past kv_len end at
// once.
template <int DT, int CT, int LG, int U>
__global__ void __launch_bounds__(256)
kv_cache_read(PagedPool p, PagedSeqs s, void* __restrict__ k, void* __restrict__ v,
              uint32_t max_seq, uint32_t nchunks) {
  constexpr uint32_t RPB = 256 / LG;
  const uint32_t chunk = blockIdx.x % nchunks, bh = blockIdx.x / nchunks;
  const uint32_t b = bh / p.nkv, h = bh % p.nkv;
  const uint32_t len = min(paged_clamp(s.kv_len[b], 0x7fffffffu), max_seq);
  const uint32_t first = chunk * (U * RPB) + threadIdx.x / LG, col = 8u * (threadIdx.x % LG);
  if (chunk * (U * RPB) >= len || col >= p.head_dim) return;
  float f[2][U][8];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t pos = first + u * RPB;
    const int32_t page = pos < len ? paged_page(s, b, pos) : -1;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[kv][u][i] = 0.0f;
      if (page >= 0) {
        const uint32_t row = paged_row(s, pos);
        const uint64_t at = pool_row(p, s, page, h, row) + col;
        const void* pool = kv ? p.v : p.k;
        if constexpr (cache_codes<CT>()) {
          const float scale =
              (kv ? p.v_scale : p.k_scale)[pool_scale(p, s, page, h, row)];
          decode8<CT>(*reinterpret_cast<const u32x2*>(static_cast<const uint8_t*>(pool) + at),
                      f[kv][u]);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            f[kv][u][i] *= scale;
            // (kept from merging with the conversion to f16, which would round once and lose the
            // sign of a zero)
            if constexpr (DT == kF16) asm("" : "+v"(f[kv][u][i]));
          }
        } else {
          widen8<CT>(load8<CT>(static_cast<const uint16_t*>(pool) + at), f[kv][u]);
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t pos = first + u * RPB;
    if (pos >= len) continue;
    const uint64_t at = (static_cast<uint64_t>(bh) * max_seq + pos) * p.head_dim + col;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      void* out = kv ? v : k;
      if constexpr (DT == kF32) store8<DT, true>(static_cast<float*>(out) + at, f[kv][u]);
      else store8<DT, true>(static_cast<uint16_t*>(out) + at, f[kv][u]);
    }
  }
}

}  // namespace th
