// th_sample (include/tilers_hip.h, section 2).
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "kernels/sample.hpp"
#include "ops_common.hpp"
#include "runtime.hpp"

using th::fail;
using namespace th::ops;

namespace {

// Rows of up to 16 vectors per thread stay in registers; the least that holds them.  (8 rows with
// all limits, us: 8000 bf16 19 so, 24 read again at each pass, 52 with room for 16; 50257 bf16
// 37, 42, 54, f32 34, 41, 40; 128256 bf16 68, 70.)
template <int DT>
int sample_go(const void* logits, int32_t* tokens, uint32_t rows, uint32_t vocab, uint64_t stride,
              const float* uniform, const float* temperature, const int32_t* top_k,
              const float* top_p, const float* min_p, hipStream_t s) {
  constexpr uint32_t E = th::smp::Row<DT>::E;
  const uint64_t blocks = (static_cast<uint64_t>(vocab) + E - 1 + E - 1) / E;   // at any alignment
  auto go = [&](auto nv) {
    hipLaunchKernelGGL((th::smp::sample_rows<DT, nv.value>), dim3(rows), dim3(th::smp::NT), 0, s,
                       logits, tokens, vocab, stride, uniform, temperature, top_k, top_p, min_p);
  };
  // Without limits a long row's one pass is divided: over many workgroups where there are few
  // rows, and always where a row does not stay in a workgroup's registers with ease.  Not divided
  // and divided, us: 8 rows of 8000 bf16 7.8, 9.9; of 50257 13.5, 10.0; of 128256 22, 10.2; 64
  // rows of 20000 f32 9.3, 10.1; of 50257 12.3, 11.3; 256 rows of 50257 f32 18.5, 19.5; of 128256
  // 47.7, 30.7, bf16 31.0, 26.8.  The parts' sums go to the stream's scratch, which a captured
  // stream does not offer.
  const uint32_t parts = static_cast<uint32_t>((blocks + th::smp::kPart - 1) / th::smp::kPart);
  if (!top_k && !top_p && !min_p &&
      (blocks > 1024 * 13 || (blocks > 1024 * 5 && 4ull * rows <= current_cu_count())) &&
      !stream_capturing(s)) {
    if (uint64_t{rows} * parts > 0xffffffffu / 256)
      return fail(TH_KERNEL_ERROR, "sample: grid too large");
    void* sums = nullptr;
    th::ScratchHold hold;
    // (without memory for them the rows stay whole)
    if (th::try_stream_scratch(s, sizeof(th::smp::PartSum) * rows * parts, &sums, &hold)) {
      auto* ps = static_cast<th::smp::PartSum*>(sums);
      hipLaunchKernelGGL((th::smp::sample_parts<DT>), dim3(rows * parts), dim3(256), 0, s, logits,
                         ps, vocab, stride, temperature, parts);
      hipLaunchKernelGGL((th::smp::sample_pick<DT>), dim3(rows), dim3(th::smp::NT), 0, s, logits,
                         tokens, vocab, stride, uniform, temperature, ps, parts);
      return launch_status("sample launch");
    }
  }
  using std::integral_constant;
  if (blocks <= 1024 * 2) go(integral_constant<int, 2>{});
  else if (blocks <= 1024 * 4) go(integral_constant<int, 4>{});
  else if (blocks <= 1024 * 8) go(integral_constant<int, 8>{});
  else if (blocks <= 1024 * 13) go(integral_constant<int, 13>{});
  else if (blocks <= 1024 * 16) go(integral_constant<int, 16>{});
  else go(integral_constant<int, 0>{});
  return launch_status("sample launch");
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace

extern "C" int th_sample(const void* logits, int32_t* tokens, uint32_t rows, uint32_t vocab,
                         uint64_t stride, th_dtype dtype, const float* uniform,
                         const float* temperature, const int32_t* top_k, const float* top_p,
                         const float* min_p, th_stream s) {
  if (!valid_dtype(dtype)) return fail(TH_KERNEL_ERROR, "sample: unknown dtype");
  if (stride == 0) stride = vocab;
  if (stride < vocab) return fail(TH_KERNEL_ERROR, "sample: stride is less than vocab");
  if (vocab > (1u << 23) || rows > 0x7fffffffu)
    return fail(TH_KERNEL_ERROR, "sample: vocab must be at most 2^23 and rows below 2^31");
  if (rows == 0) return TH_OK;
  if (vocab == 0) return fail(TH_KERNEL_ERROR, "sample: vocab == 0");
  if (stride > (uint64_t{1} << 60) / rows) return fail(TH_KERNEL_ERROR, "sample: stride is too large");
  if (rows > 0xffffffffu / th::smp::NT) return fail(TH_KERNEL_ERROR, "sample: grid too large");
  if (!logits || !tokens || !uniform) return fail(TH_KERNEL_ERROR, "sample: null pointer");
  if (!aligned(logits, dtype_size(dtype)) || !aligned(tokens, 4) || !aligned(uniform, 4) ||
      !aligned(temperature, 4) || !aligned(top_k, 4) || !aligned(top_p, 4) || !aligned(min_p, 4))
    return fail(TH_KERNEL_ERROR, "sample: pointers must be aligned to their elements");
  switch (dtype) {
    case TH_F32:
      return sample_go<th::kF32>(logits, tokens, rows, vocab, stride, uniform, temperature, top_k,
                                 top_p, min_p, as_stream(s));
    case TH_F16:
      return sample_go<th::kF16>(logits, tokens, rows, vocab, stride, uniform, temperature, top_k,
                                 top_p, min_p, as_stream(s));
    default:
      return sample_go<th::kBF16>(logits, tokens, rows, vocab, stride, uniform, temperature, top_k,
                                  top_p, min_p, as_stream(s));
  }
}
