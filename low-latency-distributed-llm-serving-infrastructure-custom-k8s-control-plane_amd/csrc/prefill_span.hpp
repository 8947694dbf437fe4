// Launches of the matrix-core prefill over part of the context, for the sources
// that hold its instances.
#pragma once

#include <algorithm>

#include "prefill_kernel.hpp"

namespace pa {

template <typename T, int D, int DM, int SPAN>
static hipError_t launch_prefill_span_d(const PrefillArgs& args, int group, int64_t num_items, hipStream_t s) {
  const int g = group / args.sub_groups;
  if (g < 1 || g > 8 || args.new_key != nullptr) return hipErrorNotSupported;
  PrefillArgs a = args;
  a.num_units = num_items * a.num_kv_heads * a.sub_groups;
  // Unit ranks are 32-bit and a workgroup's ranks reach about twice the count.
  if (a.num_units > (int64_t{1} << 30)) return hipErrorInvalidValue;
  const int cus = device_compute_units();
  const dim3 grid(static_cast<uint32_t>(cus > 0 ? std::min<int64_t>(a.num_units, cus) : a.num_units));
  if (a.key_scales != nullptr)
    hipLaunchKernelGGL((prefill_kernel<T, D, DM, false, false, true, SPAN>), grid, dim3(kPrefillThreads), 0, s, a);
  else if constexpr (SPAN == kSpanTree)
    return hipErrorNotSupported;  // (tree_attention.hip)
  else if ((1 << a.log2_block_size) >= kCopyRows)
    hipLaunchKernelGGL((prefill_kernel<T, D, DM, false, false, false, SPAN>), grid, dim3(kPrefillThreads), 0, s, a);
  else
    hipLaunchKernelGGL((prefill_kernel<T, D, DM, true, false, false, SPAN>), grid, dim3(kPrefillThreads), 0, s, a);
  return hipGetLastError();
}

template <typename T, int SPAN>
static hipError_t launch_prefill_span_t(const PrefillArgs& a, int head_dim, int group, int64_t num_items,
                                        hipStream_t s) {
  switch (head_dim) {
    case 64: return launch_prefill_span_d<T, 64, 64, SPAN>(a, group, num_items, s);
    case 80: return launch_prefill_span_d<T, 128, 80, SPAN>(a, group, num_items, s);
    case 96: return launch_prefill_span_d<T, 128, 96, SPAN>(a, group, num_items, s);
    case 128: return launch_prefill_span_d<T, 128, 128, SPAN>(a, group, num_items, s);
    default: return hipErrorNotSupported;
  }
}

template <int SPAN>
static hipError_t launch_prefill_span(const PrefillArgs& a, int dtype, int head_dim, int group, int64_t num_items,
                                      hipStream_t s) {
  if (dtype == PA_DTYPE_BF16) return launch_prefill_span_t<bf16_t, SPAN>(a, head_dim, group, num_items, s);
  if (dtype == PA_DTYPE_F16) return launch_prefill_span_t<f16_t, SPAN>(a, head_dim, group, num_items, s);
  return hipErrorNotSupported;
}

}  // namespace pa
