// The vector decode kernel's instances for windows with sinks (fp32 heads, 16-bit
// heads of 256; the matrix-core kernels hold their own).  As without a window, bound by
// the bytes of the rows seen: 64 sequences of 100-16000 tokens, window 2048, 4 sinks,
// fp32 32/8 heads of 128 182 us, 5.8 TB/s; bf16 16/4 heads of 256 113 us, 4.7 TB/s.
#include "decode_kernel.hpp"

namespace pa {

namespace {

struct WindowOp {
  const DecodeArgs& a;
  int64_t num_items;
  hipStream_t stream;
  template <typename T, int D, int G, bool SHARED, int DM>
  hipError_t run() const {
    const int64_t grid = num_items * a.num_kv_heads * a.sub_groups;
    hipLaunchKernelGGL((decode_partition_kernel<T, D, G, SHARED, DM, true>), dim3(static_cast<uint32_t>(grid)),
                       dim3(kDecodeThreads), 0, stream, a);
    return hipGetLastError();
  }
};

}  // namespace

hipError_t launch_decode_window(const DecodeArgs& a, int dtype, int head_dim, int group, int64_t num_items,
                                hipStream_t stream) {
  return visit_decode(dtype, head_dim, group, WindowOp{a, num_items, stream});
}

}  // namespace pa
