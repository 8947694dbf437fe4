// The matrix-core prefill's instances for trees of drafted tokens over 8-bit caches:
// 16 trees of 9-17 nodes after 100-6000 tokens, 32/8 heads of 128, 59 us (104 MB; a
// unit's start and its chain of steps; tree_attention.hip over 16 bits 51), the generic
// kernel 5.9 ms.
#include "prefill_span.hpp"

namespace pa {

hipError_t launch_prefill_tree(const PrefillArgs& a, int dtype, int head_dim, int group, int64_t num_items,
                               hipStream_t stream) {
  return launch_prefill_span<kSpanTree>(a, dtype, head_dim, group, num_items, stream);
}

}  // namespace pa
