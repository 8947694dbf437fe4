// The matrix-core prefill's instances for trees of drafted tokens over 8-bit caches.
#include "prefill_span.hpp"

namespace pa {

hipError_t launch_prefill_tree(const PrefillArgs& a, int dtype, int head_dim, int group, int64_t num_items,
                               hipStream_t stream) {
  return launch_prefill_span<kSpanTree>(a, dtype, head_dim, group, num_items, stream);
}

}  // namespace pa
