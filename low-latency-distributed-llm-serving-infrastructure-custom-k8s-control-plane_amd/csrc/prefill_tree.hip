// The matrix-core prefill's instances for trees of drafted tokens over 8-bit caches:
// 16 trees of 9-17 nodes after 100-6000 tokens, 32/8 heads of 128, 69 us (104 MB; a
// unit's start and its chain of steps), the generic kernel 5.9 ms.
//
// A probability goes into the product as two terms of the query's type, as in
// tree_attention.hip and in the decode over these caches.  One term took 56 us and was off
// 64 bits by 2.24e-3 (bf16, 2-norm), two are off by 1.66e-3; the registers of the second
// one spill (36 a lane for heads of 128, with V's two halves of a tile read one after the
// other; 54, 70.5 us, with both ahead).
#include "prefill_span.hpp"

namespace pa {

hipError_t launch_prefill_tree(const PrefillArgs& a, int dtype, int head_dim, int group, int64_t num_items,
                               hipStream_t stream) {
  return launch_prefill_span<kSpanTree>(a, dtype, head_dim, group, num_items, stream);
}

}  // namespace pa
