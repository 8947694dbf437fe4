// The matrix-core prefill's instances for windows with sinks.
//
// As the causal kernel, bound by the chain of its steps; what a window leaves out is
// left out in whole stages.  4 prompts of 2048 tokens at 0 to 12288, 32/8 heads of 128,
// window 2048, 4 sinks: 300 us, 803 TFLOP/s of what the queries see (over the 8-bit
// cache 334 us); the generic kernel, which walks the window row by row, 62 ms.  Masks
// from one word of bits a row and tile, not from comparisons with each limit: 308 ->
// 300 us.
//
// A probability goes into the product with V as one 16-bit term, as in the causal kernel
// and for its reason (prefill.hip): a prompt's layers with and without a window round
// alike.  Two terms, measured: these prompts 297 -> 384 us, off 64 bits (bf16, 2-norm) by
// 2.15e-3 -> 1.64e-3, of which 1.64e-3 is the result's rounding; over the 8-bit cache 336
// -> 433; 4 prompts with 16/4 heads of 256 (prefill256.hip) 398 -> 463; fp16, 5 ragged
// prompts of up to 611 tokens beside 9 decodes, heads of 80, 28.5 -> 30.6, 2.6e-4 ->
// 2.0e-4.
#include "prefill_span.hpp"

namespace pa {

hipError_t launch_prefill_window(const PrefillArgs& a, int dtype, int head_dim, int group, int64_t num_items,
                                 hipStream_t stream) {
  return launch_prefill_span<kSpanWindow>(a, dtype, head_dim, group, num_items, stream);
}

}  // namespace pa
