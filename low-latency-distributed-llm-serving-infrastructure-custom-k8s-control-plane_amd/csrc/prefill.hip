// Causal chunked prefill over the paged cache with gfx950 MFMA tiles (the kernel
// itself: prefill_kernel.hpp).
//
// A unit of work is (sequence, query tile, KV head).  The tile holds 128
// query rows = (128 / G) query tokens x the G query heads that share the KV
// head.  The launch runs one workgroup (8 waves) per CU, and each walks its
// share of the units in turn (longest first, snake order), so a unit's
// start costs no workgroup launch.  The context is walked in stages of 64
// tokens; wave w owns rows [32 (w%4), 32 (w%4) + 32) and the 32-token half
// w/4 of every stage, with flash-style online softmax in fp32, so the two
// waves of a row group split the context and merge their partial results
// through LDS at the end (this halves the longest chain of a causal tile).
// The query tile comes into LDS and the finished rows leave through it, in
// whole rows: a lane's own row in registers would take one 16-byte piece of
// 32 different rows per load or store.
//
// Both products are computed transposed so that a lane owns one query row:
//   S^T[kv][row] = sum_d K[kv][d] Q[row][d]       (A = K regs, B = Q regs)
//   O^T[d][row] += sum_kv V^T[d][kv] P^T[kv][row]  (A = V^T regs, B = P^T regs)
// with v_mfma_f32_32x32x16_bf16 (or _f16 for fp16 caches).  In the 32x32
// accumulator lane l holds column l % 32 and rows 8*(i/4) + 4*(l/32) + (i%4),
// i = 0..15, so the softmax max/sum of a query row needs only its own 16
// values plus the partner lane l ^ 32, and the probabilities a lane holds
// are the B operand of the PV product with the context index of k-slot j
// being 8*(j/4) + 4*(l/32) + (j%4) inside each 16-token step.
//
// K and V go from HBM straight into LDS with the gfx950 direct loads
// (global_load_lds_dwordx4: lane i's 16 bytes land at M0 + 16 i), into
// unpadded rows whose 16-byte chunks are XOR-swizzled (chunk_swizzle) so that
// the operand reads below are free of bank conflicts.  The V^T operand is
// read with the gfx950 LDS transpose read ds_read_b64_tr_b16: inside each
// group of 16 lanes, lane i receives element j from the 8-byte word
// addressed by lane (i/4 + 4j), element i%4.  Lane i of a group therefore
// addresses V[kv0 + (i/4)][d0 + 4*(i%4)] and receives V[kv0 + j][d0 + i],
// j = 0..3: four context tokens of its own output column.
//
// Copies.  Waves 0-3 copy 16 rows each of every stage.  One copy covers 4
// rows (8 for 64-dim heads) of one cache block, so its source is a scalar
// base (block id, row offset) plus a fixed per-lane offset: no vector
// address arithmetic.  The block ids come from an LDS ring of table entries
// that wave 0 fills eight stages ahead, read one step ahead of their use.
// (Blocks smaller than one copy take the per-lane form of the address.)
// The copies are issued from
// inline assembly and each copying wave waits for its own copies with an
// exact s_waitcnt vmcnt before the barrier that publishes them: the compiler
// would otherwise drain every copy before each LDS read, as it cannot tell
// the buffers apart.
//
// Pipeline (one barrier per stage).  K and V have separate LDS rings: the K
// of stage st+2 is read into registers during step st and consumed by the
// QK MFMAs of step st+1, so every step starts its MFMAs right after the
// barrier; the V of stage st is read during step st.  A step is two phases,
// each interleaved at the instruction level (sched_group_barrier):
//   A: QK MFMAs of stage st+1  |  softmax of stage st (exp2, pack, row sum)
//                              |  V^T reads of stage st
//   B: PV MFMAs of stage st    |  row maxima of stage st+1  |  K reads of st+2
// so each wave alternates matrix and vector work instead of running long
// runs of one kind in lock-step with the other wave of its SIMD.
// The row sum is accumulated from the rounded probabilities the PV product
// uses (v_dot2 against ones), per lane half, and the halves are added once
// at the end.  They enter that product as one 16-bit term: a weight is off by
// half a step of the type at most, about what rounding the result costs (bf16,
// four chunks of 512 at 4096: off by 0.0022 of the result where fp32
// probabilities leave 0.0017, and 0.0016 is the result's rounding).  A second
// term, as in the decode, whose products are free beside its reads, would make
// 24 products of a tile's 16 (heads of 128), in a kernel that waits for little
// else.  Masking is applied only to tiles that cross the causal
// diagonal or the end of the context (or to every tile when some block id of
// the sequence lies outside the pool: those positions are skipped, as in
// decode), in a separate loop after the unmasked one, and the accumulator is
// rescaled only when some row's maximum grew by more than 2^8 over the
// reference maximum in use.
//
// CODES (the 8-bit cache): the rings hold 16-bit rows as above, so everything
// after them is the same; only the copies differ.  A thread takes one 16-byte
// piece (16 codes) of one row of K and of V a stage, converts it on its way
// (v_cvt_scalef32_pk_*_fp8, the block's scale in the same instruction) and
// writes two chunks.  The pieces are loaded two steps before the step that
// writes them, into registers of that step's parity: K of stage st+5 and V of
// st+3 go out in step st, which writes K of st+3 and V of st+1; the block id
// comes one step earlier still.  All eight waves share the conversions (16 a
// thread and step, against its 16 exponentials), which cost what the smaller
// reads save and some more: bf16, four chunks of 512 at 4096, 32/8 heads of 128
// (146 GFLOP), 170 us, 858 TFLOP/s (the 16-bit cache 152); 2048 at 6000, 262 us
// (231): both repeated until the clocks have settled, which takes the chip tens
// of launches (the first after a pause take 201 and 169 us, the fifteenth or
// twentieth 233 and 203).
// fp16, 1457 ragged tokens, 16/4 heads of 80: 44 us, its longest unit's chain of
// 30 stages.
//
// Reference: the block-diagonal causal mask of app/model/paged_attention.py:
// 92-118 applied by SDPA (paged_attention.py:170-178); query token j of a
// sequence at position start + j attends context positions [0, start + j].
#include <algorithm>
#include <atomic>

#include "prefill_kernel.hpp"

namespace pa {

bool prefill_fast_path_supported(int dtype, int head_dim, int group, int block_size) {
  // bf16 / fp16: prefill_kernel.hpp's (heads of 80 and 96 on rows of 128)
  // and prefill256_kernel for heads of 256; fp32: prefill_f32_mfma_kernel
  // (v_mfma_f32_32x32x2_f32), heads of 64 and 128.
  if (dtype != PA_DTYPE_BF16 && dtype != PA_DTYPE_F16 && dtype != PA_DTYPE_F32) return false;
  const bool mfma_dim =
      head_dim == 64 || head_dim == 80 || head_dim == 96 || head_dim == 128 || head_dim == 256;
  if (dtype == PA_DTYPE_F32 ? head_dim != 64 && head_dim != 128 : !mfma_dim) return false;
  if (group < 1 || group > kMaxDecodeQueryGroup) return false;
  if (block_size <= 0 || (block_size & (block_size - 1)) != 0) return false;
  return true;
}

bool tree_fast_path_supported(int dtype, int head_dim, int group, int block_size) {
  if (dtype == PA_DTYPE_E4M3) return head_dim <= 128 && prefill_fast_path_supported(PA_DTYPE_BF16, head_dim, group, block_size);
  return prefill_fast_path_supported(dtype, head_dim, group, block_size);
}

bool prefill_append_supported(int dtype, int head_dim) {
  // Every fast-path kernel but the one for heads of 256.
  if (dtype == PA_DTYPE_F32) return head_dim == 64 || head_dim == 128;
  return (dtype == PA_DTYPE_BF16 || dtype == PA_DTYPE_F16) &&
         (head_dim == 64 || head_dim == 80 || head_dim == 96 || head_dim == 128);
}

bool prefill_codes_supported(int dtype, int head_dim) {
  // prefill_kernel.hpp's.
  return (dtype == PA_DTYPE_BF16 || dtype == PA_DTYPE_F16) && head_dim <= 128;
}

// Query tokens per work item: 128 rows over the heads of one workgroup (a
// sub-group of at most 8 when the group is larger).
int prefill_tile_for(int group) {
  return group > 0 ? kPrefillRows / (group / decode_sub_groups(group)) : kPrefillRows;
}

// Compute units of the current device (cached per device; 0 if unknown).
int device_compute_units() {
  constexpr int kMaxDevices = 64;
  static std::atomic<int> cached[kMaxDevices];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) return 0;
  int n = cached[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 0) n = 0;
    cached[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <typename T, int D, int DM, bool APPEND>
static hipError_t launch_prefill_d(const PrefillArgs& args, int group, int64_t num_items, hipStream_t s) {
  const int g = group / args.sub_groups;
  if (g < 1 || g > 8) return hipErrorNotSupported;
  PrefillArgs a = args;
  a.num_units = num_items * a.num_kv_heads * a.sub_groups;
  // Unit ranks are 32-bit and a workgroup's ranks reach about twice the count.
  if (a.num_units > (int64_t{1} << 30)) return hipErrorInvalidValue;
  // One workgroup per CU (the rings hold one per CU), each looping over its
  // share of the units; fewer units than CUs run one each.
  const int cus = device_compute_units();
  const int64_t wgs = cus > 0 ? std::min<int64_t>(a.num_units, cus) : a.num_units;
  const dim3 grid(static_cast<uint32_t>(wgs));
  if (a.key_scales != nullptr) {
    if constexpr (!APPEND)
      hipLaunchKernelGGL((prefill_kernel<T, D, DM, false, false, true>), grid, dim3(kPrefillThreads), 0, s, a);
    return APPEND ? hipErrorNotSupported : hipGetLastError();
  }
  // A copying wave's 16 rows of a stage share one block from blocks of 16
  // up; smaller blocks take the per-lane copy addresses (ids read per lane
  // from the ring), which beat one scalar base per copy with its id read
  // just before it.
  if ((1 << a.log2_block_size) >= kCopyRows)
    hipLaunchKernelGGL((prefill_kernel<T, D, DM, false, APPEND>), grid, dim3(kPrefillThreads), 0, s, a);
  else
    hipLaunchKernelGGL((prefill_kernel<T, D, DM, true, APPEND>), grid, dim3(kPrefillThreads), 0, s, a);
  return hipGetLastError();
}

template <typename T, int D, int DM>
static hipError_t launch_prefill_t(const PrefillArgs& a, int group, int64_t num_items, hipStream_t s) {
  return a.new_key != nullptr ? launch_prefill_d<T, D, DM, true>(a, group, num_items, s)
                              : launch_prefill_d<T, D, DM, false>(a, group, num_items, s);
}

hipError_t launch_prefill(const PrefillArgs& a, int dtype, int head_dim, int group,
                          int64_t num_items, hipStream_t stream) {
  if (num_items <= 0) return hipSuccess;
  if (dtype == PA_DTYPE_F32) return launch_prefill_f32(a, head_dim, group, num_items, stream);
  if (a.masks != nullptr)
    return a.key_scales != nullptr ? launch_prefill_tree(a, dtype, head_dim, group, num_items, stream)
                                   : launch_tree_attention(a, dtype, head_dim, group, num_items, stream);
  if (head_dim == 256)
    return a.new_key != nullptr ? hipErrorNotSupported : launch_prefill256(a, dtype, group, num_items, stream);
  if (a.window > 0) return launch_prefill_window(a, dtype, head_dim, group, num_items, stream);
  if (dtype == PA_DTYPE_BF16) {
    if (head_dim == 128) return launch_prefill_t<bf16_t, 128, 128>(a, group, num_items, stream);
    if (head_dim == 96) return launch_prefill_t<bf16_t, 128, 96>(a, group, num_items, stream);
    if (head_dim == 80) return launch_prefill_t<bf16_t, 128, 80>(a, group, num_items, stream);
    if (head_dim == 64) return launch_prefill_t<bf16_t, 64, 64>(a, group, num_items, stream);
  } else if (dtype == PA_DTYPE_F16) {
    if (head_dim == 128) return launch_prefill_t<f16_t, 128, 128>(a, group, num_items, stream);
    if (head_dim == 96) return launch_prefill_t<f16_t, 128, 96>(a, group, num_items, stream);
    if (head_dim == 80) return launch_prefill_t<f16_t, 128, 80>(a, group, num_items, stream);
    if (head_dim == 64) return launch_prefill_t<f16_t, 64, 64>(a, group, num_items, stream);
  }
  return hipErrorNotSupported;
}

}  // namespace pa
