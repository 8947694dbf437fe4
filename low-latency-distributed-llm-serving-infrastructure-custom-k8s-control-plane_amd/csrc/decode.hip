// Paged-attention decode for gfx950 on the vector units: one workgroup per
// (sequence, context partition of up to 4096 tokens, KV head), split-K merge
// after.  fp32 caches and 16-bit heads of 256 run here; 16-bit heads of 64 to
// 128 run on the matrix cores (decode_mfma.hip).  The kernel itself: decode_kernel.hpp.
//
// The workgroup (4 waves) serves the G = H_q / H_kv query heads that share
// one KV head, so every K/V row of the partition is read from HBM once
// (groups above 8 run as sub-groups of at most 8 on SHARED instances, whose
// re-reads are ordered to meet in one XCD's L2).  Heads of 64, 128 and 256
// have their own instances; heads of 80 and 96 run those of 128 with the
// pieces past the head masked (DM below).
// The partition is cut into 32-token tiles (16 for groups above 4 and for
// 512-byte rows) dealt round-robin to the waves;
// each wave runs flash-style online softmax over its tiles with no
// workgroup barrier inside the loop:
//
//  K (QK layout)  a "row group" of kL lanes holds one token's K row, each
//                 lane two 16-byte pieces (the group's loads cover the row
//                 contiguously); a wave covers 64 / kL tokens per load.
//                 Dots with the G query slices use v_dot2_f32_bf16 /
//                 v_dot2_f32_f16 (16-bit types) and a DPP butterfly sums
//                 each group; groups of more than 4 on fp32 heads of 64 (row
//                 groups of 8 lanes) use a reduce-scatter instead, after
//                 which each lane holds one head's scores (qk_softmax_rs).
//  V (PV layout)  one wave load covers one V row (4 bytes per lane of 256-byte
//                 rows, 8 of 512), so the row address of a load is
//                 wave-uniform and is formed in scalar registers from the
//                 block id fetched with v_readlane.  Every lane owns a fixed
//                 slice of the head dimension for all G heads.
//  softmax        per tile: wave-wide max per head (DPP + shuffles), rescale
//                 of the running sum / accumulator only when the max moved,
//                 p = exp2(s - max) staged in LDS.  For bf16/fp16 the p of
//                 two tokens are packed as a pair of the cache type and the
//                 PV product uses v_dot2 on the matching V pair (one v_perm_b32 per
//                 two elements); fp32 keeps fp32 FMAs throughout.
//
// At the end the four waves combine (max, sum, acc) through LDS.  A sequence
// whose context fits one partition gets its normalised output directly;
// otherwise the partials go to the workspace and decode_merge_kernel
// combines them.
//
// The reference computes the same quantity with its CPU loop nest
// (csrc/src/paged_kernels.cpp:49-104) over a flat gather list and dense mask.
#include "decode_kernel.hpp"

namespace pa {

// Combines the split-K partials (max, sum, unnormalised acc) of one
// multi-partition sequence for the G heads of one KV head.  One workgroup
// per (entry of the merge list, KV head, 256 of the G*D outputs); an entry,
// written by pa_pack, is (first full-partition item, number of full
// partitions, sequence, item of the partial last partition or -1): the full
// partitions of a sequence are contiguous items, its partial one sits among
// the short work at the end.  Every thread owns one output (merge_partials):
// no LDS and no barrier, so the only dependent global round trips are the
// entry and then the partials.  (With several outputs per thread their
// round trips queued one behind the other: eight heads of 128 at partition
// 2048 took 19 us.)
template <typename T>
__global__ __launch_bounds__(kDecodeThreads) void decode_merge_kernel(DecodeArgs a, int G, int D) {
  const int hkv = a.num_kv_heads;
  const int64_t m = blockIdx.x / hkv;
  const int kvh = static_cast<int>(blockIdx.x - m * hkv);
  const int4 e = reinterpret_cast<const int4*>(a.merge_items)[m];
  const int64_t first = e.x;
  const int nfull = static_cast<int>(min(static_cast<int64_t>(e.y), a.num_items - first));
  const bool has_rem = e.w >= 0 && e.w < a.num_items;
  const int nparts = nfull + (has_rem ? 1 : 0);
  if (nfull < 0 || nparts <= 1) return;
  const int hq = hkv * G;
  T* out = reinterpret_cast<T*>(a.output) + (a.cu_seqlens[e.z] * hq + kvh * G) * D;
  const int i = static_cast<int>(blockIdx.y) * kDecodeThreads + static_cast<int>(threadIdx.x);
  if (i >= G * D) return;
  const int h = kvh * G + i / D;
  merge_partials<T, 1>(a.part_ml + 2 * h, a.part_acc + static_cast<int64_t>(kvh) * G * D + i, 0,
                       2 * static_cast<int64_t>(hq), static_cast<int64_t>(hq) * D, first, nfull, has_rem ? e.w : -1,
                       nparts, out + i);
}

// ---- host-side dispatch ------------------------------------------------

// The merge phase, unless the partition launch merged in place (merge
// records given): all a.group query heads of a KV head merge in one
// workgroup row; out_d: elements per query head in memory.
template <typename T>
static hipError_t launch_merge_t(const DecodeArgs& a, int out_d, int phases, hipStream_t stream) {
  const int64_t grid = a.num_merge * a.num_kv_heads;
  if (!(phases & PA_DECODE_PHASE_MERGE) || grid <= 0) return hipSuccess;
  if ((phases & PA_DECODE_PHASE_PARTITIONS) && a.merge_state != nullptr) return hipSuccess;
  const int chunks = (a.group * out_d + kDecodeThreads - 1) / kDecodeThreads;
  hipLaunchKernelGGL((decode_merge_kernel<T>), dim3(static_cast<uint32_t>(grid), static_cast<uint32_t>(chunks)),
                     dim3(kDecodeThreads), 0, stream, a, a.group, out_d);
  return hipGetLastError();
}

static hipError_t launch_merge(const DecodeArgs& a, int dtype, int out_d, int phases, hipStream_t stream) {
  return dtype == PA_DTYPE_BF16  ? launch_merge_t<bf16_t>(a, out_d, phases, stream)
         : dtype == PA_DTYPE_F16 ? launch_merge_t<f16_t>(a, out_d, phases, stream)
                                 : launch_merge_t<float>(a, out_d, phases, stream);
}

// Launches both phases of one kernel instance.  D, G: the kernel's head dim
// and group.
struct LaunchOp {
  const DecodeArgs& a;
  int64_t num_items;
  int phases;
  hipStream_t stream;
  template <typename T, int D, int G, bool SHARED, int DM>
  hipError_t run() const {
    const int64_t grid = num_items * a.num_kv_heads * a.sub_groups;
    if (phases & PA_DECODE_PHASE_PARTITIONS) {
      hipLaunchKernelGGL((decode_partition_kernel<T, D, G, SHARED, DM, false>), dim3(static_cast<uint32_t>(grid)),
                         dim3(kDecodeThreads), 0, stream, a);
      const hipError_t err = hipGetLastError();
      if (err != hipSuccess) return err;
    }
    return launch_merge_t<T>(a, DM, phases, stream);
  }
};

// Resident partition workgroups per CU of one kernel instance.
struct OccupancyOp {
  int* per_cu;
  template <typename T, int D, int G, bool SHARED, int DM>
  hipError_t run() const {
    return hipOccupancyMaxActiveBlocksPerMultiprocessor(per_cu, decode_partition_kernel<T, D, G, SHARED, DM, false>,
                                                        kDecodeThreads, 0);
  }
};

int decode_unit_heads(int dtype, int head_dim, int num_kv_heads, int group) {
  return decode_uses_mfma(dtype, head_dim) && head_dim % 64 == 0 && num_kv_heads % 2 == 0 && group >= 1 && group <= 4
             ? 2
             : 1;
}

int decode_sub_groups(int group) {
  // The fewest equal sub-groups of at most kMaxDecodeGroup query heads.
  int n = (group + kMaxDecodeGroup - 1) / kMaxDecodeGroup;
  while (n < group && group % n != 0) ++n;
  return n > 0 ? n : 1;
}

int decode_workgroups_per_head(int dtype, int head_dim, int group) {
  if (!decode_uses_mfma(dtype, head_dim)) return decode_sub_groups(group);
  int n = (group + kMfmaHeads - 1) / kMfmaHeads;
  while (n < group && group % n != 0) ++n;
  return n > 0 ? n : 1;
}

bool decode_fast_path_supported(int dtype, int head_dim, int group, int block_size,
                                int partition) {
  if (dtype == PA_DTYPE_E4M3) {
    // (two tokens of a V operand's pair share a block, hence a scale)
    if (!decode_uses_mfma(dtype, head_dim) || block_size < 2) return false;
  } else if (dtype != PA_DTYPE_F32 && dtype != PA_DTYPE_BF16 && dtype != PA_DTYPE_F16) {
    return false;
  }
  // Rows of up to 512 bytes: heads of 64 and 128, and of 256 in 16-bit types;
  // heads of 80 and 96 on the lane layout of 128.
  const bool wide16 = dtype != PA_DTYPE_F32 && dtype != PA_DTYPE_E4M3 && head_dim == 256;
  if (head_dim != 64 && head_dim != 128 && head_dim != 80 && head_dim != 96 && !wide16) return false;
  if (group < 1 || group > kMaxDecodeQueryGroup) return false;
  if (block_size <= 0 || (block_size & (block_size - 1)) != 0) return false;
  if (partition <= 0 || partition > kMaxPartition || partition % 32 != 0) return false;
  return true;
}

hipError_t launch_decode(const DecodeArgs& a, int dtype, int head_dim, int group,
                         int64_t num_items, int phases, hipStream_t stream) {
  if (num_items <= 0) return hipSuccess;
  if (decode_uses_mfma(dtype, head_dim)) {
    if (phases & PA_DECODE_PHASE_PARTITIONS) {
      const int heads = decode_unit_heads(dtype, head_dim, a.num_kv_heads, group);
      const hipError_t err = a.key_scales != nullptr
                                 ? launch_decode8(a, dtype, head_dim, heads, num_items, stream)
                                 : launch_decode_mfma(a, dtype, head_dim, heads, num_items, stream);
      if (err != hipSuccess) return err;
    }
    return launch_merge(a, dtype, head_dim, phases, stream);
  }
  if (a.window > 0) return launch_decode_window(a, dtype, head_dim, group, num_items, stream);
  return visit_decode(dtype, head_dim, group, LaunchOp{a, num_items, phases, stream});
}

hipError_t decode_workgroups_per_cu(int dtype, int head_dim, int num_kv_heads, int group, int* per_cu) {
  *per_cu = 0;
  if (!decode_uses_mfma(dtype, head_dim)) return visit_decode(dtype, head_dim, group, OccupancyOp{per_cu});
  const int wgs = decode_workgroups_per_head(dtype, head_dim, group);
  const int heads = decode_unit_heads(dtype, head_dim, num_kv_heads, group);
  const hipError_t err = dtype == PA_DTYPE_E4M3
                             ? decode8_workgroups_per_cu(head_dim, wgs > 1, heads, per_cu)
                             : decode_mfma_workgroups_per_cu(dtype, head_dim, wgs > 1, heads, per_cu);
  *per_cu *= decode_sub_groups(group) / wgs;
  return err;
}

}  // namespace pa
