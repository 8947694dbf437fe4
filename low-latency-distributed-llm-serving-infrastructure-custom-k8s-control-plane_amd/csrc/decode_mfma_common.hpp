// What the matrix-core decode kernels (decode_mfma.hip, decode8.hip) share.
#pragma once

#include "decode_common.hpp"

namespace pa {

typedef float f32x4m __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8m __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8m __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4m __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2m __attribute__((ext_vector_type(2)));

template <typename T>
__device__ __forceinline__ f32x4m mfma16(u32x4m a, u32x4m b, f32x4m c);
template <>
__device__ __forceinline__ f32x4m mfma16<bf16_t>(u32x4m a, u32x4m b, f32x4m c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8m, a), __builtin_bit_cast(bf16x8m, b), c,
                                                 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4m mfma16<f16_t>(u32x4m a, u32x4m b, f32x4m c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8m, a), __builtin_bit_cast(f16x8m, b), c, 0,
                                                0, 0);
}

// NT: streaming loads, for rows no other workgroup reads.
template <typename V, bool NT>
__device__ __forceinline__ V row_load(const void* p) {
  if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
  return *reinterpret_cast<const V*>(p);
}

// Workgroup -> (item, unit of KV heads, sub-group).  Ids are dealt to the XCDs
// round-robin: the members of a gang get ids that are equal modulo the XCD
// count and close together, gang after gang going to the next XCD (runs of
// 8 gangs, the last may be shorter), so that they share an XCD's L2.  A gang is
// an item's sub-groups of one unit (SHARED), which read the same rows, and with
// GANG_UNITS all of the item's units, whose parts of a row are lines apart or
// less.
struct DecodePlace {
  int64_t item;
  int unit, sg;
};
template <bool GANG_UNITS, bool SHARED>
__device__ __forceinline__ DecodePlace decode_place(const DecodeArgs& a, uint32_t units) {
  const uint32_t sub_groups = SHARED ? a.sub_groups : 1;
  uint32_t g_id = blockIdx.x, member = 0;
  if constexpr (GANG_UNITS || SHARED) {
    const uint32_t gang = (GANG_UNITS ? units : 1) * sub_groups;
    const uint32_t gangs = static_cast<uint32_t>(a.num_items) * (GANG_UNITS ? 1 : units);
    const uint32_t run = quotient(blockIdx.x, kXcds * gang, a.run_rcp);
    const uint32_t at_run = blockIdx.x - run * (kXcds * gang);
    const uint32_t width = min(static_cast<uint32_t>(kXcds), gangs - run * kXcds);
    member = width == kXcds ? at_run / kXcds : at_run / width;
    g_id = run * kXcds + (at_run - member * width);
  }
  DecodePlace p;
  if constexpr (GANG_UNITS) {
    p.item = g_id;
    p.unit = static_cast<int>(SHARED ? member / sub_groups : member);
    p.sg = SHARED ? static_cast<int>(member - p.unit * sub_groups) : 0;
  } else {
    p.item = quotient(g_id, units, a.unit_rcp);
    p.unit = static_cast<int>(g_id - static_cast<uint32_t>(p.item) * units);
    p.sg = SHARED ? static_cast<int>(member) : 0;
  }
  return p;
}

// The end of a workgroup: its waves' running maxima m (as scores), sums l (of the
// lane's tokens only) and accumulators (acc[b][i]: dim PE * (4c + i) + b of head
// r), HEADS KV heads' waves side by side, become output rows, or partials that
// the last of the sequence's workgroups merges.  s_wave: each wave's LDS, free
// by now but for its own reads.
template <typename T, int D, int DM, int HEADS, size_t BYTES>
__device__ __forceinline__ void combine_waves(const DecodeArgs& a, const DecodePlace& at, uint32_t units, int G, int seq,
                                              int part, int ctx, int n, int64_t qtok, float m, float l,
                                              const f32x4m (&acc)[D / 16], float (&s_m)[kDecodeWaves][kMfmaHeads],
                                              float (&s_l)[kDecodeWaves][kMfmaHeads],
                                              char (&s_wave)[kDecodeWaves][BYTES]) {
  constexpr int PE = D / 16;
  constexpr int kAccRow = D + 4;  // padded LDS row of one head's accumulators
  constexpr int kHeadWaves = kDecodeWaves / HEADS;
  static_assert(BYTES >= kMfmaHeads * kAccRow * 4, "a wave's accumulators fit");
  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int r = lane & 15;
  const int c = lane >> 4;
  l = sum_halves(sum_row_pairs(l));
  float* acc_row = reinterpret_cast<float*>(s_wave[wave]) + r * kAccRow + 4 * PE * c;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int b = 0; b < PE; b += 4)
      *reinterpret_cast<float4*>(acc_row + PE * i + b) =
          make_float4(acc[b][i], acc[b + 1][i], acc[b + 2][i], acc[b + 3][i]);
  if (lane < kMfmaHeads) {
    s_m[wave][lane] = m * a.scale_log2e;
    s_l[wave][lane] = l;
  }
  __syncthreads();

  const int hq = a.num_kv_heads * a.group;
  const int nparts = ctx <= a.partition ? 1 : (ctx + a.partition - 1) / a.partition;
  const int hu = at.unit * HEADS * a.group + at.sg * G;  // first query head of the workgroup
  float* pacc = a.part_acc + (at.item * hq + hu) * DM;
  T* out = reinterpret_cast<T*>(a.output) + (qtok * hq + hu) * DM;
  for (int i = tid; i < HEADS * G * DM; i += kDecodeThreads) {
    const int hg = i / DM;
    const int kv = HEADS == 1 ? 0 : HEADS == 2 ? hg >= G : hg / G;
    const int w0 = kv * kHeadWaves;  // the head's first wave
    const int g = hg - kv * G;
    const int e = g * kAccRow + (i - hg * DM);
    float mx = s_m[w0][g];
#pragma unroll
    for (int w = 1; w < kHeadWaves; ++w) mx = fmaxf(mx, s_m[w0 + w][g]);
    float o = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kHeadWaves; ++w) {
      const float f = fast_exp2(s_m[w0 + w][g] - mx);
      o = fmaf(reinterpret_cast<const float*>(s_wave[w0 + w])[e], f, o);
      sum = fmaf(s_l[w0 + w][g], f, sum);
    }
    if (nparts <= 1) {
      store_scalar<T>(out + i, sum != 0.f ? o / sum : 0.f);
    } else {
      store_device(pacc + i, o);
      if (i % DM == 0) {
        float* pml = a.part_ml + (at.item * hq + hu + hg) * 2;
        store_device(pml, mx);
        store_device(pml + 1, sum);
      }
    }
  }
  if (nparts > 1 && n > 0 && a.merge_state != nullptr && seq >= 0 && seq < a.num_seqs)
    merge_in_launch<T, DM, kMergeOutputs>(a, HEADS * G, part, at.item, ctx, nparts,
                                          (static_cast<int64_t>(seq) * units + at.unit) * a.sub_groups + at.sg, hu, hq,
                                          reinterpret_cast<T*>(a.output) + qtok * hq * DM);
}

}  // namespace pa
