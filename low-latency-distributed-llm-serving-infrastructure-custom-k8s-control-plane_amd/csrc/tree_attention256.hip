// Attention of trees of drafted tokens over the paged cache, 16-bit heads of 256,
// with gfx950 MFMA tiles.
//
// tree_attention.hip keeps 64 rows' queries and accumulators in a wave's registers
// and a ring of K and V for each wave in LDS; at 256 dims neither fits.  Here the
// four waves of a workgroup share the rings, as in prefill256.hip: a unit is (item,
// KV head, sub-group) with 128 query rows, node after node, wave w owns rows
// [32 w, 32 w + 32), and the context goes by in steps of 32 tokens.  (Waves without
// a live row only copy.)  The rings have four slots each of K and V, filled three
// steps ahead: K of step st+5 goes out in step st, when K of st+1 is in registers
// already, and V of st+3.  Items, masks, partial results and a probability's two terms
// as there.
//
// 16 trees of 9-17 nodes after 100-6000 tokens, 16/4 heads: 60 us, 3.4 TB/s (a unit's
// start, its steps' chain between barriers, and the join); 66 us while the compiler
// moved the accumulators at each step and waited for the query in the loop.  With a
// probability in one term 55-56 us, off 64 bits by 2.2e-3 (2-norm) where two terms are
// by 1.65e-3.
#include <type_traits>

#include "tree_common.hpp"

namespace pa {

namespace {

constexpr int kThreads = 256;
constexpr int kRows = 128;
constexpr int kTile = 32;        // context tokens per step
constexpr int kBufs = 4;         // ring slots
constexpr int kCopyRows = kTile / 4;

template <typename T>
__global__ __launch_bounds__(kThreads) void tree_attention256_kernel(PrefillArgs a) {
  static_assert(Elem<T>::kBytes == 2, "16-bit caches (bf16 or fp16)");
  constexpr int D = 256;
  constexpr int KS = D / 16;       // QK k-steps
  constexpr int DB = D / 32;       // output d blocks
  constexpr int CHUNKS = D / 8;    // 16-byte pieces per LDS row
  constexpr int ROW_BYTES = D * 2;
  constexpr int kRowsPerDma = kWave / CHUNKS;
  constexpr int kDmaPerWave = kCopyRows / kRowsPerDma;  // copies per tensor and step
  constexpr int kRegion = kTile * ROW_BYTES;
  constexpr int kVBase = kBufs * kRegion;
  constexpr int kPerQk = 16 / KS;  // probabilities per QK k-step
  static_assert(kDmaPerWave >= 1 && kPerQk >= 1, "D 64 to 256");

  __shared__ __attribute__((aligned(16))) char s_lds[2 * kBufs * kRegion];
  __shared__ int s_ids[kTreeIds];  // blocks of the run's columns, -1 outside the pool

  const int G = a.group / a.sub_groups;
  const int MTOK = kRows / G;
  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int hkv = a.num_kv_heads;
  const int units = hkv * a.sub_groups;
  const int item = static_cast<int>(blockIdx.x) / units;
  const int unit = static_cast<int>(blockIdx.x) - item * units;
  const int kvh = unit / a.sub_groups;
  const int h0 = kvh * a.group + (unit - kvh * a.sub_groups) * G;  // first query head
  TreeRun run;
  if (!run.load(a, item, MTOK)) return;
  const int log2_bs = a.log2_block_size;
  const int bs_mask = (1 << log2_bs) - 1;
  const uint32_t row_bytes = static_cast<uint32_t>(hkv) * ROW_BYTES;
  const uint32_t block_bytes = row_bytes << log2_bs;
  const bool row_ok = run.trow >= 0 && run.trow < a.num_table_rows;
  const int32_t* bt = row_ok ? a.block_tables + static_cast<int64_t>(run.trow) * a.block_table_stride : kNoBlockRow;
  global_i32* btg = (global_i32*)(bt);
  const int bt_stride = row_ok ? a.block_table_stride : 1;
  const char* kbase = reinterpret_cast<const char*>(a.key_cache) + kvh * ROW_BYTES;
  const char* vbase = reinterpret_cast<const char*>(a.value_cache) + kvh * ROW_BYTES;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(s_lds));
  const float scale = a.scale_log2e;

  run.plan(log2_bs, bt_stride);
  const int ntiles = run.ntiles;
  auto id_at = [&](int t, int p) { return s_ids[run.id_index(t, p, log2_bs)]; };
  auto entry = [&](int i) {
    const int c = run.column(i);
    const int b = c < bt_stride ? btg[c] : -1;
    return static_cast<uint32_t>(b) < static_cast<uint32_t>(a.total_blocks) ? b : -1;
  };

  // ---- the wave's rows ---------------------------------------------------------
  const int row = wave * 32 + (lane & 31);
  const int half = lane >> 5;
  const int tok = row / G;
  const int g = row - tok * G;
  const bool row_live = tok < run.ntok;
  const bool wave_live = wave * 32 < run.ntok * G;
  const int64_t node = static_cast<int64_t>(run.first) + run.tok0 + (row_live ? tok : 0);
  const int h = h0 + g;
  int first_id = tid < run.ncols ? entry(tid) : 0;
  uint4 qreg[KS];
  {
    const uint16_t* qrow = reinterpret_cast<const uint16_t*>(a.query) + node * a.q_token_stride +
                           static_cast<int64_t>(row_live ? h : h0) * a.q_head_stride;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      qreg[ks] = row_live ? ld16(qrow + ks * 16 + half * 8) : make_uint4(0, 0, 0, 0);
  }
  TreeRow mine;
  mine.load(a, run, tok);
  bool bad = false;  // a seen position's block is missing
  {
    auto stage = [&](int i, int b) {
      s_ids[i] = b;
      bad |= b < 0 && run.column_seen(i, log2_bs);
    };
    if (tid < run.ncols) stage(tid, first_id);
    for (int i = tid + kThreads; i < run.ncols; i += kThreads) stage(i, entry(i));
  }
  const bool bad_ids = __syncthreads_or(bad ? 1 : 0) != 0;
  __builtin_amdgcn_s_waitcnt(kWaitLoads);  // (the query and the masks, as in tree_attention.hip)

  // ---- copies: wave w copies rows [8 w, 8 w + 8) of a step ---------------------
  const int delta = lane / CHUNKS;
  uint32_t chunk_off[kDmaPerWave], row_off[kDmaPerWave];
#pragma unroll
  for (int j = 0; j < kDmaPerWave; ++j) {
    const int r = wave * kCopyRows + j * kRowsPerDma + delta;
    const int c = (lane % CHUNKS) ^ chunk_swizzle<CHUNKS>(r);
    chunk_off[j] = static_cast<uint32_t>(c * 16);
    row_off[j] = __umul24(static_cast<uint32_t>(j * kRowsPerDma + delta), row_bytes) + chunk_off[j];
  }
  const bool one_block = (1 << log2_bs) >= kCopyRows;
  // Rows past the readable context repeat its last one, and a missing block reads
  // block 0 (their scores are masked, the latter's V rows cleared).
  auto copy = [&](int t, uint32_t region, const char* base) {
    const int p0 = run.tile_at(t) + wave * kCopyRows;
    const uint32_t dst0 = lds0 + region + wave * kCopyRows * ROW_BYTES;
    if (one_block && p0 + kCopyRows - 1 <= run.kv_last) {
      const uint32_t b = max(__builtin_amdgcn_readfirstlane(id_at(t, p0)), 0);
      const char* src = base + (static_cast<uint64_t>(b) * block_bytes + static_cast<uint32_t>(p0 & bs_mask) * row_bytes);
#pragma unroll
      for (int j = 0; j < kDmaPerWave; ++j)
        dma16_s(dst0 + j * kRowsPerDma * ROW_BYTES, row_off[j], src);
    } else {
      int pos[kDmaPerWave], b[kDmaPerWave];
#pragma unroll
      for (int j = 0; j < kDmaPerWave; ++j) {
        pos[j] = min(p0 + j * kRowsPerDma + delta, run.kv_last);
        b[j] = max(id_at(t, pos[j]), 0);
      }
#pragma unroll
      for (int j = 0; j < kDmaPerWave; ++j)
        dma16(dst0 + j * kRowsPerDma * ROW_BYTES,
              base + (static_cast<uint64_t>(static_cast<uint32_t>(b[j])) * block_bytes +
                        (static_cast<uint32_t>(pos[j] & bs_mask) * row_bytes + chunk_off[j])));
    }
  };
  auto copy_k = [&](int t, int slot) { copy(t, slot * kRegion, kbase); };
  auto copy_v = [&](int t, int slot) { copy(t, kVBase + slot * kRegion, vbase); };

  // ---- LDS operands -------------------------------------------------------------
  const int k_row = lane & 31;
  int k_off[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int c = half + 2 * ks;  // (rows of 32 chunks: the swizzle permutes within 16)
    k_off[ks] = k_row * ROW_BYTES + ((c & ~15) + ((c & 15) ^ chunk_swizzle<CHUNKS>(k_row))) * 16;
  }
  const int li = lane & 15;
  int v_off[DB][2];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) {
      const int r = 4 * half + (li >> 2) + 8 * hi;
      const int col = 16 * ((lane >> 4) & 1) + 4 * (li & 3) + 32 * db;
      v_off[db][hi] = kVBase + r * ROW_BYTES + (((col >> 3) ^ chunk_swizzle<CHUNKS>(r)) * 16) + (col & 7) * 2;
    }
  auto read_k = [&](int slot, uint4* ka) {
    const char* buf = s_lds + slot * kRegion;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) ka[ks] = *reinterpret_cast<const uint4*>(buf + k_off[ks]);
  };
  auto read_vt = [&](int slot, int kk, int db) {
    const char* base = s_lds + slot * kRegion + kk * 16 * ROW_BYTES;
    const uint2 lo = lds_read_tr16(reinterpret_cast<const uint16_t*>(base + v_off[db][0]));
    const uint2 hi = lds_read_tr16(reinterpret_cast<const uint16_t*>(base + v_off[db][1]));
    return make_uint4(lo.x, lo.y, hi.x, hi.y);
  };

  // ---- masks ------------------------------------------------------------------
  auto mask_tile = [&](int t, f32x16& s) {
    mine.mask(run, a.sinks, t, half, s);
    if (bad_ids) {
      const uint32_t gone = static_cast<uint32_t>(__ballot(id_at(t, min(run.tile_at(t) + (lane & 31), run.kv_last)) < 0)) >>
                            (4 * half);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if ((gone >> (8 * (i >> 2) + (i & 3))) & 1u) s[i] = -INFINITY;
    }
  };
  auto clear_v = [&](int t, int slot) {
    const int p = run.tile_at(t) + (lane & 31);
    if (run.hidden(p) || (bad_ids && id_at(t, min(p, run.kv_last)) < 0)) {
      char* r = s_lds + kVBase + slot * kRegion + (lane & 31) * ROW_BYTES + half * (ROW_BYTES / 2);
#pragma unroll 1
      for (int i = 0; i < ROW_BYTES / 32; ++i) st16(r + 16 * i, make_uint4(0, 0, 0, 0));
    }
  };
  f32x16 acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[db][i] = 0.f;
  float m = kScoreFloor, l = 0.f;  // l: this lane's half of the row sum
  auto rescale = [&](float tmax) {
    const bool grow = (tmax - m) * scale > kLazyRescale;
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
      const float m_new = grow ? tmax : m;
      const float alpha = fast_exp2((m - m_new) * scale);
      l *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        in_matrix_registers(acc[db]);
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[db][i] *= alpha;
        in_matrix_registers(acc[db]);
      }
      m = m_new;
    }
  };

  // ---- prologue: K of steps 0-3 and V of 0-2 in flight, K 0 and 1 awaited -------
  f32x16 s0, s1;
  uint4 ka[KS];
  {
    copy_k(0, 0);
    if (ntiles > 1) copy_k(1, 1);
    copy_v(0, 0);
    if (ntiles > 2) copy_k(2, 2);
    if (ntiles > 1) copy_v(1, 1);
    if (ntiles > 3) copy_k(3, 3);
    if (ntiles > 2) copy_v(2, 2);
    wait_vmcnt_at_most<5 * kDmaPerWave>(kDmaPerWave * (1 + 2 * min(max(ntiles - 2, 0), 1) +
                                                       min(max(ntiles - 1, 0), 1) + min(max(ntiles - 3, 0), 1)));
    stage_barrier();
#pragma unroll
    for (int i = 0; i < 16; ++i) s0[i] = 0.f;
    if (wave_live) {
      read_k(0, ka);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s0 = mfma32<T>(ka[ks], qreg[ks], s0);
      read_k(1, ka);
      mask_tile(0, s0);
      rescale(tree_tile_max(s0));
    }
    // K 0 and 1 are read, V 0 and K 2 have landed before step 0.
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    wait_vmcnt_at_most<3 * kDmaPerWave>(kDmaPerWave * (min(max(ntiles - 1, 0), 1) + min(max(ntiles - 3, 0), 1) +
                                                       min(max(ntiles - 2, 0), 1)));
    stage_barrier();
    if (ntiles > 4) copy_k(4, 0);
  }

  auto step = [&](int st, f32x16& s_cur, f32x16& s_nxt, auto masked, auto slot_c) {
    constexpr bool MASKED = decltype(masked)::value;
    constexpr int SLOT = decltype(slot_c)::value;
    if (st + 5 < ntiles) copy_k(st + 5, (SLOT + 1) & (kBufs - 1));
    if (st + 3 < ntiles) copy_v(st + 3, (SLOT + 3) & (kBufs - 1));
    if (wave_live) {
      if (MASKED && (bad_ids || run.has_hole(st))) clear_v(st, SLOT);
      // ---- A: S_next = K_next Q^T | P = exp2(S - m)
      const float msc = m * scale;
      f32x16 sn;
#pragma unroll
      for (int i = 0; i < 16; ++i) sn[i] = 0.f;
      uint4 pb[2], rest[2];
      float rsum0 = 0.f, rsum1 = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        sn = mfma32<T>(ka[ks], qreg[ks], sn);
#pragma unroll
        for (int j = ks * kPerQk; j < (ks + 1) * kPerQk; ++j) s_cur[j] = fast_exp2(fmaf(s_cur[j], scale, -msc));
        if (((ks + 1) * kPerQk) % 8 == 0) {
          const int c = (ks + 1) * kPerQk / 8 - 1;
          split_weights<T>(s_cur, c, pb[c], rest[c], rsum0, rsum1);
        }
      }
      // ---- B: O^T += V^T P^T | row maxima of S_next | K reads of step st+2
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          const uint4 v = read_vt(SLOT, kk, db);
          acc[db] = mfma32<T>(v, pb[kk], acc[db]);
          acc[db] = mfma32<T>(v, rest[kk], acc[db]);
        }
      read_k((SLOT + 2) & (kBufs - 1), ka);
      if constexpr (MASKED) mask_tile(st + 1, sn);
      l += rsum0 + rsum1;
      const float tmax = tree_tile_max(sn);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kSchedValu, 10 * 8 / KS, 0);
      }
#pragma unroll
      for (int i = 0; i < 2 * DB; ++i) {
        __builtin_amdgcn_sched_group_barrier(kSchedDsRead, 2, 0);
        __builtin_amdgcn_sched_group_barrier(kSchedMfma, 2, 0);
        __builtin_amdgcn_sched_group_barrier(kSchedDsRead, (KS + 2 * DB - 1) / (2 * DB), 0);
        __builtin_amdgcn_sched_group_barrier(kSchedValu, 2, 0);
      }
      rescale(tmax);
      s_nxt = sn;
    }
    // K of step st+3 and V of st+1 have landed before the barrier; what this step
    // and the last one issued may stay in flight (copies complete in order).
    const int n = kDmaPerWave * ((st + 4 < ntiles ? 1 : 0) + (st + 5 < ntiles ? 1 : 0) + (st + 2 < ntiles ? 1 : 0) +
                                 (st + 3 < ntiles ? 1 : 0));
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    wait_vmcnt_at_most<4 * kDmaPerWave>(n);
    stage_barrier();
  };

  using U = std::false_type;
  using M = std::true_type;
  using S0 = std::integral_constant<int, 0>;
  using S1 = std::integral_constant<int, 1>;
  using S2 = std::integral_constant<int, 2>;
  using S3 = std::integral_constant<int, 3>;
  // Steps whose next tokens every row sees whole: from the last row's window on, to
  // the tree.
  const int from = run.from(a.window), to = run.to();
  const int n_main = bad_ids ? 0 : min(max(to - 1, 0), ntiles - 1);
  int st = 0;
  for (; st < from && st + 3 < ntiles; st += 4) {
    step(st, s0, s1, M{}, S0{});
    step(st + 1, s1, s0, M{}, S1{});
    step(st + 2, s0, s1, M{}, S2{});
    step(st + 3, s1, s0, M{}, S3{});
  }
  for (; st + 3 < n_main; st += 4) {
    step(st, s0, s1, U{}, S0{});
    step(st + 1, s1, s0, U{}, S1{});
    step(st + 2, s0, s1, U{}, S2{});
    step(st + 3, s1, s0, U{}, S3{});
  }
  while (st < ntiles) {
    step(st, s0, s1, M{}, S0{});
    if (++st == ntiles) break;
    step(st, s1, s0, M{}, S1{});
    if (++st == ntiles) break;
    step(st, s0, s1, M{}, S2{});
    if (++st == ntiles) break;
    step(st, s1, s0, M{}, S3{});
    ++st;
  }
  l += __shfl_xor(l, 32, kWave);
  if (!row_live) return;
  const int64_t hq = static_cast<int64_t>(hkv) * a.group;
  if (run.part_row >= 0) {
    // One of a tile's runs: the sums as they are, for merge_tree_kernel.
    const int64_t prow = (static_cast<int64_t>(run.part_row) + tok) * hq + h;
    float* dst = a.part_acc + prow * D;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const int d = db * 32 + 8 * q4 + 4 * half;
        *reinterpret_cast<float4*>(dst + d) =
              make_float4(acc[db][4 * q4 + 0], acc[db][4 * q4 + 1], acc[db][4 * q4 + 2], acc[db][4 * q4 + 3]);
      }
    if (half == 0) *reinterpret_cast<float2*>(a.part_ml + prow * 2) = make_float2(m * scale, l);
    return;
  }
  const float inv = l > 0.f ? 1.f / l : l;  // (zero for a row that sees nothing; a NaN stays)
  uint16_t* orow = reinterpret_cast<uint16_t*>(a.output) + (node * hq + h) * static_cast<int64_t>(D);
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      const int d = db * 32 + 8 * q4 + 4 * half;
      uint2 w;
      w.x = pack_half2<T>(acc[db][4 * q4 + 0] * inv, acc[db][4 * q4 + 1] * inv);
      w.y = pack_half2<T>(acc[db][4 * q4 + 2] * inv, acc[db][4 * q4 + 3] * inv);
      *reinterpret_cast<uint2*>(orow + d) = w;
    }
}

}  // namespace

hipError_t launch_tree_attention256(const PrefillArgs& a, int dtype, int group, int64_t num_items, hipStream_t stream) {
  const int g = group / a.sub_groups;
  const int64_t units = num_items * a.num_kv_heads * a.sub_groups;
  if (g < 1 || g > 8 || units > 0x7fffffff) return hipErrorNotSupported;
  const dim3 grid(static_cast<uint32_t>(units));
  if (dtype == PA_DTYPE_BF16)
    hipLaunchKernelGGL(tree_attention256_kernel<bf16_t>, grid, dim3(kThreads), 0, stream, a);
  else if (dtype == PA_DTYPE_F16)
    hipLaunchKernelGGL(tree_attention256_kernel<f16_t>, grid, dim3(kThreads), 0, stream, a);
  else
    return hipErrorNotSupported;
  return hipGetLastError();
}

}  // namespace pa
