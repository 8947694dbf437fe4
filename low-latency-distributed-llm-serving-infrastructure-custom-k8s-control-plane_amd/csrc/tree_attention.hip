// Attention of trees of drafted tokens over the paged cache, 16-bit rows of 64 to
// 128, with gfx950 MFMA tiles.
//
// A unit of work is (item, KV head, sub-group); an item (pa_pack_tree) is a run of
// stages of one tile of a sequence's nodes, and its record holds all that a unit
// has to know of its sequence.  The tile has 64 query rows, node after node, the
// query heads of the KV head (or sub-group) side by side: two blocks of 32, of which
// a small tree fills one.  A workgroup has two or four waves (kWaves); wave w takes
// tiles w, w + kWaves, ... of 32 context tokens of the run for all rows, with
// flash-style online softmax in fp32, and keeps its own K and V in its own part of
// LDS, two tiles deep: no wave waits for another until they are joined at the end.
//   S^T[kv][row] = sum_d K[kv][d] Q[row][d]
//   O^T[d][row] += sum_kv V^T[d][kv] P^T[kv][row]     (v_mfma_f32_32x32x16)
// with the layouts, the swizzled LDS rows, the direct global -> LDS copies, the
// transpose read of V and the lazy rescale of prefill_kernel.hpp.  An operand of K or V
// read from LDS serves both blocks of rows, whose products and softmax do not
// depend on each other.
//
// What bounds it is the cache's bytes, read once for a tile's rows (32 trees of 9-17
// nodes after 100-8000 tokens, 32/8 heads of 128: 114 us and 7.5 for the join, 4.7 TB/s;
// 8 of 64 nodes after 1000-4000, 32/32 heads: 77 us, 4.5 TB/s); for trees whose tiles
// share a short context the one wave a SIMD, whose products and softmax follow each
// other (2 of 40-60 nodes under a window of 8192: 38 and 4.5 us); for short runs the
// chain of round trips at a unit's start (record; block ids, query and masks; K and V:
// one of 26 nodes after 3000, 15 and 4 us).  With one term a probability (below) the
// causal prefill's tiles, shared by eight waves, took 145, 95, and 28 us where this took
// 118, 73 and 18; V's operands read behind the softmax, and the accumulators copied out
// of the matrix registers at each tile: 133, 91 and 21 us.
//
// A probability goes into the product as two terms of the type (split_weights()), as the
// decode's does: a node that verifies a token answers as the decode of that token would,
// off 64 bits by the rounding of the result alone.  One term -> two, bf16, 2-norm and
// time: 32 trees 2.2e-3 -> 1.7e-3 and 117 -> 121.6 us; 2 under a window of 8192 2.3e-3
// -> 1.7e-3 and 37.3 -> 42.5; one of 26 nodes 2.1e-3 -> 1.65e-3 and 18.0 -> 18.7; fp16, 8
// of 64 nodes 2.9e-4 -> 2.1e-4 and 71 -> 76.
//
// Masks: a node sees the context before the tree (under a window, from where its
// own position's window starts, and the sinks) and of the tree what its mask's
// bits say.  Tiles that every row sees whole run without masks; the others are
// those at the edges.  V rows that no row of the unit sees, or of blocks outside
// the pool, become zeros in LDS, as a NaN or an infinity outlives a weight of zero.
#include <type_traits>

#include "tree_common.hpp"

namespace pa {

namespace {

constexpr int kRows = kTreeRows;
constexpr int kSlots = 2;  // tiles of K and of V a wave holds

// D: the head dim of the LDS rows and MFMA tiles, DM in memory (80 and 96 run on
// rows of 128 whose pieces past DM are zero).
template <typename T, int D, int DM, int kWaves>
__global__ __launch_bounds__(kWaves * kWave) __attribute__((amdgpu_waves_per_eu(D > 64 ? 1 : 2))) void
tree_attention_kernel(PrefillArgs a) {
  static_assert(Elem<T>::kBytes == 2, "16-bit caches (bf16 or fp16)");
  constexpr int kThreads = kWaves * kWave;
  constexpr bool MASKD = DM < D;
  constexpr int KS = D / 16;       // QK k-steps
  constexpr int DB = D / 32;       // output d blocks
  constexpr int CHUNKS = D / 8;    // 16-byte pieces per LDS row
  constexpr int ROW_BYTES = D * 2;
  constexpr int MEM_ROW = DM * 2;
  constexpr int kRegion = kTreeKvTile * ROW_BYTES;
  constexpr int kCopies = kRegion / (kWave * 16);  // of a tile of one tensor
  constexpr int kRowsPerDma = kWave / CHUNKS;
  constexpr int kWaveBytes = 2 * kSlots * kRegion;  // K slots, then V slots
  constexpr int kVBase = kSlots * kRegion;
  constexpr int kPieces = 4 * DB;  // 16-byte pieces of a lane's accumulator of a block
  static_assert(kWaveBytes >= 2 * kPieces * kWave * 16, "the accumulators fit the rings");

  __shared__ __attribute__((aligned(16))) char s_lds[kWaves * kWaveBytes];
  __shared__ int s_ids[kTreeIds];  // blocks of the run's columns, -1 outside the pool
  __shared__ float2 s_ml[kWaves][kRows];

  const int G = a.group / a.sub_groups;
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
  if (!run.load(a, item, kRows / G)) return;
  const int log2_bs = a.log2_block_size;
  const int bs_mask = (1 << log2_bs) - 1;
  const uint32_t row_bytes = static_cast<uint32_t>(hkv) * MEM_ROW;
  const uint32_t block_bytes = row_bytes << log2_bs;
  const bool row_ok = run.trow >= 0 && run.trow < a.num_table_rows;
  const int32_t* bt = row_ok ? a.block_tables + static_cast<int64_t>(run.trow) * a.block_table_stride : kNoBlockRow;
  global_i32* btg = (global_i32*)(bt);
  const int bt_stride = row_ok ? a.block_table_stride : 1;
  const char* kbase = reinterpret_cast<const char*>(a.key_cache) + kvh * MEM_ROW;
  const char* vbase = reinterpret_cast<const char*>(a.value_cache) + kvh * MEM_ROW;
  const float scale = a.scale_log2e;
  run.plan(log2_bs, bt_stride);
  auto id_at = [&](int t, int p) { return s_ids[run.id_index(t, p, log2_bs)]; };
  auto entry = [&](int i) {
    const int c = run.column(i);
    const int b = c < bt_stride ? btg[c] : -1;
    return static_cast<uint32_t>(b) < static_cast<uint32_t>(a.total_blocks) ? b : -1;
  };
  const int half = lane >> 5;
  const int li = lane & 15;
  const int64_t hq = static_cast<int64_t>(hkv) * a.group;

  // ---- copies: a wave's own tiles ------------------------------------------------
  char* const ring = s_lds + wave * kWaveBytes;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(s_lds)) + wave * kWaveBytes;
  const int delta = lane / CHUNKS;
  // Copies of 16 rows; the swizzle repeats every 16.
  constexpr int kHalfCopies = kCopies / 2;
  uint32_t chunk_off[kHalfCopies], row_off[kHalfCopies];
#pragma unroll
  for (int j = 0; j < kHalfCopies; ++j) {
    const int r = j * kRowsPerDma + delta;
    chunk_off[j] = static_cast<uint32_t>(((lane % CHUNKS) ^ chunk_swizzle<CHUNKS>(r)) * 16);
    row_off[j] = __umul24(static_cast<uint32_t>(r), row_bytes) + chunk_off[j];
  }
  // Whether no other workgroup reads the rows, nor part of their 128-byte lines.
  const bool alone = a.sub_groups == 1 && run.count <= kRows / G && MEM_ROW % 128 == 0;
  auto piece_in = [&](int j) { return !MASKD || chunk_off[j] < MEM_ROW; };
  // Where a tile's rows lie: offsets of its two halves from the tensors' bases when
  // each is within a block and all its rows are the context's; else row by row.
  struct Place {
    uint64_t at[2];
    int p0;
    bool whole;
  };
  auto place_of = [&](int t) {
    Place w;
    w.p0 = run.tile_at(t);
    w.whole = log2_bs >= 4 && w.p0 + kTreeKvTile - 1 <= run.kv_last;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int p = w.p0 + 16 * s;
      const uint32_t b = max(__builtin_amdgcn_readfirstlane(id_at(t, p)), 0);
      w.at[s] = static_cast<uint64_t>(b) * block_bytes + static_cast<uint32_t>(p & bs_mask) * row_bytes;
    }
    return w;
  };
  // Rows past the readable context repeat its last one, and a missing block reads
  // block 0 (their scores are masked, the latter's V rows cleared).
  auto copy = [&](int t, const Place& w, uint32_t region, const char* base) {
    const uint32_t dst0 = lds0 + region;
    if (w.whole) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const char* src = base + w.at[s];
        if (alone) {
#pragma unroll
          for (int j = 0; j < kHalfCopies; ++j)
            if (piece_in(j)) dma16_s_nt(dst0 + (s * kHalfCopies + j) * (kWave * 16), row_off[j], src);
        } else {
#pragma unroll
          for (int j = 0; j < kHalfCopies; ++j)
            if (piece_in(j)) dma16_s(dst0 + (s * kHalfCopies + j) * (kWave * 16), row_off[j], src);
        }
      }
    } else {
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int j = 0; j < kHalfCopies; ++j) {
          const int pos = min(w.p0 + 16 * s + j * kRowsPerDma + delta, run.kv_last);
          const uint32_t b = max(id_at(t, pos), 0);
          if (piece_in(j))
            dma16(dst0 + (s * kHalfCopies + j) * (kWave * 16),
                  base + (static_cast<uint64_t>(b) * block_bytes +
                          (static_cast<uint32_t>(pos & bs_mask) * row_bytes + chunk_off[j])));
        }
    }
  };

  // ---- LDS operands -------------------------------------------------------------
  const int k_row = lane & 31;
  int k_off[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
    k_off[ks] = k_row * ROW_BYTES + (((half + 2 * ks) ^ chunk_swizzle<CHUNKS>(k_row)) * 16);
  int v_off[DB][2];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) {
      const int r = 4 * half + (li >> 2) + 8 * hi;
      const int col = 16 * ((lane >> 4) & 1) + 4 * (li & 3) + 32 * db;
      v_off[db][hi] = kVBase + r * ROW_BYTES + (((col >> 3) ^ chunk_swizzle<CHUNKS>(r)) * 16) + (col & 7) * 2;
    }

  // The unit with its live blocks of rows, NB of two.
  auto attend = [&](auto blocks) {
    constexpr int NB = decltype(blocks)::value;
    int first_id = tid < run.ncols ? entry(tid) : 0;
    uint4 qreg[NB][KS];
    TreeRow mine[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int row = b * 32 + (lane & 31);
      const int tok = row / G;
      const bool live = tok < run.ntok;
      const int64_t node = static_cast<int64_t>(run.first) + run.tok0 + (live ? tok : 0);
      const uint16_t* qrow = reinterpret_cast<const uint16_t*>(a.query) + node * a.q_token_stride +
                             static_cast<int64_t>(h0 + (live ? row - tok * G : 0)) * a.q_head_stride;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        qreg[b][ks] = live && (!MASKD || ks * 16 + half * 8 < DM) ? ld16(qrow + ks * 16 + half * 8)
                                                                 : make_uint4(0, 0, 0, 0);
      mine[b].load(a, run, tok);
    }
    bool bad = false;  // a seen position's block is missing
    auto stage = [&](int i, int b) {
      s_ids[i] = b;
      bad |= b < 0 && run.column_seen(i, log2_bs);
    };
    if (tid < run.ncols) stage(tid, first_id);
    for (int i = tid + kThreads; i < run.ncols; i += kThreads) stage(i, entry(i));
    if constexpr (MASKD) {
      // Row pieces past the head are never copied: zero them before any copy lands.
      for (int i = tid; i < kWaves * kWaveBytes / 16; i += kThreads) st16(s_lds + 16 * i, make_uint4(0, 0, 0, 0));
    }
    const bool bad_ids = __syncthreads_or(bad ? 1 : 0) != 0;
    // The query and the masks arrive before the copies go out: a wait for them in the
    // loop would be one for the copies behind them (the compiler sees this wait).
    __builtin_amdgcn_s_waitcnt(kWaitLoads);

    f32x16 acc[NB][DB];
    float m[NB], l[NB];  // l: this lane's half of the row sum
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      m[b] = kScoreFloor;
      l[b] = 0.f;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[b][db][i] = 0.f;
    }
    const int n = (run.ntiles - wave + kWaves - 1) / kWaves;  // tiles of this wave
    const int from = run.from(a.window), to = run.to();
    if (n > 0) {
      const Place w = place_of(wave);
      copy(wave, w, 0, kbase);
      copy(wave, w, kVBase, vbase);
    }
    if (n > 1) {
      const Place w = place_of(wave + kWaves);
      copy(wave + kWaves, w, kRegion, kbase);
      copy(wave + kWaves, w, kVBase + kRegion, vbase);
    }
    auto step = [&](int i, auto which) {  // (tile i of the wave, in slot i & 1)
      constexpr int slot = decltype(which)::value * kRegion;
      const int t = wave + i * kWaves;
      const int next = i + 1 < n ? 1 : 0, after = i + 2 < n ? 1 : 0;
      const bool edge = bad_ids || t < from || t >= to;
      // K of this tile (V of it and both of the next may be in flight).
      wait_vmcnt_at_most<3 * kCopies>(kCopies * (1 + 2 * next));
      uint4 ka[KS];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) ka[ks] = *reinterpret_cast<const uint4*>(ring + slot + k_off[ks]);
      const Place w = place_of(t + 2 * kWaves);  // (past the run: some place in it, not used)
      f32x16 s[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < 16; ++j) s[b][j] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int b = 0; b < NB; ++b) s[b] = mfma32<T>(ka[ks], qreg[b][ks], s[b]);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the slot has been read)
      if (after) copy(t + 2 * kWaves, w, slot, kbase);
      uint4 pb[NB][2], rest[NB][2];
      if (edge) {
        uint32_t gone = 0;
        if (bad_ids)
          gone = static_cast<uint32_t>(__ballot(id_at(t, min(run.tile_at(t) + (lane & 31), run.kv_last)) < 0)) >>
                 (4 * half);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          mine[b].mask(run, a.sinks, t, half, s[b]);
          if (bad_ids) {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if ((gone >> (8 * (j >> 2) + (j & 3))) & 1u) s[b][j] = -INFINITY;
          }
        }
      }
      // V of this tile (both of the next and K of the one after may be in flight).
      wait_vmcnt_at_most<3 * kCopies>(kCopies * (2 * next + after));
      if (edge && (bad_ids || run.has_hole(t))) {
        const int p = run.tile_at(t) + (lane & 31);
        if (run.hidden(p) || (bad_ids && id_at(t, min(p, run.kv_last)) < 0)) {
          char* r = ring + kVBase + slot + (lane & 31) * ROW_BYTES + half * (ROW_BYTES / 2);
#pragma unroll 1
          for (int j = 0; j < ROW_BYTES / 32; ++j) st16(r + 16 * j, make_uint4(0, 0, 0, 0));
        }
      }
      // (its operands are read while the softmax runs)
      uint4 va[DB][2];
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          const char* base = ring + slot + kk * 16 * ROW_BYTES;
          const uint2 lo = lds_read_tr16(reinterpret_cast<const uint16_t*>(base + v_off[db][0]));
          const uint2 hi = lds_read_tr16(reinterpret_cast<const uint16_t*>(base + v_off[db][1]));
          va[db][kk] = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        // The reference maximum moves only when a tile's maximum exceeds it by more
        // than kLazyRescale (log2 units).
        const float tmax = tree_tile_max(s[b]);
        const bool grow = (tmax - m[b]) * scale > kLazyRescale;
        if (__builtin_amdgcn_ballot_w64(grow) != 0) {
          const float m_new = grow ? tmax : m[b];
          const float alpha = fast_exp2((m[b] - m_new) * scale);
          l[b] *= alpha;
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            if constexpr (D > 64) in_matrix_registers(acc[b][db]);
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[b][db][j] *= alpha;
            if constexpr (D > 64) in_matrix_registers(acc[b][db]);
          }
          m[b] = m_new;
        }
        const float msc = m[b] * scale;
        float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int j = 8 * c; j < 8 * c + 8; ++j) s[b][j] = fast_exp2(fmaf(s[b][j], scale, -msc));
          split_weights<T>(s[b], c, pb[b][c], rest[b][c], sum0, sum1);
        }
        l[b] += sum0 + sum1;
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (after) copy(t + 2 * kWaves, w, kVBase + slot, vbase);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int b = 0; b < NB; ++b) acc[b][db] = mfma32<T>(va[db][kk], pb[b][kk], acc[b][db]);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int b = 0; b < NB; ++b) acc[b][db] = mfma32<T>(va[db][kk], rest[b][kk], acc[b][db]);
    };
    for (int i = 0; i < n; i += 2) {
      step(i, std::integral_constant<int, 0>());
      if (i + 1 < n) step(i + 1, std::integral_constant<int, 1>());
    }

    // ---- the waves of each row joined ---------------------------------------------
    // Each wave leaves its accumulators in its own rings, in 16-byte pieces (piece c
    // of lane i at (c * 64 + i) * 16), and finishes NB DB of the pieces for all.
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      l[b] += __shfl_xor(l[b], 32, kWave);
      if (half == 0) s_ml[wave][b * 32 + (lane & 31)] = make_float2(m[b], l[b]);
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<float4*>(ring + (((b * DB + db) * 4 + q) * kWave + lane) * 16) =
              make_float4(acc[b][db][4 * q], acc[b][db][4 * q + 1], acc[b][db][4 * q + 2], acc[b][db][4 * q + 3]);
    }
    __syncthreads();
    constexpr int kMine = NB * kPieces / kWaves;
    const int b = wave * kMine / kPieces;  // block of this wave's pieces
    const int row = b * 32 + (lane & 31);
    const int tok = row / G;
    const int h = h0 + (row - tok * G);
    float mm = kScoreFloor, sum = 0.f, f[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) mm = fmaxf(mm, s_ml[w][row].x);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float2 x = s_ml[w][row];
      f[w] = fast_exp2((x.x - mm) * scale);
      sum = fmaf(x.y, f[w], sum);
    }
    if (tok >= run.ntok) return;
    const float inv = sum > 0.f ? 1.f / sum : sum;  // (zero for a row that sees nothing; a NaN stays)
    const int64_t prow = (static_cast<int64_t>(run.part_row) + tok) * hq + h;
    uint16_t* orow = reinterpret_cast<uint16_t*>(a.output) +
                     ((static_cast<int64_t>(run.first) + run.tok0 + tok) * hq + h) * static_cast<int64_t>(DM);
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      const int c = wave * kMine + k;
      const int d = ((c / 4) % DB) * 32 + 8 * (c % 4) + 4 * half;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(s_lds + w * kWaveBytes + (c * kWave + lane) * 16);
        o = make_float4(fmaf(x.x, f[w], o.x), fmaf(x.y, f[w], o.y), fmaf(x.z, f[w], o.z), fmaf(x.w, f[w], o.w));
      }
      if (MASKD && d >= DM) continue;
      if (run.part_row >= 0)  // one of a tile's runs: the sums as they are, for merge_tree_kernel
        *reinterpret_cast<float4*>(a.part_acc + prow * DM + d) = o;
      else
        *reinterpret_cast<uint2*>(orow + d) =
            make_uint2(pack_half2<T>(o.x * inv, o.y * inv), pack_half2<T>(o.z * inv, o.w * inv));
    }
    if (run.part_row >= 0 && half == 0 && (wave * kMine) % kPieces == 0)
      *reinterpret_cast<float2*>(a.part_ml + prow * 2) = make_float2(mm * scale, sum);
  };
  if (run.ntok * G <= 32)
    attend(std::integral_constant<int, 1>());
  else
    attend(std::integral_constant<int, 2>());
}

// No more units than CUs: four waves each, which halve a unit's chain where a second
// workgroup would not share its CU (us, four and two waves: one tree of 26 nodes after
// 3000, 32/8 heads of 128, 24 items 17.8 and 20.1, 4 items 29.7 and 48.3; 8 trees of 64,
// 32/32 heads, 8 items 71 and 104).  More units: two, of which a CU holds two or three (2
// trees under a window of 8192, 54 items 48.8 and 41.4; 64 trees of 9-17 nodes, 9/3 heads
// of 64, 251 items 52 and 41).
template <typename T, int D, int DM>
hipError_t launch_d(const PrefillArgs& a, dim3 grid, hipStream_t s) {
  if (static_cast<int>(grid.x) <= device_compute_units())
    hipLaunchKernelGGL((tree_attention_kernel<T, D, DM, 4>), grid, dim3(4 * kWave), 0, s, a);
  else
    hipLaunchKernelGGL((tree_attention_kernel<T, D, DM, 2>), grid, dim3(2 * kWave), 0, s, a);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_t(const PrefillArgs& a, int head_dim, dim3 grid, hipStream_t s) {
  switch (head_dim) {
    case 64: return launch_d<T, 64, 64>(a, grid, s);
    case 80: return launch_d<T, 128, 80>(a, grid, s);
    case 96: return launch_d<T, 128, 96>(a, grid, s);
    case 128: return launch_d<T, 128, 128>(a, grid, s);
    default: return hipErrorNotSupported;
  }
}

}  // namespace

int tree_tile_for(int dtype, int head_dim, int group) {
  const int g = group / decode_sub_groups(group);
  return dtype == PA_DTYPE_E4M3 || dtype == PA_DTYPE_F32 || head_dim == 256 ? prefill_tile_for(group) : kTreeRows / g;
}

hipError_t launch_tree_attention(const PrefillArgs& a, int dtype, int head_dim, int group, int64_t num_items,
                                 hipStream_t stream) {
  const int g = group / a.sub_groups;
  const int64_t units = num_items * a.num_kv_heads * a.sub_groups;
  if (g < 1 || g > 8 || units > 0x7fffffff) return hipErrorNotSupported;
  if (units <= 0) return hipSuccess;
  if (head_dim == 256) return launch_tree_attention256(a, dtype, group, num_items, stream);
  const dim3 grid(static_cast<uint32_t>(units));
  if (dtype == PA_DTYPE_BF16) return launch_t<bf16_t>(a, head_dim, grid, stream);
  if (dtype == PA_DTYPE_F16) return launch_t<f16_t>(a, head_dim, grid, stream);
  return hipErrorNotSupported;
}

}  // namespace pa
