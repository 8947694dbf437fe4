// What the tree attention kernels (tree_attention.hip, tree_attention256.hip) share:
// an item's run of the context, the blocks of its columns, and a row's masks.
#pragma once

#include "pa_common.hpp"
#include "pa_launch.hpp"
#include "prefill_common.hpp"
#include "span.hpp"

namespace pa {

constexpr int kTreeKvTile = 32;  // context tokens of an MFMA tile
constexpr int kTreePerStage = kTreeStage / kTreeKvTile;

// An item's record, and the tiles of its run (all wave-uniform).
struct TreeRun {
  int first, count, start;  // the sequence's first token, nodes, and context before them
  int tok0, ntok;           // the tile's nodes
  int part_row;
  int kv_end, kv_last;      // exclusive end of what the tile sees; last position with a table column
  int seen_lo, seen_sinks;  // positions [0, seen_sinks) and from seen_lo on are seen by some row
  int gap, sinks, stage0;   // stages left out, of the sinks, and before the run
  int stages, ntiles;
  // Columns in LDS: of the run's nsink sink stages, then of the others.
  int nsink, col_a, cols_a, col_b, ncols;
  int trow;

  // False: an entry that is not needed, or an empty run.
  __device__ __forceinline__ bool load(const PrefillArgs& a, int64_t item, int mtok) {
    const int32_t* rec = a.items + item * kTreeItemInts;
    const int seq = rec[0], split = rec[2];
    tok0 = rec[1] * mtok;
    part_row = rec[3];
    first = rec[4];
    count = rec[5];
    start = rec[6];
    trow = rec[7];
    ntok = min(mtok, count - tok0);
    kv_end = start + tok0 + ntok;
    seen_lo = min(window_start(start, a.window), start);
    seen_sinks = min(a.sinks, seen_lo);
    const StageSpan s = stage_span(seen_lo, kv_end, a.sinks, kTreeStage);
    gap = s.gap;
    sinks = s.sinks;
    const TreeSplit cut = tree_split(s.count, a.split_stages);
    stage0 = split * cut.stages;
    stages = min(s.count - stage0, cut.stages);
    return seq >= 0 && ntok > 0 && stages > 0;
  }
  __device__ __forceinline__ int stage_at(int x) const {
    const int at = x + stage0;
    return (at < sinks ? at : at + gap) * kTreeStage;
  }
  __device__ __forceinline__ int tile_at(int t) const {
    return stage_at(t / kTreePerStage) + (t % kTreePerStage) * kTreeKvTile;
  }
  __device__ __forceinline__ void plan(int log2_bs, int bt_stride) {
    kv_last = static_cast<int>(min(static_cast<int64_t>(kv_end), static_cast<int64_t>(bt_stride) << log2_bs)) - 1;
    // (tiles past the context's end are left out)
    ntiles = kTreePerStage * stages - max(0, (stage_at(stages - 1) + kTreeStage - kv_end) / kTreeKvTile);
    nsink = min(max(sinks - stage0, 0), stages);
    col_a = (stage0 * kTreeStage) >> log2_bs;
    cols_a = nsink > 0 ? (((stage0 + nsink) * kTreeStage - 1) >> log2_bs) - col_a + 1 : 0;
    col_b = stage_at(nsink) >> log2_bs;
    const int end_b = min(stage_at(stages - 1) + kTreeStage, kv_end);
    const int cols_b = nsink < stages ? ((end_b - 1) >> log2_bs) - col_b + 1 : 0;
    ncols = min(cols_a + cols_b, kTreeIds);
  }
  __device__ __forceinline__ int column(int i) const { return i < cols_a ? col_a + i : col_b + (i - cols_a); }
  // Place in LDS of the column of position p of tile t.
  __device__ __forceinline__ int id_index(int t, int p, int log2_bs) const {
    const int c = p >> log2_bs;
    const int i = t / kTreePerStage < nsink ? c - col_a : cols_a + (c - col_b);
    return min(max(i, 0), kTreeIds - 1);
  }
  // Whether column i of the run holds a position that some row sees.
  __device__ __forceinline__ bool column_seen(int i, int log2_bs) const {
    const int p = column(i) << log2_bs;
    return p < seen_sinks || (p + (1 << log2_bs) > seen_lo && p < kv_end);
  }
  // Rows of tile t that no row of the unit sees.
  __device__ __forceinline__ bool has_hole(int t) const {
    return tile_at(t) < seen_lo && tile_at(t) + kTreeKvTile > seen_sinks;
  }
  __device__ __forceinline__ bool hidden(int p) const { return p >= seen_sinks && p < seen_lo; }
  // Tiles [from, to) are seen whole by every row: from the last row's window on, to
  // the tree.
  __device__ __forceinline__ int from(int window) const {
    const int lo = min(window_start(start + count - 1, window), start);
    return (lo + kTreeKvTile - 1) / kTreeKvTile - (gap + stage0) * kTreePerStage;
  }
  __device__ __forceinline__ int to() const {
    return min(start, kv_last + 1) / kTreeKvTile - (gap + stage0) * kTreePerStage;
  }
};

// Around the only vector instructions on accumulators, a rescale's: without it the
// compiler copies all of them out of the matrix registers at each tile, for the case of
// a rescale (32 trees of 9-17 nodes, 32/8 heads of 128, one term a probability: 132 us,
// with it 122).
__device__ __forceinline__ void in_matrix_registers(f32x16& x) { asm("" : "+a"(x)); }

// s_waitcnt's immediate for vmcnt(0) alone.
constexpr int kWaitLoads = 0x0F70;

// A query row's masks.  The first 64 bits of its node's word stay in registers.
struct TreeRow {
  const uint32_t* words;
  uint32_t word0, word1;
  int num_words;
  int lo;   // where its window starts
  int lim;  // last position it may see

  __device__ __forceinline__ void load(const PrefillArgs& a, const TreeRun& r, int tok) {
    const int64_t node = static_cast<int64_t>(r.first) + r.tok0 + (tok < r.ntok ? tok : 0);
    words = a.masks + node * a.mask_words;
    num_words = a.mask_words;
    word0 = words[0];
    word1 = a.mask_words > 1 ? words[1] : 0u;
    lo = a.window > 0 ? min(window_start(static_cast<int>(a.positions[node]), a.window), r.start) : 0;
    lim = min(r.start + r.tok0 + tok, r.kv_last);
  }
  // Scores of tile t (lane half `half`) that the row does not see.  (What is
  // computed for a tile past the run's last counts for nothing.)
  __device__ __forceinline__ void mask(const TreeRun& r, int sinks, int t, int half, f32x16& s) const {
    const int tile = r.tile_at(t);
    const int at = tile + 4 * half;
    const int last = t < r.ntiles ? lim - at : -1;
    const int low = lo - at, sink = sinks - at;
    uint32_t bits = ~0u;
    if (tile + kTreeKvTile > r.start) {
      const int n = at - r.start;  // node of the first position; before the tree all bits are ones
      auto word = [&](int w) {
        if (w < 2) return w < 0 ? ~0u : w == 0 ? word0 : word1;
        return w < num_words ? words[w] : 0u;
      };
      bits = static_cast<uint32_t>(((static_cast<uint64_t>(word((n >> 5) + 1)) << 32) | word(n >> 5)) >> (n & 31));
    }
    hide(s, bits & below(last + 1) & (~below(low) | below(sink)));
  }
};

// Row maximum of a tile: v_max3 written out, because fmaxf quiets each input first.
// (Each of the first depends on an instruction that the compiler sees reading the
// product's last result, so that none comes before the product is done.)
__device__ __forceinline__ float tree_tile_max(const f32x16& s) {
  const float ready = __builtin_amdgcn_fmed3f(s[15], s[15], s[15]);
  auto first3 = [&](float x, float y, float z) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z), "v"(ready));
    return r;
  };
  auto max3 = [](float x, float y, float z) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
    return r;
  };
  const float a0 = first3(s[0], s[1], s[2]), a1 = first3(s[3], s[4], s[5]), a2 = first3(s[6], s[7], s[8]);
  const float a3 = first3(s[9], s[10], s[11]), a4 = first3(s[12], s[13], s[14]);
  return max_halves(max3(max3(a0, a1, a2), max3(a3, a4, ready), ready));
}

}  // namespace pa
