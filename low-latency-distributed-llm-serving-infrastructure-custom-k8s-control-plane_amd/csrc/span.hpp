// What part of the context a query sees under a window with sinks, and how the
// tuned kernels leave the rest out: the query at position p sees the positions
// q <= p with p - q < window or q < sinks.  Used by the kernels and, for the
// work lists, by the host (no HIP types).
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define PA_HOST_DEVICE __host__ __device__ inline
#else
#define PA_HOST_DEVICE inline
#endif

namespace pa {

// What a kernel instance's queries see: the whole context, a window with sinks of
// it, or a tree of drafted tokens behind it (or behind a window of it).
enum { kSpanAll = 0, kSpanWindow = 1, kSpanTree = 2 };

// Most nodes of one tree (pa_pack_tree keeps a sequence's parents in LDS).
constexpr int kMaxTreeNodes = 1024;

PA_HOST_DEVICE int span_min(int a, int b) { return a < b ? a : b; }
PA_HOST_DEVICE int span_max(int a, int b) { return a > b ? a : b; }

// First position of the window of the query at position p (window >= 1; 0: no
// window).
PA_HOST_DEVICE int window_start(int p, int window) { return window > 0 ? span_max(p - window + 1, 0) : 0; }

// A single query at the end of a context of ctx positions, in whole blocks of
// 2^log2_bs tokens.  The blocks between the last one that holds sinks and the
// first one of the window are left out: the kernel walks a context of `ctx`
// positions without them, whose block column c is column c of the sequence's
// table, or c + skip from column `sinks` on.  Of that shorter context the
// positions [hole, hole_end), in the two blocks beside the cut, are not seen.
struct DecodeSpan {
  int ctx;
  int sinks, skip;
  int hole, hole_end;
};
PA_HOST_DEVICE DecodeSpan decode_span(int ctx, int window, int sinks, int log2_bs) {
  const int lo = window_start(ctx - 1, window);
  const int s = span_min(sinks, lo);
  DecodeSpan d;
  d.sinks = (s >> log2_bs) + ((s & ((1 << log2_bs) - 1)) != 0 ? 1 : 0);
  d.skip = span_max((lo >> log2_bs) - d.sinks, 0);
  d.ctx = ctx - (d.skip << log2_bs);
  d.hole = s;
  d.hole_end = lo - (d.skip << log2_bs);
  return d;
}

// The queries of a tile, the first window of which starts at lo and the last
// of which sees positions below `end`, in stages of `stage` positions: those of
// the sinks first, then from the window's first stage on, `gap` stages left out
// between them.
struct StageSpan {
  int sinks, gap;
  int count;
};
PA_HOST_DEVICE StageSpan stage_span(int lo, int end, int sinks, int stage) {
  StageSpan t;
  const int s = span_min(sinks, lo);
  t.sinks = s / stage + (s % stage != 0 ? 1 : 0);
  t.gap = span_max(lo / stage - t.sinks, 0);
  t.count = span_max((end > 0 ? (end - 1) / stage + 1 : 0) - t.gap, 0);
  return t;
}

// The stages of a tree's tile, whose last query is node `nodes` - 1 of its
// sequence (the root, at position `start`, sees the first window of them all).
PA_HOST_DEVICE StageSpan tree_span(int start, int nodes, int window, int sinks, int stage) {
  return stage_span(window_start(start, window), start + nodes, sinks, stage);
}

// Positions of a stage, in which the tiles of every matrix-core kernel of trees walk
// their context.
constexpr int kTreeStage = 64;
// Query rows of a tile over 16-bit caches, heads of up to 128; nodes of a tile of
// any shape (dtype: the cache's).
constexpr int kTreeRows = 64;
int tree_tile_for(int dtype, int head_dim, int group);
// A tile's stages in runs of at most `most`, as even as whole stages allow.
struct TreeSplit {
  int runs, stages;
};
PA_HOST_DEVICE TreeSplit tree_split(int count, int most) {
  TreeSplit t;
  t.runs = count > 0 ? (count - 1) / most + 1 : 0;
  t.stages = t.runs > 0 ? (count - 1) / t.runs + 1 : 1;
  return t;
}
// An item of a tree's work list: sequence (-1: an entry that is not needed), tile,
// run of stages, first row of its partial results or -1; first token, nodes,
// context before the tree and table row of the sequence.
constexpr int kTreeItemInts = 8;
// Block ids that the kernel keeps of a run, and the most stages whose columns (and
// the two more at each end of the sinks' and the window's) they cover.
constexpr int kTreeIds = 3584;
PA_HOST_DEVICE int tree_max_stages(int block_size) {
  const long long n = static_cast<long long>(kTreeIds - 8) * block_size / kTreeStage;
  return n < (1 << 24) ? static_cast<int>(n) : 1 << 24;
}
// Whether a matrix-core kernel of trees serves the shape (dtype: the cache's, 8-bit codes
// under 16-bit queries): tree_attention.hip, for heads of 256 tree_attention256.hip, over
// 8-bit caches prefill_tree.hip, over fp32 ones prefill_f32.hip.
bool tree_fast_path_supported(int dtype, int head_dim, int group, int block_size);

}  // namespace pa
