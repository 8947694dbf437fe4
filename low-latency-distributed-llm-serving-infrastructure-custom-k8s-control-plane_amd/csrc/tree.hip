// Trees of drafted tokens: what surrounds their attention (tree_attention.hip,
// tree_attention256.hip, prefill_tree.hip, prefill_f32.hip, generic.hip) in a
// verification step.
//
//  pack_tree_kernel    the nodes' masks and positions from their parents, and
//                      the attention's work lists;
//  merge_tree_kernel   joins the partial results of tiles whose context was
//                      split over workgroups;
//  accept_tree_kernel  the path of nodes whose tokens the model itself chose;
//  keep_rows_kernel    moves the path's K and V rows behind the context, in
//                      every layer (keep_rows8_kernel: in an 8-bit cache).
//
// All four are chains of dependent reads over little data: what counts is the
// number of round trips and of launches.  Node i of a sequence names an earlier
// node as its parent, or is a root; a parent that is no earlier node of the
// sequence reads as a root, so every walk up ends.
#include <algorithm>
#include <type_traits>

#include "cache8.hpp"
#include "pa_common.hpp"
#include "pa_launch.hpp"
#include "span.hpp"

namespace pa {

namespace {

constexpr int kTreeThreads = 256;

// A sequence's tokens: first row, count (at most kMaxTreeNodes, inside the step).
struct TreeSeq {
  int64_t first;
  int count;
};
__device__ __forceinline__ TreeSeq tree_seq(const int64_t* cu_seqlens, int seq, int num_query_tokens) {
  TreeSeq s;
  s.first = cu_seqlens[seq];
  const int64_t n = min<int64_t>(cu_seqlens[seq + 1], num_query_tokens) - s.first;
  s.count = static_cast<int>(max<int64_t>(0, min<int64_t>(n, kMaxTreeNodes)));
  return s;
}
__device__ __forceinline__ int parent_of(const int32_t* parents, int64_t first, int node) {
  const int p = parents[first + node];
  return p >= 0 && p < node ? p : -1;
}

// Items, merge items and partial rows of a sequence's tiles (64-bit: contexts of the
// device's arrays may be longer than those the lists were sized for).
struct TreeWork {
  int64_t items, merges, rows;
};
__device__ __forceinline__ TreeWork tree_work(const PackTreeArgs& a, int start, int count) {
  TreeWork w{0, 0, 0};
  for (int t0 = 0; t0 < count; t0 += a.tile) {
    const int n = min(a.tile, count - t0);
    const int stages = tree_span(start, t0 + n, a.window, a.sinks, kTreeStage).count;
    const int splits = tree_split(stages, a.split_stages).runs;
    w.items += splits;
    if (splits > 1) {
      w.merges += 1;
      w.rows += static_cast<int64_t>(splits) * n;
    }
  }
  return w;
}

// One workgroup a sequence.  Each node walks up its ancestors in LDS, whose
// indices fall, so its mask's words come out from the last to the first.  For
// the work lists every workgroup adds up what the sequences before its own
// need (a step of 64 sequences: a read each); the last one marks the entries
// behind the lists' ends, so that a launch sized for more work skips them.  One tree of
// 26 nodes 3.4 us, 48 of 16-64 nodes 6.6.
__global__ __launch_bounds__(kTreeThreads) void pack_tree_kernel(PackTreeArgs a) {
  __shared__ int s_parent[kMaxTreeNodes];
  __shared__ int64_t s_sum[kTreeThreads / kWave][3];
  const int tid = threadIdx.x;
  const int seq = blockIdx.x;
  const TreeSeq s = tree_seq(a.cu_seqlens, seq, a.num_query_tokens);
  const int start = a.context_lens[seq] - s.count;
  for (int i = tid; i < s.count; i += kTreeThreads) {
    const int p = parent_of(a.parents, s.first, i);
    s_parent[i] = p;
    if (a.packed_parents != nullptr) a.packed_parents[s.first + i] = p;
  }
  int64_t items = 0, merges = 0, rows = 0;
  if (a.items != nullptr) {
    for (int j = tid; j < seq; j += kTreeThreads) {
      const TreeSeq o = tree_seq(a.cu_seqlens, j, a.num_query_tokens);
      const TreeWork w = tree_work(a, a.context_lens[j] - o.count, o.count);
      items += w.items;
      merges += w.merges;
      rows += w.rows;
    }
#pragma unroll
    for (int o = kWave / 2; o >= 1; o >>= 1) {
      items += __shfl_xor(static_cast<long long>(items), o, kWave);
      merges += __shfl_xor(static_cast<long long>(merges), o, kWave);
      rows += __shfl_xor(static_cast<long long>(rows), o, kWave);
    }
    if (tid % kWave == 0) {
      s_sum[tid / kWave][0] = items;
      s_sum[tid / kWave][1] = merges;
      s_sum[tid / kWave][2] = rows;
    }
  }
  __syncthreads();

  for (int i = tid; i < s.count; i += kTreeThreads) {
    uint32_t* mask = a.masks + (s.first + i) * a.mask_words;
    int w = i >> 5, depth = 0;
    for (int k = a.mask_words - 1; k > w; --k) mask[k] = 0;
    uint32_t bits = 1u << (i & 31);
    for (int p = s_parent[i]; p >= 0; p = s_parent[p]) {
      ++depth;
      while (w > (p >> 5)) {
        if (w < a.mask_words) mask[w] = bits;
        bits = 0;
        --w;
      }
      bits |= 1u << (p & 31);
    }
    for (; w >= 0; --w) {
      if (w < a.mask_words) mask[w] = bits;
      bits = 0;
    }
    a.positions[s.first + i] = static_cast<int64_t>(start) + depth;
  }
  if (a.items == nullptr) return;

  items = merges = rows = 0;
#pragma unroll
  for (int w = 0; w < kTreeThreads / kWave; ++w) {
    items += s_sum[w][0];
    merges += s_sum[w][1];
    rows += s_sum[w][2];
  }
  for (int t0 = 0; t0 < s.count; t0 += a.tile) {
    const int n = min(a.tile, s.count - t0);
    const int stages = tree_span(start, t0 + n, a.window, a.sinks, kTreeStage).count;
    const int splits = tree_split(stages, a.split_stages).runs;
    // (a tile whose partials would not fit is left out: the host sizes them)
    const bool fits = splits == 1 || rows + static_cast<int64_t>(splits) * n <= a.max_partial_rows;
    for (int k = tid; k < splits; k += kTreeThreads)
      if (items + k < a.max_items) {
        int4* item = a.items + 2 * (items + k);
        item[0] = make_int4(fits ? seq : -1, t0 / a.tile, k, splits > 1 && fits ? static_cast<int>(rows) + k * n : -1);
        item[1] = make_int4(static_cast<int>(s.first), s.count, start, a.rows != nullptr ? a.rows[seq] : seq);
      }
    if (splits > 1) {
      if (tid == 0 && merges < a.max_merge_items)
        a.merge_items[merges] = make_int4(fits ? seq : -1, t0 / a.tile, splits, fits ? static_cast<int>(rows) : 0);
      merges += 1;
      rows += static_cast<int64_t>(splits) * n;
    }
    items += splits;
  }
  if (seq == a.num_seqs - 1) {
    for (int64_t i = items + tid; i < a.max_items; i += kTreeThreads) a.items[2 * i] = make_int4(-1, 0, 0, -1);
    for (int64_t i = merges + tid; i < a.max_merge_items; i += kTreeThreads) a.merge_items[i] = make_int4(-1, 0, 0, 0);
  }
}

// A thread four elements of one head of a node of a split tile, kMergeRuns
// partials a round trip with a running maximum (the stored maxima are in the exp2
// domain); slots past the last partial read it again and get no weight.  The
// partials are in L2 or beside it: what counts is the number of round trips, so
// the loads of a batch go out together and a node's heads spread over workgroups
// (26 nodes of 32 heads of 128 in 16 runs: 3.9 us; one workgroup a node, eight partials
// a trip: 13.2).  Up to four runs go in a batch of four (8 trees of 64 nodes, 32 heads
// of 128, two runs each: 5.4 us; sixteen slots, most of them the last run again: 9.2),
// up to eight in one of eight (2 trees of 40-60 nodes in 5 runs, with their attention:
// 37.0 us, in sixteen slots 38.2).
constexpr int kMergeRuns = 16;
constexpr int kFewRuns = 4;
template <typename T, int D>
__global__ __launch_bounds__(kTreeThreads) void merge_tree_kernel(MergeTreeArgs a) {
  const int64_t m = blockIdx.x / a.tile;
  const int tok = static_cast<int>(blockIdx.x - m * a.tile);
  const int4 item = a.merge_items[m];
  const int r = blockIdx.y * kTreeThreads + threadIdx.x;
  const int hq = a.num_query_heads;
  if (item.x < 0 || r >= hq * (D / 4)) return;
  const int64_t first = a.cu_seqlens[item.x];
  const int64_t count = min<int64_t>(a.cu_seqlens[item.x + 1], a.num_query_tokens) - first;
  const int64_t t0 = static_cast<int64_t>(item.y) * a.tile;
  const int n = static_cast<int>(min<int64_t>(a.tile, count - t0));
  if (tok >= n) return;
  const int h = r / (D / 4);
  const int64_t row = (static_cast<int64_t>(item.w) + tok) * hq + h;  // of the first run, n * hq rows apart
  const int64_t step = static_cast<int64_t>(hq) * n;
  const float4* acc = reinterpret_cast<const float4*>(a.part_acc) + row * (D / 4) + (r - h * (D / 4));
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + row;
  float mx = kScoreFloor, sum = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto join = [&](auto runs) {
    constexpr int R = decltype(runs)::value;
    for (int p = 0; p < item.z; p += R) {
      float2 s[R];
      float4 x[R];
#pragma unroll
      for (int u = 0; u < R; ++u) {
        const int64_t at = min(p + u, item.z - 1) * step;
        s[u] = ml[at];
        x[u] = acc[at * (D / 4)];
      }
      float mn = mx;
#pragma unroll
      for (int u = 0; u < R; ++u) mn = fmaxf(mn, s[u].x);
      const float keep = fast_exp2(mx - mn);
      sum *= keep;
      o = make_float4(o.x * keep, o.y * keep, o.z * keep, o.w * keep);
#pragma unroll
      for (int u = 0; u < R; ++u) {
        const float w = p + u < item.z ? fast_exp2(s[u].x - mn) : 0.f;
        if (p + u < item.z) {
          sum = fmaf(s[u].y, w, sum);
          o = make_float4(fmaf(x[u].x, w, o.x), fmaf(x[u].y, w, o.y), fmaf(x[u].z, w, o.z), fmaf(x[u].w, w, o.w));
        }
      }
      mx = mn;
    }
  };
  if (item.z <= kFewRuns) join(std::integral_constant<int, kFewRuns>());
  else if (item.z <= 2 * kFewRuns) join(std::integral_constant<int, 2 * kFewRuns>());
  else join(std::integral_constant<int, kMergeRuns>());
  // (a sum of zero is a row that attends nothing, whose result is zero; a NaN stays)
  T* out = reinterpret_cast<T*>(a.output) + (first + t0 + tok) * hq * D + static_cast<int64_t>(r) * 4;
  o = sum != 0.f ? make_float4(o.x / sum, o.y / sum, o.z / sum, o.w / sum) : make_float4(0.f, 0.f, 0.f, 0.f);
  if constexpr (sizeof(T) == 4)
    *reinterpret_cast<float4*>(out) = o;
  else
    *reinterpret_cast<uint2*>(out) = make_uint2(pack_half2<T>(o.x, o.y), pack_half2<T>(o.z, o.w));
}

// One wave a sequence: at each node the lanes look for its first child (they
// come behind it) that drafted the token predicted there: two round trips a node of
// the path.  One tree of 26 nodes 2.6 us, 48 of 16-64 nodes 5.2.
__global__ __launch_bounds__(kWave) void accept_tree_kernel(AcceptTreeArgs a) {
  __shared__ int s_parent[kMaxTreeNodes];
  const int lane = threadIdx.x;
  const int seq = blockIdx.x;
  const TreeSeq s = tree_seq(a.cu_seqlens, seq, a.num_query_tokens);
  for (int i = lane; i < s.count; i += kWave) s_parent[i] = parent_of(a.parents, s.first, i);
  __syncthreads();
  int kept = 0;
  int64_t next = -1;
  for (int node = s.count > 0 ? 0 : -1; node >= 0;) {
    if (lane == 0) a.nodes[s.first + kept] = node;
    ++kept;
    next = a.predicted[s.first + node];
    int child = -1;
    for (int i0 = node + 1; i0 < s.count && child < 0; i0 += kWave) {
      const int i = i0 + lane;
      const bool on = i < s.count && s_parent[i] == node && a.drafted[s.first + i] == next;
      const uint64_t hits = __ballot(on);
      if (hits != 0) child = i0 + __builtin_ctzll(hits);
    }
    node = child;
  }
  for (int i = kept + lane; i < s.count; i += kWave) a.nodes[s.first + i] = -1;
  if (lane == 0) {
    a.counts[seq] = kept;
    a.next_tokens[seq] = next;
  }
}

// Where a sequence's positions lie, and what of its nodes is kept.
struct KeptSeq {
  int64_t first;
  int start, count;  // count: entries of `nodes` looked at
  int nodes;
  const int32_t* table;  // null: no blocks
};
__device__ __forceinline__ KeptSeq kept_seq(const KeepRowsArgs& a, int seq) {
  const TreeSeq s = tree_seq(a.cu_seqlens, seq, a.num_query_tokens);
  KeptSeq k;
  k.first = s.first;
  k.nodes = s.count;
  k.start = a.context_lens[seq] - s.count;
  k.count = max(0, min(a.counts[seq], s.count));
  const int64_t trow = a.rows != nullptr ? a.rows[seq] : seq;
  k.table = trow >= 0 && trow < a.num_table_rows ? a.block_tables + trow * a.block_table_stride : nullptr;
  return k;
}
// Block of a position, or -1.
__device__ __forceinline__ int kept_block(const KeepRowsArgs& a, const KeptSeq& k, int pos) {
  const int col = pos / a.block_size;
  if (k.table == nullptr || pos < 0 || col >= a.block_table_stride) return -1;
  const int b = k.table[col];
  return b >= 0 && b < a.total_blocks ? b : -1;
}
// Whether entry j of a sequence's kept nodes can follow the one before it.
__device__ __forceinline__ bool kept_ok(const KeepRowsArgs& a, const KeptSeq& k, int j) {
  const int node = a.nodes[k.first + j];
  return node >= j && node < k.nodes && (j == 0 || node > a.nodes[k.first + j - 1]);
}

// A workgroup a (sequence, layer, tensor), a thread the same 16 (or fewer)
// bytes of every row: rows move down in order (the kept nodes ascend, so no row
// is written before it has been read), and no thread waits for another but for
// the slots of the next 64 rows.  48 trees of 16-64 nodes, 32 layers, 8 heads of 128: 12
// us (20 MB, 1.6 TB/s: the counts, the nodes, the table and the rows are read one after
// the other); one tree 4.6.
template <typename V>
__global__ __launch_bounds__(kTreeThreads) void keep_rows_kernel(KeepRowsArgs a) {
  constexpr int kBatch = 8;
  __shared__ int64_t s_from[kWave], s_to[kWave];  // rows of the layer; -1: stays
  __shared__ int s_end;
  const int tid = threadIdx.x;
  const KeptSeq k = kept_seq(a, blockIdx.x);
  const int layer = blockIdx.y >> 1;
  char* base = reinterpret_cast<char*>((blockIdx.y & 1) ? a.value_cache : a.key_cache) +
               static_cast<int64_t>(layer) * a.total_blocks * a.block_size * a.row_bytes;
  const int pieces = static_cast<int>(a.row_bytes / sizeof(V));
  for (int j0 = 0; j0 < k.count; j0 += kWave) {
    if (tid < kWave) {
      const int j = j0 + tid;
      const bool ok = j < k.count && kept_ok(a, k, j);
      const int node = ok ? a.nodes[k.first + j] : 0;
      int64_t from = -1, to = -1;
      if (ok && node != j) {
        const int p = k.start + node, q = k.start + j;
        const int bp = kept_block(a, k, p), bq = kept_block(a, k, q);
        if (bp >= 0 && bq >= 0) {
          from = static_cast<int64_t>(bp) * a.block_size + p % a.block_size;
          to = static_cast<int64_t>(bq) * a.block_size + q % a.block_size;
        }
      }
      s_from[tid] = from;
      s_to[tid] = to;
      const uint64_t bad = ~__ballot(ok);
      if (tid == 0) s_end = bad == 0 ? kWave : __builtin_ctzll(bad);
    }
    __syncthreads();
    const int end = s_end;
    for (int c = tid; c < pieces; c += blockDim.x) {
      for (int j = 0; j < end; j += kBatch) {
        V v[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
          if (j + u < end && s_from[j + u] >= 0)
            v[u] = reinterpret_cast<const V*>(base + s_from[j + u] * a.row_bytes)[c];
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
          if (j + u < end && s_from[j + u] >= 0) reinterpret_cast<V*>(base + s_to[j + u] * a.row_bytes)[c] = v[u];
      }
    }
    __syncthreads();
    if (end < kWave) return;  // (the whole workgroup)
  }
}

// An 8-bit cache: a wave a (sequence, layer, tensor, KV head), a lane the same
// codes of every row.  Block after block that rows move into: its scale becomes
// the largest among its own and those of the blocks that the rows come from; if
// that is larger, its rows are re-coded with it, and so is each row that moves
// in from a block of a smaller one (to nearest even; values but those among the
// subnormal codes stay).  A block that rows come from later still has its own
// codes and scale then.  The same 48 trees: 39 us, the rows of a block one after
// another.
__global__ __launch_bounds__(kWave) void keep_rows8_kernel(KeepRowsArgs a) {
  constexpr int kCodes = 4;  // codes of a row a lane holds, kWave apart
  const int lane = threadIdx.x;
  const KeptSeq k = kept_seq(a, blockIdx.x);
  const int layer = blockIdx.y >> 1;
  const int h = blockIdx.z;
  const bool is_v = blockIdx.y & 1;
  const int64_t layer_blocks = static_cast<int64_t>(layer) * a.total_blocks;
  uint8_t* base = reinterpret_cast<uint8_t*>(is_v ? a.value_cache : a.key_cache) +
                  layer_blocks * a.block_size * a.row_bytes + static_cast<int64_t>(h) * a.head_dim;
  float* scales = (is_v ? a.value_scales : a.key_scales) + layer_blocks * a.num_kv_heads + h;
  const float least = __uint_as_float(static_cast<uint32_t>(127 + kMinScaleExp) << 23);
  auto scale_of = [&](int b) { return fmaxf(scale_pow2(scales[static_cast<int64_t>(b) * a.num_kv_heads]), least); };
  auto row = [&](int b, int at) { return base + (static_cast<int64_t>(b) * a.block_size + at) * a.row_bytes; };
  auto recode = [&](const uint8_t* from, uint8_t* to, float ratio) {
    uint8_t x[kCodes];
#pragma unroll
    for (int e = 0; e < kCodes; ++e)
      if (lane + e * kWave < a.head_dim) x[e] = from[lane + e * kWave];
#pragma unroll
    for (int e = 0; e < kCodes; ++e)
      if (lane + e * kWave < a.head_dim)
        to[lane + e * kWave] =
            ratio == 1.f ? x[e] : static_cast<uint8_t>(pack_codes2(code_to_f32<0>(x[e]) * ratio, 0.f) & 0xffu);
  };
  int j = 0;
  bool good = true;
  while (good && j < k.count) {
    const int q = k.start + j;
    const int block = kept_block(a, k, q);
    const int last = min(k.count, j + a.block_size - q % a.block_size);  // (the block's last entry, + 1)
    const float had = block >= 0 ? scale_of(block) : least;
    float scale = had;
    bool moves = false;
    int stop = last;
    for (int i = j; i < last; ++i) {
      if (!kept_ok(a, k, i)) {
        stop = i;
        good = false;
        break;
      }
      const int node = a.nodes[k.first + i];
      const int from = node != i && block >= 0 ? kept_block(a, k, k.start + node) : -1;
      if (from >= 0) {
        moves = true;
        scale = fmaxf(scale, scale_of(from));
      }
    }
    if (moves) {
      if (scale != had) {
        for (int at = 0; at < a.block_size; ++at) recode(row(block, at), row(block, at), had * inverse_pow2(scale));
      }
      for (int i = j; i < stop; ++i) {
        const int node = a.nodes[k.first + i];
        const int p = k.start + node;
        const int from = node != i ? kept_block(a, k, p) : -1;
        if (from < 0) continue;
        const float own = from == block ? scale : scale_of(from);
        recode(row(from, p % a.block_size), row(block, (k.start + i) % a.block_size), own * inverse_pow2(scale));
      }
      if (scale != had && lane == 0) scales[static_cast<int64_t>(block) * a.num_kv_heads] = scale;
    }
    j = last;
  }
}

template <typename T>
hipError_t launch_merge_t(const MergeTreeArgs& a, int head_dim, dim3 grid, hipStream_t s) {
  switch (head_dim) {
    case 64: hipLaunchKernelGGL((merge_tree_kernel<T, 64>), grid, dim3(kTreeThreads), 0, s, a); break;
    case 80: hipLaunchKernelGGL((merge_tree_kernel<T, 80>), grid, dim3(kTreeThreads), 0, s, a); break;
    case 96: hipLaunchKernelGGL((merge_tree_kernel<T, 96>), grid, dim3(kTreeThreads), 0, s, a); break;
    case 256: hipLaunchKernelGGL((merge_tree_kernel<T, 256>), grid, dim3(kTreeThreads), 0, s, a); break;
    case 128: hipLaunchKernelGGL((merge_tree_kernel<T, 128>), grid, dim3(kTreeThreads), 0, s, a); break;
    default: return hipErrorNotSupported;
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_pack_tree(const PackTreeArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(pack_tree_kernel, dim3(static_cast<uint32_t>(a.num_seqs)), dim3(kTreeThreads), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_accept_tree(const AcceptTreeArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(accept_tree_kernel, dim3(static_cast<uint32_t>(a.num_seqs)), dim3(kWave), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_keep_rows(const KeepRowsArgs& a, hipStream_t stream) {
  const uint32_t seqs = static_cast<uint32_t>(a.num_seqs), tensors = 2 * static_cast<uint32_t>(a.num_layers);
  if (a.key_scales != nullptr) {
    hipLaunchKernelGGL(keep_rows8_kernel, dim3(seqs, tensors, a.num_kv_heads), dim3(kWave), 0, stream, a);
    return hipGetLastError();
  }
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.key_cache) | reinterpret_cast<uintptr_t>(a.value_cache) |
                       static_cast<uintptr_t>(a.row_bytes);
  auto threads = [&](int64_t piece) {
    return dim3(static_cast<uint32_t>(std::min<int64_t>(kTreeThreads, (a.row_bytes / piece + kWave - 1) / kWave * kWave)));
  };
  if ((at & 15) == 0)
    hipLaunchKernelGGL(keep_rows_kernel<uint4>, dim3(seqs, tensors), threads(16), 0, stream, a);
  else if ((at & 3) == 0)
    hipLaunchKernelGGL(keep_rows_kernel<uint32_t>, dim3(seqs, tensors), threads(4), 0, stream, a);
  else
    hipLaunchKernelGGL(keep_rows_kernel<uint16_t>, dim3(seqs, tensors), threads(2), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_merge_tree(const MergeTreeArgs& a, int dtype, int head_dim, hipStream_t stream) {
  if (a.num_merge <= 0) return hipSuccess;
  const int threads = a.num_query_heads * (head_dim / 4);
  const dim3 grid(static_cast<uint32_t>(a.num_merge * a.tile), (threads + kTreeThreads - 1) / kTreeThreads);
  if (dtype == PA_DTYPE_F32) return launch_merge_t<float>(a, head_dim, grid, stream);
  if (dtype == PA_DTYPE_BF16) return launch_merge_t<bf16_t>(a, head_dim, grid, stream);
  if (dtype == PA_DTYPE_F16) return launch_merge_t<f16_t>(a, head_dim, grid, stream);
  return hipErrorNotSupported;
}

}  // namespace pa
