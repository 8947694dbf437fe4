// rotate_and_cache: the projections' Q, K and V rows of a step, Q and K
// normalised per head and rotated to their positions, Q written out, K and V
// appended to the paged cache; and the 8-bit cache's write, of rotated rows or
// of rows as they are.
//
//   norm     y_i = x_i * rsqrt(mean(x^2) + eps) * w_i
//   rotation (a, b) -> (a cos - b sin, b cos + a sin), the pairs (i, i + R/2)
//            or (2i, 2i + 1) of the first R elements, with the cosine and sine
//            of the token's position from a table; the others stay
// in fp32, rounded once, to the rows' type.
//
// A row (token, head) belongs to a group of L lanes (8 elements a lane), so
// its sum of squares is a few DPP additions, a lane holds both elements of its
// pairs, and the cosines and sines a lane needs are one 16-byte load each.
//
// What bounds it is memory once a step has some ten thousand rows, and before
// that the launch and two dependent reads (position, then table).  bf16 rows,
// cold caches: 8 tokens of 32/8 heads of 128 3.2 us; 2176 tokens with norms
// (54.6 MB) 17.5 us, 3.1 TB/s; the rotation alone, 4096 tokens with norms (86 MB)
// 25.8 us, 3.3 TB/s.  The 8-bit write: 256 decode tokens 6.8 us; 1406 tokens of
// 32/32 heads of 128, fp16 with norms (58 MB) 25.2 us; 20183 tokens of 9/3 heads
// of 64 (75 MB) 25.9 us, 2.9 TB/s: there each chunk reads the rows that may belong
// to its last run, which the next one reads again, and waits for slots, rows and
// scales one after the other.
#include "cache8.hpp"
#include "pa_common.hpp"
#include "pa_launch.hpp"

namespace pa {

constexpr int kRotateThreads = 256;

// Four elements in memory, as floats, and back (rounded to nearest even).
template <typename T>
struct Four {
  using type = uint2;
};
template <>
struct Four<float> {
  using type = float4;
};
template <typename T>
__device__ __forceinline__ typename Four<T>::type load4(const T* p) {
  return *reinterpret_cast<const typename Four<T>::type*>(p);
}
template <typename T>
__device__ __forceinline__ void unpack4(typename Four<T>::type v, float* x) {
  if constexpr (sizeof(T) == 4) {
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    x[0] = half_lo<T>(v.x), x[1] = half_hi<T>(v.x), x[2] = half_lo<T>(v.y), x[3] = half_hi<T>(v.y);
  }
}
template <typename T>
__device__ __forceinline__ typename Four<T>::type pack4(const float* x) {
  if constexpr (sizeof(T) == 4) return make_float4(x[0], x[1], x[2], x[3]);
  else return make_uint2(pack_half2<T>(x[0], x[1]), pack_half2<T>(x[2], x[3]));
}
// x as its type holds it.
template <typename T>
__device__ __forceinline__ float rounded(float x) {
  if constexpr (sizeof(T) == 4) return x;
  else return half_lo<T>(pack_half2<T>(x, x));
}

// Sum over the L lanes of a row.
template <int L>
__device__ __forceinline__ float row_sum(float x) {
  x = group_sum<(L < 16 ? L : 16)>(x);
  if constexpr (L >= 32) x = sum_row_pairs(x);
  if constexpr (L >= 64) x = sum_halves(x);
  return x;
}
template <int L>
__device__ __forceinline__ float row_max(float x) {
  x = fmaxf(x, dpp<kDppQuadXor1>(x));
  x = fmaxf(x, dpp<kDppQuadXor2>(x));
  x = fmaxf(x, dpp<kDppRowHalfMirror>(x));
  if constexpr (L >= 16) x = fmaxf(x, dpp<kDppRowMirror>(x));
  if constexpr (L >= 32) x = max_row_pairs(x);
  if constexpr (L >= 64) x = max_halves(x);
  return x;
}

// What a lane of a row's group does with its row.  VEC: 8 elements, in two
// runs of 4 at `a` and `b` (the two halves of its pairs, or 8 in a row);
// needs D and R in multiples of 8 and rows at multiples of 4 elements.  Lanes
// past the row load its first pieces, so that no load waits behind a branch.
// Else elements lane + 64 e, each with its partner read again; any D up to 256.
template <typename T, int L, bool VEC>
struct RowLane {
  static constexpr int kN = VEC ? 8 : 4;
  using Piece = typename Four<T>::type;
  struct Raw {
    Piece lo, hi;  // VEC: as they are in memory
  };
  const RotateArgs& args;
  int lane;  // in the row's group
  int a, b;  // VEC
  bool live, turns;

  __device__ __forceinline__ RowLane(const RotateArgs& r, int l) : args(r), lane(l) {
    if constexpr (VEC) {
      turns = 8 * l < r.rotary_dim;
      live = 8 * l < r.head_dim;
      const bool halves = turns && !r.interleaved;
      a = halves ? 4 * l : 8 * l;
      b = halves ? r.rotary_dim / 2 + 4 * l : 8 * l + 4;
      if (!live) a = b = 0;
    } else {
      turns = live = true;
      a = b = 0;
    }
  }
  __device__ __forceinline__ Raw load_raw(const T* row) const {
    Raw v{};
    if constexpr (VEC) {
      v.lo = load4<T>(row + a);
      v.hi = load4<T>(row + b);
    }
    return v;
  }
  // The row as floats (zeros past its end).
  __device__ __forceinline__ void unpack(const Raw& v, const T* row, float* x) const {
    if constexpr (VEC) {
      unpack4<T>(v.lo, x);
      unpack4<T>(v.hi, x + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = live ? x[i] : 0.f;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = lane + 64 * e;
        x[e] = d < args.head_dim ? load_scalar<T>(row + d) : 0.f;
      }
    }
  }
  // Stores x, or (`copy`) the raw row.
  __device__ __forceinline__ void store(T* row, const float* x, const Raw& v, bool copy) const {
    if constexpr (VEC) {
      Piece lo = pack4<T>(x), hi = pack4<T>(x + 4);
      if (copy) {
        lo = v.lo;
        hi = v.hi;
      }
      if (live) {
        *reinterpret_cast<Piece*>(row + a) = lo;
        *reinterpret_cast<Piece*>(row + b) = hi;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (lane + 64 * e < args.head_dim) store_scalar<T>(row + lane + 64 * e, x[e]);
    }
  }
  __device__ __forceinline__ float weight(const void* w, int d) const {
    return args.weight_f32 ? static_cast<const float*>(w)[d] : load_scalar<T>(static_cast<const T*>(w) + d);
  }
  // VEC: the lane's cosines and sines at a position of the table.
  __device__ __forceinline__ void angles(int64_t pos, float4* c, float4* s) const {
    *c = *s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (args.rotary_dim > 0) {
      const float* cs = args.cos_sin + pos * args.rotary_dim + (turns ? 4 * lane : 0);
      *c = *reinterpret_cast<const float4*>(cs);
      *s = *reinterpret_cast<const float4*>(cs + args.rotary_dim / 2);
    }
  }
  // VEC: the lane's norm weights.
  __device__ __forceinline__ void weights(const void* w, float* g) const {
    if (args.weight_f32) {
      unpack4<float>(load4<float>(static_cast<const float*>(w) + a), g);
      unpack4<float>(load4<float>(static_cast<const float*>(w) + b), g + 4);
    } else {
      unpack4<T>(load4<T>(static_cast<const T*>(w) + a), g);
      unpack4<T>(load4<T>(static_cast<const T*>(w) + b), g + 4);
    }
  }
  // The norm's factor of the row x holds.  (No contraction but the fmaf
  // written here, in these three: the kernels below give the same bits.)
  __device__ __forceinline__ float norm(const float* x) const {
#pragma clang fp contract(off)
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < kN; ++i) ss = fmaf(x[i], x[i], ss);
    return rsqrtf(row_sum<L>(ss) / static_cast<float>(args.head_dim) + args.eps);
  }
  // VEC: normalise (`normed`, with the weights g) and rotate the row x holds.
  __device__ __forceinline__ void apply(float* x, bool normed, const float* g, const float4& c4, const float4& s4) const {
#pragma clang fp contract(off)
    if (normed) {
      const float r = norm(x);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * r * g[i];
    }
    if (turns) {
      auto turn = [](float& p, float& q, float c, float s) {
        const float u = p, v = q;
        p = fmaf(u, c, -(v * s));
        q = fmaf(v, c, u * s);
      };
      if (args.interleaved) {
        turn(x[0], x[1], c4.x, s4.x);
        turn(x[2], x[3], c4.y, s4.y);
        turn(x[4], x[5], c4.z, s4.z);
        turn(x[6], x[7], c4.w, s4.w);
      } else {
        turn(x[0], x[4], c4.x, s4.x);
        turn(x[1], x[5], c4.y, s4.y);
        turn(x[2], x[6], c4.z, s4.z);
        turn(x[3], x[7], c4.w, s4.w);
      }
    }
  }
  // Not VEC: the same, each partner read again from the row.
  __device__ __forceinline__ void apply_any(const T* row, float* x, const void* w, int64_t pos) const {
#pragma clang fp contract(off)
    const float r = w != nullptr ? norm(x) : 1.f;
    const int rot = args.rotary_dim;
    const float* cs = args.cos_sin + pos * rot;  // (not read without rotation)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = lane + 64 * e;
      if (d >= args.head_dim) continue;
      float u = x[e];
      if (w != nullptr) u = u * r * weight(w, d);
      if (d < rot) {
        const bool second = args.interleaved ? d & 1 : d >= rot / 2;
        const int o = args.interleaved ? d ^ 1 : second ? d - rot / 2 : d + rot / 2;
        const int k = args.interleaved ? d / 2 : second ? o : d;
        float v = load_scalar<T>(row + o);
        if (w != nullptr) v = v * r * weight(w, o);
        const float vs = v * cs[rot / 2 + k];
        u = fmaf(u, cs[k], second ? vs : -vs);
      }
      x[e] = u;
    }
  }
  __device__ __forceinline__ void invalidate(float* x) const {
#pragma unroll
    for (int i = 0; i < kN; ++i) x[i] = __builtin_nanf("");
  }
};

// A token's position, 0 (and not ok) where it lies outside the table: its Q
// rows are NaN then, so that no such call passes for a result, and its K rows
// are not cached.
__device__ __forceinline__ int64_t position_of(const RotateArgs& a, int64_t t, bool* ok) {
  const int64_t pos = a.rotary_dim > 0 ? a.positions[t] : 0;
  *ok = a.rotary_dim == 0 || (pos >= 0 && pos < a.num_positions);
  return *ok ? pos : 0;
}

// Heads h0 .. h0 + NR - 1 of token t, of the heads of Q, K, V in this order
// (`heads` of them): K and V go to the cache's slot, or (no cache) K to
// key_out.  Every load is issued before the first row is finished, and the
// rows share the token's angles.
template <typename T, int L, bool VEC, int NR>
__device__ __forceinline__ void rotate_rows(const RotateArgs& a, const RowLane<T, L, VEC>& ln, int64_t t, int h0,
                                            int heads) {
  const T* src[NR];
  typename RowLane<T, L, VEC>::Raw raw[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    int h = min(h0 + i, heads - 1);
    const bool is_q = h < a.num_query_heads;
    if (!is_q) h -= a.num_query_heads;
    const bool is_v = !is_q && h >= a.num_kv_heads;
    if (is_v) h -= a.num_kv_heads;
    src[i] = reinterpret_cast<const T*>(is_q ? a.query : is_v ? a.value : a.key) +
             t * (is_q ? a.q_token_stride : is_v ? a.v_token_stride : a.k_token_stride) +
             h * (is_q ? a.q_head_stride : is_v ? a.v_head_stride : a.k_head_stride);
    raw[i] = ln.load_raw(src[i]);
  }
  const int64_t slot = a.slot_mapping != nullptr ? a.slot_mapping[t] : 0;
  bool ok;
  const int64_t pos = position_of(a, t, &ok);
  const bool any_norm = a.query_weight != nullptr || a.key_weight != nullptr;
  float qg[8] = {}, kg[8] = {};  // the weights of Q rows and of K rows
  float4 c, s;
  if constexpr (VEC) {
    if (any_norm) {
      ln.weights(a.query_weight != nullptr ? a.query_weight : a.key_weight, qg);
      ln.weights(a.key_weight != nullptr ? a.key_weight : a.query_weight, kg);
    }
    ln.angles(pos, &c, &s);
  }
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int h = h0 + i;
    const bool is_q = h < a.num_query_heads;
    const bool is_v = h >= a.num_query_heads + a.num_kv_heads;
    const void* w = is_q ? a.query_weight : a.key_weight;
    float x[RowLane<T, L, VEC>::kN];
    ln.unpack(raw[i], src[i], x);
    if constexpr (VEC) {
      float g[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) g[k] = is_q ? qg[k] : kg[k];
      ln.apply(x, any_norm && w != nullptr, g, c, s);
    } else {
      if (!is_v && h < heads) ln.apply_any(src[i], x, w, pos);
    }
    if (!is_v && !ok) ln.invalidate(x);
    T* out;
    bool keep = h < heads;
    if (is_q) {
      out = reinterpret_cast<T*>(a.query_out) + t * a.q_out_token_stride + h * a.q_out_head_stride;
    } else if (a.key_cache != nullptr) {
      keep = keep && slot >= 0 && slot < a.num_slots && (is_v || ok);
      const int kv = h - a.num_query_heads - (is_v ? a.num_kv_heads : 0);
      out = reinterpret_cast<T*>(is_v ? a.value_cache : a.key_cache) + (slot * a.num_kv_heads + kv) * a.head_dim;
    } else {
      out = reinterpret_cast<T*>(a.key_out) + t * a.k_out_token_stride + (h - a.num_query_heads) * a.k_out_head_stride;
    }
    if (keep) ln.store(out, x, raw[i], is_v);
  }
}

// Every row of the step, NR heads of a token to a group of lanes.
template <typename T, int L, bool VEC, int NR>
__global__ __launch_bounds__(kRotateThreads) void rotate_kernel(RotateArgs a) {
  const int heads = a.num_query_heads + (a.key_cache != nullptr ? 2 : 1) * a.num_kv_heads;
  const uint32_t units = (heads + NR - 1) / NR;  // per token
  const uint32_t id = blockIdx.x * (kRotateThreads / L) + threadIdx.x / L;
  const uint32_t tok = quotient(id, units, a.heads_rcp);
  if (tok >= static_cast<uint32_t>(a.num_tokens)) return;
  const RowLane<T, L, VEC> ln(a, threadIdx.x % L);
  rotate_rows<T, L, VEC, NR>(a, ln, tok, static_cast<int>(id - tok * units) * NR, heads);
}

// The 8-bit cache's write.  The first a.kv_groups workgroups take (chunk of
// tokens, KV head, tensor) each, the others rows of Q.
//
// A block's scale depends on all of its rows, so one workgroup has to see
// every row the step brings for the block.  Those follow each other in the
// step: a chunk owns the runs (tokens of one block) that begin in it, and so
// looks at up to block_size - 1 tokens past its end and leaves the first ones
// to the chunk before where their run began there.  It takes the rows' largest
// magnitudes (kept in LDS by an integer maximum of the floats' bits, which no
// order changes), settles the scales, and writes the codes.  KEPT: the span is
// at most this many rows a group, which are loaded first of all, beside the
// slots, and stay in registers; 0: the rows are read (and rotated) again.  A run
// that holds its block's first row starts the block afresh; the other rows of
// any other block are re-coded if its scale grows.
template <typename T, int L, bool VEC, int KEPT, int NR>
__global__ __launch_bounds__(kRotateThreads) void cache8_write_kernel(RotateArgs a) {
  constexpr int C = kRotateThreads / L;                 // rows at once
  constexpr int kOwn = KEPT > 0 ? (KEPT - 1) * C : C;   // tokens of a chunk
  constexpr bool KEEP = KEPT > 0;
  static_assert(kOwn <= kWave, "a lane for each of its runs");
  constexpr int kN = RowLane<T, L, VEC>::kN;
  const RowLane<T, L, VEC> ln(a, threadIdx.x % L);
  const int group = threadIdx.x / L;
  if (blockIdx.x >= a.kv_groups) {
    const uint32_t units = (a.num_query_heads + NR - 1) / NR;
    const uint32_t id = (blockIdx.x - a.kv_groups) * C + group;
    const uint32_t tok = quotient(id, units, a.heads_rcp);
    if (tok >= static_cast<uint32_t>(a.num_tokens)) return;
    rotate_rows<T, L, VEC, NR>(a, ln, tok, static_cast<int>(id - tok * units) * NR, a.num_query_heads);
    return;
  }
  // Per run that begins in the chunk (at token kOwn c + i): its block, whether it
  // holds the block's first row, its largest magnitude's bits, the scale the
  // block has (0 if it starts afresh); and one past the last run's last token.
  __shared__ int64_t s_block[kOwn];
  __shared__ int s_fresh[kOwn], s_end;
  __shared__ uint32_t s_amax[kOwn];
  __shared__ float s_old[kOwn];
  // Per token of the span: the run it belongs to (< 0: none of the chunk's),
  // and its row of the cache.
  __shared__ int16_t s_run[kOwn + kMaxCache8Block];
  __shared__ int64_t s_slot[kOwn + kMaxCache8Block];

  const uint32_t units = 2 * a.num_kv_heads;
  const uint32_t chunk = quotient(blockIdx.x, units, a.kv_rcp);
  const int u = static_cast<int>(blockIdx.x - chunk * units);
  const bool is_v = u >= a.num_kv_heads;
  const int h = is_v ? u - a.num_kv_heads : u;
  const int64_t t0 = static_cast<int64_t>(chunk) * kOwn;
  const int span = static_cast<int>(min<int64_t>(kOwn + a.block_size - 1, a.num_tokens - t0));
  const T* src = reinterpret_cast<const T*>(is_v ? a.value : a.key) + h * (is_v ? a.v_head_stride : a.k_head_stride);
  const int64_t tok_stride = is_v ? a.v_token_stride : a.k_token_stride;
  const void* w = is_v ? nullptr : a.key_weight;
  // Row j as it is given, with what turning it takes; then as the 16-bit cache
  // would hold it (false if it is not cached).
  using Raw = typename RowLane<T, L, VEC>::Raw;
  float g[8] = {};
  if constexpr (VEC)
    if (w != nullptr) ln.weights(w, g);
  auto load_row = [&](int j, Raw* raw, int64_t* pos, bool* ok, float4* c, float4* s) {
    *ok = true;
    *pos = 0;
    *raw = ln.load_raw(src + (t0 + j) * tok_stride);
    if (!is_v) {
      *pos = position_of(a, t0 + j, ok);
      if constexpr (VEC) ln.angles(*pos, c, s);
    }
  };
  auto finish_row = [&](int j, const Raw& raw, float* x, int64_t pos, const float4& c, const float4& s) {
    ln.unpack(raw, src + (t0 + j) * tok_stride, x);
    if (!is_v) {
      if constexpr (VEC) ln.apply(x, w != nullptr, g, c, s);
      else ln.apply_any(src + (t0 + j) * tok_stride, x, w, pos);
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      x[i] = rounded<T>(x[i]);
      if (fabsf(x[i]) < INFINITY) x[i] = fminf(fmaxf(x[i], -kMaxRow8<T>), kMaxRow8<T>);
    }
  };
  constexpr int kKept = KEEP ? KEPT : 1;
  float x[kKept][kN];
  Raw raw[kKept];
  float4 cs[kKept], sn[kKept];
  int64_t pos[kKept];
  bool ok[kKept];
  if constexpr (KEEP) {
#pragma unroll
    for (int k = 0; k < kKept; ++k)
      load_row(min(group + k * C, span - 1), &raw[k], &pos[k], &ok[k], &cs[k], &sn[k]);
  }

  float* scales = (is_v ? a.value_scales : a.key_scales) + h;
  float old = 0.f;  // lane i < kOwn of the first wave: the scale of run i's block
  if (threadIdx.x < kOwn) {
    s_block[threadIdx.x] = -1;
    s_end = 0;
    s_fresh[threadIdx.x] = 0;
    s_amax[threadIdx.x] = 0;
  }
  if (threadIdx.x < kWave) {
    // A slot's block, -1 outside the pool.
    auto split = [&](int64_t slot, int* row) -> int64_t {
      if (slot < 0 || slot >= a.num_slots) {
        *row = 0;
        return -1;
      }
      if (a.log2_block >= 0) {
        *row = static_cast<int>(slot) & (a.block_size - 1);
        return slot >> a.log2_block;
      }
      const int64_t b = slot / a.block_size;
      *row = static_cast<int>(slot - b * a.block_size);
      return b;
    };
    int row;
    int64_t before = t0 > 0 ? split(a.slot_mapping[t0 - 1], &row) : -1;  // the block of the token ahead of the batch
    int last = -1;                                                       // the run that token ends
    for (int base = 0; base < span; base += kWave) {
      const int j = base + threadIdx.x;
      const int64_t slot = j < span ? a.slot_mapping[t0 + j] : -1;
      const int64_t blk = split(slot, &row);
      int64_t prev = __shfl_up(blk, 1, kWave);
      if (threadIdx.x == 0) prev = before;
      before = __shfl(blk, kWave - 1, kWave);
      const bool starts = blk != prev;
      const uint64_t mask = __ballot(starts);
      const uint64_t upto = mask & (~uint64_t{0} >> (kWave - 1 - threadIdx.x));
      const int lead = upto != 0 ? base + 63 - __builtin_clzll(upto) : last;
      const bool ours = lead >= 0 && lead < kOwn && blk >= 0;
      if (j < span) {
        s_run[j] = static_cast<int16_t>(ours ? lead : -1);
        s_slot[j] = slot;
      }
      if (ours) {
        if (starts) s_block[lead] = blk;
        atomicMax(&s_end, j + 1);
        if (row == 0) s_fresh[lead] = 1;
      }
      if (mask != 0) last = base + 63 - __builtin_clzll(mask);
      // (run i begins at token i, so its lane holds its block)
      if (base == 0 && threadIdx.x < kOwn && ours && starts) old = scale_pow2(scales[blk * a.num_kv_heads]);
    }
  }
  __syncthreads();
  // Rows past the last run that begins in the chunk are not the chunk's.
  const int end = s_end;
  auto note = [&](int run, const float* y) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const float v = fabsf(y[i]);
      m = fmaxf(m, v < INFINITY ? v : 0.f);
    }
    m = row_max<L>(m);
    if (ln.lane == 0) atomicMax(&s_amax[run], __float_as_uint(m));
  };
  if constexpr (KEEP) {
#pragma unroll
    for (int k = 0; k < kKept; ++k) {
      const int j = group + k * C;
      const int run = j < end ? s_run[j] : -1;
      ok[k] = run >= 0 && ok[k];
      if (ok[k]) {
        finish_row(j, raw[k], x[k], pos[k], cs[k], sn[k]);
        note(run, x[k]);
      }
    }
  } else {
    for (int j = group; j < end; j += C) {
      if (s_run[j] < 0) continue;
      load_row(j, &raw[0], &pos[0], &ok[0], &cs[0], &sn[0]);
      finish_row(j, raw[0], x[0], pos[0], cs[0], sn[0]);
      if (ok[0]) note(s_run[j], x[0]);
    }
  }
  if (threadIdx.x < kOwn) s_old[threadIdx.x] = s_fresh[threadIdx.x] ? 0.f : old;
  __syncthreads();
  auto new_scale = [&](int run) { return fmaxf(s_old[run], scale_for(__uint_as_float(s_amax[run]))); };
  // What the other rows of a run's block are re-coded by (1: not at all).
  auto recode = [&](int run) {
    return s_block[run] < 0 || s_fresh[run] ? 1.f : s_old[run] * inverse_pow2(new_scale(run));
  };
  if (threadIdx.x < kOwn && s_block[threadIdx.x] >= 0)
    scales[s_block[threadIdx.x] * a.num_kv_heads] = new_scale(threadIdx.x);
  uint8_t* cache = reinterpret_cast<uint8_t*>(is_v ? a.value_cache : a.key_cache) + h * a.head_dim;
  const int64_t row_codes = static_cast<int64_t>(a.num_kv_heads) * a.head_dim;
  // Blocks whose scale grew: all of their rows; the run's own follow below.
  const int lane = threadIdx.x % kWave;
  if (__any(lane < kOwn && recode(min(lane, kOwn - 1)) != 1.f)) {  // (alike in every wave)
    for (int i = 0; i < kOwn; ++i) {
      const float ratio = recode(i);
      if (ratio == 1.f) continue;
      uint8_t* rows = cache + s_block[i] * a.block_size * row_codes;
      if constexpr (VEC) {
        const int words = a.head_dim / 4;
        for (int k = threadIdx.x; k < a.block_size * words; k += kRotateThreads) {
          const int r = k / words;
          uint32_t* p = reinterpret_cast<uint32_t*>(rows + r * row_codes) + (k - r * words);
          const uint32_t v = *p;
          *p = pack_codes4(code_to_f32<0>(v) * ratio, code_to_f32<1>(v) * ratio, code_to_f32<2>(v) * ratio,
                           code_to_f32<3>(v) * ratio);
        }
      } else {
        for (int k = threadIdx.x; k < a.block_size * a.head_dim; k += kRotateThreads) {
          const int r = k / a.head_dim;
          uint8_t* p = rows + r * row_codes + (k - r * a.head_dim);
          *p = static_cast<uint8_t>(pack_codes2(code_to_f32<0>(*p) * ratio, 0.f));
        }
      }
    }
    __syncthreads();  // (orders the stores of a row's two writes)
  }
  auto write = [&](int j, const float* y) {
    const float inv = inverse_pow2(new_scale(s_run[j]));
    uint8_t* out = cache + s_slot[j] * row_codes;
    if constexpr (VEC) {
      if (ln.live) {
        *reinterpret_cast<uint32_t*>(out + ln.a) = pack_codes4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
        *reinterpret_cast<uint32_t*>(out + ln.b) = pack_codes4(y[4] * inv, y[5] * inv, y[6] * inv, y[7] * inv);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (ln.lane + 64 * e < a.head_dim)
          out[ln.lane + 64 * e] = static_cast<uint8_t>(pack_codes2(y[e] * inv, 0.f));
    }
  };
  if constexpr (KEEP) {
#pragma unroll
    for (int k = 0; k < kKept; ++k)
      if (ok[k]) write(group + k * C, x[k]);
  } else {
    for (int j = group; j < end; j += C) {
      if (s_run[j] < 0) continue;
      load_row(j, &raw[0], &pos[0], &ok[0], &cs[0], &sn[0]);
      finish_row(j, raw[0], x[0], pos[0], cs[0], sn[0]);
      if (ok[0]) write(j, x[0]);
    }
  }
}

// Lanes the device holds at a time: 2048 on each of its CUs (a whole chip's 256
// where their count is unknown).
static int64_t resident_lanes() {
  const int cus = device_compute_units();
  return 2048 * static_cast<int64_t>(cus > 0 ? cus : 256);
}

template <typename T, int L, bool VEC, int NR>
static hipError_t launch_rotate_n(const RotateArgs& args, hipStream_t s) {
  constexpr int kRows = kRotateThreads / L;
  RotateArgs a = args;
  const bool codes = a.key_scales != nullptr;
  const uint32_t heads =
      codes ? a.num_query_heads : a.num_query_heads + (a.key_cache != nullptr ? 2 : 1) * a.num_kv_heads;
  const uint32_t units = (heads + NR - 1) / NR;
  const int64_t groups = static_cast<int64_t>(a.num_tokens) * units;
  const uint32_t grid = static_cast<uint32_t>((groups + kRows - 1) / kRows);
  a.heads_rcp = units > 0 ? 0xffffffffu / units : 0;
  if (!codes) {
    hipLaunchKernelGGL((rotate_kernel<T, L, VEC, NR>), dim3(grid), dim3(kRotateThreads), 0, s, a);
    return hipGetLastError();
  }
  a.kv_rcp = 0xffffffffu / (2 * a.num_kv_heads);
  // Three rows a group, so that a chunk re-reads half as much of its
  // neighbour's, once its rows of K and V alone would fill the chip (see
  // resident_lanes); a chunk of two has less to wait for.  Two against three:
  // bf16, 32/8 heads of 128, 256 tokens 6.1 / 7.5 us, 1024 10.0 / 11.2, 2048
  // 17.4 / 16.7; fp16, 32/32 of 128, 384 tokens 10.4 / 11.2, 512 13.4 / 12.8,
  // 4096 69.1 / 61.8; 9/3 heads of 64, 8192 tokens 13.5 / 13.9, 16384 23.5 /
  // 22.3; 8/2 heads of 256 in blocks of 8, 2048 tokens 10.0 / 10.8, 8192 31.7 /
  // 29.1.  Blocks longer than a group's rows at once and one (33 tokens for heads
  // of 64, 17 up to 128, 9 above) would need a span that does not fit the
  // registers: their rows are loaded, normalised and turned twice.  bf16 32/8
  // heads of 128, blocks of 16 and of 32: 256 tokens 7.2 / 7.4 us, 2048 17.5 /
  // 21.9, 8192 53.5 / 73.6; 8/2 of 256, blocks of 8 and of 16: 6.6 / 6.6, 10.3 /
  // 14.0, 29.2 / 39.1.
  const bool keep = a.block_size <= kRows + 1;
  const bool three = keep && static_cast<int64_t>(a.num_tokens) * 2 * a.num_kv_heads * L >= resident_lanes();
  const int own = three ? 2 * kRows : kRows;
  a.kv_groups = static_cast<uint32_t>((a.num_tokens + own - 1) / own * (2 * a.num_kv_heads));
  a.log2_block = -1;
  for (int i = 0; i <= 8; ++i)
    if (1 << i == a.block_size) a.log2_block = i;
  if (three)
    hipLaunchKernelGGL((cache8_write_kernel<T, L, VEC, 3, NR>), dim3(a.kv_groups + grid), dim3(kRotateThreads), 0, s, a);
  else if (keep)
    hipLaunchKernelGGL((cache8_write_kernel<T, L, VEC, 2, NR>), dim3(a.kv_groups + grid), dim3(kRotateThreads), 0, s, a);
  else
    hipLaunchKernelGGL((cache8_write_kernel<T, L, VEC, 0, NR>), dim3(a.kv_groups + grid), dim3(kRotateThreads), 0, s, a);
  return hipGetLastError();
}

// Two heads to a group of lanes once one each would take more lanes than the
// chip holds: from there on loads in flight are what counts, and below it the
// depth of one row's work.  One against two, bf16, 32/8 heads of 128 with
// norms: 256 tokens 4.6 / 4.9 us, 512 6.7 / 6.7, 768 9.7 / 8.7, 4096 36.3 /
// 28.9; 9/3 heads of 64: 1024 tokens 3.9 / 4.2 us, 4096 7.2 / 7.2; fp32, 8/8
// heads of 64: 1024 5.6 / 6.2 us, 4096 13.3 / 13.4.  Four: 18.2 us where two
// took 17.9 and one 21.3.
template <typename T, int L, bool VEC>
static hipError_t launch_rotate_l(const RotateArgs& a, hipStream_t s) {
  if constexpr (VEC) {
    const int64_t rows = static_cast<int64_t>(a.num_tokens) * (a.num_query_heads + 2 * a.num_kv_heads);
    if (rows * L > resident_lanes()) return launch_rotate_n<T, L, VEC, 2>(a, s);
  }
  return launch_rotate_n<T, L, VEC, 1>(a, s);
}

template <typename T>
static hipError_t launch_rotate_t(const RotateArgs& a, bool vec, hipStream_t s) {
  if (!vec) return launch_rotate_l<T, 64, false>(a, s);
  return a.head_dim <= 64    ? launch_rotate_l<T, 8, true>(a, s)
         : a.head_dim <= 128 ? launch_rotate_l<T, 16, true>(a, s)
                             : launch_rotate_l<T, 32, true>(a, s);
}

hipError_t launch_rotate(const RotateArgs& a, int dtype, hipStream_t s) {
  if (a.num_tokens <= 0) return hipSuccess;
  // Runs of 4 elements: rows and their strides at multiples of 4 (of 16 bytes
  // for fp32), 16 bytes of the table.
  const int64_t eb = dtype == PA_DTYPE_F32 ? 4 : 2;
  const auto fits = [&](const void* p, int64_t tok, int64_t head) {
    return reinterpret_cast<uintptr_t>(p) % (4 * eb) == 0 && tok % 4 == 0 && head % 4 == 0;
  };
  const bool q = a.num_query_heads == 0 || (fits(a.query, a.q_token_stride, a.q_head_stride) &&
                                            fits(a.query_out, a.q_out_token_stride, a.q_out_head_stride));
  const bool vec = a.head_dim % 8 == 0 && a.rotary_dim % 8 == 0 && q && fits(a.key, a.k_token_stride, a.k_head_stride) &&
                   fits(a.value, a.v_token_stride, a.v_head_stride) &&
                   fits(a.key_out, a.k_out_token_stride, a.k_out_head_stride) && fits(a.key_cache, 0, 0) &&
                   fits(a.value_cache, 0, 0) && reinterpret_cast<uintptr_t>(a.cos_sin) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(a.query_weight) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(a.key_weight) % 16 == 0;
  switch (dtype) {
    case PA_DTYPE_F32: return launch_rotate_t<float>(a, vec, s);
    case PA_DTYPE_BF16: return launch_rotate_t<bf16_t>(a, vec, s);
    case PA_DTYPE_F16: return launch_rotate_t<f16_t>(a, vec, s);
    default: return hipErrorNotSupported;
  }
}

}  // namespace pa
