// Paged-attention decode over the 8-bit cache on the matrix cores: bf16 or
// fp16 queries, heads of 64 and 128, and of 80 and 96 on the LDS rows of 128.
//
// The split, the operand layouts, the softmax and the merge are those of
// decode_mfma.hip: one workgroup per (sequence, context partition, KV head, or
// two or four adjacent ones), S^T = K Q^T and O^T = V^T P^T by v_mfma_f32_16x16x32 of
// the query's type, probabilities as two terms of it.  What differs:
//  * Codes become 16-bit values in registers, between LDS and the product (K)
//    or between the row pieces and the product (V), by v_cvt_scalef32_pk_*_fp8,
//    which takes the block's scale along: 64 conversions for the 24 products
//    of a tile (heads of 128), no multiplication.  A lane's 16-byte piece of K
//    is two operands, so the query's pieces are 8 of 16 elements each.  V is
//    transposed as bytes, two tokens' codes of a dim side by side (v_perm_b32
//    on 4 dims at once), before it is converted.
//  * The scales of a tile's blocks come into LDS with its K rows (lane i loads
//    the i-th of them), ahead of the K copies, so the wait for those covers
//    them.
// What bounds it is HBM: half the bytes a token of the 16-bit cache, and 4 to 8
// flops a byte of a group's heads, far below what the matrix units do.  bf16,
// 256 sequences of 32-8192 tokens, 32/8 heads of 128 (778 MB): 143 us, 5.4 TB/s
// (a pure read: 7.0); two of 60000-131000 (475 MB): 83 us, 5.7; fp16, 64 of
// 128-4096, 32/32 heads (1.18 GB): 198 us, 6.0.  Between these and the read
// rate lie workgroups of unequal length on a CU's last round and the reads of
// ids and scales ahead of a workgroup's first rows.  Eight sequences of 16-512
// tokens, 8/8 heads of 64: 6.9 us, a chain of dependent reads.
#include <type_traits>

#include "cache8.hpp"
#include "decode_common.hpp"
#include "decode_mfma_common.hpp"
#include "span.hpp"

namespace pa {

constexpr int kTile8 = 32;           // context tokens per wave iteration: two groups of 16
// Block ids of a partition kept in LDS: of blocks of 16 tokens or more
// (smaller ones are read from the table, token by token).
constexpr int kMaxIds8 = kMaxPartition / 16 + 2;

// A lane's piece of a V row: D / 16 codes.
template <int D>
struct VCodes;
template <>
struct VCodes<64> {
  using type = uint32_t;
};
template <>
struct VCodes<128> {
  using type = u32x2m;
};
template <typename V>
__device__ __forceinline__ uint32_t code_word(V v, int w) {
  if constexpr (sizeof(V) == 4) return v;
  else return v[w];
}

// The raw K pieces of groups G0 and G0 + 1 from the wave's LDS rows (at[j]: the
// LDS address of piece 4j + c of token r).  VM >= 0: waits first until at most
// VM vector memory operations are outstanding, the copies into those rows
// among the ones that are done (see read_k in decode_mfma.hip).
template <int KP, int ROW, int G0, int VM>
__device__ __forceinline__ void read_codes(const uint32_t (&at)[KP], u32x4m (&k)[2][KP]) {
  static_assert(KP == 1 || KP == 2, "heads of 64 to 128");
  if constexpr (VM >= 0) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(VM) : "memory");
  if constexpr (KP == 1)
    asm volatile(
        "ds_read_b128 %0, %2 offset:%3\n\tds_read_b128 %1, %2 offset:%4\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(k[0][0]), "=&v"(k[1][0])
        : "v"(at[0]), "n"(G0 * 16 * ROW), "n"((G0 + 1) * 16 * ROW)
        : "memory");
  else
    asm volatile(
        "ds_read_b128 %0, %4 offset:%6\n\tds_read_b128 %1, %5 offset:%6\n\t"
        "ds_read_b128 %2, %4 offset:%7\n\tds_read_b128 %3, %5 offset:%7\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(k[0][0]), "=&v"(k[0][1]), "=&v"(k[1][0]), "=&v"(k[1][1])
        : "v"(at[0]), "v"(at[1]), "n"(G0 * 16 * ROW), "n"((G0 + 1) * 16 * ROW)
        : "memory");
}

// SMALL: blocks of fewer than 16 tokens.  WINDOW: as in decode_mfma.hip (64 sequences of
// 128-8192 tokens, 32/32 heads of 128, window 2048, 16 sinks: 174 us, 5.8 TB/s).
template <typename T, int D, int DM, bool SHARED, int HEADS, bool SMALL, bool WINDOW>
__global__ __launch_bounds__(kDecodeThreads) __attribute__((amdgpu_waves_per_eu(4))) void
decode8_kernel(DecodeArgs a) {
  static_assert(sizeof(T) == 2, "16-bit queries");
  // (Rows of 80 or 96 bytes share 128-byte lines with the next head's.)
  constexpr bool kNt = !SHARED && DM % 128 == 0;
  constexpr int KP = (DM + 63) / 64;  // 16-byte pieces of a K row a lane takes
  constexpr int PE = D / 16;          // V codes of a lane's piece, blocks of the output
  constexpr int kRowBytes = D;        // an LDS row
  constexpr int kMemBytes = DM;       // a cache row
  constexpr int kVLoads = 8;
  using VP = typename VCodes<D>::type;

  __shared__ int s_blk[SMALL ? 1 : kMaxIds8];
  __shared__ int s_hole[kDecodeWaves];  // a wave met a missing block
  __shared__ float s_m[kDecodeWaves][kMfmaHeads];
  __shared__ float s_l[kDecodeWaves][kMfmaHeads];
  // Per wave: the scales of its tile's blocks (K's, V's; of each group, or of
  // each token).
  __shared__ __align__(16) float s_sc[kDecodeWaves][2 * kTile8];
  // Per wave: the K rows of its tile, and after the last tile its
  // accumulators.
  constexpr int kWaveBytes = kMfmaHeads * (D + 4) * 4;
  static_assert(kWaveBytes >= kTile8 * kRowBytes, "a tile's K rows fit");
  __shared__ __align__(16) char s_wave[kDecodeWaves][kWaveBytes];

  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int r = lane & 15;  // token of a K piece, query head elsewhere
  const int c = lane >> 4;
  constexpr int kHeadWaves = kDecodeWaves / HEADS;  // waves per KV head
  const int hkv = a.num_kv_heads;
  const int G = SHARED ? a.group / a.sub_groups : a.group;
  // Gangs of all of an item's workgroups: a head's part of a row is one line of
  // memory or less.
  const uint32_t units = static_cast<uint32_t>(hkv) / HEADS;
  const DecodePlace place = decode_place<true, SHARED>(a, units);
  const int64_t item = place.item;
  const int kvh = place.unit * HEADS + wave / kHeadWaves;
  const int h0 = kvh * a.group + place.sg * G;  // first query head of the wave
  const int seq = a.items[2 * item];
  const int part = a.items[2 * item + 1];
  const int64_t trow = a.rows != nullptr ? a.rows[seq] : seq;
  const bool row_ok = trow >= 0 && trow < a.num_table_rows;
  int ctx = a.context_lens[seq];
  int64_t qtok = a.cu_seqlens[seq];
  const int p0 = part * a.partition;
  const int log2_bs = a.log2_block_size;
  const int bs_mask = (1 << log2_bs) - 1;
  [[maybe_unused]] DecodeSpan span{};  // (its context is the one of this launch)
  if constexpr (WINDOW) {
    asm volatile("" : "+s"(ctx), "+s"(qtok));
    span = decode_span(ctx, a.window, a.sinks, log2_bs);
    ctx = span.ctx;
    if (part > 0 && p0 >= ctx) return;  // (a list made for a longer one)
  }
  const int first_blk = p0 >> log2_bs;
  const int nblk = SMALL ? 0 : ((p0 + a.partition - 1) >> log2_bs) - first_blk + 1;  // ids kept in LDS
  // (an id outside the pool becomes -1)
  auto table_entry = [&](int i) {
    int col = first_blk + i;
    if constexpr (WINDOW) col += col >= span.sinks ? span.skip : 0;
    const int b = row_ok && col < a.block_table_stride ? a.block_tables[trow * a.block_table_stride + col] : -1;
    return b >= a.total_blocks ? -1 : b;
  };
  const int b0 = tid < nblk ? table_entry(tid) : -1;
  // (both scalar loads issued before either is waited for: one round trip)
  asm volatile("" : "+s"(ctx), "+s"(qtok));
  const int n = max(0, min(a.partition, ctx - p0));
  const int ntiles = (n + kTile8 - 1) / kTile8;
  // Whether tokens [t, t + count) of the partition meet the hole of the span.
  [[maybe_unused]] auto in_hole = [&](int t, int count) {
    return WINDOW && p0 + t < span.hole_end && p0 + t + count > span.hole;
  };
  const int64_t row_bytes = static_cast<int64_t>(hkv) * kMemBytes;
  const char* kbase = reinterpret_cast<const char*>(a.key_cache) + kvh * kMemBytes;
  const char* vbase = reinterpret_cast<const char*>(a.value_cache) + kvh * kMemBytes;

  // The query heads (lanes past the group repeat its last one, and their
  // results are never stored; zero past the head dim): elements 0-7 and 8-15
  // of each of the lane's pieces.
  u32x4m q[2 * KP];
#pragma unroll
  for (int j = 0; j < 2 * KP; ++j) {
    const T* qrow = reinterpret_cast<const T*>(a.query) + qtok * a.q_token_stride +
                    static_cast<int64_t>(h0 + min(r, G - 1)) * a.q_head_stride;
    const int at = (4 * (j / 2) + c) * 16 + 8 * (j % 2);
    const bool in = DM == D || at < DM;
    q[j] = *reinterpret_cast<const u32x4m*>(qrow + (in ? at : 0));
    if constexpr (DM != D) q[j] = in ? q[j] : u32x4m{0, 0, 0, 0};
  }

  bool hole = false;  // a block the partition needs is missing
  {
    auto stage = [&](int i, int b) {
      s_blk[i] = b;
      hole |= b < 0 && (i << log2_bs) < n + (p0 & bs_mask);
    };
    if (tid < nblk) stage(tid, b0);
    for (int i = tid + kDecodeThreads; i < nblk; i += kDecodeThreads) stage(i, table_entry(i));
  }
  hole = __any(hole);
  if (lane == 0) s_hole[wave] = hole;
  __syncthreads();
  hole = false;
#pragma unroll
  for (int w = 0; w < kDecodeWaves; ++w) hole |= s_hole[w] != 0;
  // Block of token t < n of the partition, -1 where there is none.
  auto block_of = [&](int t) {
    const int i = ((p0 + t) >> log2_bs) - first_blk;
    return SMALL ? table_entry(i) : s_blk[i];
  };
  auto live_tokens = [&](int tile) {
    const int t = tile * kTile8 + lane % kTile8;
    return static_cast<uint32_t>(__ballot(t < n && !in_hole(t, 1) && block_of(min(t, n - 1)) >= 0));
  };

  VP vt[kVLoads];  // V of a tile: tokens 4c .. 4c+3 of each group
  // K goes straight into LDS, whole rows per load, the 16-byte chunks of token
  // t at position chunk ^ swizzle(t), which spreads the 16 rows of an operand
  // read over the banks.
  constexpr int kChunks = kRowBytes / 16;
  constexpr int kRowsPerLoad = kWave / kChunks;
  constexpr int kLoads = 16 / kRowsPerLoad;  // per group
  auto swizzle = [](int t) { return kChunks == 8 ? (t >> 1) & 7 : (t >> 2) & 3; };
  char* const s_k = s_wave[wave];
  auto k_row = [&](int i) { return kRowsPerLoad * i + lane / kChunks; };
  auto k_chunk = [&](int i) { return static_cast<uint32_t>(((lane % kChunks) ^ swizzle(k_row(i))) * 16); };
  // Lanes whose chunk lies past the head dim load nothing; those chunks stay
  // zero.
  if constexpr (DM != D) {
    constexpr int kPast = (D - DM) / 16;
    for (int i = lane; i < kPast * kTile8; i += kWave) {
      const int t = i / kPast, chunk = DM / 16 + i % kPast;
      st16(s_k + t * kRowBytes + 16 * (chunk ^ swizzle(t & 15)), make_uint4(0, 0, 0, 0));
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  typedef const __attribute__((address_space(1))) void* global_ptr;
  typedef __attribute__((address_space(3))) void* lds_ptr;
  auto load_k_lds = [&](const char* src, int s, int i) {
    if (DM != D && k_chunk(i) >= kMemBytes) return;
    __builtin_amdgcn_global_load_lds((global_ptr)(src), (lds_ptr)(s_k + (s * kLoads + i) * (kWave * 16)), 16, 0,
                                     kNt ? 2 : 0);
  };
  uint32_t koff[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) koff[i] = static_cast<uint32_t>(k_row(i) * static_cast<int>(row_bytes)) + k_chunk(i);
  // (Lanes past the head dim read the row's first piece; their output rows
  // are never stored.)
  const uint32_t vcol = DM == D || r * PE < DM ? r * PE : 0;
  const uint32_t voff = static_cast<uint32_t>(4 * c * static_cast<int>(row_bytes)) + vcol;
  // Blocks of 16 tokens or more: a group of 16 lies in one block, so it takes
  // one scalar base and per-lane offsets.  Groups past the partition's end read
  // the last one's rows, groups without a block block 0's.  Lanes 0 and 1 hold
  // the groups' blocks (2 and 3 again, for V's scales).
  int64_t at[2];  // byte offset of each group's first row
  auto locate = [&](int tile) {
    const int t = min(tile * kTile8 + 16 * (lane & 1), (n - 1) & ~15);
    const int b = max(s_blk[((p0 + t) >> log2_bs) - first_blk], 0);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int ts = min(tile * kTile8 + 16 * s, (n - 1) & ~15);
      at[s] = ((static_cast<int64_t>(__builtin_amdgcn_readlane(b, s)) << log2_bs) | ((p0 + ts) & bs_mask)) * row_bytes;
    }
    return b;
  };
  auto load_scales = [&](int b) {
    const float* from = (lane < 2 ? a.key_scales : a.value_scales) + static_cast<int64_t>(b) * hkv + kvh;
    if (lane < 4) __builtin_amdgcn_global_load_lds((global_ptr)(from), (lds_ptr)(s_sc[wave]), 4, 0, 0);
  };
  auto load_k = [&]() {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < kLoads; ++i) load_k_lds(kbase + at[s] + koff[i], s, i);
  };
  auto load_v = [&]() {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) vt[4 * s + i] = row_load<VP, kNt>(vbase + at[s] + i * row_bytes + voff);
  };
  // Smaller blocks: a slot and two scales per token; one without a block (or
  // past the end) reads slot 0.
  auto slot_of = [&](int t) -> int64_t {
    const int b = t < n ? block_of(t) : -1;
    return b < 0 ? 0 : (static_cast<int64_t>(b) << log2_bs) | ((p0 + t) & bs_mask);
  };
  auto load_any = [&](int tile) {
    const int t0 = tile * kTile8;
    const int64_t mine = (slot_of(t0 + lane % kTile8) >> log2_bs) * hkv + kvh;
    const float* from = (lane < kTile8 ? a.key_scales : a.value_scales) + mine;
    __builtin_amdgcn_global_load_lds((global_ptr)(from), (lds_ptr)(s_sc[wave]), 4, 0, 0);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        load_k_lds(kbase + slot_of(t0 + 16 * s + k_row(i)) * row_bytes + k_chunk(i), s, i);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        vt[4 * s + i] = row_load<VP, kNt>(vbase + slot_of(t0 + 16 * s + 4 * c + i) * row_bytes + vcol);
      __builtin_amdgcn_sched_barrier(0);  // (a group's addresses at a time: all of them spill)
    }
  };

  const float scale = a.scale_log2e;
  float m = kScoreFloor, l = 0.f;  // head r; l: this lane's tokens only
  f32x4m acc[PE];                  // acc[b][i]: dim PE * (4c + i) + b of head r
#pragma unroll
  for (int b = 0; b < PE; ++b) acc[b] = f32x4m{0.f, 0.f, 0.f, 0.f};

  f32x4m s[2];      // scores of tokens 4c .. 4c+3 of each group, head r
  float vs[2][2];   // V's scales of tokens 4c, 4c+1 and of 4c+2, 4c+3
  uint32_t k_at[KP];       // LDS addresses of the lane's pieces in the first group
#pragma unroll
  for (int j = 0; j < KP; ++j)
    k_at[j] = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)s_k)) +
              r * kRowBytes + 16 * ((4 * j + c) ^ swizzle(r));
  const uint32_t sc_at =
      static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) float*)s_sc[wave]));
  auto score_group = [&](int g, const u32x4m (&k)[KP], float ks) {
    s[g] = f32x4m{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < KP; ++j) {
      u32x4m lo, hi;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        lo[2 * i] = codes_to_half2<T, false>(k[j][i], ks);
        lo[2 * i + 1] = codes_to_half2<T, true>(k[j][i], ks);
        hi[2 * i] = codes_to_half2<T, false>(k[j][2 + i], ks);
        hi[2 * i + 1] = codes_to_half2<T, true>(k[j][2 + i], ks);
      }
      s[g] = mfma16<T>(hi, q[2 * j + 1], mfma16<T>(lo, q[2 * j], s[g]));
    }
  };
  // A group's scales, once the tile's copies but for its V loads have landed.
  auto scores = [&]() {
    f32x4m sc;  // K's of the two groups, V's
    asm volatile("s_waitcnt vmcnt(%2)\n\tds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(sc)
                 : "v"(sc_at), "n"(kVLoads)
                 : "memory");
    u32x4m k[2][KP];
    read_codes<KP, kRowBytes, 0, -1>(k_at, k);
    score_group(0, k[0], sc[0]);
    score_group(1, k[1], sc[1]);
#pragma unroll
    for (int g = 0; g < 2; ++g) vs[g][0] = vs[g][1] = sc[2 + g];
  };
  // A token's scales, after every load.
  auto scores_any = [&]() {
    u32x4m k[2][KP];
    read_codes<KP, kRowBytes, 0, 0>(k_at, k);
    const float* sc = s_sc[wave];
    score_group(0, k[0], sc[r]);
    score_group(1, k[1], sc[16 + r]);
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int i = 0; i < 2; ++i) vs[g][i] = sc[kTile8 + 16 * g + 4 * c + 2 * i];
  };
  // Tokens past the end or without a block get no weight, and their V codes
  // (NaN, perhaps) and scales are set aside.
  auto mask = [&](uint32_t live) {
    const uint32_t mine = live >> (4 * c);
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool on = (mine >> (16 * g + i)) & 1u;
        s[g][i] = on ? s[g][i] : -INFINITY;
        if (!on) vt[4 * g + i] = VP{};
        // (a pair's scale is set aside with both of its tokens)
        if (i % 2 == 0) vs[g][i / 2] = ((mine >> (16 * g + i)) & 3u) != 0 ? vs[g][i / 2] : 1.f;
      }
  };
  auto attend = [&]() {
    float tm = -INFINITY;
#pragma unroll
    for (int g = 0; g < 2; ++g)
      tm = fmaxf(tm, fmaxf(fmaxf(s[g][0], s[g][1]), fmaxf(s[g][2], s[g][3])));
    tm = max_halves(max_row_pairs(tm));
    const float m_new = fmaxf(m, tm);
    if (__any(m_new != m)) {
      const float alpha = fast_exp2((m - m_new) * scale);
      l *= alpha;
#pragma unroll
      for (int b = 0; b < PE; ++b) acc[b] *= alpha;
      m = m_new;
    }
    // (fp16: probabilities times 2^14, in l and acc alike, so that the second
    // term of a small one is not lost among fp16's subnormals)
    const float mc = fmaf(-m, scale, Elem<T>::kDtype == PA_DTYPE_F16 ? 14.f : 0.f);
    u32x4m p, rest;  // the probabilities, and what rounding them left
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float pa = fast_exp2(fmaf(s[i / 2][2 * (i % 2)], scale, mc));
      const float pb = fast_exp2(fmaf(s[i / 2][2 * (i % 2) + 1], scale, mc));
      l += pa + pb;
      const uint32_t w = pack_half2<T>(pa, pb);
      p[i] = w;
      rest[i] = pack_half2<T>(pa - half_lo<T>(w), pb - half_hi<T>(w));
    }
#pragma unroll
    for (int w = 0; w < PE / 4; ++w) {
      u32x4m d[4];  // dims 4w .. 4w+3 of the 8 tokens
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t v0 = code_word(vt[2 * i], w), v1 = code_word(vt[2 * i + 1], w);
        const float sc = vs[i / 2][i % 2];
        const uint32_t x = __builtin_amdgcn_perm(v1, v0, 0x05010400u);
        const uint32_t y = __builtin_amdgcn_perm(v1, v0, 0x07030602u);
        d[0][i] = codes_to_half2<T, false>(x, sc);
        d[1][i] = codes_to_half2<T, true>(x, sc);
        d[2][i] = codes_to_half2<T, false>(y, sc);
        d[3][i] = codes_to_half2<T, true>(y, sc);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[4 * w + e] = mfma16<T>(d[e], rest, mfma16<T>(d[e], p, acc[4 * w + e]));
    }
  };

  if (wave % kHeadWaves < ntiles) {
    int tile = wave % kHeadWaves;
    if constexpr (SMALL) {
      for (; tile < ntiles; tile += kHeadWaves) {
        load_any(tile);
        scores_any();
        mask(live_tokens(tile));
        attend();
      }
    } else {
      // The next tile's scales and K copies go out once the scores have used
      // the current ones, its V loads once the product has used the current V
      // (the pipeline of decode_mfma.hip, with its scheduling barriers and
      // empty statements).
#pragma unroll
      for (int j = 0; j < 2 * KP; ++j) asm volatile("" : "+v"(q[j]));
      load_scales(locate(tile));
      load_k();
      __builtin_amdgcn_sched_barrier(0);
      load_v();
      __builtin_amdgcn_sched_barrier(0);
      for (; tile + kHeadWaves < ntiles; tile += kHeadWaves) {
        const int b = locate(tile + kHeadWaves);
        scores();
        if (hole || in_hole(tile * kTile8, kTile8)) mask(live_tokens(tile));
#pragma unroll
        for (int i = 0; i < kVLoads; ++i) asm volatile("" : "+v"(vt[i]));
        __builtin_amdgcn_sched_barrier(0);
        load_scales(b);
        load_k();
        __builtin_amdgcn_sched_barrier(0);
        attend();
        load_v();
        __builtin_amdgcn_sched_barrier(0);
      }
      scores();
      if (hole || n - tile * kTile8 < kTile8 || in_hole(tile * kTile8, kTile8)) mask(live_tokens(tile));
      attend();
    }
  }

  combine_waves<T, D, DM, HEADS>(a, place, units, G, seq, part, ctx, n, qtok, m, l, acc, s_m, s_l, s_wave);
}

template <typename T, int D, int DM, typename Op>
static hipError_t visit8_t(bool shared, int heads, const Op& op) {
  if constexpr (DM == D)
    if (heads == 4) return op.template run<T, D, DM, false, 4>();
  if constexpr (DM == D)
    if (heads == 2) return op.template run<T, D, DM, false, 2>();
  return shared ? op.template run<T, D, DM, true, 1>() : op.template run<T, D, DM, false, 1>();
}

// Heads of 80 and 96 run on the LDS rows of 128.
template <typename T, typename Op>
static hipError_t visit8_dim(int head_dim, bool shared, int heads, const Op& op) {
  switch (head_dim) {
    case 64: return visit8_t<T, 64, 64>(shared, heads, op);
    case 80: return visit8_t<T, 128, 80>(shared, heads, op);
    case 96: return visit8_t<T, 128, 96>(shared, heads, op);
    case 128: return visit8_t<T, 128, 128>(shared, heads, op);
    default: return hipErrorNotSupported;
  }
}

struct Launch8 {
  const DecodeArgs& a;
  int64_t num_items;
  hipStream_t stream;
  template <typename T, int D, int DM, bool SHARED, int HEADS>
  hipError_t run() const {
    return a.window > 0 ? launch<T, D, DM, SHARED, HEADS, true>() : launch<T, D, DM, SHARED, HEADS, false>();
  }
  template <typename T, int D, int DM, bool SHARED, int HEADS, bool WINDOW>
  hipError_t launch() const {
    const uint32_t units = a.num_kv_heads / HEADS;
    const int64_t grid = num_items * units * a.sub_groups;
    DecodeArgs b = a;
    b.run_rcp = 0xffffffffu / (kXcds * units * a.sub_groups);
    if (a.log2_block_size < 4)
      hipLaunchKernelGGL((decode8_kernel<T, D, DM, SHARED, HEADS, true, WINDOW>), dim3(static_cast<uint32_t>(grid)),
                         dim3(kDecodeThreads), 0, stream, b);
    else
      hipLaunchKernelGGL((decode8_kernel<T, D, DM, SHARED, HEADS, false, WINDOW>), dim3(static_cast<uint32_t>(grid)),
                         dim3(kDecodeThreads), 0, stream, b);
    return hipGetLastError();
  }
};

struct Occupancy8 {
  int* per_cu;
  template <typename T, int D, int DM, bool SHARED, int HEADS>
  hipError_t run() const {
    return hipOccupancyMaxActiveBlocksPerMultiprocessor(per_cu, decode8_kernel<T, D, DM, SHARED, HEADS, false, false>,
                                                        kDecodeThreads, 0);
  }
};

hipError_t launch_decode8(const DecodeArgs& a, int dtype, int head_dim, int unit_heads, int64_t num_items,
                          hipStream_t stream) {
  const Launch8 op{a, num_items, stream};
  const bool shared = a.sub_groups > 1;
  // Four heads a workgroup where that still gives every CU four of them: a
  // wave each, so a row's pieces are read together and a CU touches fewer
  // pages.  Two heads -> four: 128 sequences of 128-8192 tokens, 32/8 heads of
  // 64, 132 -> 126 us; 256 of 2048, 32/8 of 128, at 1024, 206 -> 194 (512 of
  // them 367 -> 348).  With fewer workgroups a CU waits on its largest one: 16
  // of 256-1024, 32/8, 12.0 -> 13.9.
  if (unit_heads == 2 && a.num_kv_heads % 4 == 0 &&
      num_items * (a.num_kv_heads / 4) >= 4 * static_cast<int64_t>(device_compute_units()))
    unit_heads = 4;
  if (dtype == PA_DTYPE_BF16) return visit8_dim<bf16_t>(head_dim, shared, unit_heads, op);
  if (dtype == PA_DTYPE_F16) return visit8_dim<f16_t>(head_dim, shared, unit_heads, op);
  return hipErrorNotSupported;
}

// (What the partition is planned with.  The kernels of a head dim need the same
// LDS whatever their heads and query type, and registers for the same waves, so
// this holds for the four heads that launch_decode8 may take too.)
hipError_t decode8_workgroups_per_cu(int head_dim, bool shared, int unit_heads, int* per_cu) {
  return visit8_dim<bf16_t>(head_dim, shared, unit_heads, Occupancy8{per_cu});
}

}  // namespace pa
