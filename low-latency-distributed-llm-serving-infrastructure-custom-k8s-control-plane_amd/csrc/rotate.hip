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
// What bounds it is memory once a step has some thousand rows, and before that
// the launch and two dependent reads (position, then table).
#include "cache8.hpp"
#include "pa_common.hpp"
#include "pa_launch.hpp"

namespace pa {

constexpr int kRotateThreads = 256;

// Four elements at p as floats, and back (rounded to nearest even).
template <typename T>
__device__ __forceinline__ void load4(const T* p, float* x) {
  if constexpr (sizeof(T) == 4) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    x[0] = half_lo<T>(v.x), x[1] = half_hi<T>(v.x), x[2] = half_lo<T>(v.y), x[3] = half_hi<T>(v.y);
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float* x) {
  if constexpr (sizeof(T) == 4)
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  else
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_half2<T>(x[0], x[1]), pack_half2<T>(x[2], x[3]));
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
// needs D and R in multiples of 8 and rows at multiples of 4 elements.  Else
// elements lane + 64 e, each with its partner read again; any D up to 256.
template <typename T, int L, bool VEC>
struct RowLane {
  static constexpr int kN = VEC ? 8 : 4;
  const RotateArgs& args;
  int lane;  // in the row's group
  int a, b;  // VEC
  bool live, turns;

  __device__ __forceinline__ RowLane(const RotateArgs& r, int l) : args(r), lane(l) {
    if constexpr (VEC) {
      const int pairs = r.rotary_dim / 8;  // lanes that rotate
      turns = l < pairs;
      live = 8 * l < r.head_dim;
      const bool halves = turns && !r.interleaved;
      a = halves ? 4 * l : 8 * l;
      b = halves ? r.rotary_dim / 2 + 4 * l : 8 * l + 4;
    } else {
      turns = live = true;
      a = b = 0;
    }
  }
  __device__ __forceinline__ void load(const T* row, float* x) const {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.f;
      if (live) {
        load4<T>(row + a, x);
        load4<T>(row + b, x + 4);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = lane + 64 * e;
        x[e] = d < args.head_dim ? load_scalar<T>(row + d) : 0.f;
      }
    }
  }
  __device__ __forceinline__ void store(T* row, const float* x) const {
    if constexpr (VEC) {
      if (live) {
        store4<T>(row + a, x);
        store4<T>(row + b, x + 4);
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
  // Normalise (w not null) and rotate the row x holds.
  // (No contraction but the fmaf written here: the kernels below give the
  // same bits.)
  __device__ __forceinline__ void apply(const T* row, float* x, const void* w, int64_t pos) const {
#pragma clang fp contract(off)
    float r = 1.f;
    if (w != nullptr) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < kN; ++i) ss = fmaf(x[i], x[i], ss);
      r = rsqrtf(row_sum<L>(ss) / static_cast<float>(args.head_dim) + args.eps);
    }
    const int rot = args.rotary_dim;
    const float* cs = args.cos_sin + pos * rot;  // (not read without rotation)
    if constexpr (VEC) {
      if (w != nullptr && live) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = x[i] * r * weight(w, a + i);
          x[4 + i] = x[4 + i] * r * weight(w, b + i);
        }
      }
      if (turns && rot > 0) {
        const float4 c4 = *reinterpret_cast<const float4*>(cs + 4 * lane);
        const float4 s4 = *reinterpret_cast<const float4*>(cs + rot / 2 + 4 * lane);
        const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float& p = args.interleaved ? x[2 * i] : x[i];
          float& q = args.interleaved ? x[2 * i + 1] : x[4 + i];
          const float u = p, v = q;
          p = fmaf(u, c[i], -(v * s[i]));
          q = fmaf(v, c[i], u * s[i]);
        }
      }
    } else {
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
  }
};

// A row of Q (head < H_q) or K, rotated; a position outside the table makes
// it NaN, so that no such call passes for a result.
template <typename T, int L, bool VEC>
__device__ __forceinline__ bool rotated_row(const RotateArgs& a, const RowLane<T, L, VEC>& ln, const T* row, int64_t t,
                                            const void* w, float* x) {
  const int64_t pos = a.rotary_dim > 0 ? a.positions[t] : 0;
  ln.load(row, x);
  const bool ok = a.rotary_dim == 0 || (pos >= 0 && pos < a.num_positions);
  ln.apply(row, x, w, ok ? pos : 0);
  if (!ok) {
#pragma unroll
    for (int i = 0; i < RowLane<T, L, VEC>::kN; ++i) x[i] = __builtin_nanf("");
  }
  return ok;
}

// Every row of the step in turn, (token, head) with the heads of Q, K, V in
// this order; K and V go to the cache's slots, or (no cache) K to key_out.
template <typename T, int L, bool VEC>
__global__ __launch_bounds__(kRotateThreads) void rotate_kernel(RotateArgs a) {
  constexpr int kRows = kRotateThreads / L;
  const uint32_t heads = a.num_query_heads + (a.key_cache != nullptr ? 2 : 1) * a.num_kv_heads;
  const uint32_t id = blockIdx.x * kRows + threadIdx.x / L;
  const uint32_t tok = quotient(id, heads, a.heads_rcp);
  if (tok >= static_cast<uint32_t>(a.num_tokens)) return;
  const int64_t t = tok;
  int h = static_cast<int>(id - tok * heads);
  const RowLane<T, L, VEC> ln(a, threadIdx.x % L);
  float x[RowLane<T, L, VEC>::kN];
  if (h < a.num_query_heads) {
    const T* row = reinterpret_cast<const T*>(a.query) + t * a.q_token_stride + h * a.q_head_stride;
    rotated_row<T, L, VEC>(a, ln, row, t, a.query_weight, x);
    ln.store(reinterpret_cast<T*>(a.query_out) + t * a.q_out_token_stride + h * a.q_out_head_stride, x);
    return;
  }
  h -= a.num_query_heads;
  const bool is_v = h >= a.num_kv_heads;
  if (is_v) h -= a.num_kv_heads;
  T* out;
  if (a.key_cache != nullptr) {
    const int64_t slot = a.slot_mapping[t];
    if (slot < 0 || slot >= a.num_slots) return;
    out = reinterpret_cast<T*>(is_v ? a.value_cache : a.key_cache) + (slot * a.num_kv_heads + h) * a.head_dim;
  } else {
    out = reinterpret_cast<T*>(a.key_out) + t * a.k_out_token_stride + h * a.k_out_head_stride;
  }
  if (is_v) {
    ln.load(reinterpret_cast<const T*>(a.value) + t * a.v_token_stride + h * a.v_head_stride, x);
  } else {
    const T* row = reinterpret_cast<const T*>(a.key) + t * a.k_token_stride + h * a.k_head_stride;
    // (a K row without a position is not cached)
    if (!rotated_row<T, L, VEC>(a, ln, row, t, a.key_weight, x) && a.key_cache != nullptr) return;
  }
  ln.store(out, x);
}

// The 8-bit cache's write.  The first a.kv_groups workgroups take (chunk of C
// tokens, KV head, tensor) each, the others rows of Q.
//
// A block's scale depends on all of its rows, so one workgroup has to see
// every row the step brings for the block.  Those follow each other in the
// step: a chunk owns the runs (tokens of one block) that begin in it, and so
// looks at up to block_size - 1 tokens past its end and leaves the first ones
// to the chunk before where their run began there.  It goes over them twice,
// for the runs' largest magnitudes (kept in LDS by an integer maximum of the
// floats' bits, which no order changes) and then to write the codes, the rows
// coming from the L2 the second time.  A run that holds its block's first row
// starts the block afresh; the other rows of any other block are re-coded if
// its scale grows.
template <typename T, int L, bool VEC>
__global__ __launch_bounds__(kRotateThreads) void cache8_write_kernel(RotateArgs a) {
  constexpr int C = kRotateThreads / L;  // tokens a chunk owns, rows at once
  constexpr int kN = RowLane<T, L, VEC>::kN;
  const RowLane<T, L, VEC> ln(a, threadIdx.x % L);
  const int group = threadIdx.x / L;
  float x[kN];
  if (blockIdx.x >= a.kv_groups) {
    const uint32_t id = (blockIdx.x - a.kv_groups) * C + group;
    const uint32_t tok = quotient(id, a.num_query_heads, a.heads_rcp);
    if (tok >= static_cast<uint32_t>(a.num_tokens)) return;
    const int64_t t = tok;
    const int h = static_cast<int>(id - tok * a.num_query_heads);
    const T* row = reinterpret_cast<const T*>(a.query) + t * a.q_token_stride + h * a.q_head_stride;
    rotated_row<T, L, VEC>(a, ln, row, t, a.query_weight, x);
    ln.store(reinterpret_cast<T*>(a.query_out) + t * a.q_out_token_stride + h * a.q_out_head_stride, x);
    return;
  }
  // Per run that begins in the chunk (at token C c + i): its block, its first
  // and one past its last token, whether it holds the block's first row, its
  // largest magnitude's bits, the block's scales.
  __shared__ int64_t s_block[C];
  __shared__ int s_end[C], s_fresh[C];
  __shared__ uint32_t s_amax[C];
  __shared__ float s_new[C], s_ratio[C];
  // Per token of the span: the run it belongs to (< 0: none of the chunk's).
  __shared__ int16_t s_run[C + kMaxCache8Block];

  const uint32_t units = 2 * a.num_kv_heads;
  const uint32_t chunk = quotient(blockIdx.x, units, a.kv_rcp);
  const int u = static_cast<int>(blockIdx.x - chunk * units);
  const bool is_v = u >= a.num_kv_heads;
  const int h = is_v ? u - a.num_kv_heads : u;
  const int64_t t0 = static_cast<int64_t>(chunk) * C;
  const int span = static_cast<int>(min<int64_t>(C + a.block_size - 1, a.num_tokens - t0));
  auto block_of = [&](int64_t t) -> int64_t {
    if (t < 0 || t >= a.num_tokens) return -1;
    const int64_t slot = a.slot_mapping[t];
    if (slot < 0 || slot >= a.num_slots) return -1;
    return slot / a.block_size;
  };
  if (threadIdx.x < C) {
    s_block[threadIdx.x] = -1;
    s_end[threadIdx.x] = 0;
    s_fresh[threadIdx.x] = 0;
    s_amax[threadIdx.x] = 0;
  }
  __syncthreads();
  if (threadIdx.x < kWave) {
    int last = -1;  // the run the tokens before this batch end in
    for (int base = 0; base < span; base += kWave) {
      const int j = base + threadIdx.x;
      const int64_t blk = j < span ? block_of(t0 + j) : -1;
      const bool starts = j < span && blk != block_of(t0 + j - 1);
      const uint64_t mask = __ballot(starts);
      const uint64_t upto = mask & (~uint64_t{0} >> (kWave - 1 - threadIdx.x));
      const int lead = upto != 0 ? base + 63 - __builtin_clzll(upto) : last;
      const bool ours = lead >= 0 && lead < C && blk >= 0 && j < span;
      if (j < span) s_run[j] = static_cast<int16_t>(ours ? lead : -1);
      if (ours) {
        if (starts) s_block[lead] = blk;
        atomicMax(&s_end[lead], j + 1);
        if (a.slot_mapping[t0 + j] % a.block_size == 0) s_fresh[lead] = 1;
      }
      if (mask != 0) last = base + 63 - __builtin_clzll(mask);
    }
  }
  __syncthreads();
  const T* src = reinterpret_cast<const T*>(is_v ? a.value : a.key) + h * (is_v ? a.v_head_stride : a.k_head_stride);
  const int64_t tok_stride = is_v ? a.v_token_stride : a.k_token_stride;
  // Row j as the 16-bit cache would hold it; false if it is not cached.
  auto read_row = [&](int j) {
    const int64_t t = t0 + j;
    const T* row = src + t * tok_stride;
    bool ok = true;
    if (is_v) ln.load(row, x);
    else ok = rotated_row<T, L, VEC>(a, ln, row, t, a.key_weight, x);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      if constexpr (Elem<T>::kDtype == PA_DTYPE_F16) {
        if (fabsf(x[i]) < INFINITY) x[i] = fminf(fmaxf(rounded<T>(x[i]), -kMaxF16Row), kMaxF16Row);
      } else {
        x[i] = rounded<T>(x[i]);
      }
    }
    return ok;
  };
  // The run past whose end no token is the chunk's.
  int end = 0;
  for (int i = 0; i < C; ++i) end = max(end, s_end[i]);
  for (int j = group; j < end; j += C) {
    const int run = s_run[j];
    if (run < 0 || !read_row(j)) continue;
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const float v = fabsf(x[i]);
      m = fmaxf(m, v < INFINITY ? v : 0.f);
    }
    m = row_max<L>(m);
    if (ln.lane == 0) atomicMax(&s_amax[run], __float_as_uint(m));
  }
  __syncthreads();
  float* scales = is_v ? a.value_scales : a.key_scales;
  if (threadIdx.x < C && s_block[threadIdx.x] >= 0) {
    float* at = scales + s_block[threadIdx.x] * a.num_kv_heads + h;
    const float need = scale_for(__uint_as_float(s_amax[threadIdx.x]));
    const float was = s_fresh[threadIdx.x] ? 0.f : scale_pow2(*at);
    const float now = fmaxf(was, need);
    s_new[threadIdx.x] = now;
    s_ratio[threadIdx.x] = s_fresh[threadIdx.x] ? 1.f : was * inverse_pow2(now);
    *at = now;
  }
  __syncthreads();
  uint8_t* cache = reinterpret_cast<uint8_t*>(is_v ? a.value_cache : a.key_cache) + h * a.head_dim;
  const int64_t row_codes = static_cast<int64_t>(a.num_kv_heads) * a.head_dim;
  // Blocks whose scale grew: all of their rows; the run's own follow below.
  for (int i = 0; i < C; ++i) {
    if (s_block[i] < 0 || s_ratio[i] == 1.f) continue;
    const float ratio = s_ratio[i];
    uint8_t* rows = cache + s_block[i] * a.block_size * row_codes;
    for (int k = threadIdx.x; k < a.block_size * a.head_dim; k += kRotateThreads) {
      const int r = k / a.head_dim;
      uint8_t* p = rows + r * row_codes + (k - r * a.head_dim);
      *p = static_cast<uint8_t>(pack_codes2(code_to_f32<0>(*p) * ratio, 0.f));
    }
  }
  __syncthreads();  // (orders the stores of a row's two writes)
  for (int j = group; j < end; j += C) {
    const int run = s_run[j];
    if (run < 0 || !read_row(j)) continue;
    const float inv = inverse_pow2(s_new[run]);
    uint8_t* out = cache + a.slot_mapping[t0 + j] * row_codes;
    if constexpr (VEC) {
      if (ln.live) {
        *reinterpret_cast<uint32_t*>(out + ln.a) = pack_codes4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
        *reinterpret_cast<uint32_t*>(out + ln.b) = pack_codes4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (ln.lane + 64 * e < a.head_dim)
          out[ln.lane + 64 * e] = static_cast<uint8_t>(pack_codes2(x[e] * inv, 0.f));
    }
  }
}

template <typename T, int L, bool VEC>
static hipError_t launch_rotate_l(const RotateArgs& args, hipStream_t s) {
  constexpr int kRows = kRotateThreads / L;
  RotateArgs a = args;
  if (a.key_scales == nullptr) {
    const uint32_t heads = a.num_query_heads + (a.key_cache != nullptr ? 2 : 1) * a.num_kv_heads;
    a.heads_rcp = 0xffffffffu / heads;
    const int64_t rows = static_cast<int64_t>(a.num_tokens) * heads;
    const dim3 grid(static_cast<uint32_t>((rows + kRows - 1) / kRows));
    hipLaunchKernelGGL((rotate_kernel<T, L, VEC>), grid, dim3(kRotateThreads), 0, s, a);
    return hipGetLastError();
  }
  a.heads_rcp = a.num_query_heads > 0 ? 0xffffffffu / a.num_query_heads : 0;
  a.kv_rcp = 0xffffffffu / (2 * a.num_kv_heads);
  a.kv_groups = static_cast<uint32_t>((a.num_tokens + kRows - 1) / kRows * (2 * a.num_kv_heads));
  const int64_t q_rows = static_cast<int64_t>(a.num_tokens) * a.num_query_heads;
  const dim3 grid(a.kv_groups + static_cast<uint32_t>((q_rows + kRows - 1) / kRows));
  hipLaunchKernelGGL((cache8_write_kernel<T, L, VEC>), grid, dim3(kRotateThreads), 0, s, a);
  return hipGetLastError();
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
                   fits(a.value_cache, 0, 0) && reinterpret_cast<uintptr_t>(a.cos_sin) % 16 == 0;
  switch (dtype) {
    case PA_DTYPE_F32: return launch_rotate_t<float>(a, vec, s);
    case PA_DTYPE_BF16: return launch_rotate_t<bf16_t>(a, vec, s);
    case PA_DTYPE_F16: return launch_rotate_t<f16_t>(a, vec, s);
    default: return hipErrorNotSupported;
  }
}

}  // namespace pa
