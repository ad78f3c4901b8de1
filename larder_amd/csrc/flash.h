// What the attention of many rows at a time shares (prompt.hip: over keys in 16 bits; chunk.hip: over the paged cache): matrix
// products of 32 rows, the layout of keys and values in LDS, weights in 16 bits, values that are not finite, and the joining of
// rows whose keys were worked in chunks.
#pragma once
#include "lines.h"
#include "rows.h"

namespace lmoe {

constexpr int kPromptKeys = 64;  // keys a tile

// A weight is 2^(score - maximum in use + kLift), the maximum lagging at most kLag: float16 weights reach 2^15 at most, and
// one 2^-25 of the largest is still a normal number
template <bool BF>
constexpr float kLift = BF ? 0.0f : 11.0f;
template <bool BF>
constexpr float kLag = BF ? 8.0f : 4.0f;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <bool BF>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// 16-byte chunk c of key row r (rows of D / 8 chunks): eight, or sixteen, rows' same chunk lie in different banks
template <int D>
__device__ __forceinline__ int k_chunk(int r, int c) {
  return D == 64 ? c ^ ((r >> 1) & 7) : c ^ (r & 15);
}
// 32-byte chunk pair p of value row r: what 32 lanes of a transposing load take (two neighbouring pairs of four rows) lies in
// different banks
template <int D>
__device__ __forceinline__ int v_pair(int r, int p) {
  return D == 64 ? p ^ (r & 2) : p ^ ((r & 3) << 1) ^ ((r >> 2) & 1);
}

template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (BF) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{a, b}, bf16x2));
  } else {
    return __builtin_bit_cast(uint32_t, h2_t{_Float16(a), _Float16(b)});
  }
}
// a + the pair's two values
template <bool BF>
__device__ __forceinline__ float add2(uint32_t pair, float a) {
  if constexpr (BF)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), __builtin_bit_cast(bf16x2, 0x3f803f80u), a, false);
  else
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2_t, pair), h2_t{1.0f, 1.0f}, a, false);
}

// Whether a thread's share of a tile's values holds one that is not finite. In LDS order: looked at by key and channel, as
// take_bad does, 18 prompts of 512 rows take 112 us instead of 107.6 (16 heads of 256)
template <int D, bool BF, int THREADS = 256>
__device__ __forceinline__ bool any_bad(const uint8_t *vt) {
  constexpr uint32_t INF = BF ? 0x7f80u : 0x7c00u;
  uint32_t over = 0;
#pragma unroll
  for (int i = 0; i < kPromptKeys * D / 8 / THREADS; ++i) {  // a half word's magnitude of INF or more carries into its sign bit
    const u32x4 w = reinterpret_cast<const u32x4 *>(vt)[i * THREADS + threadIdx.x];
#pragma unroll
    for (int e = 0; e < 4; ++e) over |= (w[e] & 0x7fff7fffu) + (0x8000u - INF) * 0x10001u;
  }
  return over & 0x80008000u;
}

// Values that are not finite in a tile that some row does not see whole: one thread a key and 32 channels. They are set to zero
// in LDS and noted in two words of bits, pos (NaN, +inf) and neg (NaN, -inf).
template <int D, bool BF>
__device__ __forceinline__ void take_bad(uint8_t *vt, int row, int c32, uint32_t *pos, uint32_t *neg) {
  constexpr uint32_t INF = BF ? 0x7f80u : 0x7c00u;
  uint32_t up = 0, down = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    u32x4 *at = reinterpret_cast<u32x4 *>(vt + row * D * 2 + v_pair<D>(row, 2 * c32 + (j >> 1)) * 32 + (j & 1) * 16);
    u32x4 w = *at;
    bool any = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t x = (w[e >> 1] >> (16 * (e & 1))) & 0xffffu, mag = x & 0x7fffu;
      if (mag >= INF) {
        const bool nan = mag > INF, minus = x >> 15;
        any = true;
        if (nan || !minus) up |= 1u << (8 * j + e);
        if (nan || minus) down |= 1u << (8 * j + e);
        w[e >> 1] &= ~(0xffffu << (16 * (e & 1)));
      }
    }
    if (any) *at = w;
  }
  *pos = up;
  *neg = down;
}

// Rows whose keys were worked in more than one chunk: D / 4 threads a row and head, the chunks joined in order
struct JoinArgs {
  uint16_t *out;
  const float *part;  // [chunks][T][q_heads] of [D] sums and {maximum, weight}
  const int *joins;   // [T][q_heads]: how many chunks (0: the row is done)
  int T, q_heads, chunks;
  const int2 *placed = nullptr;  // PLACED: [T][q_heads] of the first piece's line in part (-1: the row is done) and the last one's
  int next = 0, step = 0, most = 0;  // from the first piece's line to the second's, from there to each further one's; lines in all
};
// G: groups of D / 4 threads that share a line's chunks, every Gth each, where there are many chunks and few lines
template <int D, bool BF, int G = 1, bool PLACED = false>
static __global__ void __launch_bounds__(256) k_join_chunks(JoinArgs a) {
  constexpr int LANES = D / 4;
  const int thread = threadIdx.x % LANES, group = threadIdx.x / LANES % G;
  const size_t line = size_t(blockIdx.x) * (256 / (LANES * G)) + threadIdx.x / (LANES * G), lines = size_t(a.T) * a.q_heads;
  if (G == 1 && line >= lines) return;
  const int d = thread * 4;
  int parts = 0, from = 0;
  if constexpr (PLACED) {
    const int2 place = line < lines ? a.placed[line] : int2{-1, 0};
    from = place.x;
    parts = joined_pieces(from, place.y, a.next, a.step, a.most);
  } else if (line < lines) {
    parts = min(a.joins[line], a.chunks);
  }
  if (G == 1 && parts < 2) return;
  f32x4 v = {};
  float top = -INFINITY, weight = 0.0f;
  auto join = [&](float m, float l, f32x4 y) {
    if (l == 0.0f) return;  // (a chunk that the row sees nothing of weighs 0; NaN goes on)
    const float to = fmaxf(top, m), f = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
    const float keep = weight == 0.0f ? 0.0f : to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - to);
    top = to;
    weight = fmaf(l, f, weight * keep);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = fmaf(y[e], f, v[e] * keep);
  };
  for (int c0 = group; c0 < parts; c0 += 4 * G) {
    float2 ml[4];
    f32x4 y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = min(c0 + j * G, parts - 1);
      const float *part =
          a.part + (PLACED ? size_t(from + (c ? a.next + (c - 1) * a.step : 0)) : size_t(c) * lines + line) * (D + 4);
      ml[j] = *reinterpret_cast<const float2 *>(part + D);
      y[j] = *reinterpret_cast<const f32x4 *>(part + d);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c0 + j * G < parts) join(ml[j].x, ml[j].y, y[j]);
  }
  if constexpr (G > 1) {
    __shared__ float sums[256][6];
    float *mine = sums[threadIdx.x];
#pragma unroll
    for (int e = 0; e < 4; ++e) mine[e] = v[e];
    mine[4] = top, mine[5] = weight;
    __syncthreads();
    if (group || parts < 2) return;
    for (int g = 1; g < G; ++g) {
      const float *other = sums[threadIdx.x + g * LANES];
      join(other[4], other[5], f32x4{other[0], other[1], other[2], other[3]});
    }
  }
  const float inv = weight == 0.0f ? 0.0f : 1.0f / weight;
  *reinterpret_cast<u32x2 *>(a.out + line * D + d) = u32x2{pack2<BF>(v[0] * inv, v[1] * inv), pack2<BF>(v[2] * inv, v[3] * inv)};
}

}  // namespace lmoe
