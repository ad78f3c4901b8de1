// Attention over whole prompts: packed sequences, causal, query heads in groups that share a key head.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - m_i),  over j <= i + (keys - rows) of the sequence
//
// One pass over the keys with a running maximum m. Bound by the matrix cores (4 width products a visible pair) beside the
// exponentials on the vector unit.
//
// A workgroup takes 128 rows of one head, a wavefront 32 of them; keys come 64 (width 256: 32) at a time, global -> LDS
// without registers, the next tile's copies in flight under the present one's products. Products are written so that
// nothing has to change lanes between them:
//   scores^T = K Q^T   A = 32 keys (lane & 31) x 16 channels from LDS, B = Q^T from registers: a lane ends with 16 of 32
//                      keys' scores of one row (lane & 31), the other 16 in lane ^ 32;
//   out^T += V^T P^T   B = eight of those weights as they lie (keys 4 h + i and 8 + 4 h + i, h = lane >> 5); A = the same
//                      keys' values of one channel, by LDS loads that transpose (ds_read_b64_tr_b16).
// Weights are rounded to the inputs' type for the matrix cores (float16: times 2^15, so that those down to 2^-29 of a row's
// largest keep all their bits), and what a row is divided by is the float32 sum of the rounded weights.
//
// Values that a row must not see are multiplied by a weight of zero; where one is not finite in a tile that some row does
// not see whole, it is taken out and given to the rows that do see it alone.
#include "rows.h"

namespace lmoe {

constexpr int kPromptRows = 128;

struct PromptArgs {
  const uint16_t *q, *k, *v;
  long long q_row, q_head, k_row, k_head, v_row, v_head;  // elements
  const int *cu, *cu_k;
  uint16_t *out;
  float scale;  // times log2 e
  int T, U, B, q_heads, heads, tiles;
};

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
// 32-byte chunk pair p of value row r: the eight rows that a transposing load takes lie in different banks
template <int D>
__device__ __forceinline__ int v_pair(int r, int p) {
  return D == 64 ? p ^ ((r >> 1) & 3) : p ^ (r & 7);
}

template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (BF) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{a, b}, bf2));
  } else {
    return __builtin_bit_cast(uint32_t, h2_t{_Float16(a), _Float16(b)});
  }
}
// a + the pair's two values
template <bool BF>
__device__ __forceinline__ float add2(uint32_t pair, float a) {
  if constexpr (BF)
    return a + (__uint_as_float(pair << 16) + __uint_as_float(pair & 0xffff0000u));
  else
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2_t, pair), h2_t{1.0f, 1.0f}, a, false);
}

// Fragment words of values: those not finite taken out (set to zero), and as ones in pos (NaN, +inf) and neg (NaN, -inf)
template <bool BF>
__device__ __forceinline__ bool take_bad(u32x4 &f, u32x4 &pos, u32x4 &neg) {
  constexpr uint32_t INF = BF ? 0x7f80u : 0x7c00u, ONE = BF ? 0x3f80u : 0x3c00u;
  bool any = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    pos[e] = neg[e] = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t v = (f[e] >> (16 * h)) & 0xffffu, mag = v & 0x7fffu;
      if (mag >= INF) {
        any = true;
        const bool nan = mag > INF, minus = v >> 15;
        if (nan || !minus) pos[e] |= ONE << (16 * h);
        if (nan || minus) neg[e] |= ONE << (16 * h);
        f[e] &= ~(0xffffu << (16 * h));
      }
    }
  }
  return any;
}

template <int D, int BN, bool BF>
__global__ void __launch_bounds__(256) k_prompt(PromptArgs a) {
  constexpr int MT = BN / 32, KS = D / 16, DT = D / 32, COPIES = BN * D / 512 / 4;
  constexpr int kTileBytes = BN * D * 2;
  extern __shared__ uint8_t lds[];  // [2 stages][K tile, V tile]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 31, h = lane >> 5;
  // heads of one XCD are neighbours (they share key heads in its L2); later tiles, which see more keys, go first
  const int slot = blockIdx.x % a.q_heads, task = a.tiles - 1 - int(blockIdx.x) / a.q_heads;
  const int head = a.q_heads % 8 == 0 ? (slot & 7) * (a.q_heads / 8) + (slot >> 3) : slot;
  const int b = last_at(a.cu, a.B, task, [](int c, int i) { return (long long)(c / kPromptRows) + i; });
  if (b < 0) return;
  int row0, nq, key0, nk;
  seq_rows(a.cu, b, a.T, &row0, &nq);
  seq_rows(a.cu_k, b, a.U, &key0, &nk);
  const int tile = task - (a.cu[b] / kPromptRows + b);
  if (tile == 0 && (b == 0 || b == a.B - 1)) {
    // rows before the first sequence or behind the last one come back zero
    const int lo = b == 0 ? min(max(a.cu[0], 0), a.T) : 0, hi = b == a.B - 1 ? min(max(a.cu[a.B], 0), a.T) : a.T;
    for (int row = int(threadIdx.x) / (D / 8); row < lo + (a.T - hi); row += 256 / (D / 8)) {
      const size_t line = size_t(row < lo ? row : hi + row - lo) * a.q_heads + head;
      *reinterpret_cast<u32x4 *>(a.out + line * D + (threadIdx.x % (D / 8)) * 8) = u32x4{};
    }
  }
  const int first = tile * kPromptRows;
  if (first >= nq) return;
  const int off = nk - nq;                                  // row i sees keys 0 .. i + off
  const int keys = off + min(first + kPromptRows, nq);      // what the workgroup's last row sees
  const int mine = min(first + 32 * wave + r, nq - 1), sees = mine + off + 1;
  const int all = first + 32 * wave + off + 1;              // what every row of the wavefront sees
  const int wave_keys = min(first + 32 * wave + 31, nq - 1) + off + 1;  // what its last row sees
  const int kv = head / (a.q_heads / a.heads);

  u32x4 qf[KS];
  {
    const uint16_t *q = a.q + size_t(row0 + mine) * a.q_row + size_t(head) * a.q_head + 8 * h;
#pragma unroll
    for (int j = 0; j < KS; ++j) qf[j] = *reinterpret_cast<const u32x4 *>(q + 16 * j);
  }
  const uint32_t base = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t *)lds));
  // copy i of this wavefront: 64 chunks of 16 bytes, in LDS order; the rows' chunks are permuted on the global side
  auto fetch = [&](int at, int stage) {
    const uint16_t *k = a.k + size_t(key0 + at) * a.k_row + size_t(kv) * a.k_head;
    const uint16_t *v = a.v + size_t(key0 + at) * a.v_row + size_t(kv) * a.v_head;
    const int most = nk - 1 - at;
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
      const int j = (wave * COPIES + i) * 64 + lane, row = j / (D / 8), c = j % (D / 8);
      const int from = min(row, most);
      dma<16>(k, uint32_t(from) * uint32_t(a.k_row * 2) + k_chunk<D>(row, c) * 16,
              base + stage * 2 * kTileBytes + (wave * COPIES + i) * 1024);
      dma<16>(v, uint32_t(from) * uint32_t(a.v_row * 2) + (v_pair<D>(row, c >> 1) * 2 + (c & 1)) * 16,
              base + (stage * 2 + 1) * kTileBytes + (wave * COPIES + i) * 1024);
    }
  };
  f32x16 o[DT] = {};
  float m = -INFINITY, l = 0.0f;
  if (keys > 0) fetch(0, 0);
  for (int at = 0, stage = 0; at < keys; at += BN, stage ^= 1) {
    wait_vm<0>();
    barrier_lds();  // the tile is there, and the other stage has been read
    if (at + BN < keys) fetch(at + BN, stage ^ 1);
    if (at >= wave_keys) continue;
    const uint8_t *kt = lds + stage * 2 * kTileBytes, *vt = kt + kTileBytes;
    f32x16 s[MT] = {};
#pragma unroll
    for (int j = 0; j < KS; ++j)
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const int row = 32 * t + r;
        s[t] = mfma32<BF>(*reinterpret_cast<const u32x4 *>(kt + row * D * 2 + k_chunk<D>(row, 2 * j + h) * 16), qf[j], s[t]);
      }
    const bool edge = at + BN > all;
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[t][e] *= a.scale;
        if (edge && at + 32 * t + 8 * (e >> 2) + 4 * h + (e & 3) >= sees) s[t][e] = -INFINITY;
        top = fmaxf(top, s[t][e]);
      }
    top = fmaxf(top, lane_xor32(top));
    if (__any(top > m)) {
      const float to = fmaxf(m, top), keep = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
      m = to;
      l *= keep;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= keep;
    }
    const float lift = m == -INFINITY ? 0.0f : m - (BF ? 0.0f : 15.0f);
    u32x4 p[MT * 2];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t w = pack2<BF>(__builtin_amdgcn_exp2f(s[t][2 * e] - lift), __builtin_amdgcn_exp2f(s[t][2 * e + 1] - lift));
        l = add2<BF>(w, l);
        p[2 * t + (e >> 2)][e & 3] = w;
      }
    // a transposing load: 16 lanes take 4 keys x 16 channels, lane i of them gets channel i of the 4
    const int vrow = 4 * h + ((lane & 15) >> 2), vpair = (lane >> 4) & 1, vbyte = (lane & 3) * 8;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int ks = 0; ks < MT * 2; ++ks) {
        u32x4 f;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int row = 16 * ks + 8 * x + vrow;
          const uint8_t *src = vt + row * D * 2 + v_pair<D>(row, 2 * d + vpair) * 32 + vbyte;
          const s16x4 g = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(src));
          const u32x2 g2 = __builtin_bit_cast(u32x2, g);
          f[2 * x] = g2.x, f[2 * x + 1] = g2.y;
        }
        if (edge) {
          u32x4 pos, neg;
          if (__any(take_bad<BF>(f, pos, neg))) {
            constexpr uint32_t ONE = BF ? 0x3f80u : 0x3c00u;
            u32x4 seen;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int place = at + 16 * ks + 8 * (e >> 1) + 4 * h + 2 * (e & 1);
              seen[e] = (place < sees ? ONE : 0) | (place + 1 < sees ? ONE << 16 : 0);
            }
            const f32x16 up = mfma32<BF>(pos, seen, f32x16{}), down = mfma32<BF>(neg, seen, f32x16{});
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              if (up[e] > 0.0f) o[d][e] += INFINITY;
              if (down[e] > 0.0f) o[d][e] -= INFINITY;
            }
          }
        }
        o[d] = mfma32<BF>(f, p[ks], o[d]);
      }
  }
  l += lane_xor32(l);
  if (first + 32 * wave + r >= nq) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t *out = a.out + (size_t(row0 + mine) * a.q_heads + head) * D;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      *reinterpret_cast<u32x2 *>(out + 32 * d + 8 * e + 4 * h) =
          u32x2{pack2<BF>(o[d][4 * e] * inv, o[d][4 * e + 1] * inv), pack2<BF>(o[d][4 * e + 2] * inv, o[d][4 * e + 3] * inv)};
}

}  // namespace lmoe

using namespace lmoe;

extern "C" int lmoe_prompt_attend(const void *q, long long q_row, long long q_head, const void *k, long long k_row,
                                  long long k_head, const void *v, long long v_row, long long v_head, int dtype, int T, int U,
                                  int q_heads, int heads, int D, const int *cu, const int *cu_k, int B, float scale, void *out,
                                  void *stream) {
  const char *fn = "lmoe_prompt_attend";
  LMOE_REQUIRE(dtype == LMOE_F16 || dtype == LMOE_BF16, LMOE_EINVAL, "%s: dtype %d (float16 and bfloat16 are served)", fn, dtype);
  LMOE_REQUIRE(D == 64 || D == 128 || D == 256, LMOE_ESHAPE, "%s: heads of %d channels (64, 128 and 256 are served)", fn, D);
  LMOE_REQUIRE(heads > 0 && q_heads > 0 && q_heads % heads == 0, LMOE_ESHAPE, "%s: %d query heads over %d key heads", fn, q_heads,
               heads);
  LMOE_REQUIRE(T >= 0 && U >= 0 && B >= 0, LMOE_ESHAPE, "%s: %d rows, %d keys, %d sequences", fn, T, U, B);
  if (T == 0) return 0;
  LMOE_REQUIRE(B > 0, LMOE_ESHAPE, "%s: %d rows of no sequence", fn, T);
  LMOE_REQUIRE(q && out && cu && cu_k && ((k && v) || U == 0), LMOE_EINVAL, "%s: null pointer", fn);
  LMOE_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out) && q_row % 8 == 0 && q_head % 8 == 0 &&
                   k_row % 8 == 0 && k_head % 8 == 0 && v_row % 8 == 0 && v_head % 8 == 0,
               LMOE_EALIGN, "%s: rows must be 16-byte aligned", fn);
  LMOE_REQUIRE(k_row >= 0 && v_row >= 0 && k_row < (1 << 23) && v_row < (1 << 23), LMOE_ESHAPE,
               "%s: rows of keys %lld and of values %lld elements apart", fn, k_row, v_row);
  const long long tiles = T / kPromptRows + (long long)B;
  LMOE_REQUIRE(tiles * q_heads < (1ll << 31), LMOE_ESHAPE, "%s: %d rows of %d heads", fn, T, q_heads);
  PromptArgs a = {static_cast<const uint16_t *>(q), static_cast<const uint16_t *>(k), static_cast<const uint16_t *>(v), q_row,
                  q_head, k_row, k_head, v_row, v_head, cu, cu_k, static_cast<uint16_t *>(out), scale * 1.4426950408889634f, T, U,
                  B, q_heads, heads, int(tiles)};
  auto go = [&](auto kernel, int bn) -> int {
    const size_t lds = size_t(bn) * D * 2 * 4;
    if (const int rc = allow_lds(kernel, lds, fn)) return rc;
    launch(kernel, dim3(unsigned(tiles * q_heads)), dim3(256), lds, (hipStream_t)stream, a);
    LMOE_LAUNCHED(fn);
    return 0;
  };
  const bool bf = dtype == LMOE_BF16;
  if (D == 64) return bf ? go(k_prompt<64, 64, true>, 64) : go(k_prompt<64, 64, false>, 64);
  if (D == 128) return bf ? go(k_prompt<128, 64, true>, 64) : go(k_prompt<128, 64, false>, 64);
  return bf ? go(k_prompt<256, 32, true>, 32) : go(k_prompt<256, 32, false>, 32);
}
