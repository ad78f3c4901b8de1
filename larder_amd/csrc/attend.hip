// Attention of the newest rows of each sequence (one token, or a speculative decoder's few) over the 8-bit paged cache.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - m),  over the places j < len - (n - 1 - r) of row r of n
//
// One pass over the keys and values with a running maximum m. Bound by the cache's bytes: 2 width a token and key head, read
// once for all the query heads of its group and all of a sequence's rows (up to 16 of these together fill a matrix-core
// tile's columns).
//
// A wavefront takes 32 tokens a step, straight from global memory to registers; no LDS until the end. Products are written
// so that nothing has to change lanes between them:
//   scores^T = K Q^T   A = 16 tokens (lane & 15) x 32 channels, 16 codes a lane from one load, B = Q^T; a lane ends with
//                      four tokens (4 (lane >> 4) + i) of one query row (lane & 15) from each of two 16-token tiles;
//   out^T += V^T P^T   B = those eight tokens' weights as they lie; A = the same eight tokens' codes of one channel. A lane
//                      loads width / 16 neighbouring channels of its eight tokens, and byte permutes pair up the tokens.
// e4m3 codes are exact in float16 and bfloat16, so q keeps its type; weights are float16, times 2^15 so that a weight down to
// 2^-29 of the row's largest keeps all eleven bits (a long context under one token that stands out lives there). The scales
// multiply float32 sums.
//
// A workgroup is four wavefronts, taking turns at the 32-token tiles of one chunk of one sequence; they join in LDS, and
// where a sequence has more than one chunk a second kernel joins those. Chunks have one length, so ragged sequences give
// equal workgroups; those past a sequence's end leave at once.
#include "rows.h"

namespace lmoe {

constexpr int kAttendWaves = 4;
constexpr float kLog2e = 1.4426950408889634f;

struct AttendArgs {
  const void *q;
  long long q_row, q_head;
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int *table, *lens, *cu;
  void *out;        // [T][q_heads][D]
  float *part;      // [T q_heads][chunks] of D sums, then [T q_heads][chunks] of {maximum, weight}; null: one chunk
  float scale;      // times log2 e
  int T, B, q_heads, heads, page_shift, pages, width, group, row_tiles, chunk, chunks;
};

template <bool BF>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// two e4m3 codes of a word (HI: its upper two) as a pair of 16-bit floats, exactly
template <bool BF, bool HI>
__device__ __forceinline__ uint32_t codes2(uint32_t w) {
  if constexpr (BF)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
}

// whether one of a word's four codes is NaN
__device__ __forceinline__ bool nan_code(uint32_t w) {
  const uint32_t m = ~w & 0x7f7f7f7fu;  // a NaN's byte is zero here, and no byte has its top bit
  return ((m - 0x01010101u) & ~m & 0x80808080u) != 0;
}

// One wavefront's raw codes of 32 tokens of a head
template <int D>
struct Codes {
  u32x4 k[2][D / 64];      // [16 tokens][64 channels]: token lane & 15, channels 64 c + 16 (lane >> 4) .. + 15
  uint32_t v[8][D / 64];   // tokens 4 (lane >> 4) + i and 16 + those, channels (lane & 15) D / 16 .. + D / 16 - 1
};

template <int D>
__device__ __forceinline__ void load_codes(Codes<D> &c, const uint8_t *kc, const uint8_t *vc, size_t at, int lane) {
  const int r = lane & 15, g = lane >> 4;
  const uint8_t *k = kc + at + size_t(r) * D + 16 * g;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int j = 0; j < D / 64; ++j) c.k[m][j] = *reinterpret_cast<const u32x4 *>(k + m * 16 * D + 64 * j);
  const uint8_t *v = vc + at + size_t(4 * g) * D + r * (D / 16);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint8_t *p = v + ((i & 3) + 16 * (i >> 2)) * D;
    if constexpr (D == 64) {
      c.v[i][0] = *reinterpret_cast<const uint32_t *>(p);
    } else if constexpr (D == 128) {
      const u32x2 w = *reinterpret_cast<const u32x2 *>(p);
      c.v[i][0] = w.x, c.v[i][1] = w.y;
    } else {
      const u32x4 w = *reinterpret_cast<const u32x4 *>(p);
      c.v[i][0] = w.x, c.v[i][1] = w.y, c.v[i][2] = w.z, c.v[i][3] = w.w;
    }
  }
}

// The float16 fragments of channels 4 w + j (j < 4) of a lane's eight tokens from their words v[i]
__device__ __forceinline__ void v_fragments(const uint32_t (&a)[8], u32x4 (&f)[4]) {
#pragma unroll
  for (int p = 0; p < 4; ++p) {  // tokens 2 p, 2 p + 1
    const uint32_t lo = __builtin_amdgcn_perm(a[2 * p + 1], a[2 * p], 0x05010400u);
    const uint32_t hi = __builtin_amdgcn_perm(a[2 * p + 1], a[2 * p], 0x07030602u);
    f[0][p] = codes2<false, false>(lo);
    f[1][p] = codes2<false, true>(lo);
    f[2][p] = codes2<false, false>(hi);
    f[3][p] = codes2<false, true>(hi);
  }
}

template <int D>
__device__ __forceinline__ void zero_rows(const AttendArgs &a, int head, int from, int to) {
  const int per = a.group * D / 8;
  for (long long i = threadIdx.x; i < (long long)(to - from) * per; i += 64 * kAttendWaves) {
    const int row = int(i / per), j = int(i - (long long)row * per);
    *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(a.out) + (size_t(from + row) * a.q_heads + head * a.group) * D +
                               j * 8) = u32x4{};
  }
}

template <int D, bool BF>
__global__ void __launch_bounds__(64 * kAttendWaves) k_attend(AttendArgs a) {
  constexpr int NC = D / 64, NT = D / 16;  // 64-channel groups, 16-channel tiles
  extern __shared__ float lds[];           // [wave][16 rows][D] sums, then [wave][16] maxima, [wave][16] weights
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int head = blockIdx.y / a.row_tiles, b = blockIdx.z;
  int row0, n;
  seq_rows(a.cu, b, a.T, &row0, &n);
  if (!a.part && blockIdx.y % a.row_tiles == 0 && a.cu) {
    // rows before the first sequence or behind the last one come back zero (the joining kernel does it where there is one)
    const int from = b == 0 ? 0 : a.T, to = b == 0 ? min(max(a.cu[0], 0), a.T) : a.T;
    zero_rows<D>(a, head, from, to);
    if (b == a.B - 1) zero_rows<D>(a, head, min(max(a.cu[a.B], 0), a.T), a.T);
  }
  const int rows = n * a.group, page_tokens = 1 << a.page_shift, len = a.lens[b];
  const int begin = blockIdx.x * a.chunk;
  // the row tiles and the last chunk go on past what the caller said of the longest sequence and the most rows
  for (int rt = blockIdx.y - head * a.row_tiles; 16 * rt < rows; rt += a.row_tiles) {
    const int last = min(16 * rt + 15, rows - 1) / a.group;
    int end = len - n + last + 1;  // this workgroup's tokens: [begin, end)
    if (int(blockIdx.x) + 1 < a.chunks) end = min(end, begin + a.chunk);
    if (begin >= end && a.part) continue;
    // the lane's row: query row `mine` of the sequence, seeing the first `sees` places; every row sees those below `all`
    const int flat = min(16 * rt + r, rows - 1), mine = flat / a.group, sub = flat - mine * a.group;
    const int sees = len - n + mine + 1, all = len - n + (16 * rt) / a.group + 1;

    u32x4 qf[2 * NC];
    {
      const uint16_t *q = static_cast<const uint16_t *>(a.q) + size_t(row0 + mine) * a.q_row +
                          size_t(head * a.group + sub) * a.q_head + 16 * g;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        qf[2 * c] = *reinterpret_cast<const u32x4 *>(q + 64 * c);
        qf[2 * c + 1] = *reinterpret_cast<const u32x4 *>(q + 64 * c + 8);
      }
    }
    f32x4 o[NT] = {};
    float m = -INFINITY, l = 0.0f;
    const int first = begin / 32 + wave, stop = (max(end, begin) + 31) / 32, tiles = max(0, (stop - first + 3) / 4);
    const size_t head_bytes = size_t(page_tokens) * D, page_bytes = head_bytes * a.heads;

    for (int t0 = 0; t0 < tiles; t0 += 64) {
      // the pages and scales of this wavefront's next 64 tiles, one a lane
      int number = -1;
      float ks = 0.0f, vs = 0.0f;
      if (t0 + lane < tiles) {
        const int p = (first + 4 * (t0 + lane)) * 32 >> a.page_shift;
        if (p < a.width) number = a.table[size_t(b) * a.width + p];
        if (number >= a.pages) number = -1;
        if (number >= 0) {
          ks = a.ks[size_t(number) * a.heads + head];
          vs = a.vs[size_t(number) * a.heads + head];
        }
      }
      const int nt = min(64, tiles - t0);
      auto fetch = [&](Codes<D> &c, int i) {
        const int page = max(0, __builtin_amdgcn_readlane(number, i));
        const int place = (first + 4 * (t0 + i)) * 32 & (page_tokens - 1);
        load_codes<D>(c, a.kc, a.vc, size_t(page) * page_bytes + size_t(head) * head_bytes + size_t(place) * D, lane);
      };
      Codes<D> next;
      fetch(next, 0);
      for (int i = 0; i < nt; ++i) {
        Codes<D> c = next;
        if (i + 1 < nt) fetch(next, i + 1);
        const int at = (first + 4 * (t0 + i)) * 32;
        const bool there = __builtin_amdgcn_readlane(number, i) >= 0;
        const float k_scale = lane_value(ks, i) * a.scale, v_scale = lane_value(vs, i);
        if (!there) continue;
        f32x4 s[2] = {};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < NC; ++j) {
            const u32x4 w = c.k[h][j];
            s[h] = mfma16<BF>(u32x4{codes2<BF, false>(w.x), codes2<BF, true>(w.x), codes2<BF, false>(w.y), codes2<BF, true>(w.y)},
                              qf[2 * j], s[h]);
            s[h] = mfma16<BF>(u32x4{codes2<BF, false>(w.z), codes2<BF, true>(w.z), codes2<BF, false>(w.w), codes2<BF, true>(w.w)},
                              qf[2 * j + 1], s[h]);
          }
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = s[e >> 2][e & 3] * k_scale;
        const bool edge = at + 32 > all || at + 32 > end;  // some row does not see all of the tile
        bool poison = false;
        if (edge) {
          bool bad = false;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int place = at + 4 * g + (e & 3) + 16 * (e >> 2);
            if (place >= min(sees, end)) x[e] = -INFINITY;
            // places past the last row's: whatever the page holds there must not reach a product (0 NaN is NaN)
#pragma unroll
            for (int w = 0; w < NC; ++w) {
              if (place >= end) c.v[e][w] = 0;
              bad |= nan_code(c.v[e][w]);
            }
          }
          poison = __any(bad);
        }
        float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        top = fmaxf(top, lane_xor16(top));
        top = fmaxf(top, lane_xor32(top));
        if (__any(top > m)) {
          const float to = fmaxf(m, top), keep = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
          m = to;
          l *= keep;
#pragma unroll
          for (int d = 0; d < NT; ++d) o[d] *= keep;
        }
        const float off = m == -INFINITY ? 0.0f : m - 15.0f;
        u32x4 p;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const h2_t w = {_Float16(__builtin_amdgcn_exp2f(x[2 * e] - off)), _Float16(__builtin_amdgcn_exp2f(x[2 * e + 1] - off))};
          l = __builtin_amdgcn_fdot2(w, h2_t{1.0f, 1.0f}, l, false);  // the rounded weights: their sum is what they are divided by
          p[e] = __builtin_bit_cast(uint32_t, w);
        }
#pragma unroll
        for (int w = 0; w < NC; ++w) {
          uint32_t v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = c.v[e][w];
          u32x4 f[4];
          v_fragments(v, f);
          if (poison) {  // a NaN among tokens that not every row sees: it goes to the rows that see it alone
            u32x4 seen;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              seen[e] = (x[2 * e] == -INFINITY ? 0u : 0x3c00u) | (x[2 * e + 1] == -INFINITY ? 0u : 0x3c000000u);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              u32x4 mark;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t lo = f[j][e] & 0x7fffu, hi = f[j][e] & 0x7fff0000u;
                mark[e] = (lo > 0x7c00u ? 0x3c00u : 0u) | (hi > 0x7c000000u ? 0x3c000000u : 0u);
                if (lo > 0x7c00u) f[j][e] &= 0xffff0000u;
                if (hi > 0x7c000000u) f[j][e] &= 0x0000ffffu;
              }
              const f32x4 hit = mfma16<false>(mark, seen, f32x4{});
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (hit[e] > 0.0f) o[4 * w + j][e] = NAN;
            }
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const f32x4 y = mfma16<false>(f[j], p, f32x4{});
#pragma unroll
            for (int e = 0; e < 4; ++e) o[4 * w + j][e] = fmaf(y[e], v_scale, o[4 * w + j][e]);
          }
        }
      }
    }
    // the four wavefronts' sums: a lane's o[4 w + j][e] is channel (4 g + e) D / 16 + 4 w + j of row r
    l += lane_xor16(l);
    l += lane_xor32(l);
    float *sums = lds, *tops = lds + kAttendWaves * 16 * D, *weights = tops + kAttendWaves * 16;
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int w = 0; w < NC; ++w) {
        const f32x4 v = {o[4 * w][e], o[4 * w + 1][e], o[4 * w + 2][e], o[4 * w + 3][e]};
        *reinterpret_cast<f32x4 *>(sums + (wave * 16 + r) * D + (4 * g + e) * NT + 4 * w) = v;
      }
    if (g == 0) tops[wave * 16 + r] = m, weights[wave * 16 + r] = l;
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * (D / 4); i += 64 * kAttendWaves) {
      const int row = i / (D / 4), d = (i - row * (D / 4)) * 4, fl = 16 * rt + row;
      if (fl >= rows) continue;
      float top = tops[row];
#pragma unroll
      for (int w = 1; w < kAttendWaves; ++w) top = fmaxf(top, tops[w * 16 + row]);
      float weight = 0.0f;
      f32x4 v = {};
#pragma unroll
      for (int w = 0; w < kAttendWaves; ++w) {
        const float mw = tops[w * 16 + row], f = mw == -INFINITY && top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw - top);
        const f32x4 y = *reinterpret_cast<const f32x4 *>(sums + (w * 16 + row) * D + d);
        weight = fmaf(weights[w * 16 + row], f, weight);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaf(y[e], f, v[e]);
      }
      const int qr = fl / a.group, h = head * a.group + (fl - qr * a.group);
      const size_t line = size_t(row0 + qr) * a.q_heads + h;
      if (a.part) {
        *reinterpret_cast<f32x4 *>(a.part + (line * a.chunks + blockIdx.x) * D + d) = v;
        if (d == 0)
          *reinterpret_cast<float2 *>(a.part + size_t(a.T) * a.q_heads * a.chunks * D + (line * a.chunks + blockIdx.x) * 2) =
              float2{top, weight};
      } else {
        const float inv = weight == 0.0f ? 0.0f : 1.0f / weight;
        const uint32_t two[2] = {
            BF ? uint32_t(f32_to_bf16(v[0] * inv)) | uint32_t(f32_to_bf16(v[1] * inv)) << 16
               : __builtin_bit_cast(uint32_t, h2_t{_Float16(v[0] * inv), _Float16(v[1] * inv)}),
            BF ? uint32_t(f32_to_bf16(v[2] * inv)) | uint32_t(f32_to_bf16(v[3] * inv)) << 16
               : __builtin_bit_cast(uint32_t, h2_t{_Float16(v[2] * inv), _Float16(v[3] * inv)})};
        *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(a.out) + line * D + d) = u32x2{two[0], two[1]};
      }
    }
    __syncthreads();
  }
}

// One workgroup a query row and head: its sequence's chunks, the same ones as k_attend wrote, joined in order
template <int D, bool BF>
__global__ void __launch_bounds__(256) k_attend_join(AttendArgs a) {
  constexpr int LANES = D / 4, GROUPS = 256 / LANES;  // threads over the channels, and over the chunks
  __shared__ float sums[GROUPS][D];
  __shared__ float weights[GROUPS];
  const int line = blockIdx.x, row = line / a.q_heads;
  const int b = a.cu ? last_at(a.cu, a.B, row, [](int c, int) { return (long long)c; }) : row;
  int row0 = 0, n = 0;
  if (b >= 0) seq_rows(a.cu, b, a.T, &row0, &n);
  const int r = row - row0;
  // the chunks that k_attend worked: those below the end of the row's tile of 16
  int chunks = 0;
  if (r < n) {
    const int flat = r * a.group + (line - row * a.q_heads) % a.group;
    const int last = min((flat | 15), n * a.group - 1) / a.group;
    chunks = min(a.chunks, max(0, (a.lens[b] - n + last + 1 + a.chunk - 1) / a.chunk));
  }
  const float2 *ml = reinterpret_cast<const float2 *>(a.part + size_t(a.T) * a.q_heads * a.chunks * D) + size_t(line) * a.chunks;
  float top = -INFINITY;
  for (int i = threadIdx.x & 63; i < chunks; i += 64) top = fmaxf(top, ml[i].x);
  top = wave_max(top);
  const int grp = threadIdx.x / LANES, d = (threadIdx.x - grp * LANES) * 4;
  f32x4 v = {};
  float weight = 0.0f;
  for (int i = grp; i < chunks; i += GROUPS) {
    const float2 c = ml[i];
    if (c.y == 0.0f) continue;  // the row sees nothing of it (the largest weight seen is 2^15; one that is NaN goes on)
    const float f = c.x == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(c.x - top);
    const f32x4 y = *reinterpret_cast<const f32x4 *>(a.part + (size_t(line) * a.chunks + i) * D + d);
    weight = fmaf(c.y, f, weight);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = fmaf(y[e], f, v[e]);
  }
  *reinterpret_cast<f32x4 *>(&sums[grp][d]) = v;
  if (d == 0) weights[grp] = weight;
  __syncthreads();
  if (threadIdx.x >= LANES) return;
#pragma unroll
  for (int j = 1; j < GROUPS; ++j) {
    const f32x4 y = *reinterpret_cast<const f32x4 *>(&sums[j][d]);
    weight += weights[j];
    v += y;
  }
  const float inv = weight == 0.0f ? 0.0f : 1.0f / weight;
  uint16_t *out = static_cast<uint16_t *>(a.out) + size_t(line) * D + d;
  u32x2 w;
#pragma unroll
  for (int j = 0; j < 2; ++j)
    w[j] = BF ? uint32_t(f32_to_bf16(v[2 * j] * inv)) | uint32_t(f32_to_bf16(v[2 * j + 1] * inv)) << 16
              : __builtin_bit_cast(uint32_t, h2_t{_Float16(v[2 * j] * inv), _Float16(v[2 * j + 1] * inv)});
  *reinterpret_cast<u32x2 *>(out) = w;
}

// The tokens a chunk: the longest that gives 1,024 workgroups (four a CU), within 128 (a tile for each wavefront) and 2,048
static int attend_chunk(int B, int heads, int row_tiles, int longest) {
  int chunk = 2048;
  while (chunk > 128 && (long long)B * heads * row_tiles * ((longest + chunk - 1) / chunk) < 1024) chunk >>= 1;
  return chunk;
}

static int attend_plan(const char *fn, int T, int q_heads, int heads, int D, int B, int most_rows, int longest, int *row_tiles,
                       int *chunk, int *chunks) {
  LMOE_REQUIRE(D == 64 || D == 128 || D == 256, LMOE_ESHAPE, "%s: heads of %d channels (64, 128 and 256 are served)", fn, D);
  LMOE_REQUIRE(heads > 0 && q_heads > 0 && q_heads % heads == 0, LMOE_ESHAPE, "%s: %d query heads over %d key heads", fn, q_heads,
               heads);
  LMOE_REQUIRE(T >= 0 && B >= 0 && B <= 65535 && most_rows > 0 && longest > 0, LMOE_ESHAPE,
               "%s: %d rows, %d sequences (65535 at most) of %d rows and %d tokens", fn, T, B, most_rows, longest);
  const long long flat = (long long)(most_rows < T ? most_rows : (T > 0 ? T : 1)) * (q_heads / heads);
  const long long tiles = (flat + 15) / 16, room = 65535 / heads;
  LMOE_REQUIRE(room > 0, LMOE_ESHAPE, "%s: %d key heads", fn, heads);
  *row_tiles = int(tiles < room ? tiles : room);
  *chunk = attend_chunk(B, heads, *row_tiles, longest);
  *chunks = (longest + *chunk - 1) / *chunk;
  return 0;
}

}  // namespace lmoe

using namespace lmoe;

extern "C" size_t lmoe_kv_attend_workspace_bytes(int T, int q_heads, int heads, int D, int B, int most_rows, int longest) {
  int row_tiles, chunk, chunks;
  if (attend_plan("lmoe_kv_attend_workspace_bytes", T, q_heads, heads, D, B, most_rows, longest, &row_tiles, &chunk, &chunks))
    return 0;
  return chunks > 1 ? size_t(T) * q_heads * chunks * (D + 2) * sizeof(float) : 0;
}

extern "C" int lmoe_kv_attend(const void *q, int dtype, long long q_row, long long q_head, int T, int q_heads, int heads, int D,
                              const int *cu, const int *lens, int B, const int *table, int width, const uint8_t *k_codes,
                              const float *k_scale, const uint8_t *v_codes, const float *v_scale, int pages, int page,
                              int most_rows, int longest, float scale, void *workspace, size_t workspace_bytes, void *out,
                              void *stream) {
  const char *fn = "lmoe_kv_attend";
  LMOE_REQUIRE(dtype == LMOE_F16 || dtype == LMOE_BF16, LMOE_EINVAL, "%s: dtype %d (float16 and bfloat16 are served)", fn, dtype);
  int row_tiles, chunk, chunks;
  if (const int rc = attend_plan(fn, T, q_heads, heads, D, B, most_rows, longest, &row_tiles, &chunk, &chunks)) return rc;
  LMOE_REQUIRE(page == 32 || page == 64 || page == 128, LMOE_ESHAPE, "%s: pages of %d tokens (32, 64 and 128 are served)", fn,
               page);
  LMOE_REQUIRE(pages > 0 && width > 0, LMOE_ESHAPE, "%s: %d pages, a table of %d", fn, pages, width);
  if (T == 0) return 0;
  LMOE_REQUIRE(B > 0 && (cu || T == B), LMOE_ESHAPE, "%s: %d rows of %d sequences need their offsets", fn, T, B);
  LMOE_REQUIRE(scale > 0.0f && scale < INFINITY, LMOE_EINVAL, "%s: scale %g", fn, double(scale));
  LMOE_REQUIRE(q && lens && table && k_codes && k_scale && v_codes && v_scale && out, LMOE_EINVAL, "%s: null pointer", fn);
  LMOE_REQUIRE(aligned16(q) && q_row % 8 == 0 && q_head % 8 == 0 && aligned16(k_codes) && aligned16(v_codes) && aligned16(out),
               LMOE_EALIGN, "%s: rows and codes must be 16-byte aligned", fn);
  const size_t need = chunks > 1 ? size_t(T) * q_heads * chunks * (D + 2) * sizeof(float) : 0;
  LMOE_REQUIRE(need == 0 || (workspace && aligned16(workspace) && workspace_bytes >= need), LMOE_EWORKSPACE,
               "%s: a 16-byte aligned workspace of %zu bytes is needed", fn, need);
  LMOE_REQUIRE((long long)T * q_heads < (1ll << 31), LMOE_ESHAPE, "%s: %d rows of %d heads", fn, T, q_heads);
  AttendArgs a = {q, q_row, q_head, k_codes, v_codes, k_scale, v_scale, table, lens, cu, out,
                  need ? static_cast<float *>(workspace) : nullptr, scale * kLog2e, T, B, q_heads, heads,
                  page == 32 ? 5 : page == 64 ? 6 : 7, pages, width, q_heads / heads, row_tiles, chunk, chunks};
  hipStream_t st = (hipStream_t)stream;
  auto go = [&](auto kernel, auto join) -> int {
    const size_t lds = size_t(kAttendWaves) * 16 * (D + 2) * sizeof(float);
    if (const int rc = allow_lds(kernel, lds, fn)) return rc;
    launch(kernel, dim3(unsigned(chunks), unsigned(heads * row_tiles), unsigned(B)), dim3(64 * kAttendWaves), lds, st, a);
    LMOE_LAUNCHED(fn);
    if (need) {
      launch(join, dim3(unsigned(T) * unsigned(q_heads)), dim3(256), 0, st, a);
      LMOE_LAUNCHED(fn);
    }
    return 0;
  };
  const bool bf = dtype == LMOE_BF16;
  if (D == 64) return bf ? go(k_attend<64, true>, k_attend_join<64, true>) : go(k_attend<64, false>, k_attend_join<64, false>);
  if (D == 128)
    return bf ? go(k_attend<128, true>, k_attend_join<128, true>) : go(k_attend<128, false>, k_attend_join<128, false>);
  return bf ? go(k_attend<256, true>, k_attend_join<256, true>) : go(k_attend<256, false>, k_attend_join<256, false>);
}
