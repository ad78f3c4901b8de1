// Attention of the newest rows of each sequence (one token, or a speculative decoder's few) over the 8-bit paged cache.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - m),  over the places j < len - (n - 1 - r) of row r of n
//
// One pass over the keys and values with a running maximum m. Bound by the cache's bytes: 2 width a token and key head, read
// once for every 16 (row, query head of the group) pairs of a sequence, which fill a matrix-core tile's columns: once for a
// token of up to 16 heads a group, three times for five draft rows of 8, eight times for sixteen.
//
// A wavefront takes 32 tokens a step, straight from global memory to registers; no LDS until the end. Products are written
// so that nothing has to change lanes between them:
//   scores^T = K Q^T   A = 16 tokens (lane & 15) x 32 channels, 16 codes a lane from one load, B = Q^T; a lane ends with
//                      four tokens (4 (lane >> 4) + i) of one query row (lane & 15) from each of two 16-token tiles;
//   out^T += V^T P^T   B = those eight tokens' weights as they lie; A = the same eight tokens' codes of one channel. A lane
//                      loads width / 16 neighbouring channels of its eight tokens, and byte permutes pair up the tokens.
// e4m3 codes are exact in float16 and bfloat16, so q keeps its type; weights are float16, times 2^11 so that a weight down to
// 2^-25 of the row's largest keeps all eleven bits (a long context under one token that stands out lives there). The scales
// multiply float32 sums.
//
// All of a call's work lies on one line of units of 128 tokens (one 32-token tile for each of a workgroup's four wavefronts):
// sequence by sequence, in it each tile of 16 rows and key head, in that the sequence's units in order. Two workgroups a CU
// take equal stretches of the line, whatever the sequences' lengths. A workgroup finishes the items that lie in its stretch
// whole; the two that may reach over its ends go to its two places in the workspace, and a second kernel joins those. Where
// sequences are short, each is one unit and there is nothing to join.
//
// Measured: 64 sequences of 1,024 to 16,384 tokens, 32 heads over 4 of 128: 75 us, 5.0 TB/s, and 4.5 to join (chunks of one
// length on a grid of the longest: 125, two thirds of the workgroups empty and the rest uneven over the XCDs); one sequence of
// 131,072: 26 and 5.4; heads of 256: 79 (190), with 256 registers and five spilled (24 bytes of scratch a lane). One unit takes
// 5.7 (width 64) to 8.4 us (256) from launch to end: lengths, pages, codes and the wavefronts' join, one after the other.
#include "rows.h"

namespace lmoe {

constexpr int kAttendWaves = 4;
constexpr float kLog2e = 1.4426950408889634f;

// A weight is 2^(score - maximum in use + kLift), the maximum lagging at most kLag behind
constexpr float kLift = 11.0f, kLag = 4.0f;

struct AttendArgs {
  const void *q;
  long long q_row, q_head;
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int *table, *lens, *cu;
  void *out;    // [T][q_heads][D]
  float *part;  // [workgroups][2] of [16 rows][D] sums and [16 rows] of {maximum, weight}; null: an item is one unit
  int2 *joins;  // [T][q_heads]: the first place of a row's item (-1: one workgroup had it all), 16 times its last workgroup
                // and the row of the tile
  float scale;  // times log2 e
  int T, B, q_heads, heads, page_shift, unit_shift, pages, width, group, groups;  // groups: workgroups of k_attend
};

// A sequence's share of the line
struct Share {
  int row0, n, len, tiles, units;  // rows, tokens, tiles of 16 (row, query head of the group) pairs, units an item
  __device__ __forceinline__ int total(int heads) const { return tiles * heads * units; }
};
__device__ __forceinline__ Share share(const AttendArgs &a, int row0, int n, int len) {
  return {row0, n, len, (n * a.group + 15) >> 4,
          a.part ? ((min(max(len, 1), a.width << a.page_shift) - 1) >> a.unit_shift) + 1 : 1};
}

// Inclusive sums over a wavefront's lanes
__device__ __forceinline__ int wave_scan(int v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int u = __shfl_up(v, d);
    if (int(threadIdx.x & 63) >= d) v += u;
  }
  return v;
}

// Workgroup w of n has the units [stretch(w), stretch(w + 1)) of a line
__device__ __forceinline__ int stretch(int line, int w, int n) { return int((long long)line * w / n); }

// 64 sequences of the line, in LDS for each wavefront (in registers they would be there through the whole loop)
struct Seqs {
  int3 *seq;  // [64] first row, rows, tokens
  int *ends;  // [64] where a sequence ends on the line
  int b0;     // the first of them
  int base;   // where that begins
  bool rising = true;  // of the lane's sequences: offsets that do not fall

  __device__ __forceinline__ void load(const AttendArgs &a, int from, int begins) {
    const int lane = threadIdx.x & 63, b = from + lane;
    int3 s = {0, 0, 0};
    if (b < a.B) {
      rising &= seq_rows(a.cu, b, a.T, &s.x, &s.y);
      s.z = a.lens[b];
    }
    seq[lane] = s;
    ends[lane] = begins + wave_scan(share(a, s.x, s.y, s.z).total(a.heads));
    b0 = from;
    base = begins;
  }
  __device__ __forceinline__ int end() const { return __builtin_amdgcn_readfirstlane(ends[63]); }
};
constexpr size_t kSeqsLds = kAttendWaves * 64 * (sizeof(int3) + sizeof(int));

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

// 0x80 in the place of each of a word's four codes that is NaN
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ~((~w & 0x7f7f7f7fu) + 0x7f7f7f7fu) & 0x80808080u; }

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
__device__ __forceinline__ void zero_rows(const AttendArgs &a, int from, int to) {
  const long long per = (long long)a.q_heads * D / 8;
  u32x4 *out = reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(a.out) + size_t(from) * a.q_heads * D);
  for (long long i = threadIdx.x; i < (to - from) * per; i += 64 * kAttendWaves) out[i] = u32x4{};
  if (a.part)
    for (long long i = threadIdx.x; i < (long long)(to - from) * a.q_heads; i += 64 * kAttendWaves)
      a.joins[(long long)from * a.q_heads + i] = int2{-1, 0};
}

template <bool BF>
__device__ __forceinline__ void store4(void *out, size_t at, f32x4 v, float weight) {
  const float inv = weight == 0.0f ? 0.0f : 1.0f / weight;
  u32x2 w;
#pragma unroll
  for (int j = 0; j < 2; ++j)
    w[j] = BF ? uint32_t(f32_to_bf16(v[2 * j] * inv)) | uint32_t(f32_to_bf16(v[2 * j + 1] * inv)) << 16
              : __builtin_bit_cast(uint32_t, h2_t{_Float16(v[2 * j] * inv), _Float16(v[2 * j + 1] * inv)});
  *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(out) + at) = w;
}

template <int D>
constexpr int kPlace = 16 * (D + 2);  // floats of a place in the workspace
template <int D>
constexpr int kRow = D + 4;  // floats of a row of sums in LDS: 16 rows' same channels lie in different banks
template <int D>
constexpr size_t kSumsLds = size_t(kAttendWaves) * 16 * (kRow<D> + 2) * sizeof(float);
template <int D>
constexpr size_t kAttendLds = kSumsLds<D> + kSeqsLds;

template <int D, bool BF>
__global__ void __launch_bounds__(64 * kAttendWaves, D == 256 ? 2 : 3) k_attend(AttendArgs a) {
  constexpr int NC = D / 64, NT = D / 16;  // 64-channel groups, 16-channel tiles
  extern __shared__ float lds[];           // [wave][16 rows][kRow] sums, then [wave][16] maxima, [wave][16] weights; then Seqs
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  if (blockIdx.x == 0 && a.cu) {  // rows before the first sequence or behind the last one come back zero
    zero_rows<D>(a, 0, min(max(a.cu[0], 0), a.T));
    zero_rows<D>(a, min(max(a.cu[a.B], 0), a.T), a.T);
  }
  char *seqs_at = reinterpret_cast<char *>(lds) + kSumsLds<D>;
  Seqs seqs = {reinterpret_cast<int3 *>(seqs_at + kAttendWaves * 64 * sizeof(int)) + wave * 64,
               reinterpret_cast<int *>(seqs_at) + wave * 64, 0, 0};
  seqs.load(a, 0, 0);
  int line = seqs.end();
  if (a.B > 64) {  // the rest of the line: a lane adds up every 64th sequence
    int more = 0;
#pragma unroll 4
    for (int b = 64 + lane; b < a.B; b += 64) {
      int row0, n;
      seqs.rising &= seq_rows(a.cu, b, a.T, &row0, &n);
      more += share(a, row0, n, a.lens[b]).total(a.heads);
    }
    line += __builtin_amdgcn_readlane(wave_scan(more), 63);
  }
  if (!__all(seqs.rising)) return;  // sequences with the same rows could have more units than 32 bits count
  // no more workgroups than units: each has one at least, so that every one between an item's first and last writes its place
  const int groups = min(a.groups, line);
  if (int(blockIdx.x) >= groups) return;
  int at_unit = stretch(line, blockIdx.x, groups);
  const int stop_unit = stretch(line, blockIdx.x + 1, groups);
  const int first_unit = at_unit;
  const int page_tokens = 1 << a.page_shift;
  const size_t head_bytes = size_t(page_tokens) * D, page_bytes = head_bytes * a.heads;

  while (at_unit < stop_unit) {
    while (at_unit >= seqs.end()) seqs.load(a, seqs.b0 + 64, seqs.end());
    const int in64 = __ffsll(__ballot(seqs.ends[opaque(lane)] > at_unit)) - 1, b = seqs.b0 + in64;
    const int3 found = seqs.seq[in64];
    const Share s = share(a, __builtin_amdgcn_readfirstlane(found.x), __builtin_amdgcn_readfirstlane(found.y),
                          __builtin_amdgcn_readfirstlane(found.z));
    const int base = in64 ? __builtin_amdgcn_readfirstlane(seqs.ends[in64 - 1]) : seqs.base;
    const int item = (at_unit - base) / s.units, unit0 = (at_unit - base) - item * s.units;
    const int units = min(s.units - unit0, stop_unit - at_unit);
    const int rt = item / a.heads, head = item - rt * a.heads, rows = s.n * a.group;
    const bool whole = units == s.units;
    const int last = min(16 * rt + 15, rows - 1) / a.group;
    // this stretch's tokens [begin, end): an item's last unit ends with what its last row sees
    const int begin = unit0 << a.unit_shift;
    int end = min(s.len - s.n + last + 1, a.width << a.page_shift);  // (the table has no places past that)
    if (unit0 + units < s.units) end = min(end, begin + (units << a.unit_shift));
    // the lane's row: query row `mine` of the sequence, seeing the first `sees` places; every row sees those below `all`
    const int flat = min(16 * rt + r, rows - 1), mine = flat / a.group, sub = flat - mine * a.group;
    const int sees = s.len - s.n + mine + 1, all = s.len - s.n + (16 * rt) / a.group + 1;

    u32x4 qf[2 * NC];
    {
      const uint16_t *q = static_cast<const uint16_t *>(a.q) + size_t(s.row0 + mine) * a.q_row +
                          size_t(head * a.group + sub) * a.q_head + 16 * g;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        qf[2 * c] = *reinterpret_cast<const u32x4 *>(q + 64 * c);
        qf[2 * c + 1] = *reinterpret_cast<const u32x4 *>(q + 64 * c + 8);
      }
    }
    f32x4 o[NT] = {};
    float m = -INFINITY, l = 0.0f;
    uint8_t *marks = reinterpret_cast<uint8_t *>(lds + wave * 16 * kRow<D>);
    const int first = begin / 32 + wave, tiles = max(0, ((max(end, begin) + 31) / 32 - first + 3) / 4);

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
      auto work = [&](Codes<D> &c, int i) {
        const int at = (first + 4 * (t0 + i)) * 32;
        const bool held = __builtin_amdgcn_readlane(number, i) >= 0;
        const float k_scale = lane_value(ks, i) * a.scale, v_scale = lane_value(vs, i);
        f32x4 sc[2] = {};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < NC; ++j) {
            const u32x4 w = c.k[h][j];
            sc[h] = mfma16<BF>(
                u32x4{codes2<BF, false>(w.x), codes2<BF, true>(w.x), codes2<BF, false>(w.y), codes2<BF, true>(w.y)}, qf[2 * j],
                sc[h]);
            sc[h] = mfma16<BF>(
                u32x4{codes2<BF, false>(w.z), codes2<BF, true>(w.z), codes2<BF, false>(w.w), codes2<BF, true>(w.w)},
                qf[2 * j + 1], sc[h]);
          }
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = sc[e >> 2][e & 3] * k_scale;
        bool poison = false;
        if (!held || at + 32 > all || at + 32 > end) {  // some row does not see all of the tile
          const int there = opaque(held ? end - at - 4 * g : 0), left = min(there, sees - at - 4 * g);
          uint32_t bad = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int place = (e & 3) + 16 * (e >> 2);
            if (place >= left) x[e] = -INFINITY;
            // places past the last row's: whatever the page holds there must not reach a product (0 NaN is NaN)
#pragma unroll
            for (int w = 0; w < NC; ++w) {
              if (place >= there) c.v[e][w] = 0;
              bad |= nan_codes(c.v[e][w]);
            }
          }
          poison = __any(bad != 0);
          if (poison) {  // NaN among tokens that not every row sees: taken out, and noted in LDS by token and four channels
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
              for (int w = 0; w < NC; ++w) {
                const uint32_t z = nan_codes(c.v[e][w]) >> 7;
                c.v[e][w] &= ~(z * 0xffu);
                marks[(4 * g + (e & 3) + 16 * (e >> 2)) * (D / 4) + r * NC + w] = uint8_t(z | z >> 7 | z >> 14 | z >> 21);
              }
          }
        }
        float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        top = fmaxf(top, lane_xor16(top));
        top = fmaxf(top, lane_xor32(top));
        if (__any(top > m + kLag)) {
          const float to = fmaxf(m, top), keep = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
          m = to;
          l *= keep;
#pragma unroll
          for (int d = 0; d < NT; ++d) o[d] *= keep;
        }
        const float lift = m == -INFINITY ? 0.0f : kLift - m;
        u32x4 p;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const h2_t w = {_Float16(__builtin_amdgcn_exp2f(x[2 * e] + lift)), _Float16(__builtin_amdgcn_exp2f(x[2 * e + 1] + lift))};
          l = __builtin_amdgcn_fdot2(w, h2_t{1.0f, 1.0f}, l, false);  // the rounded weights' sum is what the row is divided by
          p[e] = __builtin_bit_cast(uint32_t, w);
        }
#pragma unroll
        for (int w = 0; w < NC; ++w) {
          uint32_t v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = c.v[e][w];
          u32x4 f[4];
          v_fragments(v, f);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const f32x4 y = mfma16<false>(f[j], p, f32x4{});
#pragma unroll
            for (int e = 0; e < 4; ++e) o[4 * w + j][e] = fmaf(y[e], v_scale, o[4 * w + j][e]);
          }
        }
        if (poison) {  // and given to the rows that do see them
          for (int place = 0; place < 32; ++place)
#pragma unroll
            for (int i = 0; i < 4 * NC; ++i) {
              const uint32_t z = at + place < sees ? marks[place * (D / 4) + (4 * g + i / NC) * NC + i % NC] : 0;
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (z >> j & 1) o[4 * (i % NC) + j][i / NC] = NAN;
            }
        }
      };
      if constexpr (D < 256) {  // two sets of codes in turn, so that none is moved; at width 256 there are no registers for that
        Codes<D> one, two;
        fetch(one, 0);
        int i = 0;
        for (; i + 2 < nt; i += 2) {
          fetch(two, i + 1);
          work(one, i);
          fetch(one, i + 2);
          work(two, i + 1);
        }
        if (i + 1 < nt) fetch(two, i + 1);
        work(one, i);
        if (i + 1 < nt) work(two, i + 1);
      } else {
        Codes<D> next;
        fetch(next, 0);
        for (int i = 0; i < nt; ++i) {
          Codes<D> c = next;
          if (i + 1 < nt) fetch(next, i + 1);
          work(c, i);
        }
      }
    }
    // the four wavefronts' sums: a lane's o[4 w + j][e] is channel (4 g + e) D / 16 + 4 w + j of row r
    l += lane_xor16(l);
    l += lane_xor32(l);
    const int tid = opaque(int(threadIdx.x)), er = tid & 15, eg = tid >> 4 & 3;  // opaque: no address of this lives through the loop
    float *sums = lds, *tops = lds + kAttendWaves * 16 * kRow<D>, *weights = tops + kAttendWaves * 16;
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int w = 0; w < NC; ++w) {
        const f32x4 v = {o[4 * w][e], o[4 * w + 1][e], o[4 * w + 2][e], o[4 * w + 3][e]};
        *reinterpret_cast<f32x4 *>(sums + (wave * 16 + er) * kRow<D> + (4 * eg + e) * NT + 4 * w) = v;
      }
    if (eg == 0) tops[wave * 16 + er] = m, weights[wave * 16 + er] = l;
    __syncthreads();
    if (a.part && unit0 == 0) {  // what the joining kernel has to do for the item's rows
      const int2 join = {whole ? -1 : int(blockIdx.x) * 2 + (at_unit == first_unit ? 0 : 1),
                         int(((long long)(at_unit + s.units) * groups - 1) / line) * 16 + tid};
      const int fl = 16 * rt + tid, qr = fl / a.group;
      if (tid < 16 && fl < rows) a.joins[size_t(s.row0 + qr) * a.q_heads + head * a.group + (fl - qr * a.group)] = join;
    }
    float *place = whole ? nullptr : a.part + (size_t(blockIdx.x) * 2 + (at_unit == first_unit ? 0 : 1)) * kPlace<D>;
    for (int i = tid; i < 16 * (D / 4); i += 64 * kAttendWaves) {
      const int row = i / (D / 4), d = (i - row * (D / 4)) * 4, fl = 16 * rt + row;
      if (fl >= rows) break;
      float top = tops[row];
#pragma unroll
      for (int w = 1; w < kAttendWaves; ++w) top = fmaxf(top, tops[w * 16 + row]);
      float weight = 0.0f;
      f32x4 v = {};
#pragma unroll
      for (int w = 0; w < kAttendWaves; ++w) {
        const float mw = tops[w * 16 + row], f = mw == -INFINITY && top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw - top);
        const f32x4 y = *reinterpret_cast<const f32x4 *>(sums + (w * 16 + row) * kRow<D> + d);
        weight = fmaf(weights[w * 16 + row], f, weight);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaf(y[e], f, v[e]);
      }
      if (whole) {
        const int qr = fl / a.group, h = head * a.group + (fl - qr * a.group);
        store4<BF>(a.out, (size_t(s.row0 + qr) * a.q_heads + h) * D + d, v, weight);
      } else {
        *reinterpret_cast<f32x4 *>(place + row * D + d) = v;
        if (d == 0) *reinterpret_cast<float2 *>(place + 16 * D + 2 * row) = float2{top, weight};
      }
    }
    __syncthreads();
    at_unit += units;
  }
}

// One workgroup a query row and head (blockIdx.x first): where more than one workgroup of k_attend had its item, their places joined in order
template <int D, bool BF>
__global__ void __launch_bounds__(256) k_attend_join(AttendArgs a) {
  constexpr int LANES = D / 4, PARTS = 256 / LANES;  // threads over the channels, and over the places
  __shared__ float sums[PARTS][D];
  __shared__ float tops[PARTS], weights[PARTS];
  const size_t line = blockIdx.x + size_t(blockIdx.y) * gridDim.x;
  if (line >= size_t(a.T) * a.q_heads) return;
  const int2 join = a.joins[line];
  if (join.x < 0) return;
  const int in = join.y & 15, w0 = min(join.x >> 1, a.groups - 1), w1 = min(join.y >> 4, a.groups - 1);
  const int part = threadIdx.x / LANES, d = (threadIdx.x - part * LANES) * 4;
  f32x4 v = {};
  float top = -INFINITY, weight = 0.0f;
  // a place that the row sees nothing of weighs 0 (one that it sees weighs 2^(kLift - kLag) at least; NaN goes on)
  auto add = [&](float m, float l, f32x4 y) {
    const float to = fmaxf(top, l == 0.0f ? top : m);
    const float keep = weight == 0.0f ? 0.0f : to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - to);
    const float f = l == 0.0f ? 0.0f : to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
    top = to;
    weight = fmaf(l, f, weight * keep);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = fmaf(y[e], f, v[e] * keep);
  };
  for (int first = w0 + part; first <= w1; first += 4 * PARTS) {  // four places' loads at a time
    float2 c[4];
    f32x4 y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int w = min(first + j * PARTS, w1);
      const float *place = a.part + (size_t(w) * 2 + (w == w0 ? join.x & 1 : 0)) * kPlace<D>;
      c[j] = *reinterpret_cast<const float2 *>(place + 16 * D + 2 * in);
      y[j] = *reinterpret_cast<const f32x4 *>(place + in * D + d);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (first + j * PARTS <= w1) add(c[j].x, c[j].y, y[j]);
  }
  *reinterpret_cast<f32x4 *>(&sums[part][d]) = v;
  if (d == 0) tops[part] = top, weights[part] = weight;
  __syncthreads();
  if (threadIdx.x >= LANES) return;
#pragma unroll 1
  for (int j = 1; j < PARTS; ++j) add(tops[j], weights[j], *reinterpret_cast<const f32x4 *>(&sums[j][d]));
  store4<BF>(a.out, line * D + d, v, weight);
}

// Sequences of up to 512 tokens (four tiles a wavefront) are one unit each: joining would cost what splitting gains
constexpr int kShort = 512;

// Two workgroups a CU. The GPU holds three (width 128) or four (64), but three gain 1 % on 64 sequences of 16,384 tokens
// (75.7 -> 74.9 us), and every workgroup more is another place to join (131,072 tokens of one sequence: 7.5 -> 8.8 us)
constexpr int kAttendGroups = 512;

struct AttendPlan {
  int groups;      // workgroups
  int unit_shift;  // a unit's tokens
  bool split;    // items of more than one unit
  size_t places, bytes;  // the workspace's places, and all of it
};

static int attend_plan(const char *fn, int T, int q_heads, int heads, int D, int B, int most_rows, int longest, AttendPlan *plan) {
  LMOE_REQUIRE(D == 64 || D == 128 || D == 256, LMOE_ESHAPE, "%s: heads of %d channels (64, 128 and 256 are served)", fn, D);
  LMOE_REQUIRE(heads > 0 && q_heads > 0 && q_heads % heads == 0, LMOE_ESHAPE, "%s: %d query heads over %d key heads", fn, q_heads,
               heads);
  LMOE_REQUIRE(T >= 0 && B >= 0 && most_rows > 0 && longest > 0, LMOE_ESHAPE, "%s: %d rows, %d sequences of %d rows and %d tokens",
               fn, T, B, most_rows, longest);
  const long long flat = (long long)(most_rows < T ? most_rows : (T > 0 ? T : 1)) * (q_heads / heads);
  const long long items = (flat + 15) / 16 * heads * (B > 0 ? B : 1);
  plan->split = longest > kShort;
  plan->unit_shift = 7;
  long long n = items;
  if (plan->split) {
    const long long units = items * ((longest + 127ll) / 128);
    n = kAttendGroups < units ? kAttendGroups : units;
  }
  plan->groups = int(n < (1 << 20) ? n : (1 << 20));  // (a workgroup takes several items where there are more)
  plan->places = size_t(plan->groups) * 2 * 16 * (D + 2) * sizeof(float);
  plan->bytes = plan->split ? plan->places + size_t(T) * q_heads * sizeof(int2) : 0;
  return 0;
}

}  // namespace lmoe

using namespace lmoe;

extern "C" size_t lmoe_kv_attend_workspace_bytes(int T, int q_heads, int heads, int D, int B, int most_rows, int longest) {
  AttendPlan plan;
  return attend_plan("lmoe_kv_attend_workspace_bytes", T, q_heads, heads, D, B, most_rows, longest, &plan) ? 0 : plan.bytes;
}

extern "C" int lmoe_kv_attend(const void *q, int dtype, long long q_row, long long q_head, int T, int q_heads, int heads, int D,
                              const int *cu, const int *lens, int B, const int *table, int width, const uint8_t *k_codes,
                              const float *k_scale, const uint8_t *v_codes, const float *v_scale, int pages, int page,
                              int most_rows, int longest, float scale, void *workspace, size_t workspace_bytes, void *out,
                              void *stream) {
  const char *fn = "lmoe_kv_attend";
  LMOE_REQUIRE(dtype == LMOE_F16 || dtype == LMOE_BF16, LMOE_EINVAL, "%s: dtype %d (float16 and bfloat16 are served)", fn, dtype);
  AttendPlan plan;
  if (const int rc = attend_plan(fn, T, q_heads, heads, D, B, most_rows, longest, &plan)) return rc;
  LMOE_REQUIRE(page == 32 || page == 64 || page == 128, LMOE_ESHAPE, "%s: pages of %d tokens (32, 64 and 128 are served)", fn,
               page);
  const int page_shift = page == 32 ? 5 : page == 64 ? 6 : 7;
  LMOE_REQUIRE(pages > 0 && width > 0 && width <= (1 << 30) >> page_shift, LMOE_ESHAPE, "%s: %d pages, a table of %d", fn, pages,
               width);
  if (T == 0) return 0;
  LMOE_REQUIRE(B > 0 && (cu || T == B), LMOE_ESHAPE, "%s: %d rows of %d sequences need their offsets", fn, T, B);
  LMOE_REQUIRE(scale > 0.0f && scale < INFINITY, LMOE_EINVAL, "%s: scale %g", fn, double(scale));
  LMOE_REQUIRE(q && lens && table && k_codes && k_scale && v_codes && v_scale && out, LMOE_EINVAL, "%s: null pointer", fn);
  LMOE_REQUIRE(aligned16(q) && q_row % 8 == 0 && q_head % 8 == 0 && aligned16(k_codes) && aligned16(v_codes) && aligned16(out),
               LMOE_EALIGN, "%s: rows and codes must be 16-byte aligned", fn);
  LMOE_REQUIRE(!plan.split || (workspace && aligned16(workspace) && workspace_bytes >= plan.bytes), LMOE_EWORKSPACE,
               "%s: a 16-byte aligned workspace of %zu bytes is needed", fn, plan.bytes);
  LMOE_REQUIRE((long long)T * q_heads < (1ll << 27), LMOE_ESHAPE, "%s: %d rows of %d heads", fn, T, q_heads);
  // units are counted in 32 bits: longer ones where a table's room could hold more than that
  const long long most = ((long long)T * (q_heads / heads) / 16 + B) * heads;
  while ((most * ((((long long)width << page_shift) >> plan.unit_shift) + 1)) >> 31 && plan.unit_shift < 30) ++plan.unit_shift;
  LMOE_REQUIRE(most * ((((long long)width << page_shift) >> plan.unit_shift) + 1) < (1ll << 31), LMOE_ESHAPE,
               "%s: %d rows of %d sequences and %d key heads", fn, T, B, heads);
  AttendArgs a = {q, q_row, q_head, k_codes, v_codes, k_scale, v_scale, table, lens, cu, out,
                  plan.split ? static_cast<float *>(workspace) : nullptr,
                  plan.split ? reinterpret_cast<int2 *>(static_cast<char *>(workspace) + plan.places) : nullptr, scale * kLog2e, T, B, q_heads, heads, page_shift, plan.unit_shift, pages,
                  width, q_heads / heads, plan.groups};
  hipStream_t st = (hipStream_t)stream;
  auto go = [&](auto kernel, auto join, size_t lds) -> int {
    if (const int rc = allow_lds(kernel, lds, fn)) return rc;
    launch(kernel, dim3(unsigned(plan.groups)), dim3(64 * kAttendWaves), lds, st, a);
    LMOE_LAUNCHED(fn);
    if (plan.split) {
      const unsigned lines = unsigned(T) * unsigned(q_heads), x = lines < kMostGroups ? lines : 1u << 23;  // two axes past one's end
      launch(join, dim3(x, (lines + x - 1) / x), dim3(256), 0, st, a);
      LMOE_LAUNCHED(fn);
    }
    return 0;
  };
  const bool bf = dtype == LMOE_BF16;
  if (D == 64)
    return bf ? go(k_attend<64, true>, k_attend_join<64, true>, kAttendLds<64>)
              : go(k_attend<64, false>, k_attend_join<64, false>, kAttendLds<64>);
  if (D == 128)
    return bf ? go(k_attend<128, true>, k_attend_join<128, true>, kAttendLds<128>)
              : go(k_attend<128, false>, k_attend_join<128, false>, kAttendLds<128>);
  return bf ? go(k_attend<256, true>, k_attend_join<256, true>, kAttendLds<256>)
            : go(k_attend<256, false>, k_attend_join<256, false>, kAttendLds<256>);
}
