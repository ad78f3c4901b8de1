// Attention of chunks of new rows over the 8-bit paged cache, causal: a later chunk of a prompt, a message after a long history,
// a tree of drafts.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - m),  over the places j < len - (n - 1 - r) of row r of n
//
// One pass over the keys with a running maximum m. A workgroup takes 128 or 256 (row, query head of the group) pairs of one key
// head, a wavefront 32 of them, so that the heads of a group share what it reads; keys come 64 at a time. Codes go from the pages
// to registers, a tile ahead, and as 16-bit values (exact) to LDS, from where the matrix cores' operands are read as in prompt.hip:
//   scores^T = K Q^T   A = 32 keys x 16 channels, B = Q^T from registers: a lane ends with 16 of 32 keys' scores of one row
//   out^T += V^T P^T   B = those weights as they lie, A = the same keys' values by LDS loads that transpose
// Pages hold 32 tokens at least, so a half of a tile has one page, one scale of keys and one of values: the former multiplies
// float32 scores, the latter goes into the conversion (its exponent: scales are powers of two). bfloat16 takes any scale; float16
// takes it relative to a reference that moves, and the sums with it, when a page's scale leaves 2^-15 .. 2^7 of it, so that the
// conversion stays exact for a tile's two pages up to 2^22 apart.
//
// 32 keys are worked at a time: the next 32 keys' score products, these ones' exponentials, their output products and a part of the
// next tile's conversion are issued in one stream of slots, a product and about seven other instructions each. Tiles of keys lie
// half a tile off those of values for that.
//
// Bound by the matrix cores (4 width products a visible pair), at the rate that their power allows: products alone reach 2.2-2.4
// PFLOP/s on constant data and 1.84 on random data (the clock falls to 1.86 GHz); with six vector instructions beside each, which
// is what the exponentials and the conversion need, 1.56; the library's largest product 1.21. Measured (2,048 rows over 34,816
// tokens, 32 heads over 4 of 128, bf16): 1,018-1,119 us by card, 1.01-1.11 PFLOP/s, with float16, whose products take more power,
// 11 % more; without LDS reads and staging 943. One after the other instead of slots 1,252; 128 pairs a workgroup 1,158; 64 pairs a
// wavefront, which halves the LDS reads and leaves one wavefront a SIMD (it issues a vector instruction every eight or nine
// cycles, each of two every four or five), 1,156; codes two tiles ahead, or loads of single lanes' addresses, 1-3 % more. Width
// 256: one wavefront a SIMD, 0.90-0.92 PFLOP/s where all places work (float16 0.83-0.85). Width 64: 0.68-0.71 (float16 0.61-0.63),
// bound by the vector unit: a pair's exponential and the rest of its weight are the same for half of the products. A short call's
// workgroup: 3.3 us to its first scores, 1.45 a tile, 2.5 of output.
//
// Weights, their sums and values that are not finite: as in prompt.hip.
#include <cmath>
#include "flash.h"

namespace lmoe {

struct ChunkArgs {
  const uint16_t *q;
  long long q_row, q_head;  // elements
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int *table, *lens, *cu;
  uint16_t *out;  // [T][q_heads][D]
  float *part;    // [workgroups][2][pairs] of [D] sums and {maximum, weight}: of a tile that a workgroup goes on with (0), or begins
                  // and does not end (1)
  int2 *joins;    // [T][q_heads]: the first piece's line in part (-1: the row is done), the last one's
  float scale;    // times log2 e
  int T, B, q_heads, heads, group, pages, width, page_shift, tiles, stretches, per, sorted;  // per: stretches a tile
  double per_group, per_stretch;  // 1 / group, 1 / stretches
};

// The nth tile of ROWS pairs that is worked, by one wavefront. Up to 64 sequences: those that see the most keys first (to 256
// keys), so that what is left for the end is short (sorted; where all find a place at once, in the order of sequences). More: the
// sequences from the last on, each from its end, eight tiles in turn shifted against the next eight (prompt.hip says why);
// sequence b's tiles begin at cu[b] group / ROWS + b, which leaves it room for all of them. b < 0: there is none. The first and
// the last sequence have a tile even without rows.
struct ChunkTile {
  int b, tile, row0, n, len;
};
template <int ROWS>
__device__ __forceinline__ ChunkTile nth_chunk_tile(const ChunkArgs &a, int nth) {
  ChunkTile w = {-1, 0, 0, 0, 0};
  if (a.B > 64) {
    const int task = a.tiles - 1 - turned_task(nth, a.tiles);
    auto begin = [&](int c, int i) { return first_task(c, i, a.group, ROWS); };
    if (a.cu)
      w.b = last_at(a.cu, a.B, task, begin);
    else  // a row a sequence
      w.b = int(min((long long)a.B - 1, (long long)task * ROWS / (a.group + ROWS) + 1));
    if (!a.cu)
      while (w.b >= 0 && begin(w.b, w.b) > task) --w.b;
    if (w.b < 0) return w;
    seq_rows(a.cu, w.b, a.T, &w.row0, &w.n);
    w.len = max(a.lens[w.b], 0);
    w.tile = int(task - begin(a.cu ? a.cu[w.b] : w.b, w.b));
    return w;
  }
  const int lane = threadIdx.x & 63;
  int row0 = 0, n = 0, len = 0, tiles = 0;
  if (lane < a.B) {
    seq_rows(a.cu, lane, a.T, &row0, &n);
    len = max(a.lens[lane], 0);
    tiles = max(tiles_of(n, a.group, ROWS), lane == 0 || lane == a.B - 1 ? 1 : 0);
  }
  const int past = max(len - n, 0);
  auto count = [&](int x) { return tiles_that_see(x, past, tiles, a.group, ROWS); };  // of the lane's sequence
  auto from = [&](int x) { return int(wave_sum(float(count(x)))); };  // (counts below 2^24: exact in float32)
  int lo = 0, hi = !a.sorted ? 1 : (int(wave_max(tiles > 0 ? float(past) + float(tiles) * ROWS / a.group : 0.0f)) >> 8) + 2, behind = 0;
  if (nth >= from(0)) return w;
  while (hi - lo > 1) {  // the largest x with more than nth tiles from it on
    const int mid = lo + ((hi - lo) >> 1), c = from(mid);
    if (c > nth)
      lo = mid;
    else
      hi = mid, behind = c;
  }
  // of the tiles that see 256 lo keys and not 256 more, the lane's sequence has `mine`; in the order of sequences
  const int above = a.sorted ? count(lo + 1) : 0, mine = count(lo) - above;
  int ends = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int u = __shfl_up(ends, d);
    if (lane >= d) ends += u;
  }
  const int left = nth - behind;
  const unsigned long long past_it = __ballot(ends > left);
  if (!past_it) return w;
  const int b = __ffsll(past_it) - 1;
  const int at = left - (__builtin_amdgcn_readlane(ends, b) - __builtin_amdgcn_readlane(mine, b));
  w = {b, __builtin_amdgcn_readlane(tiles - above, b) - 1 - at, __builtin_amdgcn_readlane(row0, b), __builtin_amdgcn_readlane(n, b),
       __builtin_amdgcn_readlane(len, b)};
  return w;
}

// Where one workgroup of a key head takes all of a tile's keys, the longest tile decides, and few tiles leave places free. So a
// call may be laid out as one line instead, all tiles one behind another, cut into as many equal stretches as a head has places:
// a workgroup works what its stretch holds, the end of one tile, whole ones and the beginning of another, say. Tile t of a
// sequence takes START, what its beginning and end cost in keys, and a key for each that its last row sees: past + (t + 1) ROWS /
// group. START is 192 where two workgroups share a CU, which hides a part of it, and 320 where one has it alone (12 sequences of
// 48 to 700 rows over up to 9,700 tokens, 28 heads over 4 of 128: 253 -> 232 us; the former with 320 is 1 % slower).
static_assert(kLineKeys == kPromptKeys, "a stretch begins with a tile of keys");
struct LinePlace {
  int b, tile, key;  // key: a multiple of a tile of keys, below what the tile's last row sees
};
template <int ROWS, int START>
struct TileLine {
  const ChunkArgs &a;
  int row0, n, len, tiles;  // of the lane's sequence
  __device__ __forceinline__ void look(int b) {
    row0 = n = len = 0;
    if (b < a.B) {
      seq_rows(a.cu, b, a.T, &row0, &n);
      len = max(a.lens[b], 0);
    }
    tiles = tiles_of(n, a.group, ROWS);
  }
  __device__ __forceinline__ double cost(int past, int t) const { return line_cost(past, t, a.group, ROWS, START); }
  // of the lane's sequence and those before it in the wavefront (lanes past the last sequence: of some of them)
  __device__ __forceinline__ double ends() const {
    double x = cost(len - n, tiles);
    const int lane = threadIdx.x & 63;
    for (int d = 1; d < min(a.B, 64); d <<= 1) {
      const double u = __shfl_up(x, d);
      if (lane >= d) x += u;
    }
    return x;
  }
  __device__ __forceinline__ static double lane_of(double x, int i) {
    const u32x2 w = __builtin_bit_cast(u32x2, x);
    const int low = __builtin_amdgcn_readlane(int(w.x), i), high = __builtin_amdgcn_readlane(int(w.y), i);
    return __builtin_bit_cast(double, u32x2{uint32_t(low), uint32_t(high)});
  }
  // Both ends of one of `of` stretches of the line, and the sequence that it begins in (its fields in *first). Stretches shorter
  // than kLeastStretch, two of which may begin at the same key of a tile, are not made: there are fewer then.
  __device__ __forceinline__ void stretch(int one, int of, LinePlace *from, LinePlace *to, ChunkTile *first) {
    const int lane = threadIdx.x & 63;
    double all = 0.0, last = 0.0;
    for (int b = 0; b < a.B; b += 64) {
      look(b + lane);
      last = ends();
      all += lane_of(last, min(a.B - b, 64) - 1);
    }
    *from = *to = {a.B, 0, 0};
    double each = all * a.per_stretch;
    if (each * a.per_group < kLeastStretch) {
      of = max(int(all * a.per_group * (1.0 / kLeastStretch)), 1);
      each = all / of;
    }
    if (one >= of) return;
    const double x0 = floor(each * one), x1 = one + 1 < of ? floor(each * (one + 1)) : all;  // (the same number to both sides)
    double before = 0.0;
    for (int b = 0; b < a.B; b += 64) {
      if (a.B > 64) {
        look(b + lane);
        last = ends();
      }
      const double behind = before + lane_of(last, min(a.B - b, 64) - 1);
      if (x0 >= before && x0 < behind) {
        *from = place(x0 - before, b, last);
        auto its = [&](int x) { return __builtin_amdgcn_readlane(x, from->b - b); };
        *first = {from->b, 0, its(row0), its(n), its(len)};
      }
      if (x1 >= before && x1 < behind) {
        *to = place(x1 - before, b, last);
        break;
      }
      before = behind;
    }
  }
  __device__ __forceinline__ LinePlace place(double x, int b, double last) const {
    const int lane = threadIdx.x & 63;
    const int i = __ffsll((long long)__ballot(last > x)) - 1;
    x -= i ? lane_of(last, i - 1) : 0.0;
    const int its_n = __builtin_amdgcn_readlane(n, i), off = __builtin_amdgcn_readlane(len, i) - its_n;
    int lo = 0, hi = __builtin_amdgcn_readlane(tiles, i);  // the tile is in [lo, hi)
    while (hi - lo > 1) {
      const int step = (hi - lo + 63) >> 6, t = lo + lane * step;
      lo += step * (__popcll(__ballot(t < hi && cost(off, t) <= x)) - 1);
      hi = min(hi, lo + step);
    }
    int key = line_key((x - cost(off, lo)) * a.per_group - START);
    if (key && seen(off, lo, its_n * a.group) - key < kPromptKeys) ++lo, key = 0;
    return {b + i, lo, key};
  }
  // One sequence's tiles in `per` equal pieces each: what `stretch` gives, for less where all tiles see about as much
  __device__ __forceinline__ void piece(int one, int per, LinePlace *from, LinePlace *to, ChunkTile *first) {
    look(0);
    const int tile = one / per, i = one - tile * per;
    *from = *to = {a.B, 0, 0};
    if ((long long)tile * ROWS >= (long long)n * a.group) return;
    const uint32_t most = max(seen(len - n, tile, n * a.group), 1), step = piece_keys(most, per);
    const uint32_t begin = i * step;
    if (i > 0 && begin >= most) return;
    *first = {0, 0, row0, n, len};
    *from = {0, tile, int(begin)};
    *to = begin + step < most ? LinePlace{0, tile, int(begin + step)} : LinePlace{0, tile + 1, 0};
  }
  // how many keys a tile's last row sees
  __device__ __forceinline__ int seen(int off, int tile, int pairs) const {
    return tile_sees(off, tile, pairs, a.group, ROWS, a.width << a.page_shift);
  }
  // the first sequence from b on that has rows, by one wavefront
  __device__ __forceinline__ int with_rows(int b) {
    for (; b < a.B; b += 64) {
      look(b + (threadIdx.x & 63));
      const unsigned long long some = __ballot(n > 0);
      if (some) return b + __ffsll((long long)some) - 1;
    }
    return a.B;
  }
};

// Eight codes times a power of two as 16-bit floats
template <bool BF>
__device__ __forceinline__ u32x4 widen8(uint32_t a, uint32_t b, float scale) {
  if constexpr (BF)
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, true))};
  else
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, scale, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, scale, true))};
}

// The codes of half a tile (32 tokens of a page's head): rows past `rows` read as zeros
__device__ __forceinline__ u32x4 load_rows(const uint8_t *from, int bytes, int at) {
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(from), 0, bytes, 0x00020000);
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, 0));
}

constexpr int kAhead = 3;  // fragments that are read ahead of their products

// Whether every output product's weights are packed a slot before it: NM score products, NV output products, of which each 16 keys
// take `per`, over NP pairs of weights (four for 16 keys), spread over NS slots and packed one slot later
constexpr bool weights_in_time(int NM, int NV, int NP, int per, int NS) {
  for (int k = 0; k < NV; ++k) {
    const int slots = NM + k - 1 < NS ? NM + k - 1 : NS;
    if (slots * NP / NS < 4 * (k / per + 1)) return false;
  }
  return true;
}

// NW wavefronts of 32 pairs. SPLIT: in stretches of the line of tiles
template <int D, bool BF, int NW, bool SPLIT>
__global__ void __launch_bounds__(64 * NW, D == 256 ? 1 : 2) k_chunk_rows(ChunkArgs a) {
  constexpr int ROWS = 32 * NW, THREADS = 64 * NW, BN = kPromptKeys, KS = D / 16, DT = D / 32;
  constexpr int COPIES = D / (16 * NW), COPY_ROWS = 1024 * NW / D;  // 16 codes a thread
  constexpr int kTileBytes = BN * D * 2;
  extern __shared__ uint8_t lds[];  // [2 stages] of keys, [2 stages] of values
  __shared__ uint32_t marks[2 * BN * DT];  // of take_bad: [pos, neg][key][32 channels]
  __shared__ uint32_t flags[NW];           // of any_bad: a wavefront's
  const int kv = blockIdx.x % a.heads, group = a.group;
  auto zeros = [&](int lo, int hi) {  // rows before the first sequence or behind the last one come back zero
    lo = min(max(lo, 0), a.T), hi = min(max(hi, 0), a.T);
    const int per = group * (D / 8);
    for (long long i = threadIdx.x; i < (long long)(lo + (a.T - hi)) * per; i += THREADS) {
      const int row = int(i / per), c = int(i - (long long)row * per);
      const size_t line = size_t(row < lo ? row : hi + row - lo) * a.q_heads + kv * group + c / (D / 8);
      *reinterpret_cast<u32x4 *>(a.out + line * D + (c % (D / 8)) * 8) = u32x4{};
      if (SPLIT && c % (D / 8) == 0) a.joins[line].x = -1;
    }
  };
  auto uniform = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  ChunkTile work;
  [[maybe_unused]] TileLine<ROWS, line_start(D, NW)> line_of_tiles{a};
  [[maybe_unused]] LinePlace at_line, to_line;
  if constexpr (SPLIT) {
    const int one = int(blockIdx.x) / a.heads;
    if (a.per)
      line_of_tiles.piece(one, a.per, &at_line, &to_line, &work);
    else
      line_of_tiles.stretch(one, a.stretches, &at_line, &to_line, &work);
    at_line = {uniform(at_line.b), uniform(at_line.tile), uniform(at_line.key)};
    to_line = {uniform(to_line.b), uniform(to_line.tile), uniform(to_line.key)};
    if (one == 0 && a.cu) zeros(a.cu[0], a.cu[a.B]);
  } else {
    work = nth_chunk_tile<ROWS>(a, int(blockIdx.x) / a.heads);
    work = {uniform(work.b), uniform(work.tile), uniform(work.row0), uniform(work.n), uniform(work.len)};
    if (work.b < 0) return;
    if (work.tile == 0 && a.cu && (work.b == 0 || work.b == a.B - 1))
      zeros(work.b == 0 ? a.cu[0] : 0, work.b == a.B - 1 ? a.cu[a.B] : a.T);
  }
  do {
    // opaque: what is made of it belongs to this tile, and is not kept in registers from one to the next
    const int tid = SPLIT ? opaque(int(threadIdx.x)) : int(threadIdx.x), lane = tid & 63, wave = uniform(tid >> 6);
    const int r = lane & 31, h = lane >> 5;
    [[maybe_unused]] int begin = 0, end = 0x7fffffff;  // the workgroup's keys of the tile
    if constexpr (SPLIT) {
      if (at_line.b >= a.B) return;
      if ((long long)at_line.tile * ROWS >= (long long)work.n * group) {
        const int b = line_of_tiles.with_rows(at_line.b + 1);
        if (b >= a.B) return;
        at_line = {b, 0, 0};
        seq_rows(a.cu, b, a.T, &work.row0, &work.n);
        work.b = b, work.len = max(a.lens[b], 0);
      }
      const bool same = at_line.b == to_line.b, last = same && at_line.tile == to_line.tile;
      if (at_line.b > to_line.b || (same && at_line.tile > to_line.tile) || (last && at_line.key >= to_line.key)) return;
      begin = at_line.key;
      if (last) end = to_line.key;
      work = {uniform(work.b), at_line.tile, uniform(work.row0), uniform(work.n), uniform(work.len)};
      at_line = {work.b, work.tile + 1, 0};
    }
    const int b = work.b, n = work.n;
    const int pairs = n * group, first = work.tile * ROWS;
    if (uint32_t(first) >= uint32_t(pairs)) return;  // (a tile before the sequence's first: where offsets fall)
    const int off = work.len - n;  // row i sees places 0 .. i + off
    const int room = a.width << a.page_shift;
    const int most_keys = min(off + (min(first + ROWS, pairs) - 1) / group + 1, room);  // what the workgroup's last row sees
    const int keys = SPLIT ? min(most_keys, end) : most_keys;
    const int own = first + 32 * wave;  // the wavefront's first pair
    const int all = min(off + min(own, pairs - 1) / group + 1, room);  // what every row of the wavefront sees
    const int all_rows = min(off + first / group + 1, room);           // and of the workgroup
    const int flat = min(own + r, pairs - 1), mine = flat / group, sees = min(mine + off + 1, room);
    u32x4 qf[KS];
    {
      const uint16_t *q = a.q + size_t(work.row0 + mine) * a.q_row + size_t(kv * group + flat - mine * group) * a.q_head + 8 * h;
  #pragma unroll
      for (int j = 0; j < KS; ++j) qf[j] = *reinterpret_cast<const u32x4 *>(q + 16 * j);
    }
    // pages and scales of the halves of 64 tiles from `base` on, a tile a lane
    // (here and below: a table of 32-token pages may have room for 2^31 - 32 tokens, and no end of a tile is held in an int)
    const int tiles = keys > begin ? (keys - begin - 1) / BN + 1 : 0;
    int base = 0, number[2];
    float k_scale[2], v_scale[2];
    auto look_up = [&](int t0) {
      base = t0;
  #pragma unroll
      for (int x = 0; x < 2; ++x) {
        number[x] = -1, k_scale[x] = 1.0f, v_scale[x] = 0.0f;
        const int p = (begin + (t0 + lane) * BN + 32 * x) >> a.page_shift;
        if (t0 + lane < tiles && p < a.width) {
          const int page = a.table[size_t(b) * a.width + p];
          if (uint32_t(page) < uint32_t(a.pages)) {
            number[x] = page;
            k_scale[x] = a.ks[size_t(page) * a.heads + kv];
            v_scale[x] = a.vs[size_t(page) * a.heads + kv];
          }
        }
      }
    };
    // Tiles of keys are shifted by half a tile against those of values: tile T of keys are the halves 2 T - 1 and 2 T, so that
    // the scores of the next 32 keys are always to be had beside the values of the present 32
    const int page_tokens = 1 << a.page_shift;
    const uint32_t page_bytes = uint32_t(a.heads) * uint32_t(page_tokens * D);
    const uint8_t *const kc = a.kc + uint32_t(kv) * uint32_t(page_tokens * D);
    const uint8_t *const vc = a.vc + uint32_t(kv) * uint32_t(page_tokens * D);
    u32x4 kr[COPIES], vr[COPIES];
    const int crow = tid / (D / 16), cchunk = tid % (D / 16);  // the thread's row and 16 codes of copy 0; copy i is i COPY_ROWS on
    // (the wavefront's rows of a copy are in one half)
    auto half_of = [&](int i) { return COPY_ROWS == 64 ? wave / (NW / 2) : i * COPY_ROWS >> 5; };
    auto rows_at = [&](const uint8_t *codes, int t, int x, int voff) {  // 16 codes of half x of tile t
      const int found = __builtin_amdgcn_readlane(x ? number[1] : number[0], (t - base) & 63), page = t < 0 ? -1 : found;
      const int token = begin + t * BN + 32 * x, rows = __builtin_amdgcn_readfirstlane(min(32, max(0, most_keys - token)));
      const uint64_t at = uint64_t(uint32_t(max(page, 0))) * page_bytes + uint32_t((token & (page_tokens - 1)) * D);
      return load_rows(codes + at, page < 0 ? 0 : rows * D, voff);
    };
    const int voff = (crow & 31) * D + cchunk * 16;
    auto fetch_k = [&](int T, int i) {
      kr[i] = rows_at(kc, half_of(i) ? T : T - 1, half_of(i) ^ 1, voff + (i * COPY_ROWS & 31) * D);
    };
    auto fetch_v = [&](int t, int i) { vr[i] = rows_at(vc, t, half_of(i), voff + (i * COPY_ROWS & 31) * D); };
    float ref = BF ? 1.0f : 0.0f, vs[2], move = 1.0f;  // float16: values in LDS are in units of ref
    // the factors that tile t's codes of values take, and the one that brings the sums to its reference
    auto scales_of = [&](int t) {
      vs[0] = lane_value(v_scale[0], (t - base) & 63), vs[1] = lane_value(v_scale[1], (t - base) & 63);
      if constexpr (!BF) {
        const float big = fmaxf(vs[0], vs[1]), small = vs[0] == 0.0f ? vs[1] : vs[1] == 0.0f ? vs[0] : fminf(vs[0], vs[1]);
        move = 1.0f;
        if (big > 0.0f && (big > ref * 0x1p7f || small < ref * 0x1p-15f)) {
          // the larger page's own scale where the smaller one's values stay exact beside it, down to 2^-7 of it (448 2^7 is finite)
          // where they lie further apart; (2^-40 448 is nothing in float16)
          const float to = fmaxf(fmaxf(fminf(big, small * 0x1p15f), big * 0x1p-7f), 0x1p-40f);
          move = ref == 0.0f ? 1.0f : fminf(ref / to, 0x1p120f);
          ref = to;
        }
        if (ref != 0.0f) vs[0] /= ref, vs[1] /= ref;
      }
    };
    uint8_t *const k_lds = lds, *const v_lds = lds + 2 * kTileBytes;
    auto store_k = [&](int stage, int i, int part) {
      const int row = i * COPY_ROWS + crow;
      *reinterpret_cast<u32x4 *>(k_lds + stage * kTileBytes + row * D * 2 + k_chunk<D>(crow, 2 * cchunk + part) * 16) =
          widen8<BF>(kr[i][2 * part], kr[i][2 * part + 1], 1.0f);
    };
    auto store_v = [&](int stage, int i, int part) {
      const int row = i * COPY_ROWS + crow;
      *reinterpret_cast<u32x4 *>(v_lds + stage * kTileBytes + row * D * 2 + v_pair<D>(crow, cchunk) * 32 + part * 16) =
          widen8<BF>(vr[i][2 * part], vr[i][2 * part + 1], half_of(i) ? vs[1] : vs[0]);
    };
    // a transposing load: 16 lanes take 4 keys x 16 channels, lane i of them gets channel i of the 4
    const int vrow = 4 * h + ((lane & 15) >> 2), vpair = (lane >> 4) & 1, vbyte = (lane & 3) * 8;
    auto k_frag = [&](const uint8_t *kt, int x, int j) {
      // (256 bytes apart the swizzle is the same: eight addresses for all of them)
      return *reinterpret_cast<const u32x4 *>(kt + (32 * x + r) * D * 2 + k_chunk<D>(r, 2 * (j & 7) + h) * 16 + (j >> 3) * 256);
    };
    auto v_frag = [&](const uint8_t *vt, int ks, int d) {
      u32x4 f;
  #pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int row = 16 * ks + 8 * x + vrow;
        const uint8_t *src = vt + row * D * 2 + v_pair<D>(vrow, 2 * (d & 3) + vpair) * 32 + (d >> 2) * 256 + vbyte;
        const u32x2 g = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(src)));
        f[2 * x] = g.x, f[2 * x + 1] = g.y;
      }
      return f;
    };
    auto largest = [](const f32x16 &x) {
      float y[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  #pragma unroll
      for (int e = 0; e < 16; ++e) y[e & 3] = fmaxf(y[e & 3], x[e]);
      return fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
    };
    f32x16 o[DT] = {}, s = {}, other;
    float m = -INFINITY, l = 0.0f, top = -INFINITY;
    if (tiles > 0) {
      look_up(0);
      u32x4 next[COPIES];
  #pragma unroll
      for (int i = 0; i < COPIES; ++i) fetch_k(1, i), next[i] = kr[i];
  #pragma unroll
      for (int i = 0; i < COPIES; ++i) fetch_k(0, i), fetch_v(0, i);
      scales_of(0);
      move = 1.0f;
      static_for<0, 2 * COPIES>([&](auto q) { store_k(0, q / 2, q % 2), store_v(0, q / 2, q % 2); });
  #pragma unroll
      for (int i = 0; i < COPIES; ++i) kr[i] = next[i];
      static_for<0, 2 * COPIES>([&](auto q) { store_k(1, q / 2, q % 2); });
  #pragma unroll
      for (int i = 0; i < COPIES; ++i) fetch_k(2, i), fetch_v(1, i);
      barrier_lds();
  #pragma unroll
      for (int j = 0; j < KS; ++j) s = mfma32<BF>(k_frag(k_lds, 1, j), qf[j], s);
      top = largest(s);
    }
    // 32 keys, half x of tile t: their scores s become next, the following half's. Called with the two in turn, so that nothing is
    // moved. Beside the products, tile t + 2 of keys (x = 0) or t + 1 of values (x = 1) goes from registers to LDS, and the codes of
    // the one after it are asked for.
    auto half = [&](int t, auto xc, auto stage_c, f32x16 &s, f32x16 &next) {
      constexpr int x = decltype(xc)::value, stage = decltype(stage_c)::value;
      const uint8_t *kt = k_lds + (stage ^ 1) * kTileBytes, *vt = v_lds + stage * kTileBytes + 32 * x * D * 2;
      const int at = begin + t * BN + 32 * x;
      // (never zero: -infinity times that would be NaN)
      const float c = fmaxf(lane_value(k_scale[x], t - base) * a.scale, 0x1p-126f);
      const bool hole = __builtin_amdgcn_readlane(number[x], t - base) < 0;
      if (all - 32 < at || hole) {
        const int left = opaque(hole ? 0 : sees - at - 4 * h);  // opaque: a branch, not selects in every half
  #pragma unroll
        for (int e = 0; e < 16; ++e)
          if (8 * (e >> 2) + (e & 3) >= left) s[e] = -INFINITY;
        top = largest(s);
      }
      constexpr int NM = KS, NV = 2 * DT, NP = 8;
      // 192 registers of queries and sums: the queries stay in accumulation registers, which the products read as they are
      if constexpr (D == 256)
  #pragma unroll
        for (int j = 0; j < KS; ++j) asm volatile("" : "+a"(qf[j]));
      u32x4 ring[kAhead + 1];
      auto frag = [&](auto ic) {
        constexpr int i = decltype(ic)::value;
        if constexpr (i < KS)
          ring[i % (kAhead + 1)] = k_frag(kt, x, i);
        else if constexpr (i < KS + 2 * DT)
          ring[i % (kAhead + 1)] = v_frag(vt, (i - KS) / DT, (i - KS) % DT);
      };
      static_for<0, kAhead>([&](auto ic) { frag(ic); });
      __builtin_amdgcn_sched_barrier(0);
      top = fmaxf(top, lane_xor32(top)) * c;
      const float moved = x == 0 ? move : 1.0f;
      if (__any(top > m + kLag<BF>) || (!BF && moved != 1.0f)) {
        const float to = fmaxf(m, top), keep = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
        m = to;
        l *= keep;
  #pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= keep * moved;
      }
      const float lift = m == -INFINITY ? 0.0f : kLift<BF> - m;
      float peak[2] = {-INFINITY, -INFINITY}, ex[NP][2];
      if constexpr (x == 1) scales_of(t + 1);
      constexpr int NS = NM + NV / 2 - 2, NR = NM + NV - NS, PIECES = 2 * COPIES;  // slots with exponentials, and with the maximum
      static_assert(weights_in_time(NM, NV, NP, DT, NS), "an output product before its weights");
      u32x4 p[2];
      auto each = [&](auto slot, auto f) {  // the pairs of a slot
        constexpr int i = decltype(slot)::value;
        if constexpr (i >= 0 && i < NS) static_for<i * NP / NS, (i + 1) * NP / NS>(f);
      };
      static_for<0, NM + NV>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        frag(IC<i + kAhead>{});
        if constexpr (i < NM)
          next = mfma32<BF>(ring[i % (kAhead + 1)], qf[i], i == 0 ? f32x16{} : next);
        else
          o[(i - NM) % DT] = mfma32<BF>(ring[i % (kAhead + 1)], p[(i - NM) / DT], o[(i - NM) % DT]);
        each(IC<i>{}, [&](auto ec) {
          constexpr int e = decltype(ec)::value;
          ex[e][0] = __builtin_amdgcn_exp2f(fmaf(s[2 * e], c, lift));
          ex[e][1] = __builtin_amdgcn_exp2f(fmaf(s[2 * e + 1], c, lift));
        });
        each(IC<i - 1>{}, [&](auto ec) {
          constexpr int e = decltype(ec)::value;
          p[e / 4][e % 4] = pack2<BF>(ex[e][0], ex[e][1]);
        });
        each(IC<i - 2>{}, [&](auto ec) {
          constexpr int e = decltype(ec)::value;
          l = opaque(add2<BF>(p[e / 4][e % 4], l));  // opaque: here, not after the branch
        });
        // a piece of a tile: eight codes; then, a copy being out of its registers, the next one's load
        static_for<(i * PIECES + NM + NV - 1) / (NM + NV), ((i + 1) * PIECES + NM + NV - 1) / (NM + NV)>([&](auto qc) {
          constexpr int q = decltype(qc)::value;
          if constexpr (x == 0)
            store_k(stage, q / 2, q % 2);
          else
            store_v(stage ^ 1, q / 2, q % 2);
          if constexpr (q % 2) {
            if constexpr (x == 0)
              fetch_k(t + 3, q / 2);
            else
              fetch_v(t + 2, q / 2);
          }
        });
        if constexpr (i >= NS)
          static_for<(i - NS) * NP / NR, (i - NS + 1) * NP / NR>([&](auto ec) {
            constexpr int e = decltype(ec)::value;
            peak[e & 1] = opaque(fmaxf(fmaxf(next[2 * e], next[2 * e + 1]), peak[e & 1]));
          });
        __builtin_amdgcn_sched_barrier(0);
      });
      top = fmaxf(peak[0], peak[1]);
    };
    auto step = [&](int t, auto stage_c) {
      constexpr int stage = decltype(stage_c)::value;
      if (t + 4 > base + 64) look_up(t);
      barrier_lds();  // this tile's values and the next one's keys are there, and what they replace has been read
      const int at = begin + t * BN;
      uint8_t *vt = v_lds + stage * kTileBytes;
      bool bad = false;
      if (all_rows - BN < at) {  // the workgroup's first row does not see all of it
        const bool found = __any(any_bad<D, BF, THREADS>(vt));
        if (lane == 0) flags[wave] = found;
        barrier_lds();
        uint32_t any = 0;
  #pragma unroll
        for (int w = 0; w < NW; ++w) any |= flags[w];
        bad = __builtin_amdgcn_readfirstlane(any);
        if (bad) {
          for (int i = tid; i < BN * DT; i += THREADS) take_bad<D, BF>(vt, i / DT, i % DT, &marks[i], &marks[BN * DT + i]);
          barrier_lds();
        }
      }
      half(t, IC<0>{}, stage_c, s, other);
      half(t, IC<1>{}, stage_c, other, s);
      if (bad) {
        for (int j = 0; j < BN; ++j)
  #pragma unroll
          for (int d = 0; d < DT; ++d) {
            const uint32_t up = at + j < sees ? marks[j * DT + d] >> (4 * h) : 0, down = at + j < sees ? marks[BN * DT + j * DT + d] >> (4 * h) : 0;
            if (!__any((up | down) != 0)) continue;
  #pragma unroll
            for (int e = 0; e < 16; ++e) {
              if (up >> (8 * (e >> 2) + (e & 3)) & 1) o[d][e] += INFINITY;
              if (down >> (8 * (e >> 2) + (e & 3)) & 1) o[d][e] -= INFINITY;
            }
          }
      }
    };
    for (int t = 0; t < tiles; t += 2) {
      step(t, IC<0>{});
      if (t + 1 >= tiles) break;
      step(t + 1, IC<1>{});
    }
    barrier_lds();
    auto line_of = [&](int f) {  // of a pair [T][q_heads]
      const int row = f / group;
      return size_t(work.row0 + row) * a.q_heads + kv * group + (f - row * group);
    };
    const bool there = own + r < pairs;
    const float weight = l + lane_xor32(l);
    if constexpr (SPLIT) {
      const bool ended = keys == most_keys;
      if (there && h == 0) {
        const int place = 2 * int(blockIdx.x) * ROWS + 32 * wave + r;
        int2 *join = a.joins + line_of(own + r);
        if (begin == 0) join->x = ended ? -1 : place + ROWS;
        if (begin > 0 && ended) join->y = place;
      }
      if (begin > 0 || !ended) {
        float *rows = reinterpret_cast<float *>(lds) + wave * 32 * D;
  #pragma unroll
        for (int d = 0; d < DT; ++d)
  #pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<f32x4 *>(rows + r * D + ((8 * d + 2 * e + h) ^ (r & 15)) * 4) =
                f32x4{o[d][4 * e] * ref, o[d][4 * e + 1] * ref, o[d][4 * e + 2] * ref, o[d][4 * e + 3] * ref};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        float *part = a.part + (size_t(2 * blockIdx.x + (begin == 0)) * ROWS + 32 * wave) * (D + 4);
  #pragma unroll 4
        for (int i = 0; i < 32 * D / 256; ++i) {
          const int j = i * 64 + lane, row = j / (D / 4), c = j % (D / 4);
          const f32x4 w = *reinterpret_cast<const f32x4 *>(rows + row * D + (c ^ (row & 15)) * 4);
          if (own + row < pairs) *reinterpret_cast<f32x4 *>(part + size_t(row) * (D + 4) + c * 4) = w;
        }
        if (there && h == 0) *reinterpret_cast<float2 *>(part + size_t(r) * (D + 4) + D) = float2{m, weight};
        barrier_lds();
        continue;
      }
    }
    const float inv = weight == 0.0f ? 0.0f : ref / weight;
    uint8_t *rows = lds + wave * 32 * D * 2;
  #pragma unroll
    for (int d = 0; d < DT; ++d)
  #pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<u32x2 *>(rows + r * D * 2 + k_chunk<D>(r, 4 * d + e) * 16 + 8 * h) =
            u32x2{pack2<BF>(o[d][4 * e] * inv, o[d][4 * e + 1] * inv), pack2<BF>(o[d][4 * e + 2] * inv, o[d][4 * e + 3] * inv)};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  #pragma unroll 4
    for (int i = 0; i < 32 * D / 512; ++i) {
      const int j = i * 64 + lane, row = j / (D / 8), c = j % (D / 8);
      const u32x4 w = *reinterpret_cast<const u32x4 *>(rows + row * D * 2 + k_chunk<D>(row, c) * 16);
      if (own + row < pairs) *reinterpret_cast<u32x4 *>(a.out + line_of(own + row) * D + c * 8) = w;
    }
    if constexpr (SPLIT) barrier_lds();  // the next tile's codes go to the same places
  } while (SPLIT);
}

// How a call is laid out: wavefronts a workgroup, and whether in stretches, where tiles alone would not fill the GPU's places, or
// not evenly. Priced in us, as measured: what a workgroup takes for a key (all places at work, or few) and for a tile's beginning
// and end; tiles one after the other, those that see the most first (of several sequences, which rarely are as long as the
// longest: half of that on the mean); and pieces' sums written and read at 4 TB/s, by a second kernel. Eight wavefronts a
// workgroup convert each key once for 256 pairs instead of 128 (2,048 rows over 34,816 tokens, 32 heads over 4 of 128: 1,158 ->
// 1,067 us), but leave coarser work. Against one cut of all tiles at the same keys, sized for the longest sequence: 1,110 rows
// over 2,291 tokens before them, 16 heads over 2 of 256, 118 -> 91 us; 100 single rows over up to 8,000, 32 over 4 of 128, 113 ->
// 92; 64 sequences of up to 16 rows over up to 4,000 56 -> 48. Beginning and end of a stretch cost 1-2 us more to find: 106 rows of
// four sequences over up to 948 16.4 -> 17.7. Against whole tiles: those 106 rows 27 -> 18, 1,857 rows of three sequences over up to
// 9,024, 16 over 2 of 256, 332 -> 210, 12 sequences of 48 to 700 rows over up to 9,700, 28 over 4 of 128, 259 -> 241.
struct ChunkPlan {
  int waves, stretches, per;  // no stretches: a workgroup a tile; per: stretches a tile
  long long tiles;
  size_t lines, bytes;  // of the workspace: pieces' lines, and all of it
};
static ChunkPlan chunk_plan(int T, int q_heads, int heads, int D, int B, int longest) {
  const int group = q_heads / heads;
  ChunkPlan best = {4, 0, 0, 0, 0, 0};
  double least = 0.0;
  for (int waves = 4; waves <= (D == 128 ? 8 : 4); waves += 4) {
    const int rows = 32 * waves, places = D == 256 || waves == 8 ? 256 : 512;
    const long long tiles = B == 1 ? ((long long)T * group + rows - 1) / rows : (long long)T * group / rows + B;
    const double full = D == 64 ? 0.022 : D == 256 ? 0.040 : waves == 8 ? 0.031 : 0.034, rounds = double(tiles) * heads / places;
    const double ends = waves == 8 ? 8.0 : 6.0;
    auto look = [&](int n, int per, double us) {
      if (best.tiles && us >= least) return;
      least = us;
      best.waves = waves, best.tiles = tiles, best.stretches = n, best.per = per;
    };
    // tiles that see the most keys, the fewest, and the mean
    auto most = [&](double key) { return longest * key + ends; };
    auto fewest = [&](double key) { return B == 1 ? fmax(longest - T, 0.0) * key + ends : ends; };
    auto mean = [&](double key) { return B == 1 ? (most(key) + fewest(key)) / 2.0 : 0.5 * longest * key + ends; };
    const double alone = D == 256 ? 0.1 : waves == 8 ? 0.15 : 0.3, key = full * (1.0 - alone + alone * fmin(rounds, 1.0));
    // (the last round's end: of one sequence, half of a tile; of several, sorted, less the more there are)
    const double rest = B == 1 ? 0.5 * fewest(key) : 0.35 * most(key) / rounds;
    const double least_of = fmax(most(key), B == 1 ? ceil(rounds) * fewest(key) : 0.0);
    look(0, 0, rounds <= 1.0 ? most(key) : fmax(least_of, rounds * mean(key) + rest));
    const double held = double(T) * group / tiles;  // rows of a piece
    auto price = [&](long long pieces) { return pieces * heads * held * (D + 4.0) * 8.0 / 4e6; };
    auto fits = [&](long long n) { return n >= 2 && n * heads <= places && n <= tiles * longest / kLeastStretch; };
    auto line = [&](long long n) {
      if (fits(n)) look(int(n), 0, tiles * mean(full) / n + 13.0 + price(n + (n < tiles ? n : tiles)));
    };
    auto pieces = [&](long long per) {
      const double join = per > 4 && per < 8 ? 6.0 : 4.0;  // four at a time by a thread; from eight on, by more threads a line
      if (per >= 2 && fits(tiles * per)) look(int(tiles * per), int(per), longest * full / per + ends + join + price(tiles * per));
    };
    for (long long i = 1; i <= 8; ++i) {
      line(places / heads * i / 8);
      if (B == 1) pieces(i + 1), pieces(places / heads * i / 8 / tiles);
    }
  }
  if (!best.stretches) return best;
  best.lines = size_t(best.stretches) * heads * 2 * 32 * best.waves;
  best.bytes = best.lines * (D + 4) * sizeof(float) + size_t(T) * q_heads * sizeof(int2);
  return best;
}

}  // namespace lmoe

using namespace lmoe;

extern "C" size_t lmoe_kv_chunk_workspace_bytes(int T, int q_heads, int heads, int D, int B, int longest) {
  return T > 0 && B > 0 && heads > 0 && q_heads > 0 && q_heads % heads == 0 && longest > 0
             ? chunk_plan(T, q_heads, heads, D, B, longest).bytes
             : 0;
}

extern "C" int lmoe_kv_chunk(const void *q, int dtype, long long q_row, long long q_head, int T, int q_heads, int heads, int D,
                             const int *cu, const int *lens, int B, const int *table, int width, const uint8_t *k_codes,
                             const float *k_scale, const uint8_t *v_codes, const float *v_scale, int pages, int page, int longest,
                             float scale, void *workspace, size_t workspace_bytes, void *out, void *stream) {
  const char *fn = "lmoe_kv_chunk";
  LMOE_REQUIRE(dtype == LMOE_F16 || dtype == LMOE_BF16, LMOE_EINVAL, "%s: dtype %d (float16 and bfloat16 are served)", fn, dtype);
  LMOE_REQUIRE(D == 64 || D == 128 || D == 256, LMOE_ESHAPE, "%s: heads of %d channels (64, 128 and 256 are served)", fn, D);
  LMOE_REQUIRE(page == 32 || page == 64 || page == 128, LMOE_ESHAPE, "%s: pages of %d tokens (32, 64 and 128 are served)", fn, page);
  LMOE_REQUIRE(heads > 0 && q_heads > 0 && q_heads % heads == 0, LMOE_ESHAPE, "%s: %d query heads over %d key heads", fn, q_heads,
               heads);
  LMOE_REQUIRE(pages > 0 && width > 0 && width <= 0x7fffffff / page, LMOE_ESHAPE, "%s: %d pages, a table of %d places", fn, pages,
               width);
  LMOE_REQUIRE((long long)heads * page * D <= 0x7fffffff, LMOE_ESHAPE, "%s: pages of %d heads, %d tokens and %d channels", fn, heads,
               page, D);
  LMOE_REQUIRE(T >= 0 && B >= 0 && longest > 0, LMOE_ESHAPE, "%s: %d rows of %d sequences of %d tokens", fn, T, B, longest);
  if (T == 0) return 0;
  LMOE_REQUIRE(B > 0, LMOE_ESHAPE, "%s: %d rows of no sequence", fn, T);
  LMOE_REQUIRE(cu || T == B, LMOE_ESHAPE, "%s: %d rows of %d sequences need their offsets", fn, T, B);
  LMOE_REQUIRE(scale > 0.0f && scale < INFINITY, LMOE_EINVAL, "%s: scale %g", fn, double(scale));
  LMOE_REQUIRE(q && out && lens && table && k_codes && k_scale && v_codes && v_scale, LMOE_EINVAL, "%s: null pointer", fn);
  LMOE_REQUIRE(aligned16(q) && aligned16(out) && aligned16(k_codes) && aligned16(v_codes) && q_row % 8 == 0 && q_head % 8 == 0,
               LMOE_EALIGN, "%s: rows and codes must be 16-byte aligned", fn);
  LMOE_REQUIRE((long long)T * q_heads / heads <= 0x7ffff000, LMOE_ESHAPE, "%s: %d rows of %d heads a group", fn, T,
               q_heads / heads);
  const ChunkPlan plan = chunk_plan(T, q_heads, heads, D, B, longest);
  const long long groups = (plan.stretches ? plan.stretches : plan.tiles) * heads;
  // A workgroup joins one line by all of its threads from eight pieces a tile on (48 rows of 32 heads in 42 pieces: 14.4 us with
  // D / 4 threads a line, 10.3 so)
  const bool shared = plan.stretches >= 8 * plan.tiles;
  const long long join_groups = !plan.bytes ? 0 : shared ? (long long)T * q_heads : ((long long)T * q_heads * (D / 4) + 255) / 256;
  // (kMostGroups are of 256 threads)
  LMOE_REQUIRE(groups <= kMostGroups * 4 / plan.waves && join_groups <= kMostGroups, LMOE_ESHAPE,
               "%s: %d rows of %d sequences and %d heads are more than a launch takes", fn, T, B, q_heads);
  LMOE_REQUIRE(plan.bytes == 0 || (workspace && aligned16(workspace) && workspace_bytes >= plan.bytes), LMOE_EWORKSPACE,
               "%s: a 16-byte aligned workspace of %zu bytes is needed", fn, plan.bytes);
  float *part = static_cast<float *>(workspace);
  int2 *joins = plan.bytes ? reinterpret_cast<int2 *>(part + plan.lines * (D + 4)) : nullptr;
  ChunkArgs a = {static_cast<const uint16_t *>(q), q_row, q_head, k_codes, v_codes, k_scale, v_scale, table, lens, cu,
                 static_cast<uint16_t *>(out), part, joins, scale * 1.4426950408889634f, T, B, q_heads, heads, q_heads / heads, pages,
                 width, page == 32 ? 5 : page == 64 ? 6 : 7, int(plan.tiles), plan.stretches, plan.per,
                 groups > (D == 256 || plan.waves == 8 ? 256 : 512), 1.0 / (q_heads / heads),
                 plan.stretches ? 1.0 / plan.stretches : 0.0};
  auto go = [&](auto kernel, size_t lds) -> int {
    if (const int rc = allow_lds(kernel, lds + 4128, fn)) return rc;  // with what the kernel declares itself
    launch(kernel, dim3(unsigned(groups)), dim3(unsigned(64 * plan.waves)), lds, (hipStream_t)stream, a);
    LMOE_LAUNCHED(fn);
    return 0;
  };
  auto join = [&](auto kernel) -> int {
    const int step = 2 * heads * 32 * plan.waves;
    launch(kernel, dim3(unsigned(join_groups)), dim3(256), 0, (hipStream_t)stream,
           JoinArgs{a.out, part, nullptr, T, q_heads, 0, joins, step - 32 * plan.waves, step, int(plan.lines)});
    LMOE_LAUNCHED(fn);
    return 0;
  };
  // two stages of a tile of keys and of values; sums in float32, which the wavefronts store through LDS, may take more
  const size_t tile_lds = size_t(kPromptKeys) * D * 2 * 4, sums = size_t(plan.waves) * 32 * D * 4;
  auto type = [&](auto d, auto bf, auto waves) -> int {
    constexpr int W = decltype(d)::value, NW = decltype(waves)::value;
    constexpr bool BF = decltype(bf)::value;
    if (!plan.stretches) return go(k_chunk_rows<W, BF, NW, false>, tile_lds);
    if (const int rc = go(k_chunk_rows<W, BF, NW, true>, tile_lds > sums ? tile_lds : sums)) return rc;
    return shared ? join(k_join_chunks<W, BF, 1024 / W, true>) : join(k_join_chunks<W, BF, 1, true>);
  };
  auto width_of = [&](auto bf) -> int {
    if (D == 64) return type(IC<64>{}, bf, IC<4>{});
    if (D == 128) return plan.waves == 8 ? type(IC<128>{}, bf, IC<8>{}) : type(IC<128>{}, bf, IC<4>{});
    return type(IC<256>{}, bf, IC<4>{});
  };
  return dtype == LMOE_BF16 ? width_of(IC<1>{}) : width_of(IC<0>{});
}
