// Attention over whole prompts: packed sequences, causal, query heads in groups that share a key head.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - m_i),  over j <= i + (keys - rows) of the sequence
//
// One pass over the keys with a running maximum m. Bound by the matrix cores (4 width products a visible pair) beside the
// exponentials on the vector unit.
//
// A workgroup takes 128 rows of one head, a wavefront 32 of them; keys come 64 at a time, global -> LDS
// without registers, the next tile's copies in flight under the present one's products. Products are written so that
// nothing has to change lanes between them:
//   scores^T = K Q^T   A = 32 keys (lane & 31) x 16 channels from LDS, B = Q^T from registers: a lane ends with 16 of 32
//                      keys' scores of one row (lane & 31), the other 16 in lane ^ 32;
//   out^T += V^T P^T   B = eight of those weights as they lie (keys 4 h + i and 8 + 4 h + i, h = lane >> 5); A = the same
//                      keys' values of one channel, by LDS loads that transpose (ds_read_b64_tr_b16).
// Weights are rounded to the inputs' type for the matrix cores (float16: times 2^11, so that those down to 2^-25 of a row's
// largest keep all their bits), and what a row is divided by is the float32 sum of the rounded weights.
//
// The next tile's score products, this tile's exponentials and its output products are issued in one stream of slots, a
// product and about eight vector instructions each: 32 cycles of either. Measured (32 heads over 4 of 128, bf16, 8,192 rows):
// masks in every tile 714 us, full tiles without them 557, fragments read ahead and copies spread over the slots (a burst of
// them stalls a wavefront for 900 cycles) 521-530, q and output in whole rows 503-532, 1.03-1.09 PFLOP/s. What is left is LDS
// traffic: of 521, without half of the key reads 457, without the copies 453, without exponentials 488.
//
// Values that a row must not see are multiplied by a weight of zero; where one is not finite in a tile that some row does
// not see whole, it is taken out and given to the rows that do see it alone.
#include "rows.h"

namespace lmoe {

constexpr int kPromptRows = 128, kPromptKeys = 64;  // a workgroup's rows, and keys a tile
constexpr int kAhead = 3;  // products that a fragment is read ahead of its own

struct PromptArgs {
  const uint16_t *q, *k, *v;
  long long q_row, q_head, k_row, k_head, v_row, v_head;  // elements
  const int *cu, *cu_k;
  uint16_t *out;
  float *part;  // [chunks][T][q_heads] of [D] sums and {maximum, weight}: rows whose keys are worked in more than one chunk
  int *joins;   // [T][q_heads]: how many chunks (0: one, the row is done)
  float scale;  // times log2 e
  int T, U, B, q_heads, heads, tiles, chunk, chunks;  // chunk: keys, the last of `chunks` goes on to the end
};

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
// One wavefront-wide copy of 16 bytes a lane, from voff in what the descriptor covers, to LDS address lds + 16 lane
__device__ __forceinline__ void dma_rows(u32x4 rows, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(rows), "s"(lds) : "memory");
}

// The same from an address of each lane's own
__device__ __forceinline__ void dma_lanes(const void *from, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(lds) : "memory");
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
template <int D, bool BF>
__device__ __forceinline__ bool any_bad(const uint8_t *vt) {
  constexpr uint32_t INF = BF ? 0x7f80u : 0x7c00u;
  uint32_t over = 0;
#pragma unroll
  for (int i = 0; i < kPromptKeys * D / 8 / 256; ++i) {  // a half word's magnitude of INF or more carries into its sign bit
    const u32x4 w = reinterpret_cast<const u32x4 *>(vt)[i * 256 + threadIdx.x];
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

// Whether every output product's weights are packed a slot before it: NM score products, NV output products over NP pairs of
// weights, DT channel tiles, pairs spread over NS slots and packed one slot later
constexpr bool weights_in_time(int NM, int NV, int NP, int DT, int NS) {
  for (int k = 0; k < NV; ++k) {
    const int slots = NM + k - 1 < NS ? NM + k - 1 : NS;
    if (slots * NP / NS < 4 * (k / DT + 1)) return false;
  }
  return true;
}

// The nth tile of rows that is worked, by one wavefront. Up to 64 sequences: the tiles furthest into their sequences first,
// which see the most keys, so that what is left for the end is short (16 prompts of up to 4,000 rows at width 64: 160 -> 134
// us, of up to 900 at 128: 37 -> 30; long prompts lose up to 5 % by sharing less of L2: 12 of up to 3,500 rows 332 -> 345).
// More: the sequences from the last on, each from its end; sequence b's tiles begin at cu[b] / rows + b, which leaves it room
// for all of them, and for one that is empty where its rows fill their tiles. Eight tiles in turn are shifted against the next
// eight: workgroups go to the four quarters of an XCD in turn, and 72 sequences of 128 rows, every second workgroup empty, left
// half of the CUs idle (16 heads of 256: 118 -> 81 us). b < 0: there is none. The first and the last sequence have a tile even
// without rows.
struct PromptTile {
  int b, tile, row0, nq, key0, nk;
};
__device__ __forceinline__ PromptTile nth_tile(const PromptArgs &a, int nth) {
  PromptTile w = {-1, 0, 0, 0, 0, 0};
  if (a.B > 64) {
    const int turned = nth < (a.tiles & ~7) ? (nth & ~7) | ((nth + (nth >> 3)) & 7) : nth;
    const int task = a.tiles - 1 - turned;
    w.b = last_at(a.cu, a.B, task, [](int c, int i) { return (long long)(c / kPromptRows) + i; });
    if (w.b < 0) return w;
    seq_rows(a.cu, w.b, a.T, &w.row0, &w.nq);
    seq_rows(a.cu_k, w.b, a.U, &w.key0, &w.nk);
    w.tile = task - (a.cu[w.b] / kPromptRows + w.b);
    return w;
  }
  const int lane = threadIdx.x & 63;
  int row0 = 0, nq = 0, key0 = 0, nk = 0, tiles = 0;
  if (lane < a.B) {
    seq_rows(a.cu, lane, a.T, &row0, &nq);
    seq_rows(a.cu_k, lane, a.U, &key0, &nk);
    tiles = max((nq + kPromptRows - 1) / kPromptRows, lane == 0 || lane == a.B - 1 ? 1 : 0);
  }
  // how many tiles have an index of j or more (counts below 2^24: exact in float32)
  auto from = [&](int j) { return int(wave_sum(float(max(0, tiles - j)))); };
  int lo = 0, hi = int(wave_max(float(tiles))), behind = 0;
  if (nth >= from(0)) return w;
  while (hi - lo > 1) {  // the largest index with more than nth tiles from it on
    const int mid = (lo + hi) >> 1, n = from(mid);
    if (n > nth)
      lo = mid;
    else
      hi = mid, behind = n;
  }
  unsigned long long has = __ballot(tiles > lo);
  for (int i = nth - behind; i > 0; --i) has &= has - 1;
  const int b = __ffsll(has) - 1;
  w = {b, lo, __builtin_amdgcn_readlane(row0, b), __builtin_amdgcn_readlane(nq, b), __builtin_amdgcn_readlane(key0, b),
       __builtin_amdgcn_readlane(nk, b)};
  return w;
}

template <int D, bool BF>
__global__ void __launch_bounds__(256, D == 256 ? 1 : 2) k_prompt(PromptArgs a) {
  constexpr int BN = kPromptKeys, MT = BN / 32, KS = D / 16, DT = D / 32, COPIES = BN * D / 512 / 4;
  constexpr int kTileBytes = BN * D * 2;
  extern __shared__ uint8_t lds[];  // [2 stages][K tile, V tile]
  __shared__ uint32_t marks[2 * BN * DT];   // of take_bad: [pos, neg][key][32 channels]
  __shared__ uint32_t flags[4];             // of any_bad: a wavefront's
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 31, h = lane >> 5;
  // heads of one XCD are neighbours (they share key heads in its L2)
  const int slot = blockIdx.x % a.q_heads, chunk = int(blockIdx.x) / a.q_heads % a.chunks;
  const int nth = int(blockIdx.x) / (a.q_heads * a.chunks);
  const int head = a.q_heads % 8 == 0 ? (slot & 7) * (a.q_heads / 8) + (slot >> 3) : slot;
  const PromptTile work = nth_tile(a, nth);
  const int b = work.b, tile = work.tile, row0 = work.row0, nq = work.nq, key0 = work.key0, nk = work.nk;
  if (b < 0) return;
  if (tile == 0 && chunk == 0 && (b == 0 || b == a.B - 1)) {
    // rows before the first sequence or behind the last one come back zero
    const int lo = b == 0 ? min(max(a.cu[0], 0), a.T) : 0, hi = b == a.B - 1 ? min(max(a.cu[a.B], 0), a.T) : a.T;
    for (int row = int(threadIdx.x) / (D / 8); row < lo + (a.T - hi); row += 256 / (D / 8)) {
      const size_t line = size_t(row < lo ? row : hi + row - lo) * a.q_heads + head;
      *reinterpret_cast<u32x4 *>(a.out + line * D + (threadIdx.x % (D / 8)) * 8) = u32x4{};
      if (a.joins) a.joins[line] = 0;
    }
  }
  const int first = tile * kPromptRows;
  if (uint32_t(first) >= uint32_t(nq)) return;  // (a tile before the sequence's first: where offsets fall)
  const int off = nk - nq;                                  // row i sees keys 0 .. i + off
  const int most_keys = off + min(first + kPromptRows, nq);  // what the workgroup's last row sees
  const int begin = chunk * a.chunk;                         // this workgroup's keys: [begin, keys)
  if (chunk > 0 && begin >= most_keys) return;
  const int keys = chunk + 1 < a.chunks ? min(most_keys, begin + a.chunk) : most_keys;
  const int parts = a.part ? min(a.chunks, (most_keys - 1) / a.chunk + 1) : 1;  // chunks that the tile's keys take
  const int mine = min(first + 32 * wave + r, nq - 1), sees = mine + off + 1;
  const int all = first + 32 * wave + off + 1;  // what every row of the wavefront sees
  const int kv = head / (a.q_heads / a.heads);

  const uint32_t base = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t *)lds));
  // Copy i of this wavefront: 64 chunks of 16 bytes in LDS order; the rows' chunks are permuted on the global side. A tile's
  // copies go through a descriptor that ends with the sequence's last key: rows past it are not read.
  uint32_t k_off[COPIES], v_off[COPIES];
#pragma unroll
  for (int i = 0; i < COPIES; ++i) {
    const int j = (wave * COPIES + i) * 64 + lane, row = j / (D / 8), c = j % (D / 8);
    k_off[i] = uint32_t(row) * uint32_t(a.k_row * 2) + k_chunk<D>(row, c) * 16;
    v_off[i] = uint32_t(row) * uint32_t(a.v_row * 2) + (v_pair<D>(row, c >> 1) * 2 + (c & 1)) * 16;
  }
  auto tile_of_rows = [&](const uint16_t *p, long long stride, int at) {
    const uint64_t from = reinterpret_cast<uint64_t>(p + (long long)min(at, nk) * stride);
    const long long bytes = at < nk ? ((nk - 1 - at) * stride + D) * 2 : 0;
    return u32x4{uint32_t(from), uint32_t(from >> 32) & 0xffffu, uint32_t(min(bytes, 1ll << 31)), 0x00020000u};
  };
  const uint16_t *k_rows = a.k + size_t(key0) * a.k_row + size_t(kv) * a.k_head;
  const uint16_t *v_rows = a.v + size_t(key0) * a.v_row + size_t(kv) * a.v_head;
  const uint32_t to = base + wave * COPIES * 1024;
  auto fetch_k = [&](int at, int stage) {
    const u32x4 rows = tile_of_rows(k_rows, a.k_row, at);
#pragma unroll
    for (int i = 0; i < COPIES; ++i) dma_rows(rows, k_off[i], to + stage * kTileBytes + i * 1024);
  };
  auto fetch_v = [&](int at, int stage) {
    const u32x4 rows = tile_of_rows(v_rows, a.v_row, at);
#pragma unroll
    for (int i = 0; i < COPIES; ++i) dma_rows(rows, v_off[i], to + (2 + stage) * kTileBytes + i * 1024);
  };
  // The wavefront's rows of q come through LDS too, 16 of them in its part of the second key tile and 16 in its part of the
  // second value tile, and so does its output: loads and stores of whole rows, where fragments are 32 and 16 bytes of 32 rows
  // each. A workgroup's time beside its tiles at width 256: 9.6 -> 7 us (9 prompts of 1,024 rows, 16 heads: 159 -> 146; 32 heads
  // of 128: 136 -> 124)
  u32x4 qf[KS];
  if (keys > begin) {
    fetch_k(begin, 0);
    const uint16_t *q = a.q + size_t(row0) * a.q_row + size_t(head) * a.q_head;
#pragma unroll
    for (int i = 0; i < 2 * COPIES; ++i) {
      const int j = (i % COPIES) * 64 + lane, row = j / (D / 8), c = j % (D / 8);
      const int of = min(first + 32 * wave + 16 * (i / COPIES) + row, nq - 1);
      dma_lanes(q + size_t(of) * a.q_row + k_chunk<D>(row, c) * 8, to + (i < COPIES ? 1 : 3) * kTileBytes + (i % COPIES) * 1024);
    }
    fetch_v(begin, 0);
    wait_vm<COPIES>();
    const uint8_t *own = lds + (r < 16 ? 1 : 3) * kTileBytes + wave * COPIES * 1024 + (r & 15) * D * 2;
#pragma unroll
    for (int j = 0; j < KS; ++j) qf[j] = *reinterpret_cast<const u32x4 *>(own + k_chunk<D>(r & 15, 2 * j + h) * 16);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the rows are read before keys replace them
    fetch_k(begin + BN, 1);
    barrier_lds();
  }
  f32x16 o[DT] = {};
  float m = -INFINITY, l = 0.0f;
  // a transposing load: 16 lanes take 4 keys x 16 channels, lane i of them gets channel i of the 4
  const int vrow = 4 * h + ((lane & 15) >> 2), vpair = (lane >> 4) & 1, vbyte = (lane & 3) * 8;
  auto k_frag = [&](const uint8_t *kt, int t, int j) {
    const int row = 32 * t + r;
    return *reinterpret_cast<const u32x4 *>(kt + row * D * 2 + k_chunk<D>(row, 2 * j + h) * 16);
  };
  auto v_frag = [&](const uint8_t *vt, int d, int ks) {
    u32x4 f;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int row = 16 * ks + 8 * x + vrow;
      const uint8_t *src = vt + row * D * 2 + v_pair<D>(row, 2 * d + vpair) * 32 + vbyte;
      const u32x2 g = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(src)));
      f[2 * x] = g.x, f[2 * x + 1] = g.y;
    }
    return f;
  };
  auto largest = [](const f32x16 (&x)[MT]) {
    float y[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) y[e & 3] = fmaxf(y[e & 3], x[t][e]);
    return fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
  };
  f32x16 s[MT] = {};  // the scores of the tile at hand
  if (keys > begin) {
#pragma unroll
    for (int j = 0; j < KS; ++j)
#pragma unroll
      for (int t = 0; t < MT; ++t) s[t] = mfma32<BF>(k_frag(lds, t, j), qf[j], s[t]);
  }
  float top = largest(s);
  // one tile: its scores s become next, the following tile's. Called with the two in turn, so that nothing is moved.
  auto step = [&](int at, auto stage_c, f32x16 (&s)[MT], f32x16 (&next)[MT]) {
    constexpr int stage = decltype(stage_c)::value;
    wait_vm<0>();
    barrier_lds();  // this tile's values and the next one's keys are there, and what they replace has been read
    const u32x4 k_tile = tile_of_rows(k_rows, a.k_row, at + 2 * BN), v_tile = tile_of_rows(v_rows, a.v_row, at + BN);
    auto copy = [&](int i) {  // copy i of the next tile's values and of the keys after that
      if (i < COPIES)
        dma_rows(v_tile, v_off[i], to + (2 + (stage ^ 1)) * kTileBytes + i * 1024);
      else
        dma_rows(k_tile, k_off[i - COPIES], to + stage * kTileBytes + (i - COPIES) * 1024);
    };
    const uint8_t *kt = lds + (stage ^ 1) * kTileBytes, *vt = lds + (2 + stage) * kTileBytes;
    bool bad = false;
    if (at + BN > first + off + 1) {  // the workgroup's first row does not see all of it
      const bool found = __any(any_bad<D, BF>(vt));
      if (lane == 0) flags[wave] = found;
      barrier_lds();
      bad = __builtin_amdgcn_readfirstlane(flags[0] | flags[1] | flags[2] | flags[3]);
      if (bad) {
        for (int i = threadIdx.x; i < BN * DT; i += 256)
          take_bad<D, BF>(const_cast<uint8_t *>(vt), i / DT, i % DT, &marks[i], &marks[BN * DT + i]);
        barrier_lds();
      }
    }
    if (at + BN > all) {
      const int left = opaque(sees - at - 4 * h);  // opaque: a branch, not 64 selects in every tile
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (32 * t + 8 * (e >> 2) + (e & 3) >= left) s[t][e] = -INFINITY;
      top = largest(s);
    }
    // The matrix products of a tile: the next tile's scores, then this one's output, their fragments read kAhead products ahead
    constexpr int NM = MT * KS, NV = MT * 2 * DT, NP = MT * 8;
    u32x4 ring[kAhead + 1];
    auto frag = [&](auto ic) {
      constexpr int i = decltype(ic)::value;
      if constexpr (i < NM)
        ring[i % (kAhead + 1)] = k_frag(kt, i % MT, i / MT);
      else if constexpr (i < NM + NV)
        ring[i % (kAhead + 1)] = v_frag(vt, (i - NM) % DT, (i - NM) / DT);
    };
    static_for<0, kAhead>([&](auto ic) { frag(ic); });
    __builtin_amdgcn_sched_barrier(0);
    top = fmaxf(top, lane_xor32(top)) * a.scale;
    // The maximum in use may lag by kLag octaves, so that most tiles leave the sums as they are
    if (__any(top > m + kLag<BF>)) {
      const float to = fmaxf(m, top), keep = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
      m = to;
      l *= keep;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= keep;
    }
    const float lift = m == -INFINITY ? 0.0f : kLift<BF> - m;
    // Past the last tile the next scores are of whatever LDS holds, and unused. The vector unit's work goes between the
    // products, in the order that leaves no instruction waiting for the one before it: a slot's pairs of weights get their
    // exponentials, the slot before's are packed, the one before that's are summed. Half of the output products go among
    // them (their weights are ready by then), and the next scores' maximum goes among the other half.
    constexpr int NS = NM + NV / 2 - 2, NR = NM + NV - NS;  // slots with exponentials, and with the maximum
    u32x4 p[MT * 2];
    float part[2] = {l, 0.0f}, peak[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, ex[NP][2];
    static_assert(weights_in_time(NM, NV, NP, DT, NS), "an output product before its weights");
    auto each = [&](auto slot, auto f) {  // the pairs of a slot
      constexpr int i = decltype(slot)::value;
      if constexpr (i >= 0 && i < NS) static_for<i * NP / NS, (i + 1) * NP / NS>(f);
    };
    static_for<0, NM + NV>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      frag(IC<i + kAhead>{});
      if constexpr (i % 2 == 0 && i < 4 * COPIES) copy(i / 2);
      if constexpr (i < NM)
        next[i % MT] = mfma32<BF>(ring[i % (kAhead + 1)], qf[i / MT], i < MT ? f32x16{} : next[i % MT]);
      else
        o[(i - NM) % DT] = mfma32<BF>(ring[i % (kAhead + 1)], p[(i - NM) / DT], o[(i - NM) % DT]);
      each(IC<i>{}, [&](auto ec) {
        constexpr int e = decltype(ec)::value, u = e / 8, x = e % 8;
        ex[e][0] = __builtin_amdgcn_exp2f(fmaf(s[u][2 * x], a.scale, lift));
        ex[e][1] = __builtin_amdgcn_exp2f(fmaf(s[u][2 * x + 1], a.scale, lift));
      });
      each(IC<i - 1>{}, [&](auto ec) {
        constexpr int e = decltype(ec)::value;
        p[e / 4][e & 3] = pack2<BF>(ex[e][0], ex[e][1]);
      });
      each(IC<i - 2>{}, [&](auto ec) {
        constexpr int e = decltype(ec)::value;
        part[e & 1] = add2<BF>(p[e / 4][e & 3], part[e & 1]);
      });
      if constexpr (i >= NS)
        static_for<(i - NS) * NP * 2 / NR, (i - NS + 1) * NP * 2 / NR>([&](auto ec) {
          constexpr int e = decltype(ec)::value;
          peak[(e >> 1) & 3] = fmaxf(peak[(e >> 1) & 3], next[e / 16][e % 16]);
        });
      __builtin_amdgcn_sched_barrier(0);
    });
    l = part[0] + part[1];
    top = fmaxf(fmaxf(peak[0], peak[1]), fmaxf(peak[2], peak[3]));
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
  f32x16 other[MT];
  for (int at = begin; at < keys; at += 2 * BN) {
    step(at, IC<0>{}, s, other);
    if (at + BN >= keys) break;
    step(at + BN, IC<1>{}, other, s);
  }
  wait_vm<0>();  // the last tiles' copies (of nothing) land before the LDS holds rows, or is another workgroup's
  barrier_lds();
  l += lane_xor32(l);
  const bool there = first + 32 * wave + r < nq;
  const size_t line = size_t(row0 + mine) * a.q_heads + head;
  if (a.part) {
    if (there && chunk == 0 && h == 0) a.joins[line] = parts > 1 ? parts : 0;
    if (parts > 1) {
      float *rows = reinterpret_cast<float *>(lds) + wave * 32 * D;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<f32x4 *>(rows + r * D + ((8 * d + 2 * e + h) ^ (r & 15)) * 4) =
              f32x4{o[d][4 * e], o[d][4 * e + 1], o[d][4 * e + 2], o[d][4 * e + 3]};
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      float *part = a.part + (size_t(chunk) * a.T + row0 + first + 32 * wave) * a.q_heads * (D + 4) + size_t(head) * (D + 4);
#pragma unroll
      for (int i = 0; i < 32 * D / 256; ++i) {
        const int j = i * 64 + lane, row = j / (D / 4), c = j % (D / 4);
        const f32x4 w = *reinterpret_cast<const f32x4 *>(rows + row * D + (c ^ (row & 15)) * 4);
        if (first + 32 * wave + row < nq) *reinterpret_cast<f32x4 *>(part + size_t(row) * a.q_heads * (D + 4) + c * 4) = w;
      }
      if (there && h == 0) *reinterpret_cast<float2 *>(part + size_t(r) * a.q_heads * (D + 4) + D) = float2{m, l};
      return;
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  // through LDS, so that a store writes whole rows
  uint8_t *rows = lds + wave * 32 * D * 2;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      *reinterpret_cast<u32x2 *>(rows + r * D * 2 + k_chunk<D>(r, 4 * d + e) * 16 + 8 * h) =
          u32x2{pack2<BF>(o[d][4 * e] * inv, o[d][4 * e + 1] * inv), pack2<BF>(o[d][4 * e + 2] * inv, o[d][4 * e + 3] * inv)};
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  uint16_t *out = a.out + (size_t(row0 + first + 32 * wave) * a.q_heads + head) * D;
#pragma unroll
  for (int i = 0; i < 32 * D / 512; ++i) {
    const int j = i * 64 + lane, row = j / (D / 8), c = j % (D / 8);
    const u32x4 w = *reinterpret_cast<const u32x4 *>(rows + row * D * 2 + k_chunk<D>(row, c) * 16);
    if (first + 32 * wave + row < nq) *reinterpret_cast<u32x4 *>(out + size_t(row) * a.q_heads * D + c * 8) = w;
  }
}

// Rows whose keys were worked in more than one chunk: D / 4 threads a row and head, the chunks joined in order
template <int D, bool BF>
__global__ void __launch_bounds__(256) k_prompt_join(PromptArgs a) {
  constexpr int LANES = D / 4;
  const size_t line = size_t(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES, lines = size_t(a.T) * a.q_heads;
  if (line >= lines) return;
  const int parts = min(a.joins[line], a.chunks), d = (threadIdx.x % LANES) * 4;
  if (parts < 2) return;
  f32x4 v = {};
  float top = -INFINITY, weight = 0.0f;
  for (int c0 = 0; c0 < parts; c0 += 4) {
    float2 ml[4];
    f32x4 y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float *part = a.part + (size_t(min(c0 + j, parts - 1)) * lines + line) * (D + 4);
      ml[j] = *reinterpret_cast<const float2 *>(part + D);
      y[j] = *reinterpret_cast<const f32x4 *>(part + d);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (c0 + j >= parts || ml[j].y == 0.0f) continue;  // (a chunk that the row sees nothing of weighs 0; NaN goes on)
      const float to = fmaxf(top, ml[j].x), f = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ml[j].x - to);
      const float keep = weight == 0.0f ? 0.0f : to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - to);
      top = to;
      weight = fmaf(ml[j].y, f, weight * keep);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = fmaf(y[j][e], f, v[e] * keep);
    }
  }
  const float inv = weight == 0.0f ? 0.0f : 1.0f / weight;
  *reinterpret_cast<u32x2 *>(a.out + line * D + d) = u32x2{pack2<BF>(v[0] * inv, v[1] * inv), pack2<BF>(v[2] * inv, v[3] * inv)};
}

// Chunks of keys, where the rows alone would leave half of the GPU's places idle (two workgroups a CU, one at width 256): as many
// as fit the places, of 512 keys (eight tiles) at least. Rows' tiles are bounded by T / 128 + B, one more a sequence than there
// are where rows fill their tiles: one sequence's 1,024 rows over 8,024 keys are 448 workgroups on 512 places with 28 heads of
// 128, in two chunks, but with 32 heads 256 in one, and with 16 heads of 256 channels 128 on 256. Between half of the places
// and all of them nothing is split.
struct PromptPlan {
  int chunk, chunks;
  size_t rows, bytes;  // the workspace's sums, and all of it
};
static PromptPlan prompt_plan(int T, int U, int q_heads, int D, int B) {
  PromptPlan p = {1 << 30, 1, 0, 0};
  const long long work = (T / 128 + (long long)B) * q_heads, full = D == 256 ? 256 : 512;
  if (work <= 0 || 2 * work > full) return p;
  const int splits = int(full / work);
  long long chunk = ((long long)U / (B > 0 ? B : 1) + splits - 1) / splits;
  chunk = (chunk < 512 ? 512 : chunk) + kPromptKeys - 1;
  chunk -= chunk % kPromptKeys;
  const long long chunks = (U + chunk - 1) / chunk, most = 4ll * splits;
  if (chunks <= 1) return p;
  p.chunk = int(chunk);
  p.chunks = int(chunks < most ? chunks : most);
  p.rows = size_t(p.chunks) * T * q_heads * (D + 4) * sizeof(float);
  p.bytes = p.rows + size_t(T) * q_heads * sizeof(int);
  return p;
}

}  // namespace lmoe

using namespace lmoe;

extern "C" size_t lmoe_prompt_attend_workspace_bytes(int T, int U, int q_heads, int heads, int D, int B) {
  return T > 0 && U > 0 && q_heads > 0 ? prompt_plan(T, U, q_heads, D, B).bytes : 0;
}

extern "C" int lmoe_prompt_attend(const void *q, long long q_row, long long q_head, const void *k, long long k_row,
                                  long long k_head, const void *v, long long v_row, long long v_head, int dtype, int T, int U,
                                  int q_heads, int heads, int D, const int *cu, const int *cu_k, int B, float scale, void *workspace,
                                  size_t workspace_bytes, void *out, void *stream) {
  const char *fn = "lmoe_prompt_attend";
  LMOE_REQUIRE(dtype == LMOE_F16 || dtype == LMOE_BF16, LMOE_EINVAL, "%s: dtype %d (float16 and bfloat16 are served)", fn, dtype);
  LMOE_REQUIRE(D == 64 || D == 128 || D == 256, LMOE_ESHAPE, "%s: heads of %d channels (64, 128 and 256 are served)", fn, D);
  LMOE_REQUIRE(heads > 0 && q_heads > 0 && q_heads % heads == 0, LMOE_ESHAPE, "%s: %d query heads over %d key heads", fn, q_heads,
               heads);
  LMOE_REQUIRE(T >= 0 && U >= 0 && B >= 0, LMOE_ESHAPE, "%s: %d rows, %d keys, %d sequences", fn, T, U, B);
  if (T == 0) return 0;
  LMOE_REQUIRE(B > 0, LMOE_ESHAPE, "%s: %d rows of no sequence", fn, T);
  LMOE_REQUIRE(scale > 0.0f && scale < INFINITY, LMOE_EINVAL, "%s: scale %g", fn, double(scale));
  LMOE_REQUIRE(q && out && cu && cu_k && ((k && v) || U == 0), LMOE_EINVAL, "%s: null pointer", fn);
  LMOE_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out) && q_row % 8 == 0 && q_head % 8 == 0 &&
                   k_row % 8 == 0 && k_head % 8 == 0 && v_row % 8 == 0 && v_head % 8 == 0,
               LMOE_EALIGN, "%s: rows must be 16-byte aligned", fn);
  LMOE_REQUIRE(k_row >= 0 && v_row >= 0 && k_row < (1 << 23) && v_row < (1 << 23), LMOE_ESHAPE,
               "%s: rows of keys %lld and of values %lld elements apart", fn, k_row, v_row);
  const long long tiles = T / kPromptRows + (long long)B;
  const PromptPlan plan = prompt_plan(T, U, q_heads, D, B);
  LMOE_REQUIRE(tiles * q_heads * plan.chunks <= kMostGroups, LMOE_ESHAPE,
               "%s: %d rows of %d sequences and %d heads are more than a launch takes", fn, T, B, q_heads);
  LMOE_REQUIRE(plan.bytes == 0 || (workspace && aligned16(workspace) && workspace_bytes >= plan.bytes), LMOE_EWORKSPACE,
               "%s: a 16-byte aligned workspace of %zu bytes is needed", fn, plan.bytes);
  float *part = plan.bytes ? static_cast<float *>(workspace) : nullptr;
  int *joins = plan.bytes ? reinterpret_cast<int *>(static_cast<char *>(workspace) + plan.rows) : nullptr;
  PromptArgs a = {static_cast<const uint16_t *>(q), static_cast<const uint16_t *>(k), static_cast<const uint16_t *>(v), q_row,
                  q_head, k_row, k_head, v_row, v_head, cu, cu_k, static_cast<uint16_t *>(out), part, joins,
                  scale * 1.4426950408889634f, T, U, B, q_heads, heads, int(tiles), plan.chunk, plan.chunks};
  auto go = [&](auto kernel, auto join) -> int {
    const size_t lds = size_t(kPromptKeys) * D * 2 * 4;
    if (const int rc = allow_lds(kernel, lds + 4112, fn)) return rc;  // with what the kernel declares itself
    launch(kernel, dim3(unsigned(tiles * q_heads * plan.chunks)), dim3(256), lds, (hipStream_t)stream, a);
    LMOE_LAUNCHED(fn);
    if (part) {
      launch(join, dim3(unsigned(((long long)T * q_heads * (D / 4) + 255) / 256)), dim3(256), 0, (hipStream_t)stream, a);
      LMOE_LAUNCHED(fn);
    }
    return 0;
  };
  const bool bf = dtype == LMOE_BF16;
  if (D == 64) return bf ? go(k_prompt<64, true>, k_prompt_join<64, true>) : go(k_prompt<64, false>, k_prompt_join<64, false>);
  if (D == 128) return bf ? go(k_prompt<128, true>, k_prompt_join<128, true>) : go(k_prompt<128, false>, k_prompt_join<128, false>);
  return bf ? go(k_prompt<256, true>, k_prompt_join<256, true>) : go(k_prompt<256, false>, k_prompt_join<256, false>);
}
