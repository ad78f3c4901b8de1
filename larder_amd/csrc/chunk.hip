// Attention of chunks of new rows over the 8-bit paged cache, causal: a later chunk of a prompt, a message after a long history,
// a tree of drafts.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - m),  over the places j < len - (n - 1 - r) of row r of n
//
// One pass over the keys with a running maximum m. A workgroup takes 128 (row, query head of the group) pairs of one key
// head, so that the heads of a group share what it reads; keys come 64 at a time: their codes straight from the pages to
// registers, a tile ahead, then as 16-bit values (exact) to LDS, from where the matrix cores' operands are read as in prompt.hip.
// Pages hold 32 tokens at least, so a half of a tile has one page, one scale of keys and one of values: the former multiplies
// float32 scores, the latter goes into the conversion. bfloat16 takes any scale; float16 takes it relative to a reference that
// moves, and the sums with it, when a page's scale leaves 2^-15 .. 2^7 of it, so that the conversion stays exact.
//
// Products, weights, sums and values that are not finite: as in prompt.hip.
#include "flash.h"

namespace lmoe {

struct ChunkArgs {
  const uint16_t *q;
  long long q_row, q_head;  // elements
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int *table, *lens, *cu;
  uint16_t *out;  // [T][q_heads][D]
  float *part;    // [chunks][T][q_heads] of [D] sums and {maximum, weight}: rows whose keys are worked in more than one chunk
  int *joins;     // [T][q_heads]: how many chunks (0: one, the row is done)
  float scale;    // times log2 e
  int T, B, q_heads, heads, group, pages, width, page_shift, tiles, chunk, chunks;  // chunk: keys, the last goes on to the end
};

// The nth tile of ROWS pairs that is worked, by one wavefront. Up to 64 sequences: those that see the most keys first (to 256
// keys), so that what is left for the end is short. More: the sequences from the last on, each from its end, eight tiles in
// turn shifted against the next eight (prompt.hip says why); sequence b's tiles begin at cu[b] group / ROWS + b, which leaves
// it room for all of them. b < 0: there is none. The first and the last sequence have a tile even without rows.
struct ChunkTile {
  int b, tile, row0, n, len;
};
template <int ROWS>
__device__ __forceinline__ ChunkTile nth_chunk_tile(const ChunkArgs &a, int nth) {
  ChunkTile w = {-1, 0, 0, 0, 0};
  if (a.B > 64) {
    const int turned = nth < (a.tiles & ~7) ? (nth & ~7) | ((nth + (nth >> 3)) & 7) : nth;
    const int task = a.tiles - 1 - turned;
    auto begin = [&](int c, int i) { return (long long)c * a.group / ROWS + i; };
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
    tiles = max(int(((long long)n * a.group + ROWS - 1) / ROWS), lane == 0 || lane == a.B - 1 ? 1 : 0);
  }
  // A tile sees about past + tile ROWS / group keys: how many tiles of the lane's sequence see 256 x or more
  const int past = max(len - n, 0);
  auto count = [&](int x) {
    const long long rows = 256ll * x - past;
    const long long at = rows <= 0 ? 0 : (rows * a.group + ROWS - 1) / ROWS;
    return at >= tiles ? 0 : tiles - int(at);
  };
  auto from = [&](int x) { return int(wave_sum(float(count(x)))); };  // (counts below 2^24: exact in float32)
  int lo = 0, hi = (int(wave_max(tiles > 0 ? float(past) + float(tiles) * ROWS / a.group : 0.0f)) >> 8) + 2, behind = 0;
  if (nth >= from(0)) return w;
  while (hi - lo > 1) {  // the largest x with more than nth tiles from it on
    const int mid = lo + ((hi - lo) >> 1), c = from(mid);
    if (c > nth)
      lo = mid;
    else
      hi = mid, behind = c;
  }
  // of the tiles that see 256 lo keys and not 256 more, the lane's sequence has `mine`; in the order of sequences
  const int above = count(lo + 1), mine = count(lo) - above;
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

// 16 codes times a power of two as 16-bit floats
template <bool BF>
__device__ __forceinline__ void widen(u32x4 w, float scale, u32x4 &lo, u32x4 &hi) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t a, b;
    if constexpr (BF) {
      a = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[e], scale, false));
      b = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[e], scale, true));
    } else {
      a = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[e], scale, false));
      b = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[e], scale, true));
    }
    if (e < 2)
      lo[2 * e] = a, lo[2 * e + 1] = b;
    else
      hi[2 * e - 4] = a, hi[2 * e - 3] = b;
  }
}

// The codes of half a tile (32 tokens of a page's head): rows past `rows` read as zeros
__device__ __forceinline__ u32x4 load_rows(const uint8_t *from, int bytes, int at) {
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(from), 0, bytes, 0x00020000);
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, 0));
}

template <int D, bool BF>
__global__ void __launch_bounds__(256, D == 256 ? 1 : 2) k_chunk_rows(ChunkArgs a) {
  constexpr int ROWS = 128, BN = kPromptKeys, KS = D / 16, DT = D / 32, COPIES = D / 64;
  constexpr int kTileBytes = BN * D * 2;
  extern __shared__ uint8_t lds[];  // [2 stages][K tile, V tile]
  __shared__ uint32_t marks[2 * BN * DT];  // of take_bad: [pos, neg][key][32 channels]
  __shared__ uint32_t flags[4];            // of any_bad: a wavefront's
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, h = lane >> 5;
  const int kv = blockIdx.x % a.heads, chunk = int(blockIdx.x) / a.heads % a.chunks;
  const ChunkTile work = nth_chunk_tile<ROWS>(a, int(blockIdx.x) / (a.heads * a.chunks));
  const int b = work.b, n = work.n, group = a.group;
  if (b < 0) return;
  if (work.tile == 0 && chunk == 0 && a.cu && (b == 0 || b == a.B - 1)) {
    // rows before the first sequence or behind the last one come back zero
    const int lo = b == 0 ? min(max(a.cu[0], 0), a.T) : 0, hi = b == a.B - 1 ? min(max(a.cu[a.B], 0), a.T) : a.T;
    const int per = group * (D / 8);
    for (long long i = tid; i < (long long)(lo + (a.T - hi)) * per; i += 256) {
      const int row = int(i / per), c = int(i - (long long)row * per);
      const size_t line = size_t(row < lo ? row : hi + row - lo) * a.q_heads + kv * group + c / (D / 8);
      *reinterpret_cast<u32x4 *>(a.out + line * D + (c % (D / 8)) * 8) = u32x4{};
      if (a.joins && c % (D / 8) == 0) a.joins[line] = 0;
    }
  }
  const int pairs = n * group, first = work.tile * ROWS;
  if (uint32_t(first) >= uint32_t(pairs)) return;  // (a tile before the sequence's first: where offsets fall)
  const int off = work.len - n;  // row i sees places 0 .. i + off
  const int room = a.width << a.page_shift;
  const int most_keys = min(off + (min(first + ROWS, pairs) - 1) / group + 1, room);  // what the workgroup's last row sees
  const int begin = chunk * a.chunk;  // this workgroup's keys: [begin, keys)
  if (chunk > 0 && begin >= most_keys) return;
  const int keys = chunk + 1 < a.chunks ? min(most_keys, begin + a.chunk) : most_keys;
  const int parts = a.part ? min(a.chunks, (most_keys - 1) / a.chunk + 1) : 1;  // chunks that the tile's keys take
  const int flat = min(first + 32 * wave + r, pairs - 1), mine = flat / group, sees = min(mine + off + 1, room);
  const int all = min(off + (first + 32 * wave) / group + 1, room);  // what every row of the wavefront sees
  const int all_rows = min(off + first / group + 1, room);           // and of the workgroup

  u32x4 qf[KS];
  {
    const uint16_t *q = a.q + size_t(work.row0 + mine) * a.q_row + size_t(kv * group + flat - mine * group) * a.q_head + 8 * h;
#pragma unroll
    for (int j = 0; j < KS; ++j) qf[j] = *reinterpret_cast<const u32x4 *>(q + 16 * j);
  }
  // pages and scales of the halves of 64 tiles, a tile a lane
  const int tiles = keys > begin ? (keys - begin + BN - 1) / BN : 0;
  int number[2];
  float k_scale[2], v_scale[2];
  auto look_up = [&](int t0) {
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
  const int page_tokens = 1 << a.page_shift;
  u32x4 kr[COPIES], vr[COPIES];
  auto fetch = [&](int t) {  // tile t's codes to registers
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
      const int row0 = (i * 256 + 64 * wave) / (D / 16), x = row0 >> 5;  // (the wavefront's rows of a copy are in one half)
      const int page = x ? __builtin_amdgcn_readlane(number[1], t & 63) : __builtin_amdgcn_readlane(number[0], t & 63);
      const int token = begin + t * BN + 32 * x, rows = page < 0 ? 0 : min(32, max(0, most_keys - token));
      const size_t at = ((size_t(max(page, 0)) * a.heads + kv) * page_tokens + (token & (page_tokens - 1))) * D;
      const int j = i * 256 + tid, voff = (j / (D / 16) & 31) * D + j % (D / 16) * 16;
      kr[i] = load_rows(a.kc + at, rows * D, voff);
      vr[i] = load_rows(a.vc + at, rows * D, voff);
    }
  };
  float ref = BF ? 1.0f : 0.0f;  // float16: values in LDS are in units of it
  // tile t from registers to LDS; the factor that brings the sums to the tile's reference
  auto store = [&](int t, int stage) {
    float vs[2] = {lane_value(v_scale[0], t & 63), lane_value(v_scale[1], t & 63)}, move = 1.0f;
    if constexpr (!BF) {
      const float big = fmaxf(vs[0], vs[1]), small = vs[0] == 0.0f ? vs[1] : vs[1] == 0.0f ? vs[0] : fminf(vs[0], vs[1]);
      if (big > 0.0f && (big > ref * 0x1p7f || small < ref * 0x1p-15f)) {
        const float to = fmaxf(big, 0x1p-40f);  // (2^-40 448 is nothing in float16)
        move = ref == 0.0f ? 1.0f : fminf(ref / to, 0x1p120f);
        ref = to;
      }
      if (ref != 0.0f) vs[0] /= ref, vs[1] /= ref;
    }
    uint8_t *kt = lds + stage * kTileBytes, *vt = lds + (2 + stage) * kTileBytes;
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
      const int j = i * 256 + tid, row = j / (D / 16), c = j % (D / 16);
      const int x = (i * 256 + 64 * wave) / (D / 16) >> 5;
      u32x4 lo, hi;
      widen<BF>(kr[i], 1.0f, lo, hi);
      *reinterpret_cast<u32x4 *>(kt + row * D * 2 + k_chunk<D>(row, 2 * c) * 16) = lo;
      *reinterpret_cast<u32x4 *>(kt + row * D * 2 + k_chunk<D>(row, 2 * c + 1) * 16) = hi;
      widen<BF>(vr[i], vs[x], lo, hi);
      u32x4 *to = reinterpret_cast<u32x4 *>(vt + row * D * 2 + v_pair<D>(row, c) * 32);
      to[0] = lo, to[1] = hi;
    }
    return move;
  };
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
  f32x16 o[DT] = {};
  float m = -INFINITY, l = 0.0f, move = 1.0f;
  if (tiles > 0) {
    look_up(0);
    fetch(0);
    move = store(0, 0);
  }
  for (int t = 0; t < tiles; ++t) {
    const int at = begin + t * BN, stage = t & 1;
    __syncthreads();
    // (never zero: -infinity times that would be NaN)
    const float c[2] = {fmaxf(lane_value(k_scale[0], t & 63) * a.scale, 0x1p-126f), fmaxf(lane_value(k_scale[1], t & 63) * a.scale, 0x1p-126f)};
    const bool hole[2] = {__builtin_amdgcn_readlane(number[0], t & 63) < 0, __builtin_amdgcn_readlane(number[1], t & 63) < 0};
    if (t + 1 < tiles) {
      if (((t + 1) & 63) == 0) look_up(t + 1);
      fetch(t + 1);
    }
    uint8_t *kt = lds + stage * kTileBytes, *vt = lds + (2 + stage) * kTileBytes;
    bool bad = false;
    if (at + BN > all_rows) {
      const bool found = __any(any_bad<D, BF>(vt));
      if (lane == 0) flags[wave] = found;
      __syncthreads();
      bad = __builtin_amdgcn_readfirstlane(flags[0] | flags[1] | flags[2] | flags[3]);
      if (bad) {
        for (int i = tid; i < BN * DT; i += 256) take_bad<D, BF>(vt, i / DT, i % DT, &marks[i], &marks[BN * DT + i]);
        __syncthreads();
      }
    }
    f32x16 s[2] = {};
#pragma unroll
    for (int j = 0; j < KS; ++j)
#pragma unroll
      for (int x = 0; x < 2; ++x) s[x] = mfma32<BF>(k_frag(kt, x, j), qf[j], s[x]);
    if (at + BN > all || hole[0] || hole[1]) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int left = hole[x] ? 0 : sees - at - 4 * h - 32 * x;
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (8 * (e >> 2) + (e & 3) >= left) s[x][e] = -INFINITY;
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float y = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16; ++e) y = fmaxf(y, s[x][e]);
      top = fmaxf(top, y * c[x]);
    }
    top = fmaxf(top, lane_xor32(top));
    if (__any(top > m + kLag<BF>) || move != 1.0f) {
      const float to = fmaxf(m, top), keep = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
      m = to;
      l *= keep;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= keep * move;
    }
    const float lift = m == -INFINITY ? 0.0f : kLift<BF> - m;
    u32x4 p[4];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float u = __builtin_amdgcn_exp2f(fmaf(s[x][2 * e], c[x], lift)), w = __builtin_amdgcn_exp2f(fmaf(s[x][2 * e + 1], c[x], lift));
        p[2 * x + (e >> 2)][e & 3] = pack2<BF>(u, w);
        l = add2<BF>(p[2 * x + (e >> 2)][e & 3], l);
      }
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] = mfma32<BF>(v_frag(vt, d, ks), p[ks], o[d]);
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
    if (t + 1 < tiles) move = store(t + 1, stage ^ 1);
  }
  __syncthreads();
  l += lane_xor32(l);
  const int own = first + 32 * wave;  // the wavefront's first pair
  const bool there = own + r < pairs;
  auto line_of = [&](int f) {  // of a pair [T][q_heads]
    const int row = f / group;
    return size_t(work.row0 + row) * a.q_heads + kv * group + (f - row * group);
  };
  if (a.part) {
    if (there && chunk == 0 && h == 0) a.joins[line_of(own + r)] = parts > 1 ? parts : 0;
    if (parts > 1) {
      float *rows = reinterpret_cast<float *>(lds) + wave * 32 * D;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<f32x4 *>(rows + r * D + ((8 * d + 2 * e + h) ^ (r & 15)) * 4) =
              f32x4{o[d][4 * e] * ref, o[d][4 * e + 1] * ref, o[d][4 * e + 2] * ref, o[d][4 * e + 3] * ref};
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      float *part = a.part + size_t(chunk) * a.T * a.q_heads * (D + 4);
#pragma unroll 4
      for (int i = 0; i < 32 * D / 256; ++i) {
        const int j = i * 64 + lane, row = j / (D / 4), c = j % (D / 4);
        const f32x4 w = *reinterpret_cast<const f32x4 *>(rows + row * D + (c ^ (row & 15)) * 4);
        if (own + row < pairs) *reinterpret_cast<f32x4 *>(part + line_of(own + row) * (D + 4) + c * 4) = w;
      }
      if (there && h == 0) *reinterpret_cast<float2 *>(part + line_of(own + r) * (D + 4) + D) = float2{m, l};
      return;
    }
  }
  const float inv = l == 0.0f ? 0.0f : ref / l;
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
}

// Chunks of keys where the rows alone would leave half of the GPU's places idle (two workgroups a CU, one at width 256): as many
// as fit the places, of 512 keys at least
struct ChunkPlan {
  int chunk, chunks;
  size_t rows, bytes;  // the workspace's sums, and all of it
};
static long long chunk_tiles(int T, int B, int group) { return (long long)T * group / 128 + B; }
static ChunkPlan chunk_plan(int T, int q_heads, int heads, int D, int B, int longest) {
  ChunkPlan p = {1 << 30, 1, 0, 0};
  const long long work = chunk_tiles(T, B, q_heads / heads) * heads, full = D == 256 ? 256 : 512;
  if (work <= 0 || 2 * work > full) return p;
  const int splits = int(full / work);
  long long chunk = ((long long)longest + splits - 1) / splits;
  chunk = (chunk < 512 ? 512 : chunk) + kPromptKeys - 1;
  chunk -= chunk % kPromptKeys;
  const long long chunks = (longest + chunk - 1) / chunk;
  if (chunks <= 1) return p;
  p.chunk = int(chunk);
  p.chunks = int(chunks);
  p.rows = size_t(p.chunks) * T * q_heads * (D + 4) * sizeof(float);
  p.bytes = p.rows + size_t(T) * q_heads * sizeof(int);
  return p;
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
  LMOE_REQUIRE(T >= 0 && B >= 0 && longest > 0, LMOE_ESHAPE, "%s: %d rows of %d sequences of %d tokens", fn, T, B, longest);
  if (T == 0) return 0;
  LMOE_REQUIRE(B > 0, LMOE_ESHAPE, "%s: %d rows of no sequence", fn, T);
  LMOE_REQUIRE(cu || T == B, LMOE_ESHAPE, "%s: %d rows of %d sequences need their offsets", fn, T, B);
  LMOE_REQUIRE(scale > 0.0f && scale < INFINITY, LMOE_EINVAL, "%s: scale %g", fn, double(scale));
  LMOE_REQUIRE(q && out && lens && table && k_codes && k_scale && v_codes && v_scale, LMOE_EINVAL, "%s: null pointer", fn);
  LMOE_REQUIRE(aligned16(q) && aligned16(out) && aligned16(k_codes) && aligned16(v_codes) && q_row % 8 == 0 && q_head % 8 == 0,
               LMOE_EALIGN, "%s: rows and codes must be 16-byte aligned", fn);
  LMOE_REQUIRE((long long)T * q_heads / heads <= 0x7fffff00 && T <= (1 << 30), LMOE_ESHAPE, "%s: %d rows of %d heads a group", fn, T,
               q_heads / heads);
  const ChunkPlan plan = chunk_plan(T, q_heads, heads, D, B, longest);
  const long long tiles = chunk_tiles(T, B, q_heads / heads), groups = tiles * heads * plan.chunks;
  LMOE_REQUIRE(groups <= kMostGroups && ((long long)T * q_heads * (D / 4) + 255) / 256 <= (plan.bytes ? kMostGroups : 1ll << 62),
               LMOE_ESHAPE, "%s: %d rows of %d sequences and %d heads are more than a launch takes", fn, T, B, q_heads);
  LMOE_REQUIRE(plan.bytes == 0 || (workspace && aligned16(workspace) && workspace_bytes >= plan.bytes), LMOE_EWORKSPACE,
               "%s: a 16-byte aligned workspace of %zu bytes is needed", fn, plan.bytes);
  float *part = plan.bytes ? static_cast<float *>(workspace) : nullptr;
  int *joins = plan.bytes ? reinterpret_cast<int *>(static_cast<char *>(workspace) + plan.rows) : nullptr;
  ChunkArgs a = {static_cast<const uint16_t *>(q), q_row, q_head, k_codes, v_codes, k_scale, v_scale, table, lens, cu,
                 static_cast<uint16_t *>(out), part, joins, scale * 1.4426950408889634f, T, B, q_heads, heads, q_heads / heads, pages,
                 width, page == 32 ? 5 : page == 64 ? 6 : 7, int(tiles), plan.chunk, plan.chunks};
  auto go = [&](auto kernel, auto join) -> int {
    const size_t lds = size_t(kPromptKeys) * D * 2 * 4;
    if (const int rc = allow_lds(kernel, lds + 4112, fn)) return rc;  // with what the kernel declares itself
    launch(kernel, dim3(unsigned(groups)), dim3(256), lds, (hipStream_t)stream, a);
    LMOE_LAUNCHED(fn);
    if (part) {
      launch(join, dim3(unsigned(((long long)T * q_heads * (D / 4) + 255) / 256)), dim3(256), 0, (hipStream_t)stream,
             JoinArgs{a.out, part, joins, T, q_heads, plan.chunks});
      LMOE_LAUNCHED(fn);
    }
    return 0;
  };
  const bool bf = dtype == LMOE_BF16;
  if (D == 64) return bf ? go(k_chunk_rows<64, true>, k_join_chunks<64, true>) : go(k_chunk_rows<64, false>, k_join_chunks<64, false>);
  if (D == 128)
    return bf ? go(k_chunk_rows<128, true>, k_join_chunks<128, true>) : go(k_chunk_rows<128, false>, k_join_chunks<128, false>);
  return bf ? go(k_chunk_rows<256, true>, k_join_chunks<256, true>) : go(k_chunk_rows<256, false>, k_join_chunks<256, false>);
}
