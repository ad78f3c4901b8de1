// Rotary positions of the trunk's rows, and the 8-bit paged cache's writer and reader.
//
// Rotation: pair (u, w) of a head's first 2 F channels becomes gain (u cos a - w sin a, w cos a + u sin a), a = position *
// freq[f]. Pairs are (f, f + F), or (2 f, 2 f + 1) where interleaved. The reference rotates its decode rows the same way
// (route_cuda.py:549-591).
//
// The angle is a float64 product reduced to an eighth of a turn in float64: a float32 product is off by 0.06 rad at position
// 1e6. Sine and cosine of what is left are their Taylor series in float32 (remainders below 2e-9 at pi / 4), once a token and
// pair for all heads, in LDS. Everything else is one float32 multiply or add after the other, and one rounding at the end.
//
// Bound by HBM: 8,192 rows of 32 heads of 128 in float16, neighbouring pairs: 23.5 us, 5.7 TB/s. Threads run over a row's
// units, pairs and the channels that stay apart; with divisions for every unit and both kinds in one wavefront it took 29.3,
// and 54 for what takes 32 where a quarter of 256 channels turns. The choice of tensor for each unit (queries or keys) goes
// through 24 bytes of scratch a lane in k_rope<8> and k_append.
//
// The cache: e4m3 codes [page][head][token of the page][width] and one float32 scale for each page and head, of keys and of
// values. The scale is the least power of two (2^-100 at least) that brings the largest finite magnitude of the page's head
// to 448 or less. With a power of two, restating a page when a later token is larger moves exponents and rounds nothing but
// codes that become subnormal, so a page filled token by token holds what one written at once would, up to those. e4m3 has
// no infinity: infinities and NaN become NaN, and stay out of the scale.
//
// Measured: 64 sequences' tokens (32 + 8 heads of 128) 8.8 us, five dependent loads; 9,349 rows of prompts (16 + 4 heads of
// 256) with their rotation 51 us, 3.7 TB/s of 192 MB, on tensors that no cache holds (the same ones again and again: 40);
// reading those pages back in 16 bits 11.5 us, 2.5 TB/s: eight codes a thread, each behind two divisions and a scale's load.
#include "rows.h"

namespace lmoe {

constexpr int kRopeThreads = 256;
constexpr int kMostWidth = 1 << 30;  // channels of a row, counted in ints

struct Rows {  // [T][heads][D] in place, strides in elements; the last axis is dense
  const void *p;
  long long st, sh;
};

// cos and sin of pos * freq (float64 radians)
__device__ __forceinline__ float2 turn(double pos, double freq) {
  const double t = pos * freq * 0.15915494309189535;  // turns
  const double r = t - rint(t);
  const double q = rint(4.0 * r);
  const float x = float((r - 0.25 * q) * 6.283185307179586);  // |x| <= pi / 4
  const float x2 = x * x;
  float s = fmaf(x2, 1.0f / 362880.0f, -1.0f / 5040.0f);
  s = fmaf(x2, s, 1.0f / 120.0f);
  s = fmaf(x2, s, -1.0f / 6.0f);
  s = fmaf(x * x2, s, x);
  float c = fmaf(x2, -1.0f / 3628800.0f, 1.0f / 40320.0f);
  c = fmaf(x2, c, -1.0f / 720.0f);
  c = fmaf(x2, c, 1.0f / 24.0f);
  c = fmaf(x2, c, -0.5f);
  c = fmaf(x2, c, 1.0f);
  const int k = int(q) & 3;  // quarter turns
  const float a = k & 1 ? s : c, b = k & 1 ? c : s;
  return float2{k == 1 || k == 2 ? -a : a, k >= 2 ? -b : b};
}

// Channels [d, d + 8) of a head's row x, rotated where they belong to a pair; cs: the token's cos / sin [F]
__device__ __forceinline__ void rotate8(const void *x, size_t at, int d, int dt, int F, bool inter, const float2 *cs,
                                        float (&o)[8]) {
  float own[8];
  load8(x, at + d, dt, own);
  if (d >= 2 * F) {
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = own[e];
  } else if (inter) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float2 t = cs[(d + e) >> 1];
      o[e] = own[e] * t.x - own[e + 1] * t.y;
      o[e + 1] = own[e + 1] * t.x + own[e] * t.y;
    }
  } else {
    const bool lo = d < F;
    const int f0 = lo ? d : d - F;
    float other[8];
    load8(x, at + (lo ? d + F : d - F), dt, other);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 t = cs[f0 + e];
      o[e] = lo ? own[e] * t.x - other[e] * t.y : own[e] * t.x + other[e] * t.y;
    }
  }
}

struct RopeArgs {
  Rows x, k;             // k: a second tensor of the same rows (append's keys), or null
  void *xo, *ko;         // outputs; xo strided (may be x itself), ko dense
  long long xo_st, xo_sh;
  const void *positions;  // int32 / int64 [T], or null: from cu and lens
  const double *freq;
  const int *cu, *lens;
  float gain;
  int pos64, T, B, heads, k_heads, D, F, inter, dt, tokens, turn_shift, copy_shift;
};

constexpr int kNoRow = -0x7fffffff - 1;  // the position of a row of no sequence

// The positions of rows t0 .. t0 + nt - 1 (nt <= 8) from their sequences, by one wavefront, into place: the first row's
// sequence, then the 64 that follow it in one load
__device__ __forceinline__ void places_of(const RopeArgs &a, int t0, int nt, int *place) {
  const int lane = threadIdx.x & 63;
  if (!a.cu) {
    if (lane < nt) place[lane] = t0 + lane < a.B ? a.lens[t0 + lane] - 1 : kNoRow;
    return;
  }
  auto begins = [](int c, int) { return (long long)c; };
  const int b0 = last_at(a.cu, a.B, t0, begins);
  const int c = a.cu[min(b0 + 1 + lane, a.B)];
  for (int i = 0; i < nt; ++i) {
    const int row = t0 + i, past = __popcll(__ballot(b0 + 1 + lane <= a.B && c <= row));
    const int b = past < 64 ? b0 + past : last_at(a.cu, a.B, row, begins);
    int pos = kNoRow;
    if (b >= 0 && b < a.B) {
      int r0, n;
      seq_rows(a.cu, b, a.T, &r0, &n);
      if (row >= r0 && row < r0 + n) pos = a.lens[b] - n + (row - r0);
    }
    if (lane == 0) place[i] = pos;
  }
}

// One workgroup, `tokens` rows from t0 on: their cos / sin into LDS, then every head of them. A thread takes both sides of its
// pairs, so xo may be x. W 8: eight channels a load; W 1: any widths, strides and alignments.
template <int W>
__device__ __forceinline__ void rope_block(const RopeArgs &a, int t0, float2 *cs) {
  __shared__ int place[8];
  const int nt = min(a.tokens, a.T - t0);
  if (!a.positions) {
    if (threadIdx.x < 64) places_of(a, t0, nt, place);
    __syncthreads();
  }
  for (int i = threadIdx.x; i < nt * a.F; i += kRopeThreads) {
    const int t = i / a.F;
    const double pos = !a.positions ? double(place[t])
                       : a.pos64    ? double(static_cast<const long long *>(a.positions)[t0 + t])
                                    : double(static_cast<const int *>(a.positions)[t0 + t]);
    float2 v = turn(pos, a.freq[i - t * a.F]);
    v.x *= a.gain, v.y *= a.gain;
    cs[i] = v;
  }
  __syncthreads();
  // f(head's input row offset, output row offset, input, output, their row strides, unit, first row, row step) for every unit
  // of `per` a head: threads over a row's units, and over rows where a row has fewer units than there are threads
  auto units = [&](int per, int shift, auto &&f) __attribute__((always_inline)) {
    const int per_t = per * (a.heads + a.k_heads);
    for (int j = threadIdx.x & ((1 << shift) - 1); j < per_t; j += 1 << shift) {
      const int h = j / per, u = j - h * per;
      const bool key = h >= a.heads;
      const int hk = key ? h - a.heads : h;
      const size_t x_row = key ? a.k.st : a.x.st, y_row = key ? size_t(a.k_heads) * a.D : size_t(a.xo_st);
      f(size_t(t0) * x_row + size_t(hk) * (key ? a.k.sh : a.x.sh), size_t(t0) * y_row + size_t(hk) * (key ? (long long)a.D : a.xo_sh),
        key ? a.k.p : a.x.p, key ? a.ko : a.xo, x_row, y_row, u, int(threadIdx.x) >> shift, kRopeThreads >> shift);
    }
  };
  if constexpr (W == 8) {
    if (a.inter)  // four pairs inside a load
      units(a.F / 4, a.turn_shift, [&](size_t from, size_t to, const void *x, void *y, size_t xs, size_t ys, int u, int t, int step) {
        for (; t < nt; t += step) {
          const bool none = !a.positions && place[t] == kNoRow;
          float v[8], o[8];
          load8(x, from + t * xs + u * 8, a.dt, v);
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float2 r = cs[t * a.F + u * 4 + (e >> 1)];
            o[e] = none ? 0.0f : v[e] * r.x - v[e + 1] * r.y;
            o[e + 1] = none ? 0.0f : v[e + 1] * r.x + v[e] * r.y;
          }
          store8(y, to + t * ys + u * 8, a.dt, o);
        }
      });
    else  // a load of either side
      units(a.F / 8, a.turn_shift, [&](size_t from, size_t to, const void *x, void *y, size_t xs, size_t ys, int u, int t, int step) {
        for (; t < nt; t += step) {
          const bool none = !a.positions && place[t] == kNoRow;
          float v[8], w[8], p[8], q[8];
          load8(x, from + t * xs + u * 8, a.dt, v);
          load8(x, from + t * xs + u * 8 + a.F, a.dt, w);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 r = cs[t * a.F + u * 8 + e];
            p[e] = none ? 0.0f : v[e] * r.x - w[e] * r.y;
            q[e] = none ? 0.0f : w[e] * r.x + v[e] * r.y;
          }
          store8(y, to + t * ys + u * 8, a.dt, p);
          store8(y, to + t * ys + u * 8 + a.F, a.dt, q);
        }
      });
    const int wide = a.dt == LMOE_F32 ? 4 : 8;  // channels in 16 bytes
    if (a.D > 2 * a.F)                          // the other channels, four rows' loads at a time
      units((a.D - 2 * a.F) / wide, a.copy_shift, [&](size_t from, size_t to, const void *x, void *y, size_t xs, size_t ys, int u,
                                                      int t, int step) {
        if (x == y && from == to && xs == ys) return;
        const int d = (2 * a.F + u * wide) / wide;
        for (; t < nt; t += 4 * step) {
          u32x4 v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = static_cast<const u32x4 *>(x)[(from + min(t + i * step, nt - 1) * xs) / wide + d];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (t + i * step < nt) {
              const bool none = !a.positions && place[t + i * step] == kNoRow;
              static_cast<u32x4 *>(y)[(to + (t + i * step) * ys) / wide + d] = none ? u32x4{} : v[i];
            }
        }
      });
  } else {
    units(a.D - a.F, a.turn_shift, [&](size_t from, size_t to, const void *x, void *y, size_t xs, size_t ys, int u, int t, int step) {
      for (; t < nt; t += step) {
        if (u < a.F) {
          const int d = a.inter ? 2 * u : u, e = a.inter ? d + 1 : d + a.F;
          const float2 c = cs[t * a.F + u];
          const float v = load_elt(x, from + t * xs + d, a.dt), w = load_elt(x, from + t * xs + e, a.dt);
          store_elt(y, to + t * ys + d, v * c.x - w * c.y, a.dt);
          store_elt(y, to + t * ys + e, w * c.x + v * c.y, a.dt);
        } else {
          const int d = u + a.F;
          store_elt(y, to + t * ys + d, load_elt(x, from + t * xs + d, a.dt), a.dt);
        }
      }
    });
  }
}

template <int W>
__global__ void __launch_bounds__(kRopeThreads) k_rope(RopeArgs a) {
  extern __shared__ float2 cs[];
  rope_block<W>(a, blockIdx.x * a.tokens, cs);
}

// Rows a workgroup, and the threads over a row's units. One row while that gives no more than 1,024 workgroups, then up to
// eight, so that a prompt's cos / sin and sequence search serve more heads.
static void plan_rope(RopeArgs *a, bool wide) {
  a->tokens = a->T <= 1024 ? 1 : a->T >= 8192 ? 8 : (a->T + 1023) / 1024;
  auto shift = [&](int per) {
    int s = 0;
    while (s < 8 && (1 << s) < per * (a->heads + a->k_heads)) ++s;
    return s;
  };
  a->turn_shift = shift(!wide ? a->D - a->F : a->inter ? a->F / 4 : a->F / 8);
  a->copy_shift = shift((a->D - 2 * a->F) / (a->dt == LMOE_F32 ? 4 : 8));
}

static int launch_rope(const char *fn, RopeArgs a, bool wide, hipStream_t st) {
  plan_rope(&a, wide);
  const size_t lds = size_t(a.tokens) * a.F * sizeof(float2);
  const dim3 grid(unsigned((a.T + a.tokens - 1) / a.tokens));
  if (wide)
    launch(k_rope<8>, grid, dim3(kRopeThreads), lds, st, a);
  else
    launch(k_rope<1>, grid, dim3(kRopeThreads), lds, st, a);
  LMOE_LAUNCHED(fn);
  return 0;
}

// Whether rows can be read and written 8 channels at a time
static bool wide_rows(const void *p, long long st, long long sh, int D, int dt) {
  const int step = dt == LMOE_F32 ? 4 : 8;
  return aligned16(p) && st % step == 0 && sh % step == 0 && D % 8 == 0;
}

// ---- the cache -------------------------------------------------------------------------------------------------

struct AppendArgs {
  Rows k, v;
  uint8_t *kc, *vc;
  float *ks, *vs;
  const int *table, *lens, *cu;
  const double *freq;
  float gain;
  int T, B, heads, D, page, pages, width, F, inter, dt;
  int pages_at, tasks;  // the workgroups that write pages: tasks of them from pages_at on; the others rotate rows
};

// the least s >= -100 with m <= 448 2^s
__device__ __forceinline__ float scale_for(float m) {
  const uint32_t u = __float_as_uint(m);
  // m = (1 + f) 2^e with 448 = 1.75 2^8
  const int e = int(u >> 23) - 127, s = e - 8 + ((u & 0x7fffffu) > 0x600000u);
  return __uint_as_float(uint32_t(max(s, -100) + 127) << 23);
}

// four floats to e4m3 (nearest even; the values are within 448)
__device__ __forceinline__ uint32_t to_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}
// e4m3 codes 0, 1 (HI: 2, 3) of a word as floats
template <bool HI>
__device__ __forceinline__ float2 from_e4m3(uint32_t w) {
  const auto v = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), HI);
  return float2{v[0], v[1]};
}
__device__ __forceinline__ float finite_or_nan(float v) {
  return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u ? __uint_as_float(0x7fc00000u) : v;
}

// One workgroup: the new tokens of one page's head, of keys (rotated) or of values. Page task t of the call: sequence b's
// tasks begin at cu[b] / page + 2 b, which leaves it room for every page that its rows can touch, so no task list is made.
// NV: groups of 8 channels a thread (page * D / 2048). The workgroups that rotate queries share the launch.
template <int NV>
__global__ void __launch_bounds__(256) k_append(AppendArgs a, RopeArgs rope_rows) {
  extern __shared__ float2 cs[];
  __shared__ float top[4];
  const int block = int(blockIdx.x) - a.pages_at;
  if (block < 0 || block >= a.tasks) {
    rope_block<8>(rope_rows, (block < 0 ? int(blockIdx.x) : block - a.tasks) * rope_rows.tokens, cs);
    return;
  }
  const int task = block / (2 * a.heads), head = (block >> 1) % a.heads;
  const bool key = !(block & 1);
  const int page = a.page;
  int b;
  if (a.cu)
    b = last_at(a.cu, a.B, task, [page](int c, int i) { return (long long)(c / page) + 2ll * i; });
  else
    b = task;
  if (b < 0) return;
  int row0, n;
  seq_rows(a.cu, b, a.T, &row0, &n);
  if (n == 0) return;
  const int start = a.lens[b] - n;  // the first new token's place
  const int nth = a.cu ? task - (row0 / page + 2 * b) : 0;
  if (nth < 0) return;  // (where offsets fall)
  const int p = max(start, 0) / page + nth;
  const int lo = max(start, p * page), hi = min(start + n, (p + 1) * page);
  if (hi <= lo || p >= a.width) return;
  const int number = a.table[size_t(b) * a.width + p];
  if (number < 0 || number >= a.pages) return;
  const int base = p * page, rope = key ? a.F : 0;
  for (int i = threadIdx.x; i < (hi - lo) * rope; i += 256) {
    const int t = i / rope;
    float2 c = turn(double(lo + t), a.freq[i - t * rope]);
    c.x *= a.gain, c.y *= a.gain;
    cs[i] = c;
  }
  __syncthreads();
  const Rows src = key ? a.k : a.v;
  const int per = a.D >> 3;
  float x[NV][8];
  float most = 0.0f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int i = threadIdx.x + 256 * j, t = base + i / per, d = (i % per) * 8;
    if (t >= lo && t < hi) {
      const size_t at = size_t(row0 + t - start) * src.st + size_t(head) * src.sh;
      rotate8(src.p, at, d, a.dt, rope, a.inter, cs + (t - lo) * rope, x[j]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[j][e] = finite_or_nan(x[j][e]);
        most = fmaxf(most, fabsf(x[j][e]));  // passes over NaN
      }
    }
  }
  most = wave_max(most);
  if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = most;
  __syncthreads();
  most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
  float *scale = (key ? a.ks : a.vs) + size_t(number) * a.heads + head;
  uint8_t *codes = (key ? a.kc : a.vc) + (size_t(number) * a.heads + head) * size_t(page) * a.D;
  const bool held = lo > base;
  const float old = held ? *scale : 0.0f, now = fmaxf(old, scale_for(most)), inv = 1.0f / now, ratio = old / now;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int i = threadIdx.x + 256 * j, t = base + i / per;
    u32x2 *at = reinterpret_cast<u32x2 *>(codes + size_t(i) * 8);
    if (t >= lo && t < hi) {
      const float *f = x[j];
      *at = u32x2{to_e4m3(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv),
                  to_e4m3(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv)};
    } else if (t < lo && ratio != 1.0f) {  // a page that held tokens and whose scale grows
      u32x2 w = *at;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 u = from_e4m3<false>(w[h]), v = from_e4m3<true>(w[h]);
        w[h] = to_e4m3(u.x * ratio, u.y * ratio, v.x * ratio, v.y * ratio);
      }
      *at = w;
    }
  }
  __syncthreads();  // every thread has read the old scale
  if (threadIdx.x == 0) *scale = now;
}

struct ReadArgs {
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int *table, *cu;
  void *ko, *vo;
  int total, B, heads, D, page, pages, width, dt;
};

constexpr int kReadRows = 16;

// 16 rows of keys (blockIdx.y 0) or values, all heads: codes times scale, one rounding; rows whose page the table does not
// have, or of no sequence, are zero
__global__ void __launch_bounds__(256) k_read(ReadArgs a) {
  __shared__ int page_of[kReadRows], place[kReadRows];
  const int r0 = blockIdx.x * kReadRows, nr = min(kReadRows, a.total - r0);
  for (int i = threadIdx.x >> 6; i < nr; i += 4) {
    const int row = r0 + i, b = last_at(a.cu, a.B, row, [](int c, int) { return (long long)c; });
    int number = -1, at = 0;
    if (b >= 0) {
      int s0, n;
      seq_rows(a.cu, b, a.total, &s0, &n);
      at = row - s0;
      if (at >= 0 && at < n && at / a.page < a.width) number = a.table[size_t(b) * a.width + at / a.page];
      if (number >= a.pages) number = -1;
    }
    if ((threadIdx.x & 63) == 0) page_of[i] = number, place[i] = at % a.page;
  }
  __syncthreads();
  const bool key = blockIdx.y == 0;
  const uint8_t *codes = key ? a.kc : a.vc;
  const float *scales = key ? a.ks : a.vs;
  void *out = key ? a.ko : a.vo;
  const int per = a.D >> 3, per_r = per * a.heads;
  for (int i = threadIdx.x; i < nr * per_r; i += 256) {
    const int r = i / per_r, j = i - r * per_r, h = j / per, d = (j - h * per) * 8;
    const int number = page_of[r];
    float o[8] = {};
    if (number >= 0) {
      const size_t head = size_t(number) * a.heads + h;
      const float s = scales[head];
      const u32x2 w = *reinterpret_cast<const u32x2 *>(codes + (head * a.page + place[r]) * a.D + d);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const float2 u = from_e4m3<false>(w[q]), v = from_e4m3<true>(w[q]);
        o[4 * q] = u.x * s, o[4 * q + 1] = u.y * s, o[4 * q + 2] = v.x * s, o[4 * q + 3] = v.y * s;
      }
    }
    store8(out, (size_t(r0 + r) * a.heads + h) * a.D + d, a.dt, o);
  }
}

}  // namespace lmoe

using namespace lmoe;

extern "C" int lmoe_rope_rows(const void *x, int dtype, long long x_row, long long x_head, const void *positions,
                              int positions64, const double *freq, int n_freq, int T, int heads, int D, int interleaved,
                              float gain, void *out, long long out_row, long long out_head, void *stream) {
  const char *fn = "lmoe_rope_rows";
  LMOE_REQUIRE(dtype_ok(dtype), LMOE_EINVAL, "%s: dtype %d", fn, dtype);
  LMOE_REQUIRE(T >= 0 && heads > 0 && D > 0 && D <= 1024 && heads <= kMostWidth / D, LMOE_ESHAPE, "%s: %d rows of %d heads of %d", fn,
               T, heads, D);
  LMOE_REQUIRE(n_freq >= 0 && 2 * n_freq <= D, LMOE_ESHAPE, "%s: %d pairs in heads of %d", fn, n_freq, D);
  LMOE_REQUIRE((T + 7ll) / 8 <= kMostGroups, LMOE_ESHAPE, "%s: %d rows are more than a launch takes", fn, T);
  if (T == 0) return 0;
  LMOE_REQUIRE(x && out && positions && (freq || n_freq == 0), LMOE_EINVAL, "%s: null pointer", fn);
  const bool wide = wide_rows(x, x_row, x_head, D, dtype) && wide_rows(out, out_row, out_head, D, dtype) &&
                    (interleaved ? n_freq % 4 == 0 : n_freq % 8 == 0);
  RopeArgs a = {};
  a.x = {x, x_row, x_head};
  a.xo = out, a.xo_st = out_row, a.xo_sh = out_head;
  a.positions = positions, a.pos64 = positions64, a.freq = freq, a.gain = gain;
  a.T = T, a.heads = heads, a.D = D, a.F = n_freq, a.inter = interleaved, a.dt = dtype;
  return launch_rope(fn, a, wide, (hipStream_t)stream);
}

static int check_cache(const char *fn, int heads, int D, int page, int pages, int width) {
  LMOE_REQUIRE(D == 64 || D == 128 || D == 256, LMOE_ESHAPE, "%s: heads of %d channels (64, 128 and 256 are served)", fn, D);
  LMOE_REQUIRE(page == 32 || page == 64 || page == 128, LMOE_ESHAPE, "%s: pages of %d tokens (32, 64 and 128 are served)", fn,
               page);
  // a page's end is an int
  LMOE_REQUIRE(heads > 0 && heads <= 65535 && pages > 0 && width > 0 && width <= 0x7fffffff / page, LMOE_ESHAPE,
               "%s: %d heads, %d pages, a table of %d", fn, heads, pages, width);
  return 0;
}

extern "C" int lmoe_kv_append(const void *q, long long q_row, long long q_head, int q_heads, const void *k, long long k_row,
                              long long k_head, const void *v, long long v_row, long long v_head, int dtype, int T, int heads,
                              int D, const int *cu, const int *lens, int B, const int *table, int width, uint8_t *k_codes,
                              float *k_scale, uint8_t *v_codes, float *v_scale, int pages, int page, const double *freq,
                              int n_freq, int interleaved, float gain, void *q_out, void *k_out, void *stream) {
  const char *fn = "lmoe_kv_append";
  LMOE_REQUIRE(dtype_ok(dtype), LMOE_EINVAL, "%s: dtype %d", fn, dtype);
  LMOE_REQUIRE(T >= 0 && B >= 0 && (!q || q_heads > 0), LMOE_ESHAPE, "%s: %d rows, %d sequences, %d query heads", fn, T, B,
               q_heads);
  if (const int rc = check_cache(fn, heads, D, page, pages, width)) return rc;
  LMOE_REQUIRE(!q || q_heads <= kMostWidth / D - heads, LMOE_ESHAPE, "%s: %d query heads of %d", fn, q_heads, D);
  LMOE_REQUIRE(n_freq >= 0 && 2 * n_freq <= D && (interleaved ? n_freq % 4 == 0 : n_freq % 8 == 0), LMOE_ESHAPE,
               "%s: %d pairs in heads of %d (multiples of 8, of 4 where interleaved)", fn, n_freq, D);
  if (T == 0 || B == 0) return 0;
  LMOE_REQUIRE(k && v && lens && table && k_codes && k_scale && v_codes && v_scale && (freq || n_freq == 0) && (!q || q_out),
               LMOE_EINVAL, "%s: null pointer", fn);
  LMOE_REQUIRE(cu || T == B, LMOE_ESHAPE, "%s: %d rows of %d sequences need their offsets", fn, T, B);
  LMOE_REQUIRE((!q || wide_rows(q, q_row, q_head, D, dtype)) && wide_rows(k, k_row, k_head, D, dtype) &&
                   wide_rows(v, v_row, v_head, D, dtype) && aligned16(k_codes) && aligned16(v_codes),
               LMOE_EALIGN, "%s: rows and codes must be 16-byte aligned", fn);
  hipStream_t st = (hipStream_t)stream;
  const long long tasks = (cu ? T / page + 2ll * B : B) * heads * 2;
  LMOE_REQUIRE(tasks + 1024 + T / 8 <= kMostGroups, LMOE_ESHAPE,
               "%s: %d rows of %d sequences and %d heads are more than a launch takes", fn, T, B, heads);
  AppendArgs a = {{k, k_row, k_head}, {v, v_row, v_head}, k_codes, v_codes, k_scale, v_scale, table, lens, cu, freq, gain,
                  T, B, heads, D, page, pages, width, n_freq, interleaved, dtype, 0, int(tasks)};
  RopeArgs r = {};
  r.x = {q, q_row, q_head};
  r.k = {k, k_row, k_head};
  r.xo = q_out, r.xo_st = (long long)q_heads * D, r.xo_sh = D, r.ko = k_out;
  r.freq = freq, r.cu = cu, r.lens = lens, r.gain = gain;
  r.T = T, r.B = B, r.heads = q ? q_heads : 0, r.k_heads = k_out ? heads : 0, r.D = D, r.F = n_freq, r.inter = interleaved;
  r.dt = dtype;
  const bool rows = q || k_out;
  plan_rope(&r, true);
  // One launch: the rotation hides the latency of the pages' few workgroups (prompts at width 256: 18 + 33 us apart, 46
  // together), and a token's call saves a launch. Pages go first where there are many rows, so that their chain of loads is
  // not what the launch ends with. Apart only where a page's registers would leave the rotation two wavefronts a SIMD.
  // A page's cos / sin in LDS can bound it as well, which the rule does not look at: whole heads of 128 on pages of 128 (or of
  // 256 on 64) take 64 KiB a workgroup, two a CU.
  const bool together = rows && (T <= 1024 || page * D <= 16384);
  const int rotating = together ? (T + r.tokens - 1) / r.tokens : 0;
  a.pages_at = T <= 1024 ? rotating : 0;
  const size_t lds = size_t(max(cu ? page : 1, r.tokens)) * n_freq * sizeof(float2);
  const unsigned grid = unsigned(tasks + rotating);
  auto go = [&](auto kernel) -> int {
    if (const int rc = allow_lds(kernel, lds + 256, fn)) return rc;  // with what the kernel declares itself
    launch(kernel, dim3(grid), dim3(256), lds, st, a, r);
    LMOE_LAUNCHED(fn);
    return 0;
  };
  int rc;
  switch (page * D / 2048) {
    case 1: rc = go(k_append<1>); break;
    case 2: rc = go(k_append<2>); break;
    case 4: rc = go(k_append<4>); break;
    case 8: rc = go(k_append<8>); break;
    default: rc = go(k_append<16>); break;
  }
  return rc || !rows || together ? rc : launch_rope(fn, r, true, st);
}

extern "C" int lmoe_kv_read(const uint8_t *k_codes, const float *k_scale, const uint8_t *v_codes, const float *v_scale, int pages,
                            int page, int heads, int D, const int *table, int width, const int *cu, int B, int total,
                            void *k_out, void *v_out, int dtype, void *stream) {
  const char *fn = "lmoe_kv_read";
  LMOE_REQUIRE(dtype_ok(dtype), LMOE_EINVAL, "%s: dtype %d", fn, dtype);
  LMOE_REQUIRE(total >= 0 && B >= 0, LMOE_ESHAPE, "%s: %d rows, %d sequences", fn, total, B);
  if (const int rc = check_cache(fn, heads, D, page, pages, width)) return rc;
  LMOE_REQUIRE((total + kReadRows - 1ll) / kReadRows <= kMostGroups, LMOE_ESHAPE, "%s: %d rows are more than a launch takes", fn,
               total);
  if (total == 0) return 0;
  LMOE_REQUIRE(k_codes && k_scale && v_codes && v_scale && (table || B == 0) && (cu || B == 0) && k_out && v_out, LMOE_EINVAL,
               "%s: null pointer", fn);
  LMOE_REQUIRE(aligned16(k_codes) && aligned16(v_codes) && aligned16(k_out) && aligned16(v_out), LMOE_EALIGN,
               "%s: codes and rows must be 16-byte aligned", fn);
  ReadArgs a = {k_codes, v_codes, k_scale, v_scale, table, cu, k_out, v_out, total, B, heads, D, page, pages, width, dtype};
  launch(k_read, dim3(unsigned((total + kReadRows - 1) / kReadRows), 2), dim3(256), 0, (hipStream_t)stream, a);
  LMOE_LAUNCHED(fn);
  return 0;
}
