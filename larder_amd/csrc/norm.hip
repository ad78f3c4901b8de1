// Root-mean-square norm of rows, with the residual's addition before it and, where asked, an output in 8 bits with scales.
//
//   s = x + residual, y = s / sqrt(mean(s^2) + eps) * weight;  codes: c = e4m3(y / scale), scale the least power of two (2^-100
//   at least) that brings the group's largest finite |y| to 448 or less
//
// Bound by HBM: each input is read once and each output written once; a row stays in registers between the sum of squares and
// the product. float32 inside: y is of the sum before that is rounded, one rounding each for y (or its code) and for s.
//
// A row is taken by `lanes` neighbouring threads, eight channels a thread and step: 8 to 64 lanes of a wavefront (up to 512
// channels, 1,536 where rows are many; several rows a workgroup), or a workgroup of 256 (up to 16,384 in registers, longer ones
// read twice, the second time from L2). Measured: 8,192 rows of 4,096 in bf16 with their residual 53.9 us, 5.0 TB/s (with
// codes 50, read back 20); 2,048 rows of 32 heads of 128 7.9; one row 2.8 of kernel under 9 of the call; 4,000 rows of an
// odd 5,001 3.6 TB/s, 2,000 of 20,000 3.1. Rows may begin anywhere: loads and stores are of 16 bytes whatever their alignment (the
// hardware splits what crosses a line), and the last, partial eight go one by one.
#include "codes.h"

namespace lmoe {

struct NormArgs {
  const void *x, *residual, *weight;
  void *out, *sum;
  float *scales;
  long long x_row, x_head, r_row, r_head, s_row, s_head;  // elements
  long long rows;
  float eps;
  int heads, H, wdt, group;  // group: channels a scale, 0 for no codes
};

// f(0), f(1), ...: N of them unrolled, or `steps` in a loop where N is 0
template <int N, typename F>
__device__ __forceinline__ void for_steps(int steps, F &&f) {
  if constexpr (N) {
#pragma unroll
    for (int i = 0; i < N; ++i) f(i);
  } else {
    for (int i = 0; i < steps; ++i) f(i);
  }
}

__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  typedef float f2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{a, b}, b2));
}

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));

// n (8, or fewer at a row's end) neighbouring elements from any address; zeros behind them
template <int DT>
__device__ __forceinline__ void load_any(const void *p, long long i, int n, float (&v)[8]) {
  if (n >= 8) {
    if constexpr (DT == LMOE_F32) {
      const u32x4_any *q = reinterpret_cast<const u32x4_any *>(static_cast<const float *>(p) + i);
      const u32x4_any a = q[0], b = q[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(a[e]), v[4 + e] = __uint_as_float(b[e]);
    } else {
      const u32x4_any w = *reinterpret_cast<const u32x4_any *>(static_cast<const uint16_t *>(p) + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (DT == LMOE_F16) {
          const h2_t h = __builtin_bit_cast(h2_t, uint32_t(w[e]));
          v[2 * e] = float(h[0]), v[2 * e + 1] = float(h[1]);
        } else {
          v[2 * e] = __uint_as_float(w[e] << 16), v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        }
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? load_elt(p, size_t(i + e), DT) : 0.0f;
  }
}

template <int DT>
__device__ __forceinline__ void store_any(void *p, long long i, int n, const float (&v)[8]) {
  if (n >= 8) {
    if constexpr (DT == LMOE_F32) {
      u32x4_any *q = reinterpret_cast<u32x4_any *>(static_cast<float *>(p) + i);
      q[0] = u32x4_any{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
      q[1] = u32x4_any{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])};
    } else {
      u32x4_any w;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = DT == LMOE_F16 ? __builtin_bit_cast(uint32_t, h2_t{_Float16(v[2 * e]), _Float16(v[2 * e + 1])})
                              : bf16_pair(v[2 * e], v[2 * e + 1]);
      *reinterpret_cast<u32x4_any *>(static_cast<uint16_t *>(p) + i) = w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) store_elt(p, size_t(i + e), v[e], DT);
  }
}

// sums and maxima over a row's L lanes (256: a workgroup's four wavefronts, through LDS)
template <int L>
__device__ __forceinline__ float row_sum(float v, float *lds) {
  if constexpr (L == 8) return sum8(v);
  v = sum16(v);
  if constexpr (L == 16) return v;
  v += lane_xor16(v);
  if constexpr (L == 32) return v;
  v += lane_xor32(v);
  if constexpr (L == 64) return v;
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}
// maxima over aligned groups of 4, 8, 16, 32 or 64 lanes
__device__ __forceinline__ float lanes_max(float v, int lanes) {
  v = fmaxf(v, LMOE_DPP(v, kDppXor1));
  v = fmaxf(v, LMOE_DPP(v, kDppXor2));
  if (lanes >= 8) v = fmaxf(v, LMOE_DPP(v, kDppHalfMirror));
  if (lanes >= 16) v = fmaxf(v, LMOE_DPP(v, kDppMirror));
  if (lanes >= 32) v = fmaxf(v, lane_xor16(v));
  if (lanes >= 64) v = fmaxf(v, lane_xor32(v));
  return v;
}

// Where squares overflow: rows are scaled by kDown^2 for their sum (2^128 of the largest becomes 2^48, its square 2^96). A channel is
// brought back by one kDown with its division and one after it, so that what is small beside large ones is not rounded on the way
constexpr float kDown = 0x1p-40f;

// N steps of eight channels a lane in registers; N = 0: rows of any length, read twice
template <int DT, int L, int N>
__global__ void __launch_bounds__(256) k_norm(NormArgs a) {
  __shared__ float lds[12];
  constexpr int kRows = 256 / L, kHeld = N ? N : 1;
  const int lane = threadIdx.x % L;
  const long long row = (long long)blockIdx.x * kRows + threadIdx.x / L;
  const bool there = row < a.rows;
  const long long at = there ? row : a.rows - 1, t = at / a.heads;
  const int head = int(at - t * a.heads), chunks = (a.H + 7) >> 3;
  const long long xi = t * a.x_row + head * a.x_head, ri = t * a.r_row + head * a.r_head, si = t * a.s_row + head * a.s_head;
  const int steps = N ? N : (chunks + L - 1) / L;
  float v[kHeld][8];
  auto load = [&](int i, float (&u)[8]) {
    const int c = i * L + lane, n = a.H - 8 * c;
    if (n <= 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] = 0.0f;
      return;
    }
    load_any<DT>(a.x, xi + 8 * c, n, u);
    if (a.residual) {
      float r[8];
      load_any<DT>(a.residual, ri + 8 * c, n, r);
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] += r[e];
    }
  };
  auto squares = [&](float down) {
    float ss = 0.0f;
    auto add = [&](const float (&u)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = u[e] * down;
        ss = fmaf(d, d, ss);
      }
    };
    if constexpr (N) {
#pragma unroll
      for (int i = 0; i < N; ++i) add(v[i]);
    } else {
      for (int i = 0; i < steps; ++i) {
        float u[8];
        load(i, u);
        add(u);
      }
    }
    return ss;
  };
  if constexpr (N) {
#pragma unroll
    for (int i = 0; i < N; ++i) load(i, v[i]);
  }
  const float ss = row_sum<L>(squares(1.0f), lds);
  float inv = 1.0f / sqrtf(ss / float(a.H) + a.eps), down = 1.0f;
  if (__any(!(ss < INFINITY))) {  // (for a row in four wavefronts: all of them or none)
    constexpr float kSquares = kDown * kDown;
    const float low = row_sum<L>(squares(kSquares), lds + 4);
    if (!(ss < INFINITY)) inv = kDown / sqrtf(low / float(a.H) + a.eps * kSquares * kSquares), down = kDown;
  }
  auto divide = [&](float (&u)[8], const float (&w)[8]) {
    if (down == 1.0f) {
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] = u[e] * inv * w[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {  // below 1 no weight overflows; from 1 on nothing is subnormal before its weight
        const float y = u[e] * inv;
        u[e] = fabsf(y) < 1.0f ? y * w[e] * down : y * down * w[e];
      }
    }
  };
  auto normed = [&](int i, float (&u)[8]) {  // the step's y from its sums; the sums are written
    const int c = i * L + lane, n = a.H - 8 * c;
    if (n <= 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] = 0.0f;
      return;
    }
    if (a.sum && there) store_any<DT>(a.sum, si + 8 * c, n, u);
    float w[8];
    if (a.wdt == DT)
      load_any<DT>(a.weight, 8 * c, n, w);
    else
      load_any<LMOE_F32>(a.weight, 8 * c, n, w);
    divide(u, w);
  };
  if (!a.group) {
    for_steps<N>(steps, [&](int i) {
      float u[8];
      if constexpr (N) {
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = v[i][e];
      } else {
        load(i, u);
      }
      normed(i, u);
      const int c = i * L + lane;
      if (there && 8 * c < a.H) store_any<DT>(a.out, row * a.H + 8 * c, a.H - 8 * c, u);
    });
    return;
  }
  // Codes. One scale a row needs all of its y first: kept in the registers that held the sums, or (rows read twice) worked
  // out once more; the sums are written in the pass that loads them last.
  auto finite = [&](float (&u)[8]) {
    float most = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] = finite_or_nan(u[e]), most = fmaxf(most, fabsf(u[e]));  // passes over NaN
    return most;
  };
  auto write = [&](int i, const float (&u)[8], float inv_scale) {
    const int c = i * L + lane, n = a.H - 8 * c;
    if (!there || n <= 0) return;
    const float *f = u;
    const uint32_t lo = to_e4m3(f[0] * inv_scale, f[1] * inv_scale, f[2] * inv_scale, f[3] * inv_scale);
    const uint32_t hi = to_e4m3(f[4] * inv_scale, f[5] * inv_scale, f[6] * inv_scale, f[7] * inv_scale);
    uint8_t *p = static_cast<uint8_t *>(a.out) + row * a.H + 8 * c;
    if (n >= 8) {
      *reinterpret_cast<u32x2_any *>(p) = u32x2_any{lo, hi};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) p[e] = uint8_t((e < 4 ? lo : hi) >> (8 * (e & 3)));
    }
  };
  if (a.group < a.H) {  // groups of 32 to 512 channels: aligned runs of 4 to 64 lanes
    for_steps<N>(steps, [&](int i) {
      float u[8];
      if constexpr (N) {
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = v[i][e];
      } else {
        load(i, u);
      }
      normed(i, u);
      const float scale = scale_for(lanes_max(finite(u), a.group >> 3));
      const int c = i * L + lane;
      if (there && 8 * c < a.H && (8 * c) % a.group == 0) a.scales[(row * a.H + 8 * c) / a.group] = scale;
      write(i, u, 1.0f / scale);
    });
    return;
  }
  float most = 0.0f;
  if constexpr (N) {
#pragma unroll
    for (int i = 0; i < N; ++i) normed(i, v[i]), most = fmaxf(most, finite(v[i]));
  } else {
    for (int i = 0; i < steps; ++i) {
      const int c = i * L + lane, n = a.H - 8 * c;
      if (n <= 0) continue;
      float u[8], w[8];
      load(i, u);
      if (a.wdt == DT)
        load_any<DT>(a.weight, 8 * c, n, w);
      else
        load_any<LMOE_F32>(a.weight, 8 * c, n, w);
      divide(u, w);
      most = fmaxf(most, finite(u));
    }
  }
  most = lanes_max(most, min(L, 64));
  if constexpr (L == 256) {
    if ((threadIdx.x & 63) == 0) lds[8 + (threadIdx.x >> 6)] = most;
    __syncthreads();
    most = fmaxf(fmaxf(lds[8], lds[9]), fmaxf(lds[10], lds[11]));
  }
  const float scale = scale_for(most), inv_scale = 1.0f / scale;
  if (there && lane == 0) a.scales[row] = scale;
  for_steps<N>(steps, [&](int i) {
    if constexpr (N) {
      write(i, v[i], inv_scale);
    } else {
      float u[8];
      load(i, u);
      normed(i, u);
      finite(u);
      write(i, u, inv_scale);
    }
  });
}

struct CodesArgs {
  const uint8_t *codes;
  const float *scales;
  void *out;
  long long n;
  int group, dt;
};

// Eight codes a thread. A row holds a whole number of groups, so the scale of element i is i / group, whatever the rows.
__global__ void __launch_bounds__(256) k_read_codes(CodesArgs a) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 8;
  if (i >= a.n) return;
  float v[8];
  const int n = int(min(8ll, a.n - i));
  uint32_t w[2] = {0, 0};
  if (n == 8) {
    const u32x2 g = *reinterpret_cast<const u32x2 *>(a.codes + i);
    w[0] = g.x, w[1] = g.y;
  } else {
    for (int e = 0; e < n; ++e) w[e >> 2] |= uint32_t(a.codes[i + e]) << (8 * (e & 3));
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float2 lo = from_e4m3<false>(w[h]), hi = from_e4m3<true>(w[h]);
    v[4 * h] = lo.x, v[4 * h + 1] = lo.y, v[4 * h + 2] = hi.x, v[4 * h + 3] = hi.y;
  }
  if (a.group % 8 == 0) {
    const float s = a.scales[i / a.group];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= s;
  } else {
    long long g = i / a.group;
    int left = int(a.group - (i - g * a.group));
    float s = a.scales[g];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (e >= n) break;
      if (left == 0) left = a.group, s = a.scales[++g];
      v[e] *= s;
      --left;
    }
  }
  if (n == 8) {
    store8(a.out, size_t(i), a.dt, v);
  } else {
    for (int e = 0; e < n; ++e) store_elt(a.out, size_t(i + e), v[e], a.dt);
  }
}

template <int DT>
static int go_norm(const char *fn, const NormArgs &a, hipStream_t st) {
  const int chunks = (a.H + 7) / 8;
  // A wavefront a row where there are many that would leave a quarter or more of a workgroup's threads without channels (16,000
  // rows of 513, bf16, residual: 21.5 -> 16.3 us; 8,000 of 1,111: 26.4 -> 23.3; 16,384 of 2,048 lose, 45 -> 55). Few rows take a
  // workgroup each, for latency
  const bool many = a.rows >= 2048 && chunks <= 192;
  const int lanes = chunks <= 8 ? 8 : chunks <= 16 ? 16 : chunks <= 32 ? 32 : chunks <= 64 || many ? 64 : 256;
  const long long groups = (a.rows + 256 / lanes - 1) / (256 / lanes);
  LMOE_REQUIRE(groups <= (1ll << 24) - 1, LMOE_ESHAPE, "%s: %lld rows are more than a launch takes", fn, a.rows);
  auto go = [&](auto kernel) -> int {
    launch(kernel, dim3(unsigned(groups)), dim3(256), 0, st, a);
    LMOE_LAUNCHED(fn);
    return 0;
  };
  switch (lanes) {
    case 8: return go(k_norm<DT, 8, 1>);
    case 16: return go(k_norm<DT, 16, 1>);
    case 32: return go(k_norm<DT, 32, 1>);
    case 64: return chunks <= 64 ? go(k_norm<DT, 64, 1>) : chunks <= 128 ? go(k_norm<DT, 64, 2>) : go(k_norm<DT, 64, 3>);
  }
  const int steps = (chunks + 255) / 256;
  return steps == 1   ? go(k_norm<DT, 256, 1>)
         : steps == 2 ? go(k_norm<DT, 256, 2>)
         : steps <= 4 ? go(k_norm<DT, 256, 4>)
         : steps <= 8 ? go(k_norm<DT, 256, 8>)
                      : go(k_norm<DT, 256, 0>);
}

}  // namespace lmoe

using namespace lmoe;

extern "C" int lmoe_norm_rows(const void *x, int dtype, long long x_row, long long x_head, const void *residual, long long r_row,
                              long long r_head, const void *weight, int wdtype, long long T, int heads, int H, float eps, void *out,
                              int group, float *scales, void *sum, long long s_row, long long s_head, void *stream) {
  const char *fn = "lmoe_norm_rows";
  LMOE_REQUIRE(dtype_ok(dtype) && (wdtype == dtype || wdtype == LMOE_F32), LMOE_EINVAL,
               "%s: dtype %d with weights of %d (the rows' type or float32)", fn, dtype, wdtype);
  LMOE_REQUIRE(T >= 0 && heads >= 0 && H > 0 && H <= (1 << 30), LMOE_ESHAPE, "%s: %lld rows of %d heads of %d channels", fn, T,
               heads, H);
  LMOE_REQUIRE(eps > 0.0f && eps < INFINITY, LMOE_EINVAL, "%s: eps %g", fn, double(eps));
  LMOE_REQUIRE(group == 0 || group == H ||
                   ((group == 32 || group == 64 || group == 128 || group == 256 || group == 512) && H % group == 0),
               LMOE_ESHAPE, "%s: scales of %d channels in rows of %d (32, 64, 128, 256 or 512 that divide them, or whole rows)", fn,
               group, H);
  LMOE_REQUIRE(heads == 0 || T <= (1ll << 62) / heads, LMOE_ESHAPE, "%s: %lld rows of %d heads", fn, T, heads);
  if (T == 0 || heads == 0) return 0;
  LMOE_REQUIRE(x && weight && out && (scales || group == 0), LMOE_EINVAL, "%s: null pointer", fn);
  NormArgs a = {x, residual, weight, out, sum, scales, x_row, x_head, r_row, r_head, s_row, s_head, T * heads, eps, heads, H, wdtype,
                group};
  hipStream_t st = (hipStream_t)stream;
  return dtype == LMOE_F32 ? go_norm<LMOE_F32>(fn, a, st) : dtype == LMOE_F16 ? go_norm<LMOE_F16>(fn, a, st)
                                                                             : go_norm<LMOE_BF16>(fn, a, st);
}

extern "C" int lmoe_read_codes(const uint8_t *codes, const float *scales, long long n, int group, void *out, int dtype,
                               void *stream) {
  const char *fn = "lmoe_read_codes";
  LMOE_REQUIRE(dtype_ok(dtype), LMOE_EINVAL, "%s: dtype %d", fn, dtype);
  LMOE_REQUIRE(n >= 0 && group > 0 && n % group == 0, LMOE_ESHAPE, "%s: %lld codes in groups of %d", fn, n, group);
  LMOE_REQUIRE((n + 2047) / 2048 <= (1ll << 24) - 1, LMOE_ESHAPE, "%s: %lld codes are more than a launch takes", fn, n);
  if (n == 0) return 0;
  LMOE_REQUIRE(codes && scales && out, LMOE_EINVAL, "%s: null pointer", fn);
  LMOE_REQUIRE(aligned16(codes) && aligned16(out), LMOE_EALIGN, "%s: codes and rows must be 16-byte aligned", fn);
  launch(k_read_codes, dim3(unsigned((n + 2047) / 2048)), dim3(256), 0, (hipStream_t)stream, CodesArgs{codes, scales, out, n, group, dtype});
  LMOE_LAUNCHED(fn);
  return 0;
}
