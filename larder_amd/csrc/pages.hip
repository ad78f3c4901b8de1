// The pages of the paged cache (rope.hip, attend.hip) as a pool that tables share: pages given to the places that need one,
// shared, copied, given back, moved together.
//
// refs [pages] int32 counts the places of the tables that hold a page; 0: it is free. Tables have -1 where a sequence has no
// page. Everything is decided on the GPU, in an order that does not depend on how threads run: the lowest free pages go to the
// first sequences' first places; counts change by integer atomics alone.
//
// Bound by latency where sequences take a few pages (a chain of dependent loads: offsets, lengths, table, counts, free pages),
// by HBM where pages are copied.
#include "rows.h"

namespace lmoe {

constexpr int kTakers = 1024;  // threads of the one workgroup that gives pages

// Inclusive sums over a wavefront's lanes
__device__ __forceinline__ int lanes_scan(int v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int u = __shfl_up(v, d);
    if (int(threadIdx.x & 63) >= d) v += u;
  }
  return v;
}

// Exclusive sum over a workgroup's threads in order, and the total; lds [wavefronts + 1]
__device__ __forceinline__ int block_scan(int v, int *lds, int *total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int in = lanes_scan(v);
  __syncthreads();  // what lds held has been read
  if (lane == 63) lds[wave] = in;
  __syncthreads();
  if (wave == 0) {
    const int w = lane < waves ? lds[lane] : 0, s = lanes_scan(w);
    if (lane < waves) lds[lane] = s - w;
    if (lane == waves - 1) lds[waves] = s;
  }
  __syncthreads();
  *total = lds[waves];
  return lds[wave] + in - v;
}

// Ranks of the pages of a stretch of J kTakers from p0 on that `is` holds for, in order, by the whole workgroup: rank(p, k), k = how
// many come before p in the stretch. Returns how many there are. J loads are on their way at a time, and ballots count them
// (a page a thread and shuffles: 18 us instead of 11 for a pool of 8,192 compacted by one workgroup).
template <int J, typename Is, typename Rank>
__device__ __forceinline__ int rank_stretch(int p0, int pages, const int *refs, int *lds, Is &&is, Rank &&rank) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, first = p0 + wave * (64 * J) + lane;
  int held[J];
#pragma unroll
  for (int j = 0; j < J; ++j) held[j] = first + 64 * j < pages ? refs[first + 64 * j] : -1;
  unsigned long long ones[J];
  int count = 0;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    ones[j] = __ballot(first + 64 * j < pages && is(first + 64 * j, held[j]));
    count += __popcll(ones[j]);
  }
  __syncthreads();  // what lds held has been read
  if (lane == 0) lds[wave] = count;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kTakers / 64; ++w) {
    const int c = lds[w];
    before += w < wave ? c : 0;
    total += c;
  }
#pragma unroll
  for (int j = 0; j < J; ++j) {
    if (ones[j] >> lane & 1) rank(first + 64 * j, before + __popcll(ones[j] & ((1ull << lane) - 1)));
    before += __popcll(ones[j]);
  }
  return total;
}

constexpr int kStretch = 8 * kTakers;  // pages that one workgroup looks at at a time

// How many pages of each stretch are free, or held
__global__ void __launch_bounds__(kTakers) k_count(const int *refs, int pages, int *counts, int held) {
  __shared__ int sums[kTakers / 64];
  const int n = rank_stretch<8>(blockIdx.x * kStretch, pages, refs, sums, [&](int, int r) { return held ? r > 0 : r == 0; },
                                [](int, int) {});
  if (threadIdx.x == 0) counts[blockIdx.x] = n;
}

struct TakeArgs {
  int *refs, *table;
  const int *lens, *cu;
  int *src, *dst, *lacking;
  int *begins;  // [B] where a sequence's tasks begin (more than kSeqsInLds sequences)
  int *ranks;   // [tasks]
  int *given;   // [pages that are needed]
  int *counts;  // [stretches] of free pages, or null
  int pages, B, width, page_shift;
};

constexpr int kSeqsInLds = 2048;

// The places [first, first + count) that a sequence's newest rows fall into, and the tokens before those
struct Fallen {
  int first, count, start;
  __device__ __forceinline__ Fallen(const TakeArgs &a, int b) {
    int row0, n;
    seq_rows(a.cu, b, 0x7fffffff, &row0, &n);
    const int len = a.lens[b];
    start = len > n ? len - n : 0;
    first = start >> a.page_shift;
    count = n > 0 && len > 0 ? max(min((len - 1) >> a.page_shift, a.width - 1) - first + 1, 0) : 0;
  }
};

// One workgroup. A task is a place that rows fall into, in the order of sequences and places. 1: where each sequence's tasks
// begin; 2: which need a page, and their ranks; 3: as many of the lowest free pages; 4: the places get them; 5: where that was
// not enough, a page that all of its holders gave up stays with the last of those that found none.
__global__ void __launch_bounds__(kTakers) k_take(TakeArgs a) {
  __shared__ int sums[kTakers / 64 + 1], begins_lds[kSeqsInLds], counts[kTakers];
  const int tid = threadIdx.x;
  int *begins = a.B <= kSeqsInLds ? begins_lds : a.begins;
  int tasks = 0;
  for (int b0 = 0; b0 < a.B; b0 += kTakers) {
    const int b = b0 + tid;
    int count = 0, total;
    if (b < a.B) {
      a.src[b] = -1, a.dst[b] = -1, a.lacking[b] = 0;
      count = Fallen(a, b).count;
    }
    const int begin = tasks + block_scan(count, sums, &total);
    if (b < a.B) begins[b] = begin;
    tasks += total;
  }
  __syncthreads();
  auto sequence_of = [&](int t) {  // the last one whose tasks begin at t or before: it has tasks
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (begins[mid] <= t)
        lo = mid;
      else
        hi = mid;
    }
    return lo;
  };
  int needs = 0;
  for (int t0 = 0; t0 < tasks; t0 += kTakers) {
    const int t = t0 + tid;
    bool need = false;
    if (t < tasks) {
      const int b = sequence_of(t), p = a.table[size_t(b) * a.width + Fallen(a, b).first + t - begins[b]];
      need = uint32_t(p) >= uint32_t(a.pages) || a.refs[p] > 1;
    }
    int total;
    const int rank = needs + block_scan(need, sums, &total);
    if (t < tasks) a.ranks[t] = need ? rank : -1;
    needs += total;
  }
  if (needs == 0) return;
  int found = 0;
  auto free_from = [&](auto j, int p0) {
    found += rank_stretch<decltype(j)::value>(p0, a.pages, a.refs, sums, [](int, int refs) { return refs == 0; },
                                              [&](int p, int rank) {
                                                if (found + rank < needs) a.given[found + rank] = p;
                                              });
  };
  if (!a.counts) {
    free_from(IC<1>{}, 0);  // (a few pages are often found among the first ones: 6.9 us of kernel instead of 9.8)
    for (int p0 = kTakers; p0 < a.pages && found < needs; p0 += kStretch) free_from(IC<8>{}, p0);
  } else {  // only the stretches that have any
    const int stretches = (a.pages + kStretch - 1) / kStretch;
    for (int s0 = 0; s0 < stretches && found < needs; s0 += kTakers) {
      __syncthreads();
      counts[tid] = s0 + tid < stretches ? a.counts[s0 + tid] : 0;
      __syncthreads();
      for (int i = 0; i < min(kTakers, stretches - s0) && found < needs; ++i)
        if (counts[i]) free_from(IC<8>{}, (s0 + i) * kStretch);
    }
  }
  __syncthreads();
  for (int t = tid; t < tasks; t += kTakers) {
    const int rank = a.ranks[t];
    if (rank < 0) continue;
    const int b = sequence_of(t);
    const Fallen at(a, b);
    const int i = at.first + t - begins[b];
    int *place = a.table + size_t(b) * a.width + i;
    const int old = *place, page = rank < found ? a.given[rank] : -1;
    if (page >= 0) *place = page, a.refs[page] = 1;
    if (uint32_t(old) < uint32_t(a.pages)) {
      atomicSub(a.refs + old, 1);
      if (page >= 0 && at.start > i << a.page_shift) a.src[b] = old, a.dst[b] = page;
    }
  }
  if (found >= needs) return;
  // Places that found no page still hold what they shared, or none
  auto each_without = [&](auto &&f) {  // f(task, sequence, place, page)
    __syncthreads();
    for (int t = tid; t < tasks; t += kTakers) {
      const int rank = a.ranks[t];
      if (rank == -1 || (rank >= 0 && rank < found)) continue;
      const int b = sequence_of(t);
      int *place = a.table + size_t(b) * a.width + Fallen(a, b).first + t - begins[b];
      f(t, b, place, *place);
    }
  };
  auto holders = [&](int p) { return __hip_atomic_load(a.refs + p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
  constexpr int kLeft = -2;  // for a rank: nobody holds what this place shared
  each_without([&](int t, int, int *, int p) {
    if (uint32_t(p) < uint32_t(a.pages) && holders(p) == 0) a.ranks[t] = kLeft;
  });
  each_without([&](int t, int, int *, int p) {
    if (a.ranks[t] == kLeft) atomicMin(a.refs + p, -1 - t);
  });
  each_without([&](int t, int b, int *place, int p) {
    if (a.ranks[t] == kLeft && holders(p) == -1 - t) {
      a.refs[p] = 1;
    } else {
      *place = -1;
      atomicAdd(a.lacking + b, 1);
    }
  });
}

// The places of a table from keep[b] tokens on are given back
__global__ void __launch_bounds__(256) k_free(int *refs, int pages, int *table, int width, long long places, const int *keep,
                                              int page_shift) {
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  if (at >= places) return;
  const int b = int(at / width), i = int(at - (long long)b * width);
  const long long kept = max(keep[b], 0);
  if (i < (kept + (1 << page_shift) - 1) >> page_shift) return;
  const int p = table[at];
  if (uint32_t(p) < uint32_t(pages)) atomicSub(refs + p, 1);
  if (p != -1) table[at] = -1;
}

// out's rows are those of table that parents names (none: -1); the pages' counts follow from table to out
__global__ void __launch_bounds__(256) k_fork(int *refs, int pages, const int *table, int B, int width, const int *parents, int n,
                                              int *out) {
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  if (at < (long long)B * width) {
    const int p = table[at];
    if (uint32_t(p) < uint32_t(pages)) atomicSub(refs + p, 1);
  }
  if (at < (long long)n * width) {
    const int r = int(at / width), i = int(at - (long long)r * width), from = parents[r];
    const int p = uint32_t(from) < uint32_t(B) ? table[size_t(from) * width + i] : -1;
    const bool there = uint32_t(p) < uint32_t(pages);
    if (there) atomicAdd(refs + p, 1);
    out[at] = there ? p : -1;
  }
}

// A workgroup for each stretch, after k_count of the held pages: which held pages lie past the first `used` numbers, and the free
// ones among those that they go to, both in order. Held pages before p are p's rank among them; what lies before `used` itself
// is counted by every workgroup.
__global__ void __launch_bounds__(kTakers) k_moves(const int *refs, int pages, int *counts, int *src, int *dst, int *used_out,
                                                   int *to) {
  __shared__ int sums[kTakers / 64 + 1];
  const int tid = threadIdx.x, stretches = gridDim.x, mine = blockIdx.x;
  auto held_in = [&](int end) {  // in the stretches before `end`
    int n = 0, total;
    for (int i = tid; i < end; i += kTakers) n += counts[i];
    block_scan(n, sums, &total);
    return total;
  };
  const int used = held_in(stretches), edge = used / kStretch;
  if (mine == 0 && tid == 0) *used_out = used;
  int below = held_in(edge);  // held pages before `used`
  if (edge < stretches)
    below += rank_stretch<8>(edge * kStretch, pages, refs, sums, [&](int p, int r) { return p < used && r > 0; }, [](int, int) {});
  if (mine == 0 && tid == 0) counts[stretches] = used - below;  // moves: as many as are free there
  const int before = held_in(mine), first = mine * kStretch;
  if (first < used)
    rank_stretch<8>(first, pages, refs, sums, [&](int p, int r) { return p < used && r <= 0; },
                    [&](int p, int rank) { dst[first - before + rank] = p; });
  if (first + kStretch > used)
    rank_stretch<8>(first, pages, refs, sums,
                    [&](int p, int r) {
                      if (p >= used) to[p] = p;  // (a page that only a table knows of stays what it is)
                      return p >= used && r > 0;
                    },
                    [&](int p, int rank) { src[max(before - below, 0) + rank] = p; });
}

// The moved pages' counts and new numbers; -1 behind the last pair
__global__ void __launch_bounds__(256) k_move(int *refs, const int *moves, int *src, int *dst, int most, int *to) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= most) return;
  if (i < *moves) {
    const int a = src[i], b = dst[i];
    refs[b] = refs[a];
    refs[a] = 0;
    to[a] = b;
  } else {
    src[i] = -1, dst[i] = -1;
  }
}

// A table's pages of `used` and more are the ones that were moved
__global__ void __launch_bounds__(256) k_renumber(int *table, long long places, int pages, const int *used, const int *to) {
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  if (at >= places) return;
  const int p = table[at];
  if (p >= *used && p < pages) table[at] = to[p];
}

struct CopyArgs {
  uint8_t *kc, *vc;
  float *ks, *vs;
  const int *src, *dst;
  long long page_bytes;  // of keys, or of values
  int pages, heads, n;
};

// Pairs of pages, a workgroup 16 KiB of keys or values at a time, four loads of a thread on their way
constexpr int kCopied = 16384;
__global__ void __launch_bounds__(256) k_copy(CopyArgs a) {
  const int parts = int((a.page_bytes + kCopied - 1) / kCopied);
  const long long works = 2ll * a.n * parts;
  for (long long w = blockIdx.x; w < works; w += gridDim.x) {
    const int i = int(w / (2 * parts)), which = int(w - i * 2ll * parts), value = which >= parts, part = which - value * parts;
    const int from = a.src[i], to = a.dst[i];
    if (uint32_t(from) >= uint32_t(a.pages) || uint32_t(to) >= uint32_t(a.pages)) continue;
    uint8_t *codes = value ? a.vc : a.kc;
    const uint8_t *x = codes + size_t(from) * a.page_bytes;
    uint8_t *y = codes + size_t(to) * a.page_bytes;
    const long long at = (long long)part * kCopied + threadIdx.x * 16;
    u32x4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (at + j * 4096 < a.page_bytes) v[j] = *reinterpret_cast<const u32x4 *>(x + at + j * 4096);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (at + j * 4096 < a.page_bytes) *reinterpret_cast<u32x4 *>(y + at + j * 4096) = v[j];
    if (part == 0) {
      float *scales = value ? a.vs : a.ks;
      for (int h = threadIdx.x; h < a.heads; h += 256) scales[size_t(to) * a.heads + h] = scales[size_t(from) * a.heads + h];
    }
  }
}

static bool pages_ok(int pages) { return pages > 0 && pages <= 1 << 30; }

static int stretches(int pages) { return (pages + kStretch - 1) / kStretch; }

static int page_shift(int page) { return page == 32 ? 5 : page == 64 ? 6 : page == 128 ? 7 : -1; }

}  // namespace lmoe

using namespace lmoe;

extern "C" size_t lmoe_pages_take_workspace_bytes(int B, int width, int pages) {
  if (B <= 0 || width <= 0 || pages <= 0) return 0;
  const long long places = (long long)B * width;
  return size_t(B + places + (places < pages ? places : pages) + stretches(pages)) * sizeof(int);
}

extern "C" int lmoe_pages_take(int *refs, int pages, int *table, int B, int width, const int *lens, const int *cu, int page, int *src,
                               int *dst, int *lacking, void *workspace, size_t workspace_bytes, void *stream) {
  const char *fn = "lmoe_pages_take";
  LMOE_REQUIRE(pages_ok(pages) && B >= 0 && width > 0, LMOE_ESHAPE, "%s: %d pages, %d sequences of %d places", fn, pages, B, width);
  LMOE_REQUIRE(page_shift(page) > 0, LMOE_ESHAPE, "%s: pages of %d tokens (32, 64 and 128 are served)", fn, page);
  LMOE_REQUIRE(width <= 0x7fffffff / page && (long long)B * width <= 0x7fffffff - kTakers, LMOE_ESHAPE,
               "%s: %d sequences of %d places of %d tokens are more than an int counts", fn, B, width, page);
  if (B == 0) return 0;
  LMOE_REQUIRE(refs && table && lens && src && dst && lacking, LMOE_EINVAL, "%s: null pointer", fn);
  const size_t need = lmoe_pages_take_workspace_bytes(B, width, pages);
  LMOE_REQUIRE(workspace && aligned4(workspace) && workspace_bytes >= need, LMOE_EWORKSPACE, "%s: a workspace of %zu bytes is needed",
               fn, need);
  int *begins = static_cast<int *>(workspace), *ranks = begins + B, *given = ranks + (long long)B * width;
  // One workgroup looks at 8,192 pages in 3.4 us: from three times as many on, a launch that counts all of them at once is worth
  // it (65,536 pages of which the last are free: 31 us without it, 11 with it)
  int *counts = pages > 2 * kStretch ? given + ((long long)B * width < pages ? (long long)B * width : pages) : nullptr;
  if (counts) {
    launch(k_count, dim3(stretches(pages)), dim3(kTakers), 0, (hipStream_t)stream, refs, pages, counts, 0);
    LMOE_LAUNCHED(fn);
  }
  launch(k_take, dim3(1), dim3(kTakers), 0, (hipStream_t)stream,
         TakeArgs{refs, table, lens, cu, src, dst, lacking, begins, ranks, given, counts, pages, B, width, page_shift(page)});
  LMOE_LAUNCHED(fn);
  return 0;
}

extern "C" int lmoe_pages_free(int *refs, int pages, int *table, int B, int width, const int *keep, int page, void *stream) {
  const char *fn = "lmoe_pages_free";
  LMOE_REQUIRE(pages_ok(pages) && B >= 0 && width > 0, LMOE_ESHAPE, "%s: %d pages, %d sequences of %d places", fn, pages, B, width);
  LMOE_REQUIRE(page_shift(page) > 0, LMOE_ESHAPE, "%s: pages of %d tokens (32, 64 and 128 are served)", fn, page);
  const long long places = (long long)B * width, groups = (places + 255) / 256;
  LMOE_REQUIRE(groups <= kMostGroups, LMOE_ESHAPE, "%s: %d sequences of %d places are more than a launch takes", fn, B, width);
  if (B == 0) return 0;
  LMOE_REQUIRE(refs && table && keep, LMOE_EINVAL, "%s: null pointer", fn);
  launch(k_free, dim3(unsigned(groups)), dim3(256), 0, (hipStream_t)stream, refs, pages, table, width, places, keep, page_shift(page));
  LMOE_LAUNCHED(fn);
  return 0;
}

extern "C" int lmoe_pages_fork(int *refs, int pages, const int *table, int B, int width, const int *parents, int n, int *out,
                               void *stream) {
  const char *fn = "lmoe_pages_fork";
  LMOE_REQUIRE(pages_ok(pages) && B >= 0 && n >= 0 && width > 0, LMOE_ESHAPE, "%s: %d pages, %d sequences of %d places, %d new ones", fn,
               pages, B, width, n);
  const long long groups = ((long long)(B > n ? B : n) * width + 255) / 256;
  LMOE_REQUIRE(groups <= kMostGroups, LMOE_ESHAPE, "%s: %d and %d sequences of %d places are more than a launch takes", fn, B, n,
               width);
  if (groups == 0) return 0;
  LMOE_REQUIRE(refs && (table || B == 0) && ((parents && out) || n == 0), LMOE_EINVAL, "%s: null pointer", fn);
  launch(k_fork, dim3(unsigned(groups)), dim3(256), 0, (hipStream_t)stream, refs, pages, table, B, width, parents, n, out);
  LMOE_LAUNCHED(fn);
  return 0;
}

extern "C" size_t lmoe_pages_compact_workspace_bytes(int pages) { return pages_ok(pages) ? size_t(stretches(pages) + 1) * sizeof(int) : 0; }

extern "C" int lmoe_pages_compact(int *refs, int pages, int *src, int *dst, int *used, int *to, void *workspace, size_t workspace_bytes,
                                  void *stream) {
  const char *fn = "lmoe_pages_compact";
  LMOE_REQUIRE(pages_ok(pages), LMOE_ESHAPE, "%s: %d pages", fn, pages);
  LMOE_REQUIRE(refs && src && dst && used && to, LMOE_EINVAL, "%s: null pointer", fn);
  const size_t need = lmoe_pages_compact_workspace_bytes(pages);
  LMOE_REQUIRE(workspace && aligned4(workspace) && workspace_bytes >= need, LMOE_EWORKSPACE, "%s: a workspace of %zu bytes is needed",
               fn, need);
  int *counts = static_cast<int *>(workspace);
  hipStream_t st = (hipStream_t)stream;
  const int n = stretches(pages), most = pages > 1 ? pages / 2 : 1;
  launch(k_count, dim3(n), dim3(kTakers), 0, st, refs, pages, counts, 1);
  LMOE_LAUNCHED(fn);
  launch(k_moves, dim3(n), dim3(kTakers), 0, st, refs, pages, counts, src, dst, used, to);
  LMOE_LAUNCHED(fn);
  launch(k_move, dim3((most + 255) / 256), dim3(256), 0, st, refs, counts + n, src, dst, most, to);
  LMOE_LAUNCHED(fn);
  return 0;
}

extern "C" int lmoe_pages_renumber(int *table, int B, int width, int pages, const int *used, const int *to, void *stream) {
  const char *fn = "lmoe_pages_renumber";
  LMOE_REQUIRE(pages_ok(pages) && B >= 0 && width > 0, LMOE_ESHAPE, "%s: %d pages, %d sequences of %d places", fn, pages, B, width);
  const long long places = (long long)B * width, groups = (places + 255) / 256;
  LMOE_REQUIRE(groups <= kMostGroups, LMOE_ESHAPE, "%s: %d sequences of %d places are more than a launch takes", fn, B, width);
  if (B == 0) return 0;
  LMOE_REQUIRE(table && used && to, LMOE_EINVAL, "%s: null pointer", fn);
  launch(k_renumber, dim3(unsigned(groups)), dim3(256), 0, (hipStream_t)stream, table, places, pages, used, to);
  LMOE_LAUNCHED(fn);
  return 0;
}

extern "C" int lmoe_pages_copy(uint8_t *k_codes, float *k_scale, uint8_t *v_codes, float *v_scale, int pages, int page, int heads,
                               int D, const int *src, const int *dst, int n, void *stream) {
  const char *fn = "lmoe_pages_copy";
  LMOE_REQUIRE(D == 64 || D == 128 || D == 256, LMOE_ESHAPE, "%s: heads of %d channels (64, 128 and 256 are served)", fn, D);
  LMOE_REQUIRE(page_shift(page) > 0, LMOE_ESHAPE, "%s: pages of %d tokens (32, 64 and 128 are served)", fn, page);
  LMOE_REQUIRE(pages_ok(pages) && heads > 0 && n >= 0, LMOE_ESHAPE, "%s: %d pages of %d heads, %d copies", fn, pages, heads, n);
  if (n == 0) return 0;
  LMOE_REQUIRE(k_codes && k_scale && v_codes && v_scale && src && dst, LMOE_EINVAL, "%s: null pointer", fn);
  LMOE_REQUIRE(aligned16(k_codes) && aligned16(v_codes), LMOE_EALIGN, "%s: codes must be 16-byte aligned", fn);
  const long long bytes = (long long)heads * page * D, works = 2ll * n * ((bytes + kCopied - 1) / kCopied);
  launch(k_copy, dim3(unsigned(works < 4096 ? works : 4096)), dim3(256), 0, (hipStream_t)stream,
         CopyArgs{k_codes, v_codes, k_scale, v_scale, src, dst, bytes, pages, heads, n});
  LMOE_LAUNCHED(fn);
  return 0;
}
