// larder_amd/csrc/lines.h for a test: the kernels' walk over tiles and stretches as loops over sequences in place of lanes, on the
// functions that they use. Numbers in, numbers out:
//   0 from last next step most                              joined_pieces
//   1 width waves group room of B n.. len..                 stretches of the line: "stretch b tile begin end sees" a piece, -1
//   2 width waves group room per 1 n len                    one sequence's pieces, likewise
//   3 waves group sorted tasks B n.. len..                  nth tile: "b tile" for each of the tasks (-1 -1: none)
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "../../larder_amd/csrc/lines.h"

using namespace lmoe;

static long long next() {
  long long x;
  if (std::scanf("%lld", &x) != 1) std::exit(1);
  return x;
}

struct Place {
  int b, tile, key;
};

struct Call {
  int group, rows, room, start, B;
  std::vector<int> n, len;
  void sequences(int count) {
    B = count;
    n.resize(B), len.resize(B);
    for (int &x : n) x = int(next());
    for (int &x : len) x = int(next());
  }
  int tiles(int b) const { return tiles_of(n[b], group, rows); }
  int sees(int b, int t) const { return tile_sees(len[b] - n[b], t, n[b] * group, group, rows, room); }
  double cost(int b, int t) const { return line_cost(len[b] - n[b], t, group, rows, start); }
  Place place(double x) const {
    for (int b = 0; b < B; ++b) {
      if (x < cost(b, tiles(b))) {
        int t = 0;
        while (t + 1 < tiles(b) && cost(b, t + 1) <= x) ++t;
        int key = line_key((x - cost(b, t)) * (1.0 / group) - start);
        if (key && sees(b, t) - key < kLineKeys) ++t, key = 0;
        return {b, t, key};
      }
      x -= cost(b, tiles(b));
    }
    return {B, 0, 0};
  }
  void walk(int one, Place at, Place to) const {
    for (;;) {
      if (at.b >= B) return;
      if ((long long)at.tile * rows >= (long long)n[at.b] * group) {
        int b = at.b + 1;
        while (b < B && n[b] == 0) ++b;
        if (b >= B) return;
        at = {b, 0, 0};
      }
      const bool same = at.b == to.b, last = same && at.tile == to.tile;
      if (at.b > to.b || (same && at.tile > to.tile) || (last && at.key >= to.key)) return;
      const int most = sees(at.b, at.tile), end = last && to.key < most ? to.key : most;
      std::printf("%d %d %d %d %d %d\n", one, at.b, at.tile, at.key, end, most);
      at = {at.b, at.tile + 1, 0};
    }
  }
};

int main() {
  int what;
  while (std::scanf("%d", &what) == 1) {
    if (what == 0) {
      int a[5];
      for (int &x : a) x = int(next());
      std::printf("%d\n", joined_pieces(a[0], a[1], a[2], a[3], a[4]));
      continue;
    }
    Call c;
    const int width = what == 3 ? 0 : int(next()), waves = int(next());
    c.rows = 32 * waves, c.start = line_start(width, waves), c.group = int(next());
    if (what == 3) {
      const bool sorted = next();
      const int tasks = int(next());
      c.room = 0, c.sequences(int(next()));
      std::vector<int> tiles(c.B), past(c.B), cu(1, 0);
      for (int b = 0; b < c.B; ++b) {
        tiles[b] = c.tiles(b), past[b] = c.len[b] > c.n[b] ? c.len[b] - c.n[b] : 0;
        if (tiles[b] < 1 && (b == 0 || b == c.B - 1)) tiles[b] = 1;
        cu.push_back(cu[b] + c.n[b]);
      }
      for (int nth = 0; nth < tasks; ++nth) {
        int b = -1, t = -1;
        if (c.B > 64) {
          const int task = tasks - 1 - turned_task(nth, tasks);
          for (int i = 0; i < c.B; ++i)
            if (first_task(cu[i], i, c.group, c.rows) <= task) b = i;
          t = b < 0 ? -1 : int(task - first_task(cu[b], b, c.group, c.rows));
        } else {
          auto count = [&](int i, int x) { return tiles_that_see(x, past[i], tiles[i], c.group, c.rows); };
          auto from = [&](int x) {
            int sum = 0;
            for (int i = 0; i < c.B; ++i) sum += count(i, x);
            return sum;
          };
          int x = 0, end = 1;
          for (int i = 0; sorted && i < c.B; ++i) {
            const int most = int((past[i] + (long long)tiles[i] * c.rows / c.group) >> 8) + 2;
            end = most > end ? most : end;
          }
          while (end - x > 1) {  // the largest x with more than nth tiles from it on
            const int mid = x + (end - x) / 2;
            (from(mid) > nth ? x : end) = mid;
          }
          int left = nth - (sorted ? from(x + 1) : 0);
          for (int i = 0; nth < from(0) && i < c.B && b < 0; ++i) {
            const int above = sorted ? count(i, x + 1) : 0, mine = count(i, x) - above;
            if (left < mine) b = i, t = tiles[i] - above - 1 - left;
            left -= mine;
          }
        }
        std::printf("%d %d\n", b, t);
      }
      std::printf("-2\n");
      continue;
    }
    c.room = int(next());
    int of = int(next());
    c.sequences(int(next()));
    if (what == 1) {
      double all = 0.0;
      for (int b = 0; b < c.B; ++b) all += c.cost(b, c.tiles(b));
      double each = all * (1.0 / of);
      if (each * (1.0 / c.group) < kLeastStretch) {
        of = int(all * (1.0 / c.group) * (1.0 / kLeastStretch));
        if (of < 1) of = 1;
        each = all / of;
      }
      for (int one = 0; one < of; ++one) {
        const double x0 = std::floor(each * one), x1 = one + 1 < of ? std::floor(each * (one + 1)) : all;
        c.walk(one, c.place(x0), x1 < all ? c.place(x1) : Place{c.B, 0, 0});
      }
    } else {
      for (int one = 0; one < c.tiles(0) * of; ++one) {
        const int t = one / of, i = one - t * of;
        const uint32_t most = c.sees(0, t) > 1 ? c.sees(0, t) : 1, step = piece_keys(most, of), begin = i * step;
        if (i > 0 && begin >= most) continue;
        c.walk(one, {0, t, int(begin)}, begin + step < most ? Place{0, t, int(begin + step)} : Place{0, t + 1, 0});
      }
    }
    std::printf("-1\n");
  }
}
