// Whole numbers of chunk.hip's cuts that need no GPU: constexpr, so that the kernels, the host and a program of plain C++ share them.
// A sequence's n rows of `group` query heads are `pairs` pairs in tiles of `rows`; off = len - n tokens stand before them.
#pragma once
#include <stdint.h>

namespace lmoe {

constexpr int kLineKeys = 64;       // keys a tile of keys
constexpr int kLeastStretch = 128;  // keys: two stretches do not begin at the same 64 keys of a tile then

constexpr int tiles_of(int n, int group, int rows) { return int(((long long)n * group + rows - 1) / rows); }

// How many keys a tile's last row sees, of `room` that the table has
constexpr int tile_sees(int off, int tile, int pairs, int group, int rows, int room) {
  const int end = tile * rows + rows < pairs ? tile * rows + rows : pairs, sees = off + (end - 1) / group + 1;
  return sees < room ? sees : room;
}

// ---- tiles in order --------------------------------------------------------------------------------------------

// More than 64 sequences: where the tiles of sequence b begin, whose first row is c
constexpr long long first_task(int c, int b, int group, int rows) { return (long long)c * group / rows + b; }
// and eight tasks in turn shifted against the next eight
constexpr int turned_task(int nth, int tasks) { return nth < (tasks & ~7) ? (nth & ~7) | ((nth + (nth >> 3)) & 7) : nth; }

// Up to 64: how many of a sequence's tiles see 256 x keys or more; a tile sees about past + tile rows / group
constexpr int tiles_that_see(int x, int past, int tiles, int group, int rows) {
  const long long more = 256ll * x - past, at = more <= 0 ? 0 : (more * group + rows - 1) / rows;
  return at >= tiles ? 0 : tiles - int(at);
}

// ---- the line of tiles -----------------------------------------------------------------------------------------

// What a tile's beginning and end cost, in keys
constexpr int line_start(int width, int waves) { return width == 256 || waves == 8 ? 320 : 192; }

// What the first `tiles` tiles of a sequence take on the line, times group (float64: a 64-bit product is an instruction; whole
// numbers below 2^53, and past that places are rounded, in the same way for all)
constexpr double line_cost(int past, int tiles, int group, int rows, int start) {
  return double(tiles) * (double(group) * (double(past > 0 ? past : 0) + start) + double(rows / 2) * (tiles + 1));
}

// The key that a stretch begins with, `at` keys behind a tile's start on the line
constexpr int line_key(double at) { return int(at <= 0.0 ? 0.0 : at < 0x7fffffff ? at : double(0x7fffffff)) & -kLineKeys; }

// One sequence's tiles in `per` equal pieces: the keys of each but the last, of `most` (1 or more). Pieces' ends pass 31 bits
// where a table has room for as many tokens
constexpr uint32_t piece_keys(uint32_t most, int per) { return ((most - 1) / uint32_t(per * kLineKeys) + 1) * kLineKeys; }

// Of how many pieces a row's sums are joined (0: none). The first one's line is `from`, the second's `next` further on, each other
// one's `step` behind that, the last one's `last`, of `most` lines in all. Rows that no sequence owns (where offsets fall, or
// begin below zero) have whatever the workspace held for from and last: no line outside of [0, most) comes of that.
constexpr int joined_pieces(int from, int last, int next, int step, int most) {
  return from < 0 || from >= most - next || last < from + next || last >= most ? 0 : 2 + (last - from - next) / step;
}

}  // namespace lmoe
