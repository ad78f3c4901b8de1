// Whole numbers of chunk.hip's cuts that need no GPU: constexpr, so that the kernels, the host and a program of plain C++ share them.
#pragma once

namespace lmoe {

// Of how many pieces a row's sums are joined (0: none). The first one's line is `from`, the second's `next` further on, each other
// one's `step` behind that, the last one's `last`, of `most` lines in all. Rows that no sequence owns (where offsets fall, or
// begin below zero) have whatever the workspace held for from and last: no line outside of [0, most) comes of that.
constexpr int joined_pieces(int from, int last, int next, int step, int most) {
  return from < 0 || from >= most - next || last < from + next || last >= most ? 0 : 2 + (last - from - next) / step;
}

}  // namespace lmoe
