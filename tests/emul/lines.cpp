// larder_amd/csrc/lines.h for a test: lines of numbers in, one number a line out.
//   0 from last next step most        joined_pieces
#include <cstdio>
#include "../../larder_amd/csrc/lines.h"

int main() {
  int what;
  while (std::scanf("%d", &what) == 1) {
    int a[5];
    for (int &x : a)
      if (std::scanf("%d", &x) != 1) return 1;
    std::printf("%d\n", lmoe::joined_pieces(a[0], a[1], a[2], a[3], a[4]));
  }
}
