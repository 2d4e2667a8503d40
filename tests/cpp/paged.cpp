// Answers questions about the paged cache's index arithmetic, one a line:
//   add A B               ->  sat_add
//   pages TOKENS P WIDE   ->  pages_of
//   slot ID P OFF         ->  slot_of
//   owner N V AT0 .. ATN  ->  owner_of
#include <cstdio>
#include <cstring>
#include <vector>

#include "gq_paged.h"

int main() {
  char what[8];
  int a, b, c;
  while (std::scanf("%7s", what) == 1) {
    if (!std::strcmp(what, "add") && std::scanf("%d %d", &a, &b) == 2) {
      std::printf("%d\n", gq::sat_add(a, b));
    } else if (!std::strcmp(what, "pages") && std::scanf("%d %d %d", &a, &b, &c) == 3) {
      std::printf("%d\n", gq::pages_of(a, b, c));
    } else if (!std::strcmp(what, "slot") && std::scanf("%d %d %d", &a, &b, &c) == 3) {
      std::printf("%d\n", gq::slot_of(a, b, c));
    } else if (!std::strcmp(what, "owner") && std::scanf("%d %d", &a, &b) == 2) {
      std::vector<int> at(a + 1);
      for (int &v : at)
        if (std::scanf("%d", &v) != 1) return 1;
      std::printf("%d\n", gq::owner_of(at.data(), a, b));
    } else {
      return 1;
    }
  }
}
