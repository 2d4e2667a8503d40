// Answers questions about the paged cache's index arithmetic, one a line:
//   add A B               ->  sat_add
//   pages TOKENS P WIDE   ->  pages_of
//   slot ID P OFF         ->  slot_of
//   owner N V AT0 .. ATN  ->  owner_of
//   req S E CTX N WIDE PAGE MAXCTX  ->  start fresh first keys of attn_request
//   keys FRESH FIRST KEYS I0 I1 WINDOW SPLIT  ->  lo hi of attn_keys, attn_parts
//   cut TOKENS REQUESTS KV GROUP MAXNEW MAXCTX  ->  few rtiles split rparts ttiles
//                                               tsplit tparts parts of attn_cut
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
    } else if (!std::strcmp(what, "req")) {
      int s, e, ctx, n, wide, page, most;
      if (std::scanf("%d %d %d %d %d %d %d", &s, &e, &ctx, &n, &wide, &page, &most) != 7) return 1;
      const gq::AttnRequest r = gq::attn_request(s, e, ctx, n, wide, page, most);
      std::printf("%d %d %d %d\n", r.start, r.fresh, r.first, r.keys);
    } else if (!std::strcmp(what, "keys")) {
      gq::AttnRequest r{};
      int i0, i1, window, split;
      if (std::scanf("%d %d %d %d %d %d %d", &r.fresh, &r.first, &r.keys, &i0, &i1, &window, &split) != 7) return 1;
      const gq::AttnKeys k = gq::attn_keys(r, i0, i1, window);
      std::printf("%d %d %d\n", k.lo, k.hi, gq::attn_parts(k, split));
    } else if (!std::strcmp(what, "cut")) {
      int n, nr, kv, group, fresh, ctx;
      if (std::scanf("%d %d %d %d %d %d", &n, &nr, &kv, &group, &fresh, &ctx) != 6) return 1;
      const gq::AttnCut t = gq::attn_cut(n, nr, kv, group, fresh, ctx);
      std::printf("%d %lld %d %d %lld %d %d %d\n", t.few, (long long)t.rtiles, t.split, t.rparts, (long long)t.ttiles, t.tsplit,
                  t.tparts, t.parts);
    } else {
      return 1;
    }
  }
}
