// gq_paged.h -- arithmetic of the paged 8-bit KV cache that the host, the
// kernels and the CPU tests share.  No HIP headers: g++ compiles it too.
#pragma once
#include <stdint.h>

#if defined(__HIPCC__)
#define GQ_HD __host__ __device__ __forceinline__
#else
#define GQ_HD inline
#endif

namespace gq {

constexpr int KV8_PAGE_MAX = 256;            // tokens of a page: multiples of 16 up to this
constexpr int PAGE_PLAN_MAX_REQUESTS = 4096;  // both prefix sums stay in a block's LDS
constexpr float KV8_MIN_SCALE = 0x1p-60f;

// The sum of two counts >= 0, held at INT_MAX (so that it is associative).
GQ_HD int sat_add(int a, int b) {
  const uint32_t s = (uint32_t)a + (uint32_t)b;
  return s > 0x7fffffffu ? 0x7fffffff : (int)s;
}
GQ_HD int not_negative(int v) { return v < 0 ? 0 : v; }

// Pages that `tokens` >= 0 take, at most a table's width.
GQ_HD int pages_of(int tokens, int page, int wide) {
  const int p = (int)(((uint32_t)tokens + (uint32_t)page - 1u) / (uint32_t)page);
  return p < wide ? p : wide;
}

// The slot of offset `off` in page `id`, -1 where there is no such page or
// the slot does not fit an int.
GQ_HD int slot_of(int id, int page, int off) {
  if (id < 0) return -1;
  const int64_t s = (int64_t)id * page + off;
  return s > 0x7fffffff ? -1 : (int)s;
}

// First i in [0, n) with at[i + 1] > v (at[0] = 0, ascending, v < at[n]).
GQ_HD int owner_of(const int *at, int n, int v) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (at[mid + 1] > v)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

}  // namespace gq
