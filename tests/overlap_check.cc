// rows_share (ms_overlap.h) against a map of bytes, over random matrices of
// rows: neighbours, column blocks of one buffer, other strides, one row.
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>

#include "ms_overlap.h"

int main() {
  std::mt19937 rng(7);
  auto in = [&](size_t lo, size_t hi) { return lo + rng() % (hi - lo + 1); };
  long shared = 0, apart = 0;
  for (int t = 0; t < 400000; ++t) {
    const size_t M = in(1, 6), wa = in(1, 12), wb = in(1, 12);
    size_t lda = in(wa, 30), ldb = in(wb, 30);
    if (rng() % 2) lda = ldb = std::max(lda, ldb);
    const uintptr_t a = 1000 + in(0, 200), b = 1000 + in(0, 200);
    std::vector<char> map(2000, 0);
    for (size_t i = 0; i < M; ++i)
      for (size_t k = 0; k < wa; ++k) map[a + i * lda + k] = 1;
    bool want = false;
    for (size_t i = 0; i < M; ++i)
      for (size_t k = 0; k < wb; ++k) want |= map[b + i * ldb + k] != 0;
    (want ? shared : apart)++;
    if (ms::rows_share(a, lda, wa, b, ldb, wb, M) != want ||
        ms::rows_share(b, ldb, wb, a, lda, wa, M) != want) {
      printf("M %zu: a %zu + %zu x %zu, b %zu + %zu x %zu: share %d\n", M, (size_t)a, lda, wa, (size_t)b, ldb,
             wb, want);
      return 1;
    }
  }
  if (shared < 1000 || apart < 1000) return 1;
  printf("ok\n");
  return 0;
}
