// ms_overlap.h -- whether two matrices of rows share memory.  Host only.
// Internal to libmojostream_cuda.so.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace ms {

// Rows [a + i lda, + wa) and [b + j ldb, + wb), 0 <= i, j < M, all in bytes,
// widths of 1 and more, strides at least the widths: do any two share a byte?
// Exact, so that column blocks of one buffer are told apart.
inline bool rows_share(uintptr_t a, size_t lda, size_t wa, uintptr_t b, size_t ldb, size_t wb,
                       size_t M) {
  const uintptr_t a1 = a + (M - 1) * lda + wa, b1 = b + (M - 1) * ldb + wb;
  if (a >= b1 || b >= a1) return false;
  // the rows of one stride that reach into a row of the other
  auto hits = [&](uintptr_t r, size_t w, uintptr_t c, size_t ld, size_t wc) {
    if (r + w <= c) return false;
    size_t j = r > c ? (r - c) / ld : 0;  // the last row that begins at r or before
    if (j >= M) j = M - 1;
    const uintptr_t x = c + j * ld;
    if (x < r + w && r < x + wc) return true;
    return j + 1 < M && x + ld < r + w;
  };
  if (lda == ldb) {
    // offsets between rows are those of the first rows, one stride or more apart
    return b >= a ? hits(b, wb, a, lda, wa) : hits(a, wa, b, ldb, wb);
  }
  for (size_t i = 0; i < M; ++i)
    if (hits(a + i * lda, wa, b, ldb, wb)) return true;
  return false;
}

}  // namespace ms
