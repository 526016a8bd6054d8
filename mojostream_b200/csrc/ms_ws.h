// ms_ws.h -- workspace of the operators beside the token loop: how it grows.
// Host only, internal to libmojostream_cuda.so.
#pragma once

#include <stddef.h>

#include <algorithm>

namespace ms {

// Memory of at least `bytes` to follow a workspace of `old` bytes (alloc gives
// null when there is none): twice the old one, so that calls of growing sizes
// do not allocate each time, or else just what the call needs.
template <typename Alloc>
void* ws_grow(size_t bytes, size_t old, Alloc&& alloc, size_t* got) {
  const size_t want = std::max(std::max(bytes, 2 * old), (size_t)1 << 20);
  for (const size_t n : {want, bytes}) {
    *got = n;
    if (void* p = alloc(n)) return p;
  }
  *got = 0;
  return nullptr;
}

}  // namespace ms
