// ws_grow (ms_ws.h) on a device with so much memory: calls are served as long
// as what they need is there, and sizes that grow a little allocate seldom.
#include <cstdio>
#include <cstdlib>

#include "ms_ws.h"

int main() {
  size_t left = 0;
  int calls = 0;
  auto alloc = [&](size_t n) -> void* {
    ++calls;
    if (n > left) return nullptr;
    left -= n;
    return (void*)16;
  };
  auto check = [](bool ok, int line) {
    if (!ok) {
      printf("line %d\n", line);
      exit(1);
    }
  };
  const size_t G = (size_t)1 << 30;
  size_t got = 7;
  left = 100 * G;  // a workspace of 60 GB: one byte more fits, twice as much does not
  check(ms::ws_grow(60 * G + 1, 60 * G, alloc, &got) && got == 60 * G + 1, __LINE__);
  check(left == 40 * G - 1 && calls == 2, __LINE__);
  check(!ms::ws_grow(41 * G, 60 * G, alloc, &got) && got == 0 && left == 40 * G - 1, __LINE__);
  left = 1000;  // not even the least size, but the call's
  check(ms::ws_grow(1000, 0, alloc, &got) && got == 1000 && left == 0, __LINE__);
  left = 100 * G;
  calls = 0;
  size_t have = 0;
  for (size_t n = 1; n <= 4096; ++n)  // 1 MB to 4 GB in steps of 1 MB
    if (n << 20 > have) {
      check(ms::ws_grow(n << 20, have, alloc, &got) && got >= n << 20, __LINE__);
      have = got;
    }
  check(calls <= 13, __LINE__);
  printf("ok\n");
  return 0;
}
