// WsPool (ms_ws.h) on a pretended device, through random calls on streams and
// into graphs, graphs that end and memory that runs out.  After each: a
// workspace is large enough and lies in memory that is allocated; none that a
// stream with work in flight or a living graph holds is freed or given to
// another; and memory does not pile up.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>

#include "ms_ws.h"

using ms::WsPool;
typedef unsigned long long u64;

#define CHECK(c)                                  \
  do {                                            \
    if (!(c)) {                                   \
      printf("line %d: %s\n", __LINE__, #c);      \
      exit(1);                                    \
    }                                             \
  } while (0)

struct Device {
  std::map<void*, size_t> mem;
  std::map<u64, std::set<void*>> busy;      // by stream, since it was last waited for
  std::map<u64, std::set<void*>> graph;     // by living graph
  size_t left = 0;
  uintptr_t next = 4096;
  bool can_wait = true;
  int waits = 0;
  bool held(void* p) const {
    for (auto& b : busy)
      if (b.second.count(p)) return true;
    for (auto& g : graph)
      if (g.second.count(p)) return true;
    return false;
  }
  void* alloc(size_t n) {
    if (n > left) return nullptr;
    left -= n;
    void* p = (void*)next;
    next += n + 4096;
    mem[p] = n;
    return p;
  }
  void free(void* p) {
    CHECK(mem.count(p) && !held(p));
    left += mem[p];
    mem.erase(p);
  }
  void wait(u64 s) { busy.erase(s); }
  bool wait_all() {
    if (!can_wait) return false;
    ++waits;
    busy.clear();
    return true;
  }
};

int main() {
  std::mt19937 rng(3);
  Device d;
  d.left = (size_t)1 << 40;
  WsPool pool;
  u64 graphs = 0, largest = 0, refused = 0, taken = 0;
  for (int t = 0; t < 300000; ++t) {
    const int what = rng() % 100;
    size_t bytes = (size_t)1 << (rng() % 30);
    if (t % 1000 == 0) d.left = t % 3000 ? (size_t)1 << 40 : (size_t)1 << (20 + rng() % 16);
    d.can_wait = rng() % 20 != 0;
    if (what < 60) {
      const u64 s = 1 + rng() % (t % 5000 < 2500 ? 6 : 40);
      void* p = pool.for_stream(s, bytes, d);
      largest = std::max(largest, (u64)bytes);
      if (!p) continue;
      CHECK(d.mem.count(p) && d.mem[p] >= bytes);
      for (auto& b : d.busy) CHECK(b.first == s || !b.second.count(p));
      for (auto& g : d.graph) CHECK(!g.second.count(p));
      d.busy[s].insert(p);
    } else if (what < 85) {
      if (d.graph.empty() || rng() % 4 == 0) d.graph[++graphs];
      auto it = d.graph.begin();
      std::advance(it, rng() % d.graph.size());
      const u64 s = 1 + rng() % 3;  // streams that the capture spans
      if (rng() % 20 == 0) bytes = largest + 1;
      bool no = false, first = false;
      const size_t had = it->second.size();
      void* p = pool.for_graph(it->first, s, bytes, d, &no, &first);
      CHECK(no == (bytes > largest));
      refused += no;
      if (!p) continue;
      CHECK(!no && d.mem.count(p) && d.mem[p] >= bytes && first == (had == 0));
      for (auto& b : d.busy) CHECK(!b.second.count(p));
      for (auto& g : d.graph) CHECK(g.first == it->first || !g.second.count(p));
      ++taken;
      it->second.insert(p);
    } else if (!d.graph.empty()) {
      auto it = d.graph.begin();
      std::advance(it, rng() % d.graph.size());
      const u64 g = it->first;
      d.graph.erase(it);
      pool.release(g);
    }
    size_t total = 0;
    for (auto& m : d.mem) total += m.second;
    CHECK(total == pool.bytes());
  }
  CHECK(refused > 100 && taken > 1000 && d.waits > 10);
  // graphs that come and go one after the other need no more than one of them
  for (auto& g : d.graph) pool.release(g.first);
  d.graph.clear();
  d.busy.clear();
  d.left = (size_t)1 << 40;
  d.can_wait = true;
  const size_t size = (size_t)1 << 29;
  CHECK(pool.for_stream(1, size, d));
  d.busy.clear();
  size_t after = 0;
  for (int i = 0; i < 100; ++i) {
    bool no, first;
    CHECK(pool.for_graph(++graphs, 1, size, d, &no, &first) && first);
    if (i == 0) after = pool.bytes();
    CHECK(pool.bytes() == after);
    pool.release(graphs);
  }
  // two streams of one capture, and a call of another size in it
  bool no, first;
  void* a = pool.for_graph(++graphs, 1, 1000, d, &no, &first);
  void* b = pool.for_graph(graphs, 2, 1000, d, &no, &first);
  CHECK(a && b && a != b && !first);
  CHECK(pool.for_graph(graphs, 1, 1000, d, &no, &first) == a);
  pool.free_all(d);
  CHECK(d.mem.empty() && pool.bytes() == 0);
  printf("ok\n");
  return 0;
}
