// ms_ws.h -- workspaces of the operators beside the token loop: whose they are
// and how they grow.  Host only, internal to libmojostream_cuda.so.
#pragma once

#include <stddef.h>

#include <algorithm>
#include <mutex>
#include <vector>

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

// A call's workspace is written by its first kernel and read by its second, so
// calls that may run at the same time must not have one in common.  Calls of
// one stream follow one another, those of a graph (captured from one stream)
// too; so every stream has a workspace, and every captured graph one for each
// stream that it was captured from, until the graph is gone.
//   Dev: alloc(n) (null: no memory), free(p), wait(id) (the work of a stream
// has finished), wait_all() (all work has; false: it cannot be waited for now).
// One thread calls at a time; only release() may come from any other.
class WsPool {
 public:
  enum Kind { kFree, kStream, kGraph };
  // Streams come and go; beyond so many the one that called longest ago gives
  // its workspace up.
  static constexpr int kMaxStreams = 16;

  // The workspace of a call outside captures, or null: no memory.
  template <typename Dev>
  void* for_stream(unsigned long long stream, size_t bytes, Dev& dev) {
    drain();
    largest_ = std::max(largest_, bytes);
    Buf* own = find(kStream, stream, 0);
    if (own && own->bytes >= bytes) return use(*own);
    if (!own && count(kStream) >= kMaxStreams && dev.wait_all()) {
      Buf* oldest = nullptr;
      for (Buf& b : bufs_)
        if (b.kind == kStream && (!oldest || b.used < oldest->used)) oldest = &b;
      oldest->kind = kFree;
    }
    size_t old = 0;
    if (own) {
      old = own->bytes;
      dev.wait(stream);  // then nothing uses it
      own->kind = kFree;
    }
    return take(kStream, stream, 0, bytes, old, dev);
  }

  // The workspace of a call that is captured into graph `graph` from `stream`,
  // or null: no memory, or (*refused) more than any call outside captures has
  // asked for.  *first: the graph's first, release() has to follow its end.
  template <typename Dev>
  void* for_graph(unsigned long long graph, unsigned long long stream, size_t bytes, Dev& dev,
                  bool* refused, bool* first) {
    drain();
    *refused = bytes > largest_;
    *first = false;
    if (*refused) return nullptr;
    for (Buf& b : bufs_)  // (a smaller one that earlier nodes of the graph use stays as it is)
      if (b.kind == kGraph && b.owner == graph && b.stream == stream && b.bytes >= bytes) return use(b);
    *first = true;
    for (const Buf& b : bufs_)
      if (b.kind == kGraph && b.owner == graph) *first = false;
    return take(kGraph, graph, stream, bytes, 0, dev);
  }

  // Graph `graph` is gone, its executions have finished.  Only noted here: the
  // device's functions may not be called where this is.
  void release(unsigned long long graph) {
    std::lock_guard<std::mutex> lock(mu_);
    gone_.push_back(graph);
  }

  size_t largest() const { return largest_; }
  size_t bytes() const {
    size_t n = 0;
    for (const Buf& b : bufs_) n += b.bytes;
    return n;
  }
  template <typename Dev>
  void free_all(Dev& dev) {
    for (const Buf& b : bufs_) dev.free(b.p);
    bufs_.clear();
  }

 private:
  struct Buf {
    void* p;
    size_t bytes;
    Kind kind;
    unsigned long long owner, stream;  // of a graph: the stream that it was captured from
    unsigned long long used;
  };

  void drain() {
    std::lock_guard<std::mutex> lock(mu_);
    for (const unsigned long long graph : gone_)
      for (Buf& b : bufs_)
        if (b.kind == kGraph && b.owner == graph) b.kind = kFree;
    gone_.clear();
  }
  Buf* find(Kind kind, unsigned long long owner, unsigned long long stream) {
    for (Buf& b : bufs_)
      if (b.kind == kind && b.owner == owner && b.stream == stream) return &b;
    return nullptr;
  }
  int count(Kind kind) const {
    int n = 0;
    for (const Buf& b : bufs_) n += b.kind == kind;
    return n;
  }
  void* use(Buf& b) {
    b.used = ++clock_;
    return b.p;
  }
  // A free buffer that is large enough and not four times too large, or a new
  // one, for which (not inside a capture) the free ones make room.
  template <typename Dev>
  void* take(Kind kind, unsigned long long owner, unsigned long long stream, size_t bytes, size_t old,
             Dev& dev) {
    Buf* best = nullptr;
    for (Buf& b : bufs_)
      if (b.kind == kFree && b.bytes >= bytes && (!best || b.bytes < best->bytes)) best = &b;
    if (!best || best->bytes / 4 > std::max(bytes, (size_t)1 << 20)) {
      bufs_.reserve(bufs_.size() + 1);  // (throws before there is anything to lose)
      for (size_t i = bufs_.size(); i-- > 0 && kind == kStream;)
        if (bufs_[i].kind == kFree) {
          dev.free(bufs_[i].p);
          bufs_.erase(bufs_.begin() + i);
        }
      size_t got = 0;
      void* p = ws_grow(bytes, old, [&](size_t n) { return dev.alloc(n); }, &got);
      if (!p) return nullptr;
      bufs_.push_back({p, got, kFree, 0, 0, 0});
      best = &bufs_.back();
    }
    best->kind = kind;
    best->owner = owner;
    best->stream = stream;
    return use(*best);
  }

  std::mutex mu_;  // of gone_; never held while the device is asked for something
  std::vector<unsigned long long> gone_;
  std::vector<Buf> bufs_;
  size_t largest_ = 0;
  unsigned long long clock_ = 0;
};

}  // namespace ms
