// Which of a context's scratch buffers its recorded graphs hold.  A graph keeps the addresses
// that its calls had when they were recorded, so a buffer that a later call outgrows may only be
// freed when no graph holds it.  Plain C++, which the CPU tests build too.
#pragma once

#include <cstddef>
#include <new>
#include <vector>

namespace mmnb {

constexpr int kScratchSlots = 12;

class GraphBuffers {
 public:
  // A recording begins (or is given up), and a call of it takes slot's buffer p, which stays the
  // same to the recording's end.
  void begin() {
    for (void *&p : now_.held) p = nullptr;
  }
  void take(int slot, void *p) { now_.held[slot] = p; }
  // The recording has become a graph; false when host memory is out.
  bool end(void *graph) {
    now_.graph = graph;
    const bool ok = push(graphs_, now_);
    begin();
    return ok;
  }

  bool held(const void *p) const {
    for (const Graph &g : graphs_)
      for (const void *q : g.held)
        if (p && q == p) return true;
    return false;
  }
  // Keeps a held buffer that has been replaced; false when host memory is out.
  bool retire(void *p) { return push(retired_, p); }

  // The graph is gone, and with it what it alone held.
  template <typename Free>
  void destroyed(const void *graph, Free free) {
    for (size_t i = 0; i < graphs_.size(); i++)
      if (graphs_[i].graph == graph) {
        graphs_.erase(graphs_.begin() + i);
        break;
      }
    for (size_t i = 0; i < retired_.size();) {
      if (held(retired_[i])) {
        i++;
        continue;
      }
      free(retired_[i]);
      retired_.erase(retired_.begin() + i);
    }
  }
  // All of them, with the context.
  template <typename Free>
  void clear(Free free) {
    graphs_.clear();
    destroyed(nullptr, free);
  }

 private:
  struct Graph {
    void *graph = nullptr;
    void *held[kScratchSlots] = {};
  };
  template <typename T>
  static bool push(std::vector<T> &v, const T &x) {
    try {
      v.push_back(x);
    } catch (const std::bad_alloc &) {
      return false;
    }
    return true;
  }
  Graph now_;
  std::vector<Graph> graphs_;
  std::vector<void *> retired_;
};

}  // namespace mmnb
