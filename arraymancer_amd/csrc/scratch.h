// A block of device memory for the length of one call, from the library's cache of blocks. It goes back to the cache when
// the call returns, and whoever gets it next touches it behind this call's kernels on the same stream; while a graph is
// being captured the block stays with that graph.
#pragma once
#include "common.h"

namespace am {

struct Scratch {
  void* p = nullptr;
  int take(size_t bytes) { return am_hip_malloc(bytes, &p); }
  ~Scratch() { if (p) (void)am_hip_free(p); }
  Scratch() = default;
  Scratch(const Scratch&) = delete;
  Scratch& operator=(const Scratch&) = delete;
};

}  // namespace am
