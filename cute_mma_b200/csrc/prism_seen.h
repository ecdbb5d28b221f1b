// Which kernels have had their shared-memory limit raised, by function and device (plain C++, tested without CUDA).
#pragma once

#include <stdint.h>

namespace prism {

// Open addressing over 4096 places: the library has a few hundred kernels, a process up to eight devices.  Past three quarters it
// starts anew; what is forgotten is only set again.  Never allocates, so that nothing can be thrown out of a C entry point.
struct SeenKernels {
  static constexpr unsigned kPlaces = 4096;
  struct Entry { const void* fn; int dev, bytes; };
  Entry e[kPlaces];   // fn null: free
  unsigned used;

  Entry* find(const void* fn, int dev) {
    unsigned at = (unsigned)(((reinterpret_cast<uintptr_t>(fn) >> 4) * 0x9e3779b97f4a7c15ull + (unsigned)dev * 0x85ebca6bull) >> 20);
    while (true) {
      Entry* x = &e[at++ % kPlaces];
      if (x->fn == nullptr || (x->fn == fn && x->dev == dev)) return x;
    }
  }
  bool has(const void* fn, int dev, int bytes) {
    const Entry* x = find(fn, dev);
    return x->fn != nullptr && x->bytes >= bytes;
  }
  void add(const void* fn, int dev, int bytes) {
    Entry* x = find(fn, dev);
    if (x->fn == nullptr) {
      if (used >= kPlaces / 4 * 3) {
        for (unsigned i = 0; i < kPlaces; ++i) e[i].fn = nullptr;
        used = 0;
        x = find(fn, dev);
      }
      ++used;
    } else if (x->bytes > bytes) {
      return;
    }
    *x = Entry{fn, dev, bytes};
  }
};

}  // namespace prism
