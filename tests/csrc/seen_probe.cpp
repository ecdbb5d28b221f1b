// The table of launched kernels behind C functions, for tests that have no GPU.
#include "../../cute_mma_b200/csrc/prism_seen.h"

static prism::SeenKernels seen;
extern "C" int seen_has(unsigned long long fn, int dev, int bytes) { return seen.has(reinterpret_cast<const void*>(fn), dev, bytes); }
extern "C" void seen_add(unsigned long long fn, int dev, int bytes) { seen.add(reinterpret_cast<const void*>(fn), dev, bytes); }
