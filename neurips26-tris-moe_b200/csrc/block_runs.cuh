// Which rows a CTA of the append to block-scaled pages takes at a time (paged_kv_blocks.cu).  Plain C++ but for the two intrinsics, so that the rule can be tried on a host.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define TRIS_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define TRIS_HOST_DEVICE inline
#endif

namespace tris {

TRIS_HOST_DEVICE int lowest_bit(uint32_t v) {  // of a number that is not 0
#ifdef __CUDA_ARCH__
  return __ffs(static_cast<int>(v)) - 1;
#else
  return __builtin_ctz(v);
#endif
}
TRIS_HOST_DEVICE int highest_bit(uint32_t v) {
#ifdef __CUDA_ARCH__
  return 31 - __clz(static_cast<int>(v));
#else
  return 31 - __builtin_clz(v);
#endif
}

// A window of `window` tokens begins with a run's first token; bit i of `starts` says whether token i of it begins a run, `window` included.  The CTA owns the
// runs that begin in the first `own` tokens, 1 to `window` of them, and no others: the next CTA begins with the first run behind those, and two at one block would both bring its
// tokens to a new scale.  Returns how many tokens the whole runs are that it owns and the window holds; 0: the first run is longer than the window.
TRIS_HOST_DEVICE int tokens_of_whole_runs(uint32_t starts, int own, int window) {
  const uint32_t beyond = starts >> own;
  const int stop = beyond ? own + lowest_bit(beyond) : window + 1;
  if (stop <= window) return stop;
  const uint32_t behind = starts & ((1u << own) - 1) & ~1u;  // of the runs that it owns the last one goes on behind the window
  return behind ? highest_bit(behind) : 0;
}

}  // namespace tris
