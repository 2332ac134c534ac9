// What the library's translation units share and its users do not see.
#ifndef DLAGG_INTERNAL_H
#define DLAGG_INTERNAL_H

#include <cstdint>

// Sets this thread's dla_last_error() and returns `code`; clears it.
__attribute__((visibility("hidden"))) int dla_internal_fail(int code, const char* msg);
__attribute__((visibility("hidden"))) void dla_internal_clear_error();

// Workgroups of `threads` threads for `units` of work, one unit each as long as a launch has fewer than 2^32 threads, which
// is as many as HIP takes; the workgroups of a larger one walk.
inline int64_t dla_internal_grid(int64_t units, int threads) {
  const int64_t most = INT64_C(0xffffffff) / threads;
  return units < most ? units : most;
}

#endif  // DLAGG_INTERNAL_H
