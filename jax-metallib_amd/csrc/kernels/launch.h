// Host-side helpers of the launchers in this directory.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../capi_internal.h"

namespace mkc {

// Lets a kernel use `bytes` of dynamic LDS, asked for once per device (`done`:
// a bit per device, one word per kernel).
inline int lds_opt_in(const void* kernel, int bytes, std::atomic<uint64_t>& done, const char* fn) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0) dev = 64;
  const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
  if (done.load(std::memory_order_acquire) & bit) return MK_OK;
  const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) return fail(MK_ELAUNCH, "%s: LDS opt-in failed: %s", fn, hipGetErrorString(e));
  done.fetch_or(bit, std::memory_order_release);
  return MK_OK;
}

// A launch has fewer than 2^32 threads per dimension.
inline bool grid_fits(int64_t blocks, int threads) { return blocks < ((int64_t)1 << 32) / threads; }

// A stride that no element is reached by counts as 0.
inline int64_t stride_of(int64_t stride, int64_t n) { return n > 1 ? stride : 0; }

// Whether the n[0] n[1] n[2] runs of `run` elements, `stride` (>= 0) apart, have
// no element in common: where each stride passes what lies within it (every
// layout but interleaved ones), else by looking for two indices whose distance
// is less than a run.  A stride of 0 counts only where there is one index.
inline bool runs_apart(const int64_t (&n)[3], const int64_t (&stride)[3], int64_t run) {
  if (n[0] <= 0 || n[1] <= 0 || n[2] <= 0) return true;
  int at[3], dims = 0;
  for (int i = 0; i < 3; ++i) {
    if (n[i] == 1) continue;
    if (stride[i] == 0) return false;
    int j = dims++;
    for (; j > 0 && stride[at[j - 1]] > stride[i]; --j) at[j] = at[j - 1];
    at[j] = i;
  }
  typedef __int128 wide;  // a stride times an index may pass 64 bits
  wide reach = run;
  bool nested = true;
  for (int i = 0; i < dims; ++i) {
    nested = nested && stride[at[i]] >= reach;
    reach += (wide)(n[at[i]] - 1) * stride[at[i]];
  }
  if (nested) return true;
  // The distance a of two indices in the other dimensions, one of each pair
  // d, -d, and the steps along the longest one that come nearest to it.
  int longest = 0;
  for (int i = 1; i < 3; ++i) longest = n[i] > n[longest] ? i : longest;
  const int u = (longest + 1) % 3, v = (longest + 2) % 3;
  const wide s = stride[longest];
  if (s < run) return false;
  for (int64_t i = 0; i < n[u]; ++i)
    for (int64_t j = i ? 1 - n[v] : 1; j < n[v]; ++j) {
      const wide d = (wide)i * stride[u] + (wide)j * stride[v], a = d < 0 ? -d : d;
      wide steps = (a + s / 2) / s;
      if (steps > n[longest] - 1) steps = n[longest] - 1;
      const wide gap = a - steps * s;
      if ((gap < 0 ? -gap : gap) < run) return false;
    }
  return true;
}

}  // namespace mkc
