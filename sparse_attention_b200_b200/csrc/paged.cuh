// What the kernels of the paged serving path share.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>
#include "internal.h"

namespace sb {

inline int check_kernel_launch() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SB_OK : set_error(SB_ERR_CUDA, cudaGetErrorString(e));
}

constexpr int PAGED_MAX_BATCH = 4096;      // requests of a step: their sums are held in shared memory
constexpr int SELECT_SMEM = 200 * 1024;    // of a CTA that holds the keys of whole lists
constexpr int SELECT_MOST_PAGES = SELECT_SMEM / 4 - 1;       // one list of (pages | 1) keys: 51199

// First place in the ascending a[0..n) whose value is above x.
__device__ __forceinline__ int upper_bound(const int* a, int n, int x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// The largest r of [0, n) with f(r) <= x for an ascending f with f(0) <= x, by a whole warp: 32 probes a round.
template <typename F>
__device__ __forceinline__ int warp_last_at_most(int n, long long x, F f) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = n;                      // f(lo) <= x; f(hi) > x or hi == n
  while (hi - lo > 1) {
    const int step = (hi - lo + 32) / 33;
    const int at = lo + (lane + 1) * step;
    const bool below = at < hi && f(at) <= x;
    const int c = __popc(__ballot_sync(0xffffffffu, below));
    hi = min(hi, lo + (c + 1) * step);
    lo += c * step;
  }
  return lo;
}

// Row of the list of a request's first tile, for lists that `tile` consecutive tokens of a request share: with tile 1 a
// token's list has the token's own row; else cu / tile + r, which leaves every request room for its tiles.
__device__ __forceinline__ long long first_list_row(int cu, int r, int tile) {
  return tile == 1 ? cu : static_cast<long long>(cu / tile) + r;
}

}  // namespace sb
