// Tables of a serving step, from the requests' lengths alone: pages are taken from a free stack, the block table is
// extended, and the slot map, the cumulative lengths and the flat page list that the scorer, the cache writer and the
// attention read are written. One launch, no atomics.
//
//   need_r  = ceil((o_r + n_r) / 128) - ceil(o_r / 128)        new pages of request r (o_r cached, n_r new tokens)
//   upto_r  = need_0 + ... + need_r
//   request r is refused (its length stays, its slots are -1) when its pages do not fit its table row, or when it needs
//   pages and upto_r exceeds the free pages; need_r of a row that is too short counts as 0
//   page i of request r's new ones = free_pages[free_count - 1 - (upto_r - need_r) - i]
//
// What bounds it: a dependent chain of a few loads and two block scans; the arrays are small. Every CTA therefore runs the
// scans over all requests itself (they sit in L2) instead of waiting for another launch, keeps the sums in shared memory
// and writes its share of the slots and pages, whose requests it finds by binary search there. 48 requests of a token each:
// 6.3 us in a graph, 768 requests of up to 128 tokens and 32768 keys (1.2 MB): 10.3 us; the call's host side takes 18.
#include "internal.h"
#include "paged.cuh"

namespace sb {
namespace {

constexpr int THREADS = 256;

struct Sums {
  long long new_tokens, kv_tokens;
  int pages;                             // at most batch * width, below 2^31
};

__device__ __forceinline__ Sums add(const Sums& a, const Sums& b) {
  return {a.new_tokens + b.new_tokens, a.kv_tokens + b.kv_tokens, a.pages + b.pages};
}

__device__ __forceinline__ Sums shift_up(const Sums& a, int by) {
  return {__shfl_up_sync(0xffffffffu, a.new_tokens, by), __shfl_up_sync(0xffffffffu, a.kv_tokens, by),
          __shfl_up_sync(0xffffffffu, a.pages, by)};
}

__device__ __forceinline__ int saturated(long long x) { return x > 0x7fffffffLL ? 0x7fffffff : static_cast<int>(x); }

__global__ void __launch_bounds__(THREADS) extend_pages_kernel(
    int32_t* __restrict__ table, long long table_stride, int width, const int32_t* __restrict__ seq,
    const int32_t* __restrict__ added, const int32_t* __restrict__ free_pages, int free_capacity,
    const int32_t* __restrict__ free_count, int32_t* __restrict__ seq_out, int32_t* __restrict__ cu_q,
    int32_t* __restrict__ cu_k, int32_t* __restrict__ cu_pages, int32_t* __restrict__ kv_indices,
    long long* __restrict__ slots, int32_t* __restrict__ free_out, int32_t* __restrict__ status, int batch, int total_q,
    int total_pages) {
  extern __shared__ int shared[];
  int* s_q = shared;                     // cu_q, batch + 1
  int* s_pages = s_q + batch + 1;        // cu_pages, batch + 1
  int* s_taken = s_pages + batch + 1;    // upto_r - need_r; -1: refused
  int* s_old = s_taken + batch;          // cached tokens
  __shared__ Sums w_sums[THREADS / 32];
  __shared__ long long w_need[THREADS / 32];
  __shared__ int s_status, s_used;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool first = blockIdx.x == 0;
  const long long available = min(max(__ldg(free_count), 0), free_capacity);
  if (tid == 0) s_status = s_used = 0;
  // requests of this thread: [lo, hi)
  const int each = (batch + THREADS - 1) / THREADS;
  const int lo = min(tid * each, batch), hi = min(lo + each, batch);
  const auto old_of = [&](int r) { return max(__ldg(seq + r), 0); };
  const auto new_of = [&](int r) { return max(__ldg(added + r), 0); };
  const auto pages_of = [](long long n) { return (n + 127) >> 7; };
  const auto need_of = [&](int r, bool& wide) {
    const long long o = old_of(r), after = pages_of(o + new_of(r));
    wide = after > width;
    return wide ? 0LL : after - pages_of(o);
  };
  long long need = 0;
  for (int r = lo; r < hi; ++r) {
    bool wide;
    need += need_of(r, wide);
  }
  long long before = need;
  for (int by = 1; by < 32; by <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, before, by);
    if (lane >= by) before += x;
  }
  if (lane == 31) w_need[warp] = before;
  before -= need;
  __syncthreads();
  for (int w = 0; w < warp; ++w) before += w_need[w];
  Sums mine{0, 0, 0};
  int flags = 0, used = 0;
  for (int r = lo; r < hi; ++r) {
    bool wide;
    const long long n_need = need_of(r, wide);
    const bool is_short = n_need > 0 && before + n_need > available;
    const bool granted = !wide && !is_short;
    flags |= (is_short ? 1 : 0) | (wide ? 2 : 0);
    const int o = old_of(r), n = new_of(r);
    const int k = granted ? o + n : o;      // o + n <= 128 width, or n == 0
    s_old[r] = o;
    s_taken[r] = granted ? static_cast<int>(before) : -1;      // (needs add up to batch * width at most)
    if (granted && n_need > 0) used = static_cast<int>(before + n_need);     // (without need: `before` counts refused requests too)
    if (first) seq_out[r] = k;
    mine = add(mine, {n, k, static_cast<int>(min(pages_of(k), static_cast<long long>(width)))});
    before += n_need;
  }
  if (flags) atomicOr(&s_status, flags);
  if (used) atomicMax(&s_used, used);
  Sums upto = mine;
  for (int by = 1; by < 32; by <<= 1) {
    const Sums x = shift_up(upto, by);
    if (lane >= by) upto = add(upto, x);
  }
  if (lane == 31) w_sums[warp] = upto;
  upto = {upto.new_tokens - mine.new_tokens, upto.kv_tokens - mine.kv_tokens, upto.pages - mine.pages};
  __syncthreads();
  for (int w = 0; w < warp; ++w) upto = add(upto, w_sums[w]);
  for (int r = lo; r < hi; ++r) {
    const int o = s_old[r], n = new_of(r);
    const int k = s_taken[r] >= 0 ? o + n : o;
    s_q[r] = saturated(upto.new_tokens);
    s_pages[r] = upto.pages;
    if (first) {
      cu_q[r] = saturated(upto.new_tokens);
      cu_k[r] = saturated(upto.kv_tokens);
      cu_pages[r] = min(upto.pages, total_pages);      // (who reads kv_indices by it stays within)
    }
    upto = add(upto, {n, k, static_cast<int>(min(pages_of(k), static_cast<long long>(width)))});
  }
  if (hi == batch && (lo < hi || tid == 0)) {      // the thread of the last request holds the totals (batch >= 1)
    s_q[batch] = saturated(upto.new_tokens);
    s_pages[batch] = upto.pages;
    if (first) {
      cu_q[batch] = saturated(upto.new_tokens);
      cu_k[batch] = saturated(upto.kv_tokens);
      cu_pages[batch] = min(upto.pages, total_pages);
      *free_out = static_cast<int>(available) - s_used;
      *status = s_status | (upto.new_tokens > total_q ? 4 : 0) | (upto.pages > total_pages ? 8 : 0) |
                (upto.kv_tokens > 0x7fffffffLL || upto.new_tokens > 0x7fffffffLL ? 16 : 0);
    }
  }
  __syncthreads();
  const auto page_of = [&](int r, int j) {         // page j of request r after this step
    const int held = static_cast<int>(pages_of(s_old[r]));
    if (j >= held) return s_taken[r] < 0 ? -1 : __ldg(free_pages + (available - 1 - s_taken[r] - (j - held)));
    return table[r * table_stride + j];
  };
  const unsigned stride = gridDim.x * THREADS, start = blockIdx.x * THREADS + tid;      // (unsigned: ends may be near 2^31)
  const unsigned all_pages = max(s_pages[batch], total_pages);
  for (unsigned i = start; i < all_pages; i += stride) {
    const int j = static_cast<int>(i);
    int page = -1;
    if (j < s_pages[batch]) {
      const int r = upper_bound(s_pages, batch + 1, j) - 1;
      const int at = j - s_pages[r];
      page = page_of(r, at);
      // entries behind the held ones are written here and read by no other thread of this launch
      if (at >= pages_of(s_old[r])) table[r * table_stride + at] = page;
    }
    if (j < total_pages) kv_indices[j] = page;
  }
  for (unsigned i = start; i < static_cast<unsigned>(total_q); i += stride) {
    const int t = static_cast<int>(i);
    long long slot = -1;
    if (t < s_q[batch]) {
      const int r = upper_bound(s_q, batch + 1, t) - 1;
      if (s_taken[r] >= 0) {
        const int p = s_old[r] + (t - s_q[r]);
        const int page = page_of(r, p >> 7);
        if (page >= 0) slot = static_cast<long long>(page) * 128 + (p & 127);
      }
    }
    slots[t] = slot;
  }
}

}  // namespace

int launch_extend_pages(int32_t* table, long long table_stride, int width, const int32_t* seq, const int32_t* added,
                        const int32_t* free_pages, int free_capacity, const int32_t* free_count, int32_t* seq_out,
                        int32_t* cu_q, int32_t* cu_k, int32_t* cu_pages, int32_t* kv_indices, long long* slots,
                        int32_t* free_out, int32_t* status, int batch, int total_q, int total_pages, cudaStream_t stream) {
  DeviceCtx* ctx = device_ctx();
  if (!ctx) return SB_ERR_CUDA;
  const int smem = (4 * batch + 2) * static_cast<int>(sizeof(int));
  if (!ctx->paged_attr[0]) {
    if (cudaFuncSetAttribute(extend_pages_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (4 * PAGED_MAX_BATCH + 2) * static_cast<int>(sizeof(int))) != cudaSuccess)
      return set_error(SB_ERR_CUDA, "shared memory of the page tables kernel");
    ctx->paged_attr[0] = 1;
  }
  const long long most = max(total_q, total_pages);
  const int grid = static_cast<int>(max(1LL, min((most + 4 * THREADS - 1) / (4 * THREADS), static_cast<long long>(ctx->sm_count))));
  extend_pages_kernel<<<grid, THREADS, smem, stream>>>(table, table_stride, width, seq, added, free_pages, free_capacity,
                                                       free_count, seq_out, cu_q, cu_k, cu_pages, kv_indices, slots,
                                                       free_out, status, batch, total_q, total_pages);
  return check_kernel_launch();
}

}  // namespace sb
