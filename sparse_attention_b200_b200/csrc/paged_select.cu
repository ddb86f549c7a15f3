// Lists of pages from the scores of a ragged batch: what stands between the scorer and the attention over the paged cache.
//
//   best[row, page] = max over the list's tokens and the index heads of the KV head of scores[head, page, token]
//   the first `sink` and the last `recent` pages that the list's last token sees are always in the list
//   ids[kv head, row, :] = the top-k pages by (score descending, page ascending), written ascending, -1 behind them
//
// Pages that no token of the list sees, or whose scores are all -inf or NaN, are not listed. A list belongs to `tile`
// consecutive tokens of one request (first_list_row in paged.cuh).
//
// What bounds it: the latency of one pass over the scores (4 bytes per index head, page and token) in a decode step, the
// searches in a prompt. The scores lie with the tokens innermost, so a CTA takes neighbouring lists, whose tokens fill (or half
// fill) the 32-byte sectors that it reads, and leaves the maxima as ordered 32-bit keys in shared memory, a row for each list.
// A warp then takes a list's keys into registers (up to 16 a lane) and finds a border with exactly k keys at or above it, or
// the k-th key and how many of its equals are taken: it halves the interval of values (not of bits: scores of one sign and
// size agree in their leading bits) between the smallest and the largest key, about ten counts of a few instructions and a
// redux each; after 16 of them the interval of keys, which ends whatever the values. The pages above the border are written in
// page order by ballots: no sort, and a list lies as the sequence does.
#include "internal.h"
#include "paged.cuh"

namespace sb {
namespace {

constexpr int SMEM_MOST = 200 * 1024;

struct SelectArgs {
  const float* scores;
  const int32_t *cu_q, *seq;
  int32_t* ids;
  int batch, group, pages, total_q, topk, tile, sink, recent, causal, lists, heads;
  int pitch;                               // keys of a list in shared memory
};

// Ordered like the floats, the two zeros alike; -inf and NaN become 0, which no list takes.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  if (!(x > -INFINITY)) return 0;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

constexpr uint32_t FORCED = 0xffffffffu;

// Writes the list of the n keys k[0..n) (shared memory). KEYS > 0: at most 32 KEYS of them, held in registers.
template <int KEYS>
__device__ __forceinline__ void write_list(const uint32_t* k, int n, int topk, int32_t* out) {
  const int lane = threadIdx.x & 31;
  uint32_t mine[KEYS ? KEYS : 1];
  uint32_t top = 0, low = FORCED;
  int some = 0, forced = 0;
  const auto look = [&](uint32_t x) {
    some += x != 0;
    forced += x == FORCED;
    if (x != 0 && x != FORCED) {
      top = max(top, x);
      low = min(low, x);
    }
  };
  if constexpr (KEYS > 0) {
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      const int j = 32 * i + lane;
      mine[i] = j < n ? k[j] : 0;
      look(mine[i]);
    }
  } else {
    for (int j = lane; j < n; j += 32) look(k[j]);
  }
  const auto at_least = [&](uint32_t x) {
    int c = 0;
    if constexpr (KEYS > 0) {
#pragma unroll
      for (int i = 0; i < KEYS; ++i) c += mine[i] >= x;
    } else {
      for (int j = lane; j < n; j += 32) c += k[j] >= x;
    }
    return static_cast<int>(__reduce_add_sync(FORCED, c));
  };
  some = __reduce_add_sync(FORCED, some);
  forced = __reduce_add_sync(FORCED, forced);
  uint32_t border = 1;                     // taken: keys above it, and the first `equals` of those equal to it
  int equals = topk;
  if (some > topk && forced < topk) {
    top = __reduce_max_sync(FORCED, top);
    low = __reduce_min_sync(FORCED, low);
    // more than topk keys are at or above low, fewer than topk above top
    border = low;
    uint32_t over = top + 1;
    int above = forced;                    // keys at or above `over`
    equals = 0;
    for (int step = 0; over - border > 1; ++step) {
      uint32_t trial = border + ((over - border) >> 1);
      if (step < 16) {
        const float middle = 0.5f * value_of(border) + 0.5f * value_of(over);
        const uint32_t x = ordered(middle);
        if (x > border && x < over) trial = x;
      }
      const int c = at_least(trial);
      if (c == topk) {
        border = trial;
        equals = topk;
        break;
      }
      if (c > topk) {
        border = trial;
      } else {
        over = trial;
        above = c;
      }
    }
    if (equals == 0) equals = topk - above;
  } else if (some > topk) {
    border = FORCED;                       // the forced pages fill the list
  }
  int written = 0;
  const auto emit = [&](uint32_t key, int j) {
    const uint32_t equal = __ballot_sync(FORCED, key == border);
    const bool in = key > border || (key == border && __popc(equal & ((1u << lane) - 1)) < equals);
    const uint32_t taken = __ballot_sync(FORCED, in);
    if (in) out[written + __popc(taken & ((1u << lane) - 1))] = j;
    written += __popc(taken);
    equals -= min(equals, __popc(equal));
  };
  if constexpr (KEYS > 0) {
#pragma unroll
    for (int i = 0; i < KEYS; ++i)
      if (32 * i < n) emit(mine[i], 32 * i + lane);
  } else {
    for (int base = 0; base < n && written < topk; base += 32) emit(base + lane < n ? k[base + lane] : 0, base + lane);
  }
  for (int j = written + lane; j < topk; j += 32) out[j] = -1;
}

// SINGLE: a list has one token and one index head
template <int ROWS, int THREADS, int KEYS, bool SINGLE>
__global__ void __launch_bounds__(THREADS) select_pages_kernel(SelectArgs a) {
  constexpr int WARPS = THREADS / 32;
  extern __shared__ uint32_t keys[];
  __shared__ int s_first[ROWS], s_count[ROWS], s_seen[ROWS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int head = blockIdx.y;
  const int row0 = blockIdx.x * ROWS;
  // the tokens of each list and the pages that its last token sees
#pragma unroll 1
  for (int i = warp; i < ROWS; i += WARPS) {
    const int row = row0 + i;
    int first = 0, count = 0, seen = 0;
    if (row < a.lists) {
      const auto start = [&](int r) { return min(max(__ldg(a.cu_q + r), 0), a.total_q); };
      const int r = warp_last_at_most(a.batch, row, [&](int q) { return first_list_row(start(q), q, a.tile); });
      const int begin = start(r), end = start(r + 1);
      const long long at = (row - first_list_row(begin, r, a.tile)) * a.tile;
      if (at >= 0 && at < end - begin) {
        first = begin + static_cast<int>(at);
        count = min(a.tile, end - first);
        const int k = max(__ldg(a.seq + r), 0);
        const int keys_seen = a.causal ? k - (end - (first + count)) : k;
        seen = min(max((keys_seen >> 7) + ((keys_seen & 127) != 0), 0), a.pages);
      }
    }
    if (lane == 0) {
      s_first[i] = first;
      s_count[i] = count;
      s_seen[i] = seen;
    }
  }
  __syncthreads();
  const float* scores = a.scores + static_cast<long long>(head) * a.group * a.pages * a.total_q;
  const long long head_stride = static_cast<long long>(a.pages) * a.total_q;
  constexpr int STEP = THREADS / ROWS;
  const int mine = tid % ROWS, page0 = tid / ROWS;
  const int seen = s_seen[mine], count = s_count[mine];
  const float* from = scores + s_first[mine];
  uint32_t* row = keys + mine * a.pitch;
  const auto always = [&](int page) { return page < a.sink || page >= seen - a.recent; };
  if constexpr (SINGLE) {
    constexpr int AHEAD = 8;               // loads in flight
    for (int page = page0; page < seen; page += AHEAD * STEP) {
      float x[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (page + i * STEP < seen) x[i] = __ldg(from + static_cast<long long>(page + i * STEP) * a.total_q);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (page + i * STEP < seen) row[page + i * STEP] = always(page + i * STEP) ? FORCED : ordered(x[i]);
    }
  } else {
    for (int page = page0; page < seen; page += STEP) {
      uint32_t key = FORCED;
      if (!always(page)) {
        const float* p = from + static_cast<long long>(page) * a.total_q;
        float best = -INFINITY;
        for (int t = 0; t < count; ++t) {
#pragma unroll 16
          for (int h = 0; h < a.group; ++h) best = fmaxf(best, __ldg(p + h * head_stride + t));
        }
        key = ordered(best);
      }
      row[page] = key;
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int i = warp; i < ROWS; i += WARPS) {
    if (row0 + i >= a.lists) break;
    write_list<KEYS>(keys + i * a.pitch, s_seen[i], a.topk, a.ids + (static_cast<long long>(head) * a.lists + row0 + i) * a.topk);
  }
}

template <int ROWS, int THREADS, int KEYS, bool SINGLE>
int launch(const SelectArgs& a, cudaStream_t stream) {
  const auto kernel = select_pages_kernel<ROWS, THREADS, KEYS, SINGLE>;
  const int smem = ROWS * a.pitch * 4;
  if (smem > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MOST) != cudaSuccess)
    return set_error(SB_ERR_CUDA, "shared memory of the page selection");
  kernel<<<dim3((a.lists + ROWS - 1) / ROWS, a.heads), THREADS, smem, stream>>>(a);
  return check_kernel_launch();
}

template <int ROWS, int THREADS, bool SINGLE>
int launch(const SelectArgs& a, cudaStream_t stream) {
  return a.pages <= 128   ? launch<ROWS, THREADS, 4, SINGLE>(a, stream)
         : a.pages <= 512 ? launch<ROWS, THREADS, 16, SINGLE>(a, stream)
                          : launch<ROWS, THREADS, 0, SINGLE>(a, stream);
}

}  // namespace

int launch_select_pages(const float* scores, const int32_t* cu_q, const int32_t* seq, int32_t* ids, int batch, int heads_in,
                        int heads, int pages, int total_q, int topk, int tile, int sink, int recent, int causal,
                        cudaStream_t stream) {
  DeviceCtx* ctx = device_ctx();
  if (!ctx) return SB_ERR_CUDA;
  const long long lists = tile == 1 ? total_q : total_q / tile + batch;
  SelectArgs a{scores, cu_q, seq, ids, batch, heads_in / heads, pages, total_q, topk, tile, sink, recent, causal,
               static_cast<int>(lists), heads, pages | 1};      // odd pitch: neighbouring lists' keys of a page meet no bank twice
  const auto fits = [&](int rows) { return rows * a.pitch * 4 <= SMEM_MOST; };
  if (!fits(1)) return set_error(SB_ERR_INVALID, "too many pages for the page selection");
  const bool single = tile == 1 && a.group == 1;
  // 32 lists to a CTA read whole 128-byte lines; where that leaves SMs idle, four, with the loads spread over 512 threads
  if (fits(32) && lists * heads >= 32LL * ctx->sm_count) return single ? launch<32, 256, true>(a, stream) : launch<32, 256, false>(a, stream);
  if (fits(4)) return single ? launch<4, 512, true>(a, stream) : launch<4, 512, false>(a, stream);
  return launch<1, 512, 0, false>(a, stream);
}

}  // namespace sb
