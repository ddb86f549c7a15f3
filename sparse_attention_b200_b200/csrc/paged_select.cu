// Lists of pages from the scores of a ragged batch: what stands between the scorer and the attention over the paged cache.
//
//   best[row, page] = max over the list's tokens and the index heads of the KV head of scores[head, page, token]
//   the first `sink` and the last `recent` pages that the list's last token sees are always in the list
//   ids[kv head, row, :] = the top-k pages by (score descending, page ascending), written ascending, -1 behind them
//
// Pages that no token of the list sees, or whose scores are all -inf or NaN, are not listed. A list belongs to `tile`
// consecutive tokens of one request (first_list_row in paged.cuh).
//
// What bounds it: the latency of one pass over the scores (4 bytes per index head, page and token) and of the search. The
// scores lie with the tokens innermost, so a CTA takes neighbouring lists. The k-th largest key is found by halving the
// interval of values (not of bits: scores of one sign and size agree in their leading bits) between the smallest and the
// largest key until exactly k keys are at or above its lower end, about a dozen counts; after 16 of them the interval of keys,
// which ends whatever the values. The pages above the border are written in page order, at places that ballots or a prefix
// give: no sort, and a list lies as the sequence does.
//
// Many lists (select_many_kernel): 32 to a CTA, a lane's list is its lane number (a page's scores of 32 lists are one 128-byte
// line), a warp holds up to 64 pages of all of them in registers; a count is two instructions a key, a sum over the warps
// through shared memory and one barrier for 32 lists. Few lists (select_few_kernel): four to a CTA, so that a decode step uses
// more SMs, 512 threads for the loads; a warp then searches a list by itself (a count costs a redux, no barrier). 32,700 lists
// of up to 107 pages: 23 us with the first, 33 with the second; 270 lists of 256 pages and 16 index heads: 17 and 10 us. Both
// are bound by latency: the first takes 46 % of the issue slots (about 3500 instructions of a warp for its 64 places of 32
// lists), its warps wait for their loads and, once a count, for one another; the second for the requests that its lists belong
// to (about nine loads, one after another), one pass over the scores and a dozen counts.
#include "internal.h"
#include "paged.cuh"

namespace sb {
namespace {

struct SelectArgs {
  const float* scores;
  const int32_t *cu_q, *seq;
  int32_t* ids;
  int batch, group, pages, total_q, topk, tile, sink, recent, causal, lists;
};

// Ordered like the floats, the two zeros alike; -inf and NaN become 0, which no list takes.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  if (!(x > -INFINITY)) return 0;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

constexpr uint32_t FORCED = 0xffffffffu, ALL = 0xffffffffu;

struct List {
  int first, count, seen;                      // its tokens, and the pages that the last of them sees
};
__device__ __forceinline__ List find_list(const SelectArgs& a, int row) {
  List l{0, 0, 0};
  if (row >= a.lists) return l;
  const auto start = [&](int r) { return min(max(__ldg(a.cu_q + r), 0), a.total_q); };
  int r = 0, beyond = a.batch;                 // the last request whose lists begin at this row or before
  while (beyond - r > 1) {
    const int middle = (r + beyond) >> 1;
    if (first_list_row(start(middle), middle, a.tile) <= row) r = middle;
    else beyond = middle;
  }
  const int begin = start(r), end = start(r + 1), k = max(__ldg(a.seq + r), 0);
  const long long at = (row - first_list_row(begin, r, a.tile)) * a.tile;
  if (at >= 0 && at < end - begin) {
    l.first = begin + static_cast<int>(at);
    l.count = min(a.tile, end - l.first);
    const int keys_seen = a.causal ? k - (end - (l.first + l.count)) : k;
    l.seen = min(max((keys_seen >> 7) + ((keys_seen & 127) != 0), 0), a.pages);
  }
  return l;
}
__device__ __forceinline__ uint32_t middle_of(uint32_t border, uint32_t over, int step) {
  uint32_t trial = border + ((over - border) >> 1);
  if (step < 16) {
    const uint32_t x = ordered(0.5f * value_of(border) + 0.5f * value_of(over));
    if (x > border && x < over) trial = x;
  }
  return trial;
}

template <int WARPS>
__global__ void __launch_bounds__(32 * WARPS, WARPS == 2 ? 8 : 2) select_many_kernel(SelectArgs a) {
  constexpr int KEYS = 64;                     // pages of a warp at most
  __shared__ uint32_t s_top[WARPS][32], s_low[WARPS][32];
  __shared__ int s_count[2][WARPS][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int head = blockIdx.y, row = blockIdx.x * 32 + lane;
  const List list = find_list(a, row);
  const int each = (a.pages + WARPS - 1) / WARPS, page0 = warp * each, run = max(min(each, list.seen - page0), 0);
  const long long head_stride = static_cast<long long>(a.pages) * a.total_q;
  const float* from = a.scores + head * a.group * head_stride + static_cast<long long>(page0) * a.total_q + list.first;
  uint32_t key[KEYS];
#pragma unroll
  for (int i = 0; i < KEYS; ++i) key[i] = 0xff800000u;       // -inf
  for (int t = 0; t < list.count; ++t) {
    for (int h = 0; h < a.group; ++h) {
      const float* p = from + h * head_stride + t;
#pragma unroll
      for (int i = 0; i < KEYS; i += 16) {
        asm volatile("" : "+l"(p));            // one address at a time, not 64 of them in registers
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if (i + j < run) key[i + j] = __float_as_uint(fmaxf(__uint_as_float(key[i + j]), __ldg(p)));
          p += a.total_q;
        }
      }
    }
  }
  uint32_t next = 0, low = FORCED;             // one more than the largest key that is not forced, one less than the lowest
  int some = 0;                                // keys that can be taken
#pragma unroll
  for (int i = 0; i < KEYS; ++i) {
    const int page = page0 + i;
    key[i] = i >= run ? 0 : page < a.sink || page >= list.seen - a.recent ? FORCED : ordered(__uint_as_float(key[i]));
    some += key[i] != 0;
    next = max(next, key[i] + 1);
    low = min(low, key[i] - 1);
  }
  s_count[1][warp][lane] = some;
  s_top[warp][lane] = next;
  s_low[warp][lane] = low;
  __syncthreads();
  const auto over_warps = [&](int which) {
    int c = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) c += s_count[which][w][lane];
    return c;
  };
  some = over_warps(1);
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    next = max(next, s_top[w][lane]);
    low = min(low, s_low[w][lane]);
  }
  const int forced = min(a.sink + a.recent, list.seen);
  // Taken: keys above `border` and the first `equals` of those equal to it.
  uint32_t border = 1, over = 1;
  int equals = a.topk, above = forced;         // keys at or above `over`
  if (some > a.topk) {
    border = forced < a.topk ? low + 1 : FORCED;   // more than topk keys are at or above the lowest, fewer above the largest
    over = forced < a.topk ? next : FORCED;
  }
  bool open = over > border;
#pragma unroll 1
  for (int step = 0;; ++step) {
    const uint32_t trial = middle_of(border, over, step);
    if (open && over - border == 1) {
      open = false;
      equals = a.topk - above;
    }
    int c4[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < KEYS; ++i) c4[i & 3] += key[i] >= trial;
    int c = (c4[0] + c4[1]) + (c4[2] + c4[3]);
    s_count[step & 1][warp][lane] = c;
    if (!__syncthreads_or(open)) break;
    if (open) {
      c = over_warps(step & 1);
      if (c >= a.topk) {
        border = trial;
      } else {
        over = trial;
        above = c;
      }
      open = c != a.topk;                      // exactly topk: all of them are taken
    }
  }
  // places: keys above the border (65536 each) and equal to it in the runs before this one
  int here = 0;
#pragma unroll
  for (int i = 0; i < KEYS; ++i) here += key[i] > border ? 0x10000 : key[i] == border;
  __syncthreads();                             // the last counts have been read
  s_count[0][warp][lane] = here;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    const int x = s_count[0][w][lane];
    if (w < warp) before += x;
    total += x;
  }
  if (row >= a.lists) return;
  int32_t* out = a.ids + (static_cast<long long>(head) * a.lists + row) * a.topk;
  int place = (before >> 16) + min(before & 0xffff, equals);
  if ((total & 0xffff) <= equals) {            // all of those equal to the border
#pragma unroll
    for (int i = 0; i < KEYS; ++i)
      if (key[i] >= border) out[place++] = page0 + i;
  } else {
    int left = equals - min(before & 0xffff, equals);
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      const bool equal = key[i] == border;
      if (key[i] > border || (equal && left > 0)) out[place++] = page0 + i;
      left -= equal;
    }
  }
  for (int j = (total >> 16) + min(total & 0xffff, equals) + warp; j < a.topk; j += WARPS) out[j] = -1;
}

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
      const uint32_t trial = middle_of(border, over, step);
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

template <int ROWS, int KEYS>
__global__ void __launch_bounds__(512) select_few_kernel(SelectArgs a) {
  extern __shared__ uint32_t keys[];           // [ROWS][pages | 1]
  __shared__ int s_seen[ROWS];
  const int tid = threadIdx.x, mine = tid % ROWS, row0 = blockIdx.x * ROWS, head = blockIdx.y, pitch = a.pages | 1;
  const List list = find_list(a, row0 + mine);
  if (tid < ROWS) s_seen[tid] = list.seen;
  const long long head_stride = static_cast<long long>(a.pages) * a.total_q;
  const float* from = a.scores + head * a.group * head_stride + list.first;
  constexpr int STEP = 512 / ROWS;
  // two pages at a time, up to 16 heads of each in flight
  for (int page = tid / ROWS; page < list.seen; page += 2 * STEP) {
    const float* p = from + static_cast<long long>(page) * a.total_q;
    const bool two = page + STEP < list.seen;
    const long long second = two ? static_cast<long long>(STEP) * a.total_q : 0;
    float x = -INFINITY, y = -INFINITY;
    for (int t = 0; t < list.count; ++t) {
#pragma unroll 16
      for (int h = 0; h < a.group; ++h) {
        const float* at = p + h * head_stride + t;
        x = fmaxf(x, __ldg(at));
        y = fmaxf(y, __ldg(at + second));
      }
    }
    const auto key_of = [&](int j, float v) { return j < a.sink || j >= list.seen - a.recent ? FORCED : ordered(v); };
    keys[mine * pitch + page] = key_of(page, x);
    if (two) keys[mine * pitch + page + STEP] = key_of(page + STEP, y);
  }
  __syncthreads();
  const int i = tid >> 5;
  if (i < ROWS && row0 + i < a.lists)
    write_list<KEYS>(keys + i * pitch, s_seen[i], a.topk, a.ids + (static_cast<long long>(head) * a.lists + row0 + i) * a.topk);
}

template <int ROWS, int KEYS>
int launch_few(const SelectArgs& a, int heads, cudaStream_t stream) {
  const auto kernel = select_few_kernel<ROWS, KEYS>;
  const int smem = ROWS * (a.pages | 1) * 4;
  if (smem > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SELECT_SMEM) != cudaSuccess)
    return set_error(SB_ERR_CUDA, "shared memory of the page selection");
  kernel<<<dim3((a.lists + ROWS - 1) / ROWS, heads), 512, smem, stream>>>(a);
  return check_kernel_launch();
}
template <int WARPS>
int launch_many(const SelectArgs& a, int heads, cudaStream_t stream) {
  select_many_kernel<WARPS><<<dim3((a.lists + 31) / 32, heads), 32 * WARPS, 0, stream>>>(a);
  return check_kernel_launch();
}

}  // namespace

int launch_select_pages(const float* scores, const int32_t* cu_q, const int32_t* seq, int32_t* ids, int batch, int heads_in,
                        int heads, int pages, int total_q, int topk, int tile, int sink, int recent, int causal,
                        cudaStream_t stream) {
  DeviceCtx* ctx = device_ctx();
  if (!ctx) return SB_ERR_CUDA;
  const int lists = tile == 1 ? total_q : total_q / tile + batch;
  const SelectArgs a{scores, cu_q, seq, ids, batch, heads_in / heads, pages, total_q, topk, tile, sink, recent, causal, lists};
  if (static_cast<long long>(lists) * heads >= 32LL * ctx->sm_count) {
    if (pages <= 2 * 64) return launch_many<2>(a, heads, stream);
    if (pages <= 8 * 64) return launch_many<8>(a, heads, stream);
  }
  const auto fits = [&](int rows) { return rows * (pages | 1) * 4 <= SELECT_SMEM; };
  if (fits(4)) return pages <= 256 ? launch_few<4, 8>(a, heads, stream) : launch_few<4, 0>(a, heads, stream);
  return launch_few<1, 0>(a, heads, stream);       // (SELECT_MOST_PAGES)
}

}  // namespace sb
