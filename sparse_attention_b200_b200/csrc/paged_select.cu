// Lists of pages from the scores of a ragged batch: what stands between the scorer and the attention over the paged cache.
//
//   best[row, page] = max over the list's tokens and the index heads of the KV head of scores[head, page, token]
//   the first `sink` and the last `recent` pages that the list's last token sees are always in the list
//   ids[kv head, row, :] = the top-k pages by (score descending, page ascending), written ascending, -1 behind them
//
// Pages that no token of the list sees, or whose scores are all -inf or NaN, are not listed. A list belongs to `tile`
// consecutive tokens of one request (first_list_row in paged.cuh).
//
// What bounds it: one pass over the scores (4 bytes per index head, page and token). They lie with the tokens innermost, so a
// CTA takes neighbouring lists, whose tokens fill the 32-byte sectors that it reads, and leaves the maxima as ordered 32-bit
// keys in shared memory, a row for each list. A warp then finds a list's k-th largest key bit by bit (counting keys at or
// above a trial value; it stops as soon as exactly k are) and writes the pages above it in page order, by ballots: no sort,
// and the lists come out as they lie in the sequence.
#include "internal.h"
#include "paged.cuh"

namespace sb {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;
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

template <int ROWS>
__global__ void __launch_bounds__(THREADS) select_pages_kernel(SelectArgs a) {
  extern __shared__ uint32_t keys[];
  __shared__ int s_first[ROWS], s_count[ROWS], s_seen[ROWS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int head = blockIdx.y;
  const int row0 = blockIdx.x * ROWS;
  // the tokens of each list and the pages that its last token sees
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
        seen = min(max((keys_seen + 127) >> 7, 0), a.pages);
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
  const int mine = tid % ROWS;
  const int seen = s_seen[mine], count = s_count[mine];
  const float* from = scores + s_first[mine];
#pragma unroll 2
  for (int page = tid / ROWS; page < a.pages; page += STEP) {
    uint32_t key = 0;
    if (page < seen) {
      if (page < a.sink || page >= seen - a.recent) {
        key = 0xffffffffu;
      } else {
        const float* p = from + static_cast<long long>(page) * a.total_q;
        float best = -INFINITY;
        for (int t = 0; t < count; ++t) {
#pragma unroll 8
          for (int h = 0; h < a.group; ++h) best = fmaxf(best, __ldg(p + h * head_stride + t));
        }
        key = ordered(best);
      }
    }
    keys[mine * a.pitch + page] = key;
  }
  __syncthreads();
  for (int i = warp; i < ROWS; i += WARPS) {
    if (row0 + i >= a.lists) break;
    const uint32_t* k = keys + i * a.pitch;
    const int n = s_seen[i];
    int32_t* out = a.ids + (static_cast<long long>(head) * a.lists + row0 + i) * a.topk;
    const auto at_least = [&](uint32_t x) {
      int c = 0;
      for (int j = lane; j < n; j += 32) c += k[j] >= x;
      return __reduce_add_sync(0xffffffffu, c);
    };
    // the largest `least` with at least topk keys at or above it; 1 where there are not that many
    uint32_t least = 1;
    int above = at_least(1);
    bool exact = above <= a.topk;
    if (!exact) {
      least = 0;
      for (int bit = 31; bit >= 0; --bit) {
        const uint32_t trial = least | (1u << bit);
        const int c = at_least(trial);
        if (c >= a.topk) {
          least = trial;
          above = c;
          if (c == a.topk) {
            exact = true;
            break;
          }
        }
      }
    }
    // keys above `least`, and of those equal to it the first few
    int equal_room = a.topk;
    if (!exact) equal_room = a.topk - (least == 0xffffffffu ? 0 : at_least(least + 1));
    int written = 0;
    for (int base = 0; base < n && written < a.topk; base += 32) {
      const int j = base + lane;
      const uint32_t key = j < n ? k[j] : 0;
      const uint32_t equal = __ballot_sync(0xffffffffu, !exact && key == least);
      const int rank = __popc(equal & ((1u << lane) - 1));
      const bool in = exact ? key >= least : key > least || (key == least && rank < equal_room);
      const uint32_t taken = __ballot_sync(0xffffffffu, in);
      if (in) out[written + __popc(taken & ((1u << lane) - 1))] = j;
      written += __popc(taken);
      equal_room -= min(equal_room, __popc(equal));
    }
    for (int j = written + lane; j < a.topk; j += 32) out[j] = -1;
  }
}

template <int ROWS>
int launch(const SelectArgs& a, DeviceCtx* ctx, int slot, cudaStream_t stream) {
  if (!ctx->paged_attr[slot]) {
    if (cudaFuncSetAttribute(select_pages_kernel<ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MOST) != cudaSuccess)
      return set_error(SB_ERR_CUDA, "shared memory of the page selection");
    ctx->paged_attr[slot] = 1;
  }
  select_pages_kernel<ROWS><<<dim3((a.lists + ROWS - 1) / ROWS, a.heads), THREADS, ROWS * a.pitch * 4, stream>>>(a);
  return check_kernel_launch();
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
  if (fits(32) && lists * heads >= 32LL * ctx->sm_count) return launch<32>(a, ctx, 1, stream);
  if (fits(8)) return launch<8>(a, ctx, 2, stream);
  return launch<1>(a, ctx, 3, stream);
}

}  // namespace sb
