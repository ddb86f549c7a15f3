// What the two kernels of the attention over the 8-bit paged cache share: the work of a request, how it is cut in shares, the
// walk over a share's pages and what its warp tells the others, waits.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include "internal.h"
#include "paged.cuh"
#include "ptx.cuh"

namespace sb {
namespace pa {

constexpr int TILE_BYTES = 128 * 128;             // the codes of K or V of a page and head
// What the loader tells the other warps: batches of up to 32 pages of an item. Header (two int4): flags, pages, first token,
// tokens; KV head, place of the part (-1: the item lies in this share alone), first and last share of the item. Pages (int4
// each): row of the page in the cache (page * Hkv + head), keys it holds | keys its first token sees << 16, the two scales.
constexpr int BATCHES = 4, BATCH_BYTES = 32 + 32 * 16;
constexpr int FIRST = 1, LAST = 2, STOP = 4;      // first batch of an item, last one; there are no more

struct Params {
  PagedAttentionArgs a;
  int group, pack, pack_shift, tile_shift, ctas;
  int rows;                                       // of an item at most: 16, or 128 (wide kernel)
  float* part_o;                                  // [2 ctas, rows, 128]
  float* part_ml;                                 // [2 ctas, rows, 2]
  int* part_meta;                                 // [2 ctas, 8]
};


__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  f32x2_unpack(f32x2_mul(f32x2_pack(a.x, a.y), f32x2_pack(b.x, b.y)), d.x, d.y);
  return d;
}
// A wait by a whole converged warp whose slow part is not in line: a role's loop has to fit the instruction caches beside the
// others' (the first build of this kernel had 164 KB of code and ran at a fifth of its speed).
static __device__ __noinline__ bool wait_longer(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  return mbar_wait_warp(bar, parity, Guard{abort_flag, status}, code);
}
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, const Guard& g, int code) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return wait_longer(bar, parity, g.abort_flag, g.status, code);
}
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ float2 from_e4m3x2(uint32_t codes) {
  return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes), __NV_E4M3)));
}
__device__ __forceinline__ float from_e4m3(uint32_t code) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(code), __NV_E4M3)));
}

// ------------------------------------------------------------------ the work of a request
struct Request {
  int begin, n, k_len, held, tiles;
  __device__ __forceinline__ void set(const Params& p, int cu0, int cu1, int seq) {
    begin = min(max(cu0, 0), p.a.total_q);
    n = max(min(max(cu1, 0), p.a.total_q) - begin, 0);
    k_len = max(seq, 0);
    held = min((k_len >> 7) + ((k_len & 127) != 0), p.a.width);
    tiles = static_cast<int>((static_cast<long long>(n) + p.pack - 1) >> p.pack_shift);
  }
};
// Pages of the first `tiles` tiles of a request: a list's length each, or the pages that a tile's last token sees (one at
// least, so that every item has a place): min(held, ceil((k - n + (i + 1) pack) / 128)) summed over i. With pack = 128 / m the
// ceiling is floor((first + i) / m), whose sums have a closed form.
static __device__ __noinline__ long long pages_before(int topk, int causal, int shift, int k_len, int n, int held, int tiles) {
  if (topk) return static_cast<long long>(tiles) * topk;
  const long long most = max(held, 1);
  if (!causal) return tiles * most;
  const int mshift = 7 - shift, m = 1 << mshift;
  const long long first = ((static_cast<long long>(k_len) - n + 127) >> shift) + 1;
  const auto clamp = [&](long long x) { return x < 0 ? 0 : x > tiles ? tiles : x; };
  const long long ones = clamp(m - first), full = max(clamp(most * m - first), ones);
  const auto sum = [&](long long x) {             // sum of floor(t / m) over 0 <= t < x
    const long long q = x >> mshift, rest = x & (m - 1);
    return m * (q * (q - 1) / 2) + rest * q;
  };
  const long long middle = full > ones ? sum(first + full) - sum(first + ones) : 0;
  return ones + middle + (tiles - full) * most;
}
__device__ __forceinline__ long long pages_before(const Params& p, const Request& r, int tiles) {
  return pages_before(p.a.topk, p.a.causal, p.pack_shift, r.k_len, r.n, r.held, tiles);
}
__device__ __forceinline__ long long pages_of_request(const Params& p, int r) {
  Request q;
  q.set(p, __ldg(p.a.cu_q + r), __ldg(p.a.cu_q + r + 1), __ldg(p.a.seq + r));
  return pages_before(p, q, q.tiles);
}

// ------------------------------------------------------------------ shares
struct Share {
  long long share, unit0, unit1, total, off;      // pages of a CTA; this CTA's [unit0, unit1) of all; unit0 within its request
  int head, request;                              // where it begins
};
// The share of this CTA, by all its threads: a scan over the requests' pages.
template <int WARPS>
__device__ __forceinline__ Share find_share(const Params& p) {
  __shared__ long long s_scan[WARPS];
  __shared__ long long s_place[2];                // unit within the request, request
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int each = (p.a.batch + 32 * WARPS - 1) / (32 * WARPS);
  const int lo = min(tid * each, p.a.batch), hi = min(lo + each, p.a.batch);
  long long mine = 0;
#pragma unroll 1
  for (int r = lo; r < hi; ++r) mine += pages_of_request(p, r);
  long long upto = mine;
  for (int by = 1; by < 32; by <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, upto, by);
    if (lane >= by) upto += x;
  }
  if (lane == 31) s_scan[warp] = upto;
  __syncthreads();
  long long per_head = 0;
  upto -= mine;
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) upto += s_scan[w];
    per_head += s_scan[w];
  }
  Share s;
  s.total = per_head * p.a.hkv;
  s.share = max((s.total + p.ctas - 1) / p.ctas, 1LL);
  s.unit0 = blockIdx.x * s.share;
  s.unit1 = min(s.unit0 + s.share, s.total);
  s.head = s.unit0 < s.total ? static_cast<int>(s.unit0 / per_head) : 0;
  if (s.unit0 < s.total) {
    long long at = s.unit0 - s.head * per_head - upto;
    if (at >= 0 && at < mine) {
#pragma unroll 1
      for (int r = lo; r < hi; ++r) {
        const long long w = pages_of_request(p, r);
        if (at < w) {
          s_place[0] = at;
          s_place[1] = r;
          break;
        }
        at -= w;
      }
    }
  }
  __syncthreads();
  s.off = s_place[0];
  s.request = static_cast<int>(s_place[1]);
  return s;
}

// An item, or the part of it that lies in this share.
struct Item {
  int token0, tokens, head, place, x0, x1, k_len;
  long long seen0;                                // keys that its first token sees; the others one more each (causal)
};
// Walks over the items of a share, by a whole warp: batch(item, flags, pages, row, j) for up to 32 places of an item's list or
// table row, one per lane; pages: the lanes whose place holds a page that is taken, row: page * Hkv + head, j: its number in
// the request. Batches without a page are left out but for an item's last.
template <typename F>
__device__ __forceinline__ void walk_share(const Params& p, const Share& s, const bool& ok, F batch) {
  if (s.unit0 >= s.total) return;
  const int lane = threadIdx.x & 31;
  long long left = s.unit1 - s.unit0, off = s.off;
  int head = s.head, r = s.request;
  // requests come 32 at a time, one per lane
  int block = -1, c0 = 0, c1 = 0, sq = 0;
  Request q;
  const auto fetch = [&](int want) {
    if (want >> 5 != block) {
      block = want >> 5;
      const int i = block * 32 + lane;
      const bool in = i < p.a.batch;
      c0 = in ? __ldg(p.a.cu_q + i) : 0;
      c1 = in ? __ldg(p.a.cu_q + i + 1) : 0;
      sq = in ? __ldg(p.a.seq + i) : 0;
    }
    q.set(p, __shfl_sync(0xffffffffu, c0, want & 31), __shfl_sync(0xffffffffu, c1, want & 31),
          __shfl_sync(0xffffffffu, sq, want & 31));
  };
  fetch(r);
  int tile = warp_last_at_most(q.tiles, off, [&](int t) { return pages_before(p, q, t); });
  off -= pages_before(p, q, tile);
  long long start = s.unit0 - off;                // first unit of the item
  while (ok && left > 0) {
    Item item;
    const int first = tile * p.pack;
    item.tokens = min(p.pack, q.n - first);
    item.token0 = q.begin + first;
    item.head = head;
    item.k_len = q.k_len;
    item.seen0 = p.a.causal ? static_cast<long long>(q.k_len) - q.n + first + 1 : q.k_len;
    const long long seen = p.a.causal ? item.seen0 + item.tokens - 1 : q.k_len;
    const int count = static_cast<int>(pages_before(p, q, tile + 1) - pages_before(p, q, tile));
    const int from = static_cast<int>(off), to = static_cast<int>(min(static_cast<long long>(count), off + left));
    item.x0 = static_cast<int>(start / s.share);
    item.x1 = static_cast<int>((start + count - 1) / s.share);
    item.place = item.x0 == item.x1 ? -1 : 2 * static_cast<int>(blockIdx.x) + (item.x0 == static_cast<int>(blockIdx.x));
    bool posted = false;
    const int32_t* list = nullptr;
    if (p.a.ids) {
      const int sh = p.tile_shift;
      const long long lists = sh ? (p.a.total_q >> sh) + p.a.batch : p.a.total_q;
      list = p.a.ids + (head * lists + (q.begin >> sh) + (sh ? r : 0) + (first >> sh)) * p.a.topk;
    }
    const int32_t* table = p.a.table + r * p.a.table_stride;
#pragma unroll 1
    for (int at = from; ok && at < to; at += 32) {
      int j = at + lane;
      bool live = j < to;
      if (live && list) j = __ldg(list + j);
      live = live && j >= 0 && j < q.held && j * 128LL < seen;
      int row = 0;
      if (live) {
        const int page = __ldg(table + j);
        live = page >= 0 && page < p.a.pages;
        row = live ? page * p.a.hkv + head : 0;
      }
      const uint32_t pages = __ballot_sync(0xffffffffu, live);
      const bool last = at + 32 >= to;
      if (!pages && !last) continue;
      batch(item, (posted ? 0 : FIRST) | (last ? LAST : 0), pages, row, j);
      posted = true;
    }
    left -= to - from;
    start += count;
    off = 0;
    if (++tile >= q.tiles && left > 0) {          // the next request that has tokens; behind the last one the next head
      tile = 0;
      do {
        if (++r == p.a.batch) {
          r = 0;
          ++head;
        }
        fetch(r);
      } while (q.tiles == 0);
    }
  }
}
// What a batch tells, written by the walking warp to its place (see BATCH_BYTES).
__device__ __forceinline__ void write_batch(const Params& p, int4* to, const Item& item, int flags, uint32_t pages, int row, int j) {
  const int lane = threadIdx.x & 31;
  if (pages >> lane & 1) {
    const int valid = static_cast<int>(min(128LL, item.k_len - j * 128LL));
    const int limit = static_cast<int>(max(-128LL, min(128LL, item.seen0 - j * 128LL)));
    to[2 + __popc(pages & ((1u << lane) - 1))] =
        make_int4(row, valid | (limit << 16), __float_as_int(__ldg(p.a.k_scale + row)), __float_as_int(__ldg(p.a.v_scale + row)));
  }
  if (lane == 0) {
    to[0] = make_int4(flags, __popc(pages), item.token0, item.tokens);
    to[1] = make_int4(item.head, item.place, item.x0, item.x1);
  }
  __syncwarp();
}

int launch_paged_wide(const Params& p, int* status, DeviceCtx* ctx, cudaStream_t stream);     // paged_attention_wide.cu
constexpr int WIDE_ROWS = 128, WIDE_CTAS = 1;     // rows of an item of the wide kernel, its CTAs to an SM

}  // namespace pa
}  // namespace sb
