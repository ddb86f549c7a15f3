// Attention of new tokens over the 8-bit paged cache, on the tensor cores, straight from the e4m3 codes.
//
//   s_ij = scale * q_i . (k_scale * k_j)          keys j <= i + k_len - q_len of the request (causal) in the pages taken
//   o_i = sum_j softmax(s_i)_j v_scale v_j        lse_i = ln sum_j exp s_ij;  no key: o = 0, lse = -inf
//
// Mathematics. A work item is `pack` tokens of a request and a KV head: R rows (token, query head), 16 here, that share a pass
// over the pages; paged_attention_wide.cu has the kernel for more. Keys are the M dimension of both products, so that even one
// token of a few heads fills the instruction:
//   S^T [128 keys, R] = K [128 keys, 128] Q^T       O^T [128 features, R] = V^T [128 features, 128 keys] P^T
// The tensor core multiplies e4m3 by e4m3 (kind::f8f6f4), and the codes of a page are its operands as they lie in memory:
// nothing is dequantised. The other operand is split in two e4m3 terms in columns of their own, x = hi + lo / 16, hi rounded to
// nearest and lo the rest: a bf16 has eight significant bits and an e4m3 code four, so a query (scaled by a power of two to
// [128, 256) by its row's largest feature) is carried exactly where a feature is 2^-13 of the largest or more, and within 2^-21
// of the largest (half of lo's smallest step) where it is less; a probability (times 256, against the maximum of its own page,
// so that no page's weights fall below the format's range) within 2^-9 + 2^-11 of its value down to 2^-14 of the page's largest,
// and within 2^-22 of the largest below. Sums and outputs are fp32; every page's output is added to registers with the
// page's own factor exp2(page maximum - maximum of the item's first page) * v_scale.
//
// A softmax thread owns a key (a TMEM lane of S^T) and the 16 rows; a row's maximum over the page is taken in bf16 pairs by
// shuffles and an exchange between the four warps, in fp32 only where the scores are huge. In the second product the same
// thread owns a feature.
//
// Work split. Pages of all items, in the order (head, request, tile, page), are cut in equal shares, one per CTA: long and
// short requests balance whatever their lengths, known on the device only. Every CTA finds its share itself, from closed sums
// over a request's tiles and a scan over the requests. An item that lies in several shares is left as partial sums (fp32, with
// its maximum and sum) that paged_merge_kernel adds in order: no atomics, the same bits every time.
//
// CTA (two to an SM, so that one's exchanges and waits lie under the other's exponentials): four softmax warps, a loader warp
// (TMA, one 16 KB tile of K or V to a slot of a ring), an MMA warp, two warps that bring and split the queries of the next item.
// What the loader tells of items and pages goes through a ring of its own, in batches of 32 pages.
//
// What bounds it: HBM where pages are read once by 16 rows of heads (64 requests of 8192 to 32768 keys, 4 KV heads of 16: 1.41 GB
// in 221 us, 6.4 TB/s; with 64 listed pages each 0.54 GB in 98 us, 5.5 TB/s). The softmax, about 1400 cycles a page and CTA pair,
// is just under that. Items whose pages come from the L2 cache are bound by the latency of a page's chain: 32 requests of 1 to 8
// tokens, 66 us, keep no unit busy for more than half of the time (DRAM 50 %, issue slots 37 %, XU 10 %, tensor pipe 7 %). One row of 1 Mi
// keys: 57 us, 7 of them the merge of its parts. A call of 6 pages takes 12.5 us: latencies of two launches, of finding a share
// and of one page's chain.
#include "paged_attention.cuh"

namespace sb {
namespace pa {

constexpr int R = 16, N = 2 * R;                  // rows of an item, columns that carry them: hi and lo
struct Config {
  static constexpr int SOFTMAX_WARPS = 4;
  static constexpr int LOADER = SOFTMAX_WARPS, MMA = LOADER + 1, QWARP = MMA + 1, WARPS = QWARP + 2;
  static constexpr int THREADS = 32 * WARPS;
  static constexpr int CTAS = 2;                  // per SM
  static constexpr int SLOTS = 5;
  static constexpr int OFF_RING = 0;
  static constexpr int OFF_Q = OFF_RING + SLOTS * TILE_BYTES;       // two buffers of N rows of 128 bytes
  static constexpr int OFF_P = OFF_Q + 2 * N * 128;                 // 128 keys x N columns
  static constexpr int OFF_FACTOR = OFF_P + N * 128;               // float [softmax warp][4][16]
  static constexpr int OFF_MAX = OFF_FACTOR + SOFTMAX_WARPS * 256;  // bf16 [2][softmax warp][16]
  static constexpr int OFF_SUM = OFF_MAX + 2 * SOFTMAX_WARPS * 32;  // float [2][softmax warp][16]
  static constexpr int OFF_EXACT = OFF_SUM + 2 * SOFTMAX_WARPS * 64; // float [softmax warp][16]
  static constexpr int OFF_QF = OFF_EXACT + SOFTMAX_WARPS * 64;     // float [2][R]: what a row's scores are multiplied by
  static constexpr int OFF_ROW = OFF_QF + 2 * R * 4;                // int [R]: token << 16 | head of a row
  static constexpr int OFF_ROW_OUT = OFF_ROW + R * 4;               // int [R]: offset of a row in the output, from the item's first
  static constexpr int OFF_INFO = OFF_ROW_OUT + R * 4;
  static constexpr int OFF_BAR = OFF_INFO + BATCHES * BATCH_BYTES;
  static constexpr int B_INFO_FULL = 0, B_INFO_EMPTY = BATCHES, B_FULL = 2 * BATCHES, B_EMPTY = B_FULL + SLOTS;
  static constexpr int B_S_FULL = B_EMPTY + SLOTS, B_P_FULL = B_S_FULL + 2, B_O_FULL = B_P_FULL + 1, B_Q_FULL = B_O_FULL + 1,
                       B_Q_EMPTY = B_Q_FULL + 2, B_MAX = B_Q_EMPTY + 2, B_SUM = B_MAX + 2, B_EXACT = B_SUM + 2,
                       B_DONE = B_EXACT + 1, BARS = B_DONE + 1;
  static constexpr int OFF_FLAG = OFF_BAR + BARS * 8;               // int [SLOTS]: for the MMA warp, with a page's K tile
  static constexpr int OFF_MISC = (OFF_FLAG + SLOTS * 4 + 15) / 16 * 16;
  static constexpr int SMEM = OFF_MISC + 64 + 1024;                 // 1024: alignment of the tiles
  static constexpr int TMEM = 128;                                  // S of two pages and O: a power of two
};

// kind::f8f6f4 instruction descriptor: e4m3 x e4m3 -> fp32, M = 128.
__host__ __device__ constexpr uint32_t idesc_e4m3(int n, bool mn_major) {
  return (1u << 4) | (mn_major ? (1u << 15) | (1u << 16) : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24);
}
// Operands by the low words of their descriptors (start address and leading offset, in units of 16 bytes); the high words
// are constants. KMAJOR / MN128: 128-byte swizzle, eight rows 1024 bytes apart (a K tile and the queries; a V tile, whose 128
// features are one panel). MN32: panels of 32 columns, a key's 32 bytes after another, eight keys 256 bytes apart, panels 4096
// (the probabilities).
constexpr uint32_t HI_128 = (1024u >> 4) | (1u << 14) | (2u << 29), HI_MN32 = (256u >> 4) | (1u << 14) | (6u << 29);
constexpr uint32_t LO_MN128 = (static_cast<uint32_t>(TILE_BYTES) >> 4) << 16, LO_MN32 = (4096u >> 4) << 16;
template <uint32_t HI_B>
__device__ __forceinline__ void mma_e4m3(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      ".reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %5};\n\t"
      "mov.b64 db, {%2, %6};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %3, p;\n\t"
      "}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(HI_128), "n"(HI_B)
      : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
// Sums over the warp of 16 values: lane l gets that of value l % 16. Every step halves the values that a lane holds: 16
// shuffles in all.
__device__ __forceinline__ float row_sums(const float (&s)[16], int lane) {
  float a[8], b[4], c[2];
  const bool h8 = lane & 8, h4 = lane & 4, h2 = lane & 2, h1 = lane & 1;
#pragma unroll
  for (int j = 0; j < 8; ++j) a[j] = (h8 ? s[j + 8] : s[j]) + __shfl_xor_sync(0xffffffffu, h8 ? s[j] : s[j + 8], 8);
#pragma unroll
  for (int j = 0; j < 4; ++j) b[j] = (h4 ? a[j + 4] : a[j]) + __shfl_xor_sync(0xffffffffu, h4 ? a[j] : a[j + 4], 4);
#pragma unroll
  for (int j = 0; j < 2; ++j) c[j] = (h2 ? b[j + 2] : b[j]) + __shfl_xor_sync(0xffffffffu, h2 ? b[j] : b[j + 2], 2);
  const float d = (h1 ? c[1] : c[0]) + __shfl_xor_sync(0xffffffffu, h1 ? c[0] : c[1], 1);
  return d + __shfl_xor_sync(0xffffffffu, d, 16);
}
// The same for maxima, out of line.
__device__ __noinline__ float row_maxima_of(float s0, float s1, float s2, float s3, float s4, float s5, float s6, float s7, float s8, float s9,
                                             float s10, float s11, float s12, float s13, float s14, float s15, int lane) {
  const float s[16] = {s0, s1, s2, s3, s4, s5, s6, s7, s8, s9, s10, s11, s12, s13, s14, s15};
  float a[8], b[4], c[2];
  const bool h8 = lane & 8, h4 = lane & 4, h2 = lane & 2, h1 = lane & 1;
#pragma unroll
  for (int j = 0; j < 8; ++j) a[j] = fmaxf(h8 ? s[j + 8] : s[j], __shfl_xor_sync(0xffffffffu, h8 ? s[j] : s[j + 8], 8));
#pragma unroll
  for (int j = 0; j < 4; ++j) b[j] = fmaxf(h4 ? a[j + 4] : a[j], __shfl_xor_sync(0xffffffffu, h4 ? a[j] : a[j + 4], 4));
#pragma unroll
  for (int j = 0; j < 2; ++j) c[j] = fmaxf(h2 ? b[j + 2] : b[j], __shfl_xor_sync(0xffffffffu, h2 ? b[j] : b[j + 2], 2));
  const float d = fmaxf(h1 ? c[1] : c[0], __shfl_xor_sync(0xffffffffu, h1 ? c[0] : c[1], 1));
  return fmaxf(d, __shfl_xor_sync(0xffffffffu, d, 16));
}
__device__ __forceinline__ float row_maxima(const float (&s)[16], int lane) {
  return row_maxima_of(s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], s[9], s[10], s[11], s[12], s[13], s[14], s[15], lane);
}
// Maxima over the warp of 16 values in 8 pairs of bf16: lane l gets those of pair l % 8.
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t pair_maxima(const uint32_t (&s)[8], int lane) {
  uint32_t b[4], c[2];
  const bool h4 = lane & 4, h2 = lane & 2, h1 = lane & 1;
#pragma unroll
  for (int j = 0; j < 4; ++j) b[j] = max_bf16x2(h4 ? s[j + 4] : s[j], __shfl_xor_sync(0xffffffffu, h4 ? s[j] : s[j + 4], 4));
#pragma unroll
  for (int j = 0; j < 2; ++j) c[j] = max_bf16x2(h2 ? b[j + 2] : b[j], __shfl_xor_sync(0xffffffffu, h2 ? b[j] : b[j + 2], 2));
  uint32_t d = max_bf16x2(h1 ? c[1] : c[0], __shfl_xor_sync(0xffffffffu, h1 ? c[0] : c[1], 1));
  d = max_bf16x2(d, __shfl_xor_sync(0xffffffffu, d, 8));
  return max_bf16x2(d, __shfl_xor_sync(0xffffffffu, d, 16));
}
__device__ __noinline__ bool load_tile(uint32_t full, uint32_t empty, uint32_t parity, uint32_t to, const CUtensorMap* map, int row,
                                       volatile int* flag_at, int flag, volatile int* abort_flag, int* status) {
  if (!mbar_wait_warp(empty, parity, Guard{abort_flag, status}, 0xc01)) return false;
  if (elect_one()) {
    *flag_at = flag;
    if (flag == 2) {
      mbar_arrive(full);
    } else {
      mbar_expect_tx(full, TILE_BYTES);
      tma_load_2d(to, map, 0, row, full);
    }
  }
  __syncwarp();
  return true;
}
__device__ __forceinline__ uint32_t e4m3x2(__half2 x) { return __nv_cvt_halfraw2_to_fp8x2(x, __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ __half2 half2_of(uint32_t codes) {
  return __half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes), __NV_E4M3));
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
// hi + lo / 16 of 16 rows from tensor memory, eight at a time (registers)
__device__ __forceinline__ void load_sums(uint32_t at, float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 16; i += 8) {
    uint32_t h[8], w[8];
    tmem_ld8(at + i, h);
    tmem_ld8(at + R + i, w);
    tc_wait_ld();
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float2 y = fma2(make_float2(__uint_as_float(w[j]), __uint_as_float(w[j + 1])), make_float2(0.0625f, 0.0625f),
                            make_float2(__uint_as_float(h[j]), __uint_as_float(h[j + 1])));
      x[i + j] = y.x;
      x[i + j + 1] = y.y;
    }
  }
}

// o[j] where it is NaN: the sum of p v over the keys of a page that row j sees, from the probabilities in shared memory
// and a feature's codes
__device__ __noinline__ void visible_sums(float* o, const unsigned char* pr, const uint8_t* v, const int* row_of, int limit,
                                          int valid) {
#pragma unroll 1
  for (int j = 0; j < 16; ++j) {
    if (o[j] == o[j]) continue;
    const int end = min(limit + (row_of[j] >> 16), valid);
    float x = 0.f;
#pragma unroll 1
    for (int n = 0; n < end; ++n) {
      const auto at = [&](int c) { return from_e4m3(pr[(c >> 5) * 4096 + n * 32 + ((((c >> 4) ^ (n >> 2)) & 1) << 4) + (c & 15)]); };
      x = fmaf(fmaf(at(R + j), 0.0625f, at(j)), from_e4m3(__ldg(v + n * 128)), x);
    }
    o[j] = x;
  }
}

// ------------------------------------------------------------------ kernel
__global__ void __launch_bounds__(Config::THREADS, Config::CTAS)
    paged_attention_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const Params p,
                           int* status) {
  using C = Config;
  constexpr int SLOTS = C::SLOTS;
  extern __shared__ unsigned char raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  unsigned char* gbase = raw + (base - smem_u32(raw));
  volatile int* misc = reinterpret_cast<volatile int*>(gbase + C::OFF_MISC);     // [0] TMEM, [1] abort
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Guard guard{misc + 1, status};
  const auto bar = [&](int i) { return base + C::OFF_BAR + 8 * i; };

  if (tid == 0) {
    misc[1] = 0;
    for (int i = 0; i < BATCHES; ++i) {
      mbar_init(bar(C::B_INFO_FULL + i), 1);
      mbar_init(bar(C::B_INFO_EMPTY + i), C::SOFTMAX_WARPS + 2);
    }
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(bar(C::B_FULL + i), 1);
      mbar_init(bar(C::B_EMPTY + i), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(C::B_S_FULL + i), 1);
      mbar_init(bar(C::B_Q_FULL + i), 2);
      mbar_init(bar(C::B_Q_EMPTY + i), C::SOFTMAX_WARPS);
    }
    mbar_init(bar(C::B_P_FULL), C::SOFTMAX_WARPS);
    mbar_init(bar(C::B_O_FULL), 1);
    for (int i = C::B_MAX; i < C::B_DONE; ++i) mbar_init(bar(i), 4);
    mbar_init(bar(C::B_DONE), 1);
    fence_mbar_init();
    p.part_meta[16 * blockIdx.x] = 0;             // no part yet in either of this CTA's places
    p.part_meta[16 * blockIdx.x + 8] = 0;
  }
  int* row_of = reinterpret_cast<int*>(gbase + C::OFF_ROW);
  int* row_out = reinterpret_cast<int*>(gbase + C::OFF_ROW_OUT);
  if (tid < R) {
    const int token = tid / p.group, g = tid - token * p.group;
    row_of[tid] = token << 16 | g;
    row_out[tid] = (token * p.a.hq + g) * 128;
  }
  if (warp == C::MMA) {
    tmem_alloc(smem_u32(const_cast<int*>(misc)), C::TMEM);
    tmem_relinquish();
  }
  if (warp == C::LOADER && lane == 0) {
    prefetch_tmap(&k_map);
    prefetch_tmap(&v_map);
  }
  tc_fence_before();
  const Share share = find_share<C::WARPS>(p);     // (two barriers of the CTA)
  tc_fence_after();
  const uint32_t tmem = static_cast<uint32_t>(misc[0]);
  uint32_t fills = 0;

  if (warp == C::LOADER) {
    // --------------------------------------------------------------- loader
    uint32_t batches = 0;
    int slot = 0, phase = 0;
    bool ok = true;
    // flag: what the MMA warp has to know of a K tile: 1 = the first of an item, 2 = there are no more tiles
    const auto load = [&](const CUtensorMap* map, int row, int flag) {
      if (ok) ok = load_tile(bar(C::B_FULL + slot), bar(C::B_EMPTY + slot), phase ^ 1, base + C::OFF_RING + slot * TILE_BYTES, map, row,
                             reinterpret_cast<volatile int*>(gbase + C::OFF_FLAG + 4 * slot), flag, guard.abort_flag, status);
      fills += ok;
      if (++slot == SLOTS) {
        slot = 0;
        phase ^= 1;
      }
    };
    // waits for a free batch
    const auto batch = [&]() {
      const uint32_t e = batches % BATCHES;
      ok = ok && wait_warp(bar(C::B_INFO_EMPTY + e), ((batches / BATCHES) & 1) ^ 1, guard, 0xc00);
      return reinterpret_cast<int4*>(gbase + C::OFF_INFO + e * BATCH_BYTES);
    };
    bool started = false;
    walk_share(p, share, ok, [&](const Item& item, int flags, uint32_t pages, int row, int j) {
      if (flags & FIRST) started = false;
      uint32_t todo = pages;
#pragma unroll 1
      for (bool told = false; ok && (todo || !told);) {
        if (todo) {
          const int next = __shfl_sync(0xffffffffu, row, __ffs(todo) - 1) * 128;
          todo &= todo - 1;
          load(&k_map, next, started ? 0 : 1);
          load(&v_map, next, 0);
          started = true;
        }
        if (told) continue;
        told = true;                               // behind the first page's tiles: the scales have to be fetched
        int4* to = batch();
        if (!ok) break;
        write_batch(p, to, item, flags, pages, row, j);
        if (lane == 0) mbar_arrive(bar(C::B_INFO_FULL + batches % BATCHES));
        ++batches;
      }
    });
    int4* to = batch();
    if (ok) {
      if (lane == 0) {
        to[0] = make_int4(STOP, 0, 0, 0);
        mbar_arrive(bar(C::B_INFO_FULL + batches % BATCHES));
      }
      __syncwarp();
    }
    load(&k_map, 0, 2);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  } else if (warp == C::MMA) {
    // --------------------------------------------------------------- MMA issuer
    // Waits by the whole warp, issue by its elected lane. That S may be overwritten by the page after the next, and O by the
    // next, needs no barrier: the softmax warps store the probabilities of a page after they have read its S and the O
    // of the page before.
    // Everything that the issue depends on is uniform for the compiler to see (counters, votes, no call in the way): the
    // operands of tcgen05 instructions come from uniform registers, and what is not known to be uniform is moved there
    // one by one, which took 500 cycles for the four instructions and two commits of a product.
    constexpr uint32_t ID_QK = idesc_e4m3(N, false), ID_PV = idesc_e4m3(N, true);
    bool ok = true, stopped = false;
    int first = 0, second = 0, item = -1;          // pages whose first / second product has been issued
    int slot = 0, phase = 0, v_slot = 1, v_phase = 0;
    const auto next_page = [&](int& s, int& f) {   // two tiles on
      s += 2;
      if (s >= SLOTS) {
        s -= SLOTS;
        f ^= 1;
      }
    };
    const auto ready = [&](int which, int parity) { return __all_sync(0xffffffffu, mbar_test_wait(bar(which), parity)) != 0; };
    long long t0 = clock64();
    while (ok) {
      // One page ahead of the second products; where its K tile is not there yet and the probabilities of the page before
      // are, these go first.
      bool tile = false;
      if (!stopped && first - second < 2) {
        tile = ready(C::B_FULL + slot, phase);
        if (!tile && first == second) {
          ok = mbar_wait_warp(bar(C::B_FULL + slot), phase, guard, 0xc10);
          if (!ok) break;
          tile = true;
        }
      }
      if (tile) {
        const int flag = *reinterpret_cast<volatile int*>(gbase + C::OFF_FLAG + 4 * slot);
        stopped = __any_sync(0xffffffffu, flag & 2);
        const int of = item + (__any_sync(0xffffffffu, flag & 1) ? 1 : 0);
        bool queries = of == item;
        if (!stopped && !queries) {
          // A new item's queries are not waited for while second products are owed: their buffer may be that of an item whose
          // end needs those.
          queries = ready(C::B_Q_FULL + (of & 1), (of >> 1) & 1);
          if (!queries && first == second) {
            ok = mbar_wait_warp(bar(C::B_Q_FULL + (of & 1)), (of >> 1) & 1, guard, 0xc11);
            if (!ok) break;
            queries = true;
          }
        }
        if (!stopped && queries) {
          item = of;
          tc_fence_after();
          if (elect_one()) {
            const uint32_t kt = (base + C::OFF_RING + slot * TILE_BYTES) >> 4, qt = (base + C::OFF_Q + (item & 1) * N * 128) >> 4;
#pragma unroll
            for (int k = 0; k < 4; ++k) mma_e4m3<HI_128>(tmem + (first & 1) * N, kt + k * 2, qt + k * 2, ID_QK, k > 0);
            tc_commit(bar(C::B_S_FULL + (first & 1)));
            tc_commit(bar(C::B_EMPTY + slot));
          }
          __syncwarp();
          next_page(slot, phase);
          ++first;
          t0 = clock64();
        }
      }
      if (first == second) {
        if (stopped) break;
        continue;
      }
      if (!ready(C::B_P_FULL, second & 1)) {
        const bool late = clock64() - t0 > WAIT_LIMIT_CYCLES || *guard.abort_flag;
        if (!stopped && first - second < 2 && !__any_sync(0xffffffffu, late)) continue;
        ok = mbar_wait_warp(bar(C::B_P_FULL), second & 1, guard, 0xc12);
        if (!ok) break;
      }
      ok = mbar_wait_warp(bar(C::B_FULL + v_slot), v_phase, guard, 0xc13);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t v = ((base + C::OFF_RING + v_slot * TILE_BYTES) >> 4) | LO_MN128;
        const uint32_t pr = ((base + C::OFF_P) >> 4) | LO_MN32;
#pragma unroll
        for (int k = 0; k < 4; ++k) mma_e4m3<HI_MN32>(tmem + 2 * N, v + k * 256, pr + k * 64, ID_PV, k > 0);
        tc_commit(bar(C::B_O_FULL));
        tc_commit(bar(C::B_EMPTY + v_slot));
      }
      __syncwarp();
      next_page(v_slot, v_phase);
      ++second;
      t0 = clock64();
    }
    // nothing of the tensor core's is in flight when the CTA gives up its memory
    if (elect_one()) tc_commit(bar(C::B_DONE));
    __syncwarp();
    mbar_wait_drain(bar(C::B_DONE), 0);
  } else if (warp >= C::QWARP) {
    // --------------------------------------------------------------- queries of the next item
    const int half = warp - C::QWARP;
    bool ok = true;
    uint32_t batches = 0;
    int items = 0;
    const float sign = p.a.scale < 0.f ? -1.f : 1.f, factor = fabsf(p.a.scale) * 1.4426950408889634f;
    while (ok) {
      const uint32_t e = batches % BATCHES;
      ok = wait_warp(bar(C::B_INFO_FULL + e), (batches / BATCHES) & 1, guard, 0xc20);
      if (!ok) break;
      const int4 x = *reinterpret_cast<const int4*>(gbase + C::OFF_INFO + e * BATCH_BYTES);
      const int head = *reinterpret_cast<const int*>(gbase + C::OFF_INFO + e * BATCH_BYTES + 16);
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(C::B_INFO_EMPTY + e));
      ++batches;
      if (x.x & STOP) break;
      if (!(x.x & FIRST) || x.y == 0) continue;
      const int buf = items & 1;
      ok = wait_warp(bar(C::B_Q_EMPTY + buf), ((items >> 1) & 1) ^ 1, guard, 0xc21);
      if (!ok) break;
      const int rows = x.w * p.group;              // tokens x heads of the KV head
      unsigned char* q8 = gbase + C::OFF_Q + buf * N * 128;
      float* qf = reinterpret_cast<float*>(gbase + C::OFF_QF) + buf * R;
      const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(p.a.q) + x.z * p.a.q_token +
                                 static_cast<long long>(head) * p.group * p.a.q_head + lane * 4;
#pragma unroll 1
      for (int r0 = half * (R / 2); r0 < (half + 1) * (R / 2); r0 += 4) {
        uint2 w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = row_of[r0 + i];
          w[i] = r0 + i < rows ? __ldg(reinterpret_cast<const uint2*>(src + (at >> 16) * p.a.q_token + (at & 0xffff) * p.a.q_head))
                               : make_uint2(0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = r0 + i;
          const uint32_t m = __vmaxu2(w[i].x & 0x7fff7fffu, w[i].y & 0x7fff7fffu);
          const uint32_t top = __reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16));
          // times 2^e the largest feature lies in [128, 256); a row with infinities or NaN is taken as it is and ends as NaN
          const bool odd = top >= 0x7f80u;
          const int e = top == 0 || odd ? 0 : min(134 - static_cast<int>(top >> 7), 126);
          const float by = power_of_two(e) * sign;
          const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i].x));
          const float2 c = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i].y));
          const float v[4] = {a.x * by, a.y * by, c.x * by, c.y * by};
          uint32_t hi = e4m3x2(v[0], v[1]) | (e4m3x2(v[2], v[3]) << 16);
          const float2 h0 = from_e4m3x2(hi), h1 = from_e4m3x2(hi >> 16);
          const uint32_t rest = e4m3x2((v[0] - h0.x) * 16.f, (v[1] - h0.y) * 16.f) |
                                (e4m3x2((v[2] - h1.x) * 16.f, (v[3] - h1.y) * 16.f) << 16);
          if (odd) {
#pragma unroll
            for (int d = 0; d < 4; ++d)
              if (!(fabsf(v[d]) < INFINITY)) hi |= 0x7fu << (8 * d);
          }
          const int chunk = ((lane >> 2) ^ (row & 7)) * 16 + (lane & 3) * 4;
          *reinterpret_cast<uint32_t*>(q8 + row * 128 + chunk) = hi;
          *reinterpret_cast<uint32_t*>(q8 + (R + row) * 128 + chunk) = rest;
          if (lane == 0) qf[row] = factor * power_of_two(-e);
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(C::B_Q_FULL + buf));
      ++items;
    }
  } else {
    // --------------------------------------------------------------- softmax: lane = key, then lane = feature
    const int key = warp * 32 + lane, r16 = lane & 15;
    const uint32_t lane_base = static_cast<uint32_t>(warp * 32) << 16;
    // of the warp's 16 rows: score factor, exponent offset, weight of the page's sum, weight of its output
    float* factors = reinterpret_cast<float*>(gbase + C::OFF_FACTOR) + warp * 64;
    __nv_bfloat16* maxima = reinterpret_cast<__nv_bfloat16*>(gbase + C::OFF_MAX);
    float* sums = reinterpret_cast<float*>(gbase + C::OFF_SUM);
    const float* qf = reinterpret_cast<const float*>(gbase + C::OFF_QF);
    float acc[16], l[16], s[16], m = -INFINITY, scale_row = 0.f;      // m: what the sums of row r16 are relative to
    uint32_t batches = 0;
    int items = 0, ends = 0, exacts = 0, pages = 0, pending = -1, masked = 0;
    int item_pages = 0;
    // of the pending page, for rows that do not see all of its keys
    int p_row = 0, p_limit = 0, p_valid = 0;
    bool ok = true, fresh = false;
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = l[i] = 0.f;

    // adds the output of page `pending` to acc
    const auto add_output = [&](bool more) {
      ok = ok && wait_warp(bar(C::B_O_FULL), pending & 1, guard, 0xc30);
      pending = -1;
      if (!ok) return;
      tc_fence_after();
      float o[16];
      load_sums(tmem + lane_base + 2 * N, o);
      tc_fence_before();
      if (masked) {
        // A key that is hidden from a row has probability 0 there, and 0 times a NaN of its value is not 0: such a sum is
        // done again over the keys that the row sees.
        bool odd = false;
#pragma unroll
        for (int j = 0; j < 16; ++j) odd |= o[j] != o[j];
        if (odd) {
          float sums[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) sums[j] = o[j];
          visible_sums(sums, gbase + C::OFF_P,
                          static_cast<const uint8_t*>(p.a.v) + static_cast<long long>(p_row) * TILE_BYTES + key, row_of,
                          p_limit, p_valid);
#pragma unroll
          for (int j = 0; j < 16; ++j) o[j] = sums[j];
        }
        // All four warps read the probabilities there: none stores the next page's before the others have. (Out of the hot path's
        // way: with the maxima announced later instead, 68.5 us for 66 with 1 to 8 tokens.)
        if (more) {
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(C::B_EXACT));
          ok = wait_longer(bar(C::B_EXACT), exacts++ & 1, guard.abort_flag, guard.status, 0xc38);
          if (!ok) return;
        }
      }
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        const float4 c = *reinterpret_cast<const float4*>(factors + 48 + j);
        const float2 x = fma2(make_float2(o[j], o[j + 1]), make_float2(c.x, c.y), make_float2(acc[j], acc[j + 1]));
        const float2 y = fma2(make_float2(o[j + 2], o[j + 3]), make_float2(c.z, c.w), make_float2(acc[j + 2], acc[j + 3]));
        acc[j] = x.x;
        acc[j + 1] = x.y;
        acc[j + 2] = y.x;
        acc[j + 3] = y.y;
      }
    };

    while (ok) {
      const uint32_t e = batches % BATCHES;
      ok = wait_warp(bar(C::B_INFO_FULL + e), (batches / BATCHES) & 1, guard, 0xc31);
      if (!ok) break;
      const int4* info = reinterpret_cast<const int4*>(gbase + C::OFF_INFO + e * BATCH_BYTES);
      const int flags = info[0].x, count = info[0].y;
      if (flags & STOP) break;
      if (flags & FIRST) {
        m = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i] = l[i] = 0.f;
        fresh = true;
        item_pages = 0;
      }
      item_pages += count;
      // the pages of the batch, then the item's end
      const int steps = count + (flags & LAST ? 1 : 0);
#pragma unroll 1
      for (int step = 0; ok && step < steps; ++step) {
        const bool page = step < count;
        const volatile int* x = reinterpret_cast<const volatile int*>(info + 2 + min(step, 31));     // read where it is needed: registers
        const int seen = x[1], valid = seen & 0xffff, limit = seen >> 16;
        if (page) {
          const int b = pages & 1;
          if (fresh) {
            ok = wait_warp(bar(C::B_Q_FULL + (items & 1)), (items >> 1) & 1, guard, 0xc32);
            if (!ok) break;
            scale_row = qf[(items & 1) * R + r16];
            fresh = false;
          }
          ok = wait_warp(bar(C::B_S_FULL + b), (pages >> 1) & 1, guard, 0xc33);
          if (!ok) break;
          tc_fence_after();
          load_sums(tmem + lane_base + b * N, s);
          tc_fence_before();
          const bool partial = valid < 128 || limit < 128;
          if (partial) {
            // Rows are in token order: those that do not see this key are the first ones.
            const int first = p.a.causal ? (key - limit + 1) * p.group : key >= limit ? 16 : 0;
            const int unseen = key >= valid ? 16 : first;
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (j < unseen) s[j] = -INFINITY;
          }
          // Maxima in bf16: a reference, not a result. Rounded up by what the conversion may have lost they bound every score.
          uint32_t pairs[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) pairs[j] = pack_bf16x2(s[2 * j], s[2 * j + 1]);
          const uint32_t top = pair_maxima(pairs, lane);
          if (lane < 8) reinterpret_cast<uint32_t*>(maxima + b * C::SOFTMAX_WARPS * 16 + warp * 16)[lane] = top;
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(C::B_MAX + b));
        }
        // under the other warps' maxima: the output of the page before
        if (pending >= 0) {
          add_output(page);
          if (!ok) break;
        }
        int again = page;
        asm volatile("" : "+r"(again));              // one copy of add_output for pages and ends
        if (again) {
          const int b = pages & 1;
          ok = wait_warp(bar(C::B_MAX + b), (pages >> 1) & 1, guard, 0xc36);
          if (!ok) break;
          const __nv_bfloat16* mx = maxima + b * C::SOFTMAX_WARPS * 16 + r16;
          float top = fmaxf(fmaxf(__bfloat162float(mx[0]), __bfloat162float(mx[16])),
                            fmaxf(__bfloat162float(mx[32]), __bfloat162float(mx[48])));
          float f = scale_row * __int_as_float(x[2]);
          if (f == 0.f) f = 1e-37f;                  // hidden keys stay hidden with a scale of 0
          const bool none = top == -INFINITY, unset = m == -INFINITY;
          float mu = none ? -INFINITY : fmaf(fabsf(top), 0.00394f, top) * f;       // 2^-8 and a little
          float over = 1.f;                          // 0: s is relative to mu already
          // The sums stay relative to the item's first page: fp32 has room for 2^40 above it, and what lies below loses nothing.
          // Less where the page's values are huge: a rise times its value scale stays below 2^90, or the reference follows.
          const float room = static_cast<float>(max(min(216 - (x[3] >> 23 & 255), 40), 0));        // 90 - exponent - 1
          if (__any_sync(0xffffffffu, !none && (fabsf(mu) > 100.f || (!unset && mu - m > room)))) {
            // Rare: scores above that, or so large that the rounding up is more than a factor of 1.5. The maxima in fp32; all
            // four warps of the group are here.
            float* exact = reinterpret_cast<float*>(gbase + C::OFF_EXACT);
            top = row_maxima(s, lane);
            if (lane < 16) exact[warp * 16 + lane] = top;
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(C::B_EXACT));
            ok = wait_warp(bar(C::B_EXACT), exacts++ & 1, guard, 0xc37);
            if (!ok) break;
            top = fmaxf(fmaxf(exact[r16], exact[16 + r16]), fmaxf(exact[32 + r16], exact[48 + r16]));
            if (!none) mu = top * f;
            const bool jump = !unset && mu - m > room;
            if (lane < 16) {
              factors[lane] = jump ? ex2_approx(m - mu) : 1.f;
              factors[16 + lane] = none ? 0.f : top;
            }
            if (jump) m = mu;
            __syncwarp();
            // The scores relative to their maximum before they are scaled: s f - mu in one rounding is what mu was rounded by at
            // the maximum, more than the exponent's range where scores are huge.
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              acc[j] *= factors[j];
              l[j] *= factors[j];
              s[j] -= factors[16 + j];
            }
            over = 0.f;
            __syncwarp();
          }
          if (unset) m = mu;
          if (lane < 16) {
            const float w = none ? 0.f : ex2_approx(mu - m);
            factors[lane] = none ? 1.f : f;          // (a scale may be NaN)
            factors[16 + lane] = none ? 0.f : fmaf(-over, mu, 8.f);
            factors[32 + lane] = w;
            factors[48 + lane] = none ? 0.f : w * __int_as_float(x[3]) * 0.00390625f;
          }
          __syncwarp();
          uint32_t ph[4], pl[4];
#pragma unroll
          for (int j4 = 0; j4 < 4; ++j4) {
            const float4 f4 = *reinterpret_cast<const float4*>(factors + 4 * j4);
            const float4 b4 = *reinterpret_cast<const float4*>(factors + 16 + 4 * j4);
            const float4 w4 = *reinterpret_cast<const float4*>(factors + 32 + 4 * j4);
            uint32_t hi[2], lo[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int j = 4 * j4 + 2 * i;
              float2 v = fma2(make_float2(s[j], s[j + 1]), i ? make_float2(f4.z, f4.w) : make_float2(f4.x, f4.y),
                              i ? make_float2(b4.z, b4.w) : make_float2(b4.x, b4.y));
              v.x = ex2_approx(v.x);
              v.y = ex2_approx(v.y);
              const float2 n = fma2(v, i ? make_float2(w4.z, w4.w) : make_float2(w4.x, w4.y), make_float2(l[j], l[j + 1]));
              l[j] = n.x;
              l[j + 1] = n.y;
              const __half2 w = __float22half2_rn(v);      // 2^-11; what is left of it by its upper term is exact
              hi[i] = e4m3x2(w);
              lo[i] = e4m3x2(__hfma2(half2_of(hi[i]), __float2half2_rn(-16.f), __hmul2(w, __float2half2_rn(16.f))));
            }
            ph[j4] = __byte_perm(hi[0], hi[1], 0x5410);
            pl[j4] = __byte_perm(lo[0], lo[1], 0x5410);
          }
          unsigned char* to = gbase + C::OFF_P + key * 32;
          const auto column = [&](int c) { return to + (c >> 5) * 4096 + ((((c >> 4) ^ (key >> 2)) & 1) << 4); };
          *reinterpret_cast<uint4*>(column(0)) = make_uint4(ph[0], ph[1], ph[2], ph[3]);
          *reinterpret_cast<uint4*>(column(R)) = make_uint4(pl[0], pl[1], pl[2], pl[3]);
          if (valid < 128) {
            // rows behind the sequence may hold anything: they become zeros before the second product reads them
            const int n = 2 * pages + 1, vslot = n % SLOTS;
            ok = wait_warp(bar(C::B_FULL + vslot), (n / SLOTS) & 1, guard, 0xc34);
            if (!ok) break;
            if (key >= valid) {
              uint4* v = reinterpret_cast<uint4*>(gbase + C::OFF_RING + vslot * TILE_BYTES + key * 128);
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] = make_uint4(0, 0, 0, 0);
            }
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(C::B_P_FULL));
          pending = pages++;
          masked = limit < valid;
          p_row = x[0];
          p_limit = limit;
          p_valid = valid;
          continue;
        }
        // the item's end
        if (item_pages) {
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(C::B_Q_EMPTY + (items & 1)));
          ++items;
        }
        float* sm = sums + (ends & 1) * C::SOFTMAX_WARPS * 16;
        const float sum = row_sums(l, lane);
        if (lane < 16) sm[warp * 16 + lane] = sum;
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::B_SUM + (ends & 1)));
        ok = wait_warp(bar(C::B_SUM + (ends & 1)), (ends >> 1) & 1, guard, 0xc35);
        ++ends;
        if (!ok) break;
        const int token0 = info[0].z, rows = info[0].w * p.group, head = info[1].x, place = info[1].y;
        // lane r: sum of row r
        const float sum_row = ((sm[r16] + sm[16 + r16]) + (sm[32 + r16] + sm[48 + r16])) * 0.00390625f;
        if (place < 0) {
          const long long first = static_cast<long long>(token0) * p.a.hq + head * p.group;
          if (lane < 16) factors[lane] = sum_row == 0.f ? 0.f : 1.f / sum_row;
          __syncwarp();
          __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.a.out) + first * 128 + key;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (j < rows) out[row_out[j]] = __float2bfloat16(acc[j] * factors[j]);
          if (p.a.lse && warp == 0 && lane < rows)
            p.a.lse[first + (row_out[lane] >> 7)] = sum_row == 0.f ? -INFINITY : (m + log2f(sum_row)) * 0.6931471805599453f;
        } else {
          float* part = p.part_o + static_cast<long long>(place) * R * 128 + key;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (j < rows) part[j * 128] = acc[j];
          if (warp == 0 && lane < 16)
            *reinterpret_cast<float2*>(p.part_ml + (static_cast<long long>(place) * R + lane) * 2) = make_float2(m, sum_row);
          if (warp == 0 && lane == 0) {
            int* meta = p.part_meta + 8 * place;
            *reinterpret_cast<int4*>(meta) = make_int4(1, info[1].z, info[1].w, token0);
            *reinterpret_cast<int2*>(meta + 4) = make_int2(info[0].w, head);
          }
        }
        break;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(C::B_INFO_EMPTY + e));
      ++batches;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == C::LOADER && misc[1]) {               // a wait was given up: copies in flight land before the CTA leaves
    for (uint32_t f = fills > SLOTS ? fills - SLOTS : 0; f < fills; ++f) mbar_wait_drain(bar(C::B_FULL + f % SLOTS), (f / SLOTS) & 1);
  }
  if (warp == C::MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM);
  }
}

// Adds the parts of the items that lie in several shares, in order:
//   M = max_i m_i, w_i = exp2(m_i - M), out = sum w_i acc_i / sum w_i l_i, lse = ln 2 (M + log2 sum w_i l_i)
// blockIdx.x stands for the border of shares x and x + 1; the (n - 1) gridDim.y CTAs of the borders inside an item of n parts
// divide its rows: a row to a half warp (16 lanes, 8 features each) where the parts are few, 32 features of a row to a whole
// CTA (a warp takes every eighth part) where they are many. Either way a thread makes two dependent round trips to memory or
// a few more, which is the kernel's time. (Rows one after another by the CTA of the border: 130 us of the 217 of a batch of
// speculated tokens, 75 of the 293 of a decode batch over 1.4 GB.)
constexpr int MERGE_WARPS = 8, FEW = 16;
__global__ void __launch_bounds__(32 * MERGE_WARPS) paged_merge_kernel(const Params p) {
  __shared__ float s_top[MERGE_WARPS], s_l[MERGE_WARPS];
  __shared__ float s_acc[MERGE_WARPS][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int x = blockIdx.x + 1;
  const int4 meta = *reinterpret_cast<const int4*>(p.part_meta + 16 * x);        // the part that comes from the share before
  if (meta.x == 0) return;
  const int2 more = *reinterpret_cast<const int2*>(p.part_meta + 16 * x + 4);
  const int x0 = meta.y, parts = meta.z - x0 + 1, token0 = meta.w, rows = more.x * p.group, head = more.y;
  const int cta = (x - x0 - 1) * gridDim.y + blockIdx.y, ctas = (parts - 1) * gridDim.y;
  const auto part_row = [&](int i, int row) { return static_cast<long long>(2 * (x0 + i) + (i == 0)) * p.rows + row; };
  const auto out_row = [&](int row) {
    const int token = row / p.group;
    return (static_cast<long long>(token0) + token) * p.a.hq + head * p.group + (row - token * p.group);
  };
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.a.out);
  if (parts <= FEW) {
    const int l16 = lane & 15;
    const unsigned half = 0xffffu << (lane & 16);
    for (int row = cta * 2 * MERGE_WARPS + 2 * warp + (lane >> 4); row < rows; row += ctas * 2 * MERGE_WARPS) {
      float2 ml = make_float2(-INFINITY, 0.f);
      if (l16 < parts) ml = *reinterpret_cast<const float2*>(p.part_ml + part_row(l16, row) * 2);
      float top = ml.x;
#pragma unroll
      for (int by = 8; by; by >>= 1) top = fmaxf(top, __shfl_xor_sync(half, top, by));
      const float w = ml.x == -INFINITY ? 0.f : ex2_approx(ml.x - top);
      float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, l = 0.f;
#pragma unroll 4
      for (int i = 0; i < parts; ++i) {
        const float4* from = reinterpret_cast<const float4*>(p.part_o + part_row(i, row) * 128) + 2 * l16;
        const float4 a = from[0], b = from[1];
        const float wi = __shfl_sync(half, w, i, 16), li = __shfl_sync(half, ml.y, i, 16);
        l = fmaf(wi, li, l);
        acc[0] = fmaf(wi, a.x, acc[0]);
        acc[1] = fmaf(wi, a.y, acc[1]);
        acc[2] = fmaf(wi, a.z, acc[2]);
        acc[3] = fmaf(wi, a.w, acc[3]);
        acc[4] = fmaf(wi, b.x, acc[4]);
        acc[5] = fmaf(wi, b.y, acc[5]);
        acc[6] = fmaf(wi, b.z, acc[6]);
        acc[7] = fmaf(wi, b.w, acc[7]);
      }
      const long long to = out_row(row);
      const float inv = l == 0.f ? 0.f : 1.f / l;
      *reinterpret_cast<uint4*>(out + to * 128 + 8 * l16) =
          make_uint4(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv),
                     pack_bf16x2(acc[4] * inv, acc[5] * inv), pack_bf16x2(acc[6] * inv, acc[7] * inv));
      if (p.a.lse && l16 == 0) p.a.lse[to] = l == 0.f ? -INFINITY : (top + log2f(l)) * 0.6931471805599453f;
    }
    return;
  }
  for (int piece = cta; piece < 4 * rows; piece += ctas) {
    const int row = piece >> 2, d = (piece & 3) * 32 + lane;
    float top = -INFINITY, acc = 0.f, l = 0.f;
    for (int c = 0; warp + MERGE_WARPS * c < parts; c += 32) {
      const int mine = warp + MERGE_WARPS * (c + lane), count = min(32, (parts - warp + MERGE_WARPS - 1) / MERGE_WARPS - c);
      float2 ml = make_float2(-INFINITY, 0.f);
      if (mine < parts) ml = *reinterpret_cast<const float2*>(p.part_ml + part_row(mine, row) * 2);
      float now = fmaxf(top, ml.x);
#pragma unroll
      for (int by = 16; by; by >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, by));
      const float keep = top == -INFINITY ? 0.f : ex2_approx(top - now), w = ml.x == -INFINITY ? 0.f : ex2_approx(ml.x - now);
      top = now;
      acc *= keep;
      l *= keep;
      // 16 loads in flight, the last ones too (a loop's remainder would wait for each): lanes beyond the parts have weight 0
      for (int i0 = 0; i0 < count; i0 += 16) {
        float o[16];
#pragma unroll
        for (int j = 0; j < 16; ++j)
          o[j] = i0 + j < count ? p.part_o[part_row(warp + MERGE_WARPS * (c + i0 + j), row) * 128 + d] : 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float wi = __shfl_sync(0xffffffffu, w, i0 + j), li = __shfl_sync(0xffffffffu, ml.y, i0 + j);
          acc = fmaf(wi, o[j], acc);
          l = fmaf(wi, li, l);
        }
      }
    }
    s_acc[warp][lane] = acc;
    if (lane == 0) {
      s_top[warp] = top;
      s_l[warp] = l;
    }
    __syncthreads();
    if (warp == 0) {
      top = -INFINITY;
      acc = l = 0.f;
#pragma unroll
      for (int w = 0; w < MERGE_WARPS; ++w) top = fmaxf(top, s_top[w]);
#pragma unroll
      for (int w = 0; w < MERGE_WARPS; ++w) {
        const float keep = s_top[w] == -INFINITY ? 0.f : ex2_approx(s_top[w] - top);
        acc = fmaf(keep, s_acc[w][lane], acc);
        l = fmaf(keep, s_l[w], l);
      }
      const long long to = out_row(row);
      out[to * 128 + d] = __float2bfloat16(l == 0.f ? 0.f : acc / l);
      if (p.a.lse && d == 0) p.a.lse[to] = l == 0.f ? -INFINITY : (top + log2f(l)) * 0.6931471805599453f;
    }
    __syncthreads();
  }
}

// Tokens that share a pass over the pages, a power of two: as many as 128 rows hold, no more than there are. Up to 32 rows
// items of 16 rows read the pages twice (the second time from the L2 cache): the kernel for 16 rows does so quicker than the wide
// one goes once over them, which works on 128 rows always, and requests with fewer tokens need one item. Measured, 32
// requests of up to 8 tokens and 8192 keys, 4 heads to each of 8 KV heads: 67 us as 16 rows, 76 us in a variant for 32, 130 us
// in the wide one; 16 heads, lists of 16 pages for tiles of 16 tokens (4 prompts of 512 to 1024): 181 us in a variant for 64
// rows, 108 us in the wide one.
static int pack_of(int group, int tile, int max_q, bool listed) {
  int pack = 1;
  while (2 * pack * group <= WIDE_ROWS && pack < max_q && (!listed || 2 * pack <= tile)) pack *= 2;
  if (group <= R && pack * group <= 2 * R)
    while (pack * group > R) pack /= 2;
  return pack;
}
static int rows_of(int used) { return used <= R ? R : WIDE_ROWS; }
static int ctas_of(int rows, int sm_count) { return sm_count * (rows == R ? Config::CTAS : WIDE_CTAS); }

static int launch_narrow(const Params& p, DeviceCtx* ctx, cudaStream_t stream) {
  using C = Config;
  const PagedAttentionArgs& a = p.a;
  CUtensorMap km, vm;
  const cuuint64_t dims[2] = {128, static_cast<cuuint64_t>(a.pages) * a.hkv * 128};
  const cuuint64_t strides[1] = {128};
  const cuuint32_t box[2] = {128, 128}, steps[2] = {1, 1};
  for (int i = 0; i < 2; ++i)
    if (encode_tiled(i ? &vm : &km, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(i ? a.v : a.k), dims, strides, box, steps,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B))
      return set_error(SB_ERR_CUDA, "tensor map of the cache pages");
  if (!ctx->paged_attr[4]) {
    if (cudaFuncSetAttribute(paged_attention_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess)
      return set_error(SB_ERR_CUDA, "shared memory of the paged attention");
    ctx->paged_attr[4] = 1;
  }
  paged_attention_kernel<<<p.ctas, C::THREADS, C::SMEM, stream>>>(km, vm, p, ctx->status);
  return check_kernel_launch();
}

}  // namespace pa

long long paged_attention_workspace_bytes(int hq, int hkv, int tile, int max_q, bool listed, int sm_count) {
  const int group = hq / hkv, rows = pa::rows_of(pa::pack_of(group, tile, max_q, listed) * group);
  return 2LL * pa::ctas_of(rows, sm_count) * (rows * 130 * 4LL + 32);
}

int launch_paged_attention(const PagedAttentionArgs& a, cudaStream_t stream) {
  using namespace pa;
  DeviceCtx* ctx = device_ctx();
  if (!ctx) return SB_ERR_CUDA;
  if (!a.workspace || a.workspace_bytes < paged_attention_workspace_bytes(a.hq, a.hkv, a.tile, a.max_q, a.ids != nullptr, ctx->sm_count))
    return set_error(SB_ERR_INVALID, "workspace too small (see sparse_b200_paged_attention_workspace_bytes)");
  const int group = a.hq / a.hkv, pack = pack_of(group, a.tile, a.max_q, a.ids != nullptr), rows = rows_of(pack * group);
  Params p{a, group, pack, 0, 0, ctas_of(rows, ctx->sm_count), rows, nullptr, nullptr, nullptr};
  while ((1 << p.pack_shift) < pack) ++p.pack_shift;
  while (a.ids && (1 << p.tile_shift) < a.tile) ++p.tile_shift;
  if (!a.ids) p.a.topk = 0;
  p.part_o = static_cast<float*>(a.workspace);
  p.part_ml = p.part_o + 2LL * p.ctas * rows * 128;
  p.part_meta = reinterpret_cast<int*>(p.part_ml + 2LL * p.ctas * rows * 2);
  const int rc = rows == R ? launch_narrow(p, ctx, stream) : launch_paged_wide(p, ctx->status, ctx, stream);
  if (rc) return rc;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.ctas - 1, rows / 16);
  cfg.blockDim = dim3(32 * MERGE_WARPS);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_merge_kernel, p);
  return e == cudaSuccess ? SB_OK : set_error(SB_ERR_CUDA, cudaGetErrorString(e));
}

}  // namespace sb
