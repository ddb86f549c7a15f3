// Attention over the 8-bit paged cache for items of more than 16 rows (several new tokens, or many query heads to a KV head):
// the same results, shares, parts and lists as the narrow kernel (paged_attention.cu), with the rows on the tensor core's M
// dimension.
//
//   S [128 rows, 128 keys] = Q K^T      O [128 rows, 128 features] += P V          (kind::f16, fp32 sums, one page a step)
//
// Mathematics. The codes of a page become f16, exactly, on their way into shared memory. A query row is scaled by a power of
// two (largest feature in [128, 256)) and is exact in f16 but for features below 2^-24 of the largest, which lose up to 2^-32
// of it. The page's key scale joins the row's factor of the softmax. Outputs are sums of exp2(x + log2 v_scale - o + 6) and the
// codes, the weight in f16 (2^-11, floor 2^-31 of the row's largest): a page whose values are huge and whose weights are nothing
// costs the others no bits. Sums are kept relative to m. m and o are maxima of a row, of x and of x + log2 v_scale (counted from
// m), that follow where those rise by more than 8. O stays in tensor memory and is rescaled when o follows.
//
// Two threads of the softmax warps own a row, 64 keys each: S is read once, the maximum and the sum need one exchange between two
// warps. (One thread a row, two passes over S: 138 us with two CTAs to an SM, 127 us with two groups of warps at alternate pages;
// this 108.)
//
// What bounds it: a page's chain of softmax steps, 3000 cycles (exponentials 1400, of which the MUFU unit is taken 1024, maximum
// and exchange 600, factors 450, hand-over 400), where its two products take 1000. 4 prompts of 512 to 1024 tokens, 16 heads,
// lists of 16 pages for tiles of 16 tokens (50 GFLOP): 108 us, 0.47 PFLOP/s; an item's end costs two pages' time.
//
// CTA (one to an SM): eight softmax warps; eight that scale an item's queries and convert a page's codes from a ring in shared
// memory, four K and four V; an MMA warp, which issues QK of a page ahead of PV of the page before; a warp that walks over the
// share's pages and one that brings them (bulk copies, a tile of K or V is 16 KB in a row). A role may be a page or two ahead of
// another, and a wait tells only one phase from the next: barriers that such roles share are kept by page or item.
#include "paged_attention.cuh"

namespace sb {
namespace pa {
namespace {

constexpr int CONVERT = 8, MMA = 16, WALK = 17, LOAD = 18, WARPS = 19, THREADS = 32 * WARPS;
constexpr int HALF_TILE = 128 * 256;              // 128 rows of 128 f16: two panels of 64 features, 128-byte swizzle
constexpr int SLOTS = 5;
constexpr int OFF_Q = 0, OFF_K = HALF_TILE, OFF_V = OFF_K + HALF_TILE, OFF_RING = OFF_V + 2 * HALF_TILE;
constexpr int OFF_NAN = OFF_RING + SLOTS * TILE_BYTES;             // int [8][128]: by item, first key whose value has a NaN at a feature
constexpr int OFF_QF = OFF_NAN + 8 * 512;         // float [4][128]: by item, what a row's scores are multiplied by
constexpr int OFF_MAX = OFF_QF + 4 * 512;         // float [2][2][128]: by page, half and row
constexpr int OFF_SUM = OFF_MAX + 4 * 512;        // float [2][2][128]: by item, half and row
constexpr int OFF_INFO = OFF_SUM + 4 * 512;
constexpr int OFF_BAR = OFF_INFO + BATCHES * BATCH_BYTES;
constexpr int B_INFO_FULL = 0, B_INFO_EMPTY = BATCHES, B_FULL = 2 * BATCHES, B_EMPTY = B_FULL + SLOTS, B_K_FULL = B_EMPTY + SLOTS,
              B_K_EMPTY = B_K_FULL + 1, B_V_FULL = B_K_EMPTY + 2, B_V_EMPTY = B_V_FULL + 2, B_S_FULL = B_V_EMPTY + 2,
              B_P_FULL = B_S_FULL + 2, B_Q_FULL = B_P_FULL + 2, B_MAX = B_Q_FULL + 4, B_SUM = B_MAX + 8,
              B_DONE = B_SUM + 4, BARS = B_DONE + 1;
constexpr int OFF_FLAG = OFF_BAR + BARS * 8;      // int [2]: for the MMA warp, with a page's K tile: 1 = the first of an item, 2 = stop
constexpr int OFF_MISC = (OFF_FLAG + 8 + 15) / 16 * 16;
constexpr int SMEM = OFF_MISC + 64 + 1024;        // 1024: alignment of the tiles
static_assert(SMEM <= 227 * 1024 - 512, "shared memory of an SM");
constexpr int TMEM_COLUMNS = 512;                 // S of two pages (and P over it, 32 columns of every 64), O
constexpr int O_COLUMN = 256;
constexpr float LIFT = 6.f;                       // probabilities are exp2(x - m + 6): up to 2^14 before m follows

// kind::f16 instruction descriptor: f16 x f16 -> fp32, M = N = 128.
constexpr uint32_t ID_QK = (1u << 4) | (16u << 17) | (8u << 24), ID_PV = ID_QK | (1u << 16);
constexpr uint32_t HI = (1024u >> 4) | (1u << 14) | (2u << 29);

__device__ __forceinline__ uint32_t half2_of(uint32_t codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes), __NV_E4M3);
  return static_cast<uint32_t>(h.x) | (static_cast<uint32_t>(h.y) << 16);
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// Saturates: scores so huge that their references are rounded by whole numbers may leave a weight above 2^16.
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
// A tile of codes (128 rows of 128 bytes, shared memory) into f16 by 128 threads: eight chunks of 16 codes each. Eight threads
// of a warp read and write two rows, in 16-byte pieces that meet no bank twice.
__device__ __forceinline__ int chunk_row(int t, int i) { return (t >> 2) + 32 * (i & 3); }
__device__ __forceinline__ int chunk_part(int t, int i) { return (t & 3) + 4 * (((i >> 2) ^ (t >> 2)) & 1); }
__device__ __forceinline__ void store_chunk(unsigned char* tile, int row, int part, uint4 x) {
  unsigned char* to = tile + (part >> 2) * (HALF_TILE / 2) + row * 128;
  const int c = (part & 3) * 2;
  *reinterpret_cast<uint4*>(to + ((c ^ (row & 7)) << 4)) =
      make_uint4(half2_of(x.x), half2_of(x.x >> 16), half2_of(x.y), half2_of(x.y >> 16));
  *reinterpret_cast<uint4*>(to + (((c + 1) ^ (row & 7)) << 4)) =
      make_uint4(half2_of(x.z), half2_of(x.z >> 16), half2_of(x.w), half2_of(x.w >> 16));
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* from, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(from),
               "r"(bytes), "r"(bar)
               : "memory");
}
// Clears the NaN codes of a chunk of V and keeps, for each of its 16 features, the first key (counted from `key`) with one.
__device__ __noinline__ uint4 without_nan(uint4 x, int* nan_at, int key) {
  uint32_t w[4] = {x.x, x.y, x.z, x.w};
  for (int b = 0; b < 16; ++b)
    if ((w[b >> 2] >> (8 * (b & 3)) & 0x7f) == 0x7f) {
      w[b >> 2] &= ~(0xffu << (8 * (b & 3)));
      atomicMin(nan_at + b, key);
    }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The rare parts of the softmax (out of line they cost 3 us of 108). 64 columns of TMEM:
// scores from the key `sees` on become -inf; outputs are scaled.
__device__ __forceinline__ void mask_scores(uint32_t taddr, int sees) {
#pragma unroll 1
  for (int c = 0; c < 64; c += 16) {
    uint32_t s[16];
    tmem_ld16(taddr + c, s);
    tc_wait_ld();
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (c + j >= sees) s[j] = 0xff800000u;
    tmem_st16(taddr + c, s);
  }
  tc_wait_st();
}
__device__ __forceinline__ void scale_output(uint32_t taddr, float by) {
  tc_fence_after();
#pragma unroll 1
  for (int c = 0; c < 64; c += 16) {
    uint32_t o[16];
    tmem_ld16(taddr + c, o);
    tc_wait_ld();
#pragma unroll
    for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * by);
    tmem_st16(taddr + c, o);
  }
}

// Probabilities of 64 keys over their scores, and their sum, with exponents of their own. Scores are taken relative to their
// maximum before they are scaled: s f - mu in one rounding is what mu was rounded by at the maximum, more than the exponent's
// range where scores are huge.
__device__ __forceinline__ float rare_page(uint32_t taddr, float f, float top, float offset, float offset_l) {
  float sum = 0.f;
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    uint32_t s[16], h[8];
    tmem_ld16(taddr + 16 * c, s);
    tc_wait_ld();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = __uint_as_float(s[2 * j]) - top, y = __uint_as_float(s[2 * j + 1]) - top;
      sum += ex2_approx(fmaf(x, f, offset_l)) + ex2_approx(fmaf(y, f, offset_l));
      h[j] = pack_half2(ex2_approx(fmaf(x, f, offset)), ex2_approx(fmaf(y, f, offset)));
    }
    tmem_st8(taddr + 8 * c, h);
  }
  return sum;
}

__global__ void __launch_bounds__(THREADS, WIDE_CTAS) paged_wide_kernel(const Params p, int* status) {
  extern __shared__ unsigned char raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  unsigned char* gbase = raw + (base - smem_u32(raw));
  volatile int* misc = reinterpret_cast<volatile int*>(gbase + OFF_MISC);        // [0] TMEM, [1] abort
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Guard guard{misc + 1, status};
  const auto bar = [&](int i) { return base + OFF_BAR + 8 * i; };
  const auto batch_at = [&](uint32_t e) { return reinterpret_cast<int4*>(gbase + OFF_INFO + e * BATCH_BYTES); };

  if (tid == 0) {
    misc[1] = 0;
    const auto init = [&](int first, int n, int count) {
      for (int i = first; i < first + n; ++i) mbar_init(bar(i), count);
    };
    init(B_INFO_FULL, BATCHES, 1);
    init(B_INFO_EMPTY, BATCHES, 17);              // softmax, conversion, loads
    init(B_FULL, SLOTS, 1);
    init(B_EMPTY, SLOTS, 4);
    init(B_K_FULL, 1, 4);
    init(B_K_EMPTY, 2, 1);                        // by page, as all below: who waits for it may be a page ahead
    init(B_V_FULL, 2, 4);
    init(B_V_EMPTY, 2, 1);
    init(B_S_FULL, 2, 1);
    init(B_P_FULL, 2, 8);
    init(B_Q_FULL, 4, 8);                          // by item: QK may be two items of a page each ahead of the softmax
    init(B_MAX, 12, 2);
    init(B_DONE, 1, 1);
    fence_mbar_init();
    p.part_meta[16 * blockIdx.x] = 0;             // no part yet in either of this CTA's places
    p.part_meta[16 * blockIdx.x + 8] = 0;
  }
  if (warp == MMA) {
    tmem_alloc(smem_u32(const_cast<int*>(misc)), TMEM_COLUMNS);
    tmem_relinquish();
  }
  if (tid < 256) reinterpret_cast<int*>(gbase + OFF_NAN)[tid] = 0x7fffffff;
  tc_fence_before();
  const Share share = find_share<WARPS>(p);       // (two barriers of the CTA)
  tc_fence_after();
  const uint32_t tmem = static_cast<uint32_t>(misc[0]);
  uint32_t fills = 0;

  if (warp == WALK) {
    // --------------------------------------------------------------- the share's pages, told as far ahead as there is place
    bool ok = true;
    uint32_t batches = 0;
    const auto next = [&]() {
      const uint32_t e = batches % BATCHES;
      ok = ok && wait_warp(bar(B_INFO_EMPTY + e), ((batches / BATCHES) & 1) ^ 1, guard, 0xd00);
      return batch_at(e);
    };
    walk_share(p, share, ok, [&](const Item& item, int flags, uint32_t pages, int row, int j) {
      int4* to = next();
      if (!ok) return;
      write_batch(p, to, item, flags, pages, row, j);
      if (lane == 0) mbar_arrive(bar(B_INFO_FULL + batches % BATCHES));
      ++batches;
    });
    int4* to = next();
    if (ok && lane == 0) {
      to[0] = make_int4(STOP, 0, 0, 0);
      mbar_arrive(bar(B_INFO_FULL + batches % BATCHES));
    }
    __syncwarp();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  } else if (warp == LOAD) {
    // --------------------------------------------------------------- their tiles
    bool ok = true;
    uint32_t batches = 0;
    int slot = 0, phase = 0;
    const auto load = [&](const void* cache, int row) {
      ok = ok && wait_warp(bar(B_EMPTY + slot), phase ^ 1, guard, 0xd02);
      if (!ok) return;
      if (elect_one()) {
        mbar_expect_tx(bar(B_FULL + slot), TILE_BYTES);
        bulk_load(base + OFF_RING + slot * TILE_BYTES, static_cast<const uint8_t*>(cache) + static_cast<long long>(row) * TILE_BYTES,
                  TILE_BYTES, bar(B_FULL + slot));
      }
      __syncwarp();
      ++fills;
      if (++slot == SLOTS) {
        slot = 0;
        phase ^= 1;
      }
    };
    while (ok) {
      const uint32_t e = batches % BATCHES;
      ok = wait_warp(bar(B_INFO_FULL + e), (batches / BATCHES) & 1, guard, 0xd01);
      if (!ok) break;
      const int4* info = batch_at(e);
      const int flags = info[0].x, count = info[0].y;
      if (flags & STOP) break;
#pragma unroll 1
      for (int n = 0; ok && n < 2 * count; ++n) load(n & 1 ? p.a.v : p.a.k, info[2 + (n >> 1)].x);
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_INFO_EMPTY + e));
      ++batches;
    }
  } else if (warp == MMA) {
    // --------------------------------------------------------------- MMA issuer
    // QK of a page overwrites the S that the PV of the page before the last has read P from: it is issued behind that. The O of
    // an item's first page overwrites the last item's, which the softmax warps have read before they store that page's P.
    bool ok = true, stopped = false;
    int first = 0, second = 0, item = -1;         // pages whose first / second product has been issued
    bool fresh0 = false, fresh1 = false;          // the even / odd page under way is the first of its item
    const auto ready = [&](int which, int parity) { return __all_sync(0xffffffffu, mbar_test_wait(bar(which), parity)) != 0; };
    long long t0 = clock64();
    while (ok) {
      bool tile = false;
      if (!stopped && first - second < 2) {
        tile = ready(B_K_FULL, first & 1);
        if (!tile && first == second) {
          ok = mbar_wait_warp(bar(B_K_FULL), first & 1, guard, 0xd10);
          if (!ok) break;
          tile = true;
        }
      }
      if (tile) {
        const int flag = *reinterpret_cast<volatile int*>(gbase + OFF_FLAG + 4 * (first & 1));
        stopped = __any_sync(0xffffffffu, flag & 2);
        if (!stopped) {
          const bool fresh = __any_sync(0xffffffffu, flag & 1);
          if (fresh) {
            ++item;
            ok = mbar_wait_warp(bar(B_Q_FULL + (item & 3)), (item >> 2) & 1, guard, 0xd11);
            if (!ok) break;
          }
          if (first & 1) fresh1 = fresh;
          else fresh0 = fresh;
          tc_fence_after();
          if (elect_one()) {
            const uint32_t q = (base + OFF_Q) >> 4, k = (base + OFF_K) >> 4;
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) {
              const uint32_t at = (kk >> 2) * (HALF_TILE / 2 >> 4) + (kk & 3) * 2;
              mma_ss_lo<HI, HI>(tmem + (first & 1) * 128, q + at, k + at, ID_QK, kk > 0);
            }
            tc_commit(bar(B_S_FULL + (first & 1)));
            tc_commit(bar(B_K_EMPTY + (first & 1)));
          }
          __syncwarp();
          ++first;
          t0 = clock64();
        }
      }
      if (first == second) {
        if (stopped) break;
        continue;
      }
      if (!ready(B_P_FULL + (second & 1), (second >> 1) & 1)) {
        const bool late = clock64() - t0 > WAIT_LIMIT_CYCLES || *guard.abort_flag;
        if (!stopped && first - second < 2 && !__any_sync(0xffffffffu, late)) continue;
        ok = mbar_wait_warp(bar(B_P_FULL + (second & 1)), (second >> 1) & 1, guard, 0xd12);
        if (!ok) break;
      }
      ok = mbar_wait_warp(bar(B_V_FULL + (second & 1)), (second >> 1) & 1, guard, 0xd13);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t v = ((base + OFF_V + (second & 1) * HALF_TILE) >> 4) | ((HALF_TILE / 2 >> 4) << 16);
        const bool fresh = second & 1 ? fresh1 : fresh0;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          mma_ts_lo<HI>(tmem + O_COLUMN, tmem + (second & 1) * 128 + (kk >> 2) * 64 + (kk & 3) * 8, v + kk * (2048 >> 4), ID_PV, !fresh || kk > 0);
        tc_commit(bar(B_V_EMPTY + (second & 1)));
      }
      __syncwarp();
      ++second;
      t0 = clock64();
    }
    // nothing of the tensor core's is in flight when the CTA gives up its memory
    if (elect_one()) tc_commit(bar(B_DONE));
    __syncwarp();
    mbar_wait_drain(bar(B_DONE), 0);
  } else if (warp >= CONVERT) {
    // --------------------------------------------------------------- pages into f16 tiles: four warps K, four V
    const bool values = warp >= CONVERT + 4;
    const int t = tid & 127, mine = values ? 1 : 0;
    const int group_inverse = (65535 + p.group) / p.group;        // row / group = row * this >> 16 for rows below 128
    const float sign = p.a.scale < 0.f ? -1.f : 1.f, factor = fabsf(p.a.scale) * 1.4426950408889634f;
    bool ok = true, started = false;
    uint32_t batches = 0;
    int item = -1, pages = 0, slot = mine, phase = 0;
    const auto qk_done = [&](int page, int code) {
      ok = wait_warp(bar(B_K_EMPTY + (page & 1)), (page >> 1) & 1, guard, code);
      return ok;
    };
    while (ok) {
      const uint32_t e = batches % BATCHES;
      ok = wait_warp(bar(B_INFO_FULL + e), (batches / BATCHES) & 1, guard, 0xd20);
      if (!ok) break;
      const int4* info = batch_at(e);
      const int flags = info[0].x, count = info[0].y;
      if (flags & STOP) {
        if (values) break;
        if (!qk_done(pages - 1, 0xd21)) break;
        if (t == 0) *reinterpret_cast<volatile int*>(gbase + OFF_FLAG + 4 * (pages & 1)) = 2;
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_K_FULL));
        break;
      }
      if (flags & FIRST) started = false;
      if (count && !started) {
        ++item;
        // The item's queries: half a warp to a row, 8 features to a thread. A thread's pieces come to the places they keep, all
        // in flight at once, and are scaled there.
        if (!qk_done(pages - 1, 0xd27)) break;
        const int rows = info[0].w * p.group, part = lane & 15, row0 = 2 * (warp - CONVERT) + (lane >> 4);
        const auto piece = [&](int row) {
          return gbase + OFF_Q + (part >> 3) * (HALF_TILE / 2) + row * 128 + (((part & 7) ^ (row & 7)) << 4);
        };
        const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(p.a.q) + info[0].z * p.a.q_token +
                                   static_cast<long long>(info[1].x) * p.group * p.a.q_head + part * 8;
#pragma unroll 1
        for (int row = row0; row < 128; row += 16) {
          const int token = row * group_inverse >> 16, g = row - token * p.group;
          const bool in = row < rows;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(piece(row))),
                       "l"(in ? src + token * p.a.q_token + g * p.a.q_head : src), "r"(in ? 16 : 0)
                       : "memory");
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 2
        for (int row = row0; row < 128; row += 16) {
          const uint4 w = *reinterpret_cast<const uint4*>(piece(row));
          uint32_t top = __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
#pragma unroll
          for (int by = 8; by; by >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, by));
          top = max(top & 0xffffu, top >> 16);
          const bool odd = top >= 0x7f80u;        // infinities and NaN: the row ends as NaN
          const int ex = top == 0 || odd ? 0 : min(134 - static_cast<int>(top >> 7), 126);
          const float by = odd ? __int_as_float(0x7fffffff) : power_of_two(ex) * sign;
          const auto scaled = [&](uint32_t pair) {
            const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&pair));
            return pack_half2(x.x * by, x.y * by);
          };
          *reinterpret_cast<uint4*>(piece(row)) = make_uint4(scaled(w.x), scaled(w.y), scaled(w.z), scaled(w.w));
          if (part == 0) reinterpret_cast<float*>(gbase + OFF_QF)[(item & 3) * 128 + row] = factor * power_of_two(-ex);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_Q_FULL + (item & 3)));
      }
#pragma unroll 1
      for (int step = 0; step < count; ++step) {
        const int seen = info[2 + step].y, valid = values ? seen & 0xffff : 128, limit = values ? seen >> 16 : 128;
        ok = wait_warp(bar(B_FULL + slot), phase, guard, 0xd22);
        // the product that read the tile before
        ok = ok && (values ? wait_warp(bar(B_V_EMPTY + (pages & 1)), ((pages >> 1) & 1) ^ 1, guard, 0xd25) : qk_done(pages - 1, 0xd23));
        if (!ok) break;
        if (!started) {
          // V: the place of the item after the next is cleared here. Its first page comes two pages behind at least, and is
          // converted when PV of this one is done: all four warps have been here. (The item that had the place has ended.)
          if (values) reinterpret_cast<int*>(gbase + OFF_NAN)[((item + 2) & 7) * 128 + t] = 0x7fffffff;
        }
        if (t == 0 && !values) *reinterpret_cast<volatile int*>(gbase + OFF_FLAG + 4 * (pages & 1)) = started ? 0 : 1;
        started = true;
        const unsigned char* from = gbase + OFF_RING + slot * TILE_BYTES;
        unsigned char* to = gbase + (values ? OFF_V + (pages & 1) * HALF_TILE : OFF_K);
        const auto piece = [&](int i) {
          return reinterpret_cast<const uint4*>(from + chunk_row(t, i) * 128 + chunk_part(t, i) * 16);
        };
        if (limit == 128 && valid == 128) {       // nothing between the loads: their latencies overlap
#pragma unroll
          for (int i = 0; i < 8; i += 4) {
            const uint4 x0 = *piece(i), x1 = *piece(i + 1), x2 = *piece(i + 2), x3 = *piece(i + 3);
            store_chunk(to, chunk_row(t, i), chunk_part(t, i), x0);
            store_chunk(to, chunk_row(t, i + 1), chunk_part(t, i + 1), x1);
            store_chunk(to, chunk_row(t, i + 2), chunk_part(t, i + 2), x2);
            store_chunk(to, chunk_row(t, i + 3), chunk_part(t, i + 3), x3);
          }
        } else {
#pragma unroll 1
          for (int i = 0; i < 8; ++i) {
            const int row = chunk_row(t, i), part = chunk_part(t, i);
            uint4 x = *piece(i);
            if (row >= valid) {
              x = make_uint4(0, 0, 0, 0);         // what lies behind the sequence may hold anything
            } else if (limit < valid) {
              // Some rows do not see all keys of this page, and probability 0 times NaN is not 0: NaNs go, and the first key with
              // one at a feature is kept, as a distance from the keys that the first token sees; rows that see it get their NaN
              // in the end.
              const auto any = [](uint32_t w) { return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0; };
              if (any(x.x) || any(x.y) || any(x.z) || any(x.w))
                x = without_nan(x, reinterpret_cast<int*>(gbase + OFF_NAN) + (item & 7) * 128 + part * 16, row - limit);
            }
            store_chunk(to, row, part, x);
          }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar(B_EMPTY + slot));
          mbar_arrive(bar(values ? B_V_FULL + (pages & 1) : B_K_FULL));
        }
        slot += 2;
        if (slot >= SLOTS) {
          slot -= SLOTS;
          phase ^= 1;
        }
        ++pages;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_INFO_EMPTY + e));
      ++batches;
    }
  } else {
    // --------------------------------------------------------------- softmax: two threads own a row, 64 keys or features each
    const int quarter = warp & 3, half = warp >> 2, row = 32 * quarter + lane;
    const uint32_t t_row = tmem + (static_cast<uint32_t>(32 * quarter) << 16);
    const int token = row / p.group, g = row - token * p.group;
    float* maxima = reinterpret_cast<float*>(gbase + OFF_MAX);
    float* sums = reinterpret_cast<float*>(gbase + OFF_SUM);
    bool ok = true, fresh = true, odd_values = false;
    uint32_t batches = 0;
    int items = 0, ends = 0, pages = 0, joint = 0;       // joint: pages of which this warp had rows
    float m = -INFINITY, o = -INFINITY, l = 0.f, f_row = 0.f;      // what l is relative to, and O, counted from m
    while (ok) {
      const uint32_t e = batches % BATCHES;
      ok = wait_warp(bar(B_INFO_FULL + e), (batches / BATCHES) & 1, guard, 0xd30);
      if (!ok) break;
      const int4* info = batch_at(e);
      const int flags = info[0].x, count = info[0].y, rows = info[0].w * p.group;
      if (flags & STOP) break;
      if (flags & FIRST) {
        fresh = true;
        odd_values = false;
        m = o = -INFINITY;
        l = 0.f;
      }
      const bool idle = 32 * quarter >= rows;     // none of this warp's rows is one
#pragma unroll 1
      for (int step = 0; step < count; ++step) {
        const int b = pages & 1;
        if (fresh) {
          ok = wait_warp(bar(B_Q_FULL + (items & 3)), (items >> 2) & 1, guard, 0xd31);
          if (!ok) break;
          f_row = reinterpret_cast<const float*>(gbase + OFF_QF)[(items & 3) * 128 + row];
        }
        ok = wait_warp(bar(B_S_FULL + b), (pages >> 1) & 1, guard, 0xd32);
        if (!ok) break;
        const int seen = info[2 + step].y, valid = seen & 0xffff, limit = seen >> 16;
        if (!idle) {
          tc_fence_after();
          const uint32_t t_s = t_row + 128 * b + 64 * half;         // this half's S, and P over it
          if (valid < 128 || limit < 128)
            mask_scores(t_s, min(p.a.causal ? limit + token : limit, valid) - 64 * half);
          uint32_t s[2][32];
          tmem_ld32(t_s, s[0]);
          tmem_ld32(t_s + 32, s[1]);
          tc_wait_ld();
          float top = -INFINITY, other = -INFINITY;
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            top = max3(top, __uint_as_float(s[0][j]), __uint_as_float(s[0][j + 1]));
            other = max3(other, __uint_as_float(s[1][j]), __uint_as_float(s[1][j + 1]));
          }
          top = fmaxf(top, other);
          const int turn = joint & 1;
          maxima[(2 * turn + half) * 128 + row] = top;
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(B_MAX + 2 * quarter + turn));
          ok = wait_warp(bar(B_MAX + 2 * quarter + turn), (joint >> 1) & 1, guard, 0xd33);
          if (!ok) break;
          ++joint;
          top = fmaxf(top, maxima[(2 * turn + (half ^ 1)) * 128 + row]);
          float f = f_row * __int_as_float(info[2 + step].z);
          if (f == 0.f) f = 1e-37f;               // hidden keys stay hidden with a scale of 0
          const bool none = top == -INFINITY;
          if (none) f = 1.f;                      // (the page's scale may be NaN)
          const float mu = none ? -INFINITY : top * f;
          if (m == -INFINITY) {
            m = mu;
          } else if (mu - m > 8.f) {
            l *= ex2_approx(m - mu);
            o -= mu - m;
            m = mu;
          }
          const float log_v = __log2f(__int_as_float(info[2 + step].w)), reach = none ? -INFINITY : mu - m + log_v;
          float keep = 1.f;                       // of O
          if (o == -INFINITY) {
            o = reach;
          } else if (reach - o > 8.f) {
            keep = ex2_approx(o - reach);
            o = reach;
          }
          if (!fresh && __any_sync(0xffffffffu, keep != 1.f)) {
            ok = wait_warp(bar(B_V_EMPTY + (b ^ 1)), ((pages - 1) >> 1) & 1, guard, 0xd34);       // PV of the page before
            if (!ok) break;
            scale_output(t_row + O_COLUMN + 64 * half, keep);
          }
          const float apart = o - log_v;
          // One exponential serves both sums, but where their references are far apart or the scores huge.
          if (__any_sync(0xffffffffu, !none && !(fabsf(apart) <= 60.f && fabsf(mu) <= 65536.f))) {
            l += rare_page(t_s, f, none ? 0.f : top, reach == -INFINITY ? -INFINITY : reach - o + LIFT, none ? -INFINITY : mu - m + LIFT);
          } else {
            const float offset = reach == -INFINITY ? -INFINITY : log_v - o + LIFT - m;
            const float2 f2 = make_float2(f, f), o2 = make_float2(offset, offset);
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t h[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const int k = 16 * (c & 1) + 2 * j;
                float2 y = fma2(make_float2(__uint_as_float(s[c >> 1][k]), __uint_as_float(s[c >> 1][k + 1])), f2, o2);
                y.x = ex2_approx(y.x);
                y.y = ex2_approx(y.y);
                sum = add2(sum, y);
                h[j] = pack_half2(y.x, y.y);
              }
              tmem_st8(t_s + 8 * c, h);
            }
            l += (sum.x + sum.y) * (none ? 1.f : ex2_approx(apart));             // none: 0, or NaN where the scores are
          }
          tc_wait_st();
          tc_fence_before();
        }
        if (limit < valid) {
          ok = wait_warp(bar(B_V_FULL + b), (pages >> 1) & 1, guard, 0xd35);      // what the conversion has seen of NaNs
          if (!ok) break;
          odd_values = true;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_P_FULL + b));
        fresh = false;
        ++pages;
      }
      if (!ok) break;
      if (flags & LAST) {
        const int token0 = info[0].z, head = info[1].x, place = info[1].y;
        if (!fresh) {
          ok = wait_warp(bar(B_V_EMPTY + ((pages - 1) & 1)), ((pages - 1) >> 1) & 1, guard, 0xd36);         // PV of the last page
          if (!ok) break;
          tc_fence_after();
        }
        if (!idle) {
          float* sum_at = sums + (ends & 1) * 256;
          sum_at[half * 128 + row] = l;
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(B_SUM + quarter));
          ok = wait_warp(bar(B_SUM + quarter), ends & 1, guard, 0xd37);
          if (!ok) break;
          const float total = sum_at[row] + sum_at[128 + row];
          // Relative to m + 8, which no score exceeds: a part's sums hold keys * largest value, no more.
          constexpr float DOWN = LIFT + 8.f, SUNK = 1.f / 16384.f;       // 2^-DOWN
          const float of = ex2_approx(o - DOWN), by = total == 0.f ? 0.f : place >= 0 ? of : of / (total * SUNK);
          const long long out_row = (static_cast<long long>(token0) + token) * p.a.hq + head * p.group + g;
          const int* nan_at = reinterpret_cast<const int*>(gbase + OFF_NAN) + (items & 7) * 128 + 64 * half;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t x[16];
            if (fresh) {
#pragma unroll
              for (int j = 0; j < 16; ++j) x[j] = 0;
            } else {
              tmem_ld16(t_row + O_COLUMN + 64 * half + 16 * c, x);
              tc_wait_ld();
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] = __float_as_uint(total == 0.f ? 0.f : __uint_as_float(x[j]) * by);
            if (odd_values) {
#pragma unroll
              for (int j = 0; j < 16; ++j)
                if (nan_at[16 * c + j] < token) x[j] = 0x7fffffffu;
            }
            if (row < rows) {
              if (place >= 0) {
                float4* to = reinterpret_cast<float4*>(p.part_o + (static_cast<long long>(place) * WIDE_ROWS + row) * 128 + 64 * half + 16 * c);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  to[j] = make_float4(__uint_as_float(x[4 * j]), __uint_as_float(x[4 * j + 1]), __uint_as_float(x[4 * j + 2]),
                                      __uint_as_float(x[4 * j + 3]));
              } else {
                uint4* to = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.a.out) + out_row * 128 + 64 * half + 16 * c);
#pragma unroll
                for (int j = 0; j < 2; ++j)
                  to[j] = make_uint4(pack_bf16x2(__uint_as_float(x[8 * j]), __uint_as_float(x[8 * j + 1])),
                                     pack_bf16x2(__uint_as_float(x[8 * j + 2]), __uint_as_float(x[8 * j + 3])),
                                     pack_bf16x2(__uint_as_float(x[8 * j + 4]), __uint_as_float(x[8 * j + 5])),
                                     pack_bf16x2(__uint_as_float(x[8 * j + 6]), __uint_as_float(x[8 * j + 7])));
              }
            }
          }
          tc_fence_before();
          if (half == 0 && row < rows) {
            if (place >= 0)
              *reinterpret_cast<float2*>(p.part_ml + (static_cast<long long>(place) * WIDE_ROWS + row) * 2) = make_float2(m - LIFT + DOWN, total * SUNK);
            else if (p.a.lse)
              p.a.lse[out_row] = total == 0.f ? -INFINITY : (m - LIFT + log2f(total)) * 0.6931471805599453f;
          }
          ++ends;
        }
        if (tid == 0 && place >= 0) {
          int* meta = p.part_meta + 8 * place;
          *reinterpret_cast<int4*>(meta) = make_int4(1, info[1].z, info[1].w, token0);
          *reinterpret_cast<int2*>(meta + 4) = make_int2(info[0].w, head);
        }
        if (!fresh) ++items;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_INFO_EMPTY + e));
      ++batches;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == LOAD && misc[1]) {                   // a wait was given up: copies in flight land before the CTA leaves
    for (uint32_t f = fills > SLOTS ? fills - SLOTS : 0; f < fills; ++f) mbar_wait_drain(bar(B_FULL + f % SLOTS), (f / SLOTS) & 1);
  }
  if (warp == MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLUMNS);
  }
}

}  // namespace

int launch_paged_wide(const Params& p, int* status, DeviceCtx* ctx, cudaStream_t stream) {
  if (!ctx->paged_attr[5]) {
    if (cudaFuncSetAttribute(paged_wide_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess)
      return set_error(SB_ERR_CUDA, "shared memory of the paged attention");
    ctx->paged_attr[5] = 1;
  }
  paged_wide_kernel<<<p.ctas, THREADS, SMEM, stream>>>(p, status);
  return check_kernel_launch();
}

}  // namespace pa
}  // namespace sb
