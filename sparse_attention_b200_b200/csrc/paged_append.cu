// New keys and values into the 8-bit paged cache: e4m3 codes with one fp32 scale for each (page, head), and the NVFP4 index
// vectors of the keys.
//
// The new tokens of a request fill its last page and then whole pages: at most one run of rows per page. For the run of a
// (page, head)
//   a = max |x| over the run's finite values
//   s = 2^e, e the smallest whole number with a <= 448 * 2^e, at least -100
//   rows before the run in its page (a run that does not begin at row 0): s = max(s, old s), and where s grew the codes of
//   those rows are multiplied by old s / s and rounded again
//   code = e4m3(x / s), to nearest even, +-inf to +-448, NaN stays NaN
// A page whose scale was set elsewhere keeps it while it is large enough, a power of two or not: its new rows are multiplied by
// 1 / s in 32 bits then. Scales are finite and not negative.
// A scale that is a power of two costs no precision (e4m3 is a floating format) and makes growth exact but for codes that
// become subnormal: a page that is filled token by token is not rounded over and over.
//
// What bounds it: HBM, 256 B read and 128 B (+72 B of index) written per row; a decode step by latency. One CTA does one
// (run, head) of K or of V: the rows stay in registers between the maximum and the conversion, so they are read once, and
// nobody else touches the page's rows or scale, so nothing is ordered between CTAs. Thread = 16 features of a row (the group
// of an NVFP4 scale): 32 B in, 16 B out, eight threads write a row of 128 B. 64 requests of up to 8 tokens: 6.3 us; 8 prompts of
// 512 to 4096 tokens, 4 heads, with the index (55 MB): 16.7 us, 3.3 TB/s, two waves of CTAs, issue slots 58 % taken: a
// CTA loads, meets, converts and stores in turn, and waits for each. K (whose index is most of the arithmetic) before V: taken
// in turns they took 18.6 us; 512 threads 19.6.
#include <cuda_bf16.h>
#include "internal.h"
#include "nvfp4_quantize.cuh"
#include "paged.cuh"

namespace sb {
namespace {

constexpr int THREADS = 256;
constexpr int PASSES = 128 * 8 / THREADS;
constexpr int LOWEST_EXPONENT = -100;

// e of the scale for a largest magnitude given as the bits of a bf16
__device__ __forceinline__ int scale_exponent(uint32_t bf16_bits) {
  const int e = static_cast<int>(bf16_bits >> 7) - 127 - 8 + ((bf16_bits & 0x7fu) > 0x60u ? 1 : 0);   // 448 = 1.75 * 2^8
  return max(e, LOWEST_EXPONENT);
}

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }

// the four codes of two packed pairs of bf16, times inv
__device__ __forceinline__ uint32_t codes4(uint32_t x, uint32_t y, float inv) {
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&y));
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a.x * inv, a.y * inv), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(b.x * inv, b.y * inv), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

__device__ __forceinline__ uint32_t rescaled4(uint32_t codes, float by) {
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes >> (16 * i)), __NV_E4M3);
    const float2 f = __half22float2(__half2(h));
    out |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(f.x * by, f.y * by), __NV_SATFINITE, __NV_E4M3)) << (16 * i);
  }
  return out;
}

__global__ void __launch_bounds__(THREADS) append_tokens_kernel(AppendArgs a) {
  __shared__ uint32_t s_top[THREADS / 32];
  const int tid = threadIdx.x;
  const int head = blockIdx.y;
  const bool is_value = blockIdx.z != 0;
  // Run blockIdx.x: request r has the places [cu / 128 + 2r, ...) , room for its n / 128 + 2 runs at most.
  const long long item = blockIdx.x;
  const auto start_of = [&](int r) { return min(max(__ldg(a.cu_q + r), 0), a.total_q); };
  const int r = warp_last_at_most(a.batch, item, [&](int i) { return static_cast<long long>(start_of(i) >> 7) + 2LL * i; });
  const int first = start_of(r), n = start_of(r + 1) - first;
  const int run = static_cast<int>(item - ((first >> 7) + 2LL * r));
  if (n <= 0) return;
  const long long slot0 = __ldg(a.slots + first);
  if (slot0 < 0) return;                                   // a request without pages for its tokens
  const int offset0 = static_cast<int>(slot0 & 127);
  const int token = run ? 128 * run - offset0 : 0;         // first token of the run, within the request
  if (run < 0 || token >= n) return;
  const long long slot = run ? __ldg(a.slots + first + token) : slot0;
  const long long page = slot >> 7;
  if (slot < 0 || page >= a.pages) return;
  const int offset = static_cast<int>(slot & 127);
  const int count = min(n - token, 128 - offset);
  const long long page_head = page * a.heads + head;
  float* scale = (is_value ? a.v_scale : a.k_scale) + page_head;
  uint8_t* rows = static_cast<uint8_t*>(is_value ? a.v_cache : a.k_cache) + page_head * (128 * 128);
  const long long token_stride = is_value ? a.v_token : a.k_token;
  const int row0 = tid >> 3, group = tid & 7;
  const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(is_value ? a.v : a.k) +
                             head * (is_value ? a.v_head : a.k_head) + (first + token) * token_stride + group * 16;
  uint4 x[PASSES][2];
  uint32_t top = 0;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int row = row0 + p * (THREADS / 8);
    if (row < count) {
      const uint4* from = reinterpret_cast<const uint4*>(src + row * token_stride);
      x[p][0] = __ldg(from);
      x[p][1] = __ldg(from + 1);
    }
  }
  const float old = *scale;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    if (row0 + p * (THREADS / 8) >= count) continue;
    const uint32_t w[8] = {x[p][0].x, x[p][0].y, x[p][0].z, x[p][0].w, x[p][1].x, x[p][1].y, x[p][1].z, x[p][1].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t m = w[i] & 0x7fff7fffu;
      top = __vmaxu2(top, m & __vcmpltu2(m, 0x7f807f80u));   // finite magnitudes order as their bits do
    }
  }
  top = max(top & 0xffffu, top >> 16);
  top = __reduce_max_sync(0xffffffffu, top);
  if ((tid & 31) == 0) s_top[tid >> 5] = top;
  __syncthreads();                                         // every thread has read the old scale, too
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) top = max(top, s_top[w]);
  int e = scale_exponent(top);
  float s = power_of_two(e), inv = power_of_two(-e);
  if (offset > 0 && old >= s) {
    s = old;
    inv = 1.0f / old;
  } else if (offset > 0) {
    const float by = old * inv;                            // powers of two: exact; a page of scale 0 held zeros
    for (int i = tid; i < offset * 8; i += THREADS) {
      uint4* at = reinterpret_cast<uint4*>(rows) + i;
      uint4 c = *at;
      c.x = rescaled4(c.x, by);
      c.y = rescaled4(c.y, by);
      c.z = rescaled4(c.z, by);
      c.w = rescaled4(c.w, by);
      *at = c;
    }
  }
  if (tid == 0) *scale = s;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int row = row0 + p * (THREADS / 8);
    if (row >= count) continue;
    const uint32_t w[8] = {x[p][0].x, x[p][0].y, x[p][0].z, x[p][0].w, x[p][1].x, x[p][1].y, x[p][1].z, x[p][1].w};
    const uint4 c = make_uint4(codes4(w[0], w[1], inv), codes4(w[2], w[3], inv), codes4(w[4], w[5], inv), codes4(w[6], w[7], inv));
    *reinterpret_cast<uint4*>(rows + (offset + row) * 128 + group * 16) = c;
    if (!is_value && a.k_index) {
      float v[16];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
      uint32_t lo, hi;
      const uint8_t bits = quantize_nvfp4_group_bf16(v, lo, hi);
      const long long vector = page_head * 128 + offset + row;
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.k_index) + vector * 64 + group * 8) = make_uint2(lo, hi);
      static_cast<uint8_t*>(a.k_index_scale)[vector * 8 + group] = bits;
    }
  }
}

}  // namespace

int launch_append_tokens(const AppendArgs& a, cudaStream_t stream) {
  const dim3 grid(a.total_q / 128 + 2 * a.batch, a.heads, 2);
  append_tokens_kernel<<<grid, THREADS, 0, stream>>>(a);
  return check_kernel_launch();
}

}  // namespace sb
