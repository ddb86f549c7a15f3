// Attention of new tokens over the 8-bit paged cache.
//
//   s_ij = scale * q_i . (k_scale * k_j)          keys j <= i + k_len - q_len of the request (causal) in the pages taken
//   o_i = sum_j softmax(s_i)_j v_scale v_j        lse_i = ln sum_j exp s_ij;  no key: o = 0, lse = -inf
//
// One CTA per (token, KV head): thread = key for the scores, feature for the output.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include "internal.h"
#include "paged.cuh"
#include "ptx.cuh"

namespace sb {
namespace {

constexpr int THREADS = 128;
constexpr int HEADS = 8;      // query heads of one pass

__device__ __forceinline__ float2 decode2(uint32_t codes) {
  return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes), __NV_E4M3)));
}

__device__ __forceinline__ float block_max(float x, float* scratch) {
  for (int by = 16; by; by >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, by));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
  __syncthreads();
  return fmaxf(fmaxf(scratch[0], scratch[1]), fmaxf(scratch[2], scratch[3]));
}

__device__ __forceinline__ float block_sum(float x, float* scratch) {
  for (int by = 16; by; by >>= 1) x += __shfl_xor_sync(0xffffffffu, x, by);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
  __syncthreads();
  return (scratch[0] + scratch[1]) + (scratch[2] + scratch[3]);
}

__global__ void __launch_bounds__(THREADS) paged_attention_kernel(PagedAttentionArgs a) {
  __shared__ float s_q[HEADS][128], s_p[HEADS][128], scratch[4];
  const int tid = threadIdx.x, token = blockIdx.x, head = blockIdx.y;
  const int group = a.hq / a.hkv;
  const auto start = [&](int r) { return min(max(__ldg(a.cu_q + r), 0), a.total_q); };
  const int r = warp_last_at_most(a.batch, token, [&](int i) { return static_cast<long long>(start(i)); });
  const int begin = start(r), end = start(r + 1);
  if (token < begin || token >= end) return;
  const int k_len = max(__ldg(a.seq + r), 0);
  const int limit = a.causal ? k_len - (end - token) + 1 : k_len;      // keys seen
  const int held = min((k_len + 127) >> 7, a.width);
  const int32_t* list = nullptr;
  int steps = held;
  if (a.ids) {
    const long long lists = a.tile == 1 ? a.total_q : a.total_q / a.tile + a.batch;
    const long long row = first_list_row(begin, r, a.tile) + (token - begin) / a.tile;
    list = a.ids + (head * lists + row) * a.topk;
    steps = a.topk;
  }
  for (int g0 = 0; g0 < group; g0 += HEADS) {
    const int heads = min(HEADS, group - g0);
    __syncthreads();
    for (int g = 0; g < heads; ++g)
      s_q[g][tid] = __bfloat162float(static_cast<const __nv_bfloat16*>(
          a.q)[token * a.q_token + (head * group + g0 + g) * a.q_head + tid]) * a.scale;
    __syncthreads();
    float top[HEADS], sum[HEADS], o[HEADS];
    for (int g = 0; g < HEADS; ++g) top[g] = -INFINITY, sum[g] = o[g] = 0.f;
    for (int step = 0; step < steps; ++step) {
      const int j = list ? __ldg(list + step) : step;
      if (j < 0 || j >= held || j * 128LL >= limit) continue;
      const int page = __ldg(a.table + r * a.table_stride + j);
      if (page < 0 || page >= a.pages) continue;
      const int seen = min(limit - j * 128, 128);
      const long long at = static_cast<long long>(page) * a.hkv + head;
      const float k_scale = __ldg(a.k_scale + at), v_scale = __ldg(a.v_scale + at);
      const uint32_t* k = static_cast<const uint32_t*>(a.k) + (at * 128 + tid) * 32;
      const uint8_t* v = static_cast<const uint8_t*>(a.v) + at * (128 * 128);
      float x[HEADS];
      for (int g = 0; g < HEADS; ++g) x[g] = 0.f;
      for (int d = 0; d < 32; ++d) {
        const uint32_t w = __ldg(k + d);
        const float2 lo = decode2(w), hi = decode2(w >> 16);
        for (int g = 0; g < HEADS; ++g)
          x[g] += s_q[g][4 * d] * lo.x + s_q[g][4 * d + 1] * lo.y + s_q[g][4 * d + 2] * hi.x + s_q[g][4 * d + 3] * hi.y;
      }
      for (int g = 0; g < heads; ++g) {
        const float s = tid < seen ? x[g] * k_scale : -INFINITY;
        const float m = fmaxf(top[g], block_max(s, scratch));
        const float base = m == -INFINITY ? 0.f : m;
        const float p = tid < seen ? expf(s - base) : 0.f;
        const float keep = expf(top[g] - base);
        top[g] = m;
        sum[g] = sum[g] * keep + p;
        o[g] *= keep;
        s_p[g][tid] = p;
      }
      __syncthreads();
      for (int i = 0; i < seen; ++i) {
        const float value = decode2(__ldg(v + i * 128 + tid)).x * v_scale;
        for (int g = 0; g < heads; ++g) o[g] += s_p[g][i] * value;
      }
      __syncthreads();
    }
    for (int g = 0; g < heads; ++g) {
      const float total = block_sum(sum[g], scratch);
      const long long row = static_cast<long long>(token) * a.hq + head * group + g0 + g;
      const bool dead = total == 0.f;
      static_cast<__nv_bfloat16*>(a.out)[row * 128 + tid] = __float2bfloat16(dead ? 0.f : o[g] / total);
      if (a.lse && tid == 0) a.lse[row] = dead ? -INFINITY : top[g] + logf(total);
    }
  }
}

}  // namespace

long long paged_attention_workspace_bytes(int, int, int, int, bool, int) { return 0; }

int launch_paged_attention(const PagedAttentionArgs& a, cudaStream_t stream) {
  paged_attention_kernel<<<dim3(a.total_q, a.hkv), THREADS, 0, stream>>>(a);
  return check_kernel_launch();
}

}  // namespace sb
