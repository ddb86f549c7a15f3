// NVFP4 quantisation of one group of 16 features.
// Rule (no counterpart in the reference, which feeds random bytes):
//   scale_g = e4m3_rne(min(amax_g / 6, 448)); code = nearest e2m1 to x / scale_g,
//   ties to the even code, saturating at 6; scale 0 -> codes 0.
#pragma once
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace sb {

__device__ __forceinline__ uint32_t e2m1_code(float ratio) {
  const float a = fabsf(ratio);
  uint32_t c = 0;
  c = (a > 0.25f) ? 1u : c;                  // tie 0.25 -> 0
  c = (a >= 0.75f) ? 2u : c;                 // tie 0.75 -> 1.0 (code 2)
  c = (a > 1.25f) ? 3u : c;                  // tie 1.25 -> 1.0
  c = (a >= 1.75f) ? 4u : c;                 // tie 1.75 -> 2.0
  c = (a > 2.5f) ? 5u : c;                   // tie 2.5 -> 2.0
  c = (a >= 3.5f) ? 6u : c;                  // tie 3.5 -> 4.0
  c = (a > 5.0f) ? 7u : c;                   // tie 5.0 -> 4.0
  return (c != 0 && ratio < 0.f) ? (c | 8u) : c;
}

// Codes of features 0-7 and 8-15 (low nibble first) and the e4m3 bits of the scale.
__device__ __forceinline__ __nv_fp8_storage_t quantize_nvfp4_group(const float (&v)[16], uint32_t& lo, uint32_t& hi) {
  float amax = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) amax = fmaxf(amax, fabsf(v[e]));
  const float want = fminf(__fdiv_rn(amax, 6.0f), 448.0f);
  const __nv_fp8_storage_t bits = __nv_cvt_float_to_fp8(want, __NV_SATFINITE, __NV_E4M3);
  const float sc = __half2float(__half(__nv_cvt_fp8_to_halfraw(bits, __NV_E4M3)));
  lo = hi = 0;
  if (sc > 0.f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) lo |= e2m1_code(__fdiv_rn(v[e], sc)) << (4 * e);
#pragma unroll
    for (int e = 0; e < 8; ++e) hi |= e2m1_code(__fdiv_rn(v[8 + e], sc)) << (4 * e);
  }
  return bits;
}

// The same for values that are bf16 numbers, without a division. A border between two codes is t * scale with t of three
// significant bits and a scale of four: its seven bits and the eight of a value are apart by 2^-8 of their size, or equal. So a
// quotient that is off by a few 2^-23 is on the right side of every border but where it is equal, and rounding it to twelve
// bits puts it back on the border there: the conversion (to nearest even, as the rule) then sees what the division would give.
__device__ __forceinline__ __nv_fp8_storage_t quantize_nvfp4_group_bf16(const float (&v)[16], uint32_t& lo, uint32_t& hi) {
  float amax = 0.f;
  bool nan = false;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    amax = fmaxf(amax, fabsf(v[e]));
    nan |= v[e] != v[e];
  }
  if (nan) return quantize_nvfp4_group(v, lo, hi);
  const float want = fminf(__fdiv_rn(amax, 6.0f), 448.0f);
  const __nv_fp8_storage_t bits = __nv_cvt_float_to_fp8(want, __NV_SATFINITE, __NV_E4M3);
  const float sc = __half2float(__half(__nv_cvt_fp8_to_halfraw(bits, __NV_E4M3)));
  const float inv = sc > 0.f ? 1.0f / sc : 0.f;
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 16; e += 2) {
    const float a = __uint_as_float((__float_as_uint(v[e] * inv) + 0x800u) & 0xfffff000u);
    const float b = __uint_as_float((__float_as_uint(v[e + 1] * inv) + 0x800u) & 0xfffff000u);
    uint32_t pair;
    asm("{\n\t"
        ".reg .b8 c;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %1, %2;\n\t"
        "cvt.u32.u8 %0, c;\n\t"
        "}"
        : "=r"(pair)
        : "f"(b), "f"(a));
    w[e >> 3] |= pair << (4 * (e & 7));
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {                // a code of magnitude 0 has no sign
    const uint32_t magnitude = w[i] & 0x77777777u;
    w[i] = magnitude | (w[i] & (magnitude + 0x77777777u) & 0x88888888u);
  }
  lo = w[0];
  hi = w[1];
  return bits;
}

}  // namespace sb
