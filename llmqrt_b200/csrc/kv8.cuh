// A paged key/value cache in 8 bits: [pages, Hkv, page, d] codes (e4m3 or int8), one fp32 scale for each page and head.
// A page's rows of one head are contiguous: what a scale belongs to is one piece of memory.
#pragma once
#include "common.cuh"

namespace llmqrt {

constexpr float kKv8Floor = 1e-12f, kKv8Most = 3.3895314e38f;      // least and greatest (bf16's) maximum that a scale is made for

// The scale for values of at most `top`.  int8: top / 127.  e4m3: the least power of two that brings top within 448 -- a
// floating-point code loses nothing by a scale up to twice as large as it could be, and requantizing by a power of two only
// rounds where a value leaves e4m3's normal numbers.  An infinity counts as the greatest number of bf16.
template <bool INT8> __device__ __forceinline__ float kv8_scale(float top) {
  top = fminf(fmaxf(top, kKv8Floor), kKv8Most);
  if constexpr (INT8) return __fdiv_rn(top, 127.f);
  const uint32_t u = __float_as_uint(__fdiv_rn(top, 448.f));
  return __uint_as_float((u + 0x7fffffu) & 0x7f800000u);
}
// Sixteen codes of values x * inv: int8 rounded to even within +-127 (NaN: 0), e4m3 within +-448 (NaN stays one).
template <bool INT8> __device__ __forceinline__ uint4 kv8_encode(const float (&x)[16], float inv) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = __fmul_rn(x[4 * i], inv), b = __fmul_rn(x[4 * i + 1], inv), c = __fmul_rn(x[4 * i + 2], inv), d = __fmul_rn(x[4 * i + 3], inv);
    if constexpr (INT8) {
      auto r = [](float v) { return max(__float2int_rn(v), -127); };      // (the conversion saturates, NaN gives 0; the pack saturates at 127)
      w[i] = pack_sat_s8(r(a), r(b), r(c), r(d));
    } else {
      w[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3) |
             ((uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3) << 16);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Four codes (one word) as two pairs of fp16: both kinds of code are exact in fp16.
template <bool INT8> __device__ __forceinline__ void kv8_word_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (INT8) {
    // v + 128 in the mantissa of 1024 is 1152 + v: one subtraction gives two values
    const uint32_t u = w ^ 0x80808080u, a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 bias = __float2half2_rn(1152.f);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), bias), y = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(w));
  }
}
template <bool INT8> __device__ __forceinline__ void kv8_decode(const uint4& v, float (&x)[16]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t lo, hi;
    kv8_word_to_half<INT8>(w[i], lo, hi);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    x[4 * i] = a.x; x[4 * i + 1] = a.y; x[4 * i + 2] = b.x; x[4 * i + 3] = b.y;
  }
}

}  // namespace llmqrt
