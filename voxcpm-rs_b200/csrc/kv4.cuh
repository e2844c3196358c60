// The 4-bit KV cache: row format helpers and launch arguments shared by its kernels.
//
// A key or value row of d numbers is d / 2 bytes of e2m1 codes (dim 2j in the low nibble of
// byte j) and d / 16 e4m3 scales, one for each 16 dims: value = e2m1(code) * e4m3(scale).  A
// code has 2 significant bits and a scale 4, and |value| lies in [2^-10, 2688], so every value
// is exact in f16 (and in bf16 and f32).
#pragma once
#include <cstdint>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "../../include/voxcpm_b200.h"

namespace vx {

constexpr int KV4_GROUP = 16;  // dims that share a scale

// The two e2m1 numbers of a byte, low nibble first, as f16.  (The byte goes through cvt.u8.u32:
// taken apart with mov.b32 {b0, ..} straight from an 8-bit load, nvcc 12.9 converted zeros.)
__device__ __forceinline__ uint32_t e2m1x2_to_h2(uint32_t byte) {
  uint32_t h;
  asm("{\n\t.reg .b8 b;\n\t"
      "cvt.u8.u32 b, %1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b;\n\t}"
      : "=r"(h)
      : "r"(byte));
  return h;
}

// The eight e2m1 numbers of a word as four f16 pairs, byte by byte.
__device__ __forceinline__ void e2m1x8_to_h2(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}

// Two e4m3 numbers (low byte first) as f16.
__device__ __forceinline__ uint32_t e4m3x2_to_h2(uint32_t two) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short)two));
  return h;
}

__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// (lo, hi) rounded to f16
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// 2^x, to 2 ulp; results below 2^-126 are 0
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float e4m3_to_f32(uint32_t b) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)b, __NV_E4M3)));
}

__device__ __forceinline__ float h2_lo(uint32_t h) {
  return __half2float(__ushort_as_half((unsigned short)(h & 0xffff)));
}
__device__ __forceinline__ float h2_hi(uint32_t h) {
  return __half2float(__ushort_as_half((unsigned short)(h >> 16)));
}

// log2(e): scores are kept in base 2, so that a probability is one ex2
constexpr float KV4_LOG2E = 1.4426950408889634f;

}  // namespace vx
