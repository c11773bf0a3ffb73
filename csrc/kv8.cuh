// The 8-bit paged KV cache: its form and the device helpers that read it.
//
// Codes   e4m3 [pages, Hkv, 64, D]; a row (one token of one KV head) is D bytes.
// Scales  one power-of-two exponent (int8) per row, [pages, Hkv, 64].
// A row stands for code * 2^e.  e is the smallest integer in [-60, 60] that keeps
// max|x| * 2^-e <= 448 (values past 448 * 2^60 saturate); a row that held an infinity or a
// NaN has exponent -128 and codes 0, and stands for NaN throughout.
//
// Why powers of two: e4m3 is a floating-point format, so its relative precision (4 significant
// bits) is the same under any scale, and a scale that is a power of two costs one byte a row,
// makes every held value exact in bf16 and fp32, and makes the quantisation independent of the
// order of its arithmetic.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

namespace omni {
namespace kv8 {

constexpr int kPage = 64;
constexpr int kExpMin = -60;
constexpr int kExpMax = 60;
constexpr int kExpBad = -128;

// 2^e of a row's exponent byte; NaN for a row that is not finite.  Exponents outside the format's
// range (a cache that was never written) are clamped into it.
__device__ __forceinline__ float pow2_of(int e) {
  if (e == kExpBad) return __int_as_float(0x7fc00000);
  e = max(kExpMin, min(kExpMax, e));
  return __int_as_float((e + 127) << 23);
}

// Exponent of a row from the bit pattern of its largest magnitude (fp32): amax = 1.f * 2^x is
// held at x - 8 when 1.f <= 1.75 (448 = 1.75 * 2^8) and at x - 7 above.
__device__ __forceinline__ int exponent_of(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return kExpBad;
  if (amax_bits == 0u) return kExpMin;
  const int x = static_cast<int>(amax_bits >> 23) - 127;
  const int e = x - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(kExpMin, min(kExpMax, e));
}

// Four e4m3 codes (bytes 0 .. 3) as two fp16 pairs (exact).
__device__ __forceinline__ void e4m3x4_to_f16x4(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}\n"
      : "=r"(lo), "=r"(hi)
      : "r"(four));
}

__device__ __forceinline__ float4 e4m3x4_to_f32(uint32_t four) {
  uint32_t lo, hi;
  e4m3x4_to_f16x4(four, lo, hi);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return make_float4(a.x, a.y, b.x, b.y);
}

// A block-table entry outside the cache reads the reserved padding page 0.
__device__ __forceinline__ int checked_page(int page, int num_pages) {
  return static_cast<unsigned>(page) >= static_cast<unsigned>(num_pages) ? 0 : page;
}

}  // namespace kv8
}  // namespace omni
