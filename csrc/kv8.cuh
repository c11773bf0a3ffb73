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

// 2^e of a row's exponent byte; NaN for a row that is not finite.  Other exponents outside the format's
// range are clamped into it (a cache that was never written).
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

// Two fp32 lanes per instruction.
__device__ __forceinline__ uint64_t f32x2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack(uint64_t a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// Denormal inputs count as zero: 2^x of a masked score below may come out as one.
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Joins `count` partial softmax rows: ml(i) = (maximum in log2 units, sum), src(i) = D unnormalised
// outputs, both relative to that maximum.  W warps of one block take the parts in turn and add their
// sums in order, so the result does not depend on timing; the caller's block has 4 / W rows, and
// `red` 4 * D floats of shared memory.  A part without a maximum is empty (sum 0, its outputs
// unwritten) or carries a NaN.  Every thread of the block calls it; out is written by each row's first warp.
template <int D, int W, class Ml, class Src>
__device__ __forceinline__ void join_parts(int count, Ml ml, Src src, __nv_bfloat16* out, float* red) {
  constexpr int PER = D / 32;
  const int lane = threadIdx.x & 31, w = (threadIdx.x >> 5) % W;
  float mm = -INFINITY;
  for (int i = lane; i < count; i += 32) mm = fmaxf(mm, ml(i).x);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, d));
  float acc[PER], sum = 0.f;
#pragma unroll
  for (int k = 0; k < PER; ++k) acc[k] = 0.f;
  for (int base = 0; base < count; base += 32) {
    float2 v = make_float2(-INFINITY, 0.f);
    if (base + lane < count) v = ml(base + lane);
    const float f = v.x == -INFINITY ? (v.y == 0.f ? 0.f : 1.f) : ex2(v.x - mm);
    sum += v.y * f;
    const int m = min(32, count - base);
#pragma unroll 4
    for (int i = w; i < m; i += W) {
      const float fi = __shfl_sync(0xffffffffu, f, i);
      float x[PER];
#pragma unroll
      for (int k = 0; k < PER; ++k) x[k] = 0.f;
      if (fi != 0.f) {
        const float* s = src(base + i) + lane * PER;
        if constexpr (PER == 4) {
          const float4 y = *reinterpret_cast<const float4*>(s);
          x[0] = y.x, x[1] = y.y, x[2] = y.z, x[3] = y.w;
        } else {
          const float2 y = *reinterpret_cast<const float2*>(s);
          x[0] = y.x, x[1] = y.y;
        }
      }
#pragma unroll
      for (int k = 0; k < PER; ++k) acc[k] += x[k] * fi;
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if constexpr (W > 1) {
#pragma unroll
    for (int k = 0; k < PER; ++k) red[(threadIdx.x >> 5) * D + lane * PER + k] = acc[k];
    __syncthreads();
    if (w != 0) return;
#pragma unroll
    for (int u = 1; u < W; ++u)
#pragma unroll
      for (int k = 0; k < PER; ++k) acc[k] += red[((threadIdx.x >> 5) + u) * D + lane * PER + k];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int k = 0; k < PER; k += 2)
    *reinterpret_cast<__nv_bfloat162*>(out + lane * PER + k) = __floats2bfloat162_rn(acc[k] * inv, acc[k + 1] * inv);
}

}  // namespace kv8
}  // namespace omni
