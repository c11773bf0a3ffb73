// Write and read of the 8-bit paged KV cache (form: kv8.cuh).
//
// kv8_store: one launch takes a step's fused QKV rows [T, (Hq + 2 Hkv) D] and does per head
//   y = x * rsqrt(mean(x^2) + eps) * w          (q and k, optional)
//   z = y rotated by its token's positions      (q and k; RoPE / M-RoPE / partial / none)
// in fp32, then rounds once: q to bf16 rows, k and v to e4m3 codes with a power-of-two exponent
// per (token, head) at the token's slot.  Nothing is written back into the QKV rows.
//
// kv8_read: rows by slot, as bf16 (exact).
//
// Both are bound by bytes; the write waits besides for each token's position, its angles and a barrier, in turn
// (62 % of issue slots, 40 % of DRAM).  Measured, the write in a graph: 8191 tokens of 32 + 2 x 4 heads of 128 with
// norm, halves 35 us = 4.6 TB/s, adjacent pairs 35, no rotation or norm 27, halves of 24 dims (partners through
// shared memory) 81; of 32 + 2 x 8 heads of 64 24, 24, 16, 60.  130,000 rows of 2 x 4 heads of 128 read in 73 us =
// 5.5 TB/s (copy: 6.55).
//
// Reference counterpart: the fp8 KV-cache option of SGLang's token-to-KV pool behind
// sglang_omni/engines/ar/sglang_backend/server_args_builder.py:10-35 (kv_cache_dtype there).
#include <algorithm>

#include "host_util.h"
#include "kv8.cuh"
#include "omni_kernels.h"
#include "pdl.cuh"

namespace omni {
namespace {

using namespace kv8;

__device__ __forceinline__ void unpack8(const uint4& p, float (&f)[8]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&p);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __bfloat1622float2(h[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}

__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint4 p;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&p);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
  return p;
}

// Position row (0 t, 1 h, 2 w) that rotates pair j.
__device__ __forceinline__ int rope_axis(int j, const Kv8StoreArgs& a) {
  if (a.pos_rows != 3) return 0;
  if (a.interleaved) {
    if ((j % 3) == 1 && j < 3 * a.section[1]) return 1;
    if ((j % 3) == 2 && j < 3 * a.section[2]) return 2;
    return 0;
  }
  return j < a.section[0] ? 0 : (j < a.section[0] + a.section[1] ? 1 : 2);
}

// A head row is D / 16 lanes of 16 elements (two 16-byte loads), so a warp takes 32 / (D / 16) heads of one
// token at a time, `passes` such groups one after another (the next group's rows are read ahead).  With
// halves, a lane holds 8 elements and their 8 partners, so a rotation stays in the lane.  The grid's first
// dimension is the token: its angles are looked up once per block, one pair per thread.
enum Rope : int {
  kNone,        // no rotation
  kPairs,       // adjacent pairs
  kHalves,      // halves, rot a multiple of 16
  kOddHalves,   // halves of any size: partners through shared memory
};
template <int D, int kRope>
__global__ void __launch_bounds__(kRope == kOddHalves ? 256 : 128, kRope == kOddHalves ? 2 : 7) kv8_store_kernel(const Kv8StoreArgs a, int passes) {
  constexpr int L = D / 16;         // lanes per head
  constexpr int HW = 32 / L;        // heads per warp and pass
  __shared__ float rows[kRope == kOddHalves ? 8 : 1][HW][D];   // partner exchange
  __shared__ __align__(16) float angle[2][D / 2];  // cos, sin of the token's pairs
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane / L, l = lane - sub * L;
  const int heads = a.hq + 2 * a.hkv;
  const int tok = blockIdx.x;
  const int head0 = (blockIdx.y * (blockDim.x >> 5) + warp) * HW * passes + sub;
  const int half = a.rot_dim >> 1;
  // the lane's two groups of 8 elements
  const bool rotates = kRope == kHalves ? l * 16 < a.rot_dim : l * 16 < a.rot_dim && kRope != kNone;
  const int e0 = kRope == kHalves && rotates ? l * 8 : l * 16;
  const int e1 = kRope == kHalves && rotates ? l * 8 + half : l * 16 + 8;
  grid_dep_wait();
  grid_dep_launch();   // not before the wait: a dependent grid would hold its shared memory while a GEMM still runs
  const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(a.qkv) + static_cast<int64_t>(tok) * a.qkv_stride;
  uint4 raw[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
  auto fetch = [&](int head) {
    raw[0] = *reinterpret_cast<const uint4*>(src + head * D + e0);
    raw[1] = *reinterpret_cast<const uint4*>(src + head * D + e1);
  };
  if (head0 < heads) fetch(head0);
  if constexpr (kRope != kNone) {
    for (int j = threadIdx.x; j < half; j += blockDim.x) {
      const int p = max(0, min(a.positions[static_cast<int64_t>(rope_axis(j, a)) * a.tokens + tok], a.max_pos - 1));
      angle[0][j] = a.cos_tab[static_cast<int64_t>(p) * half + j];
      angle[1][j] = a.sin_tab[static_cast<int64_t>(p) * half + j];
    }
    __syncthreads();
  }
  if (head0 - sub >= heads) return;

  // angles of the lane's 8 pairs: (x[i], x[8 + i]) of halves, (x[2 i], x[2 i + 1]) of adjacent pairs; without a
  // rotation by 0.  (Odd halves: of each of the 16 elements, with the sine's sign.)
  constexpr int NA = kRope == kOddHalves ? 16 : 8;
  float c[NA], s[NA];
#pragma unroll
  for (int i = 0; i < NA; ++i) {
    c[i] = 1.f;
    s[i] = 0.f;
    if constexpr (kRope == kPairs) {
      if (l * 8 + i < half) {
        c[i] = angle[0][l * 8 + i];
        s[i] = angle[1][l * 8 + i];
      }
    } else if constexpr (kRope == kOddHalves) {
      const int e = l * 16 + i;
      if (e < a.rot_dim) {
        c[i] = angle[0][e < half ? e : e - half];
        s[i] = e < half ? -angle[1][e] : angle[1][e - half];
      }
    }
  }
  if constexpr (kRope == kHalves) {
    if (rotates) {
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const float4 u = *reinterpret_cast<const float4*>(&angle[0][l * 8 + i]), v = *reinterpret_cast<const float4*>(&angle[1][l * 8 + i]);
        c[i] = u.x, c[i + 1] = u.y, c[i + 2] = u.z, c[i + 3] = u.w;
        s[i] = v.x, s[i + 1] = v.y, s[i + 2] = v.z, s[i + 3] = v.w;
      }
    }
  }
  const int64_t slot = a.slot_mapping[tok];
  const bool store = slot >= 0 && slot < a.num_slots;
  float w[16];                      // norm weights of the current kind of head
  int kind = -1;                    // 0 q, 1 k, 2 v
  __nv_bfloat16* q_row = static_cast<__nv_bfloat16*>(a.q_out) + static_cast<int64_t>(tok) * a.q_out_stride;

  for (int it = 0; it < passes; ++it) {
    const int head = head0 + it * HW;
    if (head - sub >= heads) break;
    const bool live = head < heads;
    const bool is_q = head < a.hq, is_k = !is_q && head < a.hq + a.hkv;
    float x[16];
    unpack8(raw[0], *reinterpret_cast<float(*)[8]>(x));
    unpack8(raw[1], *reinterpret_cast<float(*)[8]>(x + 8));
    if (it + 1 < passes && head + HW < heads) fetch(head + HW);
    const __nv_bfloat16* wp = static_cast<const __nv_bfloat16*>(is_q ? a.q_norm : (is_k ? a.k_norm : nullptr));
    if (kind != (is_q ? 0 : (is_k ? 1 : 2))) {
      kind = is_q ? 0 : (is_k ? 1 : 2);
      if (wp != nullptr) {
        unpack8(*reinterpret_cast<const uint4*>(wp + e0), *reinterpret_cast<float(*)[8]>(w));
        unpack8(*reinterpret_cast<const uint4*>(wp + e1), *reinterpret_cast<float(*)[8]>(w + 8));
      }
    }
    if (__any_sync(0xffffffffu, wp != nullptr)) {
      uint64_t sq[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 16; i += 2) sq[(i >> 1) & 1] = fma2(f32x2(x[i], x[i + 1]), f32x2(x[i], x[i + 1]), sq[(i >> 1) & 1]);
      const float2 two = unpack(add2(sq[0], sq[1]));
      float ss = two.x + two.y;
#pragma unroll
      for (int d = 1; d < L; d <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
      if (wp != nullptr) {
        const float r = rsqrtf(ss * (1.f / D) + a.eps);
        const uint64_t rr = f32x2(r, r);
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float2 y = unpack(mul2(mul2(f32x2(x[i], x[i + 1]), rr), f32x2(w[i], w[i + 1])));
          x[i] = y.x;
          x[i + 1] = y.y;
        }
      }
    }
    if constexpr (kRope == kOddHalves) {
      float* row = rows[warp][sub];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 16; ++i) row[l * 16 + i] = x[i];
      __syncwarp();
      if (is_q || is_k) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int e = l * 16 + i;
          if (e < a.rot_dim) x[i] = x[i] * c[i] + row[e < half ? e + half : e - half] * s[i];
        }
      }
    } else if constexpr (kRope == kHalves) {
      if (rotates && (is_q || is_k)) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const uint64_t u = f32x2(x[i], x[i + 1]), v = f32x2(x[8 + i], x[9 + i]);
          const uint64_t cc = f32x2(c[i], c[i + 1]), sc = f32x2(s[i], s[i + 1]), ns = f32x2(-s[i], -s[i + 1]);
          const float2 y = unpack(fma2(v, ns, mul2(u, cc))), z = unpack(fma2(u, sc, mul2(v, cc)));
          x[i] = y.x, x[i + 1] = y.y, x[8 + i] = z.x, x[9 + i] = z.y;
        }
      }
    } else if constexpr (kRope == kPairs) {
      if (rotates && (is_q || is_k)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (l * 16 + 2 * i >= a.rot_dim) break;
          const float u = x[2 * i], v = x[2 * i + 1];
          x[2 * i] = u * c[i] - v * s[i];
          x[2 * i + 1] = v * c[i] + u * s[i];
        }
      }
    }
    if (is_q) {
      *reinterpret_cast<uint4*>(q_row + head * D + e0) = pack8(*reinterpret_cast<float(*)[8]>(x));
      *reinterpret_cast<uint4*>(q_row + head * D + e1) = pack8(*reinterpret_cast<float(*)[8]>(x + 8));
    }
    if (__all_sync(0xffffffffu, is_q)) continue;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
    for (int d = 1; d < L; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (!live || is_q || !store) continue;
    const int h = head - a.hq - (is_k ? 0 : a.hkv);
    const int e = exponent_of(top);
    const float inv = e == kExpBad ? 0.f : pow2_of(-e);
    const int64_t row = ((slot >> 6) * a.hkv + h) * kPage + (slot & 63);
    uint32_t out[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // NaN * 0 stays NaN: a row that is not finite stores zeros by selection
      const float2 v = e == kExpBad ? make_float2(0.f, 0.f) : make_float2(x[2 * i] * inv, x[2 * i + 1] * inv);
      const uint32_t two = __nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3);
      out[i >> 1] = (i & 1) ? (out[i >> 1] | (two << 16)) : two;
    }
    uint8_t* codes = static_cast<uint8_t*>(is_k ? a.k : a.v) + row * D;
    *reinterpret_cast<uint2*>(codes + e0) = make_uint2(out[0], out[1]);
    *reinterpret_cast<uint2*>(codes + e1) = make_uint2(out[2], out[3]);
    if (l == 0) static_cast<int8_t*>(is_k ? a.k_exp : a.v_exp)[row] = static_cast<int8_t>(e);
  }
}

// One thread: 8 codes of one row of K and of V, so that a warp's 16-byte stores lie side by side.
template <int D>
__global__ void __launch_bounds__(256) kv8_read_kernel(const Kv8ReadArgs a) {
  constexpr int L = D / 8;
  grid_dep_wait();
  grid_dep_launch();
  const uint32_t r = blockIdx.x * (256 / L) + threadIdx.x / L, l = threadIdx.x % L;
  if (r >= static_cast<uint32_t>(a.count) * a.hkv) return;   // below 2^31
  const uint32_t n = r / static_cast<uint32_t>(a.hkv), h = r - n * a.hkv;
  const int64_t slot = a.slots[n];
  uint2 raw[2] = {make_uint2(0u, 0u), make_uint2(0u, 0u)};
  float f[2] = {0.f, 0.f};
  if (slot >= 0 && slot < a.num_slots) {
    const int64_t row = ((slot >> 6) * a.hkv + h) * kPage + (slot & 63);
    raw[0] = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.k) + row * D + l * 8);
    raw[1] = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.v) + row * D + l * 8);
    f[0] = pow2_of(static_cast<const int8_t*>(a.k_exp)[row]);
    f[1] = pow2_of(static_cast<const int8_t*>(a.v_exp)[row]);
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const float4 t = e4m3x4_to_f32(raw[w].x), u = e4m3x4_to_f32(raw[w].y);
    const float v[8] = {t.x * f[w], t.y * f[w], t.z * f[w], t.w * f[w], u.x * f[w], u.y * f[w], u.z * f[w], u.w * f[w]};
    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(w == 0 ? a.k_out : a.v_out) + static_cast<int64_t>(r) * D + l * 8) = pack8(v);
  }
}

}  // namespace

namespace {

template <int D>
cudaError_t launch_store(const Kv8StoreArgs& a, cudaStream_t stream) {
  const int heads = a.hq + 2 * a.hkv;
  const int groups = (heads + 512 / D - 1) / (512 / D);   // warp passes of a token
  // One pass a warp while that leaves the launch within a few waves of the GPU (latency); beyond, two warps
  // walk a whole token, so little is looked up and set up per token (8191 tokens of 40 heads, with the read of
  // the rows: one warp 46 us, two 45, three 48, five 63).
  const int passes = static_cast<int64_t>(a.tokens) * groups <= 16384 ? 1 : (groups + 1) / 2;
  const int warps = std::min(a.rot_dim % 16 == 0 || a.neox == 0 ? 4 : 8, (groups + passes - 1) / passes);
  const dim3 grid(a.tokens, (groups + warps * passes - 1) / (warps * passes));
  if (a.rot_dim == 0)
    return launch_dependent(kv8_store_kernel<D, kNone>, grid, 32 * warps, 0, stream, a, passes);
  if (a.neox == 0)
    return launch_dependent(kv8_store_kernel<D, kPairs>, grid, 32 * warps, 0, stream, a, passes);
  if (a.rot_dim % 16 == 0)
    return launch_dependent(kv8_store_kernel<D, kHalves>, grid, 32 * warps, 0, stream, a, passes);
  return launch_dependent(kv8_store_kernel<D, kOddHalves>, grid, 32 * warps, 0, stream, a, passes);
}

}  // namespace

cudaError_t kv8_store(const Kv8StoreArgs& a, cudaStream_t stream) {
  if (a.tokens == 0) return cudaSuccess;
  if (a.head_dim == 128) return launch_store<128>(a, stream);
  if (a.head_dim == 64) return launch_store<64>(a, stream);
  return cudaErrorInvalidValue;
}

cudaError_t kv8_read(const Kv8ReadArgs& a, cudaStream_t stream) {
  if (a.count == 0) return cudaSuccess;
  const int64_t rows = static_cast<int64_t>(a.count) * a.hkv, per = 2048 / a.head_dim;
  if (rows > 0x7fffffff) return cudaErrorInvalidValue;
  const int64_t blocks = (rows + per - 1) / per;
  if (a.head_dim == 128)
    return launch_dependent(kv8_read_kernel<128>, dim3(static_cast<unsigned>(blocks)), 256, 0, stream, a);
  if (a.head_dim == 64)
    return launch_dependent(kv8_read_kernel<64>, dim3(static_cast<unsigned>(blocks)), 256, 0, stream, a);
  return cudaErrorInvalidValue;
}

}  // namespace omni
