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
// Both are bound by bytes.
//
// Reference counterpart: the fp8 KV-cache option of SGLang's token-to-KV pool behind
// sglang_omni/engines/ar/sglang_backend/server_args_builder.py:10-35 (kv_cache_dtype there).
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

// A head row is D / 8 lanes of 8 elements (16-byte loads), so a warp takes 32 / (D / 8) heads of one
// token at a time, `passes` such groups one after another (the next group's row is read ahead).  The
// grid's first dimension is the token: its positions, cos and sin are read once per warp.
// kPairs: adjacent-pair rotation; kPlain: the 8 angles of a lane lie side by side in the table (one
// position, halves a multiple of 8), so they are read as vectors.
template <int D, bool kPairs, bool kPlain>
__global__ void __launch_bounds__(128) kv8_store_kernel(const Kv8StoreArgs a, int passes) {
  grid_dep_launch();
  constexpr int L = D / 8;          // lanes per head
  constexpr int HW = 32 / L;        // heads per warp and pass
  __shared__ float rows[kPairs || kPlain ? 1 : 4][HW][D];   // partner exchange of odd halves
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane / L, l = lane - sub * L;
  const int heads = a.hq + 2 * a.hkv;
  const int tok = blockIdx.x;
  const int head0 = (blockIdx.y * 4 + warp) * HW * passes + sub;
  const int half = a.rot_dim >> 1;
  if (head0 - sub >= heads) return;
  const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(a.qkv) + static_cast<int64_t>(tok) * a.qkv_stride + l * 8;
  uint4 raw = head0 < heads ? *reinterpret_cast<const uint4*>(src + head0 * D) : make_uint4(0u, 0u, 0u, 0u);

  // cos / sin of the 8 elements of this lane; s carries the sign: x1 cos - x2 sin, x2 cos + x1 sin
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    c[i] = 1.f;
    s[i] = 0.f;
  }
  if (l * 8 < a.rot_dim) {
    if constexpr (kPlain) {
      const int64_t p = max(0, min(a.positions[tok], a.max_pos - 1));
      constexpr int n = kPairs ? 4 : 8;
      const int j = kPairs ? l * 4 : (l * 8 < half ? l * 8 : l * 8 - half);
      const float* ct = a.cos_tab + p * half + j;
      const float* st = a.sin_tab + p * half + j;
#pragma unroll
      for (int i = 0; i < n; i += 4) {
        const float4 cv = *reinterpret_cast<const float4*>(ct + i), sv = *reinterpret_cast<const float4*>(st + i);
        const float cc[4] = {cv.x, cv.y, cv.z, cv.w}, sc[4] = {sv.x, sv.y, sv.z, sv.w};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if constexpr (kPairs) {
            c[2 * u] = c[2 * u + 1] = cc[u];
            s[2 * u] = -sc[u];
            s[2 * u + 1] = sc[u];
          } else {
            c[i + u] = cc[u];
            s[i + u] = l * 8 < half ? -sc[u] : sc[u];
          }
        }
      }
    } else {
      int64_t at[3];
#pragma unroll
      for (int u = 0; u < 3; ++u) {
        const int p = u < a.pos_rows ? a.positions[static_cast<int64_t>(u) * a.tokens + tok] : 0;
        at[u] = static_cast<int64_t>(max(0, min(p, a.max_pos - 1))) * half;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = l * 8 + i;
        if (e >= a.rot_dim) continue;
        const int j = kPairs ? e >> 1 : (e < half ? e : e - half);
        const int ax = rope_axis(j, a);
        const int64_t row = ax == 0 ? at[0] : (ax == 1 ? at[1] : at[2]);
        c[i] = a.cos_tab[row + j];
        s[i] = a.sin_tab[row + j];
        if (kPairs ? (i & 1) == 0 : e < half) s[i] = -s[i];
      }
    }
  }
  const int64_t slot = a.slot_mapping[tok];
  const bool store = slot >= 0 && slot < a.num_slots;
  float wq[8], wk[8];
  if (a.q_norm != nullptr) unpack8(*reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.q_norm) + l * 8), wq);
  if (a.k_norm != nullptr) unpack8(*reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.k_norm) + l * 8), wk);

  for (int it = 0; it < passes; ++it) {
    const int head = head0 + it * HW;
    if (head - sub >= heads) break;
    const bool live = head < heads;
    const bool is_q = head < a.hq, is_k = !is_q && head < a.hq + a.hkv;
    float x[8];
    unpack8(raw, x);
    if (it + 1 < passes && head + HW < heads) raw = *reinterpret_cast<const uint4*>(src + (head + HW) * D);
    const bool norm = is_q ? a.q_norm != nullptr : (is_k && a.k_norm != nullptr);
    if (__any_sync(0xffffffffu, norm)) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
      for (int d = 1; d < L; d <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
      if (norm) {
        const float r = rsqrtf(ss / D + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * r * (is_q ? wq[i] : wk[i]);
      }
    }
    if (a.rot_dim > 0 && __any_sync(0xffffffffu, is_q || is_k)) {
      float y[8];   // the other element of each pair
      if constexpr (kPairs) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[i ^ 1];
      } else if (kPlain || (half & 7) == 0) {
        const int step = half >> 3;
        const int from = sub * L + (l < step ? l + step : (l < 2 * step ? l - step : l));
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = __shfl_sync(0xffffffffu, x[i], from);
      } else {
        float* row = rows[warp][sub];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) row[l * 8 + i] = x[i];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int e = l * 8 + i;
          y[i] = row[e < half ? e + half : (e < a.rot_dim ? e - half : e)];
        }
      }
      if (is_q || is_k) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = l * 8 + i < a.rot_dim ? x[i] * c[i] + y[i] * s[i] : x[i];
      }
    }
    if (is_q)
      *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.q_out) + static_cast<int64_t>(tok) * a.q_out_stride +
                                head * D + l * 8) = pack8(x);
    if (__all_sync(0xffffffffu, is_q)) continue;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
    for (int d = 1; d < L; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (!live || is_q || !store) continue;
    const int h = head - a.hq - (is_k ? 0 : a.hkv);
    const int e = exponent_of(top);
    const float inv = e == kExpBad ? 0.f : pow2_of(-e);
    const int64_t row = ((slot >> 6) * a.hkv + h) * kPage + (slot & 63);
    uint32_t out[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // NaN * 0 stays NaN: a row that is not finite stores zeros by selection
      const float2 v = e == kExpBad ? make_float2(0.f, 0.f) : make_float2(x[2 * i] * inv, x[2 * i + 1] * inv);
      const uint32_t two = __nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3);
      out[i >> 1] = (i & 1) ? (out[i >> 1] | (two << 16)) : two;
    }
    uint8_t* codes = static_cast<uint8_t*>(is_k ? a.k : a.v);
    *reinterpret_cast<uint2*>(codes + row * D + l * 8) = make_uint2(out[0], out[1]);
    if (l == 0) static_cast<int8_t*>(is_k ? a.k_exp : a.v_exp)[row] = static_cast<int8_t>(e);
  }
}

// One thread: 16 codes of one row -> 32 bytes of bf16.
template <int D>
__global__ void __launch_bounds__(256) kv8_read_kernel(const Kv8ReadArgs a) {
  constexpr int L = D / 16;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t rows = static_cast<int64_t>(a.count) * a.hkv;
  const int64_t r = i / L;
  if (r >= 2 * rows) return;
  const int l = static_cast<int>(i - r * L);
  const bool is_v = r >= rows;
  const int64_t rr = is_v ? r - rows : r;
  const int64_t n = rr / a.hkv;
  const int h = static_cast<int>(rr - n * a.hkv);
  const int64_t slot = a.slots[n];
  uint4 o[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
  if (slot >= 0 && slot < a.num_slots) {
    const int64_t row = ((slot >> 6) * a.hkv + h) * kPage + (slot & 63);
    const uint4 raw = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(is_v ? a.v : a.k) + row * D + l * 16);
    const float f = pow2_of(static_cast<const int8_t*>(is_v ? a.v_exp : a.k_exp)[row]);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 t = e4m3x2_to_f32((w[2 * k + (j >> 1)] >> (16 * (j & 1))) & 0xffffu);
        v[2 * j] = t.x * f;
        v[2 * j + 1] = t.y * f;
      }
      o[k] = pack8(v);
    }
  }
  uint4* dst = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(is_v ? a.v_out : a.k_out) + rr * D + l * 16);
  dst[0] = o[0];
  dst[1] = o[1];
}

}  // namespace

namespace {

template <int D, bool kPairs, bool kPlain>
cudaError_t launch_store(const Kv8StoreArgs& a, cudaStream_t stream) {
  const int heads = a.hq + 2 * a.hkv;
  const int groups = (heads + 256 / D - 1) / (256 / D);   // warp passes of a token
  // One pass a warp while that leaves the launch within a few waves of the GPU (latency); beyond,
  // four warps walk a whole token, so its positions and angles are read four times, not `groups` times.
  const int64_t blocks = static_cast<int64_t>(a.tokens) * ((groups + 3) / 4);
  const int passes = blocks <= 4096 ? 1 : (groups + 3) / 4;
  const dim3 grid(a.tokens, (groups + 4 * passes - 1) / (4 * passes));
  kv8_store_kernel<D, kPairs, kPlain><<<grid, 128, 0, stream>>>(a, passes);
  return cudaGetLastError();
}

template <int D>
cudaError_t launch_store(const Kv8StoreArgs& a, cudaStream_t stream) {
  const int half = a.rot_dim / 2;
  const bool pairs = a.neox == 0 && a.rot_dim > 0;
  const bool axes = a.pos_rows == 3 && (a.section[1] > 0 || a.section[2] > 0);
  const bool aligned = ((reinterpret_cast<uintptr_t>(a.cos_tab) | reinterpret_cast<uintptr_t>(a.sin_tab)) & 15) == 0;
  const bool plain = !axes && aligned && half % 8 == 0;
  if (pairs) return plain ? launch_store<D, true, true>(a, stream) : launch_store<D, true, false>(a, stream);
  return plain ? launch_store<D, false, true>(a, stream) : launch_store<D, false, false>(a, stream);
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
  const int64_t threads = 2 * static_cast<int64_t>(a.count) * a.hkv * (a.head_dim / 16);
  const int64_t blocks = (threads + 255) / 256;
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  if (a.head_dim == 128)
    kv8_read_kernel<128><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a);
  else if (a.head_dim == 64)
    kv8_read_kernel<64><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a);
  else
    return cudaErrorInvalidValue;
  return cudaGetLastError();
}

}  // namespace omni
