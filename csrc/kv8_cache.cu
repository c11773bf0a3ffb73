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

// A head row is D / 8 lanes of 8 elements (16-byte loads), so a warp takes 32 / (D / 8) heads of one
// token at a time, `passes` such groups one after another (the next group's row is read ahead).  The
// grid's first dimension is the token: its angles are looked up once per block, one pair per thread.
enum Rope : int {
  kNone,        // no rotation
  kPairs,       // adjacent pairs
  kHalves,      // halves, rot / 2 a multiple of 8: the other element lies in another lane at the same place
  kOddHalves,   // halves of any size: through shared memory
};
template <int D, int kRope>
__global__ void __launch_bounds__(128, 8) kv8_store_kernel(const Kv8StoreArgs a, int passes) {
  grid_dep_launch();
  constexpr int L = D / 8;          // lanes per head
  constexpr int HW = 32 / L;        // heads per warp and pass
  __shared__ float rows[kRope == kOddHalves ? 4 : 1][HW][D];   // partner exchange
  __shared__ __align__(16) float angle[2][D / 2];  // cos, sin of the token's pairs
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane / L, l = lane - sub * L;
  const int heads = a.hq + 2 * a.hkv;
  const int tok = blockIdx.x;
  const int head0 = (blockIdx.y * 4 + warp) * HW * passes + sub;
  const int half = a.rot_dim >> 1;
  grid_dep_wait();
  const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(a.qkv) + static_cast<int64_t>(tok) * a.qkv_stride + l * 8;
  uint4 raw = head0 < heads ? *reinterpret_cast<const uint4*>(src + head0 * D) : make_uint4(0u, 0u, 0u, 0u);
  if (kRope != kNone && static_cast<int>(threadIdx.x) < half) {
    const int j = threadIdx.x;
    const int p = max(0, min(a.positions[static_cast<int64_t>(rope_axis(j, a)) * a.tokens + tok], a.max_pos - 1));
    angle[0][j] = a.cos_tab[static_cast<int64_t>(p) * half + j];
    angle[1][j] = a.sin_tab[static_cast<int64_t>(p) * half + j];
  }
  __syncthreads();
  if (head0 - sub >= heads) return;

  // of this lane's 8 elements; s carries the sign: x1 cos - x2 sin, x2 cos + x1 sin
  float c[8], s[8];
  if (kRope == kHalves) {
    const int j = l * 8 < half ? l * 8 : min(l * 8, a.rot_dim - 8) - half;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const float4 cv = *reinterpret_cast<const float4*>(&angle[0][j + i]), sv = *reinterpret_cast<const float4*>(&angle[1][j + i]);
      c[i] = cv.x, c[i + 1] = cv.y, c[i + 2] = cv.z, c[i + 3] = cv.w;
      s[i] = sv.x, s[i + 1] = sv.y, s[i + 2] = sv.z, s[i + 3] = sv.w;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = l * 8 < half ? -s[i] : s[i];
  } else if (kRope != kNone) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = l * 8 + i;
      c[i] = 1.f;
      s[i] = 0.f;
      if (e < a.rot_dim) {
        const int j = kRope == kPairs ? e >> 1 : (e < half ? e : e - half);
        c[i] = angle[0][j];
        s[i] = (kRope == kPairs ? (i & 1) == 0 : e < half) ? -angle[1][j] : angle[1][j];
      }
    }
  }
  const int64_t slot = a.slot_mapping[tok];
  const bool store = slot >= 0 && slot < a.num_slots;
  float w[8];                       // norm weights of the current kind of head
  int kind = -1;                    // 0 q, 1 k, 2 v
  __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.q_out) + static_cast<int64_t>(tok) * a.q_out_stride + l * 8;
  const int step = half >> 3;       // lanes between the two elements of a pair
  const int from = sub * L + (l < step ? l + step : (l < 2 * step ? l - step : l));
  const bool rotates = l * 8 < a.rot_dim;

  for (int it = 0; it < passes; ++it) {
    const int head = head0 + it * HW;
    if (head - sub >= heads) break;
    const bool live = head < heads;
    const bool is_q = head < a.hq, is_k = !is_q && head < a.hq + a.hkv;
    float x[8];
    unpack8(raw, x);
    if (it + 1 < passes && head + HW < heads) raw = *reinterpret_cast<const uint4*>(src + (head + HW) * D);
    const void* wp = is_q ? a.q_norm : (is_k ? a.k_norm : nullptr);
    if (kind != (is_q ? 0 : (is_k ? 1 : 2))) {
      kind = is_q ? 0 : (is_k ? 1 : 2);
      if (wp != nullptr) unpack8(*reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(wp) + l * 8), w);
    }
    if (__any_sync(0xffffffffu, wp != nullptr)) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
      for (int d = 1; d < L; d <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
      if (wp != nullptr) {
        const float r = rsqrtf(ss * (1.f / D) + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i];
      }
    }
    if (kRope != kNone && __any_sync(0xffffffffu, is_q || is_k)) {
      float y[8];   // the other element of each pair
      if constexpr (kRope == kPairs) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[i ^ 1];
      } else if constexpr (kRope == kHalves) {
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
      if (rotates && (is_q || is_k)) {
        if (kRope == kHalves || (a.rot_dim & 7) == 0) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = x[i] * c[i] + y[i] * s[i];
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = l * 8 + i < a.rot_dim ? x[i] * c[i] + y[i] * s[i] : x[i];
        }
      }
    }
    if (is_q) *reinterpret_cast<uint4*>(dst + head * D) = pack8(x);
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
  grid_dep_launch();
  grid_dep_wait();
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
      for (int j = 0; j < 2; ++j) {
        const float4 t = e4m3x4_to_f32(w[2 * k + j]);
        v[4 * j] = t.x * f;
        v[4 * j + 1] = t.y * f;
        v[4 * j + 2] = t.z * f;
        v[4 * j + 3] = t.w * f;
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

template <int D>
cudaError_t launch_store(const Kv8StoreArgs& a, cudaStream_t stream) {
  const int heads = a.hq + 2 * a.hkv;
  const int groups = (heads + 256 / D - 1) / (256 / D);   // warp passes of a token
  // One pass a warp while that leaves the launch within a few waves of the GPU (latency); beyond,
  // a block walks a whole token, so its angles are looked up once and not once per four passes.
  const int64_t blocks = static_cast<int64_t>(a.tokens) * ((groups + 3) / 4);
  const int passes = blocks <= 4096 ? 1 : (groups + 3) / 4;
  const dim3 grid(a.tokens, (groups + 4 * passes - 1) / (4 * passes));
  if (a.rot_dim == 0)
    return launch_dependent(kv8_store_kernel<D, kNone>, grid, 128, 0, stream, a, passes);
  if (a.neox == 0)
    return launch_dependent(kv8_store_kernel<D, kPairs>, grid, 128, 0, stream, a, passes);
  if (a.rot_dim % 16 == 0)
    return launch_dependent(kv8_store_kernel<D, kHalves>, grid, 128, 0, stream, a, passes);
  return launch_dependent(kv8_store_kernel<D, kOddHalves>, grid, 128, 0, stream, a, passes);
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
    return launch_dependent(kv8_read_kernel<128>, dim3(static_cast<unsigned>(blocks)), 256, 0, stream, a);
  if (a.head_dim == 64)
    return launch_dependent(kv8_read_kernel<64>, dim3(static_cast<unsigned>(blocks)), 256, 0, stream, a);
  return cudaErrorInvalidValue;
}

}  // namespace omni
