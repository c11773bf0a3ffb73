// Attention over the 8-bit paged KV cache (form: kv8.cuh): one warp per (query token, query head),
// one pass over its visible keys with the running maximum and sum of the softmax.
//
//   o = sum_j p_j v_j,   p = softmax_j(q . k_j * scale) over the visible keys j
//
// A query at position i of its request sees j <= i; with a window W > 0 only j > i - W and the
// request's first `sinks` tokens.  A query that sees no key gives zeros.
#include "kv8.cuh"
#include "omni_kernels.h"

namespace omni {
namespace {

using namespace kv8;

constexpr float kLog2e = 1.4426950408889634f;

template <int D>
__global__ void __launch_bounds__(128) kv8_attention_kernel(const Kv8AttnArgs a) {
  constexpr int PER = D / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 4 + warp;
  const int tok = static_cast<int>(id / a.hq);
  const int hq = static_cast<int>(id - static_cast<int64_t>(tok) * a.hq);
  if (tok >= a.q_rows) return;
  const int h = hq / (a.hq / a.hkv);
  // request of the token: the last b with cu_q[b] <= tok
  int b = tok, pos_in = 0, q_len = 1;
  if (a.cu_q != nullptr) {
    int lo = 0, hi = a.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.cu_q[mid] <= tok) lo = mid; else hi = mid;
    }
    b = lo;
    pos_in = tok - a.cu_q[b];
    q_len = a.cu_q[b + 1] - a.cu_q[b];
  }
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + static_cast<int64_t>(tok) * a.out_stride + hq * D + lane * PER;
  float o[PER], q[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) o[i] = 0.f;
  float m = -INFINITY, sum = 0.f;
  if (pos_in < q_len) {
    const int kv_len = min(a.kv_lens[b], a.bt_pages * kPage);
    const int pos = kv_len - q_len + pos_in;
    const __nv_bfloat16* qr = static_cast<const __nv_bfloat16*>(a.q) + static_cast<int64_t>(tok) * a.q_stride + hq * D + lane * PER;
#pragma unroll
    for (int i = 0; i < PER; ++i) q[i] = __bfloat162float(qr[i]) * a.scale * kLog2e;
    const int first = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    const int sinks = min(a.sinks, first);
    const int total = max(0, pos + 1 - first) + sinks;
    for (int n = 0; n < total; ++n) {
      const int j = n < sinks ? n : first + n - sinks;
      const int page = checked_page(a.block_table[static_cast<int64_t>(b) * a.bt_stride + (j >> 6)], a.num_pages);
      const int64_t row = (static_cast<int64_t>(page) * a.hkv + h) * kPage + (j & 63);
      const uint8_t* kr = static_cast<const uint8_t*>(a.k) + row * D + lane * PER;
      const uint8_t* vr = static_cast<const uint8_t*>(a.v) + row * D + lane * PER;
      float dot = 0.f, v[PER];
#pragma unroll
      for (int i = 0; i < PER; i += 2) {
        const float2 kk = e4m3x2_to_f32(*reinterpret_cast<const uint16_t*>(kr + i));
        const float2 vv = e4m3x2_to_f32(*reinterpret_cast<const uint16_t*>(vr + i));
        dot += q[i] * kk.x + q[i + 1] * kk.y;
        v[i] = vv.x;
        v[i + 1] = vv.y;
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
      const float s = dot * pow2_of(static_cast<const int8_t*>(a.k_exp)[row]);
      const float ve = pow2_of(static_cast<const int8_t*>(a.v_exp)[row]);
      const float mn = fmaxf(m, s);
      const float old = mn == -INFINITY ? 1.f : exp2f(m - mn);
      const float p = mn == -INFINITY && s == -INFINITY ? 0.f : exp2f(s - mn);
      m = mn;
      sum = sum * old + p;
#pragma unroll
      for (int i = 0; i < PER; ++i) o[i] = o[i] * old + p * (v[i] * ve);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int i = 0; i < PER; ++i) out[i] = __float2bfloat16(o[i] * inv);
}

}  // namespace

cudaError_t kv8_attention(const Kv8AttnArgs& a, cudaStream_t stream) {
  if (a.q_rows == 0) return cudaSuccess;
  const int64_t blocks = (static_cast<int64_t>(a.q_rows) * a.hq + 3) / 4;
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  if (a.head_dim == 128)
    kv8_attention_kernel<128><<<static_cast<unsigned>(blocks), 128, 0, stream>>>(a);
  else if (a.head_dim == 64)
    kv8_attention_kernel<64><<<static_cast<unsigned>(blocks), 128, 0, stream>>>(a);
  else
    return cudaErrorInvalidValue;
  return cudaGetLastError();
}

}  // namespace omni
