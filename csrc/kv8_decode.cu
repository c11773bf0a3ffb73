// Decode attention over the 8-bit paged KV cache (form: kv8.cuh): one query token per request, or a few
// tokens of chunks, each as a request of its own over the keys up to it.
//
//   o = sum_j p_j v_j,   p = softmax_j(q . k_j * scale) over the visible keys j
//
// Bound by the cache's bytes (2 (D + 1) per key and KV head), so the design is a stream of 64-key
// tiles (one page of one KV head: contiguous) through a deep shared-memory ring, and cheap work on
// each tile:
//
// * Work split.  The visible tiles of all (request, KV head) pairs form one sequence; CTA c takes
//   the tiles [c * per, (c + 1) * per) of it, per = ceil(tiles / CTAs), found on the device from
//   kv_lens.  Every CTA streams the same number of tiles whatever the lengths are, and the launch
//   does not depend on them (CUDA graphs).  A pair that lies in several CTAs leaves partial sums,
//   which a second, dependent launch joins in a fixed order.  Many short pairs stay whole, one
//   to a CTA.
// * A producer warp issues TMA loads (K and V tile swizzled, their exponents as bulk copies);
//   two pairs of consumer warps take the tiles in turn, each warp 32 of the 64 keys, and keep their own
//   running maximum, sum and output until the pair ends, so tiles need no barrier among the warps.
// * Arithmetic on 16 keys: the codes go to fp16 (exact), S^T = K Q^T and O^T += V^T P by
//   mma.m16n8k16 with the keys / dims as the 16 rows and the query heads of the KV head as the
//   columns, so few heads waste few rows.  The contraction order inside a 16-dim chunk is free, and
//   is chosen so that an ldmatrix register's 4 codes are exactly one lane's operand values.
//   tcgen05 is not used: its 128-row tiles would be filled to 1/16 by 8 heads, and the time is the
//   memory's either way.
// * Scales.  Exponents never touch the codes.  With t_j = log2-score + ev_j (ev: V's exponent),
//   w_j = 2^(t_j - m) is key j's weight on its integer-like codes, held in fp16 for the product;
//   m is the running maximum of t (raised only when exceeded by 8), so what fp16 drops is below
//   2^-31 of the largest contribution.  The softmax sum takes w_j * 2^-ev_j in fp32.
//   q is scaled by a power of two to [2^9, 2^10) before it is rounded to fp16.
//
// Measured: 5 requests of 52,000 - 130,000 keys, 32 / 8 heads of 128: 204 - 210 us = 6.4 - 6.6 TB/s
// (copy: 6.55); 64 slots of about 1150 keys, 32 / 4 heads, out of HBM: 20.7 us = 3.6 TB/s by one CTA a
// pair, 22.6 over all tiles, of which about 8 us are launches, look-ups and joining; 48 windows of 4096 keys, 32 / 8 heads of 64: 45 us = 4.5 TB/s; one
// request of 517 keys: 6.3 us.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "host_util.h"
#include "kv8.cuh"
#include "omni_kernels.h"
#include "sm100.cuh"

namespace omni {
namespace {

using namespace kv8;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWarps = 4;                       // consumer warps
constexpr int kThreads = 32 * (kWarps + 1);
constexpr float kRaise = 8.f;                   // log2 units
constexpr float kHead = 7.f;                    // weights are held times 2^7: below 2^15

template <int D, int NT>
struct Smem {
  // CTAs per SM and ring depth: 64 slots of about 1150 keys, 5 of 52,000 - 130,000 and 48 windows of 4096
  // (head dim 64) took, in microseconds, at (CTAs, stages) (2, 5): 26.3, 212, 62; (3, 3 | 64: 5): 26.3, 208, 56;
  // (3, 3 | 64: 4 CTAs, 5 stages): 26.1, 207, 53.
  static constexpr int kCtas = D == 128 ? (NT == 1 ? 3 : 2) : (NT == 1 ? 4 : 3);
  static constexpr int kStages = D == 128 ? (NT == 1 ? 3 : 4) : 5;
  static constexpr int kTile = kPage * D;       // bytes of a K or V tile
  static constexpr int kStage = 2 * kTile;
  static constexpr int kExp = kStages * kStage;                 // exponents: [stage][2][64]
  static constexpr int kRedStride = D + 4;                      // floats; conflict-free float2 stores
  static constexpr int kRed = kExp + kStages * 2 * kPage;       // [warp][8 NT heads][D + 4]
  static constexpr int kMl = kRed + kWarps * 8 * NT * kRedStride * 4;   // [warp][8 NT][2] (m, l)
  static constexpr int kSum = kMl + kWarps * 8 * NT * 8;              // [8 NT][2]: the CTA's own (m, l)
  static constexpr int kBars = kSum + 8 * NT * 8;
  static constexpr int kBytes = kBars + 16 * kStages + 16 + 1024;
};

struct Params {
  const __nv_bfloat16* q;
  int64_t q_stride;
  const uint8_t* k_exp;
  const uint8_t* v_exp;
  const int* block_table;
  int64_t bt_stride;
  int bt_pages, num_pages;
  const int* kv_lens;
  const int* cu_q;                              // nullptr, or chunks: query row b is a token of one of `requests`
  int requests;
  int batch, hq, hkv, group, head_groups;       // head_groups: column tiles of 8 NT heads per KV head
  float scale;
  int window, sinks;
  __nv_bfloat16* out;
  int64_t out_stride;
  float* part_o;                                // [2 CTAs][8 NT][D]
  float* part_ml;                               // [2 CTAs][8 NT][2]
  int ctas;
  int cluster;                                  // CTAs of a cluster that share a pair
  int* status;
};

// Visible keys of a request and the 64-key tiles that hold them.
struct Span {
  int kv, lo, sinks;      // keys [0, sinks) and [lo, kv)
  int sink_tiles, first, tiles;
  int req;                // row of the block table
  __device__ Span(const Params& p, int b) {
    if (p.cu_q == nullptr) {
      req = b;
      kv = min(p.kv_lens[b], p.bt_pages * kPage);
    } else {              // the last request that starts at or before row b, and the keys up to its token
      int lo_r = 0, hi_r = p.requests;
      while (hi_r - lo_r > 1) {
        const int mid = (lo_r + hi_r) >> 1;
        if (p.cu_q[mid] <= b) lo_r = mid; else hi_r = mid;
      }
      req = lo_r;
      const int after = p.cu_q[req + 1] - 1 - b;           // tokens of the chunk behind this one
      kv = after < 0 ? 0 : min(p.kv_lens[req], p.bt_pages * kPage) - after;
    }
    lo = p.window > 0 ? max(0, kv - p.window) : 0;
    sinks = min(p.sinks, lo);
    first = lo >> 6;
    sink_tiles = min((sinks + 63) >> 6, first);
    tiles = kv > 0 ? sink_tiles + ((kv + 63) >> 6) - first : 0;
  }
  __device__ int tile(int i) const { return i < sink_tiles ? i : first + i - sink_tiles; }
};

// How the tiles are dealt out (whole warp; the same in every warp of both launches).
struct Plan {
  int tiles;              // of one (KV head, head group), over all requests (below 2^31)
  int before;             // of them, in the requests before `stop`
  int64_t per;            // tiles of a CTA
  int64_t pairs;          // with a visible key
  bool whole;             // a pair per CTA instead
  __device__ Plan(const Params& p, int R, int stop) {
    const int lane = threadIdx.x & 31;
    int all = 0, head = 0, live = 0, most = 0;
    for (int b = lane; b < p.batch; b += 32) {
      const int n = Span(p, b).tiles;
      all += n;
      if (b < stop) head += n;
      live += n > 0;
      most = max(most, n);
    }
    tiles = __reduce_add_sync(0xffffffffu, all);
    before = __reduce_add_sync(0xffffffffu, head);
    live = __reduce_add_sync(0xffffffffu, live);
    most = __reduce_max_sync(0xffffffffu, most);
    per = (static_cast<int64_t>(tiles) * R + p.ctas - 1) / p.ctas;
    // Short pairs that occupy a good part of the CTAs are not split: it saves each CTA a second segment and
    // the joining.  Longer ones stream faster from all CTAs.  64 slots of about 270 / 540 / 1150 / 2300 keys,
    // microseconds whole and split: 11.2, 13.4 / 13.7, 14.7 / 19.6, 19.0 / 35.4, 33.0.
    pairs = static_cast<int64_t>(live) * R;
    whole = pairs <= p.ctas && 5 * pairs >= 2 * p.ctas && most <= 12;
  }
};

// Walks a CTA's tiles pair by pair (whole warp; every warp of the CTA walks alike).
struct Walk {
  int b, r;               // request; KV head * head_groups + head group
  int i0, i1, n;          // this segment's tiles [i0, i1) of the pair's n
  int64_t left;
  int per_b;              // pairs per request
  // tiles [i0, i1) of one pair
  __device__ Walk(int b_, int r_, int n_, int i0_, int i1_) : b(b_), r(r_), i0(i0_), i1(i1_), n(n_), left(i1_ - i0_), per_b(0) {}
  // tiles [x, x + count) of all pairs', or pair x whole
  __device__ Walk(const Params& p, const Plan& plan, int64_t x, int64_t count, int R) {
    per_b = R;
    left = count;
    const int lane = threadIdx.x & 31;
    int cum = 0;
    b = 0;
    for (int base = 0; base < p.batch; base += 32) {
      const int mine = base + lane < p.batch ? Span(p, base + lane).tiles : 0;
      const int weight = plan.whole ? (mine > 0 ? 1 : 0) : mine;
      int inc = weight;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += up;
      }
      const unsigned past = __ballot_sync(0xffffffffu, static_cast<int64_t>(cum + inc) * R > x);
      if (past != 0) {
        const int at = __ffs(past) - 1;
        b = base + at;
        n = __shfl_sync(0xffffffffu, mine, at);
        cum += __shfl_sync(0xffffffffu, inc - weight, at);
        break;
      }
      cum += __shfl_sync(0xffffffffu, inc, 31);
    }
    const int64_t rel = x - static_cast<int64_t>(cum) * R;
    if (plan.whole) {
      r = static_cast<int>(rel);
      i0 = 0;
      left = n;
    } else {
      // rel < n R; 32-bit division where that fits
      r = rel < 0x7fffffff ? static_cast<int>(rel) / n : static_cast<int>(rel / n);
      i0 = static_cast<int>(rel - static_cast<int64_t>(r) * n);
    }
    i1 = static_cast<int>(min(static_cast<int64_t>(n), i0 + left));
  }
  __device__ bool next(const Params& p) {
    left -= i1 - i0;
    if (left <= 0) return false;
    if (++r == per_b) {
      r = 0;
      do {
        ++b;
        n = Span(p, b).tiles;
      } while (n == 0);
    }
    i0 = 0;
    i1 = static_cast<int>(min(static_cast<int64_t>(n), left));
    return true;
  }
};

__device__ __forceinline__ void bulk_copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ uint32_t movm_t(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void store_row4(__nv_bfloat16* dst, const float4& x, float f) {
  __nv_bfloat162 y[2] = {__floats2bfloat162_rn(x.x * f, x.y * f), __floats2bfloat162_rn(x.z * f, x.w * f)};
  *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(y);
}
__device__ __forceinline__ float2 ld_dsmem_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

// A row's exponent clamped into the format, from its lowest: min(max(e - kExpMin, 0), kExpMax - kExpMin), one
// instruction.  (64 slots of about 1150 keys: clamped so 20.7 us, in two instructions 20.9, not at all 20.5.)
__device__ __forceinline__ int clamped(int e) { return __viaddmin_s32_relu(e, -kExpMin, kExpMax - kExpMin); }

// Byte offset of 16-byte chunk c of row r in a swizzled tile (128-byte swizzle for 128-byte rows,
// 64-byte swizzle for 64-byte rows).
template <int D>
__device__ __forceinline__ int swz(int r, int c) {
  return D == 128 ? r * 128 + ((c ^ (r & 7)) << 4) : r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
}

// What CTA blockIdx.x walks: a share of all tiles, or (kCluster) of its cluster's pair.
template <bool kCluster>
__device__ __forceinline__ Walk first_walk(const Params& p, int R, bool& any) {
  if constexpr (kCluster) {
    const int pair = blockIdx.x / p.cluster, rank = static_cast<int>(cluster_ctarank());
    const int b = pair / R;
    const int n = Span(p, b).tiles;
    any = true;
    return Walk(b, pair - b * R, n, static_cast<int>(static_cast<int64_t>(n) * rank / p.cluster),
                static_cast<int>(static_cast<int64_t>(n) * (rank + 1) / p.cluster));
  } else {
    const Plan plan(p, R, 0);
    const int64_t x = plan.whole ? static_cast<int64_t>(blockIdx.x) : blockIdx.x * plan.per;
    const int64_t all = static_cast<int64_t>(plan.tiles) * R;
    any = plan.whole ? x < plan.pairs : x < all;
    if (!any) return Walk(0, 0, 0, 0, 0);
    return Walk(p, plan, x, min(plan.per, all - x), R);
  }
}

// kCluster: the CTAs of a cluster take a pair's tiles in equal shares and join their sums through
// distributed shared memory, so that there is no second launch.
template <int D, int NT, bool kCluster>
__global__ void __launch_bounds__(kThreads, Smem<D, NT>::kCtas)
    kv8_decode_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const Params p) {
  using S = Smem<D, NT>;
  constexpr int kStages = S::kStages;
  constexpr int C = D / 16;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  float* red = reinterpret_cast<float*>(smem + S::kRed);
  float2* ml = reinterpret_cast<float2*>(smem + S::kMl);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t* empty = full + kStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + kStages);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kWarps);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  __syncthreads();
  grid_dep_wait();
  grid_dep_launch();   // after the wait: the joining launch may read kv_lens at once, and waits for the sums

  const int R = p.hkv * p.head_groups;
  bool any;
  Walk w = first_walk<kCluster>(p, R, any);
  if (!any) return;

  if (warp == kWarps) {
    // ------------------------------------------------------------ producer
    int64_t t = 0;
    int s = 0;                    // ring stage and phase
    uint32_t ph = 1;
    bool ok = true;
    do {
      const Span sp(p, w.b);
      const int h = w.r / p.head_groups;
      const int* row = p.block_table + static_cast<int64_t>(sp.req) * p.bt_stride;
      for (int i = w.i0; i < w.i1 && ok; i += 32) {
        const int mine = i + lane < w.i1 ? checked_page(row[sp.tile(i + lane)], p.num_pages) : 0;
        const int m = min(32, w.i1 - i);
        for (int j = 0; j < m; ++j, ++t) {
          const int page = __shfl_sync(0xffffffffu, mine, j);
          bool go = true;
          if (lane == 0) {
            if (t >= kStages) go = mbar_wait(&empty[s], ph, abort_flag, p.status);
            if (go) {
              const int r0 = (page * p.hkv + h) * kPage;
              uint8_t* dst = smem + s * S::kStage;
              uint8_t* de = smem + S::kExp + s * 2 * kPage;
              mbar_arrive_expect_tx(&full[s], S::kStage + 2 * kPage);
              tma_load_2d(dst, &tk, &full[s], 0, r0);
              bulk_copy(de, p.k_exp + r0, kPage, &full[s]);
              tma_load_2d(dst + S::kTile, &tv, &full[s], 0, r0);
              bulk_copy(de + kPage, p.v_exp + r0, kPage, &full[s]);
            }
          }
          ok = __shfl_sync(0xffffffffu, go, 0);
          if (!ok) break;
          if (++s == kStages) s = 0, ph ^= 1;
        }
      }
    } while (ok && w.next(p));
    // every issued load has landed before the CTA's shared memory goes away
    if (lane == 0)
      for (int64_t j = t > kStages ? t - kStages : 0; j < t; ++j)
        mbar_wait(&full[j % kStages], static_cast<uint32_t>((j / kStages) & 1), nullptr, p.status);
    __syncwarp();
    if constexpr (!kCluster) return;
  }

  // -------------------------------------------------------------- consumers
  const int g = lane >> 2, t4 = lane & 3;
  const int row0 = (warp & 1) * 32;                         // keys of the tile that this warp takes
  const int lrow = row0 + (lane & 15);                      // ldmatrix row of this lane
  uint32_t t0 = 0;                // tiles before this one
  int s = 0;                      // their ring stage and phase
  uint32_t ph = 0;
  bool ok = true;
  bool more = warp < kWarps;
  while (more) {
    const Span sp(p, w.b);
    const int h = w.r / p.head_groups, hg = w.r - h * p.head_groups;
    const int head0 = h * p.group + hg * 8 * NT;            // first query head of this pair
    const int heads = min(8 * NT, p.group - hg * 8 * NT);
    // Q fragments: lane (g, t4) holds dims 16 c + 4 t4 .. + 3 of head g (and g + 8)
    uint32_t qf[NT][C][2];
    float qs[NT][2];                                        // score factor of heads 2 t4, 2 t4 + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float2 v[C][2];
      uint32_t top = 0;
      const bool live = nt * 8 + g < heads;
      const __nv_bfloat16* qr = p.q + static_cast<int64_t>(w.b) * p.q_stride + static_cast<int64_t>(head0 + (live ? nt * 8 + g : 0)) * D + 4 * t4;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const uint2 two = live ? *reinterpret_cast<const uint2*>(qr + 16 * c) : make_uint2(0u, 0u);
        v[c][0] = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&two.x));
        v[c][1] = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&two.y));
        top = max(max(top, __float_as_uint(v[c][0].x) & 0x7fffffffu), __float_as_uint(v[c][0].y) & 0x7fffffffu);
        top = max(max(top, __float_as_uint(v[c][1].x) & 0x7fffffffu), __float_as_uint(v[c][1].y) & 0x7fffffffu);
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const bool bad = top >= 0x7f800000u;                  // inf / NaN in q: its output is NaN
      const int x = max(static_cast<int>(top >> 23) - 127, -110);
      const float up = bad ? 0.f : __int_as_float((9 - x + 127) << 23);
      const float f = bad ? __int_as_float(0x7fc00000) : __int_as_float((x - 9 + 127) << 23) * p.scale * kLog2e;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i) qf[nt][c][i] = bad ? 0u : pack_h2(v[c][i].x * up, v[c][i].y * up);
      qs[nt][0] = __shfl_sync(0xffffffffu, f, 8 * t4);
      qs[nt][1] = __shfl_sync(0xffffffffu, f, 8 * t4 + 4);
    }
    float o[NT][C][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[nt][c][i] = 0.f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }

    // 32 keys of the tile in ring stage s, two groups of 16.  kEdge: some of its keys are not visible.
    auto work = [&](int stage, int key0, auto edge_tag) {
      constexpr bool kEdge = decltype(edge_tag)::value;
      const uint32_t kt = smem_u32(smem + stage * S::kStage), vt = kt + S::kTile;
      const int8_t* ex = reinterpret_cast<const int8_t*>(smem + S::kExp + stage * 2 * kPage) + row0 + g;
      auto seen = [&](int key) { return key < sp.kv && (key >= sp.lo || key < sp.sinks); };
      // S^T: 2 x 16 keys x 8 NT heads
      float x[2][NT][4];
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) x[q][nt][0] = x[q][nt][1] = x[q][nt][2] = x[q][nt][3] = 0.f;
#pragma unroll
      for (int c = 0; c < C; c += 2)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t r[4];
          ldsm4(kt + swz<D>(lrow + 16 * q, c + (lane >> 4)), r);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            uint32_t a0, a1, a2, a3;
            e4m3x4_to_f16x4(r[2 * u], a0, a2);
            e4m3x4_to_f16x4(r[2 * u + 1], a1, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma(x[q][nt], a0, a1, a2, a3, qf[nt][c + u][0], qf[nt][c + u][1]);
          }
        }
      // log2 weights on the codes: score + V's exponent; NaN where either row is marked as not finite
      float vi[2][2];
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int ke = ex[16 * q + 8 * u], ve = ex[kPage + 16 * q + 8 * u];
          const int kc = clamped(ke), vc = clamped(ve);
          const float kf = __int_as_float(((127 + kExpMin) << 23) + (kc << 23));
          const float vf = min(ke, ve) == kExpBad ? __int_as_float(0x7fc00000) : __int_as_float(0x4b400000 + vc) - (12582912.f - kExpMin);
          vi[q][u] = __int_as_float(((127 - kExpMin) << 23) - (vc << 23));
          const bool in = !kEdge || seen(key0 + row0 + 16 * q + 8 * u + g);
          if (!in) vi[q][u] = 0.f;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int v = 0; v < 2; ++v) {
              x[q][nt][2 * u + v] = fmaf(x[q][nt][2 * u + v], qs[nt][v] * kf, vf);
              if (!in) x[q][nt][2 * u + v] = -INFINITY;
            }
        }
      uint32_t pb[2][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float top[2];
#pragma unroll
        for (int v = 0; v < 2; ++v) top[v] = fmaxf(fmaxf(x[0][nt][v], x[0][nt][2 + v]), fmaxf(x[1][nt][v], x[1][nt][2 + v]));
        if (__any_sync(0xffffffffu, top[0] > m[nt][0] + kRaise || top[1] > m[nt][1] + kRaise)) {
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            float mx = top[v];
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float mn = fmaxf(m[nt][v], mx);
            const float f = m[nt][v] == -INFINITY ? 0.f : ex2(m[nt][v] - mn);
            m[nt][v] = mn;
            l[nt][v] *= f;
#pragma unroll
            for (int c = 0; c < C; ++c) {
              o[nt][c][v] *= f;
              o[nt][c][2 + v] *= f;
            }
          }
        }
        float less[2];
#pragma unroll
        for (int v = 0; v < 2; ++v) less[v] = m[nt][v] == -INFINITY ? 0.f : kHead - m[nt][v];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            x[q][nt][v] = ex2(x[q][nt][v] + less[v]);
            x[q][nt][2 + v] = ex2(x[q][nt][2 + v] + less[v]);
            l[nt][v] = fmaf(x[q][nt][v], vi[q][0], fmaf(x[q][nt][2 + v], vi[q][1], l[nt][v]));
          }
          pb[q][nt][0] = movm_t(pack_h2(x[q][nt][0], x[q][nt][1]));
          pb[q][nt][1] = movm_t(pack_h2(x[q][nt][2], x[q][nt][3]));
        }
      }
      // O^T += V^T P; keys that are not visible may hold anything: their codes become zeros
      uint32_t keep[2][2];
      if constexpr (kEdge) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int key = key0 + row0 + 16 * q + 8 * u + 2 * t4;
            keep[q][u] = (seen(key) ? 0xffffu : 0u) | (seen(key + 1) ? 0xffff0000u : 0u);
          }
      }
#pragma unroll
      for (int c = 0; c < C; c += 2)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t r[4];
          ldsm4_t(vt + swz<D>(lrow + 16 * q, c + (lane >> 4)), r);
          if constexpr (kEdge) {
            r[0] &= keep[q][0], r[2] &= keep[q][0];
            r[1] &= keep[q][1], r[3] &= keep[q][1];
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            // bytes (key 2t: dims 2g, 2g+1; key 2t+1: the same) -> two keys of a dim side by side
            uint32_t a0, a1, a2, a3;
            e4m3x4_to_f16x4(__byte_perm(r[2 * u], 0u, 0x3120), a0, a1);
            e4m3x4_to_f16x4(__byte_perm(r[2 * u + 1], 0u, 0x3120), a2, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma(o[nt][c + u], a0, a1, a2, a3, pb[q][nt][0], pb[q][nt][1]);
          }
        }
    };

    // The two pairs of warps take tiles in turn.  Every warp waits for every tile and releases it, so that
    // no stage is filled again before all have seen it: a phase's parity tells only the last two apart.
    for (int i = w.i0; i < w.i1; ++i, ++t0) {
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&full[s], ph, abort_flag, p.status));
      if (!ok) break;
      if ((t0 & 1) == static_cast<uint32_t>(warp >> 1)) {
        const int key0 = sp.tile(i) * kPage;
        if (key0 + kPage > sp.kv || (key0 < sp.lo && key0 + kPage > sp.sinks))
          work(s, key0, std::true_type{});
        else
          work(s, key0, std::false_type{});
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
      if (++s == kStages) s = 0, ph ^= 1;
    }

    // join the four warps
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        float x = l[nt][v];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        const int head = nt * 8 + 2 * t4 + v;
        if (g == 0) ml[warp * 8 * NT + head] = make_float2(m[nt][v], x);
        float* dst = red + (warp * 8 * NT + head) * S::kRedStride + 2 * g;
#pragma unroll
        for (int c = 0; c < C; ++c) *reinterpret_cast<float2*>(dst + 16 * c) = make_float2(o[nt][c][v], o[nt][c][2 + v]);
      }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    const bool whole = w.i0 == 0 && w.i1 == w.n;
    const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (w.i0 == 0 ? 1 : 0);
    for (int e = threadIdx.x; e < heads * (D / 4); e += 32 * kWarps) {
      const int head = e / (D / 4), d = (e - head * (D / 4)) * 4;
      float mm = -INFINITY;
#pragma unroll
      for (int u = 0; u < kWarps; ++u) mm = fmaxf(mm, ml[u * 8 * NT + head].x);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float ll = 0.f;
#pragma unroll
      for (int u = 0; u < kWarps; ++u) {
        const float2 v = ml[u * 8 * NT + head];
        // a warp without a finite maximum has either nothing (0) or a NaN to pass on
        const float f = v.x == -INFINITY ? 1.f : ex2(v.x - mm);
        const float4 x = *reinterpret_cast<const float4*>(red + (u * 8 * NT + head) * S::kRedStride + d);
        acc.x += x.x * f;
        acc.y += x.y * f;
        acc.z += x.z * f;
        acc.w += x.w * f;
        ll += v.y * f;
      }
      if constexpr (kCluster) {
        *reinterpret_cast<float4*>(red + head * S::kRedStride + d) = acc;   // the place of warp 0's share, read above
        if (d == 0) reinterpret_cast<float2*>(smem + S::kSum)[head] = make_float2(mm, ll);
      } else if (whole) {
        const float inv = ll == 0.f ? 0.f : 1.f / ll;
        store_row4(p.out + static_cast<int64_t>(w.b) * p.out_stride + static_cast<int64_t>(head0 + head) * D + d, acc, inv);
      } else {
        *reinterpret_cast<float4*>(p.part_o + (slot * 8 * NT + head) * D + d) = acc;
        if (d == 0) *reinterpret_cast<float2*>(p.part_ml + (slot * 8 * NT + head) * 2) = make_float2(mm, ll);
      }
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    more = w.next(p);
  }

  if constexpr (kCluster) {
    cluster_sync();
    const int rank = static_cast<int>(cluster_ctarank());
    const int h = w.r / p.head_groups, hg = w.r - h * p.head_groups;
    const int head0 = h * p.group + hg * 8 * NT, items = min(8 * NT, p.group - hg * 8 * NT) * (D / 4);
    for (int e = items * rank / p.cluster + static_cast<int>(threadIdx.x); e < items * (rank + 1) / p.cluster; e += kThreads) {
      const int head = e / (D / 4), d = (e - head * (D / 4)) * 4;
      const uint32_t sum_at = smem_u32(smem + S::kSum) + head * 8, o_at = smem_u32(red + head * S::kRedStride + d);
      float mm = -INFINITY;
      for (int u = 0; u < p.cluster; ++u) mm = fmaxf(mm, ld_dsmem_f2(dsmem_addr(sum_at, u)).x);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float ll = 0.f;
#pragma unroll 4
      for (int u = 0; u < p.cluster; ++u) {
        const float2 v = ld_dsmem_f2(dsmem_addr(sum_at, u));
        const float4 x = ld_dsmem_f4(dsmem_addr(o_at, u));
        const float f = v.x == -INFINITY ? 1.f : ex2(v.x - mm);   // nothing (0), or a NaN to pass on
        acc.x += x.x * f;
        acc.y += x.y * f;
        acc.z += x.z * f;
        acc.w += x.w * f;
        ll += v.y * f;
      }
      store_row4(p.out + static_cast<int64_t>(w.b) * p.out_stride + static_cast<int64_t>(head0 + head) * D + d, acc,
                 ll == 0.f ? 0.f : 1.f / ll);
    }
    cluster_sync();   // no CTA leaves while another reads its shared memory
  }
}

// Joins the partial sums of split pairs in the order of their CTAs, and writes zeros for requests
// without a visible key.  W warps per (request, query head).
template <int D, int NT, int W>
__global__ void __launch_bounds__(128) kv8_decode_join_kernel(const Params p) {
  __shared__ float red[4 * D];
  // One thread's exit without the wait would let what follows on the stream start before the sums are
  // written; the plan is read before it.
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (4 / W) + (threadIdx.x >> 5) / W;
  const bool live = row < static_cast<int64_t>(p.batch) * p.hq;
  const int b = live ? static_cast<int>(row / p.hq) : 0, hq = live ? static_cast<int>(row - static_cast<int64_t>(b) * p.hq) : 0;
  const int h = hq / p.group, in = hq - h * p.group, hg = in / (8 * NT), head = in - hg * 8 * NT;
  const int R = p.hkv * p.head_groups;
  const Plan plan(p, R, b);
  const int n = Span(p, b).tiles;
  int64_t c0 = 0;
  int count = 0;
  if (n > 0) {
    const int64_t x = static_cast<int64_t>(plan.before) * R + static_cast<int64_t>(h * p.head_groups + hg) * n;
    c0 = x / plan.per;
    count = plan.whole ? 1 : static_cast<int>((x + n - 1) / plan.per - c0) + 1;
  }
  grid_dep_wait();
  if (!live || count == 1) return;            // one part: written by its CTA
  auto slot = [&](int i) { return (2 * (c0 + i) + (i == 0 ? 1 : 0)) * 8 * NT + head; };
  join_parts<D, W>(
      count, [&](int i) { return *reinterpret_cast<const float2*>(p.part_ml + slot(i) * 2); },
      [&](int i) { return p.part_o + slot(i) * D; },
      p.out + static_cast<int64_t>(b) * p.out_stride + static_cast<int64_t>(hq) * D, red);
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}

// Codes of one layer as [pages * Hkv * 64, D] bytes, box one page of one head.
bool encode(CUtensorMap* map, const void* base, int d, int64_t rows) {
  auto fn = encode_fn();
  if (fn == nullptr) return false;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(d)};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(d), kPage};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, d == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int NT>
cudaError_t launch(const CUtensorMap& tk, const CUtensorMap& tv, const Params& p, cudaStream_t stream) {
  using S = Smem<D, NT>;
  cudaError_t e;
  if (p.cluster > 0) {
    if ((e = ensure_smem_attr<kv8_decode_kernel<D, NT, true>>(S::kBytes)) != cudaSuccess) return e;
    const int64_t grid = static_cast<int64_t>(p.batch) * p.hkv * p.head_groups * p.cluster;
    return launch_dependent_cluster(kv8_decode_kernel<D, NT, true>, dim3(static_cast<unsigned>(grid)), kThreads, S::kBytes, p.cluster,
                                    stream, tk, tv, p);
  }
  if ((e = ensure_smem_attr<kv8_decode_kernel<D, NT, false>>(S::kBytes)) != cudaSuccess) return e;
  e = launch_dependent(kv8_decode_kernel<D, NT, false>, dim3(p.ctas), kThreads, S::kBytes, stream, tk, tv, p);
  if (e != cudaSuccess) return e;
  // a row's parts: about ctas / pairs; four warps for many parts, one where there are few and many rows
  const int64_t rows = static_cast<int64_t>(p.batch) * p.hq;
  if (static_cast<int64_t>(p.batch) * p.hkv * p.head_groups * 4 <= p.ctas)
    return launch_dependent(kv8_decode_join_kernel<D, NT, 4>, dim3(static_cast<unsigned>(rows)), 128, 0, stream, p);
  return launch_dependent(kv8_decode_join_kernel<D, NT, 1>, dim3(static_cast<unsigned>((rows + 3) / 4)), 128, 0, stream, p);
}

}  // namespace

int kv8_decode_ctas(int sm_count, int group, int head_dim) {
  return sm_count * (head_dim == 128 ? (group > 8 ? Smem<128, 2>::kCtas : Smem<128, 1>::kCtas)
                                     : (group > 8 ? Smem<64, 2>::kCtas : Smem<64, 1>::kCtas));
}

namespace {

int64_t pairs_of(const Kv8AttnArgs& a) {
  const int group = a.hq / a.hkv, heads = group > 8 ? 16 : 8;
  return static_cast<int64_t>(a.q_rows) * a.hkv * ((group + heads - 1) / heads);
}

// Most tiles of a pair.
int64_t most_tiles(const Kv8AttnArgs& a) {
  if (a.window <= 0) return a.bt_pages;
  return std::min<int64_t>(a.bt_pages, (static_cast<int64_t>(a.window) + 63) / 64 + 1 + (static_cast<int64_t>(a.sinks) + 63) / 64);
}

// CTAs per pair so that all pairs run at once, 0 where there are more pairs than CTAs.
int widest_cluster(const Kv8AttnArgs& a) {
  for (int c = 8; c > 0; c >>= 1)
    if (pairs_of(a) * c <= a.ctas) return c;
  return 0;
}

}  // namespace

// CTAs of a cluster per pair, 0 for the launch over all tiles.  A cluster needs no joining launch and no
// look-up of the other requests, but its shares follow its own request alone: taken where the pairs
// with their clusters fit the GPU at once and no share can be long: 24 tiles at what the block table's width and
// the window allow.  In a graph, 32 / 4 heads of 128, microseconds by all tiles / by clusters: 1 request of
// 500 keys 7.2 / 5.8, of 8000 (8 CTAs, 16 tiles) 12.6 / 10.9, of 16,000 (31 tiles) 15.2 / 16.9; 16 requests of
// 2000 (4 CTAs, 8 tiles) 14.3 / 12.4, of 4000 20.3 / 18.8, of 8000 29.7 / 30.2; one CTA a pair, 64 slots of 1280
// 22.6 / 21.0, of 2000 31.1 / 30.6, of 3000 40.2 / 41.8; nearly a CTA for each pair, 100 slots of 3000 56.8 / 51.4, of
// 2200 - 4500 64.7 / 64.5.  A wider table changes neither form's time, only which is taken: 64 slots of 1280 keys in
// tables of 4096 run over all tiles, 22.6 us; 1 request of 500 in one of 32,768 7.1.
int kv8_decode_cluster(const Kv8AttnArgs& a) {
  const int64_t pairs = pairs_of(a), tiles = most_tiles(a);
  const int c = widest_cluster(a);
  return c > 0 && tiles <= (c == 1 && 4 * pairs >= 3 * a.ctas ? 64 : 24 * c) ? c : 0;
}

// Chunks of few tokens: the decode kernel reads the context once per token (mostly out of L2), the chunk
// kernel once, but expands it.  Taken where every pair runs at once with at most 16 tiles to a CTA, and for one
// or two tokens a request in the mean (requests without new tokens count; the lengths are on the device).  In a
// graph, 32 / 4 heads of 128, microseconds by the decode / chunk kernel: one request of 4 tokens on 2000 keys
// 7.6 / 12.2, on 32,000 26.1 / 27.5; 8 on 8000 17.0 / 18.6, on 16,000 23.9 / 21.4; 16 on 4000 16.9 / 19.1, on 16,000
// 36 / 24; 96 on 500 12.6 / 16.5, on 4000 50 / 24; 4 requests of 4 on 4000 17.3 / 16.6, on 8000 25.7 / 23.5; 16
// requests of 2 on 4000 28 / 38, on 32,000 164 / 228.  Uneven batches: 63 requests of one token on 500 keys beside 65
// tokens on 100,000 905 / 1362, beside 65 on 20,000 159 / 314; 15 beside 17 on 32,000 77 / 228.
bool kv8_few_tokens(const Kv8AttnArgs& a) {
  const int64_t rows = a.q_rows, requests = a.batch;
  if (rows > 512 || rows * a.bt_pages >= (int64_t{1} << 31)) return false;
  return rows <= 2 * requests || most_tiles(a) <= 16 * widest_cluster(a) || (requests == 1 && rows <= 4);
}

int64_t kv8_decode_scratch_floats(int ctas, int group, int head_dim) {
  return 2 * static_cast<int64_t>(ctas) * (group > 8 ? 16 : 8) * (head_dim + 2);
}

cudaError_t kv8_decode(const Kv8AttnArgs& a, cudaStream_t stream) {
  if (a.q_rows == 0) return cudaSuccess;
  CUtensorMap tk, tv;
  const int64_t rows = static_cast<int64_t>(a.num_pages) * a.hkv * kPage;
  if (!encode(&tk, a.k, a.head_dim, rows) || !encode(&tv, a.v, a.head_dim, rows)) return cudaErrorInvalidValue;
  Params p{};
  p.q = static_cast<const __nv_bfloat16*>(a.q);
  p.q_stride = a.q_stride;
  p.k_exp = static_cast<const uint8_t*>(a.k_exp);
  p.v_exp = static_cast<const uint8_t*>(a.v_exp);
  p.block_table = a.block_table;
  p.bt_stride = a.bt_stride;
  p.bt_pages = a.bt_pages;
  p.num_pages = a.num_pages;
  p.kv_lens = a.kv_lens;
  p.cu_q = a.cu_q;
  p.requests = a.batch;
  p.batch = a.q_rows;
  p.hq = a.hq;
  p.hkv = a.hkv;
  p.group = a.hq / a.hkv;
  const int nt = p.group > 8 ? 2 : 1;
  p.head_groups = (p.group + 8 * nt - 1) / (8 * nt);
  p.scale = a.scale;
  p.window = a.window;
  p.sinks = a.sinks;
  p.out = static_cast<__nv_bfloat16*>(a.out);
  p.out_stride = a.out_stride;
  p.ctas = a.ctas;
  p.cluster = kv8_decode_cluster(a);
  p.part_o = a.scratch;
  p.part_ml = a.scratch + 2 * static_cast<int64_t>(a.ctas) * 8 * nt * a.head_dim;
  p.status = a.status;
  if (a.head_dim == 128) return nt == 1 ? launch<128, 1>(tk, tv, p, stream) : launch<128, 2>(tk, tv, p, stream);
  if (a.head_dim == 64) return nt == 1 ? launch<64, 1>(tk, tv, p, stream) : launch<64, 2>(tk, tv, p, stream);
  return cudaErrorInvalidValue;
}

}  // namespace omni
