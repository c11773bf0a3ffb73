// Chunk attention over the 8-bit paged KV cache (form: kv8.cuh) on the 5th-generation tensor cores.
//
//   o_i = sum_j p_ij v_j,   p_i = softmax_j(q_i . k_j * scale) over the keys j visible to query i
//
// Long chunks are bound by the tensor cores (4 D operations per visible pair) and, as much, by the
// softmax's arithmetic on each score; chunks with few rows by the cache's bytes and latency.
//
// A CTA computes 128-row query tiles (GQA-packed: row r = token tok0 + r / G, head h G + r % G) over the
// 64-key blocks (one page each) that they see:
//
// * Keys and values enter the tensor cores as bf16 (exact: 4 significant bits times a power of two) in the
//   swizzled shared-memory layout.  Where several row tiles see the same blocks, a launch before expands
//   each block once into global memory as it will lie in shared memory, and one loader thread fetches it
//   by bulk copies; the CTA then works on two query tiles.  Otherwise, for one query tile, one thread
//   copies blocks of codes into a ring (four ahead) and eight loader warps expand them from there.  With
//   the codes read by the loader warps themselves, two blocks ahead, 16 tokens on 100,000 keys took 76 us, not 59.
// * One elected thread issues S = Q K^T and O += P V with S, P and O in tensor memory.  S has two
//   buffers per tile, and between a PV and the S that takes its columns lie the other tile's two
//   products, so neither the softmax nor the tensor core waits for a round trip.  P (bf16) takes
//   the place of its S and never goes through shared memory.
// * A softmax warpgroup per tile, one thread per row: running maximum (raised only when exceeded
//   by 2^8), 32-bit sums, O rescaled in tensor memory when the maximum is raised.
//
// Chunks with few row tiles split the key blocks over the grid's second dimension; the partial
// outputs are joined in order by a second, dependent launch.  The row tiles are found on the device
// from cu_q, so a launch depends on sizes alone.
//
// Measured, 32 / 4 heads of 128: 2048 new tokens on 32,768 keys 897 us = 1264 TFLOP/s cold, 1027 us when
// repeated under the power cap (cuBLAS bf16: 1627 and 1391); 8 chunks of 100 - 1024 tokens on up to 2500
// keys 168 - 178 us.  The two-tile loop takes about 1600 cycles a block: 1024 of tensor-core arithmetic
// (1280 with the shared-memory reads of 64-key S products), 1024 of exponentials.  Sixteen softmax
// warps (two threads a row) took 987 us, weights at the last maximum beside the block's own 949, persistent CTAs
// that fetch the next tile early 949.
//
// A key whose K or V row is marked as not finite enters as a NaN key row and a zero value row: its
// scores are NaN for the queries that see it, and masked by selection for those that do not.
#include <cuda.h>
#include <cuda_bf16.h>
#include <stdint.h>

#include <algorithm>

#include "host_util.h"
#include "kv8.cuh"
#include "omni_kernels.h"
#include "sm100.cuh"

namespace omni {
namespace {

using namespace kv8;

constexpr int kRows = 128;                 // rows of a query tile
constexpr int kBN = kPage;                 // keys of a block
// Ring stages of expanded blocks, and of blocks still in codes (where the CTA expands them itself).
constexpr int stages(bool expanded) { return expanded ? 5 : 4; }
constexpr int kRaw = 4;
constexpr int kExpandThreads = 128;
// Two query tiles and one loader warp where the tiles come expanded; one query tile and eight loader
// warps where the loaders expand them (the few rows of such a launch do not fill a second tile, and four
// loader warps took 3000 cycles a block, twice the softmax's time).
constexpr int tiles_of(bool expanded) { return expanded ? 2 : 1; }
constexpr int load_warps(bool expanded) { return expanded ? 1 : 8; }
constexpr int threads(bool expanded) { return 32 * (4 * tiles_of(expanded) + load_warps(expanded) + (expanded ? 1 : 2)); }
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRaise = 8.0f;             // log2 units
// Of every 8 pairs of scores, those whose exponential runs on the FMA pipe instead of the special-function
// unit.  2048 new tokens on 32,768, 32 / 4 heads of 128: none 933 us, one 912, two 921, three 956.
constexpr int kFmaPairs = 1;
constexpr int kTmemCols = 512;             // S/P: tile x buffer x 64, O: tile x D
constexpr int kRegionQ = kRows * 128;      // 64 columns of a query tile
constexpr int kRegionK = kBN * 128;        // 64 columns of a block

template <int D, bool kExpanded>
struct Smem {
  static constexpr int kQ = 0;
  static constexpr int kQBytes = kRows * D * 2;
  static constexpr int kKV = tiles_of(kExpanded) * kQBytes;
  static constexpr int kKBytes = kBN * D * 2;
  static constexpr int kRaw0 = kKV + stages(kExpanded) * 2 * kKBytes;
  static constexpr int kCodes = kBN * D;
  static constexpr int kRawBytes = 2 * kCodes + 2 * kBN;         // K codes, V codes, exponents of K, of V
  static constexpr int kBars = kRaw0 + (kExpanded ? 0 : kRaw * kRawBytes);
  static constexpr int kBytes = kBars + 512 + 1024;
};
static_assert(Smem<128, true>::kBytes <= 232448 && Smem<128, false>::kBytes <= 232448, "shared memory exceeds 227 KB");

struct Params {
  const __nv_bfloat16* q;
  int64_t q_stride;
  const uint8_t* k;
  const uint8_t* v;
  const int8_t* k_exp;
  const int8_t* v_exp;
  int num_pages;
  const int* block_table;
  int64_t bt_stride;
  int bt_pages;
  const int* cu_q;
  const int* kv_lens;
  int batch, q_rows, hq, hkv, G, tpt;      // tpt: tokens per 128-row tile
  float scale_log2;
  int window, sinks;
  __nv_bfloat16* out;
  int64_t out_stride;
  int splits;
  float* part_o;                           // [splits][q_rows * hq][D]
  float2* part_ml;                         // [splits][q_rows * hq]
  uint8_t* tiles;                          // expanded K / V tiles, or nullptr
  int slots, slots_by_tok;                 // tiles of a request begin at req * slots (+ its first query row / 64)
  int* status;
};

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
      "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
      "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D (tmem) (+)= A (tmem, bf16 pairs along the columns) * B (smem descriptor)
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n"
      " .reg .pred p;\n"
      " setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// One lane of a converged warp.  The compiler knows the election: behind it, MMA operands stay in uniform
// registers, where a test of the lane's number costs moves of every operand of every MMA.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r != 0;
}

__device__ __forceinline__ void bulk_copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void fence_proxy_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Shared-memory descriptor of an MN-major operand, 128-byte swizzle: rows of 64 bf16 along MN, 8-row
// atoms 1024 bytes apart along K, blocks of 64 columns `lbo` bytes apart.
__device__ __forceinline__ uint64_t umma_desc_mn(uint32_t smem_addr, uint32_t lbo) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

// A maximum of three; a NaN wins.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^x of two lanes on the FMA pipe, for -inf <= x <= 8: x = n + f with n the nearest integer (the low bits of
// x + 1.5 * 2^23), 2^f on [-0.5, 0.5] by 1 + c1 f + c2 f^2 + c3 f^3, and n added to the exponent.  The
// coefficients minimise the largest relative error under p(0) = 1 (a reweighted least-squares fit of this
// file's author's): 1.0e-4 = 2^-13.3, where the weight is rounded to 2^-9 next.  -inf gives 0.
__device__ __forceinline__ float2 exp2_fma(uint64_t x2) {
  const float2 x = unpack(x2);
  const uint64_t c = f32x2(fmaxf(x.x, -127.f), fmaxf(x.y, -127.f));
  const uint64_t magic = f32x2(12582912.f, 12582912.f), unmagic = f32x2(-12582912.f, -12582912.f);
  const uint64_t t = add2(c, magic);
  const uint64_t f = fma2(add2(t, unmagic), f32x2(-1.f, -1.f), c);
  uint64_t y = fma2(f, f32x2(0.055008933f, 0.055008933f), f32x2(0.24221097f, 0.24221097f));
  y = fma2(y, f, f32x2(0.6932829f, 0.6932829f));
  y = fma2(y, f, f32x2(1.f, 1.f));
  const float2 n = unpack(t), v = unpack(y);
  return make_float2(__int_as_float(__float_as_int(v.x) + (__float_as_int(n.x) << 23)),
                     __int_as_float(__float_as_int(v.y) + (__float_as_int(n.y) << 23)));
}

__device__ __forceinline__ uint32_t pack_bf16x2(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int site) {
  const bool ok = mbar_wait(bar, parity, abort_flag, status, kWaitTimeoutNs, kStatusWaitSite + site);
  return __all_sync(0xffffffffu, ok);
}

__device__ __forceinline__ uint32_t bf16x2_mul(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Multipliers that turn shifted e4m3 bits into values.  A code's 4 + 3 bits placed below the sign of
// a bf16 read as code * 2^-120 (subnormal codes included), so a row's factor is 2^(120 + e): one bf16
// while e <= 7, else two.
struct RowScale {
  uint32_t f, more;
  bool two;
};
__device__ __forceinline__ uint32_t bf16x2_pow2(int n) { return static_cast<uint32_t>(n + 127) * 0x00800080u; }

__device__ __forceinline__ RowScale row_scale(int e) {
  RowScale s;
  e = max(kExpMin, min(kExpMax, e));
  s.two = e > 7;
  s.f = bf16x2_pow2(120 + min(e, 7));
  s.more = bf16x2_pow2(max(e - 7, 0));
  return s;
}

// 4 codes -> 4 bf16 values
__device__ __forceinline__ uint2 expand4(uint32_t w, const RowScale& s) {
  uint2 o;
  uint32_t a = __byte_perm(w, 0u, 0x1404), b = __byte_perm(w, 0u, 0x3424);
  a = ((a >> 4) & 0x07f007f0u) | (a & 0x80008000u);
  b = ((b >> 4) & 0x07f007f0u) | (b & 0x80008000u);
  o.x = bf16x2_mul(a, s.f);
  o.y = bf16x2_mul(b, s.f);
  if (s.two) {
    o.x = bf16x2_mul(o.x, s.more);
    o.y = bf16x2_mul(o.y, s.more);
  }
  return o;
}

// This thread's share of a block: 16 codes of N consecutive rows of K and of V, and their exponents.
template <int N>
struct Share {
  uint4 k[N], v[N];
  uint32_t ke, ve;      // one byte per row
};

template <int N>
__device__ __forceinline__ uint32_t load_bytes(const int8_t* p) {
  if constexpr (N == 4) return *reinterpret_cast<const uint32_t*>(p);
  if constexpr (N == 2) return *reinterpret_cast<const uint16_t*>(p);
  return *reinterpret_cast<const uint8_t*>(p);
}

template <int D, int TH>
struct Part {
  static constexpr int CH = D / 16;              // 16-code chunks of a row
  static constexpr int N = kBN * CH / TH;        // rows per thread
  Share<N> x;
  // Thread `tid` of TH reads its share of a block's codes and exponents.
  __device__ __forceinline__ void fetch(const uint8_t* k, const uint8_t* v, const int8_t* ke, const int8_t* ve, int tid) {
    const int r0 = tid / CH * N, at = r0 * D + tid % CH * 16;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x.k[i] = *reinterpret_cast<const uint4*>(k + at + i * D);
      x.v[i] = *reinterpret_cast<const uint4*>(v + at + i * D);
    }
    x.ke = load_bytes<N>(ke + r0);
    x.ve = load_bytes<N>(ve + r0);
  }
  // Expands it into the block's K and V tiles (the tensor core's swizzled layout); rows from `left`
  // on lie past the context: their values become zeros (their scores are masked).
  __device__ __forceinline__ void store(uint8_t* dk, uint8_t* dv, int left, int tid) {
    const int c = tid % CH, r0 = tid / CH * N;
    dk += (c >> 2) * kRegionK;
    dv += (c >> 2) * kRegionK;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = r0 + i;
      const int ke = static_cast<int8_t>(x.ke >> (8 * i)), ve = static_cast<int8_t>(x.ve >> (8 * i));
      const bool bad = ke == kExpBad || ve == kExpBad;
      RowScale ks = row_scale(ke), vs = row_scale(ve);
      if (bad) {
        ks.f = 0x7fc07fc0u;
        ks.two = false;
        x.k[i] = make_uint4(0u, 0u, 0u, 0u);
      }
      if (bad || r >= left) x.v[i] = make_uint4(0u, 0u, 0u, 0u);
      const uint2 a0 = expand4(x.k[i].x, ks), a1 = expand4(x.k[i].y, ks);
      const uint2 a2 = expand4(x.k[i].z, ks), a3 = expand4(x.k[i].w, ks);
      const uint2 b0 = expand4(x.v[i].x, vs), b1 = expand4(x.v[i].y, vs);
      const uint2 b2 = expand4(x.v[i].z, vs), b3 = expand4(x.v[i].w, vs);
      const uint4 k0 = make_uint4(a0.x, a0.y, a1.x, a1.y), k1 = make_uint4(a2.x, a2.y, a3.x, a3.y);
      const uint4 v0 = make_uint4(b0.x, b0.y, b1.x, b1.y), v1 = make_uint4(b2.x, b2.y, b3.x, b3.y);
      // the two halves of a 128-dim row share banks: its lanes store their 16-byte pairs in opposite order
      const bool swap = c >= 4;
      const int ch = 2 * (c & 3) + (swap ? 1 : 0);
      const int at0 = r * 128 + ((ch ^ (r & 7)) << 4), at1 = r * 128 + (((ch ^ 1) ^ (r & 7)) << 4);
      *reinterpret_cast<uint4*>(dk + at0) = swap ? k1 : k0;
      *reinterpret_cast<uint4*>(dk + at1) = swap ? k0 : k1;
      *reinterpret_cast<uint4*>(dv + at0) = swap ? v1 : v0;
      *reinterpret_cast<uint4*>(dv + at1) = swap ? v0 : v1;
    }
  }
};

// Key blocks that the queries at positions past .. past + n - 1 (n > 0) of a request see: the pages of
// [0, sinks) and of [lo, end).
struct Blocks {
  int sink_blocks, first, count;
  __device__ Blocks(const Params& p, int kv_len, int past, int n) {
    const int end = max(0, min(kv_len, past + n));
    const int lo = p.window > 0 ? min(end, max(0, past - p.window + 1)) : 0;
    first = lo >> 6;
    sink_blocks = min((min(p.sinks, lo) + 63) >> 6, first);
    count = end > 0 ? sink_blocks + ((end + 63) >> 6) - first : 0;
  }
  __device__ int at(int j) const { return j < sink_blocks ? j : first + j - sink_blocks; }
  __device__ int of(int page) const { return page < sink_blocks ? page : sink_blocks + page - first; }   // at()'s inverse
};

// A request's new tokens (rows q_begin .. q_begin + q_len - 1 of q; cu_q never names rows past q) and its keys.
struct Chunk {
  int q_begin, q_len, kv_len;
  int past;                                                     // keys before the chunk's first query
  __device__ Chunk(const Params& p, int req) {
    q_begin = min(max(0, p.cu_q[req]), p.q_rows);
    q_len = min(p.cu_q[req + 1], p.q_rows) - q_begin;
    kv_len = max(0, min(p.kv_lens[req], p.bt_pages * kPage));
    past = kv_len - (p.cu_q[req + 1] - q_begin);
  }
  // Its first tile of p.tiles.  With a window a request of n tokens sees at most slots + n / 64 blocks, and
  // req * slots + q_begin / 64 leaves room for them without a look at the others' lengths.
  __device__ int64_t first_tile(const Params& p, int req) const {
    return static_cast<int64_t>(req) * p.slots + (p.slots_by_tok ? q_begin >> 6 : 0);
  }
};

// Expands every block that a request's new tokens see, once, into `tiles` (K tile, V tile of each
// [request][block][KV head], as they will lie in shared memory).
template <int D>
__global__ void __launch_bounds__(kExpandThreads) kv8_expand_kernel(const Params p) {
  grid_dep_wait();
  grid_dep_launch();
  const int req = blockIdx.y, h = blockIdx.z;
  const Chunk c(p, req);
  if (c.q_len <= 0) return;
  const Blocks bl(p, c.kv_len, c.past, c.q_len);
  if (static_cast<int>(blockIdx.x) >= bl.count) return;
  const int i = bl.at(blockIdx.x);
  const int page = checked_page(p.block_table[static_cast<int64_t>(req) * p.bt_stride + i], p.num_pages);
  Part<D, kExpandThreads> part;
  const int64_t row0 = (static_cast<int64_t>(page) * p.hkv + h) * kPage;
  part.fetch(p.k + row0 * D, p.v + row0 * D, p.k_exp + row0, p.v_exp + row0, threadIdx.x);
  constexpr int kTile = Smem<D, true>::kKBytes;
  uint8_t* dst = p.tiles + ((c.first_tile(p, req) + blockIdx.x) * p.hkv + h) * (2 * kTile);
  part.store(dst, dst + kTile, c.kv_len - i * kPage, threadIdx.x);
}

// kExpanded: the K / V tiles come ready from kv8_expand_kernel by bulk copies.
template <int D, bool kExpanded>
__global__ void __launch_bounds__(threads(kExpanded), 1) kv8_prefill_kernel(const Params p) {
  using S = Smem<D, kExpanded>;
  constexpr int kStages = stages(kExpanded);
  constexpr int kTiles = tiles_of(kExpanded), kLoadWarps = load_warps(kExpanded);
  constexpr int kLoad0 = 4 * kTiles, kMmaWarp = kLoad0 + kLoadWarps;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t* q_full = bars;                     // [2] tile
  uint64_t* kv_full = q_full + 2;              // [kStages]
  uint64_t* kv_empty = kv_full + kStages;      // [kStages]
  uint64_t* s_full = kv_empty + kStages;       // [2][2] tile, buffer
  uint64_t* p_full = s_full + 4;               // [2][2]
  uint64_t* pv_done = p_full + 4;              // [2] tile
  uint64_t* o_full = pv_done + 2;              // [2] tile: the last PV
  uint64_t* drain = o_full + 2;
  uint64_t* raw_full = drain + 1;              // [kRaw]
  uint64_t* raw_empty = raw_full + kRaw;       // [kRaw]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(raw_empty + kRaw);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  grid_dep_wait();

  // Row tile and KV head of this CTA.  The grid hands CTAs out in order, and the last to start should be
  // short: requests by falling context (up to 32 of them; by position in the batch beyond), each
  // request's tiles from its last, and all KV heads of a tile side by side.
  int req = -1, tok0 = 0;
  const int h = static_cast<int>(blockIdx.x % p.hkv), z = blockIdx.y;
  {
    const int step = kTiles * p.tpt;
    const int x = static_cast<int>(blockIdx.x / p.hkv);
    int cum = 0;
    for (int base = 0; base < p.batch && req < 0; base += 32) {
      const int r = base + lane;
      const int n = r < p.batch ? (max(0, p.cu_q[r + 1] - p.cu_q[r]) + step - 1) / step : 0;
      int before = 0, all = 0;
      if (p.batch <= 32) {
        const int key = r < p.batch ? p.kv_lens[r] : 0;
        for (int i = 0; i < p.batch; ++i) {
          const int ki = __shfl_sync(0xffffffffu, key, i), ni = __shfl_sync(0xffffffffu, n, i);
          if (ki > key || (ki == key && i < lane)) before += ni;
        }
      } else {
        before = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, before, d);
          if (lane >= d) before += up;
        }
        all = __shfl_sync(0xffffffffu, before, 31);
        before -= n;
      }
      const int in = x - cum - before;
      const unsigned mine = __ballot_sync(0xffffffffu, in >= 0 && in < n);
      if (mine != 0) {
        const int at = __ffs(mine) - 1;
        req = base + at;
        tok0 = __shfl_sync(0xffffffffu, (n - 1 - in) * step, at);
      }
      cum += all;
    }
    if (req < 0) return;
  }
  const Chunk chunk(p, req);
  const int q_begin = chunk.q_begin, q_len = chunk.q_len, kv_len = chunk.kv_len, past = chunk.past;
  const int tiles = kTiles == 2 && q_len - tok0 > p.tpt ? 2 : 1;
  const Blocks bl(p, kv_len, past + tok0, min(q_len - tok0, kTiles * p.tpt));
  const int j0 = static_cast<int>(static_cast<int64_t>(bl.count) * z / p.splits);
  const int nb = static_cast<int>(static_cast<int64_t>(bl.count) * (z + 1) / p.splits) - j0;
  auto block_of = [&](int j) { return bl.at(j0 + j); };

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 128);
      mbar_init(&pv_done[i], 1);
      mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&kv_full[i], kLoadWarps);
      mbar_init(&kv_empty[i], 1);
    }
    for (int i = 0; i < kRaw; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], kLoadWarps);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_dep_launch();   // with tensor memory in hand: a dependent may allocate its own before it waits for this grid
  const uint32_t tmem = *tmem_slot;
  auto s_col = [](int t, int b) -> uint32_t { return static_cast<uint32_t>(t * 2 + b) * 64u; };
  auto o_col = [](int t) -> uint32_t { return 256u + static_cast<uint32_t>(t) * D; };

  if (warp >= kLoad0 && warp < kMmaWarp) {
    // ------------------------------------------------------------ loaders
    int stage = 0;
    uint32_t phase = 1;                     // the first round finds the ring empty
    if constexpr (kExpanded) {
      if (elect_one()) {
        const Blocks all(p, kv_len, past, q_len);               // as the expansion numbered them
        const uint8_t* src = p.tiles + (chunk.first_tile(p, req) * p.hkv + h) * (2 * S::kKBytes);
        int j = 0;
        for (; j < nb; ++j) {
          if (j >= kStages && !mbar_wait(&kv_empty[stage], phase, abort_flag, p.status, kWaitTimeoutNs, kStatusWaitSite + 41)) break;
          mbar_arrive_expect_tx(&kv_full[stage], 2 * S::kKBytes);
          bulk_copy(smem + S::kKV + stage * 2 * S::kKBytes, src + static_cast<int64_t>(all.of(block_of(j))) * p.hkv * (2 * S::kKBytes),
                    2 * S::kKBytes, &kv_full[stage]);
          if (++stage == kStages) stage = 0, phase ^= 1;
        }
        // every issued copy has landed before the CTA's shared memory goes away
        for (int i = max(0, j - kStages); i < j; ++i) mbar_wait(&kv_full[i % kStages], (i / kStages) & 1, nullptr, p.status);
      }
      __syncwarp();
    } else {
      constexpr int TH = 32 * kLoadWarps;
      const int tid = threadIdx.x - 32 * kLoad0;
      for (int j = 0; j < nb; ++j) {
        const int rs = j % kRaw;
        if (!warp_wait(&raw_full[rs], (j / kRaw) & 1, abort_flag, p.status, 49)) break;
        const uint8_t* k = smem + S::kRaw0 + rs * S::kRawBytes;
        const int8_t* e = reinterpret_cast<const int8_t*>(k + 2 * S::kCodes);
        Part<D, TH> part;
        part.fetch(k, k + S::kCodes, e, e + kBN, tid);
        if (j >= kStages && !warp_wait(&kv_empty[stage], phase, abort_flag, p.status, 41)) break;
        uint8_t* dk = smem + S::kKV + stage * 2 * S::kKBytes;
        part.store(dk, dk + S::kKBytes, kv_len - block_of(j) * kPage, tid);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&kv_full[stage]);
          // Only now: the codes have been used.  Released right after their loads, a slot could be filled again
          // while a load was still to come, and rows of the block four ahead took their places.
          mbar_arrive(&raw_empty[rs]);
        }
        if (++stage == kStages) stage = 0, phase ^= 1;
      }
    }
  } else if (warp == kMmaWarp + 1) {
    // ------------------------------------------------------------ copies of the blocks' codes
    if (elect_one()) {
      const int* table = p.block_table + static_cast<int64_t>(req) * p.bt_stride;
      auto page_of = [&](int j) { return j < nb ? checked_page(table[block_of(j)], p.num_pages) : 0; };
      int page = page_of(0), j = 0;
      for (; j < nb; ++j) {
        const int rs = j % kRaw;
        const int64_t row0 = (static_cast<int64_t>(page) * p.hkv + h) * kPage;
        page = page_of(j + 1);
        if (j >= kRaw && !mbar_wait(&raw_empty[rs], (j / kRaw - 1) & 1, abort_flag, p.status, kWaitTimeoutNs, kStatusWaitSite + 50)) break;
        uint8_t* dst = smem + S::kRaw0 + rs * S::kRawBytes;
        mbar_arrive_expect_tx(&raw_full[rs], S::kRawBytes);
        bulk_copy(dst, p.k + row0 * D, S::kCodes, &raw_full[rs]);
        bulk_copy(dst + S::kCodes, p.v + row0 * D, S::kCodes, &raw_full[rs]);
        bulk_copy(dst + 2 * S::kCodes, p.k_exp + row0, kBN, &raw_full[rs]);
        bulk_copy(dst + 2 * S::kCodes + kBN, p.v_exp + row0, kBN, &raw_full[rs]);
      }
      // every issued copy has landed before the CTA's shared memory goes away
      for (int i = max(0, j - kRaw); i < j; ++i) mbar_wait(&raw_full[i % kRaw], (i / kRaw) & 1, nullptr, p.status);
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------ MMA issuer
    // One thread runs the whole sequence: its instructions between two MMAs are what the tensor
    // core waits for, so the descriptors are a base plus constants and nothing is warp-wide.
    if (elect_one()) {
      constexpr uint32_t idesc_s = umma_idesc_bf16_f32(kRows, kBN);
      constexpr uint32_t idesc_o = umma_idesc_bf16_f32(kRows, D) | (1u << 16);   // B MN-major
      const uint64_t dq = umma_desc_sw128(smem_u32(smem + S::kQ));
      const uint64_t dk = umma_desc_sw128(smem_u32(smem + S::kKV));
      const uint64_t dv = umma_desc_mn(smem_u32(smem + S::kKV + S::kKBytes), kRegionK);
      auto wait = [&](uint64_t* bar, uint32_t parity, int site) {
        return mbar_wait(bar, parity, abort_flag, p.status, kWaitTimeoutNs, kStatusWaitSite + site);
      };
      auto issue_s = [&](int t, int b, int s) {
        const uint64_t qa = dq + t * (S::kQBytes >> 4), ka = dk + s * (2 * S::kKBytes >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_f16_ss(tmem + s_col(t, b), qa + ((kk >> 2) * (kRegionQ >> 4) + 2 * (kk & 3)),
                      ka + ((kk >> 2) * (kRegionK >> 4) + 2 * (kk & 3)), idesc_s, kk > 0 ? 1u : 0u);
        umma_commit(&s_full[t * 2 + b]);
      };
      bool ok = nb > 0;
      for (int t = 0; t < tiles && ok; ++t) ok = wait(&q_full[t], 0, 44);
      auto issue_pv = [&](int t, int j, int s) {
        const uint64_t va = dv + s * (2 * S::kKBytes >> 4);
#pragma unroll
        for (int kk = 0; kk < kBN / 16; ++kk)
          umma_f16_ts(tmem + o_col(t), tmem + s_col(t, j & 1) + kk * 8, va + kk * (16 * 128 >> 4), idesc_o,
                      (j > 0 || kk > 0) ? 1u : 0u);
        umma_commit(j + 1 < nb ? &pv_done[t] : &o_full[t]);
        if (t == tiles - 1) umma_commit(&kv_empty[s]);
      };
      auto next = [](int s) { return s + 1 == kStages ? 0 : s + 1; };
      // Order: PV_A(j)  S_B(j + 1)  PV_B(j)  S_A(j + 2).  S of a block takes the columns that PV two
      // blocks before reads P from, so it waits for that PV; the other tile's two products lie in
      // between, and keep the tensor core busy meanwhile.
      int s0 = 0, s2 = 0;         // ring stages of blocks j and j + 2 (the next S_A)
      uint32_t sp = 0;
      for (int j = 0; j < 2 && j < nb && ok; ++j) {
        ok = wait(&kv_full[s2], sp, 42);
        if (!ok) break;
        tc_fence_after();
        issue_s(0, j, s2);
        if (j == 0 && tiles == 2) issue_s(1, 0, s2);
        s2 = next(s2);
      }
      for (int j = 0; j < nb && ok; ++j) {
        const int b = j & 1, s1 = next(s0);
        if (!(ok = wait(&p_full[b], (j >> 1) & 1, 43))) break;
        tc_fence_after();
        issue_pv(0, j, s0);
        if (tiles == 2) {
          if (j + 1 < nb) {
            if (j > 0 && !(ok = wait(&pv_done[1], b ^ 1, 48))) break;
            tc_fence_after();
            issue_s(1, b ^ 1, s1);
          }
          if (!(ok = wait(&p_full[2 + b], (j >> 1) & 1, 43))) break;
          tc_fence_after();
          issue_pv(1, j, s0);
        }
        s0 = s1;
        if (j + 2 < nb) {
          if (!(ok = wait(&kv_full[s2], sp, 42) && wait(&pv_done[0], b, 48))) break;
          tc_fence_after();
          issue_s(0, b, s2);
          s2 = next(s2);
          if (s2 == 0) sp ^= 1;
        }
      }
      umma_commit(drain);
      mbar_wait(drain, 0, nullptr, p.status);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ softmax + epilogue
    const int t = warp >> 2;
    const int r = threadIdx.x & 127;                  // row of the tile = TMEM lane
    const uint32_t lane_addr = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int in = r / p.G;                           // token of the row within the tile
    const int tok = tok0 + t * p.tpt + in;
    const int head = h * p.G + (r - in * p.G);
    const bool row_ok = t < tiles && in < p.tpt && tok < q_len;
    // a row without a query keeps every key: its results are not stored
    const int qpos = row_ok ? past + tok : 0x3fffffff;
    const int low = row_ok && p.window > 0 ? qpos - p.window : -1;   // keys <= low are seen only below `sinks`
    float m_run = -INFINITY, l_run = 0.f;
    if (t < tiles && nb > 0) {
      const __nv_bfloat16* src = p.q + static_cast<int64_t>(q_begin + (row_ok ? tok : 0)) * p.q_stride + static_cast<int64_t>(head) * D;
      uint8_t* dst = smem + S::kQ + t * S::kQBytes + r * 128;
      uint32_t top = 0;                               // largest magnitudes of the even and of the odd elements
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        const uint4 x = row_ok ? *reinterpret_cast<const uint4*>(src + c * 8) : make_uint4(0u, 0u, 0u, 0u);
        *reinterpret_cast<uint4*>(dst + (c >> 3) * kRegionQ + (((c & 7) ^ (r & 7)) << 4)) = x;
        top = __vmaxu2(__vmaxu2(top, x.x & 0x7fff7fffu), __vmaxu2(x.y & 0x7fff7fffu, __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu)));
      }
      fence_proxy_async_smem();
      mbar_arrive(&q_full[t]);
      // An infinite query whose scores are all -inf would look like one that sees nothing: its sum is NaN from
      // the start, unless it does see nothing.
      if (((top & 0xffffu) >= 0x7f80u || top >= 0x7f800000u) && qpos >= 0) l_run = NAN;
    }
    bool ok = true;
    const int n = t < tiles ? nb : 0;
    for (int j = 0; j < n && ok; ++j) {
      const int b = j & 1;
      if (!warp_wait(&s_full[t * 2 + b], (j >> 1) & 1, abort_flag, p.status, 45)) { ok = false; break; }
      tc_fence_after();
      float s[kBN];
      {
        uint32_t v[kBN];
        tmem_ld32(tmem + lane_addr + s_col(t, b), v);
        tmem_ld32(tmem + lane_addr + s_col(t, b) + 32, v + 32);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < kBN; ++i) s[i] = __uint_as_float(v[i]);
      }
      const int k0 = block_of(j) * kPage;
      if (k0 + kBN - 1 > qpos || (k0 <= low && k0 + kBN > p.sinks)) {
#pragma unroll
        for (int i = 0; i < kBN; ++i) {
          const int key = k0 + i;
          s[i] = key <= qpos && (key > low || key < p.sinks) ? s[i] : -INFINITY;
        }
      }
      float mx[4] = {max3(s[0], s[4], s[8]), max3(s[1], s[5], s[9]), max3(s[2], s[6], s[10]), max3(s[3], s[7], s[11])};
#pragma unroll
      for (int i = 12; i < 60; i += 8)
#pragma unroll
        for (int u = 0; u < 4; ++u) mx[u] = max3(mx[u], s[i + u], s[i + 4 + u]);
      const float mraw = max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], s[60], s[61]), max3(s[62], s[63], s[63]));
      float mb = mraw * p.scale_log2;                 // scale > 0: -inf stays -inf
      if (mb == INFINITY) mb = NAN;                   // an infinite score has no softmax: the row becomes NaN, as by a NaN score
      // decided per row, executed per warp: tensor-memory accesses are warp-collective
      const bool grow = !(mb <= m_run + kRaise);
      if (__any_sync(0xffffffffu, grow)) {
        const bool scale_o = grow && j > 0 && m_run > -INFINITY;
        if (__any_sync(0xffffffffu, scale_o)) {
          if (!warp_wait(&pv_done[t], (j - 1) & 1, abort_flag, p.status, 46)) { ok = false; break; }
          tc_fence_after();
          const float f = scale_o ? ex2(m_run - mb) : 1.f;
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t v[32];
            tmem_ld32(tmem + lane_addr + o_col(t) + c, v);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
            tmem_st32(tmem + lane_addr + o_col(t) + c, v);
          }
          tmem_st_wait();
          l_run *= f;
        }
        if (grow) m_run = mb;
      }
      const float msub = m_run == -INFINITY ? 0.f : m_run;
      const uint64_t scale2 = f32x2(p.scale_log2, p.scale_log2), sub2 = f32x2(-msub, -msub);
      uint64_t ls[4] = {0, 0, 0, 0};
      uint32_t pk[kBN / 2];
#pragma unroll
      for (int i = 0; i < kBN; i += 2) {
        const uint64_t x = fma2(f32x2(s[i], s[i + 1]), scale2, sub2);
        float2 e;
        if (((i >> 1) & 7) < kFmaPairs) {
          e = exp2_fma(x);
        } else {
          e = unpack(x);
          e = make_float2(ex2(e.x), ex2(e.y));
        }
        ls[(i >> 1) & 3] = add2(ls[(i >> 1) & 3], f32x2(e.x, e.y));
        pk[i / 2] = pack_bf16x2(e.x, e.y);
      }
      tmem_st32(tmem + lane_addr + s_col(t, b), pk);
      const float2 lsum = unpack(add2(add2(ls[0], ls[1]), add2(ls[2], ls[3])));
      l_run += lsum.x + lsum.y;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[t * 2 + b]);
    }
    // a barrier of its own: pv_done's phase may be one or two behind here, which its parity cannot tell
    if (n > 0 && ok) ok = warp_wait(&o_full[t], 0, abort_flag, p.status, 47);
    if (t < tiles && ok) {
      tc_fence_after();
      const int64_t row = static_cast<int64_t>(q_begin + tok) * p.hq + head;
      const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
      __nv_bfloat16* orow = p.out + static_cast<int64_t>(q_begin + tok) * p.out_stride + static_cast<int64_t>(head) * D;
      float* prow = p.part_o + (static_cast<int64_t>(z) * p.q_rows * p.hq + row) * D;
      if (p.splits > 1 && row_ok) p.part_ml[static_cast<int64_t>(z) * p.q_rows * p.hq + row] = make_float2(m_run, l_run);
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t v[32];
        if (n > 0) {
          tmem_ld32(tmem + lane_addr + o_col(t) + c, v);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0u;
        }
        if (!row_ok) continue;
        if (p.splits > 1) {
          if (n > 0) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) *reinterpret_cast<uint4*>(prow + c + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint4 o;
            o.x = pack_bf16x2(__uint_as_float(v[i]) * inv, __uint_as_float(v[i + 1]) * inv);
            o.y = pack_bf16x2(__uint_as_float(v[i + 2]) * inv, __uint_as_float(v[i + 3]) * inv);
            o.z = pack_bf16x2(__uint_as_float(v[i + 4]) * inv, __uint_as_float(v[i + 5]) * inv);
            o.w = pack_bf16x2(__uint_as_float(v[i + 6]) * inv, __uint_as_float(v[i + 7]) * inv);
            *reinterpret_cast<uint4*>(orow + c + i) = o;
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Joins the splits' partial outputs of each row in order.  W warps per (token, query head); a
// token that no request names keeps what the output held.
template <int D, int W>
__global__ void __launch_bounds__(128) kv8_prefill_join_kernel(const Params p) {
  __shared__ float red[4 * D];
  grid_dep_wait();
  const int64_t rows = static_cast<int64_t>(p.q_rows) * p.hq;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (4 / W) + (threadIdx.x >> 5) / W;
  if (row >= rows) return;
  const int64_t tok = row / p.hq;
  if (tok >= p.cu_q[p.batch]) return;
  join_parts<D, W>(
      p.splits, [&](int z) { return p.part_ml[z * rows + row]; }, [&](int z) { return p.part_o + (z * rows + row) * D; },
      p.out + tok * p.out_stride + (row - tok * p.hq) * D, red);
}

template <int D>
cudaError_t launch(const Params& p, int64_t tiles, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>(tiles), p.splits);
  cudaError_t e;
  if (p.tiles != nullptr) {
    if ((e = ensure_smem_attr<kv8_prefill_kernel<D, true>>(Smem<D, true>::kBytes)) != cudaSuccess) return e;
    const unsigned most = static_cast<unsigned>(p.slots_by_tok ? std::min(p.bt_pages, p.slots + p.q_rows / kPage) : p.bt_pages);
    e = launch_dependent(kv8_expand_kernel<D>, dim3(most, p.batch, p.hkv), kExpandThreads, 0, stream, p);
    if (e != cudaSuccess) return e;
    e = launch_dependent(kv8_prefill_kernel<D, true>, grid, threads(true), Smem<D, true>::kBytes, stream, p);
  } else {
    if ((e = ensure_smem_attr<kv8_prefill_kernel<D, false>>(Smem<D, false>::kBytes)) != cudaSuccess) return e;
    e = launch_dependent(kv8_prefill_kernel<D, false>, grid, threads(false), Smem<D, false>::kBytes, stream, p);
  }
  if (e != cudaSuccess || p.splits == 1) return e;
  const int64_t rows = static_cast<int64_t>(p.q_rows) * p.hq;
  if (p.splits > 8) return launch_dependent(kv8_prefill_join_kernel<D, 4>, dim3(static_cast<unsigned>(rows)), 128, 0, stream, p);
  return launch_dependent(kv8_prefill_join_kernel<D, 1>, dim3(static_cast<unsigned>((rows + 3) / 4)), 128, 0, stream, p);
}

int64_t row_tiles(int64_t q_rows, int batch, int group, bool expanded) {
  const int64_t step = tiles_of(expanded) * (kRows / group);
  // n tokens make at most (n - 1) / step + 1 tiles
  return std::min(q_rows, std::max<int64_t>(0, q_rows - batch) / step + batch);
}

// Blocks that requests of one batch can see, by what the host knows: a window's span, the sinks and a chunk's own
// tokens, each with its ragged ends (slots + new / 64 a request), or the whole block table.
struct Slots {
  int64_t each, all;
  bool by_tok;
  explicit Slots(const Kv8AttnArgs& a) {
    each = a.window / kPage + 3 + (static_cast<int64_t>(a.sinks) + kPage - 1) / kPage;
    all = a.batch * each + a.q_rows / kPage + 1;
    by_tok = a.window > 0 && all < static_cast<int64_t>(a.batch) * a.bt_pages;
    if (!by_tok) {
      each = a.bt_pages;
      all = a.batch * each;
    }
  }
};

}  // namespace

// Bytes of the expanded tiles; 0 where the blocks are expanded in the attention kernel itself.  A launch
// of its own costs each block a write and reads of the expanded form, but once for all row tiles of its
// request: taken from four of them on in the mean, where the CTAs have enough blocks to win the launch back: 4200
// (row tile, KV head, block) triples, 28 on each SM.  In a graph, microseconds with / without it, 32 / 4 heads of 128 (16
// tokens a row tile): one request of 64 tokens on 16,000 keys (28 an SM) 43 / 38, on 64,000 105 / 111; 96 on 8000 (20)
// 36 / 34, on 16,000 (40) 50 / 51; 128 on 3000 30 / 25, on 16,000 56 / 68; 1024 on themselves 29 / 28, on 1000 more 46 / 55;
// four of 32 (two row tiles each) on 8000 55 / 43, of 64 66 / 69.  Uneven batches: 2048 tokens on themselves beside 63
// requests of one token on 500 keys 92 / 101, on 4000 294 / 182; 512 on 2000 beside 15 of one on 500 48 / 39; 2048 on 4000
// beside 15 of 16 on 500 106 / 184.
int64_t kv8_prefill_tile_bytes(const Kv8AttnArgs& a) {
  const int64_t step = kRows / (a.hq / a.hkv);
  int64_t seen = a.bt_pages;
  if (a.window > 0)
    seen = std::min<int64_t>(seen, (static_cast<int64_t>(a.window) + a.q_rows / std::max(1, a.batch)) / kPage + 2 + (static_cast<int64_t>(a.sinks) + 63) / 64);
  const int64_t bytes = Slots(a).all * a.hkv * kPage * a.head_dim * 4;
  if (a.q_rows < 4 * step * a.batch || a.q_rows / step * a.hkv * seen < 4200) return 0;
  if (bytes > (int64_t{1} << 31) || a.batch > 65535 || a.hkv > 65535) return 0;
  return bytes;
}

// Splits of the key blocks: as many as keep the launch within one CTA per SM where the requests' chunks
// are alike, one where the row tiles alone fill the GPU.  (By the most row tiles that the lengths could make,
// 16 chunks of 4 tokens, 32 / 4 heads of 128, on 16,000 keys took 226 us without a split, 122 with two.)
int kv8_prefill_splits(const Kv8AttnArgs& a, int sm_count) {
  const int group = a.hq / a.hkv;
  const int64_t each = static_cast<int64_t>(a.batch) * tiles_of(a.tiles != nullptr) * (kRows / group);
  const int64_t alike = a.batch * ((a.q_rows + each - 1) / each);
  const int64_t base = std::min(alike, row_tiles(a.q_rows, a.batch, group, a.tiles != nullptr)) * a.hkv;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(sm_count / std::max<int64_t>(1, base), a.bt_pages)));
}

int64_t kv8_prefill_scratch_floats(const Kv8AttnArgs& a) {
  return a.splits > 1 ? static_cast<int64_t>(a.splits) * a.q_rows * a.hq * (a.head_dim + 2) : 0;
}

cudaError_t kv8_prefill(const Kv8AttnArgs& a, cudaStream_t stream) {
  if (a.q_rows == 0) return cudaSuccess;
  const int group = a.hq / a.hkv;
  if (group > kRows) return cudaErrorInvalidValue;
  Params p{};
  p.q = static_cast<const __nv_bfloat16*>(a.q);
  p.q_stride = a.q_stride;
  p.k = static_cast<const uint8_t*>(a.k);
  p.v = static_cast<const uint8_t*>(a.v);
  p.k_exp = static_cast<const int8_t*>(a.k_exp);
  p.v_exp = static_cast<const int8_t*>(a.v_exp);
  p.num_pages = a.num_pages;
  p.block_table = a.block_table;
  p.bt_stride = a.bt_stride;
  p.bt_pages = a.bt_pages;
  p.cu_q = a.cu_q;
  p.kv_lens = a.kv_lens;
  p.batch = a.batch;
  p.q_rows = a.q_rows;
  p.hq = a.hq;
  p.hkv = a.hkv;
  p.G = group;
  p.tpt = kRows / group;
  p.scale_log2 = a.scale * kLog2e;
  p.window = a.window;
  p.sinks = a.sinks;
  p.out = static_cast<__nv_bfloat16*>(a.out);
  p.out_stride = a.out_stride;
  p.splits = a.splits;
  p.part_o = a.scratch;
  p.part_ml = reinterpret_cast<float2*>(a.scratch + static_cast<int64_t>(a.splits) * a.q_rows * a.hq * a.head_dim);
  p.tiles = static_cast<uint8_t*>(a.tiles);
  const Slots slots(a);
  p.slots = static_cast<int>(slots.each);
  p.slots_by_tok = slots.by_tok ? 1 : 0;
  p.status = a.status;
  const int64_t tiles = row_tiles(a.q_rows, a.batch, group, a.tiles != nullptr) * a.hkv;
  if (tiles > 0x7fffffff) return cudaErrorInvalidValue;
  if (a.head_dim == 128) return launch<128>(p, tiles, stream);
  if (a.head_dim == 64) return launch<64>(p, tiles, stream);
  return cudaErrorInvalidValue;
}

}  // namespace omni
