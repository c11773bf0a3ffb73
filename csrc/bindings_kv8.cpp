// torch bindings of the 8-bit paged KV cache (kv8_cache.cu, kv8_decode.cu, kv8_prefill.cu).  Every argument is
// checked here, before anything is launched; a bad one raises with its name.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>

#include "omni_kernels.h"

namespace {

using OptTensor = c10::optional<torch::Tensor>;

// Messages are built from strings alone: streaming a number into a message ends the process where
// the image's C++ runtime and torch's differ.
std::string num(int64_t v) { return std::to_string(v); }

bool aligned16(const torch::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

void check_on(const torch::Tensor& t, const torch::Tensor& like, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be on the cache's CUDA device");
}

// Rows of a 2-D bf16 tensor that the kernels read or write 16 bytes at a time.
void check_rows(const torch::Tensor& t, int64_t cols, const char* name) {
  TORCH_CHECK(t.dim() == 2 && t.scalar_type() == at::kBFloat16, name, " must be a 2-D bf16 tensor");
  TORCH_CHECK(t.size(1) >= cols, name, " has " + num(t.size(1)) + " columns, needs " + num(cols));
  TORCH_CHECK(t.stride(1) == 1 && (t.size(0) <= 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= cols)) && aligned16(t), name,
              " must have contiguous rows, 16-byte aligned");
}

struct Cache {
  int64_t pages, hkv, d;
};

Cache check_cache(const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& ke, const torch::Tensor& ve) {
  TORCH_CHECK(k.is_cuda() && k.dim() == 4 && k.scalar_type() == at::kFloat8_e4m3fn && k.size(2) == 64,
              "cache.k must be a CUDA float8_e4m3fn tensor [pages, Hkv, 64, D]");
  Cache c{k.size(0), k.size(1), k.size(3)};
  TORCH_CHECK(c.d == 64 || c.d == 128, "the 8-bit cache takes head dims 64 and 128, got " + num(c.d));
  TORCH_CHECK(c.pages >= 1 && c.hkv >= 1 && c.pages * c.hkv * 64 < (int64_t{1} << 31),
              "cache.k: pages * Hkv * 64 must be in [1, 2^31)");
  check_on(v, k, "cache.v");
  check_on(ke, k, "cache.k_exp");
  check_on(ve, k, "cache.v_exp");
  TORCH_CHECK(v.scalar_type() == k.scalar_type() && v.sizes() == k.sizes(), "cache.v must match cache.k");
  const int64_t es[3] = {c.pages, c.hkv, 64};
  TORCH_CHECK(ke.scalar_type() == at::kChar && ke.sizes() == at::IntArrayRef(es) && ve.scalar_type() == at::kChar &&
                  ve.sizes() == at::IntArrayRef(es),
              "cache.k_exp / v_exp must be int8 [pages, Hkv, 64]");
  TORCH_CHECK(k.is_contiguous() && v.is_contiguous() && ke.is_contiguous() && ve.is_contiguous(),
              "the cache's tensors must be contiguous");
  TORCH_CHECK(aligned16(k) && aligned16(v) && aligned16(ke) && aligned16(ve), "the cache's tensors must be 16-byte aligned");
  return c;
}

// Uninitialised tensor from the caching allocator (the dispatcher's share of torch::empty is a
// third of a small call's host time).
torch::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const torch::Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
}

const int* int_ptr(const torch::Tensor& t, const torch::Tensor& like, const char* name) {
  check_on(t, like, name);
  TORCH_CHECK(t.scalar_type() == at::kInt && t.is_contiguous(), name, " must be a contiguous int32 tensor");
  return t.data_ptr<int>();
}

void check_launch(cudaError_t e, const char* what) {
  TORCH_CHECK(e == cudaSuccess, what, " failed: ", cudaGetErrorString(e));
}

torch::Tensor kv8_store(const torch::Tensor& qkv, const torch::Tensor& k, const torch::Tensor& v,
                        const torch::Tensor& k_exp, const torch::Tensor& v_exp, const torch::Tensor& slots, int64_t hq,
                        int64_t hkv, int64_t head_dim, const OptTensor& positions, const OptTensor& cos_tab,
                        const OptTensor& sin_tab, int64_t rot_dim, const OptTensor& q_norm, const OptTensor& k_norm,
                        double eps, bool neox, const std::vector<int64_t>& section, bool interleaved,
                        const OptTensor& q_out) {
  const Cache c = check_cache(k, v, k_exp, v_exp);
  TORCH_CHECK(head_dim == c.d && hkv == c.hkv && hq >= 1, "kv8_store: head counts / head dim do not match the cache");
  check_on(qkv, k, "qkv");
  check_rows(qkv, (hq + 2 * hkv) * head_dim, "qkv");
  const int64_t T = qkv.size(0);
  TORCH_CHECK(T < (int64_t{1} << 31), "qkv has too many rows");
  const at::cuda::CUDAGuard guard(k.device());
  omni::Kv8StoreArgs a{};
  a.slot_mapping = int_ptr(slots, k, "slot_mapping");
  TORCH_CHECK(slots.numel() == T, "slot_mapping has " + num(slots.numel()) + " entries for " + num(T) + " tokens");
  TORCH_CHECK(rot_dim >= 0 && rot_dim % 2 == 0 && rot_dim <= head_dim, "rot_dim must be even and in [0, head_dim]");
  if (rot_dim > 0) {
    TORCH_CHECK(positions.has_value() && cos_tab.has_value() && sin_tab.has_value(),
                "RoPE needs positions, cos_tab and sin_tab");
    a.positions = int_ptr(*positions, k, "positions");
    a.pos_rows = positions->dim() == 2 ? static_cast<int>(positions->size(0)) : 1;
    TORCH_CHECK((positions->dim() == 1 || positions->dim() == 2) && (a.pos_rows == 1 || a.pos_rows == 3) &&
                    positions->numel() == a.pos_rows * T,
                "positions must be [T] or [3, T]");
    TORCH_CHECK(section.empty() || (section.size() == 3 && section[0] >= 0 && section[1] >= 0 && section[2] >= 0),
                "mrope_section must be empty or three sizes");
    if (section.empty()) a.pos_rows = 1;   // without sections every pair follows the first row
    for (const auto* t : {&*cos_tab, &*sin_tab}) {
      check_on(*t, k, "cos_tab / sin_tab");
      TORCH_CHECK(t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(1) == rot_dim / 2 && t->is_contiguous() &&
                      t->size(0) >= 1 && t->size(0) == cos_tab->size(0),
                  "cos_tab / sin_tab must be contiguous fp32 [max_pos, rot_dim / 2]");
    }
    a.cos_tab = cos_tab->data_ptr<float>();
    a.sin_tab = sin_tab->data_ptr<float>();
    a.max_pos = static_cast<int>(cos_tab->size(0));
  }
  for (const auto* w : {&q_norm, &k_norm})
    if (w->has_value()) {
      check_on(**w, k, "q_norm / k_norm");
      TORCH_CHECK((*w)->scalar_type() == at::kBFloat16 && (*w)->numel() == head_dim && (*w)->is_contiguous() &&
                      aligned16(**w),
                  "q_norm / k_norm must be contiguous bf16 [head_dim]");
    }
  torch::Tensor q = q_out.has_value() ? *q_out : empty({T, hq * head_dim}, at::kBFloat16, k);
  check_on(q, k, "out");
  check_rows(q, hq * head_dim, "out");
  TORCH_CHECK(q.size(0) == T, "out has " + num(q.size(0)) + " rows for " + num(T) + " tokens");
  a.qkv = qkv.data_ptr();
  a.qkv_stride = qkv.stride(0);
  a.tokens = static_cast<int>(T);
  a.hq = static_cast<int>(hq);
  a.hkv = static_cast<int>(hkv);
  a.head_dim = static_cast<int>(head_dim);
  a.q_out = q.data_ptr();
  a.q_out_stride = q.stride(0);
  a.q_norm = q_norm.has_value() ? q_norm->data_ptr() : nullptr;
  a.k_norm = k_norm.has_value() ? k_norm->data_ptr() : nullptr;
  a.eps = static_cast<float>(eps);
  for (size_t i = 0; i < section.size() && i < 3; ++i) a.section[i] = static_cast<int>(std::min<int64_t>(section[i], head_dim));
  a.interleaved = interleaved ? 1 : 0;
  a.rot_dim = static_cast<int>(rot_dim);
  a.neox = neox ? 1 : 0;
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.k_exp = k_exp.data_ptr();
  a.v_exp = v_exp.data_ptr();
  a.num_slots = c.pages * 64;
  check_launch(omni::kv8_store(a, at::cuda::getCurrentCUDAStream()), "kv8_store");
  return q;
}

std::tuple<torch::Tensor, torch::Tensor> kv8_read(const torch::Tensor& k, const torch::Tensor& v,
                                                  const torch::Tensor& k_exp, const torch::Tensor& v_exp,
                                                  const torch::Tensor& slots) {
  const Cache c = check_cache(k, v, k_exp, v_exp);
  const at::cuda::CUDAGuard guard(k.device());
  omni::Kv8ReadArgs a{};
  a.slots = int_ptr(slots, k, "slots");
  TORCH_CHECK(slots.dim() == 1 && slots.numel() < (int64_t{1} << 31), "slots must be 1-D");
  torch::Tensor ko = empty({slots.numel(), c.hkv, c.d}, at::kBFloat16, k), vo = empty({slots.numel(), c.hkv, c.d}, at::kBFloat16, k);
  a.count = static_cast<int>(slots.numel());
  a.hkv = static_cast<int>(c.hkv);
  a.head_dim = static_cast<int>(c.d);
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.k_exp = k_exp.data_ptr();
  a.v_exp = v_exp.data_ptr();
  a.num_slots = c.pages * 64;
  a.k_out = ko.data_ptr();
  a.v_out = vo.data_ptr();
  check_launch(omni::kv8_read(a, at::cuda::getCurrentCUDAStream()), "kv8_read");
  return {ko, vo};
}

// cu_q: None for decode (one query row per request)
torch::Tensor kv8_attention(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v,
                            const torch::Tensor& k_exp, const torch::Tensor& v_exp, const torch::Tensor& block_table,
                            const OptTensor& cu_q, const torch::Tensor& kv_lens, int64_t hq, int64_t hkv,
                            int64_t head_dim, double scale, int64_t window, int64_t sinks, const OptTensor& out_,
                            const OptTensor& status) {
  const Cache c = check_cache(k, v, k_exp, v_exp);
  TORCH_CHECK(head_dim == c.d && hkv == c.hkv, "the head dim / KV heads do not match the cache");
  TORCH_CHECK(hq >= 1 && hq % hkv == 0, "num_heads must be a multiple of num_kv_heads");
  TORCH_CHECK(hq / hkv <= 128, "at most 128 query heads per KV head");
  TORCH_CHECK(scale > 0 && scale < 1e30, "scale must be positive");
  TORCH_CHECK(window >= 0 && sinks >= 0 && window < (int64_t{1} << 31) && sinks < (int64_t{1} << 31),
              "window and sinks must not be negative");
  check_on(q, k, "q");
  check_rows(q, hq * head_dim, "q");
  const int64_t T = q.size(0), B = kv_lens.numel();
  TORCH_CHECK(T < (int64_t{1} << 31) / hq, "q has too many rows");
  const at::cuda::CUDAGuard guard(k.device());
  omni::Kv8AttnArgs a{};
  a.kv_lens = int_ptr(kv_lens, k, "kv_lens");
  check_on(block_table, k, "block_table");
  TORCH_CHECK(block_table.dim() == 2 && block_table.scalar_type() == at::kInt && block_table.size(0) >= B &&
                  (block_table.size(1) <= 1 || block_table.stride(1) == 1),
              "block_table must be int32 [requests, pages] with contiguous rows");
  TORCH_CHECK(block_table.size(1) < (int64_t{1} << 25), "block_table rows are too long");
  if (cu_q.has_value()) {
    a.cu_q = int_ptr(*cu_q, k, "cu_q");
    TORCH_CHECK(cu_q->numel() == B + 1, "cu_q needs one entry more than kv_lens");
  } else {
    TORCH_CHECK(T * block_table.size(1) < (int64_t{1} << 31), "block_table is too large");
    TORCH_CHECK(T == B, "decode takes one query row per request: " + num(T) + " rows, " + num(B) + " requests");
  }
  torch::Tensor out = out_.has_value() ? *out_ : empty({T, hq * head_dim}, at::kBFloat16, k);
  check_on(out, k, "out");
  check_rows(out, hq * head_dim, "out");
  TORCH_CHECK(out.size(0) == T, "out has " + num(out.size(0)) + " rows for " + num(T) + " query rows");
  if (T == 0) return out;
  TORCH_CHECK(B > 0, "query rows without a request");
  a.q = q.data_ptr();
  a.q_stride = q.stride(0);
  a.q_rows = static_cast<int>(T);
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.k_exp = k_exp.data_ptr();
  a.v_exp = v_exp.data_ptr();
  a.num_pages = static_cast<int>(c.pages);
  a.block_table = block_table.data_ptr<int>();
  a.bt_stride = block_table.stride(0);
  a.bt_pages = static_cast<int>(block_table.size(1));
  a.batch = static_cast<int>(B);
  a.hq = static_cast<int>(hq);
  a.hkv = static_cast<int>(hkv);
  a.head_dim = static_cast<int>(head_dim);
  a.scale = static_cast<float>(scale);
  // a window that no context exceeds is none (and the kernels' 32-bit positions minus it stay in range)
  a.window = window < a.bt_pages * int64_t{64} ? static_cast<int>(window) : 0;
  a.sinks = static_cast<int>(sinks);
  a.out = out.data_ptr();
  a.out_stride = out.stride(0);
  if (status.has_value()) {
    check_on(*status, k, "status");
    TORCH_CHECK(status->scalar_type() == at::kInt, "status must be int32");
    a.status = status->data_ptr<int>();
  }
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  // scratch from the caching allocator, used on the current stream only
  torch::Tensor scratch;
  a.ctas = omni::kv8_decode_ctas(sms, static_cast<int>(hq / hkv), a.head_dim);
  if (!cu_q.has_value() || omni::kv8_few_tokens(a)) {
    if (omni::kv8_decode_cluster(a) == 0) {
      scratch = empty({omni::kv8_decode_scratch_floats(a.ctas, static_cast<int>(hq / hkv), a.head_dim)}, at::kFloat, k);
      a.scratch = scratch.data_ptr<float>();
    }
    check_launch(omni::kv8_decode(a, at::cuda::getCurrentCUDAStream()), "kv8_decode_attention");
  } else {
    torch::Tensor tiles;
    if (const int64_t bytes = omni::kv8_prefill_tile_bytes(a)) {
      // without the room for them the attention kernel expands the blocks itself
      try {
        tiles = empty({bytes}, at::kByte, k);
        a.tiles = tiles.data_ptr();
      } catch (const c10::OutOfMemoryError&) {
      }
    }
    a.splits = omni::kv8_prefill_splits(a, sms);
    if (a.splits > 1) {
      scratch = empty({omni::kv8_prefill_scratch_floats(a)}, at::kFloat, k);
      a.scratch = scratch.data_ptr<float>();
    }
    check_launch(omni::kv8_prefill(a, at::cuda::getCurrentCUDAStream()), "kv8_prefill_attention");
  }
  return out;
}

// The form that kv8_attention takes for a chunk batch of these sizes: "decode" (every token a request of its
// own), "expanded" (key blocks expanded by a launch before) or "in place" (by the attention kernel itself).
std::string kv8_chunk_form(int64_t q_rows, int64_t requests, int64_t table_pages, int64_t hq, int64_t hkv,
                           int64_t head_dim, int64_t window, int64_t sinks) {
  TORCH_CHECK(q_rows >= 0 && requests >= 1 && table_pages >= 0 && hkv >= 1 && hq >= hkv && hq / hkv <= 128 && window >= 0 && sinks >= 0,
              "kv8_chunk_form: sizes out of range");
  omni::Kv8AttnArgs a{};
  a.q_rows = static_cast<int>(q_rows);
  a.batch = static_cast<int>(requests);
  a.bt_pages = static_cast<int>(table_pages);
  a.hq = static_cast<int>(hq);
  a.hkv = static_cast<int>(hkv);
  a.head_dim = static_cast<int>(head_dim);
  a.window = window < table_pages * 64 ? static_cast<int>(window) : 0;
  a.sinks = static_cast<int>(sinks);
  a.ctas = omni::kv8_decode_ctas(at::cuda::getCurrentDeviceProperties()->multiProcessorCount, static_cast<int>(hq / hkv), a.head_dim);
  if (omni::kv8_few_tokens(a)) return "decode";
  return omni::kv8_prefill_tile_bytes(a) > 0 ? "expanded" : "in place";
}

}  // namespace

void bind_kv8(pybind11::module_& m) {
  m.def("kv8_store", &kv8_store, "QK RMSNorm + (M-)RoPE + quantised store into the 8-bit paged KV cache");
  m.def("kv8_read", &kv8_read, "rows of the 8-bit paged KV cache by slot, as bf16");
  m.def("kv8_attention", &kv8_attention, "paged GQA attention over the 8-bit KV cache (decode: cu_q None)");
  m.def("kv8_chunk_form", &kv8_chunk_form, "the form that kv8_attention takes for a chunk batch of these sizes");
}
