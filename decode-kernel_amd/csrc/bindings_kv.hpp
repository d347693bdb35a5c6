// The torch view of include/decode_kernel/dk_kv.h: checks, allocation of
// outputs and workspaces (caching allocator) and dispatch on the current
// stream. Included by bindings.cpp, whose check_status and current_stream it
// uses.
#pragma once

#include <optional>
#include <tuple>

#include "decode_kernel/dk_kv.h"

namespace {

dk_kv_cache kv_cache(const torch::Tensor& kc, const torch::Tensor& vc, const torch::Tensor& ks,
                     const torch::Tensor& vs) {
  TORCH_CHECK(kc.is_cuda() && vc.device() == kc.device() && ks.device() == kc.device() &&
                  vs.device() == kc.device(),
              "the cache must be CUDA tensors on one device");
  TORCH_CHECK(kc.scalar_type() == torch::kInt8 && vc.scalar_type() == torch::kInt8,
              "the cache's codes must be int8");
  TORCH_CHECK(ks.scalar_type() == torch::kFloat32 && vs.scalar_type() == torch::kFloat32,
              "the cache's scales must be fp32");
  TORCH_CHECK(kc.dim() == 5 && kc.size(4) == 16,
              "k_codes must be [pages, heads, head_size/16, page_size, 16]");
  const int64_t N = kc.size(0), H = kc.size(1), D = kc.size(2) * 16, P = kc.size(3);
  TORCH_CHECK(vc.dim() == 4 && vc.size(0) == N && vc.size(1) == H && vc.size(2) == D &&
                  vc.size(3) == P,
              "v_codes must be [pages, heads, head_size, page_size]");
  TORCH_CHECK(ks.dim() == 2 && ks.size(0) == N && ks.size(1) == H && ks.sizes() == vs.sizes(),
              "k_scales and v_scales must be [pages, heads]");
  TORCH_CHECK(kc.is_contiguous() && vc.is_contiguous() && ks.is_contiguous() && vs.is_contiguous(),
              "the cache must be contiguous");
  TORCH_CHECK(N <= INT32_MAX && H >= 1 && H <= 65535, "the cache needs 1..65535 heads");
  return {kc.data_ptr<int8_t>(), vc.data_ptr<int8_t>(), ks.data_ptr<float>(), vs.data_ptr<float>(),
          static_cast<int>(N), static_cast<int>(H), static_cast<int>(D), static_cast<int>(P)};
}

int kv_dtype(torch::ScalarType t, const char* what) {
  TORCH_CHECK(t == torch::kFloat16 || t == torch::kBFloat16, what, " must be fp16 or bf16");
  return t == torch::kBFloat16 ? DK_KV_BF16 : DK_KV_F16;
}

// The kernels load 16 bytes of a head at a time: a slice of a fused
// projection is read in place, anything odder through a contiguous copy.
torch::Tensor kv_rows(const torch::Tensor& t) {
  const bool ok = t.stride(2) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  if (ok || t.numel() == 0) return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

const int32_t* kv_ints(const torch::Tensor& t, int64_t n, const torch::Device& device,
                       const char* what) {
  TORCH_CHECK(t.device() == device, what, " must be on the same device");
  TORCH_CHECK(t.scalar_type() == torch::kInt32 && t.dim() == 1 && t.size(0) == n &&
                  t.is_contiguous(),
              what, " must be a contiguous int32 [", n, "] tensor");
  return t.data_ptr<int32_t>();
}

const int64_t* kv_slots(const torch::Tensor& t, int64_t n, const torch::Device& device) {
  TORCH_CHECK(t.device() == device, "slots must be on the same device");
  TORCH_CHECK(t.scalar_type() == torch::kInt64 && t.dim() == 1 && t.size(0) == n &&
                  t.is_contiguous(),
              "slots must be a contiguous int64 [tokens] tensor");
  return t.data_ptr<int64_t>();
}

int32_t* kv_tables(const torch::Tensor& t, const torch::Device& device) {
  TORCH_CHECK(t.device() == device, "block_tables must be on the same device");
  TORCH_CHECK(t.scalar_type() == torch::kInt32 && t.dim() == 2 && t.is_contiguous(),
              "block_tables must be a contiguous int32 [requests, width] tensor");
  TORCH_CHECK(t.size(0) <= INT32_MAX && t.size(1) <= INT32_MAX,
              "block_tables' sizes must fit in int32");
  return t.data_ptr<int32_t>();
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> kv_plan(
    torch::Tensor tables, const torch::Tensor& held, const torch::Tensor& added,
    const torch::Tensor& free_pages, const torch::Tensor& free_count, int64_t page_size,
    int64_t num_tokens) {
  TORCH_CHECK(tables.is_cuda(), "block_tables must be a CUDA tensor");
  const auto device = tables.device();
  int32_t* tp = kv_tables(tables, device);
  const int64_t B = tables.size(0), W = tables.size(1);
  TORCH_CHECK(num_tokens >= 0 && num_tokens <= INT32_MAX, "num_tokens must be in [0, 2^31)");
  TORCH_CHECK(page_size >= 0 && page_size <= INT32_MAX, "page_size must be 16, 32, 64 or 128");
  const int32_t* hp = kv_ints(held, B, device, "held");
  const int32_t* ap = kv_ints(added, B, device, "added");
  const int32_t* fp = kv_ints(free_pages, free_pages.numel(), device, "free_pages");
  TORCH_CHECK(free_pages.numel() <= INT32_MAX, "free_pages' size must fit in int32");
  const int32_t* cp = kv_ints(free_count, 1, device, "free_count");
  c10::DeviceGuard guard(device);
  // One allocation for all five, each from a multiple of 16 bytes: a plan takes
  // as long as its host work does, 5.2 us a call so and 7.0 with five.
  auto up = [](int64_t n) { return (n + 3) / 4 * 4; };
  const int64_t at_positions = 2 * up(num_tokens), at_offsets = at_positions + up(num_tokens),
                at_lens = at_offsets + up(B + 1), at_count = at_lens + up(B);
  const auto all = torch::empty({at_count + 4}, tables.options());
  auto part = [&](int64_t at, int64_t n, torch::ScalarType type) {
    auto t = at::detail::make_tensor<c10::TensorImpl>(
        c10::Storage(all.storage()), all.key_set(),
        c10::scalarTypeToTypeMeta(type));
    t.unsafeGetTensorImpl()->set_storage_offset(at);
    t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
    return t;
  };
  auto slots = part(0, num_tokens, torch::kInt64);
  auto positions = part(at_positions, num_tokens, torch::kInt32);
  auto offsets = part(at_offsets, B + 1, torch::kInt32);
  auto lens = part(at_lens, B, torch::kInt32);
  auto count = part(at_count, 1, torch::kInt32);
  check_status(dk_kv_plan(tp, static_cast<int>(W), hp, ap, static_cast<int>(B), fp,
                          static_cast<int>(free_pages.numel()), cp, static_cast<int>(page_size),
                          static_cast<int>(num_tokens), slots.data_ptr<int64_t>(),
                          positions.data_ptr<int32_t>(), offsets.data_ptr<int32_t>(),
                          lens.data_ptr<int32_t>(), count.data_ptr<int32_t>(),
                          current_stream(tables)),
               "plan_kv_step");
  return {slots, positions, offsets, lens, count};
}

void kv_append(torch::Tensor kc, torch::Tensor vc, torch::Tensor ks, torch::Tensor vs,
               const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& slots) {
  const dk_kv_cache cache = kv_cache(kc, vc, ks, vs);
  TORCH_CHECK(k.device() == kc.device() && v.device() == kc.device(),
              "k and v must be on the cache's device");
  TORCH_CHECK(k.scalar_type() == v.scalar_type(), "k and v must have one type");
  const int dtype = kv_dtype(k.scalar_type(), "k and v");
  TORCH_CHECK(k.dim() == 3 && k.sizes() == v.sizes() && k.size(1) == cache.heads &&
                  k.size(2) == cache.head_size,
              "k and v must be [tokens, ", cache.heads, ", ", cache.head_size, "]");
  TORCH_CHECK(k.size(0) <= INT32_MAX, "the number of tokens must fit in int32");
  const int64_t* sp = kv_slots(slots, k.size(0), kc.device());
  c10::DeviceGuard guard(kc.device());
  const auto kr = kv_rows(k), vr = kv_rows(v);
  check_status(dk_kv_append(&cache, kr.data_ptr(), vr.data_ptr(), dtype, kr.stride(0),
                            kr.stride(1), vr.stride(0), vr.stride(1), sp,
                            static_cast<int>(k.size(0)), current_stream(kc)),
               "append_kv");
}

std::tuple<torch::Tensor, torch::Tensor> kv_read(const torch::Tensor& kc, const torch::Tensor& vc,
                                                 const torch::Tensor& ks, const torch::Tensor& vs,
                                                 const torch::Tensor& slots, int dtype) {
  const dk_kv_cache cache = kv_cache(kc, vc, ks, vs);
  TORCH_CHECK(dtype == DK_KV_F16 || dtype == DK_KV_BF16 || dtype == DK_KV_F32,
              "dtype must be fp16, bf16 or fp32");
  const int64_t n = slots.numel();
  TORCH_CHECK(n <= INT32_MAX, "the number of slots must fit in int32");
  const int64_t* sp = kv_slots(slots, n, kc.device());
  c10::DeviceGuard guard(kc.device());
  const auto type = dtype == DK_KV_F16 ? torch::kFloat16
                    : dtype == DK_KV_BF16 ? torch::kBFloat16
                                          : torch::kFloat32;
  auto k = torch::empty({n, cache.heads, cache.head_size}, kc.options().dtype(type));
  auto v = torch::empty_like(k);
  check_status(dk_kv_read(&cache, sp, static_cast<int>(n), dtype, k.data_ptr(), v.data_ptr(),
                          current_stream(kc)),
               "read_kv");
  return {k, v};
}

torch::Tensor kv_attend(const torch::Tensor& q, const torch::Tensor& kc, const torch::Tensor& vc,
                        const torch::Tensor& ks, const torch::Tensor& vs,
                        const torch::Tensor& tables, const torch::Tensor& seq_lens,
                        const std::optional<torch::Tensor>& query_offsets, int64_t max_query_len,
                        double scale, bool causal) {
  const dk_kv_cache cache = kv_cache(kc, vc, ks, vs);
  const auto device = kc.device();
  TORCH_CHECK(q.device() == device, "q must be on the cache's device");
  const int dtype = kv_dtype(q.scalar_type(), "q");
  TORCH_CHECK(q.dim() == 3 && q.size(2) == cache.head_size, "q must be [tokens, q_heads, ",
              cache.head_size, "]");
  const int64_t T = q.size(0), Hq = q.size(1);
  TORCH_CHECK(Hq >= 1 && Hq % cache.heads == 0,
              "q's heads must be a multiple of the cache's ", cache.heads);
  TORCH_CHECK(T <= INT32_MAX && Hq <= INT32_MAX, "q's sizes must fit in int32");
  const int32_t* tp = kv_tables(tables, device);
  const int64_t B = tables.size(0);
  const int32_t* lp = kv_ints(seq_lens, B, device, "seq_lens");
  const int32_t* op = query_offsets ? kv_ints(*query_offsets, B + 1, device, "query_offsets") : nullptr;
  TORCH_CHECK(max_query_len >= 1, "max_query_len must be >= 1");
  max_query_len = std::min<int64_t>(max_query_len, INT32_MAX);
  c10::DeviceGuard guard(device);
  auto out = torch::empty({T, Hq, cache.head_size}, q.options());
  const auto qr = kv_rows(q);
  const size_t ws_bytes = dk_kv_attend_workspace_bytes(
      static_cast<int>(T), static_cast<int>(B), static_cast<int>(Hq), cache.heads, cache.head_size,
      static_cast<int>(tables.size(1)), cache.page_size, static_cast<int>(max_query_len));
  auto ws = torch::empty({static_cast<int64_t>(ws_bytes)}, q.options().dtype(torch::kUInt8));
  check_status(dk_kv_attend(qr.data_ptr(), dtype, qr.stride(0), qr.stride(1), &cache, tp,
                            static_cast<int>(tables.size(1)), lp, op, static_cast<int>(T),
                            static_cast<int>(B), static_cast<int>(Hq),
                            static_cast<int>(max_query_len), static_cast<float>(scale),
                            causal ? 1 : 0, out.data_ptr(), ws.data_ptr(), ws_bytes,
                            current_stream(kc)),
               "attend_kv");
  return out;
}

}  // namespace

void define_kv(pybind11::module_& m) {
  m.def("plan_kv_step", &kv_plan, "Pages and slots of a step's new tokens",
        py::arg("block_tables"), py::arg("held"), py::arg("added"), py::arg("free_pages"),
        py::arg("free_count"), py::arg("page_size"), py::arg("num_tokens"));
  m.def("append_kv", &kv_append, "Quantise k and v into the cache's pages at slots",
        py::arg("k_codes"), py::arg("v_codes"), py::arg("k_scales"), py::arg("v_scales"),
        py::arg("k"), py::arg("v"), py::arg("slots"));
  m.def("read_kv", &kv_read, "The cache's values at slots", py::arg("k_codes"),
        py::arg("v_codes"), py::arg("k_scales"), py::arg("v_scales"), py::arg("slots"),
        py::arg("dtype"));
  m.def("attend_kv", &kv_attend, "Attention over the cache", py::arg("q"), py::arg("k_codes"),
        py::arg("v_codes"), py::arg("k_scales"), py::arg("v_scales"), py::arg("block_tables"),
        py::arg("seq_lens"), py::arg("query_offsets"), py::arg("max_query_len"), py::arg("scale"),
        py::arg("causal"));
}
