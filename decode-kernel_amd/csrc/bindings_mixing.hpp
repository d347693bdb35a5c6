// The torch view of include/decode_kernel/dk_delta.h and dk_rotary.h: checks,
// allocation of outputs and workspaces (caching allocator) and dispatch on the
// current stream. Included by bindings.cpp after bindings_kv.hpp, whose checks
// it uses.
#pragma once

#include "decode_kernel/dk_delta.h"
#include "decode_kernel/dk_rotary.h"

namespace {

// Requests of a call, with the checks that delta_rule and short_conv share.
void check_requests(int64_t tokens, int64_t requests, const std::optional<torch::Tensor>& offsets,
                    int64_t max_query_len) {
  TORCH_CHECK(tokens <= INT32_MAX && requests <= INT32_MAX, "the number of tokens must fit in int32");
  TORCH_CHECK(offsets || tokens == requests,
              "without query_offsets each request has one token: ", requests, " rows are needed, not ", tokens);
  TORCH_CHECK(max_query_len >= 1, "max_query_len must be >= 1");
}

const float* gates(const torch::Tensor& t, int64_t tokens, int64_t heads, const torch::Device& device,
                   const char* what) {
  TORCH_CHECK(t.device() == device, what, " must be on the same device");
  TORCH_CHECK(t.scalar_type() == torch::kFloat32 && t.dim() == 2 && t.size(0) == tokens &&
                  t.size(1) == heads && t.is_contiguous(),
              what, " must be a contiguous fp32 [", tokens, ", ", heads, "] tensor");
  return t.data_ptr<float>();
}

torch::Tensor delta_rule(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v,
                         const torch::Tensor& log_decay, const torch::Tensor& beta, torch::Tensor states,
                         const std::optional<torch::Tensor>& held,
                         const std::optional<torch::Tensor>& offsets, int64_t max_query_len, double scale,
                         bool normalize) {
  TORCH_CHECK(states.is_cuda(), "states must be a CUDA tensor");
  const auto device = states.device();
  TORCH_CHECK(q.device() == device && k.device() == device && v.device() == device,
              "q, k and v must be on the states' device");
  TORCH_CHECK(states.scalar_type() == torch::kFloat32 && states.dim() == 4 && states.is_contiguous(),
              "states must be a contiguous fp32 [requests, v_heads, key_size, value_size] tensor");
  TORCH_CHECK(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(),
              "q, k and v must have one type");
  const int64_t B = states.size(0), Hv = states.size(1), dk = states.size(2), dv = states.size(3);
  TORCH_CHECK(q.dim() == 3 && q.sizes() == k.sizes() && q.size(2) == dk,
              "q and k must be [tokens, qk_heads, ", dk, "]");
  const int64_t T = q.size(0), H = q.size(1);
  TORCH_CHECK(v.dim() == 3 && v.size(0) == T && v.size(1) == Hv && v.size(2) == dv, "v must be [", T, ", ",
              Hv, ", ", dv, "]");
  TORCH_CHECK(H >= 1 && Hv >= 1 && Hv <= 65535 && Hv % H == 0,
              "the states' heads (1..65535) must be a multiple of q's and k's ", H);
  check_requests(T, B, offsets, max_query_len);
  dk_delta_args a;
  a.dtype = kv_dtype(q.scalar_type(), "q, k and v");
  a.log_decay = gates(log_decay, T, Hv, device, "log_decay");
  a.beta = gates(beta, T, Hv, device, "beta");
  a.held = held ? kv_ints(*held, B, device, "held") : nullptr;
  a.offsets = offsets ? kv_ints(*offsets, B + 1, device, "query_offsets") : nullptr;
  c10::DeviceGuard guard(device);
  auto out = torch::empty({T, Hv, dv}, v.options());
  auto rows = [](const torch::Tensor& t) {  // rows too far apart to be counted in 32 bits are copied, too
    return t.stride(0) > 1 << 24 ? t.clone(at::MemoryFormat::Contiguous) : kv_rows(t);
  };
  const auto qr = rows(q), kr = rows(k), vr = rows(v);
  a.q = qr.data_ptr();
  a.k = kr.data_ptr();
  a.v = vr.data_ptr();
  a.q_token_stride = qr.stride(0);
  a.q_head_stride = qr.stride(1);
  a.k_token_stride = kr.stride(0);
  a.k_head_stride = kr.stride(1);
  a.v_token_stride = vr.stride(0);
  a.v_head_stride = vr.stride(1);
  a.states = states.data_ptr<float>();
  a.num_tokens = static_cast<int>(T);
  a.requests = static_cast<int>(B);
  a.qk_heads = static_cast<int>(H);
  a.v_heads = static_cast<int>(Hv);
  a.key_size = static_cast<int>(dk);
  a.value_size = static_cast<int>(dv);
  a.max_query_len = static_cast<int>(std::min<int64_t>(max_query_len, INT32_MAX));
  a.normalize = normalize ? 1 : 0;
  a.scale = static_cast<float>(scale);
  const size_t ws_bytes =
      a.offsets ? dk_delta_workspace_bytes(a.num_tokens, a.requests, a.qk_heads, a.v_heads, a.key_size,
                                           a.max_query_len)
                : 0;
  torch::Tensor ws;
  if (ws_bytes > 0) ws = torch::empty({static_cast<int64_t>(ws_bytes)}, v.options().dtype(torch::kUInt8));
  check_status(dk_delta_rule(&a, out.data_ptr(), ws_bytes ? ws.data_ptr() : nullptr, ws_bytes,
                             current_stream(states)),
               "delta_rule");
  return out;
}

torch::Tensor short_conv(const torch::Tensor& x, const torch::Tensor& weight, torch::Tensor windows,
                         const std::optional<torch::Tensor>& held,
                         const std::optional<torch::Tensor>& offsets, int64_t max_query_len,
                         const std::optional<torch::Tensor>& bias, bool silu) {
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
  const auto device = x.device();
  TORCH_CHECK(weight.device() == device && windows.device() == device && (!bias || bias->device() == device),
              "weight, windows and bias must be on x's device");
  const int dtype = kv_dtype(x.scalar_type(), "x");
  TORCH_CHECK(weight.scalar_type() == x.scalar_type() && windows.scalar_type() == x.scalar_type() &&
                  (!bias || bias->scalar_type() == x.scalar_type()),
              "weight, windows and bias must have x's type");
  TORCH_CHECK(x.dim() == 2 && weight.dim() == 2 && weight.size(0) == x.size(1),
              "x must be [tokens, channels] and weight [channels, width]");
  const int64_t T = x.size(0), C = x.size(1), W = weight.size(1);
  TORCH_CHECK(W >= 2 && W <= 4, "width=", W, " must be 2, 3 or 4");
  TORCH_CHECK(windows.dim() == 3 && windows.size(1) == W - 1 && windows.size(2) == C && windows.is_contiguous(),
              "windows must be a contiguous [requests, ", W - 1, ", ", C, "] tensor");
  TORCH_CHECK(!bias || (bias->dim() == 1 && bias->size(0) == C && bias->is_contiguous()),
              "bias must be a contiguous [", C, "] tensor");
  TORCH_CHECK(weight.is_contiguous(), "weight must be contiguous");
  TORCH_CHECK(C <= INT32_MAX, "the number of channels must fit in int32");
  const int64_t B = windows.size(0);
  check_requests(T, B, offsets, max_query_len);
  const int32_t* hp = held ? kv_ints(*held, B, device, "held") : nullptr;
  const int32_t* op = offsets ? kv_ints(*offsets, B + 1, device, "query_offsets") : nullptr;
  c10::DeviceGuard guard(device);
  auto y = torch::empty({T, C}, x.options());
  const auto rows = x.stride(1) == 1 || x.numel() == 0 ? x : x.clone(at::MemoryFormat::Contiguous);
  check_status(dk_short_conv(rows.data_ptr(), rows.stride(0), weight.data_ptr(),
                             bias ? bias->data_ptr() : nullptr, windows.data_ptr(), hp, op, dtype,
                             static_cast<int>(T), static_cast<int>(B), static_cast<int>(C),
                             static_cast<int>(W), static_cast<int>(std::min<int64_t>(max_query_len, INT32_MAX)),
                             silu ? 1 : 0, y.data_ptr(), current_stream(x)),
               "short_conv");
  return y;
}

std::tuple<torch::Tensor, torch::Tensor> rotate_qk(const torch::Tensor& q, const torch::Tensor& k,
                                                   const torch::Tensor& positions,
                                                   const torch::Tensor& frequencies,
                                                   const std::optional<torch::Tensor>& axes, bool adjacent,
                                                   bool inverse) {
  TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
  const auto device = q.device();
  TORCH_CHECK(k.device() == device && positions.device() == device && frequencies.device() == device &&
                  (!axes || axes->device() == device),
              "k, positions, frequencies and axes must be on q's device");
  const int dtype = kv_dtype(q.scalar_type(), "q and k");
  TORCH_CHECK(k.scalar_type() == q.scalar_type(), "q and k must have one type");
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && k.size(0) == q.size(0) && k.size(2) == q.size(2),
              "q and k must be [tokens, heads, head_size]");
  const int64_t T = q.size(0), D = q.size(2), F = frequencies.numel();
  TORCH_CHECK(T <= INT32_MAX && q.size(1) <= 65535 && k.size(1) <= 65535, "q and k are too large");
  TORCH_CHECK(D <= DK_ROTARY_MAX_HEAD_SIZE, "head_size=", D, " must be at most ", DK_ROTARY_MAX_HEAD_SIZE);
  TORCH_CHECK(frequencies.scalar_type() == torch::kFloat32 && frequencies.dim() == 1 &&
                  frequencies.is_contiguous() && 2 * F <= D && F <= DK_ROTARY_MAX_FREQUENCIES,
              "frequencies must be a contiguous fp32 tensor of at most head_size / 2 = ", D / 2, " (and ",
              DK_ROTARY_MAX_FREQUENCIES, ")");
  const bool wide = positions.scalar_type() == torch::kInt64;
  TORCH_CHECK((wide || positions.scalar_type() == torch::kInt32) && positions.is_contiguous() &&
                  ((positions.dim() == 1 && positions.size(0) == T) ||
                   (positions.dim() == 2 && positions.size(0) >= 1 && positions.size(0) <= INT32_MAX &&
                    positions.size(1) == T)),
              "positions must be a contiguous int32 or int64 [tokens] or [axes, tokens] tensor");
  const int64_t A = positions.dim() == 2 ? positions.size(0) : 1;
  TORCH_CHECK(axes || A == 1, "positions of ", A, " axes need the axis of each frequency");
  const int32_t* ap = axes ? kv_ints(*axes, F, device, "axes") : nullptr;
  c10::DeviceGuard guard(device);
  // The last dimension has to be contiguous; anything odder is copied first.
  auto rows = [](const torch::Tensor& t) {
    return t.stride(2) == 1 || t.numel() == 0 ? t : t.clone(at::MemoryFormat::Contiguous);
  };
  const auto qr = rows(q), kr = rows(k);
  // One allocation for both, k's part from a multiple of 16 bytes: a decode step
  // takes as long as its host work does.
  const int64_t k_at = (q.numel() + 7) / 8 * 8;
  auto qo = torch::empty({k_at + k.numel()}, q.options());
  auto ko = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(qo.storage()), qo.key_set(), qo.dtype());
  ko.unsafeGetTensorImpl()->set_storage_offset(k_at);
  ko.unsafeGetTensorImpl()->set_sizes_contiguous(k.sizes());
  qo.unsafeGetTensorImpl()->set_sizes_contiguous(q.sizes());
  if (D == 0) return {qo, ko};
  check_status(
      dk_rotate_qk(qr.data_ptr(), qr.stride(0), qr.stride(1), static_cast<int>(q.size(1)), kr.data_ptr(),
                   kr.stride(0), kr.stride(1), static_cast<int>(k.size(1)), dtype, static_cast<int>(D),
                   static_cast<int>(T), positions.data_ptr(), wide ? 1 : 0, static_cast<int>(A),
                   frequencies.data_ptr<float>(), ap, static_cast<int>(F), adjacent ? 1 : 0, inverse ? 1 : 0,
                   qo.data_ptr(), ko.data_ptr(), current_stream(q)),
      "rotate_qk");
  return {qo, ko};
}

}  // namespace

void define_mixing(pybind11::module_& m) {
  m.def("delta_rule", &delta_rule, "The gated delta rule over each request's tokens", py::arg("q"),
        py::arg("k"), py::arg("v"), py::arg("log_decay"), py::arg("beta"), py::arg("states"), py::arg("held"),
        py::arg("query_offsets"), py::arg("max_query_len"), py::arg("scale"), py::arg("normalize"));
  m.def("short_conv", &short_conv, "The causal convolution over each request's tokens", py::arg("x"),
        py::arg("weight"), py::arg("windows"), py::arg("held"), py::arg("query_offsets"),
        py::arg("max_query_len"), py::arg("bias"), py::arg("silu"));
  m.def("rotate_qk", &rotate_qk, "Rotary positions of queries and keys", py::arg("q"), py::arg("k"),
        py::arg("positions"), py::arg("frequencies"), py::arg("axes"), py::arg("adjacent"),
        py::arg("inverse"));
}
