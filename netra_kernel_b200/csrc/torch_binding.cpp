// torch side of the dense FP8 and balance-loss entry points: argument checks, output and workspace tensors, autograd.
//
// These operators are called once per layer and step from eager Python on shapes whose kernels take a few microseconds, so
// the host's share decides what a call costs: the same path through ctypes took 26 us per fp8_linear call and 130 us with its
// gradient (Python autograd function).  Everything below the C ABI of include/netra_moe.h is unchanged; C callers need none of this.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <tuple>
#include <unordered_set>
#include <vector>

#include "../../include/netra_moe.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kBlockCols = 128;
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

uint32_t element_code(at::ScalarType t) { return t == at::kBFloat16 ? 0u : t == at::kHalf ? 1u : 2u; }
bool is_activation(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf || t == at::kFloat; }

void check_rc(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed (code ", rc, "): ", netra_moe_last_error()); }

cudaStream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// The kernels compute no tangents; an output without one would count as a constant in forward-mode differentiation.
void refuse_tangent(const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), "forward-mode derivatives are not supported: an operand carries a tangent");
}

// x as a matrix whose rows the kernels can walk: unit column stride, rows that do not overlap
Tensor as_rows(const Tensor& x, const char* what) {
  TORCH_CHECK_VALUE(x.is_cuda(), what, " must be a CUDA tensor");
  TORCH_CHECK_VALUE(is_activation(x.scalar_type()), what, " must be bfloat16, float16 or float32");
  TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0, what, " must have at least one column");
  Tensor r = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  if ((r.stride(1) != 1 && r.size(1) > 1) || (r.stride(0) < r.size(1) && r.size(0) > 1)) r = r.contiguous();
  return r;
}

// element pitches the C ABI accepts: a single row may report any stride
uint64_t pitch_of(const Tensor& t) { return (uint64_t)std::max(t.stride(0), t.size(1)); }
uint64_t code_pitch_of(const Tensor& t) { return (uint64_t)(t.size(0) > 1 ? t.stride(0) : ceil_div(t.size(1), 16) * 16); }

constexpr int64_t kMaxSize = 1 << 26;

void check_weight(const Tensor& w, const Tensor& s, const at::Device& device) {
  TORCH_CHECK_VALUE(w.device() == device && s.device() == device, "weight and weight_scale must be on the activations' device");
  TORCH_CHECK_VALUE(w.scalar_type() == at::kFloat8_e4m3fn && w.dim() == 2 && w.numel() > 0, "weight must be float8_e4m3fn [N, K]");
  const int64_t n = w.size(0), k = w.size(1);
  TORCH_CHECK_VALUE((w.stride(1) == 1 || k == 1) && (n == 1 || (w.stride(0) % 16 == 0 && w.stride(0) >= k)) && (uintptr_t)w.const_data_ptr() % 16 == 0,
                    "weight rows must be contiguous and start on 16-byte boundaries");
  TORCH_CHECK_VALUE(s.scalar_type() == at::kFloat && s.dim() == 2 && s.size(0) == ceil_div(n, kBlockCols) && s.size(1) == ceil_div(k, kBlockCols),
                    "weight_scale must be float32 [ceil(N/128), ceil(K/128)]");
  TORCH_CHECK_VALUE((s.stride(1) == 1 || s.size(1) == 1) && (s.stride(0) >= s.size(1) || s.size(0) == 1), "weight_scale must be row-major");
  refuse_tangent(w);
  refuse_tangent(s);
  TORCH_CHECK_VALUE(!w.requires_grad() && !s.requires_grad(), "the FP8 weight is frozen: it cannot require a gradient");
}

void check_weight_on(const Tensor& w, const Tensor& s, const at::Device& device) { check_weight(w, s, device); }

std::tuple<Tensor, Tensor> quantize_rows(const Tensor& input) {
  refuse_tangent(input);
  const Tensor x = as_rows(input.detach(), "x");
  TORCH_CHECK_VALUE(x.size(0) <= kMaxSize && x.size(1) <= kMaxSize, "sizes must not exceed 2^26");
  const int64_t m = x.size(0), k = x.size(1), blocks = ceil_div(k, kBlockCols), pitch = blocks * kBlockCols;
  Tensor codes = at::empty_strided({m, k}, {pitch, 1}, x.options().dtype(at::kFloat8_e4m3fn));
  Tensor scale = at::empty_strided({m, blocks}, {1, std::max<int64_t>(m, 1)}, x.options().dtype(at::kFloat));
  if (m > 0) {
    const c10::cuda::CUDAGuard guard(x.device());
    check_rc(netra_dense_quantize_rows_launch(codes.data_ptr(), pitch, scale.data_ptr<float>(), 1, m, x.const_data_ptr(), element_code(x.scalar_type()),
                                              pitch_of(x), (uint32_t)m, (uint32_t)k, stream_of(x)),
             "dense_quantize_rows_launch");
  }
  return {codes, scale};
}

void check_sizes(int64_t m, const Tensor& w) {
  TORCH_CHECK_VALUE(m <= kMaxSize && w.size(0) <= kMaxSize && w.size(1) <= kMaxSize, "sizes must not exceed 2^26");
}

Tensor block_scaled_matmul(const Tensor& a, const Tensor& a_scale, const Tensor& w, const Tensor& ws, bool transpose_weight,
                           at::ScalarType out_dtype, const std::optional<Tensor>& out_given) {
  TORCH_CHECK_VALUE(a.is_cuda() && a.scalar_type() == at::kFloat8_e4m3fn && a.dim() == 2, "a must be a float8_e4m3fn CUDA matrix");
  check_weight(w, ws, a.device());
  TORCH_CHECK_VALUE(!at::GradMode::is_enabled() || !(a.requires_grad() || a_scale.requires_grad()),
                    "a product of ready codes carries no gradient, so a and a_scale must not require one (fp8_linear differentiates)");
  refuse_tangent(a);
  refuse_tangent(a_scale);
  const int64_t m = a.size(0), k = w.size(transpose_weight ? 0 : 1), n = w.size(transpose_weight ? 1 : 0);
  check_sizes(m, w);
  TORCH_CHECK_VALUE(a.size(1) == k, "a has ", a.size(1), " columns, the weight reduces over ", k);
  TORCH_CHECK_VALUE(a_scale.device() == a.device() && a_scale.scalar_type() == at::kFloat && a_scale.dim() == 2 && a_scale.size(0) == m &&
                        a_scale.size(1) == ceil_div(k, kBlockCols), "a_scale must be float32 [M, ceil(K/128)] on a's device");
  TORCH_CHECK_VALUE((a.stride(1) == 1 || k == 1) && (m <= 1 || (a.stride(0) % 16 == 0 && a.stride(0) >= k)) && (uintptr_t)a.const_data_ptr() % 16 == 0,
                    "the rows of a must be contiguous and start on 16-byte boundaries");
  Tensor out;
  if (out_given.has_value()) {
    out = *out_given;
    refuse_tangent(out);
    TORCH_CHECK_VALUE(out.device() == a.device() && is_activation(out.scalar_type()) && out.dim() == 2 && out.size(0) == m && out.size(1) == n &&
                          (out.stride(1) == 1 || n == 1) && (out.stride(0) >= n || m <= 1) && !out.requires_grad(),
                      "out must be a row-major [M, N] matrix of BF16, FP16 or FP32 on a's device");
    for (const Tensor* operand : {&a, &a_scale, &w, &ws}) {        // as far as torch can tell without walking strided views
      const auto overlap = at::get_overlap_status(out, *operand);
      TORCH_CHECK_VALUE(overlap != at::MemOverlapStatus::Full && overlap != at::MemOverlapStatus::Partial, "out must not share memory with an operand");
    }
  } else {
    TORCH_CHECK_VALUE(is_activation(out_dtype), "out_dtype must be bfloat16, float16 or float32");
    out = at::empty({m, n}, a.options().dtype(out_dtype));
  }
  if (m > 0) {
    const c10::cuda::CUDAGuard guard(a.device());
    check_rc(netra_dense_fp8_matmul_launch(out.data_ptr(), element_code(out.scalar_type()), pitch_of(out), a.const_data_ptr(), code_pitch_of(a),
                                           a_scale.const_data_ptr<float>(), a_scale.stride(0), a_scale.stride(1), w.const_data_ptr(), code_pitch_of(w),
                                           ws.const_data_ptr<float>(), pitch_of(ws), transpose_weight, (uint32_t)m, (uint32_t)w.size(0),
                                           (uint32_t)w.size(1), stream_of(a)),
             "dense_fp8_matmul_launch");
    // written in place: autograd may have saved it for some backward pass (an inference tensor it cannot)
    if (out_given.has_value() && !out.is_inference()) torch::autograd::impl::bump_version(out);
  }
  return out;
}

Tensor linear(const Tensor& input, const Tensor& w, const Tensor& ws, bool transposed) {
  refuse_tangent(input);
  const Tensor x = as_rows(input, "x");
  const int64_t m = x.size(0), k = w.size(transposed ? 0 : 1), n = w.size(transposed ? 1 : 0);
  check_sizes(m, w);
  auto shape = input.sizes().vec();
  shape.back() = n;
  Tensor out = at::empty(shape, x.options());          // not a view of a matrix, which autograd would not let a caller modify in place
  if (m > 0) {
    const c10::cuda::CUDAGuard guard(x.device());
    uint64_t bytes = 0;
    Tensor workspace;
    if (netra_dense_fp8_linear_needs_workspace(x.const_data_ptr(), element_code(x.scalar_type()), pitch_of(x), transposed, (uint32_t)m, (uint32_t)k)) {
      bytes = netra_dense_fp8_linear_workspace_bytes((uint32_t)m, (uint32_t)k);
      workspace = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    }
    check_rc(netra_dense_fp8_linear_launch(out.data_ptr(), n, x.const_data_ptr(), element_code(x.scalar_type()), pitch_of(x), w.const_data_ptr(),
                                           code_pitch_of(w), ws.const_data_ptr<float>(), pitch_of(ws), transposed, (uint32_t)m, (uint32_t)w.size(0),
                                           (uint32_t)w.size(1), bytes > 0 ? workspace.data_ptr() : nullptr, bytes, stream_of(x)),
             "dense_fp8_linear_launch");
  }
  return out;
}

// The gradients have no derivatives of their own.  A backward pass that is itself being differentiated (create_graph) computes its
// gradient through a node that hangs on everything the gradient depends on and raises once a second derivative reaches it; a
// tensor without that node would count as a constant, and its terms would be missing from a sum without a word.
[[noreturn]] variable_list refuse_second_derivative() { TORCH_CHECK(false, "this gradient cannot be differentiated again"); }

// A leaf keeps its gradient node, with the stream it was made on, for as long as any graph of it lives.  If that was the default
// stream, a backward pass captured on another one makes torch tie the two together, which CUDA forbids and which invalidates the
// capture; so such a call is refused while the capture can still be ended: the forward call of the leaf itself, and, since the leaf
// may lie behind other operations, the operator's step of the backward pass.
bool capturing() { return c10::cuda::device_count() > 0 && c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None; }

void refuse_default_stream(torch::autograd::Node& leaf) {
  const auto made_on = leaf.stream();
  TORCH_CHECK(!made_on.has_value() || made_on->id() != 0 || *made_on == c10::cuda::getCurrentCUDAStream(made_on->device_index()).unwrap(),
              "an eager graph of this leaf, made on the default stream, is still alive: drop it (its loss and outputs) before capturing a "
              "forward and backward pass of the same leaf, or capture with a fresh leaf (or, for the forward pass alone, under torch.no_grad())");
}

void check_capture(const Tensor& x) {
  if (x.grad_fn()) return;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(x);
  if (node && capturing()) refuse_default_stream(*node);
}

// Called in a backward step: looks at every leaf that this backward pass will reach from here.
void check_captured_backward() {
  const auto node = torch::autograd::get_current_node();
  if (!node || !capturing()) return;
  const auto* wanted = torch::autograd::get_current_graph_task_exec_info();       // empty: every node
  std::unordered_set<torch::autograd::Node*> seen;
  std::vector<torch::autograd::Node*> stack{node.get()};
  while (!stack.empty()) {
    const auto* at = stack.back();
    stack.pop_back();
    for (const auto& edge : at->next_edges()) {
      auto* next = edge.function.get();
      if (!next || !seen.insert(next).second) continue;
      if (wanted && !wanted->empty()) {
        const auto it = wanted->find(next);
        if (it == wanted->end() || !it->second.should_execute()) continue;
      }
      if (dynamic_cast<torch::autograd::AccumulateGrad*>(next)) refuse_default_stream(*next);
      stack.push_back(next);
    }
  }
}

struct LinearGradFunction : torch::autograd::Function<LinearGradFunction> {
  static Tensor forward(AutogradContext*, const Tensor& dy, const Tensor& w, const Tensor& ws) { return linear(dy, w, ws, true); }
  static variable_list backward(AutogradContext*, const variable_list&) { return refuse_second_derivative(); }
};

struct LinearFunction : torch::autograd::Function<LinearFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& ws) {
    ctx->save_for_backward({w, ws});
    return linear(x, w, ws, false);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    check_captured_backward();
    const auto saved = ctx->get_saved_variables();
    const Tensor& dy = grads[0];
    return {at::GradMode::is_enabled() ? LinearGradFunction::apply(dy, saved[0], saved[1]) : linear(dy, saved[0], saved[1], true), Tensor(), Tensor()};
  }
};

Tensor fp8_linear(const Tensor& x, const Tensor& w, const Tensor& ws) {
  TORCH_CHECK_VALUE(x.is_cuda(), "x must be a CUDA tensor");
  TORCH_CHECK_VALUE(x.dim() > 0 && w.dim() == 2 && x.size(-1) == w.size(1), "x must have as many columns as the weight");
  check_weight(w, ws, x.device());
  if (x.requires_grad() && at::GradMode::is_enabled()) {
    check_capture(x);
    return LinearFunction::apply(x, w, ws);
  }
  return linear(x, w, ws, false);
}

constexpr int64_t kMaxExperts = 1024;

const uint8_t* mask_of(const std::optional<Tensor>& mask, int64_t tokens, const at::Device& device) {
  if (!mask.has_value() || !mask->defined()) return nullptr;
  TORCH_CHECK_VALUE(mask->scalar_type() == at::kBool && mask->device() == device && mask->dim() == 1 && mask->size(0) == tokens && mask->is_contiguous(),
                    "token_mask must be a contiguous bool [tokens] tensor on the same device (True = counted)");
  return reinterpret_cast<const uint8_t*>(mask->const_data_ptr());
}

Tensor expert_counts(const Tensor& topk_ids, int64_t experts, const std::optional<Tensor>& token_mask) {
  TORCH_CHECK_VALUE(topk_ids.is_cuda() && (topk_ids.scalar_type() == at::kInt || topk_ids.scalar_type() == at::kLong) && topk_ids.dim() == 2,
                    "topk_ids must be an int32 or int64 CUDA matrix [tokens, slots]");
  TORCH_CHECK_VALUE(experts >= 1 && experts <= kMaxExperts, "num_experts must be 1..", kMaxExperts);
  const int64_t tokens = topk_ids.size(0), slots = topk_ids.size(1);
  TORCH_CHECK_VALUE(slots <= kMaxExperts, "topk_ids has more than ", kMaxExperts, " slots");
  const uint8_t* mask = mask_of(token_mask, tokens, topk_ids.device());
  const Tensor ids = (slots > 1 && topk_ids.stride(1) != 1) || (tokens > 1 && topk_ids.stride(0) < slots) ? topk_ids.contiguous() : topk_ids;
  Tensor counts = at::empty({experts}, ids.options().dtype(at::kInt));
  const c10::cuda::CUDAGuard guard(ids.device());
  check_rc(netra_expert_counts_launch(counts.data_ptr<int32_t>(), ids.const_data_ptr(), (uint32_t)ids.element_size(), pitch_of(ids), mask,
                                      (uint64_t)tokens, (uint32_t)slots, (uint32_t)experts, stream_of(ids)),
           "expert_counts_launch");
  return counts;
}

std::tuple<Tensor, Tensor> balance_forward(const Tensor& z, const Tensor& counts, const uint8_t* mask) {
  const int64_t tokens = z.size(0), experts = z.size(1);
  const auto options = z.options().dtype(at::kFloat);
  if (tokens == 0) return {at::zeros({}, options), at::zeros({}, options)};
  Tensor loss = at::empty({}, options), scale = at::empty({}, options);
  const c10::cuda::CUDAGuard guard(z.device());
  const uint64_t bytes = netra_balance_loss_workspace_bytes((uint64_t)tokens, (uint32_t)experts);
  const Tensor workspace = bytes > 0 ? at::empty({(int64_t)bytes}, z.options().dtype(at::kByte)) : Tensor();
  check_rc(netra_balance_loss_launch(loss.data_ptr<float>(), scale.data_ptr<float>(), z.const_data_ptr(), element_code(z.scalar_type()), pitch_of(z),
                                     counts.const_data_ptr<int32_t>(), mask, bytes > 0 ? workspace.data_ptr() : nullptr, bytes, (uint64_t)tokens, (uint32_t)experts,
                                     stream_of(z)),
           "balance_loss_launch");
  return {loss, scale};
}

Tensor balance_backward(const Tensor& z, const Tensor& counts, const uint8_t* mask, const Tensor& scale, const Tensor& upstream) {
  refuse_tangent(upstream);
  const int64_t tokens = z.size(0), experts = z.size(1);
  Tensor grad = at::empty({tokens, experts}, z.options());
  if (tokens > 0) {
    const c10::cuda::CUDAGuard guard(z.device());
    check_rc(netra_balance_loss_grad_launch(grad.data_ptr(), experts, z.const_data_ptr(), element_code(z.scalar_type()), pitch_of(z),
                                            counts.const_data_ptr<int32_t>(), mask, scale.const_data_ptr<float>(), upstream.const_data_ptr<float>(),
                                            (uint64_t)tokens, (uint32_t)experts, stream_of(z)),
             "balance_loss_grad_launch");
  }
  return grad;
}

const uint8_t* saved_mask(const std::optional<Tensor>& mask) {
  return mask.has_value() && mask->defined() ? reinterpret_cast<const uint8_t*>(mask->const_data_ptr()) : nullptr;
}

struct BalanceGradFunction : torch::autograd::Function<BalanceGradFunction> {
  static Tensor forward(AutogradContext*, const Tensor& upstream, const Tensor& z, const Tensor& counts, const Tensor& scale,
                        const std::optional<Tensor>& mask) {
    return balance_backward(z, counts, saved_mask(mask), scale, upstream);
  }
  static variable_list backward(AutogradContext*, const variable_list&) { return refuse_second_derivative(); }
};

// z: logits as rows the kernels can walk; a copy, where it is one, was made outside, so that z still hangs on them
struct BalanceFunction : torch::autograd::Function<BalanceFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& z, const Tensor& counts, const std::optional<Tensor>& token_mask) {
    auto [loss, scale] = balance_forward(z, counts, saved_mask(token_mask));
    ctx->save_for_backward({z, counts, scale, token_mask.value_or(Tensor())});
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    check_captured_backward();
    const auto saved = ctx->get_saved_variables();
    const Tensor &z = saved[0], &counts = saved[1], &scale = saved[2];
    const auto mask = saved[3].defined() ? std::optional<Tensor>(saved[3]) : std::nullopt;
    return {at::GradMode::is_enabled() ? BalanceGradFunction::apply(grads[0], z, counts, scale, mask)
                                       : balance_backward(z, counts, saved_mask(mask), scale, grads[0]),
            Tensor(), Tensor()};
  }
};

const uint8_t* check_balance(const Tensor& logits, const Tensor& counts, const std::optional<Tensor>& token_mask) {
  TORCH_CHECK_VALUE(logits.is_cuda() && logits.dim() == 2 && is_activation(logits.scalar_type()),
                    "logits must be a BF16, FP16 or FP32 CUDA matrix [tokens, experts]");
  refuse_tangent(logits);
  const int64_t tokens = logits.size(0), experts = logits.size(1);
  TORCH_CHECK_VALUE(experts >= 1 && experts <= kMaxExperts, "experts must be 1..", kMaxExperts);
  TORCH_CHECK_VALUE(counts.scalar_type() == at::kInt && counts.device() == logits.device() && counts.dim() == 1 && counts.size(0) == experts &&
                        counts.is_contiguous(), "counts must be a contiguous int32 [experts] tensor on the same device");
  return mask_of(token_mask, tokens, logits.device());
}

// the gradient alone (a traced graph's backward pass): the loss is computed again for its scale
Tensor balance_loss_grad(const Tensor& upstream, const Tensor& logits, const Tensor& counts, const std::optional<Tensor>& token_mask) {
  const uint8_t* mask = check_balance(logits, counts, token_mask);
  TORCH_CHECK_VALUE(upstream.scalar_type() == at::kFloat && upstream.numel() == 1 && upstream.device() == logits.device(),
                    "upstream must be an FP32 scalar on the same device");
  const Tensor z = as_rows(logits.detach(), "logits");
  return balance_backward(z, counts, mask, std::get<1>(balance_forward(z, counts, mask)), upstream);
}

Tensor balance_loss(const Tensor& logits, const Tensor& counts, const std::optional<Tensor>& token_mask) {
  const uint8_t* mask = check_balance(logits, counts, token_mask);
  if (logits.requires_grad() && at::GradMode::is_enabled()) {
    check_capture(logits);
    return BalanceFunction::apply(as_rows(logits, "logits"), counts, token_mask);
  }
  return std::get<0>(balance_forward(as_rows(logits, "logits"), counts, mask));
}

}  // namespace

PYBIND11_MODULE(_netra_torch, m) {
  // argument errors are ValueError, errors of the C ABI RuntimeError; the interpreter lock is released during a call
  m.def("check_weight", torch::wrap_pybind_function_no_gil(check_weight_on));
  m.def("check_captured_backward", torch::wrap_pybind_function_no_gil(check_captured_backward));
  m.def("quantize_rows", torch::wrap_pybind_function_no_gil(quantize_rows));
  m.def("block_scaled_matmul", torch::wrap_pybind_function_no_gil(block_scaled_matmul));
  m.def("fp8_linear", torch::wrap_pybind_function_no_gil(fp8_linear));
  m.def("expert_counts", torch::wrap_pybind_function_no_gil(expert_counts));
  m.def("balance_loss_grad", torch::wrap_pybind_function_no_gil(balance_loss_grad));
  m.def("balance_loss", torch::wrap_pybind_function_no_gil(balance_loss));
}
