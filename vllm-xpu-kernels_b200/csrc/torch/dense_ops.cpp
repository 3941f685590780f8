// The dense layers beside the routed experts: torch.ops._xpu_C.b200_int8_linear, b200_gated_linear,
// b200_gated_linear_backward and, with gradients, b200_gated_product over the C ABI.  No counterpart in the reference, which multiplies dense layers by library calls.
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/variable.h>

#include <unordered_set>

#include "layer.h"

using namespace b200shim;

namespace {

void same_device(const at::Tensor& t, const at::Tensor& input, const char* op, const char* name) {
  TORCH_CHECK(t.device() == input.device(), op, ": ", name, " must be on the input's device");
}
// A tensor that is written shares no byte with itself or with one of the others (rows may lie between another's).
Pieces pieces_of(const at::Tensor& t, const char* op, const char* name) { return pieces_of_rows(t, row_stride(t, op, name)); }
void writable(const at::Tensor& t, const char* op, const char* name, std::initializer_list<const at::Tensor*> others) {
  if (t.numel() == 0) return;
  const Pieces mine = pieces_of(t, op, name);
  TORCH_CHECK(mine.n * mine.length == (int64_t)t.numel() * (int64_t)t.element_size() && (mine.n <= 1 || mine.stride >= mine.length), op,
              ": the rows of ", name, " must not overlap");
  for (const at::Tensor* o : others)
    if (o != nullptr && o->numel() > 0)
      TORCH_CHECK(!overlap(mine, pieces_of(*o, op, "another tensor")), op, ": ", name, " must not share memory with another tensor of the call");
}
bool same_leading(const at::Tensor& a, const at::Tensor& b) {
  return a.dim() == b.dim() && a.sizes().slice(0, a.dim() - 1) == b.sizes().slice(0, b.dim() - 1);
}
int64_t rows_of(const at::Tensor& t) {
  int64_t rows = 1;
  for (int64_t d = 0; d + 1 < t.dim(); ++d) rows *= t.size(d);
  return rows;
}
int32_t* status_word(const at::Tensor& like) {
  int32_t* word = device_status_word(like.get_device());
  raise_if_timed_out(word);   // an earlier call on this device gave up a wait
  return word;
}

// out = input weight^T with 8-bit integers: input int8 rows with their scales, or rows that are quantised on the way.
void b200_int8_linear(const at::Tensor& out, const at::Tensor& input, const std::optional<at::Tensor>& input_scales,
                      const at::Tensor& weight, const at::Tensor& weight_scales, const std::optional<at::Tensor>& bias) {
  const char* const op = "b200_int8_linear";
  check_cuda(input, "input");
  TORCH_CHECK(input.dim() >= 1 && out.dim() >= 1 && weight.dim() == 2, op, ": input must be [..., K], weight [N, K], out [..., N]");
  const int64_t K = input.size(-1), N = weight.size(0), rows = rows_of(input);
  TORCH_CHECK(weight.size(1) == K, op, ": input and weight must have the same K");
  TORCH_CHECK(same_leading(out, input) && out.size(-1) == N, op, ": out must be [..., N]");
  TORCH_CHECK(rows <= 0x7fffffff && N <= 0x7fffffff && K <= B200MOE_INT8_MAX_K, op, ": too large (K is at most ", B200MOE_INT8_MAX_K, ")");
  TORCH_CHECK(weight.scalar_type() == at::kChar && weight.is_contiguous(), op, ": weight must be contiguous int8");
  TORCH_CHECK(weight_scales.scalar_type() == at::kFloat && weight_scales.is_contiguous() && weight_scales.numel() == N, op,
              ": weight_scales must be contiguous float32 [N]");
  TORCH_CHECK(K > 0 && K % 16 == 0, op, ": K must be a multiple of 16");
  for (const auto& [t, name] : {std::pair<const at::Tensor&, const char*>{out, "out"}, {weight, "weight"}, {weight_scales, "weight_scales"}})
    same_device(t, input, op, name);
  const bool codes = input.scalar_type() == at::kChar;
  TORCH_CHECK(codes == input_scales.has_value(), op, ": int8 rows come with input_scales, other rows without");
  b200moe_int8_linear_args a = {};
  a.d_dtype = float_dtype(out, op);
  if (bias.has_value()) {
    same_device(*bias, input, op, "bias");
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == N && bias->is_contiguous(), op, ": bias must be contiguous [N]");
    TORCH_CHECK(bias->scalar_type() == at::kHalf || bias->scalar_type() == at::kBFloat16, op, ": bias must be float16 or bfloat16");
    a.bias = bias->data_ptr();
    a.bias_dtype = float_dtype(*bias, op);
  }
  if (codes) {
    same_device(*input_scales, input, op, "input_scales");
    TORCH_CHECK(input_scales->scalar_type() == at::kFloat && input_scales->is_contiguous() && input_scales->numel() == rows, op,
                ": input_scales must be contiguous float32, one a row");
  } else {
    float_dtype(input, op);
  }
  const int64_t in_stride = row_stride(input, op, "input");
  a.d_stride = row_stride(out, op, "out");
  TORCH_CHECK(rows <= 1 || a.d_stride >= N, op, ": the rows of out must not overlap");
  writable(out, op, "out", {&input, &weight, &weight_scales, bias.has_value() ? &*bias : nullptr, codes ? &*input_scales : nullptr});
  if (rows == 0 || N == 0) return;
  const c10::cuda::CUDAGuard guard(input.device());
  a.status = status_word(input);
  a.x = input.data_ptr();
  a.x_stride = in_stride;
  a.x_dtype = codes ? B200MOE_I8 : float_dtype(input, op);
  if (codes) a.x_scale = input_scales->data_ptr<float>();
  a.w = (const int8_t*)weight.data_ptr();
  a.w_scale = weight_scales.data_ptr<float>();
  a.d = out.data_ptr();
  a.rows = rows; a.n = (int)N; a.k = (int)K;
  // A few rows are asked for without a workspace first: where the product's kernel quantises them itself, an allocation would be a quarter of
  // the call (1 x 4096 x 4096 6.4 us of the host's time with it).
  int rc = B200MOE_E_WORKSPACE;
  if (codes || rows <= 8) rc = b200moe_int8_linear(&a, current_stream());
  at::Tensor workspace;
  if (!codes && rc == B200MOE_E_WORKSPACE) {
    a.workspace_bytes = b200moe_int8_linear_workspace_bytes(rows, (int)K);
    workspace = at::empty({(int64_t)a.workspace_bytes}, input.options().dtype(at::kByte));
    a.workspace = workspace.data_ptr();
    rc = b200moe_int8_linear(&a, current_stream());
  }
  check_status(rc);
}

// What the gated product's passes have in common; weight [2 I, H], gate rows first.
b200moe_gated_linear_args gated_args(const at::Tensor& input, const at::Tensor& weight, const char* op) {
  check_cuda(input, "input");
  TORCH_CHECK(input.dim() >= 1 && weight.dim() == 2, op, ": input must be [..., H], weight [2 I, H]");
  TORCH_CHECK(weight.size(1) == input.size(-1) && weight.size(0) % 2 == 0, op, ": weight must be [2 I, H] for an input [..., H]");
  TORCH_CHECK(input.scalar_type() == at::kBFloat16 || input.scalar_type() == at::kHalf, op, ": only float16 and bfloat16 are supported");
  TORCH_CHECK(weight.scalar_type() == input.scalar_type(), op, ": weight must have the input's dtype");
  TORCH_CHECK(weight.is_contiguous(), op, ": weight must be contiguous");
  same_device(weight, input, op, "weight");
  b200moe_gated_linear_args a = {};
  const int64_t rows = rows_of(input);
  TORCH_CHECK(rows <= 0x7fffffff && weight.size(0) <= 1 << 30 && weight.size(1) <= 1 << 29, op,
              ": too large (rows of at most 2^29 values, 2^30 of them in weight)");
  a.x = input.data_ptr(); a.w = weight.data_ptr();
  a.rows = rows; a.inter = (int)(weight.size(0) / 2); a.hidden = (int)weight.size(1);
  a.x_stride = row_stride(input, op, "input");
  a.dtype = float_dtype(input, op);
  TORCH_CHECK(a.hidden % 8 == 0 && a.x_stride % 8 == 0, op, ": rows must be multiples of 8 values apart and long");
  return a;
}
void check_pre(const at::Tensor& pre, const at::Tensor& input, const b200moe_gated_linear_args& a, const char* op) {
  same_device(pre, input, op, "pre");
  TORCH_CHECK(pre.scalar_type() == at::kFloat && pre.is_contiguous() && pre.numel() == a.rows * 2 * a.inter &&
                  (pre.dim() == 0 || pre.size(-1) == 2 * (int64_t)a.inter),
              op, ": pre must be contiguous float32 [..., 2 I]");
}

void b200_gated_linear(const at::Tensor& out, const at::Tensor& input, const at::Tensor& weight, const std::optional<at::Tensor>& pre) {
  const char* const op = "b200_gated_linear";
  b200moe_gated_linear_args a = gated_args(input, weight, op);
  same_device(out, input, op, "out");
  TORCH_CHECK(same_leading(out, input) && out.size(-1) == a.inter, op, ": out must be [..., I]");
  TORCH_CHECK(out.scalar_type() == input.scalar_type(), op, ": out must have the input's dtype");
  a.out = out.data_ptr();
  a.out_stride = row_stride(out, op, "out");
  TORCH_CHECK(a.rows <= 1 || a.out_stride >= a.inter, op, ": the rows of out must not overlap");
  writable(out, op, "out", {&input, &weight, pre.has_value() ? &*pre : nullptr});
  if (pre.has_value()) {
    check_pre(*pre, input, a, op);
    writable(*pre, op, "pre", {&input, &weight});
    a.pre = pre->data_ptr<float>();
  }
  TORCH_CHECK(a.hidden > 0, op, ": rows have no values");
  if (a.rows == 0 || a.inter == 0) return;
  const c10::cuda::CUDAGuard guard(input.device());
  a.status = status_word(input);
  check_status(b200moe_gated_linear(&a, current_stream()));
}

void b200_gated_linear_backward(const at::Tensor& grad_out, const at::Tensor& pre, const at::Tensor& input, const at::Tensor& weight,
                                const std::optional<at::Tensor>& grad_input, const std::optional<at::Tensor>& grad_weight) {
  const char* const op = "b200_gated_linear_backward";
  b200moe_gated_linear_args a = gated_args(input, weight, op);
  same_device(grad_out, input, op, "grad_out");
  TORCH_CHECK(same_leading(grad_out, input) && grad_out.size(-1) == a.inter, op, ": grad_out must be [..., I]");
  TORCH_CHECK(grad_out.scalar_type() == input.scalar_type(), op, ": grad_out must have the input's dtype");
  check_pre(pre, input, a, op);
  a.grad = grad_out.data_ptr();
  a.grad_stride = row_stride(grad_out, op, "grad_out");
  a.pre = pre.data_ptr<float>();
  if (grad_input.has_value()) {
    const at::Tensor& t = *grad_input;
    same_device(t, input, op, "grad_input");
    TORCH_CHECK(t.sizes() == input.sizes() && t.scalar_type() == input.scalar_type(), op, ": grad_input must have the input's shape and dtype");
    a.grad_x = t.data_ptr();
    a.grad_x_stride = row_stride(t, op, "grad_input");
    TORCH_CHECK(a.rows <= 1 || a.grad_x_stride >= a.hidden, op, ": the rows of grad_input must not overlap");
    writable(t, op, "grad_input", {&grad_out, &pre, &input, &weight, grad_weight.has_value() ? &*grad_weight : nullptr});
  }
  if (grad_weight.has_value()) {
    const at::Tensor& t = *grad_weight;
    same_device(t, input, op, "grad_weight");
    TORCH_CHECK(t.sizes() == weight.sizes() && t.scalar_type() == weight.scalar_type() && t.is_contiguous(), op,
                ": grad_weight must be contiguous, with the weight's shape and dtype");
    a.grad_w = t.data_ptr();
    writable(t, op, "grad_weight", {&grad_out, &pre, &input, &weight});
  }
  const c10::cuda::CUDAGuard guard(input.device());
  a.status = status_word(input);
  a.workspace_bytes = b200moe_gated_linear_backward_workspace_bytes(a.rows, a.inter);
  const at::Tensor workspace = at::empty({(int64_t)a.workspace_bytes}, input.options().dtype(at::kByte));
  a.workspace = workspace.data_ptr();
  check_status(b200moe_gated_linear_backward(&a, current_stream()));
}

// ---- with gradients ------------------------------------------------------------------
// b200_gated_product(input, weight): the gated product as a value, with its gradients.  Native, as a layer call is: as a Python function
// of autograd a step of 48 rows took 107 us of the host's time for 30 of the kernels'.

// `t` as the kernels read it: rows that are dense, evenly spaced and on 16-byte boundaries (a copy where they are not).
at::Tensor readable(const at::Tensor& t, bool aligned) {
  if (t.numel() == 0) return t;
  bool fits = t.stride(-1) == 1 || t.size(-1) == 1;
  int64_t next = -1;
  for (int64_t d = t.dim() - 2; d >= 0 && fits; --d) {
    if (t.size(d) == 1) continue;
    if (next < 0) fits = !aligned || t.stride(d) % 8 == 0;
    else fits = t.stride(d) == next;
    next = t.stride(d) * t.size(d);
  }
  if (aligned && (uintptr_t)t.data_ptr() % 16 != 0) fits = false;
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}

std::vector<int64_t> with_last(const at::Tensor& t, int64_t n) {
  std::vector<int64_t> sizes = t.sizes().vec();
  sizes.back() = n;
  return sizes;
}

at::Tensor gated_product(const at::Tensor& input, const at::Tensor& weight, at::Tensor* pre) {
  TORCH_CHECK(input.dim() >= 1 && weight.dim() == 2, "b200_gated_product: input must be [..., H], weight [2 I, H]");
  at::Tensor out = at::empty(with_last(input, weight.size(0) / 2), input.options());
  std::optional<at::Tensor> keep;
  if (pre != nullptr) keep = *pre = at::empty(with_last(input, weight.size(0) / 2 * 2), input.options().dtype(at::kFloat));
  b200_gated_linear(out, input, weight, keep);
  return out;
}
at::Tensor b200_gated_product(const at::Tensor& input, const at::Tensor& weight) {
  check_cuda(input, "input");
  return gated_product(readable(input, true), weight.contiguous(), nullptr);
}

// Whether forward-mode differentiation (make_dual, torch.func.jvp) is on its way through `t`.
bool has_tangent(const at::Tensor& t) { return t._fw_grad(0).defined(); }

class GatedProduct : public torch::autograd::Function<GatedProduct> {
 public:
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& input, const at::Tensor& weight) {
    at::AutoDispatchBelowADInplaceOrView below;
    const at::Tensor x = readable(input, true), w = weight.contiguous();
    at::Tensor pre, out = gated_product(x, w, &pre);
    ctx->save_for_backward({x.is_same(input) ? input : x, w.is_same(weight) ? weight : w, pre});
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(grads[0]), "b200_gated_product: its gradients have no forward-mode derivative");
    const at::Tensor &x = saved[0], &w = saved[1], grad = readable(grads[0], false);
    at::AutoDispatchBelowADInplaceOrView below;
    std::optional<at::Tensor> dx, dw;
    // (those that this pass wants: either is a product of its own, half of the work)
    if (ctx->needs_input_grad(0)) dx = at::empty(x.sizes(), x.options());
    if (ctx->needs_input_grad(1)) dw = at::empty(w.sizes(), w.options());
    b200_gated_linear_backward(grad, saved[2], x, w, dx, dw);
    if (at::GradMode::is_enabled()) refuse_twice(grads[0], {dx.has_value() ? &*dx : nullptr, dw.has_value() ? &*dw : nullptr});
    return {dx.has_value() ? *dx : at::Tensor(), dw.has_value() ? *dw : at::Tensor()};
  }

 private:
  // Gradients that are part of a graph (create_graph) depend on both operands and on the incoming gradient, whether or not that one has a graph
  // itself.  Their own derivative raises on the way to any of the three: without a node there it would be left out of a sum of
  // losses in silence.
  static void refuse_twice(const at::Tensor& grad, std::initializer_list<at::Tensor*> gradients) {
    const auto self = torch::autograd::get_current_node();
    TORCH_CHECK(self != nullptr, "b200_gated_product is not differentiable twice");   // (called by no engine: no edges to lead on)
    torch::autograd::edge_list to = self->next_edges();
    if (grad.requires_grad()) to.push_back(torch::autograd::impl::gradient_edge(grad));
    const auto node = std::make_shared<torch::autograd::Error>("b200_gated_product is not differentiable twice", std::move(to));
    for (at::Tensor* t : gradients)
      if (t != nullptr) torch::autograd::set_history(*t, node);
  }
};
bool is_capturing(cudaStream_t stream) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  // (the default stream cannot be asked while another one captures, and does not itself)
  if (cudaStreamIsCapturing(stream, &status) != cudaSuccess) {
    (void)cudaGetLastError();
    return false;
  }
  return status != cudaStreamCaptureStatusNone;
}
// A leaf's gradient is waited for on the stream that its first live graph was made on.  Another stream than the capturing one joins the capture by
// that; the default stream cannot, and the error ends the process in the captured backward pass: refused here, while it is one call's.  That goes
// for leaves that `t` is made of (a view or a copy of a parameter, the layers before) as for `t` itself.
void check_capture(const at::Tensor& t, const char* name) {
  if (!t.requires_grad()) return;
  std::vector<std::shared_ptr<torch::autograd::Node>> to_do;
  std::unordered_set<torch::autograd::Node*> seen;
  auto add = [&](std::shared_ptr<torch::autograd::Node> node) {
    if (node != nullptr && seen.insert(node.get()).second) to_do.push_back(std::move(node));
  };
  add(t.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(t) : t.grad_fn());
  while (!to_do.empty()) {
    const auto node = std::move(to_do.back());
    to_do.pop_back();
    const auto edges = node->next_edges();
    for (const auto& edge : edges) add(edge.function);
    if (dynamic_cast<torch::autograd::AccumulateGrad*>(node.get()) == nullptr) continue;
    const auto stream = node->stream();
    TORCH_CHECK(!stream.has_value() || c10::cuda::CUDAStream(*stream).stream() != nullptr, "b200_gated_product: ", name,
                " is part of a graph that lives outside this stream capture, on the default stream; let go of what was computed from it first");
  }
}
at::Tensor b200_gated_product_autograd(const at::Tensor& input, const at::Tensor& weight) {
  // (below autograd a tangent would be dropped, and the derivative be zero)
  TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(input) && !has_tangent(weight), "b200_gated_product has no forward-mode derivative");
  if (at::GradMode::is_enabled() && (input.requires_grad() || weight.requires_grad()) && input.is_cuda()) {
    if (is_capturing(at::cuda::getCurrentCUDAStream(input.get_device()))) {
      check_capture(input, "input");
      check_capture(weight, "weight");
    }
    return GatedProduct::apply(input, weight);
  }
  at::AutoDispatchBelowADInplaceOrView below;
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("_xpu_C::b200_gated_product", "")
                             .typed<at::Tensor(const at::Tensor&, const at::Tensor&)>();
  return op.call(input, weight);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(_xpu_C, m) {
  m.def("b200_gated_product(Tensor input, Tensor weight) -> Tensor");
  m.def(
      "b200_int8_linear(Tensor(a!) out, Tensor input, Tensor? input_scales, Tensor weight, Tensor weight_scales, "
      "Tensor? bias=None) -> ()");
  m.def("b200_gated_linear(Tensor(a!) out, Tensor input, Tensor weight, Tensor(b!)? pre=None) -> ()");
  m.def(
      "b200_gated_linear_backward(Tensor grad_out, Tensor pre, Tensor input, Tensor weight, Tensor(a!)? grad_input, "
      "Tensor(b!)? grad_weight) -> ()");
}

TORCH_LIBRARY_IMPL(_xpu_C, CUDA, m) {
  m.impl("b200_int8_linear", &b200_int8_linear);
  m.impl("b200_gated_linear", &b200_gated_linear);
  m.impl("b200_gated_linear_backward", &b200_gated_linear_backward);
  m.impl("b200_gated_product", &b200_gated_product);
}

TORCH_LIBRARY_IMPL(_xpu_C, Autograd, m) { m.impl("b200_gated_product", &b200_gated_product_autograd); }
