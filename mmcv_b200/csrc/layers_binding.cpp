// Tensor front of the transformer-layer entries of the C ABI (dcn_linear_*, dcn_layer_norm_*): argument
// checks, row strides, workspaces, streams and autograd nodes.  It is C++ and not Python because the
// kernels of a layer on a few hundred tokens take microseconds: a node written in Python costs more
// host time than its kernels run (a layer norm's training step on 300 rows: 121 us of host time with
// Python nodes).  mmcv_b200/_layers.py loads it; mmcv_b200.ops documents the operators.
#include <atomic>
#include <initializer_list>
#include <memory>
#include <mutex>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>

#include "dcn_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

std::atomic<bool> g_check_status{false};

int dtype_code(const char *op, at::ScalarType t) {
  switch (t) {
    case at::kFloat: return DCN_DTYPE_F32;
    case at::kBFloat16: return DCN_DTYPE_BF16;
    case at::kHalf: return DCN_DTYPE_F16;
    default:
      TORCH_CHECK(false, "dcn_b200: ", op, ": unsupported dtype ", t, " (float32, bfloat16 and float16 only)");
  }
}

void check(int rc) { TORCH_CHECK(rc == DCN_OK, "dcn_b200: ", dcn_last_error(), " (code ", rc, ")"); }

bool has(const OptTensor &t) { return t.has_value() && t->defined(); }

void require(const char *op, const char *name, const Tensor &t, const Tensor &like) {
  TORCH_CHECK(t.is_cuda(), "dcn_b200: ", op, ": ", name,
              " must be a CUDA tensor (this build has no CPU implementation)");
  TORCH_CHECK(t.device() == like.device(), "dcn_b200: ", op, ": ", name, " is on ", t.device(), ", expected ",
              like.device());
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), "dcn_b200: ", op, ": ", name, " has dtype ", t.scalar_type(),
              ", expected ", like.scalar_type());
}

// A tensor as [rows, cols] with neighbouring columns next to each other in memory.  Whatever a row
// stride can describe is taken as it lies; the rest is copied.
struct Rows {
  Tensor keep;
  const void *p = nullptr;
  int64_t ld = 0, rows = 0;
  Rows() = default;
  Rows(const Tensor &t, int64_t cols) {
    rows = t.numel() / cols;
    ld = cols;
    if (t.is_contiguous()) {
      keep = t;
    } else {
      keep = t.dim() == 2 && t.size(1) == cols ? t : t.reshape({rows, cols});
      if ((keep.stride(1) != 1 && cols > 1) || (keep.stride(0) < cols && rows > 1)) keep = keep.contiguous();
      if (rows > 1) ld = keep.stride(0);
    }
    p = keep.const_data_ptr();
  }
};

const void *ptr(const OptTensor &t) { return has(t) ? t->const_data_ptr() : nullptr; }
void *out_ptr(const Tensor &t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

// A dense tensor on `like`'s device, straight from the allocator.
Tensor make(at::IntArrayRef sizes, at::ScalarType type, const Tensor &like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

Tensor workspace(const Tensor &like, size_t bytes) {
  return bytes ? make({(int64_t)bytes}, at::kByte, like) : Tensor();
}

// The status word is read after the call where that was asked for (set_check_status).  A stream that is being
// captured cannot be waited for: what a replay leaves in the word is found by the next call outside a capture.
void after(int device, void *stream) {
  if (!g_check_status.load(std::memory_order_relaxed)) return;
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return;
  int32_t status = 0;
  check(dcn_linear_read_status(device, stream, &status));
  TORCH_CHECK(status == 0, "dcn_b200: device-side wait ", status, " timed out; the output is not valid");
}

// ---- matrix product ---------------------------------------------------------------------------

std::pair<Tensor, Tensor> linear_forward(const Tensor &x, const Tensor &w, const OptTensor &bias, const OptTensor &res,
                                         int act, bool save) {
  const int code = dtype_code("linear", x.scalar_type());
  const int64_t cout = w.size(0), cin = w.size(1), es = x.element_size();
  const c10::cuda::CUDAGuard guard(x.device());
  const int dev = x.device().index();
  void *stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  const Rows xr(x, cin), wr(w, cin), rr = has(res) ? Rows(*res, cout) : Rows();
  auto shape = x.sizes().vec();
  shape.back() = cout;
  Tensor y = make(shape, x.scalar_type(), x), saved;
  const Tensor b = has(bias) ? bias->contiguous() : Tensor();
  if (save && act == DCN_ACT_RELU) saved = make({xr.rows, (cout + 31) / 32}, at::kInt, x);
  if (save && act == DCN_ACT_GELU) saved = make({xr.rows, (cout + 7) / 8 * 8}, code == DCN_DTYPE_F32 ? at::kFloat : at::kShort, x);
  const int64_t align = (int64_t)(uintptr_t)xr.p | (int64_t)(uintptr_t)wr.p | ((xr.ld | wr.ld) * es);
  size_t bytes = 0;
  check(dcn_linear_workspace_bytes(code, xr.rows, cin, cout, align, &bytes));
  const Tensor ws = workspace(x, bytes);
  check(dcn_linear_forward(xr.p, xr.ld, wr.p, wr.ld, ptr(b), rr.p, rr.ld, out_ptr(y), out_ptr(saved), code, act,
                           xr.rows, cin, cout, dev, out_ptr(ws), bytes, stream));
  after(dev, stream);
  return {y, saved};
}

struct Want { bool x, w, b, x_sum; };
struct LinearGrads { Tensor x, w, b, x_sum; };

// The gradients of linear_forward that `want` asks for.  in_saved / in_act: the gradient of x is taken on
// through the activation that made x; gx_add is added to it; x_sum: its column sums.
LinearGrads linear_backward(const Tensor &gy, const Tensor &x, const Tensor &w, int64_t cin,
                                                   const std::vector<int64_t> &x_shape, const Tensor &saved, int act,
                                                   Want want, const Tensor &in_saved, int in_act,
                                                   const Tensor &gx_add) {
  const int code = dtype_code("linear", gy.scalar_type());
  const int64_t cout = gy.size(-1), es = gy.element_size();
  const c10::cuda::CUDAGuard guard(gy.device());
  const int dev = gy.device().index();
  void *stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  const Rows gr(gy, cout), xr = want.w ? Rows(x, cin) : Rows(), wr = want.x ? Rows(w, cin) : Rows();
  LinearGrads g;
  const at::ScalarType type = gy.scalar_type();
  if (want.x) g.x = make(x_shape, type, gy);
  if (want.w) g.w = make({cout, cin}, type, gy);
  if (want.b) g.b = make({cout}, type, gy);
  if (want.x_sum) g.x_sum = make({cin}, type, gy);
  const Tensor add = gx_add.defined() ? gx_add.contiguous() : Tensor();
  const int64_t align = (int64_t)(uintptr_t)gr.p | (int64_t)(uintptr_t)xr.p | (int64_t)(uintptr_t)wr.p |
                        ((gr.ld | xr.ld | wr.ld) * es);
  size_t bytes = 0;
  check(dcn_linear_backward_workspace_bytes(code, act, gr.rows, cin, cout, align, want.x ? want.x_sum ? 2 : 1 : 0,
                                            want.w, want.b, &bytes));
  const Tensor ws = workspace(gy, bytes);
  check(dcn_linear_backward(gr.p, gr.ld, xr.p, xr.ld, wr.p, wr.ld, out_ptr(saved), out_ptr(in_saved), out_ptr(add),
                            out_ptr(g.x), out_ptr(g.x_sum), out_ptr(g.w), out_ptr(g.b), code, act, in_act, gr.rows, cin, cout, dev,
                            out_ptr(ws), bytes, stream));
  after(dev, stream);
  return g;
}

// The kernels' gradients are values, not functions of the inputs: a second derivative is an error, not zero.
variable_list once(const char *op, variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list given;
  for (const Tensor &g : grads)
    if (g.defined()) given.push_back(g.detach().requires_grad_(true));
  auto fail = std::make_shared<torch::autograd::DelayedError>(
      std::string("dcn_b200: ") + op + ": the gradient cannot be differentiated again", (int64_t)given.size());
  variable_list wrapped = (*fail)(std::move(given));
  size_t k = 0;
  for (Tensor &g : grads)
    if (g.defined()) g = wrapped[k++];
  return grads;
}

bool needs(const Tensor &t) { return t.defined() && t.requires_grad(); }
bool needs(const OptTensor &t) { return has(t) && t->requires_grad(); }

// A tangent of forward-mode differentiation would be lost without a word.
void refuse_tangents(const char *op, std::initializer_list<const Tensor *> tensors) {
  for (const Tensor *t : tensors)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), "dcn_b200: ", op,
                ": forward-mode differentiation is not supported");
}

// A view that negates lazily has the opposite sign in memory.
bool negated(std::initializer_list<const Tensor *> tensors) {
  for (const Tensor *t : tensors)
    if (t->defined() && t->is_neg()) return true;
  return false;
}
Tensor resolved(const Tensor &t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }

// A tracer records dispatched operations, and there is none here: the results of the example's values would
// stand in the traced program as constants.
void refuse_tracing(const char *op) {
  using Mode = c10::impl::TorchDispatchModeKey;
  using Modes = c10::impl::TorchDispatchModeTLS;
  TORCH_CHECK(!torch::jit::tracer::isTracing() && !Modes::get_mode(Mode::PROXY).has_value() &&
                  !Modes::get_mode(Mode::FAKE).has_value(),
              "dcn_b200: ", op, ": tracing is not supported (the traced program would keep this call's values)");
}

const Tensor &get(const OptTensor &t) {
  static const Tensor none;
  return t.has_value() ? *t : none;
}

// Nodes are written against the engine's own interface: the convenience class for custom functions keeps
// its values in a dictionary of boxed ones, 6 us more for a forward call and a backward pass.
template <typename N, typename... T>
std::shared_ptr<N> make_node(const T &...inputs) {
  std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
  return node;
}

struct LinearNode final : torch::autograd::Node {
  SavedVariable x, w, saved;
  std::vector<int64_t> shape;
  int64_t cin = 0;
  int act = 0;
  std::string name() const override { return "FusedLinearBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data();
    w.reset_data();
    saved.reset_data();
  }
  variable_list apply(variable_list &&gys) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(4);
    if (!gys[0].defined()) return out;
    const Want want{task_should_compute_output(0), task_should_compute_output(1), task_should_compute_output(2), false};
    if (want.x || want.w || want.b) {
      LinearGrads g;
      {
        const c10::AutoGradMode off(false);
        g = linear_backward(resolved(gys[0]), x.unpack(), w.unpack(), cin, shape, saved.unpack(), act, want, Tensor(),
                            DCN_ACT_NONE, Tensor());
      }
      out = {g.x, g.w, g.b, Tensor()};
    }
    if (task_should_compute_output(3)) out[3] = gys[0];
    return once("fused_linear", std::move(out));
  }
};

void check_weight(const char *op, const char *name, const Tensor &input, int64_t cin, const Tensor &w) {
  require(op, name, w, input);
  TORCH_CHECK(w.dim() == 2 && w.size(1) == cin, "dcn_b200: ", op, ": ", name, " has shape ", w.sizes(),
              ", which does not fit rows of ", cin, " (expected [out, ", cin, "])");
  TORCH_CHECK(w.size(0) > 0 && cin > 0, "dcn_b200: ", op, ": ", name, " must not be empty");
}
void check_bias(const char *op, const char *name, const Tensor &input, const OptTensor &b, int64_t cout) {
  if (!has(b)) return;
  require(op, name, *b, input);
  TORCH_CHECK(b->dim() == 1 && b->size(0) == cout, "dcn_b200: ", op, ": ", name, " has shape ", b->sizes(),
              ", expected [", cout, "]");
}
void check_input(const char *op, const Tensor &input) {
  dtype_code(op, input.scalar_type());
  TORCH_CHECK(input.is_cuda(), "dcn_b200: ", op,
              ": input must be a CUDA tensor (this build has no CPU implementation)");
  TORCH_CHECK(input.dim() >= 1, "dcn_b200: ", op, ": input must have at least one dimension");
}
OptTensor check_residual(const char *op, const Tensor &input, const OptTensor &res, int64_t cout) {
  if (!has(res)) return std::nullopt;
  require(op, "residual", *res, input);
  auto shape = input.sizes().vec();
  shape.back() = cout;
  return res->sizes() == shape ? *res : res->expand(shape);   // its gradient is summed where it was broadcast
}

Tensor fused_linear(const Tensor &input, const Tensor &weight, const OptTensor &bias, const OptTensor &residual,
                    int64_t act) {
  refuse_tracing("fused_linear");
  check_input("fused_linear", input);
  check_weight("fused_linear", "weight", input, input.size(-1), weight);
  check_bias("fused_linear", "bias", input, bias, weight.size(0));
  if (negated({&input, &weight, &get(bias), &get(residual)}))
    return fused_linear(resolved(input), resolved(weight), resolved(get(bias)), resolved(get(residual)), act);
  const OptTensor res = check_residual("fused_linear", input, residual, weight.size(0));
  refuse_tangents("fused_linear", {&input, &weight, &get(bias), &get(res)});
  const bool grad = at::GradMode::is_enabled(), nx = grad && needs(input), nw = grad && needs(weight),
             nb = grad && needs(bias), nr = grad && needs(res);
  std::pair<Tensor, Tensor> made;
  {
    const c10::AutoGradMode off(false);
    made = linear_forward(input, weight, bias, res, (int)act, nx || nw || nb);
  }
  if (nx || nw || nb || nr) {
    auto node = make_node<LinearNode>(input, weight, get(bias), get(res));
    if (nw) node->x = SavedVariable(input, false);
    if (nx) node->w = SavedVariable(weight, false);
    if (made.second.defined()) node->saved = SavedVariable(made.second, false);
    node->shape = input.sizes().vec();
    node->cin = weight.size(1);
    node->act = (int)act;
    torch::autograd::set_history(made.first, node);
  }
  return made.first;
}

// ---- two products back to back ----------------------------------------------------------------

struct FeedForwardNode final : torch::autograd::Node {
  SavedVariable x, w1, w2, h, saved;
  std::vector<int64_t> shape;
  int64_t cin = 0, hidden = 0;
  int act = 0;
  bool identity = false;   // the residual is the input itself
  std::string name() const override { return "FeedForwardBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable *v : {&x, &w1, &w2, &h, &saved}) v->reset_data();
  }
  variable_list apply(variable_list &&gys) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(6);
    const Tensor gy = resolved(gys[0]);
    if (!gy.defined()) return out;
    const bool nx = task_should_compute_output(0), nw1 = task_should_compute_output(1),
               nb1 = task_should_compute_output(2), nw2 = task_should_compute_output(3),
               nb2 = task_should_compute_output(4), inner = nx || nw1 || nb1;
    // bias1's gradient from the hidden gradient before its rounding, in the epilogue of the product that makes
    // it, up to 2^22 hidden values; beyond, where that takes 8 to 13 % of the step, from the rounded one, beside
    // weight1's: two roundings, not one.  us of a bf16 training step with relu, before / after the rounding: 300 x 256 x 1024
    // 47.5 / 47.5, 1200 x 256 x 1024 61.8 / 59.8, 4000 x 256 x 1024 68.0 / 65.9, 8000 x 256 x 1024 85.6 / 79.0,
    // 35642 x 256 x 512 123.7 / 108.5, 35642 x 256 x 1024 187 / 165.  fp32 gradients are not rounded; without an
    // activation there is no such epilogue.
    const bool early = nb1 && act != DCN_ACT_NONE && gy.scalar_type() != at::kFloat &&
                       gy.numel() / gy.size(-1) * hidden <= 1 << 22;
    {
      const c10::AutoGradMode off(false);
      Tensor gz;
      if (inner || nw2 || nb2) {
        auto h_shape = shape;
        h_shape.back() = hidden;
        LinearGrads g = linear_backward(gy, h.unpack(), w2.unpack(), hidden, h_shape, Tensor(), DCN_ACT_NONE,
                                        Want{inner, nw2, nb2, early}, saved.unpack(), act, Tensor());
        gz = g.x;
        out[2] = g.x_sum;
        out[3] = g.w;
        out[4] = g.b;
      }
      if (nx || nw1 || (nb1 && !early)) {
        LinearGrads g = linear_backward(gz, x.unpack(), w1.unpack(), cin, shape, Tensor(), DCN_ACT_NONE,
                                        Want{nx, nw1, nb1 && !early, false}, Tensor(), DCN_ACT_NONE,
                                        nx && identity ? gy : Tensor());
        out[0] = g.x;
        out[1] = g.w;
        if (!early) out[2] = g.b;
      }
    }
    if (task_should_compute_output(5)) out[5] = gy;
    return once("feed_forward", std::move(out));
  }
};

Tensor feed_forward(const Tensor &input, const Tensor &w1, const OptTensor &b1, const Tensor &w2, const OptTensor &b2,
                    const OptTensor &residual, int64_t act) {
  const char *op = "feed_forward";
  refuse_tracing(op);
  check_input(op, input);
  check_weight(op, "weight1", input, input.size(-1), w1);
  check_bias(op, "bias1", input, b1, w1.size(0));
  check_weight(op, "weight2", input, w1.size(0), w2);
  check_bias(op, "bias2", input, b2, w2.size(0));
  if (negated({&input, &w1, &get(b1), &w2, &get(b2), &get(residual)})) {
    const Tensor x = resolved(input);
    return feed_forward(x, resolved(w1), resolved(get(b1)), resolved(w2), resolved(get(b2)),
                        has(residual) && residual->is_same(input) ? x : resolved(get(residual)), act);
  }
  const bool identity = has(residual) && residual->is_same(input) && w2.size(0) == input.size(-1);
  const OptTensor res = identity ? OptTensor() : check_residual(op, input, residual, w2.size(0));
  refuse_tangents(op, {&input, &w1, &get(b1), &w2, &get(b2), &get(res)});
  const bool grad = at::GradMode::is_enabled(), nx = grad && needs(input), nw1 = grad && needs(w1),
             nb1 = grad && needs(b1), nw2 = grad && needs(w2), nb2 = grad && needs(b2), nr = grad && needs(res);
  const bool inner = nx || nw1 || nb1;
  std::pair<Tensor, Tensor> first;
  Tensor y;
  {
    const c10::AutoGradMode off(false);
    first = linear_forward(input, w1, b1, std::nullopt, (int)act, inner);
    y = linear_forward(first.first, w2, b2, identity ? OptTensor(input) : res, DCN_ACT_NONE, false).first;
  }
  if (inner || nw2 || nb2 || nr) {
    auto node = make_node<FeedForwardNode>(input, w1, get(b1), w2, get(b2), get(res));
    if (nw1) node->x = SavedVariable(input, false);
    if (nx) node->w1 = SavedVariable(w1, false);
    if (inner) node->w2 = SavedVariable(w2, false);
    if (nw2) node->h = SavedVariable(first.first, false);
    if (first.second.defined()) node->saved = SavedVariable(first.second, false);
    node->shape = input.sizes().vec();
    node->cin = input.size(-1);
    node->hidden = w1.size(0);
    node->act = (int)act;
    node->identity = identity;
    torch::autograd::set_history(y, node);
  }
  return y;
}

// ---- layer norm -------------------------------------------------------------------------------

std::pair<Tensor, Tensor> norm_forward(const Tensor &x, const OptTensor &w, const OptTensor &b, int64_t cols,
                                       double eps, bool save) {
  const int code = dtype_code("layer_norm", x.scalar_type());
  const c10::cuda::CUDAGuard guard(x.device());
  const int dev = x.device().index();
  const Rows xr(x, cols);
  Tensor y = make(x.sizes(), x.scalar_type(), x), stats;
  if (save) stats = make({3, xr.rows}, at::kFloat, x);
  const int wcode = has(w) ? dtype_code("layer_norm", w->scalar_type()) : has(b) ? dtype_code("layer_norm", b->scalar_type()) : code;
  check(dcn_layer_norm_forward(xr.p, xr.ld, ptr(w), ptr(b), out_ptr(y), (float *)out_ptr(stats), code, wcode, xr.rows,
                               cols, (float)eps, dev, c10::cuda::getCurrentCUDAStream(dev).stream()));
  return {y, stats};
}

struct NormNode final : torch::autograd::Node {
  SavedVariable x, w, stats;
  int64_t cols = 0;
  std::vector<int64_t> shape;        // of weight and bias
  at::ScalarType type = at::kFloat;  // of weight and bias
  std::string name() const override { return "LayerNormBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data();
    w.reset_data();
    stats.reset_data();
  }
  variable_list apply(variable_list &&gys) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(3);
    if (!gys[0].defined()) return out;
    {
      const c10::AutoGradMode off(false);
      const Tensor in = x.unpack(), weight = w.unpack(), st = stats.unpack();
      const c10::cuda::CUDAGuard guard(in.device());
      const int dev = in.device().index();
      if (task_should_compute_output(0)) out[0] = make(in.sizes(), in.scalar_type(), in);
      if (task_should_compute_output(1)) out[1] = make(shape, type, in);
      if (task_should_compute_output(2)) out[2] = make(shape, type, in);
      const Rows gr(resolved(gys[0]), cols), xr(in, cols);
      size_t bytes = 0;
      if (out[1].defined() || out[2].defined()) check(dcn_layer_norm_workspace_bytes(xr.rows, cols, &bytes));
      const Tensor ws = workspace(in, bytes);
      check(dcn_layer_norm_backward(gr.p, gr.ld, xr.p, xr.ld, weight.defined() ? weight.const_data_ptr() : nullptr,
                                    (const float *)st.const_data_ptr(), out_ptr(out[0]), out_ptr(out[1]),
                                    out_ptr(out[2]), dtype_code("layer_norm", in.scalar_type()),
                                    dtype_code("layer_norm", type), xr.rows, cols, dev, out_ptr(ws), bytes,
                                    c10::cuda::getCurrentCUDAStream(dev).stream()));
    }
    return once("layer_norm", std::move(out));
  }
};

Tensor layer_norm(const Tensor &input, const std::vector<int64_t> &shape, const OptTensor &weight,
                  const OptTensor &bias, double eps) {
  const char *op = "layer_norm";
  refuse_tracing(op);
  check_input(op, input);
  const int64_t n = (int64_t)shape.size();
  TORCH_CHECK(n > 0 && input.dim() >= n && input.sizes().slice(input.dim() - n) == at::IntArrayRef(shape), "dcn_b200: ",
              op, ": input of shape ", input.sizes(), " does not end in normalized_shape ", at::IntArrayRef(shape));
  int64_t cols = 1;
  for (int64_t v : shape) cols *= v;
  TORCH_CHECK(cols > 0, "dcn_b200: ", op, ": normalized_shape ", at::IntArrayRef(shape), " has no elements");
  for (const auto &[name, p] : {std::make_pair("weight", &weight), std::make_pair("bias", &bias)}) {
    if (!has(*p)) continue;
    const Tensor &t = **p;
    TORCH_CHECK(t.sizes() == at::IntArrayRef(shape), "dcn_b200: ", op, ": ", name, " has shape ", t.sizes(),
                ", expected ", at::IntArrayRef(shape));
    TORCH_CHECK(t.scalar_type() == input.scalar_type() || t.scalar_type() == at::kFloat, "dcn_b200: ", op, ": ", name,
                " has dtype ", t.scalar_type(), ", expected ", input.scalar_type(), " or float32");
    TORCH_CHECK(t.device() == input.device(), "dcn_b200: ", op, ": ", name, " is on ", t.device(), ", expected ",
                input.device());
  }
  TORCH_CHECK(!has(weight) || !has(bias) || weight->scalar_type() == bias->scalar_type(), "dcn_b200: ", op,
              ": weight and bias have different dtypes");
  if (negated({&input, &get(weight), &get(bias)}))
    return layer_norm(resolved(input), shape, resolved(get(weight)), resolved(get(bias)), eps);
  const OptTensor w = has(weight) ? OptTensor(weight->contiguous()) : OptTensor();
  const OptTensor b = has(bias) ? OptTensor(bias->contiguous()) : OptTensor();
  refuse_tangents(op, {&input, &get(w), &get(b)});
  const bool grad = at::GradMode::is_enabled() && (needs(input) || needs(w) || needs(b));
  std::pair<Tensor, Tensor> made;
  {
    const c10::AutoGradMode off(false);
    made = norm_forward(input, w, b, cols, eps, grad);
  }
  if (grad) {
    auto node = make_node<NormNode>(input, get(w), get(b));
    node->x = SavedVariable(input, false);
    if (has(w)) node->w = SavedVariable(*w, false);
    node->stats = SavedVariable(made.second, false);
    node->cols = cols;
    const Tensor &p = has(w) ? *w : has(b) ? *b : input;
    node->shape = p.sizes().vec();
    node->type = p.scalar_type();
    torch::autograd::set_history(made.first, node);
  }
  return made.first;
}

}  // namespace

PYBIND11_MODULE(_layers_native, m) {
  namespace py = pybind11;
  m.def("fused_linear", &fused_linear);
  m.def("feed_forward", &feed_forward);
  m.def("layer_norm", &layer_norm);
  m.def("set_check_status", [](bool flag) { g_check_status.store(flag); });
}
