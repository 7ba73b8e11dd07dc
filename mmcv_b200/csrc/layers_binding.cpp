// Tensor front of the transformer-layer entries of the C ABI (dcn_linear_*, dcn_layer_norm_*): argument
// checks, row strides, workspaces, streams and autograd nodes.  It is C++ and not Python because the
// kernels of a layer on a few hundred tokens take microseconds: a node written in Python costs more
// host time than its kernels run (a layer norm's training step on 300 rows: 121 us of host time with
// Python nodes).  mmcv_b200/_layers.py loads it; mmcv_b200.ops documents the operators.
#include <atomic>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>
#include <ATen/ATen.h>

#include "dcn_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
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
      keep = t.dim() == 2 ? t : t.reshape({rows, cols});
      if ((keep.stride(1) != 1 && cols > 1) || (keep.stride(0) < cols && rows > 1)) keep = keep.contiguous();
      if (rows > 1) ld = keep.stride(0);
    }
    p = keep.const_data_ptr();
  }
};

const void *ptr(const OptTensor &t) { return has(t) ? t->const_data_ptr() : nullptr; }
void *out_ptr(const Tensor &t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

Tensor workspace(const Tensor &like, size_t bytes) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

void after(int device, void *stream) {
  if (!g_check_status.load(std::memory_order_relaxed)) return;
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
  Tensor y = at::empty(shape, x.options()), saved;
  const Tensor b = has(bias) ? bias->contiguous() : Tensor();
  if (save && act == DCN_ACT_RELU) saved = at::empty({xr.rows, (cout + 31) / 32}, x.options().dtype(at::kInt));
  if (save && act == DCN_ACT_GELU) saved = at::empty({xr.rows, (cout + 7) / 8 * 8}, x.options().dtype(code == DCN_DTYPE_F32 ? at::kFloat : at::kHalf));
  const int64_t align = (int64_t)(uintptr_t)xr.p | (int64_t)(uintptr_t)wr.p | ((xr.ld | wr.ld) * es);
  size_t bytes = 0;
  check(dcn_linear_workspace_bytes(code, xr.rows, cin, cout, align, &bytes));
  const Tensor ws = workspace(x, bytes);
  check(dcn_linear_forward(xr.p, xr.ld, wr.p, wr.ld, ptr(b), rr.p, rr.ld, out_ptr(y), out_ptr(saved), code, act,
                           xr.rows, cin, cout, dev, out_ptr(ws), bytes, stream));
  after(dev, stream);
  return {y, saved};
}

struct Want { bool x, w, b; };

// The gradients of linear_forward that `want` asks for.  in_saved / in_act: the gradient of x is taken on
// through the activation that made x; gx_add is added to it.
std::tuple<Tensor, Tensor, Tensor> linear_backward(const Tensor &gy, const Tensor &x, const Tensor &w, int64_t cin,
                                                   const std::vector<int64_t> &x_shape, const Tensor &saved, int act,
                                                   Want want, const Tensor &in_saved, int in_act,
                                                   const Tensor &gx_add) {
  const int code = dtype_code("linear", gy.scalar_type());
  const int64_t cout = gy.size(-1), es = gy.element_size();
  const c10::cuda::CUDAGuard guard(gy.device());
  const int dev = gy.device().index();
  void *stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  const Rows gr(gy, cout), xr = want.w ? Rows(x, cin) : Rows(), wr = want.x ? Rows(w, cin) : Rows();
  Tensor gx, gw, gb;
  if (want.x) gx = at::empty(x_shape, gy.options());
  if (want.w) gw = at::empty({cout, cin}, gy.options());
  if (want.b) gb = at::empty({cout}, gy.options());
  const Tensor add = gx_add.defined() ? gx_add.contiguous() : Tensor();
  const int64_t align = (int64_t)(uintptr_t)gr.p | (int64_t)(uintptr_t)xr.p | (int64_t)(uintptr_t)wr.p |
                        ((gr.ld | xr.ld | wr.ld) * es);
  size_t bytes = 0;
  check(dcn_linear_backward_workspace_bytes(code, act, gr.rows, cin, cout, align, want.x, want.w, want.b, &bytes));
  const Tensor ws = workspace(gy, bytes);
  check(dcn_linear_backward(gr.p, gr.ld, xr.p, xr.ld, wr.p, wr.ld, out_ptr(saved), out_ptr(in_saved), out_ptr(add),
                            out_ptr(gx), out_ptr(gw), out_ptr(gb), code, act, in_act, gr.rows, cin, cout, dev,
                            out_ptr(ws), bytes, stream));
  after(dev, stream);
  return {gx, gw, gb};
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

struct LinearNode : torch::autograd::Function<LinearNode> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const OptTensor &bias,
                        const OptTensor &res, int64_t act) {
    const bool nx = needs(x), nw = needs(w), nb = needs(bias);
    auto [y, saved] = linear_forward(x, w, bias, res, (int)act, nx || nw || nb);
    ctx->saved_data["act"] = act;
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["cin"] = w.size(1);
    ctx->saved_data["bias"] = has(bias);
    ctx->saved_data["res"] = has(res);
    ctx->save_for_backward({nw ? x : Tensor(), nx ? w : Tensor(), saved});
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list gys) {
    const variable_list s = ctx->get_saved_variables();
    const bool bias = ctx->saved_data["bias"].toBool(), res = ctx->saved_data["res"].toBool();
    const Want want{ctx->needs_input_grad(0), ctx->needs_input_grad(1), bias && ctx->needs_input_grad(2)};
    variable_list out(5);
    if (!gys[0].defined()) return out;
    if (want.x || want.w || want.b)
      std::tie(out[0], out[1], out[2]) =
          linear_backward(gys[0], s[0], s[1], ctx->saved_data["cin"].toInt(), ctx->saved_data["shape"].toIntVector(),
                          s[2], (int)ctx->saved_data["act"].toInt(), want, Tensor(), DCN_ACT_NONE, Tensor());
    if (res && ctx->needs_input_grad(2 + (bias ? 1 : 0))) out[3] = gys[0];
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
  check_input("fused_linear", input);
  check_weight("fused_linear", "weight", input, input.size(-1), weight);
  check_bias("fused_linear", "bias", input, bias, weight.size(0));
  const OptTensor res = check_residual("fused_linear", input, residual, weight.size(0));
  if (at::GradMode::is_enabled() && (needs(input) || needs(weight) || needs(bias) || needs(res)))
    return LinearNode::apply(input, weight, bias, res, act);
  return linear_forward(input, weight, bias, res, (int)act, false).first;
}

// ---- two products back to back ----------------------------------------------------------------

struct FeedForwardNode : torch::autograd::Function<FeedForwardNode> {
  // identity: the residual is the input itself (res is empty then)
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w1, const OptTensor &b1,
                        const Tensor &w2, const OptTensor &b2, const OptTensor &res, int64_t act, bool identity) {
    const bool inner = needs(x) || needs(w1) || needs(b1), keep_h = needs(w2);
    auto [h, saved] = linear_forward(x, w1, b1, std::nullopt, (int)act, inner);
    Tensor y = linear_forward(h, w2, b2, identity ? OptTensor(x) : res, DCN_ACT_NONE, false).first;
    ctx->saved_data["act"] = act;
    ctx->saved_data["identity"] = identity;
    ctx->saved_data["b1"] = has(b1);
    ctx->saved_data["b2"] = has(b2);
    ctx->saved_data["res"] = has(res);
    ctx->save_for_backward({x, w1, w2, keep_h ? h : Tensor(), saved});
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list gys) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w1 = s[1], &w2 = s[2];
    const bool hb1 = ctx->saved_data["b1"].toBool(), hb2 = ctx->saved_data["b2"].toBool();
    size_t edge = 0;   // edges exist for the tensors that were given
    const bool nx = ctx->needs_input_grad(edge++), nw1 = ctx->needs_input_grad(edge++);
    const bool nb1 = hb1 && ctx->needs_input_grad(edge++);
    const bool nw2 = ctx->needs_input_grad(edge++);
    const bool nb2 = hb2 && ctx->needs_input_grad(edge++);
    const bool nres = ctx->saved_data["res"].toBool() && ctx->needs_input_grad(edge);
    const bool inner = nx || nw1 || nb1;
    variable_list out(8);
    if (!gys[0].defined()) return out;
    const int64_t hidden = w1.size(0);
    auto h_shape = x.sizes().vec();
    h_shape.back() = hidden;
    Tensor gz;
    if (inner || nw2 || nb2)
      std::tie(gz, out[3], out[4]) =
          linear_backward(gys[0], s[3], w2, hidden, h_shape, Tensor(), DCN_ACT_NONE, Want{inner, nw2, nb2}, s[4],
                          (int)ctx->saved_data["act"].toInt(), Tensor());
    if (inner)
      std::tie(out[0], out[1], out[2]) =
          linear_backward(gz, x, w1, x.size(-1), x.sizes().vec(), Tensor(), DCN_ACT_NONE, Want{nx, nw1, nb1}, Tensor(),
                          DCN_ACT_NONE, nx && ctx->saved_data["identity"].toBool() ? gys[0] : Tensor());
    if (nres) out[5] = gys[0];
    return once("feed_forward", std::move(out));
  }
};

Tensor feed_forward(const Tensor &input, const Tensor &w1, const OptTensor &b1, const Tensor &w2, const OptTensor &b2,
                    const OptTensor &residual, int64_t act) {
  const char *op = "feed_forward";
  check_input(op, input);
  check_weight(op, "weight1", input, input.size(-1), w1);
  check_bias(op, "bias1", input, b1, w1.size(0));
  check_weight(op, "weight2", input, w1.size(0), w2);
  check_bias(op, "bias2", input, b2, w2.size(0));
  const bool identity = has(residual) && residual->is_same(input) && w2.size(0) == input.size(-1);
  const OptTensor res = identity ? OptTensor() : check_residual(op, input, residual, w2.size(0));
  if (at::GradMode::is_enabled() &&
      (needs(input) || needs(w1) || needs(b1) || needs(w2) || needs(b2) || needs(res)))
    return FeedForwardNode::apply(input, w1, b1, w2, b2, res, act, identity);
  const Tensor h = linear_forward(input, w1, b1, std::nullopt, (int)act, false).first;
  return linear_forward(h, w2, b2, identity ? OptTensor(input) : res, DCN_ACT_NONE, false).first;
}

// ---- layer norm -------------------------------------------------------------------------------

std::pair<Tensor, Tensor> norm_forward(const Tensor &x, const OptTensor &w, const OptTensor &b, int64_t cols,
                                       double eps, bool save) {
  const int code = dtype_code("layer_norm", x.scalar_type());
  const c10::cuda::CUDAGuard guard(x.device());
  const int dev = x.device().index();
  const Rows xr(x, cols);
  Tensor y = at::empty(x.sizes(), x.options()), stats;
  if (save) stats = at::empty({3, xr.rows}, x.options().dtype(at::kFloat));
  const int wcode = has(w) ? dtype_code("layer_norm", w->scalar_type()) : has(b) ? dtype_code("layer_norm", b->scalar_type()) : code;
  check(dcn_layer_norm_forward(xr.p, xr.ld, ptr(w), ptr(b), out_ptr(y), (float *)out_ptr(stats), code, wcode, xr.rows,
                               cols, (float)eps, dev, c10::cuda::getCurrentCUDAStream(dev).stream()));
  return {y, stats};
}

struct NormNode : torch::autograd::Function<NormNode> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const OptTensor &w, const OptTensor &b, int64_t cols,
                        double eps) {
    auto [y, stats] = norm_forward(x, w, b, cols, eps, true);
    ctx->saved_data["cols"] = cols;
    ctx->saved_data["w"] = has(w);
    ctx->saved_data["b"] = has(b);
    const Tensor &p = has(w) ? *w : has(b) ? *b : x;
    ctx->saved_data["type"] = (int64_t)p.scalar_type();
    ctx->saved_data["shape"] = p.sizes().vec();
    ctx->save_for_backward({x, has(w) ? *w : Tensor(), stats});
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list gys) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0];
    const int64_t cols = ctx->saved_data["cols"].toInt();
    const bool hw = ctx->saved_data["w"].toBool(), hb = ctx->saved_data["b"].toBool();
    variable_list out(5);
    if (!gys[0].defined()) return out;
    const c10::cuda::CUDAGuard guard(x.device());
    const int dev = x.device().index();
    const at::ScalarType type = (at::ScalarType)ctx->saved_data["type"].toInt();
    const auto shape = ctx->saved_data["shape"].toIntVector();
    const auto options = x.options().dtype(type);
    if (ctx->needs_input_grad(0)) out[0] = at::empty(x.sizes(), x.options());
    if (hw && ctx->needs_input_grad(1)) out[1] = at::empty(shape, options);
    if (hb && ctx->needs_input_grad(hw ? 2 : 1)) out[2] = at::empty(shape, options);
    const Rows gr(gys[0], cols), xr(x, cols);
    size_t bytes = 0;
    if (out[1].defined() || out[2].defined()) check(dcn_layer_norm_workspace_bytes(xr.rows, cols, &bytes));
    const Tensor ws = workspace(x, bytes);
    check(dcn_layer_norm_backward(gr.p, gr.ld, xr.p, xr.ld, s[1].defined() ? s[1].const_data_ptr() : nullptr,
                                  (const float *)s[2].const_data_ptr(), out_ptr(out[0]), out_ptr(out[1]),
                                  out_ptr(out[2]), dtype_code("layer_norm", x.scalar_type()),
                                  dtype_code("layer_norm", type), xr.rows, cols, dev, out_ptr(ws), bytes,
                                  c10::cuda::getCurrentCUDAStream(dev).stream()));
    return once("layer_norm", std::move(out));
  }
};

Tensor layer_norm(const Tensor &input, const std::vector<int64_t> &shape, const OptTensor &weight,
                  const OptTensor &bias, double eps) {
  const char *op = "layer_norm";
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
  const OptTensor w = has(weight) ? OptTensor(weight->contiguous()) : OptTensor();
  const OptTensor b = has(bias) ? OptTensor(bias->contiguous()) : OptTensor();
  if (at::GradMode::is_enabled() && (needs(input) || needs(w) || needs(b)))
    return NormNode::apply(input, w, b, cols, eps);
  return norm_forward(input, w, b, cols, eps, false).first;
}

}  // namespace

PYBIND11_MODULE(_layers_native, m) {
  namespace py = pybind11;
  m.def("fused_linear", &fused_linear);
  m.def("feed_forward", &feed_forward);
  m.def("layer_norm", &layer_norm);
  m.def("set_check_status", [](bool flag) { g_check_status.store(flag); });
}
