// The host side of optimi_b200/activations.py: argument checks, buffers, autograd nodes, and the calls of the C ABI in
// include/optimi_b200.h.  Everything below could be Python over ctypes and was at first; a layer's forward and backward pass
// then cost the host 40 to 60 us more than the plain layer's (12 linear layers 1151 against 682 us), which is more than the
// kernels of a small layer take.
#include <torch/extension.h>

#include <ATen/SavedTensorHooks.h>
#include <ATen/autocast_mode.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/PyInterpreter.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "../../include/optimi_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kGroup = 32;  // channels that share an exponent byte

std::optional<Tensor> some(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
Tensor or_none(const std::optional<Tensor>& t) { return t ? *t : Tensor(); }

void check_rc(int rc) { TORCH_CHECK(rc == 0, "optimi_b200 (code ", rc, "): ", optimi_b200_last_error()); }

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return OPTIMI_F32;
    case at::kBFloat16: return OPTIMI_BF16;
    case at::kHalf: return OPTIMI_F16;
    default: return -1;
  }
}

void refuse_tracing(const char* name) {
  // a trace would record the buffers without the kernel that fills them
  TORCH_CHECK(!torch::jit::tracer::isTracing(), name, ": the kernels cannot be recorded by torch.jit.trace");
}

std::string type_name(const Tensor& t) { return "torch." + std::string(c10::getDtypeNames(t.scalar_type()).first); }

void check(const char* name, const char* what, const Tensor& t, const Tensor* like = nullptr) {
  TORCH_CHECK(t.is_cuda(), name, ": `", what, "` lives on ", t.device(), "; optimi_b200 takes CUDA tensors only (there is no CPU path)");
  TORCH_CHECK(dtype_code(t.scalar_type()) >= 0, name, ": `", what, "` has unsupported dtype ", type_name(t), " (float32, bfloat16 and float16 are)");
  TORCH_CHECK(t.layout() == at::kStrided, name, ": `", what, "` must be a dense tensor");
  if (like)
    TORCH_CHECK(t.device() == like->device() && t.scalar_type() == like->scalar_type(), name, ": `", what, "` (", type_name(t), ", ", t.device(),
                ") does not match ", type_name(*like), " on ", like->device());
}

int64_t rows_of(at::IntArrayRef shape) {
  int64_t n = 1;
  for (size_t i = 0; i + 1 < shape.size(); i++) n *= shape[i];
  return n;
}

int64_t groups_of(int64_t cols) { return (cols + kGroup - 1) / kGroup; }

// `t` as a matrix of its last dimension whose rows are contiguous and do not overlap: itself where that holds, else a copy.
Tensor as_rows(const Tensor& given) {
  Tensor t = given.detach();
  if (t.is_neg()) t = t.resolve_neg();  // a lazily negated view: its memory holds the opposite
  if (t.dim() != 2) t = t.reshape({rows_of(t.sizes()), t.size(-1)});
  if (t.is_contiguous()) return t;
  if ((t.size(1) != 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < t.size(1))) t = t.contiguous();
  return t;
}

// A norm's weight or the scale of the channels: its values one after another in memory (not those of a lazily negated view).
Tensor as_channels(const Tensor& t) { return t.defined() ? t.detach().resolve_neg().contiguous() : Tensor(); }

Tensor dense_like(const Tensor& t) { return at::empty(t.sizes(), t.options().memory_format(at::MemoryFormat::Contiguous)); }
Tensor bytes(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte)); }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// Where codes and exponents lie: in one buffer (codes, exponents, and behind them, at the next 16 bytes, a norm's 1 / rms), or in
// two tensors of the caller's.
struct Kept {
  void* codes;
  int64_t pitch;
  void* exponents;
  int64_t epitch;
};

int64_t buffer_bytes(int64_t rows, int64_t cols) { return rows * groups_of(cols) * (kGroup + 1); }
int64_t behind(int64_t n) { return (n + 15) / 16 * 16; }

Kept kept_in(const Tensor& buffer, int64_t rows, int64_t cols) {
  char* at = static_cast<char*>(buffer.data_ptr());
  const int64_t groups = groups_of(cols);
  return {at, groups * kGroup, at + rows * groups * kGroup, groups};
}

Kept kept_in(const std::vector<Tensor>& tensors, int64_t rows, int64_t cols) {
  if (tensors.size() == 1) return kept_in(tensors[0], rows, cols);
  if (rows <= 1) return {tensors[0].data_ptr(), groups_of(cols) * kGroup, tensors[1].data_ptr(), groups_of(cols)};  // strides of one row mean nothing
  return {tensors[0].data_ptr(), tensors[0].stride(0), tensors[1].data_ptr(), tensors[1].stride(0)};
}

Tensor compress(const Tensor& x) {
  refuse_tracing("compress");
  check("compress", "x", x);
  TORCH_CHECK(x.dim() > 0, "compress: `x` must have at least one dimension");
  c10::cuda::CUDAGuard guard(x.device());
  const Tensor m = as_rows(x);
  const Tensor buffer = bytes(buffer_bytes(m.size(0), m.size(1)), x);
  const Kept k = kept_in(buffer, m.size(0), m.size(1));
  check_rc(optimi_b200_compress(m.data_ptr(), m.stride(0), m.size(0), m.size(1), dtype_code(x.scalar_type()), k.codes, k.pitch, k.exponents,
                                k.epitch, stream_of(x)));
  return buffer;
}

Tensor decompress(const std::vector<Tensor>& tensors, const std::vector<int64_t>& shape, at::ScalarType dtype, const std::optional<Tensor>& scale) {
  refuse_tracing("decompress");
  TORCH_CHECK(tensors[0].is_cuda(), "decompress: `saved` lives on ", tensors[0].device(), "; optimi_b200 takes CUDA tensors only (there is no CPU path)");
  c10::cuda::CUDAGuard guard(tensors[0].device());
  const Tensor out = at::empty(shape, tensors[0].options().dtype(dtype));
  const Tensor s = as_channels(or_none(scale));
  const int64_t rows = rows_of(shape), cols = shape.back();
  const Kept k = kept_in(tensors, rows, cols);
  check_rc(optimi_b200_decompress(k.codes, k.pitch, k.exponents, k.epitch, ptr(s), rows, cols, dtype_code(dtype), out.data_ptr(), stream_of(out)));
  return out;
}

// grad^T @ (what `tensors` hold: a (rows, channels) matrix of grad's type).
Tensor weight_gradient_of(const Tensor& grad, const std::vector<Tensor>& tensors, int64_t channels, const Tensor& scale) {
  c10::cuda::CUDAGuard guard(grad.device());
  Tensor m = as_rows(grad);
  const int64_t rows = m.size(0), outputs = m.size(1), pitch = (outputs + 7) / 8 * 8;
  const int code = dtype_code(grad.scalar_type());
  void* stream = stream_of(grad);
  int64_t stride = rows > 1 ? m.stride(0) : pitch;
  if (reinterpret_cast<uintptr_t>(m.data_ptr()) % 16 || (rows > 1 ? stride : outputs) % 8) {  // the kernel loads rows that begin on 16 bytes
    const Tensor copy = at::empty({rows, pitch}, m.options());
    check_rc(optimi_b200_align_rows(m.data_ptr(), m.stride(0), rows, outputs, code, copy.data_ptr(), pitch, stream));
    m = copy, stride = pitch;
  }
  const Tensor dw = at::empty({outputs, channels}, m.options());
  const size_t need = optimi_b200_weight_gradient_workspace_bytes(rows, outputs, channels);
  const Tensor workspace = need ? bytes((int64_t)need, m) : Tensor();
  const Tensor s = as_channels(scale);
  const Kept k = kept_in(tensors, rows, channels);
  check_rc(optimi_b200_weight_gradient(m.data_ptr(), stride, k.codes, k.pitch, k.exponents, k.epitch, ptr(s), rows, outputs, channels, code,
                                       dw.data_ptr(), ptr(workspace), need, stream));
  return dw;
}

Tensor weight_gradient(const Tensor& grad, const std::vector<Tensor>& tensors, const std::vector<int64_t>& shape, at::ScalarType dtype,
                       const std::optional<Tensor>& scale) {
  const char* name = "weight_gradient";
  refuse_tracing(name);
  check(name, "grad", grad);
  TORCH_CHECK(grad.scalar_type() != at::kFloat, name, ": `grad` is float32; bfloat16 and float16 are supported");
  TORCH_CHECK(dtype == grad.scalar_type() && tensors[0].device() == grad.device(), name, ": `saved` (torch.", c10::getDtypeNames(dtype).first,
              ", ", tensors[0].device(), ") does not match `grad` (", type_name(grad), ", ", grad.device(), ")");
  TORCH_CHECK(grad.dim() > 0 && rows_of(grad.sizes()) == rows_of(shape), name, ": `grad` ", grad.sizes(), " and `saved` ", at::IntArrayRef(shape),
              " have different numbers of tokens");
  return weight_gradient_of(grad, tensors, shape.back(), or_none(scale));
}

void refuse_double_backward(const char* name) {
  // gradients are recorded inside a backward pass only under create_graph=True, and these kernels' would come out as constants
  TORCH_CHECK(!at::GradMode::is_enabled(), name, ": differentiating the backward pass (create_graph=True) is not supported");
}

void refuse_tangent(const char* name, const char* what, const Tensor& t) {
  // forward mode needs no input that requires a gradient, so the way past the node would drop the tangent without a word
  TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), name, ": `", what, "` carries a forward-mode tangent; forward-mode differentiation is not supported");
}

struct Normed {
  Tensor output, sum, buffer;
};

Normed norm_forward(const Tensor& x, const Tensor& weight, const Tensor& residual, double eps, bool keep) {
  c10::cuda::CUDAGuard guard(x.device());
  const Tensor m = as_rows(x), r = residual.defined() ? as_rows(residual) : Tensor();
  const Tensor w = as_channels(weight);
  const int64_t rows = m.size(0), cols = m.size(1);
  Normed out;
  out.output = dense_like(x);
  if (r.defined()) out.sum = dense_like(x);
  Kept k = {nullptr, 0, nullptr, 0};
  float* rstd = nullptr;
  if (keep) {
    const int64_t at = behind(buffer_bytes(rows, cols));
    out.buffer = bytes(at + 4 * rows, x);
    k = kept_in(out.buffer, rows, cols);
    rstd = reinterpret_cast<float*>(static_cast<char*>(out.buffer.data_ptr()) + at);
  }
  check_rc(optimi_b200_rms_norm(m.data_ptr(), m.stride(0), ptr(r), r.defined() ? r.stride(0) : 0, ptr(w), rows, cols, eps,
                                dtype_code(x.scalar_type()), out.output.data_ptr(), ptr(out.sum), k.codes, k.pitch, k.exponents, k.epitch, rstd,
                                stream_of(x)));
  return out;
}

struct RMSNormNode : torch::autograd::Function<RMSNormNode> {
  // inputs that are not given do not count among the node's
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight_, const std::optional<Tensor>& residual,
                               double eps) {
    const Tensor weight = or_none(weight_);
    const Normed out = norm_forward(x, weight, or_none(residual), eps, true);
    ctx->save_for_backward({out.buffer, weight});
    ctx->mark_non_differentiable({out.buffer});
    ctx->set_materialize_grads(false);
    if (out.sum.defined()) return {out.output, out.buffer, out.sum};
    return {out.output, out.buffer};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_double_backward("rms_norm");
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &buffer = saved[0], &weight = saved[1], &grad = grads[0];
    const bool has_sum = grads.size() > 2;
    const Tensor grad_sum = has_sum ? grads[2] : Tensor();
    const bool need_x = ctx->needs_input_grad(0), need_w = weight.defined() && ctx->needs_input_grad(1),
               need_r = has_sum && ctx->needs_input_grad(weight.defined() ? 2 : 1);
    if (!grad.defined()) {  // only the residual was used: it passes through
      const Tensor dw = need_w ? at::zeros_like(weight) : Tensor();
      return {need_x ? grad_sum : Tensor(), dw, need_r ? grad_sum : Tensor(), Tensor()};
    }
    c10::cuda::CUDAGuard guard(grad.device());
    const Tensor g = as_rows(grad), s = grad_sum.defined() ? as_rows(grad_sum) : Tensor();
    const Tensor w = as_channels(weight);
    const int64_t rows = g.size(0), cols = g.size(1);
    const int code = dtype_code(grad.scalar_type());
    const Tensor dx = need_x || need_r ? dense_like(grad) : Tensor(), dw = need_w ? at::empty({cols}, g.options()) : Tensor();
    const size_t need = need_w ? optimi_b200_rms_norm_backward_workspace_bytes(rows, cols, code) : 0;
    const Tensor workspace = need ? bytes((int64_t)need, g) : Tensor();
    const Kept k = kept_in(buffer, rows, cols);
    const float* rstd = reinterpret_cast<const float*>(static_cast<const char*>(buffer.data_ptr()) + behind(buffer_bytes(rows, cols)));
    check_rc(optimi_b200_rms_norm_backward(g.data_ptr(), g.stride(0), ptr(s), s.defined() ? s.stride(0) : 0, k.codes, k.pitch, k.exponents,
                                           k.epitch, rstd, ptr(w), rows, cols, code, ptr(dx), ptr(dw), ptr(workspace), need, stream_of(grad)));
    return {need_x ? dx : Tensor(), dw, need_r ? dx : Tensor(), Tensor()};
  }
};

// (output, updated residual, buffer of the 8-bit row)
std::tuple<Tensor, std::optional<Tensor>, std::optional<Tensor>> rms_norm(const Tensor& x, const std::optional<Tensor>& weight_,
                                                                          const std::optional<Tensor>& residual_, std::optional<double> eps_,
                                                                          bool keep) {
  const char* name = "rms_norm";
  refuse_tracing(name);
  const Tensor weight = or_none(weight_), residual = or_none(residual_);
  check(name, "x", x);
  TORCH_CHECK(x.dim() > 0, name, ": `x` must have at least one dimension");
  if (weight.defined()) {
    check(name, "weight", weight, &x);
    TORCH_CHECK(weight.dim() == 1 && weight.size(0) == x.size(-1), name, ": `weight` ", weight.sizes(), " does not match the last dimension of `x` ",
                x.sizes());
  }
  if (residual.defined()) {
    check(name, "residual", residual, &x);
    TORCH_CHECK(residual.sizes() == x.sizes(), name, ": `residual` ", residual.sizes(), " does not match `x` ", x.sizes());
  }
  const double eps = eps_ ? *eps_ : 0x1p-23;  // float32's epsilon for 16-bit types too, as in torch.nn.RMSNorm
  TORCH_CHECK_VALUE(eps >= 0, name, ": eps=", eps, " must not be negative");
  refuse_tangent(name, "x", x), refuse_tangent(name, "weight", weight), refuse_tangent(name, "residual", residual);
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || (weight.defined() && weight.requires_grad()) || (residual.defined() && residual.requires_grad()))) {
    const variable_list out = RMSNormNode::apply(x, some(weight), some(residual), eps);
    return {out[0], some(out.size() > 2 ? out[2] : Tensor()), out[1]};
  }
  const Normed out = norm_forward(x, weight, residual, eps, keep);
  return {out.output, some(out.sum), some(out.buffer)};
}

// The 8-bit form of a layer's input, where the caller has it (no tensors: none).
struct Saved {
  std::vector<Tensor> tensors;
  Tensor scale;
};

struct LinearNode : torch::autograd::Function<LinearNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias, const Saved& saved) {
    const Tensor out = at::linear(x, weight, bias);
    // not ctx->needs_input_grad: inside a backward pass (recomputation) that answers for the pass under way
    const bool need_x = x.requires_grad(), need_w = weight.requires_grad();
    ctx->saved_data["channels"] = x.size(-1);
    ctx->saved_data["bias"] = bias.has_value();
    variable_list keep = {need_x ? weight : Tensor(), need_w ? saved.scale : Tensor()};
    if (need_w) {
      if (saved.tensors.empty()) keep.push_back(compress(x));
      else keep.insert(keep.end(), saved.tensors.begin(), saved.tensors.end());
    }
    ctx->save_for_backward(std::move(keep));
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_double_backward("linear");
    const variable_list kept = ctx->get_saved_variables();
    const Tensor& grad = grads[0];
    Tensor dx, dw, db;
    if (grad.defined()) {
      if (ctx->needs_input_grad(0)) dx = at::matmul(grad, kept[0]);
      if (ctx->needs_input_grad(1)) dw = weight_gradient_of(grad, {kept.begin() + 2, kept.end()}, ctx->saved_data["channels"].toInt(), kept[1]);
      if (ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2)) db = grad.reshape({rows_of(grad.sizes()), grad.size(-1)}).sum(0);
    }
    return {dx, dw, db, Tensor()};
  }
};

Tensor linear(const Tensor& x_, const Tensor& weight_, const std::optional<Tensor>& bias_, const std::vector<Tensor>& tensors,
              const std::vector<int64_t>& shape, std::optional<at::ScalarType> dtype, const std::optional<Tensor>& scale) {
  const char* name = "linear";
  if (at::GradMode::is_enabled()) refuse_tracing(name);
  Tensor x = x_, weight = weight_, bias = or_none(bias_);
  if (at::autocast::is_autocast_enabled(at::kCUDA) && x.is_cuda()) {
    const at::ScalarType to = at::autocast::get_autocast_dtype(at::kCUDA);
    const auto cast = [&](const Tensor& t) { return t.is_cuda() && t.is_floating_point() && t.scalar_type() != at::kDouble ? t.to(to) : t; };
    x = cast(x), weight = cast(weight);
    if (bias.defined()) bias = cast(bias);
  }
  check(name, "x", x);
  check(name, "weight", weight, &x);
  if (bias.defined()) check(name, "bias", bias, &x);
  TORCH_CHECK(x.scalar_type() != at::kFloat, name, ": float32 is not supported (bfloat16 and float16 are); use torch.nn.functional.linear");
  TORCH_CHECK(x.dim() > 0 && weight.dim() == 2 && x.size(-1) == weight.size(1), name, ": `x` ", x.sizes(), " and `weight` ", weight.sizes(),
              " do not match");
  TORCH_CHECK(!bias.defined() || (bias.dim() == 1 && bias.size(0) == weight.size(0)), name, ": `bias` ", bias.sizes(), " does not match `weight` ",
              weight.sizes());
  if (!tensors.empty())
    TORCH_CHECK(rows_of(shape) == rows_of(x.sizes()) && shape.back() == x.size(-1) && dtype == x.scalar_type() && tensors[0].device() == x.device(),
                name, ": `saved` (", at::IntArrayRef(shape), ", torch.", c10::getDtypeNames(*dtype).first, ", ", tensors[0].device(),
                ") does not stand for `x` (", x.sizes(), ", ", type_name(x), ", ", x.device(), ")");
  if (!at::GradMode::is_enabled()) return at::linear(x, weight, some(bias));
  c10::cuda::CUDAGuard guard(x.device());
  // The backward pass reads the row on this stream, and whoever made it on another one does not know of that: a prepared norm's
  // row is not even seen by the caller.
  for (const Tensor& t : tensors) c10::cuda::CUDACachingAllocator::recordStream(t.storage().data_ptr(), c10::cuda::getCurrentCUDAStream(x.device().index()));
  return LinearNode::apply(x, weight, some(bias), Saved{tensors, or_none(scale)});
}

// The function that tensors saved for a backward pass go through now (None: they are kept as they are).
py::object saving_hook() {
  const auto hooks = at::SavedTensorDefaultHooks::get_hooks();
  return hooks ? py::reinterpret_borrow<py::object>(hooks->first.ptr(getPyInterpreter())) : py::none();
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("compress", torch::wrap_pybind_function_no_gil(compress));
  m.def("decompress", torch::wrap_pybind_function_no_gil(decompress));
  m.def("weight_gradient", torch::wrap_pybind_function_no_gil(weight_gradient));
  m.def("rms_norm", torch::wrap_pybind_function_no_gil(rms_norm));
  m.def("linear", torch::wrap_pybind_function_no_gil(linear));
  m.def("saving_hook", saving_hook);
}
