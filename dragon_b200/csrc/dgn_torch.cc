// Python calls of the norm and expert operators on torch tensors: checks of the
// arguments, outputs from torch's allocator, the current stream, and one call of
// the C-ABI each.  A call through ctypes spends 10 to 25 us on the host with its
// allocations, several times what the kernel of a small batch takes; this one 5 to 8.
//
// Refusals are ValueError and TypeError as elsewhere in the package; a status of
// the C-ABI becomes dragon_b200._C.DgnError.  Works on shapes, types and addresses
// alone: nothing is copied, converted or synchronised, no autograd graph is recorded (of
// which a caller whose inputs require gradients is told once).
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <initializer_list>
#include <optional>
#include <string>
#include <tuple>

#include "../../include/dgn.h"

namespace py = pybind11;
using at::ScalarType;
using at::Tensor;
typedef std::optional<Tensor> MaybeTensor;

namespace {

std::string name_of(ScalarType t) { return py::str(py::cast(t)).cast<std::string>(); }
std::string name_of(at::IntArrayRef shape) {
  std::string s = "(";
  for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
  return s + (shape.size() == 1 ? ",)" : ")");
}
[[noreturn]] void value_error(const std::string& what) { throw py::value_error(what); }
[[noreturn]] void type_error(const std::string& what) { throw py::type_error(what); }
[[noreturn]] void unsupported(const char* name, ScalarType t) {
  type_error(std::string("Unsupported data type of <") + name + ">: " + name_of(t));
}

// -1 for a type that the operators do not take.
int dgn_type(ScalarType t) {
  switch (t) {
    case ScalarType::Half: return DGN_F16;
    case ScalarType::BFloat16: return DGN_BF16;
    case ScalarType::Float: return DGN_F32;
    default: return -1;
  }
}

void check(int status) {
  if (status != DGN_OK) py::module_::import("dragon_b200._C").attr("check")(status);
}

Tensor empty(at::IntArrayRef shape, ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(shape, type, like.device(), std::nullopt);
}
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
const void* address(const MaybeTensor& t) { return t ? t->const_data_ptr() : nullptr; }

void check_cuda(const Tensor& t, const char* name) {
  if (!t.is_cuda()) value_error(std::string("<") + name + "> must be a CUDA tensor (got " + t.device().str() + ")");
}
// Views that stand for other values than their memory holds (x.conj(), the imaginary part of one).
void check_plain(const Tensor& t, const char* name) {
  if (t.is_conj() || t.is_neg())
    value_error(std::string("<") + name + "> is a conjugate or negative view: resolve_conj() and resolve_neg() make its values");
}
void check_device(const Tensor& t, const Tensor& like, const char* name) {
  if (t.device() != like.device())
    value_error(std::string("<") + name + "> must live on " + like.device().str() + " (got " + t.device().str() + ")");
}
void check_shape(const Tensor& t, at::IntArrayRef shape, const char* name) {
  if (t.sizes() != shape)
    value_error(std::string("<") + name + "> must have the shape " + name_of(shape) + ", got " + name_of(t.sizes()));
}
// A contiguous tensor of one device, shape and type.
void check_exactly(const Tensor& t, const Tensor& like, at::IntArrayRef shape, ScalarType type, const char* name) {
  if (t.scalar_type() != type) unsupported(name, t.scalar_type());
  check_plain(t, name);
  check_device(t, like, name);
  check_shape(t, shape, name);
  if (!t.is_contiguous()) value_error(std::string("<") + name + "> must be contiguous");
}

// Rows that lie at one distance: a matrix, or more dimensions that fold into one.
struct Rows {
  int64_t rows, cols, stride;
};
Rows rows_of(const Tensor& t, const char* name) {
  const std::string n = std::string("<") + name + ">";
  if (t.dim() == 0) value_error(n + " needs at least one dimension");
  check_plain(t, name);
  const int64_t cols = t.size(-1);
  if (t.is_contiguous()) return {cols ? t.numel() / cols : 0, cols, cols};
  if (t.stride(-1) != 1 && cols > 1) value_error("the last dimension of " + n + " must be contiguous");
  int64_t stride = 0, rows = 1;
  for (int64_t d = t.dim() - 2; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (rows == 1) stride = t.stride(d);
    else if (t.stride(d) != stride * rows) value_error("the rows of " + n + " must lie at one distance");
    rows *= t.size(d);
  }
  if (rows == 1) stride = cols;
  if (stride < cols) value_error("the rows of " + n + " must not overlap");
  return {rows, cols, stride};
}
// Row stride of a CUDA matrix of one of the three types.
int64_t matrix(const Tensor& t, const char* name, bool any_type = false) {
  if (!any_type && dgn_type(t.scalar_type()) < 0) unsupported(name, t.scalar_type());
  if (t.dim() != 2) value_error(std::string("<") + name + "> must have two dimensions");
  check_cuda(t, name);
  return rows_of(t, name).stride;
}

const Tensor* maybe(const MaybeTensor& t) { return t ? &*t : nullptr; }
// One warning of the process, for the mistake of taking a forward call for one that autograd follows.
void tell_of_no_graph(const char* call, const char* backward, std::initializer_list<const Tensor*> inputs) {
  static bool told = false;
  if (told || !at::GradMode::is_enabled()) return;
  for (const Tensor* t : inputs) {
    if (!t || !t->requires_grad()) continue;
    const std::string what = std::string(call) + ": an input requires a gradient, but the call records no autograd graph; its backward pass is " +
                             backward + " (call both in a torch.autograd.Function, or the forward call under torch.no_grad())";
    if (PyErr_WarnEx(PyExc_UserWarning, what.c_str(), 1) != 0) throw py::error_already_set();
    told = true;
    return;
  }
}

// ---- norm ------------------------------------------------------------------------------

void check_norm_input(const Tensor& x, const char* name) {
  if (dgn_type(x.scalar_type()) < 0) type_error("Unsupported data type: " + name_of(x.scalar_type()));
  check_cuda(x, name);
}
void check_like(const Tensor& t, const Tensor& x, const char* name) {
  check_device(t, x, name);
  check_shape(t, x.sizes(), name);
  if (t.scalar_type() != x.scalar_type()) unsupported(name, t.scalar_type());
}
void check_weight(const Tensor& weight, const Tensor& x, int64_t cols) {
  if (weight.scalar_type() != x.scalar_type() && weight.scalar_type() != ScalarType::Float)
    type_error("<weight> must be float32 or " + name_of(x.scalar_type()) + ", got " + name_of(weight.scalar_type()));
  check_plain(weight, "weight");
  check_device(weight, x, "weight");
  if (weight.dim() != 1 || weight.size(0) != cols || !weight.is_contiguous())
    value_error("<weight> must be a contiguous vector of " + std::to_string(cols) + " elements");
}

std::tuple<Tensor, Tensor, Tensor, MaybeTensor> rms_norm(const Tensor& x, const MaybeTensor& weight,
                                                          const MaybeTensor& residual, double eps,
                                                          std::optional<ScalarType> out_type, int64_t group,
                                                          bool in_place) {
  check_norm_input(x, "x");
  tell_of_no_graph("rms_norm", "rms_norm_grad", {&x, maybe(weight), maybe(residual)});
  const Rows r = rows_of(x, "x");
  if (!(eps >= 0x1p-126) || eps > 3.4e38) value_error("<eps> must be a positive number, 2^-126 at least");
  if (group != 0 && group != 32 && group != 64 && group != 128)
    value_error("<group_size> must be one of (0, 32, 64, 128), got " + std::to_string(group));
  const ScalarType type = x.scalar_type(), out = out_type.value_or(type);
  int code = DGN_CODE_NONE;
  if (out != type) {
    code = out == ScalarType::Char            ? DGN_CODE_I8
           : out == ScalarType::Float8_e4m3fn ? DGN_CODE_E4M3
           : out == ScalarType::Float8_e5m2   ? DGN_CODE_E5M2
                                              : -1;
    if (code < 0) type_error("Unsupported output type: " + name_of(out));
  }
  if (weight) check_weight(*weight, x, r.cols);
  Tensor hidden = x;
  int64_t residual_stride = 0, hidden_stride = 0;
  if (residual) {
    check_like(*residual, x, "residual");
    residual_stride = rows_of(*residual, "residual").stride;
    hidden = in_place ? *residual : empty(x.sizes(), type, x);
    hidden_stride = in_place ? residual_stride : r.cols;
  } else if (in_place) {
    value_error("<inplace_residual> needs a residual");
  }
  Tensor output = empty(x.sizes(), out, x), rstd = empty(x.sizes().slice(0, x.dim() - 1), ScalarType::Float, x);
  MaybeTensor scale;
  if (code) {
    at::DimVector shape(x.sizes());
    shape.back() = group ? (r.cols + group - 1) / group : 1;
    scale = empty(shape, ScalarType::Float, x);
  }
  check(dgn_rms_norm(x.const_data_ptr(), r.stride, address(residual), residual_stride, address(weight),
                     weight ? dgn_type(weight->scalar_type()) : dgn_type(type),
                     residual ? hidden.mutable_data_ptr() : nullptr, hidden_stride, output.mutable_data_ptr(), code, group,
                     code ? scale->mutable_data_ptr<float>() : nullptr, rstd.mutable_data_ptr<float>(), r.rows, r.cols,
                     (float)eps, dgn_type(type), x.device().index(), stream_of(x)));
  return {output, hidden, rstd, scale};
}

std::tuple<Tensor, MaybeTensor> rms_norm_grad(const Tensor& grad_output, const Tensor& hidden, const Tensor& rstd,
                                              const MaybeTensor& weight, const MaybeTensor& grad_hidden) {
  check_norm_input(hidden, "hidden");
  const Rows r = rows_of(hidden, "hidden");
  check_like(grad_output, hidden, "grad_output");
  const int64_t grad_stride = rows_of(grad_output, "grad_output").stride;
  if (rstd.device() != hidden.device() || rstd.scalar_type() != ScalarType::Float || rstd.numel() != r.rows ||
      !rstd.is_contiguous())
    value_error("<rstd> must be the forward call's");
  int64_t grad_hidden_stride = 0;
  if (grad_hidden) {
    check_like(*grad_hidden, hidden, "grad_hidden");
    grad_hidden_stride = rows_of(*grad_hidden, "grad_hidden").stride;
  }
  const int type = dgn_type(hidden.scalar_type());
  int weight_type = type;
  int64_t bytes = 0;
  MaybeTensor grad_weight;
  Tensor workspace;
  if (weight) {
    check_weight(*weight, hidden, r.cols);
    weight_type = dgn_type(weight->scalar_type());
    grad_weight = empty(weight->sizes(), weight->scalar_type(), hidden);
    bytes = dgn_rms_norm_grad_workspace(r.rows, r.cols, type);
    workspace = empty({bytes}, ScalarType::Byte, hidden);
  }
  Tensor grad_x = empty(hidden.sizes(), hidden.scalar_type(), hidden);
  check(dgn_rms_norm_grad(grad_output.const_data_ptr(), grad_stride, address(grad_hidden), grad_hidden_stride,
                          hidden.const_data_ptr(), r.stride, address(weight), weight_type, rstd.const_data_ptr<float>(),
                          grad_x.mutable_data_ptr(), weight ? grad_weight->mutable_data_ptr() : nullptr,
                          weight ? workspace.mutable_data_ptr() : nullptr, bytes, r.rows, r.cols, type,
                          hidden.device().index(), stream_of(hidden)));
  return {grad_x, grad_weight};
}

// ---- experts ---------------------------------------------------------------------------

void check_experts(int64_t experts) {
  if (experts < 1 || experts > DGN_MAX_EXPERTS)
    value_error("there must be 1 to " + std::to_string(DGN_MAX_EXPERTS) + " experts, got " + std::to_string(experts));
}
void check_choice(int64_t k, int64_t experts) {
  check_experts(experts);
  if (k < 1 || k > DGN_MAX_CHOICES || k > experts)
    value_error("<k> must be 1 to " + std::to_string(DGN_MAX_CHOICES) + " and at most the number of experts, got " +
                std::to_string(k));
}
const float* floats(const MaybeTensor& t) { return t ? t->const_data_ptr<float>() : nullptr; }

std::tuple<Tensor, Tensor> route(const Tensor& logits, int64_t k, const MaybeTensor& bias, const MaybeTensor& mask,
                                 int score, int64_t groups, int64_t keep, int64_t best, bool renormalize, double scale) {
  const int64_t stride = matrix(logits, "logits"), tokens = logits.size(0), experts = logits.size(1);
  check_choice(k, experts);
  tell_of_no_graph("route", "route_grad", {&logits});
  if (groups < 1 || groups > DGN_MAX_GROUPS || experts % groups)
    value_error("<groups> must be 1 to " + std::to_string(DGN_MAX_GROUPS) + " and divide the number of experts");
  if (keep < 1 || keep > groups) value_error("<keep_groups> must be 1 to <groups>, got " + std::to_string(keep));
  if (best != 1 && best != 2) value_error("<group_best> must be 1 or 2, got " + std::to_string(best));
  if (bias) check_exactly(*bias, logits, {experts}, ScalarType::Float, "bias");
  if (mask) check_exactly(*mask, logits, {tokens}, ScalarType::Bool, "mask");
  Tensor indices = empty({tokens, k}, ScalarType::Int, logits), weights = empty({tokens, k}, ScalarType::Float, logits);
  check(dgn_route(logits.const_data_ptr(), stride, floats(bias), static_cast<const uint8_t*>(address(mask)),
                  indices.mutable_data_ptr<int>(), weights.mutable_data_ptr<float>(), tokens, (int)experts, (int)k, score,
                  (int)groups, (int)keep, (int)best, renormalize, (float)scale, dgn_type(logits.scalar_type()),
                  logits.device().index(), stream_of(logits)));
  return {indices, weights};
}

Tensor route_grad(const Tensor& grad_weights, const Tensor& logits, const Tensor& indices, int score, bool renormalize,
                  double scale) {
  const int64_t stride = matrix(logits, "logits"), tokens = logits.size(0), experts = logits.size(1);
  if (indices.dim() != 2) value_error("<indices> must have two dimensions");
  const int64_t k = indices.size(1);
  check_choice(k, experts);
  check_exactly(indices, logits, {tokens, k}, ScalarType::Int, "indices");
  check_exactly(grad_weights, logits, {tokens, k}, ScalarType::Float, "grad_weights");
  Tensor grad = empty({tokens, experts}, logits.scalar_type(), logits);
  check(dgn_route_grad(grad_weights.const_data_ptr<float>(), logits.const_data_ptr(), stride, indices.const_data_ptr<int>(),
                       grad.mutable_data_ptr(), tokens, (int)experts, (int)k, score, renormalize, (float)scale,
                       dgn_type(logits.scalar_type()), logits.device().index(), stream_of(logits)));
  return grad;
}

std::tuple<Tensor, Tensor, Tensor, Tensor> plan(const Tensor& indices, int64_t experts, int64_t align) {
  if (indices.scalar_type() != ScalarType::Int) unsupported("indices", indices.scalar_type());
  matrix(indices, "indices", true);
  if (!indices.is_contiguous()) value_error("<indices> must be contiguous");
  const int64_t tokens = indices.size(0), k = indices.size(1), slots = tokens * k;
  check_experts(experts);
  if (k < 1 || k > DGN_MAX_CHOICES)
    value_error("a token has 1 to " + std::to_string(DGN_MAX_CHOICES) + " choices, got " + std::to_string(k));
  if (align < 1 || align > INT32_MAX || slots > INT32_MAX || slots + std::min(experts, slots) * (align - 1) > INT32_MAX)
    value_error("<align> must be positive and the rows fewer than 2^31");
  Tensor counts = empty({experts}, ScalarType::Int, indices), offsets = empty({experts + 1}, ScalarType::Int, indices),
         ends = empty({experts}, ScalarType::Int, indices), positions = empty({tokens, k}, ScalarType::Int, indices), workspace;
  const int64_t bytes = dgn_expert_plan_workspace(slots, (int)experts);
  if (bytes) workspace = empty({bytes}, ScalarType::Byte, indices);
  check(dgn_expert_plan(indices.const_data_ptr<int>(), slots, (int)experts, (int)align, counts.mutable_data_ptr<int>(),
                        offsets.mutable_data_ptr<int>(), ends.mutable_data_ptr<int>(), positions.mutable_data_ptr<int>(),
                        bytes ? workspace.mutable_data_ptr() : nullptr, bytes, indices.device().index(),
                        stream_of(indices)));
  return {counts, offsets, ends, positions};
}

// A plan's tensors, as plan() made them.
struct Plan {
  const Tensor &offsets, &ends, &positions;
  int64_t tokens() const { return positions.size(0); }
  int64_t k() const { return positions.size(1); }
  int experts() const { return (int)ends.size(0); }
};
void check_plan(const Plan& p, const Tensor& like) {
  if (p.positions.device() != like.device())
    value_error("the plan must live on " + like.device().str() + " (got " + p.positions.device().str() + ")");
}

Tensor dispatch(const Tensor& x, const Tensor& offsets, const Tensor& ends, const Tensor& positions, int64_t capacity,
                const MaybeTensor& to) {
  const Plan p = {offsets, ends, positions};
  const int64_t stride = matrix(x, "x", true), tokens = x.size(0), cols = x.size(1), size = x.element_size();
  check_plan(p, x);
  tell_of_no_graph("dispatch", "dispatch_grad", {&x});
  if (tokens != p.tokens())
    value_error("<x> must have the plan's " + std::to_string(p.tokens()) + " rows, got " + std::to_string(tokens));
  if (cols == 0) value_error("<x> has no columns");
  if (to) {
    if (to->dim() != 2) value_error("<out> must have two dimensions");
    check_exactly(*to, x, {to->size(0), cols}, x.scalar_type(), "out");
  }
  Tensor out = to ? *to : empty({capacity, cols}, x.scalar_type(), x);
  check(dgn_expert_dispatch(x.const_data_ptr(), stride * size, cols * size, positions.const_data_ptr<int>(),
                            offsets.const_data_ptr<int>(), ends.const_data_ptr<int>(), out.mutable_data_ptr(), tokens,
                            (int)p.k(), p.experts(), out.size(0), x.device().index(), stream_of(x)));
  return out;
}

// Checks the experts' rows; their number of columns.
int64_t check_rows(const Tensor& rows, const Plan& p) {
  matrix(rows, "rows");
  if (!rows.is_contiguous()) value_error("<rows> must be contiguous");
  check_plan(p, rows);
  if (rows.size(1) == 0) value_error("<rows> has no columns");
  return rows.size(1);
}
// Row stride of a matrix of the tokens, of the rows' type.
int64_t of_tokens(const Tensor& t, const Tensor& rows, const Plan& p, const char* name) {
  if (t.scalar_type() != rows.scalar_type()) unsupported(name, t.scalar_type());
  const int64_t stride = matrix(t, name);
  check_device(t, rows, name);
  check_shape(t, {p.tokens(), rows.size(1)}, name);
  return stride;
}

Tensor combine(const Tensor& rows, const Tensor& offsets, const Tensor& ends, const Tensor& positions,
               const MaybeTensor& weights, const MaybeTensor& residual) {
  const Plan p = {offsets, ends, positions};
  const int64_t cols = check_rows(rows, p);
  tell_of_no_graph("combine", "combine_grad", {&rows, maybe(weights), maybe(residual)});
  if (weights) check_exactly(*weights, rows, {p.tokens(), p.k()}, ScalarType::Float, "weights");
  const int64_t residual_stride = residual ? of_tokens(*residual, rows, p, "residual") : 0;
  Tensor out = empty({p.tokens(), cols}, rows.scalar_type(), rows);
  check(dgn_expert_combine(rows.const_data_ptr(), positions.const_data_ptr<int>(), floats(weights), address(residual),
                           residual_stride, out.mutable_data_ptr(), p.tokens(), (int)p.k(), cols, rows.size(0),
                           dgn_type(rows.scalar_type()), rows.device().index(), stream_of(rows)));
  return out;
}

std::tuple<Tensor, Tensor> combine_grad(const Tensor& grad_output, const Tensor& rows, const Tensor& offsets,
                                        const Tensor& ends, const Tensor& positions, const Tensor& weights,
                                        const MaybeTensor& to) {
  const Plan p = {offsets, ends, positions};
  const int64_t cols = check_rows(rows, p), stride = of_tokens(grad_output, rows, p, "grad_output");
  check_exactly(weights, rows, {p.tokens(), p.k()}, ScalarType::Float, "weights");
  if (to) check_exactly(*to, rows, rows.sizes(), rows.scalar_type(), "out");
  Tensor out = to ? *to : empty(rows.sizes(), rows.scalar_type(), rows),
         grad_weights = empty(weights.sizes(), ScalarType::Float, rows);
  check(dgn_expert_combine_grad(grad_output.const_data_ptr(), stride, rows.const_data_ptr(),
                                positions.const_data_ptr<int>(), weights.const_data_ptr<float>(),
                                offsets.const_data_ptr<int>(), ends.const_data_ptr<int>(), out.mutable_data_ptr(),
                                grad_weights.mutable_data_ptr<float>(), p.tokens(), (int)p.k(), p.experts(), cols,
                                rows.size(0), dgn_type(rows.scalar_type()), rows.device().index(), stream_of(rows)));
  return {out, grad_weights};
}

Tensor update_bias(const Tensor& bias, const Tensor& counts, double rate, const MaybeTensor& to) {
  if (bias.dim() != 1 || bias.size(0) < 1 || bias.size(0) > DGN_MAX_EXPERTS)
    value_error("<bias> must be a vector of 1 to " + std::to_string(DGN_MAX_EXPERTS) + " elements");
  check_cuda(bias, "bias");
  check_exactly(bias, bias, bias.sizes(), ScalarType::Float, "bias");
  check_exactly(counts, bias, bias.sizes(), ScalarType::Int, "counts");
  if (to) check_exactly(*to, bias, bias.sizes(), ScalarType::Float, "out");
  Tensor out = to ? *to : bias;
  check(dgn_expert_update_bias(bias.const_data_ptr<float>(), counts.const_data_ptr<int>(), out.mutable_data_ptr<float>(),
                               (int)bias.size(0), (float)rate, bias.device().index(), stream_of(bias)));
  return out;
}

}  // namespace

PYBIND11_MODULE(dgn_torch, m) {
  m.def("rms_norm", &rms_norm);
  m.def("rms_norm_grad", &rms_norm_grad);
  m.def("route", &route);
  m.def("route_grad", &route_grad);
  m.def("plan", &plan);
  m.def("dispatch", &dispatch);
  m.def("combine", &combine);
  m.def("combine_grad", &combine_grad);
  m.def("update_bias", &update_bias);
}
