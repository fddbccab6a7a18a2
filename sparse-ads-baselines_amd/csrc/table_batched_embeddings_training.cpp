// Expert routing, gradient clipping and the clipped table updates of the pybind11 module
// table_batched_embeddings_cpp (no counterpart in the reference).  Host code over the C ABI: checks, outputs,
// autograd; the kernels are in the library.  The smallest calls are bound by what the host does for them,
// which is why these operators live here and not in the ctypes module.
//
// Scratch memory that a call needs comes from PyTorch's allocator for that call alone: calls on different streams, and
// graphs captured on one stream and replayed on several, share none of it.
#include "table_batched_embeddings_binding.h"

#include <torch/csrc/autograd/custom_function.h>

#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>

#include <cmath>
#include <limits>
#include <tuple>
#include <vector>

namespace tbe_binding {
namespace {

namespace py = pybind11;

// element types of expert routing and clipping: those of the tables and bfloat16
int32_t float_code(const at::Tensor &t, const char *name) {
  switch (t.scalar_type()) {
    case at::kFloat: return TBE_DTYPE_F32;
    case at::kHalf: return TBE_DTYPE_F16;
    case at::kDouble: return TBE_DTYPE_F64;
    case at::kBFloat16: return TBE_DTYPE_BF16;
    default: TORCH_CHECK(false, name, " must be float16, bfloat16, float32 or float64");
  }
  return -1;
}

// An uninitialised tensor on the device of `like`, straight from the allocator (a third of the host time of a call
// through the dispatcher, which would end up there).
at::Tensor empty_on(const at::Tensor &like, at::IntArrayRef sizes, at::ScalarType type) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt));
}

// Part of `whole` as a tensor of its own: several outputs of one call share an allocation.
at::Tensor part_of(const at::Tensor &whole, int64_t offset, at::IntArrayRef sizes) {
  at::Tensor part = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), whole.dtype());
  part.unsafeGetTensorImpl()->set_storage_offset(offset);
  part.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return part;
}

// ------------------------------------------------------------------------------ expert routing
struct Plan {
  int64_t tokens;
  int32_t choices, experts;
};

Plan check_plan(const at::Tensor &places, const at::Tensor &expert_offsets, const at::Device &device) {
  TORCH_CHECK(places.scalar_type() == at::kInt && expert_offsets.scalar_type() == at::kInt,
              "places and expert_offsets must be int32");
  TORCH_CHECK(places.device() == device && expert_offsets.device() == device,
              "places and expert_offsets must live on the rows' device");
  TORCH_CHECK(places.dim() == 2 && places.is_contiguous() && places.size(1) > 0,
              "places must be a contiguous [tokens, choices] tensor with choices > 0");
  TORCH_CHECK(expert_offsets.dim() == 1 && expert_offsets.is_contiguous() && expert_offsets.numel() > 1,
              "expert_offsets must be a contiguous 1-D tensor of num_experts + 1 entries");
  TORCH_CHECK(places.numel() < std::numeric_limits<int32_t>::max() &&
                  expert_offsets.numel() < std::numeric_limits<int32_t>::max(),
              "tokens * choices must stay below 2^31 - 1");
  return Plan{places.size(0), static_cast<int32_t>(places.size(1)), static_cast<int32_t>(expert_offsets.numel() - 1)};
}

// Rows at any distance from each other are read in place; anything else is laid out first.
at::Tensor check_rows(const at::Tensor &rows, const char *name, int64_t count) {
  TORCH_CHECK(rows.is_cuda(), name, " must be a GPU tensor");
  TORCH_CHECK(rows.dim() == 2 && rows.size(1) > 0, name, " must be a [rows, D] tensor with D > 0");
  TORCH_CHECK(rows.size(0) == count, name, " must have ", count, " rows (one row per row of places, or per pair), got ",
              rows.size(0));
  return rows.stride(1) == 1 && rows.stride(0) >= 0 ? rows : rows.contiguous();
}
int64_t row_stride(const at::Tensor &rows) { return rows.size(0) > 1 ? rows.stride(0) : rows.size(1); }

at::Tensor check_gates(const at::Tensor &weights, const at::Tensor &rows, const at::Tensor &places) {
  TORCH_CHECK(weights.scalar_type() == rows.scalar_type() || weights.scalar_type() == at::kFloat,
              "weights must be float32 or have the rows' dtype");
  TORCH_CHECK(weights.device() == rows.device(), "weights must live on the rows' device");
  TORCH_CHECK(weights.sizes() == places.sizes(), "weights must be [tokens, choices]");
  return weights.contiguous();
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> expert_plan(at::Tensor expert_ids, int64_t num_experts) {
  TORCH_CHECK(expert_ids.is_cuda(), "expert_ids must be a GPU tensor");
  TORCH_CHECK(expert_ids.scalar_type() == at::kInt || expert_ids.scalar_type() == at::kLong,
              "expert_ids must be int32 or int64");
  TORCH_CHECK(expert_ids.dim() == 2 && expert_ids.size(1) > 0, "expert_ids must be [tokens, choices] with choices > 0");
  const int64_t pairs = expert_ids.numel();
  TORCH_CHECK(pairs < std::numeric_limits<int32_t>::max(), "tokens * choices must stay below 2^31 - 1");
  TORCH_CHECK(num_experts > 0 && num_experts <= TBE_MAX_EXPERTS, "num_experts must be 1 to ", TBE_MAX_EXPERTS, " (got ",
              num_experts, ")");
  c10::DeviceGuard guard(expert_ids.device());
  expert_ids = expert_ids.contiguous();
  // places, order, expert_offsets, each from a 64-byte boundary on
  const int64_t padded = (pairs + 15) / 16 * 16;
  const at::Tensor whole = empty_on(expert_ids, {2 * padded + num_experts + 1}, at::kInt);
  at::Tensor places = part_of(whole, 0, expert_ids.sizes());
  at::Tensor order = part_of(whole, padded, {pairs});
  at::Tensor expert_offsets = part_of(whole, 2 * padded, {num_experts + 1});
  const uint64_t bytes = tbe_expert_plan_workspace_bytes(pairs, static_cast<int32_t>(num_experts));
  // (a call of its own scratch: two graphs captured on one stream do not share it)
  at::Tensor scratch;
  if (bytes > 0) scratch = empty_on(expert_ids, {static_cast<int64_t>(bytes)}, at::kByte);
  check(tbe_expert_plan(expert_ids.data_ptr(), static_cast<int32_t>(expert_ids.element_size()), pairs,
                        static_cast<int32_t>(num_experts), expert_offsets.data_ptr<int32_t>(),
                        order.data_ptr<int32_t>(), places.data_ptr<int32_t>(), bytes > 0 ? scratch.data_ptr() : nullptr,
                        bytes, stream_of(expert_ids)));
  return {expert_offsets, order, places};
}

at::Tensor dispatch(const at::Tensor &tokens_in, const at::Tensor &places, const at::Tensor &expert_offsets) {
  const at::Tensor tokens = check_rows(tokens_in, "tokens", places.dim() > 0 ? places.size(0) : 0);
  const Plan p = check_plan(places, expert_offsets, tokens.device());
  const int32_t dtype = float_code(tokens, "tokens");
  c10::DeviceGuard guard(tokens.device());
  at::Tensor rows = empty_on(tokens, {p.tokens * p.choices, tokens.size(1)}, tokens.scalar_type());
  check(tbe_expert_dispatch(tokens.data_ptr(), row_stride(tokens), dtype, p.tokens, p.choices, p.experts, tokens.size(1),
                            places.data_ptr<int32_t>(), expert_offsets.data_ptr<int32_t>(), rows.data_ptr(),
                            stream_of(tokens)));
  return rows;
}

at::Tensor combine(const at::Tensor &rows_in, const at::Tensor &places, const at::Tensor &expert_offsets,
                   const c10::optional<at::Tensor> &weights_in) {
  const at::Tensor rows = check_rows(rows_in, "rows", places.numel());
  const Plan p = check_plan(places, expert_offsets, rows.device());
  const int32_t dtype = float_code(rows, "rows");
  c10::optional<at::Tensor> weights;
  if (weights_in.has_value()) weights = check_gates(*weights_in, rows, places);
  c10::DeviceGuard guard(rows.device());
  at::Tensor output = empty_on(rows, {p.tokens, rows.size(1)}, rows.scalar_type());
  check(tbe_expert_combine(rows.data_ptr(), row_stride(rows), dtype, p.tokens, p.choices, p.experts, rows.size(1),
                           places.data_ptr<int32_t>(), expert_offsets.data_ptr<int32_t>(), ptr(weights),
                           weights.has_value() ? float_code(*weights, "weights") : dtype, output.data_ptr(),
                           stream_of(rows)));
  return output;
}

// (gradient of the rows, gradient of the weights), either of them only where it is wanted
std::tuple<c10::optional<at::Tensor>, c10::optional<at::Tensor>> combine_backward(
    const at::Tensor &grad_in, const at::Tensor &rows_in, const at::Tensor &places, const at::Tensor &expert_offsets,
    const at::Tensor &weights_in, bool want_rows, bool want_weights) {
  const at::Tensor rows = check_rows(rows_in, "rows", places.numel());
  const Plan p = check_plan(places, expert_offsets, rows.device());
  const int32_t dtype = float_code(rows, "rows");
  const at::Tensor weights = check_gates(weights_in, rows, places);
  TORCH_CHECK(grad_in.scalar_type() == rows.scalar_type(), "grad_output must have the rows' dtype");
  TORCH_CHECK(grad_in.device() == rows.device(), "grad_output must live on the rows' device");
  TORCH_CHECK(grad_in.dim() == 2 && grad_in.size(0) == p.tokens && grad_in.size(1) == rows.size(1),
              "grad_output must be [tokens, D]");
  const at::Tensor grad = check_rows(grad_in, "grad_output", p.tokens);
  c10::DeviceGuard guard(rows.device());
  c10::optional<at::Tensor> grad_rows, grad_weights;
  if (want_rows) grad_rows = empty_on(rows, {rows.size(0), rows.size(1)}, rows.scalar_type());
  if (want_weights) grad_weights = empty_on(rows, places.sizes(), weights.scalar_type());
  if (!want_rows && !want_weights) return {grad_rows, grad_weights};
  check(tbe_expert_combine_backward(
      grad.data_ptr(), row_stride(grad), rows.data_ptr(), row_stride(rows), dtype, p.tokens, p.choices, p.experts,
      rows.size(1), places.data_ptr<int32_t>(), expert_offsets.data_ptr<int32_t>(), weights.data_ptr(),
      float_code(weights, "weights"), const_cast<void *>(ptr(grad_rows)), const_cast<void *>(ptr(grad_weights)),
      stream_of(rows)));
  return {grad_rows, grad_weights};
}

// The kernels' results carry no graph of their own, so that a second derivative would silently be a wrong one.
void refuse_second_derivative() {
  TORCH_CHECK(!at::GradMode::is_enabled(), "expert routing is differentiable once (create_graph=True is not served)");
}

// (nor do they carry a tangent)
void refuse_tangent(const at::Tensor &t) {
  TORCH_CHECK(!t._fw_grad(0).defined(), "expert routing has no forward-mode derivative");
}

struct Dispatch : torch::autograd::Function<Dispatch> {
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &tokens, const at::Tensor &places,
                            const at::Tensor &expert_offsets) {
    ctx->save_for_backward({places, expert_offsets});
    return dispatch(tokens, places, expert_offsets);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                 torch::autograd::variable_list grads) {
    refuse_second_derivative();
    const auto saved = ctx->get_saved_variables();
    return {combine(grads[0], saved[0], saved[1], c10::nullopt), at::Tensor(), at::Tensor()};
  }
};

struct Combine : torch::autograd::Function<Combine> {
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &rows, const at::Tensor &places,
                            const at::Tensor &expert_offsets, const c10::optional<at::Tensor> &weights) {
    ctx->saved_data["weighted"] = weights.has_value();
    if (weights.has_value()) ctx->save_for_backward({rows, places, expert_offsets, *weights});
    else ctx->save_for_backward({places, expert_offsets});
    return combine(rows, places, expert_offsets, weights);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                 torch::autograd::variable_list grads) {
    refuse_second_derivative();
    const auto saved = ctx->get_saved_variables();
    if (!ctx->saved_data["weighted"].toBool())
      return {dispatch(grads[0], saved[0], saved[1]), at::Tensor(), at::Tensor(), at::Tensor()};
    const auto wanted = combine_backward(grads[0], saved[0], saved[1], saved[2], saved[3], ctx->needs_input_grad(0),
                                         ctx->needs_input_grad(3));
    return {std::get<0>(wanted).value_or(at::Tensor()), at::Tensor(), at::Tensor(),
            std::get<1>(wanted).value_or(at::Tensor())};
  }
};

at::Tensor expert_dispatch(const at::Tensor &tokens, const at::Tensor &places, const at::Tensor &expert_offsets) {
  refuse_tangent(tokens);
  if (at::GradMode::is_enabled() && tokens.requires_grad()) return Dispatch::apply(tokens, places, expert_offsets);
  return dispatch(tokens, places, expert_offsets);
}

at::Tensor expert_combine(const at::Tensor &rows, const at::Tensor &places, const at::Tensor &expert_offsets,
                          const c10::optional<at::Tensor> &weights) {
  refuse_tangent(rows);
  if (weights.has_value()) refuse_tangent(*weights);
  if (at::GradMode::is_enabled() && (rows.requires_grad() || (weights.has_value() && weights->requires_grad())))
    return Combine::apply(rows, places, expert_offsets, weights);
  return combine(rows, places, expert_offsets, weights);
}

// -------------------------------------------------------------------- gradient norm and clipping
// The tensors of a Python sequence (or any iterable), looked at where they are: lists of hundreds of tensors are bound
// by what the host does for each of them.
class TensorSequence {
 public:
  TensorSequence(const py::object &source, const char *name)
      : items_(py::reinterpret_steal<py::object>(PySequence_Fast(source.ptr(), "a list of tensors is needed"))) {
    if (!items_) throw py::error_already_set();
    const Py_ssize_t count = size();
    for (Py_ssize_t i = 0; i < count; ++i)
      TORCH_CHECK_TYPE(THPVariable_Check(item(i)), name, " must be tensors (entry ", i, " is none)");
  }
  Py_ssize_t size() const { return PySequence_Fast_GET_SIZE(items_.ptr()); }
  const at::Tensor &operator[](Py_ssize_t i) const { return THPVariable_Unpack(item(i)); }

 private:
  PyObject *item(Py_ssize_t i) const { return PySequence_Fast_GET_ITEM(items_.ptr(), i); }
  py::object items_;
};

struct GradientList {
  std::vector<const void *> gradients;
  std::vector<void *> outputs;
  std::vector<int64_t> numels;
  std::vector<int32_t> dtypes;
  bool f64 = false;
  int32_t count() const { return static_cast<int32_t>(gradients.size()); }
};

GradientList check_gradients(const TensorSequence &gradients, const TensorSequence *outputs) {
  const Py_ssize_t count = gradients.size();
  TORCH_CHECK(count > 0, "there must be at least one gradient");
  TORCH_CHECK(count < (1 << 24), "too many gradients");
  TORCH_CHECK(!outputs || outputs->size() == count, "out must hold one tensor per gradient");
  GradientList list;
  list.gradients.reserve(count);
  list.numels.reserve(count);
  list.dtypes.reserve(count);
  list.outputs.reserve(count);
  const at::Device device = gradients[0].device();
  for (Py_ssize_t i = 0; i < count; ++i) {
    const at::Tensor &g = gradients[i];
    TORCH_CHECK(g.is_cuda(), "gradients must be GPU tensors");
    TORCH_CHECK(g.layout() == at::kStrided, "gradients must be strided (dense) tensors");
    TORCH_CHECK(g.device() == device, "gradients must live on one device");
    // (any order of the dimensions, transposed ones among them: the elements are one block of memory)
    TORCH_CHECK(g.is_non_overlapping_and_dense(), "gradients must be dense: gradient ", i, " has gaps or repeats elements");
    list.dtypes.push_back(float_code(g, "gradients"));
    list.f64 = list.f64 || g.scalar_type() == at::kDouble;
    list.gradients.push_back(g.data_ptr());
    list.numels.push_back(g.numel());
    if (!outputs) {
      list.outputs.push_back(g.data_ptr());
      continue;
    }
    const at::Tensor &o = (*outputs)[i];
    TORCH_CHECK(o.device() == device && o.layout() == at::kStrided && o.scalar_type() == g.scalar_type() &&
                    o.sizes() == g.sizes() && o.strides() == g.strides(),
                "out must have the gradients' shapes, strides, types and device (tensor ", i, ")");
    list.outputs.push_back(o.data_ptr());
  }
  return list;
}

at::Tensor empty_norm(const at::Tensor &like, bool f64) {
  return empty_on(like, {}, f64 ? at::kDouble : at::kFloat);
}
int32_t norm_code(bool f64) { return f64 ? TBE_DTYPE_F64 : TBE_DTYPE_F32; }

at::Tensor gradient_norm(const py::object &source) {
  const TensorSequence gradients(source, "gradients");
  const GradientList list = check_gradients(gradients, nullptr);
  const at::Tensor &first = gradients[0];
  c10::DeviceGuard guard(first.device());
  at::Tensor norm = empty_norm(first, list.f64);
  const uint64_t bytes = tbe_gradient_norm_workspace_bytes(list.count());
  at::Tensor scratch = empty_on(first, {static_cast<int64_t>(bytes)}, at::kByte);
  check(tbe_gradient_norm(list.gradients.data(), list.numels.data(), list.dtypes.data(), list.count(), norm.data_ptr(),
                          norm_code(list.f64), scratch.data_ptr(), bytes, stream_of(first)));
  return norm;
}

at::Tensor clip_gradients(const py::object &source, double max_norm, const py::object &out) {
  const TensorSequence gradients(source, "gradients");
  c10::optional<TensorSequence> outputs;
  if (!out.is_none()) outputs.emplace(out, "out");
  const GradientList list = check_gradients(gradients, outputs.has_value() ? &*outputs : nullptr);
  TORCH_CHECK(max_norm >= 0.0, "max_norm must not be negative");
  const at::Tensor &first = gradients[0];
  c10::DeviceGuard guard(first.device());
  at::Tensor norm = empty_norm(first, list.f64);
  const uint64_t bytes = tbe_gradient_norm_workspace_bytes(list.count());
  at::Tensor scratch = empty_on(first, {static_cast<int64_t>(bytes)}, at::kByte);
  check(tbe_clip_gradients(list.gradients.data(), list.outputs.data(), list.numels.data(), list.dtypes.data(),
                           list.count(), max_norm, norm.data_ptr(), norm_code(list.f64), scratch.data_ptr(), bytes,
                           stream_of(first)));
  // autograd learns that the tensors were written
  const TensorSequence &written = outputs.has_value() ? *outputs : gradients;
  for (Py_ssize_t i = 0; i < written.size(); ++i)
    if (!written[i].is_inference()) written[i].unsafeGetTensorImpl()->bump_version();
  return norm;
}

// ------------------------------------------------------------------------ clipped table updates

// The batch's plan into `ws` and the norm of the tables' exact gradient.
at::Tensor plan_and_norm(const at::Tensor &grad_output, const at::Tensor &weights, const at::Tensor &table_offsets,
                         const at::Tensor &indices, const at::Tensor &offsets,
                         const c10::optional<at::Tensor> &indice_weights, const Shape &s, int32_t dtype,
                         const at::Tensor &ws) {
  const bool f64 = weights.scalar_type() == at::kDouble;
  at::Tensor norm = empty_norm(weights, f64);
  void *stream = stream_of(weights);
  const uint64_t bytes = static_cast<uint64_t>(ws.numel());
  check(tbe_plan_batch(table_offsets.data_ptr<int32_t>(), s.T, indices.data_ptr<int32_t>(), s.n,
                       offsets.data_ptr<int32_t>(), s.B, s.rows, max_table_rows(table_offsets, s.rows), s.D, dtype,
                       ws.data_ptr(), bytes, stream));
  check(tbe_table_gradient_norm(grad_output.data_ptr(), dtype, s.D, s.T, s.B, s.n, ptr(indice_weights), ws.data_ptr(),
                                bytes, norm.data_ptr(), norm_code(f64), stream));
  return norm;
}

// `gradient` scaled down to max_norm by a norm that is on the device.
at::Tensor scaled(const at::Tensor &gradient, double max_norm, const at::Tensor &norm) {
  at::Tensor out = empty_on(gradient, gradient.sizes(), gradient.scalar_type());
  const void *from = gradient.data_ptr();
  void *to = out.data_ptr();
  const int64_t numel = gradient.numel();
  const int32_t dtype = float_code(gradient, "grad_output");
  check(tbe_scale_gradients(&from, &to, &numel, &dtype, 1, max_norm, norm.data_ptr(),
                            norm_code(norm.scalar_type() == at::kDouble), stream_of(gradient)));
  return out;
}

// Whether a scaled copy of an fp16 gradient is too coarse for the update, whatever the gradient's values.  Below 2^-14
// fp16 has steps of 2^-24, so that scaling moves an element by up to 2^-25, always to the same side for equal elements:
// n lookups of D columns move the tables' gradient by up to n * sqrt(D) * 2^-25 (all of them in one row) times the largest
// per-sample weight, or make it vanish.  The copy serves where that is no more than max_norm * 2^-11, the half step that
// every larger element may be off by; else the update takes the factor itself, in 32 bits, on the gradient as it came.  The
// host does not know the weights: up to kLargestWeight is allowed for.
constexpr double kLargestWeight = 32.0;
bool copy_is_too_coarse(const at::Tensor &weights, const Shape &s, bool weighted, double max_norm) {
  return weights.scalar_type() == at::kHalf &&
         max_norm < static_cast<double>(s.n) * std::sqrt(static_cast<double>(s.D)) * 0x1p-14 * (weighted ? kLargestWeight : 1.0);
}

at::Tensor plan_scratch(const at::Tensor &weights, const Shape &s, int32_t dtype) {
  tbe_workspace_layout_t layout;
  check(tbe_backward_workspace_layout(s.n, s.D, dtype, s.T, &layout));
  return empty_on(weights, {static_cast<int64_t>(layout.total_bytes)}, at::kByte);
}

std::tuple<at::Tensor, at::Tensor> clip_table_gradient(at::Tensor grad_output, at::Tensor weights,
                                                       at::Tensor table_offsets, at::Tensor indices, at::Tensor offsets,
                                                       double max_norm, c10::optional<at::Tensor> indice_weights) {
  const Shape s = check_common(weights, table_offsets, indices, offsets);
  grad_output = check_grad(grad_output, weights, s);
  check_weights_of_lookups(indice_weights, weights, indices);
  TORCH_CHECK(max_norm >= 0.0, "max_norm must not be negative");
  const int32_t dtype = dtype_code(weights);
  c10::DeviceGuard guard(weights.device());
  const at::Tensor ws = plan_scratch(weights, s, dtype);
  const at::Tensor norm = plan_and_norm(grad_output, weights, table_offsets, indices, offsets, indice_weights, s, dtype, ws);
  return {scaled(grad_output, max_norm, norm), norm};
}

// backward_sgd / backward_exact_adagrad on the clipped gradient, one plan for the norm and the update, or
// backward_approx_adagrad, which makes its own.
at::Tensor backward_clipped(int64_t optimizer, at::Tensor grad_output, at::Tensor weights, at::Tensor table_offsets,
                            at::Tensor indices, at::Tensor offsets, c10::optional<at::Tensor> indice_weights,
                            c10::optional<at::Tensor> optimizer_state, double learning_rate, double eps,
                            bool stochastic_rounding, double max_norm) {
  const Shape s = check_common(weights, table_offsets, indices, offsets);
  grad_output = check_grad(grad_output, weights, s);
  check_weights_of_lookups(indice_weights, weights, indices);
  TORCH_CHECK(max_norm >= 0.0, "max_norm must not be negative");
  TORCH_CHECK(optimizer == TBE_OPT_SGD || optimizer == TBE_OPT_ROWWISE_ADAGRAD ||
                  optimizer == TBE_OPT_APPROX_ROWWISE_ADAGRAD,
              "optimizer must be SGD or a row-wise Adagrad");
  const bool adagrad = optimizer != TBE_OPT_SGD;
  TORCH_CHECK(adagrad || !indice_weights.has_value(), "SGD takes no per-sample weights");
  TORCH_CHECK(!adagrad || optimizer_state.has_value(), "row-wise Adagrad needs its state");
  if (adagrad) check_state(*optimizer_state, weights);
  const int32_t dtype = dtype_code(weights);
  c10::DeviceGuard guard(weights.device());
  const bool rounds = adagrad && stochastic_rounding && weights.scalar_type() == at::kHalf;
  std::pair<uint64_t, uint64_t> stream_of_bits{0, 0};
  if (rounds) stream_of_bits = rounding_stream(weights);
  const at::Tensor ws = plan_scratch(weights, s, dtype);
  const at::Tensor norm = plan_and_norm(grad_output, weights, table_offsets, indices, offsets, indice_weights, s, dtype, ws);
  const float *factor = nullptr;
  at::Tensor one;
  if (copy_is_too_coarse(weights, s, indice_weights.has_value(), max_norm)) {
    one = scaled(at::ones({1}, weights.options().dtype(at::kFloat)), max_norm, norm);
    factor = one.data_ptr<float>();
  } else {
    grad_output = scaled(grad_output, max_norm, norm);
  }
  // (the clipped gradient's dot products with the rows, which nobody asks for: the update writes them)
  c10::optional<at::Tensor> unused;
  if (indice_weights.has_value()) unused = at::empty_like(*indice_weights);
  if (optimizer == TBE_OPT_APPROX_ROWWISE_ADAGRAD)
    check(tbe_backward_approx_adagrad_scaled(
        grad_output.data_ptr(), factor, weights.data_ptr(), dtype, s.rows, max_table_rows(table_offsets, s.rows), s.D,
        table_offsets.data_ptr<int32_t>(), s.T, indices.data_ptr<int32_t>(), s.n, offsets.data_ptr<int32_t>(), s.B,
        ptr(indice_weights), optimizer_state->data_ptr(), static_cast<float>(learning_rate), static_cast<float>(eps),
        const_cast<void *>(ptr(unused)), rounds ? 1 : 0, stream_of_bits.first, stream_of_bits.second, ws.data_ptr(),
        static_cast<uint64_t>(ws.numel()), stream_of(weights)));
  else
    check(tbe_backward_planned_scaled(
        static_cast<int32_t>(optimizer), grad_output.data_ptr(), factor, weights.data_ptr(), dtype, s.rows, s.D, s.T, s.B,
        s.n, ptr(indice_weights), adagrad ? optimizer_state->data_ptr() : nullptr, static_cast<float>(learning_rate),
        static_cast<float>(eps), const_cast<void *>(ptr(unused)), rounds ? 1 : 0, stream_of_bits.first,
        stream_of_bits.second, ws.data_ptr(), static_cast<uint64_t>(ws.numel()), stream_of(weights)));
  return norm;
}

}  // namespace

void bind_training(pybind11::module &m) {
  using release = py::call_guard<py::gil_scoped_release>;
  m.def("expert_plan", &expert_plan, "stable order of the (token, choice) pairs by expert", py::arg("expert_ids"),
        py::arg("num_experts"), release());
  m.def("expert_dispatch", &expert_dispatch, "rows of the tokens in expert order", py::arg("tokens"), py::arg("places"),
        py::arg("expert_offsets"), release());
  m.def("expert_combine", &expert_combine, "weighted sums of the experts' rows in token order", py::arg("rows"),
        py::arg("places"), py::arg("expert_offsets"), py::arg("weights") = py::none(), release());
  m.def("expert_combine_backward", &combine_backward, "gradients of expert_combine", py::arg("grad_output"),
        py::arg("rows"), py::arg("places"), py::arg("expert_offsets"), py::arg("weights"), py::arg("want_rows") = true,
        py::arg("want_weights") = true, release());
  m.def("gradient_norm", &gradient_norm, "global norm of a list of gradients", py::arg("gradients"));
  m.def("clip_gradients", &clip_gradients, "scales a list of gradients down to a global norm", py::arg("gradients"),
        py::arg("max_norm"), py::arg("out") = py::none());
  m.def("clip_table_gradient", &clip_table_gradient, "grad_output scaled by the norm of the tables' exact gradient",
        py::arg("grad_output"), py::arg("weights"), py::arg("table_offsets"), py::arg("indices"), py::arg("offsets"),
        py::arg("max_norm"), py::arg("indice_weights") = py::none(), release());
  m.def("backward_clipped", &backward_clipped, "table update with the clipped gradient", py::arg("optimizer"),
        py::arg("grad_output"), py::arg("weights"), py::arg("table_offsets"), py::arg("indices"), py::arg("offsets"),
        py::arg("indice_weights"), py::arg("optimizer_state"), py::arg("learning_rate"), py::arg("eps"),
        py::arg("stochastic_rounding"), py::arg("max_norm"), release());
}

}  // namespace tbe_binding
