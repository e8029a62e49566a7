// torch_binding.cpp -- the PyTorch side of the routing, of the products with
// 4-bit weights and of the 8-bit norm and products: argument checks, outputs, the current stream and the autograd
// node, ahead of the C entry points of include/grouped_gemm_amd_kernels.h.
//
// In C++ because these calls last a few microseconds on the GPU: made from
// Python through ctypes the same call took 10 to 20 us, and its backward pass,
// which autograd runs on a thread of its own, waited for the interpreter.
//
// A call returns its outputs, or None where the arguments are not in order
// (the Python caller then says what is wrong), or the hipError_t of a launch.
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <unordered_set>
#include <vector>

#include "grouped_gemm_amd_kernels.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

int type_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return GGK_TYPE_F32;
    case at::kHalf: return GGK_TYPE_F16;
    case at::kBFloat16: return GGK_TYPE_BF16;
    default: return -1;
  }
}

// Rows contiguous and not overlapping; the strides of an empty matrix do not matter.
bool rows_in_order(const Tensor& t, int64_t rows, int64_t columns, int64_t row_stride, int64_t column_stride) {
  if (t.numel() == 0) return true;
  return (columns <= 1 || column_stride == 1) && (rows <= 1 || row_stride >= std::max<int64_t>(1, columns));
}

// Does the memory hold the values?  Not where they are its negatives (the negative bit, as of the imaginary part of a
// conjugate) or it is not there (a zero tensor).
bool is_stored(const Tensor& t) { return !t.is_neg() && !t._is_zerotensor(); }

bool matrix_in_order(const Tensor& t) {
  return t.dim() == 2 && is_stored(t) && rows_in_order(t, t.size(0), t.size(1), t.stride(0), t.stride(1));
}

int64_t row_stride(const Tensor& t) {
  return t.size(0) <= 1 || t.numel() == 0 ? std::max<int64_t>(1, t.size(1)) : t.stride(0);
}

bool vector_in_order(const Tensor& t, at::ScalarType type, int64_t count, c10::Device device) {
  return t.scalar_type() == type && t.device() == device && t.numel() == count && t.is_contiguous() &&
         is_stored(t);
}

// A tangent of forward-mode differentiation: a dual tensor does not have to require a gradient.
bool has_tangent(const Tensor& t) { return torch::autograd::isFwGradDefined(t); }

// The address of a tensor's data, by its type: this form of the accessor throws where a tensor has elements but no data
// (a fake one), for which the one without a type gives the null pointer that stands for an argument left out.
const void* data(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return t.const_data_ptr<float>();
    case at::kHalf: return t.const_data_ptr<at::Half>();
    case at::kBFloat16: return t.const_data_ptr<at::BFloat16>();
    case at::kFloat8_e4m3fn: return t.const_data_ptr<at::Float8_e4m3fn>();
    case at::kInt: return t.const_data_ptr<int>();
    case at::kBool: return t.const_data_ptr<bool>();
    default: return t.const_data_ptr<uint8_t>();
  }
}

template <class Args>
int launch(hipError_t (*entry)(const Args*, hipStream_t), const Args& args, c10::Device device) {
  const c10::OptionalDeviceGuard guard(device);
  return entry(&args, c10::hip::getCurrentHIPStream(device.index()).stream());
}

// ---------------------------------------------------------------- routing

struct RouteCall {
  Tensor logits;
  MaybeTensor ids, mask;
  int64_t slots;
  bool normalize;
  double scale;
  bool balance;
};

struct RouteOutputs {
  Tensor weights, ids, counts, order, loss, slope;
  int status = 0;
};

bool route_in_order(const RouteCall& c) {
  const Tensor& z = c.logits;
  if (!z.is_cuda() || type_of(z.scalar_type()) < 0 || !matrix_in_order(z) || has_tangent(z)) return false;
  const int64_t tokens = z.size(0), experts = z.size(1);
  if (experts < 1 || experts > GGK_MOE_MAX_EXPERTS || c.slots < 1 || c.slots > GGK_ROUTE_MAX_SLOTS ||
      (!c.ids && c.slots > experts) || tokens > GGK_ROUTE_MAX_TOTAL_SLOTS / c.slots) {
    return false;
  }
  if (c.ids && (c.ids->dim() != 2 || c.ids->size(0) != tokens ||
                !vector_in_order(*c.ids, at::kInt, tokens * c.slots, z.device()))) {
    return false;
  }
  return !c.mask || vector_in_order(*c.mask, at::kBool, tokens, z.device());
}

RouteOutputs route(const RouteCall& c) {
  const Tensor& z = c.logits;
  const int64_t tokens = z.size(0), experts = z.size(1);
  const auto f32 = z.options().dtype(at::kFloat).requires_grad(false), i32 = f32.dtype(at::kInt);
  RouteOutputs o;
  o.weights = at::empty({tokens, c.slots}, f32);
  o.ids = at::empty({tokens, c.slots}, i32);
  o.order = at::empty({tokens * c.slots}, i32);
  if (tokens == 0) {
    o.counts = at::zeros({experts}, i32);
    if (c.balance) {
      o.loss = at::zeros({}, f32);
      o.slope = at::zeros({experts}, f32);
    }
    return o;
  }
  o.counts = at::empty({experts}, i32);
  if (c.balance) {
    o.loss = at::empty({}, f32);
    o.slope = at::empty({experts}, f32);
  }
  ggk_route_args a{};
  a.tokens = static_cast<int>(tokens);
  a.experts = static_cast<int>(experts);
  a.slots = static_cast<int>(c.slots);
  a.type = type_of(z.scalar_type());
  a.logits = data(z);
  a.ld = row_stride(z);
  a.token_mask = c.mask ? static_cast<const unsigned char*>(data(*c.mask)) : nullptr;
  a.given_ids = c.ids ? c.ids->const_data_ptr<int>() : nullptr;
  a.normalize = c.normalize;
  a.scale = static_cast<float>(c.scale);
  a.weights = o.weights.mutable_data_ptr<float>();
  a.ids = o.ids.mutable_data_ptr<int>();
  a.counts = o.counts.mutable_data_ptr<int>();
  a.order = o.order.mutable_data_ptr<int>();
  a.loss = c.balance ? o.loss.mutable_data_ptr<float>() : nullptr;
  a.slope = c.balance ? o.slope.mutable_data_ptr<float>() : nullptr;
  a.workspace_bytes = ggk_route_workspace(a.tokens, a.experts);
  Tensor workspace;
  if (a.workspace_bytes > 0) {
    workspace = at::empty({static_cast<int64_t>(a.workspace_bytes)}, f32.dtype(at::kByte));
    a.workspace = workspace.mutable_data_ptr();
  }
  o.status = launch(ggk_route, a, z.device());
  return o;
}

bool is_capturing(c10::Device device) {
  const c10::OptionalDeviceGuard guard(device);
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  return hipStreamIsCapturing(c10::hip::getCurrentHIPStream(device.index()).stream(), &status) == hipSuccess &&
         status != hipStreamCaptureStatusNone;
}

// Does the graph go on from `node` to one that belongs to the default stream: a leaf that an eager graph made there holds,
// or an operator of such a graph itself?
bool reaches_default_stream(torch::autograd::Node* node) {
  std::vector<torch::autograd::Node*> left{node};
  std::unordered_set<torch::autograd::Node*> seen;
  while (!left.empty()) {
    torch::autograd::Node* at = left.back();
    left.pop_back();
    if (at == nullptr || !seen.insert(at).second) continue;
    const auto stream = at->stream();
    if (stream && stream->id() == 0) return true;
    for (const auto& edge : at->next_edges()) left.push_back(edge.function.get());
  }
  return false;
}

struct Route : torch::autograd::Function<Route> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const RouteCall& c) {
    RouteOutputs o = route(c);
    TORCH_CHECK(o.status == 0, "ggk_route failed with hipError_t ", o.status);
    ctx->save_for_backward({logits, o.ids, o.slope});
    ctx->saved_data["distinct"] = !c.ids.has_value();
    ctx->saved_data["normalize"] = c.normalize;
    ctx->saved_data["scale"] = c.scale;
    ctx->mark_non_differentiable({o.ids, o.counts, o.order});
    ctx->set_materialize_grads(false);
    variable_list out{o.weights, o.ids, o.counts, o.order};
    if (c.balance) out.push_back(o.loss);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &z = saved[0], &ids = saved[1], &slope = saved[2];
    // Incoming gradients may be expanded (a sum's) or in any strides, and hold their values' negatives, or none where all
    // are zero.
    const auto incoming = [&](size_t i) {
      return i >= grads.size() || !grads[i].defined() || grads[i]._is_zerotensor() ? Tensor()
                                                                                   : grads[i].resolve_neg().contiguous();
    };
    if (!grads[0].defined() && (grads.size() < 5 || !grads[4].defined())) return {Tensor(), Tensor()};
    TORCH_CHECK(!has_tangent(grads[0]) && (grads.size() < 5 || !has_tangent(grads[4])),
                "moe_route's gradient has no forward-mode derivative: it was given a dual tensor");
    const Tensor d_weights = incoming(0), d_loss = incoming(4);
    // The engine would join the next node's stream to the capture, which for the default stream ends the process.
    TORCH_CHECK(!is_capturing(z.device()) || !reaches_default_stream(torch::autograd::get_current_node().get()),
                "moe_route: a backward pass is being captured while an eager graph of the same leaves, made on the default "
                "stream, is alive (the logits' own, or another): free it first, or make it on a side stream");
    Tensor d = at::empty({z.size(0), z.size(1)}, z.options().requires_grad(false));
    if (z.size(0) > 0) {
      ggk_route_gradient_args a{};
      a.tokens = static_cast<int>(z.size(0));
      a.experts = static_cast<int>(z.size(1));
      a.slots = static_cast<int>(ids.size(1));
      a.type = type_of(z.scalar_type());
      a.logits = data(z);
      a.ld = row_stride(z);
      a.ids = ids.const_data_ptr<int>();
      a.distinct = ctx->saved_data["distinct"].toBool();
      a.slope = slope.defined() ? slope.const_data_ptr<float>() : nullptr;
      a.normalize = ctx->saved_data["normalize"].toBool();
      a.scale = static_cast<float>(ctx->saved_data["scale"].toDouble());
      a.d_weights = d_weights.defined() ? d_weights.const_data_ptr<float>() : nullptr;
      a.d_loss = d_loss.defined() ? d_loss.const_data_ptr<float>() : nullptr;
      a.d_logits = d.mutable_data_ptr();
      const int status = launch(ggk_route_gradient, a, z.device());
      TORCH_CHECK(status == 0, "ggk_route_gradient failed with hipError_t ", status);
    }
    if (at::GradMode::is_enabled()) {  // create_graph: a second derivative raises instead of being left out
      d.set_requires_grad(true);
      const auto refuse = std::make_shared<torch::autograd::DelayedError>(
          "moe_route's gradient is once_differentiable: it has no second derivative", 1);
      d = (*refuse)({d})[0];
    }
    return {d, Tensor()};
  }
};

py::object route_call(const Tensor& logits, std::optional<int64_t> top_k, const MaybeTensor& ids, const MaybeTensor& mask,
                      bool normalize, double scale, bool balance) {
  if (top_k.has_value() == ids.has_value()) return py::none();
  if (ids && ids->dim() != 2) return py::none();
  const RouteCall c{logits, ids, mask, ids ? ids->size(1) : *top_k, normalize, scale, balance};
  if (!route_in_order(c)) return py::none();
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    const variable_list o = Route::apply(logits, c);
    return py::make_tuple(o[0], o[1], o[2], o[3], balance ? py::cast(o[4]) : py::none());
  }
  const RouteOutputs o = route(c);
  if (o.status != 0) return py::int_(o.status);
  return py::make_tuple(o.weights, o.ids, o.counts, o.order, balance ? py::cast(o.loss) : py::none());
}

// ---------------------------------------------------------------- 4-bit weights

// [N, columns] or [experts, N, columns], rows contiguous and not overlapping, row and matrix starts on multiples of
// `align` elements.
bool weights_in_order(const Tensor& t, const Tensor& q, at::ScalarType type, c10::Device device, int64_t align) {
  const int64_t dim = q.dim(), n = q.size(dim - 2);
  if (t.scalar_type() != type || t.device() != device || t.dim() != dim || !is_stored(t)) return false;
  for (int64_t i = 0; i + 1 < dim; ++i) {
    if (t.size(i) != q.size(i)) return false;
  }
  const int64_t columns = t.size(dim - 1);
  return (columns <= 1 || t.stride(dim - 1) == 1) &&
         (n <= 1 || (t.stride(dim - 2) >= columns && t.stride(dim - 2) % align == 0)) &&
         (dim == 2 || t.size(0) <= 1 || t.stride(0) % align == 0);
}

py::object w4_call(const Tensor& x, const Tensor& q, const Tensor& scales, const MaybeTensor& zeros,
                   const MaybeTensor& counts, const MaybeTensor& order, const MaybeTensor& row_weights,
                   at::ScalarType out_type) {
  const int64_t dim = counts ? 3 : 2;
  if (!x.is_cuda() || x.scalar_type() != at::kHalf || !matrix_in_order(x) || q.dim() != dim ||
      (out_type != at::kFloat && out_type != at::kHalf)) {
    return py::none();
  }
  const c10::Device device = x.device();
  const int64_t n = q.size(dim - 2), half = q.size(dim - 1), k = 2 * half, x_rows = x.size(0);
  const int64_t experts = counts ? q.size(0) : 0;
  if (!weights_in_order(q, q, at::kByte, device, 16) || !weights_in_order(scales, q, at::kHalf, device, 1) ||
      (zeros && !weights_in_order(*zeros, q, at::kByte, device, 1))) {
    return py::none();
  }
  const int64_t groups = scales.size(dim - 1);
  if (x.size(1) != k || k == 0 || groups < 1 || k % (32 * groups) != 0 || (zeros && zeros->size(dim - 1) != groups) ||
      reinterpret_cast<uintptr_t>(q.const_data_ptr()) % 16 != 0) {
    return py::none();
  }
  int64_t rows = x_rows;
  if (counts) {
    if (!order || experts < 1 || experts > GGK_MOE_MAX_EXPERTS || !vector_in_order(*counts, at::kInt, experts, device)) {
      return py::none();
    }
    rows = order->numel();
    if (!vector_in_order(*order, at::kInt, rows, device) || (rows > 0 && (x_rows == 0 || rows % x_rows != 0)) ||
        (row_weights && !vector_in_order(*row_weights, at::kFloat, rows, device))) {
      return py::none();
    }
  }
  if (rows > GGK_ROUTE_MAX_TOTAL_SLOTS || n > GGK_W4_MAX_EXTENT || k > GGK_W4_MAX_EXTENT) return py::none();
  if (has_tangent(x) || has_tangent(scales) || (row_weights && has_tangent(*row_weights))) return py::none();
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || scales.requires_grad() || (row_weights && row_weights->requires_grad()))) {
    return py::none();
  }
  Tensor y = at::empty({rows, n}, x.options().dtype(out_type).requires_grad(false));
  if (rows == 0 || n == 0) return py::cast(y);
  const auto ld = [&](const Tensor& t) { return n > 1 ? t.stride(dim - 2) : t.size(dim - 1); };
  const auto matrix = [&](const Tensor& t) { return experts > 1 ? t.stride(0) : 0; };
  ggk_w4_args a{};
  a.rows = static_cast<int>(rows);
  a.x_rows = static_cast<int>(x_rows);
  a.n = static_cast<int>(n);
  a.k = static_cast<int>(k);
  a.group = static_cast<int>(k / groups);
  a.experts = static_cast<int>(experts);
  a.x = data(x);
  a.ldx = row_stride(x);
  a.q = static_cast<const unsigned char*>(data(q));
  a.ldq = ld(q);
  a.stride_q = matrix(q);
  a.scales = data(scales);
  a.lds = ld(scales);
  a.stride_s = matrix(scales);
  if (zeros) {
    a.zeros = static_cast<const unsigned char*>(data(*zeros));
    a.ldz = ld(*zeros);
    a.stride_z = matrix(*zeros);
  }
  if (counts) {
    a.counts = counts->const_data_ptr<int>();
    a.order = order->const_data_ptr<int>();
    a.row_weights = row_weights ? row_weights->const_data_ptr<float>() : nullptr;
  }
  a.y = y.mutable_data_ptr();
  a.ldy = n;
  a.y_type = type_of(out_type);
  const int status = launch(ggk_w4_multiply, a, device);
  return status == 0 ? py::cast(y) : py::object(py::int_(status));
}

// ---------------------------------------------------------------- 8-bit rows

constexpr int64_t blocks_of(int64_t n) { return (n + GGK_FP8_BLOCK - 1) / GGK_FP8_BLOCK; }

bool wants_gradient(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors) {
    if (t != nullptr && t->requires_grad()) return true;
  }
  return false;
}

const Tensor* given(const MaybeTensor& t) { return t ? &*t : nullptr; }

py::object norm_fp8_call(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& residual, double eps, bool plain) {
  if (!x.is_cuda() || type_of(x.scalar_type()) < 0 || !matrix_in_order(x) || has_tangent(x)) return py::none();
  const c10::Device device = x.device();
  const int64_t rows = x.size(0), columns = x.size(1);
  if (columns < 1 || columns > GGK_NORM_MAX_COLUMNS || rows > GGK_ROUTE_MAX_TOTAL_SLOTS) return py::none();
  if (weight) {
    if ((weight->scalar_type() != x.scalar_type() && weight->scalar_type() != at::kFloat) || weight->dim() != 1 ||
        !vector_in_order(*weight, weight->scalar_type(), columns, device) || has_tangent(*weight)) {
      return py::none();
    }
  }
  if (residual && (residual->scalar_type() != x.scalar_type() || residual->device() != device ||
                   !matrix_in_order(*residual) || residual->sizes() != x.sizes() || has_tangent(*residual))) {
    return py::none();
  }
  if (wants_gradient({&x, given(weight), given(residual)})) return py::none();
  const auto like_x = x.options().requires_grad(false);
  Tensor q = at::empty({rows, columns}, like_x.dtype(at::kFloat8_e4m3fn));
  Tensor scales = at::empty({rows, blocks_of(columns)}, like_x.dtype(at::kFloat));
  MaybeTensor y, sum;
  if (plain) y = at::empty({rows, columns}, like_x);
  if (residual) sum = at::empty({rows, columns}, like_x);
  if (rows > 0) {
    ggk_norm_fp8_args a{};
    a.rows = static_cast<int>(rows);
    a.columns = static_cast<int>(columns);
    a.type = type_of(x.scalar_type());
    a.x = data(x);
    a.ldx = row_stride(x);
    if (weight) {
      a.weight = data(*weight);
      a.weight_type = type_of(weight->scalar_type());
    }
    a.eps = static_cast<float>(eps);
    a.q = static_cast<unsigned char*>(q.mutable_data_ptr());
    a.ldq = columns;
    a.scales = scales.mutable_data_ptr<float>();
    a.lds = scales.size(1);
    if (residual) {
      a.residual = data(*residual);
      a.ldr = row_stride(*residual);
      a.sum = sum->mutable_data_ptr();
      a.ldsum = columns;
    }
    if (plain) {
      a.y = y->mutable_data_ptr();
      a.ldy = columns;
    }
    const int status = launch(ggk_norm_fp8, a, device);
    if (status != 0) return py::int_(status);
  }
  const auto or_none = [](const MaybeTensor& t) { return t ? py::cast(*t) : py::object(py::none()); };
  return py::make_tuple(q, scales, or_none(y), or_none(sum));
}

// A weight matrix (or one an expert) of 8-bit numbers, rows on multiples of 16 bytes, with its blocks' scales.
bool fp8_matrix_in_order(const Tensor& w, const Tensor& scales, int64_t dim, c10::Device device) {
  if (w.scalar_type() != at::kFloat8_e4m3fn || w.device() != device || w.dim() != dim || !is_stored(w) ||
      scales.scalar_type() != at::kFloat || scales.device() != device || scales.dim() != dim || !is_stored(scales)) {
    return false;
  }
  const int64_t n = w.size(dim - 2), k = w.size(dim - 1), rows = scales.size(dim - 2), columns = scales.size(dim - 1);
  if (rows != blocks_of(n) || columns != blocks_of(k) || (dim == 3 && scales.size(0) != w.size(0))) return false;
  if (k > 1 && w.stride(dim - 1) != 1) return false;
  if (n > 1 && (w.stride(dim - 2) < k || w.stride(dim - 2) > GGK_FP8_MAX_LD || w.stride(dim - 2) % 16 != 0)) return false;
  if (columns > 1 && scales.stride(dim - 1) != 1) return false;
  if (rows > 1 && scales.stride(dim - 2) < columns) return false;
  return (dim == 2 || w.size(0) <= 1 || w.stride(0) % 16 == 0) && reinterpret_cast<uintptr_t>(w.const_data_ptr()) % 16 == 0;
}

py::object fp8_call(const Tensor& x, const Tensor& x_scales, const Tensor& w, const Tensor& w_scales, const MaybeTensor& up,
                    const MaybeTensor& up_scales, int gate, const MaybeTensor& counts, const MaybeTensor& order,
                    const MaybeTensor& row_weights, at::ScalarType out_type, bool fast) {
  const int64_t dim = counts ? 3 : 2;
  const bool gated = gate != GGK_GATE_NONE;
  if (!x.is_cuda() || x.scalar_type() != at::kFloat8_e4m3fn || !matrix_in_order(x) || w.dim() != dim ||
      gated != up.has_value() || gated != up_scales.has_value() || gate < GGK_GATE_NONE || gate > GGK_GATE_GELU ||
      type_of(out_type) < 0 || (fast && (gated || out_type == at::kFloat))) {
    return py::none();
  }
  const c10::Device device = x.device();
  const int64_t n = w.size(dim - 2), k = w.size(dim - 1), x_rows = x.size(0), experts = counts ? w.size(0) : 0;
  if (x.size(1) != k || k < 16 || k % 16 != 0 || k > GGK_FP8_MAX_K || n > GGK_FP8_MAX_N ||
      (x_rows > 1 && x.stride(0) % 16 != 0) || reinterpret_cast<uintptr_t>(x.const_data_ptr()) % 16 != 0 ||
      x_scales.scalar_type() != at::kFloat || x_scales.device() != device || !matrix_in_order(x_scales) ||
      x_scales.size(0) != x_rows || x_scales.size(1) != blocks_of(k) ||
      !fp8_matrix_in_order(w, w_scales, dim, device) ||
      (gated && (up->sizes() != w.sizes() || !fp8_matrix_in_order(*up, *up_scales, dim, device)))) {
    return py::none();
  }
  int64_t rows = x_rows;
  if (counts) {
    if (!order || experts < 1 || experts > GGK_MOE_MAX_EXPERTS || !vector_in_order(*counts, at::kInt, experts, device)) {
      return py::none();
    }
    rows = order->numel();
    if (!vector_in_order(*order, at::kInt, rows, device) || (rows > 0 && (x_rows == 0 || rows % x_rows != 0)) ||
        (row_weights && !vector_in_order(*row_weights, at::kFloat, rows, device))) {
      return py::none();
    }
  }
  if (rows > GGK_ROUTE_MAX_TOTAL_SLOTS) return py::none();
  for (const Tensor* t : {&x, &x_scales, &w, &w_scales, given(up), given(up_scales), given(row_weights)}) {
    if (t != nullptr && has_tangent(*t)) return py::none();
  }
  if (wants_gradient({&x, &x_scales, &w, &w_scales, given(up), given(up_scales), given(row_weights)})) return py::none();
  const auto like_x = x.options().requires_grad(false);
  Tensor y = at::empty({rows, n}, gated ? like_x : like_x.dtype(out_type)), y_scales;
  if (gated) y_scales = at::empty({rows, blocks_of(n)}, like_x.dtype(at::kFloat));
  if (rows > 0 && n > 0) {
    const auto ld = [&](const Tensor& t) { return t.size(dim - 2) > 1 ? t.stride(dim - 2) : t.size(dim - 1); };
    const auto matrix = [&](const Tensor& t) { return experts > 1 ? t.stride(0) : 0; };
    ggk_fp8_args a{};
    a.rows = static_cast<int>(rows);
    a.x_rows = static_cast<int>(x_rows);
    a.n = static_cast<int>(n);
    a.k = static_cast<int>(k);
    a.experts = static_cast<int>(experts);
    a.gate = gate;
    a.x = static_cast<const unsigned char*>(data(x));
    a.ldx = row_stride(x);
    a.x_scales = x_scales.const_data_ptr<float>();
    a.ldxs = row_stride(x_scales);
    a.w = static_cast<const unsigned char*>(data(w));
    a.ldw = ld(w);
    a.stride_w = matrix(w);
    a.w_scales = w_scales.const_data_ptr<float>();
    a.ldws = ld(w_scales);
    a.stride_ws = matrix(w_scales);
    if (gated) {
      a.up = static_cast<const unsigned char*>(data(*up));
      a.ldu = ld(*up);
      a.stride_u = matrix(*up);
      a.up_scales = up_scales->const_data_ptr<float>();
      a.ldus = ld(*up_scales);
      a.stride_us = matrix(*up_scales);
      a.y_scales = y_scales.mutable_data_ptr<float>();
      a.ldys = y_scales.size(1);
    }
    if (counts) {
      a.counts = counts->const_data_ptr<int>();
      a.order = order->const_data_ptr<int>();
      a.row_weights = row_weights ? row_weights->const_data_ptr<float>() : nullptr;
    }
    a.y = y.mutable_data_ptr();
    a.ldy = n;
    a.y_type = type_of(out_type);
    a.fast = fast ? 1 : 0;
    Tensor workspace;  // goes back to the allocator in the stream's order
    long long floats = 0;
    if (const int status = ggk_fp8_workspace(&a, &floats); status != 0) return py::int_(status);
    if (floats > 0) {
      workspace = at::empty({floats}, like_x.dtype(at::kFloat));
      a.workspace = workspace.mutable_data_ptr<float>();
      a.workspace_floats = floats;
    }
    const int status = launch(ggk_fp8_multiply, a, device);
    if (status != 0) return py::int_(status);
  }
  return gated ? py::object(py::make_tuple(y, y_scales)) : py::cast(y);
}

}  // namespace

PYBIND11_MODULE(gg_torch, m) {
  m.attr("torch_version") = GG_TORCH_VERSION;  // whose classes this was compiled with; the loader compares
  m.def("route", &route_call);
  m.def("w4", &w4_call);
  m.def("norm_fp8", &norm_fp8_call);
  m.def("fp8", &fp8_call);
}
