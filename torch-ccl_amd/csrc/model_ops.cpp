// Tensor front end of the operators that compute around the collectives (embedding, router,
// mixture-of-experts layer): checks, output and workspace allocation, and the call of the C ABI on the
// current stream of the tensors' device.  In C++ because these calls are short: an interpreter's share of a
// decode step's layer, 14 us of host time, was more than its kernels' 10.
#include "model_ops.hpp"

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/utils/pybind.h>

#include <initializer_list>
#include <optional>
#include <sstream>
#include <stdexcept>
#include <string>
#include <tuple>

#include "mccl.h"

namespace {

namespace py = pybind11;
using at::ScalarType;
using at::Tensor;
using MaybeTensor = std::optional<Tensor>;

// RuntimeError in Python, with the message alone.
[[noreturn]] void refuse(const char* what, const std::string& why) { throw std::runtime_error(std::string(what) + ": " + why); }

const char* name_of(ScalarType t) {
  switch (t) {
    case at::kBFloat16: return "bfloat16";
    case at::kHalf: return "float16";
    case at::kFloat: return "float32";
    case at::kDouble: return "float64";
    case at::kInt: return "int32";
    case at::kLong: return "int64";
    default: return c10::toString(t);
  }
}

int code_of(ScalarType t) {
  switch (t) {
    case at::kBFloat16: return MCCL_BF16;
    case at::kHalf: return MCCL_F16;
    case at::kFloat: return MCCL_F32;
    case at::kInt: return MCCL_I32;
    default: return MCCL_I64;
  }
}

bool is_float(const Tensor& t) {
  const ScalarType s = t.scalar_type();
  return s == at::kBFloat16 || s == at::kHalf || s == at::kFloat;
}
bool is_id(const Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }

struct Named {
  const char* name;
  const Tensor& t;
};

// Every tensor on the GPU, contiguous, all on one device.
void check_gpu(const char* what, std::initializer_list<Named> tensors) {
  const c10::Device device = tensors.begin()->t.device();
  for (const Named& n : tensors) {
    if (!n.t.is_cuda()) refuse(what, "tensors must be on the GPU (got " + n.t.device().str() + ")");
    if (!n.t.is_contiguous()) refuse(what, std::string(n.name) + " has to be contiguous");
    if (n.t.device() != device) refuse(what, "tensors must share one device");
  }
}

void check_shape(const char* what, const char* name, const Tensor& t, at::IntArrayRef shape, std::initializer_list<ScalarType> types) {
  bool fits = t.sizes() == shape, typed = false;
  for (const ScalarType s : types) typed |= t.scalar_type() == s;
  if (fits && typed) return;
  std::ostringstream why;
  why << name << " must be ";
  const char* between = "";
  for (const ScalarType s : types) { why << between << name_of(s); between = " or "; }
  why << " of shape " << shape << " (got " << name_of(t.scalar_type()) << " " << t.sizes() << ")";
  refuse(what, why.str());
}

// The calls are no autograd nodes.  Who passes a tensor that wants a gradient, and has not switched gradients off, is told
// so once per place in the program: the result has none.
void check_grad(const char* what, std::initializer_list<Named> inputs) {
  if (!at::GradMode::is_enabled()) return;
  for (const Named& n : inputs) {
    if (!n.t.requires_grad()) continue;
    const std::string why = std::string(what) + ": " + n.name + " requires grad, but the call is no autograd node and its result has no "
                            "gradient (gradients are calls of their own; torch.no_grad() or detach() says that none is meant)";
    if (PyErr_WarnEx(PyExc_UserWarning, why.c_str(), 2)) throw py::error_already_set();
    return;
  }
}

void check(int rc) {
  if (rc != MCCL_OK) throw std::runtime_error("mccl error " + std::to_string(rc) + ": " + mccl_last_error());
}

// The device made current, if it is not, and its current stream.
struct OnDevice {
  explicit OnDevice(const Tensor& t) : guard(t.device()), stream(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream()) {}
  c10::DeviceGuard guard;
  void* stream;
};

// The caller's workspace (uint8, large enough) or one from torch's allocator for this call.
struct Workspace {
  Workspace(const char* what, const MaybeTensor& given, size_t bytes, c10::Device device) {
    if (given) {
      const Tensor& g = *given;
      if (g.scalar_type() != at::kByte || g.device() != device || !g.is_contiguous() || (size_t)g.numel() < bytes)
        refuse(what, "workspace must be " + std::to_string(bytes) + " bytes of uint8 on " + device.str());
      held = g;
    } else if (bytes) {
      held = at::empty({(int64_t)bytes}, at::TensorOptions(at::kByte).device(device));
    }
  }
  void* data() const { return held.defined() ? held.data_ptr() : nullptr; }
  size_t size() const { return held.defined() ? (size_t)held.numel() : 0; }
  Tensor held;
};

// The caller's tensors have new values: autograd notices where it has kept one for a backward pass.
void written(const MaybeTensor& given) {
  if (given && !given->is_inference()) given->unsafeGetTensorImpl()->bump_version();
}

Tensor embedding(const Tensor& table, const Tensor& ids, double scale, int64_t first_row, const MaybeTensor& given) {
  const char* what = "embedding";
  if (table.dim() != 2 || !is_float(table)) refuse(what, "table must be a matrix in bf16, f16 or f32");
  if (!is_id(ids)) refuse(what, "ids must be int32 or int64");
  c10::SmallVector<int64_t, 6> shape(ids.sizes().begin(), ids.sizes().end());
  shape.push_back(table.size(1));
  if (given) check_shape(what, "out", *given, shape, {table.scalar_type()});
  check_gpu(what, {{"table", table}, {"ids", ids}, {"out", given ? *given : table}});
  check_grad(what, {{"table", table}});
  const OnDevice on(table);
  const Tensor out = given ? *given : at::empty(shape, table.options().memory_format(std::nullopt));
  check(mccl_embedding(table.data_ptr(), table.size(0), ids.data_ptr(), code_of(ids.scalar_type()), ids.numel(), first_row, table.size(1),
                       (float)scale, code_of(table.scalar_type()), out.data_ptr(), on.stream));
  written(given);
  return out;
}

std::tuple<Tensor, Tensor> sort_ids(const Tensor& ids, int64_t rows, int64_t first_row, const MaybeTensor& workspace) {
  const char* what = "sort_ids";
  if (!is_id(ids)) refuse(what, "ids must be int32 or int64");
  if (rows < 0) refuse(what, "negative row count");
  check_gpu(what, {{"ids", ids}});
  const OnDevice on(ids);
  const int64_t n = ids.numel();
  const auto options = at::TensorOptions(at::kLong).device(ids.device());
  const Tensor order = at::empty({n}, options), offsets = at::empty({rows + 1}, options);
  const Workspace ws(what, workspace, mccl_sort_ids_workspace(n), ids.device());
  check(mccl_sort_ids(ids.data_ptr(), code_of(ids.scalar_type()), n, first_row, rows, ws.data(), ws.size(), order.data_ptr<int64_t>(),
                      offsets.data_ptr<int64_t>(), on.stream));
  return {order, offsets};
}

Tensor embedding_grad(const Tensor& grad, const Tensor& order, const Tensor& offsets, double scale, std::optional<ScalarType> dtype,
                      const MaybeTensor& given, bool accumulate, const MaybeTensor& workspace) {
  const char* what = "embedding_grad";
  if (grad.dim() < 1 || !is_float(grad)) refuse(what, "grad must be bf16, f16 or f32");
  const int64_t hidden = grad.size(-1), n = order.numel();
  if (grad.numel() != n * hidden) refuse(what, "grad must hold one row per sorted id");
  check_shape(what, "order", order, {n}, {at::kLong});
  if (offsets.dim() != 1 || offsets.numel() < 1) refuse(what, "offsets must hold rows + 1 entries");
  check_shape(what, "offsets", offsets, offsets.sizes(), {at::kLong});
  const int64_t rows = offsets.numel() - 1;
  const ScalarType type = dtype.value_or(given ? given->scalar_type() : grad.scalar_type());
  if (type != grad.scalar_type() && type != at::kFloat)
    refuse(what, std::string("out must be float32 or of grad's type ") + name_of(grad.scalar_type()));
  if (accumulate && !given) refuse(what, "accumulate needs the tensor to add to (out)");
  if (given) check_shape(what, "out", *given, {rows, hidden}, {type});
  check_gpu(what, {{"grad", grad}, {"order", order}, {"offsets", offsets}, {"out", given ? *given : grad}});
  check_grad(what, {{"grad", grad}});
  const OnDevice on(grad);
  const Tensor out = given ? *given : at::empty({rows, hidden}, at::TensorOptions(type).device(grad.device()));
  const Workspace ws(what, workspace, mccl_embedding_grad_workspace(n, hidden), grad.device());
  check(mccl_embedding_grad(grad.data_ptr(), order.data_ptr<int64_t>(), offsets.data_ptr<int64_t>(), n, rows, hidden, (float)scale,
                            code_of(grad.scalar_type()), out.data_ptr(), code_of(type), accumulate, ws.data(), ws.size(), on.stream));
  written(given);
  return out;
}

std::tuple<Tensor, Tensor> moe_route(const Tensor& logits, int64_t topk, bool normalize, const MaybeTensor& given_ids,
                                     const MaybeTensor& given_weights) {
  const char* what = "moe_route";
  if (logits.dim() != 2 || !is_float(logits)) refuse(what, "logits must be [tokens, experts] in bf16, f16 or f32");
  if (topk < 1 || topk > INT32_MAX) refuse(what, "topk must be positive");
  const int64_t tokens = logits.size(0);
  if (given_ids) check_shape(what, "expert_ids", *given_ids, {tokens, topk}, {at::kInt});
  if (given_weights) check_shape(what, "weights", *given_weights, {tokens, topk}, {at::kFloat});
  check_gpu(what, {{"logits", logits}, {"expert_ids", given_ids ? *given_ids : logits}, {"weights", given_weights ? *given_weights : logits}});
  check_grad(what, {{"logits", logits}});
  const OnDevice on(logits);
  const Tensor ids = given_ids ? *given_ids : at::empty({tokens, topk}, at::TensorOptions(at::kInt).device(logits.device()));
  const Tensor weights = given_weights ? *given_weights : at::empty({tokens, topk}, at::TensorOptions(at::kFloat).device(logits.device()));
  check(mccl_moe_route(logits.data_ptr(), tokens, logits.size(1), (int)topk, normalize, code_of(logits.scalar_type()),
                       ids.data_ptr<int32_t>(), weights.data_ptr<float>(), on.stream));
  written(given_ids);
  written(given_weights);
  return {ids, weights};
}

Tensor moe_route_grad(const Tensor& grad_weights, const Tensor& logits, const Tensor& ids, bool normalize, const MaybeTensor& given) {
  const char* what = "moe_route_grad";
  if (logits.dim() != 2 || !is_float(logits)) refuse(what, "logits must be [tokens, experts] in bf16, f16 or f32");
  if (ids.dim() != 2) refuse(what, "expert_ids must be [tokens, topk]");
  const int64_t tokens = logits.size(0), topk = ids.size(1);
  check_shape(what, "expert_ids", ids, {tokens, topk}, {at::kInt});
  check_shape(what, "grad_weights", grad_weights, {tokens, topk}, {at::kFloat});
  if (given) check_shape(what, "out", *given, logits.sizes(), {logits.scalar_type()});
  check_gpu(what, {{"grad_weights", grad_weights}, {"logits", logits}, {"expert_ids", ids}, {"out", given ? *given : logits}});
  check_grad(what, {{"grad_weights", grad_weights}, {"logits", logits}});
  const OnDevice on(logits);
  const Tensor out = given ? *given : at::empty(logits.sizes(), logits.options().memory_format(std::nullopt));
  check(mccl_moe_route_grad(grad_weights.data_ptr<float>(), logits.data_ptr(), ids.data_ptr<int32_t>(), tokens, logits.size(1), (int)topk,
                            normalize, code_of(logits.scalar_type()), out.data_ptr(), on.stream));
  written(given);
  return out;
}

Tensor moe_layer(const Tensor& x, const Tensor& w_in, const Tensor& w_out, const Tensor& ids, const Tensor& weights, int64_t first_expert,
                 const std::string& activation, const MaybeTensor& given, const MaybeTensor& workspace) {
  const char* what = "moe_layer";
  if (activation != "silu" && activation != "gelu") refuse(what, "activation must be one of gelu, silu");
  if (x.dim() != 2 || w_in.dim() != 3 || w_out.dim() != 3 || ids.dim() != 2 || (x.scalar_type() != at::kBFloat16 && x.scalar_type() != at::kHalf))
    refuse(what, "x [tokens, hidden], w_in [experts, 2 * inter, hidden] and w_out [experts, hidden, inter] in bf16 or f16");
  const int64_t tokens = x.size(0), hidden = x.size(1), experts = w_out.size(0), inter = w_out.size(2), topk = ids.size(1);
  const ScalarType type = x.scalar_type();
  check_shape(what, "w_in", w_in, {experts, 2 * inter, hidden}, {type});
  check_shape(what, "w_out", w_out, {experts, hidden, inter}, {type});
  check_shape(what, "expert_ids", ids, {tokens, topk}, {at::kInt});
  check_shape(what, "weights", weights, {tokens, topk}, {at::kFloat});
  if (given) check_shape(what, "out", *given, x.sizes(), {type});
  check_gpu(what, {{"x", x}, {"w_in", w_in}, {"w_out", w_out}, {"expert_ids", ids}, {"weights", weights}, {"out", given ? *given : x}});
  check_grad(what, {{"x", x}, {"w_in", w_in}, {"w_out", w_out}, {"weights", weights}});
  const OnDevice on(x);
  const Tensor out = given ? *given : at::empty({tokens, hidden}, at::TensorOptions(type).device(x.device()));
  const int act = activation == "silu" ? MCCL_ACT_SILU : MCCL_ACT_GELU;
  if (experts == 0) {  // a rank that holds none: zeros for the sum, within the limits on tokens that the other ranks have
    check(mccl_moe_layer(nullptr, nullptr, nullptr, nullptr, nullptr, tokens, (int)topk, 1, first_expert, 0, inter, act, code_of(type), nullptr,
                         nullptr, 0, on.stream));
    return out.zero_();
  }
  const Workspace ws(what, workspace, mccl_moe_layer_workspace(tokens, (int)topk, experts, hidden, inter), x.device());
  check(mccl_moe_layer(x.data_ptr(), w_in.data_ptr(), w_out.data_ptr(), ids.data_ptr<int32_t>(), weights.data_ptr<float>(), tokens, (int)topk,
                       experts, first_expert, hidden, inter, act, code_of(type),
                       out.data_ptr(), ws.data(), ws.size(), on.stream));
  written(given);
  return out;
}

}  // namespace

void register_model_ops(py::module_& m) {
  m.def("embedding", &embedding);
  m.def("sort_ids", &sort_ids);
  m.def("embedding_grad", &embedding_grad);
  m.def("moe_route", &moe_route);
  m.def("moe_route_grad", &moe_route_grad);
  m.def("moe_layer", &moe_layer);
}
