// The language-model operators' calls from torch in C++ (lib/ndt_torch_calls.so).
//
// For a few tokens the host takes longer than the GPU: a call through Python
// costs 9 - 15 us and a Python autograd Function 30 us more than one in C++
// (the thread that runs the backward pass has to get the interpreter).  These
// functions make the plain calls - CUDA tensors of the current device, types
// and strides that need no copy - and return nothing for any other, which the
// Python functions of the same names then check, lay out or refuse.  A call that
// was made and failed raises what it would raise from Python: it is not made
// again, since its entry point may have reported an earlier call's failure,
// which it does once.
//
// They call the C entry points of libndtensors_capi.so through addresses that
// bind() is given, so this file needs torch alone.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <optional>
#include <vector>

#include "../../include/ndtensors_capi.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

struct Entries {
  decltype(&ndt_b200_scaled_linear_dev) scaled_linear;
  decltype(&ndt_b200_scaled_linear_fwd_dev) scaled_linear_fwd;
  decltype(&ndt_b200_scaled_linear_vjp_dev) scaled_linear_vjp;
  decltype(&ndt_b200_embedding_dev) embedding;
  decltype(&ndt_b200_embedding_grad_dev) embedding_grad;
  decltype(&ndt_b200_last_error) last_error;
} entry;

template <typename F>
void set(F& f, uintptr_t address) {
  f = reinterpret_cast<F>(address);
}
PyObject* failure = nullptr;  // the package's exception for a status

void bind(const std::vector<uintptr_t>& at, py::object exception) {
  TORCH_CHECK(at.size() == 6, "bind: six addresses");
  set(entry.scaled_linear, at[0]), set(entry.scaled_linear_fwd, at[1]), set(entry.scaled_linear_vjp, at[2]);
  set(entry.embedding, at[3]), set(entry.embedding_grad, at[4]), set(entry.last_error, at[5]);
  failure = exception.release().ptr();
}

// The C ABI's code of a 32- or 16-bit floating type, or 0.
int real_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat:
      return NDT_F32;
    case at::kBFloat16:
      return NDT_BF16;
    case at::kHalf:
      return NDT_F16;
    default:
      return 0;
  }
}
int code8(at::ScalarType t) { return t == at::kFloat8_e4m3fn ? NDT_E4M3 : t == at::kFloat8_e5m2 ? NDT_E5M2 : 0; }
// (with the negative bit memory holds the opposite of the tensor's numbers)
bool here(const Tensor& t) { return t.is_cuda() && !t.is_neg() && t.get_device() == c10::cuda::current_device(); }
// A call without a gradient of its own refuses these.
bool asks(const Tensor& t) { return (at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined(); }
bool beside(const Tensor& t, const Tensor& x) { return t.is_cuda() && !t.is_neg() && t.get_device() == x.get_device(); }
void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
void* data(const Tensor& t) { return t.data_ptr(); }
long at_least(int64_t a, int64_t b) { return (long)std::max(a, b); }
bool unit_rows(const Tensor& t) { return t.stride(1) == 1 && t.stride(0) >= t.size(1); }

// x as a matrix of its last axis, where that is a view.
Maybe rows_of(const Tensor& x) {
  if (x.dim() == 2) return x;
  if (x.dim() < 1 || !x.is_contiguous() || x.size(-1) == 0) return std::nullopt;
  return x.view({-1, x.size(-1)});
}
// An empty result in x's shape with another last axis.  (Not a view of a matrix:
// torch refuses to change a view that comes out of a Function in place.)
Tensor result(const Tensor& x, int64_t last, at::ScalarType type) {
  auto sizes = x.sizes().vec();
  sizes.back() = last;
  return at::empty(sizes, x.options().dtype(type).requires_grad(false));
}
// Raises as the Python functions do (from a backward pass's thread too).
void check(int status) {
  if (status == NDT_SUCCESS) return;
  const std::string text = entry.last_error();  // (of this thread)
  py::gil_scoped_acquire gil;
  if (status == NDT_SHAPE_MISMATCH)
    PyErr_SetString(PyExc_ValueError, text.c_str());
  else
    PyErr_SetString(failure, (text + " (status " + std::to_string(status) + ")").c_str());
  python_error e;
  e.persist();
  throw e;
}

// A gradient that a graph was asked of: differentiating it again is an error.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list defined;
  for (auto& g : grads)
    if (g.defined()) defined.push_back(g.detach().set_requires_grad(true));
  auto refuse = std::make_shared<torch::autograd::DelayedError>("this operator's gradient cannot be differentiated", (int64_t)defined.size());
  auto out = (*refuse)(std::move(defined));
  size_t i = 0;
  for (auto& g : grads)
    if (g.defined()) g = out[i++];
  return grads;
}

// ---------------------------------------------------------------- embedding
bool plain_embedding(const Tensor& table, const Tensor& ids) {
  return here(table) && beside(ids, table) && table.dim() == 2 && real_code(table) &&
         unit_rows(table) && (ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt) && ids.is_contiguous();
}
Tensor lookup(const Tensor& table, const Tensor& ids, double scale, int64_t first) {
  const int64_t v = table.size(0), d = table.size(1);
  auto sizes = ids.sizes().vec();
  sizes.push_back(d);
  Tensor out = at::empty(sizes, table.options().requires_grad(false));
  check(entry.embedding(real_code(table), data(table), v, d, at_least(d, table.stride(0)), data(ids), ids.scalar_type() == at::kLong,
                        ids.numel(), first, (float)scale, data(out), d, stream()));
  return out;
}
Maybe embedding(const Tensor& table, const Tensor& ids, double scale, int64_t first) {
  if (!plain_embedding(table, ids) || asks(table)) return std::nullopt;
  return lookup(table, ids, scale, first);
}

struct EmbeddingFunction : torch::autograd::Function<EmbeddingFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& ids, double scale, int64_t first) {
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = table.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["first"] = first;
    ctx->saved_data["type"] = (int64_t)table.scalar_type();
    return lookup(table, ids, scale, first);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Tensor grad = grads[0];
    if (!grad.defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const c10::cuda::CUDAGuard guard(grad.device());
    const Tensor ids = ctx->get_saved_variables()[0];
    const int64_t rows = ctx->saved_data["rows"].toInt(), d = grad.size(-1), n = ids.numel();
    at::AutoDispatchBelowADInplaceOrView below;
    grad = grad.resolve_neg();
    if (grad.dim() != 2) grad = grad.reshape({n, d});
    if (!unit_rows(grad)) grad = grad.contiguous();
    const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
    Tensor out = at::empty({rows, d}, grad.options().dtype(type));
    check(entry.embedding_grad(real_code(grad), data(grad), at_least(d, grad.stride(0)), data(ids), ids.scalar_type() == at::kLong, n,
                               rows, d, ctx->saved_data["first"].toInt(), (float)ctx->saved_data["scale"].toDouble(), real_code(out),
                               data(out), d, 0, stream()));
    return once({out, Tensor(), Tensor(), Tensor()});
  }
};
Maybe torch_embedding(const Tensor& table, const Tensor& ids, double scale, int64_t first) {
  if (!plain_embedding(table, ids)) return std::nullopt;
  return EmbeddingFunction::apply(table, ids, scale, first);
}

// ------------------------------------------------------------ scaled linear
Maybe scaled_linear(const Tensor& x, const Tensor& w, const Tensor& scales, std::optional<at::ScalarType> out_type) {
  if (!here(x) || !beside(w, x) || !beside(scales, x) || asks(x) || asks(w) || asks(scales) || !real_code(x) || !code8(w.scalar_type()) || w.dim() != 2 || scales.dim() != 2 || scales.scalar_type() != at::kFloat)
    return std::nullopt;
  const int64_t n = w.size(0), k = w.size(1);
  if (x.dim() < 1 || x.size(-1) != k || scales.size(0) != (n + 127) / 128 || scales.size(1) != (k + 127) / 128) return std::nullopt;
  const Maybe x2 = rows_of(x);
  if (!x2) return std::nullopt;
  const int64_t t = x2->size(0);
  Tensor y = result(x, n, out_type.value_or(x.scalar_type()));
  if (!real_code(y)) return std::nullopt;
  check(entry.scaled_linear(real_code(x), data(*x2), t, k, x2->stride(0), x2->stride(1), code8(w.scalar_type()), data(w), n, w.stride(0),
                            w.stride(1), static_cast<const float*>(data(scales)), scales.stride(0), scales.stride(1), real_code(y),
                            data(y), n, stream()));
  return y;
}

struct ScaledLinearFunction : torch::autograd::Function<ScaledLinearFunction> {
  // (ctx has no needs_input_grad where nothing needs a gradient)
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, int64_t grad8, bool need_x, bool need_w) {
    const int64_t n = w.size(0), k = w.size(1);
    const Tensor x2 = *rows_of(x);
    const int64_t t = x2.size(0);
    Tensor y = result(x, n, x.scalar_type());
    // the weights' 8-bit transpose, kept for x's gradient: values and scales in one buffer
    const int64_t ld = (n + 15) / 16 * 16, kb = (k + 127) / 128, nb = (n + 127) / 128;
    Tensor kept = need_x ? at::empty({k * ld + 4 * kb * nb}, x.options().dtype(at::kByte).requires_grad(false)) : Tensor();
    char* at = need_x ? (char*)data(kept) : nullptr;
    check(entry.scaled_linear_fwd(real_code(x), data(x2), t, k, x2.stride(0), x2.stride(1), real_code(w), data(w), n, w.stride(0),
                                  w.stride(1), data(y), at_least(1, n), at, ld, need_x ? (float*)(at + k * ld) : nullptr, stream()));
    ctx->save_for_backward({need_w ? x2 : Tensor(), kept});
    ctx->saved_data["x"] = x.sizes().vec();
    ctx->saved_data["n"] = n;
    ctx->saved_data["grad8"] = grad8;
    ctx->saved_data["w_type"] = (int64_t)w.scalar_type();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Tensor dy = grads[0];
    if (!dy.defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    const c10::cuda::CUDAGuard guard(dy.device());
    const auto saved = ctx->get_saved_variables();
    const Tensor &x2 = saved[0], &kept = saved[1];
    const auto x_sizes = ctx->saved_data["x"].toIntVector();
    const int64_t n = ctx->saved_data["n"].toInt(), k = x_sizes.back(), ld = (n + 15) / 16 * 16;
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    at::AutoDispatchBelowADInplaceOrView below;
    dy = dy.resolve_neg();
    if (dy.dim() != 2) dy = dy.reshape({dy.numel() / std::max<int64_t>(n, 1), n});
    const int64_t t = dy.size(0);
    Tensor dx = need_x ? at::empty({t, k}, dy.options()) : Tensor();
    Tensor dw = need_w ? at::empty({n, k}, dy.options().dtype((at::ScalarType)ctx->saved_data["w_type"].toInt())) : Tensor();
    char* at = need_x ? (char*)data(kept) : nullptr;
    check(entry.scaled_linear_vjp(real_code(dy), data(dy), t, n, dy.stride(0), dy.stride(1), need_w ? data(x2) : nullptr, k,
                                  need_w ? x2.stride(0) : 0, need_w ? x2.stride(1) : 0, at, ld, need_x ? (float*)(at + k * ld) : nullptr,
                                  (int)ctx->saved_data["grad8"].toInt(), need_x ? data(dx) : nullptr, at_least(1, k),
                                  need_w ? real_code(dw) : NDT_F32, need_w ? data(dw) : nullptr, at_least(1, k), stream()));
    if (need_x && x_sizes.size() != 2) dx = dx.view(x_sizes);
    return once({dx, dw, Tensor(), Tensor(), Tensor()});
  }
};
Maybe torch_scaled_linear(const Tensor& x, const Tensor& w, at::ScalarType grad_type) {
  if (!here(x) || !beside(w, x) || !real_code(x) || !real_code(w) || !code8(grad_type) ||
      w.dim() != 2 || x.dim() < 1 || x.size(-1) != w.size(1) || w.size(0) == 0 || !rows_of(x))
    return std::nullopt;
  const bool graph = at::GradMode::is_enabled();
  return ScaledLinearFunction::apply(x, w, (int64_t)code8(grad_type), graph && x.requires_grad(), graph && w.requires_grad());
}

}  // namespace

PYBIND11_MODULE(ndt_torch_calls, m) {
  m.def("bind", &bind);
  m.def("embedding", &embedding);
  m.def("torch_embedding", &torch_embedding);
  m.def("scaled_linear", &scaled_linear);
  m.def("torch_scaled_linear", &torch_scaled_linear);
}
