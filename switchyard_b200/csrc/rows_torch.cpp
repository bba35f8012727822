// The row operators as calls on torch tensors, with their autograd nodes: what rows.py and kernels.Ext
// hand on to. In C++ because the host is what a small batch waits for: permute_rows and its gradient, 64 tokens of
// 2048 columns, took 90 us through Python autograd functions and ctypes; they take 52 (unpermute_rows 103, 60), where
// torch's own negation and its gradient take 49 and index_select and its gradient 61: the engine hands a
// GPU's gradients to a thread of its own. Without a gradient 5 us (11). No work is done here but checks,
// allocation of the results, and the launches of the C ABI library (include/switchyard_b200.h).
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/switchyard_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

[[noreturn]] void refuse(const std::string& why) { throw std::runtime_error(why); }

void done(const char* name, int rc) {
  if (rc != SY_OK) refuse("switchyard_b200." + std::string(name) + " failed (" + std::to_string(rc) + "): " + sy_last_error());
}

std::string shape_of(const Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}

int row_code(const char* name, const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kHalf: return SY_DTYPE_F16;
    case at::kBFloat16: return SY_DTYPE_BF16;
    case at::kFloat: return SY_DTYPE_F32;
    default: refuse(std::string(name) + ": fp16, bf16 or fp32 expected, got " + c10::toString(t.scalar_type()));
  }
}

// Contiguous, on a GPU (device `dev` when not negative), with memory of its own (a wrapper of a
// functional transform has none).
bool usable(const Tensor& t, int dev) {
  return t.is_cuda() && t.has_storage() && t.is_contiguous() && (dev < 0 || t.get_device() == dev);
}

int on_device(const char* name, const Tensor& t, const char* what) {
  if (!usable(t, -1)) refuse(std::string(name) + ": " + what + " must be a contiguous CUDA tensor");
  return t.get_device();
}

void check_places(const char* name, const Tensor& pos_of, int dev) {
  if (pos_of.scalar_type() != at::kInt || pos_of.dim() != 2 || !usable(pos_of, dev))
    refuse(std::string(name) + ": pos_of must be contiguous int32 [tokens, top_k] on the rows' CUDA device");
}

void check_offsets(const char* name, const Tensor& offsets, int dev) {
  if (offsets.scalar_type() != at::kInt || offsets.dim() != 1 || !usable(offsets, dev))
    refuse(std::string(name) + ": offsets must be contiguous int32 [experts + 1] on the rows' CUDA device");
}

int check_weights(const char* name, const Tensor& w, const Tensor& rows, int64_t N, int64_t k, int dev) {
  if ((w.scalar_type() != rows.scalar_type() && w.scalar_type() != at::kFloat) || w.dim() != 2 || w.size(0) != N ||
      w.size(1) != k || !usable(w, dev))
    refuse(std::string(name) + ": w must be contiguous [" + std::to_string(N) + ", " + std::to_string(k) +
           "], float32 or of the rows' dtype, on their CUDA device");
  return row_code(name, w);
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// A size as the C ABI takes it: past 32 bits it is refused there, as the largest one.
int as_int(int64_t v) { return (int)std::min<int64_t>(v, 0x7fffffff); }

Tensor permute(const Tensor& h, const Tensor& pos_of, const Tensor& offsets) {
  const char* name = "permute_rows";
  const int dev = on_device(name, h, "h"), code = row_code(name, h);
  check_places(name, pos_of, dev);
  check_offsets(name, offsets, dev);
  const int64_t N = pos_of.size(0), k = pos_of.size(1);
  if (h.dim() != 2 || h.size(0) != N) refuse(std::string(name) + ": h must be [" + std::to_string(N) + ", hidden], got " + shape_of(h));
  const int64_t H = h.size(1);
  c10::cuda::CUDAGuard guard(dev);
  Tensor x = at::empty({N * k, H}, h.options());
  done(name, sy_permute_rows(ptr(h), pos_of.const_data_ptr<int32_t>(), offsets.const_data_ptr<int32_t>(), as_int(N), as_int(k),
                             as_int(offsets.numel() - 1), as_int(H), code, ptr(x), c10::cuda::getCurrentCUDAStream(dev).stream()));
  return x;
}

Tensor unpermute(const Tensor& y, const Tensor& w, const Tensor& pos_of) {
  const char* name = "unpermute_rows";
  const int dev = on_device(name, y, "y"), code = row_code(name, y);
  check_places(name, pos_of, dev);
  const int64_t N = pos_of.size(0), k = pos_of.size(1);
  if (y.dim() != 2 || y.size(0) != N * k)
    refuse(std::string(name) + ": y must be [" + std::to_string(N * k) + ", hidden], got " + shape_of(y));
  const int wcode = w.defined() ? check_weights(name, w, y, N, k, dev) : code;
  const int64_t H = y.size(1);
  c10::cuda::CUDAGuard guard(dev);
  Tensor out = at::empty({N, H}, y.options());
  done(name, sy_unpermute_rows(ptr(y), ptr(w), wcode, pos_of.const_data_ptr<int32_t>(), as_int(N), as_int(k), as_int(H), code, ptr(out),
                               c10::cuda::getCurrentCUDAStream(dev).stream()));
  return out;
}

std::pair<Tensor, Tensor> unpermute_grad(const Tensor& dout, const Tensor& y, const Tensor& w, const Tensor& pos_of,
                                         const Tensor& offsets, bool need_dy, bool need_dw) {
  const char* name = "unpermute_rows_grad";
  const int dev = on_device(name, dout, "dout"), code = row_code(name, dout);
  check_places(name, pos_of, dev);
  check_offsets(name, offsets, dev);
  const int64_t N = pos_of.size(0), k = pos_of.size(1);
  if (dout.dim() != 2 || dout.size(0) != N)
    refuse(std::string(name) + ": dout must be [" + std::to_string(N) + ", hidden], got " + shape_of(dout));
  const int64_t H = dout.size(1);
  if (y.defined() && (y.scalar_type() != dout.scalar_type() || y.dim() != 2 || y.size(0) != N * k || y.size(1) != H || !usable(y, dev)))
    refuse(std::string(name) + ": y must be a contiguous CUDA tensor [" + std::to_string(N * k) + ", " + std::to_string(H) +
           "] in dout's dtype and on its device");
  if (need_dw && !(y.defined() && w.defined())) refuse(std::string(name) + ": the weights' gradient needs y and w");
  const int wcode = w.defined() ? check_weights(name, w, dout, N, k, dev) : code;
  c10::cuda::CUDAGuard guard(dev);
  Tensor dy, dw;
  if (need_dy) dy = at::empty({N * k, H}, dout.options());
  if (need_dw) dw = at::empty({N, k}, w.options());
  done(name, sy_unpermute_rows_grad(ptr(dout), ptr(y), ptr(w), wcode, pos_of.const_data_ptr<int32_t>(), offsets.const_data_ptr<int32_t>(),
                                    as_int(N), as_int(k), as_int(offsets.numel() - 1), as_int(H), code, ptr(dy), ptr(dw),
                                    c10::cuda::getCurrentCUDAStream(dev).stream()));
  return {dy, dw};
}

// An argument of an autograd node that may be absent (an undefined tensor may not be one).
using Maybe = std::optional<Tensor>;
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }

// A gradient as the kernels take it. Autograd may hand over any view of its producer's: expanded, strided, or
// a slice of a flat buffer that starts between 16-byte boundaries.
Tensor incoming(const Tensor& d) {
  Tensor c = d.contiguous();
  return (uintptr_t)c.data_ptr() % 16 == 0 ? c : c.clone();
}

// Hands a gradient on, in a graph with what it was made from, and has no gradient.
struct NoSecond : torch::autograd::Function<NoSecond> {
  static Tensor forward(AutogradContext*, const Tensor& g, const Tensor&, const Maybe&, const Maybe&) { return g; }
  static variable_list backward(AutogradContext*, const variable_list&) {
    refuse("permute_rows and unpermute_rows have no second derivatives");
  }
};

// The gradient g, made from d, y and w. Where a graph of it is being recorded it is tied to those: a derivative of
// it is then refused, wherever it is asked for, and not left out of a sum.
Tensor last(const Tensor& g, const Tensor& d, const Tensor& y, const Tensor& w) {
  const auto asks = [](const Tensor& t) { return t.defined() && t.requires_grad(); };
  if (!(g.defined() && at::GradMode::is_enabled() && (asks(d) || asks(y) || asks(w)))) return g;
  return NoSecond::apply(g, d, maybe(y), maybe(w));
}

struct Permute : torch::autograd::Function<Permute> {
  static Tensor forward(AutogradContext* ctx, const Tensor& h, const Tensor& offsets, const Tensor& pos_of) {
    ctx->save_for_backward({pos_of});
    return permute(h, pos_of, offsets);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor dh = unpermute(incoming(grads[0]), Tensor(), saved[0]);
    return {last(dh, grads[0], Tensor(), Tensor()), Tensor(), Tensor()};
  }
};

struct Unpermute : torch::autograd::Function<Unpermute> {
  static Tensor forward(AutogradContext* ctx, const Tensor& y, const Maybe& weights, const Tensor& offsets, const Tensor& pos_of) {
    const Tensor w = weights.value_or(Tensor());
    const bool dw = w.defined() && w.requires_grad();  // (y is kept for the weights' gradient alone)
    ctx->save_for_backward({dw ? y : Tensor(), w, offsets, pos_of});
    return unpermute(y, w, pos_of);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &y = saved[0], &w = saved[1];
    const auto [dy, dw] = unpermute_grad(incoming(grads[0]), y, w, saved[3], saved[2], ctx->needs_input_grad(0),
                                         ctx->needs_input_grad(1) && y.defined());
    return {last(dy, grads[0], y, w), last(dw, grads[0], y, w), Tensor(), Tensor()};
  }
};

void refuse_tangent(const char* name, const Tensor& t) {
  if (t.defined() && t._fw_grad(0).defined()) refuse(std::string(name) + " has no forward-mode derivative: unpack its dual inputs first");
}

// ---- Python ---------------------------------------------------------------------------------
Tensor tensor_arg(PyObject* const* args, Py_ssize_t n, Py_ssize_t i, bool may_be_none = false) {
  if (may_be_none && args[i] == Py_None) return Tensor();
  if (i >= n || !THPVariable_Check(args[i])) refuse("argument " + std::to_string(i + 1) + " must be a tensor");
  return THPVariable_Unpack(args[i]);
}
void expect(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) refuse("expected " + std::to_string(want) + " arguments, got " + std::to_string(n));
}
PyObject* wrap(Tensor t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(t));
}

// (h, pos_of, offsets)
PyObject* py_permute(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 3);
  const Tensor h = tensor_arg(args, n, 0), pos_of = tensor_arg(args, n, 1), offsets = tensor_arg(args, n, 2);
  Tensor x;
  {
    pybind11::gil_scoped_release no_gil;
    x = permute(h, pos_of, offsets);
  }
  return wrap(x);
  END_HANDLE_TH_ERRORS
}

PyObject* py_permute_autograd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 3);
  const Tensor given = tensor_arg(args, n, 0), pos_of = tensor_arg(args, n, 1), offsets = tensor_arg(args, n, 2);
  Tensor x;
  {
    pybind11::gil_scoped_release no_gil;
    refuse_tangent("permute_rows", given);
    const Tensor h = given.contiguous();
    x = at::GradMode::is_enabled() && h.requires_grad() ? Permute::apply(h, offsets, pos_of) : permute(h, pos_of, offsets);
  }
  return wrap(x);
  END_HANDLE_TH_ERRORS
}

// (y, w or None, pos_of)
PyObject* py_unpermute(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 3);
  const Tensor y = tensor_arg(args, n, 0), w = tensor_arg(args, n, 1, true), pos_of = tensor_arg(args, n, 2);
  Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    out = unpermute(y, w, pos_of);
  }
  return wrap(out);
  END_HANDLE_TH_ERRORS
}

// (y, w or None, pos_of, offsets)
PyObject* py_unpermute_autograd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 4);
  const Tensor given = tensor_arg(args, n, 0), given_w = tensor_arg(args, n, 1, true), pos_of = tensor_arg(args, n, 2),
               offsets = tensor_arg(args, n, 3);
  Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    refuse_tangent("unpermute_rows", given);
    refuse_tangent("unpermute_rows", given_w);
    const Tensor y = given.contiguous(), w = given_w.defined() ? given_w.contiguous() : given_w;
    const bool graph = at::GradMode::is_enabled() && (y.requires_grad() || (w.defined() && w.requires_grad()));
    out = graph ? Unpermute::apply(y, maybe(w), offsets, pos_of) : unpermute(y, w, pos_of);
  }
  return wrap(out);
  END_HANDLE_TH_ERRORS
}

// (dout, y or None, w or None, pos_of, offsets, need_dy, need_dw) -> (dy or None, dw or None)
PyObject* py_unpermute_grad(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 7);
  const Tensor dout = tensor_arg(args, n, 0), y = tensor_arg(args, n, 1, true), w = tensor_arg(args, n, 2, true),
               pos_of = tensor_arg(args, n, 3), offsets = tensor_arg(args, n, 4);
  const int need_dy = PyObject_IsTrue(args[5]), need_dw = PyObject_IsTrue(args[6]);
  if (need_dy < 0 || need_dw < 0) return nullptr;
  std::pair<Tensor, Tensor> grads;
  {
    pybind11::gil_scoped_release no_gil;
    grads = unpermute_grad(dout, y, w, pos_of, offsets, need_dy, need_dw);
  }
  PyObject* pair = PyTuple_New(2);
  if (!pair) return nullptr;
  PyTuple_SET_ITEM(pair, 0, wrap(grads.first));
  PyTuple_SET_ITEM(pair, 1, wrap(grads.second));
  return pair;
  END_HANDLE_TH_ERRORS
}

// (tensors or None...) -> what they ask of a call that has no derivatives: 2 one has a forward-mode tangent, 1
// gradients are being recorded and one requires its own, 0 nothing
PyObject* py_asks(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  long asks = 0;
  for (Py_ssize_t i = 0; i < n; ++i) {
    const Tensor t = tensor_arg(args, n, i, true);
    if (!t.defined()) continue;
    if (t._fw_grad(0).defined()) return PyLong_FromLong(2);
    if (t.requires_grad() && at::GradMode::is_enabled()) asks = 1;
  }
  return PyLong_FromLong(asks);
  END_HANDLE_TH_ERRORS
}

#define SY_METHOD(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {SY_METHOD("permute", py_permute),
                         SY_METHOD("permute_autograd", py_permute_autograd),
                         SY_METHOD("unpermute", py_unpermute),
                         SY_METHOD("unpermute_autograd", py_unpermute_autograd),
                         SY_METHOD("unpermute_grad", py_unpermute_grad),
                         SY_METHOD("asks", py_asks),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_rows_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__rows_torch(void) { return PyModule_Create(&module); }
