// The layer operators on torch tensors, as a Python extension module
// (ferrograd_b200._layer; the documented functions are in kernels.py).  It
// checks the tensors, allocates outputs and workspace and calls the C ABI
// (include/ferro_cuda.h): what ctypes and the interpreter took 10 of a small
// call's 16 us for.  torch gives memory and the current stream, nothing else.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <string>

#include "../../include/ferro_cuda.h"

namespace {

// A Python error is set; carries no more.
struct Raised {};

[[noreturn]] void value_error(const std::string &message) {
  PyErr_SetString(PyExc_ValueError, message.c_str());
  throw Raised{};
}

// Raises FerroError(code, fg_last_error()) for a failed C-ABI call.
void check(int code) {
  if (code == FG_OK) return;
  PyObject *mod = PyImport_ImportModule("ferrograd_b200._lib");
  PyObject *cls = mod ? PyObject_GetAttrString(mod, "FerroError") : nullptr;
  PyObject *err = cls ? PyObject_CallFunction(cls, "is", code, fg_last_error()) : nullptr;
  if (err) PyErr_SetObject(cls, err);
  Py_XDECREF(err);
  Py_XDECREF(cls);
  Py_XDECREF(mod);
  throw Raised{};
}

const at::Tensor &tensor(PyObject *o, const char *name) {
  if (!THPVariable_Check(o)) value_error(std::string(name) + ": expected a tensor");
  const at::Tensor &t = THPVariable_Unpack(o);
  // (such a view's memory holds the values before the sign, or nothing)
  if (t.is_neg() || t._is_zerotensor())
    value_error(std::string(name) + ": a lazily negated or zero tensor (see resolve_neg)");
  return t;
}

double real(PyObject *o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised{};
  return v;
}
unsigned long long word(PyObject *o) {  // modulo 2^64
  const unsigned long long v = PyLong_AsUnsignedLongLongMask(o);
  if (PyErr_Occurred()) throw Raised{};
  return v;
}
int integer(PyObject *o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  return (int)v;
}
bool truth(PyObject *o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Raised{};
  return v != 0;
}

std::string shape_text(at::IntArrayRef s) {
  std::string t = "(";
  for (size_t i = 0; i < s.size(); i++)
    t += (i ? ", " : "") + std::to_string(s[i]) + (s.size() == 1 ? "," : "");
  return t + ")";
}

// What every tensor of a call shares with x.
struct Like {
  const at::Tensor &x;
  int code;
  explicit Like(const at::Tensor &x_) : x(x_) {
    if (!x.is_cuda()) value_error("expected a CUDA tensor, got " + x.device().str());
    switch (x.scalar_type()) {
      case at::kFloat:
        code = FG_F32;
        break;
      case at::kBFloat16:
        code = FG_BF16;
        break;
      case at::kHalf:
        code = FG_F16;
        break;
      default:
        value_error(std::string("unsupported dtype ") + c10::toString(x.scalar_type()));
    }
  }
  // A tensor of x's dtype and device and this shape (unit_cols: its last
  // dimension has stride 1).
  void check(const char *name, const at::Tensor &t, at::IntArrayRef shape, bool unit_cols) const {
    if (t.device() != x.device())
      value_error(std::string(name) + ": expected a CUDA tensor on " + x.device().str() + ", got " +
                  t.device().str());
    if (t.scalar_type() != x.scalar_type())
      value_error(std::string(name) + ": expected " + c10::toString(x.scalar_type()) + ", got " +
                  c10::toString(t.scalar_type()));
    if (t.sizes() != shape)
      value_error(std::string(name) + ": expected shape " + shape_text(shape) + ", got " +
                  shape_text(t.sizes()));
    if (unit_cols && !shape.empty() && t.strides().back() != 1 && shape.back() > 1 && t.numel() > 0)
      value_error(std::string(name) + ": expected unit stride in the last dimension");
  }
};

// Row pitch of a 2-D tensor with unit column stride (rows of one row, or of one
// element, may carry any stride).
int64_t pitch(const at::Tensor &t) {
  return t.size(0) <= 1 ? std::max(t.stride(0), t.size(1)) : t.stride(0);
}

int32_t extent(int64_t n) {  // the C ABI refuses what is beyond its range
  return n > 0x7fffffff ? 0x7fffffff : (int32_t)n;
}

at::Tensor empty(const at::Tensor &x, at::IntArrayRef shape) {
  return at::empty(shape, x.options().memory_format(at::MemoryFormat::Contiguous));
}

// The stream of a call: torch's current one, or the one given.  On another
// stream than the current one the call's memory has to be that stream's own:
// the allocator hands out blocks whose last use is over in the order of the
// stream they are allocated for, and of no other.  So everything is allocated
// with that stream current; arguments are kept from reuse until it is done with
// them, and results until the caller's stream is.
class Launch {
 public:
  cudaStream_t st;

  Launch(const at::Tensor &x, PyObject *stream)
      : device_(x.device()), caller_(c10::cuda::getCurrentCUDAStream(x.device().index())) {
    st = caller_.stream();
    if (stream == Py_None) return;
    cudaStream_t given = (cudaStream_t)word(stream);
    if (given == cudaStreamLegacy) given = nullptr;  // the same stream by its other name
    if (given == st) return;
    st = given;
    guard_.reset_stream(c10::cuda::getStreamFromExternal(st, x.device().index()));
  }
  void uses(const at::Tensor &t) {
    if (guard_.current_stream().has_value())
      t.record_stream(guard_.current_stream().value().unwrap());
  }
  void gives(const at::Tensor &t) {
    if (guard_.current_stream().has_value() && t.defined()) t.record_stream(caller_.unwrap());
  }

 private:
  c10::cuda::CUDAGuard device_;
  c10::cuda::CUDAStream caller_;
  c10::cuda::OptionalCUDAStreamGuard guard_;
};

// Runs a C-ABI call with the workspace it asks for.
template <typename Args>
void run(const at::Tensor &x, const Launch &on, Args &a, int (*ask)(const Args *, size_t *),
         int (*call)(const Args *, void *)) {
  size_t need = 0;
  check(ask(&a, &need));
  at::Tensor ws;
  if (need) {
    ws = at::empty({(int64_t)need}, x.options().dtype(at::kByte));
    a.workspace = ws.data_ptr();
    a.workspace_bytes = need;
  }
  check(call(&a, on.st));
}

void set_drop(fg_dropout_spec &d, PyObject *p, PyObject *seed, PyObject *offset) {
  d.p = real(p);
  d.seed = word(seed);
  d.offset = word(offset);
}

struct Product {
  int64_t M, N, K;
};
Product product(const Like &like, const at::Tensor &x, const at::Tensor &w) {
  if (x.dim() != 2 || w.dim() != 2) value_error("expected 2-D x and w");
  const Product s{x.size(0), w.size(0), x.size(1)};
  like.check("w", w, {s.N, s.K}, false);
  return s;
}

// linear(x, w, bias, act, residual, p, seed, offset, save_pre, out, stream)
PyObject *linear(PyObject *const *o) {
  const at::Tensor &x = tensor(o[0], "x"), &w = tensor(o[1], "w");
  const Like like(x);
  const Product s = product(like, x, w);
  Launch on(x, o[10]);
  on.uses(x), on.uses(w);
  fg_linear_args a{};
  a.dtype = like.code;
  a.M = extent(s.M), a.N = extent(s.N), a.K = extent(s.K);
  a.x = x.data_ptr(), a.x_row = x.stride(0), a.x_col = x.stride(1);
  a.w = w.data_ptr(), a.w_row = w.stride(0), a.w_col = w.stride(1);
  if (o[2] != Py_None) {
    const at::Tensor &bias = tensor(o[2], "bias");
    like.check("bias", bias, {s.N}, true);
    on.uses(bias);
    a.bias = bias.data_ptr();
  }
  a.act = integer(o[3]);
  if (o[4] != Py_None) {
    const at::Tensor &r = tensor(o[4], "residual");
    like.check("residual", r, {s.M, s.N}, true);
    on.uses(r);
    a.residual = r.data_ptr(), a.ld_residual = pitch(r);
  }
  set_drop(a.drop, o[5], o[6], o[7]);
  const bool save_pre = truth(o[8]);
  at::Tensor out, pre;
  if (o[9] == Py_None) {
    out = empty(x, {s.M, s.N});
    on.gives(out);
  } else {
    out = tensor(o[9], "out");
    like.check("out", out, {s.M, s.N}, true);
    on.uses(out);
  }
  a.out = out.data_ptr(), a.ld_out = pitch(out);
  if (save_pre) {
    pre = empty(x, {s.M, s.N});
    on.gives(pre);
    a.pre = pre.data_ptr(), a.ld_pre = s.N;
  }
  run(x, on, a, fg_linear_workspace, fg_linear);
  PyObject *result = o[9] == Py_None ? THPVariable_Wrap(out) : Py_NewRef(o[9]);
  if (!save_pre) return result;
  return Py_BuildValue("(NN)", result, THPVariable_Wrap(pre));
}

// linear_grad(dy, x, w, pre, act, p, seed, offset, need_dx, need_dw, need_db,
//             dx_residual, stream)
PyObject *linear_grad(PyObject *const *o) {
  const at::Tensor &dy = tensor(o[0], "dy"), &x = tensor(o[1], "x"), &w = tensor(o[2], "w");
  const Like like(x);
  const Product s = product(like, x, w);
  like.check("dy", dy, {s.M, s.N}, false);
  Launch on(x, o[12]);
  on.uses(dy), on.uses(x), on.uses(w);
  fg_linear_grad_args a{};
  a.dtype = like.code;
  a.M = extent(s.M), a.N = extent(s.N), a.K = extent(s.K);
  a.dy = dy.data_ptr(), a.dy_row = dy.stride(0), a.dy_col = dy.stride(1);
  a.x = x.data_ptr(), a.x_row = x.stride(0), a.x_col = x.stride(1);
  a.w = w.data_ptr(), a.w_row = w.stride(0), a.w_col = w.stride(1);
  a.act = integer(o[4]);
  if (a.act != FG_ACT_NONE) {
    const at::Tensor &pre = tensor(o[3], "pre");
    like.check("pre", pre, {s.M, s.N}, true);
    on.uses(pre);
    a.pre = pre.data_ptr(), a.ld_pre = pitch(pre);
  }
  set_drop(a.drop, o[5], o[6], o[7]);
  at::Tensor dx, dw, db;
  if (truth(o[8])) {
    dx = empty(x, {s.M, s.K});
    a.dx = dx.data_ptr(), a.ld_dx = s.K;
    if (o[11] != Py_None) {
      const at::Tensor &r = tensor(o[11], "dx_residual");
      like.check("dx_residual", r, {s.M, s.K}, true);
      on.uses(r);
      a.dx_residual = r.data_ptr(), a.ld_dx_residual = pitch(r);
    }
  } else if (o[11] != Py_None) {
    value_error("dx_residual without dx");
  }
  if (truth(o[9])) {
    dw = empty(x, {s.N, s.K});
    a.dw = dw.data_ptr(), a.ld_dw = s.K;
  }
  if (truth(o[10])) {
    db = empty(x, {s.N});
    a.db = db.data_ptr();
  }
  on.gives(dx), on.gives(dw), on.gives(db);
  run(x, on, a, fg_linear_grad_workspace, fg_linear_grad);
  // an undefined tensor wraps as None
  return Py_BuildValue("(NNN)", THPVariable_Wrap(dx), THPVariable_Wrap(dw), THPVariable_Wrap(db));
}

// dropout(x, residual, p, seed, offset, out, stream)
PyObject *dropout(PyObject *const *o) {
  const at::Tensor &x = tensor(o[0], "x");
  const Like like(x);
  Launch on(x, o[6]);
  on.uses(x);
  const auto shape = x.sizes();
  const bool flat = shape.size() != 2;  // rows are then a contiguous tensor's
  const int64_t cols = shape.empty() ? 1 : shape.back();
  const int64_t rows = cols ? x.numel() / cols : 0;
  auto rows_of = [&](const char *name, const at::Tensor &t) {
    like.check(name, t, shape, !flat);
    if (flat && !t.is_contiguous())
      value_error(std::string(name) + ": expected a 2-D or a contiguous tensor");
    return flat ? cols : pitch(t);
  };
  const int64_t ldx = rows_of("x", x);
  at::Tensor r, out;
  int64_t ldr = 0;
  if (o[1] != Py_None) {
    r = tensor(o[1], "residual");
    ldr = rows_of("residual", r);
    on.uses(r);
  }
  fg_dropout_spec drop{};
  set_drop(drop, o[2], o[3], o[4]);
  out = o[5] == Py_None ? empty(x, shape) : tensor(o[5], "out");
  const int64_t ldo = rows_of("out", out);
  o[5] == Py_None ? on.gives(out) : on.uses(out);
  check(fg_dropout(like.code, (size_t)rows, (size_t)cols, x.data_ptr(), ldx,
                   r.defined() ? r.data_ptr() : nullptr, ldr, out.data_ptr(), ldo, &drop, on.st));
  return o[5] == Py_None ? THPVariable_Wrap(out) : Py_NewRef(o[5]);
}

// Sets the error module.name(message).
void raise(const char *module, const char *name, const char *message) {
  PyObject *mod = PyImport_ImportModule(module);
  PyObject *cls = mod ? PyObject_GetAttrString(mod, name) : nullptr;
  if (cls) PyErr_SetString(cls, message);
  Py_XDECREF(cls);
  Py_XDECREF(mod);
}

// No C++ exception leaves the module.
template <PyObject *(*F)(PyObject *const *), Py_ssize_t N>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  if (nargs != N) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", N, nargs);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Raised &) {
    return nullptr;
  } catch (const c10::OutOfMemoryError &e) {
    raise("torch", "OutOfMemoryError", e.what_without_backtrace());
  } catch (const c10::Error &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

template <PyObject *(*F)(PyObject *const *), Py_ssize_t N>
PyMethodDef method(const char *name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, N>)),
          METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {method<linear, 11>("linear"), method<linear_grad, 13>("linear_grad"),
                         method<dropout, 7>("dropout"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_layer", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__layer(void) { return PyModule_Create(&module); }
