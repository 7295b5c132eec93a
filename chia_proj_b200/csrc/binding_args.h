// binding_args.h -- what the functions of the CPython module share: reading of
// arguments, checks of tensors, errors.
#pragma once
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstring>
#include <map>
#include <stdexcept>
#include <string>
#include <utility>

#include "../../include/chia_draft.h"

namespace {

using at::Tensor;

struct ValueError : std::runtime_error {
  using std::runtime_error::runtime_error;
};

std::string str(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + ")";
}

// ------------------------------------------------------------------ arguments
struct Args {
  PyObject *const *v;
  Py_ssize_t n;
  Args(PyObject *const *args, Py_ssize_t nargs, Py_ssize_t want) : v(args), n(nargs) {
    if (nargs != want) throw ValueError("wrong number of arguments");
  }
  int64_t integer(int i) const {
    const long long x = PyLong_AsLongLong(v[i]);
    if (x == -1 && PyErr_Occurred()) throw 0;
    return x;
  }
  double number(int i) const {
    const double x = PyFloat_AsDouble(v[i]);
    if (x == -1.0 && PyErr_Occurred()) throw 0;
    return x;
  }
  bool none(int i) const { return v[i] == Py_None; }
  // A tensor of `dim` dimensions on a GPU.
  const Tensor &tensor(int i, const char *name, int64_t dim) const {
    if (!THPVariable_Check(v[i])) throw ValueError(std::string(name) + " must be a " + std::to_string(dim) + "-D tensor");
    const Tensor &t = THPVariable_Unpack(v[i]);
    if (t.dim() != dim) throw ValueError(std::string(name) + " must be a " + std::to_string(dim) + "-D tensor");
    if (!t.is_cuda())
      throw std::runtime_error(std::string(name) + " is on " + t.device().str() +
                               ": the library runs on CUDA only (no CPU fallback)");
    return t;
  }
  // int32 of this shape and device, unit stride in the last dimension.
  const Tensor &ints(int i, const char *name, at::IntArrayRef shape, const at::Device &dev) const {
    const Tensor &t = tensor(i, name, static_cast<int64_t>(shape.size()));
    if (t.scalar_type() != at::kInt || t.sizes() != shape || t.device() != dev)
      throw ValueError(std::string(name) + " must be int32 " + str(shape) + " on " + dev.str() + ", got " +
                       c10::toString(t.scalar_type()) + " " + str(t.sizes()) + " on " + t.device().str());
    if (t.size(-1) > 1 && t.stride(-1) != 1) throw ValueError(std::string(name) + " must have unit stride");
    return t;
  }
};

template <class T>
T *ptr(const Tensor &t) {
  return static_cast<T *>(t.data_ptr());
}

bool page_ok(int64_t p) { return p == 16 || p == 32 || p == 64 || p == 128; }
void check_page(int64_t p) {
  if (!page_ok(p)) throw ValueError("page_size " + std::to_string(p) + " unsupported (16, 32, 64 or 128)");
}

int value_type(const Tensor &t) {
  return t.scalar_type() == at::kBFloat16 ? CHIA_DTYPE_BF16 : t.scalar_type() == at::kHalf ? CHIA_DTYPE_F16 : -1;
}

// A dense copy at an address of its own (contiguous() gives back a dense tensor as it is, wherever it begins).
Tensor fitting(const Tensor &t) { return t.detach().clone(at::MemoryFormat::Contiguous); }

// Unit stride on the channels, 16-byte aligned rows; a copy where it is not so.
bool fits(const Tensor &t) {
  return t.stride(2) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && t.stride(0) >= 0 &&
         t.stride(1) >= 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

// No two elements of [rows, heads, channels] share memory.
bool apart(const Tensor &t) {
  if (t.numel() == 0) return true;
  const int near = t.stride(0) < t.stride(1) ? 0 : 1;  // the dimension of the smaller stride
  const int64_t one = t.size(near) > 1 ? t.stride(near) : t.size(2);
  const int64_t all = (t.size(near) - 1) * one + t.size(2);
  return one >= t.size(2) && (t.size(1 - near) == 1 || t.stride(1 - near) >= all);
}

// The kernels write below autograd; this tells it (a tensor that a graph has saved
// must not change unseen).
void written(const Tensor &t) {
  if (!t.unsafeGetTensorImpl()->is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void no_tangent(const Tensor &t, const char *name) {
  if (t._fw_grad(0).defined())
    throw ValueError(std::string(name) + " has a forward-mode tangent: there is no derivative");
}

struct Cache {
  const Tensor &k, &v, &ks, &vs;
  int type;
  at::Device dev;
  int64_t pages, heads, page, dim;
  Cache(const Args &a, int i)
      : k(a.tensor(i, "k_cache", 4)), v(a.tensor(i + 1, "v_cache", 4)), ks(a.tensor(i + 2, "k_scale", 2)),
        vs(a.tensor(i + 3, "v_scale", 2)), dev(k.device()) {
    const auto ty = k.scalar_type();
    type = ty == at::kFloat8_e4m3fn ? CHIA_CACHE_E4M3 : ty == at::kChar ? CHIA_CACHE_INT8 : -1;
    if (type < 0 || v.scalar_type() != ty)
      throw ValueError(std::string("k_cache, v_cache must share a type, float8_e4m3fn or int8; got ") +
                       c10::toString(ty) + ", " + c10::toString(v.scalar_type()));
    if (v.sizes() != k.sizes() || v.device() != dev)
      throw ValueError("k_cache, v_cache must match in shape and device");
    if (!k.is_contiguous() || !v.is_contiguous()) throw ValueError("k_cache, v_cache must be contiguous");
    pages = k.size(0), heads = k.size(1), page = k.size(2), dim = k.size(3);
    check_page(page);
    if (dim != 64 && dim != 128) throw ValueError("head_dim " + std::to_string(dim) + " unsupported (64 or 128)");
    if (pages < 1 || heads < 1) throw ValueError("empty cache");
    for (const Tensor *s : {&ks, &vs})
      if (s->scalar_type() != at::kFloat || s->size(0) != pages || s->size(1) != heads || s->device() != dev ||
          !s->is_contiguous())
        throw ValueError(std::string(s == &ks ? "k_scale" : "v_scale") + " must be contiguous fp32 (" +
                         std::to_string(pages) + ", " + std::to_string(heads) + ") on " + dev.str());
  }
};

// Any C++ exception ends here as a Python one; one that Python threw below (a hook of saved tensors: a
// checkpoint stops its second run by one) goes on as it is.
template <class F>
PyObject *guarded(F f) {
  try {
    return f();
  } catch (int) {
    return nullptr;  // the Python error is set
  } catch (python_error &e) {
    e.restore();
  } catch (py::error_already_set &e) {
    e.restore();
  } catch (const ValueError &e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const c10::Error &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// Elements [at, at + n) of a 1-D tensor, sharing its storage (narrow() takes ten
// times as long to set up).
Tensor piece(const Tensor &buf, int64_t at, int64_t n) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(buf.storage()),
                                                      buf.key_set(), buf.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(at);
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return t;
}

}  // namespace
