// The general operators' calls on torch tensors (module arctic_tensors, used by arctic_embed_s_int8.Engine): reads the
// tensors' sizes, strides and addresses, checks them, and calls the C ABI. The same checks through the tensors'
// Python attributes cost 3.5 us a call, as much as the launch itself; these take a few tenths.
//
// Each function takes the context's address, the GPU's index and the tensors, raises ValueError for a tensor that
// does not fit, and returns the C ABI's status code. bind() receives the C functions' addresses, so that this
// module and the ctypes binding use one loaded library.
#include <Python.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <exception>

#include "../../include/arctic_cuda.h"

namespace {

decltype(&ae_matmul_i8) g_matmul = nullptr;
decltype(&ae_linear_i8) g_linear = nullptr;
decltype(&ae_qk_norm_rope) g_qk = nullptr;

struct Refused {};  // a Python exception is set

[[noreturn]] void refuse(const char* fmt, const char* what, const char* detail = "") {
  PyErr_Format(PyExc_ValueError, fmt, what, detail);
  throw Refused{};
}

const at::Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) refuse("%s must be a torch tensor%s", what);
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.is_neg()) refuse("%s holds the negatives of its values: call resolve_neg() on it%s", what);
  // as torch refuses operations with out=: a gradient would end here without a word
  if (t.requires_grad() && c10::GradMode::is_enabled())
    refuse("%s requires grad, but no gradients are computed: call this under torch.no_grad()%s", what);
  return t;
}

// For autograd, which otherwise takes what it saved of a result for what it still holds.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

const char* type_name(at::ScalarType t) {
  switch (t) {
    case at::kChar: return "int8";
    case at::kInt: return "int32";
    case at::kFloat: return "float32";
    case at::kHalf: return "float16";
    case at::kBFloat16: return "bfloat16";
    default: return "of its type";
  }
}

int float_type(const at::Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return AE_F32;
    case at::kHalf: return AE_F16;
    case at::kBFloat16: return AE_BF16;
    default: refuse("%s must be float32, float16 or bfloat16%s", what);
  }
}

void on_gpu(const at::Tensor& t, const char* what, int64_t device) {
  if (!t.is_cuda() || t.get_device() != device) refuse("%s must be in device memory of the engine's GPU%s", what);
}

void of_type(const at::Tensor& t, const char* what, at::ScalarType type) {
  if (t.scalar_type() != type) refuse("%s must be %s", what, type_name(type));
}

// Sizes as the C ABI takes them; larger ones are refused there.
uint32_t count(int64_t n) { return n > 0xffffffffll ? 0xffffffffu : uint32_t(n); }

template <class T>
T* at_address(const at::Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}

// A contiguous [n] tensor.
const at::Tensor& vector(PyObject* o, const char* what, int64_t n, at::ScalarType type, int64_t device) {
  const at::Tensor& t = tensor(o, what);
  if (t.dim() != 1 || t.size(0) != n) {
    PyErr_Format(PyExc_ValueError, "%s must have %lld elements in one axis", what, (long long)n);
    throw Refused{};
  }
  of_type(t, what, type);
  on_gpu(t, what, device);
  if (n > 1 && t.stride(0) != 1) refuse("%s must be contiguous%s", what);
  return t;
}

const float* floats_or_none(PyObject* o, const char* what, int64_t n, int64_t device) {
  return o == Py_None ? nullptr : at_address<const float>(vector(o, what, n, at::kFloat, device));
}

// A [rows, cols] tensor whose rows are contiguous.
const at::Tensor& matrix(PyObject* o, const char* what, int64_t rows, int64_t cols, int64_t device) {
  const at::Tensor& t = tensor(o, what);
  if (t.dim() != 2 || t.size(0) != rows || t.size(1) != cols) {
    PyErr_Format(PyExc_ValueError, "%s must be [%lld, %lld]", what, (long long)rows, (long long)cols);
    throw Refused{};
  }
  on_gpu(t, what, device);
  if (rows && cols > 1 && t.stride(1) != 1) refuse("%s must be contiguous along its last axis%s", what);
  return t;
}

// Row pitch in elements; that of a single row is the row's own length.
uint64_t pitch(const at::Tensor& t) {
  return uint64_t(t.size(0) > 1 && t.size(1) ? t.stride(0) : t.size(1));
}

// None, a closed engine's, is the null context, which the C ABI refuses.
ae_ctx* context(PyObject* o) {
  if (o == Py_None) return nullptr;
  void* p = PyLong_AsVoidPtr(o);
  if (!p && PyErr_Occurred()) throw Refused{};
  return static_cast<ae_ctx*>(p);
}

int64_t whole(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Refused{};
  return v;
}

// The C call without the interpreter's lock, as ctypes makes it. `call` holds plain values: a tensor that is asked for its
// address throws where it has none, which needs the lock.
template <class F>
int unlocked(F&& call) {
  int code;
  Py_BEGIN_ALLOW_THREADS;
  code = call();
  Py_END_ALLOW_THREADS;
  return code;
}

template <class F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want, bool bound, F&& body) {
  if (n != want || !bound) {
    PyErr_SetString(PyExc_TypeError, bound ? "wrong number of arguments" : "bind() first");
    return nullptr;
  }
  try {
    return body();
  } catch (const Refused&) {
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// (context, device, a, a_scale, w, w_scale, out, bias or None)
PyObject* matmul_i8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 8, g_matmul != nullptr, [&] {
    ae_ctx* ctx = context(args[0]);
    const int64_t dev = whole(args[1]);
    const at::Tensor &a0 = tensor(args[2], "a"), &w0 = tensor(args[4], "w");
    if (a0.dim() != 2) refuse("%s must be [tokens, in_features]%s", "a");
    if (w0.dim() != 2) refuse("%s must be [out_features, in_features]%s", "w");
    const int64_t M = a0.size(0), K = a0.size(1), N = w0.size(0);
    const at::Tensor &a = matrix(args[2], "a", M, K, dev), &w = matrix(args[4], "w", N, K, dev);
    const at::Tensor& out = matrix(args[6], "out", M, N, dev);
    of_type(a, "a", at::kChar);
    of_type(w, "w", at::kChar);
    const int out_type = float_type(out, "out");
    const float* a_scale = at_address<const float>(vector(args[3], "a_scale", M, at::kFloat, dev));
    const float* w_scale = at_address<const float>(vector(args[5], "w_scale", N, at::kFloat, dev));
    const float* bias = floats_or_none(args[7], "bias", N, dev);
    const int8_t *pa = at_address<const int8_t>(a), *pw = at_address<const int8_t>(w);
    void* po = out.data_ptr();
    const uint64_t lda = pitch(a), ldw = pitch(w), ldo = pitch(out);
    const int code = unlocked([=] {
      return g_matmul(ctx, count(M), count(N), count(K), pa, lda, a_scale, pw, ldw, w_scale, bias, out_type, po, ldo);
    });
    if (code == AE_OK) written(out);
    return PyLong_FromLong(code);
  });
}

// (context, device, x, inv_smooth or None, w, w_scale, out, bias or None)
PyObject* linear_i8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 8, g_linear != nullptr, [&] {
    ae_ctx* ctx = context(args[0]);
    const int64_t dev = whole(args[1]);
    const at::Tensor &x0 = tensor(args[2], "x"), &w0 = tensor(args[4], "w");
    if (x0.dim() != 2) refuse("%s must be [tokens, in_features]%s", "x");
    if (w0.dim() != 2) refuse("%s must be [out_features, in_features]%s", "w");
    const int64_t M = x0.size(0), K = x0.size(1), N = w0.size(0);
    const at::Tensor &x = matrix(args[2], "x", M, K, dev), &w = matrix(args[4], "w", N, K, dev);
    const at::Tensor& out = matrix(args[6], "out", M, N, dev);
    of_type(w, "w", at::kChar);
    const int x_type = float_type(x, "x"), out_type = float_type(out, "out");
    const float* smooth = floats_or_none(args[3], "inv_smooth", K, dev);
    const float* w_scale = at_address<const float>(vector(args[5], "w_scale", N, at::kFloat, dev));
    const float* bias = floats_or_none(args[7], "bias", N, dev);
    const int8_t* pw = at_address<const int8_t>(w);
    void *px = x.data_ptr(), *po = out.data_ptr();
    const uint64_t ldx = pitch(x), ldw = pitch(w), ldo = pitch(out);
    const int code = unlocked([=] {
      return g_linear(ctx, count(M), count(N), count(K), x_type, px, ldx, smooth, pw, ldw, w_scale, bias, out_type, po,
                      ldo);
    });
    if (code == AE_OK) written(out);
    return PyLong_FromLong(code);
  });
}

struct Heads {
  void* p;
  uint64_t token, head;
};

// A [tokens, heads, dim] tensor with contiguous heads.
Heads heads(PyObject* o, const char* what, int64_t T, int64_t H, int64_t D, at::ScalarType type, int64_t device) {
  const at::Tensor& t = tensor(o, what);
  if (t.dim() != 3 || t.size(0) != T || t.size(1) != H || t.size(2) != D) {
    PyErr_Format(PyExc_ValueError, "%s must be [%lld, %lld, %lld]", what, (long long)T, (long long)H, (long long)D);
    throw Refused{};
  }
  of_type(t, what, type);
  on_gpu(t, what, device);
  if (t.numel() && D > 1 && t.stride(2) != 1) refuse("%s must be contiguous along its last axis%s", what);
  return {t.data_ptr(), uint64_t(t.stride(0)), uint64_t(t.stride(1))};
}

// (context, device, q, k, q_out, k_out, table, positions, cu, q_weight, k_weight, eps, flags); table to k_weight or None
PyObject* qk_norm_rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 13, g_qk != nullptr, [&] {
    ae_ctx* ctx = context(args[0]);
    const int64_t dev = whole(args[1]);
    const at::Tensor &q0 = tensor(args[2], "q"), &k0 = tensor(args[3], "k");
    if (q0.dim() != 3) refuse("%s must be [tokens, heads, dim]%s", "q");
    if (k0.dim() != 3) refuse("%s must be [tokens, heads, dim]%s", "k");
    const int type = float_type(q0, "q");
    const at::ScalarType st = q0.scalar_type();
    const int64_t T = q0.size(0), Hq = q0.size(1), D = q0.size(2), Hk = k0.size(1);
    const Heads q = heads(args[2], "q", T, Hq, D, st, dev), k = heads(args[3], "k", T, Hk, D, st, dev);
    const Heads qo = heads(args[4], "q_out", T, Hq, D, st, dev), ko = heads(args[5], "k_out", T, Hk, D, st, dev);
    int64_t rows = 0, rotary = 0, seqs = 0;
    const float* table = nullptr;
    const int32_t* positions = nullptr;
    const uint32_t* cu = nullptr;
    if (args[6] != Py_None) {
      const at::Tensor& t0 = tensor(args[6], "table");
      if (t0.dim() != 2) refuse("%s must be [rows, rotary_dim]%s", "table");
      rows = t0.size(0), rotary = t0.size(1);
      const at::Tensor& t = matrix(args[6], "table", rows, rotary, dev);
      of_type(t, "table", at::kFloat);
      if (int64_t(pitch(t)) != rotary) refuse("%s must be contiguous%s", "table");
      table = at_address<const float>(t);
      if (args[7] != Py_None) {
        positions = at_address<const int32_t>(vector(args[7], "positions", T, at::kInt, dev));
      } else if (args[8] != Py_None) {
        const at::Tensor& c = tensor(args[8], "cu");
        if (c.scalar_type() != at::kInt && c.scalar_type() != at::kUInt32) refuse("%s must be int32 or uint32%s", "cu");
        if (c.dim() != 1 || c.size(0) < 1) refuse("%s must have an entry more than there are sequences%s", "cu");
        seqs = c.size(0) - 1;
        cu = at_address<const uint32_t>(vector(args[8], "cu", seqs + 1, c.scalar_type(), dev));
      } else {
        refuse("%s needs positions or cu%s", "a rotation");
      }
    }
    const float* qw = floats_or_none(args[9], "q_weight", D, dev);
    const float* kw = floats_or_none(args[10], "k_weight", D, dev);
    const double eps = PyFloat_AsDouble(args[11]);
    if (eps == -1.0 && PyErr_Occurred()) throw Refused{};
    const int flags = int(whole(args[12]));
    const int code = unlocked([=] {
      return g_qk(ctx, type, count(T), count(Hq), count(Hk), count(D), count(rotary), flags, q.p, q.token, q.head, k.p,
                  k.token, k.head, qo.p, qo.token, qo.head, ko.p, ko.token, ko.head, qw, kw, float(eps), table,
                  count(rows), positions, cu, count(seqs));
    });
    if (code == AE_OK) {
      written(tensor(args[4], "q_out"));
      written(tensor(args[5], "k_out"));
    }
    return PyLong_FromLong(code);
  });
}

// (ae_matmul_i8, ae_linear_i8, ae_qk_norm_rope) as addresses
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 3, true, [&]() -> PyObject* {
    void* p[3];
    for (int i = 0; i < 3; ++i) {
      p[i] = PyLong_AsVoidPtr(args[i]);
      if (!p[i]) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null function");
        throw Refused{};
      }
    }
    g_matmul = reinterpret_cast<decltype(g_matmul)>(p[0]);
    g_linear = reinterpret_cast<decltype(g_linear)>(p[1]);
    g_qk = reinterpret_cast<decltype(g_qk)>(p[2]);
    Py_RETURN_NONE;
  });
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}

PyMethodDef g_methods[] = {method<matmul_i8>("matmul_i8"), method<linear_i8>("linear_i8"),
                           method<qk_norm_rope>("qk_norm_rope"), method<bind>("bind"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "arctic_tensors", nullptr, -1, g_methods, nullptr, nullptr, nullptr,
                        nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_arctic_tensors() { return PyModule_Create(&g_module); }
