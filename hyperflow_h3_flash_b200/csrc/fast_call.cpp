// The common calls of the attention operators without the interpreter in between (module hyperflow_h3_flash_b200._fast).
//
// Each function looks at its arguments as attention.py does and, where nothing about them needs a second look (CUDA
// tensors on the current device, no gradient wanted, sizes that the library takes), takes the given outputs or allocates
// them, calls the C entry on torch's current stream and returns the result.  In every other case it returns None, and attention.py goes
// through its own checks and names what is wrong: nothing is decided here alone.  At a few tokens the checks and the
// foreign-function call take three times as long as the launch (17 us against 6 for the norm and rotation of 17 tokens).
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "../../include/convrot.h"

namespace {

decltype(&convrot_rotary_table) g_table;
decltype(&convrot_qk_norm_rope) g_rope;
decltype(&convrot_attention) g_attention;
decltype(&convrot_attention_workspace_size) g_workspace;

// The tensor behind an object, or null: a plain CUDA tensor on `device` that wants no gradient.
const at::Tensor* plain(PyObject* o, int device) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.get_device() != device || t.layout() != at::kStrided) return nullptr;
  if (t.requires_grad() && c10::GradMode::is_enabled()) return nullptr;
  if (t._fw_grad(/*level=*/0).defined()) return nullptr;  // a forward-mode tangent (there is one level)
  return &t;
}

int type_of(const at::Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? CONVROT_BF16 : t.scalar_type() == at::kHalf ? CONVROT_FP16 : -1;
}

// A [tokens, heads, head_dim] tensor with neighbouring channels, of the given type (-1: any of the two).
const at::Tensor* heads(PyObject* o, int device, int type) {
  const at::Tensor* t = plain(o, device);
  if (!t || t->dim() != 3 || t->stride(2) != 1 || t->size(1) > (1 << 16) || t->size(2) > 256) return nullptr;
  const int own = type_of(*t);
  return own < 0 || (type >= 0 && own != type) ? nullptr : t;
}

at::Tensor fresh(const at::Tensor& t) {
  return t.is_contiguous() ? at::empty_like(t) : at::empty(t.sizes(), t.options());
}

void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }

template <class F>
PyObject* guarded(F&& f) {
  try {
    PyObject* r = f();
    if (r || PyErr_Occurred()) return r;
  } catch (const std::exception&) {  // an allocation that failed: attention.py makes it again, and torch reports it
    PyErr_Clear();
  }
  Py_RETURN_NONE;
}

bool number(PyObject* o, double* v) {
  *v = PyFloat_AsDouble(o);
  if (*v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

bool truth(PyObject* o, int* v) {
  if (!PyBool_Check(o)) return false;
  *v = o == Py_True;
  return true;
}

// The tensor to write into: a given output (null if it needs a second look: an inference tensor has no version to count
// the write in), else a fresh one, which `made` then holds.
const at::Tensor* target(PyObject* given, const at::Tensor& like, int device, int type, at::Tensor* made) {
  if (given == Py_None) {
    *made = fresh(like);
    return made;
  }
  const at::Tensor* t = heads(given, device, type);
  return t && t->sizes() == like.sizes() && !t->is_inference() ? t : nullptr;
}

// An output as the call returns it; the write into a given one counts as torch's own in-place operations do.
PyObject* returned(PyObject* given, at::Tensor& made) {
  if (given == Py_None) return THPVariable_Wrap(std::move(made));
  THPVariable_Unpack(given).unsafeGetTensorImpl()->bump_version();
  Py_INCREF(given);
  return given;
}

// qk_norm_rope(q, k, q_weight, k_weight, eps, norm, table, interleaved[, q_out, k_out])
PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (!g_rope || (n != 8 && n != 10)) return nullptr;
    PyObject* const given[2] = {n == 10 ? a[8] : Py_None, n == 10 ? a[9] : Py_None};
    const int device = c10::cuda::current_device();
    const at::Tensor* q = heads(a[0], device, -1);
    if (!q) return nullptr;
    const int type = type_of(*q);
    const at::Tensor* k = nullptr;
    if (a[1] != Py_None) {
      k = heads(a[1], device, type);
      if (!k || k->size(0) != q->size(0) || k->size(2) != q->size(2) || k->size(1) < 1) return nullptr;
    }
    const int64_t T = q->size(0), D = q->size(2);
    double eps;
    int norm, interleaved, f32 = -1;
    if (!number(a[4], &eps) || !truth(a[5], &norm) || !truth(a[7], &interleaved)) return nullptr;
    if (!(eps >= 0.0) || !std::isfinite(eps) || q->size(1) < 1) return nullptr;
    const void* weight[2] = {nullptr, nullptr};
    for (int i = 0; i < 2; ++i) {
      if (a[2 + i] == Py_None) continue;
      const at::Tensor* w = plain(a[2 + i], device);
      if (!w || !norm || (i == 1 && !k) || w->dim() != 1 || w->size(0) != D || !w->is_contiguous()) return nullptr;
      const int is_f32 = w->scalar_type() == at::kFloat;
      if ((!is_f32 && type_of(*w) != type) || (f32 >= 0 && f32 != is_f32)) return nullptr;
      f32 = is_f32;
      weight[i] = w->data_ptr();
    }
    const at::Tensor* table = nullptr;
    if (a[6] != Py_None) {
      table = plain(a[6], device);
      if (!table || table->dim() != 3 || table->size(0) != T || table->size(2) != 2 ||
          table->scalar_type() != at::kFloat || !table->is_contiguous())
        return nullptr;
    }
    const int64_t pairs = table ? table->size(1) : 0;
    if (!k && given[1] != Py_None) return nullptr;
    at::Tensor made[2];
    const at::Tensor* qo = target(given[0], *q, device, type, &made[0]);
    const at::Tensor* ko = k ? target(given[1], *k, device, type, &made[1]) : nullptr;
    if (!qo || (k && !ko)) return nullptr;
    if (k && T > 0) {
      const void *x = qo->data_ptr(), *y = ko->data_ptr();
      if (x == k->data_ptr() || x == y || y == q->data_ptr()) return nullptr;
    }
    const int rc = g_rope(q->data_ptr(), q->stride(0), q->stride(1), qo->data_ptr(), qo->stride(0), qo->stride(1),
                          static_cast<int>(q->size(1)), k ? k->data_ptr() : nullptr, k ? k->stride(0) : 0,
                          k ? k->stride(1) : 0, k ? ko->data_ptr() : nullptr, k ? ko->stride(0) : 0,
                          k ? ko->stride(1) : 0, k ? static_cast<int>(k->size(1)) : 0, T, static_cast<int>(D), type,
                          norm, weight[0], weight[1], f32 == 1, static_cast<float>(eps),
                          table ? static_cast<const float*>(table->data_ptr()) : nullptr, pairs,
                          static_cast<int>(2 * pairs), interleaved, stream_of(device));
    if (rc) return nullptr;
    if (!k) return returned(given[0], made[0]);
    PyObject* x = returned(given[0], made[0]);
    PyObject* y = returned(given[1], made[1]);
    PyObject* r = x && y ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return r;
  });
}

// attention(q, k, v, cu_q, cu_k, causal, scale, return_lse[, out])
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (!g_attention || !g_workspace || (n != 8 && n != 9)) return nullptr;
    PyObject* const given = n == 9 ? a[8] : Py_None;
    const int device = c10::cuda::current_device();
    const at::Tensor* q = heads(a[0], device, -1);
    if (!q) return nullptr;
    const int type = type_of(*q);
    const at::Tensor *k = heads(a[1], device, type), *v = heads(a[2], device, type);
    if (!k || !v || k->sizes() != v->sizes() || k->size(2) != q->size(2)) return nullptr;
    const int64_t Tq = q->size(0), Tk = k->size(0), D = q->size(2);
    int64_t batch = 1;
    const int32_t* cu[2] = {nullptr, nullptr};
    if ((a[3] == Py_None) != (a[4] == Py_None)) return nullptr;
    if (a[3] != Py_None) {
      for (int i = 0; i < 2; ++i) {
        const at::Tensor* c = plain(a[3 + i], device);
        if (!c || c->dim() != 1 || c->size(0) < 1 || c->scalar_type() != at::kInt || !c->is_contiguous())
          return nullptr;
        if (i == 1 && c->size(0) != batch + 1) return nullptr;
        batch = c->size(0) - 1;
        cu[i] = static_cast<const int32_t*>(c->data_ptr());
      }
    }
    int causal, return_lse;
    double scale = 1.0 / std::sqrt(static_cast<double>(D > 0 ? D : 1));
    if (!truth(a[5], &causal) || !truth(a[7], &return_lse)) return nullptr;
    if (a[6] != Py_None && !number(a[6], &scale)) return nullptr;
    if (!(scale > 0.0) || !std::isfinite(scale)) return nullptr;
    const int hq = static_cast<int>(q->size(1)), hkv = static_cast<int>(k->size(1));
    const int64_t size = g_workspace(Tq, Tk, batch, hq, hkv, static_cast<int>(D));
    if (size < 0) return nullptr;
    at::Tensor made, lse, space;
    const at::Tensor* out = target(given, *q, device, type, &made);
    if (!out) return nullptr;
    if (Tq > 0) {
      const void* o = out->data_ptr();
      if (o == q->data_ptr() || o == k->data_ptr() || o == v->data_ptr()) return nullptr;
    }
    if (return_lse) lse = at::empty({Tq, hq}, q->options().dtype(at::kFloat));
    if (size) space = at::empty({size}, q->options().dtype(at::kByte));
    const int rc = g_attention(q->data_ptr(), q->stride(0), q->stride(1), k->data_ptr(), k->stride(0), k->stride(1),
                               v->data_ptr(), v->stride(0), v->stride(1), cu[0], cu[1], batch, Tq, Tk, hq, hkv,
                               static_cast<int>(D), type, static_cast<float>(scale), causal, out->data_ptr(),
                               out->stride(0), out->stride(1),
                               return_lse ? static_cast<float*>(lse.data_ptr()) : nullptr,
                               size ? space.data_ptr() : nullptr, static_cast<size_t>(size), stream_of(device));
    if (rc) return nullptr;
    if (!return_lse) return returned(given, made);
    PyObject* x = returned(given, made);
    PyObject* y = THPVariable_Wrap(std::move(lse));
    PyObject* r = x && y ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return r;
  });
}

// rotary_table(positions, axes, theta): theta a float for every axis
PyObject* rotary_table(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (!g_table || n != 3 || !PyTuple_CheckExact(a[1]) || !PyFloat_CheckExact(a[2])) return nullptr;
    const int device = c10::cuda::current_device();
    const at::Tensor* pos = plain(a[0], device);
    const Py_ssize_t axes = PyTuple_GET_SIZE(a[1]);
    if (!pos || axes < 1 || axes > 8 || pos->dim() != 2 || pos->size(1) != axes || !pos->is_contiguous()) return nullptr;
    int kind;
    switch (pos->scalar_type()) {
      case at::kInt: kind = CONVROT_POS_I32; break;
      case at::kLong: kind = CONVROT_POS_I64; break;
      case at::kFloat: kind = CONVROT_POS_F32; break;
      case at::kDouble: kind = CONVROT_POS_F64; break;
      default: return nullptr;
    }
    int dims[8];
    double theta[8];
    int64_t pairs = 0;
    for (Py_ssize_t i = 0; i < axes; ++i) {
      PyObject* d = PyTuple_GET_ITEM(a[1], i);
      if (!PyLong_CheckExact(d)) return nullptr;
      int overflow = 0;
      const long v = PyLong_AsLongAndOverflow(d, &overflow);
      if (overflow || v <= 0 || v > 256 || v % 2) return nullptr;
      dims[i] = static_cast<int>(v);
      theta[i] = PyFloat_AS_DOUBLE(a[2]);
      pairs += v / 2;
    }
    if (pairs > 128) return nullptr;
    at::Tensor out = at::empty({pos->size(0), pairs, 2}, pos->options().dtype(at::kFloat));
    if (g_table(pos->data_ptr(), kind, axes, pos->size(0), static_cast<int>(axes), dims, theta,
                static_cast<float*>(out.data_ptr()), stream_of(device)))
      return nullptr;
    return THPVariable_Wrap(std::move(out));
  });
}

// init(rotary_table, qk_norm_rope, attention, attention_workspace_size): addresses of the C entries
PyObject* init(PyObject*, PyObject* args) {
  unsigned long long t, r, x, w;
  if (!PyArg_ParseTuple(args, "KKKK", &t, &r, &x, &w)) return nullptr;
  g_table = reinterpret_cast<decltype(g_table)>(t);
  g_rope = reinterpret_cast<decltype(g_rope)>(r);
  g_attention = reinterpret_cast<decltype(g_attention)>(x);
  g_workspace = reinterpret_cast<decltype(g_workspace)>(w);
  Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"init", init, METH_VARARGS, nullptr},
    {"rotary_table", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rotary_table)), METH_FASTCALL, nullptr},
    {"qk_norm_rope", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(qk_norm_rope)), METH_FASTCALL, nullptr},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attention)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_fast", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fast() { return PyModule_Create(&g_module); }
