// host.cpp -- the optimiser's walk over its tensors, as a CPython extension (fsgs_amd/lib/_fsgs_host.so).
//
// A step over hundreds of small tensors is bound by the host: reading some twenty attributes of four tensors costs Python
// 5 us a parameter, more than the GPU needs for most of them; here it is 0.2 us, half of that the hash of the parameter.
// Every function checks all that the kernels take for granted and returns None, with nothing changed, when something
// is not the ordinary case (other types, devices or layouts, missing or replaced state): the caller then takes the
// general path in optim.py, which converts, makes or refuses.  Rows are those of include/fsgs.h, as bytes.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty_like.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <exception>
#include <vector>

#include "../../include/fsgs.h"

namespace {

PyObject *k_step, *k_m, *k_v, *k_mq, *k_vq, *k_scales, *k_master;

// a plain tensor on the GPU whose elements follow each other in memory
bool plain(PyObject *o) { return o && THPVariable_CheckExact(o); }
bool packed(const at::Tensor &t) {
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.is_contiguous() && !t.is_neg();
}
int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? FSGS_DTYPE_F32 : t == at::kBFloat16 ? FSGS_DTYPE_BF16 : t == at::kHalf ? FSGS_DTYPE_F16 : -1;
}
bool fits(const at::Tensor &t, at::ScalarType type, c10::Device device, int64_t numel) {
  return packed(t) && t.scalar_type() == type && t.device() == device && t.numel() == numel;
}
int64_t address(const at::Tensor &t) { return (int64_t)(uintptr_t)t.data_ptr(); }
const at::Tensor *entry(PyObject *state, PyObject *key) {  // state[key] as a plain tensor, or nullptr
  PyObject *o = PyDict_GetItemWithError(state, key);
  return plain(o) ? &THPVariable_Unpack(o) : nullptr;
}

struct Ref {  // an owned reference
  PyObject *o;
  explicit Ref(PyObject *p) : o(p) {}
  ~Ref() { Py_XDECREF(o); }
  PyObject *release() { PyObject *p = o; o = nullptr; return p; }
  Ref(const Ref &) = delete;
  Ref &operator=(const Ref &) = delete;
};

PyObject *rows_of(const std::vector<int64_t> &rows) {
  return PyBytes_FromStringAndSize((const char *)rows.data(), (Py_ssize_t)(rows.size() * sizeof(int64_t)));
}
PyObject *other_case() {
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

template <class F> PyObject *guarded(F body) {  // no C++ exception leaves an entry
  try {
    return body();
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// step_rows(groups, state, bits, masters, dtype) -> (rows, params, states, counts, dtype, others, device index) or None.
// groups: list of parameter lists, row i of group k has hyper k; counts[k]: steps that group k's tensors have done (-1: no
// gradient in it).  Of the tensors of `dtype` (-1: that of the first); others: bit c is set where one of type c was passed
// over.  All on one device.
PyObject *step_rows(PyObject *, PyObject *args) {
  PyObject *groups, *state;
  int bits, masters, want;
  if (!PyArg_ParseTuple(args, "O!O!iii", &PyList_Type, &groups, &PyDict_Type, &state, &bits, &masters, &want)) return nullptr;
  return guarded([&]() -> PyObject * {
    Ref params(PyList_New(0)), states(PyList_New(0)), counts(PyList_New(0));
    if (!params.o || !states.o || !counts.o) return nullptr;
    std::vector<int64_t> rows;
    PyObject *const km = bits == 8 ? k_mq : k_m, *const kv = bits == 8 ? k_vq : k_v;
    const at::ScalarType moment = bits == 8 ? at::kFloat8_e4m3fn : at::kFloat;
    c10::Device device(c10::kCPU);
    int others = 0;
    for (Py_ssize_t k = 0; k < PyList_GET_SIZE(groups); k++) {
      PyObject *group = PyList_GET_ITEM(groups, k);
      if (!PyList_Check(group)) return other_case();
      long long count = -1;
      for (Py_ssize_t i = 0; i < PyList_GET_SIZE(group); i++) {
        PyObject *o = PyList_GET_ITEM(group, i);
        if (!plain(o)) return other_case();
        const at::Tensor &p = THPVariable_Unpack(o);
        const at::Tensor &g = p.grad();
        if (!g.defined()) continue;
        const at::ScalarType type = p.scalar_type();
        const int code = dtype_code(type);
        if (code < 0) return other_case();
        if (want < 0) want = code;
        if (want != code) {
          others |= 1 << code;
          continue;
        }
        if (rows.empty()) device = p.device();
        const int64_t n = p.numel();
        if (!fits(p, type, device, n) || !fits(g, type, device, n)) return other_case();
        PyObject *st = PyDict_GetItemWithError(state, o);
        if (!st || !PyDict_Check(st)) return other_case();
        PyObject *step = PyDict_GetItemWithError(st, k_step);
        if (!step || !PyLong_CheckExact(step)) return other_case();
        const long long done = PyLong_AsLongLong(step);
        if (done < 0 || (count >= 0 && done != count)) return other_case();
        count = done;
        const at::Tensor *m = entry(st, km), *v = m ? entry(st, kv) : nullptr, *s = nullptr, *w = nullptr;
        if (!m || !v || !fits(*m, moment, device, n) || !fits(*v, moment, device, n)) return other_case();
        if (bits == 8) {
          s = entry(st, k_scales);
          if (!s || !fits(*s, at::kByte, device, 2 * ((n + FSGS_ADAMW_BLOCK - 1) / FSGS_ADAMW_BLOCK))) return other_case();
        }
        if (masters && type != at::kFloat) {
          w = entry(st, k_master);
          if (!w || !fits(*w, at::kFloat, device, n)) return other_case();
        }
        if (PyList_Append(params.o, o) || PyList_Append(states.o, st)) return nullptr;
        const int64_t row[] = {address(p), address(g), address(*m), address(*v), s ? address(*s) : 0, w ? address(*w) : 0, n, k};
        static_assert(sizeof(row) == sizeof(FsgsAdamWTensor), "a row");
        rows.insert(rows.end(), row, row + 8);
      }
      Ref c(PyLong_FromLongLong(count));
      if (!c.o || PyList_Append(counts.o, c.o)) return nullptr;
    }
    Ref bytes(rows_of(rows));
    if (!bytes.o) return nullptr;
    return Py_BuildValue("(OOOOiii)", bytes.o, params.o, states.o, counts.o, want, others,
                         rows.empty() ? -1 : (int)device.index());
  });
}

// stepped(params, states): one more step counted in every state that counts on the host, and the parameters' versions raised
PyObject *stepped(PyObject *, PyObject *args) {
  PyObject *params, *states;
  if (!PyArg_ParseTuple(args, "O!O!", &PyList_Type, &params, &PyList_Type, &states)) return nullptr;
  return guarded([&]() -> PyObject * {
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(states); i++) {
      PyObject *st = PyList_GET_ITEM(states, i), *step = PyDict_GetItemWithError(st, k_step);
      if (!step) return other_case();
      if (!PyLong_CheckExact(step)) continue;  // a count on the device
      Ref next(PyLong_FromLongLong(PyLong_AsLongLong(step) + 1));
      if (!next.o || PyDict_SetItem(st, k_step, next.o)) return nullptr;
    }
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(params); i++)
      if (THPVariable_Check(PyList_GET_ITEM(params, i)))
        THPVariable_Unpack(PyList_GET_ITEM(params, i)).unsafeGetTensorImpl()->bump_version();
    Py_RETURN_NONE;
  });
}

// grad_rows(params) -> (rows, device index) of the gradients that there are, or None; all on one device
PyObject *grad_rows(PyObject *, PyObject *params) {
  if (!PyList_Check(params)) Py_RETURN_NONE;
  return guarded([&]() -> PyObject * {
    std::vector<int64_t> rows;
    int device = -1;
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(params); i++) {
      PyObject *o = PyList_GET_ITEM(params, i);
      if (!plain(o)) return other_case();
      const at::Tensor &g = THPVariable_Unpack(o).grad();
      if (!g.defined()) continue;
      const int code = dtype_code(g.scalar_type());
      if (code < 0 || !packed(g) || (device >= 0 && g.device().index() != device)) return other_case();
      device = g.device().index();
      const int64_t row[] = {address(g), g.numel(), code};
      static_assert(sizeof(row) == sizeof(FsgsGradTensor), "a row");
      rows.insert(rows.end(), row, row + 3);
    }
    Ref bytes(rows_of(rows));
    if (!bytes.o) return nullptr;
    return Py_BuildValue("(Oi)", bytes.o, device);
  });
}

// grads_written(params): the versions of their gradients raised
PyObject *grads_written(PyObject *, PyObject *params) {
  if (!PyList_Check(params)) { PyErr_SetString(PyExc_TypeError, "a list"); return nullptr; }
  return guarded([&]() -> PyObject * {
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(params); i++) {
      PyObject *o = PyList_GET_ITEM(params, i);
      if (!plain(o)) return other_case();
      const at::Tensor &g = THPVariable_Unpack(o).grad();
      if (g.defined()) g.unsafeGetTensorImpl()->bump_version();
    }
    Py_RETURN_NONE;
  });
}

// moment_rows(states, dtype) -> ([(m, v)], rows, device index) for states whose moments are in 8 bits, or None: new tensors
// of `dtype` for the values
PyObject *moment_rows(PyObject *, PyObject *args) {
  PyObject *states, *dtype;
  if (!PyArg_ParseTuple(args, "O!O", &PyList_Type, &states, &dtype)) return nullptr;
  if (!THPDtype_Check(dtype)) { PyErr_SetString(PyExc_TypeError, "a dtype"); return nullptr; }
  return guarded([&]() -> PyObject * {
    const at::ScalarType type = ((THPDtype *)dtype)->scalar_type;
    std::vector<int64_t> rows;
    Ref pairs(PyList_New(0));
    if (!pairs.o) return nullptr;
    c10::Device device(c10::kCPU);
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(states); i++) {
      PyObject *st = PyList_GET_ITEM(states, i);
      if (!PyDict_Check(st)) return other_case();
      const at::Tensor *mq = entry(st, k_mq), *vq = mq ? entry(st, k_vq) : nullptr, *s = vq ? entry(st, k_scales) : nullptr;
      if (!s) return other_case();
      const int64_t n = mq->numel();
      if (i == 0) device = mq->device();
      if (!fits(*mq, at::kFloat8_e4m3fn, device, n) || !fits(*vq, at::kFloat8_e4m3fn, device, n) ||
          !fits(*s, at::kByte, device, 2 * ((n + FSGS_ADAMW_BLOCK - 1) / FSGS_ADAMW_BLOCK)))
        return other_case();
      const at::Tensor m = at::empty_like(*mq, mq->options().dtype(type)), v = at::empty_like(*mq, mq->options().dtype(type));
      const int64_t row[] = {address(*mq), address(*vq), address(*s), address(m), address(v), n};
      static_assert(sizeof(row) == sizeof(FsgsAdamWMoments), "a row");
      rows.insert(rows.end(), row, row + 6);
      Ref a(THPVariable_Wrap(m)), b(THPVariable_Wrap(v));
      if (!a.o || !b.o) return nullptr;
      Ref pair(PyTuple_Pack(2, a.o, b.o));
      if (!pair.o || PyList_Append(pairs.o, pair.o)) return nullptr;
    }
    Ref bytes(rows_of(rows));
    if (!bytes.o) return nullptr;
    return Py_BuildValue("(OOi)", pairs.o, bytes.o, (int)device.index());
  });
}

PyMethodDef methods[] = {
    {"step_rows", step_rows, METH_VARARGS, "(rows, params, states, counts, dtype, others, device) of an ordinary step, or None"},
    {"stepped", stepped, METH_VARARGS, "count a step in every state and raise the parameters' versions"},
    {"grad_rows", grad_rows, METH_O, "(rows, device) of the parameters' gradients, or None"},
    {"grads_written", grads_written, METH_O, "raise the versions of the parameters' gradients"},
    {"moment_rows", moment_rows, METH_VARARGS, "(pairs, rows, device) of 8-bit moments, or None"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fsgs_host", "the optimiser's walk over its tensors", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fsgs_host(void) {
  struct { PyObject **key; const char *name; } keys[] = {
      {&k_step, "step"}, {&k_m, "exp_avg"}, {&k_v, "exp_avg_sq"}, {&k_mq, "exp_avg_q"},
      {&k_vq, "exp_avg_sq_q"}, {&k_scales, "scales"}, {&k_master, "master"}};
  for (auto &k : keys)
    if (!(*k.key = PyUnicode_InternFromString(k.name))) return nullptr;
  return PyModule_Create(&module);
}
