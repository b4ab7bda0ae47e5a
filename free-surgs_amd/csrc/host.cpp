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
#include <ATen/hip/EmptyTensor.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>
#include <exception>
#include <vector>

#include "../../include/fsgs.h"

namespace {

PyObject *k_step, *k_m, *k_v, *k_mq, *k_vq, *k_scales, *k_master;
PyObject *k_params, *k_lr, *k_betas, *k_eps, *k_decay, *k_bits, *k_masters, *k_maximize, *k_capturable;

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
  static PyObject *more(PyObject *p) { Py_XINCREF(p); return p; }
  ~Ref() { Py_XDECREF(o); }
  PyObject *release() { PyObject *p = o; o = nullptr; return p; }
  Ref(const Ref &) = delete;
  Ref &operator=(const Ref &) = delete;
};

// torch's own function behind torch.empty, without the dispatch of an operator
PyObject *fresh(at::IntArrayRef sizes, at::ScalarType type, int device) {
  return THPVariable_Wrap(at::Tensor(
      at::detail::empty_cuda(sizes, type, c10::Device(c10::kCUDA, (c10::DeviceIndex)device), std::nullopt)));
}

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

struct Bucket {  // tensors of one launch sequence
  int dtype, bits, device;
  bool masters, maximize;
  std::vector<int64_t> rows;
  std::vector<FsgsAdamWHyper> hypers;
  PyObject *params, *states;
};
struct Buckets : std::vector<Bucket> {
  ~Buckets() {
    for (Bucket &b : *this) {
      Py_XDECREF(b.params);
      Py_XDECREF(b.states);
    }
  }
};

bool number(PyObject *o, double *x) {  // a float or an int, and nothing that may have a reading of its own
  if (!o || (!PyFloat_CheckExact(o) && !PyLong_CheckExact(o))) return false;
  *x = PyFloat_CheckExact(o) ? PyFloat_AS_DOUBLE(o) : PyLong_AsDouble(o);
  return true;
}
bool truth(PyObject *o, bool *x) {
  if (o != Py_True && o != Py_False) return false;
  *x = o == Py_True;
  return true;
}

// step_rows(param_groups, state) -> [(device index, dtype, bits, maximize, rows, hypers, params, states)] or None
PyObject *step_rows(PyObject *, PyObject *args) {
  PyObject *groups, *state;
  if (!PyArg_ParseTuple(args, "O!O!", &PyList_Type, &groups, &PyDict_Type, &state)) return nullptr;
  return guarded([&]() -> PyObject * {
    Buckets buckets;
    for (Py_ssize_t k = 0; k < PyList_GET_SIZE(groups); k++) {
      PyObject *group = PyList_GET_ITEM(groups, k);
      if (!PyDict_Check(group)) return other_case();
      PyObject *betas = PyDict_GetItemWithError(group, k_betas), *list = PyDict_GetItemWithError(group, k_params);
      FsgsAdamWHyper h = {};
      double bits;
      bool masters, maximize, capturable;
      if (!betas || !PyTuple_CheckExact(betas) || PyTuple_GET_SIZE(betas) != 2 || !list || !PyList_Check(list) ||
          !number(PyDict_GetItemWithError(group, k_lr), &h.lr) || !number(PyTuple_GET_ITEM(betas, 0), &h.beta1) ||
          !number(PyTuple_GET_ITEM(betas, 1), &h.beta2) || !number(PyDict_GetItemWithError(group, k_eps), &h.eps) ||
          !number(PyDict_GetItemWithError(group, k_decay), &h.weight_decay) ||
          !number(PyDict_GetItemWithError(group, k_bits), &bits) || (bits != 8 && bits != 32) ||
          !truth(PyDict_GetItemWithError(group, k_masters), &masters) ||
          !truth(PyDict_GetItemWithError(group, k_maximize), &maximize) ||
          !truth(PyDict_GetItemWithError(group, k_capturable), &capturable) || capturable)
        return other_case();
      if (!(h.lr >= 0.0 && h.beta1 >= 0.0 && h.beta1 < 1.0 && h.beta2 >= 0.0 && h.beta2 < 1.0 && h.eps >= 0.0 && h.weight_decay >= 0.0))
        return other_case();
      PyObject *const km = bits == 8 ? k_mq : k_m, *const kv = bits == 8 ? k_vq : k_v;
      const at::ScalarType moment = bits == 8 ? at::kFloat8_e4m3fn : at::kFloat;
      // a parameter's hash is Python code, during which other threads may run: what is used after it is held
      const Ref hold_list(Ref::more(list));
      for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); i++) {
        PyObject *o = PyList_GET_ITEM(list, i);
        if (!plain(o)) return other_case();
        const Ref hold(Ref::more(o));
        const at::Tensor &p = THPVariable_Unpack(o);
        const at::Tensor g = p.grad();
        if (!g.defined()) continue;
        const at::ScalarType type = p.scalar_type();
        const c10::Device device = p.device();
        const int64_t n = p.numel();
        const int code = dtype_code(type);
        if (code < 0 || !packed(p) || !fits(g, type, device, n)) return other_case();
        PyObject *st = PyDict_GetItemWithError(state, o);
        if (!st || !PyDict_Check(st)) return other_case();
        PyObject *step = PyDict_GetItemWithError(st, k_step);
        if (!step || !PyLong_CheckExact(step)) return other_case();
        h.step = PyLong_AsLongLong(step) + 1;
        if (h.step < 1) return other_case();
        const at::Tensor *m = entry(st, km), *v = m ? entry(st, kv) : nullptr, *s = nullptr, *w = nullptr;
        if (!m || !v || !fits(*m, moment, device, n) || !fits(*v, moment, device, n)) return other_case();
        if (bits == 8) {
          s = entry(st, k_scales);
          if (!s || !fits(*s, at::kByte, device, 2 * ((n + FSGS_ADAMW_BLOCK - 1) / FSGS_ADAMW_BLOCK))) return other_case();
        }
        if (masters && type != at::kFloat) {
          w = entry(st, k_master);
          if (!w || !fits(*w, at::kFloat, device, n)) return other_case();
        } else if (PyDict_GetItemWithError(st, k_master)) {
          return other_case();  // master weights that the step would leave behind
        }
        Bucket *b = nullptr;
        for (Bucket &x : buckets)
          if (x.dtype == code && x.bits == (int)bits && x.device == device.index() && x.masters == (w != nullptr) && x.maximize == maximize)
            b = &x;
        if (!b) {
          buckets.push_back({code, (int)bits, device.index(), w != nullptr, maximize, {}, {}, PyList_New(0), PyList_New(0)});
          b = &buckets.back();
          if (!b->params || !b->states) return nullptr;
        }
        // most tensors share the scalars of the one in front of them; other repetitions cost a place in the list
        if (b->hypers.empty() || std::memcmp(&b->hypers.back(), &h, sizeof(h))) b->hypers.push_back(h);
        if (PyList_Append(b->params, o) || PyList_Append(b->states, st)) return nullptr;
        const int64_t row[] = {address(p), address(g), address(*m), address(*v), s ? address(*s) : 0, w ? address(*w) : 0, n,
                               (int64_t)b->hypers.size() - 1};
        static_assert(sizeof(row) == sizeof(FsgsAdamWTensor), "a row");
        b->rows.insert(b->rows.end(), row, row + 8);
      }
    }
    Ref out(PyList_New(0));
    if (!out.o) return nullptr;
    for (const Bucket &b : buckets) {
      Ref rows(rows_of(b.rows));
      Ref hypers(PyBytes_FromStringAndSize((const char *)b.hypers.data(), (Py_ssize_t)(b.hypers.size() * sizeof(FsgsAdamWHyper))));
      if (!rows.o || !hypers.o) return nullptr;
      Ref item(Py_BuildValue("(iiiOOOOO)", b.device, b.dtype, b.bits, b.maximize ? Py_True : Py_False, rows.o, hypers.o, b.params,
                             b.states));
      if (!item.o || PyList_Append(out.o, item.o)) return nullptr;
    }
    return out.release();
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

// grad_rows(params, nbytes) -> (rows, device index, norm, scratch) of the gradients that there are, or None; all on one device.
// norm, scratch: a new 0-d float32 tensor and one of nbytes bytes there, None without gradients.
PyObject *grad_rows(PyObject *, PyObject *args) {
  PyObject *params;
  long long nbytes;
  if (!PyArg_ParseTuple(args, "OL", &params, &nbytes)) return nullptr;
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
    if (device < 0) return Py_BuildValue("(OiOO)", bytes.o, device, Py_None, Py_None);
    Ref norm(fresh({}, at::kFloat, device)), scratch(fresh({(int64_t)nbytes}, at::kByte, device));
    if (!norm.o || !scratch.o) return nullptr;
    return Py_BuildValue("(OiOO)", bytes.o, device, norm.o, scratch.o);
  });
}

// norm_buffers(device index, nbytes) -> (norm, scratch): a new 0-d float32 tensor and one of nbytes bytes
PyObject *norm_buffers(PyObject *, PyObject *args) {
  int device;
  long long nbytes;
  if (!PyArg_ParseTuple(args, "iL", &device, &nbytes)) return nullptr;
  return guarded([&]() -> PyObject * {
    Ref norm(fresh({}, at::kFloat, device)), scratch(fresh({(int64_t)nbytes}, at::kByte, device));
    return norm.o && scratch.o ? PyTuple_Pack(2, norm.o, scratch.o) : nullptr;
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

int64_t padded(int64_t n) { return (n + 255) / 256 * 256; }

// moment_rows(param_groups, state, dtype) -> ([(m, v)], rows, device index) of the parameters that have a state, in order, or None:
// tensors of `dtype` for the values of 8-bit moments, cut from one new buffer
PyObject *moment_rows(PyObject *, PyObject *args) {
  PyObject *groups, *state, *dtype;
  if (!PyArg_ParseTuple(args, "O!O!O", &PyList_Type, &groups, &PyDict_Type, &state, &dtype)) return nullptr;
  if (!THPDtype_Check(dtype)) { PyErr_SetString(PyExc_TypeError, "a dtype"); return nullptr; }
  return guarded([&]() -> PyObject * {
    const at::ScalarType type = ((THPDtype *)dtype)->scalar_type;
    struct Item { at::Tensor m, v, s; };  // held, as in step_rows
    std::vector<Item> items;
    c10::Device device(c10::kCPU);
    for (Py_ssize_t k = 0; k < PyList_GET_SIZE(groups); k++) {
      PyObject *group = PyList_GET_ITEM(groups, k), *list = PyDict_Check(group) ? PyDict_GetItemWithError(group, k_params) : nullptr;
      if (!list || !PyList_Check(list)) return other_case();
      const Ref hold_list(Ref::more(list));
      for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); i++) {
        PyObject *o = PyList_GET_ITEM(list, i);
        const Ref hold(Ref::more(o));
        PyObject *st = PyDict_GetItemWithError(state, o);
        if (PyErr_Occurred()) return nullptr;
        if (!st) continue;
        if (!plain(o) || !PyDict_Check(st)) return other_case();
        const int64_t n = THPVariable_Unpack(o).numel();
        const at::Tensor *mq = entry(st, k_mq), *vq = mq ? entry(st, k_vq) : nullptr, *s = vq ? entry(st, k_scales) : nullptr;
        if (!s) return other_case();
        if (items.empty()) device = mq->device();
        if (!fits(*mq, at::kFloat8_e4m3fn, device, n) || !fits(*vq, at::kFloat8_e4m3fn, device, n) ||
            mq->sizes() != THPVariable_Unpack(o).sizes() ||
            !fits(*s, at::kByte, device, 2 * ((n + FSGS_ADAMW_BLOCK - 1) / FSGS_ADAMW_BLOCK)))
          return other_case();
        items.push_back({*mq, *vq, *s});
      }
    }
    if (items.empty()) return other_case();
    Ref pairs(PyList_New((Py_ssize_t)items.size()));
    if (!pairs.o) return nullptr;
    std::vector<int64_t> rows;
    rows.reserve(6 * items.size());
    // all values in one allocation, cut on 512-byte boundaries: 0.3 us a tensor where one of its own takes 0.7
    int64_t total = 0;
    for (const Item &x : items) total += 2 * padded(x.m.numel());
    const at::Tensor all(at::detail::empty_cuda({total}, type, device, std::nullopt));
    int64_t used = 0;
    const auto cut = [&](at::IntArrayRef sizes, int64_t n) {
      at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
      t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
      t.unsafeGetTensorImpl()->set_storage_offset(used);
      used += padded(n);
      return THPVariable_Wrap(std::move(t));
    };
    for (size_t i = 0; i < items.size(); i++) {
      const Item &x = items[i];
      Ref a(cut(x.m.sizes(), x.m.numel())), b(cut(x.m.sizes(), x.m.numel()));
      if (!a.o || !b.o) return nullptr;
      const int64_t row[] = {address(x.m), address(x.v), address(x.s), address(THPVariable_Unpack(a.o)),
                             address(THPVariable_Unpack(b.o)), x.m.numel()};
      static_assert(sizeof(row) == sizeof(FsgsAdamWMoments), "a row");
      rows.insert(rows.end(), row, row + 6);
      PyObject *pair = PyTuple_Pack(2, a.o, b.o);
      if (!pair) return nullptr;
      PyList_SET_ITEM(pairs.o, (Py_ssize_t)i, pair);
    }
    Ref bytes(rows_of(rows));
    if (!bytes.o) return nullptr;
    return Py_BuildValue("(OOi)", pairs.o, bytes.o, (int)device.index());
  });
}

PyMethodDef methods[] = {
    {"step_rows", step_rows, METH_VARARGS, "the launch sequences of an ordinary step, or None"},
    {"stepped", stepped, METH_VARARGS, "count a step in every state and raise the parameters' versions"},
    {"grad_rows", grad_rows, METH_VARARGS, "(rows, device, norm, scratch) for the parameters' gradients, or None"},
    {"norm_buffers", norm_buffers, METH_VARARGS, "(norm, scratch) on a device"},
    {"grads_written", grads_written, METH_O, "raise the versions of the parameters' gradients"},
    {"moment_rows", moment_rows, METH_VARARGS, "(pairs, rows, device) of the 8-bit moments of all parameters, or None"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fsgs_host", "the optimiser's walk over its tensors", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fsgs_host(void) {
  struct { PyObject **key; const char *name; } keys[] = {
      {&k_step, "step"}, {&k_m, "exp_avg"}, {&k_v, "exp_avg_sq"}, {&k_mq, "exp_avg_q"},
      {&k_vq, "exp_avg_sq_q"}, {&k_scales, "scales"}, {&k_master, "master"}, {&k_params, "params"},
      {&k_lr, "lr"}, {&k_betas, "betas"}, {&k_eps, "eps"}, {&k_decay, "weight_decay"}, {&k_bits, "state_bits"},
      {&k_masters, "master_weights"}, {&k_maximize, "maximize"}, {&k_capturable, "capturable"}};
  for (auto &k : keys)
    if (!(*k.key = PyUnicode_InternFromString(k.name))) return nullptr;
  PyObject *m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", FSGS_TORCH_VERSION)) {  // _lib.host() compares it
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
