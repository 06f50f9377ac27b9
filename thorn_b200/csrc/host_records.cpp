// Host side of the functional multi-tensor calls: checks whole lists of tensors and writes
// their pointers, sizes and scalars into the C records that the library takes.  In Python the
// same work costs about 3 us per tensor, 200 us for the 65 norm weights of a decoder whose
// step is 10 us on the device.
//
// A CPython extension over libtorch.  Checks only report whether a list is as expected; the
// caller looks for the offender and raises.
#include <ATen/core/LegacyTypeDispatch.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstring>
#include <exception>
#include <utility>
#include <vector>

namespace {

constexpr int64_t kBlock = 128;

int64_t numel_of(const at::Tensor& t) { return t.numel(); }

// A record buffer: a writable contiguous object that holds n records of `stride` bytes.
struct Records {
  Py_buffer view{};
  bool ok = false;
  Records(PyObject* o) { ok = PyObject_GetBuffer(o, &view, PyBUF_WRITABLE) == 0; }
  ~Records() {
    if (ok) PyBuffer_Release(&view);
  }
  bool holds(Py_ssize_t n, Py_ssize_t offset, Py_ssize_t stride, Py_ssize_t width) const {
    return offset >= 0 && stride >= offset + width && n <= view.len / stride;
  }
  template <class T>
  void put(Py_ssize_t i, Py_ssize_t offset, Py_ssize_t stride, T v) {
    std::memcpy((char*)view.buf + i * stride + offset, &v, sizeof(T));
  }
};

PyObject* bad_records() {
  PyErr_SetString(PyExc_ValueError, "the record buffer is too short");
  return nullptr;
}

// The list's tensors; false (with an error set) when an element is none.
bool tensors_of(PyObject* list, std::vector<const at::Tensor*>& out) {
  if (!PyList_Check(list)) {
    PyErr_SetString(PyExc_TypeError, "expected a list of tensors");
    return false;
  }
  const Py_ssize_t n = PyList_GET_SIZE(list);
  out.reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PyList_GET_ITEM(list, i);
    if (!THPVariable_Check(o)) {
      PyErr_Format(PyExc_TypeError, "element %zd is not a tensor", i);
      return false;
    }
    out.push_back(&THPVariable_Unpack(o));
  }
  return true;
}

enum Like { kAny = 0, kSameShape = 1, kFlatBlocks = 2, kMatrixBlocks = 3 };

bool as_expected(const at::Tensor& t, const at::Tensor& like, int mode) {
  if (mode == kSameShape) return t.sizes() == like.sizes();
  if (mode == kFlatBlocks) return t.dim() == 1 && t.size(0) == (numel_of(like) + kBlock - 1) / kBlock;
  const int64_t d = like.dim();
  if (d < 2) return false;
  int64_t batch = 1;
  for (int64_t i = 0; i + 2 < d; ++i) batch *= like.size(i);
  return t.dim() == 2 && t.size(0) == batch && t.size(1) == (like.size(d - 2) * like.size(d - 1) + kBlock - 1) / kBlock;
}

// pointers(records, offset, stride, tensors, dtype, device index or -1, like or None, mode,
// distinct) -> bool: whether every tensor is a contiguous one of this dtype and device, of the
// shape that `mode` derives from its partner in `like`, and (distinct) no two share memory;
// their pointers are then in the records.
PyObject* pointers(PyObject*, PyObject* args) {
  PyObject *buf, *list, *dtype, *like;
  Py_ssize_t offset, stride;
  int device, mode, distinct;
  if (!PyArg_ParseTuple(args, "OnnOOiOip", &buf, &offset, &stride, &list, &dtype, &device, &like, &mode, &distinct))
    return nullptr;
  if (!THPDtype_Check(dtype)) {
    PyErr_SetString(PyExc_TypeError, "expected a dtype");
    return nullptr;
  }
  try {
    std::vector<const at::Tensor*> ts, ls;
    if (!tensors_of(list, ts)) return nullptr;
    if (mode != kAny && (!tensors_of(like, ls) || ls.size() != ts.size())) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "lists of different lengths");
      return nullptr;
    }
    Records rec(buf);
    if (!rec.ok) return nullptr;
    if (!rec.holds((Py_ssize_t)ts.size(), offset, stride, 8)) return bad_records();
    const at::ScalarType want = reinterpret_cast<THPDtype*>(dtype)->scalar_type;
    std::vector<std::pair<uint64_t, uint64_t>> seen;  // first byte, the one behind the last
    if (distinct) seen.reserve(ts.size());
    bool ascending = true;
    for (size_t i = 0; i < ts.size(); ++i) {
      const at::Tensor& t = *ts[i];
      if (t.scalar_type() != want || t.layout() != at::kStrided || !t.is_contiguous()) Py_RETURN_FALSE;
      if (device < 0 ? !t.is_cpu() : !(t.is_cuda() && t.get_device() == device)) Py_RETURN_FALSE;
      if (mode != kAny && !as_expected(t, *ls[i], mode)) Py_RETURN_FALSE;
      const uint64_t p = (uint64_t)(uintptr_t)t.data_ptr();
      rec.put(i, offset, stride, p);
      if (distinct && numel_of(t) > 0) {  // empty tensors may share an address
        ascending = ascending && (seen.empty() || seen.back().second <= p);
        seen.emplace_back(p, p + (uint64_t)numel_of(t) * t.element_size());
      }
    }
    if (!ascending) {
      std::sort(seen.begin(), seen.end());
      for (size_t i = 1; i < seen.size(); ++i)
        if (seen[i].first < seen[i - 1].second) Py_RETURN_FALSE;
    }
  } catch (const std::exception& ex) {
    PyErr_SetString(PyExc_RuntimeError, ex.what());
    return nullptr;
  }
  Py_RETURN_TRUE;
}

// numels(records, offset, stride, tensors): the element counts as int64
PyObject* numels(PyObject*, PyObject* args) {
  PyObject *buf, *list;
  Py_ssize_t offset, stride;
  if (!PyArg_ParseTuple(args, "OnnO", &buf, &offset, &stride, &list)) return nullptr;
  try {
    std::vector<const at::Tensor*> ts;
    if (!tensors_of(list, ts)) return nullptr;
    Records rec(buf);
    if (!rec.ok) return nullptr;
    if (!rec.holds((Py_ssize_t)ts.size(), offset, stride, 8)) return bad_records();
    for (size_t i = 0; i < ts.size(); ++i) rec.put(i, offset, stride, numel_of(*ts[i]));
  } catch (const std::exception& ex) {
    PyErr_SetString(PyExc_RuntimeError, ex.what());
    return nullptr;
  }
  Py_RETURN_NONE;
}

// values(records, offset, stride, n, kind, x): n scalars, x one number or a list of n; kind
// 'f' float, 'i' int32, 'Q' 64 bits of an int (taken modulo 2^64)
PyObject* values(PyObject*, PyObject* args) {
  PyObject *buf, *x;
  Py_ssize_t offset, stride, n;
  int kind;
  if (!PyArg_ParseTuple(args, "OnnnCO", &buf, &offset, &stride, &n, &kind, &x)) return nullptr;
  Records rec(buf);
  if (!rec.ok) return nullptr;
  if (!rec.holds(n, offset, stride, kind == 'Q' ? 8 : 4)) return bad_records();
  const bool many = PyList_Check(x);
  if (many && PyList_GET_SIZE(x) != n) {
    PyErr_SetString(PyExc_ValueError, "as many values as records are needed");
    return nullptr;
  }
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = many ? PyList_GET_ITEM(x, i) : x;
    if (kind == 'f') rec.put(i, offset, stride, (float)PyFloat_AsDouble(o));
    else if (kind == 'i') rec.put(i, offset, stride, (int32_t)PyLong_AsLong(o));
    else rec.put(i, offset, stride, (uint64_t)PyLong_AsUnsignedLongLongMask(o));
    if (PyErr_Occurred()) return nullptr;
  }
  Py_RETURN_NONE;
}

// matrices(records, offset, stride, tensors, scratch function) -> (elements, bytes): writes
// int64 batch, rows, cols and leading dimension (= cols); returns the elements of the outputs,
// each padded to 8, and the bytes of all tensors' scratch.  The function is the library's
// int64 (batch, rows, cols) -> bytes, as an address.
using ScratchBytes = int64_t (*)(int64_t, int64_t, int64_t);
PyObject* matrices(PyObject*, PyObject* args) {
  PyObject *buf, *list;
  Py_ssize_t offset, stride;
  unsigned long long fn;
  if (!PyArg_ParseTuple(args, "OnnOK", &buf, &offset, &stride, &list, &fn)) return nullptr;
  long long elems = 0, bytes = 0;
  try {
    std::vector<const at::Tensor*> ts;
    if (!tensors_of(list, ts)) return nullptr;
    Records rec(buf);
    if (!rec.ok) return nullptr;
    if (!rec.holds((Py_ssize_t)ts.size(), offset, stride, 32)) return bad_records();
    for (size_t i = 0; i < ts.size(); ++i) {
      const at::Tensor& t = *ts[i];
      const int64_t d = t.dim();
      if (d < 2) {
        PyErr_SetString(PyExc_ValueError, "grads must be matrices or stacks of matrices");
        return nullptr;
      }
      int64_t v[4] = {1, t.size(d - 2), t.size(d - 1), t.size(d - 1)};
      for (int64_t k = 0; k + 2 < d; ++k) v[0] *= t.size(k);
      for (int k = 0; k < 4; ++k) rec.put(i, offset + 8 * k, stride, v[k]);
      elems += (t.numel() + 7) / 8 * 8;
      bytes += ((ScratchBytes)fn)(v[0], v[1], v[2]);
    }
  } catch (const std::exception& ex) {
    PyErr_SetString(PyExc_RuntimeError, ex.what());
    return nullptr;
  }
  return Py_BuildValue("(LL)", elems, bytes);
}

// scratch(records, offset, at, stride, n, scratch function, base): writes each record's part of
// the scratch at `base` at `at`, from the batch, rows and cols at `offset`
PyObject* scratch(PyObject*, PyObject* args) {
  PyObject* buf;
  Py_ssize_t offset, at, stride, n;
  unsigned long long fn, base;
  if (!PyArg_ParseTuple(args, "OnnnnKK", &buf, &offset, &at, &stride, &n, &fn, &base)) return nullptr;
  Records rec(buf);
  if (!rec.ok) return nullptr;
  if (!rec.holds(n, offset, stride, 24) || !rec.holds(n, at, stride, 8)) return bad_records();
  for (Py_ssize_t i = 0; i < n; ++i) {
    int64_t v[3];
    std::memcpy(v, (const char*)rec.view.buf + i * stride + offset, sizeof(v));
    rec.put(i, at, stride, (uint64_t)base);
    base += (uint64_t)((ScratchBytes)fn)(v[0], v[1], v[2]);
  }
  Py_RETURN_NONE;
}

// views(flat, like, records, offset, stride) -> list of tensors of the shapes of `like` that
// lie one after another in `flat`, each starting at a multiple of 8 elements (the caller has
// allocated enough); their pointers are written into the records
PyObject* views(PyObject*, PyObject* args) {
  PyObject *flat, *list, *buf;
  Py_ssize_t offset, stride;
  if (!PyArg_ParseTuple(args, "OOOnn", &flat, &list, &buf, &offset, &stride)) return nullptr;
  if (!THPVariable_Check(flat)) {
    PyErr_SetString(PyExc_TypeError, "expected a tensor");
    return nullptr;
  }
  PyObject* out = nullptr;
  try {
    std::vector<const at::Tensor*> ts;
    if (!tensors_of(list, ts)) return nullptr;
    Records rec(buf);
    if (!rec.ok) return nullptr;
    if (!rec.holds((Py_ssize_t)ts.size(), offset, stride, 8)) return bad_records();
    const at::Tensor& f = THPVariable_Unpack(flat);
    int64_t total = 0;
    for (const at::Tensor* t : ts) total += (t->numel() + 7) / 8 * 8;
    if (f.numel() < total || !f.is_contiguous()) {
      PyErr_SetString(PyExc_ValueError, "the buffer is too short");
      return nullptr;
    }
    at::AutoDispatchBelowAutograd no_autograd;  // plain buffers: no view tracking
    const uint64_t base = (uint64_t)(uintptr_t)f.data_ptr();
    const int64_t width = f.element_size();
    out = PyList_New((Py_ssize_t)ts.size());
    int64_t at = 0;
    std::vector<int64_t> strides;
    for (size_t i = 0; out && i < ts.size(); ++i) {
      const int64_t n = ts[i]->numel();
      strides.assign(ts[i]->dim(), 1);
      for (int64_t k = ts[i]->dim() - 1; k > 0; --k) strides[k - 1] = strides[k] * std::max<int64_t>(1, ts[i]->size(k));
      PyObject* o = THPVariable_Wrap(f.as_strided(ts[i]->sizes(), strides, f.storage_offset() + at));
      if (!o) {
        Py_CLEAR(out);
        break;
      }
      PyList_SET_ITEM(out, (Py_ssize_t)i, o);
      rec.put(i, offset, stride, base + (uint64_t)(at * width));
      at += (n + 7) / 8 * 8;
    }
  } catch (const std::exception& ex) {
    Py_XDECREF(out);
    PyErr_SetString(PyExc_RuntimeError, ex.what());
    return nullptr;
  }
  return out;
}

// written(list or None, ...): counts every tensor of the lists as modified in place, which a graph
// that saved it looks at.  Inference tensors have no count.
PyObject* written(PyObject*, PyObject* args) {
  try {
    for (Py_ssize_t k = 0; k < PyTuple_GET_SIZE(args); ++k) {
      PyObject* list = PyTuple_GET_ITEM(args, k);
      if (list == Py_None) continue;
      std::vector<const at::Tensor*> ts;
      if (!tensors_of(list, ts)) return nullptr;
      for (const at::Tensor* t : ts)
        if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    }
  } catch (const std::exception& ex) {
    PyErr_SetString(PyExc_RuntimeError, ex.what());
    return nullptr;
  }
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"pointers", pointers, METH_VARARGS, "check a list of tensors and write their pointers"},
    {"numels", numels, METH_VARARGS, "write element counts"},
    {"values", values, METH_VARARGS, "write scalars"},
    {"matrices", matrices, METH_VARARGS, "write batch, rows and columns"},
    {"scratch", scratch, METH_VARARGS, "write scratch pointers"},
    {"views", views, METH_VARARGS, "views of one buffer"},
    {"written", written, METH_VARARGS, "count tensors as modified in place"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "thorn_b200_host", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_thorn_b200_host(void) { return PyModule_Create(&kModule); }
