// The calls on a paged cache from tensors to launch: a CPython module around pbs_paged_append, pbs_paged_attn_fwd and pbs_paged_read.
//
// A decoding step's calls take the GPU 3 to 12 us, and reading eight to twelve tensors in Python takes longer: the next token of a chat into
// the cache 17.1 us a call in Python, 6.5 here.  Tensors are read through torch's C++ interface here (an attribute read through Python takes 0.1 us, and a
// call reads fifty), so the module is built for one interpreter and one torch, and says which: with another one, or without the module, the calls go
// through Python.
//
// Whatever is not the plain case returns None with nothing done, and the general path in Python takes the call, or refuses it with its message.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/pbs_hip.h"

namespace {

constexpr int HEAD_DIM = 128;

decltype(&pbs_paged_append) append_fn;
decltype(&pbs_paged_attn_workspace_bytes) attn_bytes_fn;
decltype(&pbs_paged_attn_fwd) attn_fn;
decltype(&pbs_paged_read) read_fn;
PyObject *pages_type, *current_device, *current_stream, *check;
PyObject *s_k, *s_v, *s_k_scale, *s_v_scale;

// a tensor of that type on the GPU, itself and no subclass
const at::Tensor* tensor(PyObject* x, at::ScalarType type, int64_t dims) {
  if (!THPVariable_CheckExact(x)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(x);
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.scalar_type() == type && t.dim() == dims && !t.is_neg() && !t.is_conj() ? &t : nullptr;
}
bool is_shape(const at::Tensor& t, std::initializer_list<int64_t> shape) { return t.sizes() == at::IntArrayRef(shape); }
bool aligned(const void* p) { return (uintptr_t)p % 16 == 0; }
// rows of 128 that the kernels read where they are
bool rows(const at::Tensor& t) {
  const int64_t last = t.dim() - 1;
  if (t.size(last) != HEAD_DIM || t.stride(last) != 1 || !aligned(t.const_data_ptr())) return false;
  for (int64_t i = 0; i < last; ++i)
    if (t.stride(i) % 8) return false;
  return true;
}

struct Pages {
  at::Tensor k, v, k_scale, v_scale;   // held: another thread may change the pages object while the GIL is released
  int64_t n, heads, size;
  bool read(PyObject* pk, PyObject* pv, PyObject* pks, PyObject* pvs) {
    const bool bf16 = pks == Py_None && pvs == Py_None;
    const at::ScalarType type = bf16 ? at::kBFloat16 : at::kByte;
    const at::Tensor *tk = tensor(pk, type, 4), *tv = tensor(pv, type, bf16 ? 5 : 6);
    if (!tk || !tv) return false;
    k = *tk, v = *tv;
    if (!bf16) {
      const at::Tensor *tks = tensor(pks, type, 5), *tvs = tensor(pvs, type, 5);
      if (!tks || !tvs) return false;
      k_scale = *tks, v_scale = *tvs;
    }
    n = k.size(0), heads = k.size(1), size = k.size(2);
    if (n <= 0 || heads <= 0 || (size != 32 && size != 64 && size != 128 && size != 256)) return false;
    if (bf16 ? !is_shape(k, {n, heads, size, HEAD_DIM}) || !is_shape(v, {n, heads, size / 8, HEAD_DIM, 8})
             : !is_shape(k, {n, heads, size, HEAD_DIM / 2}) || !is_shape(v, {n, heads, size / 4, 16, 4, 4}) ||
                   !is_shape(k_scale, {n, heads, size / 32, 4, 32}) || !is_shape(v_scale, {n, heads, size / 32, 4, 32}))
      return false;
    for (const at::Tensor* t : {&k, &v, &k_scale, &v_scale})
      if (t->defined() && (!t->is_contiguous() || !aligned(t->const_data_ptr()) || t->device() != k.device())) return false;
    return true;
  }
  bool read(PyObject* pages) {
    if ((PyObject*)Py_TYPE(pages) != pages_type) return false;
    PyObject* x[4] = {PyObject_GetAttr(pages, s_k), PyObject_GetAttr(pages, s_v), PyObject_GetAttr(pages, s_k_scale), PyObject_GetAttr(pages, s_v_scale)};
    const bool fine = x[0] && x[1] && x[2] && x[3] && read(x[0], x[1], x[2], x[3]);
    for (PyObject* o : x) Py_XDECREF(o);
    return fine;
  }
  const void* kp() const { return k.const_data_ptr(); }
  const void* vp() const { return v.const_data_ptr(); }
  const void* ksp() const { return k_scale.defined() ? k_scale.const_data_ptr() : nullptr; }
  const void* vsp() const { return v_scale.defined() ? v_scale.const_data_ptr() : nullptr; }
  int bits() const { return k_scale.defined() ? 4 : 16; }
};

const at::Tensor* table_of(PyObject* x, int64_t B) {
  const at::Tensor* t = tensor(x, at::kInt, 2);
  return t && t->size(0) == B && t->size(1) > 0 && t->stride(1) == 1 ? t : nullptr;
}
const at::Tensor* lengths(PyObject* x, int64_t B) {
  const at::Tensor* t = tensor(x, at::kInt, 1);
  return t && t->size(0) == B && t->is_contiguous() ? t : nullptr;
}
bool fits(int64_t x) { return x >= 0 && x <= INT32_MAX; }

// the current stream, where the current device is the tensors'
bool stream_of(const at::Tensor& t, void** stream) {
  PyObject* device = PyObject_CallNoArgs(current_device);
  if (!device) return false;
  const long index = PyLong_AsLong(device);
  PyObject* raw = index == t.device().index() ? PyObject_CallOneArg(current_stream, device) : nullptr;
  Py_DECREF(device);
  if (!raw) return false;
  *stream = (void*)(uintptr_t)PyLong_AsUnsignedLongLong(raw);
  Py_DECREF(raw);
  return !PyErr_Occurred();
}
bool modes_are_on() { return at::impl::torch_function_mode_enabled() || c10::impl::TorchDispatchModeTLS::any_modes_set(); }

PyObject* not_taken() {
  if (PyErr_Occurred() && !PyErr_ExceptionMatches(PyExc_Exception)) return nullptr;   // an interrupt, an exit
  PyErr_Clear();   // the general path meets the same error again
  Py_RETURN_NONE;
}
PyObject* failed(int rc, const char* what) { return PyObject_CallFunction(check, "is", rc, what); }   // raises
bool several(Py_ssize_t n, Py_ssize_t want, const char* what) {
  if (n != want) PyErr_Format(PyExc_TypeError, "%s takes %zd arguments", what, want);
  return n == want;
}

// pages_ok(k, v, k_scale, v_scale) -> bool
PyObject* pages_ok(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!several(n, 4, "pages_ok")) return nullptr;
  Pages p;
  return PyBool_FromLong(!modes_are_on() && p.read(args[0], args[1], args[2], args[3]));
  END_HANDLE_TH_ERRORS
}

// append(pages, page_table, past_lens, k, v, q, cos, sin, new_lens, want_k) -> (q, k), or None
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!several(n, 10, "append")) return nullptr;
  Pages pages;
  if (!pages_type || modes_are_on() || !pages.read(args[0]) || !PyBool_Check(args[9])) return not_taken();
  const at::Tensor *k = tensor(args[3], at::kBFloat16, 4), *v = tensor(args[4], at::kBFloat16, 4);
  if (!k || !v || k->sizes() != v->sizes() || k->size(1) != pages.heads || !rows(*k) || !rows(*v)) return not_taken();
  const int64_t B = k->size(0), Hkv = k->size(1), S = k->size(2);
  const at::Tensor *table = table_of(args[1], B), *past = lengths(args[2], B), *fresh = args[8] == Py_None ? nullptr : lengths(args[8], B);
  const at::Tensor *q = args[5] == Py_None ? nullptr : tensor(args[5], at::kBFloat16, 4), *cos = nullptr, *sin = nullptr;
  if (!table || !past || (!fresh && args[8] != Py_None) || (!q && args[5] != Py_None)) return not_taken();
  if (q && (q->size(0) != B || q->size(2) != S || !rows(*q))) return not_taken();
  if (args[6] != Py_None || args[7] != Py_None) {
    cos = tensor(args[6], at::kBFloat16, 3), sin = tensor(args[7], at::kBFloat16, 3);
    if (!cos || !sin || cos->sizes() != sin->sizes() || cos->strides() != sin->strides() || (cos->size(0) != 1 && cos->size(0) != B) ||
        cos->size(1) != S || !rows(*cos) || !rows(*sin))
      return not_taken();
  }
  const int64_t Hq = q ? q->size(1) : 0;
  for (const at::Tensor* t : {k, v, table, past, fresh, q, cos, sin})
    if (t && t->device() != pages.k.device()) return not_taken();
  if (!fits(B) || !fits(Hq) || !fits(Hkv) || !fits(S) || !fits(pages.n) || !fits(table->size(1))) return not_taken();
  void* stream;
  if (!stream_of(*k, &stream)) return not_taken();
  at::Tensor q_out, k_out;
  if (q) q_out = at::empty({B, Hq, S, HEAD_DIM}, q->options());
  if (args[9] == Py_True) k_out = at::empty({B, Hkv, S, HEAD_DIM}, k->options());
  const auto address = [](const at::Tensor* t) { return t ? t->const_data_ptr() : nullptr; };
  // (written: a lazy copy becomes a copy here)
  void *kp = pages.k.mutable_data_ptr(), *vp = pages.v.mutable_data_ptr();
  void *ksp = pages.k_scale.defined() ? pages.k_scale.mutable_data_ptr() : nullptr, *vsp = pages.v_scale.defined() ? pages.v_scale.mutable_data_ptr() : nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = append_fn(address(q), address(k), address(v), address(cos), address(sin), q ? q_out.mutable_data_ptr() : nullptr,
                 k_out.defined() ? k_out.mutable_data_ptr() : nullptr, kp, vp, ksp, vsp,
                 (const int32_t*)address(table), (const int32_t*)address(past), (const int32_t*)address(fresh), (int)B, (int)Hq, (int)Hkv, (int)S, HEAD_DIM,
                 (int)pages.n, (int)table->size(1), (int)pages.size, pages.bits(), q ? q->stride(0) : 0, q ? q->stride(1) : 0, q ? q->stride(2) : 0,
                 k->stride(0), k->stride(1), k->stride(2), v->stride(0), v->stride(1), v->stride(2), cos && cos->size(0) > 1 ? cos->stride(0) : 0,
                 cos ? cos->stride(1) : 0, table->stride(0), stream);
  Py_END_ALLOW_THREADS
  if (rc) return failed(rc, "pbs_paged_append");
  PyObject* a = q ? THPVariable_Wrap(std::move(q_out)) : (Py_INCREF(Py_None), Py_None);
  PyObject* b = k_out.defined() ? THPVariable_Wrap(std::move(k_out)) : (Py_INCREF(Py_None), Py_None);
  PyObject* both = a && b ? PyTuple_Pack(2, a, b) : nullptr;
  Py_XDECREF(a);
  Py_XDECREF(b);
  return both;
  END_HANDLE_TH_ERRORS
}

// attn(q, pages, page_table, past_lens, new_lens, softmax_scale, max_len) -> tensor, or None
PyObject* attn(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!several(n, 7, "attn")) return nullptr;
  Pages pages;
  if (!pages_type || modes_are_on() || !pages.read(args[1])) return not_taken();
  const at::Tensor* q = tensor(args[0], at::kBFloat16, 4);
  if (!q || !rows(*q)) return not_taken();
  const int64_t B = q->size(0), Hq = q->size(1), S = q->size(2);
  const at::Tensor *table = table_of(args[2], B), *past = lengths(args[3], B), *fresh = args[4] == Py_None ? nullptr : lengths(args[4], B);
  if (!table || !past || (!fresh && args[4] != Py_None) || Hq % pages.heads) return not_taken();
  for (const at::Tensor* t : {q, table, past, fresh})
    if (t && t->device() != pages.k.device()) return not_taken();
  if (!fits(B) || !fits(Hq) || !fits(S) || !fits(pages.heads) || !fits(pages.n) || !fits(table->size(1) * pages.size)) return not_taken();
  if ((args[5] != Py_None && !PyFloat_CheckExact(args[5])) || (args[6] != Py_None && !PyLong_CheckExact(args[6]))) return not_taken();
  const float scale = args[5] == Py_None ? 0.08838834764831845f : (float)PyFloat_AS_DOUBLE(args[5]);
  const int64_t room = table->size(1) * pages.size;
  long long max_len = args[6] == Py_None ? room : PyLong_AsLongLong(args[6]);
  if (max_len == -1 && PyErr_Occurred()) return not_taken();
  if (max_len > room) max_len = room;
  if (max_len <= 0) return not_taken();
  void* stream;
  if (!stream_of(*q, &stream)) return not_taken();
  const size_t bytes = attn_bytes_fn((int)B, (int)Hq, (int)pages.heads, (int)S, HEAD_DIM, pages.bits(), (int)max_len);
  at::Tensor out = at::empty({B, Hq, S, HEAD_DIM}, q->options()), ws;
  if (bytes) ws = at::empty({(int64_t)bytes}, q->options().dtype(at::kByte));
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = attn_fn(q->const_data_ptr(), pages.kp(), pages.vp(), pages.ksp(), pages.vsp(), (const int32_t*)table->const_data_ptr(),
               (const int32_t*)past->const_data_ptr(), fresh ? (const int32_t*)fresh->const_data_ptr() : nullptr, out.mutable_data_ptr(), (int)B, (int)Hq,
               (int)pages.heads, (int)S, HEAD_DIM, (int)pages.n, (int)table->size(1), (int)pages.size, pages.bits(), (int)max_len, q->stride(0),
               q->stride(1), q->stride(2), Hq * S * HEAD_DIM, S * HEAD_DIM, HEAD_DIM, table->stride(0), scale,
               bytes ? ws.mutable_data_ptr() : nullptr, bytes, stream);
  Py_END_ALLOW_THREADS
  return rc ? failed(rc, "pbs_paged_attn_fwd") : THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// read(pages, page_table, lens, max_len) -> (k, v), or None
PyObject* read(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!several(n, 4, "read")) return nullptr;
  Pages pages;
  if (!pages_type || modes_are_on() || !pages.read(args[0]) || !THPVariable_CheckExact(args[1]) || !PyLong_CheckExact(args[3])) return not_taken();
  const int64_t B = THPVariable_Unpack(args[1]).dim() ? THPVariable_Unpack(args[1]).size(0) : 0;
  const at::Tensor *table = table_of(args[1], B), *lens = lengths(args[2], B);
  if (!table || !lens || table->device() != pages.k.device() || lens->device() != pages.k.device()) return not_taken();
  const long long L = PyLong_AsLongLong(args[3]);
  if (L <= 0 || !fits(L) || !fits(B) || !fits(pages.heads) || !fits(pages.n) || !fits(table->size(1))) return not_taken();
  void* stream;
  if (!stream_of(*table, &stream)) return not_taken();
  const auto options = table->options().dtype(at::kBFloat16);
  at::Tensor k = at::empty({B, pages.heads, L, HEAD_DIM}, options), v = at::empty({B, pages.heads, L, HEAD_DIM}, options);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = read_fn(pages.kp(), pages.vp(), pages.ksp(), pages.vsp(), (const int32_t*)table->const_data_ptr(), (const int32_t*)lens->const_data_ptr(),
               k.mutable_data_ptr(), v.mutable_data_ptr(), (int)B, (int)pages.heads, (int)L, HEAD_DIM, (int)pages.n, (int)table->size(1), (int)pages.size,
               pages.bits(), table->stride(0), stream);
  Py_END_ALLOW_THREADS
  if (rc) return failed(rc, "pbs_paged_read");
  PyObject *a = THPVariable_Wrap(std::move(k)), *b = THPVariable_Wrap(std::move(v));
  PyObject* both = a && b ? PyTuple_Pack(2, a, b) : nullptr;
  Py_XDECREF(a);
  Py_XDECREF(b);
  return both;
  END_HANDLE_TH_ERRORS
}

// setup(KVPages, current device, its current raw stream, check, addresses of the library's four functions), once
PyObject* setup(PyObject*, PyObject* args) {
  PyObject *type, *dev, *st, *ck;
  unsigned long long f[4];
  if (!PyArg_ParseTuple(args, "OOOOKKKK", &type, &dev, &st, &ck, &f[0], &f[1], &f[2], &f[3])) return nullptr;
  for (PyObject* o : {type, dev, st, ck}) Py_INCREF(o);
  pages_type = type, current_device = dev, current_stream = st, check = ck;
  append_fn = (decltype(append_fn))(uintptr_t)f[0];
  attn_bytes_fn = (decltype(attn_bytes_fn))(uintptr_t)f[1];
  attn_fn = (decltype(attn_fn))(uintptr_t)f[2];
  read_fn = (decltype(read_fn))(uintptr_t)f[3];
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) { return {name, (PyCFunction)(void (*)(void))F, METH_FASTCALL, nullptr}; }
PyMethodDef methods[] = {method<pages_ok>("pages_ok"), method<append>("append"), method<attn>("attn"), method<read>("read"),
                         {"setup", setup, METH_VARARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_pbs_paged", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__pbs_paged() {
  s_k = PyUnicode_InternFromString("k");
  s_v = PyUnicode_InternFromString("v");
  s_k_scale = PyUnicode_InternFromString("k_scale");
  s_v_scale = PyUnicode_InternFromString("v_scale");
  PyObject* m = s_k && s_v && s_k_scale && s_v_scale ? PyModule_Create(&module) : nullptr;
  if (m && !PyModule_AddStringConstant(m, "torch_version", PBS_TORCH_VERSION) && !PyModule_AddIntConstant(m, "abi_version", PBS_ABI_VERSION)) return m;
  Py_XDECREF(m);
  return nullptr;
}
