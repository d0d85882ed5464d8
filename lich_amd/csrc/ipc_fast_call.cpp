// ipc_fast_call.cpp - calls of the microscaled entry points from Python (host code only).
//
// A small call of lich_amd.microscale lasts longer on the host than on the GPU.
// MI355X's host, us a call: quantisation 5.3 through ctypes, 2.85 here; a
// prediction of six tensors 6.5, 2.85; a packed matrix's two allocations 3.7, 2.0 (a
// launch alone 2.6, one torch.empty 1.75).
//
//   Call(entry address, shape of its arguments, ((sizes, dtype), ...) of its pointers,
//        constants, stream function)
//   Call(tensor or pair of tensors, ... [, workspace])  ->  0 done, < 0 the entry
//        point's error, 1 nothing was called: an argument is not what it has to be
//   Packed(sizes, dtype, sizes, dtype, pair type)(device or None)  ->  pair of new tensors
//
// What a 1 means is for the caller to find out and to raise: the checks with messages are
// written once, in Python.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <torch/csrc/Device.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <new>
#include <utility>
#include <tuple>

namespace {

constexpr int kPointers = 6, kInts = 6, kDims = 3;

struct Spec {
  int dims = 0;
  int64_t size[kDims] = {};
  at::ScalarType type{};
  bool is(const at::Tensor& t) const {
    if (!t.is_cuda() || t.scalar_type() != type || t.dim() != dims) return false;
    const auto s = t.sizes();
    for (int i = 0; i < dims; ++i)
      if (s[i] != size[i]) return false;
    return t.is_contiguous();
  }
};

bool read_sizes(PyObject* sizes, Spec& o) {
  if (!PyTuple_Check(sizes) || PyTuple_GET_SIZE(sizes) > kDims) return false;
  o.dims = (int)PyTuple_GET_SIZE(sizes);
  for (int i = 0; i < o.dims; ++i) o.size[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(sizes, i));
  return !PyErr_Occurred();
}

// An entry point's arguments: NP pointers, NA ints, a float (F), NB ints, a lent
// workspace and its bytes (W), the stream.
struct Arguments {
  void* entry;
  void* p[kPointers];
  int i[kInts];
  float f;
  void* workspace;
  long long bytes;
  void* stream;
};
template <size_t... P, size_t... A, size_t... B, typename... FW>
int call_with(const Arguments& a, std::index_sequence<P...>, std::index_sequence<A...>, std::index_sequence<B...>,
              std::tuple<FW...> f, std::true_type) {
  using Fn = int (*)(decltype((void)P, (void*)nullptr)..., decltype((void)A, 0)..., FW..., decltype((void)B, 0)..., void*,
                     long long, void*);
  return std::apply([&](auto... x) {
    return reinterpret_cast<Fn>(a.entry)(a.p[P]..., a.i[A]..., x..., a.i[sizeof...(A) + B]..., a.workspace, a.bytes, a.stream);
  }, f);
}
template <size_t... P, size_t... A, size_t... B, typename... FW>
int call_with(const Arguments& a, std::index_sequence<P...>, std::index_sequence<A...>, std::index_sequence<B...>,
              std::tuple<FW...> f, std::false_type) {
  using Fn = int (*)(decltype((void)P, (void*)nullptr)..., decltype((void)A, 0)..., FW..., decltype((void)B, 0)..., void*);
  return std::apply([&](auto... x) {
    return reinterpret_cast<Fn>(a.entry)(a.p[P]..., a.i[A]..., x..., a.i[sizeof...(A) + B]..., a.stream);
  }, f);
}
template <int NP, int NA, bool F, int NB, bool W>
int enter(const Arguments& a) {
  const auto ptr = std::make_index_sequence<NP>(), first = std::make_index_sequence<NA>(), rest = std::make_index_sequence<NB>();
  if constexpr (F) return call_with(a, ptr, first, rest, std::tuple<float>(a.f), std::bool_constant<W>());
  else return call_with(a, ptr, first, rest, std::tuple<>(), std::bool_constant<W>());
}

struct Kind {
  const char* name;
  int pointers, ints;
  bool number, workspace;
  int (*enter)(const Arguments&);
};
// pointers, ints before a float, float, ints after it, workspace, as in ipc_hip.h
#define KIND(NAME, NP, NA, F, NB, W) {NAME, NP, NA + NB, F, W, enter<NP, NA, F, NB, W>}
const Kind kKinds[] = {
    KIND("ipc_mx_quantize", 3, 6, false, 0, false),        KIND("ipc_mx_dequantize", 3, 4, false, 0, false),
    KIND("ipc_mx_pred_err", 6, 4, false, 0, false),        KIND("ipc_mx_forward", 5, 4, false, 0, false),
    KIND("ipc_mx_infer_update", 6, 3, true, 2, false),     KIND("ipc_mx_weight_update", 5, 3, true, 1, false),
    KIND("ipc_mx_predict", 4, 5, false, 0, true),          KIND("ipc_ckpt_weight_update", 4, 3, true, 3, true),
    KIND("ipc_ckpt_gradient", 5, 6, false, 0, true),
};

// ------------------------------------------------------------------ Call
struct Call {
  PyObject_HEAD
  vectorcallfunc vectorcall;
  const Kind* kind;
  Arguments args;  // entry and constants
  Spec spec[kPointers];
  PyObject* stream;  // f(device index) -> handle
};

PyObject* call_run(PyObject* self, PyObject* const* argv, size_t nargsf, PyObject* names) {
  const Call& c = *reinterpret_cast<Call*>(self);
  const Kind& k = *c.kind;
  const Py_ssize_t n = PyVectorcall_NARGS(nargsf);
  PyObject* refuse = PyLong_FromLong(1);
  if (names && PyTuple_GET_SIZE(names)) return refuse;
  Arguments a = c.args;
  int got = 0;
  c10::DeviceIndex device = -1;
  auto take = [&](PyObject* o) {
    if (got == k.pointers || !THPVariable_Check(o)) return false;
    try {
      const at::Tensor& t = THPVariable_Unpack(o);
      if (!c.spec[got].is(t)) return false;
      const c10::DeviceIndex d = t.get_device();
      if (device >= 0 && d != device) return false;
      device = d;
      a.p[got++] = t.data_ptr();
    } catch (const std::exception&) {  // (a tensor without strides or storage)
      return false;
    }
    return true;
  };
  Py_ssize_t at = 0;
  for (; at < n && got < k.pointers; ++at) {
    PyObject* o = argv[at];
    if (PyTuple_Check(o)) {
      if (PyTuple_GET_SIZE(o) != 2 || !take(PyTuple_GET_ITEM(o, 0)) || !take(PyTuple_GET_ITEM(o, 1))) return refuse;
    } else if (!take(o)) {
      return refuse;
    }
  }
  if (got != k.pointers) return refuse;
  a.workspace = nullptr;
  a.bytes = 0;
  if (k.workspace && at < n) {
    PyObject* o = argv[at++];
    if (o != Py_None) {
      if (!THPVariable_Check(o)) return refuse;
      try {
        const at::Tensor& t = THPVariable_Unpack(o);
        if (!t.is_cuda() || t.get_device() != device || !t.is_contiguous()) return refuse;
        a.workspace = t.data_ptr();
        a.bytes = (long long)t.nbytes();
      } catch (const std::exception&) {
        return refuse;
      }
    }
  }
  if (at != n) return refuse;
  PyObject* index = PyLong_FromLong(device);
  PyObject* handle = index ? PyObject_CallOneArg(c.stream, index) : nullptr;
  Py_XDECREF(index);
  if (!handle) {
    Py_DECREF(refuse);
    return nullptr;
  }
  a.stream = PyLong_AsVoidPtr(handle);
  Py_DECREF(handle);
  Py_DECREF(refuse);
  if (PyErr_Occurred()) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = k.enter(a);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

PyObject* call_new(PyTypeObject* type, PyObject* args, PyObject*) {
  const char* name;
  PyObject *address, *specs, *constants, *stream;
  if (!PyArg_ParseTuple(args, "sOO!O!O", &name, &address, &PyTuple_Type, &specs, &PyTuple_Type, &constants, &stream)) return nullptr;
  const Kind* kind = nullptr;
  for (const Kind& k : kKinds)
    if (!std::strcmp(k.name, name)) kind = &k;
  if (!kind || PyTuple_GET_SIZE(specs) != kind->pointers ||
      PyTuple_GET_SIZE(constants) != kind->ints + (kind->number ? 1 : 0)) {
    PyErr_Format(PyExc_ValueError, "no such call of %s", name);
    return nullptr;
  }
  Call* c = reinterpret_cast<Call*>(type->tp_alloc(type, 0));
  if (!c) return nullptr;
  c->vectorcall = call_run;
  c->kind = kind;
  c->args = Arguments{};
  c->args.entry = PyLong_AsVoidPtr(address);
  int ints = 0;
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(constants); ++i) {
    PyObject* v = PyTuple_GET_ITEM(constants, i);
    if (PyFloat_Check(v)) c->args.f = (float)PyFloat_AS_DOUBLE(v);
    else if (ints < kInts) c->args.i[ints++] = (int)PyLong_AsLong(v);
  }
  bool good = !PyErr_Occurred() && ints == kind->ints;
  for (int i = 0; good && i < kind->pointers; ++i) {
    PyObject* s = PyTuple_GET_ITEM(specs, i);
    new (&c->spec[i]) Spec();
    good = PyTuple_Check(s) && PyTuple_GET_SIZE(s) == 2 && read_sizes(PyTuple_GET_ITEM(s, 0), c->spec[i]) &&
           THPDtype_Check(PyTuple_GET_ITEM(s, 1));
    if (good) c->spec[i].type = reinterpret_cast<THPDtype*>(PyTuple_GET_ITEM(s, 1))->scalar_type;
  }
  if (!good) {
    Py_DECREF(c);
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "Call: constants or specs");
    return nullptr;
  }
  Py_INCREF(stream);
  c->stream = stream;
  return reinterpret_cast<PyObject*>(c);
}

void call_free(PyObject* self) {
  Py_XDECREF(reinterpret_cast<Call*>(self)->stream);
  Py_TYPE(self)->tp_free(self);
}

// ---------------------------------------------------------------- Packed
struct Packed {
  PyObject_HEAD
  vectorcallfunc vectorcall;
  Spec part[2];
  PyTypeObject* pair;
};

PyObject* packed_run(PyObject* self, PyObject* const* argv, size_t nargsf, PyObject*) {
  const Packed& p = *reinterpret_cast<Packed*>(self);
  at::Device device(at::kCUDA);
  if (PyVectorcall_NARGS(nargsf) > 0 && argv[0] != Py_None) {
    if (!THPDevice_Check(argv[0])) {
      PyErr_SetString(PyExc_TypeError, "device must be a torch.device or None");
      return nullptr;
    }
    device = reinterpret_cast<THPDevice*>(argv[0])->device;
  }
  HANDLE_TH_ERRORS  // (no memory, no such device)
  at::Tensor t[2];
  for (int i = 0; i < 2; ++i)
    t[i] = at::empty(at::IntArrayRef(p.part[i].size, p.part[i].dims),
                     at::TensorOptions().dtype(p.part[i].type).device(device));
  PyObject *codes = THPVariable_Wrap(std::move(t[0])), *scales = codes ? THPVariable_Wrap(std::move(t[1])) : nullptr;
  PyObject* both = scales ? PyTuple_Pack(2, codes, scales) : nullptr;
  PyObject* args = both ? PyTuple_Pack(1, both) : nullptr;
  PyObject* pair = args ? PyTuple_Type.tp_new(p.pair, args, nullptr) : nullptr;
  Py_XDECREF(args);
  Py_XDECREF(both);
  Py_XDECREF(scales);
  Py_XDECREF(codes);
  return pair;
  END_HANDLE_TH_ERRORS
}

PyObject* packed_new(PyTypeObject* type, PyObject* args, PyObject*) {
  PyObject *s0, *t0, *s1, *t1, *pair;
  if (!PyArg_ParseTuple(args, "OOOOO", &s0, &t0, &s1, &t1, &pair)) return nullptr;
  Spec part[2];
  if (!read_sizes(s0, part[0]) || !read_sizes(s1, part[1]) || !THPDtype_Check(t0) || !THPDtype_Check(t1) ||
      !PyType_Check(pair) || !PyType_IsSubtype(reinterpret_cast<PyTypeObject*>(pair), &PyTuple_Type)) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "Packed: sizes, types or pair");
    return nullptr;
  }
  part[0].type = reinterpret_cast<THPDtype*>(t0)->scalar_type;
  part[1].type = reinterpret_cast<THPDtype*>(t1)->scalar_type;
  Packed* p = reinterpret_cast<Packed*>(type->tp_alloc(type, 0));
  if (!p) return nullptr;
  p->vectorcall = packed_run;
  p->part[0] = part[0];
  p->part[1] = part[1];
  Py_INCREF(pair);
  p->pair = reinterpret_cast<PyTypeObject*>(pair);
  return reinterpret_cast<PyObject*>(p);
}

void packed_free(PyObject* self) {
  Py_XDECREF(reinterpret_cast<PyObject*>(reinterpret_cast<Packed*>(self)->pair));
  Py_TYPE(self)->tp_free(self);
}

PyTypeObject make_type(const char* name, Py_ssize_t size, Py_ssize_t vectorcall, newfunc make, destructor free) {
  PyTypeObject t = {PyVarObject_HEAD_INIT(nullptr, 0)};
  t.tp_name = name;
  t.tp_basicsize = size;
  t.tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_VECTORCALL;
  t.tp_vectorcall_offset = vectorcall;
  t.tp_call = PyVectorcall_Call;
  t.tp_new = make;
  t.tp_dealloc = free;
  return t;
}
PyTypeObject call_type = make_type("_fast_call.Call", sizeof(Call), offsetof(Call, vectorcall), call_new, call_free);
PyTypeObject packed_type = make_type("_fast_call.Packed", sizeof(Packed), offsetof(Packed, vectorcall), packed_new, packed_free);

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast_call", nullptr, -1, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fast_call() {
  if (PyType_Ready(&call_type) < 0 || PyType_Ready(&packed_type) < 0) return nullptr;
  PyObject* m = PyModule_Create(&module);
  if (!m) return nullptr;
  if (PyModule_AddObjectRef(m, "Call", reinterpret_cast<PyObject*>(&call_type)) < 0 ||
      PyModule_AddObjectRef(m, "Packed", reinterpret_cast<PyObject*>(&packed_type)) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
