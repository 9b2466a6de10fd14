// The Python binding of the entry points that a serving step calls once per layer, over the CPython C API.
//
// ctypes takes 4 to 5 us to convert the 25 to 30 arguments of such a call, more than the kernel runs for when
// the step is a few decode tokens; here they take 0.3.  The functions are the ones of include/prism_kv.h, found in
// the library that the package has loaded (attach); arguments are its arguments, pointers and strides as ints.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <dlfcn.h>

#include <tuple>
#include <type_traits>
#include <utility>

#include "../../include/prism_kv.h"

namespace {

template <typename T>
T convert(PyObject* o) {
  if constexpr (std::is_pointer<T>::value) {
    return reinterpret_cast<T>(PyLong_AsVoidPtr(o));
  } else if constexpr (std::is_floating_point<T>::value) {
    return static_cast<T>(PyFloat_AsDouble(o));
  } else if constexpr (std::is_same<T, size_t>::value) {
    return PyLong_AsSize_t(o);
  } else {
    const long long v = PyLong_AsLongLong(o);
    if (v != static_cast<long long>(static_cast<T>(v)))
      PyErr_Format(PyExc_OverflowError, "argument %lld does not fit %d bytes", v, int(sizeof(T)));
    return static_cast<T>(v);
  }
}

// One entry point: its address in the attached library, and the call.
template <typename F>
struct Entry;
template <typename... A>
struct Entry<int(A...)> {
  using Fn = int (*)(A...);
  template <size_t... I>
  static PyObject* invoke(void* fn, PyObject* const* args, std::index_sequence<I...>) {
    const std::tuple<A...> a{convert<A>(args[I])...};  // in order: the first error is the one reported
    if (PyErr_Occurred()) return nullptr;
    return PyLong_FromLong(reinterpret_cast<Fn>(fn)(std::get<I>(a)...));
  }
  static PyObject* call(const char* name, void* fn, PyObject* const* args, Py_ssize_t n) {
    if (!fn) return PyErr_Format(PyExc_RuntimeError, "%s: no library attached", name);
    if (n != Py_ssize_t(sizeof...(A)))
      return PyErr_Format(PyExc_TypeError, "%s takes %d arguments (%zd given)", name, int(sizeof...(A)), n);
    return invoke(fn, args, std::index_sequence_for<A...>{});
  }
};

#define ENTRIES(X) X(pkv_rotate_qk) X(pkv_packed_rope_append) X(pkv_packed_attn)
#define DEFINE(name)                                                                       \
  void* g_##name = nullptr;                                                                \
  PyObject* py_##name(PyObject*, PyObject* const* args, Py_ssize_t n) {                    \
    return Entry<decltype(::name)>::call(#name, g_##name, args, n);                        \
  }
ENTRIES(DEFINE)

PyObject* attach(PyObject*, PyObject* arg) {
  void* lib = PyLong_AsVoidPtr(arg);
  if (PyErr_Occurred()) return nullptr;
#define FIND(name) \
  if (!(g_##name = dlsym(lib, #name))) return PyErr_Format(PyExc_RuntimeError, "%s not in the library", #name);
  ENTRIES(FIND)
  Py_RETURN_NONE;
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_##name)), METH_FASTCALL, nullptr},
PyMethodDef methods[] = {
    {"attach", attach, METH_O, "attach(handle): take the entry points from a loaded libprism_kv.so"},
    ENTRIES(METHOD){nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fastcall", "libprism_kv entry points without ctypes", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fastcall() { return PyModule_Create(&module); }
