// Calls of the step operators from Python without ctypes' cost per argument: a decode step's operators run
// for a few microseconds each, and ctypes takes 4 to 6 us to convert their 18 to 29 arguments (this:
// under one). bind(name, address, function) gives a callable that converts numbers and None by the C
// prototype and calls `address`; a call with any other kind of argument, or a wrong number of them, goes to
// `function`, the ctypes one, which knows the rest (and raises what it raises).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cstring>
#include <tuple>
#include <type_traits>
#include <utility>

#include "s1_executor.h"

namespace {

// One argument by its C type; false leaves the call to ctypes.
template <class T>
bool convert(PyObject* o, T& out) {
    if constexpr (std::is_pointer_v<T>) {
        if (o == Py_None) {
            out = nullptr;
            return true;
        }
        if (!PyLong_CheckExact(o)) return false;
        void* p = PyLong_AsVoidPtr(o);
        if (!p && PyErr_Occurred()) return PyErr_Clear(), false;
        out = static_cast<T>(p);
        return true;
    } else if constexpr (std::is_floating_point_v<T>) {
        if (!PyFloat_CheckExact(o)) return false;
        out = static_cast<T>(PyFloat_AS_DOUBLE(o));
        return true;
    } else if constexpr (std::is_same_v<T, size_t>) {
        if (!PyLong_CheckExact(o)) return false;
        out = PyLong_AsSize_t(o);
        if (out == static_cast<size_t>(-1) && PyErr_Occurred()) return PyErr_Clear(), false;
        return true;
    } else {
        static_assert(std::is_same_v<T, int>);
        if (!PyLong_CheckExact(o)) return false;
        const long v = PyLong_AsLong(o);
        if ((v == -1 && PyErr_Occurred()) || v != static_cast<int>(v)) return PyErr_Clear(), false;
        out = static_cast<int>(v);
        return true;
    }
}

using Invoke = bool (*)(void* fn, PyObject* const* args, Py_ssize_t n, int* result);

template <class F>
struct Call;
template <class... A>
struct Call<int (*)(A...)> {
    template <size_t... I>
    static bool run(void* fn, PyObject* const* args, int* result, std::index_sequence<I...>) {
        std::tuple<A...> a{};
        if (!(convert(args[I], std::get<I>(a)) && ...)) return false;
        Py_BEGIN_ALLOW_THREADS
        *result = reinterpret_cast<int (*)(A...)>(fn)(std::get<I>(a)...);
        Py_END_ALLOW_THREADS
        return true;
    }
    static bool invoke(void* fn, PyObject* const* args, Py_ssize_t n, int* result) {
        return n == sizeof...(A) && run(fn, args, result, std::index_sequence_for<A...>{});
    }
};

struct Name {
    const char* name;
    Invoke invoke;
};
#define NAME(f) {#f, Call<decltype(&f)>::invoke}  // the type alone: nothing is linked here
const Name NAMES[] = {NAME(s1_gdn_step), NAME(s1_gdn_conv_gates_step), NAME(s1_attn_prep_paged), NAME(s1_attention_paged),
                      NAME(s1_pages_copy)};
#undef NAME

struct Bound {
    PyObject_HEAD
    vectorcallfunc vectorcall;
    void* fn;
    Invoke invoke;
    PyObject* other;
};

PyObject* bound_call(PyObject* self, PyObject* const* args, size_t nargsf, PyObject* kwnames) {
    Bound* b = reinterpret_cast<Bound*>(self);
    int result = 0;
    if ((!kwnames || PyTuple_GET_SIZE(kwnames) == 0) && b->invoke(b->fn, args, PyVectorcall_NARGS(nargsf), &result))
        return PyLong_FromLong(result);
    return PyObject_Vectorcall(b->other, args, nargsf, kwnames);
}
void bound_dealloc(PyObject* self) {
    Py_XDECREF(reinterpret_cast<Bound*>(self)->other);
    Py_TYPE(self)->tp_free(self);
}

PyTypeObject make_type() {
    PyTypeObject t = {PyVarObject_HEAD_INIT(nullptr, 0)};
    t.tp_name = "system1_omni_b200._fastcall.Bound";
    t.tp_basicsize = sizeof(Bound);
    t.tp_dealloc = bound_dealloc;
    t.tp_vectorcall_offset = offsetof(Bound, vectorcall);
    t.tp_call = PyVectorcall_Call;
    t.tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_VECTORCALL;
    return t;
}
PyTypeObject bound_type = make_type();

PyObject* bind(PyObject*, PyObject* args) {
    const char* name;
    PyObject *address, *other;
    if (!PyArg_ParseTuple(args, "sO!O", &name, &PyLong_Type, &address, &other)) return nullptr;
    for (const Name& n : NAMES) {
        if (std::strcmp(n.name, name) != 0) continue;
        void* fn = PyLong_AsVoidPtr(address);
        if (!fn) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "%s: no address", name);
        Bound* b = PyObject_New(Bound, &bound_type);
        if (!b) return nullptr;
        b->vectorcall = bound_call;
        b->fn = fn;
        b->invoke = n.invoke;
        b->other = Py_NewRef(other);
        return reinterpret_cast<PyObject*>(b);
    }
    return PyErr_Format(PyExc_KeyError, "%s", name);
}

PyMethodDef METHODS[] = {{"bind", bind, METH_VARARGS, "bind(name, address, function) -> callable"}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef MODULE = {PyModuleDef_HEAD_INIT, "_fastcall", nullptr, -1, METHODS, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fastcall(void) {
    if (PyType_Ready(&bound_type) < 0) return nullptr;
    PyObject* m = PyModule_Create(&MODULE);
    if (!m) return nullptr;
    PyObject* names = PyTuple_New(sizeof(NAMES) / sizeof(NAMES[0]));
    if (!names) return nullptr;
    for (size_t i = 0; i < sizeof(NAMES) / sizeof(NAMES[0]); i++) PyTuple_SET_ITEM(names, i, PyUnicode_FromString(NAMES[i].name));
    if (PyModule_AddObject(m, "NAMES", names) < 0) return nullptr;
    return m;
}
