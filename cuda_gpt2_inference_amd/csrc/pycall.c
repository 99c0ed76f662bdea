// pycall.c -- calls of libkvattn.so's entry points from Python.  An eager call of a few microseconds on the
// GPU is bound by the host: 3.3 us of the runtime's launch, and in ctypes, with an address asked of every
// tensor in Python, 2.3 to 3.8 more.  A Call takes tensors, addresses, integers and None as they are and
// needs 0.9 to 1.5 (paged_reserve with 17 arguments 3.8 -> 1.5 us of host time, paged_store 2.3 -> 0.9).
// Where the entry point has an integer it takes an integer's value alone, as ctypes does: a tensor's address, or
// None's zero, would be a count there.
//
// Every parameter of the entry points is a pointer or an integer, which on x86-64 System V each take a
// register or a stack word of 64 bits that the callee reads its own width of, and the caller takes
// off again: so one call with the most words there are serves them all, the unused ones zero.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stddef.h>

#if !defined(__x86_64__) || !defined(__linux__)
#error "words of a call are laid out for x86-64 System V"
#endif

#define MOST 24
typedef long long Word;

typedef struct {
    PyObject_HEAD
    vectorcallfunc call;
    void* entry;
    Py_ssize_t words;
    unsigned long long integers;   // bit i: word i is no address
} Call;

static PyObject* data_ptr;         // the name
static PyObject* argument_error;   // ctypes.ArgumentError

// An integer's low 64 bits, zero for None, a tensor's address.
static int word_of(PyObject* x, Word* w) {
    PyObject* n;
    if (x == Py_None) {
        *w = 0;
        return 0;
    }
    if (PyLong_Check(x)) {
        *w = (Word)PyLong_AsUnsignedLongLongMask(x);
        return *w == -1 && PyErr_Occurred() ? -1 : 0;
    }
    n = PyObject_CallMethodNoArgs(x, data_ptr);
    if (!n && PyErr_ExceptionMatches(PyExc_AttributeError)) {
        PyErr_Clear();
        n = PyNumber_Index(x);
    }
    if (!n) return -1;
    *w = (Word)PyLong_AsUnsignedLongLongMask(n);
    Py_DECREF(n);
    return *w == -1 && PyErr_Occurred() ? -1 : 0;
}

// The low 64 bits of an integer, or of what stands for one (a tensor of one integer is its value).
static int integer_of(PyObject* x, Py_ssize_t i, Word* w) {
    PyObject* const n = PyNumber_Index(x);
    if (!n) {
        if (PyErr_ExceptionMatches(PyExc_TypeError))
            PyErr_Format(argument_error, "argument %zd: an integer expected, not %s", i + 1, Py_TYPE(x)->tp_name);
        return -1;
    }
    *w = (Word)PyLong_AsUnsignedLongLongMask(n);
    Py_DECREF(n);
    return *w == -1 && PyErr_Occurred() ? -1 : 0;
}

static PyObject* call_entry(PyObject* self, PyObject* const* args, size_t nargsf, PyObject* names) {
    const Call* const c = (const Call*)self;
    const Py_ssize_t n = PyVectorcall_NARGS(nargsf);
    Word w[MOST] = {0};
    int status;
    if (n != c->words || (names && PyTuple_GET_SIZE(names) > 0))
        return PyErr_Format(PyExc_TypeError, "%zd positional arguments expected, %zd given", c->words, n);
    for (Py_ssize_t i = 0; i < n; ++i)
        if ((c->integers >> i & 1 ? integer_of(args[i], i, w + i) : word_of(args[i], w + i)) < 0) return NULL;
    Py_BEGIN_ALLOW_THREADS
    status = ((int (*)(Word, Word, Word, Word, Word, Word, Word, Word, Word, Word, Word, Word, Word, Word, Word, Word, Word,
                       Word, Word, Word, Word, Word, Word, Word))c->entry)(
        w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7], w[8], w[9], w[10], w[11], w[12], w[13], w[14], w[15], w[16], w[17],
        w[18], w[19], w[20], w[21], w[22], w[23]);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(status);
}

static PyObject* call_new(PyTypeObject* type, PyObject* args, PyObject* kwargs) {
    unsigned long long entry, integers = 0;
    Py_ssize_t words;
    Call* c;
    if (kwargs && PyDict_GET_SIZE(kwargs) > 0) return PyErr_Format(PyExc_TypeError, "Call(address, words, integers)");
    if (!PyArg_ParseTuple(args, "Kn|K", &entry, &words, &integers)) return NULL;
    if (!entry || words < 0 || words > MOST) return PyErr_Format(PyExc_ValueError, "Call: no address, or more than %d words", MOST);
    c = (Call*)type->tp_alloc(type, 0);
    if (!c) return NULL;
    c->call = call_entry;
    c->entry = (void*)(size_t)entry;
    c->words = words;
    c->integers = integers;
    return (PyObject*)c;
}

static PyTypeObject call_type = {
    PyVarObject_HEAD_INIT(NULL, 0)
    .tp_name = "_pycall.Call",
    .tp_doc = "Call(address, words, integers=0): the C function int f(words words) at address, as a callable.  Words "
              "whose bit of integers is set take an integer's value alone.",
    .tp_basicsize = sizeof(Call),
    .tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_VECTORCALL,
    .tp_vectorcall_offset = offsetof(Call, call),
    .tp_call = PyVectorcall_Call,
    .tp_new = call_new,
};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_pycall", NULL, -1, NULL};

PyMODINIT_FUNC PyInit__pycall(void) {
    PyObject *m, *ctypes;
    data_ptr = PyUnicode_InternFromString("data_ptr");
    ctypes = data_ptr ? PyImport_ImportModule("ctypes") : NULL;
    if (!ctypes) return NULL;
    argument_error = PyObject_GetAttrString(ctypes, "ArgumentError");
    Py_DECREF(ctypes);
    if (!argument_error || PyType_Ready(&call_type) < 0) return NULL;
    m = PyModule_Create(&module);
    if (!m) return NULL;
    Py_INCREF(&call_type);
    if (PyModule_AddObject(m, "Call", (PyObject*)&call_type) < 0) {
        Py_DECREF(&call_type);
        Py_DECREF(m);
        return NULL;
    }
    return m;
}
