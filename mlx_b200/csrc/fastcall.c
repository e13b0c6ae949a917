/* The short calls of lux_gpu_quant_vtbl for Python: mx4_quantize, mx4_dequantize, mx4_matmul, block_norm, qmatmul_epi, moe_route,
 * qmatmul_experts, moe_combine.
 *
 * plugin.py mirrors the whole interface with ctypes, which takes 1.1 us to turn a dozen arguments into C ones (0.2 us here): a
 * third of the time of a call whose kernel takes two or three.  Same entries, same arguments, same codes. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <string.h>

#include "lux_cuda_quant.h"

typedef struct {
    PyObject_HEAD
    const lux_gpu_quant_vtbl* q;
} Entries;

/* None or an address */
static int as_pointer(PyObject* o, void** p) {
    *p = NULL;
    if (o == Py_None) return 1;
    *p = PyLong_AsVoidPtr(o);
    return *p != NULL || !PyErr_Occurred();
}
static int as_int(PyObject* o, int* v) {
    const long n = PyLong_AsLong(o);
    if (n == -1 && PyErr_Occurred()) return 0;
    *v = (int)n;
    if (*v == n) return 1;
    PyErr_SetString(PyExc_OverflowError, "argument does not fit a C int");
    return 0;
}
static int as_size(PyObject* o, size_t* v) {
    PyObject* const n = PyNumber_Index(o); /* (PyLong_AsSize_t takes Python's own integers only) */
    if (!n) return 0;
    *v = PyLong_AsSize_t(n);
    Py_DECREF(n);
    return *v != (size_t)-1 || !PyErr_Occurred();
}
static int as_float(PyObject* o, float* v) {
    const double d = PyFloat_AsDouble(o);
    *v = (float)d;
    return d != -1.0 || !PyErr_Occurred();
}
static int pointers(PyObject* const* a, void** p, int n) {
    for (int i = 0; i < n; i++)
        if (!as_pointer(a[i], p + i)) return 0;
    return 1;
}
static int ints(PyObject* const* a, int* v, int n) {
    for (int i = 0; i < n; i++)
        if (!as_int(a[i], v + i)) return 0;
    return 1;
}
static int count(Py_ssize_t n, Py_ssize_t need) {
    if (n != need) PyErr_Format(PyExc_TypeError, "%zd arguments, %zd expected", n, need);
    return n == need;
}

static PyObject* quantize(Entries* self, PyObject* const* a, Py_ssize_t n) {
    void* p[4];
    int rk[2], fd[2], r;
    size_t ld;
    float pre;
    if (!count(n, 10) || !pointers(a, p, 4) || !ints(a + 4, rk, 2) || !as_size(a[6], &ld) || !ints(a + 7, fd, 2) || !as_float(a[9], &pre)) return NULL;
    Py_BEGIN_ALLOW_THREADS
    r = self->q->mx4_quantize(p[0], p[1], p[2], p[3], rk[0], rk[1], ld, fd[0], fd[1], pre);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(r);
}
static PyObject* dequantize(Entries* self, PyObject* const* a, Py_ssize_t n) {
    void* p[4];
    int v[4], r;
    float post;
    if (!count(n, 9) || !pointers(a, p, 4) || !ints(a + 4, v, 4) || !as_float(a[8], &post)) return NULL;
    Py_BEGIN_ALLOW_THREADS
    r = self->q->mx4_dequantize(p[0], p[1], p[2], p[3], v[0], v[1], v[2], v[3], post);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(r);
}
static PyObject* matmul(Entries* self, PyObject* const* a, Py_ssize_t n) {
    void* p[6];
    int v[5], r;
    float alpha;
    if (!count(n, 12) || !pointers(a, p, 6) || !ints(a + 6, v, 5) || !as_float(a[11], &alpha)) return NULL;
    Py_BEGIN_ALLOW_THREADS
    r = self->q->mx4_matmul(p[0], p[1], p[2], p[3], p[4], p[5], v[0], v[1], v[2], v[3], v[4], alpha);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(r);
}
/* A parameter block (None: no block), copied: another thread may change the caller's while this one is in the call.  1: there is one. */
static int block(PyObject* o, void* dst, size_t size, const char* what) {
    Py_buffer b;
    if (o == Py_None) return 0;
    if (PyObject_GetBuffer(o, &b, PyBUF_SIMPLE)) return -1;
    const int fits = b.len == (Py_ssize_t)size;
    if (fits) memcpy(dst, b.buf, size);
    PyBuffer_Release(&b);
    if (fits) return 1;
    PyErr_SetString(PyExc_TypeError, what);
    return -1;
}
/* entry(context, parameters, N buffers) */
#define WITH_BLOCK(NAME, TYPE, N, CLASS, ...)                                                              \
    static PyObject* NAME(Entries* self, PyObject* const* a, Py_ssize_t n) {                               \
        void *ctx, *p[N];                                                                                  \
        TYPE prm;                                                                                          \
        int r;                                                                                             \
        if (!count(n, N + 2) || !as_pointer(a[0], &ctx) || !pointers(a + 2, p, N)) return NULL;            \
        const int there = block(a[1], &prm, sizeof prm, #NAME ": not a " CLASS);                           \
        if (there < 0) return NULL;                                                                        \
        Py_BEGIN_ALLOW_THREADS                                                                             \
        r = self->q->NAME(ctx, there ? &prm : NULL, __VA_ARGS__);                                          \
        Py_END_ALLOW_THREADS                                                                               \
        return PyLong_FromLong(r);                                                                         \
    }
WITH_BLOCK(block_norm, lux_block_norm_params, 10, "BlockNormParams", p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7], p[8], p[9])
WITH_BLOCK(qmatmul_epi, lux_qmm_epi_params, 7, "QmmEpiParams", p[0], p[1], p[2], p[3], p[4], p[5], p[6])
WITH_BLOCK(moe_route, lux_moe_route_params, 7, "MoeRouteParams", p[0], p[1], p[2], p[3], p[4], p[5], p[6])
WITH_BLOCK(qmatmul_experts, lux_experts_params, 8, "ExpertsParams", p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7])
WITH_BLOCK(moe_combine, lux_moe_combine_params, 5, "MoeCombineParams", p[0], p[1], p[2], p[3], p[4])

static PyMethodDef methods[] = {
    {"mx4_quantize", (PyCFunction)(void (*)(void))quantize, METH_FASTCALL, NULL},
    {"mx4_dequantize", (PyCFunction)(void (*)(void))dequantize, METH_FASTCALL, NULL},
    {"mx4_matmul", (PyCFunction)(void (*)(void))matmul, METH_FASTCALL, NULL},
    {"block_norm", (PyCFunction)(void (*)(void))block_norm, METH_FASTCALL, NULL},
    {"qmatmul_epi", (PyCFunction)(void (*)(void))qmatmul_epi, METH_FASTCALL, NULL},
    {"moe_route", (PyCFunction)(void (*)(void))moe_route, METH_FASTCALL, NULL},
    {"qmatmul_experts", (PyCFunction)(void (*)(void))qmatmul_experts, METH_FASTCALL, NULL},
    {"moe_combine", (PyCFunction)(void (*)(void))moe_combine, METH_FASTCALL, NULL},
    {NULL, NULL, 0, NULL},
};
/* Entries(address of a lux_gpu_quant_vtbl) */
static PyObject* entries_new(PyTypeObject* type, PyObject* args, PyObject* kw) {
    PyObject* o;
    void* p;
    if (kw && PyDict_GET_SIZE(kw)) return PyErr_Format(PyExc_TypeError, "no keywords");
    if (!PyArg_ParseTuple(args, "O", &o) || !as_pointer(o, &p)) return NULL;
    const lux_gpu_quant_vtbl* q = p;
    if (!q || !LUX_CUDA_QUANT_HAS(q, moe_combine)) return PyErr_Format(PyExc_ValueError, "no table of a library with these entries");
    Entries* self = (Entries*)type->tp_alloc(type, 0);
    if (self) self->q = q;
    return (PyObject*)self;
}
static PyTypeObject entries_type = {
    PyVarObject_HEAD_INIT(NULL, 0).tp_name = "fastcall.Entries",
    .tp_basicsize = sizeof(Entries),
    .tp_flags = Py_TPFLAGS_DEFAULT,
    .tp_methods = methods,
    .tp_new = entries_new,
};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "fastcall", NULL, -1, NULL, NULL, NULL, NULL, NULL};
PyMODINIT_FUNC PyInit_fastcall(void) {
    PyObject* m = PyType_Ready(&entries_type) ? NULL : PyModule_Create(&module);
    if (m && PyModule_AddObjectRef(m, "Entries", (PyObject*)&entries_type)) Py_CLEAR(m);
    return m;
}
