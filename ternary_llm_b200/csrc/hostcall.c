/* The three operators on prepared weights and those of the 4-bit cache, from Python to the C ABI in one native call.
 *
 * A call of a small projection is bound by the host: through ctypes and checks written in Python it
 * takes 9.7 us, of which 3.2 are an object for the current stream, 2.5 the checks of three tensors and 1
 * the conversion of arguments, in front of a kernel of 3.2 us.  The functions here ask the tensors the same
 * questions and call the library, 4.1 us with the launch; where an answer is not the expected one, or an argument is not a plain
 * int or float, they return None and do nothing, and the caller goes through the checks in Python, which
 * say what is wrong.  Nothing is kept from one call for the next; the structs of a cache and a rotary table are made with
 * them, and each call asks whether their memory is still there.
 *
 * The library's functions are handed over as addresses, so that whichever build of it is loaded is used. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <limits.h>

#include "tllm_b200_cache4.h"

typedef int (*gemv_fn)(const void*, const void*, void*, int, int, int, void*);
typedef int (*gemv_int8_fn)(const void*, const void*, float, void*, int, int, void*);
typedef int (*gemm_fn)(const void*, const void*, void*, int, int, int, void*);

static gemv_fn f_gemv;
static gemv_int8_fn f_gemv_int8;
static gemm_fn f_gemm;
static PyObject *current_device, *raw_stream;                   /* callables of torch */
static PyObject *d_half, *d_int8, *d_uint8;                     /* its dtypes */
static PyObject *s_is_cuda, *s_dtype, *s_is_contiguous, *s_get_device, *s_numel, *s_data_ptr;

/* Consumes a new reference; 1: it is True, 0: it is not (or an exception, which is dropped). */
static int is_true(PyObject* o)
{
    const int r = o == Py_True;
    if (!o) PyErr_Clear();
    Py_XDECREF(o);
    return r;
}
/* Consumes a new reference; -1 where it is no number of the range 0 .. LLONG_MAX. */
static long long number(PyObject* o)
{
    long long v = -1;
    if (o) v = PyLong_AsLongLong(o);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        v = -1;
    }
    Py_XDECREF(o);
    return v;
}
static PyObject* method(PyObject* t, PyObject* name) { return PyObject_CallMethodNoArgs(t, name); }

/* 1 and the address: a contiguous CUDA tensor of this type on the current device with at least `need` elements. */
static int tensor(PyObject* t, PyObject* dtype, long long device, long long need, void** p)
{
    if (!is_true(PyObject_GetAttr(t, s_is_cuda))) return 0;
    PyObject* d = PyObject_GetAttr(t, s_dtype);
    if (!d) PyErr_Clear();
    Py_XDECREF(d);
    if (d != dtype) return 0;
    if (!is_true(method(t, s_is_contiguous)) || number(method(t, s_get_device)) != device || number(method(t, s_numel)) < need) return 0;
    /* an address is unsigned: above 2^63 number() refuses it and the call takes the other way */
    const long long a = number(method(t, s_data_ptr));
    if (a < 0) return 0;
    *p = (void*)a;
    return 1;
}

/* a plain int of 1 .. INT_MAX, else 0 */
static int positive(PyObject* o)
{
    if (!PyLong_CheckExact(o)) return 0;
    int over = 0;
    const long long v = PyLong_AsLongLongAndOverflow(o, &over);
    return over || v < 1 || v > INT_MAX ? 0 : (int)v;
}

static int where(long long* device, void** stream)
{
    PyObject* dev = PyObject_CallNoArgs(current_device);
    PyObject* st = dev ? PyObject_CallOneArg(raw_stream, dev) : NULL;
    if (!st) PyErr_Clear();
    *device = number(dev);
    const long long s = number(st);
    *stream = (void*)s;
    return f_gemv && *device >= 0 && s >= 0;
}

/* (packed, rows, cols, input, output, batch) */
static PyObject* gemv_packed(PyObject* self, PyObject* const* a, Py_ssize_t n)
{
    long long dev;
    void *w, *x, *y, *stream;
    const int rows = n == 6 ? positive(a[1]) : 0, cols = n == 6 ? positive(a[2]) : 0, batch = n == 6 ? positive(a[5]) : 0;
    if (!rows || !batch || cols < 128 || cols % 128 || !where(&dev, &stream) || !tensor(a[0], d_uint8, dev, 0, &w) ||
        !tensor(a[3], d_half, dev, (long long)batch * cols, &x) || !tensor(a[4], d_half, dev, (long long)batch * rows, &y))
        Py_RETURN_NONE;
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = f_gemv(w, x, y, batch, rows, cols, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(status);
}

/* (packed, rows, cols, input, scale, output) */
static PyObject* gemv_int8_packed(PyObject* self, PyObject* const* a, Py_ssize_t n)
{
    long long dev;
    void *w, *x, *y, *stream;
    const int rows = n == 6 ? positive(a[1]) : 0, cols = n == 6 ? positive(a[2]) : 0;
    if (!rows || !cols || !PyFloat_CheckExact(a[4]) || !where(&dev, &stream) || !tensor(a[0], d_uint8, dev, 0, &w) ||
        !tensor(a[3], d_int8, dev, cols, &x) || !tensor(a[5], d_half, dev, rows, &y))
        Py_RETURN_NONE;
    const float scale = (float)PyFloat_AS_DOUBLE(a[4]);
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = f_gemv_int8(w, x, scale, y, rows, cols, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(status);
}

/* (A, packed, rows, cols, C, M) */
static PyObject* gemm_packed(PyObject* self, PyObject* const* a, Py_ssize_t n)
{
    long long dev;
    void *w, *x, *y, *stream;
    const int rows = n == 6 ? positive(a[2]) : 0, cols = n == 6 ? positive(a[3]) : 0, m = n == 6 ? positive(a[5]) : 0;
    if (!rows || !m || cols < 128 || cols % 128 || !where(&dev, &stream) || !tensor(a[0], d_half, dev, (long long)m * cols, &x) ||
        !tensor(a[1], d_uint8, dev, 0, &w) || !tensor(a[4], d_half, dev, (long long)m * rows, &y))
        Py_RETURN_NONE;
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = f_gemm(x, w, y, m, rows, cols, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(status);
}

/* ---- 4-bit cache: handles are C structs made once by the Python objects that own the memory, and its tensors, which are asked each time whether they
 * are still there ---- */
static int (*f_rotary)(int, const tllm_b200_rotary_table*, const int*, int, const tllm_b200_heads*, const tllm_b200_heads*, int, const tllm_b200_heads*,
                       const tllm_b200_heads*, int, int, int, void*);
static int (*f_append)(const tllm_b200_cache4*, int, const tllm_b200_rotary_table*, const int*, const int*, int, const tllm_b200_heads*,
                       const tllm_b200_heads*, int, const tllm_b200_heads*, const tllm_b200_heads*, void*);
static int (*f_read)(const tllm_b200_cache4*, int, const int*, const int*, int, const tllm_b200_heads*, const tllm_b200_heads*, void*);
static int (*f_attention)(const tllm_b200_cache4*, int, const int*, const int*, int, const tllm_b200_heads*, const tllm_b200_heads*, int, float, int, int,
                          void*, size_t, void*);
static int (*f_workspace)(const tllm_b200_cache4*, int, int, int, int, size_t*);
static PyObject *d_types[3], *d_int32;                          /* FP16, BF16, FP32 as the C ABI numbers them */
static PyObject *s_shape, *s_stride, *s_new_empty, *s_nbytes;

/* Three numbers of a tuple; consumes the reference. */
static int triple(PyObject* o, long long* v)
{
    int ok = o && PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 3;
    for (int i = 0; ok && i < 3; i++) {
        v[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(o, i));
        ok = !PyErr_Occurred();
    }
    PyErr_Clear();
    Py_XDECREF(o);
    return ok;
}

/* 1 and the rows of a CUDA tensor [tokens, heads, dim] whose heads lie behind one another; *type, and entries of `shape`, are set where
 * they are -1 and must agree otherwise.  Empty tensors go the other way. */
static int rows3(PyObject* t, long long device, int* type, long long* shape, tllm_b200_heads* r)
{
    long long n[3], st[3];
    if (!is_true(PyObject_GetAttr(t, s_is_cuda))) return 0;
    PyObject* d = PyObject_GetAttr(t, s_dtype);
    if (!d) PyErr_Clear();
    Py_XDECREF(d);
    int k = 0;
    while (k < 3 && d != d_types[k]) k++;
    if (k == 3 || (*type >= 0 && *type != k) || number(method(t, s_get_device)) != device) return 0;
    *type = k;
    if (!triple(PyObject_GetAttr(t, s_shape), n) || !triple(method(t, s_stride), st)) return 0;
    for (int i = 0; i < 3; i++) {
        if (n[i] < 1 || n[i] > INT_MAX || (shape[i] >= 0 && shape[i] != n[i])) return 0;
        shape[i] = n[i];
    }
    if ((n[2] > 1 && st[2] != 1) || (n[1] > 1 && st[1] != n[2])) return 0;
    const long long a = number(method(t, s_data_ptr));
    if (a <= 0) return 0;
    r->p = (void*)a;
    r->ld = n[0] > 1 ? st[0] : n[1] * n[2];
    return 1;
}

/* 1: tensor and storage are still the memory that a handle was made of, `bytes` of storage and the tensor at `p` in it.  The handle holds the
 * storage, so that its memory can only go by a change of its size. */
static int same(PyObject* t, PyObject* storage, PyObject* bytes, const void* p)
{
    return p && number(method(t, s_data_ptr)) == (long long)p && number(method(storage, s_nbytes)) == PyLong_AsLongLong(bytes);
}

/* The C struct that `o`, (struct, its device, then a tensor, its storage and the storage's bytes for each address that the struct begins with), holds,
 * where they are the memory they were. */
static const void* handle(PyObject* o, long long current, size_t size, int addresses)
{
    if (!PyTuple_CheckExact(o) || PyTuple_GET_SIZE(o) != 2 + 3 * addresses) return NULL;
    PyObject *b = PyTuple_GET_ITEM(o, 0), *device = PyTuple_GET_ITEM(o, 1);
    if (!PyBytes_CheckExact(b) || (size_t)PyBytes_GET_SIZE(b) != size || !PyLong_CheckExact(device) || PyLong_AsLongLong(device) != current) return NULL;
    void* const* p = (void* const*)PyBytes_AS_STRING(b);
    for (int i = 0; i < addresses; i++)
        if (!same(PyTuple_GET_ITEM(o, 2 + 3 * i), PyTuple_GET_ITEM(o, 3 + 3 * i), PyTuple_GET_ITEM(o, 4 + 3 * i), p[i])) return NULL;
    return p;
}
static const tllm_b200_cache4* cache_of(PyObject* o, long long device) { return handle(o, device, sizeof(tllm_b200_cache4), 4); }
static const tllm_b200_rotary_table* table_of(PyObject* o, long long device) { return handle(o, device, sizeof(tllm_b200_rotary_table), 1); }

/* int32 tensors of batch + 1 and batch entries */
static int sequences(const tllm_b200_cache4* c, PyObject* first, PyObject* lens, long long dev, void** f, void** n)
{
    return c->batch > 0 && tensor(first, d_int32, dev, (long long)c->batch + 1, f) && number(method(first, s_numel)) == (long long)c->batch + 1 &&
           tensor(lens, d_int32, dev, c->batch, n) && number(method(lens, s_numel)) == c->batch;
}

/* a plain int of 0 .. INT_MAX, else -1 */
static int not_negative(PyObject* o)
{
    if (!PyLong_CheckExact(o)) return -1;
    int over = 0;
    const long long v = PyLong_AsLongLongAndOverflow(o, &over);
    return over || v < 0 || v > INT_MAX ? -1 : (int)v;
}

/* (table, q, k or None, positions, q_out or None, k_out or None, inverse) */
static PyObject* rotary(PyObject* self, PyObject* const* a, Py_ssize_t n)
{
    long long dev, q3[3] = {-1, -1, -1}, k3[3];
    void *positions, *stream;
    int type = -1;
    tllm_b200_heads q, qo, k, ko;
    const tllm_b200_rotary_table* t;
    if (n != 7 || !f_rotary || !where(&dev, &stream) || !(t = table_of(a[0], dev)) || !rows3(a[1], dev, &type, q3, &q) || !PyBool_Check(a[6])) Py_RETURN_NONE;
    const int keys = a[2] != Py_None;
    k3[0] = q3[0], k3[1] = -1, k3[2] = q3[2];
    if (!rows3(a[4] == Py_None ? a[1] : a[4], dev, &type, q3, &qo) || (!keys && a[5] != Py_None) ||
        (keys && (!rows3(a[2], dev, &type, k3, &k) || !rows3(a[5] == Py_None ? a[2] : a[5], dev, &type, k3, &ko))) ||
        !tensor(a[3], d_int32, dev, q3[0], &positions))
        Py_RETURN_NONE;
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = f_rotary(type, t, positions, (int)q3[0], &q, &qo, (int)q3[1], keys ? &k : NULL, keys ? &ko : NULL, keys ? (int)k3[1] : 0, (int)q3[2],
                      a[6] == Py_True, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(status);
}

/* (cache, table or None, q or None, k, v, first, lens, q_out or None) */
static PyObject* cache4_append(PyObject* self, PyObject* const* a, Py_ssize_t n)
{
    long long dev, q3[3], k3[3] = {-1, -1, -1};
    void *first, *lens, *stream;
    int type = -1;
    tllm_b200_heads q, qo, k, v;
    const tllm_b200_cache4* c;
    const tllm_b200_rotary_table* t = NULL;
    if (n != 8 || !f_append || !where(&dev, &stream) || !(c = cache_of(a[0], dev)) || (a[1] != Py_None && !(t = table_of(a[1], dev)))) Py_RETURN_NONE;
    k3[1] = c->kv_heads, k3[2] = c->dim;
    const int queries = a[2] != Py_None;
    if (!rows3(a[3], dev, &type, k3, &k) || type == TLLM_FP32 || !rows3(a[4], dev, &type, k3, &v) || !sequences(c, a[5], a[6], dev, &first, &lens))
        Py_RETURN_NONE;
    q3[0] = k3[0], q3[1] = -1, q3[2] = c->dim;
    if ((!queries && a[7] != Py_None) || (queries && (!rows3(a[2], dev, &type, q3, &q) || !rows3(a[7] == Py_None ? a[2] : a[7], dev, &type, q3, &qo))))
        Py_RETURN_NONE;
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = f_append(c, type, t, first, lens, (int)k3[0], queries ? &q : NULL, queries ? &qo : NULL, queries ? (int)q3[1] : 0, &k, &v, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(status);
}

/* (cache, k or None, v or None, first, lens) */
static PyObject* cache4_read(PyObject* self, PyObject* const* a, Py_ssize_t n)
{
    long long dev, k3[3] = {-1, -1, -1};
    void *first, *lens, *stream;
    int type = -1;
    tllm_b200_heads k, v;
    const tllm_b200_cache4* c;
    if (n != 5 || !f_read || !where(&dev, &stream) || !(c = cache_of(a[0], dev)) || (a[1] == Py_None && a[2] == Py_None)) Py_RETURN_NONE;
    k3[1] = c->kv_heads, k3[2] = c->dim;
    if ((a[1] != Py_None && !rows3(a[1], dev, &type, k3, &k)) || (a[2] != Py_None && !rows3(a[2], dev, &type, k3, &v)) ||
        !sequences(c, a[3], a[4], dev, &first, &lens))
        Py_RETURN_NONE;
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = f_read(c, type, first, lens, (int)k3[0], a[1] != Py_None ? &k : NULL, a[2] != Py_None ? &v : NULL, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(status);
}

/* (cache, q, out, first, lens, scale, max_new, max_len); the workspace is a tensor of the call's own */
static PyObject* cache4_attention(PyObject* self, PyObject* const* a, Py_ssize_t n)
{
    long long dev, q3[3] = {-1, -1, -1};
    void *first, *lens, *stream, *ws = NULL;
    int type = -1;
    size_t need = 0;
    tllm_b200_heads q, out;
    const tllm_b200_cache4* c;
    if (n != 8 || !f_attention || !where(&dev, &stream) || !(c = cache_of(a[0], dev)) || !PyFloat_CheckExact(a[5])) Py_RETURN_NONE;
    const int max_new = not_negative(a[6]), max_len = not_negative(a[7]);
    q3[2] = c->dim;
    if (max_new < 0 || max_len < 0 || !rows3(a[1], dev, &type, q3, &q) || type == TLLM_FP32 || !rows3(a[2], dev, &type, q3, &out) ||
        !sequences(c, a[3], a[4], dev, &first, &lens))
        Py_RETURN_NONE;
    int status = f_workspace(c, (int)q3[0], (int)q3[1], max_new, max_len, &need);
    if (status) return PyLong_FromLong(status);
    PyObject* memory = NULL;
    if (need) {
        PyObject* size = PyLong_FromSize_t((need + 1) / 2);               /* q's type has two bytes */
        memory = size ? PyObject_CallMethodOneArg(a[1], s_new_empty, size) : NULL;
        Py_XDECREF(size);
        if (!memory) return NULL;                                         /* out of memory, as torch says it */
        const long long p = number(method(memory, s_data_ptr));
        if (p <= 0) {
            Py_DECREF(memory);
            Py_RETURN_NONE;
        }
        ws = (void*)p;
    }
    const float scale = (float)PyFloat_AS_DOUBLE(a[5]);
    Py_BEGIN_ALLOW_THREADS
    status = f_attention(c, type, first, lens, (int)q3[0], &q, &out, (int)q3[1], scale, max_new, max_len, ws, need, stream);
    Py_END_ALLOW_THREADS
    Py_XDECREF(memory);
    return PyLong_FromLong(status);
}

/* (rotary, append, read, attention, workspace addresses, bfloat16, float32, int32), after bind */
static PyObject* bind_cache4(PyObject* self, PyObject* args)
{
    unsigned long long f[5];
    PyObject *b, *s, *i;
    if (!PyArg_ParseTuple(args, "KKKKKOOO", &f[0], &f[1], &f[2], &f[3], &f[4], &b, &s, &i)) return NULL;
    Py_INCREF(b);
    Py_INCREF(s);
    Py_INCREF(i);
    d_types[0] = d_half, d_types[1] = b, d_types[2] = s, d_int32 = i;
    f_append = (void*)(uintptr_t)f[1];
    f_read = (void*)(uintptr_t)f[2];
    f_workspace = (void*)(uintptr_t)f[4];
    f_attention = (void*)(uintptr_t)f[3];
    f_rotary = (void*)(uintptr_t)f[0];
    Py_RETURN_NONE;
}

/* (gemv, gemv_int8, gemm addresses, current_device, raw_stream, float16, int8, uint8) */
static PyObject* bind(PyObject* self, PyObject* args)
{
    unsigned long long g, i, m;
    PyObject *o[5], **d[5] = {&current_device, &raw_stream, &d_half, &d_int8, &d_uint8};
    if (!PyArg_ParseTuple(args, "KKKOOOOO", &g, &i, &m, &o[0], &o[1], &o[2], &o[3], &o[4])) return NULL;
    for (int k = 0; k < 5; k++) {
        Py_INCREF(o[k]);
        Py_XSETREF(*d[k], o[k]);
    }
    f_gemv_int8 = (gemv_int8_fn)(uintptr_t)i;
    f_gemm = (gemm_fn)(uintptr_t)m;
    f_gemv = (gemv_fn)(uintptr_t)g;
    Py_RETURN_NONE;
}

static PyMethodDef methods[] = {
    {"gemv_packed", (PyCFunction)(void*)gemv_packed, METH_FASTCALL, NULL},
    {"gemv_int8_packed", (PyCFunction)(void*)gemv_int8_packed, METH_FASTCALL, NULL},
    {"gemm_packed", (PyCFunction)(void*)gemm_packed, METH_FASTCALL, NULL},
    {"bind", bind, METH_VARARGS, NULL},
    {"rotary", (PyCFunction)(void*)rotary, METH_FASTCALL, NULL},
    {"cache4_append", (PyCFunction)(void*)cache4_append, METH_FASTCALL, NULL},
    {"cache4_read", (PyCFunction)(void*)cache4_read, METH_FASTCALL, NULL},
    {"cache4_attention", (PyCFunction)(void*)cache4_attention, METH_FASTCALL, NULL},
    {"bind_cache4", bind_cache4, METH_VARARGS, NULL},
    {NULL, NULL, 0, NULL},
};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_hostcall", "Operators on prepared weights and on the 4-bit cache in one native call.", -1, methods,
                                    NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__hostcall(void)
{
    s_is_cuda = PyUnicode_InternFromString("is_cuda");
    s_dtype = PyUnicode_InternFromString("dtype");
    s_is_contiguous = PyUnicode_InternFromString("is_contiguous");
    s_get_device = PyUnicode_InternFromString("get_device");
    s_numel = PyUnicode_InternFromString("numel");
    s_data_ptr = PyUnicode_InternFromString("data_ptr");
    s_shape = PyUnicode_InternFromString("shape");
    s_stride = PyUnicode_InternFromString("stride");
    s_new_empty = PyUnicode_InternFromString("new_empty");
    s_nbytes = PyUnicode_InternFromString("nbytes");
    if (!s_shape || !s_stride || !s_new_empty || !s_nbytes) return NULL;
    if (!s_is_cuda || !s_dtype || !s_is_contiguous || !s_get_device || !s_numel || !s_data_ptr) return NULL;
    return PyModule_Create(&module);
}
