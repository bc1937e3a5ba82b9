/*
 * q8call.c -- the calls of kv_b200.Q8Cache: checks of the tensors handed over,
 * then the library's entry points, which take 9 to 17 arguments each.
 *
 * A decoded token's call runs for a few microseconds on the GPU; through
 * ctypes, its arguments and tensor checks took about 10 us on the host, here
 * about 2 us.  Tensors are read through their Python attributes (no torch
 * headers); the entry points' addresses come from the loaded library.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>

#include "kv_api.h"

static PyObject *g_f32, *g_f16, *g_i32;   /* torch.float32, torch.float16, torch.int32 */
static PyObject *s_dtype, *s_shape, *s_stride, *s_get_device, *s_data_ptr, *s_cuda_stream, *s_is_contiguous, *s_nbytes;
static int (*p_store)(const kv_q8_cache *, int64_t, int32_t, const void *, int64_t, const void *, int64_t, int32_t, void *);
static int (*p_load)(const kv_q8_cache *, int64_t, int64_t, void *, void *, int64_t, int32_t, void *);
static int (*p_attend)(const kv_q8_cache *, int32_t, int64_t, int32_t, const void *, int64_t, int32_t, const void *, int32_t,
                       int64_t, uint32_t, void *, int64_t, int32_t, void *, uint64_t, void *);
static int (*p_evict)(const kv_q8_cache *, int64_t, int64_t, int64_t, const kv_q8_cache *, int32_t *, void *);

/* an integer attribute, or the integer a method without arguments returns; -1 with an error set */
static int64_t int_of(PyObject *o, PyObject *name, int call)
{
    PyObject *v = call ? PyObject_CallMethodNoArgs(o, name) : PyObject_GetAttr(o, name);
    if (!v) return -1;
    const int64_t x = PyLong_AsLongLong(v);
    Py_DECREF(v);
    return x;
}

static int32_t type_of(PyObject *t)
{
    PyObject *d = PyObject_GetAttr(t, s_dtype);
    if (!d) return -1;
    const int32_t k = d == g_f32 ? KV_F32 : d == g_f16 ? KV_F16 : -1;
    Py_DECREF(d);
    return k;
}

typedef struct {
    void *ptr;
    int64_t stride;
    int32_t type;
} rows_t;

/* A tensor of n rows of `width` contiguous elements on device `dev`.  0 with a ValueError set otherwise. */
static int rows_of(const char *name, PyObject *t, int64_t n, int64_t width, int64_t dev, rows_t *out)
{
    out->type = type_of(t);
    if (out->type < 0) {
        if (!PyErr_Occurred()) PyErr_Format(PyExc_ValueError, "%s must be float32 or float16", name);
        return 0;
    }
    PyObject *shape = PyObject_GetAttr(t, s_shape), *stride = shape ? PyObject_CallMethodNoArgs(t, s_stride) : NULL;
    const int64_t on = stride ? int_of(t, s_get_device, 1) : -1;
    int ok = 0;
    if (stride && !PyErr_Occurred() && PyTuple_Check(shape) && PyTuple_Check(stride)) {
        const Py_ssize_t dims = PyTuple_GET_SIZE(shape);
        int64_t inner = 1;
        ok = 1;
        for (Py_ssize_t i = dims - 1; ok && i > 0; i--) {
            const int64_t x = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, i)), s = PyLong_AsLongLong(PyTuple_GET_ITEM(stride, i));
            if (x != 1 && s != inner) ok = 0;
            inner *= x;
        }
        if (!ok) {
            PyErr_Format(PyExc_ValueError, "the rows of %s must be contiguous", name);
        } else if (dims < 1 || on != dev || inner != width || PyLong_AsLongLong(PyTuple_GET_ITEM(shape, 0)) != n) {
            PyErr_Format(PyExc_ValueError, "%s must hold %lld rows of %lld elements on the cache's device", name, (long long)n,
                         (long long)width);
            ok = 0;
        } else {
            out->stride = PyLong_AsLongLong(PyTuple_GET_ITEM(stride, 0));
            out->ptr = (void *)(intptr_t)int_of(t, s_data_ptr, 1);
            ok = !PyErr_Occurred();
        }
    }
    Py_XDECREF(shape);
    Py_XDECREF(stride);
    return ok;
}

/* None, an integer, or an object with cuda_stream */
static void *stream_of(PyObject *s)
{
    if (s == Py_None) return NULL;
    if (PyLong_Check(s)) return PyLong_AsVoidPtr(s);
    return (void *)(intptr_t)int_of(s, s_cuda_stream, 0);
}

static int64_t as_i64(PyObject *o) { return PyLong_AsLongLong(o); }

/* a 32-bit argument: one that does not fit is out of every range */
static int32_t as_i32(PyObject *o)
{
    const int64_t x = PyLong_AsLongLong(o);
    return x < INT32_MIN || x > INT32_MAX ? -1 : (int32_t)x;
}

static int arity(const char *name, Py_ssize_t n, Py_ssize_t want)
{
    if (n == want) return 1;
    PyErr_Format(PyExc_TypeError, "%s takes %zd arguments", name, want);
    return 0;
}

/* store(cache, device, width, row0, n_new, k, v, stream) */
static PyObject *q8_store(PyObject *self, PyObject *const *a, Py_ssize_t n)
{
    if (!arity("store", n, 8)) return NULL;
    const kv_q8_cache *c = PyLong_AsVoidPtr(a[0]);
    const int64_t dev = as_i64(a[1]), width = as_i64(a[2]), row0 = as_i64(a[3]), count = as_i64(a[4]);
    void *st = stream_of(a[7]);
    rows_t k, v;
    if (PyErr_Occurred() || !rows_of("k", a[5], count, width, dev, &k) || !rows_of("v", a[6], count, width, dev, &v)) return NULL;
    if (k.type != v.type) {
        PyErr_SetString(PyExc_ValueError, "k and v must have one type");
        return NULL;
    }
    return PyLong_FromLong(p_store(c, row0, as_i32(a[4]), k.ptr, k.stride, v.ptr, v.stride, k.type, st));
}

/* load(cache, device, width, row0, n, k_out or None, v_out or None, stream) */
static PyObject *q8_load(PyObject *self, PyObject *const *a, Py_ssize_t n)
{
    if (!arity("load", n, 8)) return NULL;
    const kv_q8_cache *c = PyLong_AsVoidPtr(a[0]);
    const int64_t dev = as_i64(a[1]), width = as_i64(a[2]), row0 = as_i64(a[3]), count = as_i64(a[4]);
    void *st = stream_of(a[7]);
    rows_t k = {NULL, 0, 0}, v = {NULL, 0, 0};
    if (PyErr_Occurred()) return NULL;
    if (a[5] != Py_None && !rows_of("k_out", a[5], count, width, dev, &k)) return NULL;
    if (a[6] != Py_None && !rows_of("v_out", a[6], count, width, dev, &v)) return NULL;
    if (k.ptr && v.ptr && (k.type != v.type || k.stride != v.stride)) {
        PyErr_SetString(PyExc_ValueError, "k_out and v_out must have one type and row stride");
        return NULL;
    }
    const rows_t *x = k.ptr ? &k : &v;
    return PyLong_FromLong(p_load(c, row0, count, k.ptr, v.ptr, x->stride, x->type, st));
}

/* attend(cache, device, head_dim, n_head, n_past, n_new, q, out, mask or None, flash, workspace, stream) */
static PyObject *q8_attend(PyObject *self, PyObject *const *a, Py_ssize_t n)
{
    if (!arity("attend", n, 12)) return NULL;
    const kv_q8_cache *c = PyLong_AsVoidPtr(a[0]);
    const int64_t dev = as_i64(a[1]), n_head = as_i64(a[3]), past = as_i64(a[4]), count = as_i64(a[5]);
    const int64_t width = n_head * as_i64(a[2]);
    const int flash = PyObject_IsTrue(a[9]);
    void *st = stream_of(a[11]);
    rows_t q, out;
    if (PyErr_Occurred() || !rows_of("q", a[6], count, width, dev, &q) || !rows_of("out", a[7], count, width, dev, &out))
        return NULL;
    void *mask = NULL;
    int32_t mask_type = 0;
    int64_t mask_stride = 0;
    if (a[8] != Py_None) {
        PyObject *shape = PyObject_GetAttr(a[8], s_shape), *stride = shape ? PyObject_CallMethodNoArgs(a[8], s_stride) : NULL;
        mask_type = stride ? type_of(a[8]) : -1;
        int ok = stride && mask_type >= 0 && PyTuple_Check(shape) && PyTuple_Check(stride) && PyTuple_GET_SIZE(shape) == 2;
        if (ok) {
            mask_stride = PyLong_AsLongLong(PyTuple_GET_ITEM(stride, 0));
            ok = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, 0)) == count &&
                 PyLong_AsLongLong(PyTuple_GET_ITEM(shape, 1)) >= past + count &&
                 PyLong_AsLongLong(PyTuple_GET_ITEM(stride, 1)) == 1 && int_of(a[8], s_get_device, 1) == dev;
        }
        Py_XDECREF(shape);
        Py_XDECREF(stride);
        if (ok) mask = (void *)(intptr_t)int_of(a[8], s_data_ptr, 1);
        if (!ok && !PyErr_Occurred())
            PyErr_SetString(PyExc_ValueError,
                            "mask must be [n_new][>= n_past + n_new], float32 or float16, on the cache's device");
        if (PyErr_Occurred()) return NULL;
    }
    PyObject *whole = a[10] == Py_None ? NULL : PyObject_CallMethodNoArgs(a[10], s_is_contiguous);
    const int ok = whole == Py_True && int_of(a[10], s_get_device, 1) == dev;
    Py_XDECREF(whole);
    if (!ok) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "attend needs a contiguous workspace tensor on the cache's device");
        return NULL;
    }
    void *ws = (void *)(intptr_t)int_of(a[10], s_data_ptr, 1);
    const int64_t bytes = int_of(a[10], s_nbytes, 0);
    if (PyErr_Occurred()) return NULL;
    return PyLong_FromLong(p_attend(c, as_i32(a[3]), past, as_i32(a[5]), q.ptr, q.stride, q.type, mask, mask_type, mask_stride,
                                    flash ? KV_ATTN_FLASH : 0u, out.ptr, out.stride, out.type, ws, (uint64_t)bytes, st));
}

/* evict(cache, device, n_head_kv, n_rows, keep, recent, dst, dst's device, kept, stream) */
static PyObject *q8_evict(PyObject *self, PyObject *const *a, Py_ssize_t n)
{
    if (!arity("evict", n, 10)) return NULL;
    const kv_q8_cache *c = PyLong_AsVoidPtr(a[0]), *dst = PyLong_AsVoidPtr(a[6]);
    const int64_t dev = as_i64(a[1]), heads = as_i64(a[2]), keep = as_i64(a[4]), ddev = as_i64(a[7]);
    void *st = stream_of(a[9]);
    PyObject *type = PyErr_Occurred() ? NULL : PyObject_GetAttr(a[8], s_dtype);
    PyObject *shape = type ? PyObject_GetAttr(a[8], s_shape) : NULL, *whole = shape ? PyObject_CallMethodNoArgs(a[8], s_is_contiguous) : NULL;
    const int ok = whole == Py_True && type == g_i32 && PyTuple_Check(shape) && PyTuple_GET_SIZE(shape) == 2 &&
                   PyLong_AsLongLong(PyTuple_GET_ITEM(shape, 0)) == heads && PyLong_AsLongLong(PyTuple_GET_ITEM(shape, 1)) == keep &&
                   ddev == dev && int_of(a[8], s_get_device, 1) == dev;
    Py_XDECREF(type);
    Py_XDECREF(shape);
    Py_XDECREF(whole);
    if (!ok) {
        if (!PyErr_Occurred())
            PyErr_Format(PyExc_ValueError, "kept must be a contiguous int32 [%lld][%lld] tensor on the cache's device, dst there too",
                         (long long)heads, (long long)keep);
        return NULL;
    }
    int32_t *kept = (int32_t *)(intptr_t)int_of(a[8], s_data_ptr, 1);
    const int64_t rows = as_i64(a[3]), recent = as_i64(a[5]);
    if (PyErr_Occurred()) return NULL;
    return PyLong_FromLong(p_evict(c, rows, keep, recent, dst, kept, st));
}

/* init(torch.float32, torch.float16, torch.int32, address of kv_q8_store, _load, _attend, _evict) */
static PyObject *q8_init(PyObject *self, PyObject *args)
{
    PyObject *f32, *f16, *i32;
    unsigned long long s, l, a, e;
    if (!PyArg_ParseTuple(args, "OOOKKKK", &f32, &f16, &i32, &s, &l, &a, &e)) return NULL;
    Py_INCREF(f32);
    Py_INCREF(f16);
    Py_INCREF(i32);
    Py_XSETREF(g_f32, f32);
    Py_XSETREF(g_f16, f16);
    Py_XSETREF(g_i32, i32);
    *(void **)&p_store = (void *)(uintptr_t)s;
    *(void **)&p_load = (void *)(uintptr_t)l;
    *(void **)&p_attend = (void *)(uintptr_t)a;
    *(void **)&p_evict = (void *)(uintptr_t)e;
    Py_RETURN_NONE;
}

static PyMethodDef methods[] = {{"init", q8_init, METH_VARARGS, NULL},
                                {"store", (PyCFunction)(void (*)(void))q8_store, METH_FASTCALL, NULL},
                                {"load", (PyCFunction)(void (*)(void))q8_load, METH_FASTCALL, NULL},
                                {"attend", (PyCFunction)(void (*)(void))q8_attend, METH_FASTCALL, NULL},
                                {"evict", (PyCFunction)(void (*)(void))q8_evict, METH_FASTCALL, NULL},
                                {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_q8call", NULL, -1, methods};

PyMODINIT_FUNC PyInit__q8call(void)
{
    s_dtype = PyUnicode_InternFromString("dtype");
    s_shape = PyUnicode_InternFromString("shape");
    s_stride = PyUnicode_InternFromString("stride");
    s_get_device = PyUnicode_InternFromString("get_device");
    s_data_ptr = PyUnicode_InternFromString("data_ptr");
    s_cuda_stream = PyUnicode_InternFromString("cuda_stream");
    s_is_contiguous = PyUnicode_InternFromString("is_contiguous");
    s_nbytes = PyUnicode_InternFromString("nbytes");
    if (!s_dtype || !s_shape || !s_stride || !s_get_device || !s_data_ptr || !s_cuda_stream || !s_is_contiguous || !s_nbytes)
        return NULL;
    return PyModule_Create(&module);
}
