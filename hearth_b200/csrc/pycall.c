/* Python's way into the calls of the 8-bit linear path that a decode loop makes for every token.  Through ctypes and
 * checks in Python, two such calls cost more host time (about 4 us) than their kernels run; here the checks of the usual
 * case - two-dimensional CUDA tensors of the right type on the handle's device - and the call itself take a tenth of it.
 * Anything else (another shape, type or device, a missing tensor) returns None, and api.py's own checks then refuse or
 * serve it; a number is the call's status code.  The C entry points are those of the library that ctypes loaded; like
 * ctypes, the calls let other Python threads run meanwhile (a full launch queue blocks). */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stddef.h>

typedef int (*quantize_fn)(void *, const float *, size_t, size_t, void *);
typedef int (*norm_fn)(void *, const float *, const float *, size_t, const float *, float, size_t, float *, size_t, void *);
typedef int (*silu_fn)(void *, const float *, const float *, size_t, size_t, void *);
typedef int (*dequantize_fn)(void *, float *, size_t, size_t, void *);
typedef int (*matmul_fn)(void *, void *, size_t, float *, size_t, int, void *);

static quantize_fn f_quantize;
static norm_fn f_norm;
static silu_fn f_silu;
static dequantize_fn f_dequantize;
static matmul_fn f_matmul;
static PyObject *g_f32, *g_raw_stream;
static PyObject *s_dtype, *s_shape, *s_stride, *s_data_ptr, *s_get_device, *s_cuda_stream;

/* A non-negative integer; 0 if it is none. */
static int number(PyObject *o, size_t *out) {
    if (!o || !PyLong_Check(o)) return 0;
    *out = PyLong_AsSize_t(o);
    if (*out == (size_t)-1 && PyErr_Occurred()) { PyErr_Clear(); return 0; }
    return 1;
}

static int of_tensor(PyObject *t, size_t device, void **p) {
    PyObject *d = PyObject_GetAttr(t, s_dtype);
    if (!d) { PyErr_Clear(); return 0; }
    const int f32 = d == g_f32;
    Py_DECREF(d);
    if (!f32) return 0;
    PyObject *dev = PyObject_CallMethodNoArgs(t, s_get_device);
    if (!dev) { PyErr_Clear(); return 0; }
    size_t n;
    const int same = number(dev, &n) && n == device;
    Py_DECREF(dev);
    if (!same) return 0;
    PyObject *a = PyObject_CallMethodNoArgs(t, s_data_ptr);
    if (!a) { PyErr_Clear(); return 0; }
    const int ok = number(a, &n);
    Py_DECREF(a);
    *p = (void *)n;
    return ok;
}

/* Address and row stride of a float32 tensor of at least `rows` rows of n_cols adjacent values on `device`. */
static int rows_of(PyObject *t, size_t n_cols, size_t rows, size_t device, float **p, size_t *ld) {
    if (!of_tensor(t, device, (void **)p)) return 0;
    PyObject *shape = PyObject_GetAttr(t, s_shape);
    if (!shape) { PyErr_Clear(); return 0; }
    PyObject *stride = PyObject_CallMethodNoArgs(t, s_stride);
    if (!stride) { PyErr_Clear(); Py_DECREF(shape); return 0; }
    size_t n0 = 0, n1 = 0, s0 = 0, s1 = 0;
    const int ok = PyTuple_Check(shape) && PyTuple_Check(stride) && PyTuple_GET_SIZE(shape) == 2 && PyTuple_GET_SIZE(stride) == 2 &&
                   number(PyTuple_GET_ITEM(shape, 0), &n0) && number(PyTuple_GET_ITEM(shape, 1), &n1) &&
                   number(PyTuple_GET_ITEM(stride, 0), &s0) && number(PyTuple_GET_ITEM(stride, 1), &s1) && n0 >= rows && n1 >= n_cols &&
                   (s1 == 1 || n1 <= 1);
    Py_DECREF(shape);
    Py_DECREF(stride);
    *ld = n0 > 1 || s0 > n_cols ? s0 : n_cols;
    return ok;
}

static int vector_of(PyObject *t, size_t n, size_t device, float **p) {
    if (!of_tensor(t, device, (void **)p)) return 0;
    PyObject *shape = PyObject_GetAttr(t, s_shape);
    if (!shape) { PyErr_Clear(); return 0; }
    PyObject *stride = PyObject_CallMethodNoArgs(t, s_stride);
    if (!stride) { PyErr_Clear(); Py_DECREF(shape); return 0; }
    size_t n0 = 0, s0 = 0;
    const int ok = PyTuple_Check(shape) && PyTuple_Check(stride) && PyTuple_GET_SIZE(shape) == 1 && PyTuple_GET_SIZE(stride) == 1 &&
                   number(PyTuple_GET_ITEM(shape, 0), &n0) && number(PyTuple_GET_ITEM(stride, 0), &s0) && n0 >= n && (s0 == 1 || n0 <= 1);
    Py_DECREF(shape);
    Py_DECREF(stride);
    return ok;
}

/* The stream given, or the device's current one. */
static int stream_of(PyObject *stream, PyObject *device, void **out) {
    PyObject *v = stream == Py_None ? PyObject_CallOneArg(g_raw_stream, device) : PyObject_GetAttr(stream, s_cuda_stream);
    if (!v) { PyErr_Clear(); return 0; }
    size_t n;
    const int ok = number(v, &n);
    Py_DECREF(v);
    *out = (void *)n;
    return ok;
}

/* quantize(act, device, n_cols, x, seq_len, stream) */
static PyObject *quantize(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    size_t h, dev, cols, seq, ld;
    float *x;
    void *st;
    if (n != 6 || !number(a[0], &h) || !number(a[1], &dev) || !number(a[2], &cols) || !number(a[4], &seq) ||
        !rows_of(a[3], cols, seq, dev, &x, &ld) || !stream_of(a[5], a[1], &st))
        Py_RETURN_NONE;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f_quantize((void *)h, x, ld, seq, st);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

/* add_rms_norm(act, device, n_cols, x, residual or None, weight, eps, seq_len, sum or None, stream) */
static PyObject *add_rms_norm(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    size_t h, dev, cols, seq, ld, ld_r, ld_s = 0;
    float *x, *r = NULL, *w, *s = NULL;
    void *st;
    if (n != 10 || !number(a[0], &h) || !number(a[1], &dev) || !number(a[2], &cols) || !number(a[7], &seq) || !PyFloat_Check(a[6]) ||
        !rows_of(a[3], cols, seq, dev, &x, &ld) || !vector_of(a[5], cols, dev, &w))
        Py_RETURN_NONE;
    if (a[4] != Py_None && (!rows_of(a[4], cols, seq, dev, &r, &ld_r) || (ld_r != ld && seq > 1))) Py_RETURN_NONE;
    if (a[8] != Py_None && !rows_of(a[8], cols, seq, dev, &s, &ld_s)) Py_RETURN_NONE;
    if (!stream_of(a[9], a[1], &st)) Py_RETURN_NONE;
    if (s && seq <= 1) ld_s = ld;
    const float eps = (float)PyFloat_AS_DOUBLE(a[6]);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f_norm((void *)h, x, r, ld, w, eps, seq, s, ld_s, st);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

/* silu_mul(act, device, n_cols, gate, up, seq_len, stream) */
static PyObject *silu_mul(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    size_t h, dev, cols, seq, ld, ld_u;
    float *g, *u;
    void *st;
    if (n != 7 || !number(a[0], &h) || !number(a[1], &dev) || !number(a[2], &cols) || !number(a[5], &seq) ||
        !rows_of(a[3], cols, seq, dev, &g, &ld) || !rows_of(a[4], cols, seq, dev, &u, &ld_u) || (ld_u != ld && seq > 1) ||
        !stream_of(a[6], a[1], &st))
        Py_RETURN_NONE;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f_silu((void *)h, g, u, ld, seq, st);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

/* dequantize(act, device, n_cols, out, seq_len, stream) */
static PyObject *dequantize(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    size_t h, dev, cols, seq, ld;
    float *o;
    void *st;
    if (n != 6 || !number(a[0], &h) || !number(a[1], &dev) || !number(a[2], &cols) || !number(a[4], &seq) ||
        !rows_of(a[3], cols, seq, dev, &o, &ld) || !stream_of(a[5], a[1], &st))
        Py_RETURN_NONE;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f_dequantize((void *)h, o, ld, seq, st);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

/* matmul(weight, act, device, n_rows, seq_len, out, accumulate, stream) */
static PyObject *matmul(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    size_t w, h, dev, rows, seq, ld;
    float *o;
    void *st;
    if (n != 8 || !number(a[0], &w) || !number(a[1], &h) || !number(a[2], &dev) || !number(a[3], &rows) || !number(a[4], &seq) ||
        !rows_of(a[5], rows, seq, dev, &o, &ld) || !stream_of(a[7], a[2], &st))
        Py_RETURN_NONE;
    const int acc = PyObject_IsTrue(a[6]);
    if (acc < 0) { PyErr_Clear(); Py_RETURN_NONE; }
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f_matmul((void *)w, (void *)h, seq, o, ld, acc, st);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

/* bind(torch.float32, raw_stream, addresses of quantize, add_rms_norm, silu_mul, dequantize, matmul) */
static PyObject *bind(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    size_t p[5];
    int ok = n == 7;
    for (int i = 0; ok && i < 5; i++) ok = number(a[2 + i], &p[i]) && p[i] != 0;
    if (!ok) {
        PyErr_SetString(PyExc_TypeError, "bind(dtype, raw_stream, five addresses)");
        return NULL;
    }
    f_quantize = (quantize_fn)p[0];
    f_norm = (norm_fn)p[1];
    f_silu = (silu_fn)p[2];
    f_dequantize = (dequantize_fn)p[3];
    f_matmul = (matmul_fn)p[4];
    Py_INCREF(a[0]);
    Py_XSETREF(g_f32, a[0]);
    Py_INCREF(a[1]);
    Py_XSETREF(g_raw_stream, a[1]);
    Py_RETURN_NONE;
}

static PyMethodDef methods[] = {{"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, NULL},
                                {"quantize", (PyCFunction)(void (*)(void))quantize, METH_FASTCALL, NULL},
                                {"add_rms_norm", (PyCFunction)(void (*)(void))add_rms_norm, METH_FASTCALL, NULL},
                                {"silu_mul", (PyCFunction)(void (*)(void))silu_mul, METH_FASTCALL, NULL},
                                {"dequantize", (PyCFunction)(void (*)(void))dequantize, METH_FASTCALL, NULL},
                                {"matmul", (PyCFunction)(void (*)(void))matmul, METH_FASTCALL, NULL},
                                {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_pycall", "Checked calls of the 8-bit linear path.", -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__pycall(void) {
    s_dtype = PyUnicode_InternFromString("dtype");
    s_shape = PyUnicode_InternFromString("shape");
    s_stride = PyUnicode_InternFromString("stride");
    s_data_ptr = PyUnicode_InternFromString("data_ptr");
    s_get_device = PyUnicode_InternFromString("get_device");
    s_cuda_stream = PyUnicode_InternFromString("cuda_stream");
    if (!s_dtype || !s_shape || !s_stride || !s_data_ptr || !s_get_device || !s_cuda_stream) return NULL;
    return PyModule_Create(&module);
}
