// Python's way into the calls of the 8-bit linear path that a decode loop makes for every token.  Through ctypes and checks
// in Python, two such calls cost more host time (about 4 us) than their kernels run; here the checks of the usual case -
// two-dimensional float32 CUDA tensors on the handle's device - read the tensors directly and cost next to nothing.
// Anything else (another shape, type or device, a missing tensor) returns None, and api.py's own checks then refuse or serve
// it; a number is the call's status code.  The C entry points are those of the library that ctypes loaded; like ctypes,
// the calls let other Python threads run meanwhile (a full launch queue blocks).
#include <torch/csrc/autograd/python_variable.h>

#include <c10/cuda/CUDAStream.h>

namespace {

typedef int (*quantize_fn)(void*, const float*, size_t, size_t, void*);
typedef int (*norm_fn)(void*, const float*, const float*, size_t, const float*, float, size_t, float*, size_t, void*);
typedef int (*silu_fn)(void*, const float*, const float*, size_t, size_t, void*);
typedef int (*dequantize_fn)(void*, float*, size_t, size_t, void*);
typedef int (*matmul_fn)(void*, void*, size_t, float*, size_t, int, void*);

quantize_fn f_quantize;
norm_fn f_norm;
silu_fn f_silu;
dequantize_fn f_dequantize;
matmul_fn f_matmul;
PyObject* s_cuda_stream;

// A non-negative integer; false if it is none.
bool number(PyObject* o, size_t* out) {
    if (!PyLong_Check(o)) return false;
    *out = PyLong_AsSize_t(o);
    if (*out == (size_t)-1 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}
// A device index (-1: the host's memory, which only tests hand in).
bool device_of(PyObject* o, int64_t* out) {
    if (!PyLong_Check(o)) return false;
    *out = PyLong_AsLongLong(o);
    if (*out == -1 && PyErr_Occurred()) PyErr_Clear();
    return true;
}

const at::Tensor* tensor_of(PyObject* o, int64_t device) {
    if (!THPVariable_Check(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || t.layout() != at::kStrided || t.scalar_type() != at::kFloat) return nullptr;
    if (device < 0 ? !t.is_cpu() : !t.is_cuda() || t.get_device() != device) return nullptr;
    return &t;
}

// Address and row stride of a float32 tensor of at least `rows` rows of n_cols adjacent values on `device`.
bool rows_of(PyObject* o, size_t n_cols, size_t rows, int64_t device, float** p, size_t* ld) {
    const at::Tensor* t = tensor_of(o, device);
    if (!t || t->dim() != 2) return false;
    const int64_t n0 = t->size(0), n1 = t->size(1), s0 = t->stride(0), s1 = t->stride(1);
    if ((uint64_t)n0 < rows || (uint64_t)n1 < n_cols || (s1 != 1 && n1 > 1)) return false;
    *ld = n0 > 1 || (uint64_t)s0 > n_cols ? (size_t)s0 : n_cols;
    *p = (float*)t->data_ptr();
    return true;
}

bool vector_of(PyObject* o, size_t n, int64_t device, float** p) {
    const at::Tensor* t = tensor_of(o, device);
    if (!t || t->dim() != 1 || (uint64_t)t->size(0) < n || (t->stride(0) != 1 && t->size(0) > 1)) return false;
    *p = (float*)t->data_ptr();
    return true;
}

// The stream given, or the device's current one.
bool stream_of(PyObject* stream, int64_t device, void** out) {
    if (stream == Py_None) {
        if (device < 0) return false;
        *out = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
        return true;
    }
    PyObject* v = PyObject_GetAttr(stream, s_cuda_stream);
    size_t n = 0;
    const bool ok = v && number(v, &n);
    if (!v) PyErr_Clear();
    Py_XDECREF(v);
    *out = (void*)n;
    return ok;
}

// The body of a call: nothing thrown by torch crosses into Python's C code.
template <typename F>
PyObject* guarded(F body) {
    try {
        return body();
    } catch (...) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
}
template <typename F>
PyObject* call(F f) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f();
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

// quantize(act, device, n_cols, x, seq_len, stream)
PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        size_t h, cols, seq, ld;
        int64_t dev;
        float* x;
        void* st;
        if (n != 6 || !number(a[0], &h) || !device_of(a[1], &dev) || !number(a[2], &cols) || !number(a[4], &seq) ||
            !rows_of(a[3], cols, seq, dev, &x, &ld) || !stream_of(a[5], dev, &st))
            Py_RETURN_NONE;
        return call([&] { return f_quantize((void*)h, x, ld, seq, st); });
    });
}

// add_rms_norm(act, device, n_cols, x, residual or None, weight, eps, seq_len, sum or None, stream)
PyObject* add_rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        size_t h, cols, seq, ld, ld_r, ld_s = 0;
        int64_t dev;
        float *x, *r = nullptr, *w, *s = nullptr;
        void* st;
        if (n != 10 || !number(a[0], &h) || !device_of(a[1], &dev) || !number(a[2], &cols) || !number(a[7], &seq) || !PyFloat_Check(a[6]) ||
            !rows_of(a[3], cols, seq, dev, &x, &ld) || !vector_of(a[5], cols, dev, &w))
            Py_RETURN_NONE;
        if (a[4] != Py_None && (!rows_of(a[4], cols, seq, dev, &r, &ld_r) || (ld_r != ld && seq > 1))) Py_RETURN_NONE;
        if (a[8] != Py_None && !rows_of(a[8], cols, seq, dev, &s, &ld_s)) Py_RETURN_NONE;
        if (!stream_of(a[9], dev, &st)) Py_RETURN_NONE;
        if (s && seq <= 1) ld_s = ld;
        const float eps = (float)PyFloat_AS_DOUBLE(a[6]);
        return call([&] { return f_norm((void*)h, x, r, ld, w, eps, seq, s, ld_s, st); });
    });
}

// silu_mul(act, device, n_cols, gate, up, seq_len, stream)
PyObject* silu_mul(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        size_t h, cols, seq, ld, ld_u;
        int64_t dev;
        float *g, *u;
        void* st;
        if (n != 7 || !number(a[0], &h) || !device_of(a[1], &dev) || !number(a[2], &cols) || !number(a[5], &seq) ||
            !rows_of(a[3], cols, seq, dev, &g, &ld) || !rows_of(a[4], cols, seq, dev, &u, &ld_u) || (ld_u != ld && seq > 1) ||
            !stream_of(a[6], dev, &st))
            Py_RETURN_NONE;
        return call([&] { return f_silu((void*)h, g, u, ld, seq, st); });
    });
}

// dequantize(act, device, n_cols, out, seq_len, stream)
PyObject* dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        size_t h, cols, seq, ld;
        int64_t dev;
        float* o;
        void* st;
        if (n != 6 || !number(a[0], &h) || !device_of(a[1], &dev) || !number(a[2], &cols) || !number(a[4], &seq) ||
            !rows_of(a[3], cols, seq, dev, &o, &ld) || !stream_of(a[5], dev, &st))
            Py_RETURN_NONE;
        return call([&] { return f_dequantize((void*)h, o, ld, seq, st); });
    });
}

// matmul(weight, act, device, n_rows, seq_len, out, accumulate, stream)
PyObject* matmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        size_t w, h, rows, seq, ld;
        int64_t dev;
        float* o;
        void* st;
        if (n != 8 || !number(a[0], &w) || !number(a[1], &h) || !device_of(a[2], &dev) || !number(a[3], &rows) || !number(a[4], &seq) ||
            !rows_of(a[5], rows, seq, dev, &o, &ld) || !stream_of(a[7], dev, &st))
            Py_RETURN_NONE;
        const int acc = PyObject_IsTrue(a[6]);
        if (acc < 0) {
            PyErr_Clear();
            Py_RETURN_NONE;
        }
        return call([&] { return f_matmul((void*)w, (void*)h, seq, o, ld, acc, st); });
    });
}

// bind(addresses of quantize, add_rms_norm, silu_mul, dequantize, matmul)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    size_t p[5];
    bool ok = n == 5;
    for (int i = 0; ok && i < 5; i++) ok = number(a[i], &p[i]) && p[i] != 0;
    if (!ok) {
        PyErr_SetString(PyExc_TypeError, "bind(five addresses)");
        return nullptr;
    }
    f_quantize = (quantize_fn)p[0];
    f_norm = (norm_fn)p[1];
    f_silu = (silu_fn)p[2];
    f_dequantize = (dequantize_fn)p[3];
    f_matmul = (matmul_fn)p[4];
    Py_RETURN_NONE;
}

#define HB_METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {HB_METHOD(bind),       HB_METHOD(quantize), HB_METHOD(add_rms_norm), HB_METHOD(silu_mul),
                         HB_METHOD(dequantize), HB_METHOD(matmul),   {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_pycall", "Checked calls of the 8-bit linear path.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__pycall(void) {
    s_cuda_stream = PyUnicode_InternFromString("cuda_stream");
    PyObject* m = s_cuda_stream ? PyModule_Create(&module) : nullptr;
    // the interpreter and torch whose headers were read above (build.py); api.py compares
    if (m && PyModule_AddStringConstant(m, "built_for", HB_BUILT_FOR) != 0) {
        Py_DECREF(m);
        m = nullptr;
    }
    return m;
}
