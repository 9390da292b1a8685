/* The layer operators for Python without ctypes: a call costs about 0.5 us in place of 3, which is what a decode step's smallest operators
 * take on the GPU.  The functions are the C ABI's (include/w4a8_b200.h), found in the library that the package has loaded (bind); arguments in its order.  A
 * pointer is a number, None, or a tensor (its data_ptr()), which has to lie on the current GPU: a kernel would follow a pointer to host memory, or to another
 * GPU's, to a fault.  A struct is a ctypes Structure, whose _gpu says where the tensors behind it lie; a stream is a number, an object with a cuda_stream, or None: what the two functions given to
 * streams() say is torch's current one.  Each returns the status code. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <limits.h>
typedef struct w4a8_arena w4a8_arena;
#include "../../include/w4a8_b200.h"

static PyObject *data_ptr_name, *cuda_stream_name, *is_cuda_name, *get_device_name, *gpu_name;
static PyObject *current_device, *current_stream;         /* of torch: device(), raw stream(device) */
static int gpus;                                          /* 0: nothing can be launched, and tensors may lie anywhere */
/* The tensor type's own C functions behind is_cuda and data_ptr(), called without a look-up: 0.1 us less for a call of five tensors. */
static PyTypeObject *tensor_type;
static getter tensor_is_cuda;
static void *tensor_is_cuda_closure;
static PyCFunction tensor_data_ptr;

/* Whether a tensor lies on the current GPU; which one that is, is asked for only where there are several. */
static int on_gpu(PyObject *o) {
    if (gpus == 0) return 1;
    PyObject *there = Py_TYPE(o) == tensor_type ? tensor_is_cuda(o, tensor_is_cuda_closure) : PyObject_GetAttr(o, is_cuda_name);
    if (!there) return 0;
    const int yes = there == Py_True;
    Py_DECREF(there);
    if (!yes) {
        PyErr_SetString(PyExc_ValueError, "a tensor that is not on a GPU");
        return 0;
    }
    if (gpus == 1) return 1;
    PyObject *its = PyObject_CallMethodNoArgs(o, get_device_name), *now = its ? PyObject_CallNoArgs(current_device) : NULL;
    const int same = now ? PyObject_RichCompareBool(its, now, Py_EQ) : -1;
    if (same == 0) PyErr_Format(PyExc_ValueError, "a tensor on GPU %S, the current one is %S", its, now);
    Py_XDECREF(its);
    Py_XDECREF(now);
    return same == 1;
}
/* Each conversion does nothing once one before it has failed. */
static void *as_pointer(PyObject *o, int *ok) {
    if (!*ok || o == Py_None) return NULL;
    if (PyLong_Check(o)) {
        void *p = PyLong_AsVoidPtr(o);
        if (!p && PyErr_Occurred()) *ok = 0;
        return p;
    }
    PyObject *n = !on_gpu(o) ? NULL : Py_TYPE(o) == tensor_type ? tensor_data_ptr(o, NULL) : PyObject_CallMethodNoArgs(o, data_ptr_name);
    if (!n) { *ok = 0; return NULL; }
    void *p = PyLong_AsVoidPtr(n);
    if (!p && PyErr_Occurred()) *ok = 0;
    Py_DECREF(n);
    return p;
}
static void *as_stream(PyObject *o, int *ok) {
    if (!*ok) return NULL;
    if (PyLong_Check(o)) return as_pointer(o, ok);
    PyObject *n = NULL;
    if (o != Py_None) n = PyObject_GetAttr(o, cuda_stream_name);
    else if (!current_stream) PyErr_SetString(PyExc_RuntimeError, "no current stream: streams() has not been called");
    else {
        PyObject *device = PyObject_CallNoArgs(current_device);
        if (device) {
            n = PyObject_CallOneArg(current_stream, device);
            Py_DECREF(device);
        }
    }
    if (!n) { *ok = 0; return NULL; }
    void *p = PyLong_AsVoidPtr(n);
    if (!p && PyErr_Occurred()) *ok = 0;
    Py_DECREF(n);
    return p;
}
static int64_t as_int64(PyObject *o, int *ok) {
    if (!*ok) return 0;
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) *ok = 0;
    return v;
}
static int as_int(PyObject *o, int *ok) {
    const int64_t v = as_int64(o, ok);
    if (v < INT_MIN || v > INT_MAX) {
        if (*ok) PyErr_Format(PyExc_OverflowError, "%lld does not fit 32 bits", (long long)v);
        *ok = 0;
    }
    return (int)v;
}
/* Whether what a struct points to lies on the current GPU: its _gpu, if it has one that is not None. */
static int struct_on_gpu(PyObject *o) {
    PyObject *its = PyObject_GetAttr(o, gpu_name);
    if (!its) {
        if (!PyErr_ExceptionMatches(PyExc_AttributeError)) return 0;
        PyErr_Clear();
        return 1;
    }
    int same = its == Py_None;
    if (!same) {
        PyObject *now = PyObject_CallNoArgs(current_device);
        same = now ? PyObject_RichCompareBool(its, now, Py_EQ) : -1;
        if (same == 0) PyErr_Format(PyExc_ValueError, "a struct of tensors on GPU %S, the current one is %S", its, now);
        Py_XDECREF(now);
    }
    Py_DECREF(its);
    return same == 1;
}
/* A struct's memory: it outlives the call, in which the library reads it. */
static const void *as_struct(PyObject *o, size_t size, int *ok) {
    Py_buffer view;
    if (!*ok) return NULL;
    if (gpus > 1 && !struct_on_gpu(o)) { *ok = 0; return NULL; }
    if (PyObject_GetBuffer(o, &view, PyBUF_SIMPLE) != 0) { *ok = 0; return NULL; }
    const void *p = view.buf;
    if ((size_t)view.len != size) {
        PyErr_Format(PyExc_TypeError, "a struct of %zu bytes, not %zd", size, view.len);
        *ok = 0;
    }
    PyBuffer_Release(&view);
    return p;
}
static int count(Py_ssize_t n, Py_ssize_t want) {
    if (n == want) return 1;
    PyErr_Format(PyExc_TypeError, "%zd arguments, %zd expected", n, want);
    return 0;
}

static __typeof__(&w4a8_add_norm) f_add_norm;
static __typeof__(&w4a8_rope_qk) f_rope_qk;
static __typeof__(&w4a8_moe_route) f_moe_route;
static __typeof__(&w4a8_quantize_rows_q8) f_quantize_rows_q8;
static __typeof__(&w4a8_gemm_w8a8) f_gemm_w8a8;
static __typeof__(&w4a8_linear_w8a8) f_linear_w8a8;

#define P(i) as_pointer(a[i], &ok)
#define I(i) as_int(a[i], &ok)
#define L(i) as_int64(a[i], &ok)
/* arguments are converted one after the other before the call, which is made only if all could be */
#define ENTRY(name, arguments)                                                       \
    static PyObject *name(PyObject *self, PyObject *const *a, Py_ssize_t n) {        \
        int ok = 1;                                                                  \
        if (!count(n, arguments)) return NULL;
#define CALL(name, ...)                                                              \
        if (!ok) return NULL;                                                        \
        return PyLong_FromLong(f_##name(__VA_ARGS__));                               \
    }

ENTRY(add_norm, 15)
        const w4a8_norm *norm = as_struct(a[0], sizeof(w4a8_norm), &ok); const void *h = P(1); const int64_t ldh = L(2); const void *y = P(3); const int64_t ldy = L(4);
        void *ho = P(5); const int64_t ldo = L(6); void *no = P(7); const int64_t ldn = L(8); int8_t *xq = P(9); float *xs = P(10); int32_t *xsum = P(11);
        const int group = I(12), S = I(13); void *stream = as_stream(a[14], &ok);
    CALL(add_norm, norm, h, ldh, y, ldy, ho, ldo, no, ldn, xq, xs, xsum, group, S, stream)
ENTRY(rope_qk, 15)
        const w4a8_rope *rope = as_struct(a[0], sizeof(w4a8_rope), &ok); const void *q = P(1); const int64_t ldq = L(2); const int hq = I(3); const void *k = P(4);
        const int64_t ldk = L(5); const int hk = I(6); const int32_t *position = P(7); const int T = I(8); void *qo = P(9); const int64_t ldqo = L(10); void *ko = P(11);
        const int64_t ldko = L(12); const int dtype = I(13); void *stream = as_stream(a[14], &ok);
    CALL(rope_qk, rope, q, ldq, hq, k, ldk, hk, position, T, qo, ldqo, ko, ldko, dtype, stream)
ENTRY(moe_route, 8)
        const w4a8_router *router = as_struct(a[0], sizeof(w4a8_router), &ok); const void *logits = P(1); const int64_t ld = L(2); const int S = I(3), dtype = I(4);
        int32_t *idx = P(5); float *weight = P(6); void *stream = as_stream(a[7], &ok);
    CALL(moe_route, router, logits, ld, S, dtype, idx, weight, stream)
ENTRY(quantize_rows_q8, 8)
        const void *x = P(0); const int64_t ldx = L(1); const int S = I(2), K = I(3), dtype = I(4); int8_t *xq = P(5); float *xs = P(6); void *stream = as_stream(a[7], &ok);
    CALL(quantize_rows_q8, x, ldx, S, K, dtype, xq, xs, stream)
ENTRY(gemm_w8a8, 12)
        const int8_t *xq = P(0); const float *xs = P(1); const int8_t *wq = P(2); const float *ws = P(3); const float *bias = P(4); void *Y = P(5); const int64_t ldy = L(6);
        const int M = I(7), N = I(8), K = I(9), dtype = I(10); void *stream = as_stream(a[11], &ok);
    CALL(gemm_w8a8, xq, xs, wq, ws, bias, Y, ldy, M, N, K, dtype, stream)
ENTRY(linear_w8a8, 16)
        const void *x = P(0); const int64_t ldx = L(1); int8_t *xq = P(2); float *xs = P(3); const int8_t *wq = P(4); const float *ws = P(5); const float *bias = P(6);
        void *Y = P(7); const int64_t ldy = L(8); const int S = I(9), N = I(10), K = I(11), xd = I(12), yd = I(13), skip = I(14); void *stream = as_stream(a[15], &ok);
    CALL(linear_w8a8, x, ldx, xq, xs, wq, ws, bias, Y, ldy, S, N, K, xd, yd, skip, stream)

/* bind(addresses of the six functions, in the order of the table below) */
static PyObject *bind(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    int ok = 1;
    if (!count(n, 6)) return NULL;
    void *p[6];
    for (int i = 0; i < 6; i++) p[i] = P(i);
    if (!ok) return NULL;
    f_add_norm = (__typeof__(f_add_norm))p[0];
    f_rope_qk = (__typeof__(f_rope_qk))p[1];
    f_moe_route = (__typeof__(f_moe_route))p[2];
    f_quantize_rows_q8 = (__typeof__(f_quantize_rows_q8))p[3];
    f_gemm_w8a8 = (__typeof__(f_gemm_w8a8))p[4];
    f_linear_w8a8 = (__typeof__(f_linear_w8a8))p[5];
    Py_RETURN_NONE;
}

/* What the two names are in a type: a getter and a method without arguments, or it is looked at as any object is. */
static void tensors_of(PyObject *type) {
    tensor_type = NULL;
    if (!PyType_Check(type)) return;
    PyObject *is_cuda = PyObject_GetAttr(type, is_cuda_name), *data_ptr = PyObject_GetAttr(type, data_ptr_name);
    if (is_cuda && data_ptr && Py_IS_TYPE(is_cuda, &PyGetSetDescr_Type) && Py_IS_TYPE(data_ptr, &PyMethodDescr_Type) &&
        ((PyMethodDescrObject *)data_ptr)->d_method->ml_flags == METH_NOARGS) {
        tensor_is_cuda = ((PyGetSetDescrObject *)is_cuda)->d_getset->get;
        tensor_is_cuda_closure = ((PyGetSetDescrObject *)is_cuda)->d_getset->closure;
        tensor_data_ptr = ((PyMethodDescrObject *)data_ptr)->d_method->ml_meth;
        Py_INCREF(type);                                  /* for good: the functions are the type's */
        tensor_type = (PyTypeObject *)type;
    }
    PyErr_Clear();
    Py_XDECREF(is_cuda);
    Py_XDECREF(data_ptr);
}

/* streams(device(), stream(device), number of GPUs, type of tensors) */
static PyObject *streams(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    int ok = 1;
    if (!count(n, 4)) return NULL;
    const int there = I(2);
    if (!ok) return NULL;
    gpus = there;
    tensors_of(a[3]);
    Py_INCREF(a[0]);
    Py_INCREF(a[1]);
    Py_XSETREF(current_device, a[0]);
    Py_XSETREF(current_stream, a[1]);
    Py_RETURN_NONE;
}

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, NULL}
static PyMethodDef methods[] = {METHOD(bind), METHOD(streams), METHOD(add_norm), METHOD(rope_qk), METHOD(moe_route), METHOD(quantize_rows_q8), METHOD(gemm_w8a8), METHOD(linear_w8a8), {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", NULL, -1, methods};
PyMODINIT_FUNC PyInit__binding(void) {
    data_ptr_name = PyUnicode_InternFromString("data_ptr");
    cuda_stream_name = PyUnicode_InternFromString("cuda_stream");
    is_cuda_name = PyUnicode_InternFromString("is_cuda");
    get_device_name = PyUnicode_InternFromString("get_device");
    gpu_name = PyUnicode_InternFromString("_gpu");
    return data_ptr_name && cuda_stream_name && is_cuda_name && get_device_name && gpu_name ? PyModule_Create(&module) : NULL;
}
