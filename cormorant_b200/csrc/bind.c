/* bind.c -- the Python side of the block-scaled 8-bit floating-point entries (cormorant_b200._bind).
 *
 * A decode step makes many small calls, and looking at the tensors of one in Python took longer than
 * the kernel behind it (a matrix product of one token: 11 us of Python before a 7 us kernel).  Each
 * function here takes the arguments of its Python entry by position, looks at the tensors through
 * their Python attributes, and calls the C ABI; it returns the C status.  What is checked and raised:
 * see `matrix` and `kernels.py`.  The C ABI's addresses come from setup().
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>

#include "cormorant_cuda.h"

/* ---- the C ABI, by address ------------------------------------------------------------------ */
static struct {
    int (*device)(void);
    __typeof__(&cm_quant_fp8) quant;
    __typeof__(&cm_quant_fp8_async) quant_async;
    __typeof__(&cm_rmsnorm_fp8) norm;
    __typeof__(&cm_rmsnorm_fp8_async) norm_async;
    __typeof__(&cm_matmul_fp8) matmul;
    __typeof__(&cm_matmul_fp8_async) matmul_async;
    __typeof__(&cm_matmul_fp8_grouped) grouped;
    __typeof__(&cm_matmul_fp8_grouped_async) grouped_async;
} api;

/* ---- element types --------------------------------------------------------------------------- */
enum { D_I16, D_F32, D_F16, D_BF16, D_E4M3, D_E5M2, D_U8, D_I32, D_COUNT };
static const char* const kDtypeNames[D_COUNT] = {"int16", "float32", "float16", "bfloat16", "float8_e4m3fn", "float8_e5m2", "uint8", "int32"};
static PyObject* dtypes[D_COUNT];

enum { K_TYPE, K_FORMAT, K_SCALE, K_OFFSETS };   /* what an operand may hold */
#define ANY (-1)                                   /* a raw address, or bytes of either format */

static PyObject *s_data_ptr, *s_stride, *s_shape, *s_dtype, *s_get_device, *s_cuda_stream;

static int find_dtypes(void) {
    PyObject* torch = PyImport_ImportModule("torch");      /* a tensor is at hand: it is loaded */
    if (!torch) return -1;
    for (int i = D_COUNT - 1; i >= 0; --i) {               /* the first one, which says that all are there, last */
        dtypes[i] = PyObject_GetAttrString(torch, kDtypeNames[i]);
        if (!dtypes[i]) { Py_DECREF(torch); return -1; }
    }
    Py_DECREF(torch);
    return 0;
}

static int code_of(int dtype, int kind) {
    switch (kind) {
        case K_TYPE: return dtype <= D_BF16 ? dtype : -2;             /* CM_T_* in this order */
        case K_FORMAT: return dtype == D_E4M3 ? 0 : dtype == D_E5M2 ? 1 : dtype == D_U8 ? ANY : -2;
        case K_SCALE: return dtype == D_F32 ? 0 : -2;
        default: return dtype == D_I32 ? 0 : -2;
    }
}

/* ---- numbers ----------------------------------------------------------------------------------- */
static int as_u64(PyObject* o, uint64_t* v) {
    *v = PyLong_AsUnsignedLongLong(o);
    if (*v != (uint64_t)-1 || !PyErr_Occurred()) return 0;
    if (!PyErr_ExceptionMatches(PyExc_TypeError)) return -1;
    PyErr_Clear();                                          /* an integer of another kind */
    PyObject* i = PyNumber_Index(o);
    if (!i) return -1;
    *v = PyLong_AsUnsignedLongLong(i);
    Py_DECREF(i);
    return *v == (uint64_t)-1 && PyErr_Occurred() ? -1 : 0;
}

static int as_size(PyObject* o, const char* what, unsigned* v) {
    uint64_t u;
    if (as_u64(o, &u)) return -1;
    if (u > 0xffffffffull) { PyErr_Format(PyExc_ValueError, "%s: %llu does not fit 32 bits", what, (unsigned long long)u); return -1; }
    *v = (unsigned)u;
    return 0;
}

/* an int64 of a shape or stride tuple; negative ones do not occur in torch */
static uint64_t item(PyObject* tuple, Py_ssize_t i) { return (uint64_t)PyLong_AsLongLong(PyTuple_GET_ITEM(tuple, i)); }

static int call_u64(PyObject* o, PyObject* name, uint64_t* v) {
    PyObject* r = PyObject_CallMethodNoArgs(o, name);
    if (!r) return -1;
    const int rc = as_u64(r, v);
    Py_DECREF(r);
    return rc;
}

/* ---- operands ------------------------------------------------------------------------------------ */
typedef struct {
    void* p;
    uint64_t ld, bs;      /* row pitch, batch stride, in elements */
    int code;             /* element type or format, or ANY */
} Mat;

/* Elements from t's first one to its last. */
static uint64_t room_of(PyObject* shape, PyObject* stride) {
    uint64_t last = 0;
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(shape); ++i) {
        if (!item(shape, i)) return 0;
        last += (item(shape, i) - 1) * item(stride, i);
    }
    return last + 1;
}

/* The [batch][rows][cols] operand t: None, a raw address, or a CUDA tensor of the kind's types on
 * the library's device with contiguous rows.  A tensor of two or more dimensions has its own pitch
 * unless the pitch is given, one of three or more its own batch stride unless the batch stride is
 * given (the dimensions before the last two are one batch as far as their matrices lie an even stride
 * apart); what is missing is dense.  Nothing beyond a tensor's own last element is reached. */
static int matrix(PyObject* t, uint64_t rows, uint64_t cols, PyObject* ld, int kind, const char* what, uint64_t batch, PyObject* bs, Mat* m) {
    m->p = NULL; m->ld = m->bs = 0; m->code = ANY;
    if (t == Py_None) return 0;
    const int has_ld = ld && ld != Py_None, has_bs = bs && bs != Py_None;
    if (has_ld && as_u64(ld, &m->ld)) return -1;
    if (has_bs && as_u64(bs, &m->bs)) return -1;
    if (PyLong_Check(t)) {
        uint64_t a;
        if (as_u64(t, &a)) return -1;
        m->p = (void*)(uintptr_t)a;
        if (!has_ld) m->ld = cols;
        if (!has_bs) m->bs = rows * m->ld;
        return 0;
    }
    PyObject* r = PyObject_CallMethodNoArgs(t, s_get_device);
    if (!r) {
        if (!PyErr_ExceptionMatches(PyExc_AttributeError)) return -1;
        PyErr_Format(PyExc_TypeError, "%s: buffers must be CUDA tensors or device addresses", what);
        return -1;
    }
    const long dev = PyLong_AsLong(r);
    Py_DECREF(r);
    if (dev < 0) {
        PyErr_Clear();
        PyErr_Format(PyExc_TypeError, "%s: buffers must be CUDA tensors or device addresses", what);
        return -1;
    }
    const int own = api.device();
    if (own >= 0 && dev != own) {
        PyErr_Format(PyExc_ValueError, "%s: a tensor of cuda:%ld, but the library runs on cuda:%d", what, dev, own);
        return -1;
    }
    r = PyObject_GetAttr(t, s_dtype);
    if (!r) return -1;
    if (!dtypes[0] && find_dtypes()) { Py_DECREF(r); return -1; }
    int dtype = 0;
    while (dtype < D_COUNT && dtypes[dtype] != r) ++dtype;
    m->code = dtype < D_COUNT ? code_of(dtype, kind) : -2;
    if (m->code == -2) {
        PyErr_Format(PyExc_TypeError, "%s: a tensor of %R is not supported here", what, r);
        Py_DECREF(r);
        return -1;
    }
    Py_DECREF(r);
    uint64_t a;
    if (call_u64(t, s_data_ptr, &a)) return -1;
    m->p = (void*)(uintptr_t)a;
    PyObject* shape = PyObject_GetAttr(t, s_shape);
    PyObject* stride = shape ? PyObject_CallMethodNoArgs(t, s_stride) : NULL;
    int rc = -1;
    if (!stride) goto done;
    if (!PyTuple_Check(shape) || !PyTuple_Check(stride) || PyTuple_GET_SIZE(shape) != PyTuple_GET_SIZE(stride)) {
        PyErr_Format(PyExc_TypeError, "%s: not a tensor", what);
        goto done;
    }
    const Py_ssize_t nd = PyTuple_GET_SIZE(shape);
    if (nd && item(shape, nd - 1) > 1 && item(stride, nd - 1) != 1) {
        PyErr_Format(PyExc_ValueError, "%s: the elements of a row must be contiguous", what);
        goto done;
    }
    if (nd >= 2 && !has_ld) {
        if (item(shape, nd - 2) < rows || item(shape, nd - 1) < cols) {
            PyErr_Format(PyExc_ValueError, "%s: %R holds no %llu x %llu matrix", what, shape, (unsigned long long)rows, (unsigned long long)cols);
            goto done;
        }
        m->ld = item(stride, nd - 2);
        if (rows <= 1 && m->ld < cols) m->ld = cols;
    }
    if (!has_ld && nd < 2) m->ld = cols;
    if (!has_bs) {
        m->bs = rows * m->ld;
        if (nd >= 3) {                       /* its own, whether or not the pitch is given */
            uint64_t have = item(shape, nd - 3);
            m->bs = item(stride, nd - 3);
            for (Py_ssize_t i = nd - 4; i >= 0; --i) {
                if (item(shape, i) == 1) continue;
                if (have == 1) m->bs = item(stride, i);
                else if (item(stride, i) != have * m->bs) break;
                have *= item(shape, i);
            }
            if (have < batch) {
                PyErr_Format(PyExc_ValueError, "%s: %R holds fewer than %llu matrices an even stride apart", what, shape, (unsigned long long)batch);
                goto done;
            }
        }
    }
    if (nd >= 2 && !has_ld && (batch <= 1 || (nd >= 3 && !has_bs))) {        /* its shape has said that it is large enough */
        rc = 0;
        goto done;
    }
    if (rows && cols && batch) {
        const uint64_t room = room_of(shape, stride);
        if ((unsigned __int128)(batch - 1) * m->bs + (unsigned __int128)(rows - 1) * m->ld + cols > room) {
            PyErr_Format(PyExc_ValueError, "%s: the buffer is too short for %llu x %llu x %llu at pitch %llu", what, (unsigned long long)batch,
                         (unsigned long long)rows, (unsigned long long)cols, (unsigned long long)m->ld);
            goto done;
        }
    }
    rc = 0;
done:
    Py_XDECREF(shape);
    Py_XDECREF(stride);
    return rc;
}

/* An element type or format: the tensor's own, or the one given for a raw address or bytes. */
static int pick(const Mat* m, PyObject* given, int fallback, const char* what, unsigned* v) {
    unsigned want = 0;
    const int has = given != Py_None;
    if (has && as_size(given, what, &want)) return -1;
    if (m->code == ANY) {
        if (!has && fallback < 0) { PyErr_Format(PyExc_TypeError, "%s: a raw address needs its type", what); return -1; }
        *v = has ? want : (unsigned)fallback;
        return 0;
    }
    if (has && want != (unsigned)m->code) { PyErr_Format(PyExc_TypeError, "%s: the tensor's type is not the one given", what); return -1; }
    *v = (unsigned)m->code;
    return 0;
}

static int stream_of(PyObject* s, void** p) {
    uint64_t v;
    if (PyLong_Check(s)) {
        if (as_u64(s, &v)) return -1;
    } else {
        PyObject* r = PyObject_GetAttr(s, s_cuda_stream);
        if (!r) return -1;
        const int rc = as_u64(r, &v);
        Py_DECREF(r);
        if (rc) return -1;
    }
    *p = (void*)(uintptr_t)v;
    return 0;
}

static uint64_t blocks(uint64_t v) { return (v + 127) / 128; }

static int arguments(Py_ssize_t n, Py_ssize_t want) {
    if (!api.device) { PyErr_SetString(PyExc_RuntimeError, "_bind.setup has not been called"); return -1; }
    if (n != want) { PyErr_Format(PyExc_TypeError, "%zd arguments, %zd are wanted", n, want); return -1; }
    return 0;
}

#define TRY(x) do { if (x) return NULL; } while (0)
#define CALL(rc, stream, plain, twin)                        \
    do {                                                     \
        void* s_ = NULL;                                     \
        const int async_ = (stream) != Py_None;              \
        if (async_) TRY(stream_of(stream, &s_));             \
        Py_BEGIN_ALLOW_THREADS                               \
        rc = async_ ? twin : plain;                          \
        Py_END_ALLOW_THREADS                                 \
    } while (0)

/* x, q, scale, rows, cols, batch, ldx, ldq, lds, x_bs, q_bs, scale_bs, fmt, block_rows, x_type, stream */
static PyObject* quant_fp8(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    (void)self;
    TRY(arguments(n, 16));
    unsigned rows, cols, batch, block_rows, xt, qf;
    TRY(as_size(a[3], "rows", &rows) || as_size(a[4], "cols", &cols) || as_size(a[5], "batch", &batch) || as_size(a[13], "block_rows", &block_rows));
    const int wide = block_rows != 1;
    const uint64_t sr = wide ? blocks(rows) : blocks(cols), sc = wide ? blocks(cols) : rows;
    Mat x, q, s;
    TRY(matrix(a[0], rows, cols, a[6], K_TYPE, "x", batch, a[9], &x) || matrix(a[1], rows, cols, a[7], K_FORMAT, "q", batch, a[10], &q) ||
        matrix(a[2], sr, sc, a[8], K_SCALE, "scale", batch, a[11], &s) || pick(&x, a[14], -1, "x", &xt) || pick(&q, a[12], CM_F8_E4M3, "q", &qf));
    int rc;
#define ARGS x.p, xt, q.p, s.p, rows, cols, batch, x.ld, q.ld, s.ld, x.bs, q.bs, s.bs, qf, block_rows
    CALL(rc, a[15], api.quant(ARGS), api.quant_async(ARGS, s_));
#undef ARGS
    return PyLong_FromLong(rc);
}

/* x, weight, q, scale, rows, cols, eps, resid, resid_out, y, ldx, ldr, ldo, ldy, ldq, lds, fmt, x_type, weight_type, stream */
static PyObject* rmsnorm_fp8(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    (void)self;
    TRY(arguments(n, 20));
    unsigned rows, cols, xt, wt, qf;
    TRY(as_size(a[4], "rows", &rows) || as_size(a[5], "cols", &cols));
    const double eps = PyFloat_AsDouble(a[6]);
    if (eps == -1.0 && PyErr_Occurred()) return NULL;
    Mat x, w, q, s, r, o, y;
    TRY(matrix(a[0], rows, cols, a[10], K_TYPE, "x", 1, NULL, &x) || pick(&x, a[17], -1, "x", &xt) ||
        matrix(a[7], rows, cols, a[11], K_TYPE, "resid", 1, NULL, &r) || matrix(a[8], rows, cols, a[12], K_TYPE, "resid_out", 1, NULL, &o) ||
        matrix(a[9], rows, cols, a[13], K_TYPE, "y", 1, NULL, &y));
    if ((r.code != ANY && (unsigned)r.code != xt) || (o.code != ANY && (unsigned)o.code != xt) || (y.code != ANY && (unsigned)y.code != xt)) {
        PyErr_SetString(PyExc_TypeError, "resid, resid_out and y are of x's type");
        return NULL;
    }
    TRY(matrix(a[1], 1, cols, NULL, K_TYPE, "weight", 1, NULL, &w) || pick(&w, a[18], (int)xt, "weight", &wt) ||
        matrix(a[2], rows, cols, a[14], K_FORMAT, "q", 1, NULL, &q) || matrix(a[3], blocks(cols), rows, a[15], K_SCALE, "scale", 1, NULL, &s) ||
        pick(&q, a[16], CM_F8_E4M3, "q", &qf));
    int rc;
#define ARGS x.p, r.p, w.p, o.p, y.p, q.p, s.p, rows, cols, x.ld, r.ld, o.ld, y.ld, q.ld, s.ld, xt, wt, (float)eps, qf
    CALL(rc, a[19], api.norm(ARGS), api.norm_async(ARGS, s_));
#undef ARGS
    return PyLong_FromLong(rc);
}

/* a, a_scale, b, b_scale, c, n, k, m, lda, a_scale_ld, ldb, b_scale_ld, ldc, a_fmt, b_fmt, c_type, stream */
static PyObject* matmul_fp8(PyObject* self, PyObject* const* v, Py_ssize_t cnt) {
    (void)self;
    TRY(arguments(cnt, 17));
    unsigned n, k, m, af, bf, ct;
    TRY(as_size(v[5], "n", &n) || as_size(v[6], "k", &k) || as_size(v[7], "m", &m));
    Mat a, as, b, bs, c;
    TRY(matrix(v[0], n, k, v[8], K_FORMAT, "a", 1, NULL, &a) || matrix(v[2], m, k, v[10], K_FORMAT, "b", 1, NULL, &b) ||
        matrix(v[1], blocks(k), n, v[9], K_SCALE, "a_scale", 1, NULL, &as) || matrix(v[3], blocks(m), blocks(k), v[11], K_SCALE, "b_scale", 1, NULL, &bs) ||
        matrix(v[4], n, m, v[12], K_TYPE, "c", 1, NULL, &c) || pick(&a, v[13], CM_F8_E4M3, "a", &af) || pick(&b, v[14], CM_F8_E4M3, "b", &bf) ||
        pick(&c, v[15], -1, "c", &ct));
    int rc;
#define ARGS a.p, as.p, b.p, bs.p, c.p, n, k, m, a.ld, as.ld, b.ld, bs.ld, c.ld, af, bf, ct
    CALL(rc, v[16], api.matmul(ARGS), api.matmul_async(ARGS, s_));
#undef ARGS
    return PyLong_FromLong(rc);
}

/* a, a_scale, b, b_scale, c, offsets, groups, n, k, m, lda, a_scale_ld, ldb, b_scale_ld, b_gs, b_scale_gs, ldc,
 * a_fmt, b_fmt, c_type, stream */
static PyObject* matmul_fp8_grouped(PyObject* self, PyObject* const* v, Py_ssize_t cnt) {
    (void)self;
    TRY(arguments(cnt, 21));
    unsigned g, n, k, m, af, bf, ct;
    TRY(as_size(v[6], "groups", &g) || as_size(v[7], "n", &n) || as_size(v[8], "k", &k) || as_size(v[9], "m", &m));
    Mat a, as, b, bs, c, o;
    TRY(matrix(v[0], n, k, v[10], K_FORMAT, "a", 1, NULL, &a) || matrix(v[2], m, k, v[12], K_FORMAT, "b", g, v[14], &b) ||
        matrix(v[1], blocks(k), n, v[11], K_SCALE, "a_scale", 1, NULL, &as) || matrix(v[3], blocks(m), blocks(k), v[13], K_SCALE, "b_scale", g, v[15], &bs) ||
        matrix(v[4], n, m, v[16], K_TYPE, "c", 1, NULL, &c) || matrix(v[5], 1, (uint64_t)g + 1, NULL, K_OFFSETS, "offsets", 1, NULL, &o) ||
        pick(&a, v[17], CM_F8_E4M3, "a", &af) || pick(&b, v[18], CM_F8_E4M3, "b", &bf) || pick(&c, v[19], -1, "c", &ct));
    int rc;
#define ARGS a.p, as.p, b.p, bs.p, c.p, o.p, g, n, k, m, a.ld, as.ld, b.ld, bs.ld, b.bs, bs.bs, c.ld, af, bf, ct
    CALL(rc, v[20], api.grouped(ARGS), api.grouped_async(ARGS, s_));
#undef ARGS
    return PyLong_FromLong(rc);
}

/* setup(cm_device, cm_quant_fp8, its _async, cm_rmsnorm_fp8, .., cm_matmul_fp8, .., cm_matmul_fp8_grouped, ..): addresses */
static PyObject* setup(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    (void)self;
    if (n != 9) { PyErr_SetString(PyExc_TypeError, "setup: nine addresses are wanted"); return NULL; }
    uint64_t p[9];
    for (int i = 0; i < 9; ++i) TRY(as_u64(a[i], &p[i]));
    void** const f[9] = {(void**)&api.device, (void**)&api.quant, (void**)&api.quant_async, (void**)&api.norm, (void**)&api.norm_async,
                         (void**)&api.matmul, (void**)&api.matmul_async, (void**)&api.grouped, (void**)&api.grouped_async};
    for (int i = 0; i < 9; ++i) *f[i] = (void*)(uintptr_t)p[i];
    Py_RETURN_NONE;
}

static PyMethodDef methods[] = {
    {"setup", (PyCFunction)(void (*)(void))setup, METH_FASTCALL, NULL},
    {"quant_fp8", (PyCFunction)(void (*)(void))quant_fp8, METH_FASTCALL, NULL},
    {"rmsnorm_fp8", (PyCFunction)(void (*)(void))rmsnorm_fp8, METH_FASTCALL, NULL},
    {"matmul_fp8", (PyCFunction)(void (*)(void))matmul_fp8, METH_FASTCALL, NULL},
    {"matmul_fp8_grouped", (PyCFunction)(void (*)(void))matmul_fp8_grouped, METH_FASTCALL, NULL},
    {NULL, NULL, 0, NULL},
};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__bind(void) {
    static PyObject** const names[] = {&s_data_ptr, &s_stride, &s_shape, &s_dtype, &s_get_device, &s_cuda_stream};
    static const char* const text[] = {"data_ptr", "stride", "shape", "dtype", "get_device", "cuda_stream"};
    for (size_t i = 0; i < sizeof(names) / sizeof(*names); ++i)
        if (!(*names[i] = PyUnicode_InternFromString(text[i]))) return NULL;
    return PyModule_Create(&module);
}
