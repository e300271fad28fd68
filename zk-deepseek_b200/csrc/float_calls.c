/* Argument structures of the calls over pages and of sampling, from torch tensors: what Python needs a microsecond a tensor for.
 * Every function looks its tensors over (types, shapes, strides, device), raises ValueError for what does not belong together
 * and gives the bytes of the structure that the call takes; it launches nothing and keeps nothing.  Tensors are read through DLPack's C
 * exchange interface (a versioned one: 0.05 us a tensor), and where that declines (a tensor that requires gradients, say), or torch's headers or
 * torch itself do not have it, through their Python attributes (0.4 us); nothing here depends on how torch was built. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdarg.h>
#include <string.h>
#ifdef __has_include
#if __has_include(<ATen/dlpack.h>)
#include <ATen/dlpack.h>
#endif
#endif
/* the interface came with version 1.3 of the header */
#if defined(DLPACK_MAJOR_VERSION) && DLPACK_MAJOR_VERSION == 1 && DLPACK_MINOR_VERSION >= 3
#define EXCHANGE 1
#else
#define EXCHANGE 0
#endif

#include "zkds_float.h"

enum { kDims = 8 };

/* what `setup` was given, and names of attributes */
static PyObject *tensor_type, *bfloat16, *float32, *int32, *int64, *empty, *current_device, *empty_names;
static PyObject *n_dtype, *n_shape, *n_stride, *n_data_ptr, *n_get_device, *n_element_size;
static long long (*paged_scratch)(const zkfp_paged_attention_args*);
#if EXCHANGE
static DLPackDLTensorFromPyObjectNoSync exchange;
#endif

static int refuse(const char* what, const char* format, ...)
{
    va_list v;
    va_start(v, format);
    PyObject* text = PyUnicode_FromFormatV(format, v);
    va_end(v);
    if (text) PyErr_Format(PyExc_ValueError, "%s: %U", what, text);
    Py_XDECREF(text);
    return -1;
}

/* ---- tensors ---------------------------------------------------------------------------------------------------- */
typedef struct {
    PyObject* dtype;                 /* one of torch's, which live as long as torch */
    char* at;
    long long n[kDims], step[kDims];
    int dims, device, element;       /* element: its bytes, 0 where they are not known */
} Tensor;

static int numbers(PyObject* tuple, long long* to)
{
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(tuple); ++i) {
        to[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(tuple, i));
        if (to[i] == -1 && PyErr_Occurred()) return -1;
    }
    return 0;
}

static int is_tensor(PyObject* t) { return PyObject_TypeCheck(t, (PyTypeObject*)tensor_type); }

static int see(const char* what, const char* name, PyObject* t, Tensor* s)
{
    if (!is_tensor(t)) return refuse(what, "%s is no tensor", name);
#if EXCHANGE
    DLTensor d;
    if (exchange && exchange(t, &d)) PyErr_Clear();
    else if (exchange) {
        const int type = d.dtype.code << 8 | d.dtype.bits;
        s->dtype = d.dtype.lanes != 1 ? NULL : type == (kDLBfloat << 8 | 16) ? bfloat16 : type == (kDLFloat << 8 | 32) ? float32 : type == (kDLInt << 8 | 32) ? int32 : type == (kDLInt << 8 | 64) ? int64 : NULL;
        if (s->dtype && d.ndim <= kDims && (!d.ndim || d.strides)) {
            s->dims = d.ndim;
            s->at = (char*)d.data + d.byte_offset;
            s->device = d.device.device_type == kDLCUDA ? d.device.device_id : -1;
            s->element = d.dtype.bits / 8;
            for (int i = 0; i < d.ndim; ++i) {
                s->n[i] = d.shape[i];
                s->step[i] = d.strides[i];
            }
            return 0;
        }
    }
#endif
    int rc = -1;
    s->element = 0;
    PyObject *dtype = PyObject_GetAttr(t, n_dtype), *shape = NULL, *stride = NULL, *at = NULL, *device = NULL;
    if (dtype && (shape = PyObject_GetAttr(t, n_shape)) && (stride = PyObject_CallMethodNoArgs(t, n_stride)) &&
        (at = PyObject_CallMethodNoArgs(t, n_data_ptr)) && (device = PyObject_CallMethodNoArgs(t, n_get_device))) {
        s->dtype = dtype;
        if (!PyTuple_Check(shape) || !PyTuple_Check(stride) || PyTuple_GET_SIZE(shape) != PyTuple_GET_SIZE(stride) || PyTuple_GET_SIZE(shape) > kDims) {
            refuse(what, "%s has %zd dimensions", name, PyObject_Length(shape));
        } else {
            s->dims = (int)PyTuple_GET_SIZE(shape);
            s->at = (char*)(uintptr_t)PyLong_AsUnsignedLongLong(at);
            s->device = (int)PyLong_AsLong(device);
            if (!PyErr_Occurred()) rc = numbers(shape, s->n) || numbers(stride, s->step) ? -1 : 0;
        }
    }
    Py_XDECREF(dtype);
    Py_XDECREF(shape);
    Py_XDECREF(stride);
    Py_XDECREF(at);
    Py_XDECREF(device);
    return rc;
}

/* the device that the call goes to: the current one.  `t` is the tensor that says whether there is one */
static int device_of(const char* what, const char* name, PyObject* t, Tensor* s)
{
    if (see(what, name, t, s)) return -1;
    if (s->device < 0) return refuse(what, "%s is no tensor on a GPU", name);
    PyObject* d = PyObject_CallNoArgs(current_device);
    const long device = d ? PyLong_AsLong(d) : -1;
    Py_XDECREF(d);
    return device < 0 ? -1 : (int)device;
}

static int fits(const char* what, const char* name, const Tensor* s, PyObject* dtype, int dims, int device)
{
    if (s->dims != dims) return refuse(what, "%s has %d dimensions, not %d", name, s->dims, dims);
    if (s->dtype != dtype) return refuse(what, "%s is %S, not %S", name, s->dtype, dtype);
    if (s->device != device) return refuse(what, "%s is on device %d, the call goes to cuda:%d", name, s->device, device);
    return 0;
}

static int takes(const char* what, const char* name, PyObject* t, Tensor* s, PyObject* dtype, int dims, int device)
{
    return see(what, name, t, s) || fits(what, name, s, dtype, dims, device) ? -1 : 0;
}

static int shaped(const char* what, const char* name, const Tensor* s, const long long* n)
{
    for (int i = 0; i < s->dims; ++i)
        if (s->n[i] != n[i]) return refuse(what, "%s has %lld in dimension %d, not %lld", name, s->n[i], i, n[i]);
    return 0;
}

/* of one dimension, without gaps */
static int row(const char* what, const char* name, PyObject* t, Tensor* s, PyObject* dtype, int device, long long n)
{
    if (takes(what, name, t, s, dtype, 1, device) || shaped(what, name, s, &n)) return -1;
    return n > 1 && s->step[0] != 1 ? refuse(what, "%s is not contiguous", name) : 0;
}

/* a tensor of heads: the elements of a head adjacent, everything on 16-byte pieces (eight elements of bfloat16, and two of float32's); a
 * dimension of one element has no stride of its own, and gets 0 */
static int heads(const char* what, const char* name, Tensor* s)
{
    const int last = s->dims - 1;
    int bad = (uintptr_t)s->at & 15 || (s->n[last] > 1 && s->step[last] != 1);
    for (int i = 0; i < last; ++i) {
        if (s->n[i] <= 1) s->step[i] = 0;
        bad |= (s->step[i] & 7) != 0;
    }
    return bad ? refuse(what, "%s: heads must be contiguous, its strides multiples of 8 elements, its address one of 16 bytes", name) : 0;
}

/* results: no head on another one (a tensor that was expanded) */
static int apart(const char* what, const char* name, const Tensor* s)
{
    for (int i = 0; i + 1 < s->dims; ++i)
        if (s->n[i] > 1 && s->step[i] == 0) return refuse(what, "the heads of %s lie on one another", name);
    return 0;
}

typedef struct {
    Tensor k, v, table, rows, lengths;
    int device;
    long long batch, cols, ld;
} Pool;

static int see_pool(const char* what, PyObject* const* x, Pool* p)
{
    const int dev = p->device = device_of(what, "k_pages", x[0], &p->k);
    if (dev < 0) return -1;
    if (p->k.dtype != bfloat16 && p->k.dtype != float32) return refuse(what, "pages hold float32 or bfloat16");
    if (fits(what, "k_pages", &p->k, p->k.dtype, 4, dev) || heads(what, "k_pages", &p->k) || takes(what, "v_pages", x[1], &p->v, p->k.dtype, 4, dev) ||
        heads(what, "v_pages", &p->v))
        return -1;
    const long long page = p->k.n[1];
    if (memcmp(p->k.n, p->v.n, 3 * sizeof(long long))) return refuse(what, "pages of keys and of values differ in number, positions or heads");
    if (page < 8 || page > 1024 || page & (page - 1)) return refuse(what, "pages of %lld positions", page);
    if (!p->k.n[3] || !p->v.n[3] || (p->k.n[3] | p->v.n[3]) & 7) return refuse(what, "head sizes %lld and %lld are no multiples of 8", p->k.n[3], p->v.n[3]);
    if (takes(what, "table", x[2], &p->table, int32, 2, dev)) return -1;
    p->batch = p->table.n[0];
    p->cols = p->table.n[1];
    if (row(what, "rows", x[3], &p->rows, int32, dev, p->batch + 1) || row(what, "lengths", x[4], &p->lengths, int32, dev, p->batch)) return -1;
    if (!p->batch || !p->cols || !p->k.n[0] || !p->k.n[2]) return refuse(what, "no sequences, no columns, no pages or no heads");
    p->ld = p->batch > 1 ? p->table.step[0] : p->cols;
    if ((p->cols > 1 && p->table.step[1] != 1) || p->ld < p->cols) return refuse(what, "rows of the table must be contiguous");
    return 0;
}

static int code(PyObject* dtype) { return dtype == bfloat16 ? ZKFP_BF16 : ZKFP_F32; }

/* a whole number, those beyond 64 bits cut off */
static int whole(PyObject* x, long long* to)
{
    int over = 0;
    PyObject* i = PyNumber_Index(x);
    if (!i) return -1;
    *to = PyLong_AsLongLongAndOverflow(i, &over);
    Py_DECREF(i);
    if (over) *to = over > 0 ? 0x7fffffffffffffffll : -0x7fffffffffffffffll;
    return *to == -1 && PyErr_Occurred() ? -1 : 0;
}

static PyObject* new_tensor(long long n, PyObject* dtype, int device)
{
    PyObject *size = PyLong_FromLongLong(n), *dev = PyLong_FromLong(device), *t = NULL;
    if (size && dev) {
        PyObject* args[3] = {size, dtype, dev};
        t = PyObject_Vectorcall(empty, args, 1, empty_names);
    }
    Py_XDECREF(size);
    Py_XDECREF(dev);
    return t;
}

static PyObject* bytes_of(const void* a, size_t n) { return PyBytes_FromStringAndSize((const char*)a, (Py_ssize_t)n); }

/* ---- calls ------------------------------------------------------------------------------------------------------ */
/* (q, k_pages, v_pages, table, rows, lengths, out, scale, window, max_tokens, gate, out_scale): structure and scratch, or None */
static PyObject* paged_attention(PyObject* self, PyObject* const* x, Py_ssize_t count)
{
    const char* what = "paged_attention";
    Pool p;
    Tensor q, out, gate;
    long long window, most;
    if (count != 12) return PyErr_Format(PyExc_TypeError, "%s: 12 arguments", what);
    if (see_pool(what, x + 1, &p) || takes(what, "q", x[0], &q, p.k.dtype, 3, p.device) || heads(what, "q", &q)) return NULL;
    const long long tokens = q.n[0], h = q.n[1], kv = p.k.n[2], d = p.k.n[3], shape[3] = {tokens, h, p.v.n[3]};
    if (!h || h % kv || d != q.n[2]) {
        refuse(what, "%lld query heads of %lld over %lld key heads of %lld", h, q.n[2], kv, d);
        return NULL;
    }
    if (takes(what, "out", x[6], &out, p.k.dtype, 3, p.device) || shaped(what, "out", &out, shape) || heads(what, "out", &out) || apart(what, "out", &out))
        return NULL;
    memset(&gate, 0, sizeof gate);
    if (x[10] != Py_None && (takes(what, "gate", x[10], &gate, p.k.dtype, 3, p.device) || shaped(what, "gate", &gate, shape) || heads(what, "gate", &gate)))
        return NULL;
    const double scale = PyFloat_AsDouble(x[7]), out_scale = PyFloat_AsDouble(x[11]);
    if (PyErr_Occurred() || whole(x[8], &window)) return NULL;
    most = tokens < p.batch ? 1 : tokens - p.batch + 1;        /* if the other sequences bring one row each; it only chooses the kernel */
    if (x[9] != Py_None && whole(x[9], &most)) return NULL;
    if (window < 0 || most < 0 || !(scale >= 0 && scale < 3e38)) {
        refuse(what, "a negative window, bound or scale");
        return NULL;
    }
    if (tokens == 0) Py_RETURN_NONE;
    if (out.at == q.at || out.at == gate.at || out.at == p.k.at || out.at == p.v.at) {
        refuse(what, "out lies on an input");
        return NULL;
    }
    zkfp_paged_attention_args a;
    memset(&a, 0, sizeof a);
    a.q = q.at; a.k = p.k.at; a.v = p.v.at; a.out = out.at; a.gate = gate.at;
    a.table = (const int*)p.table.at; a.rows = (const int*)p.rows.at; a.lengths = (const int*)p.lengths.at;
    a.q_tok = q.step[0]; a.q_head = q.step[1];
    a.k_page = p.k.step[0]; a.k_pos = p.k.step[1]; a.k_head = p.k.step[2];
    a.v_page = p.v.step[0]; a.v_pos = p.v.step[1]; a.v_head = p.v.step[2];
    a.o_tok = out.step[0]; a.o_head = out.step[1];
    a.gate_tok = gate.step[0]; a.gate_head = gate.step[1];
    a.tokens = tokens; a.pages = p.k.n[0]; a.table_cols = p.cols; a.table_ld = p.ld; a.batch = p.batch; a.max_tokens = most;
    a.heads = (int)h; a.kv_heads = (int)kv; a.d = (int)d; a.dv = (int)p.v.n[3]; a.page = (int)p.k.n[1];
    a.window = (int)(window < 0x7fffffff ? window : 0x7fffffff);
    a.dtype = code(p.k.dtype);
    a.scale = (float)scale; a.out_scale = (float)out_scale;
    const long long floats = paged_scratch(&a);
    PyObject *scratch = Py_NewRef(Py_None), *result = NULL;
    if (floats > 0) {
        Py_SETREF(scratch, new_tensor(floats, float32, p.device));
        PyObject* at = scratch ? PyObject_CallMethodNoArgs(scratch, n_data_ptr) : NULL;
        if (at) a.scratch = (float*)(uintptr_t)PyLong_AsUnsignedLongLong(at);
        Py_XDECREF(at);
        if (!at || PyErr_Occurred()) goto done;
    }
    PyObject* bytes = bytes_of(&a, sizeof a);
    if (bytes) result = PyTuple_Pack(2, bytes, scratch);
    Py_XDECREF(bytes);
done:
    Py_XDECREF(scratch);
    return result;
}

/* (k, v, k_pages, v_pages, table, rows, lengths, q, q_out, cos_sin, half): structure, or None */
static PyObject* write_pages(PyObject* self, PyObject* const* x, Py_ssize_t count)
{
    const char* what = "write_pages";
    Pool p;
    Tensor k, v, q, out, angles;
    if (count != 11) return PyErr_Format(PyExc_TypeError, "%s: 11 arguments", what);
    if (see_pool(what, x + 2, &p) || apart(what, "k_pages", &p.k) || apart(what, "v_pages", &p.v)) return NULL;
    if (takes(what, "k", x[0], &k, p.k.dtype, 3, p.device) || heads(what, "k", &k)) return NULL;
    const long long tokens = k.n[0], kv = p.k.n[2], d = p.k.n[3], shape[3] = {tokens, kv, d}, vshape[3] = {tokens, kv, p.v.n[3]};
    if (shaped(what, "k", &k, shape) || takes(what, "v", x[1], &v, p.k.dtype, 3, p.device) || shaped(what, "v", &v, vshape) || heads(what, "v", &v)) return NULL;
    memset(&q, 0, sizeof q);
    memset(&out, 0, sizeof out);
    memset(&angles, 0, sizeof angles);
    if ((x[7] == Py_None) != (x[8] == Py_None)) {
        refuse(what, "q and q_out come together");
        return NULL;
    }
    if (x[7] != Py_None) {
        if (takes(what, "q", x[7], &q, p.k.dtype, 3, p.device) || heads(what, "q", &q)) return NULL;
        if (!q.n[1] || q.n[0] != tokens || q.n[2] != d) {
            refuse(what, "q is [%lld, %lld, %lld] beside %lld keys of %lld", q.n[0], q.n[1], q.n[2], tokens, d);
            return NULL;
        }
        if (takes(what, "q_out", x[8], &out, p.k.dtype, 3, p.device) || shaped(what, "q_out", &out, q.n) || heads(what, "q_out", &out) ||
            apart(what, "q_out", &out))
            return NULL;
    }
    if (x[9] != Py_None) {
        if (takes(what, "cos_sin", x[9], &angles, float32, 3, p.device)) return NULL;
        const long long* n = angles.n;
        const int adjacent = (n[2] <= 1 || angles.step[2] == 1) && (n[1] <= 1 || angles.step[1] == 2) && (n[0] <= 1 || angles.step[0] == 2 * n[1]);
        if (n[2] != 2 || (!adjacent && n[0] && n[1]) || 2 * n[1] > d) {
            refuse(what, "cos_sin [%lld, %lld, %lld] is no contiguous [positions, pairs, 2] for heads of %lld", n[0], n[1], n[2], d);
            return NULL;
        }
    }
    const int half = PyObject_IsTrue(x[10]);
    if (half < 0) return NULL;
    if (tokens == 0) Py_RETURN_NONE;
    zkfp_write_pages_args a;
    memset(&a, 0, sizeof a);
    a.q = q.at; a.k = k.at; a.v = v.at; a.q_out = out.at; a.k_pages = p.k.at; a.v_pages = p.v.at; a.cos_sin = (const float*)angles.at;
    a.table = (const int*)p.table.at; a.rows = (const int*)p.rows.at; a.lengths = (const int*)p.lengths.at;
    a.q_tok = q.step[0]; a.q_head = q.step[1]; a.k_tok = k.step[0]; a.k_head = k.step[1]; a.v_tok = v.step[0]; a.v_head = v.step[1];
    a.qo_tok = out.step[0]; a.qo_head = out.step[1];
    a.k_page = p.k.step[0]; a.k_pos = p.k.step[1]; a.kp_head = p.k.step[2];
    a.v_page = p.v.step[0]; a.v_pos = p.v.step[1]; a.vp_head = p.v.step[2];
    a.tokens = tokens; a.pages = p.k.n[0]; a.table_cols = p.cols; a.table_ld = p.ld; a.batch = p.batch; a.positions = angles.n[0];
    a.heads = (int)q.n[1]; a.kv_heads = (int)kv; a.d = (int)d; a.dv = (int)p.v.n[3]; a.page = (int)p.k.n[1];
    a.pairs = (int)angles.n[1]; a.half = half; a.dtype = code(p.k.dtype);
    return bytes_of(&a, sizeof a);
}

/* page numbers as an array of int, which the caller frees, and the smallest and largest of them */
static int* page_numbers(const char* what, PyObject* list, Py_ssize_t* n, long long* least, long long* most)
{
    PyObject* fast = PySequence_Fast(list, "page numbers are a sequence");
    if (!fast) return NULL;
    *n = PySequence_Fast_GET_SIZE(fast);
    int* to = (int*)PyMem_Malloc(sizeof(int) * (size_t)(*n ? *n : 1));
    if (!to) PyErr_NoMemory();
    for (Py_ssize_t i = 0; to && i < *n; ++i) {
        long long page;
        int bad = whole(PySequence_Fast_GET_ITEM(fast, i), &page);
        if (!bad && (page < 0 || page > 0x7fffffff)) bad = refuse(what, "page %lld", page);
        if (bad) {
            PyMem_Free(to);
            to = NULL;
            break;
        }
        to[i] = (int)page;
        if (page < *least) *least = page;
        if (page > *most) *most = page;
    }
    Py_DECREF(fast);
    return to;
}

/* one buffer: bytes between pages, bytes of one that are copied, pages */
static int page_buffer(const char* what, PyObject* t, int i, int device, long long most, long long positions, zkfp_page_buffer* b)
{
    Tensor s;
    char name[32];
    PyOS_snprintf(name, sizeof name, "buffer %d", i);
    if (see(what, name, t, &s)) return -1;
    if (s.device != device) return refuse(what, "%s is not on cuda:%d", name, device);
    if (s.dims < 2) return refuse(what, "%s is no [pages, page, ...] tensor", name);
    const long long pages = s.n[0], lines = s.n[1];
    if (positions > lines) return refuse(what, "%lld positions of pages of %lld", positions, lines);
    if (pages <= most) return refuse(what, "pages that %s of %lld does not have", name, pages);
    long long element = s.element;
    if (!element) {
        PyObject* e = PyObject_CallMethodNoArgs(t, n_element_size);
        element = e ? PyLong_AsLongLong(e) : -1;
        Py_XDECREF(e);
        if (element < 0) return -1;
    }
    long long whole_page = element;
    int gaps = 0;
    for (int k = s.dims - 1; k > 0; --k) {
        gaps |= s.n[k] > 1 && s.step[k] * element != whole_page;
        whole_page *= s.n[k];
    }
    b->base = s.at;
    b->pages = pages;
    b->stride = b->bytes = 0;
    if (whole_page) {
        if (gaps) return refuse(what, "pages of %s are not contiguous", name);
        b->bytes = positions < 0 ? whole_page : whole_page / lines * positions;
        b->stride = pages > 1 ? s.step[0] * element : whole_page;
        if ((b->stride | b->bytes) & 15 || b->stride < whole_page)
            return refuse(what, "pages of %s, or the part of them that is copied, do not lie on 16-byte pieces of their own", name);
    }
    return (uintptr_t)s.at & 15 ? refuse(what, "%s does not lie on 16-byte pieces", name) : 0;
}

/* (buffers, source, target, positions): buffers, their number, sources, targets and their number, or None */
static PyObject* copy_pages(PyObject* self, PyObject* const* x, Py_ssize_t count)
{
    const char* what = "copy_pages";
    if (count != 4) return PyErr_Format(PyExc_TypeError, "%s: 4 arguments", what);
    Py_ssize_t n = 0, m = 0;
    long long least = 0x7fffffff, most = -1, positions = -1;
    PyObject *result = NULL, *buffers = PySequence_Fast(x[0], "buffers are a sequence"), *list = NULL;
    int *source = NULL, *target = NULL;
    if (!buffers || !(source = page_numbers(what, x[1], &n, &least, &most)) || !(target = page_numbers(what, x[2], &m, &least, &most))) goto done;
    if (n != m) {
        refuse(what, "%zd sources, %zd targets", n, m);
        goto done;
    }
    if (x[3] != Py_None && (whole(x[3], &positions) || (positions < 0 && refuse(what, "%lld positions", positions)))) goto done;
    const Py_ssize_t many = PySequence_Fast_GET_SIZE(buffers);
    if (!many || !n) {
        result = Py_NewRef(Py_None);
        goto done;
    }
    Tensor first;
    const int device = device_of(what, "a buffer", PySequence_Fast_GET_ITEM(buffers, 0), &first);
    if (device < 0 || !(list = PyBytes_FromStringAndSize(NULL, many * (Py_ssize_t)sizeof(zkfp_page_buffer)))) goto done;
    for (Py_ssize_t i = 0; i < many; ++i)
        if (page_buffer(what, PySequence_Fast_GET_ITEM(buffers, i), (int)i, device, most, positions, (zkfp_page_buffer*)PyBytes_AS_STRING(list) + i)) goto done;
    result = Py_BuildValue("Oiy#y#n", list, (int)many, (const char*)source, n * (Py_ssize_t)sizeof(int), (const char*)target, n * (Py_ssize_t)sizeof(int), n);
done:
    PyMem_Free(source);
    PyMem_Free(target);
    Py_XDECREF(buffers);
    Py_XDECREF(list);
    return result;
}

/* (logits, random, out, temperature, top_k, top_p, min_p): structure (or None: no rows) and out, which is made where it is None */
static PyObject* sample(PyObject* self, PyObject* const* x, Py_ssize_t count)
{
    const char* what = "sample";
    static const char* const names[4] = {"temperature", "top_k", "top_p", "min_p"};
    Tensor l, t;
    zkfp_sample_args a;
    if (count != 7) return PyErr_Format(PyExc_TypeError, "%s: 7 arguments", what);
    const int device = device_of(what, "logits", x[0], &l);
    if (device < 0) return NULL;
    if (l.dtype != bfloat16 && l.dtype != float32) {
        refuse(what, "logits are float32 or bfloat16");
        return NULL;
    }
    if (fits(what, "logits", &l, l.dtype, 2, device)) return NULL;
    memset(&a, 0, sizeof a);
    a.logits = l.at;
    a.rows = l.n[0];
    a.vocab = l.n[1];
    a.ld = a.rows == 1 ? a.vocab : l.step[0];
    a.dtype = code(l.dtype);
    if (!a.vocab || (a.vocab > 1 && l.step[1] != 1) || (a.rows && a.ld < a.vocab)) {
        refuse(what, "logits [%lld, %lld] with strides [%lld, %lld]", l.n[0], l.n[1], l.step[0], l.step[1]);
        return NULL;
    }
    if (row(what, "random", x[1], &t, float32, device, a.rows)) return NULL;
    a.random = (const float*)t.at;
    const void* at[4] = {NULL, NULL, NULL, NULL};
    double value[4] = {0, 0, 0, 0};
    for (int i = 0; i < 4; ++i) {
        if (is_tensor(x[3 + i])) {
            if (row(what, names[i], x[3 + i], &t, i == 1 ? int32 : float32, device, a.rows)) return NULL;
            at[i] = t.at;
        } else {
            value[i] = PyFloat_AsDouble(x[3 + i]);
            if (value[i] == -1 && PyErr_Occurred()) return NULL;
            if (!(value[i] >= 0) || (i == 1 && value[i] < 1e15 && value[i] != (double)(long long)value[i])) {
                refuse(what, "%s is %R", names[i], x[3 + i]);
                return NULL;
            }
        }
    }
    a.temperature = (const float*)at[0]; a.top_k = (const int*)at[1]; a.top_p = (const float*)at[2]; a.min_p = (const float*)at[3];
    a.value_temperature = (float)value[0]; a.value_top_k = (int)(value[1] < 0x7fffffff ? value[1] : 0x7fffffff);
    a.value_top_p = (float)value[2]; a.value_min_p = (float)value[3];
    PyObject *out = x[2] == Py_None ? new_tensor(a.rows, int64, device) : Py_NewRef(x[2]), *result = NULL;
    if (out && !row(what, "out", out, &t, int64, device, a.rows)) {
        a.out = (long long*)t.at;
        PyObject* bytes = a.rows ? bytes_of(&a, sizeof a) : Py_NewRef(Py_None);
        if (bytes) result = PyTuple_Pack(2, bytes, out);
        Py_XDECREF(bytes);
    }
    Py_XDECREF(out);
    return result;
}

/* (torch.Tensor, bfloat16, float32, int32, int64, torch.empty, current device, address of zkfp_paged_scratch, capsule of the exchange interface) */
static PyObject* setup(PyObject* self, PyObject* const* x, Py_ssize_t count)
{
    PyObject** to[7] = {&tensor_type, &bfloat16, &float32, &int32, &int64, &empty, &current_device};
    if (count != 9 || !PyType_Check(x[0])) return PyErr_Format(PyExc_TypeError, "setup: 9 arguments, a type first");
    const unsigned long long at = PyLong_AsUnsignedLongLong(x[7]);
    if (PyErr_Occurred()) return NULL;
#if EXCHANGE
    const DLPackExchangeAPI* api = x[8] == Py_None ? NULL : (const DLPackExchangeAPI*)PyCapsule_GetPointer(x[8], "dlpack_exchange_api");
    if (PyErr_Occurred()) return NULL;
    exchange = api && api->header.version.major == DLPACK_MAJOR_VERSION ? api->dltensor_from_py_object_no_sync : NULL;
#endif
    for (int i = 0; i < 7; ++i) Py_XSETREF(*to[i], Py_NewRef(x[i]));
    paged_scratch = (long long (*)(const zkfp_paged_attention_args*))(uintptr_t)at;
    Py_RETURN_NONE;
}

static PyMethodDef methods[] = {{"setup", (PyCFunction)(void (*)(void))setup, METH_FASTCALL, NULL},
                                {"paged_attention", (PyCFunction)(void (*)(void))paged_attention, METH_FASTCALL, NULL},
                                {"write_pages", (PyCFunction)(void (*)(void))write_pages, METH_FASTCALL, NULL},
                                {"copy_pages", (PyCFunction)(void (*)(void))copy_pages, METH_FASTCALL, NULL},
                                {"sample", (PyCFunction)(void (*)(void))sample, METH_FASTCALL, NULL},
                                {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "float_calls", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit_float_calls(void)
{
    n_dtype = PyUnicode_InternFromString("dtype");
    n_shape = PyUnicode_InternFromString("shape");
    n_stride = PyUnicode_InternFromString("stride");
    n_data_ptr = PyUnicode_InternFromString("data_ptr");
    n_get_device = PyUnicode_InternFromString("get_device");
    n_element_size = PyUnicode_InternFromString("element_size");
    empty_names = Py_BuildValue("(ss)", "dtype", "device");
    if (!n_dtype || !n_shape || !n_stride || !n_data_ptr || !n_get_device || !n_element_size || !empty_names) return NULL;
    return PyModule_Create(&module);
}
