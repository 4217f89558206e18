// torch tensors in, the token-step operators of include/hipvoc_ops.h out: the CPython module behind qwen3-tts_amd/ops.py.
//
// A token step makes some hundred calls of a few microseconds each, so what a call costs the host counts as much as its kernel.  Looking at the tensors,
// allocating the results and converting the arguments costs 4.4 us in Python with ctypes (8.2 us for an add_rmsnorm of one row, of them 3.0 the launch);
// here the same things are C++ on the tensors themselves.  The entry points stay those of the C ABI, whose addresses ops.py hands over (bind): this
// module links nothing of it.
#include <torch/csrc/python_headers.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Device.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>

#include "../../include/hipvoc_ops.h"

namespace {

struct {
    decltype(&hipvoc_kv_write) kv_write;
    decltype(&hipvoc_kv_read) kv_read;
    decltype(&hipvoc_attention_workspace) attention_workspace;
    decltype(&hipvoc_attention) attention;
    decltype(&hipvoc_add_rmsnorm) add_rmsnorm;
    decltype(&hipvoc_q4_matvec) q4_matvec;
    decltype(&hipvoc_last_error) last_error;
} api;
PyObject *error_type, *str_p, *str_device;            // HipVocError, and the names of a cache's attributes

struct Raised {};                                      // a Python exception is set
[[noreturn]] void fail(int code, const std::string &why) {
    PyObject *e = PyObject_CallFunction(error_type, "is", code, why.c_str());
    if (e) PyErr_SetObject(error_type, e);
    Py_XDECREF(e);
    throw Raised();
}
[[noreturn]] void refuse(const std::string &why) { fail(HIPVOC_E_ARG, why); }
std::string say(long long v) { return std::to_string(v); }

// ---- arguments -----------------------------------------------------------------------------------------------------------------------
struct Call {                                          // (handle, device) that every function starts with
    void *h;
    c10::Device device{c10::kCUDA, 0};
    hipStream_t stream;
    PyObject *const *arg;
};
Call call_of(PyObject *const *args, Py_ssize_t n, Py_ssize_t want) {
    if (n != want + 2) {
        PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
        throw Raised();
    }
    Call c;
    if (args[0] == Py_None) refuse("the handle is closed");
    c.h = PyLong_AsVoidPtr(args[0]);
    const long index = PyLong_AsLong(args[1]);
    if (PyErr_Occurred()) throw Raised();
    c.device = c10::Device(c10::kCUDA, (c10::DeviceIndex)index);
    c.stream = c10::hip::getCurrentHIPStream((c10::DeviceIndex)index).stream();
    c.arg = args + 2;
    return c;
}
void answered(const Call &c, int rc) {
    if (rc) fail(rc, api.last_error(c.h));
}
int number(PyObject *o, const char *name) {
    int overflow = 0;
    const long long v = PyLong_AsLongLongAndOverflow(o, &overflow);
    if (v == -1 && PyErr_Occurred()) throw Raised();
    if (overflow || v < 0 || v >= 1LL << 31) refuse(std::string(name) + " is negative or does not fit 32 bits");
    return (int)v;
}
float real(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised();
    return (float)v;
}
const at::Tensor &tensor(const Call &c, PyObject *o, const char *name) {
    if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
    const at::Tensor &t = THPVariable_Unpack(o);
    if (t.layout() != c10::kStrided) refuse(std::string(name) + " must be a strided tensor");
    if (t.device() != c.device) refuse(std::string(name) + " is on " + t.device().str() + ", the handle on " + c.device.str());
    // a result without a graph would end the gradient without a word
    if (t.requires_grad() && at::GradMode::is_enabled()) refuse(std::string(name) + " requires grad, and the operators have no backward: call them under torch.no_grad() or on " + name + ".detach()");
    if (t.is_neg()) refuse(std::string(name) + " is a view whose memory holds its negative: resolve_neg() makes it a tensor of its own");
    return t;
}
int type_of(c10::ScalarType t) {
    switch (t) {
        case c10::kFloat: return HIPVOC_T_F32;
        case c10::kHalf: return HIPVOC_T_F16;
        case c10::kBFloat16: return HIPVOC_T_BF16;
        case c10::kChar: return HIPVOC_T_INT8;
        case c10::kFloat8_e4m3fn: return HIPVOC_T_E4M3;
        default: refuse(std::string("unsupported dtype ") + c10::toString(t));
    }
}
c10::ScalarType scalar_of(int type) {
    static const c10::ScalarType t[] = {c10::kFloat, c10::kHalf, c10::kBFloat16, c10::kChar, c10::kFloat8_e4m3fn};
    return t[type];
}
c10::ScalarType dtype_of(PyObject *o, c10::ScalarType none) {
    if (o == Py_None) return none;
    if (!THPDtype_Check(o)) refuse("dtype must be a torch dtype");
    return ((THPDtype *)o)->scalar_type;
}
int rows32(int64_t n, const char *name) {
    if (n >> 31) refuse(std::string(name) + " has " + say(n) + " rows or columns");
    return (int)n;
}

const hipvoc_kv_cache *cache_of(const Call &c, PyObject *o) {
    PyObject *p = PyObject_GetAttr(o, str_p), *d = p ? PyObject_GetAttr(o, str_device) : nullptr;
    const void *at = p && d ? PyLong_AsVoidPtr(p) : nullptr;
    const bool device = d && THPDevice_Check(d), here = device && ((THPDevice *)d)->device == c.device;
    Py_XDECREF(p);
    Py_XDECREF(d);
    PyErr_Clear();
    if (!at || !device) refuse("cache must be a KvCache");
    if (!here) refuse("the cache is on another device than the handle, " + c.device.str());
    return (const hipvoc_kv_cache *)at;
}
// A contiguous int32 vector of n values
const int32_t *ints(const Call &c, PyObject *o, int64_t n, const char *name) {
    const at::Tensor &t = tensor(c, o, name);
    if (t.scalar_type() != c10::kInt || t.dim() != 1 || t.size(0) != n || (n > 1 && t.stride(0) != 1)) refuse(std::string(name) + " must be a contiguous int32 vector of " + say(n));
    return (const int32_t *)t.data_ptr();
}
struct Table { const int32_t *p; int64_t stride; int width, rows; };
Table table_of(const Call &c, PyObject *o) {
    const at::Tensor &t = tensor(c, o, "table");
    if (t.scalar_type() != c10::kInt || t.dim() != 2 || (t.size(1) > 1 && t.stride(1) != 1)) refuse("table must be int32 [seqs, pages] with contiguous rows");
    return {(const int32_t *)t.data_ptr(), t.stride(0), rows32(t.size(1), "table"), rows32(t.size(0), "table")};
}
struct Heads { void *p; int64_t stride; int rows; c10::ScalarType type; };
// [rows, heads, head_dim] with contiguous rows
Heads heads_of(const Call &c, PyObject *o, int64_t heads, int64_t hd, const char *name) {
    const at::Tensor &t = tensor(c, o, name);
    if (t.dim() != 3 || t.size(1) != heads || t.size(2) != hd || t.stride(2) != 1 || (heads > 1 && t.stride(1) != hd))
        refuse(std::string(name) + " must be [rows, " + say(heads) + ", " + say(hd) + "] with contiguous rows");
    const int rows = rows32(t.size(0), name);
    return {t.data_ptr(), rows > 1 ? t.stride(0) : heads * hd, rows, t.scalar_type()};
}
struct Matrix { void *p; int64_t stride; int rows, cols; c10::ScalarType type; };
Matrix matrix_of(const Call &c, PyObject *o, const char *name) {
    const at::Tensor &t = tensor(c, o, name);
    if (t.dim() != 2 || (t.size(1) > 1 && t.stride(1) != 1)) refuse(std::string(name) + " must be a matrix with contiguous rows");
    const int rows = rows32(t.size(0), name), cols = rows32(t.size(1), name);
    return {t.data_ptr(), rows > 1 ? t.stride(0) : cols, rows, cols, t.scalar_type()};
}
at::Tensor fresh(const Call &c, c10::IntArrayRef shape, c10::ScalarType t) { return at::Tensor(at::detail::empty_cuda(shape, t, c.device, std::nullopt)); }

// The call itself, with Python free to run other threads
template <typename F> int apart(F &&f) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f();
    Py_END_ALLOW_THREADS
    return rc;
}

// ---- results -------------------------------------------------------------------------------------------------------------------------
PyObject *given(PyObject *o) {
    Py_INCREF(o);
    return o;
}
PyObject *wrapped(const at::Tensor &t) {
    if (!t.defined()) return given(Py_None);
    PyObject *o = THPVariable_Wrap(t);
    if (!o) throw Raised();
    return o;
}
PyObject *tuple_of(std::initializer_list<PyObject *> items) {
    PyObject *t = PyTuple_New((Py_ssize_t)items.size());
    if (!t) throw Raised();
    Py_ssize_t i = 0;
    for (PyObject *o : items) PyTuple_SET_ITEM(t, i++, o);
    return t;
}

// ---- the operators ----------------------------------------------------------------------------------------------------------------------
hipvoc_kv_rows rows_of(const Call &c, PyObject *table, PyObject *cu, PyObject *first) {
    const Table t = table_of(c, table);
    return {t.p, ints(c, cu, (int64_t)t.rows + 1, "cu"), ints(c, first, t.rows, "first"), t.stride, t.width, t.rows};
}

PyObject *kv_write(const Call &c) {                    // cache, k, v, table, cu, first
    const hipvoc_kv_cache *cache = cache_of(c, c.arg[0]);
    const Heads k = heads_of(c, c.arg[1], cache->kv_heads, cache->head_dim, "k"), v = heads_of(c, c.arg[2], cache->kv_heads, cache->head_dim, "v");
    if (k.rows != v.rows || k.type != v.type) refuse("k and v must be alike");
    const hipvoc_kv_rows r = rows_of(c, c.arg[3], c.arg[4], c.arg[5]);
    const int t = type_of(k.type);
    answered(c, apart([&] { return api.kv_write(c.h, cache, k.p, v.p, k.stride, v.stride, t, &r, k.rows, c.stream); }));
    return given(Py_None);
}

PyObject *kv_read(const Call &c) {                     // cache, table, cu, first, n_rows, dtype, out
    const hipvoc_kv_cache *cache = cache_of(c, c.arg[0]);
    const int64_t heads = cache->kv_heads, hd = cache->head_dim;
    const int n = number(c.arg[4], "n_rows");
    at::Tensor tk, tv;
    Heads k, v;
    if (c.arg[6] == Py_None) {
        const c10::ScalarType type = dtype_of(c.arg[5], scalar_of(cache->dtype));
        type_of(type);
        tk = fresh(c, {n, heads, hd}, type);
        tv = fresh(c, {n, heads, hd}, type);
        k = {tk.data_ptr(), heads * hd, n, type};
        v = {tv.data_ptr(), heads * hd, n, type};
    } else {
        if (!PyTuple_Check(c.arg[6]) || PyTuple_GET_SIZE(c.arg[6]) != 2) refuse("out must be a tuple of two tensors");
        if (c.arg[5] != Py_None) refuse("dtype is out's where out is given");
        k = heads_of(c, PyTuple_GET_ITEM(c.arg[6], 0), heads, hd, "k");
        v = heads_of(c, PyTuple_GET_ITEM(c.arg[6], 1), heads, hd, "v");
        if (k.rows < n || v.rows < n || k.type != v.type) refuse("out must be two tensors of n_rows rows, alike in type");
    }
    const hipvoc_kv_rows r = rows_of(c, c.arg[1], c.arg[2], c.arg[3]);
    const int t = type_of(k.type);
    answered(c, apart([&] { return api.kv_read(c.h, cache, k.p, v.p, k.stride, v.stride, t, &r, n, c.stream); }));
    if (!tk.defined()) return given(c.arg[6]);
    return tuple_of({wrapped(tk), wrapped(tv)});
}

PyObject *attention(const Call &c) {                   // q, cache, table, lens, scale, window, max_len, lse, out
    const hipvoc_kv_cache *cache = cache_of(c, c.arg[1]);
    const at::Tensor &tq = tensor(c, c.arg[0], "q");
    if (tq.dim() != 3) refuse("q must be [seqs, heads, head_dim]");
    const int heads = rows32(tq.size(1), "q");
    const int64_t hd = cache->head_dim;
    const Heads q = heads_of(c, c.arg[0], heads, hd, "q");
    const Table t = table_of(c, c.arg[2]);
    if (t.rows != q.rows) refuse("table must have a row per sequence");
    const int32_t *lens = ints(c, c.arg[3], q.rows, "lens");
    const float scale = c.arg[4] == Py_None ? (float)(1.0 / std::sqrt((double)hd)) : real(c.arg[4]);
    const int window = number(c.arg[5], "window"), type = type_of(q.type);
    const int64_t all = (int64_t)t.width * cache->page;
    if (c.arg[6] == Py_None && all >> 31) refuse("table: a sequence may have up to 2^31 - 256 positions");
    const int max_len = c.arg[6] == Py_None ? (int)all : number(c.arg[6], "max_len"), want = PyObject_IsTrue(c.arg[7]);
    if (want < 0) throw Raised();
    at::Tensor to, ts, work;
    Heads out;
    if (c.arg[8] == Py_None) {
        to = fresh(c, {q.rows, heads, hd}, q.type);
        out = {to.data_ptr(), heads * hd, q.rows, q.type};
    } else {
        out = heads_of(c, c.arg[8], heads, hd, "out");
        if (out.rows != q.rows || out.type != q.type) refuse("out must be like q");
    }
    if (want) ts = fresh(c, {q.rows, heads}, c10::kFloat);
    const size_t need = api.attention_workspace(cache, heads, q.rows, max_len, window);
    if (need) work = fresh(c, {(int64_t)(need / 4)}, c10::kInt);
    float *lse = want ? (float *)ts.data_ptr() : nullptr;
    void *ws = need ? work.data_ptr() : nullptr;
    answered(c, apart([&] {
        return api.attention(c.h, cache, q.p, q.stride, out.p, out.stride, lse, type, heads, t.p, t.stride, t.width, lens, q.rows, max_len, window, scale, ws, need, c.stream);
    }));
    PyObject *o = to.defined() ? wrapped(to) : given(c.arg[8]);
    return want ? tuple_of({o, wrapped(ts)}) : o;
}

PyObject *add_rmsnorm(const Call &c) {                 // x, weight, residual, eps, quant (a type or None), group
    const Matrix x = matrix_of(c, c.arg[0], "x");
    const at::Tensor &w = tensor(c, c.arg[1], "weight");
    const int type = type_of(x.type), group = number(c.arg[5], "group"), rows = x.rows, cols = x.cols;
    if (w.scalar_type() != x.type || w.dim() != 1 || w.size(0) != cols || (cols > 1 && w.stride(0) != 1)) refuse("weight must be a contiguous [cols] of x's type");
    const float eps = real(c.arg[3]);
    Matrix r = {};
    at::Tensor sum, y, scales;
    if (c.arg[2] != Py_None) {
        r = matrix_of(c, c.arg[2], "residual");
        if (r.type != x.type || r.rows != rows || r.cols != cols) refuse("residual must have x's type and shape");
        sum = fresh(c, {rows, cols}, x.type);
    }
    int out = type;
    if (c.arg[4] == Py_None) {
        y = fresh(c, {rows, cols}, x.type);
    } else {
        out = number(c.arg[4], "quant");
        if (group && ((group != 32 && group != 64 && group != 128) || cols % group))
            refuse("group " + say(group) + " must be 0, or 32, 64 or 128 and a divisor of cols " + say(cols));
        y = fresh(c, {rows, cols}, scalar_of(out));
        scales = fresh(c, {rows, group ? cols / group : 1}, c10::kFloat);
    }
    void *sp = sum.defined() ? sum.data_ptr() : nullptr, *yp = y.data_ptr(), *wp = w.data_ptr();
    float *cp = scales.defined() ? (float *)scales.data_ptr() : nullptr;
    answered(c, apart([&] { return api.add_rmsnorm(c.h, x.p, x.stride, r.p, r.stride, wp, sp, cols, yp, cols, cp, type, out, group, eps, rows, cols, c.stream); }));
    if (!scales.defined()) return tuple_of({wrapped(sum), wrapped(y)});
    return tuple_of({wrapped(sum), wrapped(y), wrapped(scales)});
}

PyObject *q4_matvec(const Call &c) {                   // codes, scales, x, mins, x_scale, dtype
    const at::Tensor &codes = tensor(c, c.arg[0], "codes"), &scales = tensor(c, c.arg[1], "scales");
    if (codes.dim() != 2 || codes.scalar_type() != c10::kByte || !codes.is_contiguous()) refuse("codes must be a contiguous uint8 [n_out, n_in / 2]");
    const int n_out = rows32(codes.size(0), "codes"), n_in = rows32(codes.size(1) * 2, "codes");
    if (scales.dim() != 2 || scales.size(0) != n_out || scales.scalar_type() != c10::kHalf || !scales.is_contiguous() || scales.size(1) < 1 || n_in % scales.size(1))
        refuse("scales must be a contiguous float16 [n_out, n_in / group]");
    const void *mins = nullptr;
    if (c.arg[3] != Py_None) {
        const at::Tensor &t = tensor(c, c.arg[3], "mins");
        if (t.scalar_type() != c10::kHalf || t.sizes() != scales.sizes() || !t.is_contiguous()) refuse("mins must be like scales");
        mins = t.data_ptr();
    }
    const Matrix x = matrix_of(c, c.arg[2], "x");
    if (x.cols != n_in) refuse("x must have " + say(n_in) + " columns");
    const int type = type_of(x.type), group = (int)(n_in / scales.size(1));
    const float *x_scale = nullptr;
    int x_groups = 0;
    c10::ScalarType out = x.type;
    if (type == HIPVOC_T_INT8) {
        if (c.arg[4] == Py_None) refuse("int8 rows need x_scale, a contiguous float32 [rows, n_in / group] or [rows, 1]");
        const at::Tensor &t = tensor(c, c.arg[4], "x_scale");
        if (t.scalar_type() != c10::kFloat || t.dim() != 2 || t.size(0) != x.rows || !t.is_contiguous()) refuse("int8 rows need x_scale, a contiguous float32 [rows, n_in / group] or [rows, 1]");
        x_groups = rows32(t.size(1), "x_scale");
        x_scale = (const float *)t.data_ptr();
        out = c10::kFloat;
    } else if (c.arg[4] != Py_None) {
        refuse("only int8 rows have scales");
    }
    out = dtype_of(c.arg[5], out);
    const int y_type = type_of(out);
    const at::Tensor y = fresh(c, {x.rows, n_out}, out);
    const uint8_t *cp = (const uint8_t *)codes.data_ptr();
    const void *sp = scales.data_ptr();
    void *yp = y.data_ptr();
    answered(c, apart([&] { return api.q4_matvec(c.h, cp, sp, mins, n_out, n_in, group, x.p, x.stride, type, x_scale, x_groups, yp, n_out, y_type, x.rows, c.stream); }));
    return wrapped(y);
}

// No C++ exception passes into Python: ours are set there already, torch's (out of memory, a bad device) become RuntimeError.
template <PyObject *(*F)(const Call &), int ARGS> PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
    try {
        return F(call_of(args, n, ARGS));
    } catch (const Raised &) {
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}

// (HipVocError, addresses of the C entry points in api's order)
PyObject *bind(PyObject *, PyObject *args) {
    unsigned long long a[7];
    PyObject *e;
    if (!PyArg_ParseTuple(args, "OKKKKKKK", &e, a, a + 1, a + 2, a + 3, a + 4, a + 5, a + 6)) return nullptr;
    Py_INCREF(e);
    Py_XDECREF(error_type);
    error_type = e;
    api = {(decltype(api.kv_write))a[0], (decltype(api.kv_read))a[1], (decltype(api.attention_workspace))a[2], (decltype(api.attention))a[3],
           (decltype(api.add_rmsnorm))a[4], (decltype(api.q4_matvec))a[5], (decltype(api.last_error))a[6]};
    return given(Py_None);
}

#define ENTRY(f, args) {#f, (PyCFunction)(void (*)(void))(PyObject * (*)(PyObject *, PyObject *const *, Py_ssize_t)) entry<f, args>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, nullptr}, ENTRY(kv_write, 6), ENTRY(kv_read, 7), ENTRY(attention, 9), ENTRY(add_rmsnorm, 6), ENTRY(q4_matvec, 6), {}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops_torch", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__ops_torch(void) {
    str_p = PyUnicode_InternFromString("_p");
    str_device = PyUnicode_InternFromString("device");
    return str_p && str_device ? PyModule_Create(&module) : nullptr;
}
