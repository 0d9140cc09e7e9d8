// front.cpp - the Python front end's calls into the C ABI (include/ffkv.h) as a CPython extension.
//
// A decode step of a small model is a handful of calls of a few microseconds of GPU work each, issued from Python
// once per layer.  Through ctypes a call cost 6 to 8 us before anything was launched: about 20 argument conversions,
// and a Python call for every pointer, shape and dtype.  Here the wrappers of firefly_amd/__init__.py hand their
// tensors over as they are, and shapes, dtypes, pointers and the current stream are read natively: 1 to 2 us.  The fused
// append + decode of 4 rows of up to 255 tokens (16/8 heads), one launch: 10.1 -> 6.9 us in a row, where the GPU now sets
// the pace, and 24.2 -> 19.1 us for a call that is waited for.
// The library is the one firefly_amd loaded: bind() gets the addresses of its functions, so nothing is linked here.
// Only CPython's own API is used; tensors are read through their attributes (shape, dtype, data_ptr(), nbytes).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <climits>
#include <cstdarg>
#include <cstdint>
#include <initializer_list>
#include <vector>

#include "ffkv.h"

namespace
{

struct Functions
{
    decltype(&ffkv_append)                     append;
    decltype(&ffkv_paged_decode)               decode;
    decltype(&ffkv_append_paged_decode)        append_decode;
    decltype(&ffkv_paged_decode_shared_prefix) decode_shared;
    decltype(&ffkv_paged_decode_noalloc)       decode_noalloc;
    decltype(&ffkv_prefill_workspace_bytes)    prefill_bytes;
    decltype(&ffkv_paged_prefill_ws)           prefill;
    decltype(&ffkv_rope)                       rope;
    decltype(&ffkv_rope_append)                rope_append;
    decltype(&ffkv_paged_decode_scored)        decode_scored;
    decltype(&ffkv_prefill_scored_workspace_bytes) prefill_scored_bytes;
    decltype(&ffkv_paged_prefill_scored)       prefill_scored;
    decltype(&ffkv_evict)                      evict;
    decltype(&ffkv_attention_weights)          attention_weights;
    decltype(&ffkv_decode_scored_scratch_bytes)       decode_scored_bytes;
    decltype(&ffkv_attention_weights_workspace_bytes) weights_bytes;
    decltype(&ffkv_evict_workspace_bytes)             evict_bytes;
};
Functions fn{};

PyObject *s_shape, *s_dtype, *s_data_ptr, *s_nbytes, *s_cuda_stream, *s_device, *s_index, *s_is_contiguous, *s_is_cuda;
constexpr int kInt32 = 4;  // int32 among bind()'s dtypes: tables and lengths, no dtype of activations or caches
struct DtypeCode
{
    PyObject* dtype;
    int       code;
};
std::vector<DtypeCode> dtypes;
PyObject *              get_device, *raw_stream, *first_stream;  // set by bind()
bool                    stream_ready = false;

// Reads a call's arguments one after the other; after the first failure (a Python exception is set) the rest read as
// zero.
struct Reader
{
    PyObject* const* a;
    bool             ok = true;

    void* ptr(PyObject* t)
    {
        if (!ok || t == Py_None) return nullptr;
        PyObject* p = PyObject_CallMethodNoArgs(t, s_data_ptr);
        void*     v = p ? PyLong_AsVoidPtr(p) : nullptr;
        Py_XDECREF(p);
        if (PyErr_Occurred()) ok = false;
        return v;
    }
    template <typename T>
    T* ptr(PyObject* t)
    {
        return static_cast<T*>(ptr(t));
    }
    // The sizes of t (a tuple), at least `least` and, when exactly is set, as many.
    PyObject* shape(PyObject* t, Py_ssize_t least, bool exactly)
    {
        if (!ok) return nullptr;
        PyObject* s = PyObject_GetAttr(t, s_shape);
        if (s != nullptr && PyTuple_Check(s))
        {
            const Py_ssize_t n = PyTuple_GET_SIZE(s);
            if (n >= least && (!exactly || n == least)) return s;
            if (exactly)
                PyErr_Format(PyExc_ValueError, "%s values to unpack (expected %zd, got %zd)",
                             n > least ? "too many" : "not enough", least, n);
            else
                PyErr_SetString(PyExc_IndexError, "tuple index out of range");
        }
        else if (s != nullptr)
            PyErr_SetString(PyExc_TypeError, "shape is not a tuple");
        Py_XDECREF(s);
        ok = false;
        return nullptr;
    }
    int item(PyObject* shape, Py_ssize_t i)
    {
        return ok ? static_cast<int>(PyLong_AsLongLong(PyTuple_GET_ITEM(shape, i))) : 0;
    }
    void dims4(PyObject* t, int& d0, int& d1, int& d2, int& d3)
    {
        PyObject* s = shape(t, 4, true);
        d0 = item(s, 0), d1 = item(s, 1), d2 = item(s, 2), d3 = item(s, 3);
        Py_XDECREF(s);
    }
    int dim(PyObject* t, Py_ssize_t i)  // negative: from the end
    {
        PyObject* s = shape(t, i < 0 ? -i : i + 1, false);
        const int v = s ? item(s, i < 0 ? PyTuple_GET_SIZE(s) + i : i) : 0;
        Py_XDECREF(s);
        return v;
    }
    int dtype(PyObject* t)
    {
        if (!ok) return 0;
        PyObject* d = PyObject_GetAttr(t, s_dtype);
        if (d != nullptr)
        {
            for (const DtypeCode& c : dtypes)
                if (c.dtype == d && c.code != kInt32)
                {
                    Py_DECREF(d);
                    return c.code;
                }
            PyErr_Format(PyExc_TypeError, "unsupported dtype %S", d);
            Py_DECREF(d);
        }
        ok = false;
        return 0;
    }
    int integer(PyObject* o)  // a Python int: nothing that merely converts to one (a device tensor would synchronize)
    {
        if (!ok) return 0;
        if (!PyLong_Check(o))
        {
            PyErr_Format(PyExc_TypeError, "an int is required, not %.100s", Py_TYPE(o)->tp_name);
            ok = false;
            return 0;
        }
        const long long v = PyLong_AsLongLong(o);
        if (v == -1 && PyErr_Occurred())
            ok = false;
        else if (v < INT_MIN || v > INT_MAX)
            refuse(PyExc_OverflowError, "%lld does not fit in 32 bits", v);
        return ok ? static_cast<int>(v) : 0;
    }
    int blocks(PyObject* num_blocks, PyObject* cache) { return num_blocks == Py_None ? dim(cache, 0) : integer(num_blocks); }
    float real(PyObject* o)  // whatever float() takes
    {
        if (!ok) return 0.0f;
        PyObject*    f = PyNumber_Float(o);
        const double v = f ? PyFloat_AS_DOUBLE(f) : 0.0;
        Py_XDECREF(f);
        if (f == nullptr) ok = false;
        return static_cast<float>(v);
    }
    bool refuse(PyObject* error, const char* format, ...)
    {
        va_list va;
        va_start(va, format);
        PyErr_FormatV(error, format, va);
        va_end(va);
        return ok = false;
    }
    // t's (or None's, where that is allowed) dtype is `code`, its sizes are `dims` (-1: any), it is contiguous, and it lies
    // on the device of `like`.
    bool holds(PyObject* t, const char* name, int code, std::initializer_list<long long> dims, PyObject* like, bool optional)
    {
        if (!ok || (optional && t == Py_None)) return ok;
        if (t == Py_None) return refuse(PyExc_TypeError, "%s is missing", name);
        PyObject* d = PyObject_GetAttr(t, s_dtype);
        if (d == nullptr) return ok = false;
        bool known = false;
        for (const DtypeCode& c : dtypes) known = known || (c.dtype == d && c.code == code);
        if (!known) refuse(PyExc_TypeError, "%s has the wrong dtype (%S)", name, d);
        Py_DECREF(d);
        if (!ok) return false;
        PyObject* s = shape(t, 0, false);
        if (s == nullptr) return false;
        bool same = PyTuple_GET_SIZE(s) == static_cast<Py_ssize_t>(dims.size());
        Py_ssize_t i = 0;
        for (long long v : dims)
        {
            if (same && v >= 0) same = PyLong_AsLongLong(PyTuple_GET_ITEM(s, i)) == v;
            ++i;
        }
        if (!same) refuse(PyExc_ValueError, "%s has the wrong shape %S", name, s);
        Py_DECREF(s);
        return ok && plain(t, name, like);
    }
    // t is contiguous and on the device of `like`.
    bool plain(PyObject* t, const char* name, PyObject* like)
    {
        if (!ok || t == Py_None) return ok;
        PyObject* c = PyObject_CallMethodNoArgs(t, s_is_contiguous);
        if (c == nullptr) return ok = false;
        const bool yes = c == Py_True;
        Py_DECREF(c);
        if (!yes) return refuse(PyExc_ValueError, "%s must be contiguous", name);
        if (t == like) return true;
        PyObject* a = PyObject_GetAttr(t, s_device);
        PyObject* b = a ? PyObject_GetAttr(like, s_device) : nullptr;
        const int eq = b ? PyObject_RichCompareBool(a, b, Py_EQ) : -1;
        Py_XDECREF(a);
        Py_XDECREF(b);
        if (eq < 0) return ok = false;
        return eq == 1 || refuse(PyExc_ValueError, "%s is on another device than the other tensors", name);
    }
    // t lies on the current device (a call without rows touches no device and may have its tensors anywhere).
    void current(PyObject* t, bool rows)
    {
        if (!ok || !rows) return;
        PyObject* c = PyObject_GetAttr(t, s_is_cuda);
        const bool gpu = c == Py_True;
        Py_XDECREF(c);
        if (c == nullptr) ok = false;
        else if (!gpu) refuse(PyExc_ValueError, "the tensors must be on the GPU");
        if (!ok) return;
        PyObject* d = PyObject_GetAttr(t, s_device);
        PyObject* i = d ? PyObject_GetAttr(d, s_index) : nullptr;
        PyObject* n = i ? PyObject_CallNoArgs(get_device) : nullptr;
        const int eq = n ? PyObject_RichCompareBool(i, n, Py_EQ) : -1;
        Py_XDECREF(d);
        Py_XDECREF(i);
        Py_XDECREF(n);
        if (eq < 0) ok = false;
        else if (eq == 0) refuse(PyExc_ValueError, "the tensors are on another device than the current one");
    }
    size_t nbytes(PyObject* t)
    {
        if (!ok || t == Py_None) return 0;
        PyObject*    n = PyObject_GetAttr(t, s_nbytes);
        const size_t v = n ? PyLong_AsSize_t(n) : 0;
        Py_XDECREF(n);
        if (PyErr_Occurred()) ok = false;
        return v;
    }
    // A stream argument: None is torch's current stream, else an object with cuda_stream, or a raw handle.
    void* stream(PyObject* o)
    {
        if (!ok) return nullptr;
        PyObject* h = nullptr;
        if (o == Py_None && !stream_ready)
        {
            h = PyObject_CallNoArgs(first_stream);
            stream_ready = h != nullptr;
        }
        else if (o == Py_None)
        {
            PyObject* dev = PyObject_CallNoArgs(get_device);
            h = dev ? PyObject_CallOneArg(raw_stream, dev) : nullptr;
            Py_XDECREF(dev);
        }
        else
        {
            h = PyObject_GetAttr(o, s_cuda_stream);
            if (h == nullptr && PyErr_ExceptionMatches(PyExc_AttributeError))
            {
                PyErr_Clear();
                h = PyNumber_Long(o);
            }
        }
        void* v = h ? PyLong_AsVoidPtr(h) : nullptr;
        Py_XDECREF(h);
        if (PyErr_Occurred()) ok = false;
        return v;
    }
};

bool count(Py_ssize_t got, Py_ssize_t want)
{
    if (got == want) return true;
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, got);
    return false;
}

// The C call, without the interpreter lock (as ctypes made it).
template <typename F>
PyObject* finish(const Reader& r, F call)
{
    if (!r.ok) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = call();
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

// k, v, k_cache, v_cache, block_table, context_lens, k_scale, v_scale, num_blocks, stream
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (!count(n, 10)) return nullptr;
    Reader r{a};
    int    B, S, Hkv, D;
    r.dims4(a[0], B, S, Hkv, D);
    const int  mb = r.dim(a[4], -1), N = r.blocks(a[8], a[2]), st = r.dtype(a[0]), ct = r.dtype(a[2]);
    void *     k = r.ptr(a[0]), *v = r.ptr(a[1]), *kc = r.ptr(a[2]), *vc = r.ptr(a[3]);
    auto *     bt = r.ptr<int32_t>(a[4]), *cx = r.ptr<int32_t>(a[5]);
    auto *     ks = r.ptr<float>(a[6]), *vs = r.ptr<float>(a[7]);
    void*      s = r.stream(a[9]);
    return finish(r, [&] { return fn.append(k, v, st, kc, vc, ct, ks, vs, bt, cx, B, S, Hkv, D, FFKV_BLOCK_SIZE, mb, N, s); });
}

// The tensors of a decode: q, out, k_cache, v_cache, k_scale, v_scale, block_table, context_lens at a[0 .. 7],
// max_context_len, scale, num_blocks at a[8 .. 10].
struct Decode
{
    int      B, Hq, D, Hkv, mb, N, qt, ct, mcl;
    float    scale;
    void *   q, *out, *kc, *vc;
    float *  ks, *vs;
    int32_t *bt, *cx;
    Decode(Reader& r, PyObject* const* a)
    {
        B = r.dim(a[0], 0), Hq = r.dim(a[0], -2), D = r.dim(a[0], -1), Hkv = r.dim(a[2], 2);
        mb = r.dim(a[6], -1), N = r.blocks(a[10], a[2]);
        q = r.ptr(a[0]), out = r.ptr(a[1]), qt = r.dtype(a[0]), kc = r.ptr(a[2]), vc = r.ptr(a[3]), ct = r.dtype(a[2]);
        ks = r.ptr<float>(a[4]), vs = r.ptr<float>(a[5]), bt = r.ptr<int32_t>(a[6]), cx = r.ptr<int32_t>(a[7]);
        mcl = r.integer(a[8]), scale = r.real(a[9]);
    }
};

// decode's 11, workspace, stream
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (!count(n, 13)) return nullptr;
    Reader       r{a};
    Decode       d(r, a);
    void*        ws = r.ptr(a[11]);
    const size_t wb = r.nbytes(a[11]);
    void*        s = r.stream(a[12]);
    return finish(r, [&] {
        return fn.decode(d.q, d.out, d.qt, d.kc, d.vc, d.ct, d.ks, d.vs, d.bt, d.cx, d.B, d.Hq, d.Hkv, d.D,
                         FFKV_BLOCK_SIZE, d.mb, d.N, d.mcl, d.scale, ws, wb, s);
    });
}

// decode's 11, shared_blocks, workspace, stream
PyObject* decode_shared(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (!count(n, 14)) return nullptr;
    Reader       r{a};
    Decode       d(r, a);
    const int    sb = r.integer(a[11]);
    void*        ws = r.ptr(a[12]);
    const size_t wb = r.nbytes(a[12]);
    void*        s = r.stream(a[13]);
    return finish(r, [&] {
        return fn.decode_shared(d.q, d.out, d.qt, d.kc, d.vc, d.ct, d.ks, d.vs, d.bt, d.cx, d.B, d.Hq, d.Hkv, d.D,
                                FFKV_BLOCK_SIZE, d.mb, d.N, d.mcl, d.scale, sb, ws, wb, s);
    });
}

// decode's 11, k_new, v_new, workspace, stream
PyObject* append_decode(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (!count(n, 15)) return nullptr;
    Reader       r{a};
    Decode       d(r, a);
    void *       k = r.ptr(a[11]), *v = r.ptr(a[12]);
    const int    st = r.dtype(a[11]);
    void*        ws = r.ptr(a[13]);
    const size_t wb = r.nbytes(a[13]);
    void*        s = r.stream(a[14]);
    return finish(r, [&] {
        return fn.append_decode(k, v, st, d.q, d.out, d.qt, d.kc, d.vc, d.ct, d.ks, d.vs, d.bt, d.cx, d.B, d.Hq, d.Hkv,
                                d.D, FFKV_BLOCK_SIZE, d.mb, d.N, d.mcl, d.scale, ws, wb, s);
    });
}

// A score rule at r: score_cap, slopes, window, key_begin [, key_end].
struct Rule
{
    float    cap = 0.0f;
    float*   slopes = nullptr;
    int      window = 0;
    int32_t *begin = nullptr, *end = nullptr;
};

// weights, prior, decay at w: fp32 [B, Hkv, T] or None, the same or None, a number.
struct Weights
{
    float * w = nullptr, *prior = nullptr;
    float   decay = 0.0f;
    int64_t stride = 0;
    Weights(Reader& r, PyObject* const* a, int B, int Hkv, PyObject* like)
    {
        r.holds(a[0], "weights", FFKV_DTYPE_F32, {B, Hkv, -1}, like, true);
        if (r.ok && a[0] != Py_None) stride = r.dim(a[0], 2);
        if (r.ok && a[0] == Py_None && a[1] != Py_None) r.refuse(PyExc_ValueError, "prior without weights");
        r.holds(a[1], "prior", FFKV_DTYPE_F32, {B, Hkv, stride}, like, true);
        decay = r.real(a[2]);
        w = r.ptr<float>(a[0]), prior = r.ptr<float>(a[1]);
    }
};

// The scales of an int8 [N, 16, Hkv] or fp8 [Hkv] cache; another cache's are not read.
void check_scales(Reader& r, PyObject* s, const char* name, int ct, PyObject* cache, int Hkv, PyObject* like)
{
    if (ct == FFKV_DTYPE_I8) r.holds(s, name, FFKV_DTYPE_F32, {r.dim(cache, 0), FFKV_BLOCK_SIZE, Hkv}, like, true);
    if (ct == FFKV_DTYPE_FP8_E4M3) r.holds(s, name, FFKV_DTYPE_F32, {Hkv}, like, true);
}

// num_blocks: at most the pool's pages
void check_blocks(Reader& r, int n, PyObject* cache)
{
    if (r.ok && n > r.dim(cache, 0)) r.refuse(PyExc_ValueError, "num_blocks %d is more than the caches' pages", n);
}

// Scratch of `need` bytes for one call without a workspace, from `make` (bytes, like, stream) -> a tensor or None: torch's
// allocator keeps it, where the library's stream-ordered memory is given back whenever the stream is waited for (a call that
// is waited for: 125 us against 59 in a row).  Owned until the call has been issued.
struct Scratch
{
    PyObject* t = nullptr;
    void*     ptr = nullptr;
    size_t    bytes = 0;
    Scratch(Reader& r, PyObject* given, PyObject* make, size_t need, PyObject* like, PyObject* stream)
    {
        if (!r.ok) return;
        if (given != Py_None)
        {
            t = Py_NewRef(given);
        }
        else if (need > 0)
        {
            PyObject* n = PyLong_FromSize_t(need);
            t = n ? PyObject_CallFunctionObjArgs(make, n, like, stream, nullptr) : nullptr;
            Py_XDECREF(n);
            if (t == nullptr) r.ok = false;
        }
        if (t == nullptr) return;
        ptr = r.ptr(t), bytes = r.nbytes(t);
    }
    ~Scratch() { Py_XDECREF(t); }
    Scratch(const Scratch&) = delete;
    Scratch& operator=(const Scratch&) = delete;
};

// decode's 11, k_new, v_new, score_cap, slopes, window, key_begin, weights, prior, decay, workspace, stream, scratch
PyObject* decode_scored(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (!count(n, 23)) return nullptr;
    Reader     r{a};
    Decode     d(r, a);
    PyObject*  q = a[0];
    PyObject*  sh = r.shape(q, 3, false);
    const bool four = r.ok && PyTuple_GET_SIZE(sh) == 4;
    if (r.ok && (PyTuple_GET_SIZE(sh) > 4 || (four && r.item(sh, 1) != 1)))
        r.refuse(PyExc_ValueError, "q must be [B, 1, Hq, D] or [B, Hq, D], got %S", sh);
    Py_XDECREF(sh);
    r.plain(q, "q", q);
    r.plain(a[1], "out", q);
    if (r.ok && r.dtype(a[1]) != d.qt) r.refuse(PyExc_TypeError, "out must have q's dtype");
    if (r.ok && r.nbytes(a[1]) != r.nbytes(q)) r.refuse(PyExc_ValueError, "out must have as many values as q");
    r.holds(a[2], "k_cache", d.ct, {-1, FFKV_BLOCK_SIZE, d.Hkv, d.D}, q, false);
    r.holds(a[3], "v_cache", d.ct, {r.dim(a[2], 0), FFKV_BLOCK_SIZE, d.Hkv, d.D}, q, false);
    check_scales(r, a[4], "k_scale", d.ct, a[2], d.Hkv, q);
    check_scales(r, a[5], "v_scale", d.ct, a[2], d.Hkv, q);
    r.holds(a[6], "block_table", kInt32, {d.B, -1}, q, false);
    r.holds(a[7], "context_lens", kInt32, {d.B}, q, false);
    check_blocks(r, d.N, a[2]);
    int st = d.qt;
    if (r.ok && (a[11] == Py_None) != (a[12] == Py_None)) r.refuse(PyExc_ValueError, "k_new and v_new come together");
    if (r.ok && a[11] != Py_None)
    {
        st = r.dtype(a[11]);
        r.holds(a[11], "k_new", st, {d.B, 1, d.Hkv, d.D}, q, false);
    }
    if (r.ok && a[12] != Py_None) r.holds(a[12], "v_new", st, {d.B, 1, d.Hkv, d.D}, q, false);
    Rule u;
    u.cap = r.real(a[13]);
    r.holds(a[14], "slopes", FFKV_DTYPE_F32, {d.Hq}, q, true);
    u.window = r.integer(a[15]);
    r.holds(a[16], "key_begin", kInt32, {d.B}, q, true);
    Weights w(r, a + 17, d.B, d.Hkv, q);
    r.plain(a[20], "workspace", q);
    r.current(q, d.B > 0);
    void *       k = r.ptr(a[11]), *v = r.ptr(a[12]);
    u.slopes = r.ptr<float>(a[14]), u.begin = r.ptr<int32_t>(a[16]);
    void*         s = r.stream(a[21]);
    const size_t  need = r.ok && a[20] == Py_None ? fn.decode_scored_bytes(d.qt, d.ct, d.B, d.Hq, d.Hkv, d.D, d.mb, d.mcl,
                                                                           u.window, w.w != nullptr)
                                                  : 0;
    const Scratch ws(r, a[20], a[22], need, q, a[21]);
    return finish(r, [&] {
        return fn.decode_scored(d.q, d.out, d.qt, d.kc, d.vc, d.ct, d.ks, d.vs, d.bt, d.cx, d.B, d.Hq, d.Hkv, d.D,
                                FFKV_BLOCK_SIZE, d.mb, d.N, d.mcl, d.scale, u.cap, u.slopes, u.window, u.begin, k, v, st,
                                w.w, w.prior, w.decay, w.stride, ws.ptr, ws.bytes, s);
    });
}

// decode's 11, stream
PyObject* decode_noalloc(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (!count(n, 12)) return nullptr;
    Reader r{a};
    Decode d(r, a);
    void*  s = r.stream(a[11]);
    return finish(r, [&] {
        return fn.decode_noalloc(d.q, d.out, d.qt, d.kc, d.vc, d.ct, d.ks, d.vs, d.bt, d.cx, d.B, d.Hq, d.Hkv, d.D,
                                 FFKV_BLOCK_SIZE, d.mb, d.N, d.mcl, d.scale, s);
    });
}

// q, out, k_cache, v_cache, k_scale, v_scale, block_table, context_lens, max_context_len, scale, num_blocks, stream,
// scratch (bytes, q, stream) -> a tensor or None
PyObject* prefill(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (!count(n, 13)) return nullptr;
    Reader r{a};
    int    B, S, Hq, D;
    r.dims4(a[0], B, S, Hq, D);
    const int   Hkv = r.dim(a[2], 2);
    const bool  paged = a[6] != Py_None;
    const int   mb = paged ? r.dim(a[6], -1) : 0, N = paged ? r.blocks(a[10], a[2]) : 0;
    void *      q = r.ptr(a[0]), *out = r.ptr(a[1]), *kc = r.ptr(a[2]), *vc = r.ptr(a[3]);
    const int   qt = r.dtype(a[0]), ct = r.dtype(a[2]);
    auto *      ks = r.ptr<float>(a[4]), *vs = r.ptr<float>(a[5]);
    auto *      bt = r.ptr<int32_t>(a[6]), *cx = r.ptr<int32_t>(a[7]);
    const int   mcl = r.integer(a[8]);
    const float scale = r.real(a[9]);
    void*       s = r.stream(a[11]);
    if (!r.ok) return nullptr;
    PyObject*    ws = nullptr;
    const size_t need = fn.prefill_bytes(qt, ct, B, S, Hq, Hkv, D, paged, mb, mcl);
    if (need > 0)
    {
        PyObject* nb = PyLong_FromSize_t(need);
        ws = nb ? PyObject_CallFunctionObjArgs(a[12], nb, a[0], a[11], nullptr) : nullptr;
        Py_XDECREF(nb);
        if (ws == nullptr) return nullptr;
    }
    void*        w = ws ? r.ptr(ws) : nullptr;
    const size_t wb = ws ? r.nbytes(ws) : 0;
    PyObject*    rc = finish(r, [&] {
        return fn.prefill(q, out, qt, kc, vc, ct, ks, vs, bt, cx, B, S, Hq, Hkv, D, FFKV_BLOCK_SIZE, mb, N, mcl, scale,
                             w, wb, s);
    });
    Py_XDECREF(ws);  // its memory goes back to the allocator of the call's stream, whose later work may reuse it
    return rc;
}

// q, out, k_cache, v_cache, k_scale, v_scale, block_table, context_lens, max_context_len, scale, num_blocks, score_cap,
// slopes, window, key_begin, key_end, stream, scratch (as prefill's)
PyObject* prefill_scored(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (!count(n, 18)) return nullptr;
    Reader    r{a};
    PyObject* q = a[0];
    int       B, S, Hq, D;
    r.dims4(q, B, S, Hq, D);
    const int  Hkv = r.dim(a[2], 2), qt = r.dtype(q), ct = r.dtype(a[2]);
    const bool paged = a[6] != Py_None;
    r.plain(q, "q", q);
    if (r.ok && r.dtype(a[1]) != qt) r.refuse(PyExc_TypeError, "out must have q's dtype");
    r.plain(a[1], "out", q);
    if (r.ok && r.nbytes(a[1]) != r.nbytes(q)) r.refuse(PyExc_ValueError, "out must have as many values as q");
    const int pages = paged ? r.dim(a[2], 0) : B, slots = paged ? FFKV_BLOCK_SIZE : S;
    r.holds(a[2], "k_cache", ct, {pages, slots, Hkv, D}, q, false);
    r.holds(a[3], "v_cache", ct, {pages, slots, Hkv, D}, q, false);
    check_scales(r, a[4], "k_scale", ct, a[2], Hkv, q);
    check_scales(r, a[5], "v_scale", ct, a[2], Hkv, q);
    int mb = 0, N = 0;
    if (paged)
    {
        r.holds(a[6], "block_table", kInt32, {B, -1}, q, false);
        r.holds(a[7], "context_lens", kInt32, {B}, q, false);
        mb = r.dim(a[6], 1), N = r.blocks(a[10], a[2]);
        check_blocks(r, N, a[2]);
    }
    else if (r.ok && a[7] != Py_None)
        r.refuse(PyExc_ValueError, "context_lens without a block table: contiguous keys begin at position 0");
    const int   mcl = r.integer(a[8]);
    const float scale = r.real(a[9]);
    Rule        u;
    u.cap = r.real(a[11]);
    r.holds(a[12], "slopes", FFKV_DTYPE_F32, {Hq}, q, true);
    u.window = r.integer(a[13]);
    r.holds(a[14], "key_begin", kInt32, {B, S}, q, true);
    r.holds(a[15], "key_end", kInt32, {B, S}, q, true);
    r.current(q, B > 0 && S > 0);
    void *out = r.ptr(a[1]), *qp = r.ptr(q), *kc = r.ptr(a[2]), *vc = r.ptr(a[3]);
    auto *ks = r.ptr<float>(a[4]), *vs = r.ptr<float>(a[5]);
    auto *bt = r.ptr<int32_t>(a[6]), *cx = r.ptr<int32_t>(a[7]);
    u.slopes = r.ptr<float>(a[12]), u.begin = r.ptr<int32_t>(a[14]), u.end = r.ptr<int32_t>(a[15]);
    void* s = r.stream(a[16]);
    if (!r.ok) return nullptr;
    PyObject*    ws = nullptr;
    const size_t need =
        fn.prefill_scored_bytes(qt, ct, B, S, Hq, Hkv, D, paged, mb, mcl, u.window, u.end != nullptr);
    if (need > 0)
    {
        PyObject* nb = PyLong_FromSize_t(need);
        ws = nb ? PyObject_CallFunctionObjArgs(a[17], nb, q, a[16], nullptr) : nullptr;
        Py_XDECREF(nb);
        if (ws == nullptr) return nullptr;
    }
    void*        w = ws ? r.ptr(ws) : nullptr;
    const size_t wb = ws ? r.nbytes(ws) : 0;
    PyObject*    rc = finish(r, [&] {
        return fn.prefill_scored(qp, out, qt, kc, vc, ct, ks, vs, bt, cx, B, S, Hq, Hkv, D, FFKV_BLOCK_SIZE, mb, N, mcl,
                                    scale, u.cap, u.slopes, u.window, u.begin, u.end, w, wb, s);
    });
    Py_XDECREF(ws);
    return rc;
}

// q, k_cache, k_scale, block_table, context_lens, max_context_len, scale, num_blocks, score_cap, slopes, window, key_begin,
// key_end, weights, prior, decay, workspace, stream, scratch
PyObject* attention_weights(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (!count(n, 19)) return nullptr;
    Reader    r{a};
    PyObject* q = a[0];
    int       B, S, Hq, D;
    r.dims4(q, B, S, Hq, D);
    const int Hkv = r.dim(a[1], 2), qt = r.dtype(q), ct = r.dtype(a[1]);
    r.plain(q, "q", q);
    r.holds(a[1], "k_cache", ct, {-1, FFKV_BLOCK_SIZE, Hkv, D}, q, false);
    check_scales(r, a[2], "k_scale", ct, a[1], Hkv, q);
    r.holds(a[3], "block_table", kInt32, {B, -1}, q, false);
    r.holds(a[4], "context_lens", kInt32, {B}, q, false);
    const int   mb = r.dim(a[3], 1), mcl = r.integer(a[5]);
    const float scale = r.real(a[6]);
    const int   N = r.blocks(a[7], a[1]);
    check_blocks(r, N, a[1]);
    Rule u;
    u.cap = r.real(a[8]);
    r.holds(a[9], "slopes", FFKV_DTYPE_F32, {Hq}, q, true);
    u.window = r.integer(a[10]);
    r.holds(a[11], "key_begin", kInt32, {B, S}, q, true);
    r.holds(a[12], "key_end", kInt32, {B, S}, q, true);
    Weights w(r, a + 13, B, Hkv, q);
    r.plain(a[16], "workspace", q);
    r.current(q, B > 0);  // (without queries the earlier weights still decay)
    void *qp = r.ptr(q), *kc = r.ptr(a[1]);
    auto* ks = r.ptr<float>(a[2]);
    auto *bt = r.ptr<int32_t>(a[3]), *cx = r.ptr<int32_t>(a[4]);
    u.slopes = r.ptr<float>(a[9]), u.begin = r.ptr<int32_t>(a[11]), u.end = r.ptr<int32_t>(a[12]);
    void*         s = r.stream(a[17]);
    const size_t  need = r.ok && a[16] == Py_None ? fn.weights_bytes(B, S, Hq, Hkv, D, mb, mcl) : 0;
    const Scratch ws(r, a[16], a[18], need, q, a[17]);
    return finish(r, [&] {
        return fn.attention_weights(qp, qt, kc, ct, ks, bt, cx, B, S, Hq, Hkv, D, FFKV_BLOCK_SIZE, mb, N, mcl, scale, u.cap,
                                    u.slopes, u.window, u.begin, u.end, w.w, w.prior, w.decay, w.stride, ws.ptr, ws.bytes,
                                    s);
    });
}

// weights, k_cache, v_cache, k_scale, v_scale, block_table, context_lens, keep, sinks, recent, dst_table, kept,
// kept_lens, weights_out, num_blocks, workspace, stream, scratch
PyObject* evict(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (!count(n, 18)) return nullptr;
    Reader    r{a};
    PyObject* w = a[0];
    const int B = r.dim(w, 0), Hkv = r.dim(a[1], 2), D = r.dim(a[1], 3), ct = r.dtype(a[1]);
    r.holds(w, "weights", FFKV_DTYPE_F32, {B, Hkv, -1}, w, false);
    r.holds(a[1], "k_cache", ct, {-1, FFKV_BLOCK_SIZE, Hkv, D}, w, false);
    r.holds(a[2], "v_cache", ct, {r.dim(a[1], 0), FFKV_BLOCK_SIZE, Hkv, D}, w, false);
    if (ct == FFKV_DTYPE_I8)
    {
        check_scales(r, a[3], "k_scale", ct, a[1], Hkv, w);
        check_scales(r, a[4], "v_scale", ct, a[1], Hkv, w);
    }
    r.holds(a[5], "block_table", kInt32, {B, -1}, w, false);
    r.holds(a[6], "context_lens", kInt32, {B}, w, false);
    const int keep = r.integer(a[7]), sinks = r.integer(a[8]), recent = r.integer(a[9]);
    r.holds(a[10], "dst_table", kInt32, {B, -1}, w, true);
    r.holds(a[11], "kept", kInt32, {B, Hkv, keep}, w, false);
    r.holds(a[12], "kept_lens", kInt32, {B}, w, false);
    r.holds(a[13], "weights_out", FFKV_DTYPE_F32, {B, Hkv, -1}, w, true);
    const int       mb = r.dim(a[5], 1), N = r.blocks(a[14], a[1]);
    const int       db = r.ok && a[10] != Py_None ? r.dim(a[10], 1) : 0;
    const long long stride = r.dim(w, 2), ostride = r.ok && a[13] != Py_None ? r.dim(a[13], 2) : 0;
    check_blocks(r, N, a[1]);
    r.current(w, B > 0);
    auto *wp = r.ptr<float>(w), *wo = r.ptr<float>(a[13]);
    void *kc = r.ptr(a[1]), *vc = r.ptr(a[2]);
    auto *ks = r.ptr<float>(a[3]), *vs = r.ptr<float>(a[4]);
    auto *bt = r.ptr<int32_t>(a[5]), *cx = r.ptr<int32_t>(a[6]), *dt = r.ptr<int32_t>(a[10]), *kp = r.ptr<int32_t>(a[11]),
         *kl = r.ptr<int32_t>(a[12]);
    r.plain(a[15], "workspace", w);
    void*         s = r.stream(a[16]);
    const size_t  need = r.ok && a[15] == Py_None ? fn.evict_bytes(B, Hkv, keep, stride, mb) : 0;
    const Scratch ws(r, a[15], a[17], need, w, a[16]);
    return finish(r, [&] {
        return fn.evict(wp, stride, cx, keep, sinks, recent, kc, vc, ct, ks, vs, bt, mb, dt, db, kp, kl, wo, ostride, B, Hkv,
                        D, FFKV_BLOCK_SIZE, N, ws.ptr, ws.bytes, s);
    });
}

// q or None, k, context_lens, theta, stream
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (!count(n, 5)) return nullptr;
    Reader r{a};
    int    B, S, Hkv, D;
    r.dims4(a[1], B, S, Hkv, D);
    const int   Hq = a[0] == Py_None ? 0 : r.dim(a[0], 2), st = r.dtype(a[1]);
    void *      q = r.ptr(a[0]), *k = r.ptr(a[1]);
    auto*       cx = r.ptr<int32_t>(a[2]);
    const float theta = r.real(a[3]);
    void*       s = r.stream(a[4]);
    return finish(r, [&] { return fn.rope(q, k, st, cx, B, S, Hq, Hkv, D, theta, s); });
}

// q or None, k, v, k_cache, v_cache, block_table, context_lens, theta, k_scale, v_scale, num_blocks, stream
PyObject* rope_append(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    if (!count(n, 12)) return nullptr;
    Reader r{a};
    int    B, S, Hkv, D;
    r.dims4(a[1], B, S, Hkv, D);
    const int   Hq = a[0] == Py_None ? 0 : r.dim(a[0], 2), mb = r.dim(a[5], -1), N = r.blocks(a[10], a[3]);
    const int   st = r.dtype(a[1]), ct = r.dtype(a[3]);
    void *      q = r.ptr(a[0]), *k = r.ptr(a[1]), *v = r.ptr(a[2]), *kc = r.ptr(a[3]), *vc = r.ptr(a[4]);
    auto *      bt = r.ptr<int32_t>(a[5]), *cx = r.ptr<int32_t>(a[6]);
    const float theta = r.real(a[7]);
    auto *      ks = r.ptr<float>(a[8]), *vs = r.ptr<float>(a[9]);
    void*       s = r.stream(a[11]);
    return finish(r, [&] {
        return fn.rope_append(q, k, v, st, kc, vc, ct, ks, vs, bt, cx, B, S, Hq, Hkv, D, FFKV_BLOCK_SIZE, mb, N, theta, s);
    });
}

// bind(addresses, [(dtype, code), ..], get_device, raw_stream, first_stream): the library's functions in Functions'
// order, torch's dtypes, and how the current stream's handle is found (first_stream() until it has succeeded once,
// which initialises torch's GPU state; then raw_stream(get_device())).
PyObject* bind(PyObject*, PyObject* args)
{
    PyObject *addrs, *types, *dev, *raw, *first;
    if (!PyArg_ParseTuple(args, "O!O!OOO", &PyTuple_Type, &addrs, &PyList_Type, &types, &dev, &raw, &first)) return nullptr;
    constexpr Py_ssize_t kFns = sizeof(Functions) / sizeof(void*);
    if (!count(PyTuple_GET_SIZE(addrs), kFns)) return nullptr;
    void* p[kFns];
    for (Py_ssize_t i = 0; i < kFns; ++i) p[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(addrs, i));
    std::vector<DtypeCode> d;
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(types); ++i)
    {
        DtypeCode c{};
        if (!PyArg_ParseTuple(PyList_GET_ITEM(types, i), "Oi", &c.dtype, &c.code)) return nullptr;
        d.push_back(c);
    }
    if (PyErr_Occurred()) return nullptr;
    for (const DtypeCode& c : d) Py_INCREF(c.dtype);
    dtypes = d;  // an earlier binding's references are kept: dtypes live as long as torch
    Py_INCREF(dev), Py_INCREF(raw), Py_INCREF(first);
    get_device = dev, raw_stream = raw, first_stream = first, stream_ready = false;
    __builtin_memcpy(&fn, p, sizeof(fn));
    Py_RETURN_NONE;
}

// The next call looks the stream up through first_stream() again (a forked child has no GPU state of its own).
PyObject* forget_stream(PyObject*, PyObject*)
{
    stream_ready = false;
    Py_RETURN_NONE;
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(decode_scored),  FAST(prefill_scored), FAST(evict), FAST(attention_weights),
                         FAST(append),         FAST(decode),  FAST(decode_shared), FAST(append_decode),
                         FAST(decode_noalloc), FAST(prefill), FAST(rope),          FAST(rope_append),
                         {"bind", bind, METH_VARARGS, nullptr},
                         {"forget_stream", forget_stream, METH_NOARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_front", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__front(void)
{
    s_shape = PyUnicode_InternFromString("shape");
    s_dtype = PyUnicode_InternFromString("dtype");
    s_data_ptr = PyUnicode_InternFromString("data_ptr");
    s_nbytes = PyUnicode_InternFromString("nbytes");
    s_cuda_stream = PyUnicode_InternFromString("cuda_stream");
    s_device = PyUnicode_InternFromString("device");
    s_index = PyUnicode_InternFromString("index");
    s_is_contiguous = PyUnicode_InternFromString("is_contiguous");
    s_is_cuda = PyUnicode_InternFromString("is_cuda");
    if (PyErr_Occurred()) return nullptr;
    return PyModule_Create(&module);
}
