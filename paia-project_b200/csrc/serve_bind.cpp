// CPython extension _paia_serve: the checks and the struct of a serving call (paia_gemv.serve) in C, 0.5 us instead of 5 us
// in Python. It reads tensors through the DLPack exchange functions that torch.Tensor publishes
// (__dlpack_c_exchange_api__), links neither torch nor the GEMV library (the caller passes the entry points' addresses),
// and decides nothing: whatever it does not find exactly as a plain call has it (another type, shape, layout or device, a
// tensor subclass, an error), it answers None, and the Python code makes the call or raises.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/dlpack.h>
#include <math.h>
#include <stdint.h>
#include "paia_gemv.h"

namespace {

const DLPackExchangeAPI* g_api = nullptr;
PyObject* g_tensor = nullptr;                    // torch.Tensor
using Call = int (*)(const void*, void*);
using Device = int (*)(void);

enum Kind { kBf16, kF32, kF64, kI32, kE4m3, kU8 };

bool is_kind(const DLDataType& t, Kind k) {
    if (t.lanes != 1) return false;
    switch (k) {
        case kBf16: return t.code == kDLBfloat && t.bits == 16;
        case kF32: return t.code == kDLFloat && t.bits == 32;
        case kF64: return t.code == kDLFloat && t.bits == 64;
        case kI32: return t.code == kDLInt && t.bits == 32;
        case kU8: return t.code == kDLUInt && t.bits == 8;
        default: return t.code == kDLFloat8_e4m3fn && t.bits == 8;
    }
}

// A tensor argument: plain torch.Tensor on CUDA device `device`; a stride along a dimension of one is 0 (never used).
struct Arg {
    DLTensor t;
    bool read(PyObject* o, int device) {
        if ((PyObject*)Py_TYPE(o) != g_tensor) return false;
        if (g_api->dltensor_from_py_object_no_sync(o, &t)) {
            PyErr_Clear();
            return false;
        }
        return t.device.device_type == kDLCUDA && t.device.device_id == device && (t.strides || t.ndim == 0);
    }
    bool is(PyObject* o, int device, Kind k, int ndim) { return read(o, device) && t.ndim == ndim && is_kind(t.dtype, k); }
    long long n(int i) const { return t.shape[i]; }
    long long stride(int i) const { return t.shape[i] == 1 ? 0 : t.strides[i]; }
    bool dense_last() const { return t.shape[t.ndim - 1] == 1 || t.strides[t.ndim - 1] == 1; }
    void* ptr() const { return static_cast<char*>(t.data) + t.byte_offset; }
    // contiguous [count], or None: a null pointer
    bool flat(PyObject* o, int device, Kind k, long long count, const void** p) {
        *p = nullptr;
        if (o == Py_None) return true;
        if (!is(o, device, k, 1) || n(0) != count || !dense_last()) return false;
        *p = ptr();
        return true;
    }
};

bool small(long long v) { return v >= 0 && v <= 0x7fffffff; }

bool integer(PyObject* o, long long* v) {
    if (!PyLong_CheckExact(o)) return false;
    int over = 0;
    *v = PyLong_AsLongLongAndOverflow(o, &over);
    return !over;
}
bool number(PyObject* o, double* v) {
    if (PyFloat_CheckExact(o)) *v = PyFloat_AS_DOUBLE(o);
    else if (PyLong_CheckExact(o)) *v = PyLong_AsDouble(o);
    else return false;
    if (PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}
// The stream argument (None: torch's current one).
bool stream_of(PyObject* o, int device, void** s) {
    if (o == Py_None) return g_api->current_work_stream(kDLCUDA, device, s) == 0;
    long long v = 0;
    if (!integer(o, &v)) return false;
    *s = reinterpret_cast<void*>((uintptr_t)v);
    return true;
}
template <class T>
T address(PyObject* o) { return reinterpret_cast<T>(PyLong_AsVoidPtr(o)); }

// The current device through the library's own runtime; -1 where there is none.
int current(PyObject* entry, PyObject* device) {
    const Device f = address<Device>(device);
    return !f || !address<Call>(entry) ? -1 : f();
}

PyObject* none() {
    if (PyErr_Occurred()) PyErr_Clear();
    Py_RETURN_NONE;
}

struct Pools {
    Arg k, v;
    int cache;
    bool read(PyObject* ko, PyObject* vo, int device) {
        if (!k.read(ko, device) || !v.read(vo, device) || k.t.ndim != 4 || v.t.ndim != 4) return false;
        cache = is_kind(k.t.dtype, kBf16) ? 0 : is_kind(k.t.dtype, kE4m3) ? 1 : -1;
        if (cache < 0 || !is_kind(v.t.dtype, cache ? kE4m3 : kBf16)) return false;
        for (int i = 0; i < 4; ++i)
            if (k.n(i) != v.n(i) || !small(k.n(i))) return false;
        return k.dense_last() && v.dense_last();
    }
};

// (entry, device, q, k_pages, v_pages, page_table, lens, out, workspace pointer, workspace sizes, scale, window, k_scale,
//  v_scale, lse, stream)
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 16) return none();
    const int dev = current(a[0], a[1]);
    Arg q, out, table, lens, ks, vs, lse;
    Pools pool;
    paia_gemv_attn s{};
    const void *lp, *kp, *vp;
    long long window = 0;
    double scale = 0.0;
    if (dev < 0 || !q.is(a[2], dev, kBf16, 3) || !pool.read(a[3], a[4], dev) || !table.is(a[5], dev, kI32, 2) ||
        !out.is(a[7], dev, kBf16, 3))
        return none();
    const long long b = q.n(0), h = q.n(1), hd = q.n(2), kv = pool.k.n(2);
    if (!small(b) || !small(h) || !small(hd) || !small(table.n(1)) || pool.k.n(3) != hd || !kv || h % kv || table.n(0) != b ||
        out.n(0) != b || out.n(1) != h || out.n(2) != hd || !q.dense_last() || !out.dense_last() || !table.dense_last() ||
        !lens.flat(a[6], dev, kI32, b, &lp) || !lp || !ks.flat(a[12], dev, kF32, kv, &kp) ||
        !vs.flat(a[13], dev, kF32, kv, &vp) || !integer(a[11], &window) || !small(window))
        return none();
    // the workspace's (device, heads, kv_heads, head_dim)
    PyObject* z = a[9];
    const long long want[4] = {dev, h, kv, hd};
    if (!PyTuple_CheckExact(z) || PyTuple_GET_SIZE(z) != 4) return none();
    for (int i = 0; i < 4; ++i) {
        long long v = -1;
        if (!integer(PyTuple_GET_ITEM(z, i), &v) || v != want[i]) return none();
    }
    if (a[14] != Py_None) {
        if (!lse.is(a[14], dev, kF32, 2) || lse.n(0) != b || lse.n(1) != h || !lse.dense_last()) return none();
        s.lse = static_cast<float*>(lse.ptr());
        s.lse_batch = lse.stride(0);
    }
    if (a[10] == Py_None) scale = pow((double)hd, -0.5);
    else if (!number(a[10], &scale)) return none();
    void* stream = nullptr;
    if (!stream_of(a[15], dev, &stream)) return none();
    s.q = q.ptr();
    s.k = pool.k.ptr();
    s.v = pool.v.ptr();
    s.page_table = static_cast<const int*>(table.ptr());
    s.lens = static_cast<const int*>(lp);
    s.k_scale = static_cast<const float*>(kp);
    s.v_scale = static_cast<const float*>(vp);
    s.out = out.ptr();
    s.workspace = address<void*>(a[8]);
    s.q_batch = q.stride(0);
    s.q_head = q.stride(1);
    s.out_batch = out.stride(0);
    s.out_head = out.stride(1);
    s.table_batch = table.stride(0);
    s.k_page = pool.k.stride(0);
    s.k_token = pool.k.stride(1);
    s.k_head = pool.k.stride(2);
    s.v_page = pool.v.stride(0);
    s.v_token = pool.v.stride(1);
    s.v_head = pool.v.stride(2);
    s.batch = (int)b;
    s.heads = (int)h;
    s.kv_heads = (int)kv;
    s.head_dim = (int)hd;
    s.cache = pool.cache;
    s.num_pages = (int)pool.k.n(0);
    s.page_size = (int)pool.k.n(1);
    s.max_pages = (int)table.n(1);
    s.window = (int)window;
    s.scale = (float)scale;
    return PyErr_Occurred() ? none() : PyLong_FromLong(address<Call>(a[0])(&s, stream));
}

// (entry, device, qkv, positions, inv_freq, q_out, k_pages, v_pages, page_table, seq, q_norm, k_norm, eps, interleaved,
//  k_scale, v_scale, k_out, stream): calls with a cache
PyObject* qkv_rope_cache(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 18) return none();
    const int dev = current(a[0], a[1]);
    Arg x, q, table, pos, freq, seq, qn, kn, ks, vs, ko;
    Pools pool;
    paia_gemv_rope_cache s{};
    const void *pp, *sp, *qp, *np, *kp, *vp;
    double eps = 0.0;
    if (dev < 0 || !x.is(a[2], dev, kBf16, 2) || !q.is(a[5], dev, kBf16, 3) || !pool.read(a[6], a[7], dev) ||
        !table.is(a[8], dev, kI32, 2) || !freq.is(a[4], dev, kF64, 1))
        return none();
    const long long t = q.n(0), h = q.n(1), hd = q.n(2), kv = pool.k.n(2);
    if (!small(t) || !small(h) || !small(hd) || !small(2 * freq.n(0)) || !small(table.n(0)) || !small(table.n(1)) ||
        pool.k.n(3) != hd || x.n(0) != t || x.n(1) != (h + 2 * kv) * hd || !x.dense_last() || !q.dense_last() ||
        !table.dense_last() || !freq.dense_last() || !pos.flat(a[3], dev, kI32, t, &pp) || !pp ||
        !seq.flat(a[9], dev, kI32, t, &sp) || (!sp && table.n(0) < t) || !qn.flat(a[10], dev, kF32, hd, &qp) ||
        !kn.flat(a[11], dev, kF32, hd, &np) || !ks.flat(a[14], dev, kF32, kv, &kp) || !vs.flat(a[15], dev, kF32, kv, &vp) ||
        !number(a[12], &eps))
        return none();
    if (a[16] != Py_None) {
        if (!ko.is(a[16], dev, kBf16, 3) || ko.n(0) != t || ko.n(1) != kv || ko.n(2) != hd || !ko.dense_last()) return none();
        s.k_out = ko.ptr();
        s.ko_token = ko.stride(0);
        s.ko_head = ko.stride(1);
    }
    const int inter = PyObject_IsTrue(a[13]);
    void* stream = nullptr;
    if (inter < 0 || !stream_of(a[17], dev, &stream)) return none();
    s.qkv = x.ptr();
    s.pos = static_cast<const int*>(pp);
    s.seq = static_cast<const int*>(sp);
    s.inv_freq = static_cast<const double*>(freq.ptr());
    s.q_norm = static_cast<const float*>(qp);
    s.k_norm = static_cast<const float*>(np);
    s.page_table = static_cast<const int*>(table.ptr());
    s.k_scale = static_cast<const float*>(kp);
    s.v_scale = static_cast<const float*>(vp);
    s.q_out = q.ptr();
    s.k = pool.k.ptr();
    s.v = pool.v.ptr();
    s.qkv_token = x.stride(0);
    s.q_token = q.stride(0);
    s.q_head = q.stride(1);
    s.table_seq = table.stride(0);
    s.k_page = pool.k.stride(0);
    s.k_row = pool.k.stride(1);
    s.k_head = pool.k.stride(2);
    s.v_page = pool.v.stride(0);
    s.v_row = pool.v.stride(1);
    s.v_head = pool.v.stride(2);
    s.tokens = (int)t;
    s.sequences = (int)table.n(0);
    s.heads = (int)h;
    s.kv_heads = (int)kv;
    s.head_dim = (int)hd;
    s.rot = (int)(2 * freq.n(0));
    s.interleaved = inter;
    s.cache = pool.cache;
    s.num_pages = (int)pool.k.n(0);
    s.page_size = (int)pool.k.n(1);
    s.max_pages = (int)table.n(1);
    s.eps = (float)eps;
    return PyErr_Occurred() ? none() : PyLong_FromLong(address<Call>(a[0])(&s, stream));
}

// (entry, device, x, a, b, adapter, out, base, scaling, ranks, stream)
PyObject* lora(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 11) return none();
    const int dev = current(a[0], a[1]);
    Arg x, A, B, out, base, ad, sc, rk;
    paia_gemv_lora_args s{};
    const void *ap, *cp, *rp;
    if (dev < 0 || !x.is(a[2], dev, kBf16, 2) || !A.is(a[3], dev, kBf16, 3) || !B.is(a[4], dev, kBf16, 3) ||
        !out.is(a[6], dev, kBf16, 2))
        return none();
    const long long m = x.n(0), k = x.n(1), ads = A.n(0), r = A.n(1), cols = B.n(1);
    if (!small(m) || !small(k) || !small(ads) || !small(r) || !small(cols) || A.n(2) != k || B.n(0) != ads || B.n(2) != r ||
        out.n(0) != m || out.n(1) != cols || !x.dense_last() || !A.dense_last() || !B.dense_last() || !out.dense_last() ||
        !ad.flat(a[5], dev, kI32, m, &ap) || !ap || !sc.flat(a[8], dev, kF32, ads, &cp) || !rk.flat(a[9], dev, kI32, ads, &rp))
        return none();
    if (a[7] != Py_None) {
        if (!base.is(a[7], dev, kBf16, 2) || base.n(0) != m || base.n(1) != cols || !base.dense_last()) return none();
        s.base = base.ptr();
        s.base_row = base.stride(0);
    }
    void* stream = nullptr;
    if (!stream_of(a[10], dev, &stream)) return none();
    s.x = x.ptr();
    s.a = A.ptr();
    s.b = B.ptr();
    s.adapter = static_cast<const int*>(ap);
    s.ranks = static_cast<const int*>(rp);
    s.scaling = static_cast<const float*>(cp);
    s.out = out.ptr();
    s.x_row = x.stride(0);
    s.out_row = out.stride(0);
    s.a_adapter = A.stride(0);
    s.a_row = A.stride(1);
    s.b_adapter = B.stride(0);
    s.b_row = B.stride(1);
    s.M = (int)m;
    s.N = (int)cols;
    s.K = (int)k;
    s.rank = (int)r;
    s.adapters = (int)ads;
    return PyErr_Occurred() ? none() : PyLong_FromLong(address<Call>(a[0])(&s, stream));
}

// The integers of a tuple of n.
bool integers(PyObject* o, int n, long long* v) {
    if (!PyTuple_CheckExact(o) || PyTuple_GET_SIZE(o) != n) return false;
    for (int i = 0; i < n; ++i)
        if (!integer(PyTuple_GET_ITEM(o, i), v + i)) return false;
    return true;
}

// (entry, device, logits, routing pointers (weights, experts, places, rows, offsets, workspace), routing sizes (device, tokens,
//  experts, top_k), scoring, bias, renormalise, scale, positions, stream)
PyObject* route(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 11) return none();
    const int dev = current(a[0], a[1]);
    Arg x, bias, pos;
    long long ptr[6], size[4];
    const void *bp, *pp;
    double scale = 0.0;
    paia_gemv_route_args s{};
    if (dev < 0 || !x.read(a[2], dev) || x.t.ndim != 2 || !x.dense_last() || !integers(a[3], 6, ptr) || !integers(a[4], 4, size) ||
        size[0] != dev || x.n(0) != size[1] || x.n(1) != size[2] || !small(size[1]) || !small(size[2]) || !small(size[3]))
        return none();
    s.logits_type = is_kind(x.t.dtype, kBf16) ? 0 : is_kind(x.t.dtype, kF32) ? 1 : -1;
    if (s.logits_type < 0 || !PyUnicode_CheckExact(a[5])) return none();
    s.scoring = PyUnicode_CompareWithASCIIString(a[5], "softmax") == 0 ? 0
                : PyUnicode_CompareWithASCIIString(a[5], "sigmoid") == 0 ? 1 : -1;
    if (s.scoring < 0 || !bias.flat(a[6], dev, kF32, size[2], &bp) || (bp && !s.scoring) ||
        !pos.flat(a[9], dev, kI32, size[1], &pp) || !number(a[8], &scale))
        return none();
    const int renorm = PyObject_IsTrue(a[7]);
    void* stream = nullptr;
    if (renorm < 0 || !stream_of(a[10], dev, &stream)) return none();
    s.logits = x.ptr();
    s.bias = static_cast<const float*>(bp);
    s.pos = static_cast<const int*>(pp);
    s.weights = reinterpret_cast<float*>((uintptr_t)ptr[0]);
    s.ids = reinterpret_cast<int*>((uintptr_t)ptr[1]);
    s.places = reinterpret_cast<int*>((uintptr_t)ptr[2]);
    s.rows = reinterpret_cast<int*>((uintptr_t)ptr[3]);
    s.offsets = reinterpret_cast<int*>((uintptr_t)ptr[4]);
    s.workspace = reinterpret_cast<void*>((uintptr_t)ptr[5]);
    s.logits_row = x.stride(0);
    s.tokens = (int)size[1];
    s.experts = (int)size[2];
    s.top_k = (int)size[3];
    s.renormalise = renorm;
    s.scale = (float)scale;
    return PyErr_Occurred() ? none() : PyLong_FromLong(address<Call>(a[0])(&s, stream));
}

// (entry, device, w, x, offsets, out, workspace pointer, workspace device, scales, rows, silu, stream)
PyObject* expert_matmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 12) return none();
    const int dev = current(a[0], a[1]);
    Arg w, x, off, out, sc, rows;
    const void *op, *rp;
    long long ws_dev = -1;
    paia_gemv_expert_args s{};
    if (dev < 0 || !w.read(a[2], dev) || w.t.ndim != 3 || !w.dense_last() || !x.is(a[3], dev, kBf16, 2) || !x.dense_last() ||
        !out.is(a[5], dev, kBf16, 2) || !out.dense_last() || !integer(a[7], &ws_dev) || ws_dev != dev)
        return none();
    s.kind = is_kind(w.t.dtype, kBf16) ? 0 : is_kind(w.t.dtype, kE4m3) || is_kind(w.t.dtype, kU8) ? 1 : -1;
    const int silu = PyObject_IsTrue(a[10]);
    const long long e = w.n(0), rn = w.n(1), k = w.n(2), m = out.n(0), cols = silu > 0 ? rn / 2 : rn;
    if (s.kind < 0 || silu < 0 || !small(e) || !small(rn) || !small(k) || !small(m) || !small(x.n(0)) || x.n(1) != k ||
        out.n(1) != cols || (silu && rn % 2) || !off.flat(a[4], dev, kI32, e + 1, &op) || !op ||
        !rows.flat(a[9], dev, kI32, m, &rp) || (!rp && x.n(0) < m))
        return none();
    if (s.kind == 1) {
        if (!sc.is(a[8], dev, kF32, 2) || sc.n(0) != e || sc.n(1) != rn || !sc.dense_last()) return none();
        s.scales = static_cast<const float*>(sc.ptr());
        s.scale_expert = sc.stride(0);
    } else if (a[8] != Py_None) {
        return none();
    }
    void* stream = nullptr;
    if (!stream_of(a[11], dev, &stream)) return none();
    s.w = w.ptr();
    s.x = x.ptr();
    s.rows = static_cast<const int*>(rp);
    s.offsets = static_cast<const int*>(op);
    s.out = out.ptr();
    s.workspace = address<void*>(a[6]);
    s.w_expert = w.stride(0);
    s.w_row = rn > 1 ? w.stride(1) : k;
    s.x_row = x.stride(0);
    s.out_row = out.stride(0);
    s.experts = (int)e;
    s.M = (int)m;
    s.N = (int)rn;
    s.K = (int)k;
    s.x_rows = (int)x.n(0);
    s.silu = silu;
    return PyErr_Occurred() ? none() : PyLong_FromLong(address<Call>(a[0])(&s, stream));
}

// (entry, device, h, x, h_out, out, places, weights, post, gate, scale, pre, eps, stream)
PyObject* block_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 14) return none();
    const int dev = current(a[0], a[1]);
    Arg h, x, ho, out, pl, wt, post, pre, gate;
    const void *qp, *np;
    double scale = 0.0, eps = 0.0;
    paia_gemv_block_norm_args s{};
    if (dev < 0 || !h.is(a[2], dev, kBf16, 2) || !h.dense_last() || (a[3] == Py_None) != (a[4] == Py_None)) return none();
    const long long t = h.n(0), hid = h.n(1);
    if (!small(t) || !small(hid) || !post.flat(a[8], dev, kF32, hid, &qp) || !pre.flat(a[11], dev, kF32, hid, &np) ||
        !number(a[10], &scale) || !number(a[12], &eps))
        return none();
    if (a[6] != Py_None) {
        if (!pl.is(a[6], dev, kI32, 2) || !wt.is(a[7], dev, kF32, 2) || pl.n(0) != t || wt.n(0) != t || wt.n(1) != pl.n(1) ||
            !small(pl.n(1)) || pl.n(1) < 1 || !pl.dense_last() || !wt.dense_last())
            return none();
        s.places = static_cast<const int*>(pl.ptr());
        s.weights = static_cast<const float*>(wt.ptr());
        s.places_row = pl.stride(0);
        s.weights_row = wt.stride(0);
        s.top_k = (int)pl.n(1);
    } else if (a[7] != Py_None) {
        return none();
    }
    if (a[3] != Py_None) {
        if (!x.is(a[3], dev, kBf16, 2) || !ho.is(a[4], dev, kBf16, 2) || x.n(1) != hid || !small(x.n(0)) || ho.n(0) != t ||
            ho.n(1) != hid || !x.dense_last() || !ho.dense_last() || (!s.places && x.n(0) < t))
            return none();
        s.x = x.ptr();
        s.x_row = x.stride(0);
        s.x_rows = (int)x.n(0);
        s.h_out = ho.ptr();
        s.h_out_row = ho.stride(0);
    }
    if (a[5] != Py_None) {
        if (!out.is(a[5], dev, kBf16, 2) || out.n(0) != t || out.n(1) != hid || !out.dense_last()) return none();
        s.out = out.ptr();
        s.out_row = out.stride(0);
    }
    if (a[9] != Py_None) {
        if (!gate.read(a[9], dev) || !is_kind(gate.t.dtype, kBf16) || gate.t.ndim < 1 || gate.t.ndim > 2 || !gate.dense_last())
            return none();
        const long long cols = gate.n(gate.t.ndim - 1);
        if (!(gate.t.ndim == 1 ? cols == hid : gate.n(0) == t && (cols == hid || cols == 1))) return none();
        s.gate = gate.ptr();
        s.gate_row = gate.t.ndim == 2 ? gate.stride(0) : 0;
        s.gate_col = cols == hid;
    }
    void* stream = nullptr;
    if (!stream_of(a[13], dev, &stream)) return none();
    s.h = h.ptr();
    s.h_row = h.stride(0);
    s.post = static_cast<const float*>(qp);
    s.pre = static_cast<const float*>(np);
    s.tokens = (int)t;
    s.hidden = (int)hid;
    s.eps = (float)eps;
    s.scale = (float)scale;
    return PyErr_Occurred() ? none() : PyLong_FromLong(address<Call>(a[0])(&s, stream));
}

// (torch.Tensor, its __dlpack_c_exchange_api__ capsule) -> whether calls can be made
PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 2 || !PyCapsule_IsValid(a[1], "dlpack_exchange_api")) Py_RETURN_FALSE;
    const auto* api = static_cast<const DLPackExchangeAPI*>(PyCapsule_GetPointer(a[1], "dlpack_exchange_api"));
    if (!api || api->header.version.major != DLPACK_MAJOR_VERSION || !api->dltensor_from_py_object_no_sync ||
        !api->current_work_stream)
        Py_RETURN_FALSE;
    Py_INCREF(a[0]);
    g_tensor = a[0];
    g_api = api;
    Py_RETURN_TRUE;
}

PyMethodDef kMethods[] = {
    {"init", (PyCFunction)(void (*)(void))init, METH_FASTCALL, nullptr},
    {"paged_attention", (PyCFunction)(void (*)(void))paged_attention, METH_FASTCALL, nullptr},
    {"qkv_rope_cache", (PyCFunction)(void (*)(void))qkv_rope_cache, METH_FASTCALL, nullptr},
    {"lora", (PyCFunction)(void (*)(void))lora, METH_FASTCALL, nullptr},
    {"route", (PyCFunction)(void (*)(void))route, METH_FASTCALL, nullptr},
    {"expert_matmul", (PyCFunction)(void (*)(void))expert_matmul, METH_FASTCALL, nullptr},
    {"block_norm", (PyCFunction)(void (*)(void))block_norm, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_paia_serve", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paia_serve(void) { return PyModule_Create(&kModule); }
