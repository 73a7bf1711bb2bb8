// The per-layer entry points of a decode step, called straight from torch
// tensors. Through ctypes a fused append + attend spends about half of its 11.4
// us on the host in Python: four descriptors keyed by (pointer, type, shape,
// strides), a slot tuple, two foreign calls with nine converted arguments. Read
// from the tensors here, the call takes 7.7 us (30-layer frame of one stream),
// less than its two short launches do on the GPU.
//
// Every function returns the runtime's code (0 or negative), or 1 where an
// argument is not in the plain form it reads: an exact torch.Tensor on the GPU
// (contiguous where the Python wrapper would have made it so), exact ints in
// lists or tuples. Nothing has happened then, and the caller takes its general
// path, which converts or refuses the call; a stream that cannot be bound goes
// there too. Nothing is kept between calls.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <climits>

#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/impl/DeviceGuardImplInterface.h>
#include <torch/csrc/autograd/python_variable.h>

#include "kvrt.h"

namespace {

constexpr int kMaxSlots = 64, kMaxPositions = 256;
constexpr long kGeneral = 1;

struct Api {
    decltype(&kvrt_bind_stream) bind;
    decltype(&kvrt_append_attend_async) append_attend;
    decltype(&kvrt_attend_decode_async) attend;
    decltype(&kvrt_attend_talker_async) talker;
    decltype(&kvrt_write_positions_async) write;
    decltype(&kvrt_append_gather_async) gather;
    decltype(&kvrt_attend_tensors_async) tensors;
    decltype(&kvrt_attend_shared_async) shared;
} api;

PyObject *talker_mask_type;

bool read_int(PyObject *o, int32_t &out) {
    if (!PyLong_CheckExact(o)) return false;
    int over = 0;
    const long v = PyLong_AsLongAndOverflow(o, &over);
    if (over || v < INT_MIN || v > INT_MAX) return false;
    out = (int32_t)v;
    return true;
}

bool read_float(PyObject *o, float &out) {
    if (!PyFloat_CheckExact(o)) return false;
    out = (float)PyFloat_AS_DOUBLE(o);
    return true;
}

// Items of an exact list or tuple (borrowed), or -1.
Py_ssize_t items(PyObject *o, PyObject **&at) {
    if (!PyList_CheckExact(o) && !PyTuple_CheckExact(o)) return -1;
    at = PySequence_Fast_ITEMS(o);
    return PySequence_Fast_GET_SIZE(o);
}

int read_ints(PyObject *o, int32_t *out, int cap) {
    PyObject **at;
    const Py_ssize_t n = items(o, at);
    if (n < 0 || n > cap) return -1;
    for (Py_ssize_t i = 0; i < n; ++i)
        if (!read_int(at[i], out[i])) return -1;
    return (int)n;
}

int dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kBFloat16: return KVRT_BF16;
        case at::kChar: return KVRT_INT8;
        case at::kFloat: return KVRT_FP32;
        case at::kBool: return KVRT_BOOL;
        case at::kInt: return KVRT_INT32;
        case at::kLong: return KVRT_INT64;
        default: return -1;
    }
}

bool read_tensor(PyObject *o, bool contiguous, kvrt_tensor &d) {
    if (!THPVariable_CheckExact(o)) return false;
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.dim() > KVRT_MAX_RANK) return false;
    if (contiguous && !t.is_contiguous()) return false;
    d = kvrt_tensor{};
    d.dtype = dtype_code(t.scalar_type());
    if (d.dtype < 0) return false;
    d.data = t.data_ptr();
    d.ndim = (int32_t)t.dim();
    for (int i = 0; i < d.ndim; ++i) {
        d.dims[i] = t.size(i);
        d.strides[i] = t.stride(i);
    }
    return true;
}

bool read_mask(PyObject *o, kvrt_talker_mask &m) {
    if ((PyObject *)Py_TYPE(o) != talker_mask_type) return false;
    static const char *const names[6] = {"prefix_start",   "audio_start",           "prefix_position",
                                         "audio_position", "prefix_attention_mode", "visible_prefix_count"};
    int32_t *const at[6] = {&m.prefix_start,   &m.audio_start,           &m.prefix_position,
                            &m.audio_position, &m.prefix_attention_mode, &m.visible_prefix_count};
    for (int i = 0; i < 6; ++i) {
        PyObject *v = PyObject_GetAttrString(o, names[i]);
        const bool ok = v && read_int(v, *at[i]);
        Py_XDECREF(v);
        if (!ok) return false;
    }
    PyObject *v = PyObject_GetAttrString(o, "prefix_log_gate");
    const bool ok = v && read_float(v, m.prefix_log_gate);
    Py_XDECREF(v);
    return ok;
}

// The leading arguments of a runtime call: context, stream, layer, slots.
struct Head {
    kvrt_ctx *ctx;
    void *stream;
    int32_t layer, n, slots[kMaxSlots];

    bool read(PyObject *const *a) {
        ctx = static_cast<kvrt_ctx *>(PyLong_AsVoidPtr(a[0]));
        stream = PyLong_AsVoidPtr(a[1]);
        if (!ctx || !read_int(a[2], layer)) return false;
        n = read_ints(a[3], slots, kMaxSlots);
        return n >= 0;
    }
    bool bind() const { return api.bind(ctx, stream) == KVRT_OK; }
};

// Runs body (parse, then call), any C++ or Python error of the parse meaning
// the general path.
template <class F>
PyObject *guarded(Py_ssize_t nargs, Py_ssize_t want, F body) {
    long rc = kGeneral;
    try {
        if (nargs == want) rc = body();
    } catch (...) {  // e.g. a tensor without storage
        rc = kGeneral;
    }
    if (PyErr_Occurred()) PyErr_Clear();
    return PyLong_FromLong(rc);
}

// The runtime call, the parse done. An exception out of it (its vectors can
// fail to allocate) is a device error and not the general path's to repeat: the
// call may have mapped pages or enqueued work. The interpreter lock is held
// again before anything else runs.
template <class F>
long without_gil(F call) {
    long rc;
    PyThreadState *const thread = PyEval_SaveThread();
    try {
        rc = call();
    } catch (...) {
        rc = KVRT_EDEVICE;
    }
    PyEval_RestoreThread(thread);
    return rc;
}

// (ctx, stream, layer, slots, scale, q, k, v, out)
PyObject *append_attend(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded(nargs, 9, [&]() -> long {
        Head h;
        float scale;
        kvrt_tensor q, k, v, o;
        if (!h.read(a) || !read_float(a[4], scale) || !read_tensor(a[5], true, q) || !read_tensor(a[6], true, k) ||
            !read_tensor(a[7], true, v) || !read_tensor(a[8], false, o) || !h.bind())
            return kGeneral;
        return without_gil([&] { return api.append_attend(h.ctx, h.layer, h.n, h.slots, &q, &k, &v, &o, scale); });
    });
}

// (ctx, stream, layer, slots, scale, q, out)
PyObject *attend(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded(nargs, 7, [&]() -> long {
        Head h;
        float scale;
        kvrt_tensor q, o;
        if (!h.read(a) || !read_float(a[4], scale) || !read_tensor(a[5], true, q) || !read_tensor(a[6], false, o) ||
            !h.bind())
            return kGeneral;
        return without_gil([&] { return api.attend(h.ctx, h.layer, h.n, h.slots, &q, &o, scale); });
    });
}

// (ctx, stream, layer, slots, scale, q, out, prefix slot or -1, softcap, slopes or None)
PyObject *attend_shared(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded(nargs, 10, [&]() -> long {
        Head h;
        float scale, cap;
        int32_t prefix;
        kvrt_tensor q, o, slopes;
        const bool biased = a[9] != Py_None;
        if (!h.read(a) || !read_float(a[4], scale) || !read_tensor(a[5], true, q) || !read_tensor(a[6], false, o) ||
            !read_int(a[7], prefix) || !read_float(a[8], cap) || (biased && !read_tensor(a[9], true, slopes)) || !h.bind())
            return kGeneral;
        return without_gil([&] {
            return api.shared(h.ctx, h.layer, h.n, h.slots, prefix, &q, &o, scale, cap,
                              biased ? static_cast<const float *>(slopes.data) : nullptr);
        });
    });
}

// (ctx, stream, layer, slots, scale, q, out, masks)
PyObject *attend_talker(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded(nargs, 8, [&]() -> long {
        Head h;
        float scale;
        kvrt_tensor q, o;
        kvrt_talker_mask m[kMaxSlots];
        PyObject **at = nullptr;
        if (!h.read(a) || !read_float(a[4], scale) || !read_tensor(a[5], true, q) || !read_tensor(a[6], false, o) ||
            items(a[7], at) != h.n)
            return kGeneral;
        for (int i = 0; i < h.n; ++i)
            if (!read_mask(at[i], m[i])) return kGeneral;
        if (!h.bind()) return kGeneral;
        return without_gil([&] { return api.talker(h.ctx, h.layer, h.n, h.slots, &q, &o, scale, m); });
    });
}

// (ctx, stream, layer, slots, positions, k, v)
PyObject *write_positions(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded(nargs, 7, [&]() -> long {
        Head h;
        kvrt_tensor k, v;
        int32_t pos[kMaxPositions];
        PyObject **rows;
        Py_ssize_t n_rows;
        if (!h.read(a) || (n_rows = items(a[4], rows)) < 0 || !read_tensor(a[5], false, k) ||
            !read_tensor(a[6], false, v))
            return kGeneral;
        int n = 0;
        for (Py_ssize_t i = 0; i < n_rows; ++i) {
            const int got = read_ints(rows[i], pos + n, kMaxPositions - n);
            if (got < 0) return kGeneral;
            n += got;
        }
        // other counts and empty writes are the general path's to answer
        if (k.ndim != 4 || k.dims[2] == 0 || n != k.dims[0] * k.dims[2] || !h.bind()) return kGeneral;
        return without_gil([&] { return api.write(h.ctx, h.layer, h.n, h.slots, pos, &k, &v); });
    });
}

// (ctx, stream, layer, slots, k, v, out_k, out_v, mask or None)
PyObject *append_gather(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded(nargs, 9, [&]() -> long {
        Head h;
        kvrt_tensor k, v, ok, ov, m;
        const bool masked = a[8] != Py_None;
        if (!h.read(a) || !read_tensor(a[4], false, k) || !read_tensor(a[5], false, v) ||
            !read_tensor(a[6], false, ok) || !read_tensor(a[7], false, ov) ||
            (masked && !read_tensor(a[8], false, m)) || !h.bind())
            return kGeneral;
        return without_gil([&] {
            return api.gather(h.ctx, h.layer, h.n, h.slots, &k, &v, nullptr, &ok, &ov, masked ? &m : nullptr);
        });
    });
}

// (stream, scale, window, q, k, v, lengths, out)
PyObject *attend_tensors(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded(nargs, 8, [&]() -> long {
        float scale;
        int32_t window;
        kvrt_tensor q, k, v, len, o;
        void *stream = PyLong_AsVoidPtr(a[0]);
        if (!read_float(a[1], scale) || !read_int(a[2], window) || !read_tensor(a[3], true, q) ||
            !read_tensor(a[4], false, k) || !read_tensor(a[5], false, v) || !read_tensor(a[6], true, len) ||
            len.dtype != KVRT_INT32 || !read_tensor(a[7], false, o))
            return kGeneral;
        return without_gil([&] {
            return api.tensors(&q, &k, &v, static_cast<const int32_t *>(len.data), nullptr, &o, scale, window, stream);
        });
    });
}

// (mask type, address of each Api member in order): once, after loading
PyObject *connect(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    void *p[7];
    if (nargs != 8) {
        PyErr_SetString(PyExc_TypeError, "connect takes the mask type and seven addresses");
        return nullptr;
    }
    for (int i = 0; i < 7; ++i) {
        p[i] = PyLong_AsVoidPtr(a[i + 1]);
        if (PyErr_Occurred()) return nullptr;
    }
    Py_INCREF(a[0]);
    Py_XDECREF(talker_mask_type);
    talker_mask_type = a[0];
    api.bind = reinterpret_cast<decltype(api.bind)>(p[0]);
    api.append_attend = reinterpret_cast<decltype(api.append_attend)>(p[1]);
    api.attend = reinterpret_cast<decltype(api.attend)>(p[2]);
    api.talker = reinterpret_cast<decltype(api.talker)>(p[3]);
    api.write = reinterpret_cast<decltype(api.write)>(p[4]);
    api.gather = reinterpret_cast<decltype(api.gather)>(p[5]);
    api.tensors = reinterpret_cast<decltype(api.tensors)>(p[6]);
    Py_RETURN_NONE;
}

// (address of kvrt_attend_shared_async): once, after connect
PyObject *connect_shared(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    void *p = nargs == 1 ? PyLong_AsVoidPtr(a[0]) : nullptr;
    if (PyErr_Occurred()) return nullptr;
    if (!p) {
        PyErr_SetString(PyExc_TypeError, "connect_shared takes one address");
        return nullptr;
    }
    api.shared = reinterpret_cast<decltype(api.shared)>(p);
    Py_RETURN_NONE;
}

// ---- 8-bit pages (kvrt/block8.py) --------------------------------------------------
//
// Through ctypes and torch.empty an update of the page tables spends 14 us on the host;
// its launches take 4 on the GPU. Here it allocates its answers, checks its tensors
// and launches in one call. A call that is not in the plain form is
// the general path's, which says what is wrong with it.

struct BlockApi {
    decltype(&kvrt_block_tables_update_async) update;
    decltype(&kvrt_block8_append_async) append;
    decltype(&kvrt_block8_gather_async) gather;
    decltype(&kvrt_block8_attend_async) attend;
    decltype(&kvrt_block8_attend_work) attend_work;
} block_api;

// The tensor in o where it is a plain GPU tensor on device dev.
const at::Tensor *plain(PyObject *o, int dev) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.get_device() != dev || t.layout() != at::kStrided || t.requires_grad())
        return nullptr;
    return &t;
}

// A contiguous int32 tensor of n elements on dev.
const int32_t *ints(PyObject *o, int dev, int ndim, int64_t n) {
    const at::Tensor *t = plain(o, dev);
    if (!t || t->scalar_type() != at::kInt || t->dim() != ndim || t->numel() != n || !t->is_contiguous()) return nullptr;
    return t->const_data_ptr<int32_t>();
}

bool describe(const at::Tensor *t, kvrt_tensor &d) {
    if (!t || t->dim() > KVRT_MAX_RANK) return false;
    d = kvrt_tensor{};
    d.dtype = dtype_code(t->scalar_type());
    if (d.dtype < 0) return false;
    d.data = t->data_ptr();
    d.ndim = (int32_t)t->dim();
    for (int i = 0; i < d.ndim; ++i) {
        d.dims[i] = t->size(i);
        d.strides[i] = t->stride(i);
    }
    return true;
}

bool current_device(int dev) {
    return c10::impl::getDeviceGuardImpl(c10::DeviceType::CUDA)->getDevice().index() == dev;
}

at::Tensor fresh(at::IntArrayRef size, at::ScalarType type, int dev) {
    return at::empty(size, at::TensorOptions().dtype(type).device(c10::DeviceType::CUDA, (c10::DeviceIndex)dev));
}

// As guarded(), for calls that answer with tensors: body's object, or the code.
template <class F>
PyObject *guarded_object(Py_ssize_t nargs, Py_ssize_t want, F body) {
    PyObject *out = nullptr;
    long rc = kGeneral;
    try {
        if (nargs == want) rc = body(out);
    } catch (...) {
        rc = kGeneral;
    }
    if (PyErr_Occurred()) PyErr_Clear();
    if (rc == KVRT_OK && out) return out;
    Py_XDECREF(out);
    return PyLong_FromLong(rc);
}

// (tables: sizes, scratch and status, stream, device, table, mapped, free, free_count, lengths, new, rows)
// -> (starts, slot_map, lengths, granted)
PyObject *block_update(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded_object(nargs, 10, [&](PyObject *&out) -> long {
        int32_t dev, rows;
        const auto *base = static_cast<const kvrt_block_tables *>(PyLong_AsVoidPtr(a[0]));
        void *stream = PyLong_AsVoidPtr(a[1]);
        if (!base || !read_int(a[2], dev) || !read_int(a[9], rows) || rows < 0 || !current_device(dev)) return kGeneral;
        kvrt_block_tables t = *base;
        t.table = const_cast<int32_t *>(ints(a[3], dev, 2, (int64_t)t.n * t.max_pages));
        t.mapped = const_cast<int32_t *>(ints(a[4], dev, 1, t.n));
        t.free_pages = const_cast<int32_t *>(ints(a[5], dev, 1, t.pool_pages));
        t.free_count = const_cast<int32_t *>(ints(a[6], dev, 1, 1));
        const int32_t *lengths = ints(a[7], dev, 1, t.n), *fresh_rows = ints(a[8], dev, 1, t.n);
        if (!t.table || THPVariable_Unpack(a[3]).size(0) != t.n || !t.mapped || !t.free_pages || !t.free_count ||
            !lengths || !fresh_rows)
            return kGeneral;
        const at::Tensor starts = fresh({t.n + 1}, at::kInt, dev), slots = fresh({rows}, at::kInt, dev),
                         lens = fresh({t.n}, at::kInt, dev), granted = fresh({t.n}, at::kInt, dev);
        int32_t *const p[4] = {starts.data_ptr<int32_t>(), rows ? slots.data_ptr<int32_t>() : nullptr,
                               lens.data_ptr<int32_t>(), granted.data_ptr<int32_t>()};
        const long rc =
            without_gil([&] { return block_api.update(&t, lengths, fresh_rows, rows, p[0], p[1], p[2], p[3], stream); });
        if (rc == KVRT_OK)
            out = Py_BuildValue("(NNNN)", THPVariable_Wrap(starts), THPVariable_Wrap(slots), THPVariable_Wrap(lens),
                                THPVariable_Wrap(granted));
        return rc;
    });
}

// The leading arguments of a pool's call: sizes and status, stream, device, then the pool's
// tensors k, v, k_scale, v_scale, which may be others than the last call's.
struct PoolHead {
    static constexpr int kArgs = 7;
    kvrt_block8 pages;
    void *stream;
    int32_t dev;

    template <class T>
    bool take(PyObject *o, at::ScalarType type, at::IntArrayRef size, T *&p) {
        const at::Tensor *t = plain(o, dev);
        if (!t || t->scalar_type() != type || t->sizes() != size || !t->is_contiguous()) return false;
        p = static_cast<T *>(t->data_ptr());
        return true;
    }
    bool read(PyObject *const *a) {
        const auto *base = static_cast<const kvrt_block8 *>(PyLong_AsVoidPtr(a[0]));
        stream = PyLong_AsVoidPtr(a[1]);
        if (!base || !read_int(a[2], dev) || !current_device(dev)) return false;
        pages = *base;
        const int64_t size[4] = {pages.pages, pages.kv_heads, pages.block, pages.head_dim};
        const at::IntArrayRef codes(size, 4), scales(size, 2);
        const at::ScalarType type = pages.dtype == KVRT_INT8 ? at::kChar : at::kFloat8_e4m3fn;
        return take(a[3], type, codes, pages.k) && take(a[4], type, codes, pages.v) &&
               take(a[5], at::kFloat, scales, pages.k_scale) && take(a[6], at::kFloat, scales, pages.v_scale);
    }
};

// (pool, k, v, slot_map)
PyObject *block_append(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded(nargs, PoolHead::kArgs + 3, [&]() -> long {
        PoolHead h;
        kvrt_tensor k, v;
        if (!h.read(a)) return kGeneral;
        a += PoolHead::kArgs;
        if (!describe(plain(a[0], h.dev), k) || !describe(plain(a[1], h.dev), v) || k.ndim < 1) return kGeneral;
        const int32_t *slots = ints(a[2], h.dev, 1, k.dims[0]);
        if (!slots) return kGeneral;
        return without_gil([&] { return block_api.append(&h.pages, &k, &v, slots, h.stream); });
    });
}

// What both forms of gather share.
struct GatherHead : PoolHead {
    static constexpr int kArgs = PoolHead::kArgs + 3;
    kvrt_tensor table;
    const int32_t *lengths, *from = nullptr;

    bool read(PyObject *const *a) {
        if (!PoolHead::read(a)) return false;
        a += PoolHead::kArgs;
        if (!describe(plain(a[0], dev), table) || table.ndim != 2 || table.dtype != KVRT_INT32) return false;
        lengths = ints(a[1], dev, 1, table.dims[0]);
        return lengths && (a[2] == Py_None || (from = ints(a[2], dev, 1, table.dims[0])));
    }
};

// (pool, table, lengths, start_pos or None, out_k, out_v, mask or None)
PyObject *block_gather(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded(nargs, GatherHead::kArgs + 3, [&]() -> long {
        GatherHead h;
        kvrt_tensor k, v, m;
        if (!h.read(a)) return kGeneral;
        a += GatherHead::kArgs;
        const bool masked = a[2] != Py_None;
        if (!describe(plain(a[0], h.dev), k) || !describe(plain(a[1], h.dev), v) ||
            (masked && !describe(plain(a[2], h.dev), m)))
            return kGeneral;
        return without_gil(
            [&] { return block_api.gather(&h.pages, &h.table, h.lengths, h.from, &k, &v, masked ? &m : nullptr, h.stream); });
    });
}

// (pool, table, lengths, start_pos or None, lmax, fp32, mask: 0 none, 1 bool, 2 fp32, 3 bf16)
// -> (k, v, mask or None)
PyObject *block_gather_new(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded_object(nargs, GatherHead::kArgs + 3, [&](PyObject *&out) -> long {
        GatherHead h;
        int32_t lmax, fp32, kind;
        if (!h.read(a)) return kGeneral;
        a += GatherHead::kArgs;
        if (!read_int(a[0], lmax) || lmax < 0 || !read_int(a[1], fp32) || !read_int(a[2], kind) || kind < 0 || kind > 3)
            return kGeneral;
        const int64_t size[4] = {h.table.dims[0], h.pages.kv_heads, lmax, h.pages.head_dim}, flat[2] = {size[0], lmax};
        const at::ScalarType kinds[3] = {at::kBool, at::kFloat, at::kBFloat16};
        const at::Tensor kt = fresh(size, fp32 ? at::kFloat : at::kBFloat16, h.dev), vt = at::empty_like(kt);
        at::Tensor mt;
        if (kind) mt = fresh(flat, kinds[kind - 1], h.dev);
        kvrt_tensor k, v, m;
        if (!describe(&kt, k) || !describe(&vt, v) || (kind && !describe(&mt, m))) return kGeneral;
        const long rc = without_gil(
            [&] { return block_api.gather(&h.pages, &h.table, h.lengths, h.from, &k, &v, kind ? &m : nullptr, h.stream); });
        if (rc == KVRT_OK) {
            PyObject *mask = Py_None;
            if (kind) mask = THPVariable_Wrap(mt);
            else Py_INCREF(mask);
            out = Py_BuildValue("(NNN)", THPVariable_Wrap(kt), THPVariable_Wrap(vt), mask);
        }
        return rc;
    });
}

// (pool, scale, window, max_q, q, table, lengths, starts, granted or None, out or None) -> out
PyObject *block_attend(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded_object(nargs, PoolHead::kArgs + 9, [&](PyObject *&answer) -> long {
        PoolHead h;
        int32_t window, max_q;
        float scale;
        kvrt_tensor q, table, o;
        const at::Tensor *qt;
        if (!h.read(a)) return kGeneral;
        a += PoolHead::kArgs;
        const int32_t dev = h.dev;
        if (!read_float(a[0], scale) || !read_int(a[1], window) || !read_int(a[2], max_q) || !(qt = plain(a[3], dev)) ||
            !describe(qt, q) || q.ndim != 3 || !describe(plain(a[4], dev), table) || table.ndim != 2 ||
            table.dtype != KVRT_INT32)
            return kGeneral;
        const int64_t n = table.dims[0];
        const int32_t *lengths = ints(a[5], dev, 1, n), *starts = ints(a[6], dev, 1, n + 1), *granted = nullptr;
        if (!lengths || !starts || (a[7] != Py_None && !(granted = ints(a[7], dev, 1, n)))) return kGeneral;
        if (max_q > q.dims[0]) max_q = (int32_t)q.dims[0];
        at::Tensor out;
        if (a[8] == Py_None) {
            out = fresh(qt->sizes(), qt->scalar_type(), dev);
            if (!describe(&out, o)) return kGeneral;
        } else if (!describe(plain(a[8], dev), o)) {
            return kGeneral;
        }
        const uint64_t size = block_api.attend_work(&h.pages, n, table.dims[1], q.dims[0], q.dims[1], max_q);
        at::Tensor work;
        if (size) work = fresh({(int64_t)size}, at::kByte, dev);
        const long rc = without_gil([&] {
            return block_api.attend(&h.pages, &q, &table, lengths, starts, granted, &o, scale, window, max_q,
                                    size ? work.data_ptr() : nullptr, size, h.stream);
        });
        if (rc == KVRT_OK) {
            if (out.defined()) answer = THPVariable_Wrap(out);
            else Py_INCREF(answer = a[8]);
        }
        return rc;
    });
}

// (address of each BlockApi member in order): once, after loading
PyObject *connect_blocks(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    void *p[5];
    if (nargs != 5) {
        PyErr_SetString(PyExc_TypeError, "connect_blocks takes five addresses");
        return nullptr;
    }
    for (int i = 0; i < 5; ++i) {
        p[i] = PyLong_AsVoidPtr(a[i]);
        if (PyErr_Occurred()) return nullptr;
    }
    block_api.update = reinterpret_cast<decltype(block_api.update)>(p[0]);
    block_api.append = reinterpret_cast<decltype(block_api.append)>(p[1]);
    block_api.gather = reinterpret_cast<decltype(block_api.gather)>(p[2]);
    block_api.attend = reinterpret_cast<decltype(block_api.attend)>(p[3]);
    block_api.attend_work = reinterpret_cast<decltype(block_api.attend_work)>(p[4]);
    Py_RETURN_NONE;
}

// ---- heads normed and rotated (kvrt/rotation.py) -------------------------------------

decltype(&kvrt_rotate_heads_async) rotate_api;

// Heads [n, H, Q, D] or packed [T, H, D] as kvrt_rotate_heads_async takes them.
bool describe_heads(const at::Tensor *t, kvrt_tensor &d) {
    if (!t || (t->dim() != 3 && t->dim() != 4) || !describe(t, d)) return false;
    if (d.ndim == 3) {
        d.ndim = 4;
        d.dims[3] = d.dims[2], d.strides[3] = d.strides[2];
        d.dims[2] = 1, d.strides[2] = 0;
    }
    return true;
}

// (rotation, stream, device, q, k, v, positions, out_q, out_k, out_v; each tensor may be None)
// -> (q, k, v)
PyObject *rotate_heads(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded_object(nargs, 10, [&](PyObject *&answer) -> long {
        int32_t dev;
        const auto *rot = static_cast<const kvrt_rotation *>(PyLong_AsVoidPtr(a[0]));
        void *stream = PyLong_AsVoidPtr(a[1]);
        if (!rot || !read_int(a[2], dev) || !current_device(dev)) return kGeneral;
        kvrt_tensor in[3], to[3], pos;
        at::Tensor fresh_out[3];
        int64_t rank = 0;
        for (int i = 0; i < 3; ++i) {
            PyObject *const x = a[3 + i], *const o = a[7 + i];
            if (x == Py_None) {
                if (o != Py_None) return kGeneral;
                continue;
            }
            const at::Tensor *t = plain(x, dev);
            if (!describe_heads(t, in[i]) || (rank && rank != t->dim())) return kGeneral;
            rank = t->dim();
            if (o == Py_None) {
                fresh_out[i] = fresh(t->sizes(), t->scalar_type(), dev);
                if (!describe_heads(&fresh_out[i], to[i])) return kGeneral;
            } else {
                const at::Tensor *d = plain(o, dev);
                if (!d || d->sizes() != t->sizes() || !describe_heads(d, to[i])) return kGeneral;
            }
        }
        if (!rank) return kGeneral;
        const bool turns = rot->n_freq > 0;
        if (turns) {
            const at::Tensor *p = plain(a[6], dev);
            const int own = rank == 3 ? 1 : 2;  // dims of one axis' positions
            if (!p || (p->dim() != own && p->dim() != own + 1) || !describe(p, pos)) return kGeneral;
            const int lead = p->dim() == own ? 0 : 1;
            kvrt_tensor x = pos;
            x.ndim = 3;
            x.dims[0] = lead ? pos.dims[0] : 1, x.strides[0] = lead ? pos.strides[0] : 0;
            x.dims[1] = pos.dims[lead], x.strides[1] = pos.strides[lead];
            x.dims[2] = own == 2 ? pos.dims[lead + 1] : 1, x.strides[2] = own == 2 ? pos.strides[lead + 1] : 0;
            pos = x;
        }
        const auto at = [&](int i, kvrt_tensor *of) { return a[3 + i] == Py_None ? nullptr : of + i; };
        const long rc = without_gil([&] {
            return rotate_api(rot, at(0, in), at(1, in), at(2, in), turns ? &pos : nullptr, at(0, to), at(1, to), at(2, to),
                              stream);
        });
        if (rc == KVRT_OK) {
            PyObject *got[3];
            for (int i = 0; i < 3; ++i) {
                if (fresh_out[i].defined()) got[i] = THPVariable_Wrap(fresh_out[i]);
                else Py_INCREF(got[i] = a[7 + i]);
            }
            answer = Py_BuildValue("(NNN)", got[0], got[1], got[2]);
        }
        return rc;
    });
}

// (address of kvrt_rotate_heads_async): once, after loading
PyObject *connect_rotate(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    void *p = nargs == 1 ? PyLong_AsVoidPtr(a[0]) : nullptr;
    if (PyErr_Occurred()) return nullptr;
    if (!p) {
        PyErr_SetString(PyExc_TypeError, "connect_rotate takes one address");
        return nullptr;
    }
    rotate_api = reinterpret_cast<decltype(rotate_api)>(p);
    Py_RETURN_NONE;
}

#define KVRT_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {KVRT_METHOD(append_attend),   KVRT_METHOD(attend),        KVRT_METHOD(attend_talker),
                         KVRT_METHOD(write_positions), KVRT_METHOD(append_gather), KVRT_METHOD(attend_tensors),
                         KVRT_METHOD(connect),         KVRT_METHOD(block_update),  KVRT_METHOD(block_append),
                         KVRT_METHOD(block_gather),    KVRT_METHOD(block_gather_new), KVRT_METHOD(block_attend),
                         KVRT_METHOD(connect_blocks),  KVRT_METHOD(rotate_heads),  KVRT_METHOD(connect_rotate),
                         KVRT_METHOD(attend_shared),   KVRT_METHOD(connect_shared),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "kvrt_pycall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_kvrt_pycall() { return PyModule_Create(&module); }
