// CPython module of the package's host paths that run once per layer and step: what a call costs before its
// launches.  A decode call's argument checks and launch arguments took ~5.6 us of Python and ctypes next to
// ~6.8 us for the launches themselves, more than a small cache's time on the GPU: 11.8 -> 9.2 us per call at
// 3B's heads over 4k tokens, 11.7 -> 10.7 (GPU-bound) over 32k.  A cache build's allocations, launch
// arguments and ~45 metadata views took ~80 us next to 9 us of kernels: 92 -> 68 us (4k tokens), 99 -> 75
// (64k, 38 us of kernels).
//
// A call on a paged cache or a prompt's rows took 16 to 20 us in Python, more than a decode step's kernels.
//
// The decode entry takes the forms that a model's step uses and returns None for every other (strided or
// misaligned rows, other types, a full ring, a folded rotation, any error): those keep the Python path and
// its checks and messages.  It keeps nothing from a call.  The library's functions come as addresses, so
// that the module follows whichever library the package loaded.
#include <Python.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <vector>

#include "r2o_sspa.h"

namespace {

const at::Tensor* exact_tensor(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

bool on_device(const at::Tensor& t, int64_t device) {
    return t.device().type() == at::kCUDA && t.device().index() == device && t.layout() == at::kStrided;
}

int row_code(const at::Tensor& t) {
    return t.scalar_type() == at::kBFloat16 ? 0 : (t.scalar_type() == at::kHalf ? 1 : -1);
}

bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

struct WithoutGil {
    PyThreadState* state = PyEval_SaveThread();
    ~WithoutGil() { PyEval_RestoreThread(state); }
};

// ------------------------------------------------------------------------------------ decode call
struct Decode {
    r2o_decode_params params;  // what stays from call to call (SplitKExecutor._static_params)
    int (*launch)(const r2o_decode_params*, void*);
    int64_t device;
};

void decode_free(PyObject* capsule) { delete static_cast<Decode*>(PyCapsule_GetPointer(capsule, "r2o_decode")); }

// decode_handle(params address, r2o_decode address, device index)
PyObject* decode_handle(PyObject*, PyObject* args) {
    unsigned long long params, fn;
    long long device;
    if (!PyArg_ParseTuple(args, "KKL", &params, &fn, &device)) return nullptr;
    auto* d = new Decode;
    std::memcpy(&d->params, reinterpret_cast<const void*>(params), sizeof(d->params));
    d->launch = reinterpret_cast<int (*)(const r2o_decode_params*, void*)>(fn);
    d->device = device;
    PyObject* capsule = PyCapsule_New(d, "r2o_decode", decode_free);
    if (!capsule) delete d;
    return capsule;
}

bool plain_int(PyObject* o, int64_t& v) {
    if (!PyLong_CheckExact(o)) return false;
    int overflow = 0;
    v = PyLong_AsLongLongAndOverflow(o, &overflow);
    return overflow == 0;
}

// One value per request: an int for all, or a list or tuple of b ints.
bool per_request(PyObject* o, int64_t b, int64_t* out) {
    if (plain_int(o, out[0])) {
        std::fill(out + 1, out + b, out[0]);
        return true;
    }
    if (!(PyList_CheckExact(o) || PyTuple_CheckExact(o)) || PySequence_Fast_GET_SIZE(o) != b) return false;
    for (int64_t i = 0; i < b; ++i)
        if (!plain_int(PySequence_Fast_GET_ITEM(o, i), out[i])) return false;
    return true;
}

PyObject* const kRecentPool = PyUnicode_InternFromString("recent_fp_pool");
PyObject* const kActiveLength = PyUnicode_InternFromString("active_length");
PyObject* const kCapacity = PyUnicode_InternFromString("capacity");

// An int attribute of o; false (with no exception set) if it is anything else.
bool int_attr(PyObject* o, PyObject* name, int64_t& v) {
    PyObject* a = PyObject_GetAttr(o, name);
    if (!a) {
        PyErr_Clear();
        return false;
    }
    const bool ok = plain_int(a, v);
    Py_DECREF(a);
    return ok;
}

// decode(handle, query, append or None, output, caches list, own ring lengths list or None): the status of
// r2o_decode, or None for a call that the Python path makes.  With ring lengths of its own (a stacked
// executor) a call with an append advances them.
PyObject* decode_call(PyObject* const* args) {
    auto* d = static_cast<Decode*>(PyCapsule_GetPointer(args[0], "r2o_decode"));
    if (!d) return nullptr;
    r2o_decode_params p = d->params;
    const int64_t b = p.batch;
    if (b < 1 || b > R2O_MAX_BATCH) Py_RETURN_NONE;
    const at::Tensor *q = exact_tensor(args[1]), *out = exact_tensor(args[3]);
    if (!q || !out || !on_device(*q, d->device) || !on_device(*out, d->device)) Py_RETURN_NONE;
    const bool token_axis = q->dim() == 4 && q->size(2) == 1;
    if (!(q->dim() == 3 || token_axis) || q->size(0) != b || q->size(1) != p.hq || q->size(-1) != R2O_HEAD_DIM ||
        !q->is_contiguous() || !aligned16(*q) || row_code(*q) < 0)
        Py_RETURN_NONE;
    if (out->dim() != 3 || out->size(0) != b || out->size(1) != p.hq || out->size(2) != R2O_HEAD_DIM) Py_RETURN_NONE;
    p.query = static_cast<const uint16_t*>(q->data_ptr());
    p.q_dtype = row_code(*q);
    p.out = static_cast<uint16_t*>(out->data_ptr());

    PyObject *caches = args[4], *own = args[5];
    if (!PyList_CheckExact(caches) || PyList_GET_SIZE(caches) != b) Py_RETURN_NONE;
    const bool stacked = own != Py_None;
    if (stacked && (!PyList_CheckExact(own) || PyList_GET_SIZE(own) != b)) Py_RETURN_NONE;
    bool room = true;
    int64_t lengths[R2O_MAX_BATCH];
    for (int64_t i = 0; i < b; ++i) {
        int64_t capacity = 0;
        if (stacked && i > 0) {  // one capacity for all, as the Python path checks
            if (!plain_int(PyList_GET_ITEM(own, i), lengths[i])) Py_RETURN_NONE;
            room = room && lengths[i] < p.recent_len[0];
            continue;
        }
        PyObject* pool = PyObject_GetAttr(PyList_GET_ITEM(caches, i), kRecentPool);
        if (!pool) {
            PyErr_Clear();
            Py_RETURN_NONE;
        }
        const bool ok = int_attr(pool, kCapacity, capacity) &&
                        (stacked ? plain_int(PyList_GET_ITEM(own, i), lengths[i]) : int_attr(pool, kActiveLength, lengths[i]));
        Py_DECREF(pool);
        if (!ok || capacity > 0x7fffffff) Py_RETURN_NONE;
        room = room && lengths[i] < capacity;
        if (stacked) p.recent_len[0] = (int32_t)capacity;
    }
    for (int64_t i = 0; i < b; ++i) {
        if (lengths[i] < 0 || lengths[i] > 0x7fffffff) Py_RETURN_NONE;
        p.recent_len[i] = (int32_t)lengths[i];
    }

    PyObject* append = args[2];
    if (append != Py_None) {
        if (!PyTuple_CheckExact(append) || PyTuple_GET_SIZE(append) != 4 || !room) Py_RETURN_NONE;
        const at::Tensor *k = exact_tensor(PyTuple_GET_ITEM(append, 0)), *v = exact_tensor(PyTuple_GET_ITEM(append, 1));
        const int64_t n = b * p.hkv * R2O_HEAD_DIM;
        for (const at::Tensor* t : {k, v})
            if (!t || !on_device(*t, d->device) || !t->is_contiguous() || t->numel() != n || !aligned16(*t) ||
                row_code(*t) != p.row_dtype)
                Py_RETURN_NONE;
        if (!per_request(PyTuple_GET_ITEM(append, 2), b, p.append_global) ||
            !per_request(PyTuple_GET_ITEM(append, 3), b, p.append_logical))
            Py_RETURN_NONE;
        p.append_k = static_cast<const uint16_t*>(k->data_ptr());
        p.append_v = static_cast<const uint16_t*>(v->data_ptr());
        p.do_append = 1;
    }
    void* stream = c10::hip::getCurrentHIPStream((c10::DeviceIndex)d->device).stream();
    int rc;
    {
        WithoutGil released;
        rc = d->launch(&p, stream);
    }
    if (rc == R2O_OK && stacked && append != Py_None)
        for (int64_t i = 0; i < b; ++i) {
            PyObject* next = PyLong_FromLongLong(lengths[i] + 1);
            if (!next || PyList_SetItem(own, i, next)) return nullptr;
        }
    return PyLong_FromLong(rc);
}

PyObject* decode(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 6) Py_RETURN_NONE;
    try {
        return decode_call(args);
    } catch (...) {  // a tensor without memory of its own (vmap, a subclass): the Python path's error
        Py_RETURN_NONE;
    }
}

// ------------------------------------------------------------------------------------- cache build
int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

PyObject* wrap(const at::Tensor& t) {
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(t);
}

// A tuple of the tensors (None where undefined).
PyObject* wrap_all(const std::vector<at::Tensor>& ts) {
    PyObject* tuple = PyTuple_New((Py_ssize_t)ts.size());
    for (size_t i = 0; tuple && i < ts.size(); ++i) {
        PyObject* o = wrap(ts[i]);
        if (!o) {
            Py_DECREF(tuple);
            return nullptr;
        }
        PyTuple_SET_ITEM(tuple, (Py_ssize_t)i, o);
    }
    return tuple;
}

// cache_build(key, value, global, logical, page table [3, pages] on the host, r2o_cache_page_words address,
// r2o_cache_build address, tier pages (4), tier tokens (4), page size, ring capacity, append capacity,
// superblock, INT2 group, key bits (4, 2, 16), INT4 generated values): allocates every tensor of the cache,
// uploads the page words and launches; the callers have checked shapes, types and devices.  Returns
// (status, payload tensors, metadata tensors) in the order that cache.py unpacks.
PyObject* cache_build(PyObject*, PyObject* args) {
    PyObject *key_o, *value_o, *global_o, *logical_o, *table_o;
    unsigned long long words_fn, build_fn;
    long long tp[4], tt[4], page_size, ring, append, superblock, group, k_bits;
    int gen_int4;
    if (!PyArg_ParseTuple(args, "OOOOOKK(LLLL)(LLLL)LLLLLLp", &key_o, &value_o, &global_o, &logical_o, &table_o, &words_fn,
                          &build_fn, tp, tp + 1, tp + 2, tp + 3, tt, tt + 1, tt + 2, tt + 3, &page_size, &ring, &append,
                          &superblock, &group, &k_bits, &gen_int4))
        return nullptr;
    for (PyObject* o : {key_o, value_o, global_o, logical_o, table_o})
        if (!THPVariable_Check(o)) {
            PyErr_SetString(PyExc_TypeError, "cache_build takes tensors");
            return nullptr;
        }
    int rc = 0;
    std::vector<at::Tensor> payload, meta;
    try {
        WithoutGil released;
        const at::Tensor &key = THPVariable_Unpack(key_o), &value = THPVariable_Unpack(value_o),
                         &global = THPVariable_Unpack(global_o), &logical = THPVariable_Unpack(logical_o),
                         &table = THPVariable_Unpack(table_o);
        const int64_t h = key.size(0), s = key.size(1), n_pages = table.size(1);
        const int64_t s_fp = tt[0], s_i4 = tt[1], s_i2 = tt[2], n = s_fp + s_i4 + s_i2;
        const auto opt = at::TensorOptions().device(key.device());
        const auto u8 = opt.dtype(at::kByte), f16 = opt.dtype(at::kHalf), i64 = opt.dtype(at::kLong);

        at::Tensor fp_v, i4_v, i4_scale, k_packed, k_scale, k_zero, k_ops;
        if (s_fp) fp_v = at::empty({h, s_fp, 128}, opt.dtype(value.scalar_type()));
        int64_t i4_capacity = gen_int4 ? std::max<int64_t>(1, s_i4 + append) : s_i4;
        if (gen_int4) i4_v = at::empty({h, i4_capacity, 64}, u8);
        else if (s_i4) i4_v = at::empty({h * s_i4 * 64}, u8);
        if (i4_capacity) i4_scale = at::empty({h, i4_capacity, 1}, opt.dtype(at::kFloat));
        const int64_t i2_capacity = std::max<int64_t>(128, round_up(s_i2 + (gen_int4 ? 0 : append), 128));
        at::Tensor i2_v = at::empty({h, i2_capacity, 32}, u8), i2_scale = at::empty({h, i2_capacity, 128 / group, 1}, f16),
                   i2_zero = at::empty({h, i2_capacity, 128 / group, 1}, u8);
        const int64_t capacity = std::max<int64_t>(128, round_up(n + append, 128)), blocks = capacity / superblock;
        int64_t reserve2 = 0, reserve4 = 0;
        if (k_bits == 16) {  // no compact K arena to flush into: nothing is reserved
            k_packed = at::empty({h, capacity, 128}, opt.dtype(key.scalar_type()));
        } else {
            k_packed = at::empty({h, capacity, 16 * k_bits}, u8);
            k_scale = at::empty({h, blocks, 128}, f16);
            k_zero = at::empty({h, blocks, 128}, k_bits == 4 ? u8 : f16);
            k_ops = at::empty({h, blocks, 128}, opt.dtype(at::kInt));
            reserve2 = std::min(i2_capacity - s_i2, capacity - n) / page_size * page_size;
            if (gen_int4) reserve4 = std::min(i4_capacity - s_i4, capacity - n) / page_size * page_size;
        }
        at::Tensor ring_k = at::empty({h, ring, 128}, opt.dtype(key.scalar_type())), ring_v = at::empty_like(ring_k);

        const int64_t spans[3] = {tp[0], tp[1] + reserve4 / page_size, tp[2] + reserve2 / page_size};
        const int64_t tokens[3] = {s_fp, s_i4 + reserve4, s_i2 + reserve2};
        const int64_t ring_pages = ring / page_size;
        const int64_t page_words = 3 * (spans[0] + spans[1] + spans[2] + ring_pages) + 1;
        at::Tensor words = at::empty({page_words + 3 * n_pages}, at::TensorOptions().dtype(at::kLong).pinned_memory(true));
        rc = reinterpret_cast<decltype(&r2o_cache_page_words)>(words_fn)(
            table.data_ptr<int64_t>(), n_pages, page_size, reserve4, reserve2, ring, words.data_ptr<int64_t>(), words.numel());
        if (!rc) {
            // pinned: a copy from pageable memory would wait for the stream's earlier work
            at::Tensor pages = words.to(i64, /*non_blocking=*/true);
            at::Tensor storage = at::empty({page_words + 2 * (tokens[0] + tokens[1] + tokens[2]) + tt[3] + 2 * ring}, i64);
            at::Tensor index = at::empty({n}, i64);

            auto ptr = [](const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
            r2o_cache_build_params p{};
            p.key = static_cast<const uint16_t*>(ptr(key));
            p.value = static_cast<const uint16_t*>(ptr(value));
            p.key_dtype = row_code(key);
            p.value_dtype = row_code(value);
            p.hkv = h;
            p.tokens = s;
            p.plan_global = static_cast<const int64_t*>(ptr(global));
            p.plan_logical = static_cast<const int64_t*>(ptr(logical));
            p.pages = static_cast<const int64_t*>(ptr(pages));
            p.page_words = page_words;
            p.n_pages = n_pages;
            for (int t = 0; t < 4; ++t) p.tier_tokens[t] = tt[t];
            p.reserve4 = reserve4;
            p.reserve2 = reserve2;
            p.storage = static_cast<int64_t*>(ptr(storage));
            p.index = static_cast<int64_t*>(ptr(index));
            p.ring_k = static_cast<uint16_t*>(ptr(ring_k));
            p.ring_v = static_cast<uint16_t*>(ptr(ring_v));
            p.ring_capacity = ring;
            p.k_bits = k_bits;
            p.superblock = superblock;
            p.k_packed = static_cast<uint8_t*>(ptr(k_packed));
            p.k_scale = static_cast<uint16_t*>(ptr(k_scale));
            p.k_zero = ptr(k_zero);
            p.k_operands = static_cast<uint32_t*>(ptr(k_ops));
            p.k_capacity = capacity;
            p.k_superblocks = blocks;
            p.fp_v = static_cast<uint16_t*>(ptr(fp_v));
            p.i4_v = static_cast<uint8_t*>(ptr(i4_v));
            p.i4_scale = static_cast<float*>(ptr(i4_scale));
            p.i4_capacity = i4_capacity;
            p.i2_v = static_cast<uint8_t*>(ptr(i2_v));
            p.i2_scale = static_cast<uint16_t*>(ptr(i2_scale));
            p.i2_zero = static_cast<uint8_t*>(ptr(i2_zero));
            p.i2_capacity = i2_capacity;
            p.i2_group = group;
            void* stream = c10::hip::getCurrentHIPStream(key.device().index()).stream();
            rc = reinterpret_cast<decltype(&r2o_cache_build)>(build_fn)(&p, stream);

            // the metadata storage's fields: per tier and for the ring ids, offsets, lengths; the length word; global
            // and logical indices per tier; evicted; ring global and logical; then the INT4 and INT2 pools' five
            // fields without their reserve
            meta.push_back(storage);
            int64_t at_word = 0;
            auto take = [&](int64_t len) {
                meta.push_back(storage.narrow(0, at_word, len));
                at_word += len;
            };
            for (int64_t span : {spans[0], spans[1], spans[2], ring_pages})
                for (int f = 0; f < 3; ++f) take(span);
            take(1);
            for (int f = 0; f < 2; ++f)
                for (int64_t span : tokens) take(span);
            take(tt[3]);
            take(ring);
            take(ring);
            meta[13] = meta[13].view(at::kInt).select(0, 0);
            for (int t = 1; t < 3; ++t)  // active views
                for (int f = 0; f < 5; ++f) {
                    const at::Tensor& full = f < 3 ? meta[1 + 3 * t + f] : meta[14 + 3 * (f - 3) + t];
                    const int64_t len = f < 3 ? tp[t] : tt[t];
                    meta.push_back(full.size(0) == len ? full : full.narrow(0, 0, len));
                }
            payload = {fp_v, i4_v, i4_scale, i2_v, i2_scale, i2_zero, k_packed, k_scale, k_zero, k_ops, ring_k, ring_v};
        }
    } catch (...) {
        torch::translate_exception_to_python(std::current_exception());
        return nullptr;
    }
    PyObject* tensors = wrap_all(payload);
    PyObject* fields = tensors ? wrap_all(meta) : nullptr;
    if (!fields) {
        Py_XDECREF(tensors);
        return nullptr;
    }
    return Py_BuildValue("(iNN)", rc, tensors, fields);
}

// ------------------------------------------------------------------------- prompt and paged calls
// Each takes the forms that a model's layer uses, allocates its results and scratch and launches; None for every other
// (strides or alignments that need a copy, other types, an operand that a check refuses, another device than the
// current one): those keep the Python path and its checks and messages.
int current_device() {
    int d = -1;
    return hipGetDevice(&d) == hipSuccess ? d : -1;
}

int64_t compute_units(int device) {
    static int known[64] = {};
    if (device < 0 || device >= 64) return 0;
    if (!known[device]) {
        int n = 0;
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess) return 0;
        known[device] = n;
    }
    return known[device];
}

// A derivative through the tensor, of either mode, would be lost.
bool needs_grad(const at::Tensor& t) { return (at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined(); }

// Strides of the axes before the channels: multiples of 8 elements, the rows' within 32-bit offsets; 0 for an axis of one.
bool row_strides(const at::Tensor& t, int64_t n, int64_t* out, bool own_memory = false) {
    if (t.stride(-1) != 1 || !aligned16(t)) return false;
    for (int64_t i = 0; i < n; ++i) {
        out[i] = t.size(i) > 1 ? t.stride(i) : 0;
        if (out[i] % 8 || out[i] < 0 || (own_memory && t.size(i) > 1 && out[i] == 0)) return false;
    }
    return true;
}

// None, or a contiguous int32 tensor [batch] on the device.
bool lengths_arg(PyObject* o, int64_t batch, int64_t device, const int32_t*& out) {
    out = nullptr;
    if (o == Py_None) return true;
    const at::Tensor* t = exact_tensor(o);
    if (!t || !on_device(*t, device) || t->scalar_type() != at::kInt || t->dim() != 1 || t->size(0) != batch || !t->is_contiguous())
        return false;
    out = static_cast<const int32_t*>(t->data_ptr());
    return true;
}

// window and sinks as Python ints (window None: 0), the scale as a float (None: 1 / sqrt(128)).
bool mask_args(PyObject* window_o, PyObject* sinks_o, PyObject* scale_o, int64_t& window, int64_t& sinks, float& scale) {
    window = 0;
    if (window_o != Py_None && (!plain_int(window_o, window) || window < 1)) return false;
    if (!plain_int(sinks_o, sinks) || sinks < 0 || sinks > (1 << 29)) return false;
    if (scale_o == Py_None) {
        scale = 0.08838834764831845f;
        return true;
    }
    if (!PyFloat_CheckExact(scale_o)) return false;
    const double x = PyFloat_AS_DOUBLE(scale_o);
    scale = (float)x;
    return x > 0.0 && scale > 0.f && scale < INFINITY;
}

int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Workgroups that share the keys of one tile of 128 packed rows: as many as give a compute unit one, at most one for each 256
// keys, begun ones among them, that the tile sees: its rows stand at 128 / group neighbouring positions, so with a window
// these are the window's, 128 / group more, the sinks and what else the first of its key tiles holds.  257 rows of 16 heads over
// 4097 keys take 28.4 us in 7 splits (one a compute unit), 30 in 6, 32 in 8, 91 in one; 512 rows of 16 heads with a window of
// 256 15.9 in 2, 19.8 in 4, 14.0 in one; one row of 28 heads over 300 keys 10.7 in 2, 11.2 in one.
int64_t attention_splits(int64_t batch, int64_t hq, int64_t hkv, int64_t queries, int64_t keys, int64_t window, int64_t sinks, int64_t cus) {
    const int64_t group = hq / hkv, tiles = div_up(group * queries, 128) * batch * hkv;
    const int64_t seen = window ? std::min(keys, std::min(window, keys) + div_up(128, group) + std::min(sinks, keys) + 64) : keys;
    return std::max<int64_t>(1, std::min(cus / tiles, div_up(seen, 256)));
}

// Workgroups that share the query rows of one key tile: as many as give a compute unit three, at most one for each (query
// head, 64-row tile) pair.  8192 rows of 16 heads over as many keys take 173 us in 12 splits (three a compute unit), 181 in
// 16, 237 in 8; 64 rows of 28 heads over 32641 keys 30 us in one (two a compute unit), 37 in two.
int64_t weight_splits(int64_t batch, int64_t hq, int64_t hkv, int64_t queries, int64_t keys, int64_t cus) {
    const int64_t tiles = div_up(keys, 256) * batch * hkv, pairs = hq / hkv * div_up(queries, 64);
    return std::max<int64_t>(1, std::min(pairs, 3 * cus / tiles));
}

// Workgroups that share the slots of a call: one a compute unit (their LDS fills it), fewer when the page tables hold
// fewer than four tiles of 32 slots for each.
int64_t paged_workers(int64_t batch, int64_t hkv, int64_t capacity, int64_t cus) {
    return std::max<int64_t>(1, std::min(cus, batch * hkv * div_up(capacity, 128)));
}

// The fields that attention and weights share; false for what the Python path has to look at.
bool prompt_operands(const at::Tensor* q, const at::Tensor* k, PyObject* const* masks, r2o_prompt_params& p, int64_t& device) {
    if (!q || !k || q->dim() != 4 || k->dim() != 4 || q->size(3) != R2O_HEAD_DIM || k->size(3) != R2O_HEAD_DIM) return false;
    device = current_device();
    if (!on_device(*q, device) || !on_device(*k, device) || row_code(*q) < 0 || q->scalar_type() != k->scalar_type() ||
        needs_grad(*q) || needs_grad(*k))
        return false;
    constexpr int64_t kMost = 1 << 29;
    p.batch = q->size(0);
    p.hq = q->size(1);
    p.hkv = k->size(1);
    p.queries = q->size(2);
    p.keys = k->size(2);
    p.dtype = row_code(*q);
    if (k->size(0) != p.batch || p.batch < 1 || p.hkv < 1 || p.hq < 1 || p.hq % p.hkv || p.queries < 1 || p.keys < 1 ||
        p.queries > kMost || p.keys > kMost || p.batch * p.hq > 65535 || p.hq / p.hkv * p.queries > 2 * kMost)
        return false;
    if (!row_strides(*q, 3, p.q_strides) || !row_strides(*k, 3, p.k_strides) || p.q_strides[2] > R2O_MAX_ROW_STRIDE ||
        p.k_strides[2] > R2O_MAX_ROW_STRIDE)
        return false;
    p.query = static_cast<const uint16_t*>(q->data_ptr());
    p.key = static_cast<const uint16_t*>(k->data_ptr());
    return mask_args(masks[0], masks[1], masks[4], p.window, p.sinks, p.sm_scale) &&
           lengths_arg(masks[2], p.batch, device, p.query_lengths) && lengths_arg(masks[3], p.batch, device, p.key_lengths);
}

template <class Params>
int launch_on(PyObject* fn, const Params& p, int64_t device) {
    auto* f = reinterpret_cast<int (*)(const Params*, void*)>(PyLong_AsVoidPtr(fn));
    void* stream = c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream();
    WithoutGil released;
    return f(&p, stream);
}

// (status, tensors ...)
PyObject* status_and(int rc, const std::vector<at::Tensor>& ts) {
    PyObject* tuple = PyTuple_New(1 + (Py_ssize_t)ts.size());
    if (!tuple) return nullptr;
    PyTuple_SET_ITEM(tuple, 0, PyLong_FromLong(rc));
    for (size_t i = 0; i < ts.size(); ++i) {
        PyObject* o = wrap(ts[i]);
        if (!o) {
            Py_DECREF(tuple);
            return nullptr;
        }
        PyTuple_SET_ITEM(tuple, 1 + (Py_ssize_t)i, o);
    }
    return tuple;
}

// prompt(function, query, key, value, window, sinks, query_lengths, key_lengths, scale): (status, out, lse) or None
PyObject* prompt_call(PyObject* const* args) {
    r2o_prompt_params p{};
    int64_t device;
    const at::Tensor *q = exact_tensor(args[1]), *k = exact_tensor(args[2]), *v = exact_tensor(args[3]);
    if (!prompt_operands(q, k, args + 4, p, device) || !v || v->sizes() != k->sizes() || !on_device(*v, device) ||
        v->scalar_type() != k->scalar_type() || needs_grad(*v) || !row_strides(*v, 3, p.v_strides) || p.v_strides[2] > R2O_MAX_ROW_STRIDE)
        Py_RETURN_NONE;
    at::Tensor out = at::empty_like(*q);
    if (!row_strides(out, 3, p.o_strides, true) || p.o_strides[2] > R2O_MAX_ROW_STRIDE) Py_RETURN_NONE;
    const auto f32 = at::TensorOptions().device(q->device()).dtype(at::kFloat);
    at::Tensor lse = at::empty({p.batch, p.hq, p.queries}, f32), scratch;
    p.splits = attention_splits(p.batch, p.hq, p.hkv, p.queries, p.keys, p.window, p.sinks, compute_units((int)device));
    if (p.splits > 1) {
        p.scratch_floats = 130 * p.splits * p.batch * p.hq * p.queries;
        scratch = at::empty({p.scratch_floats}, f32);
        p.scratch = scratch.data_ptr<float>();
    }
    p.value = static_cast<const uint16_t*>(v->data_ptr());
    p.out = static_cast<uint16_t*>(out.data_ptr());
    p.lse = lse.data_ptr<float>();
    return status_and(launch_on(args[0], p, device), {out, lse});
}

// weights(function, query, key, lse, window, sinks, query_lengths, key_lengths, scale): (status, weights) or None
PyObject* weights_call(PyObject* const* args) {
    r2o_prompt_params p{};
    int64_t device;
    const at::Tensor *q = exact_tensor(args[1]), *k = exact_tensor(args[2]), *lse = exact_tensor(args[3]);
    if (!prompt_operands(q, k, args + 4, p, device) || !lse || !on_device(*lse, device) || lse->scalar_type() != at::kFloat ||
        lse->dim() != 3 || lse->size(0) != p.batch || lse->size(1) != p.hq || lse->size(2) != p.queries || !lse->is_contiguous() || needs_grad(*lse))
        Py_RETURN_NONE;
    const auto f32 = at::TensorOptions().device(q->device()).dtype(at::kFloat);
    at::Tensor out = at::empty({p.batch, p.hkv, p.keys}, f32), scratch;
    p.splits = weight_splits(p.batch, p.hq, p.hkv, p.queries, p.keys, compute_units((int)device));
    if (p.splits > 1) {
        p.scratch_floats = p.splits * out.numel();
        scratch = at::empty({p.scratch_floats}, f32);
        p.scratch = scratch.data_ptr<float>();
    }
    p.lse_in = lse->data_ptr<float>();
    p.weights = out.data_ptr<float>();
    return status_and(launch_on(args[0], p, device), {out});
}

PyObject* const kCacheFields[5] = {PyUnicode_InternFromString("key_pages"), PyUnicode_InternFromString("value_pages"),
                                   PyUnicode_InternFromString("page_table"), PyUnicode_InternFromString("lengths"),
                                   PyUnicode_InternFromString("weight_pages")};

// A PagedCache's tensors, held for a call, and where they lie now: nothing is kept from its making, so a copy, a loaded
// one and one whose tensors got other memory are what they say.
struct Cache {
    PyObject* fields[5] = {};
    r2o_paged_cache c{};
    int64_t device = -1;
    ~Cache() {
        for (PyObject* o : fields) Py_XDECREF(o);
    }
    bool read(PyObject* cache);  // false for what the Python path has to look at
    bool callable() const {      // in a call: the tensors lie on the current device, and no derivative would be lost
        if (device != current_device()) return false;
        for (int i : {0, 1, 4})
            if (fields[i] != Py_None && needs_grad(THPVariable_Unpack(fields[i]))) return false;
        return true;
    }
};

bool Cache::read(PyObject* cache) {
    for (int i = 0; i < 5; ++i)
        if (!(fields[i] = PyObject_GetAttr(cache, kCacheFields[i]))) {
            PyErr_Clear();
            return false;
        }
    const at::Tensor *k = exact_tensor(fields[0]), *v = exact_tensor(fields[1]), *table = exact_tensor(fields[2]), *n = exact_tensor(fields[3]);
    const at::Tensor* w = fields[4] == Py_None ? nullptr : exact_tensor(fields[4]);
    if (!k || !v || !table || !n || (fields[4] != Py_None && !w) || k->dim() != 4 || k->device().type() != at::kCUDA) return false;
    device = k->device().index();
    c.pages = k->size(0);
    c.hkv = k->size(1);
    c.page_size = k->size(2);
    c.dtype = row_code(*k);
    for (const at::Tensor* t : {k, v, table, n})
        if (!on_device(*t, device)) return false;
    if (c.dtype < 0 || k->size(3) != R2O_HEAD_DIM || c.pages < 1 || c.pages > 0x7fffffff || c.hkv < 1 || c.hkv > 1024 ||
        v->sizes() != k->sizes() || v->scalar_type() != k->scalar_type() ||
        (c.page_size != 16 && c.page_size != 32 && c.page_size != 64 && c.page_size != 128))
        return false;
    if (!row_strides(*k, 3, c.key_strides, true) || !row_strides(*v, 3, c.value_strides, true)) return false;
    for (int i = 0; i < 3; ++i)
        if (std::max(c.key_strides[i], c.value_strides[i]) > (i == 2 ? R2O_PAGED_MAX_SLOT_STRIDE : 0x7fffffff)) return false;
    if (table->scalar_type() != at::kInt || table->dim() != 2 || table->size(0) < 1 || table->size(1) < 1 ||
        (table->size(1) > 1 && table->stride(1) != 1) || n->scalar_type() != at::kInt || n->dim() != 1 || n->size(0) != table->size(0) ||
        !n->is_contiguous())
        return false;
    c.batch = table->size(0);
    c.max_pages = table->size(1);
    c.table_stride = c.batch > 1 ? table->stride(0) : c.max_pages;
    if (c.table_stride && c.table_stride < c.max_pages) return false;  // rows that overlap
    if (c.batch > R2O_PAGED_MAX_BATCH || c.max_pages * c.page_size > (1 << 29) || c.table_stride > 0x7fffffff) return false;
    if (w) {
        if (!on_device(*w, device) || w->scalar_type() != at::kFloat || w->dim() != 3 || w->size(0) != c.pages || w->size(1) != c.hkv ||
            w->size(2) != c.page_size || w->stride(2) != 1)
            return false;
        for (int i = 0; i < 2; ++i) {
            c.weight_strides[i] = w->size(i) > 1 ? w->stride(i) : 0;
            if (w->size(i) > 1 && (c.weight_strides[i] < 1 || c.weight_strides[i] > 0x7fffffff)) return false;
        }
        c.weight_pages = w->data_ptr<float>();
    }
    c.key_pages = static_cast<uint16_t*>(k->data_ptr());
    c.value_pages = static_cast<uint16_t*>(v->data_ptr());
    c.page_table = table->data_ptr<int32_t>();
    c.lengths = n->data_ptr<int32_t>();
    return true;
}

// One row of page ids for all requests (an expanded table): their pages may be read, not written.
bool one_row(const r2o_paged_cache& c) { return c.batch > 1 && c.table_stride == 0; }

// paged_cache(cache): True if its tensors need no look by the Python path, or None
PyObject* paged_cache_call(PyObject* const* args) {
    Cache cache;
    if (!cache.read(args[0])) Py_RETURN_NONE;
    Py_RETURN_TRUE;
}

bool cache_rows(const at::Tensor* t, const r2o_paged_cache& c, int64_t device) {
    return t && on_device(*t, device) && row_code(*t) == c.dtype && !needs_grad(*t);
}

// paged_extend(function, cache, key, value, counts, weights): (status,) or None
PyObject* paged_extend_call(PyObject* const* args) {
    r2o_paged_extend_params p{};
    Cache cache;
    const at::Tensor *k = exact_tensor(args[2]), *v = exact_tensor(args[3]);
    if (!cache.read(args[1]) || !cache.callable()) Py_RETURN_NONE;
    const int64_t device = cache.device;
    p.cache = cache.c;
    if (one_row(p.cache)) Py_RETURN_NONE;
    if (!cache_rows(k, p.cache, device) || !cache_rows(v, p.cache, device) ||
        k->dim() != 4 || k->size(0) != p.cache.batch || k->size(1) != p.cache.hkv || k->size(3) != R2O_HEAD_DIM || v->sizes() != k->sizes())
        Py_RETURN_NONE;
    p.rows = k->size(2);
    if (p.rows < 1 || p.rows > p.cache.max_pages * p.cache.page_size || !row_strides(*k, 3, p.key_strides) ||
        !row_strides(*v, 3, p.value_strides) || p.key_strides[2] > R2O_MAX_ROW_STRIDE || p.value_strides[2] > R2O_MAX_ROW_STRIDE ||
        !lengths_arg(args[4], p.cache.batch, device, p.counts))
        Py_RETURN_NONE;
    if (args[5] != Py_None) {
        const at::Tensor* w = exact_tensor(args[5]);
        if (!w || !p.cache.weight_pages || needs_grad(*w) || !on_device(*w, device) || w->scalar_type() != at::kFloat || w->dim() != 3 ||
            w->size(0) != k->size(0) || w->size(1) != k->size(1) || w->size(2) != k->size(2) || !w->is_contiguous())
            Py_RETURN_NONE;
        p.weights = w->data_ptr<float>();
        p.weights_strides[0] = w->stride(0);
        p.weights_strides[1] = w->stride(1);
    }
    p.key = static_cast<const uint16_t*>(k->data_ptr());
    p.value = static_cast<const uint16_t*>(v->data_ptr());
    return status_and(launch_on(args[0], p, device), {});
}

// paged_attention(function, cache, query, append or None, window, sinks, scale): (status, out, lse) or None
PyObject* paged_attention_call(PyObject* const* args) {
    r2o_paged_attention_params p{};
    r2o_paged_cache& c = p.cache;
    Cache cache;
    const at::Tensor* q = exact_tensor(args[2]);
    if (!cache.read(args[1]) || !cache.callable()) Py_RETURN_NONE;
    const int64_t device = cache.device;
    c = cache.c;
    if (one_row(c) && (c.weight_pages || args[3] != Py_None)) Py_RETURN_NONE;
    if (!cache_rows(q, c, device) ||
        !(q->dim() == 3 || (q->dim() == 4 && q->size(2) == 1)) || q->size(0) != c.batch || q->size(-1) != R2O_HEAD_DIM)
        Py_RETURN_NONE;
    p.hq = q->size(1);
    if (p.hq < 1 || p.hq % c.hkv || p.hq / c.hkv > R2O_MAX_GQA || !row_strides(*q, 2, p.query_strides) ||
        !mask_args(args[4], args[5], args[6], p.window, p.sinks, p.sm_scale) ||
        std::max(p.query_strides[0], p.query_strides[1]) > 0x7fffffff)
        Py_RETURN_NONE;
    if (args[3] != Py_None) {
        if (!PyTuple_CheckExact(args[3]) || PyTuple_GET_SIZE(args[3]) != 2) Py_RETURN_NONE;
        for (int i = 0; i < 2; ++i) {
            const at::Tensor* t = exact_tensor(PyTuple_GET_ITEM(args[3], i));
            if (!cache_rows(t, c, device) || !(t->dim() == 3 || (t->dim() == 4 && t->size(2) == 1)) || t->size(0) != c.batch ||
                t->size(1) != c.hkv || t->size(-1) != R2O_HEAD_DIM || !row_strides(*t, 2, p.append_strides + 2 * i) ||
                std::max(p.append_strides[2 * i], p.append_strides[2 * i + 1]) > 0x7fffffff)
                Py_RETURN_NONE;
            (i ? p.append_value : p.append_key) = static_cast<const uint16_t*>(t->data_ptr());
        }
    }
    const int64_t capacity = c.max_pages * c.page_size, group = p.hq / c.hkv;
    if (c.batch * c.hkv * div_up(capacity, 32) > 0x7fffffff - R2O_PAGED_MAX_WORKERS) Py_RETURN_NONE;
    p.workers = paged_workers(c.batch, c.hkv, capacity, compute_units((int)device));
    p.partial_states = (p.workers + c.batch * c.hkv) * group;
    p.logits_floats = c.weight_pages ? c.batch * p.hq * div_up(capacity, 32) * 32 : 0;
    const auto f32 = at::TensorOptions().device(q->device()).dtype(at::kFloat);
    at::Tensor out = at::empty({c.batch, p.hq, R2O_HEAD_DIM}, q->options()), lse = at::empty({c.batch, p.hq}, f32);
    at::Tensor scratch = at::empty({130 * p.partial_states + 2 + p.logits_floats}, f32);
    p.query = static_cast<const uint16_t*>(q->data_ptr());
    p.out = static_cast<uint16_t*>(out.data_ptr());
    p.lse = lse.data_ptr<float>();
    p.partial_out = scratch.data_ptr<float>();  // then the (maximum, sum) pairs and, 16-byte aligned, the logits
    p.partial_ml = p.partial_out + 128 * p.partial_states;
    if (p.logits_floats) p.logits = p.partial_out + div_up(130 * p.partial_states, 4) * 4;
    return status_and(launch_on(args[0], p, device), {out, lse});
}

// paged_evict(function, cache, target, keep, sinks, recent): (status, kept) or None
PyObject* paged_evict_call(PyObject* const* args) {
    r2o_paged_evict_params p{};
    Cache source, target;
    if (!source.read(args[1]) || !target.read(args[2]) || !source.callable() || !target.callable() ||
        !plain_int(args[3], p.keep) || !plain_int(args[4], p.sinks) || !plain_int(args[5], p.recent))
        Py_RETURN_NONE;
    const r2o_paged_cache &c = p.source = source.c, &o = p.target = target.c;
    if (!c.weight_pages || one_row(o) || c.batch != o.batch || c.hkv != o.hkv || c.dtype != o.dtype || std::abs(c.lengths - o.lengths) < c.batch ||
        c.page_table == o.page_table || p.keep < 1 || p.keep > o.max_pages * o.page_size || p.sinks < 0 || p.recent < 0 ||
        p.sinks > p.keep || p.recent > p.keep - p.sinks)
        Py_RETURN_NONE;
    const at::Tensor& lengths = THPVariable_Unpack(target.fields[3]);
    at::Tensor kept = at::empty({c.batch, c.hkv, p.keep}, lengths.options());
    p.kept = kept.data_ptr<int32_t>();
    p.target_lengths = lengths.data_ptr<int32_t>();
    return status_and(launch_on(args[0], p, source.device), {kept});
}

template <PyObject* (*CALL)(PyObject* const*), Py_ssize_t N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != N) Py_RETURN_NONE;
    try {
        return CALL(args);
    } catch (...) {  // no memory, or a tensor without memory of its own: the Python path's error
        Py_RETURN_NONE;
    }
}

PyObject* attention_splits_rule(PyObject*, PyObject* args) {
    long long x[8];
    if (!PyArg_ParseTuple(args, "LLLLLLLL", x, x + 1, x + 2, x + 3, x + 4, x + 5, x + 6, x + 7)) return nullptr;
    return PyLong_FromLongLong(attention_splits(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]));
}

PyObject* weight_splits_rule(PyObject*, PyObject* args) {
    long long x[6];
    if (!PyArg_ParseTuple(args, "LLLLLL", x, x + 1, x + 2, x + 3, x + 4, x + 5)) return nullptr;
    return PyLong_FromLongLong(weight_splits(x[0], x[1], x[2], x[3], x[4], x[5]));
}

PyObject* paged_workers_rule(PyObject*, PyObject* args) {
    long long x[4];
    if (!PyArg_ParseTuple(args, "LLLL", x, x + 1, x + 2, x + 3)) return nullptr;
    return PyLong_FromLongLong(paged_workers(x[0], x[1], x[2], x[3]));
}

#define FAST(call, n) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<call, n>)), METH_FASTCALL, nullptr

PyMethodDef kMethods[] = {
    {"decode_handle", decode_handle, METH_VARARGS, nullptr},
    {"decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(decode)), METH_FASTCALL, nullptr},
    {"cache_build", cache_build, METH_VARARGS, nullptr},
    {"prompt", FAST(prompt_call, 9)},
    {"weights", FAST(weights_call, 9)},
    {"paged_cache", FAST(paged_cache_call, 1)},
    {"paged_extend", FAST(paged_extend_call, 6)},
    {"paged_attention", FAST(paged_attention_call, 7)},
    {"paged_evict", FAST(paged_evict_call, 6)},
    {"attention_splits", attention_splits_rule, METH_VARARGS, nullptr},
    {"weight_splits", weight_splits_rule, METH_VARARGS, nullptr},
    {"paged_workers", paged_workers_rule, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_r2o_host", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__r2o_host() { return PyModule_Create(&kModule); }
