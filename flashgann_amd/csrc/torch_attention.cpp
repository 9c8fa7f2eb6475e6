// torch_attention.cpp -- the cache and attention entry points for torch tensors:
// a CPython module, flashgann_amd._attention.
//
// It checks what the C ABI cannot see (types, shapes, devices), allocates outputs
// and workspace from torch's allocator and queues the call on torch's current
// stream.  In Python the same took 6 to 10 us a call, as much as the kernels of a
// decode step.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <stdexcept>
#include <string>

#include "../../include/flashgann.h"

namespace {

struct Refused : std::runtime_error {  // ValueError
    using std::runtime_error::runtime_error;
};
struct Failed {  // FlashGannError
    int code;
};

PyObject *g_error = nullptr;  // flashgann_amd._lib.FlashGannError

void need(bool ok, const char *what) {
    if (!ok) throw Refused(what);
}

const at::Tensor &tensor(PyObject *o, const char *name) {
    if (!THPVariable_Check(o)) throw Refused(std::string(name) + " must be a tensor");
    return THPVariable_Unpack(o);
}

// No operator here has a gradient: one that autograd would have to pass on is not
// dropped in silence.
void no_gradient(std::initializer_list<const at::Tensor *> ts) {
    if (!c10::GradMode::is_enabled()) return;
    for (const at::Tensor *t : ts)
        need(!t->requires_grad(), "cache_append and attention have no gradient: detach their tensors or call them under torch.no_grad()");
}

// What a call writes in place: autograd has to see it where it saved the tensor.
void written(std::initializer_list<const at::Tensor *> ts) {
    for (const at::Tensor *t : ts)
        if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

int64_t integer(PyObject *o, const char *name, int64_t lo, int64_t hi) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        throw Refused(std::string(name) + " must be an integer");
    }
    if (v < lo || v > hi) throw Refused(std::string(name) + " must be in [" + std::to_string(lo) + ", " + std::to_string(hi) + "]");
    return v;
}

constexpr int64_t kMost = (1ll << 31) - 1;

// The device that all tensors of a call must be on: torch's current one.
struct Call {
    c10::Device device;
    void *stream;
    explicit Call(const at::Tensor &t) : device(t.device()), stream(nullptr) {
        need(t.is_cuda() && t.device().index() == c10::hip::current_device(), "tensors must be on the current CUDA device");
        stream = c10::hip::getCurrentHIPStream(t.device().index()).stream();
    }
    bool has(const at::Tensor &t) const { return t.device() == device; }
    at::Tensor empty(at::IntArrayRef shape, at::ScalarType type) const {
        return at::empty(shape, at::TensorOptions().dtype(type).device(device));
    }
};

void *vector_of(const Call &c, PyObject *o, int64_t n, at::ScalarType type, const char *name) {
    const at::Tensor &t = tensor(o, name);
    if (t.dim() != 1 || t.size(0) != n || t.scalar_type() != type || !c.has(t) || !t.is_contiguous())
        throw Refused(std::string(name) + " must be a contiguous " + c10::toString(type) + " vector of " + std::to_string(n) + " on the same device");
    return t.data_ptr();
}

int dtype_of(at::ScalarType t) {
    need(t == at::kBFloat16 || t == at::kHalf, "k_cache and v_cache must be bfloat16 or float16");
    return t == at::kBFloat16 ? FG_BF16 : FG_F16;
}

uint32_t u32(int64_t v) { return static_cast<uint32_t>(v); }

fg_kv_cache cache_of(const Call &c, const at::Tensor &k, const at::Tensor &v) {
    need(k.dim() == 4 && v.sizes() == k.sizes(), "k_cache and v_cache must have shape (pages, page_size, heads_kv, dim)");
    const int dtype = dtype_of(k.scalar_type());
    need(v.scalar_type() == k.scalar_type(), "k_cache and v_cache must be bfloat16 or float16");
    need(c.has(k) && c.has(v), "k_cache and v_cache must be on the same device");
    need(k.stride(3) == 1 && v.stride(3) == 1, "the last dimension of k_cache and v_cache must be contiguous");
    for (int i = 0; i < 4; ++i) need(k.size(i) <= kMost, "k_cache and v_cache are too large");
    return {k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), v.stride(0), v.stride(1), v.stride(2),
            u32(k.size(0)), u32(k.size(1)), u32(k.size(2)), u32(k.size(3)), dtype, 0};
}

struct Table {
    int32_t *at;
    int64_t row;
    uint32_t width;
};
Table table_of(const Call &c, PyObject *o, int64_t requests) {
    const at::Tensor &t = tensor(o, "block_table");
    if (t.dim() != 2 || t.size(0) != requests || t.scalar_type() != at::kInt || !c.has(t) ||
        (t.stride(1) != 1 && t.size(1) > 1) || t.size(1) > kMost)
        throw Refused("block_table must be int32 of shape (" + std::to_string(requests) + ", width), its rows contiguous, on the same device");
    return {static_cast<int32_t *>(t.data_ptr()), t.stride(0), u32(t.size(1))};
}

PyObject *wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }

PyObject *pack(std::initializer_list<at::Tensor> ts) {
    PyObject *out = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
    Py_ssize_t i = 0;
    for (const at::Tensor &t : ts) {
        PyObject *o = out ? wrap(t) : nullptr;
        if (!o) {
            Py_XDECREF(out);
            return nullptr;
        }
        PyTuple_SET_ITEM(out, i++, o);
    }
    return out;
}

// Runs `body`, its C++ exceptions as Python ones.
template <class F>
PyObject *guarded(F body) {
    try {
        return body();
    } catch (const Refused &e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const Failed &f) {
        PyObject *e = PyObject_CallFunction(g_error, "is", f.code, fg_last_error());
        if (e) {
            PyErr_SetObject(g_error, e);
            Py_DECREF(e);
        }
    } catch (const std::exception &e) {  // torch's allocator
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}

void check(int rc) {
    if (rc != FG_OK) throw Failed{rc};
}

// (lens, new_lens, block_table, free_pages, page_size, max_tokens) -> (q_starts, kv_lens, slots, positions, used)
PyObject *cache_plan(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&] {
        need(n == 6, "cache_plan takes 6 arguments");
        const at::Tensor &lens = tensor(a[0], "lens"), &free_pages = tensor(a[3], "free_pages");
        const Call c(lens);
        need(lens.dim() == 1 && free_pages.dim() == 1 && lens.size(0) <= kMost && free_pages.size(0) <= kMost, "lens and free_pages must be vectors");
        const int64_t requests = lens.size(0), nfree = free_pages.size(0);
        const int64_t page = integer(a[4], "page_size", 1, kMost), tokens = integer(a[5], "max_tokens", 0, kMost);
        const Table t = table_of(c, a[2], requests);
        const auto *l = static_cast<int32_t *>(vector_of(c, a[0], requests, at::kInt, "lens"));
        const auto *m = static_cast<int32_t *>(vector_of(c, a[1], requests, at::kInt, "new_lens"));
        const auto *f = static_cast<int32_t *>(vector_of(c, a[3], nfree, at::kInt, "free_pages"));
        at::Tensor q_starts = c.empty({requests + 1}, at::kInt), kv_lens = c.empty({requests}, at::kInt), slots = c.empty({tokens}, at::kLong),
                   positions = c.empty({tokens}, at::kInt), used = c.empty({1}, at::kInt);
        check(fg_cache_plan(l, m, u32(requests), t.at, t.row, t.width, f, u32(nfree), u32(page), u32(tokens),
                            static_cast<int32_t *>(q_starts.data_ptr()), static_cast<int32_t *>(kv_lens.data_ptr()),
                            static_cast<int64_t *>(slots.data_ptr()), static_cast<int32_t *>(positions.data_ptr()),
                            static_cast<int32_t *>(used.data_ptr()), c.stream));
        written({&tensor(a[2], "block_table")});
        return pack({q_starts, kv_lens, slots, positions, used});
    });
}

// (k, v, k_cache, v_cache, slots)
PyObject *cache_append(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        need(n == 5, "cache_append takes 5 arguments");
        const at::Tensor &k = tensor(a[0], "k"), &v = tensor(a[1], "v"), &kc = tensor(a[2], "k_cache"), &vc = tensor(a[3], "v_cache");
        no_gradient({&k, &v, &kc, &vc});
        const Call c(kc);
        const fg_kv_cache cache = cache_of(c, kc, vc);
        const at::Tensor &slots = tensor(a[4], "slots");
        need(slots.dim() == 1 && slots.size(0) <= kMost, "slots must be a vector");
        const int64_t tokens = slots.size(0);
        need(k.dim() == 3 && k.size(0) == tokens && k.size(1) == kc.size(2) && k.size(2) == kc.size(3) && v.sizes() == k.sizes(),
             "k and v must have shape (tokens, heads_kv, dim), one row a slot");
        need(k.scalar_type() == kc.scalar_type() && v.scalar_type() == kc.scalar_type(), "k and v must have the cache's type");
        need(c.has(k) && c.has(v), "k and v must be on the same device");
        const auto *at = static_cast<int64_t *>(vector_of(c, a[4], tokens, at::kLong, "slots"));
        if (tokens) {
            need(k.stride(2) == 1 && v.stride(2) == 1, "the last dimension of k and v must be contiguous");
            check(fg_cache_append(&cache, k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), v.stride(0), v.stride(1), at, u32(tokens), c.stream));
            written({&kc, &vc});
        }
        Py_RETURN_NONE;
    });
}

// (q, k_cache, v_cache, block_table, q_starts | None, kv_lens, ids | None, max_q, scale | None, window, sinks, out | None, lse | None) -> (out, lse)
PyObject *attend(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&] {
        need(n == 13, "attend takes 13 arguments");
        const at::Tensor &q = tensor(a[0], "q"), &kc = tensor(a[1], "k_cache"), &vc = tensor(a[2], "v_cache");
        no_gradient({&q, &kc, &vc});
        const Call c(q);
        const fg_kv_cache cache = cache_of(c, kc, vc);
        need(q.dim() == 3 && q.size(2) == kc.size(3) && q.scalar_type() == kc.scalar_type(), "q must have shape (tokens, heads, dim) and the cache's type");
        const int64_t tokens = q.size(0), heads = q.size(1), dim = q.size(2);
        need(tokens <= kMost && heads <= kMost, "q is too large");
        need(q.stride(2) == 1 || !tokens, "the last dimension of q must be contiguous");
        at::Tensor out = a[11] == Py_None ? c.empty({tokens, heads, dim}, q.scalar_type()) : tensor(a[11], "out");
        no_gradient({&out});
        need(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && c.has(out) && (out.stride(2) == 1 || !tokens),
             "out must have q's shape and type, its last dimension contiguous, on the same device");
        at::Tensor lse = a[12] == Py_None ? c.empty({tokens, heads}, at::kFloat) : tensor(a[12], "lse");
        no_gradient({&lse});
        need(lse.dim() == 2 && lse.size(0) == tokens && lse.size(1) == heads && lse.scalar_type() == at::kFloat && c.has(lse) && lse.is_contiguous(),
             "lse must be contiguous float32 of shape (tokens, heads) on the same device");
        const at::Tensor &kv_lens = tensor(a[5], "kv_lens");
        need(kv_lens.dim() == 1 && kv_lens.size(0) <= kMost, "kv_lens must be a vector");
        const int64_t requests = kv_lens.size(0);
        const Table t = table_of(c, a[3], requests);
        fg_attention p{};
        p.q = q.data_ptr();
        p.out = out.data_ptr();
        p.lse = static_cast<float *>(lse.data_ptr());
        p.q_token = q.stride(0), p.q_head = q.stride(1), p.out_token = out.stride(0), p.out_head = out.stride(1);
        p.table = t.at;
        p.table_row = t.row;
        p.table_width = t.width;
        p.kv_lens = static_cast<int32_t *>(vector_of(c, a[5], requests, at::kInt, "kv_lens"));
        const bool found = a[6] != Py_None;
        if (found) {
            const at::Tensor &ids = tensor(a[6], "ids");
            need(ids.dim() == 3 && ids.size(0) == requests && (ids.scalar_type() == at::kInt || ids.scalar_type() == at::kUInt32) && c.has(ids) &&
                     ids.is_contiguous() && ids.size(1) <= kMost && ids.size(2) <= kMost,
                 "ids must be contiguous int32 or uint32 of shape (requests, lists, K) on the same device");
            p.ids = static_cast<uint32_t *>(ids.data_ptr());
            p.lists = u32(ids.size(1));
            p.nids = u32(ids.size(2));
        } else {
            p.q_starts = static_cast<int32_t *>(vector_of(c, a[4], requests + 1, at::kInt, "q_starts"));
        }
        p.requests = u32(requests);
        p.tokens = u32(tokens);
        p.heads = u32(heads);
        p.max_q = u32(integer(a[7], "max_q", 0, kMost));
        p.scale = a[8] == Py_None ? static_cast<float>(1.0 / std::sqrt(static_cast<double>(dim))) : static_cast<float>(PyFloat_AsDouble(a[8]));
        if (PyErr_Occurred()) {
            PyErr_Clear();
            throw Refused("scale must be a number");
        }
        p.window = a[9] == Py_None ? -1 : static_cast<int32_t>(integer(a[9], "window", found ? 0 : 1, kMost));
        p.sinks = u32(integer(a[10], "sinks", 0, kMost));
        if (found && (p.lists == 0 || tokens != requests)) need(false, "ids must have a list or more, and q one row a request");
        const int64_t bytes = fg_attend_workspace_bytes(&cache, &p);
        if (bytes < 0) throw Failed{static_cast<int>(bytes)};
        at::Tensor work;
        if (bytes) work = c.empty({bytes}, at::kByte);
        check((found ? fg_attend_retrieved : fg_attend)(&cache, &p, bytes ? work.data_ptr() : nullptr, static_cast<uint64_t>(bytes), c.stream));
        if (a[11] != Py_None) written({&out});
        if (a[12] != Py_None) written({&lse});
        return pack({out, lse});
    });
}

// What calls over rows of q share: q, its requests and their table.
struct Rows {
    int64_t tokens, heads, requests;
    fg_attention p{};
};
Rows rows_of(const Call &c, const at::Tensor &q, int64_t dim, PyObject *table, PyObject *q_starts, PyObject *lens) {
    Rows w;
    need(q.dim() == 3 && q.size(2) == dim && c.has(q), "q must have shape (tokens, heads, dim), on the same device");
    w.tokens = q.size(0), w.heads = q.size(1);
    need(w.tokens <= kMost && w.heads <= kMost, "q is too large");
    need(q.stride(2) == 1 || !w.tokens, "the last dimension of q must be contiguous");
    const at::Tensor &kv_lens = tensor(lens, "kv_lens");
    need(kv_lens.dim() == 1 && kv_lens.size(0) <= kMost, "kv_lens must be a vector");
    w.requests = kv_lens.size(0);
    const Table t = table_of(c, table, w.requests);
    w.p.q = q.data_ptr();
    w.p.q_token = q.stride(0), w.p.q_head = q.stride(1);
    w.p.table = t.at, w.p.table_row = t.row, w.p.table_width = t.width;
    w.p.kv_lens = static_cast<int32_t *>(vector_of(c, lens, w.requests, at::kInt, "kv_lens"));
    w.p.q_starts = static_cast<int32_t *>(vector_of(c, q_starts, w.requests + 1, at::kInt, "q_starts"));
    w.p.requests = u32(w.requests);
    w.p.tokens = u32(w.tokens);
    w.p.heads = u32(w.heads);
    return w;
}

float scale_of(PyObject *o, int64_t dim) {
    const float s = static_cast<float>(o == Py_None ? 1.0 / std::sqrt(static_cast<double>(dim)) : PyFloat_AsDouble(o));
    if (PyErr_Occurred()) {
        PyErr_Clear();
        throw Refused("scale must be a number");
    }
    return s;
}

at::Tensor workspace(const Call &c, int64_t bytes) {
    if (bytes < 0) throw Failed{static_cast<int>(bytes)};
    return bytes ? c.empty({bytes}, at::kByte) : at::Tensor();
}
void *start_of(const at::Tensor &work) { return work.defined() ? work.data_ptr() : nullptr; }

// (codes, scales) of a cache's pages
void bounds_of(const Call &c, const at::Tensor &bounds, const at::Tensor &scales) {
    need(bounds.dim() == 4 && bounds.size(2) == 2 && bounds.scalar_type() == at::kChar && c.has(bounds) && bounds.is_contiguous(),
         "bounds must be contiguous int8 of shape (pages, heads_kv, 2, dim) on the same device");
    need(scales.dim() == 2 && scales.size(0) == bounds.size(0) && scales.size(1) == bounds.size(1) && scales.scalar_type() == at::kFloat &&
             c.has(scales) && scales.is_contiguous(),
         "scales must be contiguous float32 of shape (pages, heads_kv) on the same device");
}

// (k_cache, slots, bounds, scales)
PyObject *cache_bounds(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        need(n == 4, "cache_bounds takes 4 arguments");
        const at::Tensor &k = tensor(a[0], "k_cache"), &slots = tensor(a[1], "slots"), &bounds = tensor(a[2], "bounds"), &scales = tensor(a[3], "scales");
        no_gradient({&k, &scales});
        const Call c(k);
        const fg_kv_cache cache = cache_of(c, k, k);
        bounds_of(c, bounds, scales);
        need(bounds.size(0) == k.size(0) && bounds.size(1) == k.size(2) && bounds.size(3) == k.size(3), "bounds must have shape (pages, heads_kv, 2, dim)");
        need(slots.dim() == 1 && slots.size(0) <= kMost, "slots must be a vector");
        const int64_t tokens = slots.size(0);
        const auto *at = static_cast<int64_t *>(vector_of(c, a[1], tokens, at::kLong, "slots"));
        check(fg_cache_bounds(&cache, at, u32(tokens), static_cast<int8_t *>(bounds.data_ptr()), static_cast<float *>(scales.data_ptr()), c.stream));
        if (tokens) written({&bounds, &scales});
        Py_RETURN_NONE;
    });
}

// (q, bounds, scales, block_table, q_starts, kv_lens, page_size, k, lists | None, first_blocks, last_blocks) -> ids
PyObject *select_blocks(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&] {
        need(n == 11, "select_blocks takes 11 arguments");
        const at::Tensor &q = tensor(a[0], "q"), &bounds = tensor(a[1], "bounds"), &scales = tensor(a[2], "scales");
        no_gradient({&q, &scales});
        const Call c(q);
        bounds_of(c, bounds, scales);
        need(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf, "q must be bfloat16 or float16");
        for (int i = 0; i < 4; ++i) need(bounds.size(i) <= kMost, "bounds are too large");
        fg_kv_cache cache{};
        cache.pages = u32(bounds.size(0)), cache.heads_kv = u32(bounds.size(1)), cache.dim = u32(bounds.size(3));
        cache.page_size = u32(integer(a[6], "page_size", 1, kMost));
        cache.dtype = q.scalar_type() == at::kBFloat16 ? FG_BF16 : FG_F16;
        Rows w = rows_of(c, q, bounds.size(3), a[3], a[4], a[5]);
        w.p.nids = u32(integer(a[7], "k", 1, kMost));
        w.p.lists = a[8] == Py_None ? cache.heads_kv : u32(integer(a[8], "lists", 1, kMost));
        w.p.sinks = u32(integer(a[9], "first_blocks", 0, kMost));
        w.p.window = static_cast<int32_t>(integer(a[10], "last_blocks", 1, kMost));
        const int64_t bytes = fg_select_blocks_workspace_bytes(&cache, &w.p);
        const at::Tensor work = workspace(c, bytes);
        at::Tensor ids = c.empty({w.tokens, static_cast<int64_t>(w.p.lists), static_cast<int64_t>(w.p.nids)}, at::kInt);
        check(fg_select_blocks(&cache, &w.p, static_cast<int8_t *>(bounds.data_ptr()), static_cast<float *>(scales.data_ptr()),
                               static_cast<int32_t *>(ids.data_ptr()), start_of(work), static_cast<uint64_t>(bytes), c.stream));
        return wrap(ids);
    });
}

// (q, k_cache, v_cache, block_table, q_starts, kv_lens, ids, first_blocks, last_blocks, scale | None, out | None, lse | None) -> (out, lse)
PyObject *attend_blocks(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&] {
        need(n == 12, "attend_blocks takes 12 arguments");
        const at::Tensor &q = tensor(a[0], "q"), &kc = tensor(a[1], "k_cache"), &vc = tensor(a[2], "v_cache"), &ids = tensor(a[6], "ids");
        no_gradient({&q, &kc, &vc});
        const Call c(q);
        const fg_kv_cache cache = cache_of(c, kc, vc);
        need(q.scalar_type() == kc.scalar_type(), "q must have the cache's type");
        Rows w = rows_of(c, q, kc.size(3), a[3], a[4], a[5]);
        need(ids.dim() == 3 && ids.size(0) == w.tokens && ids.scalar_type() == at::kInt && c.has(ids) && ids.is_contiguous() && ids.size(1) <= kMost &&
                 ids.size(2) <= kMost,
             "ids must be contiguous int32 of shape (tokens, lists, k) on the same device");
        at::Tensor out = a[10] == Py_None ? c.empty({w.tokens, w.heads, q.size(2)}, q.scalar_type()) : tensor(a[10], "out");
        at::Tensor lse = a[11] == Py_None ? c.empty({w.tokens, w.heads}, at::kFloat) : tensor(a[11], "lse");
        no_gradient({&out, &lse});
        need(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && c.has(out) && (out.stride(2) == 1 || !w.tokens),
             "out must have q's shape and type, its last dimension contiguous, on the same device");
        need(lse.dim() == 2 && lse.size(0) == w.tokens && lse.size(1) == w.heads && lse.scalar_type() == at::kFloat && c.has(lse) && lse.is_contiguous(),
             "lse must be contiguous float32 of shape (tokens, heads) on the same device");
        w.p.out = out.data_ptr();
        w.p.out_token = out.stride(0), w.p.out_head = out.stride(1);
        w.p.lse = static_cast<float *>(lse.data_ptr());
        w.p.ids = reinterpret_cast<uint32_t *>(ids.data_ptr());
        w.p.lists = u32(ids.size(1)), w.p.nids = u32(ids.size(2));
        w.p.sinks = u32(integer(a[7], "first_blocks", 0, kMost));
        w.p.window = static_cast<int32_t>(integer(a[8], "last_blocks", 1, kMost));
        w.p.scale = scale_of(a[9], q.size(2));
        const int64_t bytes = fg_attend_blocks_workspace_bytes(&cache, &w.p);
        const at::Tensor work = workspace(c, bytes);
        check(fg_attend_blocks(&cache, &w.p, start_of(work), static_cast<uint64_t>(bytes), c.stream));
        if (a[10] != Py_None) written({&out});
        if (a[11] != Py_None) written({&lse});
        return pack({out, lse});
    });
}

void weights_of(const Call &c, const at::Tensor &weights, const at::Tensor &k) {
    need(weights.dim() == 3 && weights.size(0) == k.size(0) && weights.size(1) == k.size(2) && weights.size(2) == k.size(1) &&
             weights.scalar_type() == at::kFloat && c.has(weights) && weights.is_contiguous(),
         "weights must be contiguous float32 of shape (pages, heads_kv, page_size) on the same device");
}

// (q, k_cache, block_table, q_starts, kv_lens, lse, weights, known, scale | None)
PyObject *cache_weigh(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        need(n == 9, "cache_weigh takes 9 arguments");
        const at::Tensor &q = tensor(a[0], "q"), &kc = tensor(a[1], "k_cache"), &lse = tensor(a[5], "lse"), &weights = tensor(a[6], "weights");
        no_gradient({&q, &kc, &lse, &weights});
        const Call c(q);
        const fg_kv_cache cache = cache_of(c, kc, kc);
        need(q.scalar_type() == kc.scalar_type(), "q must have the cache's type");
        Rows w = rows_of(c, q, kc.size(3), a[2], a[3], a[4]);
        need(lse.dim() == 2 && lse.size(0) == w.tokens && lse.size(1) == w.heads && lse.scalar_type() == at::kFloat && c.has(lse) && lse.is_contiguous(),
             "lse must be contiguous float32 of shape (tokens, heads) on the same device");
        weights_of(c, weights, kc);
        const auto *known = static_cast<int32_t *>(vector_of(c, a[7], w.requests, at::kInt, "known"));
        w.p.lse = static_cast<float *>(lse.data_ptr());
        w.p.scale = scale_of(a[8], q.size(2));
        check(fg_cache_weigh(&cache, &w.p, static_cast<float *>(weights.data_ptr()), known, c.stream));
        written({&weights});
        Py_RETURN_NONE;
    });
}

// (k_cache, v_cache, weights, block_table, kv_lens, budget, window, sinks) -> (kv_lens, freed, released)
PyObject *cache_evict(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&] {
        need(n == 8, "cache_evict takes 8 arguments");
        const at::Tensor &kc = tensor(a[0], "k_cache"), &vc = tensor(a[1], "v_cache"), &weights = tensor(a[2], "weights");
        no_gradient({&kc, &vc, &weights});
        const Call c(kc);
        const fg_kv_cache cache = cache_of(c, kc, vc);
        weights_of(c, weights, kc);
        const at::Tensor &kv_lens = tensor(a[4], "kv_lens");
        need(kv_lens.dim() == 1 && kv_lens.size(0) <= kMost, "kv_lens must be a vector");
        const int64_t requests = kv_lens.size(0);
        const Table t = table_of(c, a[3], requests);
        const auto *lens = static_cast<int32_t *>(vector_of(c, a[4], requests, at::kInt, "kv_lens"));
        const uint32_t budget = u32(integer(a[5], "budget", 1, kMost)), window = u32(integer(a[6], "window", 0, kMost)), sinks = u32(integer(a[7], "sinks", 0, kMost));
        const int64_t bytes = fg_cache_evict_workspace_bytes(&cache, t.width, u32(requests), budget);
        const at::Tensor work = workspace(c, bytes);
        at::Tensor left = c.empty({requests}, at::kInt), freed = c.empty({requests * t.width}, at::kInt), released = c.empty({1}, at::kInt);
        check(fg_cache_evict(&cache, static_cast<float *>(weights.data_ptr()), t.at, t.row, t.width, lens, u32(requests), budget, window, sinks,
                             static_cast<int32_t *>(left.data_ptr()), static_cast<int32_t *>(freed.data_ptr()), static_cast<int32_t *>(released.data_ptr()),
                             start_of(work), static_cast<uint64_t>(bytes), c.stream));
        written({&kc, &vc, &weights});
        return pack({left, freed, released});
    });
}

#define FG_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {FG_METHOD(cache_plan), FG_METHOD(cache_append), FG_METHOD(attend), FG_METHOD(cache_bounds), FG_METHOD(select_blocks),
                          FG_METHOD(attend_blocks), FG_METHOD(cache_weigh), FG_METHOD(cache_evict), {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_attention", "The cache and attention entry points for torch tensors.", -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__attention(void) {
    PyObject *lib = PyImport_ImportModule("flashgann_amd._lib");
    if (!lib) return nullptr;
    g_error = PyObject_GetAttrString(lib, "FlashGannError");
    Py_DECREF(lib);
    return g_error ? PyModule_Create(&kModule) : nullptr;
}
