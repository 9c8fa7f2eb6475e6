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

PyMethodDef kMethods[] = {{"cache_plan", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(cache_plan)), METH_FASTCALL, nullptr},
                          {"cache_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(cache_append)), METH_FASTCALL, nullptr},
                          {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attend)), METH_FASTCALL, nullptr},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_attention", "The cache and attention entry points for torch tensors.", -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__attention(void) {
    PyObject *lib = PyImport_ImportModule("flashgann_amd._lib");
    if (!lib) return nullptr;
    g_error = PyObject_GetAttrString(lib, "FlashGannError");
    Py_DECREF(lib);
    return g_error ? PyModule_Create(&kModule) : nullptr;
}
