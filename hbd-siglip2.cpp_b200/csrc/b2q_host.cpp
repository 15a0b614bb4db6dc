// b2q_host.cpp — the decode calls from Python in one native step: checks of the
// tensors, their addresses, and the C entry point.
//
// A decode step makes these calls on tensors of a few rows, where the GPU needs 2 to 5
// us a launch and the interpreter, reading a dozen attributes of a dozen tensors and
// handing them to ctypes, took 3 to 4 us on top of the 4.5 of the C call.  Each function
// here takes what its Python namesake takes and returns the C entry point's status, or
// None where anything is not as it should be (a type, a shape, a stride, a device):
// the caller then goes through its own checks, which say what is wrong.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>

#include "../../include/b2q.h"

namespace {

// The entry points of the library that the binding has loaded.
decltype(&b2q_kv_plan) f_plan;
decltype(&b2q_qk_norm_rope) f_rope;
decltype(&b2q_attention_paged) f_paged;
decltype(&b2q_attention_paged_scratch_bytes) f_scratch;
decltype(&b2q_mul_vec_q4) f_vec;

// Reads the arguments in order; `ok` falls where one is not as it should be.
struct Args {
    PyObject* const* a;
    int device;
    bool ok = true;
    int i = 0;

    PyObject* next() { return a[i++]; }
    // A strided tensor on the current device, or nullptr.
    const at::Tensor* tensor() {
        PyObject* o = next();
        if (!THPVariable_CheckExact(o)) return fail();
        const at::Tensor& t = THPVariable_Unpack(o);
        if (t.layout() != at::kStrided || !t.is_cuda() || t.get_device() != device) return fail();
        return &t;
    }
    const at::Tensor* optional() {
        if (a[i] != Py_None) return tensor();
        ++i;
        return nullptr;
    }
    const at::Tensor* fail() {
        ok = false;
        return nullptr;
    }
    int64_t integer() {
        const long long v = PyLong_AsLongLong(next());
        if (v == -1 && PyErr_Occurred()) {
            PyErr_Clear();
            ok = false;
        }
        return v;
    }
    int32_t small() { return narrow(integer()); }
    double real() {
        const double v = PyFloat_AsDouble(next());
        if (v == -1.0 && PyErr_Occurred()) {
            PyErr_Clear();
            ok = false;
        }
        return v;
    }
    int32_t narrow(int64_t v) {
        if (v != static_cast<int32_t>(v)) ok = false;
        return static_cast<int32_t>(v);
    }
    // A cache's description and its device.
    const b2q_kv_cache* cache() {
        const auto* c = static_cast<const b2q_kv_cache*>(PyLong_AsVoidPtr(next()));
        if (!c) {
            PyErr_Clear();
            ok = false;
        }
        if (integer() != device) ok = false;
        return c;
    }
    void* stream() {
        PyObject* o = next();
        if (o == Py_None) return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
        PyObject* v = PyObject_GetAttrString(o, "cuda_stream");
        void* s = v ? PyLong_AsVoidPtr(v) : nullptr;
        Py_XDECREF(v);
        if (PyErr_Occurred()) {
            PyErr_Clear();
            ok = false;
        }
        return s;
    }

    int32_t type(const at::Tensor& t) {
        switch (t.scalar_type()) {
            case at::kFloat: return B2Q_TYPE_F32;
            case at::kHalf: return B2Q_TYPE_F16;
            case at::kBFloat16: return B2Q_TYPE_BF16;
            default: ok = false; return -1;
        }
    }
    // Row stride of a [rows][width] tensor whose columns are contiguous.
    int64_t rows(const at::Tensor& t, int64_t width) {
        if (t.dim() != 2 || t.size(1) != width || (t.stride(1) != 1 && width > 1)) {
            ok = false;
            return 0;
        }
        return t.size(0) > 1 && !t.is_contiguous() ? t.stride(0) : width;
    }
    // Address of a contiguous tensor of n entries of a type; nullptr for none.
    void* entries(const at::Tensor* t, at::ScalarType type, int64_t n) {
        if (!t) return nullptr;
        if (t->scalar_type() != type || t->numel() != n || !t->is_contiguous()) ok = false;
        return t->data_ptr();
    }
};

PyObject* result(b2q_status s) { return PyLong_FromLong(s); }

template <class Fn>
b2q_status unlocked(Fn fn) {   // a full launch queue blocks: not with the interpreter's lock held
    b2q_status s;
    Py_BEGIN_ALLOW_THREADS
    s = fn();
    Py_END_ALLOW_THREADS
    return s;
}

// fn(Args&) with the number of arguments and the current device; exceptions are left to the caller's checks
template <class Fn>
PyObject* guarded(PyObject* const* a, Py_ssize_t n, Py_ssize_t want, bool ready, Fn fn) {
    if (n == want && ready) {
        try {
            Args g{a, static_cast<int>(c10::cuda::current_device())};
            PyObject* r = fn(g);
            if (r) return r;
        } catch (const std::exception&) {
        }
    }
    Py_RETURN_NONE;
}

// ctx_len, new_len, page_size, free_pages, block_table, seq_of, pos, slot, kv_len, counts, stream
PyObject* kv_plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(a, n, 11, f_plan, [](Args& g) -> PyObject* {
        const at::Tensor *ctx = g.tensor(), *add = g.tensor();
        const int32_t page = g.small();
        const at::Tensor *free_pages = g.tensor(), *table = g.tensor();
        const at::Tensor* out[5];
        for (auto& t : out) t = g.tensor();
        void* stream = g.stream();
        if (!g.ok || table->scalar_type() != at::kInt || table->dim() != 2 || table->size(0) != ctx->numel())
            return nullptr;
        const int64_t n_seq = ctx->numel(), rows = out[0]->numel(), n_free = free_pages->numel();
        const auto i32 = [&](const at::Tensor* t, int64_t k) { return static_cast<int32_t*>(g.entries(t, at::kInt, k)); };
        const int32_t *pc = i32(ctx, n_seq), *pa = i32(add, n_seq), *pf = i32(free_pages, n_free);
        int32_t* po[5];
        for (int k = 0; k < 5; ++k) po[k] = i32(out[k], k < 4 ? rows : 2);
        const int64_t width = table->size(1), stride = g.rows(*table, width);
        const int32_t s32 = g.narrow(n_seq), f32 = g.narrow(n_free), w32 = g.narrow(width), r32 = g.narrow(rows);
        if (!g.ok) return nullptr;
        return result(unlocked([&] {
            return f_plan(pc, pa, s32, page, pf, f32, static_cast<int32_t*>(table->data_ptr()), stride, w32, r32, po[0],
                          po[1], po[2], po[3], po[4], stream);
        }));
    });
}

// qkv, n_head, cache's description, its device, q_out, pos, slot, q_weight, k_weight, eps, rope, interleaved, stream
PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(a, n, 13, f_rope, [](Args& g) -> PyObject* {
        const at::Tensor* x = g.tensor();
        const int32_t n_head = g.small();
        const b2q_kv_cache* c = g.cache();
        const at::Tensor *q = g.tensor(), *pos = g.tensor(), *slot = g.tensor(), *qw = g.optional(), *kw = g.optional();
        const double eps = g.real();
        const at::Tensor* rope = g.optional();
        const int interleaved = PyObject_IsTrue(g.next());
        void* stream = g.stream();
        if (!g.ok || interleaved < 0) {
            PyErr_Clear();
            return nullptr;
        }
        const int64_t d = c->d_head;
        const int64_t ld = g.rows(*x, (n_head + 2ll * c->n_kv_head) * d), ldq = g.rows(*q, n_head * d);
        if (!g.ok) return nullptr;
        const int64_t rows = x->size(0);
        if (q->size(0) != rows || g.type(*q) != c->dtype) return nullptr;
        const int32_t type = g.type(*x);
        int32_t n_pos = 0, rot = 0;
        if (rope) {
            if (rope->dim() != 2) return nullptr;
            n_pos = g.narrow(rope->size(0));
            rot = g.narrow(rope->size(1));
            g.entries(rope, at::kFloat, rope->numel());
        }
        const auto* pq = static_cast<const float*>(g.entries(qw, at::kFloat, d));
        const auto* pk = static_cast<const float*>(g.entries(kw, at::kFloat, d));
        const auto* pp = static_cast<const int32_t*>(g.entries(pos, at::kInt, rows));
        const auto* ps = static_cast<const int32_t*>(g.entries(slot, at::kInt, rows));
        if (!g.ok) return nullptr;
        const float* pr = rope && rot ? static_cast<const float*>(rope->data_ptr()) : nullptr;
        return result(unlocked([&] {
            return f_rope(x->data_ptr(), type, ld, rows, n_head, pq, pk, static_cast<float>(eps), pr, n_pos, rot,
                          interleaved, pp, ps, q->data_ptr(), ldq, c, stream);
        }));
    });
}

// q, cache's description, its device, block_table, kv_len, out, scratch, seq_of, scale, window, lse, stream
PyObject* attention_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(a, n, 12, f_paged && f_scratch, [](Args& g) -> PyObject* {
        const at::Tensor* q = g.tensor();
        const b2q_kv_cache* c = g.cache();
        const at::Tensor *table = g.tensor(), *len = g.tensor(), *out = g.tensor(), *scratch = g.tensor();
        const at::Tensor* seq = g.optional();
        if (!g.ok) return nullptr;
        const int64_t d = c->d_head;
        double scale = 0.0;
        if (g.a[g.i] == Py_None) {
            ++g.i;
            scale = std::pow(static_cast<double>(d), -0.5);
        } else {
            scale = g.real();
        }
        const int32_t window = g.small();
        const at::Tensor* lse = g.optional();
        void* stream = g.stream();
        if (!g.ok || q->dim() != 2 || out->sizes() != q->sizes() || g.type(*q) != c->dtype || table->dim() != 2 ||
            table->scalar_type() != at::kInt)
            return nullptr;
        const int64_t rows = q->size(0), width = q->size(1);
        const int32_t n_head = g.narrow(width / d);
        const int64_t ldq = g.rows(*q, n_head * d), ldo = g.rows(*out, width), stride = g.rows(*table, table->size(1));
        const int32_t type = g.type(*out), blocks = g.narrow(table->size(1)), requests = g.narrow(table->size(0));
        const auto* pl = static_cast<const int32_t*>(g.entries(len, at::kInt, rows));
        const auto* ps = static_cast<const int32_t*>(g.entries(seq, at::kInt, rows));
        auto* pe = static_cast<float*>(g.entries(lse, at::kFloat, rows * n_head));
        if (!g.ok) return nullptr;
        const size_t need = f_scratch(n_head, c->n_kv_head, c->d_head);
        if (!need || static_cast<size_t>(scratch->numel()) < need || !scratch->is_contiguous()) return nullptr;
        return result(unlocked([&] {
            return f_paged(q->data_ptr(), ldq, rows, n_head, c, static_cast<const int32_t*>(table->data_ptr()), stride,
                           blocks, requests, ps, pl, static_cast<float>(scale), window, out->data_ptr(), type, ldo, pe,
                           scratch->data_ptr(), stream);
        }));
    });
}

// handle, n, x, m, y, bias, residual, stream
PyObject* mul_vec_q4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(a, n, 8, f_vec, [](Args& g) -> PyObject* {
        const auto* w = static_cast<const b2q_weight_q4*>(PyLong_AsVoidPtr(g.next()));
        if (!w) {   // a released weight (None) among them
            PyErr_Clear();
            return nullptr;
        }
        const int64_t cols = g.integer();
        const at::Tensor* x = g.tensor();
        const int64_t m = g.integer();
        const at::Tensor *y = g.tensor(), *bias = g.optional(), *res = g.optional();
        void* stream = g.stream();
        if (!g.ok || x->dim() != 2) return nullptr;
        const int64_t x_cols = x->size(1), ldx = g.rows(*x, x_cols), ldy = g.rows(*y, cols);
        if (!g.ok || x->size(0) < m || y->size(0) < m) return nullptr;
        if (res && (res->scalar_type() != at::kFloat || res->sizes() != y->sizes() || g.rows(*res, cols) != ldy))
            return nullptr;
        const int32_t xt = g.type(*x), yt = g.type(*y);
        const auto* pb = static_cast<const float*>(g.entries(bias, at::kFloat, cols));
        if (!g.ok) return nullptr;
        return result(unlocked([&] {
            return f_vec(w, x->data_ptr(), xt, m, x_cols, ldx, y->data_ptr(), yt, ldy, pb,
                         res ? static_cast<const float*>(res->data_ptr()) : nullptr, stream);
        }));
    });
}

// The addresses of kv_plan, qk_norm_rope, attention_paged, its scratch_bytes, mul_vec_q4.
PyObject* setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 5) {
        PyErr_SetString(PyExc_TypeError, "setup takes five addresses");
        return nullptr;
    }
    void* p[5];
    for (int i = 0; i < 5; ++i) p[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) return nullptr;
    f_plan = reinterpret_cast<decltype(f_plan)>(p[0]);
    f_rope = reinterpret_cast<decltype(f_rope)>(p[1]);
    f_paged = reinterpret_cast<decltype(f_paged)>(p[2]);
    f_scratch = reinterpret_cast<decltype(f_scratch)>(p[3]);
    f_vec = reinterpret_cast<decltype(f_vec)>(p[4]);
    Py_RETURN_NONE;
}

template <PyObject* (*fn)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL, nullptr};
}

}  // namespace

PyMODINIT_FUNC PyInit_b2q_host() {
    static PyMethodDef methods[] = {method<setup>("setup"),
                                    method<kv_plan>("kv_plan"),
                                    method<qk_norm_rope>("qk_norm_rope"),
                                    method<attention_paged>("attention_paged"),
                                    method<mul_vec_q4>("mul_vec_q4"),
                                    {nullptr, nullptr, 0, nullptr}};
    static PyModuleDef module = {PyModuleDef_HEAD_INIT, "b2q_host", nullptr, -1, methods, nullptr, nullptr, nullptr,
                                 nullptr};
    return PyModule_Create(&module);
}
