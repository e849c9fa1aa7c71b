// Token-loop calls from Python: a call's tensors looked at and handed to libkq in one step.
//
// The operators of a token loop run for a few microseconds, less than Python takes to look at six to ten tensors'
// device, type, shape and strides and to convert their numbers for a foreign call (append of one token 7.3 us through
// ops.py's checks, 2.9 us of it on the GPU).  Each function here makes exactly those checks.  Tensors that are as they should be go
// to the C ABI of include/kq.h, whose status is returned; anything else returns None, and ops.py's own checks say what
// is wrong.  What an object holds for its life (cache layout, page table, workspace) comes as a plan, made once.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <new>

#include "kq.h"

namespace {

struct Plan {
    const int32_t* table;
    int64_t ldt;
    int seqs, width, q_heads, heads, dim, max_len, rope_rows, rot, interleaved;
    const float* rope;
    float scale;
    void* ws;
    size_t ws_bytes;
};

// A device tensor of one type; ok turns false when a tensor is not as it should be.
struct Look {
    bool ok = true;
    const at::Tensor* tensor(PyObject* o, at::ScalarType type) {
        if (!ok || !THPVariable_Check(o)) return ok = false, nullptr;
        const at::Tensor& t = THPVariable_Unpack(o);
        if (!t.is_cuda() || t.scalar_type() != type) return ok = false, nullptr;
        return &t;
    }
    // [rows][cols] at least, rows contiguous
    template <class T>
    T* mat(PyObject* o, at::ScalarType type, int64_t rows, int64_t cols, int64_t* ld) {
        const at::Tensor* t = tensor(o, type);
        if (!t) return nullptr;
        if (t->dim() != 2 || t->size(0) < rows || t->size(1) < cols || (t->stride(1) != 1 && t->size(1) > 1))
            return ok = false, nullptr;
        *ld = t->stride(0);
        return static_cast<T*>(t->data_ptr());
    }
    // n values at least, contiguous; None where it may be left out
    template <class T>
    T* list(PyObject* o, at::ScalarType type, int64_t n, bool needed) {
        if (o == Py_None) return ok = ok && !needed, nullptr;
        const at::Tensor* t = tensor(o, type);
        if (!t) return nullptr;
        if (t->numel() < n || !t->is_contiguous()) return ok = false, nullptr;
        return static_cast<T*>(t->data_ptr());
    }
    // its second size, or -1
    int64_t cols(PyObject* o) {
        if (!THPVariable_Check(o)) return ok = false, -1;
        const at::Tensor& t = THPVariable_Unpack(o);
        return t.dim() == 2 ? t.size(1) : (ok = false, -1);
    }
    int64_t rows(PyObject* o) {
        if (!THPVariable_Check(o)) return ok = false, -1;
        const at::Tensor& t = THPVariable_Unpack(o);
        return t.dim() == 2 ? t.size(0) : (ok = false, -1);
    }
};

constexpr auto F32 = at::kFloat, I32 = at::kInt;

void* pointer(PyObject* o) { return o == Py_None ? nullptr : PyLong_AsVoidPtr(o); }

Plan* plan_of(PyObject* o) { return static_cast<Plan*>(PyCapsule_GetPointer(o, "kq plan")); }

void drop_plan(PyObject* o) { delete plan_of(o); }

// A C++ exception out of a tensor's accessors ends here; ops.py meets the same tensor and raises in its own words.
template <class F>
PyObject* guarded(F f) {
    try {
        return f();
    } catch (...) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
}

bool sizes_fit(int64_t a, int64_t b = 0) { return a <= INT_MAX && b <= INT_MAX; }

// plan(table, rope, q_heads, heads, dim, max_len, interleaved, scale, ws): table (pointer, row stride, rows, columns),
// rope (pointer or None, rows, columns), ws (pointer, bytes)
PyObject* plan(PyObject*, PyObject* args) {
    Plan p = {};
    PyObject *table, *rope, *ws;
    long long ldt = 0;
    Py_ssize_t bytes = 0;
    if (!PyArg_ParseTuple(args, "(OLii)(Oii)iiiiif(On)", &table, &ldt, &p.seqs, &p.width, &rope, &p.rope_rows, &p.rot, &p.q_heads,
                          &p.heads, &p.dim, &p.max_len, &p.interleaved, &p.scale, &ws, &bytes))
        return nullptr;
    p.ldt = ldt;
    p.ws_bytes = (size_t)bytes;
    p.table = static_cast<const int32_t*>(pointer(table));
    p.rope = static_cast<const float*>(pointer(rope));
    p.ws = pointer(ws);
    if (PyErr_Occurred()) return nullptr;
    Plan* held = new (std::nothrow) Plan(p);
    if (!held) return PyErr_NoMemory();
    return PyCapsule_New(held, "kq plan", drop_plan);
}

// append(plan, cache, stream, q, k, v, seq, pos, q_out)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 9) Py_RETURN_NONE;
        const Plan* p = plan_of(a[0]);
        const auto* kv = static_cast<const kq_kv*>(pointer(a[1]));
        void* stream = pointer(a[2]);
        if (PyErr_Occurred()) return nullptr;
        Look see;
        const int64_t N = see.rows(a[4]);
        int64_t ldq = 0, ldo = 0, ldk = 0, ldv = 0;
        const float* q = nullptr;
        float* out = nullptr;
        if (a[3] != Py_None || a[8] != Py_None) {
            q = see.mat<float>(a[3], F32, N, (int64_t)p->q_heads * p->dim, &ldq);
            out = see.mat<float>(a[8], F32, N, (int64_t)p->q_heads * p->dim, &ldo);
        }
        const float* k = see.mat<float>(a[4], F32, N, (int64_t)p->heads * p->dim, &ldk);
        const float* v = see.mat<float>(a[5], F32, N, (int64_t)p->heads * p->dim, &ldv);
        const int32_t* seq = see.list<int32_t>(a[6], I32, N, true);
        const int32_t* pos = see.list<int32_t>(a[7], I32, N, true);
        if (!see.ok || !sizes_fit(N)) Py_RETURN_NONE;
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = kq_kv_append(kv, p->table, p->ldt, p->seqs, p->width, (int)N, seq, pos, q, ldq, p->q_heads, out, ldo,
            k, ldk, v, ldv, p->rope, p->rope_rows, p->rot, p->interleaved, stream);
        Py_END_ALLOW_THREADS
        return PyLong_FromLong(rc);
    });
}

// attend(plan, cache, stream, q, lens, out, tokens)
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 7) Py_RETURN_NONE;
        const Plan* p = plan_of(a[0]);
        const auto* kv = static_cast<const kq_kv*>(pointer(a[1]));
        void* stream = pointer(a[2]);
        const long T = PyLong_AsLong(a[6]);
        if (PyErr_Occurred()) return nullptr;
        if (T < 1 || T > KQ_MAX_BATCH) Py_RETURN_NONE;
        Look see;
        int64_t ldq = 0, ldo = 0;
        const int64_t rows = (int64_t)p->seqs * T, cols = (int64_t)p->q_heads * p->dim;
        const float* q = see.mat<float>(a[3], F32, rows, cols, &ldq);
        float* out = see.mat<float>(a[5], F32, rows, cols, &ldo);
        const int32_t* lens = see.list<int32_t>(a[4], I32, p->seqs, true);
        if (!see.ok) Py_RETURN_NONE;
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = kq_attn_paged(kv, p->table, p->ldt, p->seqs, p->width, lens, p->max_len, (int)T, q, ldq, p->q_heads,
            p->scale, out, ldo, p->ws, p->ws_bytes, stream);
        Py_END_ALLOW_THREADS
        return PyLong_FromLong(rc);
    });
}

// pick(picked, ws, ws_bytes, stream, logits, history, length, prompt, repetition, frequency, presence, bias_ids,
// bias_values, allowed, out)
PyObject* pick(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 15) Py_RETURN_NONE;
        auto* picked = static_cast<int32_t*>(pointer(a[0]));
        void *ws = pointer(a[1]), *stream = pointer(a[3]);
        const size_t bytes = PyLong_AsSize_t(a[2]);
        if (PyErr_Occurred()) return nullptr;
        Look see;
        const int64_t B = see.rows(a[4]), V = see.cols(a[4]);
        int64_t ldx = 0, ldh = 0, ldb = 0, ldm = 0, ldy = 0, L = 0, nb = 0;
        const float* x = see.mat<float>(a[4], F32, B, V, &ldx);
        const int32_t *hist = nullptr, *ids = nullptr, *allowed = nullptr;
        const float* values = nullptr;
        float* y = nullptr;
        if (a[5] != Py_None) {
            L = see.cols(a[5]);
            hist = see.mat<int32_t>(a[5], I32, B, L, &ldh);
        }
        if (a[11] != Py_None) {
            int64_t ldv = 0;
            nb = see.cols(a[11]);
            ids = see.mat<int32_t>(a[11], I32, B, nb, &ldb);
            values = see.mat<float>(a[12], F32, B, nb, &ldv);
            if (see.ok && (see.cols(a[12]) != nb || see.rows(a[12]) != see.rows(a[11]) || ldv != ldb)) see.ok = false;
        }
        if (a[13] != Py_None) {
            const bool shared = B > 1 && see.rows(a[13]) == 1;
            allowed = see.mat<int32_t>(a[13], I32, shared ? 1 : B, (V + 31) / 32, &ldm);
            if (shared) ldm = 0;
        }
        if (a[14] != Py_None) y = see.mat<float>(a[14], F32, B, V, &ldy);
        const int32_t* length = see.list<int32_t>(a[6], I32, B, hist != nullptr);
        const int32_t* prompt = see.list<int32_t>(a[7], I32, B, false);
        const float* rep = see.list<float>(a[8], F32, B, false);
        const float* freq = see.list<float>(a[9], F32, B, false);
        const float* pres = see.list<float>(a[10], F32, B, false);
        if (!see.ok || !sizes_fit(B, V) || !sizes_fit(L, nb)) Py_RETURN_NONE;
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = kq_logits_penalize(x, ldx, (int)B, (int)V, hist, ldh, (int)L, length, prompt, rep, freq, pres, ids,
            values, ldb, (int)nb, reinterpret_cast<const uint32_t*>(allowed), ldm, y, ldy, ws,
            bytes, picked, stream);
        Py_END_ALLOW_THREADS
        return PyLong_FromLong(rc);
    });
}

PyMethodDef methods[] = {{"plan", plan, METH_VARARGS, nullptr},
                         {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(append)), METH_FASTCALL, nullptr},
                         {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attend)), METH_FASTCALL, nullptr},
                         {"pick", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(pick)), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", "Token-loop calls of libkq.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&module); }
