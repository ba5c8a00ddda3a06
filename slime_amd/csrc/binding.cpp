// binding.cpp — the attention calls of include/slime_ca.h as a CPython module over torch tensors
// (slime_amd/_binding.so), for slime_amd/attention.py.
//
// Small calls are bound by the host: an attend through ctypes, with its checks and structures in
// Python, takes 16.2 us, from here 5.3, of which the launch is about half. Each function checks its
// arguments, allocates outputs and workspace on the current stream, and makes the one C call.
// It returns the outputs; None if an argument is not as it must be (the caller then says which);
// or the status of a C call that failed.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>

#include "overlap.hpp"
#include "slime_ca.h"

namespace {

using at::Tensor;

// Arguments in turn; ok falls, and stays so, at the first that is not as it must be.
struct Args {
    PyObject* const* at;
    Py_ssize_t left;
    bool ok = true;
    int dtype = -1;
    c10::Device device{c10::DeviceType::CPU};

    PyObject* next() {
        if (left < 1) {
            ok = false;
            return Py_None;
        }
        --left;
        return *at++;
    }
    const Tensor* tensor() {
        PyObject* o = next();
        if (!THPVariable_Check(o)) {
            ok = false;
            return nullptr;
        }
        return &THPVariable_Unpack(o);
    }
    const Tensor* tensor_or_none(bool* none) {
        *none = left > 0 && *at == Py_None;
        if (*none) {
            next();
            return nullptr;
        }
        return tensor();
    }
    // [B, N, heads, D] of float32 or bfloat16 on the GPU, dense along D; of the first one's type and
    // device.
    const Tensor* heads(slime_ca_heads* h) {
        const Tensor* t = tensor();
        if (!t || t->dim() != 4 || !t->is_cuda() || t->stride(3) != 1) {
            ok = false;
            return nullptr;
        }
        const auto type = t->scalar_type();
        const int code = type == at::kFloat ? SLIME_F32 : type == at::kBFloat16 ? SLIME_BF16 : -1;
        if (dtype < 0) {
            dtype = code;
            device = t->device();
        }
        ok = ok && code >= 0 && code == dtype && t->device() == device;
        *h = slime_ca_heads{t->data_ptr(), t->stride(0), t->stride(1), t->stride(2)};
        return t;
    }
    // As heads(), for an output: no memory twice.
    const Tensor* output(slime_ca_heads* h) {
        const Tensor* t = heads(h);
        for (int d = 0; t && d < 3; ++d) ok = ok && (t->size(d) < 2 || t->stride(d) != 0);
        return t;
    }
    // n contiguous values.
    void* vector(at::ScalarType type, int64_t n, const Tensor** found) {
        const Tensor* t = *found = tensor();
        ok = ok && t && t->dim() == 1 && t->size(0) == n && t->scalar_type() == type && t->device() == device &&
             t->is_contiguous();
        return ok ? t->data_ptr() : nullptr;
    }
    double number() {
        const double v = PyFloat_AsDouble(next());
        if (v == -1.0 && PyErr_Occurred()) {
            PyErr_Clear();
            ok = false;
        }
        return v;
    }
    // 0 or 1: which of the two words.
    int either(const char* a, const char* b) {
        PyObject* o = next();
        if (!PyUnicode_Check(o)) return ok = false;
        if (PyUnicode_CompareWithASCIIString(o, a) == 0) return 0;
        ok = ok && PyUnicode_CompareWithASCIIString(o, b) == 0;
        return 1;
    }
    bool truth() {
        const int v = PyObject_IsTrue(next());
        if (v < 0) {
            PyErr_Clear();
            ok = false;
        }
        return v > 0;
    }
};

bool alike(const Tensor* a, const Tensor* b) { return a && b && a->sizes() == b->sizes(); }
bool fits(const Tensor& t) {
    for (int d = 0; d < 4; ++d)
        if (t.size(d) > INT_MAX) return false;
    return true;
}

slime::Region region_of(const Tensor& t) {
    const long long e = (long long)t.element_size();
    slime::Region r{(long long)(intptr_t)t.data_ptr(), e, (int)t.dim(), {}, {}};
    for (int d = 0; d < r.dims; ++d) {
        r.size[d] = t.size(d);
        r.stride[d] = t.stride(d) * e;
    }
    return r;
}
// An output apart from an input, or (may_be) the input itself, place by place: each element is read
// by the workgroup that writes it, and before.
bool apart(const Tensor& out, const Tensor& in, bool may_be) {
    if (may_be && out.data_ptr() == in.data_ptr() && out.sizes() == in.sizes()) {
        bool same = true;
        for (int d = 0; d < out.dim(); ++d) same = same && (out.size(d) < 2 || out.stride(d) == in.stride(d));
        if (same) return true;
    }
    return !slime::Overlap::of(region_of(out), region_of(in));
}

Tensor empty_as(const Tensor& t) { return at::empty(t.sizes(), t.options()); }
slime_ca_heads heads_of(const Tensor& t) {
    return slime_ca_heads{t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}
void* current_stream(const c10::Device& d) { return (void*)c10::hip::getCurrentHIPStream(d.index()).stream(); }

template <typename... T>
PyObject* results(const T&... t) {
    PyObject* tuple = PyTuple_New(sizeof...(T));
    if (!tuple) return nullptr;
    Py_ssize_t i = 0;
    bool ok = true;
    ((ok = ok && [&] {
         PyObject* o = THPVariable_Wrap(t);
         if (o) PyTuple_SET_ITEM(tuple, i++, o);
         return o != nullptr;
     }()),
     ...);
    if (ok) return tuple;
    Py_DECREF(tuple);
    return nullptr;
}

// q, k, v, scale, causal, window, align, lengths, alive
struct Attend {
    slime_ca_attend_config c{};
    slime_ca_heads hq, hk, hv;
    const Tensor *q, *k, *v, *lengths = nullptr, *alive = nullptr;
    explicit Attend(Args& a) {
        q = a.heads(&hq);
        k = a.heads(&hk);
        v = a.heads(&hv);
        a.ok = a.ok && alike(k, v) && fits(*q) && fits(*k) && q->size(0) == k->size(0) && q->size(3) == k->size(3);
        const bool plain = a.left > 0 && *a.at == Py_None;
        const double scale = plain ? (a.next(), 0.0) : a.number();
        c.causal = a.truth();
        PyObject* w = PyNumber_Index(a.next());
        int over = 0;
        const long long window = w ? PyLong_AsLongLongAndOverflow(w, &over) : -1;
        if (!w) PyErr_Clear();
        Py_XDECREF(w);
        c.window = over > 0 || window > INT_MAX ? INT_MAX : (int)window;
        a.ok = a.ok && over >= 0 && window >= (over > 0 ? -1 : 0);
        c.align = a.either("end", "start");
        bool none;
        const Tensor* n = a.tensor_or_none(&none);
        if (!a.ok) return;
        c.B = (int)q->size(0);
        c.Nq = (int)q->size(1);
        c.Nk = (int)k->size(1);
        c.Hq = (int)q->size(2);
        c.Hkv = (int)k->size(2);
        c.D = (int)q->size(3);
        c.dtype = a.dtype;
        c.scale = plain ? (float)(1.0 / std::sqrt((double)c.D)) : (float)scale;
        if (!none) {
            a.ok = n->dim() == 1 && n->size(0) == c.B && n->scalar_type() == at::kInt && n->device() == a.device &&
                   n->is_contiguous();
            if (a.ok) c.lengths = static_cast<const int*>((lengths = n)->data_ptr());
        }
        const Tensor* m = a.tensor_or_none(&none);
        if (!none && a.ok) {
            a.ok = m->dim() == 2 && m->size(0) == c.B && m->size(1) == c.Nk &&
                   (m->scalar_type() == at::kBool || m->scalar_type() == at::kByte) && m->device() == a.device &&
                   (c.Nk < 2 || m->stride(1) == 1);
            if (a.ok) {
                c.alive = static_cast<const unsigned char*>((alive = m)->data_ptr());
                c.alive_batch = m->stride(0);
            }
        }
    }
    bool takes(const Tensor& out) const {
        return alike(&out, q) && apart(out, *q, true) && apart(out, *k, false) && apart(out, *v, false) &&
               (!lengths || apart(out, *lengths, false)) && (!alive || apart(out, *alive, false));
    }
};

PyObject* attend(PyObject*, PyObject* const* at, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a{at, n};
    Attend x(a);
    bool none = true;
    slime_ca_heads ho;
    none = a.left > 0 && *a.at == Py_None;
    const Tensor* given = none ? (a.next(), nullptr) : a.output(&ho);
    if (!a.ok || (given && !x.takes(*given))) Py_RETURN_NONE;
    const c10::hip::HIPGuard guard(a.device.index());
    size_t bytes = 0;
    if (int rc = slime_ca_attend_workspace(&x.c, 0, &bytes)) return PyLong_FromLong(rc);
    const Tensor out = given ? *given : empty_as(*x.q);
    const auto f32 = x.q->options().dtype(at::kFloat);
    const Tensor lse = at::empty({x.c.B, x.c.Hq, x.c.Nq}, f32);
    const Tensor ws = bytes ? at::empty({(int64_t)(bytes / 4)}, f32) : Tensor();
    ho = heads_of(out);
    const int rc = slime_ca_attend(&x.c, &x.hq, &x.hk, &x.hv, &ho, static_cast<float*>(lse.data_ptr()),
                                   bytes ? ws.data_ptr() : nullptr, bytes, current_stream(a.device));
    return rc ? PyLong_FromLong(rc) : results(out, lse);
    END_HANDLE_TH_ERRORS
}

PyObject* attend_backward(PyObject*, PyObject* const* at, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a{at, n};
    Attend x(a);
    slime_ca_heads hg, ho;
    const Tensor *g = a.heads(&hg), *o = a.heads(&ho), *lse = a.tensor();
    if (!a.ok || !alike(g, x.q) || !alike(o, x.q) || lse->dim() != 3 || lse->size(0) != x.c.B ||
        lse->size(1) != x.c.Hq || lse->size(2) != x.c.Nq || lse->scalar_type() != at::kFloat ||
        lse->device() != a.device || !lse->is_contiguous())
        Py_RETURN_NONE;
    const c10::hip::HIPGuard guard(a.device.index());
    size_t bytes = 0;
    if (int rc = slime_ca_attend_workspace(&x.c, 1, &bytes)) return PyLong_FromLong(rc);
    const Tensor dq = empty_as(*x.q), dk = empty_as(*x.k), dv = empty_as(*x.v);
    const Tensor ws = bytes ? at::empty({(int64_t)(bytes / 4)}, x.q->options().dtype(at::kFloat)) : Tensor();
    const slime_ca_heads hdq = heads_of(dq), hdk = heads_of(dk), hdv = heads_of(dv);
    const int rc = slime_ca_attend_backward(&x.c, &hg, &x.hq, &x.hk, &x.hv, &ho,
                                            static_cast<const float*>(lse->data_ptr()), &hdq, &hdk, &hdv,
                                            bytes ? ws.data_ptr() : nullptr, bytes, current_stream(a.device));
    return rc ? PyLong_FromLong(rc) : results(dq, dk, dv);
    END_HANDLE_TH_ERRORS
}

// q, k, wq, wk, positions, freqs, eps, pairs
struct Norm {
    slime_ca_norm_config c{};
    slime_ca_heads hq, hk;
    const Tensor *q, *k, *small[4];  // the gains, positions and frequencies
    const float *wq = nullptr, *wk = nullptr;
    explicit Norm(Args& a) {
        q = a.heads(&hq);
        k = a.heads(&hk);
        a.ok = a.ok && fits(*q) && fits(*k) && q->size(0) == k->size(0) && q->size(1) == k->size(1) &&
               q->size(3) == k->size(3);
        if (!a.ok) return;
        c.B = (int)q->size(0);
        c.N = (int)q->size(1);
        c.Hq = (int)q->size(2);
        c.Hkv = (int)k->size(2);
        c.D = (int)q->size(3);
        c.dtype = a.dtype;
        wq = static_cast<const float*>(a.vector(at::kFloat, c.D, &small[0]));
        wk = static_cast<const float*>(a.vector(at::kFloat, c.D, &small[1]));
        const Tensor* p = small[2] = a.tensor();
        a.ok = a.ok && p && p->dim() == 3 && p->size(0) == c.B && p->size(1) == c.N &&
               (p->size(2) == 1 || (p->size(2) == 2 && p->stride(2) == 1)) && p->scalar_type() == at::kInt &&
               p->device() == a.device;
        if (!a.ok) return;
        c.axes = (int)p->size(2);
        c.positions = static_cast<const int*>(p->data_ptr());
        c.pos_batch = p->stride(0);
        c.pos_row = p->stride(1);
        c.freqs = static_cast<const double*>(a.vector(at::kDouble, c.D / 2, &small[3]));
        c.eps = (float)a.number();
        c.adjacent = a.either("halves", "adjacent");
    }
    bool takes(const Tensor& oq, const Tensor& ok) const {
        bool fine = apart(oq, *q, true) && apart(oq, *k, false) && apart(ok, *k, true) && apart(ok, *q, false) &&
                    apart(oq, ok, false);
        for (const Tensor* t : small) fine = fine && apart(oq, *t, false) && apart(ok, *t, false);
        return fine;
    }
};

PyObject* norm(PyObject*, PyObject* const* at, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a{at, n};
    Norm x(a);
    slime_ca_heads hoq, hok;
    const bool none = a.left == 2 && a.at[0] == Py_None && a.at[1] == Py_None;
    const Tensor *gq = nullptr, *gk = nullptr;
    if (!none) {
        gq = a.output(&hoq);
        gk = a.output(&hok);
        a.ok = a.ok && alike(gq, x.q) && alike(gk, x.k) && x.takes(*gq, *gk);
    }
    if (!a.ok) Py_RETURN_NONE;
    const c10::hip::HIPGuard guard(a.device.index());
    const Tensor oq = gq ? *gq : empty_as(*x.q), ok = gk ? *gk : empty_as(*x.k);
    hoq = heads_of(oq);
    hok = heads_of(ok);
    const int rc = slime_ca_qk_norm_rotate(&x.c, &x.hq, &x.hk, x.wq, x.wk, &hoq, &hok, current_stream(a.device));
    return rc ? PyLong_FromLong(rc) : results(oq, ok);
    END_HANDLE_TH_ERRORS
}

PyObject* norm_backward(PyObject*, PyObject* const* at, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a{at, n};
    Norm x(a);
    slime_ca_heads hgq, hgk;
    const Tensor *gq = a.ok ? a.heads(&hgq) : nullptr, *gk = a.ok ? a.heads(&hgk) : nullptr;
    if (!a.ok || !alike(gq, x.q) || !alike(gk, x.k)) Py_RETURN_NONE;
    const c10::hip::HIPGuard guard(a.device.index());
    size_t bytes = 0;
    if (int rc = slime_ca_qk_norm_rotate_workspace(&x.c, &bytes)) return PyLong_FromLong(rc);
    const Tensor dq = empty_as(*x.q), dk = empty_as(*x.k);
    const auto f32 = x.q->options().dtype(at::kFloat);
    const Tensor dwq = at::empty({x.c.D}, f32), dwk = at::empty({x.c.D}, f32);
    const Tensor ws = bytes ? at::empty({(int64_t)(bytes / 4)}, f32) : Tensor();
    const slime_ca_heads hdq = heads_of(dq), hdk = heads_of(dk);
    const int rc = slime_ca_qk_norm_rotate_backward(
        &x.c, &hgq, &hgk, &x.hq, &x.hk, x.wq, x.wk, &hdq, &hdk, static_cast<float*>(dwq.data_ptr()),
        static_cast<float*>(dwk.data_ptr()), bytes ? ws.data_ptr() : nullptr, bytes, current_stream(a.device));
    return rc ? PyLong_FromLong(rc) : results(dq, dk, dwq, dwk);
    END_HANDLE_TH_ERRORS
}

// (output, input, whether it may be the input itself) -> whether they share memory otherwise.
PyObject* overlaps(PyObject*, PyObject* const* at, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Args a{at, n};
    const Tensor *out = a.tensor(), *in = a.tensor();
    const bool may_be = a.truth();
    if (!a.ok || out->dim() > slime::Region::kDims || in->dim() > slime::Region::kDims) Py_RETURN_NONE;
    return PyBool_FromLong(!apart(*out, *in, may_be));
    END_HANDLE_TH_ERRORS
}

#define SLIME_FN(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {SLIME_FN(attend), SLIME_FN(attend_backward), SLIME_FN(norm), SLIME_FN(norm_backward),
                         SLIME_FN(overlaps), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", "Attention calls over torch tensors.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", SLIME_TORCH) < 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
