// The calls a decode loop makes, as a CPython extension over the C ABI: arguments go from Python objects straight to
// the entry points of krk_cuda.h. A small matrix takes 5 us on the device; through ctypes a call cost 9-14 us of
// interpreter time (argument objects, a Python-level current_stream(), the foreign-function layer), so a token of
// eager calls ran at the host's pace. Nothing is computed or kept here: kraken_b200/capi.py is the interface, and an error code
// of the library becomes the exception capi registers.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <cmath>
#include <optional>

#include "krk_cuda.h"

namespace {

PyObject *g_raise = nullptr;     // capi's (rc, where) -> raises
PyObject *g_address = nullptr;   // capi's ctypes pointer -> int

PyObject *fail(int rc, const char *where) {
    PyObject *r = PyObject_CallFunction(g_raise, "is", rc, where);
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "%s failed with %d", where, rc);
    return nullptr;
}

// One argument list; a conversion that fails leaves a Python error set and `ok` false.
struct Args {
    PyObject *const *a;
    bool ok = true;
    int64_t i(int k) {
        const long long v = PyLong_AsLongLong(a[k]);
        if (v == -1 && PyErr_Occurred()) ok = false;
        return v;
    }
    // An address: an integer, None, or whatever ctypes takes for a void pointer.
    uintptr_t addr(int k) {
        if (a[k] == Py_None) return 0;
        PyObject *o = PyLong_Check(a[k]) ? nullptr : PyObject_CallOneArg(g_address, a[k]);
        if (!o && !PyLong_Check(a[k])) {
            ok = false;
            return 0;
        }
        const uintptr_t v = (uintptr_t)PyLong_AsUnsignedLongLongMask(o ? o : a[k]);
        Py_XDECREF(o);
        if (PyErr_Occurred()) ok = false;
        return v;
    }
    void *backend(int k) {
        if (!PyLong_Check(a[k])) {
            if (ok) PyErr_SetString(PyExc_TypeError, "the backend is closed");
            ok = false;
            return nullptr;
        }
        return (void *)addr(k);
    }
    float f(int k) {
        const double v = PyFloat_AsDouble(a[k]);
        if (v == -1.0 && PyErr_Occurred()) ok = false;
        return (float)v;
    }
    bool b(int k) {
        const int v = PyObject_IsTrue(a[k]);
        if (v < 0) ok = false;
        return v > 0;
    }
    const at::Tensor *tensor(PyObject *o) {
        if (!THPVariable_Check(o)) {
            if (ok) PyErr_Format(PyExc_TypeError, "expected a torch tensor, got %s", Py_TYPE(o)->tp_name);
            ok = false;
            return nullptr;
        }
        return &THPVariable_Unpack(o);
    }
    const at::Tensor *t(int k) { return tensor(a[k]); }
    static void *ptr(const at::Tensor *x) { return x ? const_cast<void *>(x->const_data_ptr()) : nullptr; }
    void *p(int k) { return ptr(t(k)); }
    const at::Tensor *t_or_none(int k) { return a[k] == Py_None ? nullptr : t(k); }
    void *stream(int k) {
        if (a[k] == Py_None) return c10::cuda::getCurrentCUDAStream().stream();
        PyObject *s = PyObject_GetAttrString(a[k], "cuda_stream");
        if (!s) {
            ok = false;
            return nullptr;
        }
        void *v = PyLong_AsVoidPtr(s);
        Py_DECREF(s);
        if (!v && PyErr_Occurred()) ok = false;
        return v;
    }
};

at::Tensor empty_like_device(const at::Tensor &like, at::IntArrayRef sizes, at::ScalarType type) {
    return at::empty(sizes, like.options().dtype(type).requires_grad(false));
}

#define KRK_NARGS(count, name)                                                                                    \
    if (n != (count)) {                                                                                           \
        PyErr_Format(PyExc_TypeError, name " takes %d arguments, got %zd", (count), n);                           \
        return nullptr;                                                                                           \
    }
#define KRK_TRY try {
#define KRK_CATCH                                                                                                 \
    }                                                                                                             \
    catch (const std::exception &e) {                                                                             \
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());                                     \
        return nullptr;                                                                                           \
    }

PyObject *set_raise(PyObject *, PyObject *f) {
    Py_INCREF(f);
    Py_XSETREF(g_raise, f);
    Py_RETURN_NONE;
}
PyObject *set_address(PyObject *, PyObject *f) {
    Py_INCREF(f);
    Py_XSETREF(g_address, f);
    Py_RETURN_NONE;
}

PyObject *gemv(PyObject *, PyObject *const *a, Py_ssize_t n) {   // x, w, wt, n_out, n_in, out, accumulate, stream
    KRK_NARGS(8, "gemv")
    KRK_TRY
    Args g{a};
    const at::Tensor *x = g.t(0);
    const void *w = g.p(1);
    const int wt = (int)g.i(2);
    const int64_t n_out = g.i(3), n_in = g.i(4);
    const bool acc = g.b(6);
    const at::Tensor *out = g.t_or_none(5);
    void *st = g.stream(7);
    if (!g.ok) return nullptr;
    const int64_t rows = x->dim() == 1 ? 1 : x->size(0);
    at::Tensor made;
    if (!out) {
        if (acc) {
            PyErr_SetString(PyExc_ValueError, "accumulate needs an existing output");
            return nullptr;
        }
        made = empty_like_device(*x, {rows, n_out}, at::kFloat);
        out = &made;
    }
    void *y = Args::ptr(out), *xp = Args::ptr(x);
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = krk_cuda_gemv(y, xp, w, wt, n_out, n_in, rows, acc, st);
    Py_END_ALLOW_THREADS
    if (rc != 0) return fail(rc, "gemv");
    if (made.defined()) return THPVariable_Wrap(made);
    Py_INCREF(a[5]);
    return a[5];
    KRK_CATCH
}

// A list or tuple argument of up to KRK_CUDA_MAX_GROUP items, as a borrowed fast sequence.
struct Seq {
    PyObject *s;
    Py_ssize_t n = 0;
    explicit Seq(PyObject *o) : s(PySequence_Fast(o, "expected a sequence")) {
        if (s) n = PySequence_Fast_GET_SIZE(s);
    }
    ~Seq() { Py_XDECREF(s); }
    PyObject *operator[](Py_ssize_t i) const { return PySequence_Fast_GET_ITEM(s, i); }
};

PyObject *gemv_group(PyObject *, PyObject *const *a, Py_ssize_t n) {   // xs, ws, wts, n_outs, n_in, outs, fuse, stream
    KRK_NARGS(8, "gemv_group")
    KRK_TRY
    Args g{a};
    Seq xs(a[0]), ws(a[1]), wts(a[2]), nos(a[3]);
    if (!xs.s || !ws.s || !wts.s || !nos.s) return nullptr;
    const Py_ssize_t m = ws.n;
    if (m > KRK_CUDA_MAX_GROUP) return fail(KRK_CUDA_EARG, "gemv_group");
    if (xs.n != m || wts.n != m || nos.n != m) {
        PyErr_SetString(PyExc_ValueError, "gemv_group: argument lists of unequal length");
        return nullptr;
    }
    void *y[KRK_CUDA_MAX_GROUP];
    const void *x[KRK_CUDA_MAX_GROUP], *w[KRK_CUDA_MAX_GROUP];
    int wt[KRK_CUDA_MAX_GROUP];
    int64_t n_out[KRK_CUDA_MAX_GROUP];
    PyObject *outs = a[5];
    if (outs == Py_None) {
        outs = PyList_New(m);
        if (!outs) return nullptr;
    } else {
        Py_INCREF(outs);
    }
    for (Py_ssize_t i = 0; i < m && g.ok; i++) {
        const at::Tensor *wi = g.tensor(ws[i]);
        x[i] = Args::ptr(g.tensor(xs[i]));
        w[i] = Args::ptr(wi);
        Args item{PySequence_Fast_ITEMS(wts.s)}, size{PySequence_Fast_ITEMS(nos.s)};
        wt[i] = (int)item.i((int)i);
        n_out[i] = size.i((int)i);
        g.ok = g.ok && item.ok && size.ok;
        if (g.ok && a[5] == Py_None) PyList_SET_ITEM(outs, i, THPVariable_Wrap(empty_like_device(*wi, {n_out[i]}, at::kFloat)));
    }
    const int64_t n_in = g.i(4);
    const bool fuse = g.b(6);
    void *st = g.stream(7);
    if (g.ok) {
        Seq ys(outs);
        if (!ys.s || ys.n != m) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "gemv_group: as many outputs as matrices are needed");
            g.ok = false;
        }
        for (Py_ssize_t i = 0; i < m && g.ok; i++) y[i] = Args::ptr(g.tensor(ys[i]));
    }
    if (!g.ok) {
        Py_DECREF(outs);
        return nullptr;
    }
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = krk_cuda_gemv_group(y, x, w, wt, n_out, n_in, (int)m, fuse, st);
    Py_END_ALLOW_THREADS
    if (rc != 0) {
        Py_DECREF(outs);
        return fail(rc, "gemv_group");
    }
    return outs;
    KRK_CATCH
}

PyObject *gemm(PyObject *, PyObject *const *a, Py_ssize_t n) {   // x, w, wt, n_out, n_in, out, workspace, stream
    KRK_NARGS(8, "gemm")
    KRK_TRY
    Args g{a};
    const at::Tensor *x = g.t(0);
    const void *w = g.p(1);
    const int wt = (int)g.i(2);
    const int64_t n_out = g.i(3), n_in = g.i(4);
    const at::Tensor *out = g.t_or_none(5), *ws = g.t_or_none(6);
    void *st = g.stream(7);
    if (!g.ok) return nullptr;
    const int64_t rows = x->size(0);
    const int xt = x->scalar_type() == at::kHalf ? KRK_CUDA_X_F16 : KRK_CUDA_X_F32;
    at::Tensor made_ws, made;
    if (!ws) {
        const size_t need = krk_cuda_gemm_workspace_bytes(xt, n_out, n_in, rows);
        if (need) {
            made_ws = empty_like_device(*x, {(int64_t)need}, at::kByte);
            ws = &made_ws;
        }
    }
    if (!out) {
        made = empty_like_device(*x, {rows, n_out}, at::kFloat);
        out = &made;
    }
    void *y = Args::ptr(out), *xp = Args::ptr(x), *wp = Args::ptr(ws);
    const size_t ws_bytes = ws ? (size_t)ws->numel() : 0;
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = krk_cuda_gemm(y, xp, xt, w, wt, n_out, n_in, rows, wp, ws_bytes, st);
    Py_END_ALLOW_THREADS
    if (rc != 0) return fail(rc, "gemm");
    if (made.defined()) return THPVariable_Wrap(made);
    Py_INCREF(a[5]);
    return a[5];
    KRK_CATCH
}

PyObject *silu_mul(PyObject *, PyObject *const *a, Py_ssize_t n) {   // gate, up, out, stream
    KRK_NARGS(4, "silu_mul")
    KRK_TRY
    Args g{a};
    const at::Tensor *gate = g.t(0), *out = g.t_or_none(2);
    const void *up = g.p(1);
    void *st = g.stream(3);
    if (!g.ok) return nullptr;
    at::Tensor made;
    if (!out) {
        made = at::empty_like(*gate, gate->options().requires_grad(false));   // with its strides: the kernel goes through the memory as it lies
        out = &made;
    }
    void *y = Args::ptr(out), *gp = Args::ptr(gate);
    const int64_t count = gate->numel();
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = krk_cuda_silu_mul(y, gp, up, count, st);
    Py_END_ALLOW_THREADS
    if (rc != 0) return fail(rc, "silu_mul");
    if (made.defined()) return THPVariable_Wrap(made);
    Py_INCREF(a[2]);
    return a[2];
    KRK_CATCH
}

PyObject *embed(PyObject *, PyObject *const *a, Py_ssize_t n) {   // table, wt, n_vocab, n_embd, tokens, out, stream
    KRK_NARGS(7, "embed")
    KRK_TRY
    Args g{a};
    const at::Tensor *table = g.t(0), *tokens = g.t(4), *out = g.t_or_none(5);
    const int wt = (int)g.i(1);
    const int64_t n_vocab = g.i(2), n_embd = g.i(3);
    void *st = g.stream(6);
    if (!g.ok) return nullptr;
    at::Tensor made;
    if (!out) {
        made = empty_like_device(*table, {tokens->numel(), n_embd}, at::kFloat);
        out = &made;
    }
    void *y = Args::ptr(out), *tp = Args::ptr(table), *ip = Args::ptr(tokens);
    const int64_t n_tok = tokens->numel();
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = krk_cuda_embed(y, tp, wt, n_vocab, n_embd, ip, n_tok, st);
    Py_END_ALLOW_THREADS
    if (rc != 0) return fail(rc, "embed");
    if (made.defined()) return THPVariable_Wrap(made);
    Py_INCREF(a[5]);
    return a[5];
    KRK_CATCH
}

// logits, k, pen_mask, rep_pen, softcap, temp, want_mass, workspace, stream -> (ids, vals, mass or None)
PyObject *logits_topk(PyObject *, PyObject *const *a, Py_ssize_t n) {
    KRK_NARGS(9, "logits_topk")
    KRK_TRY
    Args g{a};
    const at::Tensor *logits = g.t(0), *pen = g.t_or_none(2), *ws = g.t_or_none(7);
    const int64_t k = g.i(1);
    const float rep_pen = g.f(3), softcap = g.f(4), temp = g.f(5);
    const bool want_mass = g.b(6);
    void *st = g.stream(8);
    if (!g.ok) return nullptr;
    at::Tensor made_ws, mass;
    if (!ws) {
        const size_t need = krk_cuda_logits_topk_workspace_bytes(logits->numel(), (int)k);
        made_ws = empty_like_device(*logits, {(int64_t)(need > 16 ? need : 16)}, at::kByte);
        ws = &made_ws;
    }
    at::Tensor ids = empty_like_device(*logits, {k}, at::kInt), vals = empty_like_device(*logits, {k}, at::kFloat);
    if (want_mass) mass = empty_like_device(*logits, {1}, at::kFloat);
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = krk_cuda_logits_topk(Args::ptr(logits), logits->numel(), (int)k, Args::ptr(pen), rep_pen, softcap, temp, Args::ptr(&ids),
                                                     Args::ptr(&vals), want_mass ? Args::ptr(&mass) : nullptr, Args::ptr(ws), (size_t)ws->numel(), st);
    Py_END_ALLOW_THREADS
    if (rc != 0) return fail(rc, "logits_topk");
    PyObject *r = PyTuple_New(3);
    if (!r) return nullptr;
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(ids));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(vals));
    if (want_mass) {
        PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(mass));
    } else {
        Py_INCREF(Py_None);
        PyTuple_SET_ITEM(r, 2, Py_None);
    }
    return r;
    KRK_CATCH
}

// The krk_cuda_expert_bank behind capi's ctypes structure (which offers its memory as a buffer).
struct Bank {
    Py_buffer view{};
    bool ok;
    explicit Bank(PyObject *o) : ok(PyObject_GetBuffer(o, &view, PyBUF_SIMPLE) == 0) {
        if (ok && view.len < (Py_ssize_t)sizeof(krk_cuda_expert_bank)) {
            PyErr_SetString(PyExc_TypeError, "expected an ExpertBank");
            PyBuffer_Release(&view);
            ok = false;
        }
    }
    ~Bank() {
        if (ok) PyBuffer_Release(&view);
    }
    const krk_cuda_expert_bank *get() const { return static_cast<const krk_cuda_expert_bank *>(view.buf); }
};

PyObject *moe_ffn(PyObject *, PyObject *const *a, Py_ssize_t n) {   // x, ids, wts, bank, out, workspace, stream
    KRK_NARGS(7, "moe_ffn")
    KRK_TRY
    Args g{a};
    Bank bank(a[3]);
    if (!bank.ok) return nullptr;
    const at::Tensor *x = g.t(0), *ids = g.t(1), *wts = g.t(2), *out = g.t_or_none(4), *ws = g.t_or_none(5);
    void *st = g.stream(6);
    if (!g.ok) return nullptr;
    const int64_t n_tok = ids->size(0);
    const int k = (int)ids->size(1);
    at::Tensor made, made_ws;
    if (!ws) {
        const size_t need = krk_cuda_moe_workspace_bytes(bank.get(), k, n_tok);
        made_ws = empty_like_device(*x, {(int64_t)(need > 16 ? need : 16)}, at::kByte);
        ws = &made_ws;
    }
    if (!out) {
        made = empty_like_device(*x, {n_tok, bank.get()->n_embd}, at::kFloat);
        out = &made;
    }
    void *y = Args::ptr(out), *wp = Args::ptr(ws);
    const size_t ws_bytes = (size_t)ws->numel();
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = krk_cuda_moe_ffn(y, Args::ptr(x), Args::ptr(ids), Args::ptr(wts), bank.get(), k, n_tok, wp, ws_bytes, st);
    Py_END_ALLOW_THREADS
    if (rc != 0) return fail(rc, "moe_ffn");
    if (made.defined()) return THPVariable_Wrap(made);
    Py_INCREF(a[4]);
    return a[4];
    KRK_CATCH
}

PyObject *moe_ffn_routed(PyObject *, PyObject *const *a, Py_ssize_t n) {   // x, logits, k, bank, out, workspace, stream -> (y, ids, wts)
    KRK_NARGS(7, "moe_ffn_routed")
    KRK_TRY
    Args g{a};
    Bank bank(a[3]);
    if (!bank.ok) return nullptr;
    const at::Tensor *x = g.t(0), *logits = g.t(1), *out = g.t_or_none(4), *ws = g.t_or_none(5);
    const int64_t k = g.i(2);
    void *st = g.stream(6);
    if (!g.ok) return nullptr;
    const int64_t n_tok = logits->size(0), n_expert = logits->size(1);
    at::Tensor ids = empty_like_device(*x, {n_tok, k}, at::kInt), wts = empty_like_device(*x, {n_tok, k}, at::kFloat), made, made_ws;
    if (!ws) {
        const size_t need = krk_cuda_moe_workspace_bytes(bank.get(), (int)k, n_tok);
        made_ws = empty_like_device(*x, {(int64_t)(need > 16 ? need : 16)}, at::kByte);
        ws = &made_ws;
    }
    if (!out) {
        made = empty_like_device(*x, {n_tok, bank.get()->n_embd}, at::kFloat);
        out = &made;
    }
    void *y = Args::ptr(out), *wp = Args::ptr(ws);
    const size_t ws_bytes = (size_t)ws->numel();
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = krk_cuda_moe_ffn_routed(y, Args::ptr(x), Args::ptr(logits), (int)n_expert, Args::ptr(&ids), Args::ptr(&wts),
                                                        bank.get(), (int)k, n_tok, wp, ws_bytes, st);
    Py_END_ALLOW_THREADS
    if (rc != 0) return fail(rc, "moe_ffn_routed");
    PyObject *r = PyTuple_New(3);
    if (!r) return nullptr;
    if (made.defined()) {
        PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(made));
    } else {
        Py_INCREF(a[4]);
        PyTuple_SET_ITEM(r, 0, a[4]);
    }
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(ids));
    PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(wts));
    return r;
    KRK_CATCH
}

// ---- the CudaBackend object: device and host addresses are plain integers -------------------------------------

PyObject *backend_upload(PyObject *, PyObject *const *a, Py_ssize_t n) {   // be, dst, host_src, bytes, off
    KRK_NARGS(5, "backend_upload")
    Args g{a};
    void *be = g.backend(0), *dst = (void *)g.addr(1);
    const void *src = (const void *)g.addr(2);
    const size_t bytes = (size_t)g.i(3), off = (size_t)g.i(4);
    if (!g.ok) return nullptr;
    Py_BEGIN_ALLOW_THREADS krk_cuda_backend_upload(be, dst, src, bytes, off);
    Py_END_ALLOW_THREADS Py_RETURN_NONE;
}
PyObject *backend_download(PyObject *, PyObject *const *a, Py_ssize_t n) {   // be, host_dst, src, bytes, off
    KRK_NARGS(5, "backend_download")
    Args g{a};
    void *be = g.backend(0), *dst = (void *)g.addr(1);
    const void *src = (const void *)g.addr(2);
    const size_t bytes = (size_t)g.i(3), off = (size_t)g.i(4);
    if (!g.ok) return nullptr;
    Py_BEGIN_ALLOW_THREADS krk_cuda_backend_download(be, dst, src, bytes, off);
    Py_END_ALLOW_THREADS Py_RETURN_NONE;
}
PyObject *backend_gemm(PyObject *, PyObject *const *a, Py_ssize_t n) {   // be, out, x, w, wt, n_out, n_in, rows
    KRK_NARGS(8, "backend_gemm")
    Args g{a};
    void *be = g.backend(0), *out = (void *)g.addr(1);
    const void *x = (const void *)g.addr(2), *w = (const void *)g.addr(3);
    const int wt = (int)g.i(4);
    const int64_t n_out = g.i(5), n_in = g.i(6), rows = g.i(7);
    if (!g.ok) return nullptr;
    Py_BEGIN_ALLOW_THREADS krk_cuda_backend_gemm(be, out, x, w, wt, n_out, n_in, rows);
    Py_END_ALLOW_THREADS Py_RETURN_NONE;
}
PyObject *backend_gemm_accumulate(PyObject *, PyObject *const *a, Py_ssize_t n) {   // be, dst, x, w, wt, n_out, n_in, rows
    KRK_NARGS(8, "backend_gemm_accumulate")
    Args g{a};
    void *be = g.backend(0), *dst = (void *)g.addr(1);
    const void *x = (const void *)g.addr(2), *w = (const void *)g.addr(3);
    const int wt = (int)g.i(4);
    const int64_t n_out = g.i(5), n_in = g.i(6), rows = g.i(7);
    if (!g.ok) return nullptr;
    int r;
    Py_BEGIN_ALLOW_THREADS r = krk_cuda_backend_gemm_accumulate(be, dst, x, w, wt, n_out, n_in, rows);
    Py_END_ALLOW_THREADS
    return PyBool_FromLong(r);
}
// be, outs, x, ws, wt, n_outs, n_in, rows, silu, wts or None, xs or None -> (ran in one launch, silu folded)
PyObject *backend_gemm_group(PyObject *, PyObject *const *a, Py_ssize_t n) {
    KRK_NARGS(11, "backend_gemm_group")
    KRK_TRY
    Args g{a};
    Seq outs(a[1]), ws(a[3]), nos(a[5]);
    if (!outs.s || !ws.s || !nos.s) return nullptr;
    const size_t m = (size_t)ws.n;
    PyObject *empty = PyTuple_New(0);
    Seq wts(a[9] == Py_None ? empty : a[9]), xs(a[10] == Py_None ? empty : a[10]);
    Py_DECREF(empty);
    if (!wts.s || !xs.s) return nullptr;
    if ((size_t)outs.n != m || (size_t)nos.n != m || (a[9] != Py_None && (size_t)wts.n != m) || (a[10] != Py_None && (size_t)xs.n != m)) {
        PyErr_SetString(PyExc_ValueError, "gemm_group: argument lists of unequal length");
        return nullptr;
    }
    std::vector<void *> y(m);
    std::vector<const void *> w(m), x(m);
    std::vector<int64_t> n_out(m);
    std::vector<int> wt(m);
    Args fo{PySequence_Fast_ITEMS(outs.s)}, fw{PySequence_Fast_ITEMS(ws.s)}, fn{PySequence_Fast_ITEMS(nos.s)}, ft{PySequence_Fast_ITEMS(wts.s)},
        fx{PySequence_Fast_ITEMS(xs.s)};
    for (size_t i = 0; i < m; i++) {
        y[i] = (void *)fo.addr((int)i);
        w[i] = (const void *)fw.addr((int)i);
        n_out[i] = fn.i((int)i);
        if (a[9] != Py_None) wt[i] = (int)ft.i((int)i);
        if (a[10] != Py_None) x[i] = (const void *)fx.addr((int)i);
    }
    void *be = g.backend(0);
    const void *x0 = (const void *)g.addr(2);
    const int wt0 = (int)g.i(4);
    const int64_t n_in = g.i(6), rows = g.i(7);
    const bool silu = g.b(8);
    if (!g.ok || !fo.ok || !fw.ok || !fn.ok || !ft.ok || !fx.ok) return nullptr;
    int fused = 0, ran;
    Py_BEGIN_ALLOW_THREADS ran = krk_cuda_backend_gemm_group_ex(be, y.data(), x0, w.data(), wt0, n_out.data(), n_in, (int)m, rows, silu, &fused,
                                                                a[9] != Py_None ? wt.data() : nullptr, a[10] != Py_None ? x.data() : nullptr);
    Py_END_ALLOW_THREADS
    return PyTuple_Pack(2, ran ? Py_True : Py_False, fused ? Py_True : Py_False);
    KRK_CATCH
}

// ---- query and key heads, the cache, attention, logits --------------------------------------------------------------
// These look at what they are given: types, shapes and strides become sizes of the C call, so a wrong one is an error here.

bool refuse(const char *what) {
    PyErr_SetString(PyExc_ValueError, what);
    return false;
}
// The device of the tensors, and the stream of the call, for as long as this lives; what is allocated meanwhile belongs to that stream.
struct Where {
    c10::cuda::CUDAGuard device;
    std::optional<c10::cuda::CUDAStreamGuard> other;
    void *stream;
    Where(const at::Tensor &t, bool given, void *st) : device(t.device()) {
        if (given) {
            other.emplace(c10::cuda::getStreamFromExternal((cudaStream_t)st, t.device().index()));
            stream = st;
        } else {
            stream = c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
        }
    }
};
bool on_device(const at::Tensor *t, const at::Tensor *first, const char *name) {
    if (t->is_cuda() && t->device() == first->device()) return true;
    PyErr_Format(PyExc_ValueError, "%s: not on the device of the first tensor, or not on a GPU", name);
    return false;
}
bool typed(const at::Tensor *t, const at::Tensor *first, at::ScalarType type, const char *name) {
    if (!on_device(t, first, name)) return false;
    if (t->scalar_type() == type) return true;
    PyErr_Format(PyExc_ValueError, "%s: expected %s", name, c10::toString(type));
    return false;
}
// A list of n elements one behind the other (n < 0: of any number).
bool listed(const at::Tensor *t, const at::Tensor *first, at::ScalarType type, int64_t n, const char *name) {
    if (!t) return true;
    if (!typed(t, first, type, name)) return false;
    if (t->dim() == 1 && (n < 0 || t->numel() == n) && t->is_contiguous()) return true;
    PyErr_Format(PyExc_ValueError, "%s: expected a contiguous list%s", name, n < 0 ? "" : " of as many elements as there are rows");
    return false;
}
// f32 [rows][heads][d], heads behind each other; the stride of the rows is free.
bool headed(const at::Tensor *t, const at::Tensor *first, int64_t rows, int64_t heads, int64_t d, const char *name) {
    if (!typed(t, first, at::kFloat, name)) return false;
    if (t->dim() == 3 && (rows < 0 || t->size(0) == rows) && (heads < 0 || t->size(1) == heads) && t->size(2) == d &&
        (t->numel() == 0 || ((d <= 1 || t->stride(2) == 1) && (t->size(1) <= 1 || t->stride(1) == d))))
        return true;
    PyErr_Format(PyExc_ValueError, "%s: expected [rows][heads][values] with the heads of a row behind each other", name);
    return false;
}
// [rows][n], the elements of a row behind each other.
bool tabled(const at::Tensor *t, const at::Tensor *first, at::ScalarType type, int64_t rows, const char *name) {
    if (!t) return true;
    if (!typed(t, first, type, name)) return false;
    if (t->dim() == 2 && (rows < 0 || t->size(0) == rows) && (t->numel() == 0 || t->size(1) <= 1 || t->stride(1) == 1)) return true;
    PyErr_Format(PyExc_ValueError, "%s: expected [rows][elements]", name);
    return false;
}
PyObject *given_or_made(PyObject *given, const at::Tensor &made) {
    if (given == Py_None) return THPVariable_Wrap(made);
    Py_INCREF(given);
    return given;
}
int64_t row_stride(const at::Tensor *t) { return t->size(0) > 1 ? t->stride(0) : t->dim() == 3 ? t->size(1) * t->size(2) : t->size(1); }

// q, k, pos, inv_freq, q_weight, k_weight, norm, eps, interleaved, q_out, k_out, stream -> (q_out, k_out)
PyObject *qk_norm_rope(PyObject *, PyObject *const *a, Py_ssize_t n) {
    KRK_NARGS(12, "qk_norm_rope")
    KRK_TRY
    Args g{a};
    const at::Tensor *q = g.t(0), *k = g.t_or_none(1), *pos = g.t_or_none(2), *freq = g.t_or_none(3), *wq = g.t_or_none(4), *wk = g.t_or_none(5), *qo = g.t_or_none(9),
                     *ko = g.t_or_none(10);
    krk_cuda_rope r = {};
    r.norm = g.b(6), r.eps = g.f(7), r.interleaved = g.b(8);
    void *st = a[11] == Py_None ? nullptr : g.stream(11);
    if (!g.ok) return nullptr;
    if (q->dim() != 3) return refuse("q: expected [rows][heads][values]"), nullptr;
    const int64_t rows = q->size(0), d = q->size(2);
    if (!headed(q, q, rows, -1, d, "q") || (k && !headed(k, q, rows, -1, d, "k")) || !listed(freq, q, at::kFloat, -1, "inv_freq") ||
        !listed(pos, q, at::kInt, rows, "pos") || !listed(wq, q, at::kFloat, d, "q_weight") || !listed(wk, q, at::kFloat, d, "k_weight"))
        return nullptr;
    Where where(*q, a[11] != Py_None, st);
    at::Tensor made_q, made_k;
    if (!qo) qo = &(made_q = empty_like_device(*q, {rows, q->size(1), d}, at::kFloat));
    else if (!headed(qo, q, rows, q->size(1), d, "q_out")) return nullptr;
    if (k && !ko) ko = &(made_k = empty_like_device(*q, {rows, k->size(1), d}, at::kFloat));
    else if (k && !headed(ko, q, rows, k->size(1), d, "k_out")) return nullptr;
    r.pos = pos ? Args::ptr(pos) : nullptr, r.inv_freq = freq ? Args::ptr(freq) : nullptr;
    r.q_weight = Args::ptr(wq), r.k_weight = Args::ptr(wk);
    r.n_tok = rows, r.n_heads = (int)q->size(1), r.n_kv_heads = k ? (int)k->size(1) : 0, r.head_dim = (int)d, r.rot_dim = freq ? (int)(2 * freq->numel()) : 0;
    r.q_stride = row_stride(q), r.q_out_stride = row_stride(qo);
    if (k) r.k_stride = row_stride(k), r.k_out_stride = row_stride(ko);
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = krk_cuda_qk_norm_rope(Args::ptr(qo), k ? Args::ptr(ko) : nullptr, Args::ptr(q), k ? Args::ptr(k) : nullptr, &r, where.stream);
    Py_END_ALLOW_THREADS
    if (rc != 0) return fail(rc, "qk_norm_rope");
    PyObject *y = given_or_made(a[9], made_q), *z = k ? given_or_made(a[10], made_k) : Py_NewRef(Py_None);
    PyObject *both = y && z ? PyTuple_Pack(2, y, z) : nullptr;
    Py_XDECREF(y);
    Py_XDECREF(z);
    return both;
    KRK_CATCH
}

PyObject *kv_append(PyObject *, PyObject *const *a, Py_ssize_t n) {   // cache, k, v, slots, stream
    KRK_NARGS(5, "kv_append")
    KRK_TRY
    Args g{a};
    const auto *c = (const krk_cuda_kv_cache *)g.addr(0);
    const at::Tensor *k = g.t(1), *v = g.t(2), *slots = g.t(3);
    void *st = a[4] == Py_None ? nullptr : g.stream(4);
    if (!g.ok) return nullptr;
    if (k->dim() != 3) return refuse("k: expected [rows][heads][values]"), nullptr;
    const int64_t rows = k->size(0);
    if (!headed(k, k, rows, c->n_kv_heads, c->head_dim, "k") || !headed(v, k, rows, c->n_kv_heads, c->head_dim, "v") || !listed(slots, k, at::kLong, rows, "slots")) return nullptr;
    Where where(*k, a[4] != Py_None, st);
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = krk_cuda_kv_append(c, Args::ptr(k), Args::ptr(v), row_stride(k), row_stride(v), Args::ptr(slots), rows, where.stream);
    Py_END_ALLOW_THREADS
    if (rc != 0) return fail(rc, "kv_append");
    Py_RETURN_NONE;
    KRK_CATCH
}

PyObject *kv_read(PyObject *, PyObject *const *a, Py_ssize_t n) {   // cache, slots, k_out, v_out, stream -> (k, v)
    KRK_NARGS(5, "kv_read")
    KRK_TRY
    Args g{a};
    const auto *c = (const krk_cuda_kv_cache *)g.addr(0);
    const at::Tensor *slots = g.t(1), *k = g.t_or_none(2), *v = g.t_or_none(3);
    void *st = a[4] == Py_None ? nullptr : g.stream(4);
    if (!g.ok || !listed(slots, slots, at::kLong, -1, "slots")) return nullptr;
    const int64_t rows = slots->numel(), h = c->n_kv_heads, d = c->head_dim;
    Where where(*slots, a[4] != Py_None, st);
    at::Tensor made_k, made_v;
    if (!k) k = &(made_k = empty_like_device(*slots, {rows, h, d}, at::kFloat));
    if (!v) v = &(made_v = empty_like_device(*slots, {rows, h, d}, at::kFloat));
    if (!headed(k, slots, rows, h, d, "k") || !headed(v, slots, rows, h, d, "v")) return nullptr;
    if (!k->is_contiguous() || !v->is_contiguous()) return refuse("kv_read writes contiguous tensors"), nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = krk_cuda_kv_read(c, Args::ptr(k), Args::ptr(v), Args::ptr(slots), rows, where.stream);
    Py_END_ALLOW_THREADS
    if (rc != 0) return fail(rc, "kv_read");
    PyObject *y = given_or_made(a[2], made_k), *z = given_or_made(a[3], made_v);
    PyObject *both = y && z ? PyTuple_Pack(2, y, z) : nullptr;
    Py_XDECREF(y);
    Py_XDECREF(z);
    return both;
    KRK_CATCH
}

// q, cache, q_start, kv_len, page_table, max_q, tree, scale, softcap, window, sinks, max_kv_len, out, workspace, stream -> out
PyObject *attention_tree(PyObject *, PyObject *const *a, Py_ssize_t n) {
    KRK_NARGS(15, "attention_tree")
    KRK_TRY
    Args g{a};
    const at::Tensor *q = g.t(0), *start = g.t(2), *len = g.t(3), *table = g.t(4), *tree = g.t_or_none(6), *sinks = g.t_or_none(10), *out = g.t_or_none(12), *ws = g.t_or_none(13);
    const auto *c = (const krk_cuda_kv_cache *)g.addr(1);
    krk_cuda_attention t = {};
    const int64_t max_q = g.i(5), window = g.i(9);
    t.max_kv_len = g.i(11), t.softcap = g.f(8);
    if (a[7] != Py_None) t.scale = g.f(7);
    void *st = a[14] == Py_None ? nullptr : g.stream(14);
    if (!g.ok) return nullptr;
    if (a[7] == Py_None) t.scale = 1.0f / std::sqrt((float)c->head_dim);
    if (!headed(q, q, -1, -1, c->head_dim, "q") || !tabled(table, q, at::kInt, -1, "page_table")) return nullptr;
    const int64_t rows = q->size(0), heads = q->size(1), n_seq = table->size(0);
    if (!listed(start, q, at::kInt, n_seq + 1, "q_start") || !listed(len, q, at::kInt, n_seq, "kv_len") || !listed(sinks, q, at::kFloat, heads, "sinks")) return nullptr;
    if (tree && !listed(tree, q, tree->scalar_type() == at::kUInt64 ? at::kUInt64 : at::kLong, rows, "tree")) return nullptr;
    if (!table->is_contiguous()) return refuse("page_table: expected a contiguous table"), nullptr;
    if (max_q < 0 || max_q > KRK_CUDA_MAX_DRAFT || window < 0 || window > INT32_MAX || heads > 65536 || table->size(1) > INT32_MAX)
        return refuse("attention_tree: max_q, window, heads or pages out of range"), nullptr;
    Where where(*q, a[14] != Py_None, st);
    at::Tensor made, made_ws;
    if (!out) out = &(made = empty_like_device(*q, {rows, heads, (int64_t)c->head_dim}, at::kFloat));
    else if (!headed(out, q, rows, heads, c->head_dim, "out")) return nullptr;
    t.q_start = Args::ptr(start), t.kv_len = Args::ptr(len), t.page_table = Args::ptr(table), t.tree = Args::ptr(tree), t.sinks = Args::ptr(sinks);
    t.q_stride = row_stride(q), t.out_stride = row_stride(out);
    t.n_seq = (int)n_seq, t.n_heads = (int)heads, t.max_q = (int)max_q, t.table_width = (int)table->size(1), t.window = (int)window;
    if (rows == 0) return given_or_made(a[12], made);   // (no sequence has a row)
    if (ws) {
        if (!typed(ws, q, at::kByte, "workspace")) return nullptr;
        if (!ws->is_contiguous()) return refuse("workspace: expected contiguous bytes"), nullptr;
    } else if (const size_t need = krk_cuda_attention_tree_workspace_bytes(c, &t)) {
        ws = &(made_ws = empty_like_device(*q, {(int64_t)need}, at::kByte));
    }
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = krk_cuda_attention_tree(Args::ptr(out), Args::ptr(q), c, &t, Args::ptr(ws), ws ? (size_t)ws->numel() : 0, where.stream);
    Py_END_ALLOW_THREADS
    if (rc != 0) return fail(rc, "attention_tree");
    return given_or_made(a[12], made);
    KRK_CATCH
}

// logits, hist, hist_len, rep, freq, pres, bias_ids, bias, mask, mask_row, bias_len, out, stream -> out
PyObject *logits_adjust(PyObject *, PyObject *const *a, Py_ssize_t n) {
    KRK_NARGS(13, "logits_adjust")
    KRK_TRY
    Args g{a};
    const at::Tensor *x = g.t(0), *hist = g.t_or_none(1), *hist_len = g.t_or_none(2), *rep = g.t_or_none(3), *freq = g.t_or_none(4), *pres = g.t_or_none(5), *ids = g.t_or_none(6),
                     *bias = g.t_or_none(7), *mask = g.t_or_none(8), *mask_row = g.t_or_none(9), *bias_len = g.t_or_none(10), *out = g.t_or_none(11);
    void *st = a[12] == Py_None ? nullptr : g.stream(12);
    if (!g.ok || !typed(x, x, at::kFloat, "logits")) return nullptr;
    at::Tensor one;
    const bool flat = x->dim() == 1;
    if (flat) x = &(one = x->unsqueeze(0));
    if (!tabled(x, x, at::kFloat, -1, "logits")) return nullptr;
    const int64_t rows = x->size(0), vocab = x->size(1);
    const at::ScalarType words = mask && mask->scalar_type() == at::kUInt32 ? at::kUInt32 : at::kInt;
    if (!tabled(hist, x, at::kInt, rows, "hist") || !listed(hist_len, x, at::kInt, rows, "hist_len") || !listed(rep, x, at::kFloat, rows, "rep") ||
        !listed(freq, x, at::kFloat, rows, "freq") || !listed(pres, x, at::kFloat, rows, "pres") || !tabled(ids, x, at::kInt, rows, "bias_ids") ||
        !tabled(bias, x, at::kFloat, rows, "bias") || !listed(bias_len, x, at::kInt, rows, "bias_len") || !tabled(mask, x, words, -1, "mask") ||
        !listed(mask_row, x, at::kInt, rows, "mask_row"))
        return nullptr;
    if ((bias == nullptr) != (ids == nullptr) || (bias && (bias->size(1) != ids->size(1) || (rows > 1 && bias->stride(0) != ids->stride(0)))))
        return refuse("bias and bias_ids: expected two tables of one shape and layout"), nullptr;
    if (mask && mask->size(1) < (vocab + 31) / 32) return refuse("mask: expected a bit for each logit of a row"), nullptr;
    Where where(*x, a[12] != Py_None, st);
    at::Tensor made, out_one;
    if (!out) {
        made = flat ? empty_like_device(*x, {vocab}, at::kFloat) : empty_like_device(*x, {rows, vocab}, at::kFloat);
        out = &made;
    }
    if (out->dim() == 1) out = &(out_one = out->unsqueeze(0));
    if (!tabled(out, x, at::kFloat, rows, "out")) return nullptr;
    if (out->size(1) != vocab) return refuse("out: expected the shape of logits"), nullptr;
    krk_cuda_adjust j = {};
    j.n_rows = rows, j.n_vocab = vocab, j.stride = row_stride(x), j.out_stride = row_stride(out);
    j.hist = Args::ptr(hist), j.hist_len = Args::ptr(hist_len), j.rep = Args::ptr(rep), j.freq = Args::ptr(freq), j.pres = Args::ptr(pres);
    j.bias_ids = Args::ptr(ids), j.bias = Args::ptr(bias), j.bias_len = Args::ptr(bias_len), j.mask = Args::ptr(mask), j.mask_row = Args::ptr(mask_row);
    if (hist) j.hist_n = hist->size(1), j.hist_stride = row_stride(hist);
    if (bias) j.bias_n = bias->size(1), j.bias_stride = row_stride(bias);
    if (mask) j.n_masks = mask->size(0), j.mask_stride = row_stride(mask);
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = krk_cuda_logits_adjust(Args::ptr(out), Args::ptr(x), &j, where.stream);
    Py_END_ALLOW_THREADS
    if (rc != 0) return fail(rc, "logits_adjust");
    return given_or_made(a[11], made);
    KRK_CATCH
}

bool headed16(const at::Tensor *t, const at::Tensor *first, int64_t rows, int64_t heads, int64_t d, const char *name) {   // as headed, f32 or f16
    if (!on_device(t, first, name)) return false;
    if (t->scalar_type() == at::kFloat) return headed(t, first, rows, heads, d, name);
    if (!typed(t, first, at::kHalf, name)) return false;
    if (t->dim() == 3 && (rows < 0 || t->size(0) == rows) && (heads < 0 || t->size(1) == heads) && t->size(2) == d &&
        (t->numel() == 0 || ((d <= 1 || t->stride(2) == 1) && (t->size(1) <= 1 || t->stride(1) == d))))
        return true;
    PyErr_Format(PyExc_ValueError, "%s: expected [rows][heads][values] with the heads of a row behind each other", name);
    return false;
}
int x_dtype(const at::Tensor *t) { return t->scalar_type() == at::kHalf ? KRK_CUDA_X_F16 : KRK_CUDA_X_F32; }

// q, cache, q_start, kv_len, page_table, max_q, scale, softcap, window, sinks, max_kv_len, out, workspace, stream -> out
PyObject *attention_chunk(PyObject *, PyObject *const *a, Py_ssize_t n) {
    KRK_NARGS(14, "attention_chunk")
    KRK_TRY
    Args g{a};
    const at::Tensor *q = g.t(0), *start = g.t(2), *len = g.t(3), *table = g.t(4), *sinks = g.t_or_none(9), *out = g.t_or_none(11), *ws = g.t_or_none(12);
    const auto *c = (const krk_cuda_kv_cache *)g.addr(1);
    krk_cuda_attention t = {};
    const int64_t max_q = g.i(5), window = g.i(8);
    t.max_kv_len = g.i(10), t.softcap = g.f(7);
    if (a[6] != Py_None) t.scale = g.f(6);
    void *st = a[13] == Py_None ? nullptr : g.stream(13);
    if (!g.ok) return nullptr;
    if (a[6] == Py_None) t.scale = 1.0f / std::sqrt((float)c->head_dim);
    if (!headed16(q, q, -1, -1, c->head_dim, "q") || !tabled(table, q, at::kInt, -1, "page_table")) return nullptr;
    const int64_t rows = q->size(0), heads = q->size(1), n_seq = table->size(0);
    if (!listed(start, q, at::kInt, n_seq + 1, "q_start") || !listed(len, q, at::kInt, n_seq, "kv_len") || !listed(sinks, q, at::kFloat, heads, "sinks")) return nullptr;
    if (!table->is_contiguous()) return refuse("page_table: expected a contiguous table"), nullptr;
    if (max_q < 0 || max_q > INT32_MAX || window < 0 || window > INT32_MAX || heads > 65536 || table->size(1) > INT32_MAX || n_seq > INT32_MAX)
        return refuse("attention_chunk: max_q, window, heads or pages out of range"), nullptr;
    Where where(*q, a[13] != Py_None, st);
    at::Tensor made, made_ws;
    if (!out) out = &(made = empty_like_device(*q, {rows, heads, (int64_t)c->head_dim}, q->scalar_type()));
    else if (!headed16(out, q, rows, heads, c->head_dim, "out")) return nullptr;
    t.q_start = Args::ptr(start), t.kv_len = Args::ptr(len), t.page_table = Args::ptr(table), t.sinks = Args::ptr(sinks);
    t.q_stride = row_stride(q), t.out_stride = row_stride(out);
    t.n_seq = (int)n_seq, t.n_heads = (int)heads, t.max_q = (int)(max_q < rows ? max_q : rows), t.table_width = (int)table->size(1), t.window = (int)window;
    if (rows == 0) return given_or_made(a[11], made);   // (no sequence has a row)
    if (ws) {
        if (!typed(ws, q, at::kByte, "workspace")) return nullptr;
        if (!ws->is_contiguous()) return refuse("workspace: expected contiguous bytes"), nullptr;
    } else if (const size_t need = krk_cuda_attention_chunk_workspace_bytes(c, &t, x_dtype(out))) {
        ws = &(made_ws = empty_like_device(*q, {(int64_t)need}, at::kByte));
    }
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = krk_cuda_attention_chunk(Args::ptr(out), x_dtype(out), Args::ptr(q), x_dtype(q), c, &t, Args::ptr(ws), ws ? (size_t)ws->numel() : 0, where.stream);
    Py_END_ALLOW_THREADS
    if (rc != 0) return fail(rc, "attention_chunk");
    return given_or_made(a[11], made);
    KRK_CATCH
}

// kv_before, n_new, page_table, free_pages, n_free, page_size, max_tok, out (seven tensors) or None, stream -> q_start, kv_len, positions, slots, last, counts, page_table
PyObject *step_plan(PyObject *, PyObject *const *a, Py_ssize_t n) {
    KRK_NARGS(9, "step_plan")
    KRK_TRY
    Args g{a};
    const at::Tensor *before = g.t(0), *fresh = g.t(1), *table = g.t(2), *free = g.t(3), *n_free = g.t(4);
    const int64_t page = g.i(5), max_tok = g.i(6);
    void *st = a[8] == Py_None ? nullptr : g.stream(8);
    if (!g.ok) return nullptr;
    if (!listed(before, before, at::kInt, -1, "kv_before")) return nullptr;
    const int64_t n_seq = before->numel();
    if (!listed(fresh, before, at::kInt, n_seq, "n_new") || !tabled(table, before, at::kInt, n_seq, "page_table") || !listed(free, before, at::kInt, -1, "free_pages") ||
        !listed(n_free, before, at::kInt, 1, "n_free"))
        return nullptr;
    if (!table->is_contiguous()) return refuse("page_table: expected a contiguous table"), nullptr;
    if (page < 1 || page > INT32_MAX || max_tok < 0 || max_tok > INT32_MAX || n_seq >= INT32_MAX || table->size(1) > INT32_MAX)
        return refuse("step_plan: page_size, max_tok, sequences or pages out of range"), nullptr;
    Where where(*before, a[8] != Py_None, st);
    static const char *const names[6] = {"q_start", "kv_len", "positions", "slots", "last", "counts"};
    const int64_t sizes[6] = {n_seq + 1, n_seq, max_tok, max_tok, n_seq, 4};
    std::array<at::Tensor, 6> made;
    std::array<PyObject *, 6> objects{};
    std::array<const at::Tensor *, 6> to{};
    if (a[7] != Py_None) {
        if (!PyTuple_Check(a[7]) || PyTuple_GET_SIZE(a[7]) != 7) return refuse("out: expected a StepPlan"), nullptr;
        Args o{&PyTuple_GET_ITEM(a[7], 0)};
        for (int i = 0; i < 6; i++) {
            to[i] = o.t(i);
            if (!o.ok || !listed(to[i], before, i == 3 ? at::kLong : at::kInt, sizes[i], names[i])) return nullptr;
            objects[i] = PyTuple_GET_ITEM(a[7], i);
        }
    } else {
        for (int i = 0; i < 6; i++) to[i] = &(made[i] = empty_like_device(*before, {sizes[i]}, i == 3 ? at::kLong : at::kInt));
    }
    krk_cuda_step s = {};
    s.kv_before = Args::ptr(before), s.n_new = Args::ptr(fresh), s.page_table = Args::ptr(table), s.free_pages = Args::ptr(free), s.n_free = Args::ptr(n_free);
    s.q_start = Args::ptr(to[0]), s.kv_len = Args::ptr(to[1]), s.positions = Args::ptr(to[2]), s.slots = Args::ptr(to[3]), s.last = Args::ptr(to[4]), s.counts = Args::ptr(to[5]);
    s.max_tok = max_tok, s.free_cap = free->numel(), s.n_seq = (int)n_seq, s.table_width = (int)table->size(1), s.page_size = (int)page;
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = krk_cuda_step_plan(&s, where.stream);
    Py_END_ALLOW_THREADS
    if (rc != 0) return fail(rc, "step_plan");
    PyObject *all = PyTuple_New(7);
    if (!all) return nullptr;
    for (int i = 0; i < 6; i++) {
        PyObject *x = objects[i] ? Py_NewRef(objects[i]) : THPVariable_Wrap(made[i]);
        if (!x) {
            Py_DECREF(all);
            return nullptr;
        }
        PyTuple_SET_ITEM(all, i, x);
    }
    PyTuple_SET_ITEM(all, 6, Py_NewRef(a[2]));
    return all;
    KRK_CATCH
}

// x, weight, residual, post_weight, post_norm, gate, alpha, eps, offset, half, h_out, out, stream -> (y, h)
PyObject *block_norm(PyObject *, PyObject *const *a, Py_ssize_t n) {
    KRK_NARGS(13, "block_norm")
    KRK_TRY
    Args g{a};
    const at::Tensor *x = g.t(0), *w = g.t_or_none(1), *res = g.t_or_none(2), *post = g.t_or_none(3), *gate = g.t_or_none(5), *h = g.t_or_none(10), *y = g.t_or_none(11);
    krk_cuda_norm m = {};
    m.post_norm = g.b(4), m.alpha = g.f(6), m.eps = g.f(7), m.offset = g.f(8);
    const bool half = g.b(9);
    void *st = a[12] == Py_None ? nullptr : g.stream(12);
    if (!g.ok || !tabled(x, x, at::kFloat, -1, "x")) return nullptr;
    const int64_t rows = x->size(0), width = x->size(1);
    if (!listed(w, x, at::kFloat, width, "weight") || !tabled(res, x, at::kFloat, rows, "residual") || !listed(post, x, at::kFloat, width, "post_weight")) return nullptr;
    if (res && res->size(1) != width) return refuse("residual: expected the shape of x"), nullptr;
    if (post && !m.post_norm) return refuse("post_weight without post_norm"), nullptr;
    if (gate && gate->dim() == 1) {
        if (!listed(gate, x, at::kFloat, width, "gate")) return nullptr;
    } else if (gate) {
        if (!tabled(gate, x, at::kFloat, rows, "gate")) return nullptr;
        if (gate->size(1) != width) return refuse("gate: expected a row of x, or one for each"), nullptr;
        m.gate_stride = rows > 1 ? gate->stride(0) : width;
    }
    Where where(*x, a[12] != Py_None, st);
    at::Tensor made_y, made_h;
    if (!h) h = &(made_h = empty_like_device(*x, {rows, width}, at::kFloat));
    else if (!tabled(h, x, at::kFloat, rows, "h_out")) return nullptr;
    if (!y) y = &(made_y = empty_like_device(*x, {rows, width}, half ? at::kHalf : at::kFloat));
    else if (!on_device(y, x, "out") || !tabled(y, x, y->scalar_type() == at::kHalf ? at::kHalf : at::kFloat, rows, "out")) return nullptr;
    if (h->size(1) != width || y->size(1) != width) return refuse("out, h_out: expected the shape of x"), nullptr;
    m.residual = Args::ptr(res), m.gate = Args::ptr(gate), m.post_weight = Args::ptr(post), m.weight = Args::ptr(w);
    m.rows = rows, m.n = width, m.x_stride = row_stride(x), m.h_stride = row_stride(h), m.y_stride = row_stride(y);
    if (res) m.residual_stride = row_stride(res);
    m.y_dtype = x_dtype(y);
    if (rows > 0 && width > 0) {
        int rc;
        Py_BEGIN_ALLOW_THREADS rc = krk_cuda_block_norm(Args::ptr(y), Args::ptr(h), Args::ptr(x), &m, where.stream);
        Py_END_ALLOW_THREADS
        if (rc != 0) return fail(rc, "block_norm");
    }
    PyObject *oy = given_or_made(a[11], made_y), *oh = given_or_made(a[10], made_h);
    PyObject *both = oy && oh ? PyTuple_Pack(2, oy, oh) : nullptr;
    Py_XDECREF(oy);
    Py_XDECREF(oh);
    return both;
    KRK_CATCH
}

// logits, row_start, draft, accept_u, sample_u, draft_logits, temp, draft_temp, tokens, n_accepted, logprob, workspace, stream -> (tokens, n_accepted, logprob)
PyObject *verify_draft(PyObject *, PyObject *const *a, Py_ssize_t n) {
    KRK_NARGS(13, "verify_draft")
    KRK_TRY
    Args g{a};
    const at::Tensor *x = g.t(0), *start = g.t(1), *draft = g.t(2), *au = g.t(3), *su = g.t(4), *q = g.t_or_none(5), *temp = g.t_or_none(6), *qt = g.t_or_none(7),
                     *tokens = g.t_or_none(8), *count = g.t_or_none(9), *lp = g.t_or_none(10), *ws = g.t_or_none(11);
    void *st = a[12] == Py_None ? nullptr : g.stream(12);
    if (!g.ok || !tabled(x, x, at::kFloat, -1, "logits")) return nullptr;
    const int64_t rows = x->size(0), vocab = x->size(1);
    if (!listed(start, x, at::kInt, -1, "row_start")) return nullptr;
    const int64_t n_seq = start->numel() - 1;
    if (n_seq < 0 || n_seq > INT32_MAX) return refuse("row_start: expected one more element than there are sequences"), nullptr;
    if (!listed(draft, x, at::kInt, rows, "draft") || !listed(au, x, at::kFloat, rows, "accept_u") || !listed(su, x, at::kFloat, n_seq, "sample_u") ||
        !tabled(q, x, at::kFloat, rows, "draft_logits") || !listed(temp, x, at::kFloat, n_seq, "temp") || !listed(qt, x, at::kFloat, n_seq, "draft_temp") ||
        !listed(tokens, x, at::kInt, rows, "tokens") || !listed(count, x, at::kInt, n_seq, "n_accepted") || !listed(lp, x, at::kFloat, rows, "logprob"))
        return nullptr;
    if (q && q->size(1) != vocab) return refuse("draft_logits: expected the shape of logits"), nullptr;
    Where where(*x, a[12] != Py_None, st);
    at::Tensor made_t, made_c, made_l, made_ws;
    if (!tokens) tokens = &(made_t = empty_like_device(*x, {rows}, at::kInt));
    if (!count) count = &(made_c = empty_like_device(*x, {n_seq}, at::kInt));
    if (!lp) lp = &(made_l = empty_like_device(*x, {rows}, at::kFloat));
    krk_cuda_verify v = {};
    v.row_start = Args::ptr(start), v.draft = Args::ptr(draft), v.accept_u = Args::ptr(au), v.sample_u = Args::ptr(su), v.temp = Args::ptr(temp), v.draft_temp = Args::ptr(qt);
    v.draft_logits = Args::ptr(q);
    v.n_rows = rows, v.n_vocab = vocab, v.stride = row_stride(x), v.n_seq = (int)n_seq;
    if (q) v.draft_stride = row_stride(q);
    if (ws) {
        if (!typed(ws, x, at::kByte, "workspace")) return nullptr;
        if (!ws->is_contiguous()) return refuse("workspace: expected contiguous bytes"), nullptr;
    } else if (const size_t need = krk_cuda_verify_draft_workspace_bytes(&v)) {
        ws = &(made_ws = empty_like_device(*x, {(int64_t)need}, at::kByte));
    }
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = krk_cuda_verify_draft(Args::ptr(tokens), Args::ptr(count), Args::ptr(lp), Args::ptr(x), &v, Args::ptr(ws), ws ? (size_t)ws->numel() : 0, where.stream);
    Py_END_ALLOW_THREADS
    if (rc != 0) return fail(rc, "verify_draft");
    PyObject *ot = given_or_made(a[8], made_t), *oc = given_or_made(a[9], made_c), *ol = given_or_made(a[10], made_l);
    PyObject *all = ot && oc && ol ? PyTuple_Pack(3, ot, oc, ol) : nullptr;
    Py_XDECREF(ot);
    Py_XDECREF(oc);
    Py_XDECREF(ol);
    return all;
    KRK_CATCH
}

#define KRK_FAST(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {{"set_raise", set_raise, METH_O, nullptr},
                         {"set_address", set_address, METH_O, nullptr},
                         KRK_FAST(gemv),
                         KRK_FAST(gemv_group),
                         KRK_FAST(gemm),
                         KRK_FAST(silu_mul),
                         KRK_FAST(embed),
                         KRK_FAST(logits_topk),
                         KRK_FAST(qk_norm_rope),
                         KRK_FAST(kv_append),
                         KRK_FAST(kv_read),
                         KRK_FAST(attention_tree),
                         KRK_FAST(logits_adjust),
                         KRK_FAST(attention_chunk),
                         KRK_FAST(step_plan),
                         KRK_FAST(block_norm),
                         KRK_FAST(verify_draft),
                         KRK_FAST(moe_ffn),
                         KRK_FAST(moe_ffn_routed),
                         KRK_FAST(backend_upload),
                         KRK_FAST(backend_download),
                         KRK_FAST(backend_gemm),
                         KRK_FAST(backend_gemm_accumulate),
                         KRK_FAST(backend_gemm_group),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fastcall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}   // namespace

PyMODINIT_FUNC PyInit__fastcall(void) { return PyModule_Create(&module); }
