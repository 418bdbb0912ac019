// dtts.serving's calls as CPython functions: a step is a few microseconds of GPU work, and reading ten tensors'
// sizes, types and addresses from Python takes as long again (a paged append: 7.3 us of Python and 3.9 of ctypes and
// launch). Each function here checks what its Python caller would, allocates what it would, and enqueues on torch's
// current stream. What it does not take (a wrong argument, another device than the current one, sizes that are
// no Python ints) returns None, and the Python path makes the call or says what is wrong with it.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "dtts.h"

namespace {

using at::Tensor;

// Arguments one after another; ok turns false at the first that is not what the caller says it is.
struct Args {
    PyObject *const *v;
    bool ok = true;
    int device = -1;  // the first tensor's: the current one

    explicit Args(PyObject *const *args) : v(args) {}
    const Tensor *tensor(int i) {
        if (!ok || !THPVariable_Check(v[i])) return fail();
        const Tensor &t = THPVariable_Unpack(v[i]);
        if (!t.is_cuda() || t.layout() != at::kStrided) return fail();
        const int d = t.get_device();
        if (device < 0) {
            device = d;
            if (d != c10::hip::current_device()) return fail();
        }
        return d == device ? &t : fail();
    }
    const Tensor *tensor(int i, at::ScalarType type) {  // contiguous, of one type
        const Tensor *t = tensor(i);
        return t && t->scalar_type() == type && t->is_contiguous() ? t : fail();
    }
    const Tensor *maybe(int i, at::ScalarType type) { return v[i] == Py_None ? nullptr : tensor(i, type); }
    int64_t integer(int i) {
        if (!ok || !PyLong_Check(v[i])) return fail(), 0;
        int over = 0;
        const int64_t x = PyLong_AsLongLongAndOverflow(v[i], &over);
        return over ? (fail(), 0) : x;
    }
    float real(int i) {
        if (!ok || !(PyFloat_Check(v[i]) || PyLong_Check(v[i]))) return fail(), 0.0f;
        const double x = PyFloat_AsDouble(v[i]);
        if (PyErr_Occurred()) {  // an int past a double
            PyErr_Clear();
            fail();
        }
        return static_cast<float>(x);
    }
    bool truth(int i) {
        if (!ok || !PyBool_Check(v[i])) return fail(), false;
        return v[i] == Py_True;
    }
    const Tensor *fail() {
        ok = false;
        return nullptr;
    }
    void need(bool c) { ok = ok && c; }
    hipStream_t stream() const { return c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(device)).stream(); }
};

template <typename T>
T *data(const Tensor *t) {
    return t ? static_cast<T *>(t->data_ptr()) : nullptr;
}

// [rows, heads, D] with contiguous rows: the elements between rows. (Torch leaves any number as the stride of a size of 1.)
int64_t rows_of(Args &a, const Tensor *t) {
    if (!t || t->dim() != 3 || t->stride(2) != 1 || (t->stride(1) != t->size(2) && t->size(1) != 1)) return a.fail(), 0;
    return t->size(0) > 1 ? t->stride(0) : t->size(1) * t->size(2);
}

// [n_pages, n_kv, page, D] with contiguous pages: the elements between them.
int64_t page_stride_of(Args &a, const Tensor *t) {
    const int64_t rows = t->size(2) * t->size(3);
    if (t->stride(3) != 1 || t->stride(2) != t->size(3) || (t->stride(1) != rows && t->size(1) != 1)) return a.fail(), 0;
    return t->size(0) > 1 ? t->stride(0) : t->size(1) * rows;
}

struct Paged {
    const Tensor *k, *v, *start, *context, *table;
    int64_t b, n_kv, hd, page, n_pages, max_pages, stride;
    Paged(Args &a, int i)
        : k(a.tensor(i)), v(a.tensor(i + 1)), start(a.tensor(i + 2, at::kInt)), context(a.tensor(i + 3, at::kInt)),
          table(a.tensor(i + 4, at::kInt)) {
        a.need(a.ok && k->dim() == 4 && k->scalar_type() == at::kHalf && v->scalar_type() == at::kHalf && k->sizes() == v->sizes() &&
               table->dim() == 2);
        if (!a.ok) return;
        n_pages = k->size(0), n_kv = k->size(1), page = k->size(2), hd = k->size(3);
        b = table->size(0), max_pages = table->size(1);
        stride = page_stride_of(a, k);
        a.need(page_stride_of(a, v) == stride && context->numel() == b && start->numel() == b + 1);
    }
};

// `given`, or a new f16 [tokens, heads, hd].
Tensor out_of(Args &a, int i, const Tensor &like, int64_t tokens, int64_t heads, int64_t hd) {
    if (a.v[i] != Py_None) {
        const Tensor *t = a.tensor(i, at::kHalf);
        a.need(t && t->numel() == tokens * heads * hd);
        return a.ok ? *t : Tensor();
    }
    return a.ok ? at::empty({tokens, heads, hd}, like.options().dtype(at::kHalf).requires_grad(false)) : Tensor();
}

Tensor workspace_of(Args &a, int i, size_t need, const Tensor &like) {
    if (a.v[i] != Py_None) {
        const Tensor *t = a.tensor(i, at::kByte);
        return t ? *t : Tensor();
    }
    return a.ok && need ? at::empty({static_cast<int64_t>(need)}, like.options().dtype(at::kByte).requires_grad(false)) : Tensor();
}

PyObject *none() { Py_RETURN_NONE; }

// (x, cos, sin, pos, interleaved, out) -> out
PyObject *rotary(PyObject *const *args) {
    Args a(args);
    const Tensor *x = a.tensor(0), *cos = a.tensor(1, at::kFloat), *sin = a.tensor(2, at::kFloat), *pos = a.tensor(3, at::kInt);
    const int layout = a.truth(4) ? DTTS_ROPE_INTERLEAVED : DTTS_ROPE_HALF;
    const int64_t xs = rows_of(a, x);
    a.need(a.ok && cos->dim() == 2 && cos->sizes() == sin->sizes() && pos->numel() == x->size(0));
    if (!a.ok) return none();
    const bool f32 = x->scalar_type() == at::kFloat;
    a.need(f32 || x->scalar_type() == at::kHalf);
    Tensor y;
    if (args[5] != Py_None) {
        const Tensor *t = a.tensor(5);
        a.need(t && t->scalar_type() == x->scalar_type() && t->sizes() == x->sizes());
        if (a.ok) y = *t;
    } else if (a.ok) {
        y = at::empty(x->sizes(), x->options().requires_grad(false));
    }
    const int64_t ys = a.ok ? rows_of(a, &y) : 0;
    if (!a.ok) return none();
    const int64_t rows = x->size(0), heads = x->size(1), hd = x->size(2), rot = 2 * cos->size(1), len = cos->size(0);
    const int status =
        f32 ? dtts_rotary_f32(data<float>(x), data<float>(cos), data<float>(sin), data<int32_t>(pos), data<float>(&y), rows, heads,
                              hd, rot, layout, xs, ys, len, a.stream())
            : dtts_rotary_f16(data<dtts_f16>(x), data<float>(cos), data<float>(sin), data<int32_t>(pos), data<dtts_f16>(&y), rows,
                              heads, hd, rot, layout, xs, ys, len, a.stream());
    return status == DTTS_OK ? THPVariable_Wrap(y) : none();
}

// (qkv, cos, sin, k_pages, v_pages, q_start, context, pages, heads, norms, eps, interleaved, out) -> out
PyObject *append(PyObject *const *args) {
    Args a(args);
    const Tensor *qkv = a.tensor(0), *cos = a.tensor(1, at::kFloat), *sin = a.tensor(2, at::kFloat);
    const Paged p(a, 3);
    const int64_t heads = a.integer(8);
    const Tensor *norms = a.maybe(9, at::kFloat);
    const float eps = a.real(10);
    const int layout = a.truth(11) ? DTTS_ROPE_INTERLEAVED : DTTS_ROPE_HALF;
    a.need(a.ok && cos->dim() == 2 && cos->sizes() == sin->sizes() && qkv->dim() == 2 && qkv->is_contiguous() && heads > 0 &&
           heads <= 65536 && qkv->size(1) == (heads + 2 * p.n_kv) * p.hd && (!norms || norms->numel() == 2 * p.hd));
    if (!a.ok) return none();
    const bool f32 = qkv->scalar_type() == at::kFloat;
    a.need(f32 || qkv->scalar_type() == at::kHalf);
    const int64_t tokens = qkv->size(0);
    const Tensor out = out_of(a, 12, *qkv, tokens, heads, p.hd);
    if (!a.ok) return none();
    const auto call = [&](auto fn, auto x) {
        return fn(x, data<float>(norms), data<float>(cos), data<float>(sin), data<int32_t>(p.start), data<int32_t>(p.context),
                  data<int32_t>(p.table), data<dtts_f16>(&out), data<dtts_f16>(p.k), data<dtts_f16>(p.v), tokens, p.b, heads, p.n_kv,
                  p.hd, 2 * cos->size(1), layout, p.page, p.n_pages, p.max_pages, p.stride, cos->size(0), eps, a.stream());
    };
    const int status = f32 ? call(dtts_qk_rope_append_paged_f32, data<const float>(qkv))
                           : call(dtts_qk_rope_append_paged_f16, data<const dtts_f16>(qkv));
    return status == DTTS_OK ? THPVariable_Wrap(out) : none();
}

// (q, k_pages, v_pages, q_start, context, pages, max_q, max_context, scale, window, out, workspace) -> out
PyObject *attention(PyObject *const *args) {
    Args a(args);
    const Tensor *q = a.tensor(0);
    const int64_t qs = rows_of(a, q);
    const Paged p(a, 1);
    const int64_t max_q = a.integer(6), max_context = a.integer(7), window = a.integer(9);
    const float scale = a.real(8);
    a.need(a.ok && q->scalar_type() == at::kHalf && q->size(2) == p.hd);
    if (!a.ok) return none();
    const int64_t tokens = q->size(0), heads = q->size(1);
    const Tensor out = out_of(a, 10, *q, tokens, heads, p.hd);
    const size_t need = args[11] == Py_None ? dtts_paged_attention_workspace_bytes(tokens, p.b, heads, p.n_kv, p.hd, max_q, max_context, window) : 0;
    const Tensor ws = workspace_of(a, 11, need, *q);
    if (!a.ok) return none();
    const int status = dtts_paged_attention_f16(
        data<dtts_f16>(q), data<dtts_f16>(p.k), data<dtts_f16>(p.v), data<int32_t>(p.start), data<int32_t>(p.context),
        data<int32_t>(p.table), data<dtts_f16>(&out), tokens, p.b, heads, p.n_kv, p.hd, p.page, p.n_pages, p.max_pages, p.stride, qs,
        max_q, max_context, window, scale, ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? ws.numel() : 0, a.stream());
    return status == DTTS_OK ? THPVariable_Wrap(out) : none();
}

// (logits, u, temperature, top_k, top_p, min_p, workspace) -> (tokens, log-probabilities)
PyObject *sample(PyObject *const *args) {
    Args a(args);
    const Tensor *x = a.tensor(0), *u = a.tensor(1, at::kFloat), *t = a.maybe(2, at::kFloat), *k = a.maybe(3, at::kInt),
                 *p = a.maybe(4, at::kFloat), *m = a.maybe(5, at::kFloat);
    a.need(a.ok && x->dim() == 2);
    if (!a.ok) return none();
    const int64_t rows = x->size(0), vocab = x->size(1);
    const bool f32 = x->scalar_type() == at::kFloat;
    const auto one = [&](const Tensor *s) { return !s || s->numel() == rows; };
    a.need((f32 || x->scalar_type() == at::kHalf) && (x->stride(1) == 1 || vocab <= 1) && one(u) && one(t) && one(k) && one(p) && one(m));
    if (!a.ok) return none();
    const int64_t stride = rows > 1 ? x->stride(0) : std::max(x->stride(0), vocab);
    const Tensor ws = workspace_of(a, 6, args[6] == Py_None ? dtts_sample_workspace_bytes(rows, vocab) : 0, *x);
    if (!a.ok) return none();
    const auto like = x->options().requires_grad(false);
    const Tensor token = at::empty({rows}, like.dtype(at::kInt)), logprob = at::empty({rows}, like.dtype(at::kFloat));
    const auto call = [&](auto fn, auto logits) {
        return fn(logits, data<float>(t), data<int32_t>(k), data<float>(p), data<float>(m), data<float>(u), data<int32_t>(&token),
                  data<float>(&logprob), rows, vocab, stride, ws.defined() ? ws.data_ptr() : nullptr,
                  ws.defined() ? static_cast<size_t>(ws.numel()) : 0, a.stream());
    };
    const int status = f32 ? call(dtts_sample_f32, data<const float>(x)) : call(dtts_sample_f16, data<const dtts_f16>(x));
    if (status != DTTS_OK) return none();
    PyObject *both = PyTuple_New(2);
    if (!both) return nullptr;
    PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(token));
    PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(logprob));
    return both;
}

// No C++ exception leaves: where torch refuses an allocation, nothing is enqueued yet, and the Python path meets the
// same refusal.
template <PyObject *(*F)(PyObject *const *), int N>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "%d arguments expected, got %zd", N, n);
        return nullptr;
    }
    try {
        return F(args);
    } catch (...) {
        return none();
    }
}

template <PyObject *(*F)(PyObject *const *), int N>
PyMethodDef method(const char *name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(entry<F, N>)), METH_FASTCALL, nullptr};
}

PyMethodDef kMethods[] = {method<rotary, 6>("rotary"), method<append, 13>("qk_rope_append_paged"),
                          method<attention, 12>("paged_attention"), method<sample, 7>("sample"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving(void) { return PyModule_Create(&kModule); }
