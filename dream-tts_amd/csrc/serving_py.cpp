// dtts.serving's calls as CPython functions: a step is a few microseconds of GPU work, and reading ten tensors'
// sizes, types and addresses from Python takes as long again (a paged append: 7.3 us of Python and 3.9 of ctypes and
// launch). Each function here checks what its Python caller would, allocates what it would, and enqueues on torch's
// current stream. What it does not take (a wrong argument, another device than the current one, sizes that are
// no Python ints) returns None, and the Python path makes the call or says what is wrong with it.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/util/SmallVector.h>
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

// Pages of f16 values, or of bytes that hold 4-bit ones (5 D / 8 a row).
struct Cache {
    const Tensor *k, *v;
    int64_t n_kv = 0, hd = 0, page = 0, n_pages = 0, stride = 0;
    bool q4 = false;
    Cache(Args &a, int i) : k(a.tensor(i)), v(a.tensor(i + 1)) {
        a.need(a.ok && k->dim() == 4 && k->scalar_type() == v->scalar_type() && k->sizes() == v->sizes());
        if (!a.ok) return;
        q4 = k->scalar_type() == at::kByte;
        n_pages = k->size(0), n_kv = k->size(1), page = k->size(2), hd = q4 ? k->size(3) / 5 * 8 : k->size(3);
        a.need((q4 && k->size(3) % 5 == 0) || k->scalar_type() == at::kHalf);
        stride = page_stride_of(a, k);
        a.need(page_stride_of(a, v) == stride);
    }
};

struct Paged : Cache {
    const Tensor *start, *context, *table;
    int64_t b = 0, max_pages = 0;
    Paged(Args &a, int i)
        : Cache(a, i), start(a.tensor(i + 2, at::kInt)), context(a.tensor(i + 3, at::kInt)), table(a.tensor(i + 4, at::kInt)) {
        a.need(a.ok && table->dim() == 2);
        if (!a.ok) return;
        b = table->size(0), max_pages = table->size(1);
        a.need(context->numel() == b && start->numel() == b + 1);
    }
};

// A page table and its pages' counts.
struct Table {
    const Tensor *pages, *refs;
    int64_t b = 0, max_pages = 0, n_pages = 0;
    explicit Table(Args &a) : pages(a.tensor(0, at::kInt)), refs(a.tensor(1, at::kInt)) {
        a.need(a.ok && pages->dim() == 2 && refs->dim() == 1);
        if (!a.ok) return;
        b = pages->size(0), max_pages = pages->size(1), n_pages = refs->numel();
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

// Several int32 arrays in one allocation: `of` takes the next n of them (each allocation, or view by torch's own way, takes as
// long as a quarter of a launch). Whoever keeps one of them keeps all, so scratch of more than kScratchHere is apart.
constexpr int64_t kScratchHere = 1 << 18;
struct Ints {
    Tensor all;
    int64_t at = 0;
    Ints(const Tensor &like, int64_t n) : all(at::empty({n}, like.options().dtype(at::kInt).requires_grad(false))) {}
    // The last of the arrays: n ints of scratch, of which `all` was made with scratch_here(n).
    Tensor scratch(int64_t n) { return n > kScratchHere ? at::empty({n}, all.options()) : of(n); }
    static int64_t scratch_here(int64_t n) { return n > kScratchHere ? 0 : n; }
    Tensor of(int64_t n) {
        Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
        t.unsafeGetTensorImpl()->set_storage_offset(at);
        t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
        at += n;
        return t;
    }
};

PyObject *tuple_of(std::initializer_list<Tensor> all) {
    PyObject *t = PyTuple_New(static_cast<Py_ssize_t>(all.size()));
    if (!t) return nullptr;
    Py_ssize_t i = 0;
    for (const Tensor &x : all) PyTuple_SET_ITEM(t, i++, THPVariable_Wrap(x));
    return t;
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
    const auto call_on = [&](auto fn, auto x, auto k, auto v) {
        return fn(x, data<float>(norms), data<float>(cos), data<float>(sin), data<int32_t>(p.start), data<int32_t>(p.context),
                  data<int32_t>(p.table), data<dtts_f16>(&out), k, v, tokens, p.b, heads, p.n_kv,
                  p.hd, 2 * cos->size(1), layout, p.page, p.n_pages, p.max_pages, p.stride, cos->size(0), eps, a.stream());
    };
    const auto call = [&](auto f16_pages, auto q4_pages, auto x) {
        return p.q4 ? call_on(q4_pages, x, p.k->data_ptr(), p.v->data_ptr()) : call_on(f16_pages, x, data<dtts_f16>(p.k), data<dtts_f16>(p.v));
    };
    const int status = f32 ? call(dtts_qk_rope_append_paged_f32, dtts_qk_rope_append_paged_q4_f32, data<const float>(qkv))
                           : call(dtts_qk_rope_append_paged_f16, dtts_qk_rope_append_paged_q4_f16, data<const dtts_f16>(qkv));
    return status == DTTS_OK ? THPVariable_Wrap(out) : none();
}

// (q, k_pages, v_pages, q_start, context, pages, max_q, max_context, scale, window, out, workspace, sinks) -> out
PyObject *attention(PyObject *const *args) {
    Args a(args);
    const Tensor *q = a.tensor(0);
    const int64_t qs = rows_of(a, q);
    const Paged p(a, 1);
    const int64_t max_q = a.integer(6), max_context = a.integer(7), window = a.integer(9), sinks = args[12] == Py_None ? 0 : a.integer(12);
    const float scale = a.real(8);
    a.need(a.ok && q->scalar_type() == at::kHalf && q->size(2) == p.hd);
    if (!a.ok) return none();
    const int64_t tokens = q->size(0), heads = q->size(1);
    const Tensor out = out_of(a, 10, *q, tokens, heads, p.hd);
    const size_t need = args[11] == Py_None ? dtts_paged_attention_sinks_workspace_bytes(p.q4 ? 4 : 16, tokens, p.b, heads, p.n_kv,
                                                                                         p.hd, max_q, max_context, window, sinks) : 0;
    const Tensor ws = workspace_of(a, 11, need, *q);
    if (!a.ok) return none();
    const int status = dtts_paged_attention(
        p.q4 ? 4 : 16, data<dtts_f16>(q), p.k->data_ptr(), p.v->data_ptr(), data<int32_t>(p.start), data<int32_t>(p.context),
        data<int32_t>(p.table), data<dtts_f16>(&out), tokens, p.b, heads, p.n_kv, p.hd, p.page, p.n_pages, p.max_pages, p.stride, qs,
        max_q, max_context, window, sinks, scale, ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? ws.numel() : 0, a.stream());
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
    return tuple_of({token, logprob});
}

// (k_pages, v_pages, ids) -> (k, v)
PyObject *unpack(PyObject *const *args) {
    Args a(args);
    const Cache c(a, 0);
    const Tensor *ids = a.maybe(2, at::kInt);
    a.need(a.ok && c.q4);
    if (!a.ok) return none();
    const int64_t n = ids ? ids->numel() : c.n_pages;
    const auto like = c.k->options().dtype(at::kHalf).requires_grad(false);
    const Tensor k = at::empty({n, c.n_kv, c.page, c.hd}, like), v = at::empty({n, c.n_kv, c.page, c.hd}, like);
    const int status = dtts_unpack_pages_q4(c.k->data_ptr(), c.v->data_ptr(), data<int32_t>(ids), data<dtts_f16>(&k), data<dtts_f16>(&v), n,
                                            c.n_kv, c.hd, c.page, c.n_pages, c.stride, a.stream());
    return status == DTTS_OK ? tuple_of({k, v}) : none();
}

// (pages, refs, parent, out, workspace) -> out
PyObject *fork(PyObject *const *args) {
    Args a(args);
    const Table t(a);
    const Tensor *parent = a.tensor(2, at::kInt);
    if (!a.ok) return none();
    const int64_t n = parent->numel();
    Tensor out;
    if (args[3] != Py_None) {
        const Tensor *o = a.tensor(3, at::kInt);
        a.need(o && o->dim() == 2 && o->size(0) == n && o->size(1) == t.max_pages);
        if (a.ok) out = *o;
    } else {
        out = at::empty({n, t.max_pages}, t.pages->options().requires_grad(false));
    }
    if (!a.ok) return none();
    const bool in_place = out.data_ptr() == t.pages->data_ptr();
    const Tensor ws = workspace_of(a, 4, in_place ? 4 * t.b * t.max_pages : 0, *t.pages);
    if (!a.ok) return none();
    const int status = dtts_fork_pages(data<int32_t>(t.pages), data<int32_t>(t.refs), data<int32_t>(parent), data<int32_t>(&out), t.b, n,
                                       t.max_pages, t.n_pages, ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? ws.numel() : 0,
                                       a.stream());
    return status == DTTS_OK ? THPVariable_Wrap(out) : none();
}

// (pages, refs, q_start, context, page, workspace) -> (src, dst, lacking)
PyObject *claim(PyObject *const *args) {
    Args a(args);
    const Table t(a);
    const Tensor *start = a.tensor(2, at::kInt), *context = a.tensor(3, at::kInt);
    const int64_t page = a.integer(4);
    a.need(a.ok && start->numel() == t.b + 1 && context->numel() == t.b);
    if (!a.ok) return none();
    const int64_t need = args[5] == Py_None ? static_cast<int64_t>(dtts_claim_pages_workspace_bytes(t.b, t.max_pages, t.n_pages)) / 4 : 0;
    const Tensor *given = a.maybe(5, at::kByte);
    if (!a.ok) return none();
    Ints all(*t.pages, 2 * t.b + 1 + Ints::scratch_here(need));
    const Tensor src = all.of(t.b), dst = all.of(t.b), lacking = all.of(1), ws = given ? *given : all.scratch(need);
    const int status = dtts_claim_pages(data<int32_t>(t.pages), data<int32_t>(t.refs), data<int32_t>(start), data<int32_t>(context),
                                        data<int32_t>(&src), data<int32_t>(&dst), data<int32_t>(&lacking), t.b, page, t.max_pages,
                                        t.n_pages, ws.data_ptr(), ws.nbytes(), a.stream());
    return status == DTTS_OK ? tuple_of({src, dst, lacking}) : none();
}

// (pages, refs, context, page, window, sinks) -> True
PyObject *trim(PyObject *const *args) {
    Args a(args);
    const Table t(a);
    const Tensor *context = a.tensor(2, at::kInt);
    const int64_t page = a.integer(3), window = a.integer(4), sinks = a.integer(5);
    a.need(a.ok && context->numel() == t.b);
    if (!a.ok) return none();
    const int status = dtts_trim_pages(data<int32_t>(t.pages), data<int32_t>(t.refs), data<int32_t>(context), t.b, page, t.max_pages,
                                       t.n_pages, window, sinks, a.stream());
    if (status != DTTS_OK) return none();
    Py_RETURN_TRUE;
}

// (pages, refs, workspace) -> (src, dst, used)
PyObject *compact(PyObject *const *args) {
    Args a(args);
    const Table t(a);
    const Tensor *given = a.maybe(2, at::kByte);
    if (!a.ok) return none();
    const int64_t need = given ? 0 : static_cast<int64_t>(dtts_compact_pages_workspace_bytes(t.n_pages)) / 4;
    Ints all(*t.pages, 2 * t.n_pages + 1 + Ints::scratch_here(need));
    const Tensor src = all.of(t.n_pages), dst = all.of(t.n_pages), used = all.of(1), ws = given ? *given : all.scratch(need);
    const int status = dtts_compact_pages(data<int32_t>(t.pages), data<int32_t>(t.refs), data<int32_t>(&src), data<int32_t>(&dst),
                                          data<int32_t>(&used), t.b, t.max_pages, t.n_pages, ws.data_ptr(), ws.nbytes(), a.stream());
    return status == DTTS_OK ? tuple_of({src, dst, used}) : none();
}

// (caches, src, dst) -> True; caches a list or a tuple
PyObject *copy(PyObject *const *args) {
    Args a(args);
    const Tensor *src = a.tensor(1, at::kInt), *dst = a.tensor(2, at::kInt);
    a.need(a.ok && src->numel() == dst->numel() && (PyList_Check(args[0]) || PyTuple_Check(args[0])));
    if (!a.ok) return none();
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(args[0]);
    Args of(PySequence_Fast_ITEMS(args[0]));
    of.device = a.device;
    c10::SmallVector<void *, 8> at(n);
    c10::SmallVector<int64_t, 8> size(n), stride(n);
    int64_t n_pages = 0;
    for (Py_ssize_t i = 0; i < n; ++i) {
        const Tensor *t = of.tensor(static_cast<int>(i));
        if (!t || t->dim() < 2 || t->numel() == 0 || (i && t->size(0) != n_pages)) return none();
        n_pages = t->size(0);
        int64_t row = 1;  // contiguous pages; the stride of a size of 1 is no one's
        for (int64_t d = t->dim() - 1; d > 0; row *= t->size(d), --d)
            if (t->size(d) != 1 && t->stride(d) != row) return none();
        at[i] = t->data_ptr();
        size[i] = row * t->element_size();
        stride[i] = n_pages > 1 ? t->stride(0) * static_cast<int64_t>(t->element_size()) : size[i];
    }
    if (n > 0 && dtts_copy_pages(at.data(), size.data(), stride.data(), n, data<int32_t>(src), data<int32_t>(dst), src->numel(), n_pages,
                                 a.stream()) != DTTS_OK)
        return none();
    Py_RETURN_TRUE;
}

// No C++ exception leaves: where torch refuses an allocation, nothing is enqueued yet, and the Python path meets the
// same refusal.
template <PyObject *(*F)(PyObject *const *), int N, int OPTIONAL>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (n > N || n < N - OPTIONAL) {
        PyErr_Format(PyExc_TypeError, "%d arguments expected, got %zd", N, n);
        return nullptr;
    }
    PyObject *all[N];
    for (int i = 0; i < N; ++i) all[i] = i < n ? args[i] : Py_None;
    try {
        return F(all);
    } catch (...) {
        return none();
    }
}

template <PyObject *(*F)(PyObject *const *), int N, int OPTIONAL = 0>
PyMethodDef method(const char *name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(entry<F, N, OPTIONAL>)), METH_FASTCALL, nullptr};
}

PyMethodDef kMethods[] = {method<rotary, 6>("rotary"), method<append, 13>("qk_rope_append_paged"),
                          method<attention, 13, 1>("paged_attention"), method<sample, 7>("sample"),
                          method<unpack, 3>("unpack_pages"), method<fork, 5>("fork_pages"), method<claim, 6>("claim_pages"),
                          method<trim, 6>("trim_pages"), method<compact, 3>("compact_pages"), method<copy, 3>("copy_pages"),
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving(void) { return PyModule_Create(&kModule); }
