// Calls of mtpx.ops as one native step each (module mtpx._calls):
// tensors are looked at, a request filled and the library called without
// Python's steps between, which take longer than the kernels of small calls do
// (one row's queries and keys: 11.3 us a call through the checks in Python, 4.8 us
// so; its gradients: 19.8 and 9.7; appended: 13.0 and 4.1; attended: 13.7 and 7.2, its
// two kernels' own time).
//
// A call that is not plainly right -- another type, shape, device or kind of
// object -- returns None, and mtpx.ops goes through its own checks, which say
// what is wrong with it.  Otherwise a call returns its results, or the library's
// error code.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/python_cpp_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include "mtpx.h"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <exception>
#include <type_traits>

namespace {

struct Entries {
    decltype(&mtpx_head_norm_rotary) head_norm_rotary, head_norm_rotary_backward;
    decltype(&mtpx_head_norm_rotary_workspace) head_norm_rotary_workspace;
    decltype(&mtpx_append_paged) append_paged;
    decltype(&mtpx_diff_attention_paged) diff_attention_paged;
    decltype(&mtpx_diff_attention_paged_workspace) diff_attention_paged_workspace;
} entries;

int type_code(at::ScalarType t)
{
    switch (t) {
    case at::kFloat: return MTPX_F32;
    case at::kBFloat16: return MTPX_BF16;
    case at::kHalf: return MTPX_F16;
    case at::kDouble: return MTPX_F64;
    case at::kInt: return MTPX_I32;
    case at::kLong: return MTPX_I64;
    default: return -1;
    }
}

// A call's arguments and what they share; `good` as long as all are plainly right.
struct Call {
    PyObject *const *args;
    int64_t device;
    bool good = true;

    // Argument i as a tensor of so many dimensions on the device (NULL: not so).
    const at::Tensor *tensor(int i, int64_t dims)
    {
        if (good && THPVariable_Check(args[i])) {
            const at::Tensor &t = THPVariable_Unpack(args[i]);
            if (t.layout() == at::kStrided && t.is_cuda() && t.get_device() == device && t.dim() == dims)
                return &t;
        }
        good = false;
        return nullptr;
    }
    bool absent(int i) const { return args[i] == Py_None; }
    // The same of a type whose last dimension is contiguous.
    const at::Tensor *rows(int i, int64_t dims, at::ScalarType type)
    {
        const at::Tensor *t = tensor(i, dims);
        if (t && t->scalar_type() == type && (t->stride(dims - 1) == 1 || t->size(dims - 1) <= 1))
            return t;
        good = false;
        return nullptr;
    }
    void need(bool condition) { good = good && condition; }
    long integer(int i)
    {
        const long v = PyLong_Check(args[i]) ? PyLong_AsLong(args[i]) : -1;
        if (!PyLong_Check(args[i]) || (v == -1 && PyErr_Occurred())) {
            PyErr_Clear();
            good = false;
        }
        return v;
    }
    float real(int i)
    {
        const double v = PyFloat_Check(args[i]) ? PyFloat_AS_DOUBLE(args[i]) : INFINITY;
        need(std::fabs(v) <= FLT_MAX);
        return good ? (float)v : 0.f;
    }
    // torch's current stream on the device: argument 2 is what says so.
    void *stream()
    {
        PyObject *s = good ? PyObject_CallOneArg(args[2], args[1]) : nullptr;
        void *p = s ? PyLong_AsVoidPtr(s) : nullptr;
        Py_XDECREF(s);
        if (PyErr_Occurred()) {
            PyErr_Clear();
            good = false;
        }
        return p;
    }
    bool truth(int i)
    {
        need(PyBool_Check(args[i]));
        return args[i] == Py_True;
    }
};

// [rows][heads][(2)][dim]
mtpx_rows rows_of(const at::Tensor &t)
{
    const auto s = t.strides();
    return {t.data_ptr(), s[0], s[1], t.dim() == 4 ? s[2] : 0};
}
// [rows][heads][2 dim]
mtpx_rows values_of(const at::Tensor &t, int64_t dim)
{
    return {t.data_ptr(), t.stride(0), t.stride(1), dim};
}
at::Tensor like(const at::Tensor &t) { return at::empty(t.sizes(), t.options()); }

// positions, freq and axis from argument i on
template <class R>
void turn(Call &c, int i, R &r)
{
    const at::Tensor *p = c.tensor(i, 2), *f = c.rows(i + 1, 1, at::kFloat), *a = c.rows(i + 2, 1, at::kInt);
    if (!c.good)
        return;
    r.position_dtype = type_code(p->scalar_type());
    c.need(r.position_dtype == MTPX_F32 || r.position_dtype >= MTPX_F64);
    c.need(p->size(0) == r.rows && f->size(0) == a->size(0) && f->size(0) <= r.dim);
    r.positions = p->data_ptr();
    r.position_row = p->stride(0);
    r.position_axis = p->stride(1);
    r.axes = (int)p->size(1);
    r.rotated = 2 * (int)f->size(0);
    r.freq = (const float *)f->data_ptr();
    r.axis = (const int *)a->data_ptr();
}
const void *weight(Call &c, int i, int64_t dim, at::ScalarType type)
{
    if (c.absent(i))
        return nullptr;
    const at::Tensor *w = c.rows(i, 1, type);
    c.need(w && w->size(0) == dim);
    return c.good ? w->data_ptr() : nullptr;
}
// k_pages, v_pages from argument i on, table, offsets and lengths from argument j on
template <class R>
void pages(Call &c, int i, int j, int64_t kv, int64_t dim, at::ScalarType type, R &r)
{
    const at::Tensor *k = c.rows(i, 5, type), *v = c.rows(i + 1, 4, type);
    const at::Tensor *t = c.rows(j, 2, at::kInt), *o = c.rows(j + 1, 1, at::kInt), *l = c.rows(j + 2, 1, at::kInt);
    if (!c.good)
        return;
    const int64_t n = k->size(0), page = k->size(1), sequences = l->size(0);
    c.need(k->size(2) == kv && k->size(3) == 2 && k->size(4) == dim);
    c.need(v->size(0) == n && v->size(1) == page && v->size(2) == kv && v->size(3) == 2 * dim);
    c.need(t->size(0) == sequences && o->size(0) == sequences + 1);
    c.need(page <= INT32_MAX && sequences <= INT32_MAX && t->size(1) <= INT32_MAX);
    r.sequences = (int)sequences;
    r.offsets = (const int *)o->data_ptr();
    r.lengths = (const int *)l->data_ptr();
    r.cache.k = {k->data_ptr(), k->stride(1), k->stride(2), k->stride(3)};
    r.cache.v = {v->data_ptr(), v->stride(1), v->stride(2), dim};
    r.cache.k_page = k->stride(0);
    r.cache.v_page = v->stride(0);
    r.cache.pages = n;
    r.cache.page_rows = (int)page;
    r.cache.table = (const int *)t->data_ptr();
    r.cache.table_row = t->stride(0);
    r.cache.table_width = (int)t->size(1);
}

template <class F, class R>
int enter(F f, mtpx_context *context, const R &r)
{
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f(context, &r);
    Py_END_ALLOW_THREADS
    return rc;
}

// Arguments 0 and 1 are the context's handle and its device.  No C++
// exception leaves into Python: one (a tensor without memory of its own, memory
// that is used up) leaves the call to mtpx.ops, which meets its cause again.
template <class F>
PyObject *guarded(PyObject *const *args, Py_ssize_t given, Py_ssize_t wanted, const F &f)
{
    if (given != wanted)
        return PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd", given, wanted);
    if (!PyLong_Check(args[0]) || !PyLong_Check(args[1]))
        Py_RETURN_NONE;
    auto *const context = static_cast<mtpx_context *>(PyLong_AsVoidPtr(args[0]));
    Call call{args, PyLong_AsLong(args[1])};
    if (PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    try {
        return f(context, call);
    } catch (const std::exception &) {
        Py_RETURN_NONE;
    }
}

bool is_type(const at::Tensor &t) { return type_code(t.scalar_type()) >= 0 && type_code(t.scalar_type()) <= MTPX_F16; }

// q and k from argument i on, weights and rotation behind them, kind, eps and
// interleaved from argument j on
bool heads(Call &c, int i, int j, mtpx_head_norm_rotary_request &r, const at::Tensor *&q, const at::Tensor *&k)
{
    const int64_t dims = THPVariable_Check(c.args[i]) && THPVariable_Unpack(c.args[i]).dim() == 4 ? 4 : 3;
    q = c.tensor(i, dims);
    if (!q || !is_type(*q) || !c.rows(i, dims, q->scalar_type()))
        return false;
    const auto type = q->scalar_type();
    r.dtype = type_code(type);
    r.rows = q->size(0);
    r.maps = dims == 4 ? (int)q->size(2) : 1;
    r.dim = (int)q->size(dims - 1);
    r.heads = (int)q->size(1);
    c.need(q->size(1) <= INT32_MAX && q->size(dims - 1) <= INT32_MAX && (r.maps == 1 || r.maps == 2));
    r.q = rows_of(*q);
    if (!c.absent(i + 1)) {
        k = c.rows(i + 1, dims, type);
        if (!k)
            return false;
        c.need(k->size(0) == r.rows && k->size(1) > 0 && k->size(1) <= INT32_MAX && k->size(dims - 1) == r.dim);
        c.need(dims == 3 || k->size(2) == r.maps);
        r.kv_heads = (int)k->size(1);
        r.k = rows_of(*k);
    }
    turn(c, i + 4, r);
    r.q_weight = weight(c, i + 2, r.dim, type);
    r.k_weight = weight(c, i + 3, r.dim, type);
    r.kind = (int)c.integer(j);
    r.eps = c.real(j + 1);
    r.interleaved = c.truth(j + 2);
    r.stream = c.stream();
    return c.good;
}
PyObject *wrapped(const at::Tensor &t)
{
    if (t.defined())
        return THPVariable_Wrap(t);
    Py_RETURN_NONE;
}

// (context, device, stream, q, k, q_weight, k_weight, positions, freq, axis, kind, eps, interleaved): (q, k)
PyObject *head_norm_rotary(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return guarded(args, n, 13, [&](mtpx_context *context, Call &c) -> PyObject * {
        const at::Tensor *q = nullptr, *k = nullptr;
        mtpx_head_norm_rotary_request r{};
        if (!heads(c, 3, 10, r, q, k))
            Py_RETURN_NONE;
        const at::Tensor qo = like(*q);
        r.q_out = rows_of(qo);
        at::Tensor ko;
        if (k) {
            ko = like(*k);
            r.k_out = rows_of(ko);
        }
        const int rc = enter(entries.head_norm_rotary, context, r);
        return rc ? PyLong_FromLong(rc) : Py_BuildValue("NN", wrapped(qo), wrapped(ko));
    });
}

// (context, device, stream, dq, dk, q, k, q_weight, k_weight, positions, freq, axis, kind, eps, interleaved,
//  dpositions): (dq, dk, dq_weight, dk_weight, dpositions)
PyObject *head_norm_rotary_backward(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return guarded(args, n, 16, [&](mtpx_context *context, Call &c) -> PyObject * {
        const at::Tensor *q = nullptr, *k = nullptr;
        mtpx_head_norm_rotary_request r{};
        const bool moved = c.truth(15);
        if (!heads(c, 5, 12, r, q, k) || c.absent(4) != !k)
            Py_RETURN_NONE;
        const at::Tensor *dy = c.rows(3, q->dim(), q->scalar_type());
        if (!dy || dy->sizes() != q->sizes())
            Py_RETURN_NONE;
        r.dq_out = rows_of(*dy);
        const at::Tensor gq = like(*q);
        r.dq = rows_of(gq);
        at::Tensor gk, wq, wk, dpos;
        if (k) {
            const at::Tensor *dz = c.rows(4, k->dim(), k->scalar_type());
            if (!dz || dz->sizes() != k->sizes())
                Py_RETURN_NONE;
            r.dk_out = rows_of(*dz);
            gk = like(*k);
            r.dk = rows_of(gk);
        }
        if (r.q_weight) {
            wq = at::empty({r.dim}, q->options());
            r.dq_weight = wq.data_ptr();
        }
        if (r.k_weight) {
            wk = at::empty({r.dim}, q->options());
            r.dk_weight = wk.data_ptr();
        }
        if (moved) {
            dpos = like(THPVariable_Unpack(args[9]));
            r.dpositions = dpos.data_ptr();
        }
        int rc = entries.head_norm_rotary_workspace(context, &r, &r.workspace_bytes);
        if (rc)
            return PyLong_FromLong(rc);
        const at::Tensor work = at::empty({(int64_t)r.workspace_bytes}, q->options().dtype(at::kByte));
        r.workspace = work.data_ptr();  // held until the kernels are queued
        rc = enter(entries.head_norm_rotary_backward, context, r);
        return rc ? PyLong_FromLong(rc)
                  : Py_BuildValue("NNNNN", wrapped(gq), wrapped(gk), wrapped(wq), wrapped(wk), wrapped(dpos));
    });
}

// (context, device, stream, k, v, k_pages, v_pages, table, offsets, lengths, positions, freq, axis, q,
//  kind, q_weight, k_weight, eps, interleaved, out): the queries' result, () without queries
PyObject *append_paged(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return guarded(args, n, 20, [&](mtpx_context *context, Call &c) -> PyObject * {
        const at::Tensor *k = c.tensor(3, 4);
        if (!k || !is_type(*k) || !c.rows(3, 4, k->scalar_type()))
            Py_RETURN_NONE;
        const auto type = k->scalar_type();
        const at::Tensor *v = c.rows(4, 3, type), *q = nullptr;
        mtpx_append_paged_request r{};
        r.dtype = type_code(type);
        r.rows = k->size(0);
        r.kv_heads = (int)k->size(1);
        r.dim = (int)k->size(3);
        c.need(v && k->size(2) == 2 && k->size(1) <= INT32_MAX && k->size(3) <= INT32_MAX / 2);
        c.need(c.good && v->size(0) == r.rows && v->size(1) == r.kv_heads && v->size(2) == 2 * r.dim);
        pages(c, 5, 7, r.kv_heads, r.dim, type, r);
        turn(c, 10, r);
        r.kind = (int)c.integer(14);
        r.q_weight = weight(c, 15, r.dim, type);
        r.k_weight = weight(c, 16, r.dim, type);
        c.need(r.kind != MTPX_NORM_NONE || (!r.q_weight && !r.k_weight));
        r.eps = c.real(17);
        r.interleaved = c.truth(18);
        at::Tensor out;
        if (!c.absent(13)) {
            q = c.rows(13, 4, type);
            c.need(q && q->size(0) == r.rows && q->size(2) == 2 && q->size(3) == r.dim && q->size(1) <= INT32_MAX);
            if (!c.good)
                Py_RETURN_NONE;
            r.heads = (int)q->size(1);
            r.q = rows_of(*q);
            if (c.absent(19)) {
                out = like(*q);
            } else {
                const at::Tensor *o = c.rows(19, 4, type);
                if (!o || o->sizes() != q->sizes())
                    Py_RETURN_NONE;
                out = *o;
            }
            r.q_out = rows_of(out);
        } else {
            c.need(c.absent(19));
        }
        r.stream = c.stream();
        if (!c.good)
            Py_RETURN_NONE;
        r.k = rows_of(*k);
        r.v = values_of(*v, r.dim);
        const int rc = enter(entries.append_paged, context, r);
        if (rc)
            return PyLong_FromLong(rc);
        return q ? THPVariable_Wrap(out) : PyTuple_New(0);
    });
}

// (context, device, stream, q, k_pages, v_pages, lam, table, offsets, lengths, causal, scale, max_rows, out)
PyObject *diff_attention_paged(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return guarded(args, n, 14, [&](mtpx_context *context, Call &c) -> PyObject * {
        const at::Tensor *q = c.tensor(3, 4), *k = c.tensor(4, 5);
        if (!c.good || !is_type(*q) || !c.rows(3, 4, q->scalar_type()))
            Py_RETURN_NONE;
        const auto type = q->scalar_type();
        const at::Tensor *lambda = c.rows(6, 1, at::kFloat);
        mtpx_diff_attention_paged_request r{};
        r.dtype = type_code(type);
        r.rows = q->size(0);
        r.heads = (int)q->size(1);
        r.kv_heads = (int)k->size(2);
        r.dim = (int)q->size(3);
        c.need(lambda && q->size(2) == 2 && q->size(1) <= INT32_MAX && k->size(2) <= INT32_MAX && q->size(3) <= INT32_MAX / 2);
        pages(c, 4, 7, r.kv_heads, r.dim, type, r);
        c.need(c.good && lambda->size(0) == r.heads);
        r.causal = c.truth(10);
        r.scale = c.absent(11) ? (float)std::pow((double)r.dim, -0.5) : c.real(11);
        if (!c.absent(12)) {
            const long most = c.integer(12);
            c.need(most >= 1);
            r.max_rows = (int)std::min<int64_t>(most, std::max<int64_t>(r.rows, 1));
        }
        c.need(r.rows <= INT32_MAX);
        r.stream = c.stream();
        if (!c.good)
            Py_RETURN_NONE;
        at::Tensor out, work;
        if (c.absent(13)) {
            out = at::empty({r.rows, r.heads, 2 * (int64_t)r.dim}, q->options());
        } else {
            const at::Tensor *o = c.rows(13, 3, type);
            if (!o || o->size(0) != r.rows || o->size(1) != r.heads || o->size(2) != 2 * (int64_t)r.dim)
                Py_RETURN_NONE;
            out = *o;
        }
        r.lambda = (const float *)lambda->data_ptr();
        r.q = rows_of(*q);
        r.out = values_of(out, r.dim);
        int rc = entries.diff_attention_paged_workspace(context, &r, &r.workspace_bytes);
        if (rc)
            return PyLong_FromLong(rc);
        if (r.workspace_bytes) {  // held until the kernels are queued
            work = at::empty({(int64_t)r.workspace_bytes}, q->options().dtype(at::kByte));
            r.workspace = work.data_ptr();
        }
        rc = enter(entries.diff_attention_paged, context, r);
        return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
    });
}

// The stream that was current when a graph's end at a leaf was made: (id, index and
// type of its device), None of anything else.
PyObject *stream_of(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    if (n != 1)
        return PyErr_Format(PyExc_TypeError, "%zd arguments, not 1", n);
    try {
        if (torch::autograd::THPCppFunction_Check(args[0]))
            if (const auto s = reinterpret_cast<torch::autograd::THPCppFunction *>(args[0])->cdata->stream())
                return Py_BuildValue("Lii", (long long)s->id(), (int)s->device_index(), (int)s->device_type());
    } catch (const std::exception &) {
    }
    Py_RETURN_NONE;
}

// The addresses of the library's entries, in the order of Entries.
PyObject *setup(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    constexpr int kEntries = 6;
    if (n != kEntries)
        return PyErr_Format(PyExc_TypeError, "%d addresses", kEntries);
    void *p[kEntries];
    for (int i = 0; i < kEntries; ++i)
        if (!(p[i] = PyLong_AsVoidPtr(args[i])))
            return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "a null address");
    int i = 0;
    auto take = [&](auto &entry) { entry = reinterpret_cast<std::decay_t<decltype(entry)>>(p[i++]); };
    take(entries.head_norm_rotary);
    take(entries.head_norm_rotary_backward);
    take(entries.head_norm_rotary_workspace);
    take(entries.append_paged);
    take(entries.diff_attention_paged);
    take(entries.diff_attention_paged_workspace);
    Py_RETURN_NONE;
}

#define MTPX_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {MTPX_METHOD(setup), MTPX_METHOD(head_norm_rotary), MTPX_METHOD(head_norm_rotary_backward),
                         MTPX_METHOD(append_paged), MTPX_METHOD(diff_attention_paged), MTPX_METHOD(stream_of), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "mtpx._calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&module); }
