// Host side of the calls that are short on the GPU: arguments checked, results allocated and the library's C entries called in one
// step.  From Python the same checks are some forty interpreted operations, 6 us beside a kernel of 6 us, and those of an
// optimizer step over hundreds of tensors some ten for each tensor.
//
// A Python extension (`image_generator_amd/_host.so`); the entries it calls are handed over by bind(), from the library that the
// process has loaded.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <cmath>
#include <cstdarg>
#include <string>
#include "../../include/mi355_denoiser.h"

namespace {

#define ENTRIES(X)                                                                                                     \
    X(mi355_doc_attention_fwd_workspace_bytes) X(mi355_doc_attention_fwd) X(mi355_doc_attention_bwd_workspace_bytes)   \
    X(mi355_doc_attention_bwd) X(mi355_embedding_fwd) X(mi355_embedding_bwd_workspace_bytes) X(mi355_embedding_bwd)
struct {
#define X(name) decltype(&::name) name = nullptr;
    ENTRIES(X)
#undef X
} lib;
PyObject* check_fn = nullptr;        // (return code, what) -> raises

struct Raise {                       // thrown inside, turned into a Python error at the entry
    PyObject* type;
    std::string text;
};
__attribute__((noreturn, format(printf, 2, 3))) void raise(PyObject* type, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    throw Raise{type, buf};
}
struct Failed {};                    // a Python error is set already

template <typename F>
PyObject* guarded(F f) {
    try {
        return f();
    } catch (const Failed&) {
    } catch (const Raise& e) {
        PyErr_SetString(e.type, e.text.c_str());
    } catch (...) {                  // torch's own, out of memory among them
        torch::translate_exception_to_python(std::current_exception());
    }
    return nullptr;
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) raise(PyExc_TypeError, "%s must be a tensor, not %s", name, Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}
const at::Tensor* maybe(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }
long long whole(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Failed{};
    return v;
}
// sizes and heads reach the library as int
int whole32(PyObject* o, const char* name) {
    const long long v = whole(o);
    if (v > 0x7fffffff || v < -0x7fffffff) raise(PyExc_ValueError, "%s %lld", name, v);
    return (int)v;
}
double real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Failed{};
    return v;
}
bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Failed{};
    return v != 0;
}
int as_int(int64_t n, const char* what) {
    if (n > 0x7fffffff) raise(PyExc_ValueError, "%s: 2^31 or more", what);
    return (int)n;
}
void checked(int rc, const char* what) {
    if (rc == 0) return;
    PyObject* r = PyObject_CallFunction(check_fn, "is", rc, what);
    Py_XDECREF(r);
    if (r) raise(PyExc_RuntimeError, "%s failed (%d)", what, rc);
    throw Failed{};
}
template <typename F>
int without_gil(F f) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f();
    Py_END_ALLOW_THREADS
    return rc;
}
void* address(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }

// operands of one launch: all on the current device (a launch goes to its stream)
void here(std::initializer_list<const at::Tensor*> all, int current) {
    const at::Tensor& first = **all.begin();
    for (const at::Tensor* t : all)
        if (t && t->device() != first.device())
            raise(PyExc_RuntimeError, "tensors on %s and %s; HIP device tensors required (no CPU path)", first.device().str().c_str(), t->device().str().c_str());
    if (!first.is_cuda()) raise(PyExc_RuntimeError, "HIP device tensors required (no CPU path)");
    if (first.get_device() != current) raise(PyExc_RuntimeError, "tensors on %s, the current device is %d", first.device().str().c_str(), current);
}

bool adjacent(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 && t.dim() == 2 && (t.stride(1) == 1 || t.size(1) <= 1 || t.size(0) == 0); }
// the stride between the rows of one row is whatever made the tensor (a transposed column, say) and is not looked at
long long row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

std::string shape(const at::Tensor& t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + ")";
}

// ---- document attention ----------------------------------------------------------------------------------------------------
struct Docs {
    const at::Tensor *q, *k, *v, *q_off, *k_off, *prefix, *slopes;
    int heads, kv_heads, width, docs, Tq, Tk;
    bool causal, start;
    float cap, scale, drop_p;
    unsigned seed;
};

void matrix(const char* name, const at::Tensor& t, int heads, int64_t width) {
    if (!adjacent(t)) raise(PyExc_RuntimeError, "doc_attention: %s must be a bf16 matrix [tokens, heads * width] with adjacent columns", name);
    if (t.size(1) != heads * width) raise(PyExc_ValueError, "doc_attention: %s %s for %d heads of width %lld", name, shape(t).c_str(), heads, (long long)width);
}
void values(const char* name, const at::Tensor* t, int64_t n, at::ScalarType type) {
    if (t && (t->numel() != n || t->scalar_type() != type || !t->is_contiguous()))
        raise(PyExc_ValueError, "doc_attention: %s must be %lld contiguous %s values, got %lld %s", name, (long long)n, c10::toString(type), (long long)t->numel(),
              c10::toString(t->scalar_type()));
}

// q, k, v, heads, q_offsets, k_offsets, kv_heads, causal, prefix, slopes, cap, scale, align, drop_p, seed
constexpr int DOC_ARGS = 15;
Docs docs_of(PyObject* const* a, int current) {
    Docs d;
    d.q = &tensor(a[0], "q");
    d.k = &tensor(a[1], "k");
    d.v = &tensor(a[2], "v");
    d.heads = whole32(a[3], "heads");
    d.q_off = &tensor(a[4], "q_offsets");
    d.k_off = a[5] == Py_None ? d.q_off : &tensor(a[5], "k_offsets");
    d.kv_heads = a[6] == Py_None ? d.heads : whole32(a[6], "kv_heads");
    d.causal = truth(a[7]);
    d.prefix = maybe(a[8], "prefix");
    d.slopes = maybe(a[9], "slopes");
    here({d.q, d.k, d.v, d.q_off, d.k_off, d.prefix, d.slopes}, current);
    if (d.heads < 1 || d.kv_heads < 1 || d.heads % d.kv_heads) raise(PyExc_ValueError, "doc_attention: %d query heads on %d key heads", d.heads, d.kv_heads);
    const int64_t width = d.q->dim() ? d.q->size(-1) / d.heads : 0;
    matrix("q", *d.q, d.heads, width);
    matrix("k", *d.k, d.kv_heads, width);
    matrix("v", *d.v, d.kv_heads, width);
    if (d.k->size(0) != d.v->size(0)) raise(PyExc_ValueError, "doc_attention: %lld keys, %lld values", (long long)d.k->size(0), (long long)d.v->size(0));
    const int64_t docs = d.q_off->numel() - 1;
    if (docs < 1) raise(PyExc_ValueError, "doc_attention: offsets hold at least two entries");
    values("q_offsets", d.q_off, docs + 1, at::kInt);
    if (d.k_off != d.q_off) values("k_offsets", d.k_off, docs + 1, at::kInt);
    values("prefix", d.prefix, docs, at::kInt);
    values("slopes", d.slopes, d.heads, at::kFloat);
    if (d.slopes && d.slopes->requires_grad() && c10::GradMode::is_enabled())
        raise(PyExc_RuntimeError, "doc_attention: no gradient reaches the slopes (detach them)");
    const char* align = PyUnicode_Check(a[12]) ? PyUnicode_AsUTF8(a[12]) : "";
    if (!align) throw Failed{};
    d.start = !strcmp(align, "start");
    if (!d.start && strcmp(align, "end")) raise(PyExc_ValueError, "doc_attention: align '%s' is neither 'end' nor 'start'", align);
    d.cap = a[10] == Py_None ? 0.f : (float)real(a[10]);
    d.scale = a[11] == Py_None ? (float)std::pow((double)width, -0.5) : (float)real(a[11]);
    d.drop_p = (float)real(a[13]);
    d.seed = (unsigned)PyLong_AsUnsignedLongLongMask(a[14]);
    if (PyErr_Occurred()) throw Failed{};
    d.width = as_int(width, "doc_attention: head width");
    d.docs = as_int(docs, "doc_attention: documents");
    d.Tq = as_int(d.q->size(0), "doc_attention: queries");
    d.Tk = as_int(d.k->size(0), "doc_attention: keys");
    return d;
}

// doc_attention_fwd(DOC_ARGS..., current device, stream) -> (out, lse)
PyObject* doc_attention_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != DOC_ARGS + 2) raise(PyExc_TypeError, "doc_attention_fwd: %zd arguments", n);
        const Docs d = docs_of(a, whole32(a[DOC_ARGS], "device"));
        void* stream = (void*)whole(a[DOC_ARGS + 1]);
        at::Tensor out = at::empty(d.q->sizes(), d.q->options()), lse = at::empty({d.heads, d.Tq}, d.q->options().dtype(at::kFloat)), ws;
        const size_t need = lib.mi355_doc_attention_fwd_workspace_bytes(d.Tq, d.Tk, d.heads, d.kv_heads, d.width, d.docs);
        if (need) ws = at::empty({(int64_t)need}, d.q->options().dtype(at::kByte));
        checked(without_gil([&] {
            return lib.mi355_doc_attention_fwd(d.q->data_ptr(), d.k->data_ptr(), d.v->data_ptr(), out.data_ptr(), (float*)lse.data_ptr(),
                                               (const int*)d.q_off->data_ptr(), (const int*)d.k_off->data_ptr(), d.docs, (const int*)address(d.prefix),
                                               (const float*)address(d.slopes), d.cap, d.causal, d.start, d.Tq, d.Tk, d.heads, d.kv_heads, d.width,
                                               row_stride(*d.q), row_stride(*d.k), row_stride(*d.v), row_stride(out), d.scale, d.drop_p, d.seed,
                                               need ? ws.data_ptr() : nullptr, need, stream);
        }), "doc_attention_fwd");
        PyObject* r = PyTuple_New(2);
        if (!r) throw Failed{};
        PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(out)));
        PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(lse)));
        return r;
    });
}

// doc_attention_bwd(DOC_ARGS..., do, o, lse, dq, dk, dv, current device, stream) -> (dq, dk, dv)
PyObject* doc_attention_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != DOC_ARGS + 8) raise(PyExc_TypeError, "doc_attention_bwd: %zd arguments", n);
        PyObject* const* b = a + DOC_ARGS;
        const int current = whole32(b[6], "device");
        const Docs d = docs_of(a, current);
        const at::Tensor &dout = tensor(b[0], "do"), &o = tensor(b[1], "o"), &lse = tensor(b[2], "lse");
        const at::Tensor *to[3], *like[3] = {d.q, d.k, d.v};
        at::Tensor made[3];
        const char* names[3] = {"dq", "dk", "dv"};
        for (int i = 0; i < 3; ++i) to[i] = maybe(b[3 + i], names[i]);
        here({d.q, &dout, &o, &lse, to[0], to[1], to[2]}, current);
        for (int i = 0; i < 3; ++i)
            if (!to[i]) {
                made[i] = at::empty(like[i]->sizes(), like[i]->options());
                to[i] = &made[i];
            }
        auto same = [](const char* name, const at::Tensor& t, const at::Tensor& as) {
            if (!adjacent(t) || t.sizes() != as.sizes())
                raise(PyExc_RuntimeError, "doc_attention_bwd: %s must be a bf16 matrix %s with adjacent columns", name, shape(as).c_str());
        };
        same("do", dout, *d.q);
        same("o", o, *d.q);
        for (int i = 0; i < 3; ++i) same(names[i], *to[i], *like[i]);
        for (int i = 0; i < 3; ++i) {
            if (to[i]->numel() == 0) continue;
            const void* at = to[i]->data_ptr();
            bool taken = at == d.q->data_ptr() || at == d.k->data_ptr() || at == d.v->data_ptr() || at == o.data_ptr() || at == dout.data_ptr();
            for (int j = 0; j < i; ++j) taken = taken || (to[j]->numel() && at == to[j]->data_ptr());
            if (taken) raise(PyExc_ValueError, "doc_attention_bwd: a gradient in the place of an operand or of another gradient");
        }
        if (lse.dim() != 2 || lse.size(0) != d.heads || lse.size(1) != d.Tq || lse.scalar_type() != at::kFloat || !lse.is_contiguous())
            raise(PyExc_RuntimeError, "doc_attention_bwd: lse is not the forward pass's");
        const size_t need = lib.mi355_doc_attention_bwd_workspace_bytes(d.Tq, d.Tk, d.heads, d.kv_heads, d.width, d.docs, d.causal);
        const at::Tensor ws = at::empty({(int64_t)need}, d.q->options().dtype(at::kByte));
        void* stream = (void*)whole(b[7]);
        checked(without_gil([&] {
            return lib.mi355_doc_attention_bwd(d.q->data_ptr(), d.k->data_ptr(), d.v->data_ptr(), o.data_ptr(), dout.data_ptr(), (const float*)lse.data_ptr(),
                                               to[0]->data_ptr(), to[1]->data_ptr(), to[2]->data_ptr(), (const int*)d.q_off->data_ptr(),
                                               (const int*)d.k_off->data_ptr(), d.docs, (const int*)address(d.prefix), (const float*)address(d.slopes), d.cap,
                                               d.causal, d.start, d.Tq, d.Tk, d.heads, d.kv_heads, d.width, row_stride(*d.q), row_stride(*d.k),
                                               row_stride(*d.v), row_stride(o), row_stride(dout), row_stride(*to[0]), row_stride(*to[1]),
                                               row_stride(*to[2]), d.scale, d.drop_p, d.seed, ws.data_ptr(), need, stream);
        }), "doc_attention_bwd");
        PyObject* r = PyTuple_New(3);
        if (!r) throw Failed{};
        for (int i = 0; i < 3; ++i) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(*to[i]));
        return r;
    });
}

// ---- embedding -------------------------------------------------------------------------------------------------------------
bool ids64(const at::Tensor& ids) {
    if (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong) raise(PyExc_RuntimeError, "embedding: ids must be int32 or int64, got %s", c10::toString(ids.scalar_type()));
    return ids.scalar_type() == at::kLong;
}
bool is_float(const at::Tensor& t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16; }

// embedding_fwd(ids, table, scale, bf16 result, current device, stream)
PyObject* embedding_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 6) raise(PyExc_TypeError, "embedding_fwd: %zd arguments", n);
        const at::Tensor &given = tensor(a[0], "ids"), &table = tensor(a[1], "table");
        here({&table, &given}, whole32(a[4], "device"));
        if (table.dim() != 2 || !is_float(table) || !table.is_contiguous()) raise(PyExc_RuntimeError, "embedding: the table must be a contiguous fp32 or bf16 matrix");
        const bool wide = ids64(given), out16 = truth(a[3]);
        const at::Tensor ids = given.contiguous();
        const float scale = (float)real(a[2]);
        const int width = as_int(table.size(1), "embedding: columns");
        void* stream = (void*)whole(a[5]);
        c10::SmallVector<int64_t, 5> sizes(ids.sizes().begin(), ids.sizes().end());
        sizes.push_back(width);
        at::Tensor out = at::empty(sizes, table.options().dtype(out16 ? at::kBFloat16 : at::kFloat));
        checked(without_gil([&] {
            return lib.mi355_embedding_fwd(ids.data_ptr(), wide, ids.numel(), table.data_ptr(), table.scalar_type() == at::kBFloat16, table.size(0), width, scale,
                                           out.data_ptr(), out16, stream);
        }), "embedding_fwd");
        return THPVariable_Wrap(std::move(out));
    });
}

// embedding_bwd(ids, dy, rows, scale, bf16 result, current device, stream)
PyObject* embedding_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 7) raise(PyExc_TypeError, "embedding_bwd: %zd arguments", n);
        const at::Tensor &given = tensor(a[0], "ids"), &dgiven = tensor(a[1], "dy");
        here({&dgiven, &given}, whole32(a[5], "device"));
        if (!is_float(dgiven)) raise(PyExc_RuntimeError, "embedding_bwd: gradients are fp32 or bf16");
        if (dgiven.dim() != given.dim() + 1 || dgiven.sizes().slice(0, given.dim()) != given.sizes())
            raise(PyExc_RuntimeError, "embedding_bwd: gradient %s of ids %s", shape(dgiven).c_str(), shape(given).c_str());
        const bool wide = ids64(given), out16 = truth(a[4]);
        const at::Tensor ids = given.contiguous(), dy = dgiven.contiguous();
        const long long rows = whole(a[2]);
        const float scale = (float)real(a[3]);
        const int width = as_int(dy.size(-1), "embedding: columns");
        void* stream = (void*)whole(a[6]);
        const size_t need = lib.mi355_embedding_bwd_workspace_bytes(ids.numel(), rows, width);
        const at::Tensor ws = at::empty({(int64_t)need}, dy.options().dtype(at::kByte));
        at::Tensor out = at::empty({rows, width}, dy.options().dtype(out16 ? at::kBFloat16 : at::kFloat));
        checked(without_gil([&] {
            return lib.mi355_embedding_bwd(ids.data_ptr(), wide, ids.numel(), dy.data_ptr(), dy.scalar_type() == at::kBFloat16, rows, width, scale, out.data_ptr(),
                                           out16, ws.data_ptr(), need, stream);
        }), "embedding_bwd");
        return THPVariable_Wrap(std::move(out));
    });
}

// ---- lists of tensors ------------------------------------------------------------------------------------------------------
PyObject** items(PyObject* list, Py_ssize_t& n) {
    if (!PyList_Check(list)) raise(PyExc_TypeError, "a list is expected, not %s", Py_TYPE(list)->tp_name);
    n = PyList_GET_SIZE(list);
    return ((PyListObject*)list)->ob_item;
}

// gradient_words(gradients, parameters, device, address of int64[n], address of int64[n] or nothing): what the device table holds for
// each gradient - its address, the lowest bit set for bf16, 0 for None - and -1, or the index of the first that is no contiguous
// fp32 or bf16 tensor of its parameter's shape on the device.  The second array: the parameters' sizes as the device knows them; one
// that has another by now raises.
PyObject* gradient_words(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 4 && n != 5) raise(PyExc_TypeError, "gradient_words: %zd arguments", n);
        Py_ssize_t count, others;
        PyObject** g = items(a[0], count);
        PyObject** p = items(a[1], others);
        if (count != others) raise(PyExc_ValueError, "gradient_words: %zd gradients of %zd parameters", count, others);
        const int device = whole32(a[2], "device");
        long long* to = (long long*)whole(a[3]);
        const long long* sizes = n == 5 ? (const long long*)whole(a[4]) : nullptr;
        for (Py_ssize_t i = 0; i < count; ++i) {
            if (g[i] == Py_None) { to[i] = 0; continue; }
            const at::Tensor &t = tensor(g[i], "a gradient"), &like = tensor(p[i], "a parameter");
            if (sizes && like.numel() != sizes[i])
                raise(PyExc_ValueError, "TensorAdamW: parameter %zd has become %lld elements, its states are of %lld", i, (long long)like.numel(), sizes[i]);
            if (!t.is_cuda() || t.get_device() != device || !is_float(t) || t.sizes() != like.sizes() || !t.is_contiguous()) return PyLong_FromSsize_t(i);
            to[i] = (long long)t.data_ptr() | (t.scalar_type() == at::kBFloat16);
        }
        return PyLong_FromLong(-1);
    });
}

// places(tensors, address of int64[n], keep): their addresses written there (keep), or whether one differs from what stands there
PyObject* places(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 3) raise(PyExc_TypeError, "places: %zd arguments", n);
        Py_ssize_t count;
        PyObject** t = items(a[0], count);
        long long* at = (long long*)whole(a[1]);
        const bool keep = truth(a[2]);
        for (Py_ssize_t i = 0; i < count; ++i) {
            const long long here = (long long)tensor(t[i], "an entry").data_ptr();
            if (keep) at[i] = here;
            else if (at[i] != here) Py_RETURN_TRUE;
        }
        Py_RETURN_FALSE;
    });
}

// bump(tensors): their versions, behind a kernel that wrote them
PyObject* bump(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 1) raise(PyExc_TypeError, "bump: %zd arguments", n);
        Py_ssize_t count;
        PyObject** t = items(a[0], count);
        for (Py_ssize_t i = 0; i < count; ++i) {
            const at::Tensor& x = tensor(t[i], "an entry");
            if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
        }
        Py_RETURN_NONE;
    });
}

// bind({entry: address}, check)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 2 || !PyDict_Check(a[0])) raise(PyExc_TypeError, "bind: {entry: address}, check");
        auto entry = [&](const char* name) {
            PyObject* v = PyDict_GetItemString(a[0], name);
            if (!v) raise(PyExc_KeyError, "%s", name);
            return (void*)whole(v);
        };
#define X(name) lib.name = (decltype(lib.name))entry(#name);
        ENTRIES(X)
#undef X
        Py_INCREF(a[1]);
        Py_XDECREF(check_fn);
        check_fn = a[1];
        Py_RETURN_NONE;
    });
}

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind), METHOD(doc_attention_fwd), METHOD(doc_attention_bwd), METHOD(embedding_fwd), METHOD(embedding_bwd),
                         METHOD(gradient_words), METHOD(places), METHOD(bump), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
