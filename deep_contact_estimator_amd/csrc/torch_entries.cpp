// torch_entries.cpp -- ops.py's entries on torch tensors: their checks, their results, one call of libdce's C ABI each (include/dce.h: dce_quantize,
// dce_matmul, dce_group_rows, dce_decide).  A CPython extension module: the smallest of these products take the GPU 4 us, which checks and allocations
// in Python took twice over (9.5 us a call for one row of 2048 x 4736; 5.7 here).  The library's functions come by address (bind): it is bound to the
// process's HIP runtime by _lib.py and not linked here.
#include <Python.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>

#include "../../include/dce.h"

#include <cstdarg>
#include <string>

namespace {

decltype(&dce_quantize) f_quantize;
decltype(&dce_matmul) f_matmul;
decltype(&dce_group_rows) f_group_rows;
decltype(&dce_group_rows_work) f_group_rows_work;
decltype(&dce_decide) f_decide;
decltype(&dce_last_error) f_last_error;
PyObject *raw_stream, *dce_error;

struct Refused {};                                              // the Python error is set

[[noreturn]] void refuse(const char* fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    PyErr_FormatV(PyExc_RuntimeError, fmt, ap);
    va_end(ap);
    throw Refused{};
}

std::string text(at::IntArrayRef s)
{
    std::string t = "(";
    for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
    return t + (s.size() == 1 ? ",)" : ")");
}

// a tensor argument; None: an undefined tensor.  What the kernels read is a tensor's memory, so a view that stands for the negative of its memory is made
// into what it stands for; written to, it would hold the negative of the result.
at::Tensor tensor(PyObject* o, const char* what, bool written = false)
{
    if (o == Py_None) return {};
    if (!THPVariable_Check(o)) refuse("%s: expected a tensor, got %s", what, Py_TYPE(o)->tp_name);
    at::Tensor t = THPVariable_Unpack(o);
    if (!t.is_neg()) return t;
    if (written) refuse("%s: out and out_scale cannot be views that stand for the negative of their memory", what);
    return t.resolve_neg();
}

int device_of(const at::Tensor& t, const char* what)
{
    if (!t.defined()) refuse("%s: expected a tensor, got None", what);
    if (!t.is_cuda()) refuse("%s: deep_contact_estimator_amd runs on MI355X only; there is no CPU path (got a tensor on %s)", what, t.device().str().c_str());
    return t.get_device();
}

void same(int dev, const char* what, std::initializer_list<const at::Tensor*> all)
{
    const bool grad = at::GradMode::is_enabled(), forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
    for (const at::Tensor* t : all) {
        if (!t->defined()) continue;
        if (!t->is_cuda() || t->get_device() != dev) refuse("%s: tensors on cuda:%d and on %s", what, dev, t->device().str().c_str());
        if (grad && t->requires_grad()) refuse("%s: deep_contact_estimator_amd implements the inference path only: detach the tensor, or call under torch.no_grad()", what);
        if (forward && t->_fw_grad(0).defined()) refuse("%s: deep_contact_estimator_amd implements the inference path only: this tensor has a tangent, which the result would lose; unpack the dual tensor", what);
    }
}

void* stream_of(int dev)
{
    PyObject* i = PyLong_FromLong(dev);
    PyObject* s = i ? PyObject_CallOneArg(raw_stream, i) : nullptr;
    Py_XDECREF(i);
    if (!s) throw Refused{};
    void* p = PyLong_AsVoidPtr(s);
    Py_DECREF(s);
    if (!p && PyErr_Occurred()) throw Refused{};
    return p;
}

void check(int64_t rc)
{
    if (rc >= 0) return;
    const char* m = f_last_error(nullptr);
    PyErr_Format(dce_error, "libdce error %d: %s", (int)rc, m ? m : "?");
    throw Refused{};
}

// the row stride of a tensor's last two axes, made contiguous where rows overlap or have gaps between their values (an axis of one entry: its stride
// says nothing)
int64_t rows_of(at::Tensor& t)
{
    const int64_t d = t.dim(), n = t.size(d - 1), m = t.size(d - 2);
    if ((n > 1 && t.stride(d - 1) != 1) || (m > 1 && t.stride(d - 2) < n)) t = t.contiguous();
    return m > 1 ? t.stride(d - 2) : n > 1 ? n : 1;
}

bool scale_code(at::ScalarType t, int32_t& code)
{
    code = t == at::kFloat ? DCE_SCALE_F32 : DCE_SCALE_E8M0;
    return t == at::kFloat || t == at::kFloat8_e8m0fnu;
}

PyObject* pair(at::Tensor a, at::Tensor b)
{
    PyObject* x = THPVariable_Wrap(std::move(a));
    PyObject* y = x ? THPVariable_Wrap(std::move(b)) : nullptr;
    PyObject* t = y ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return t;
}

// ---- quantize(x, rows, e8m0)
PyObject* quantize(PyObject* const* a)
{
    at::Tensor x = tensor(a[0], "quantize");
    const long rows = PyLong_AsLong(a[1]);
    if (rows == -1 && PyErr_Occurred()) throw Refused{};
    const bool e8 = a[2] == Py_True;
    if (!x.defined() || (x.scalar_type() != at::kFloat && x.scalar_type() != at::kBFloat16))
        refuse("quantize: x must be float32 or bfloat16, not %s", x.defined() ? c10::toString(x.scalar_type()) : "None");
    if (rows != 1 && rows != DCE_BLOCK) refuse("quantize: a block has 1 row or %d, not %ld", DCE_BLOCK, rows);
    const int64_t dims = x.dim();
    if (dims != 2 && (rows == 1 || dims != 3)) refuse("quantize: expected (m, k)%s, got %s", rows == 1 ? "" : " or (groups, n, k)", text(x.sizes()).c_str());
    const int dev = device_of(x, "quantize");
    same(dev, "quantize", {&x});
    dce_quantize_desc d{};
    d.ldx = rows_of(x);
    const int64_t m = x.size(-2), k = x.size(-1), kb = (k + 127) / 128, mb = (m + 127) / 128;
    at::Tensor q = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
    const auto so = x.options().dtype(e8 ? at::kFloat8_e8m0fnu : at::kFloat);
    at::Tensor s = rows == 1 ? at::empty({kb, m}, so) : dims == 3 ? at::empty({x.size(0), mb, kb}, so) : at::empty({mb, kb}, so);
    d.x = x.data_ptr(); d.x_batch = dims == 3 ? x.stride(0) : 0;
    d.q = static_cast<uint8_t*>(q.data_ptr()); d.ldq = k; d.q_batch = m * k;
    d.scale = s.data_ptr(); d.ld_scale = m;
    d.batch = dims == 3 ? x.size(0) : 1; d.rows = m; d.k = k;
    d.x_type = x.scalar_type() == at::kFloat ? DCE_TYPE_F32 : DCE_TYPE_BF16;
    d.scale_type = e8 ? DCE_SCALE_E8M0 : DCE_SCALE_F32;
    d.block_rows = (int32_t)rows;
    check(f_quantize(dev, stream_of(dev), &d));
    return pair(std::move(q), std::move(s));
}

// ---- matmul(what, a, a_scale, b, b_scale, bias, relu, out type, out, out_scale, offsets, index)
PyObject* matmul(PyObject* const* arg)
{
    const char* what = PyUnicode_AsUTF8(arg[0]);
    if (!what) throw Refused{};
    at::Tensor a = tensor(arg[1], what), as = tensor(arg[2], what), b = tensor(arg[3], what), bs = tensor(arg[4], what), bias = tensor(arg[5], what), out = tensor(arg[8], what, true),
               outs = tensor(arg[9], what, true), offsets = tensor(arg[10], what), index = tensor(arg[11], what);
    const int relu = PyObject_IsTrue(arg[6]);
    const long out_type = PyLong_AsLong(arg[7]);
    if (relu < 0 || (out_type == -1 && PyErr_Occurred())) throw Refused{};
    if (!a.defined() || !b.defined()) refuse("%s: expected tensors a and b", what);
    const auto kind = a.scalar_type();
    const bool f8 = kind == at::kFloat8_e4m3fn, grouped = offsets.defined();
    if (b.scalar_type() != kind || !(f8 || kind == at::kBFloat16))
        refuse("%s: operands must both be bfloat16 or float8_e4m3fn, not %s and %s", what, c10::toString(kind), c10::toString(b.scalar_type()));
    if (out_type == DCE_TYPE_E4M3 && !f8) refuse("%s: results of float8_e4m3fn from bfloat16", what);
    if (a.dim() != 2 || b.dim() != (grouped ? 3 : 2))
        refuse("%s: expected a (rows, k) and b (%sn, k), got %s and %s", what, grouped ? "groups, " : "", text(a.sizes()).c_str(), text(b.sizes()).c_str());
    if (grouped) {
        if (b.size(0) < 1 || b.size(0) > DCE_GROUPS_MAX) refuse("%s: expected b (1 .. %d groups, n, k), got %s", what, DCE_GROUPS_MAX, text(b.sizes()).c_str());
        if (offsets.scalar_type() != at::kInt || offsets.dim() != 1 || offsets.size(0) != b.size(0) + 1)
            refuse("%s: offsets must be int32 (%lld,), got %s %s", what, (long long)b.size(0) + 1, c10::toString(offsets.scalar_type()), text(offsets.sizes()).c_str());
        if (index.defined() && (index.scalar_type() != at::kInt || index.dim() != 1))
            refuse("%s: index must be int32 (m,), got %s %s", what, c10::toString(index.scalar_type()), text(index.sizes()).c_str());
    }
    const int dev = device_of(a, what);
    same(dev, what, {&a, &as, &b, &bs, &bias, &out, &outs, &offsets, &index});
    if (grouped && !offsets.is_contiguous()) offsets = offsets.contiguous();
    if (index.defined() && !index.is_contiguous()) index = index.contiguous();
    dce_matmul_desc d{};
    d.lda = rows_of(a);
    d.ldb = rows_of(b);
    const int64_t rows = a.size(0), k = a.size(1), n = b.size(-2), count = grouped ? b.size(0) : 1, m = index.defined() ? index.size(0) : rows;
    const int64_t kb = (k + 127) / 128, nb = (n + 127) / 128;
    if (b.size(-1) != k) refuse("%s: a has %lld columns, b %lld", what, (long long)k, (long long)b.size(-1));
    if (f8) {
        if (!as.defined() || !bs.defined()) refuse("%s: float8_e4m3fn operands need a_scale and b_scale", what);
        int32_t other;
        if (!scale_code(as.scalar_type(), d.scale_type) || !scale_code(bs.scalar_type(), other) || other != d.scale_type)
            refuse("%s: scales must both be float8_e8m0fnu or float32, not %s and %s", what, c10::toString(as.scalar_type()), c10::toString(bs.scalar_type()));
        if (as.dim() != 2 || as.size(0) != kb || as.size(1) != rows || bs.dim() != (grouped ? 3 : 2) || bs.size(-1) != kb || bs.size(-2) != nb || (grouped && bs.size(0) != count))
            refuse("%s: expected a_scale (%lld, %lld) and b_scale (%s%lld, %lld), got %s and %s", what, (long long)kb, (long long)rows, grouped ? "groups, " : "", (long long)nb, (long long)kb,
                   text(as.sizes()).c_str(), text(bs.sizes()).c_str());
        d.ld_a_scale = rows_of(as);
        d.ld_b_scale = rows_of(bs);
        d.b_scale_group = grouped ? bs.stride(0) : 0;
        d.a_scale = as.data_ptr();
        d.b_scale = bs.data_ptr();
    } else if (as.defined() || bs.defined()) refuse("%s: bfloat16 operands have no scales", what);
    if (bias.defined()) {
        if (bias.scalar_type() != at::kFloat || bias.dim() != (grouped ? 2 : 1) || bias.size(-1) != n || (grouped && bias.size(0) != count))
            refuse("%s: bias must be float32 (%s%lld), got %s %s", what, grouped ? "groups, " : "", (long long)n, c10::toString(bias.scalar_type()), text(bias.sizes()).c_str());
        if (n > 1 && bias.stride(-1) != 1) bias = bias.contiguous();
        d.bias = static_cast<const float*>(bias.data_ptr());
        d.bias_group = grouped ? bias.stride(0) : 0;
    }
    const auto want = out_type == DCE_TYPE_F32 ? at::kFloat : out_type == DCE_TYPE_BF16 ? at::kBFloat16 : at::kFloat8_e4m3fn;
    if (!out.defined()) {
        out = at::empty({m, n}, a.options().dtype(want));
        d.ldy = n;
    } else {
        if (out.scalar_type() != want || out.dim() != 2 || out.size(0) != m || out.size(1) != n || (n > 1 && out.stride(1) != 1) || (m > 1 && out.stride(0) < n))
            refuse("%s: out must be a %s (%lld, %lld) tensor whose rows have no gaps and do not overlap", what, c10::toString(want), (long long)m, (long long)n);
        d.ldy = m > 1 ? out.stride(0) : n;
    }
    if (out_type == DCE_TYPE_E4M3) {
        if (!outs.defined()) outs = at::empty({nb, m}, as.options());
        else if (outs.scalar_type() != as.scalar_type() || outs.dim() != 2 || outs.size(0) != nb || outs.size(1) != m || !outs.is_contiguous())
            refuse("%s: out_scale must be a contiguous %s (%lld, %lld) tensor", what, c10::toString(as.scalar_type()), (long long)nb, (long long)m);
        d.y_scale = outs.data_ptr();
        d.ld_y_scale = m;
    } else if (outs.defined()) refuse("%s: out_scale belongs to float8_e4m3fn results", what);
    d.a = a.data_ptr();
    d.b = b.data_ptr();
    d.b_group = grouped ? b.stride(0) : 0;
    d.y = out.data_ptr();
    d.offsets = grouped ? static_cast<const int32_t*>(offsets.data_ptr()) : nullptr;
    d.index = index.defined() ? static_cast<const int32_t*>(index.data_ptr()) : nullptr;
    d.a_rows = rows; d.m = m; d.n = n; d.k = k;
    d.groups = (int32_t)count;
    d.in_type = f8 ? DCE_TYPE_E4M3 : DCE_TYPE_BF16;
    d.out_type = (int32_t)out_type;
    d.relu = relu;
    check(f_matmul(dev, stream_of(dev), &d));
    for (PyObject* o : {arg[8], arg[9]})                            // a caller's tensors were written in place: autograd has to know, as of torch's own operators
        if (o != Py_None && !THPVariable_Unpack(o).is_inference()) THPVariable_Unpack(o).unsafeGetTensorImpl()->bump_version();
    return out_type == DCE_TYPE_E4M3 ? pair(std::move(out), std::move(outs)) : THPVariable_Wrap(std::move(out));
}

// ---- group_rows(ids, groups)
PyObject* group_rows(PyObject* const* a)
{
    at::Tensor ids = tensor(a[0], "group_rows");
    const long groups = PyLong_AsLong(a[1]);
    if (groups == -1 && PyErr_Occurred()) throw Refused{};
    if (!ids.defined() || ids.dim() != 1 || (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong))
        refuse("group_rows: ids must be int32 or int64 (n,), got %s %s", ids.defined() ? c10::toString(ids.scalar_type()) : "None", ids.defined() ? text(ids.sizes()).c_str() : "");
    if (groups < 1 || groups > DCE_GROUPS_MAX) refuse("group_rows: 1 .. %d groups, not %ld", DCE_GROUPS_MAX, groups);
    const int dev = device_of(ids, "group_rows");
    if (!ids.is_contiguous()) ids = ids.contiguous();
    const int64_t n = ids.size(0), need = f_group_rows_work(n, (int)groups);
    check(need);
    const auto o = ids.options().dtype(at::kInt);
    at::Tensor offsets = at::empty({groups + 1}, o), order = at::empty({n}, o), place = at::empty({n}, o), work;
    if (need) work = at::empty({need}, o);
    auto p = [](const at::Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); };
    check(f_group_rows(dev, stream_of(dev), ids.data_ptr(), (int)ids.element_size(), n, (int)groups, p(offsets), p(order), p(place), need ? p(work) : nullptr));
    PyObject* r = PyTuple_New(3);
    if (!r) throw Refused{};
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(offsets)));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(order)));
    PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(place)));
    return r;
}

// ---- decide(logits, index)
PyObject* decide(PyObject* const* a)
{
    at::Tensor v = tensor(a[0], "decide"), index = tensor(a[1], "decide");
    if (!v.defined() || v.scalar_type() != at::kFloat || v.dim() != 2 || v.size(1) != DCE_CLASSES)
        refuse("decide: expected float32 (rows, 16) logits, got %s %s", v.defined() ? c10::toString(v.scalar_type()) : "None", v.defined() ? text(v.sizes()).c_str() : "");
    if (index.defined() && (index.scalar_type() != at::kInt || index.dim() != 1)) refuse("decide: index must be int32 (n,), got %s %s", c10::toString(index.scalar_type()), text(index.sizes()).c_str());
    const int dev = device_of(v, "decide");
    same(dev, "decide", {&v, &index});
    if (!v.is_contiguous()) v = v.contiguous();
    if (index.defined() && !index.is_contiguous()) index = index.contiguous();
    const int64_t n = index.defined() ? index.size(0) : v.size(0);
    at::Tensor logits = at::empty({n, DCE_CLASSES}, v.options()), pred = at::empty({n}, v.options().dtype(at::kInt)), contacts = at::empty({n, DCE_LEGS}, v.options().dtype(at::kByte));
    check(f_decide(dev, stream_of(dev), static_cast<const float*>(v.data_ptr()), v.size(0), index.defined() ? static_cast<const int32_t*>(index.data_ptr()) : nullptr, n,
                   static_cast<float*>(logits.data_ptr()), static_cast<int32_t*>(pred.data_ptr()), static_cast<uint8_t*>(contacts.data_ptr())));
    return Py_BuildValue("{s:N,s:N,s:N}", "logits", THPVariable_Wrap(std::move(logits)), "pred", THPVariable_Wrap(std::move(pred)), "contacts", THPVariable_Wrap(std::move(contacts)));
}

// ---- bind(quantize, matmul, group_rows, group_rows_work, decide, last_error: addresses; the stream lookup; the error class)
PyObject* bind(PyObject* const* a)
{
    void* p[6];
    for (int i = 0; i < 6; ++i) { p[i] = PyLong_AsVoidPtr(a[i]); if (!p[i]) { if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: a null address"); throw Refused{}; } }
    f_quantize = reinterpret_cast<decltype(f_quantize)>(p[0]);
    f_matmul = reinterpret_cast<decltype(f_matmul)>(p[1]);
    f_group_rows = reinterpret_cast<decltype(f_group_rows)>(p[2]);
    f_group_rows_work = reinterpret_cast<decltype(f_group_rows_work)>(p[3]);
    f_decide = reinterpret_cast<decltype(f_decide)>(p[4]);
    f_last_error = reinterpret_cast<decltype(f_last_error)>(p[5]);
    Py_INCREF(a[6]); Py_XSETREF(raw_stream, a[6]);
    Py_INCREF(a[7]); Py_XSETREF(dce_error, a[7]);
    Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject* const*), int N, bool BOUND>
PyObject* entry(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    if (n != N) return PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
    if (BOUND && !f_matmul) { PyErr_SetString(PyExc_RuntimeError, "the library is not bound"); return nullptr; }
    try { return F(a); } catch (const Refused&) { return nullptr; }
    END_HANDLE_TH_ERRORS
}
template <PyObject* (*F)(PyObject* const*), int N, bool BOUND = true>
constexpr PyCFunction as_entry() { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, N, BOUND>)); }

PyMethodDef methods[] = {
    {"quantize", as_entry<quantize, 3>(), METH_FASTCALL, "quantize(x, rows, e8m0)"},
    {"matmul", as_entry<matmul, 12>(), METH_FASTCALL, "matmul(what, a, a_scale, b, b_scale, bias, relu, out_type, out, out_scale, offsets, index)"},
    {"group_rows", as_entry<group_rows, 2>(), METH_FASTCALL, "group_rows(ids, groups)"},
    {"decide", as_entry<decide, 2>(), METH_FASTCALL, "decide(logits, index)"},
    {"bind", as_entry<bind, 8, false>(), METH_FASTCALL, "bind(addresses .., stream lookup, error class)"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_entries", "ops.py's entries on torch tensors", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__entries()
{
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "ABI", DCE_ENTRIES_ABI) != 0) { Py_DECREF(m); return nullptr; }       // (the torch and the interpreter it was compiled for: build.py)
    return m;
}
