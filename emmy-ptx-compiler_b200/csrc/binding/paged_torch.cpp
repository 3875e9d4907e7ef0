// emmy_ptx._paged: the paged-cache operators on torch tensors, in front of libemmyb200.so's C ABI.
//
// A serving step makes three calls a layer, each of a few microseconds on the GPU. Checking a tensor's type, shape, strides
// and device through Python's attributes costs about a third of a microsecond apiece, 15 to 20 a call (18 to 28 us a call
// were measured that way); here they are reads of the tensor's own fields. emmy_ptx/paged.py has the documented functions.

#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <initializer_list>
#include <limits>

#include "emmy_b200.h"

namespace {

PyObject* g_error = nullptr;  // emmy_ptx.driver.EmbError

struct Refused {};  // the Python error is set

[[noreturn]] void raise(int code, const char* text) {
    PyObject* args = Py_BuildValue("(is)", code, text);
    PyObject* e = args ? PyObject_CallObject(g_error, args) : nullptr;
    Py_XDECREF(args);
    if (e) {
        PyErr_SetObject(g_error, e);
        Py_DECREF(e);
    }
    throw Refused();
}

[[noreturn]] __attribute__((format(printf, 1, 2))) void refuse(const char* fmt, ...) {
    char text[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof text, fmt, ap);
    va_end(ap);
    raise(EMB_E_ARGUMENT, text);
}

struct Arg {  // one argument: a tensor, or None where it may be left out
    const char* name;
    const at::Tensor* t;
    bool given() const { return t != nullptr; }
    const at::Tensor* operator->() const { return t; }
};

Arg tensor(const char* who, const char* name, PyObject* o, bool optional = false) {
    if (optional && o == Py_None) return {name, nullptr};
    if (!THPVariable_Check(o)) refuse("%s: %s is not a tensor", who, name);
    return {name, &THPVariable_Unpack(o)};
}

[[noreturn]] void refuse_shape(const char* who, const Arg& x, const char* is, std::initializer_list<int64_t> shape) {
    char want[96] = "", have[96] = "";
    size_t at = 0;
    for (int64_t n : shape) at += snprintf(want + at, sizeof want - at, at ? ", %lld" : "%lld", static_cast<long long>(n));
    at = 0;
    for (int64_t n : x->sizes())
        if (at + 24 < sizeof have) at += snprintf(have + at, sizeof have - at, at ? ", %lld" : "%lld", static_cast<long long>(n));
    refuse("%s: %s is %s [%s], not %s [%s]", who, x.name, is, want, c10::toString(x->scalar_type()), have);
}

bool shaped(const Arg& x, std::initializer_list<int64_t> shape) {
    return x->sizes().equals(c10::IntArrayRef(shape.begin(), shape.size()));
}

const int32_t* int32(const char* who, const Arg& x, int64_t n) {
    if (x->scalar_type() != at::kInt || !shaped(x, {n}) || !x->is_contiguous()) refuse_shape(who, x, "a contiguous int32 tensor", {n});
    return static_cast<const int32_t*>(x->data_ptr());
}

// C sizes are 32 bits wide
int32_t narrow(const char* who, const char* name, int64_t n) {
    if (n < std::numeric_limits<int32_t>::min() || n > std::numeric_limits<int32_t>::max()) refuse("%s: %s is beyond 31 bits", who, name);
    return static_cast<int32_t>(n);
}

int32_t integer(const char* who, const char* name, PyObject* o) {
    const long long n = PyLong_AsLongLong(o);
    if (n == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse("%s: %s is not an integer of 64 bits", who, name);
    }
    return narrow(who, name, n);
}

float real(const char* who, const char* name, PyObject* o) {
    const double x = PyFloat_AsDouble(o);
    if (x == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse("%s: %s is not a number", who, name);
    }
    return static_cast<float>(x);
}

int dtype_code(at::ScalarType t) { return t == at::kHalf ? EMB_F16 : t == at::kBFloat16 ? EMB_BF16 : t == at::kFloat8_e4m3fn ? EMB_U8 : -1; }

int q_type(const char* who, const Arg& q) {
    if (q->dim() != 3) refuse("%s: q is a tensor [rows, heads, dim]", who);
    const int code = dtype_code(q->scalar_type());
    if (code != EMB_F16 && code != EMB_BF16) refuse("%s: q is f16 or bf16, not %s", who, c10::toString(q->scalar_type()));
    return code;
}

// [rows, heads, dim] with a contiguous last dimension; the strides of the others (of one element: 0, since any will do)
void rows(const char* who, const Arg& x, at::ScalarType type, int64_t n, int64_t heads, int64_t dim, int64_t (&stride)[2]) {
    if (x->scalar_type() != type || !shaped(x, {n, heads, dim})) refuse_shape(who, x, c10::toString(type), {n, heads, dim});
    const auto s = x->strides();
    if (dim > 1 && s[2] != 1) refuse("%s: the last dimension of %s is not contiguous", who, x.name);
    stride[0] = n > 1 ? s[0] : 0;
    stride[1] = heads > 1 ? s[1] : 0;
}

emb_paged_cache_t cache(const char* who, const Arg& k, const Arg& v, int q_code, int64_t dim, PyObject* k_scale, PyObject* v_scale) {
    if (k->dim() != 4 || v->dim() != 4 || !k->sizes().equals(v->sizes()) || k->scalar_type() != v->scalar_type())
        refuse("%s: key and value pages are two tensors [pages, page size, key heads, dim] of one type", who);
    emb_paged_cache_t c;
    std::memset(&c, 0, sizeof c);
    c.dtype = dtype_code(k->scalar_type());
    if (c.dtype != EMB_U8 && c.dtype != q_code)
        refuse("%s: pages of %s: q's type, the same 16-bit type, or float8_e4m3fn are taken", who, c10::toString(k->scalar_type()));
    const auto n = k->sizes();
    if (n[3] != dim) refuse("%s: heads of %lld, pages of %lld", who, static_cast<long long>(dim), static_cast<long long>(n[3]));
    const auto ks = k->strides(), vs = v->strides();
    if (dim > 1 && (ks[3] != 1 || vs[3] != 1)) refuse("%s: the last dimension of the pages is not contiguous", who);
    c.k_scale = real(who, "k_scale", k_scale);
    c.v_scale = real(who, "v_scale", v_scale);
    if (c.dtype != EMB_U8 && (c.k_scale != 1.f || c.v_scale != 1.f)) refuse("%s: scales belong to a float8_e4m3fn cache", who);
    c.k = k->data_ptr();
    c.v = v->data_ptr();
    for (int i = 0; i < 3; ++i) {
        c.k_stride[i] = n[i] > 1 ? ks[i] : 0;
        c.v_stride[i] = n[i] > 1 ? vs[i] : 0;
    }
    c.pages = narrow(who, "the number of pages", n[0]);
    c.page_size = narrow(who, "the page size", n[1]);
    c.kv_heads = narrow(who, "the number of key heads", n[2]);
    c.dim = narrow(who, "the head dim", n[3]);
    return c;
}

// the row stride of a table [requests, width]
int64_t table_stride(const char* who, const Arg& table, int64_t requests) {
    if (table->scalar_type() != at::kInt || table->dim() != 2 || table->size(0) != requests || (table->size(1) > 1 && table->stride(1) != 1))
        refuse("%s: table is an int32 tensor [%lld, width] with contiguous rows", who, static_cast<long long>(requests));
    return requests > 1 ? table->stride(0) : table->size(1);
}

int device_of(const char* who, std::initializer_list<Arg> all) {
    const c10::Device first = (*all.begin())->device();
    for (const Arg& x : all)
        if (x.given() && x->device() != first) refuse("%s: the tensors are on different devices (%s)", who, x.name);
    if (!first.is_cuda()) refuse("%s: the tensors are not on a CUDA device: the kernels run on the GPU only", who);
    return first.index();
}

// a tensor that wants its gradient would silently get none (and one that is written would lose what it had); so would the
// tangent of forward differentiation, which torch.no_grad() does not end
void no_graph(const char* who, std::initializer_list<Arg> all) {
    const bool backward = c10::GradMode::is_enabled();
    const bool forward = c10::AutogradState::get_tls_state().get_fw_grad_mode() && torch::autograd::ForwardADLevel::try_get_by_idx(0);  // (a level is open)
    for (const Arg& x : all) {
        if (!x.given()) continue;
        if (backward && x->requires_grad()) refuse("%s: %s requires a gradient, and this operator has none (call it under torch.no_grad())", who, x.name);
        if (forward && x->_fw_grad(0).defined()) refuse("%s: %s has a tangent, and this operator has none", who, x.name);
    }
}

// what an operator wrote into, for autograd: a graph that saved one of these tensors finds that it changed. (Tensors made in
// inference mode have no count.)
void wrote(std::initializer_list<Arg> all) {
    for (const Arg& x : all)
        if (x.given() && !x->is_inference()) x->unsafeGetTensorImpl()->bump_version();
}

at::Tensor empty(c10::IntArrayRef shape, at::ScalarType type, int device) {
    return at::empty(shape, at::TensorOptions().dtype(type).device(c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(device))));
}

void check(int code) {
    if (code) raise(code, emb_last_error());
}

// ---------------------------------------------------------------- the calls

PyObject* assign(PyObject* const* o) {
    const char* who = "assign";
    const Arg cached = tensor(who, "cached", o[0]), fresh = tensor(who, "fresh", o[1]), table = tensor(who, "table", o[2]);
    const Arg free_pages = tensor(who, "free_pages", o[3]), free_head = tensor(who, "free_head", o[4]);
    emb_paged_assign_t a;
    std::memset(&a, 0, sizeof a);
    a.page_size = integer(who, "page_size", o[5]);
    a.tokens = integer(who, "tokens", o[6]);
    if (a.tokens < 0) refuse("assign: tokens is negative");
    if (cached->dim() != 1 || free_pages->dim() != 1) refuse("assign: cached is [requests], free_pages is [n]");
    const int64_t requests = cached->size(0);
    a.requests = narrow(who, "the number of requests", requests);
    a.cached = int32(who, cached, requests);
    a.fresh = int32(who, fresh, requests);
    a.table_stride = table_stride(who, table, requests);
    a.table = static_cast<int32_t*>(table->data_ptr());
    a.table_width = narrow(who, "the table's width", table->size(1));
    a.free_pages = int32(who, free_pages, free_pages->size(0));
    a.free_count = narrow(who, "the number of free pages", free_pages->size(0));
    a.free_head = int32(who, free_head, 1);
    static const char* const names[6] = {"out.slots", "out.positions", "out.starts", "out.lengths", "out.free_head", "out.report"};
    const int64_t sizes[6] = {a.tokens, a.tokens, requests + 1, requests, 1, 4};
    at::Tensor made[6];
    int32_t* to[6];
    PyObject* given = o[7];
    if (given != Py_None) {
        if (!PyTuple_Check(given) || PyTuple_GET_SIZE(given) != 6) refuse("assign: out is a tuple of six tensors");
        for (int i = 0; i < 6; ++i) {
            const Arg x = tensor(who, names[i], PyTuple_GET_ITEM(given, i));
            to[i] = const_cast<int32_t*>(int32(who, x, sizes[i]));
            if (x->device() != cached->device()) refuse("assign: the tensors are on different devices (%s)", x.name);
        }
    }
    const int device = device_of(who, {cached, fresh, table, free_pages, free_head});
    if (given == Py_None) {
        for (int i = 0; i < 6; ++i) {
            made[i] = empty({sizes[i]}, at::kInt, device);
            to[i] = static_cast<int32_t*>(made[i].data_ptr());
        }
    }
    a.slots = to[0], a.positions = to[1], a.starts = to[2], a.lengths = to[3], a.free_head_out = to[4], a.report = to[5];
    const c10::cuda::OptionalCUDAGuard guard(static_cast<c10::DeviceIndex>(device));
    check(emb_paged_assign(&a, c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream()));
    wrote({table});
    if (given != Py_None) {
        for (int i = 0; i < 6; ++i) wrote({tensor(who, names[i], PyTuple_GET_ITEM(given, i))});
        Py_INCREF(given);
        return given;
    }
    PyObject* r = PyTuple_New(6);
    for (int i = 0; r && i < 6; ++i) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(made[i]));
    return r;
}

PyObject* store(PyObject* const* o) {
    const char* who = "store";
    const Arg q = tensor(who, "q", o[0]), k = tensor(who, "k", o[1]), v = tensor(who, "v", o[2]);
    const Arg k_pages = tensor(who, "k_pages", o[3]), v_pages = tensor(who, "v_pages", o[4]), slots = tensor(who, "slots", o[5]);
    const Arg positions = tensor(who, "positions", o[6], true), rope = tensor(who, "rope", o[7], true);
    const Arg weights[2] = {tensor(who, "q_weight", o[8], true), tensor(who, "k_weight", o[9], true)};
    const Arg out = tensor(who, "out", o[14], true);
    no_graph(who, {q, k, v, k_pages, v_pages, rope, weights[0], weights[1], out});
    emb_paged_store_t a;
    std::memset(&a, 0, sizeof a);
    a.dtype = q_type(who, q);
    const auto type = q->scalar_type();
    const int64_t n = q->size(0), heads = q->size(1), dim = q->size(2);
    a.cache = cache(who, k_pages, v_pages, a.dtype, dim, o[12], o[13]);
    rows(who, q, type, n, heads, dim, a.q_stride);
    rows(who, k, type, n, a.cache.kv_heads, dim, a.k_stride);
    rows(who, v, type, n, a.cache.kv_heads, dim, a.v_stride);
    a.q = q->data_ptr(), a.k = k->data_ptr(), a.v = v->data_ptr();
    a.tokens = narrow(who, "the number of rows", n);
    a.heads = narrow(who, "the number of heads", heads);
    a.slots = int32(who, slots, n);
    if (rope.given()) {
        if (rope->scalar_type() != at::kFloat || rope->dim() != 2 || !rope->is_contiguous()) refuse("store: rope is a contiguous float32 tensor [positions, rot]");
        if (!positions.given()) refuse("store: a rotation needs positions");
        a.rope_rows = narrow(who, "the length of rope", rope->size(0));
        a.rot = narrow(who, "the width of rope", rope->size(1));
        a.rope = static_cast<const float*>(rope->data_ptr());
        a.positions = int32(who, positions, n);
    }
    for (int i = 0; i < 2; ++i) {
        if (!weights[i].given()) continue;
        if (weights[i]->scalar_type() != type || !shaped(weights[i], {dim}) || !weights[i]->is_contiguous())
            refuse_shape(who, weights[i], type == at::kHalf ? "a contiguous Half tensor" : "a contiguous BFloat16 tensor", {dim});
        (i ? a.k_weight : a.q_weight) = weights[i]->data_ptr();
    }
    a.eps = real(who, "eps", o[10]);
    const int truth = PyObject_IsTrue(o[11]);
    if (truth < 0) throw Refused();
    a.interleaved = truth;
    if (out.given()) rows(who, out, type, n, heads, dim, a.out_stride);
    const int device = device_of(who, {q, k, v, k_pages, v_pages, slots, rope, rope.given() ? positions : rope, weights[0], weights[1], out});
    at::Tensor made;
    if (!out.given()) {
        made = empty({n, heads, dim}, type, device);
        a.out_stride[0] = heads * dim, a.out_stride[1] = dim;
    }
    a.q_out = out.given() ? out->data_ptr() : made.data_ptr();
    const c10::cuda::OptionalCUDAGuard guard(static_cast<c10::DeviceIndex>(device));
    check(emb_paged_store(&a, c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream()));
    wrote({k_pages, v_pages, out});
    if (!out.given()) return THPVariable_Wrap(std::move(made));
    Py_INCREF(o[14]);
    return o[14];
}

PyObject* attend(PyObject* const* o) {
    const char* who = "attend";
    const Arg q = tensor(who, "q", o[0]), k_pages = tensor(who, "k_pages", o[1]), v_pages = tensor(who, "v_pages", o[2]);
    const Arg table = tensor(who, "table", o[3]), lengths = tensor(who, "lengths", o[4]);
    const Arg out = tensor(who, "out", o[9], true), lse = tensor(who, "lse", o[10], true);
    no_graph(who, {q, k_pages, v_pages, out, lse});
    emb_paged_attend_t a;
    std::memset(&a, 0, sizeof a);
    a.dtype = q_type(who, q);
    const auto type = q->scalar_type();
    const int64_t n = q->size(0), heads = q->size(1), dim = q->size(2);
    a.cache = cache(who, k_pages, v_pages, a.dtype, dim, o[7], o[8]);
    rows(who, q, type, n, heads, dim, a.q_stride);
    a.q = q->data_ptr();
    a.requests = narrow(who, "the number of requests", n);
    a.heads = narrow(who, "the number of heads", heads);
    a.lengths = int32(who, lengths, n);
    a.table_stride = table_stride(who, table, n);
    a.table = static_cast<const int32_t*>(table->data_ptr());
    a.table_width = narrow(who, "the table's width", table->size(1));
    a.scale = o[5] == Py_None ? 1.f / std::sqrt(static_cast<float>(dim)) : real(who, "scale", o[5]);
    a.window = integer(who, "window", o[6]);
    if (out.given()) rows(who, out, type, n, heads, dim, a.out_stride);
    if (lse.given()) {
        if (lse->scalar_type() != at::kFloat || !shaped(lse, {n, heads}) || !lse->is_contiguous()) refuse_shape(who, lse, "a contiguous float32 tensor", {n, heads});
        a.lse = static_cast<float*>(lse->data_ptr());
    }
    const int device = device_of(who, {q, k_pages, v_pages, table, lengths, out, lse});
    const c10::cuda::OptionalCUDAGuard guard(static_cast<c10::DeviceIndex>(device));
    a.workspace_bytes = emb_paged_attend_workspace(&a);
    if (a.workspace_bytes < 0) check(static_cast<int>(a.workspace_bytes));
    at::Tensor made;
    if (!out.given()) {
        made = empty({n, heads, dim}, type, device);
        a.out_stride[0] = heads * dim, a.out_stride[1] = dim;
    }
    a.out = out.given() ? out->data_ptr() : made.data_ptr();
    // a workspace of the call's own from torch's allocator: calls on other streams and captured graphs never share one
    c10::DataPtr workspace;
    if (a.workspace_bytes) {
        workspace = c10::cuda::CUDACachingAllocator::get()->allocate(static_cast<size_t>(a.workspace_bytes));
        a.workspace = workspace.get();
    }
    check(emb_paged_attend(&a, c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream()));
    wrote({out, lse});
    if (!out.given()) return THPVariable_Wrap(std::move(made));
    Py_INCREF(o[9]);
    return o[9];
}

template <PyObject* (*CALL)(PyObject* const*), Py_ssize_t COUNT> PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if (count != COUNT) {
        PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd", COUNT, count);
        return nullptr;
    }
    if (!g_error) {
        PyErr_SetString(PyExc_RuntimeError, "init() comes first");
        return nullptr;
    }
    try {
        return CALL(args);
    } catch (const Refused&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

PyObject* init(PyObject*, PyObject* error) {
    Py_INCREF(error);
    Py_XSETREF(g_error, error);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"init", init, METH_O, "init(EmbError): the exception that refusals raise"},
    {"assign", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<assign, 8>)), METH_FASTCALL, "see emmy_ptx.paged.assign"},
    {"store", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<store, 15>)), METH_FASTCALL, "see emmy_ptx.paged.store"},
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<attend, 11>)), METH_FASTCALL, "see emmy_ptx.paged.attend"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged", "the paged-cache operators on torch tensors", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged() { return PyModule_Create(&module); }
