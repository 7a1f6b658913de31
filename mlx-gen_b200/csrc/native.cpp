// native.cpp -- the Python side of the decoder operators as a compiled module (qlinear._native):
// checks of the tensors, allocation of the outputs, one call of the C ABI.  In a decode step
// these operators run for 2 - 5 us each, less than the interpreter needs for the same checks
// (a residual norm through ctypes 16.5 us of host time a call), so the host would be what a
// step waits for.
//
// It holds no arithmetic and does not link libqlinear: init() receives the addresses of the
// functions that the ctypes binding has loaded.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/api/include/torch/version.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <sstream>
#include <vector>

#include "../../include/qlinear.h"

namespace {

decltype(&ql_last_error) p_last_error;
decltype(&ql_norm_residual) p_norm_residual;
decltype(&ql_rope) p_rope;
decltype(&ql_rope_append) p_rope_append;
decltype(&ql_paged_attention) p_paged_attention;
decltype(&ql_paged_attention_workspace_size) p_paged_attention_workspace_size;
decltype(&ql_copy_pages) p_copy_pages;
PyObject *g_error;  // QlError(status, message)

struct PythonError {};  // a Python exception is set

template <typename... A>
[[noreturn]] void refuse(PyObject *type, const A &...a) {
    std::ostringstream s;
    (s << ... << a);
    PyErr_SetString(type, s.str().c_str());
    throw PythonError();
}
#define VALUE(cond, ...) \
    if (!(cond)) refuse(PyExc_ValueError, __VA_ARGS__)
#define TYPE(cond, ...) \
    if (!(cond)) refuse(PyExc_TypeError, __VA_ARGS__)

void check(int status) {
    if (status == QL_OK) return;
    PyObject *e = PyObject_CallFunction(g_error, "is", status, p_last_error());
    if (e) {
        PyErr_SetObject(g_error, e);
        Py_DECREF(e);
    }
    throw PythonError();
}

const at::Tensor &tensor(PyObject *o, const char *name) {
    TYPE(THPVariable_Check(o), name, " must be a tensor");
    return THPVariable_Unpack(o);
}
int64_t integer(PyObject *o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw PythonError();
    return v;
}
double real(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw PythonError();
    return v;
}
bool truth(PyObject *o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw PythonError();
    return v;
}
int int32(PyObject *o, const char *name) {
    const int64_t v = integer(o);
    VALUE(v >= INT32_MIN && v <= INT32_MAX, name, " is out of range: ", v);
    return (int)v;
}

int dtype_code(const at::Tensor &t) {
    switch (t.scalar_type()) {
        case at::kFloat: return QL_F32;
        case at::kBFloat16: return QL_BF16;
        case at::kHalf: return QL_F16;
        default: refuse(PyExc_TypeError, "unsupported dtype ", t.scalar_type(), "; expected float32, bfloat16 or float16");
    }
}

// The tensor that decides a call's device.
c10::Device on_cuda(const at::Tensor &t) {
    VALUE(t.is_cuda(), "libqlinear operates on CUDA tensors only");
    return t.device();
}
void *stream_of(c10::Device d) { return c10::cuda::getCurrentCUDAStream(d.index()).stream(); }
at::Tensor fresh(at::IntArrayRef size, at::ScalarType t, c10::Device d) {
    return at::detail::empty_cuda(size, t, d, c10::nullopt);
}

// A contiguous [rows.., D] operand in y's dtype, or None.
const void *row_operand(PyObject *o, const char *name, const at::Tensor &y, int64_t D, int64_t rows) {
    if (o == Py_None) return nullptr;
    const at::Tensor &t = tensor(o, name);
    TYPE(t.scalar_type() == y.scalar_type() && t.device() == y.device(), name, " must be ", y.scalar_type(), " on ",
         y.device(), ", got ", t.scalar_type(), " on ", t.device());
    VALUE(t.dim() > 0 && t.size(-1) == D && t.numel() >= rows * D, name, " must hold ", rows, " row(s) of ", D,
          " elements, got ", t.sizes());
    VALUE(t.is_contiguous(), name, " must be contiguous");
    return t.const_data_ptr();
}

// x as [M, D] with contiguous rows (a copy where its strides do not allow that) and its row stride.
at::Tensor as_rows(const at::Tensor &x, int64_t M, int64_t D, int64_t &stride) {
    if (x.is_contiguous()) {
        stride = D;
        return x;
    }
    at::Tensor t = x.dim() == 2 ? x : x.reshape({M, D});
    if ((D > 1 && t.stride(1) != 1) || (M > 1 && t.stride(0) < D)) t = t.contiguous();
    stride = M > 1 ? t.stride(0) : D;
    return t;
}

// (y, residual, weight, post_weight, gate, gate_period, alpha, scale, scale_period, eps, weight_offset) -> (h, r)
PyObject *norm_residual(PyObject *const *a) {
    const at::Tensor &y = tensor(a[0], "y"), &res = tensor(a[1], "residual");
    const c10::Device dev = on_cuda(y);
    VALUE(y.dim() > 0, "y must be [.., D]");
    VALUE(res.sizes() == y.sizes(), "residual ", res.sizes(), " must have y's shape ", y.sizes());
    VALUE(res.device() == dev, "residual is on ", res.device(), ", expected ", dev);
    const int ydt = dtype_code(y), rdt = dtype_code(res);
    const int64_t D = y.size(-1), M = D ? y.numel() / D : 0;
    const int64_t gp = integer(a[5]), sp = integer(a[8]);
    const auto rows = [&](int64_t period) { return period > 0 ? (M + period - 1) / period : 1; };
    TYPE(a[2] != Py_None, "weight must be a tensor");
    const void *w = row_operand(a[2], "weight", y, D, 1), *post = row_operand(a[3], "post_weight", y, D, 1);
    const void *gate = row_operand(a[4], "gate", y, D, rows(gp)), *scale = row_operand(a[7], "scale", y, D, rows(sp));
    const c10::cuda::CUDAGuard guard(dev);
    int64_t ys, rs;
    const at::Tensor y2 = as_rows(y, M, D, ys), r2 = as_rows(res, M, D, rs);
    at::Tensor h = fresh(y.sizes(), y.scalar_type(), dev), r = fresh(y.sizes(), res.scalar_type(), dev);
    check(p_norm_residual(y2.const_data_ptr(), ydt, ys, r2.const_data_ptr(), rdt, rs, M, D, w, (float)real(a[10]), post, gate,
                          gp, (float)real(a[6]), scale, sp, (float)real(a[9]), h.mutable_data_ptr(), r.mutable_data_ptr(),
                          stream_of(dev)));
    return Py_BuildValue("NN", THPVariable_Wrap(std::move(h)), THPVariable_Wrap(std::move(r)));
}

struct RopeArgs {
    c10::Device dev;
    int64_t T, Hq, D;
};
RopeArgs rope_args(const at::Tensor &q, const at::Tensor &table, const at::Tensor &pos) {
    const c10::Device dev = on_cuda(q);
    VALUE(q.dim() == 3, "q must be [tokens, heads, head_dim], got ", q.sizes());
    VALUE(table.dim() == 2 && table.scalar_type() == at::kFloat && table.is_contiguous(),
          "table must be a contiguous float32 [positions, rotary_dim] (see rope_table)");
    VALUE(pos.scalar_type() == at::kLong && pos.dim() == 1 && pos.size(0) == q.size(0) && pos.is_contiguous(),
          "positions must be a contiguous int64 [tokens]");
    VALUE(table.device() == dev && pos.device() == dev, "table and positions must be on ", dev);
    return {dev, q.size(0), q.size(1), q.size(2)};
}
at::Tensor heads(const at::Tensor &x, const char *name, const RopeArgs &r, const at::Tensor &q) {
    VALUE(x.dim() == 3 && x.size(0) == r.T && x.size(2) == r.D, name, " must be [", r.T, ", heads, ", r.D, "], got ", x.sizes());
    TYPE(x.scalar_type() == q.scalar_type() && x.device() == q.device(), name, " must be ", q.scalar_type(), " on ",
         q.device(), ", got ", x.scalar_type(), " on ", x.device());
    return x.stride(2) == 1 || r.D == 1 ? x : x.contiguous();
}
int head_count(int64_t n) {
    VALUE(n <= INT32_MAX, "too many heads");
    return (int)n;
}

// (q, k, table, positions, layout) -> (q', k')
PyObject *rope(PyObject *const *a) {
    const at::Tensor &q0 = tensor(a[0], "q"), &table = tensor(a[2], "table"), &pos = tensor(a[3], "positions");
    const RopeArgs r = rope_args(q0, table, pos);
    const c10::cuda::CUDAGuard guard(r.dev);
    const at::Tensor q = heads(q0, "q", r, q0), k = heads(tensor(a[1], "k"), "k", r, q0);
    at::Tensor qo = fresh(q.sizes(), q.scalar_type(), r.dev), ko = fresh(k.sizes(), q.scalar_type(), r.dev);
    check(p_rope(q.const_data_ptr(), q.stride(0), q.stride(1), k.const_data_ptr(), k.stride(0), k.stride(1), dtype_code(q),
                 r.T, head_count(r.Hq), head_count(k.size(1)), head_count(r.D), head_count(table.size(1)), int32(a[4], "layout"),
                 table.const_data_ptr<float>(), table.size(0), pos.const_data_ptr<int64_t>(), qo.mutable_data_ptr(),
                 ko.mutable_data_ptr(), stream_of(r.dev)));
    return Py_BuildValue("NN", THPVariable_Wrap(std::move(qo)), THPVariable_Wrap(std::move(ko)));
}

struct Cache {
    int64_t pages, heads, page_size, D, stride;
};
Cache cache_of(const at::Tensor &k, const at::Tensor &v, const at::Tensor &q) {
    for (const at::Tensor *c : {&k, &v})
        VALUE(c->dim() == 4 && c->scalar_type() == q.scalar_type() && c->device() == q.device(), c == &k ? "k" : "v",
              "_cache must be [pages, heads, page_size, head_dim] in ", q.scalar_type(), " on ", q.device(), ", got ",
              c->sizes(), " ", c->scalar_type(), " on ", c->device());
    VALUE(k.sizes() == v.sizes() && k.strides() == v.strides(), "k_cache and v_cache must have the same shape and strides");
    const int64_t P = k.size(0), H = k.size(1), ps = k.size(2), D = k.size(3);
    VALUE((D <= 1 || k.stride(3) == 1) && (ps <= 1 || k.stride(2) == D) && (H <= 1 || k.stride(1) == ps * D) &&
              (P <= 1 || k.stride(0) >= H * ps * D),
          "the [heads, page_size, head_dim] of a page must be contiguous");
    VALUE(H <= INT32_MAX && ps <= INT32_MAX && D <= INT32_MAX, "cache too large");
    return {P, H, ps, D, P > 1 ? k.stride(0) : H * ps * D};
}

// (q, k, v, table, positions, k_cache, v_cache, slots, layout) -> q'
PyObject *rope_append(PyObject *const *a) {
    const at::Tensor &q0 = tensor(a[0], "q"), &table = tensor(a[3], "table"), &pos = tensor(a[4], "positions");
    const at::Tensor &kc = tensor(a[5], "k_cache"), &vc = tensor(a[6], "v_cache"), &slots = tensor(a[7], "slots");
    const RopeArgs r = rope_args(q0, table, pos);
    const c10::cuda::CUDAGuard guard(r.dev);
    const at::Tensor q = heads(q0, "q", r, q0), k = heads(tensor(a[1], "k"), "k", r, q0), v = heads(tensor(a[2], "v"), "v", r, q0);
    const Cache c = cache_of(kc, vc, q0);
    VALUE(k.size(1) == c.heads && v.size(1) == c.heads && c.D == r.D, "k and v must have the cache's ", c.heads, " heads of ",
          c.D, ", got ", k.sizes(), " and ", v.sizes());
    VALUE(slots.scalar_type() == at::kLong && slots.sizes() == pos.sizes() && slots.is_contiguous() && slots.device() == r.dev,
          "slots must be a contiguous int64 [tokens] on ", r.dev);
    at::Tensor qo = fresh(q.sizes(), q.scalar_type(), r.dev);
    check(p_rope_append(q.const_data_ptr(), q.stride(0), q.stride(1), k.const_data_ptr(), k.stride(0), k.stride(1),
                        v.const_data_ptr(), v.stride(0), v.stride(1), dtype_code(q), r.T, head_count(r.Hq), (int)c.heads,
                        (int)c.D, head_count(table.size(1)), int32(a[8], "layout"), table.const_data_ptr<float>(),
                        table.size(0), pos.const_data_ptr<int64_t>(), slots.const_data_ptr<int64_t>(), kc.mutable_data_ptr(),
                        vc.mutable_data_ptr(), c.pages, c.stride, (int)c.page_size, qo.mutable_data_ptr(), stream_of(r.dev)));
    return THPVariable_Wrap(std::move(qo));
}

const int32_t *index_tensor(const at::Tensor &t, const char *name, c10::Device dev) {
    VALUE(t.scalar_type() == at::kInt && t.device() == dev && (t.size(-1) <= 1 || t.stride(-1) == 1), name, " must be int32 on ",
          dev, " with a contiguous last axis");
    return t.const_data_ptr<int32_t>();
}

// (q, k_cache, v_cache, page_table, q_starts, kv_lens, max_q, max_kv, scale, causal, window, out, workspace) -> out
PyObject *paged_attention(PyObject *const *a) {
    at::Tensor q = tensor(a[0], "q");
    const at::Tensor &kc = tensor(a[1], "k_cache"), &vc = tensor(a[2], "v_cache"), &table = tensor(a[3], "page_table");
    const at::Tensor &starts = tensor(a[4], "q_starts"), &lens = tensor(a[5], "kv_lens");
    const int64_t max_q = integer(a[6]), max_kv = integer(a[7]), window = integer(a[10]);
    const c10::Device dev = on_cuda(q);
    VALUE(q.dim() == 3, "q must be [tokens, heads, head_dim], got ", q.sizes());
    const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2);
    const Cache c = cache_of(kc, vc, q);
    VALUE(c.D == D, "q's head dimension ", D, " differs from the cache's ", c.D);
    VALUE(lens.dim() == 1 && table.dim() == 2 && table.size(0) == lens.size(0) && starts.dim() == 1 &&
              starts.size(0) == lens.size(0) + 1,
          "expected kv_lens [B], q_starts [B + 1] and page_table [B, pages], got ", lens.sizes(), ", ", starts.sizes(), ", ",
          table.sizes());
    const int64_t B = lens.size(0);
    const int32_t *tp = index_tensor(table, "page_table", dev), *sp = index_tensor(starts, "q_starts", dev),
                  *lp = index_tensor(lens, "kv_lens", dev);
    VALUE(max_kv <= table.size(1) * c.page_size, "page_table's ", table.size(1), " pages of ", c.page_size,
          " do not hold max_kv=", max_kv, " positions");
    const c10::cuda::CUDAGuard guard(dev);
    if (q.stride(2) != 1 || q.stride(0) % 8 || q.stride(1) % 8 || reinterpret_cast<uintptr_t>(q.const_data_ptr()) % 16)
        q = q.clone(at::MemoryFormat::Contiguous);
    at::Tensor out;
    if (a[11] == Py_None) out = fresh(q.sizes(), q.scalar_type(), dev);
    else {
        out = tensor(a[11], "out");
        VALUE(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.device() == dev && out.is_contiguous(),
              "out must be contiguous, of q's shape, dtype and device");
    }
    const int hq = head_count(Hq), hkv = (int)c.heads, d = (int)D;
    const size_t need = p_paged_attention_workspace_size(T, hq, hkv, d, B, max_q, max_kv, window);
    at::Tensor ws;
    if (need) {
        if (a[12] != Py_None) {
            ws = tensor(a[12], "workspace");
            VALUE(ws.device() == dev && ws.is_contiguous(), "workspace must be contiguous on ", dev);
        }
        if (!ws.defined() || ws.nbytes() < need) ws = fresh({(int64_t)need}, at::kByte, dev);
    }
    const float scale = a[8] == Py_None ? (float)(1.0 / std::sqrt((double)D)) : (float)real(a[8]);
    check(p_paged_attention(q.const_data_ptr(), dtype_code(q), q.stride(0), q.stride(1), T, hq, hkv, d, kc.const_data_ptr(),
                            vc.const_data_ptr(), c.pages, c.stride, (int)c.page_size, tp,
                            B > 1 ? table.stride(0) : table.size(1), sp, lp, B, max_q, max_kv, scale, truth(a[9]),
                            window, out.mutable_data_ptr(), need ? ws.mutable_data_ptr() : nullptr, need,
                            stream_of(dev)));
    return THPVariable_Wrap(std::move(out));
}

std::vector<int32_t> indices(PyObject *o, const char *name) {
    PyObject *s = PySequence_Fast(o, "src and dst must be sequences of page indices");
    if (!s) throw PythonError();
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(s);
    std::vector<int32_t> v;
    try {
        v.resize((size_t)n);
        for (Py_ssize_t i = 0; i < n; ++i) v[(size_t)i] = int32(PySequence_Fast_GET_ITEM(s, i), name);
    } catch (...) {
        Py_DECREF(s);
        throw;
    }
    Py_DECREF(s);
    return v;
}

// (pool, src, dst) -> None
PyObject *copy_pages(PyObject *const *a) {
    const at::Tensor &pool = tensor(a[0], "pool");
    const c10::Device dev = on_cuda(pool);
    VALUE(pool.dim() >= 4 && pool.is_contiguous(), "pool must be a contiguous [.., pages, heads, page_size, head_dim]");
    const std::vector<int32_t> src = indices(a[1], "src"), dst = indices(a[2], "dst");
    VALUE(src.size() == dst.size(), src.size(), " sources for ", dst.size(), " destinations");
    const int64_t pages = pool.size(-4);
    const int64_t bytes = pool.size(-3) * pool.size(-2) * pool.size(-1) * (int64_t)pool.element_size();
    const int64_t planes = pages && bytes ? (int64_t)pool.nbytes() / (pages * bytes) : 0;
    const c10::cuda::CUDAGuard guard(dev);
    check(p_copy_pages(pool.mutable_data_ptr(), planes, pages * bytes, pages, bytes, bytes, src.data(), dst.data(),
                       (int64_t)src.size(), stream_of(dev)));
    Py_RETURN_NONE;
}

template <PyObject *(*F)(PyObject *const *), int N>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != N || !p_last_error) {
        PyErr_SetString(PyExc_TypeError, n != N ? "wrong number of arguments" : "qlinear._native is not initialised");
        return nullptr;
    }
    try {
        return F(args);
    } catch (const PythonError &) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// (error class, addresses in the order below)
PyObject *init(PyObject *, PyObject *args) {
    unsigned long long f[7];
    PyObject *err;
    if (!PyArg_ParseTuple(args, "OKKKKKKK", &err, &f[0], &f[1], &f[2], &f[3], &f[4], &f[5], &f[6])) return nullptr;
    Py_INCREF(err);
    g_error = err;
    p_norm_residual = reinterpret_cast<decltype(p_norm_residual)>(f[1]);
    p_rope = reinterpret_cast<decltype(p_rope)>(f[2]);
    p_rope_append = reinterpret_cast<decltype(p_rope_append)>(f[3]);
    p_paged_attention = reinterpret_cast<decltype(p_paged_attention)>(f[4]);
    p_paged_attention_workspace_size = reinterpret_cast<decltype(p_paged_attention_workspace_size)>(f[5]);
    p_copy_pages = reinterpret_cast<decltype(p_copy_pages)>(f[6]);
    p_last_error = reinterpret_cast<decltype(p_last_error)>(f[0]);
    Py_RETURN_NONE;
}

template <PyObject *(*F)(PyObject *const *), int N>
PyMethodDef method(const char *name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&entry<F, N>)), METH_FASTCALL, nullptr};
}
PyMethodDef g_methods[] = {
    {"init", init, METH_VARARGS, nullptr},  method<norm_residual, 11>("norm_residual"), method<rope, 5>("rope"),
    method<rope_append, 9>("rope_append"),  method<paged_attention, 13>("paged_attention"),
    method<copy_pages, 3>("copy_pages"),    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native() {
    PyObject *m = PyModule_Create(&g_module);
    if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) < 0) Py_CLEAR(m);
    return m;
}
