// The paged-cache calls of kernels.py on torch tensors: what a call of a few microseconds of device work spends in Python (attribute reads, checks, allocation of
// outputs: 10 us of an append and its read back) in C++. Each function does what its namesake in kernels.py does, for arguments that are in order; for
// any other (and where the library refuses) it returns None, and kernels.py, which holds the checks with their messages, takes the call. Built where torch's headers
// are (build.py); without it kernels.py takes every call. The library is not linked: bind() takes the addresses of its functions.
#define PY_SSIZE_T_CLEAN
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/version.h>
#include <climits>
#include <cmath>
#include <cstring>
#include "../../include/hipster_b200.h"

namespace {

decltype(&hp_kv_append) f_append = nullptr;
decltype(&hp_kv_read) f_read = nullptr;
decltype(&hp_attn_paged) f_attn = nullptr;
decltype(&hp_attn_paged_workspace_bytes) f_bytes = nullptr;
decltype(&hp_rope_table) f_table = nullptr;

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }
bool on(const at::Tensor* t, int dev, at::ScalarType type) { return t && t->is_cuda() && t->get_device() == dev && t->scalar_type() == type && t->layout() == at::kStrided; }
struct Rows { float* p; long long ld, hs; };
bool rows(PyObject* o, int dev, int64_t R, int64_t heads, int64_t D, Rows* out) {
    const at::Tensor* t = tensor(o);
    if (!on(t, dev, at::kFloat) || t->dim() != 3 || t->size(0) != R || t->size(1) != heads || t->size(2) != D || t->stride(2) != 1) return false;
    out->p = static_cast<float*>(t->data_ptr()); out->ld = t->stride(0); out->hs = t->stride(1);
    return true;
}
struct Batch { const int* table; int ld, cols; const int* row_start; const int* kv_len; int S; };
bool batch(PyObject* table, PyObject* row_start, PyObject* kv_len, int dev, Batch* out) {
    const at::Tensor *t = tensor(table), *r = tensor(row_start), *k = tensor(kv_len);
    if (!on(t, dev, at::kInt) || !on(r, dev, at::kInt) || !on(k, dev, at::kInt) || t->dim() != 2) return false;
    const int64_t S = k->numel(), cols = t->size(1);
    if (S < 1 || S > INT_MAX || t->size(0) != S || r->numel() != S + 1 || t->stride(1) != 1 || cols < 1 || (S > 1 && t->stride(0) < cols) || !r->is_contiguous() || !k->is_contiguous()) return false;
    const int64_t ld = S > 1 ? t->stride(0) : cols;
    if (ld > INT_MAX) return false;
    *out = Batch{static_cast<const int*>(t->data_ptr()), (int)ld, (int)cols, static_cast<const int*>(r->data_ptr()), static_cast<const int*>(k->data_ptr()), (int)S};
    return true;
}
bool norm_weight(PyObject* o, int dev, int64_t D, const void** out) {
    if (o == Py_None) { *out = nullptr; return true; }
    const at::Tensor* t = tensor(o);
    if (!t || !(on(t, dev, at::kBFloat16) || on(t, dev, at::kShort)) || t->dim() != 1 || t->size(0) != D || !t->is_contiguous()) return false;
    *out = t->data_ptr();
    return true;
}
const hp_kv_pages* pages(PyObject* o) { return reinterpret_cast<const hp_kv_pages*>(PyLong_AsSsize_t(o)); }
// the cache as this call sees it: a table that is part of a wider one ends with its own columns
hp_kv_pages with_columns(const hp_kv_pages* c, const Batch& b) { hp_kv_pages o = *c; o.columns = b.cols; return o; }
bool whole(PyObject* o, int64_t* out) {   // an int that fits; floats and the like are for kernels.py to judge
    if (!PyLong_CheckExact(o)) return false;
    int over; *out = PyLong_AsLongLongAndOverflow(o, &over);
    return !over && *out >= INT_MIN && *out <= INT_MAX;
}
bool real(PyObject* o, double* out) {
    if (PyFloat_CheckExact(o)) { *out = PyFloat_AS_DOUBLE(o); return true; }
    int64_t i; if (!whole(o, &i)) return false;
    *out = (double)i; return true;
}
at::TensorOptions options(int dev, at::ScalarType type) { return at::TensorOptions().dtype(type).device(at::Device(at::kCUDA, (c10::DeviceIndex)dev)); }
template <typename F> int outside(F f) { int rc; Py_BEGIN_ALLOW_THREADS rc = f(); Py_END_ALLOW_THREADS return rc; }
#define TRY try {
#define CATCH } catch (...) { PyErr_Clear(); Py_RETURN_NONE; }   // kernels.py meets the same and says it

// kv_append(pages, device, k, v, table, row_start, kv_len, rope, q, q_out, interleaved, q_norm, k_norm, eps) -> q_out; True without q
PyObject* py_kv_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    int64_t dev; double eps; Batch b; Rows q{}, qo{}, k, v; const void *qn, *kn;
    if (n != 14 || !f_append || !whole(a[1], &dev) || !real(a[13], &eps)) Py_RETURN_NONE;
    TRY
    const hp_kv_pages* c = pages(a[0]);
    const at::Tensor* kt = tensor(a[2]);
    if (c10::cuda::current_device() != dev || !kt || kt->dim() != 3 || kt->size(0) < 1 || kt->size(0) > INT_MAX || !batch(a[4], a[5], a[6], (int)dev, &b)) Py_RETURN_NONE;
    const int64_t R = kt->size(0);
    if (!rows(a[2], (int)dev, R, c->n_kv, c->head_dim, &k) || !rows(a[3], (int)dev, R, c->n_kv, c->head_dim, &v) || !norm_weight(a[11], (int)dev, c->head_dim, &qn) || !norm_weight(a[12], (int)dev, c->head_dim, &kn)) Py_RETURN_NONE;
    const float* rope = nullptr; int n_pos = 0, n_rot = 0, n_head = 0;
    if (a[7] != Py_None) {
        const at::Tensor* t = tensor(a[7]);
        if (!on(t, (int)dev, at::kFloat) || t->dim() != 3 || t->size(2) != 2 || !t->is_contiguous() || t->size(0) > INT_MAX || t->size(1) > 1024) Py_RETURN_NONE;
        rope = static_cast<const float*>(t->data_ptr()); n_pos = (int)t->size(0); n_rot = 2 * (int)t->size(1);
    }
    at::Tensor out;
    if (a[8] != Py_None) {
        const at::Tensor* t = tensor(a[8]);
        if (!t || t->dim() != 3 || t->size(1) > INT_MAX || !rows(a[8], (int)dev, R, t->size(1), c->head_dim, &q)) Py_RETURN_NONE;
        n_head = (int)t->size(1);
        if (a[9] == Py_None) { out = at::empty({R, n_head, c->head_dim}, options((int)dev, at::kFloat)); qo = Rows{static_cast<float*>(out.data_ptr()), (long long)n_head * c->head_dim, c->head_dim}; }
        else { if (!rows(a[9], (int)dev, R, n_head, c->head_dim, &qo)) Py_RETURN_NONE; out = *tensor(a[9]); }
    } else if (a[9] != Py_None) Py_RETURN_NONE;
    const hp_kv_pages view = with_columns(c, b);
    const int inter = PyObject_IsTrue(a[10]);
    if (inter < 0) PyErr_Clear();
    void* s = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
    if (inter < 0 || outside([&] { return f_append(q.p, q.ld, q.hs, qo.p, qo.ld, qo.hs, n_head, k.p, k.ld, k.hs, v.p, v.ld, v.hs, qn, kn, rope, n_pos, n_rot, inter, b.table, b.ld, b.row_start, b.kv_len, b.S, (int)R, &view, (float)eps, s); })) Py_RETURN_NONE;
    if (a[8] == Py_None) Py_RETURN_TRUE;
    if (a[9] != Py_None) { Py_INCREF(a[9]); return a[9]; }
    return THPVariable_Wrap(std::move(out));
    CATCH
}
// kv_read(pages, device, table, row_start, kv_len, R) -> (k, v)
PyObject* py_kv_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    int64_t dev, R; Batch b;
    if (n != 6 || !f_read || !whole(a[1], &dev) || !whole(a[5], &R) || R < 1) Py_RETURN_NONE;
    TRY
    const hp_kv_pages* c = pages(a[0]);
    if (c10::cuda::current_device() != dev || !batch(a[2], a[3], a[4], (int)dev, &b)) Py_RETURN_NONE;
    const hp_kv_pages view = with_columns(c, b);
    at::Tensor k = at::empty({R, c->n_kv, c->head_dim}, options((int)dev, at::kHalf)), v = at::empty({R, c->n_kv, c->head_dim}, options((int)dev, at::kHalf));
    void* s = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
    if (outside([&] { return f_read(b.table, b.ld, b.row_start, b.kv_len, b.S, (int)R, &view, k.data_ptr(), v.data_ptr(), (long long)c->n_kv * c->head_dim, c->head_dim, s); })) Py_RETURN_NONE;
    PyObject *pk = THPVariable_Wrap(std::move(k)), *pv = THPVariable_Wrap(std::move(v)), *r = pk && pv ? PyTuple_Pack(2, pk, pv) : nullptr;
    Py_XDECREF(pk); Py_XDECREF(pv);
    return r;
    CATCH
}
// attn_paged(pages, device, q, gate, table, row_start, kv_len, max_rows, max_kv, scale, window, n_sink) -> out
PyObject* py_attn_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
    int64_t dev, max_rows, max_kv, window, n_sink; double scale; Batch b; Rows q, g{};
    if (n != 12 || !f_attn || !f_bytes || !whole(a[1], &dev) || !whole(a[7], &max_rows) || !whole(a[8], &max_kv) || !whole(a[10], &window) || !whole(a[11], &n_sink)) Py_RETURN_NONE;
    TRY
    const hp_kv_pages* c = pages(a[0]);
    const at::Tensor* t = tensor(a[2]);
    if (a[9] == Py_None) scale = 1.0 / std::sqrt((double)c->head_dim); else if (!real(a[9], &scale)) Py_RETURN_NONE;
    if (c10::cuda::current_device() != dev || !t || t->dim() != 3 || t->size(0) < 1 || t->size(0) > INT_MAX || t->size(1) > INT_MAX || !batch(a[4], a[5], a[6], (int)dev, &b)) Py_RETURN_NONE;
    const int64_t R = t->size(0), H = t->size(1);
    if (!rows(a[2], (int)dev, R, H, c->head_dim, &q) || (a[3] != Py_None && !rows(a[3], (int)dev, R, H, c->head_dim, &g))) Py_RETURN_NONE;
    const hp_kv_pages view = with_columns(c, b);
    const size_t bytes = f_bytes(b.ld, b.S, (int)R, (int)max_rows, (int)max_kv, (int)H, (int)window, (int)n_sink, &view);
    if (!bytes) Py_RETURN_NONE;
    at::Tensor out = at::empty({R, H, c->head_dim}, options((int)dev, at::kFloat)), ws = at::empty({(int64_t)bytes}, options((int)dev, at::kByte));
    void* s = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
    if (outside([&] { return f_attn(q.p, q.ld, q.hs, g.p, g.ld, g.hs, (int)H, b.table, b.ld, b.row_start, b.kv_len, b.S, (int)R, (int)max_rows, (int)max_kv, &view, (float)scale, (int)window, (int)n_sink,
                                    static_cast<float*>(out.data_ptr()), nullptr, nullptr, ws.data_ptr(), s); })) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
    CATCH
}
// rope_table(n_pos, n_rot, base, scaling, factor, orig_ctx, beta_fast, beta_slow, attn_factor) -> table on the current device
PyObject* py_rope_table(PyObject*, PyObject* const* a, Py_ssize_t n) {
    int64_t n_pos, n_rot, kind, orig; double base, factor, fast, slow, mul;
    if (n != 9 || !f_table || !whole(a[0], &n_pos) || !whole(a[1], &n_rot) || !real(a[2], &base) || !whole(a[3], &kind) || !real(a[4], &factor) || !whole(a[5], &orig) || !real(a[6], &fast) || !real(a[7], &slow) || !real(a[8], &mul) ||
        n_pos < 1 || n_rot < 2 || n_rot > 256) Py_RETURN_NONE;
    TRY
    const int dev = c10::cuda::current_device();
    at::Tensor out = at::empty({n_pos, n_rot / 2, 2}, options(dev, at::kFloat));
    void* s = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
    if (outside([&] { return f_table(static_cast<float*>(out.data_ptr()), (int)n_pos, (int)n_rot, base, (int)kind, factor, (int)orig, fast, slow, mul, s); })) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
    CATCH
}
// bind(name, address)
PyObject* py_bind(PyObject*, PyObject* args) {
    const char* name; Py_ssize_t at;
    if (!PyArg_ParseTuple(args, "sn", &name, &at)) return nullptr;
    void* p = reinterpret_cast<void*>(at);
    if (!std::strcmp(name, "hp_kv_append")) f_append = reinterpret_cast<decltype(f_append)>(p);
    else if (!std::strcmp(name, "hp_kv_read")) f_read = reinterpret_cast<decltype(f_read)>(p);
    else if (!std::strcmp(name, "hp_attn_paged")) f_attn = reinterpret_cast<decltype(f_attn)>(p);
    else if (!std::strcmp(name, "hp_attn_paged_workspace_bytes")) f_bytes = reinterpret_cast<decltype(f_bytes)>(p);
    else if (!std::strcmp(name, "hp_rope_table")) f_table = reinterpret_cast<decltype(f_table)>(p);
    else { PyErr_Format(PyExc_KeyError, "%s", name); return nullptr; }
    Py_RETURN_NONE;
}
#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f))
PyMethodDef methods[] = {{"bind", py_bind, METH_VARARGS, nullptr}, {"kv_append", FAST(py_kv_append), METH_FASTCALL, nullptr}, {"kv_read", FAST(py_kv_read), METH_FASTCALL, nullptr},
                         {"attn_paged", FAST(py_attn_paged), METH_FASTCALL, nullptr}, {"rope_table", FAST(py_rope_table), METH_FASTCALL, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace
PyMODINIT_FUNC PyInit__tensors(void) {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch", TORCH_VERSION) < 0) { Py_DECREF(m); return nullptr; }   // kernels.py uses it with this version alone
    return m;
}
