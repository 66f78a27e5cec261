// serving_binding.cpp -- the Python side of the batched decode operators
// (serving.py) as a CPython module: checks the torch tensors, allocates the
// results on torch's current stream and calls the C ABI (include/tmac_cuda.h).  A
// step of a small batch takes a few microseconds on the GPU, so the checks must
// not take more; from Python through ctypes they took 15 to 20.
//
// Every entry takes its arguments by position, in the order of its comment; None
// stands for an absent tensor.  Refusals raise the class given to set_error_class
// with a TMAC_ERR_* code and a message.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>
#include <string>

#include "../../include/tmac_cuda.h"

namespace {

PyObject* g_error = nullptr;  // TmacError(code, message)

struct Refusal {
    int code;
    std::string message;
};
[[noreturn]] void refuse(int code, const std::string& message) { throw Refusal{code, message}; }
void check(int rc)
{
    if (rc) refuse(rc, tmac_last_error());
}
// Calls f without the interpreter's lock: a launch waits while a stream's queue is full,
// and other Python threads must not wait with it.
template <typename F>
int unlocked(F&& f)
{
    struct Lock {
        PyThreadState* state = PyEval_SaveThread();
        ~Lock() { PyEval_RestoreThread(state); }
    } lock;
    return f();
}
PyObject* raise(const Refusal& r)
{
    PyObject* e = g_error ? PyObject_CallFunction(g_error, "is", r.code, r.message.c_str()) : nullptr;
    if (e) {
        PyErr_SetObject(g_error, e);
        Py_DECREF(e);
    } else if (!PyErr_Occurred()) {
        PyErr_SetString(PyExc_RuntimeError, r.message.c_str());
    }
    return nullptr;
}

int type_of(const at::Tensor& t)
{
    switch (t.scalar_type()) {
    case at::kFloat: return TMAC_TYPE_F32;
    case at::kHalf: return TMAC_TYPE_F16;
    case at::kBFloat16: return TMAC_TYPE_BF16;
    default: return -1;
    }
}
const at::Tensor& tensor(PyObject* o, const char* name)
{
    if (!THPVariable_Check(o)) refuse(TMAC_ERR_INVALID, std::string(name) + " must be a torch tensor");
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.requires_grad() && c10::GradMode::is_enabled())
        refuse(TMAC_ERR_INVALID, std::string(name) + " requires grad, and these operators have no gradient: detach it, or call under torch.no_grad()");
    return t;
}
int whole(PyObject* o, const char* name)
{
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    if (v < INT_MIN || v > INT_MAX) refuse(TMAC_ERR_SHAPE, std::string(name) + " is out of range");
    return (int)v;
}
int whole(int64_t v, const char* name)
{
    if (v > INT_MAX) refuse(TMAC_ERR_SHAPE, std::string(name) + " is out of range");
    return (int)v;
}
// The address of a contiguous tensor of that type and size on the device; null for None.
const void* vector(PyObject* o, const char* name, at::ScalarType type, at::IntArrayRef sizes, const at::Device& device)
{
    if (o == Py_None) return nullptr;
    const at::Tensor& t = tensor(o, name);
    if (t.scalar_type() != type || t.sizes() != sizes || t.device() != device || !t.is_contiguous()) {
        std::string s = std::string(name) + " must be a contiguous " + at::toString(type) + " tensor of sizes [";
        for (int64_t n : sizes) s += std::to_string(n) + (n == sizes.back() ? "" : ", ");
        refuse(TMAC_ERR_INVALID, s + "] on the cache's or logits' device");
    }
    return t.data_ptr();
}
// Checks [tokens, heads, dim] whose heads adjoin; the distance of two tokens.
int64_t rows(const at::Tensor& t, const char* name, int64_t dim, const at::Device& device)
{
    if (t.dim() != 3 || t.size(2) != dim)
        refuse(TMAC_ERR_SHAPE, std::string(name) + " must be [tokens, heads, " + std::to_string(dim) + "]");
    if (t.device() != device || (t.stride(2) != 1 && dim > 1) || (t.stride(1) != dim && t.size(1) > 1))
        refuse(TMAC_ERR_INVALID, std::string(name) + " must lie on the cache's device with the heads of a token adjoining");
    return t.size(0) > 1 ? t.stride(0) : t.size(1) * dim;
}
tmac_paged_cache cache_of(PyObject* ko, PyObject* vo)
{
    const at::Tensor &k = tensor(ko, "k"), &v = tensor(vo, "v");
    if (k.dim() != 4 || k.sizes() != v.sizes())
        refuse(TMAC_ERR_SHAPE, "k and v must both be [n_pages, kv_heads, page_size, head_dim]");
    const int type = type_of(k);
    if (type < 0 || v.scalar_type() != k.scalar_type())
        refuse(TMAC_ERR_TYPE, "k and v must both be float32, float16 or bfloat16");
    if (!k.is_cuda() || v.device() != k.device() || !k.is_contiguous() || !v.is_contiguous())
        refuse(TMAC_ERR_INVALID, "k and v must be contiguous tensors on one CUDA device");
    tmac_paged_cache c = {};
    c.k = k.data_ptr();
    c.v = v.data_ptr();
    c.n_pages = k.size(0);
    c.type = type;
    c.kv_heads = whole(k.size(1), "kv_heads");
    c.page_size = whole(k.size(2), "page_size");
    c.head_dim = whole(k.size(3), "head_dim");
    c.device = k.device().index();
    return c;
}
void* stream_of(const at::Device& device) { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }

template <typename F>
PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F&& f)
{
    HANDLE_TH_ERRORS
    if (got != want) return PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, got);
    try {
        return f();
    } catch (const Refusal& r) {
        return raise(r);
    }
    END_HANDLE_TH_ERRORS
}

// check_cache(k, v)
PyObject* py_check_cache(PyObject*, PyObject* const* o, Py_ssize_t n)
{
    return guarded(n, 2, [&]() -> PyObject* {
        cache_of(o[0], o[1]);
        Py_RETURN_NONE;
    });
}

// rope_append(k_pages, v_pages, q, k, v, pos, tables, cos, sin, seq, starts, interleaved, bias, q_out)
PyObject* py_rope_append(PyObject*, PyObject* const* o, Py_ssize_t n)
{
    return guarded(n, 14, [&]() -> PyObject* {
        const tmac_paged_cache c = cache_of(o[0], o[1]);
        const at::Tensor &pages = THPVariable_Unpack(o[0]), &q = tensor(o[2], "q"), &k = tensor(o[3], "k"), &v = tensor(o[4], "v");
        const at::Device dev = pages.device();
        const int type = type_of(q), dim = c.head_dim;
        if (type < 0 || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
            refuse(TMAC_ERR_TYPE, "q, k and v must be of one type: float32, float16 or bfloat16");
        const int64_t qs = rows(q, "q", dim, dev), ks = rows(k, "k", dim, dev), vs = rows(v, "v", dim, dev);
        const int64_t tokens = q.size(0), heads = q.size(1);
        if (k.sizes() != v.sizes() || k.size(0) != tokens || k.size(1) != c.kv_heads)
            refuse(TMAC_ERR_SHAPE, "k and v must have q's tokens and the cache's heads");
        const at::Tensor &tables = tensor(o[6], "tables"), &cos = tensor(o[7], "cos");
        if (tables.dim() != 2 || cos.dim() != 2)
            refuse(TMAC_ERR_SHAPE, "tables must be [n_seq, width] and cos [max_pos, rot_dim / 2]");
        const auto* bias = (const float*)vector(o[12], "bias", at::kFloat, {(heads + 2 * c.kv_heads) * dim}, dev);
        const auto* pos = (const int32_t*)vector(o[5], "pos", at::kInt, {tokens}, dev);
        const auto* seq = (const int32_t*)vector(o[9], "seq", at::kInt, {tokens}, dev);
        const auto* starts = (const int32_t*)vector(o[10], "starts", at::kInt, {tables.size(0)}, dev);
        const auto* table = (const int32_t*)vector(o[6], "tables", at::kInt, tables.sizes(), dev);
        const auto* cosp = (const float*)vector(o[7], "cos", at::kFloat, cos.sizes(), dev);
        const auto* sinp = (const float*)vector(o[8], "sin", at::kFloat, cos.sizes(), dev);
        const int interleaved = PyObject_IsTrue(o[11]);
        if (interleaved < 0) throw python_error();
        at::Tensor out;
        if (o[13] == Py_None) {
            out = at::empty({tokens, heads, dim}, pages.options());
        } else {
            vector(o[13], "q_out", pages.scalar_type(), {tokens, heads, dim}, dev);
            out = THPVariable_Unpack(o[13]);
        }
        const int n_heads = whole(heads, "heads"), n_tokens = whole(tokens, "tokens"), n_seq = whole(tables.size(0), "n_seq");
        const int width = whole(tables.size(1), "width"), max_pos = whole(cos.size(0), "max_pos"), rot = whole(2 * cos.size(1), "rot_dim");
        check(unlocked([&] {
            return tmac_rope_append(&c, type, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, n_heads, n_tokens, bias, seq, pos, starts,
                                    table, n_seq, width, cosp, sinp, max_pos, rot, interleaved, out.data_ptr(), stream_of(dev));
        }));
        return THPVariable_Wrap(out);
    });
}

// prefix_attention(q, k_pages, v_pages, tables, own_lens, prefix_pages, prefix_len, prefix_lens, q_start, max_q,
//                  max_own, scale, out)
PyObject* py_prefix_attention(PyObject*, PyObject* const* o, Py_ssize_t n)
{
    return guarded(n, 13, [&]() -> PyObject* {
        const tmac_paged_cache c = cache_of(o[1], o[2]);
        const at::Tensor &pages = THPVariable_Unpack(o[1]), &q = tensor(o[0], "q"), &tables = tensor(o[3], "tables");
        const at::Device dev = pages.device();
        if (q.scalar_type() != pages.scalar_type()) refuse(TMAC_ERR_TYPE, "q must have the cache's type");
        const int64_t qs = rows(q, "q", c.head_dim, dev);
        if (tables.dim() != 2) refuse(TMAC_ERR_SHAPE, "tables must be [batch, width]");
        const int tokens = whole(q.size(0), "tokens"), heads = whole(q.size(1), "heads"), batch = whole(tables.size(0), "batch");
        const int width = whole(tables.size(1), "width"), max_q = whole(o[9], "max_q"), prefix_len = whole(o[6], "prefix_len");
        const int max_own = o[10] == Py_None ? whole(tables.size(1) * c.page_size, "max_own") : whole(o[10], "max_own");
        const int32_t* list = nullptr;
        if (o[5] != Py_None) {
            const int64_t count = tensor(o[5], "prefix_pages").numel();
            list = (const int32_t*)vector(o[5], "prefix_pages", at::kInt, {count}, dev);
            if (prefix_len > count * c.page_size) refuse(TMAC_ERR_SHAPE, "prefix_pages do not cover prefix_len");
        }
        const auto* own = (const int32_t*)vector(o[4], "own_lens", at::kInt, {batch}, dev);
        const auto* table = (const int32_t*)vector(o[3], "tables", at::kInt, tables.sizes(), dev);
        const auto* shared = (const int32_t*)vector(o[7], "prefix_lens", at::kInt, {batch}, dev);
        const auto* starts = (const int32_t*)vector(o[8], "q_start", at::kInt, {batch + 1}, dev);
        double scale = 1.0 / std::sqrt((double)c.head_dim);
        if (o[11] != Py_None) {
            scale = PyFloat_AsDouble(o[11]);
            if (scale == -1.0 && PyErr_Occurred()) throw python_error();
        }
        size_t need = 0;
        check(tmac_prefix_attention_workspace(&c, heads, tokens, batch, max_q, prefix_len, max_own, &need));
        at::Tensor out, work;
        if (o[12] == Py_None) {
            out = at::empty({tokens, heads, c.head_dim}, pages.options());
        } else {
            out = tensor(o[12], "out");
            if (out.scalar_type() != q.scalar_type() || out.sizes() != q.sizes())
                refuse(TMAC_ERR_INVALID, "out must have q's type and shape");
        }
        const int64_t os = rows(out, "out", c.head_dim, dev);
        if (need) work = at::empty({(int64_t)need}, pages.options().dtype(at::kByte));
        check(unlocked([&] {
            return tmac_prefix_attention(&c, q.data_ptr(), qs, heads, tokens, batch, starts, max_q, list, prefix_len, shared, table, width, own,
                                         max_own, (float)scale, out.data_ptr(), os, need ? work.data_ptr() : nullptr, need, stream_of(dev));
        }));
        if (o[12] != Py_None) {
            Py_INCREF(o[12]);
            return o[12];
        }
        return THPVariable_Wrap(out);
    });
}

// sample(logits, u, temperature, top_k, top_p, min_p)
PyObject* py_sample(PyObject*, PyObject* const* o, Py_ssize_t n)
{
    return guarded(n, 6, [&]() -> PyObject* {
        const at::Tensor& l = tensor(o[0], "logits");
        const int type = type_of(l);
        if (type < 0) refuse(TMAC_ERR_TYPE, "logits must be float32, float16 or bfloat16");
        if (l.dim() != 2 || (l.size(1) > 1 && l.stride(1) != 1))
            refuse(TMAC_ERR_SHAPE, "logits must be [batch, vocab] with adjoining values");
        if (!l.is_cuda()) refuse(TMAC_ERR_INVALID, "logits must lie on a CUDA device");
        const at::Device dev = l.device();
        const int batch = whole(l.size(0), "batch"), vocab = whole(l.size(1), "vocab");
        const auto* u = (const float*)vector(o[1], "u", at::kFloat, {batch}, dev);
        const auto* temperature = (const float*)vector(o[2], "temperature", at::kFloat, {batch}, dev);
        const auto* top_k = (const int32_t*)vector(o[3], "top_k", at::kInt, {batch}, dev);
        const auto* top_p = (const float*)vector(o[4], "top_p", at::kFloat, {batch}, dev);
        const auto* min_p = (const float*)vector(o[5], "min_p", at::kFloat, {batch}, dev);
        at::Tensor tokens = at::empty({batch}, l.options().dtype(at::kInt)), probs = at::empty({batch}, l.options().dtype(at::kFloat));
        check(unlocked([&] {
            return tmac_sample(l.data_ptr(), type, batch > 1 ? l.stride(0) : vocab, batch, vocab, u, temperature, top_k, top_p, min_p,
                               tokens.data_ptr<int32_t>(), probs.data_ptr<float>(), dev.index(), stream_of(dev));
        }));
        return Py_BuildValue("NN", THPVariable_Wrap(tokens), THPVariable_Wrap(probs));
    });
}

// set_error_class(class)
PyObject* py_set_error_class(PyObject*, PyObject* const* o, Py_ssize_t n)
{
    return guarded(n, 1, [&]() -> PyObject* {
        Py_INCREF(o[0]);
        Py_XDECREF(g_error);
        g_error = o[0];
        Py_RETURN_NONE;
    });
}

#define ENTRY(name) {#name, (PyCFunction)(void (*)(void))py_##name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(check_cache), ENTRY(rope_append), ENTRY(prefix_attention), ENTRY(sample), ENTRY(set_error_class),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" PyMODINIT_FUNC PyInit__serving() { return PyModule_Create(&module); }
