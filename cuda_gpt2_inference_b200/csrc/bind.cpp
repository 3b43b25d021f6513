// bind.cpp -- Python entries of the operators for batches of requests and drafted tokens.
//
// A step of a small batch launches kernels of 3 to 10 us.  Checking ten tensors in Python and
// converting twenty arguments with ctypes costs 11 to 18 us a call, so these operators take
// their tensors here: the same checks, the C ABI of libgpt2b.so behind them (by the addresses
// that the package looked up), and 3 to 3.5 us a call with its launch (the attention, two launches: 5.5).
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cstring>
#include <exception>
#include <initializer_list>
#include <optional>
#include <string>

#include "gpt2_b200.h"

namespace {

PyObject* g_error = nullptr;  // Gpt2bError(status, where)

#define GPT2B_BOUND(X)              \
    X(gpt2b_kv_block_tables)        \
    X(gpt2b_kv_cache_write_w4)      \
    X(gpt2b_kv_cache_read_w4)       \
    X(gpt2b_attention_forward_paged_w4) \
    X(gpt2b_softmax_probs)          \
    X(gpt2b_verify_draft_tokens)
#define X(f) decltype(&f) p_##f = nullptr;
GPT2B_BOUND(X)
#undef X

struct Refused {
    int status;
    std::string what;
};
struct PyRaised {};  // a Python error is set

[[noreturn]] void refuse(const std::string& what, int status = GPT2B_ERR_INVALID_ARG) { throw Refused{status, what}; }

const char* type_name(at::ScalarType t) {
    switch (t) {
        case at::kInt: return "torch.int32";
        case at::kLong: return "torch.int64";
        case at::kFloat: return "torch.float32";
        case at::kBFloat16: return "torch.bfloat16";
        default: return "torch.uint8";
    }
}

// A tensor of that type and rank, contiguous (rows: only within its rows).
const at::Tensor& tensor(PyObject* o, const char* name, at::ScalarType type, int64_t ndim, bool rows = false) {
    const at::Tensor* t = THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr;
    if (!t || t->scalar_type() != type || t->dim() != ndim || t->layout() != at::kStrided)
        refuse(std::string(name) + " must be a " + std::to_string(ndim) + "-d " + type_name(type) + " tensor");
    if (!t->is_contiguous() &&
        !(rows && ndim == 2 && (t->size(1) <= 1 || t->stride(1) == 1) && (t->size(0) <= 1 || t->stride(0) >= t->size(1))))
        refuse(std::string(name) + " must be contiguous");
    return *t;
}
int size32(int64_t n, const char* what) {
    if (n < 0 || n > INT_MAX) refuse(std::string(what) + " does not fit 32 bits", GPT2B_ERR_UNSUPPORTED);
    return (int)n;
}
int dim32(const at::Tensor& t, int64_t d) { return size32(t.size(d), "a tensor's size"); }
int integer(PyObject* o, const char* name) {
    int over = 0;
    const long long v = PyLong_AsLongLongAndOverflow(o, &over);
    if (v == -1 && !over && PyErr_Occurred()) throw PyRaised{};
    if (over || v < INT_MIN || v > INT_MAX) refuse(std::string(name) + " does not fit 32 bits");
    return (int)v;
}
double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw PyRaised{};
    return v;
}
// elements between the rows of a 2-d tensor (its width where it has one row: the stride then says nothing)
int pitch(const at::Tensor& t) { return size32(t.size(0) > 1 ? t.stride(0) : t.size(1), "a row pitch"); }

// the same of 16-byte rows: a single row has no pitch that could be odd
int qkv_pitch(const at::Tensor& t) { return t.size(0) > 1 ? pitch(t) : size32((t.size(1) + 7) / 8 * 8, "a row pitch"); }

template <typename T> T* ptr(const at::Tensor& t) { return static_cast<T*>(t.data_ptr()); }

// The one CUDA device that holds every tensor, made current, and the stream to launch on.
struct Where {
    std::optional<c10::cuda::CUDAGuard> guard;
    gpt2b_stream_t stream = nullptr;
    Where(std::initializer_list<const at::Tensor*> all, PyObject* given) {
        const at::Device dev = (*all.begin())->device();
        bool same = dev.is_cuda();
        for (const at::Tensor* t : all) same = same && t->device() == dev;
        if (!same) refuse("the tensors must be on one CUDA device");
        if (dev.index() != c10::cuda::current_device()) guard.emplace(dev);
        if (given == Py_None) {
            stream = (gpt2b_stream_t)c10::cuda::getCurrentCUDAStream(dev.index()).stream();
        } else {
            PyObject* s = PyObject_GetAttrString(given, "cuda_stream");
            if (!s) throw PyRaised{};
            stream = (gpt2b_stream_t)PyLong_AsVoidPtr(s);
            Py_DECREF(s);
            if (!stream && PyErr_Occurred()) throw PyRaised{};
        }
    }
};

void raise(const char* where, int status, const std::string& what) {
    const std::string text = what.empty() ? std::string(where) : std::string(where) + ": " + what;
    PyObject* e = PyObject_CallFunction(g_error, "is", status, text.c_str());
    if (!e) return;
    PyErr_SetObject(g_error, e);
    Py_DECREF(e);
}

// Runs body(args) -> status; no C++ exception leaves it.
template <typename F> PyObject* entry(const char* where, Py_ssize_t want, Py_ssize_t got, F&& body) {
    if (want != got) return PyErr_Format(PyExc_TypeError, "%s takes %zd arguments (%zd given)", where, want, got);
    if (!g_error) return PyErr_Format(PyExc_RuntimeError, "the binding is not initialised");
    try {
        const int status = body();
        if (status == GPT2B_OK) Py_RETURN_NONE;
        raise(where, status, "");
    } catch (const Refused& r) {
        raise(where, r.status, r.what);
    } catch (const PyRaised&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}
// Without the interpreter lock, which comes back however f is left (a size or a data pointer may be refused in it).
struct Unlocked {
    PyThreadState* state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
};
template <typename F> int launch(F&& f) {
    const Unlocked u;
    return f();
}

struct Cache {
    const at::Tensor &codes, &scales;
    int blocks, NKV, bs, hs;
};
Cache cache_of(PyObject* kv_cache, PyObject* kv_scale) {
    const at::Tensor& c = tensor(kv_cache, "kv_cache", at::kByte, 5);
    const at::Tensor& s = tensor(kv_scale, "kv_scale", at::kBFloat16, 6);
    const int64_t half = c.size(4);
    if (c.size(1) != 2 || s.size(0) != c.size(0) || s.size(1) != 2 || s.size(2) != c.size(2) || s.size(3) != c.size(3) ||
        s.size(4) != half / 32 || s.size(5) != 2)
        refuse("kv_cache is [blocks, 2, NKV, block_size, hs/2] and kv_scale [blocks, 2, NKV, block_size, hs/64, 2]");
    if ((half != 32 && half != 64) || c.size(3) % 16 != 0 || c.size(3) == 0)
        refuse("head size 64 or 128, block size a multiple of 16", GPT2B_ERR_UNSUPPORTED);
    return Cache{c, s, dim32(c, 0), dim32(c, 2), dim32(c, 3), (int)(2 * half)};
}

PyObject* kv_block_tables(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return entry("kv_block_tables", 14, n, [&] {
        const at::Tensor& table = tensor(a[0], "block_table", at::kInt, 2);
        const at::Tensor& slots = tensor(a[1], "slot_map", at::kLong, 1);
        const int64_t B = table.size(0), R = slots.size(0);
        static const char* names[] = {"positions", "row_start", "seq_lens", "blocks_out", "free_left",
                                      "ctx_lens", "new_lens", "blocks_have", "free_list", "free_count"};
        const int64_t sizes[] = {R, B + 1, B, B, 1, B, B, B, -1, 1};
        const at::Tensor* t[10];
        for (int i = 0; i < 10; i++) {
            t[i] = &tensor(a[2 + i], names[i], at::kInt, 1);
            if (sizes[i] >= 0 && t[i]->size(0) != sizes[i])
                refuse(std::string(names[i]) + " must have " + std::to_string(sizes[i]) + " entries");
        }
        const int bs = integer(a[12], "block_size");
        const Where w({&table, &slots, t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7], t[8], t[9]}, a[13]);
        return launch([&] {
            return p_gpt2b_kv_block_tables(ptr<int>(table), ptr<long long>(slots), ptr<int>(*t[0]), ptr<int>(*t[1]), ptr<int>(*t[2]),
                                           ptr<int>(*t[3]), ptr<int>(*t[4]), ptr<int>(*t[5]), ptr<int>(*t[6]), ptr<int>(*t[7]),
                                           ptr<int>(*t[8]), ptr<int>(*t[9]), dim32(table, 0), dim32(table, 1), bs,
                                           dim32(slots, 0), dim32(*t[8], 0), w.stream);
        });
    });
}

PyObject* kv_cache_write_w4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return entry("kv_cache_write_w4", 6, n, [&] {
        const Cache c = cache_of(a[0], a[1]);
        const at::Tensor& qkv = tensor(a[2], "qkv", at::kBFloat16, 2, true);
        const at::Tensor& slots = tensor(a[3], "slot_map", at::kLong, 1);
        const int NH = integer(a[4], "NH"), rows = dim32(qkv, 0), ld = qkv_pitch(qkv);
        if (slots.size(0) != rows || qkv.size(1) < ((int64_t)NH + 2 * c.NKV) * c.hs)
            refuse("slot_map has one entry a row, a row Q, K and V of every head");
        const Where w({&c.codes, &c.scales, &qkv, &slots}, a[5]);
        return launch([&] {
            return p_gpt2b_kv_cache_write_w4(ptr<uint8_t>(c.codes), ptr<uint16_t>(c.scales), ptr<uint16_t>(qkv), ptr<long long>(slots),
                                             rows, NH, c.NKV, c.hs, ld, c.blocks, c.bs, w.stream);
        });
    });
}

PyObject* kv_cache_read_w4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return entry("kv_cache_read_w4", 5, n, [&] {
        const at::Tensor& out = tensor(a[0], "out", at::kBFloat16, 4);
        const Cache c = cache_of(a[1], a[2]);
        const at::Tensor& slots = tensor(a[3], "slot_map", at::kLong, 1);
        if (out.size(0) != slots.size(0) || out.size(1) != 2 || out.size(2) != c.NKV || out.size(3) != c.hs)
            refuse("out is [rows, 2, NKV, hs]");
        const int rows = dim32(out, 0);
        const Where w({&out, &c.codes, &c.scales, &slots}, a[4]);
        return launch([&] {
            return p_gpt2b_kv_cache_read_w4(ptr<uint16_t>(out), ptr<uint8_t>(c.codes), ptr<uint16_t>(c.scales), ptr<long long>(slots),
                                            rows, c.NKV, c.hs, c.blocks, c.bs, w.stream);
        });
    });
}

PyObject* attention_forward_paged_w4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return entry("attention_forward_paged_w4", 12, n, [&] {
        const at::Tensor& out = tensor(a[0], "out", at::kBFloat16, 2);
        const at::Tensor& qkv = tensor(a[1], "qkv", at::kBFloat16, 2, true);
        const Cache c = cache_of(a[2], a[3]);
        const at::Tensor& table = tensor(a[4], "block_table", at::kInt, 2);
        const at::Tensor& lens = tensor(a[5], "seq_lens", at::kInt, 1);
        const at::Tensor& start = tensor(a[6], "row_start", at::kInt, 1);
        const int NH = integer(a[7], "NH"), max_q = integer(a[8], "max_q");
        const at::Tensor& ws = tensor(a[9], "workspace", at::kByte, 1);
        const int rows = dim32(qkv, 0), ld = qkv_pitch(qkv), B = dim32(table, 0), max_blocks = dim32(table, 1);
        if (qkv.size(1) < ((int64_t)NH + 2 * c.NKV) * c.hs || out.size(0) != rows || out.size(1) != (int64_t)NH * c.hs)
            refuse("qkv is [rows, >= (NH + 2 NKV) hs] and out [rows, NH hs]");
        if (lens.size(0) != B || start.size(0) != (int64_t)B + 1) refuse("seq_lens has B entries and row_start B + 1");
        const float scale = a[10] == Py_None ? (c.hs == 64 ? 0.125f : 0.08838834764831845f) : (float)number(a[10]);
        const Where w({&out, &qkv, &c.codes, &c.scales, &table, &lens, &start, &ws}, a[11]);
        return launch([&] {
            return p_gpt2b_attention_forward_paged_w4(ptr<uint16_t>(out), ptr<uint16_t>(qkv), ptr<uint8_t>(c.codes),
                                                      ptr<uint16_t>(c.scales), ptr<int>(table), ptr<int>(lens), ptr<int>(start), B,
                                                      rows, NH, c.NKV, c.hs, ld, c.blocks, c.bs, max_blocks, max_q, scale,
                                                      ptr<void>(ws), (size_t)ws.size(0), w.stream);
        });
    });
}

PyObject* softmax_probs(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return entry("softmax_probs", 5, n, [&] {
        const at::Tensor& probs = tensor(a[0], "probs", at::kFloat, 2, true);
        const at::Tensor& logits = tensor(a[1], "logits", at::kFloat, 2, true);
        const double T64 = number(a[2]);
        const float T = (float)T64;
        if (T == 0.0f && T64 != 0.0) refuse("temperature is 0 or at least 1e-30");  // not rounded to 0, which is greedy
        const int V = a[3] == Py_None ? dim32(logits, 1) : integer(a[3], "V");
        if (probs.size(0) != logits.size(0) || probs.size(1) < V || logits.size(1) < V)
            refuse("probs and logits have the same rows, of at least V columns");
        const Where w({&probs, &logits}, a[4]);
        return launch([&] {
            return p_gpt2b_softmax_probs(ptr<float>(probs), ptr<float>(logits), dim32(logits, 0), V, pitch(logits), pitch(probs), T,
                                         w.stream);
        });
    });
}

PyObject* verify_draft_tokens(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return entry("verify_draft_tokens", 9, n, [&] {
        const at::Tensor& out = tensor(a[0], "out_tokens", at::kInt, 2);
        const at::Tensor& taken = tensor(a[1], "n_accepted", at::kInt, 1);
        const at::Tensor& tokens = tensor(a[2], "tokens", at::kInt, 1);
        const at::Tensor& p = tensor(a[3], "target_probs", at::kFloat, 2, true);
        const at::Tensor& q = a[4] == Py_None ? p : tensor(a[4], "draft_probs", at::kFloat, 2, true);
        const at::Tensor& start = tensor(a[5], "row_start", at::kInt, 1);
        const at::Tensor& ua = tensor(a[6], "u_accept", at::kFloat, 1);
        const at::Tensor& us = tensor(a[7], "u_sample", at::kFloat, 1);
        const int B = dim32(out, 0), rows = dim32(p, 0), V = dim32(p, 1);
        if (taken.size(0) != B || start.size(0) != (int64_t)B + 1 || us.size(0) != B)
            refuse("n_accepted and u_sample have B entries, row_start B + 1");
        if (tokens.size(0) != rows || ua.size(0) != rows) refuse("tokens and u_accept have one entry a row");
        if (q.size(0) != rows || q.size(1) != V) refuse("draft_probs has target_probs' shape");
        const Where w({&out, &taken, &tokens, &p, &q, &start, &ua, &us}, a[8]);
        return launch([&] {
            return p_gpt2b_verify_draft_tokens(ptr<int>(out), ptr<int>(taken), ptr<int>(tokens), ptr<float>(p),
                                               a[4] == Py_None ? nullptr : ptr<float>(q), ptr<int>(start), ptr<float>(ua),
                                               ptr<float>(us), B, rows, V, pitch(p), pitch(q), dim32(out, 1), w.stream);
        });
    });
}

// init(error class, {function name: address})
PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 2 || !PyType_Check(a[0]) || !PyDict_Check(a[1])) return PyErr_Format(PyExc_TypeError, "init(error, addresses)");
#define X(f)                                                                                \
    {                                                                                       \
        PyObject* v = PyDict_GetItemString(a[1], #f);                                       \
        void* p = v ? PyLong_AsVoidPtr(v) : nullptr;                                        \
        if (!p) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_KeyError, "%s", #f); \
        p_##f = reinterpret_cast<decltype(p_##f)>(p);                                       \
    }
    GPT2B_BOUND(X)
#undef X
    Py_INCREF(a[0]);
    Py_XSETREF(g_error, a[0]);
    Py_RETURN_NONE;
}

#define ENTRY(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {ENTRY(init), ENTRY(kv_block_tables), ENTRY(kv_cache_write_w4), ENTRY(kv_cache_read_w4),
                           ENTRY(attention_forward_paged_w4), ENTRY(softmax_probs), ENTRY(verify_draft_tokens),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_bind", "operators on torch tensors", -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind(void) { return PyModule_Create(&g_module); }
