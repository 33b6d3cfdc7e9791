// Python binding of the operators on device memory for torch tensors (smelt_b200.paged,
// smelt_b200.logprobs): checks of shape, type, strides and device, the outputs and the workspace
// from torch's allocator (so that a call on another stream or in a captured graph has its own), the
// current torch stream, and one call of the C-ABI. In C++ because a decode step's calls take less
// time on the GPU than the same checks take in Python (attention of one short row: 17 us a call
// through ctypes).
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <string>

#include "gpt2q.h"

namespace {

PyObject* g_error = nullptr;  // smelt_b200._ffi.Gpt2qError

struct Refused {};  // a Python exception is set

[[noreturn]] void refuse(const std::string& msg) {
    PyErr_SetString(PyExc_ValueError, msg.c_str());
    throw Refused{};
}

void check(int rc) {
    if (rc == GPT2Q_OK) return;
    PyObject* e = PyObject_CallFunction(g_error, "is", rc, gpt2q_last_error(nullptr));
    if (e) {
        PyErr_SetObject(g_error, e);
        Py_DECREF(e);
    }
    throw Refused{};
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a torch tensor");
    return THPVariable_Unpack(o);
}
const at::Tensor* optional(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }

long long whole(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Refused{};
    return v;
}
// an int argument that the C-ABI takes as int32
int small(PyObject* o, const char* name) {
    const long long v = whole(o);
    if (v < INT32_MIN || v > INT32_MAX) refuse(std::string(name) + " out of range");
    return (int)v;
}
double real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Refused{};
    return v;
}
int size32(int64_t n, const char* name) {
    if (n > INT32_MAX) refuse(std::string(name) + " is too long");
    return (int)n;
}

int type_code(at::ScalarType t) {
    return t == at::kFloat ? GPT2Q_F32 : t == at::kHalf ? GPT2Q_F16 : t == at::kBFloat16 ? GPT2Q_BF16 : -1;
}
const char* type_name(int code) { return code == GPT2Q_F32 ? "float32" : code == GPT2Q_F16 ? "float16" : "bfloat16"; }

void on_device(const at::Tensor& t, int index, const char* name) {
    if (!t.is_cuda() || t.get_device() != index)
        refuse(std::string(name) + " must be a tensor on cuda:" + std::to_string(index));
}

// a contiguous vector of n elements of a type
void* vector(const at::Tensor& t, int index, const char* name, int64_t n, at::ScalarType type, const char* type_text) {
    on_device(t, index, name);
    if (t.scalar_type() != type || t.dim() != 1 || t.size(0) != n || !t.is_contiguous())
        refuse(std::string(name) + " must be a contiguous " + type_text + " tensor of " + std::to_string(n) + " elements");
    return t.data_ptr();
}
int32_t* ints(const at::Tensor& t, int index, const char* name, int64_t n) {
    return static_cast<int32_t*>(vector(t, index, name, n, at::kInt, "int32"));
}

gpt2q_heads heads(const at::Tensor& t, int index, const char* name, int64_t n, int64_t h, int64_t dim, at::ScalarType type) {
    on_device(t, index, name);
    if (t.dim() != 3 || t.size(0) != n || t.size(1) != h || t.size(2) != dim || t.scalar_type() != type)
        refuse(std::string(name) + " must be [" + std::to_string(n) + ", " + std::to_string(h) + ", " + std::to_string(dim) +
               "] of " + type_name(type_code(type)));
    if (t.stride(2) != 1 && dim > 1) refuse(std::string(name) + " must have unit stride over the head dim");
    return gpt2q_heads{t.data_ptr(), t.stride(0), t.stride(1)};
}

// The cache and the type of the call's tensors: its own or float32.
const gpt2q_paged_kv* cache_of(PyObject* o) { return static_cast<const gpt2q_paged_kv*>(PyLong_AsVoidPtr(o)); }
at::ScalarType io_type(const gpt2q_paged_kv* kv, const at::Tensor& t) {
    const int code = type_code(t.scalar_type());
    if (code != kv->dtype && code != GPT2Q_F32)
        refuse(std::string("tensors must be ") + type_name(kv->dtype) + " like the cache, or float32");
    return t.scalar_type();
}
gpt2q_page_table page_table(const at::Tensor& t, int index) {
    on_device(t, index, "table");
    if (t.scalar_type() != at::kInt || t.dim() != 2 || (t.size(1) > 1 && t.stride(1) != 1))
        refuse("table must be int32 [rows, pages] with unit stride over the pages");
    const int rows = size32(t.size(0), "table"), width = size32(t.size(1), "table");
    return gpt2q_page_table{static_cast<const int32_t*>(t.data_ptr()), rows, width,
                            rows > 1 ? t.stride(0) : std::max<int64_t>(t.stride(0), width)};
}

struct Stream {
    c10::OptionalDeviceGuard guard;
    void* handle;
    explicit Stream(int index) {
        guard.reset_device(c10::Device(c10::kCUDA, (c10::DeviceIndex)index));
        handle = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)index).stream();
    }
};

template <class F>
PyObject* guarded(F&& f) {
    HANDLE_TH_ERRORS
    try {
        return f();
    } catch (const Refused&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

bool arity(Py_ssize_t n, Py_ssize_t want) {
    if (n == want) return true;
    PyErr_Format(PyExc_TypeError, "expected %zd arguments", want);
    return false;
}

// append(cache, device, k, v, table, pos, seq, rotary, q, q_out, status) -> q_out or None
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (!arity(n_args, 11)) return nullptr;
    return guarded([&]() -> PyObject* {
        const gpt2q_paged_kv* kv = cache_of(a[0]);
        const int index = small(a[1], "device");
        const at::Tensor &k = tensor(a[2], "k"), &v = tensor(a[3], "v");
        const at::ScalarType type = io_type(kv, k);
        if (k.dim() != 3) refuse("k must be [tokens, kv heads, head dim]");
        const int64_t n = k.size(0);
        const gpt2q_heads kh = heads(k, index, "k", n, kv->n_kv_heads, kv->head_dim, type);
        const gpt2q_heads vh = heads(v, index, "v", n, kv->n_kv_heads, kv->head_dim, type);
        const gpt2q_page_table t = page_table(tensor(a[4], "table"), index);
        const int32_t* pos = ints(tensor(a[5], "pos"), index, "pos", n);
        const at::Tensor *seq = optional(a[6], "seq"), *q = optional(a[8], "q"), *q_out = optional(a[9], "q_out");
        const at::Tensor* status = optional(a[10], "status");
        const int32_t* sp = seq ? ints(*seq, index, "seq", n) : nullptr;
        int32_t* st = status ? ints(*status, index, "status", 1) : nullptr;
        const gpt2q_rotary* rot = a[7] == Py_None ? nullptr : static_cast<const gpt2q_rotary*>(PyLong_AsVoidPtr(a[7]));
        gpt2q_heads qh{}, oh{};
        at::Tensor fresh;
        int64_t hq = 0;
        if (q) {
            if (q->dim() != 3) refuse("q must be [tokens, heads, head dim]");
            hq = q->size(1);
            qh = heads(*q, index, "q", n, hq, kv->head_dim, type);
            if (!q_out) {
                fresh = at::empty({n, hq, kv->head_dim}, q->options().memory_format(at::MemoryFormat::Contiguous));
                q_out = &fresh;
            }
            oh = heads(*q_out, index, "q_out", n, hq, kv->head_dim, type);
        } else if (q_out) {
            refuse("q_out without q");
        }
        Stream s(index);
        check(gpt2q_paged_append(kv, &t, &kh, &vh, q ? &qh : nullptr, q ? &oh : nullptr, type_code(type),
                                 size32(hq, "q"), size32(n, "k"), pos, sp, rot, st, s.handle));
        if (!q) Py_RETURN_NONE;
        if (fresh.defined()) return THPVariable_Wrap(fresh);
        return Py_NewRef(a[9]);
    });
}

// attend(cache, device, q, table, lens, scale, window, out, lse, status) -> out
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (!arity(n_args, 10)) return nullptr;
    return guarded([&]() -> PyObject* {
        const gpt2q_paged_kv* kv = cache_of(a[0]);
        const int index = small(a[1], "device");
        const at::Tensor& q = tensor(a[2], "q");
        const at::ScalarType type = io_type(kv, q);
        if (q.dim() != 3) refuse("q must be [rows, heads, head dim]");
        const int64_t n = q.size(0), hq = q.size(1);
        const gpt2q_heads qh = heads(q, index, "q", n, hq, kv->head_dim, type);
        const gpt2q_page_table t = page_table(tensor(a[3], "table"), index);
        if (t.n_rows != n) refuse("table must have " + std::to_string(n) + " rows");
        const int32_t* lens = ints(tensor(a[4], "lens"), index, "lens", n);
        const float scale = a[5] == Py_None ? 1.f / std::sqrt((float)kv->head_dim) : (float)real(a[5]);
        const int window = small(a[6], "window");
        const at::Tensor *out = optional(a[7], "out"), *lse = optional(a[8], "lse"), *status = optional(a[9], "status");
        at::Tensor fresh;
        if (!out) {
            fresh = at::empty({n, hq, kv->head_dim}, q.options().memory_format(at::MemoryFormat::Contiguous));
            out = &fresh;
        }
        const gpt2q_heads oh = heads(*out, index, "out", n, hq, kv->head_dim, type);
        if (lse) {
            on_device(*lse, index, "lse");
            if (lse->scalar_type() != at::kFloat || lse->dim() != 2 || lse->size(0) != n || lse->size(1) != hq || !lse->is_contiguous())
                refuse("lse must be a contiguous float32 tensor [" + std::to_string(n) + ", " + std::to_string(hq) + "]");
        }
        int32_t* st = status ? ints(*status, index, "status", 1) : nullptr;
        const int64_t bytes = (int64_t)gpt2q_paged_attention_workspace(kv, size32(hq, "q"));
        const at::Tensor work = at::empty({std::max<int64_t>(16, bytes)}, q.options().dtype(at::kByte));
        Stream s(index);
        check(gpt2q_paged_attention(kv, &t, lens, &qh, &oh, type_code(type), (int)hq, scale, window,
                                    lse ? static_cast<float*>(lse->data_ptr()) : nullptr, st, work.data_ptr(), s.handle));
        if (fresh.defined()) return THPVariable_Wrap(fresh);
        return Py_NewRef(a[7]);
    });
}

struct Logits {
    int index, rows, vocab, code;
    int64_t ld;
    void* data;
};
Logits logits_of(const at::Tensor& x, const char* name) {
    Logits l{};
    l.code = type_code(x.scalar_type());
    if (!x.is_cuda() || x.dim() != 2 || l.code < 0)
        refuse(std::string(name) + " must be a CUDA tensor [rows, vocab] of float32, float16 or bfloat16");
    l.index = x.get_device();
    l.rows = size32(x.size(0), name), l.vocab = size32(x.size(1), name);
    if (l.vocab < 1 || (x.stride(1) != 1 && l.vocab > 1)) refuse(std::string(name) + " must have unit stride over the vocabulary");
    l.ld = l.rows > 1 ? x.stride(0) : l.vocab;
    if (l.ld < l.vocab) refuse(std::string("the rows of ") + name + " must not overlap");
    l.data = x.data_ptr();
    return l;
}
void* targets_of(const at::Tensor* t, const Logits& l, int* wide) {
    *wide = 0;
    if (!t) return nullptr;
    *wide = t->scalar_type() == at::kLong;
    return *wide ? vector(*t, l.index, "targets", l.rows, at::kLong, "int32 or int64")
                 : vector(*t, l.index, "targets", l.rows, at::kInt, "int32 or int64");
}

// logprobs(logits, targets, top, temperature) -> (lp, entropy, top_ids, top_lp, stats)
PyObject* logprobs(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (!arity(n_args, 4)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor& x = tensor(a[0], "logits");
        const Logits l = logits_of(x, "logits");
        const at::Tensor* t = optional(a[1], "targets");
        int wide = 0;
        const void* tp = targets_of(t, l, &wide);
        const int top = small(a[2], "top");
        const double temperature = real(a[3]);
        if (top < 0 || top > GPT2Q_TOP_MAX || top > l.vocab)
            refuse("top must be from 0 to min(vocab, " + std::to_string(GPT2Q_TOP_MAX) + ")");
        const auto f32 = x.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous);
        // one block for all float outputs: lp, entropy, stats, top_lp
        const int64_t R = l.rows;
        const at::Tensor all = at::empty({R * (5 + top)}, f32);
        float* at0 = static_cast<float*>(all.data_ptr());
        at::Tensor ids;
        if (top) ids = at::empty({R, top}, f32.dtype(at::kInt));
        Stream s(l.index);
        check(gpt2q_logprobs(l.data, l.code, l.ld, l.rows, l.vocab, (float)temperature, tp, wide, top, t ? at0 : nullptr, at0 + R,
                             at0 + 2 * R, top ? static_cast<int32_t*>(ids.data_ptr()) : nullptr, top ? at0 + 5 * R : nullptr, s.handle));
        auto view = [&](int64_t from, at::IntArrayRef size, at::IntArrayRef stride) {
            return THPVariable_Wrap(all.as_strided(size, stride, from));
        };
        PyObject* out = PyTuple_New(5);
        PyTuple_SET_ITEM(out, 0, t ? view(0, {R}, {1}) : Py_NewRef(Py_None));
        PyTuple_SET_ITEM(out, 1, view(R, {R}, {1}));
        PyTuple_SET_ITEM(out, 2, top ? THPVariable_Wrap(ids) : Py_NewRef(Py_None));
        PyTuple_SET_ITEM(out, 3, top ? view(5 * R, {R, top}, {top, 1}) : Py_NewRef(Py_None));
        PyTuple_SET_ITEM(out, 4, view(2 * R, {R, 3}, {3, 1}));
        return out;
    });
}

// logprobs_grad(logits, targets, stats, d_lp, d_entropy, temperature, out) -> out
PyObject* logprobs_grad(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (!arity(n_args, 7)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor& x = tensor(a[0], "logits");
        const Logits l = logits_of(x, "logits");
        const at::Tensor* t = optional(a[1], "targets");
        int wide = 0;
        const void* tp = targets_of(t, l, &wide);
        const at::Tensor& stats = tensor(a[2], "stats");
        on_device(stats, l.index, "stats");
        if (stats.scalar_type() != at::kFloat || stats.dim() != 2 || stats.size(0) != l.rows || stats.size(1) != 3 || !stats.is_contiguous())
            refuse("stats must be a contiguous float32 tensor [" + std::to_string(l.rows) + ", 3]");
        const at::Tensor *dl = optional(a[3], "d_lp"), *de = optional(a[4], "d_entropy");
        if (dl && !t) refuse("d_lp without targets");
        const float* dlp = dl ? static_cast<const float*>(vector(*dl, l.index, "d_lp", l.rows, at::kFloat, "float32")) : nullptr;
        const float* dep = de ? static_cast<const float*>(vector(*de, l.index, "d_entropy", l.rows, at::kFloat, "float32")) : nullptr;
        const double temperature = real(a[5]);
        const at::Tensor* out = optional(a[6], "out");
        at::Tensor fresh;
        if (!out) {
            fresh = at::empty({l.rows, l.vocab}, x.options().memory_format(at::MemoryFormat::Contiguous));
            out = &fresh;
        }
        const Logits o = logits_of(*out, "out");
        if (o.index != l.index || o.rows != l.rows || o.vocab != l.vocab || o.code != l.code)
            refuse("out must have the shape, type and device of logits");
        Stream s(l.index);
        check(gpt2q_logprobs_grad(l.data, l.code, l.ld, l.rows, l.vocab, (float)temperature, tp, wide,
                                  static_cast<const float*>(stats.data_ptr()), dlp, dep, o.data, o.ld, s.handle));
        if (fresh.defined()) return THPVariable_Wrap(fresh);
        return Py_NewRef(a[6]);
    });
}

PyObject* set_error(PyObject*, PyObject* cls) {
    Py_XSETREF(g_error, Py_NewRef(cls));
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(append)), METH_FASTCALL, nullptr},
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(attend)), METH_FASTCALL, nullptr},
    {"logprobs", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(logprobs)), METH_FASTCALL, nullptr},
    {"logprobs_grad", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(logprobs_grad)), METH_FASTCALL, nullptr},
    {"set_error", set_error, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "gpt2q_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_gpt2q_torch() { return PyModule_Create(&module); }
