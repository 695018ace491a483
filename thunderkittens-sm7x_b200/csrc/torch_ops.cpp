// torch_ops.cpp — the Python helpers' way into the C ABI for the prompt and serving
// operators (include/tk_b200.h): takes torch tensors, checks them, allocates what is not
// given, and calls the entry point on the tensors' device and its current stream.
//
// It computes nothing, and no gradients: an output of inputs that require them carries a node that raises in
// backward, tangents of forward mode are refused, and tensors written in place get a new version. It exists because the smallest of these calls take a few
// microseconds on the GPU, and looking at a dozen tensors from Python takes longer than
// that (kv_append of 64 tokens: 11 us in Python with ctypes, 4.9 us here).
//
// Built as the extension module tk_b200/_ops.so against the installed torch; the library
// itself, libtk_b200.so, needs neither torch nor Python.

#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <memory>
#include <optional>
#include <string>
#include <utility>

#include "tk_b200.h"

namespace {

PyObject* g_error = nullptr;  // tk_b200.TkError

// What a helper throws for a tensor that does not fit: ValueError in Python.
struct Refused {
    std::string why;
};

std::string shape_of(const at::Tensor& t) {
    std::string s = "[";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + "]";
}

[[noreturn]] void refuse(std::string why) { throw Refused{std::move(why)}; }

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a torch tensor");
    return THPVariable_Unpack(o);
}

// Empty for None.
std::optional<at::Tensor> maybe(PyObject* o, const char* name) {
    if (o == Py_None) return std::nullopt;
    return tensor(o, name);
}

double number(PyObject* o, const char* name) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse(std::string(name) + " must be a number");
    }
    return v;
}

// A cap in 32 bits; 0 means none, so what only becomes 0 there is not that.
float cap_of(PyObject* o) {
    const double v = number(o, "softcap");
    const float cap = static_cast<float>(v);
    if (cap == 0.0f && v != 0.0) refuse("softcap must be 0 (none) or from 1e-6 to 1e30");
    return cap;
}

int whole(PyObject* o, const char* name) {
    int overflow = 0;
    const long v = PyLong_AsLongAndOverflow(o, &overflow);
    if (overflow != 0 || (v == -1 && PyErr_Occurred()) || v != static_cast<int>(v)) {
        PyErr_Clear();
        refuse(std::string(name) + " must be a whole number of 32 bits");
    }
    return static_cast<int>(v);
}

int fits_int(int64_t v, const char* name) {
    if (v > INT32_MAX) refuse(std::string(name) + " has a dimension of more than 2^31 - 1");
    return static_cast<int>(v);
}

void on_cuda(const at::Tensor& t, const char* name) {
    if (!t.is_cuda()) refuse(std::string(name) + " must be on a CUDA device");
}

void same_device(const at::Tensor& t, const at::Tensor& as, const char* name) {
    if (t.device() != as.device()) refuse(std::string(name) + " is on " + t.device().str() + ", expected " + as.device().str());
}

void half_type(const at::Tensor& t, const char* name) {
    if (t.scalar_type() != at::kHalf && t.scalar_type() != at::kBFloat16) refuse(std::string(name) + " must be float16 or bfloat16");
}

// A contiguous tensor of this type and shape, on the device of `as`.
void vector(const at::Tensor& t, const at::Tensor& as, const char* name, at::ScalarType type, at::IntArrayRef shape) {
    if (t.scalar_type() != type || t.sizes() != shape || !t.is_contiguous()) {
        std::string want = "[";
        for (size_t i = 0; i < shape.size(); ++i) want += (i ? ", " : "") + std::to_string(shape[i]);
        refuse(std::string(name) + " must be a contiguous " + c10::toString(type) + " tensor of shape " + want + "], got " +
               c10::toString(t.scalar_type()) + " " + shape_of(t));
    }
    same_device(t, as, name);
}

template <class T>
T* data(const std::optional<at::Tensor>& t) {
    return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}

// ---- autograd

// Whether forward mode is in use at all; only then are tensors asked for tangents.
bool forward_mode() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }

// What a call reads: whether gradients have to reach any of it.
bool tracked(std::initializer_list<const at::Tensor*> reads) {
    bool some = false;
    const bool forward = forward_mode();
    for (const at::Tensor* t : reads) {
        if (t == nullptr) continue;
        some = some || t->requires_grad();
        if (forward && t->_fw_grad(0).defined()) refuse("there is no forward-mode derivative");
    }
    return some && at::GradMode::is_enabled();
}

// Before a call writes tensors of the caller's.
struct Target {
    const at::Tensor* t;
    const char* name;
};

void writable(std::initializer_list<Target> targets) {
    const bool grads = at::GradMode::is_enabled(), forward = forward_mode();
    for (const Target& x : targets) {
        if (grads && x.t->requires_grad()) refuse(std::string(x.name) + " is written in place and must not require gradients");
        if (forward && x.t->_fw_grad(0).defined()) refuse("there is no forward-mode derivative");
    }
}

// After it has.
void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Backward through `out` raises instead of leaving gradients out.
void no_backward(const at::Tensor& out, const char* name, std::initializer_list<const at::Tensor*> reads) {
    torch::autograd::edge_list edges;
    for (const at::Tensor* t : reads)
        if (t != nullptr && t->requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(*t));
    std::shared_ptr<torch::autograd::Node> node(new torch::autograd::NotImplemented(name, std::move(edges)), torch::autograd::deleteNode);
    torch::autograd::set_history(out, node);
}

const at::Tensor* if_given(const std::optional<at::Tensor>& t) { return t ? &*t : nullptr; }

struct Failed {
    const char* name;
    int code;
};

void check(const char* name, cudaError_t code) {
    if (code != cudaSuccess) throw Failed{name, static_cast<int>(code)};
}

// A call's device, current while it allocates and launches, and the stream that is current there.
struct Scope {
    c10::cuda::CUDAGuard guard;
    cudaStream_t stream;
    explicit Scope(const at::Tensor& t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};

// Runs a helper's body; its refusals and errors become Python exceptions.
template <class F>
PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F&& body) {
    HANDLE_TH_ERRORS
    try {
        if (got != want) refuse("wrong number of arguments");
        return body();
    } catch (const Refused& r) {
        PyErr_SetString(PyExc_ValueError, r.why.c_str());
    } catch (const Failed& f) {
        PyObject* e = g_error != nullptr ? PyObject_CallFunction(g_error, "si", f.name, f.code) : nullptr;
        if (e != nullptr) {
            PyErr_SetObject(g_error, e);
            Py_DECREF(e);
        } else if (!PyErr_Occurred()) {
            PyErr_Format(PyExc_RuntimeError, "%s returned cudaError %d", f.name, f.code);
        }
    }
    return nullptr;
    END_HANDLE_TH_ERRORS
}

// attention_masked(q, k, v, scale, causal, softcap, alibi_slopes, doc_ids, prefix_lens, out)
PyObject* attention_masked(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 10, [&]() -> PyObject* {
        const at::Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k"), &v = tensor(a[2], "v");
        half_type(q, "q");
        if (q.dim() != 4 || k.dim() != 4 || v.sizes() != k.sizes()) refuse("q, k, v must be [B, H, S, D], k and v alike");
        if (k.size(0) != q.size(0) || k.size(3) != q.size(3)) refuse("k has shape " + shape_of(k) + ", q " + shape_of(q));
        if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) refuse("q, k, v must have one type");
        const int b = fits_int(q.size(0), "q"), h = fits_int(q.size(1), "q"), sq = fits_int(q.size(2), "q"), d = fits_int(q.size(3), "q");
        const int hkv = fits_int(k.size(1), "k"), skv = fits_int(k.size(2), "k");
        const float scale = static_cast<float>(number(a[3], "scale"));
        const int causal = PyObject_IsTrue(a[4]);
        if (causal < 0) return nullptr;
        const float cap = cap_of(a[5]);
        const auto slopes = maybe(a[6], "alibi_slopes"), ids = maybe(a[7], "doc_ids"), prefix = maybe(a[8], "prefix_lens");
        auto out = maybe(a[9], "out");
        if (slopes) vector(*slopes, q, "alibi_slopes", at::kFloat, {h});
        if (ids) vector(*ids, q, "doc_ids", at::kInt, {b, sq});
        if (prefix) vector(*prefix, q, "prefix_lens", at::kInt, {b});
        if (out && (out->scalar_type() != q.scalar_type() || out->sizes() != q.sizes())) refuse("out must have q's type and shape");
        const bool grad = tracked({&q, &k, &v, if_given(slopes)});
        const bool given = out.has_value();
        if (given) {
            writable({{&*out, "out"}});
            if (grad) refuse("out cannot be given where an input requires gradients");
        }
        if (d > 1 && (q.stride(3) != 1 || k.stride(3) != 1 || v.stride(3) != 1 || (out && out->stride(3) != 1)))
            refuse("the last strides of q, k, v and out must be 1");
        on_cuda(q, "q");
        same_device(k, q, "k");
        same_device(v, q, "v");
        if (out) same_device(*out, q, "out");
        const Scope scope(q);
        if (!out) out = at::empty_like(q);
        int64_t strides[12];
        const at::Tensor* views[4] = {&q, &k, &v, &*out};
        for (int i = 0; i < 4; ++i)
            for (int j = 0; j < 3; ++j) strides[3 * i + j] = views[i]->stride(j);
        const bool bf16 = q.scalar_type() == at::kBFloat16;
        check(bf16 ? "tk_attention_masked_bf16" : "tk_attention_masked_f16",
              (bf16 ? tk_attention_masked_bf16 : tk_attention_masked_f16)(
                  q.data_ptr(), k.data_ptr(), v.data_ptr(), out->data_ptr(), strides, b, h, hkv, sq, skv, d, scale, cap,
                  data<float>(slopes), data<int32_t>(ids), data<int32_t>(prefix), causal, scope.stream));
        if (given) written(*out);
        if (grad) no_backward(*out, "tk_b200.attention_masked", {&q, &k, &v, if_given(slopes)});
        return THPVariable_Wrap(*out);
    });
}

// Elements [from, from + n) of a buffer, without the 1 us of a dispatched view.
at::Tensor part_of(const at::Tensor& buffer, int64_t from, int64_t n) {
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(buffer.storage()), buffer.key_set(),
                                                            buffer.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(from);
    t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
    return t;
}

// kv_plan(cached_lens, new_lens, block_table, free_pages, n_free, page_size, max_tokens, lens_out, seq_lens,
//         starts, slots, n_free_out)
PyObject* kv_plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 12, [&]() -> PyObject* {
        const at::Tensor &cached = tensor(a[0], "cached_lens"), &fresh = tensor(a[1], "new_lens"), &table = tensor(a[2], "block_table");
        const at::Tensor &free = tensor(a[3], "free_pages"), &n_free = tensor(a[4], "n_free");
        const int page = whole(a[5], "page_size"), max_tokens = whole(a[6], "max_tokens");
        if (max_tokens < 0) refuse("max_tokens must not be negative");
        if (cached.dim() != 1) refuse("cached_lens must be [R]");
        if (table.dim() != 2) refuse("block_table must be [R, max_pages]");
        const int r = fits_int(cached.size(0), "cached_lens"), width = fits_int(table.size(1), "block_table");
        vector(cached, cached, "cached_lens", at::kInt, {r});
        vector(fresh, cached, "new_lens", at::kInt, {r});
        vector(table, cached, "block_table", at::kInt, {r, width});
        vector(free, cached, "free_pages", at::kInt, free.sizes());
        vector(n_free, cached, "n_free", at::kInt, {1});
        const char* names[5] = {"lens_out", "seq_lens", "starts", "slots", "n_free_out"};
        const int64_t sizes[5] = {r, r, static_cast<int64_t>(r) + 1, max_tokens, 1};
        at::Tensor outs[5];
        bool missing = false;
        for (int i = 0; i < 5; ++i) {
            if (a[7 + i] == Py_None) {
                missing = true;
                continue;
            }
            outs[i] = tensor(a[7 + i], names[i]);
            vector(outs[i], cached, names[i], i == 3 ? at::kLong : at::kInt, {sizes[i]});
        }
        on_cuda(cached, "cached_lens");
        const Scope scope(cached);
        if (missing) {
            // The 32-bit outputs that are not given are parts of one buffer.
            at::Tensor buffer;
            int64_t at_ = 0;
            for (int i = 0; i < 5; ++i) {
                if (outs[i].defined()) continue;
                if (i == 3) {
                    outs[3] = at::empty({max_tokens}, cached.options().dtype(at::kLong));
                    continue;
                }
                if (!buffer.defined()) buffer = at::empty({3 * static_cast<int64_t>(r) + 2}, cached.options());
                outs[i] = part_of(buffer, at_, sizes[i]);
                at_ += sizes[i];
            }
        }
        check("tk_kv_plan",
              tk_kv_plan(cached.data_ptr<int>(), fresh.data_ptr<int>(), r, page, table.data_ptr<int>(), width, free.data_ptr<int>(),
                         fits_int(free.numel(), "free_pages"), n_free.data_ptr<int>(), outs[0].data_ptr<int>(), outs[1].data_ptr<int>(),
                         outs[2].data_ptr<int>(), outs[3].data_ptr<int64_t>(), max_tokens, outs[4].data_ptr<int>(), scope.stream));
        written(table);
        for (int i = 0; i < 5; ++i)
            if (a[7 + i] != Py_None) written(outs[i]);
        PyObject* result = PyTuple_New(5);
        for (int i = 0; i < 5 && result != nullptr; ++i) PyTuple_SET_ITEM(result, i, THPVariable_Wrap(outs[i]));
        return result;
    });
}

// The cache's tensors, checked against each other and the device of `as`.
struct Cache {
    const at::Tensor &k, &v, &ks, &vs;
    int pages, heads, page, dim;
};

Cache cache_of(PyObject* const* a, const at::Tensor& as) {
    const at::Tensor &k = tensor(a[0], "k_cache"), &v = tensor(a[1], "v_cache"), &ks = tensor(a[2], "k_scale"), &vs = tensor(a[3], "v_scale");
    if (k.dim() != 4) refuse("k_cache must be [pages, Hkv, page_size, D]");
    for (const at::Tensor* t : {&k, &v})
        if (t->scalar_type() != at::kByte && t->scalar_type() != at::kFloat8_e4m3fn) refuse("k_cache and v_cache must be uint8 or float8_e4m3fn");
    vector(k, as, "k_cache", k.scalar_type(), k.sizes());
    vector(v, as, "v_cache", v.scalar_type(), k.sizes());
    vector(ks, as, "k_scale", at::kFloat, k.sizes().slice(0, 2));
    vector(vs, as, "v_scale", at::kFloat, k.sizes().slice(0, 2));
    return Cache{k, v, ks, vs, fits_int(k.size(0), "k_cache"), fits_int(k.size(1), "k_cache"), fits_int(k.size(2), "k_cache"),
                 fits_int(k.size(3), "k_cache")};
}

// Elements between the tokens of a packed [T, heads, dim] tensor.
int64_t token_stride(const at::Tensor& t, const char* name) {
    const int64_t row = t.size(1) * t.size(2);
    if (t.stride(2) != 1 || (t.size(1) > 1 && t.stride(1) != t.size(2))) refuse(std::string("the heads of a token of ") + name + " must be adjacent");
    return t.size(0) > 1 ? t.stride(0) : row;
}

// kv_append(k, v, slots, k_cache, v_cache, k_scale, v_scale)
PyObject* kv_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 7, [&]() -> PyObject* {
        const at::Tensor &k = tensor(a[0], "k"), &v = tensor(a[1], "v"), &slots = tensor(a[2], "slots");
        half_type(k, "k");
        const Cache c = cache_of(a + 3, k);
        if (k.dim() != 3 || k.size(1) != c.heads || k.size(2) != c.dim)
            refuse("k must be [T, " + std::to_string(c.heads) + ", " + std::to_string(c.dim) + "], got " + shape_of(k));
        if (v.scalar_type() != k.scalar_type() || v.sizes() != k.sizes()) refuse("k and v must have one type and shape");
        same_device(v, k, "v");
        vector(slots, k, "slots", at::kLong, {k.size(0)});
        writable({{&c.k, "k_cache"}, {&c.v, "v_cache"}, {&c.ks, "k_scale"}, {&c.vs, "v_scale"}});
        on_cuda(k, "k");
        const int tokens = fits_int(k.size(0), "k");
        if (tokens > 0) {
            const int64_t k_stride = token_stride(k, "k"), v_stride = token_stride(v, "v");
            const Scope scope(k);
            const bool bf16 = k.scalar_type() == at::kBFloat16;
            check(bf16 ? "tk_kv_append_e4m3_bf16" : "tk_kv_append_e4m3_f16",
                  (bf16 ? tk_kv_append_e4m3_bf16 : tk_kv_append_e4m3_f16)(
                      k.data_ptr(), v.data_ptr(), k_stride, v_stride, slots.data_ptr<int64_t>(), tokens, c.heads, c.dim, c.k.data_ptr(),
                      c.v.data_ptr(), c.ks.data_ptr<float>(), c.vs.data_ptr<float>(), c.pages, c.page, scope.stream));
            for (const at::Tensor* t : {&c.k, &c.v, &c.ks, &c.vs}) written(*t);
        }
        Py_RETURN_NONE;
    });
}

// attention_paged(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, starts, scale, softcap, alibi_slopes,
//                 max_query_len, max_seq_len, out)
PyObject* attention_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 14, [&]() -> PyObject* {
        const at::Tensor& q = tensor(a[0], "q");
        half_type(q, "q");
        const Cache c = cache_of(a + 1, q);
        const at::Tensor &table = tensor(a[5], "block_table"), &lens = tensor(a[6], "seq_lens"), &starts = tensor(a[7], "starts");
        if (q.dim() != 3 || q.size(2) != c.dim) refuse("q must be [T, Hq, " + std::to_string(c.dim) + "], got " + shape_of(q));
        if (table.dim() != 2) refuse("block_table must be [R, max_pages]");
        const int tokens = fits_int(q.size(0), "q"), heads = fits_int(q.size(1), "q");
        const int r = fits_int(table.size(0), "block_table"), width = fits_int(table.size(1), "block_table");
        vector(table, q, "block_table", at::kInt, table.sizes());
        vector(lens, q, "seq_lens", at::kInt, {r});
        vector(starts, q, "starts", at::kInt, {static_cast<int64_t>(r) + 1});
        const float scale = static_cast<float>(number(a[8], "scale")), cap = cap_of(a[9]);
        const auto slopes = maybe(a[10], "alibi_slopes");
        if (slopes) vector(*slopes, q, "alibi_slopes", at::kFloat, {heads});
        const int most_queries = whole(a[11], "max_query_len");
        const int64_t room = static_cast<int64_t>(width) * c.page;
        const int most_keys = a[12] != Py_None ? whole(a[12], "max_seq_len") : room > INT32_MAX ? INT32_MAX : static_cast<int>(room);
        auto out = maybe(a[13], "out");
        if (out && (out->scalar_type() != q.scalar_type() || out->sizes() != q.sizes())) refuse("out must have q's type and shape");
        const int64_t q_stride = token_stride(q, "q");
        const bool grad = tracked({&q, &c.k, &c.v, &c.ks, &c.vs, if_given(slopes)});
        const bool given = out.has_value();
        if (given) {
            writable({{&*out, "out"}});
            if (grad) refuse("out cannot be given where an input requires gradients");
        }
        on_cuda(q, "q");
        if (out) same_device(*out, q, "out");
        const Scope scope(q);
        if (!out) out = at::empty(q.sizes(), q.options());
        const int64_t out_stride = token_stride(*out, "out");
        if (tokens > 0 && r > 0) {
            const bool bf16 = q.scalar_type() == at::kBFloat16;
            check(bf16 ? "tk_attention_paged_e4m3_bf16" : "tk_attention_paged_e4m3_f16",
                  (bf16 ? tk_attention_paged_e4m3_bf16 : tk_attention_paged_e4m3_f16)(
                      q.data_ptr(), q_stride, out->data_ptr(), out_stride, tokens, c.k.data_ptr(), c.v.data_ptr(), c.ks.data_ptr<float>(),
                      c.vs.data_ptr<float>(), c.pages, c.page, table.data_ptr<int>(), width, lens.data_ptr<int>(), starts.data_ptr<int>(), r,
                      heads, c.heads, c.dim, most_queries, most_keys, scale, cap, data<float>(slopes), scope.stream));
            if (given) written(*out);
        }
        if (grad) no_backward(*out, "tk_b200.attention_paged", {&q, &c.k, &c.v, &c.ks, &c.vs, if_given(slopes)});
        return THPVariable_Wrap(*out);
    });
}

// set_error(cls): the class of errors that the entry points return.
PyObject* set_error(PyObject*, PyObject* cls) {
    Py_INCREF(cls);
    Py_XDECREF(g_error);
    g_error = cls;
    Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef fast(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}

PyMethodDef g_methods[] = {
    fast<attention_masked>("attention_masked"), fast<kv_plan>("kv_plan"), fast<kv_append>("kv_append"),
    fast<attention_paged>("attention_paged"),   {"set_error", set_error, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr},
};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_ops", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops() { return PyModule_Create(&g_module); }
