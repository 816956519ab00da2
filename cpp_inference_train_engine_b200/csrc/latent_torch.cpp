// Binding of the shared-prompt decode operators (include/mm_latent.h) to torch tensors: argument
// checks, outputs and workspace from torch's allocator on the tensors' current stream, and the C
// call. Written against the CPython C API because a small decode step is bound by this path: the
// same checks through Python attributes took 9 to 21 us a call, the kernels 2 to 12.
//
// The functions take their arguments by position; latent.py documents them and gives names and
// defaults. Every refusal is an EngineError with the C code.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Dtype.h>

#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <string>

#include "../../include/mm_latent.h"

namespace {

struct Refusal {
    int code;
    std::string what;
};
[[noreturn]] void bad(std::string what) { throw Refusal{MM_INVALID_ARGUMENT, std::move(what)}; }
void require(bool ok, const char* what) {
    if (!ok) bad(what);
}

PyObject* raise(const Refusal& r) {
    PyObject* module = PyImport_ImportModule("cpp_inference_train_engine_b200.engine");
    PyObject* cls = module ? PyObject_GetAttrString(module, "EngineError") : nullptr;
    PyObject* e = cls ? PyObject_CallFunction(cls, "is", r.code, r.what.c_str()) : nullptr;
    if (e) PyErr_SetObject(cls, e);
    Py_XDECREF(e);
    Py_XDECREF(cls);
    Py_XDECREF(module);
    return nullptr;
}

// Runs f; refusals become EngineError, torch's own errors (out of memory) what torch raises.
template <class F> PyObject* guarded(F&& f) {
    HANDLE_TH_ERRORS
    try {
        return f();
    } catch (const Refusal& r) {
        return raise(r);
    }
    END_HANDLE_TH_ERRORS
}

void call(int rc) {
    if (!rc) return;
    char text[512];
    mm_latent_last_error(text, sizeof text);
    throw Refusal{rc, text};
}

// The calls go past autograd: a result would silently be a constant of its inputs.
const at::Tensor& no_gradient(const at::Tensor& t) {
    if (t.requires_grad() && at::GradMode::is_enabled())
        bad("no gradient flows through these operators: detach the tensors that require one, or call under torch.no_grad()");
    return t;
}
const at::Tensor& tensor(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) bad(std::string(what) + " must be a tensor");
    return no_gradient(THPVariable_Unpack(o));
}
const at::Tensor& cuda_tensor(PyObject* o, const char* what) {
    const at::Tensor& t = tensor(o, what);
    if (!t.is_cuda()) bad("a CUDA tensor is needed, got one on " + t.device().str());
    return t;
}
void on(const at::Tensor& t, c10::Device d) {
    if (t.device() != d) bad("tensors must be on one CUDA device: got " + t.device().str() + " beside " + d.str());
}
int kind_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return MM_F32;
        case at::kHalf: return MM_F16;
        case at::kBFloat16: return MM_BF16;
        default: return -1;
    }
}
bool half(int kind) { return kind == MM_F16 || kind == MM_BF16; }
bool last_adjacent(const at::Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1; }

double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        bad("scale must be a number");
    }
    return v;
}
// An int argument, or `absent` for None.
int64_t integer(PyObject* o, int64_t absent, const char* what) {
    if (o == Py_None) return absent;
    const long long v = PyLong_AsLongLong(o);
    if ((v == -1 && PyErr_Occurred()) || v > INT32_MAX || v < INT32_MIN) {
        PyErr_Clear();
        bad(std::string(what) + " must be an int of 32 bits");
    }
    return v;
}
int32_t size32(int64_t v) {
    if (v > INT32_MAX) bad("a dimension exceeds 32 bits");
    return static_cast<int32_t>(v);
}

// A 16-bit cache (a tensor, whose latent width is kv) or an 8-bit one (a tuple of three tensors;
// kv < 0: of any width).
mm_latent_cache cache(PyObject* o, c10::Device d, int64_t kv) {
    mm_latent_cache c{};
    if (THPVariable_Check(o)) {
        if (kv < 0) bad("an 8-bit cache (LatentCache) is needed");
        const at::Tensor& t = no_gradient(THPVariable_Unpack(o));
        const int kind = kind_of(t.scalar_type());
        if (t.dim() != 3 || !half(kind) || !last_adjacent(t))
            bad("a 16-bit cache is fp16 or bf16 [rows, positions, kv + rope] with adjacent values");
        on(t, d);
        c.latent = t.data_ptr();
        c.row_stride = t.stride(0);
        c.pos_stride = t.stride(1);
        c.rows = size32(t.size(0));
        c.positions = size32(t.size(1));
        c.kv = static_cast<int32_t>(kv);
        c.rope_dim = size32(t.size(2)) - c.kv;
        c.kind = c.rope_kind = kind;
        return c;
    }
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 3) bad("a cache is a tensor or a LatentCache");
    const at::Tensor& lat = tensor(PyTuple_GET_ITEM(o, 0), "a cache's latent");
    const at::Tensor& rope = tensor(PyTuple_GET_ITEM(o, 1), "a cache's rope");
    const at::Tensor& scale = tensor(PyTuple_GET_ITEM(o, 2), "a cache's scale");
    if (lat.dim() != 3 || rope.dim() != 3 || scale.dim() != 2 || rope.size(0) != lat.size(0) || rope.size(1) != lat.size(1) ||
        scale.size(0) != lat.size(0) || scale.size(1) != lat.size(1))
        bad("an 8-bit cache is latent [rows, positions, kv], rope [rows, positions, rope], scale [rows, positions]");
    const int kind = kind_of(rope.scalar_type());
    if (lat.scalar_type() != at::kFloat8_e4m3fn || !half(kind) || scale.scalar_type() != at::kFloat)
        bad("an 8-bit cache is float8_e4m3fn latents, fp16 or bf16 rope keys and fp32 scales");
    if (!last_adjacent(lat) || !last_adjacent(rope) || !last_adjacent(scale))
        bad("the last dimension of a cache must be contiguous");
    if (kv >= 0 && lat.size(2) != kv) bad("cache width differs from kv_rank");
    on(lat, d);
    on(rope, d);
    on(scale, d);
    c.latent = lat.data_ptr();
    c.rope = rope.data_ptr();
    c.scale = static_cast<float*>(scale.data_ptr());
    c.row_stride = lat.stride(0);
    c.pos_stride = lat.stride(1);
    c.rope_row_stride = rope.stride(0);
    c.rope_pos_stride = rope.stride(1);
    c.scale_row_stride = scale.stride(0);
    c.rows = size32(lat.size(0));
    c.positions = size32(lat.size(1));
    c.kv = size32(lat.size(2));
    c.rope_dim = size32(rope.size(2));
    c.kind = MM_E4M3;
    c.rope_kind = kind;
    return c;
}

const int64_t* slots(PyObject* o, c10::Device d, int64_t* n) {
    const at::Tensor& t = tensor(o, "slots");
    if (t.dim() != 1 || t.scalar_type() != at::kLong || !t.is_contiguous())
        bad("slots is a contiguous int64 vector (row * positions + position)");
    on(t, d);
    *n = t.size(0);
    return static_cast<const int64_t*>(t.data_ptr());
}
const int32_t* ints(PyObject* o, c10::Device d, int64_t n, const char* what) {
    if (!THPVariable_Check(o)) bad(std::string(what) + " is a contiguous int32 vector of " + std::to_string(n));
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != n || !t.is_contiguous())
        bad(std::string(what) + " is a contiguous int32 vector of " + std::to_string(n));
    on(t, d);
    return static_cast<const int32_t*>(t.data_ptr());
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, c10::Device d) {
    return at::detail::empty_cuda(sizes, type, d, std::nullopt);
}
void* stream_of(c10::Device d) { return c10::cuda::getCurrentCUDAStream(d.index()).stream(); }

void arguments(Py_ssize_t n, Py_ssize_t want) {
    if (n != want) bad("wrong number of arguments");
}

// cache, latent, rope, slots
PyObject* cache_write(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        arguments(n_args, 4);
        const at::Tensor& latent = cuda_tensor(a[1], "latent");
        const c10::Device d = latent.device();
        const mm_latent_cache c = cache(a[0], d, -1);
        const at::Tensor& rope = tensor(a[2], "rope");
        const int kind = kind_of(latent.scalar_type());
        require(latent.dim() == 2 && rope.dim() == 2 && rope.scalar_type() == latent.scalar_type() && kind >= 0,
                "latent [n, kv] and rope [n, rope] share one floating type");
        int64_t n = 0;
        const int64_t* s = slots(a[3], d, &n);
        require(latent.size(0) == n && latent.size(1) == c.kv && rope.size(0) == n && rope.size(1) == c.rope_dim,
                "latent, rope and slots do not match the cache");
        require(last_adjacent(latent) && last_adjacent(rope), "the last dimension must be contiguous");
        on(rope, d);
        const c10::cuda::CUDAGuard guard(d);
        call(mm_latent_cache_write(&c, latent.data_ptr(), latent.stride(0), rope.data_ptr(), rope.stride(0), kind, s, n,
                                   stream_of(d)));
        // written in place: what autograd has kept of these tensors is no longer theirs
        for (int i = 0; i < 3; ++i) {
            const at::Tensor& t = THPVariable_Unpack(PyTuple_GET_ITEM(a[0], i));
            if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
        }
        Py_RETURN_NONE;
    });
}

// cache, slots, dtype (None: the rope key's)
PyObject* cache_read(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        arguments(n_args, 3);
        const at::Tensor& first = cuda_tensor(a[1], "slots");
        const c10::Device d = first.device();
        const mm_latent_cache c = cache(a[0], d, -1);
        int64_t n = 0;
        const int64_t* s = slots(a[1], d, &n);
        at::ScalarType type = c.rope_kind == MM_BF16 ? at::kBFloat16 : at::kHalf;
        if (a[2] != Py_None) {
            if (!THPDtype_Check(a[2])) bad("dtype must be a torch dtype");
            type = reinterpret_cast<THPDtype*>(a[2])->scalar_type;
        }
        const int kind = kind_of(type);
        require(kind >= 0, "cache_read writes fp32, fp16 or bf16");
        const c10::cuda::CUDAGuard guard(d);
        const int64_t width = c.kv + c.rope_dim;
        at::Tensor out = empty({n, width}, type, d);
        call(mm_latent_cache_read(&c, s, n, out.data_ptr(), width, kind, stream_of(d)));
        return THPVariable_Wrap(std::move(out));
    });
}

// q, prefix, suffix, group_start, prefix_len, suffix_len, scale, kv_rank, max_group, max_prefix,
// max_suffix, return_lse
PyObject* shared_prefix_attention(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        arguments(n_args, 12);
        const at::Tensor& q = cuda_tensor(a[0], "q");
        const c10::Device d = q.device();
        const int kind = kind_of(q.scalar_type());
        require(q.dim() == 4 && half(kind) && last_adjacent(q),
                "q is fp16 or bf16 [rows, tokens, heads, kv + rope] with adjacent values");
        const int64_t B = q.size(0), T = q.size(1), H = q.size(2), W = q.size(3), kv = integer(a[7], 0, "kv_rank");
        require(kv > 0 && kv <= W && T > 0 && H > 0, "kv_rank must be in (0, q's width]");
        mm_shared_prefix_desc p{};
        p.q = q.data_ptr();
        p.q_row_stride = q.stride(0);
        p.q_token_stride = q.stride(1);
        p.q_head_stride = q.stride(2);
        p.dtype = kind;
        p.rows = size32(B);
        p.tokens = size32(T);
        p.heads = size32(H);
        p.scale = static_cast<float>(number(a[6]));
        mm_latent_cache prefix, suffix;
        const bool has_prefix = a[1] != Py_None, has_suffix = a[2] != Py_None;
        if (has_prefix) {
            prefix = cache(a[1], d, kv);
            require(prefix.kv + prefix.rope_dim == W, "prefix width differs from q's");
            require(THPVariable_Check(a[3]) && THPVariable_Unpack(a[3]).dim() == 1 && THPVariable_Unpack(a[3]).size(0) > 0 &&
                        a[4] != Py_None,
                    "a prefix needs group_start [groups + 1] and prefix_len [groups]");
            const int64_t groups = THPVariable_Unpack(a[3]).size(0) - 1;
            p.groups = size32(groups);
            p.group_start = ints(a[3], d, groups + 1, "group_start");
            p.prefix_len = ints(a[4], d, groups, "prefix_len");
            p.max_group = static_cast<int32_t>(integer(a[8], B, "max_group"));
            p.max_prefix = static_cast<int32_t>(integer(a[9], prefix.positions, "max_prefix"));
        }
        if (has_suffix) {
            suffix = cache(a[2], d, kv);
            require(suffix.kv + suffix.rope_dim == W, "suffix width differs from q's");
            p.suffix_len = ints(a[5], d, B, "suffix_len");
            p.max_suffix = static_cast<int32_t>(integer(a[10], suffix.positions, "max_suffix"));
        }
        const int want_lse = PyObject_IsTrue(a[11]);
        const c10::cuda::CUDAGuard guard(d);
        at::Tensor out = empty({B, T, H, kv}, q.scalar_type(), d), lse;
        p.out = out.data_ptr();
        if (want_lse) {
            lse = empty({B, T, H}, at::kFloat, d);
            p.lse = static_cast<float*>(lse.data_ptr());
        }
        const mm_latent_cache *pre = has_prefix ? &prefix : nullptr, *suf = has_suffix ? &suffix : nullptr;
        const int64_t bytes = mm_shared_prefix_attention_workspace(&p, pre, suf);
        if (bytes < 0) call(static_cast<int>(-bytes));
        at::Tensor work;
        if (bytes > 0) work = empty({bytes}, at::kByte, d);
        call(mm_shared_prefix_attention(&p, pre, suf, bytes > 0 ? work.data_ptr() : nullptr, static_cast<size_t>(bytes),
                                        stream_of(d)));
        if (!want_lse) return THPVariable_Wrap(std::move(out));
        PyObject* both = PyTuple_New(2);
        if (!both) return nullptr;
        PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(std::move(out)));
        PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(std::move(lse)));
        return both;
    });
}

// target_probs, draft_tokens, draft_len, u_accept, u_sample, draft_probs
PyObject* verify_drafts(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        arguments(n_args, 6);
        const at::Tensor& p = cuda_tensor(a[0], "target_probs");
        const c10::Device d = p.device();
        const int kind = kind_of(p.scalar_type());
        require(p.dim() == 3 && kind >= 0 && p.is_contiguous() && p.size(1) > 0,
                "target_probs is contiguous [rows, drafts + 1, vocab]");
        const int64_t B = p.size(0), K = p.size(1) - 1, V = p.size(2);
        const at::Tensor& x = tensor(a[1], "draft_tokens");
        require(x.dim() == 2 && x.size(0) == B && x.size(1) == K && x.scalar_type() == at::kInt && x.is_contiguous(),
                "draft_tokens is contiguous int32 [rows, drafts]");
        const at::Tensor& ua = tensor(a[3], "u_accept");
        const at::Tensor& us = tensor(a[4], "u_sample");
        require(ua.dim() == 2 && ua.size(0) == B && ua.size(1) == K && ua.scalar_type() == at::kFloat && ua.is_contiguous() &&
                    us.dim() == 1 && us.size(0) == B && us.scalar_type() == at::kFloat && us.is_contiguous(),
                "u_accept is contiguous fp32 [rows, drafts], u_sample fp32 [rows]");
        on(x, d);
        on(ua, d);
        on(us, d);
        const void* draft = nullptr;
        if (a[5] != Py_None) {
            const at::Tensor& q = tensor(a[5], "draft_probs");
            require(q.dim() == 3 && q.size(0) == B && q.size(1) == K && q.size(2) == V && q.scalar_type() == p.scalar_type() &&
                        q.is_contiguous(),
                    "draft_probs is contiguous [rows, drafts, vocab] of target_probs' type");
            on(q, d);
            draft = K > 0 ? q.data_ptr() : nullptr;
        }
        const int32_t* lens = ints(a[2], d, B, "draft_len");
        const c10::cuda::CUDAGuard guard(d);
        at::Tensor tokens = empty({B, K + 1}, at::kInt, d), accepted = empty({B}, at::kInt, d);
        call(mm_verify_drafts(p.data_ptr(), draft, kind, static_cast<const int32_t*>(x.data_ptr()), lens,
                              static_cast<const float*>(ua.data_ptr()), static_cast<const float*>(us.data_ptr()), size32(B),
                              size32(K), size32(V), static_cast<int32_t*>(tokens.data_ptr()),
                              static_cast<int32_t*>(accepted.data_ptr()), stream_of(d)));
        PyObject* both = PyTuple_New(2);
        if (!both) return nullptr;
        PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(std::move(tokens)));
        PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(std::move(accepted)));
        return both;
    });
}

PyMethodDef kMethods[] = {
    {"cache_write", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(cache_write)), METH_FASTCALL, nullptr},
    {"cache_read", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(cache_read)), METH_FASTCALL, nullptr},
    {"shared_prefix_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(shared_prefix_attention)), METH_FASTCALL, nullptr},
    {"verify_drafts", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(verify_drafts)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_latent_torch", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__latent_torch() { return PyModule_Create(&kModule); }
