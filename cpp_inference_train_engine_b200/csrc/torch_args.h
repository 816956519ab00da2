// Arguments and results of the C operators' torch bindings: refusals, tensor checks, outputs from
// torch's allocator. Written against the CPython C API because a small decode step is bound by this
// path: the same checks through Python attributes took 9 to 21 us a call, the kernels 2 to 12.
#pragma once
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Dtype.h>

#include <ATen/core/grad_mode.h>
#include <c10/core/AutogradState.h>
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

// The calls read the storage: a view that stands for other values than it holds (a negated one, as of a conjugate's
// imaginary part, or one of zeros without storage) would be taken for what is stored.
const at::Tensor& as_stored(const at::Tensor& t) {
    if (t.is_neg() || t.is_conj() || t._is_zerotensor())
        bad("a tensor whose storage does not hold its values: call resolve_neg() or clone() on it");
    return t;
}
// The calls go past autograd: a result would silently be a constant of its inputs, in backward and in forward mode.
const at::Tensor& no_gradient(const at::Tensor& t) {
    if (t.requires_grad() && at::GradMode::is_enabled())
        bad("no gradient flows through these operators: detach the tensors that require one, or call under torch.no_grad()");
    if (t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
        bad("no tangent flows through these operators: unpack the dual tensors");
    return as_stored(t);
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

double number(PyObject* o, const char* what = "scale") {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        bad(std::string(what) + " must be a number");
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
// An object's truth value, where it has one.
bool truth(PyObject* o, const char* what) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) {
        PyErr_Clear();
        bad(std::string(what) + " must be true or false");
    }
    return v != 0;
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
    const at::Tensor& t = as_stored(THPVariable_Unpack(o));
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

}  // namespace
