// Binding of the paged-cache and beam-search operators (include/mm_paged.h) to torch tensors, beside
// the shared-prompt ones in _latent_torch: argument checks, outputs and workspace from torch's allocator
// on the tensors' current stream, and the C call. paged.py documents the functions and gives names
// and defaults; every refusal is an EngineError with the C code.
#include <algorithm>

#include "torch_args.h"

#include "../../include/mm_paged.h"

namespace {

const int32_t* int_table(PyObject* o, c10::Device d, mm_paged_cache* c) {
    const at::Tensor& t = tensor(o, "table");
    if (t.dim() != 2 || t.scalar_type() != at::kInt || !last_adjacent(t)) bad("table is int32 [rows, pages] with adjacent pages");
    on(t, d);
    c->table = static_cast<const int32_t*>(t.data_ptr());
    c->table_stride = t.stride(0);
    c->table_rows = size32(t.size(0));
    c->table_columns = size32(t.size(1));
    return c->table;
}

// What was written in place is no longer what autograd has kept of these tensors.
void written(PyObject* o) {
    auto bump = [](const at::Tensor& t) {
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    };
    if (THPVariable_Check(o)) return bump(THPVariable_Unpack(o));
    for (int i = 0; i < 3; ++i) bump(THPVariable_Unpack(PyTuple_GET_ITEM(o, i)));
}

PyObject* tuple(std::initializer_list<at::Tensor> ts) {
    PyObject* t = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
    if (!t) return nullptr;
    Py_ssize_t i = 0;
    for (const at::Tensor& x : ts) PyTuple_SET_ITEM(t, i++, THPVariable_Wrap(x));
    return t;
}

// cache, values, table, positions, kv_rank, rows, theta, norm, eps
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        arguments(n_args, 9);
        const at::Tensor& values = cuda_tensor(a[1], "values");
        const c10::Device d = values.device();
        const int64_t kv = integer(a[4], 0, "kv_rank");
        require(kv > 0, "kv_rank must be positive");
        mm_paged_cache c{};
        c.pool = cache(a[0], d, kv);
        int_table(a[2], d, &c);
        const int kind = kind_of(values.scalar_type());
        require(values.dim() == 2 && kind >= 0 && last_adjacent(values) && values.size(1) == static_cast<int64_t>(c.pool.kv) + c.pool.rope_dim,
                "values is fp32, fp16 or bf16 [tokens, kv + rope] of the cache's width with adjacent values");
        const int64_t n = values.size(0);
        const int32_t* positions = ints(a[3], d, n, "positions");
        const int32_t* rows = nullptr;
        if (a[5] != Py_None) rows = ints(a[5], d, n, "rows");
        else require(n == c.table_rows, "without rows there is one token per table row");
        const float* norm = nullptr;
        if (a[7] != Py_None) {
            const at::Tensor& w = tensor(a[7], "norm");
            require(w.dim() == 1 && w.size(0) == kv && w.scalar_type() == at::kFloat && w.is_contiguous(), "norm is contiguous fp32 [kv]");
            on(w, d);
            norm = static_cast<const float*>(w.data_ptr());
        }
        const c10::cuda::CUDAGuard guard(d);
        call(mm_paged_append(&c, values.data_ptr(), values.stride(0), kind, rows, positions, n, number(a[6], "theta"), norm,
                             static_cast<float>(number(a[8], "eps")), stream_of(d)));
        written(a[0]);
        Py_RETURN_NONE;
    });
}

// q, cache, table, lengths, scale, kv_rank, window, sinks, max_length, return_lse
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        arguments(n_args, 10);
        const at::Tensor& q = cuda_tensor(a[0], "q");
        const c10::Device d = q.device();
        const int kind = kind_of(q.scalar_type());
        require(q.dim() == 3 && half(kind) && last_adjacent(q), "q is fp16 or bf16 [rows, heads, kv + rope] with adjacent values");
        const int64_t B = q.size(0), H = q.size(1), W = q.size(2), kv = integer(a[5], 0, "kv_rank");
        require(kv > 0 && kv <= W && H > 0, "kv_rank must be in (0, q's width]");
        mm_paged_cache c{};
        c.pool = cache(a[1], d, kv);
        require(c.pool.kv + c.pool.rope_dim == W, "the cache's width differs from q's");
        int_table(a[2], d, &c);
        require(c.table_rows == B, "a table row per row");
        mm_paged_attention_desc p{};
        p.q = q.data_ptr();
        p.q_row_stride = q.stride(0);
        p.q_head_stride = q.stride(1);
        p.lengths = ints(a[3], d, B, "lengths");
        p.dtype = kind;
        p.rows = size32(B);
        p.heads = size32(H);
        const int64_t most = static_cast<int64_t>(c.table_columns) * c.pool.positions;
        p.max_length = static_cast<int32_t>(integer(a[8], size32(most), "max_length"));
        if (a[6] != Py_None) {
            p.window = static_cast<int32_t>(integer(a[6], 0, "window"));
            require(p.window > 0, "window must be positive (None: the whole row)");
        }
        p.sinks = static_cast<int32_t>(integer(a[7], 0, "sinks"));
        p.scale = static_cast<float>(number(a[4]));
        const bool want_lse = truth(a[9], "return_lse");
        const c10::cuda::CUDAGuard guard(d);
        at::Tensor out = empty({B, H, kv}, q.scalar_type(), d), lse;
        p.out = out.data_ptr();
        if (want_lse) {
            lse = empty({B, H}, at::kFloat, d);
            p.lse = static_cast<float*>(lse.data_ptr());
        }
        const int64_t bytes = mm_paged_attention_workspace(&p, &c);
        if (bytes < 0) call(static_cast<int>(-bytes));
        at::Tensor work;
        if (bytes > 0) work = empty({bytes}, at::kByte, d);
        call(mm_paged_attention(&p, &c, bytes > 0 ? work.data_ptr() : nullptr, static_cast<size_t>(bytes), stream_of(d)));
        if (!want_lse) return THPVariable_Wrap(std::move(out));
        return tuple({out, lse});
    });
}

// logits, scores, beams, finished, eos
PyObject* beam_select(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        arguments(n_args, 5);
        const at::Tensor& x = cuda_tensor(a[0], "logits");
        const c10::Device d = x.device();
        const int kind = kind_of(x.scalar_type());
        require(x.dim() == 3 && kind >= 0 && last_adjacent(x) && x.size(1) > 0 && x.size(2) > 0,
                "logits is fp32, fp16 or bf16 [batch, beams, vocab] with adjacent tokens");
        const int64_t B = x.size(0), K = x.size(1), V = x.size(2), n = integer(a[2], K, "beams");
        const at::Tensor& s = tensor(a[1], "scores");
        require(s.dim() == 2 && s.size(0) == B && s.size(1) == K && s.scalar_type() == at::kFloat && s.is_contiguous(),
                "scores is contiguous fp32 [batch, beams]");
        on(s, d);
        const uint8_t* finished = nullptr;
        if (a[3] != Py_None) {
            const at::Tensor& f = tensor(a[3], "finished");
            require(f.dim() == 2 && f.size(0) == B && f.size(1) == K && f.scalar_type() == at::kBool && f.is_contiguous(),
                    "finished is contiguous bool [batch, beams]");
            on(f, d);
            finished = static_cast<const uint8_t*>(f.data_ptr());
            require(a[4] != Py_None, "finished beams need eos");
        }
        const int64_t eos = integer(a[4], 0, "eos");
        require(n > 0, "beams must be positive");
        const c10::cuda::CUDAGuard guard(d);
        const int64_t bytes = mm_beam_select_workspace(size32(B), size32(K), size32(V), size32(n));
        if (bytes < 0) call(static_cast<int>(-bytes));
        at::Tensor scores = empty({B, n}, at::kFloat, d), parents = empty({B, n}, at::kInt, d), tokens = empty({B, n}, at::kInt, d), work;
        if (bytes > 0) work = empty({bytes}, at::kByte, d);
        call(mm_beam_select(x.data_ptr(), x.stride(0), x.stride(1), kind, static_cast<const float*>(s.data_ptr()), finished,
                            static_cast<int>(eos), size32(B), size32(K), size32(V), size32(n), static_cast<float*>(scores.data_ptr()),
                            static_cast<int32_t*>(parents.data_ptr()), static_cast<int32_t*>(tokens.data_ptr()),
                            bytes > 0 ? work.data_ptr() : nullptr, static_cast<size_t>(bytes), stream_of(d)));
        return tuple({scores, parents, tokens});
    });
}

// cache (with layers ahead), table, spare, lengths, parents
PyObject* beam_reorder(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        arguments(n_args, 5);
        const at::Tensor& t = cuda_tensor(a[1], "table");
        const c10::Device d = t.device();
        mm_paged_cache c{};
        int_table(a[1], d, &c);
        int64_t strides[3] = {0, 0, 0}, layers = 0;
        if (THPVariable_Check(a[0])) {
            const at::Tensor& x = no_gradient(THPVariable_Unpack(a[0]));
            require(x.dim() == 4, "the cache has its layers ahead: [layers, pages, page_size, kv + rope]");
            const int kind = kind_of(x.scalar_type());
            require(half(kind) && last_adjacent(x) && x.size(3) > 0, "a 16-bit cache is fp16 or bf16 with adjacent values");
            on(x, d);
            c.pool.latent = x.data_ptr();
            c.pool.row_stride = x.stride(1);
            c.pool.pos_stride = x.stride(2);
            c.pool.rows = size32(x.size(1));
            c.pool.positions = size32(x.size(2));
            // (kv_rank is not an argument: the copies take positions whole, so that any cut which the C entry takes will do)
            c.pool.kv = std::min(size32(x.size(3)), 1024);
            c.pool.rope_dim = size32(x.size(3)) - c.pool.kv;
            c.pool.kind = c.pool.rope_kind = kind;
            layers = x.size(0);
            strides[0] = x.stride(0);
        } else {
            require(PyTuple_Check(a[0]) && PyTuple_GET_SIZE(a[0]) == 3, "a cache is a tensor or a LatentCache");
            const at::Tensor& lat = tensor(PyTuple_GET_ITEM(a[0], 0), "a cache's latent");
            const at::Tensor& rope = tensor(PyTuple_GET_ITEM(a[0], 1), "a cache's rope");
            const at::Tensor& scale = tensor(PyTuple_GET_ITEM(a[0], 2), "a cache's scale");
            const int kind = kind_of(rope.scalar_type());
            require(lat.dim() == 4 && rope.dim() == 4 && scale.dim() == 3, "the cache has its layers ahead: [layers, pages, page_size, ...]");
            for (int i = 0; i < 3; ++i)
                require(rope.size(i) == lat.size(i) && scale.size(i) == lat.size(i), "a cache's tensors differ in size");
            require(lat.scalar_type() == at::kFloat8_e4m3fn && half(kind) && scale.scalar_type() == at::kFloat && last_adjacent(lat) &&
                        last_adjacent(rope) && last_adjacent(scale),
                    "an 8-bit cache is float8_e4m3fn latents, fp16 or bf16 rope keys and fp32 scales with adjacent values");
            on(lat, d);
            on(rope, d);
            on(scale, d);
            c.pool.latent = lat.data_ptr();
            c.pool.rope = rope.data_ptr();
            c.pool.scale = static_cast<float*>(scale.data_ptr());
            c.pool.row_stride = lat.stride(1);
            c.pool.pos_stride = lat.stride(2);
            c.pool.rope_row_stride = rope.stride(1);
            c.pool.rope_pos_stride = rope.stride(2);
            c.pool.scale_row_stride = scale.stride(1);
            c.pool.rows = size32(lat.size(1));
            c.pool.positions = size32(lat.size(2));
            c.pool.kv = size32(lat.size(3));
            c.pool.rope_dim = size32(rope.size(3));
            c.pool.kind = MM_E4M3;
            c.pool.rope_kind = kind;
            layers = lat.size(0);
            strides[0] = lat.stride(0);
            strides[1] = rope.stride(0);
            strides[2] = scale.stride(0);
        }
        const int64_t rows = c.table_rows, columns = c.table_columns;
        const int32_t* spare = ints(a[2], d, rows, "spare");
        const int32_t* lengths = ints(a[3], d, rows, "lengths");
        const int32_t* parents = ints(a[4], d, rows, "parents");
        const c10::cuda::CUDAGuard guard(d);
        at::Tensor table = empty({rows, columns}, at::kInt, d), out_spare = empty({rows}, at::kInt, d), out_lengths = empty({rows}, at::kInt, d);
        call(mm_beam_reorder(&c, size32(layers), strides, spare, lengths, parents, static_cast<int32_t*>(table.data_ptr()),
                             static_cast<int32_t*>(out_spare.data_ptr()), static_cast<int32_t*>(out_lengths.data_ptr()), stream_of(d)));
        written(a[0]);
        return tuple({table, out_spare, out_lengths});
    });
}

}  // namespace

// Added to _latent_torch's methods when the module is made.
PyMethodDef kPagedMethods[] = {
    {"paged_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(append)), METH_FASTCALL, nullptr},
    {"paged_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(attention)), METH_FASTCALL, nullptr},
    {"beam_select", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(beam_select)), METH_FASTCALL, nullptr},
    {"beam_reorder", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(beam_reorder)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
