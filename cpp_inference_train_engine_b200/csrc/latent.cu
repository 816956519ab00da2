// C entries of the shared-prompt decode operators (include/mm_latent.h): argument checks,
// variant selection and launches. Everything is enqueued on the caller's stream; no entry
// allocates or throws, and none but mm_latent_status waits.
#include <algorithm>
#include <cstring>

#include "draft_verify.cuh"
#include "entries.cuh"
#include "latent_cache.cuh"
#include "shared_prefix.cuh"
#include "shared_prefix_tc.cuh"

#include "../../include/mm_latent.h"

using namespace mm::entry;

namespace {

static_assert(sizeof(mm_latent_cache) == 88 && sizeof(mm_shared_prefix_desc) == 112, "callers without this header pack these field by field");

// The vector forms of cache write and read: the models' widths, 16-byte aligned rows.
template <class F> bool with_width(const mm_latent_cache* c, bool aligned, F&& f) {
    if (!aligned || !aligned_e4m3(c)) return false;
    if (c->kv == 128 && c->rope_dim == 16) f(std::integral_constant<int, 128>{}, std::integral_constant<int, 16>{});
    else if (c->kv == 512 && c->rope_dim == 32) f(std::integral_constant<int, 512>{}, std::integral_constant<int, 32>{});
    else return false;
    return true;
}

mm::spa::Problem problem(const mm_shared_prefix_desc* d, const mm_latent_cache* prefix, const mm_latent_cache* suffix) {
    require(d != nullptr, "null description");
    require(d->rows >= 0 && d->tokens >= 1 && d->heads >= 1 && d->groups >= 0, "shared-prefix attention: invalid sizes");
    require(d->dtype == MM_F16 || d->dtype == MM_BF16, "shared-prefix attention: q must be fp16 or bf16");
    require(prefix || suffix, "shared-prefix attention: a prefix or a suffix cache is needed");
    require(static_cast<long long>(d->rows) * d->tokens <= kMaxBlocks / d->heads,
            "shared-prefix attention: too many query rows");
    for (const mm_latent_cache* c : {prefix, suffix})
        if (c) {
            check_cache(c);
            require(c->kind == d->dtype || (c->kind == MM_E4M3 && c->rope_kind == d->dtype),
                    "shared-prefix attention: the cache's type must be q's (an e4m3 cache's rope type)");
        }
    if (prefix && suffix)
        require(prefix->kv == suffix->kv && prefix->rope_dim == suffix->rope_dim,
                "shared-prefix attention: prefix and suffix widths differ");
    require(d->groups == 0 || (prefix && prefix->rows >= d->groups), "shared-prefix attention: a prefix row per group");
    require(!suffix || suffix->rows >= d->rows, "shared-prefix attention: a suffix row per row");
    require(d->max_group >= 0 && d->max_prefix >= 0 && d->max_suffix >= 0 &&
                d->max_prefix <= (prefix ? prefix->positions : 0) &&
                d->max_suffix <= (suffix ? suffix->positions : 0),
            "shared-prefix attention: max_prefix / max_suffix exceed the cache's positions");
    if (d->rows > 0) {
        require(d->q && d->out, "shared-prefix attention: null q or out");
        require(multiple(d->q, 2) && multiple(d->out, 2) && multiple(d->lse, 4),
                "shared-prefix attention: q, out or lse not aligned to its elements");
        require(d->groups == 0 || (d->group_start && d->prefix_len), "shared-prefix attention: null group_start or prefix_len");
        require(d->max_suffix == 0 || d->suffix_len, "shared-prefix attention: null suffix_len");
    }
    const mm_latent_cache* any = prefix ? prefix : suffix;
    mm::spa::Problem p{};
    p.q = d->q;
    p.q_row = d->q_row_stride;
    p.q_tok = d->q_token_stride;
    p.q_head = d->q_head_stride;
    p.B = d->rows;
    p.T = d->tokens;
    p.H = d->heads;
    p.prefix = view(prefix);
    p.suffix = view(suffix);
    p.group_start = d->group_start;
    p.prefix_len = d->prefix_len;
    p.suffix_len = d->suffix_len;
    p.G = d->max_prefix > 0 && d->max_group > 0 ? d->groups : 0;
    p.max_group = std::min(d->max_group, d->rows);
    p.max_prefix = d->max_prefix;
    p.max_suffix = d->max_suffix;
    p.kv = any->kv;
    p.rd = any->rope_dim;
    p.scale = d->scale;
    p.out = d->out;
    p.lse = d->lse;
    return p;
}

template <typename T, bool Q8P, bool Q8S> void launch_any_width(const mm::spa::Problem& p, cudaStream_t s) {
    using namespace mm::spa;
    const int smem = kAnyWarps * (2 * p.kv + p.rd) * 4;  // at most 36 KB
    launch(s, any_width_kernel<T, Q8P, Q8S>, dim3(blocks(static_cast<long long>(p.B) * p.T * p.H, kAnyWarps)),
           dim3(32 * kAnyWarps), smem, p);
}

// ------------------------------------------------------------------ tensor-core plan
// The tensor-core form covers the two latent widths of the framework's models when every row
// can be read in 16-byte pieces and the results written in 8-byte ones (the join kernel).
bool aligned_cache(const mm_latent_cache* c) {
    if (c->kind == MM_E4M3) return aligned_e4m3(c);
    // 16-bit caches come by tensor maps: strides of up to 40 bits in bytes, rows that may be one and the same
    constexpr int64_t kMost = 1LL << 39;
    return multiple(c->latent, 16) && c->row_stride % 8 == 0 && c->pos_stride % 8 == 0 && c->pos_stride > 0 && c->pos_stride < kMost &&
           c->row_stride >= 0 && c->row_stride < kMost;
}
bool tensor_core_form(const mm::spa::Problem& p, const mm_latent_cache* prefix, const mm_latent_cache* suffix) {
    if (!((p.kv == 128 && p.rd == 16) || (p.kv == 512 && p.rd == 32))) return false;
    if (!multiple(p.q, 16) || p.q_row % 8 || p.q_tok % 8 || p.q_head % 8 || !multiple(p.out, 8)) return false;
    return (p.G == 0 || aligned_cache(prefix)) && (p.max_suffix == 0 || aligned_cache(suffix));
}

struct Plan {
    int pre_n = 0, pre_splits = 0, pre_kps = 128;  // queries per block (0: no prefix launch), ranges, keys per range
    int suf_n = 0, suf_splits = 0, suf_kps = 128;
    long long pre_blocks = 0, suf_blocks = 0;      // upper bounds of the query blocks
    bool join = false;                             // a join launch: not every row is one suffix range
    long long rows = 0;                            // query rows
    long long pre_part = 0, suf_part = 0;          // partial query rows held by the workspace
    bool span = false;                             // suffix rows in even shares of their tiles (TcArgs::pieces)
    long long pieces = 0;                          // rows whose parts the workspace lists
    long long bytes(int kv) const { return (pre_part + suf_part) * (kv + 2) * 4 + pieces * 8; }
};

// Key ranges per query block: the waves of (block, range) items over the SMs times an item's
// tiles, plus what an item costs beside its tiles (two) and the join of several ranges (one). Measured
// with other costs: items at one, 600 rows of 2,048 positions, 128 + 16 wide, 79.5 us instead of 79.9; the
// join at four, prompts of 512 under 512 + 32 wide ragged rows are not split, 63.6 us instead of 61.6.
void pick_splits(long long blocks, int keys, int most, int& splits, int& kps) {
    const int tiles = (keys + 127) / 128, sms = sm_count();
    double best = 0;
    splits = 0;
    for (int s = 1; s <= std::min(tiles, most); ++s) {
        const int per = (tiles + s - 1) / s, n = (tiles + per - 1) / per;
        if (n != s) continue;
        const double cost = static_cast<double>((blocks * n + sms - 1) / sms) * (per + 2.0) + (n > 1 ? 1.0 + 0.05 * n : 0.0);
        if (!splits || cost < best) {
            best = cost;
            splits = n;
            kps = per * 128;
        }
    }
}

Plan plan(const mm::spa::Problem& p) {
    Plan r;
    const long long th = static_cast<long long>(p.T) * p.H;
    r.rows = th * p.B;
    if (p.G > 0) {
        r.pre_n = p.max_group * th <= 16 ? 16 : 64;
        r.pre_blocks = std::min((r.rows + r.pre_n - 1) / r.pre_n + p.G, p.G * ((p.max_group * th + r.pre_n - 1) / r.pre_n));
        pick_splits(r.pre_blocks, p.max_prefix, 64, r.pre_splits, r.pre_kps);
        r.pre_part = r.rows * r.pre_splits;
    }
    if (p.max_suffix > 0) {
        r.suf_n = th <= 16 ? 16 : 64;
        r.suf_blocks = p.B * ((th + r.suf_n - 1) / r.suf_n);
        pick_splits(r.suf_blocks, p.max_suffix, 16, r.suf_splits, r.suf_kps);
        // Rows long enough to be worth cutting, one range each: the launch may divide them by their lengths
        using C = mm::spa::TcCfg<512, 32, 16, false>;
        const long long ctas = sm_count() * C::kCtas, tiles = (p.max_suffix + C::KT - 1) / C::KT, weight = p.B * (tiles + 1);
        r.span = p.kv == 512 && r.suf_n == 16 && r.suf_splits == 1 && tiles >= 8 && r.pre_splits <= mm::spa::kMaxJoin &&
                 weight + ctas * mm::spa::kMinSpan <= kMaxBlocks;
        if (r.span) {
            r.suf_blocks = std::min(ctas, weight);
            r.suf_part = 2 * r.suf_blocks * 16;
            r.pieces = p.B;
        }
    }
    r.join = r.span || r.suf_n != 16 || r.suf_splits > 1 || r.pre_splits > mm::spa::kMaxJoin;
    if (r.join && !r.span) r.suf_part = r.rows * r.suf_splits;
    if (r.pre_blocks * std::max(1, r.pre_splits) > kMaxBlocks || r.suf_blocks * std::max(1, r.suf_splits) > kMaxBlocks)
        refuse(MM_UNSUPPORTED, "shared-prefix attention: too many query rows");
    return r;
}

// The tensor maps of a 16-bit cache: whole tiles, blocks of 32 positions, and their rope columns.
struct Maps {
    CUtensorMap tile{}, block{}, rope{};
};

// Boxes of `box` columns x `keys` positions of one cache row. False where the encoder does not take
// the cache's strides.
bool cache_map(CUtensorMap* map, const mm_latent_cache* c, int box, int keys, CUtensorMapSwizzle swizzle) {
    const bool rows = c->rows > 1 && c->row_stride > 0;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(c->kv + c->rope_dim), static_cast<cuuint64_t>(c->positions),
                                static_cast<cuuint64_t>(rows ? c->rows : 1)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(c->pos_stride) * 2,
                                   static_cast<cuuint64_t>(rows ? c->row_stride : c->pos_stride) * 2};
    const cuuint32_t boxes[3] = {static_cast<cuuint32_t>(box), static_cast<cuuint32_t>(keys), 1}, steps[3] = {1, 1, 1};
    return tensor_map_encoder()(map, c->kind == MM_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                                c->latent, dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool cache_maps(Maps& m, const mm_latent_cache* c) {
    if (c->kind == MM_E4M3) return true;  // read without maps
    const int keys = c->kv == 512 ? mm::spa::TcCfg<512, 32, 16, false>::KT : mm::spa::TcCfg<128, 16, 16, false>::KT;
    return cache_map(&m.tile, c, 64, keys, CU_TENSOR_MAP_SWIZZLE_128B) && cache_map(&m.block, c, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B) &&
           cache_map(&m.rope, c, c->rope_dim, 32, c->rope_dim == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B);
}

template <int KV, int R, int N, typename T, bool Q8, bool CAUSAL>
void launch_tc(mm::spa::TcArgs a, const Maps& m, long long items, cudaStream_t s) {
    using C = mm::spa::TcCfg<KV, R, N, Q8>;
    const mm::lat::CacheView& c = a.suffix ? a.p.suffix : a.p.prefix;
    a.apart = std::min(a.p.T - 1, (N + a.p.H - 2) / a.p.H);
    a.map_rows = c.rows > 1 && c.row_stride > 0 ? 1 : 0;
    set_dynamic_smem<mm::spa::shared_prefix_tc_kernel<KV, R, N, T, Q8, CAUSAL>>(C::kSmem);
    launch(s, mm::spa::shared_prefix_tc_kernel<KV, R, N, T, Q8, CAUSAL>,
           dim3(static_cast<unsigned>(std::min<long long>(items, sm_count() * C::kCtas))), dim3(C::kThreads), C::kSmem, a,
           m.tile, m.block, m.rope);
}
template <int KV, int R, typename T>
void launch_tc_n(const mm::spa::TcArgs& a, const Maps& m, int n, bool q8, long long items, cudaStream_t s) {
    auto go = [&](auto size, auto codes) {
        constexpr int N = decltype(size)::value;
        constexpr bool Q8 = decltype(codes)::value;
        if (a.p.T > 1) launch_tc<KV, R, N, T, Q8, true>(a, m, items, s);
        else launch_tc<KV, R, N, T, Q8, false>(a, m, items, s);
    };
    using N16 = std::integral_constant<int, 16>;
    using N64 = std::integral_constant<int, 64>;
    if (n == 16) q8 ? go(N16{}, std::true_type{}) : go(N16{}, std::false_type{});
    else q8 ? go(N64{}, std::true_type{}) : go(N64{}, std::false_type{});
}

template <int KV, int R, typename T>
void run_tc(const mm::spa::Problem& p, const Plan& r, const Maps& pre, const Maps& suf, bool q8p, bool q8s, void* workspace,
            cudaStream_t s) {
    using namespace mm::spa;
    float* w = static_cast<float*>(workspace);
    float* pre_o = w;
    float* suf_o = pre_o + r.pre_part * KV;
    float2* pre_ml = reinterpret_cast<float2*>(suf_o + r.suf_part * KV);
    float2* suf_ml = pre_ml + r.pre_part;
    int2* pieces = r.span ? reinterpret_cast<int2*>(suf_ml + r.suf_part) : nullptr;
    TcArgs a{};
    a.p = p;
    if (r.pre_n) {
        a.splits = r.pre_splits;
        a.kps = r.pre_kps;
        a.part_o = pre_o;
        a.part_ml = pre_ml;
        launch_tc_n<KV, R, T>(a, pre, r.pre_n, q8p, r.pre_blocks * r.pre_splits, s);
    }
    if (r.suf_n) {
        a.suffix = 1;
        a.splits = r.suf_splits;
        a.kps = r.suf_kps;
        a.part_o = suf_o;
        a.part_ml = suf_ml;
        a.pre_o = pre_o;
        a.pre_ml = pre_ml;
        a.prefix_kps = r.pre_kps;
        a.overlap = r.pre_n ? 1 : 0;
        a.pieces = pieces;
        launch_tc_n<KV, R, T>(a, suf, r.suf_n, q8s, r.suf_blocks * r.suf_splits, s);
    }
    if (r.join)
        launch(s, r.span ? shared_prefix_join_kernel<KV, T, true> : shared_prefix_join_kernel<KV, T, false>, dim3(blocks(r.rows, 8)),
               dim3(256), 0, p, static_cast<const float*>(pre_o), static_cast<const float2*>(pre_ml), r.pre_kps,
               static_cast<const float*>(suf_o), static_cast<const float2*>(suf_ml), r.suf_kps, r.suf_n == 16 ? 1 : 0,
               static_cast<const int2*>(pieces));
}

}  // namespace

extern "C" {

size_t mm_latent_last_error(char* buf, size_t cap) {
    if (buf && cap > 0) {
        const size_t n = std::min(cap - 1, g_error.size());
        std::memcpy(buf, g_error.data(), n);
        buf[n] = 0;
    }
    return g_error.size();
}

int mm_latent_status(void* stream) {
    return guarded([&] {
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        int bits = 0;
        const int none = 0;
        check(cudaMemcpyFromSymbolAsync(&bits, mm::spa::latent_status, sizeof bits, 0, cudaMemcpyDeviceToHost, s), "status");
        check(cudaStreamSynchronize(s), "status");
        if (!bits) return;
        check(cudaMemcpyToSymbolAsync(mm::spa::latent_status, &none, sizeof none, 0, cudaMemcpyHostToDevice, s), "status");
        check(cudaStreamSynchronize(s), "status");
        refuse(MM_GPU_ERROR, "shared-prefix attention: a kernel gave up on a wait; its results are NaN");
    });
}

int mm_latent_cache_write(const mm_latent_cache* cache, const void* latent, int64_t latent_stride, const void* rope,
                          int64_t rope_stride, int dtype, const int64_t* slots, int64_t n, void* stream) {
    return guarded([&] {
        require(cache != nullptr && n >= 0, "cache write: null cache or negative count");
        check_cache(cache);
        require(cache->kind == MM_E4M3, "cache write: the cache must be an e4m3 one");
        if (n == 0 || cache->rows == 0 || cache->positions == 0) return;
        require(latent && slots && (rope || cache->rope_dim == 0), "cache write: null input");
        mm::lat::CacheOut c{static_cast<uint8_t*>(cache->latent), static_cast<uint8_t*>(cache->rope), cache->scale,
                            cache->row_stride, cache->pos_stride, cache->rope_row_stride, cache->rope_pos_stride,
                            cache->scale_row_stride, cache->rows, cache->positions};
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        with_type(dtype, [&](auto in) {
            with_half(cache->rope_kind, [&](auto half) {
                using T = typename decltype(in)::type;
                using T16 = typename decltype(half)::type;
                require(multiple(latent, sizeof(T)) && multiple(rope, sizeof(T)), "cache write: input not aligned to its elements");
                const long long e = 16 / sizeof(T);
                const bool aligned = reinterpret_cast<uintptr_t>(latent) % 16 == 0 && latent_stride % e == 0 &&
                                     reinterpret_cast<uintptr_t>(rope) % 16 == 0 && rope_stride % e == 0;
                if (with_width(cache, aligned, [&](auto kv, auto rd) {
                        // 8 warps of 512 / kv positions each; at most the CTAs that are resident together
                        constexpr int kKv = decltype(kv)::value, kRd = decltype(rd)::value;
                        const unsigned ctas = std::min(blocks(n, 8 * (512 / kKv)),
                                                       static_cast<unsigned>(sm_count() * mm::lat::kWriteCtas<T>));
                        launch(s, mm::lat::latent_write_vec_kernel<T, T16, kKv, kRd>, dim3(ctas), dim3(256), 0, c,
                               static_cast<const T*>(latent), static_cast<long long>(latent_stride), static_cast<const T*>(rope),
                               static_cast<long long>(rope_stride), reinterpret_cast<const long long*>(slots),
                               static_cast<long long>(n));
                    }))
                    return;
                launch(s, mm::lat::latent_write_kernel<T, T16>, dim3(blocks(n, 8)), dim3(256), 0, c,
                       static_cast<const T*>(latent), static_cast<long long>(latent_stride), static_cast<const T*>(rope),
                       static_cast<long long>(rope_stride), reinterpret_cast<const long long*>(slots),
                       static_cast<long long>(n), cache->kv, cache->rope_dim);
            });
        });
    });
}

int mm_latent_cache_read(const mm_latent_cache* cache, const int64_t* slots, int64_t n, void* out, int64_t out_stride,
                         int out_dtype, void* stream) {
    return guarded([&] {
        require(cache != nullptr && n >= 0, "cache read: null cache or negative count");
        check_cache(cache);
        require(cache->kind == MM_E4M3, "cache read: the cache must be an e4m3 one");
        if (n == 0) return;
        require(slots && out, "cache read: null argument");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        with_type(out_dtype, [&](auto o) {
            with_half(cache->rope_kind, [&](auto half) {
                using TO = typename decltype(o)::type;
                using T16 = typename decltype(half)::type;
                require(multiple(out, sizeof(TO)), "cache read: out not aligned to its elements");
                const bool aligned = reinterpret_cast<uintptr_t>(out) % 16 == 0 && out_stride * sizeof(TO) % 16 == 0;
                if (with_width(cache, aligned, [&](auto kv, auto rd) {
                        constexpr int kKv = decltype(kv)::value, kRd = decltype(rd)::value, kU = 2;
                        launch(s, mm::lat::latent_read_vec_kernel<T16, TO, kKv, kRd, kU>,
                               dim3(blocks(n, 8 * kU * (512 / kKv))), dim3(256), 0, view(cache),
                               reinterpret_cast<const long long*>(slots), static_cast<long long>(n), static_cast<TO*>(out),
                               static_cast<long long>(out_stride));
                    }))
                    return;
                launch(s, mm::lat::latent_read_kernel<T16, TO>, dim3(blocks(n, 8)), dim3(256), 0, view(cache),
                       reinterpret_cast<const long long*>(slots), static_cast<long long>(n), static_cast<TO*>(out),
                       static_cast<long long>(out_stride), cache->kv, cache->rope_dim);
            });
        });
    });
}

int64_t mm_shared_prefix_attention_workspace(const mm_shared_prefix_desc* desc, const mm_latent_cache* prefix,
                                             const mm_latent_cache* suffix) {
    int64_t bytes = 0;
    const int rc = guarded([&] {
        const mm::spa::Problem p = problem(desc, prefix, suffix);
        if (p.B > 0 && tensor_core_form(p, prefix, suffix)) bytes = plan(p).bytes(p.kv);
    });
    return rc ? -static_cast<int64_t>(rc) : bytes;
}

int mm_shared_prefix_attention(const mm_shared_prefix_desc* desc, const mm_latent_cache* prefix, const mm_latent_cache* suffix,
                               void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&] {
        const mm::spa::Problem p = problem(desc, prefix, suffix);
        if (p.B == 0) return;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const bool q8p = prefix && prefix->kind == MM_E4M3;
        const bool q8s = suffix && suffix->kind == MM_E4M3;
        Maps pre, suf;
        if (tensor_core_form(p, prefix, suffix) && (p.G == 0 || cache_maps(pre, prefix)) && (p.max_suffix == 0 || cache_maps(suf, suffix))) {
            const Plan r = plan(p);
            const long long need = r.bytes(p.kv);
            require(need == 0 || (workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 &&
                                  workspace_bytes >= static_cast<size_t>(need)),
                    "shared-prefix attention: workspace too small or not 16-byte aligned");
            with_half(desc->dtype, [&](auto half) {
                using T = typename decltype(half)::type;
                if (p.kv == 128) run_tc<128, 16, T>(p, r, pre, suf, q8p, q8s, workspace, s);
                else run_tc<512, 32, T>(p, r, pre, suf, q8p, q8s, workspace, s);
            });
            return;
        }
        with_half(desc->dtype, [&](auto half) {
            using T = typename decltype(half)::type;
            if (q8p && q8s) launch_any_width<T, true, true>(p, s);
            else if (q8p) launch_any_width<T, true, false>(p, s);
            else if (q8s) launch_any_width<T, false, true>(p, s);
            else launch_any_width<T, false, false>(p, s);
        });
    });
}

int mm_verify_drafts(const void* target_probs, const void* draft_probs, int dtype, const int32_t* draft_tokens,
                     const int32_t* draft_len, const float* u_accept, const float* u_sample, int rows, int drafts,
                     int vocab, int32_t* out_tokens, int32_t* accepted, void* stream) {
    return guarded([&] {
        require(rows >= 0 && drafts >= 0 && vocab >= 1, "draft verification: invalid sizes");
        if (vocab > mm::ver::kMaxVocab) refuse(MM_UNSUPPORTED, "draft verification: vocabulary over 262,144");
        if (rows == 0) return;
        require(target_probs && draft_len && u_sample && out_tokens && accepted &&
                    (drafts == 0 || (draft_tokens && u_accept)),
                "draft verification: null argument");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        with_type(dtype, [&](auto t) {
            using T = typename decltype(t)::type;
            const T* p = static_cast<const T*>(target_probs);
            const T* q = drafts > 0 ? static_cast<const T*>(draft_probs) : nullptr;
            require(multiple(p, sizeof(T)) && multiple(q, sizeof(T)), "draft verification: probabilities not aligned to their elements");
            auto fits = [&](const void* x) { return reinterpret_cast<uintptr_t>(x) % (4 * sizeof(T)) == 0; };
            auto run = [&](auto kernel, int threads) {
                launch(s, kernel, dim3(rows), dim3(threads), 0, p, q, draft_tokens, draft_len, u_accept, u_sample, drafts, vocab,
                       out_tokens, accepted);
            };
            const bool aligned = vocab % 4 == 0 && fits(p) && fits(q);
            if (rows > 2 * sm_count())
                aligned ? run(mm::ver::verify_drafts_kernel<T, true, 512>, 512) : run(mm::ver::verify_drafts_kernel<T, false, 512>, 512);
            else
                aligned ? run(mm::ver::verify_drafts_kernel<T, true, 1024>, 1024) : run(mm::ver::verify_drafts_kernel<T, false, 1024>, 1024);
        });
    });
}

}  // extern "C"
