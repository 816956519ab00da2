// C entries of the paged-cache and beam-search operators (include/mm_paged.h): argument checks,
// variant selection and launches. Everything is enqueued on the caller's stream; no entry
// allocates or throws, and none but mm_paged_status waits.
#include <algorithm>
#include <cmath>

#include "beam_select.cuh"
#include "entries.cuh"
#include "paged_attention.cuh"
#include "paged_attention_mma.cuh"
#include "paged_cache.cuh"

#include "../../include/mm_paged.h"

using namespace mm::entry;

namespace {

static_assert(sizeof(mm_paged_cache) == 112 && sizeof(mm_paged_attention_desc) == 80, "callers without this header pack these field by field");

mm::paged::Table table_of(const mm_paged_cache* c) {
    const int page = c->pool.positions;
    int shift = 0;
    while (1LL << shift < page) ++shift;
    return {c->table, c->table_stride, c->table_rows, c->table_columns, 1LL << shift == page ? shift : -1};
}

void check_paged(const mm_paged_cache* c) {
    require(c != nullptr, "paged cache: null description");
    check_cache(&c->pool);
    require(c->pool.positions >= 1, "paged cache: a page holds one position or more");
    require(c->table_rows >= 0 && c->table_columns >= 0, "paged cache: negative size");
    require(static_cast<long long>(c->table_columns) * c->pool.positions <= INT32_MAX, "paged cache: a row's positions exceed 32 bits");
    require((c->table && multiple(c->table, 4)) || c->table_rows == 0 || c->table_columns == 0, "paged cache: null or misaligned table");
}

mm::lat::CacheOut out_view(const mm_latent_cache* c) {
    return {static_cast<uint8_t*>(c->latent), static_cast<uint8_t*>(c->rope), c->scale, c->row_stride, c->pos_stride,
            c->rope_row_stride, c->rope_pos_stride, c->scale_row_stride, c->rows, c->positions};
}

// The vector form of append: the models' widths, 16-byte aligned rows.
template <typename T> bool append_vector_form(const mm_latent_cache& c, const void* values, int64_t stride, const float* norm) {
    if (!((c.kv == 128 && c.rope_dim == 16) || (c.kv == 512 && c.rope_dim == 32))) return false;
    if (!multiple(values, 16) || stride * static_cast<int64_t>(sizeof(T)) % 16 || !multiple(norm, 16)) return false;
    if (c.kind == MM_E4M3) return aligned_e4m3(&c);
    return multiple(c.latent, 16) && c.row_stride % 8 == 0 && c.pos_stride % 8 == 0;
}

mm::paged::Attention problem(const mm_paged_attention_desc* d, const mm_paged_cache* c) {
    require(d != nullptr, "null description");
    check_paged(c);
    require(d->rows >= 0 && d->heads >= 1 && d->rows <= kMaxBlocks / d->heads, "paged attention: invalid sizes");
    require(d->dtype == MM_F16 || d->dtype == MM_BF16, "paged attention: q must be fp16 or bf16");
    const int kind = c->pool.kind == MM_E4M3 ? c->pool.rope_kind : c->pool.kind;
    require(kind == d->dtype, "paged attention: the cache's type must be q's (an e4m3 cache's rope type)");
    require(d->rows <= c->table_rows, "paged attention: a table row per row");
    require(d->window >= 0 && d->sinks >= 0, "paged attention: negative window or sinks");
    require(d->max_length >= 0 && d->max_length <= static_cast<long long>(c->table_columns) * c->pool.positions,
            "paged attention: max_length exceeds the table");
    if (d->rows > 0) {
        require(d->q && d->out, "paged attention: null q or out");
        require(multiple(d->q, 2) && multiple(d->out, 2) && multiple(d->lse, 4) && multiple(d->lengths, 4),
                "paged attention: q, out, lse or lengths not aligned to its elements");
        require(d->lengths || d->max_length == 0, "paged attention: null lengths");
    }
    mm::paged::Attention p{};
    p.q = d->q;
    p.q_row = d->q_row_stride;
    p.q_head = d->q_head_stride;
    p.B = d->rows;
    p.H = d->heads;
    p.pool = view(&c->pool);
    p.table = table_of(c);
    p.lengths = d->lengths;
    p.max_length = d->max_length;
    p.window = d->window;
    p.sinks = d->window > 0 ? d->sinks : 0;
    p.kv = c->pool.kv;
    p.rd = c->pool.rope_dim;
    p.scale = d->scale;
    p.out = d->out;
    p.lse = d->lse;
    return p;
}

template <typename T, bool Q8> void launch_any_width(const mm::paged::Attention& p, cudaStream_t s) {
    using namespace mm::paged;
    const int smem = kAnyWarps * (2 * p.kv + p.rd) * 4;  // at most 36 KB
    launch(s, any_width_kernel<T, Q8>, dim3(blocks(static_cast<long long>(p.B) * p.H, kAnyWarps)), dim3(32 * kAnyWarps), smem, p);
}

// ------------------------------------------------------------------ tensor-core form of attention
// The models' two widths, pages of whole boxes of 16 positions, and what tensor maps and the kernel's 8-byte
// loads of q take.
bool mma_form(const mm::paged::Attention& p, const mm_latent_cache& c) {
    if (!((p.kv == 128 && p.rd == 16) || (p.kv == 512 && p.rd == 32)) || c.positions % 16 || c.rows == 0 || p.max_length == 0) return false;
    if (!multiple(p.q, 8) || p.q_row % 4 || p.q_head % 4 || !multiple(p.out, 8)) return false;
    constexpr int64_t kMost = 1LL << 39;  // strides of up to 40 bits in bytes
    auto strides = [&](const void* base, int64_t page, int64_t position, int size) {
        return multiple(base, 16) && position > 0 && position < kMost && position * size % 16 == 0 &&
               (c.rows == 1 || (page > 0 && page < kMost && page * size % 16 == 0));
    };
    if (c.kind != MM_E4M3) return strides(c.latent, c.row_stride, c.pos_stride, 2);
    return strides(c.latent, c.row_stride, c.pos_stride, 1) && strides(c.rope, c.rope_row_stride, c.rope_pos_stride, 2) &&
           strides(c.scale, c.scale_row_stride, 4, 4);
}

// Boxes of `width` columns x `box` positions of a page of one of the pool's arrays (its scales: of `box`
// positions). False where the encoder does not take the strides.
bool pool_map(CUtensorMap* map, CUtensorMapDataType type, int size, const mm_latent_cache& c, const void* base, int columns,
              int64_t page_stride, int64_t position_stride, int width, int box, CUtensorMapSwizzle swizzle) {
    if (c.rows == 1) page_stride = std::max<int64_t>(page_stride, 16 * position_stride);  // any: there is one
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(columns), static_cast<cuuint64_t>(c.positions), static_cast<cuuint64_t>(c.rows)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(position_stride) * size, static_cast<cuuint64_t>(page_stride) * size};
    const cuuint32_t boxes[3] = {static_cast<cuuint32_t>(width), static_cast<cuuint32_t>(box), 1}, steps[3] = {1, 1, 1};
    return tensor_map_encoder()(map, type, 3, const_cast<void*>(base), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool scale_map(CUtensorMap* map, const mm_latent_cache& c, int box) {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(c.positions), static_cast<cuuint64_t>(c.rows)};
    const cuuint64_t stride = static_cast<cuuint64_t>(c.rows == 1 ? std::max<int64_t>(c.scale_row_stride, 16) & ~3LL : c.scale_row_stride) * 4;
    const cuuint32_t boxes[2] = {static_cast<cuuint32_t>(box), 1}, steps[2] = {1, 1};
    return tensor_map_encoder()(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, c.scale, dims, &stride, boxes, steps,
                                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
struct PoolMaps {
    CUtensorMap latent{}, rope{}, scale{};
};
bool pool_maps(PoolMaps& m, const mm_latent_cache& c, int box) {
    const CUtensorMapSwizzle by_rope = c.rope_dim == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
    const CUtensorMapDataType half = (c.kind == MM_E4M3 ? c.rope_kind : c.kind) == MM_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                                          : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    if (c.kind == MM_E4M3)
        return pool_map(&m.latent, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, c, c.latent, c.kv, c.row_stride, c.pos_stride, 128, box,
                        CU_TENSOR_MAP_SWIZZLE_128B) &&
               pool_map(&m.rope, half, 2, c, c.rope, c.rope_dim, c.rope_row_stride, c.rope_pos_stride, c.rope_dim, box, by_rope) &&
               scale_map(&m.scale, c, box);
    return pool_map(&m.latent, half, 2, c, c.latent, c.kv + c.rope_dim, c.row_stride, c.pos_stride, 64, box, CU_TENSOR_MAP_SWIZZLE_128B) &&
           pool_map(&m.rope, half, 2, c, c.latent, c.kv + c.rope_dim, c.row_stride, c.pos_stride, c.rope_dim, box, by_rope);
}

struct MmaPlan {
    int blocks = 0, grid = 0, entries = 0;
    bool shares = false;
    int64_t units = 0;
    int64_t bytes(int kv) const { return shares ? int64_t(2) * grid * 16 * (kv * 4 + 8) + int64_t(entries) * 16 : 0; }
};
MmaPlan mma_plan(const mm::paged::Attention& p) {
    using namespace mm::paged;
    MmaPlan r;
    r.blocks = (p.H + 15) / 16;
    r.units = static_cast<int64_t>(p.B) * r.blocks;
    const int64_t all = (static_cast<int64_t>(p.max_length) + kTile - 1) / kTile;
    const int64_t tiles = p.window > 0 ? std::min(all, (static_cast<int64_t>(p.window) + p.sinks) / kTile + 3) : all;
    const int64_t ctas = 2 * sm_count(), least = min_share(p.kv);
    // rows of few tiles are not worth cutting (and weights are 32-bit)
    r.shares = tiles > least && r.units * (tiles + row_cost(p.kv)) < INT32_MAX / 2;
    r.grid = static_cast<int>(std::min(ctas, r.shares ? (r.units * (tiles + row_cost(p.kv)) + least - 1) / least : r.units));
    r.entries = static_cast<int>(std::min<int64_t>(r.units, r.grid));
    return r;
}

template <int KV, int R, typename T, bool Q8, bool HALF = false>
void run_mma(const mm::paged::Attention& p, const MmaPlan& r, const PoolMaps& maps, void* workspace, int give_up, cudaStream_t s) {
    using namespace mm::paged;
    using C = MmaCfg<KV, R, Q8>;
    if (KV == 128 && !HALF && p.H <= 8) return run_mma<KV, R, T, Q8, KV == 128>(p, r, maps, workspace, give_up, s);
    MmaArgs a{};
    a.p = p;
    a.box = p.pool.positions % 32 == 0 ? 32 : 16;
    a.blocks = r.blocks;
    a.shares = r.shares;
    a.by_unit = r.units <= r.grid;
    a.give_up = give_up;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + int64_t(2) * r.grid * 16 * KV);
    a.cut = reinterpret_cast<int4*>(a.part_ml + int64_t(2) * r.grid * 16);
    set_dynamic_smem<paged_mma_kernel<KV, R, T, Q8, HALF>>(C::kSmem);
    launch(s, paged_mma_kernel<KV, R, T, Q8, HALF>, dim3(r.grid), dim3(kMmaThreads), C::kSmem, a, maps.latent, maps.rope, maps.scale);
    if (r.shares) {
        // the fewer units, the more parts each has and the more warps join one (a block for 128 columns of a head where
        // the parts are many): 512 wide with 4, 2 or 1 times 128 columns a warp, us of the whole call, 250 rows of up to
        // 3,000 positions 67.3 / 68.2 / 70.0, 96 of 8,192 80.4 / 79.1 / 79.7, 48 of 8,000 56.6 / 56.6 / 53.4
        constexpr int kMost = KV / 128;
        auto join = [&](auto ng) {
            constexpr int NG = decltype(ng)::value;
            const int y = std::max(2 * kMost / NG, std::min(2 * sm_count() / r.entries, 16 * kMost));
            launch(s, paged_join_kernel<KV, NG, T>, dim3(r.entries, y), dim3(256), 0, a);
        };
        if (r.entries > sm_count()) join(std::integral_constant<int, kMost>{});
        else if (r.entries > sm_count() * 2 / 5) join(std::integral_constant<int, kMost == 4 ? 2 : 1>{});
        else join(std::integral_constant<int, 1>{});
    }
}

// give_up: MmaArgs::give_up.
void attend(const mm_paged_attention_desc* desc, const mm_paged_cache* cache, void* workspace, size_t workspace_bytes, int give_up,
            cudaStream_t s) {
    const mm::paged::Attention p = problem(desc, cache);
    if (p.B == 0) return;
    const bool q8 = cache->pool.kind == MM_E4M3;
    PoolMaps maps;
    const bool mma = mma_form(p, cache->pool);
    const MmaPlan r = mma ? mma_plan(p) : MmaPlan{};
    const int64_t need = r.bytes(p.kv);  // also of a pool whose strides the encoder turns out not to take
    require(need == 0 || (workspace && multiple(workspace, 16) && workspace_bytes >= static_cast<size_t>(need)),
            "paged attention: workspace too small or not 16-byte aligned");
    if (mma && pool_maps(maps, cache->pool, cache->pool.positions % 32 == 0 ? 32 : 16)) {
        with_half(desc->dtype, [&](auto half) {
            using T = typename decltype(half)::type;
            if (p.kv == 128) q8 ? run_mma<128, 16, T, true>(p, r, maps, workspace, give_up, s) : run_mma<128, 16, T, false>(p, r, maps, workspace, give_up, s);
            else q8 ? run_mma<512, 32, T, true>(p, r, maps, workspace, give_up, s) : run_mma<512, 32, T, false>(p, r, maps, workspace, give_up, s);
        });
        return;
    }
    if (give_up >= 0) refuse(MM_UNSUPPORTED, "paged attention: this form waits for nothing");
    with_half(desc->dtype, [&](auto half) {
        using T = typename decltype(half)::type;
        if (q8) launch_any_width<T, true>(p, s);
        else launch_any_width<T, false>(p, s);
    });
}

void check_select(int batch, int beams, int vocab, int count) {
    require(batch >= 0 && beams >= 1 && vocab >= 1 && count >= 1, "beam selection: invalid sizes");
    if (beams > mm::beam::kMaxBeams || count > mm::beam::kMaxBeams) refuse(MM_UNSUPPORTED, "beam selection: more than 32 beams");
    if (vocab > mm::beam::kMaxVocab) refuse(MM_UNSUPPORTED, "beam selection: vocabulary over 1,048,576");
}

// How a selection is launched: parts of a beam's tokens, a block each, as many as fill the multiprocessors with 32
// warps, of 4,096 tokens or more. Blocks have eight warps, where there are many beams fewer, whose lists have to be joined:
// us with 8 / 4 / 2, 400 beams of 50,000 26.8 / 26.7 / 35.5, 512 of 32,768 24.0 / 22.2 / 26.7, 1,800 of 20,000 (fp16) 42.7 /
// 32.8 / 32.7, 1,000 of 4,000 19.2 / 16.3 / 13.9.
// In clusters where a batch entry's blocks can be one, none has more than 32,768 tokens then and there are few: us in
// clusters / with a second kernel, 1 x 4 beams of 16,384 8.8 / 13.0, 4 x 16 of 32,768 13.8 / 16.6, 16 x 8 (256 blocks)
// 15.7 / 15.8, 64 x 8 (512) 22.0 / 22.2.
struct SelectPlan {
    int parts, warps;
    bool cluster;
    int64_t bytes;
};
SelectPlan select_plan(int batch, int beams, int vocab) {
    const int64_t rows = std::max<int64_t>(1, static_cast<int64_t>(batch) * beams), most = std::min((vocab + 4095) / 4096, mm::beam::kMaxParts);
    SelectPlan r{static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most, 4 * sm_count() / rows))), 8, false, 0};
    const int fits = mm::beam::kMaxCluster / beams;
    const int parts = std::min(fits, r.parts);
    if (parts > 0 && (vocab + parts - 1) / parts <= 32768 && rows * parts <= sm_count() / 2) {
        r.parts = parts;
        r.cluster = true;
    } else {
        if (rows >= 3 * sm_count()) r.warps = vocab <= 8192 ? 2 : 4;
        r.bytes = static_cast<int64_t>(batch) * beams * r.parts * (32 * sizeof(mm::beam::Pair) + sizeof(float2));
    }
    return r;
}

template <typename T, bool SHIFTED> void launch_select(const mm::beam::Select& a, const SelectPlan& r, cudaStream_t s) {
    using namespace mm::beam;
    const unsigned grid = blocks(static_cast<long long>(a.batch) * a.beams * r.parts, 1);
    if (!r.cluster) {
        auto parts = [&](auto n) {
            constexpr int W = decltype(n)::value;
            set_dynamic_smem<select_parts_kernel<T, W, false, SHIFTED>>(ring_bytes(W));
            launch(s, select_parts_kernel<T, W, false, SHIFTED>, dim3(grid), dim3(32 * W), ring_bytes(W), a);
        };
        if (r.warps == 8) parts(std::integral_constant<int, 8>{});
        else if (r.warps == 4) parts(std::integral_constant<int, 4>{});
        else parts(std::integral_constant<int, 2>{});
        launch(s, select_join_kernel, dim3(a.batch), dim3(32 * a.beams), 512 * a.beams, a);
        return;
    }
    constexpr int kWarps = 8, kRing = ring_bytes(kWarps);
    static_assert(512 * kWarps <= kRing, "the join's scratch");
    constexpr auto kernel = select_parts_kernel<T, kWarps, true, SHIFTED>;
    set_dynamic_smem<kernel>(kRing);
    check(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "cluster size");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(32 * kWarps);
    cfg.dynamicSmemBytes = kRing;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = static_cast<unsigned>(a.beams * r.parts);
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    check(cudaLaunchKernelEx(&cfg, kernel, a), "kernel launch");
}

}  // namespace

extern "C" {

int mm_paged_status(void* stream) {
    return guarded([&] {
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        int bits = 0;
        const int none = 0;
        check(cudaMemcpyFromSymbolAsync(&bits, mm::paged::paged_status, sizeof bits, 0, cudaMemcpyDeviceToHost, s), "status");
        check(cudaStreamSynchronize(s), "status");
        if (!bits) return;
        check(cudaMemcpyToSymbolAsync(mm::paged::paged_status, &none, sizeof none, 0, cudaMemcpyHostToDevice, s), "status");
        check(cudaStreamSynchronize(s), "status");
        refuse(MM_GPU_ERROR, "paged attention: a kernel gave up on a wait; its results are NaN");
    });
}

int mm_paged_append(const mm_paged_cache* cache, const void* values, int64_t values_stride, int dtype, const int32_t* rows,
                    const int32_t* positions, int64_t n, double theta, const float* norm, float eps, void* stream) {
    return guarded([&] {
        check_paged(cache);
        require(n >= 0 && (rows || n <= INT32_MAX), "paged append: invalid count");
        require(cache->pool.rope_dim % 2 == 0, "paged append: rope_dim must be even");
        require(theta > 0 && std::isfinite(theta) && (!norm || eps >= 0), "paged append: theta must be positive and eps not negative");
        if (n == 0 || cache->pool.rows == 0 || cache->table_rows == 0 || cache->table_columns == 0) return;
        require(values && positions, "paged append: null input");
        require(multiple(positions, 4) && multiple(rows, 4) && multiple(norm, 4), "paged append: input not aligned to its elements");
        mm::paged::Rotation rot;
        for (int j = 0; j < cache->pool.rope_dim / 2; ++j)
            rot.f[j] = std::pow(theta, -2.0 * j / cache->pool.rope_dim) / 6.283185307179586476925;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const bool q8 = cache->pool.kind == MM_E4M3;
        with_type(dtype, [&](auto in) {
            with_half(q8 ? cache->pool.rope_kind : cache->pool.kind, [&](auto half) {
                using T = typename decltype(in)::type;
                using T16 = typename decltype(half)::type;
                require(multiple(values, sizeof(T)), "paged append: input not aligned to its elements");
                if (append_vector_form<T>(cache->pool, values, values_stride, norm)) {
                    auto run = [&](auto kv, auto rd, auto codes) {
                        constexpr int kKv = decltype(kv)::value, kRd = decltype(rd)::value;
                        constexpr bool kQ8 = decltype(codes)::value;
                        const unsigned ctas = std::min(blocks(n, 8 * (512 / kKv)),
                                                       static_cast<unsigned>(sm_count() * mm::paged::AppendRing<T, kQ8>::kCtas));
                        // (8-bit codes with and without a norm in one instance: 43.7 us instead of 41 for 131,072 fp16 tokens;
                        // 16-bit values in two instances 52.6 instead of 51.5)
                        launch(s, kQ8 && !norm ? mm::paged::append_vec_kernel<T, T16, kKv, kRd, kQ8, !kQ8>
                                               : mm::paged::append_vec_kernel<T, T16, kKv, kRd, kQ8, true>,
                               dim3(ctas), dim3(256), 0, out_view(&cache->pool), table_of(cache), static_cast<const T*>(values),
                               static_cast<long long>(values_stride), rows, positions, static_cast<long long>(n), norm, eps, rot);
                    };
                    using Narrow = std::integral_constant<int, 128>;
                    using Wide = std::integral_constant<int, 512>;
                    using R16 = std::integral_constant<int, 16>;
                    using R32 = std::integral_constant<int, 32>;
                    if (cache->pool.kv == 128) q8 ? run(Narrow{}, R16{}, std::true_type{}) : run(Narrow{}, R16{}, std::false_type{});
                    else q8 ? run(Wide{}, R32{}, std::true_type{}) : run(Wide{}, R32{}, std::false_type{});
                    return;
                }
                launch(s, q8 ? mm::paged::append_kernel<T, T16, true> : mm::paged::append_kernel<T, T16, false>, dim3(blocks(n, 8)),
                       dim3(256), 0, out_view(&cache->pool), table_of(cache), static_cast<const T*>(values),
                       static_cast<long long>(values_stride), rows, positions, static_cast<long long>(n), cache->pool.kv,
                       cache->pool.rope_dim, norm, eps, rot);
            });
        });
    });
}

int64_t mm_paged_attention_workspace(const mm_paged_attention_desc* desc, const mm_paged_cache* cache) {
    int64_t bytes = 0;
    const int rc = guarded([&] {
        const mm::paged::Attention p = problem(desc, cache);
        if (p.B > 0 && mma_form(p, cache->pool)) bytes = mma_plan(p).bytes(p.kv);
    });
    return rc ? -static_cast<int64_t>(rc) : bytes;
}

int mm_paged_attention(const mm_paged_attention_desc* desc, const mm_paged_cache* cache, void* workspace, size_t workspace_bytes,
                       void* stream) {
    return guarded([&] { attend(desc, cache, workspace, workspace_bytes, -1, static_cast<cudaStream_t>(stream)); });
}

int mm_paged_selftest_wait_timeout(const mm_paged_attention_desc* desc, const mm_paged_cache* cache, void* workspace,
                                   size_t workspace_bytes, int steps, void* stream) {
    return guarded([&] {
        require(steps >= 0 && steps <= 1 << 24, "paged attention: invalid number of steps");
        attend(desc, cache, workspace, workspace_bytes, steps, static_cast<cudaStream_t>(stream));
    });
}

int64_t mm_beam_select_workspace(int batch, int beams, int vocab, int count) {
    int64_t bytes = 0;
    const int rc = guarded([&] {
        check_select(batch, beams, vocab, count);
        if (batch > 0) bytes = select_plan(batch, beams, vocab).bytes;
    });
    return rc ? -static_cast<int64_t>(rc) : bytes;
}

int mm_beam_select(const void* logits, int64_t batch_stride, int64_t beam_stride, int dtype, const float* scores,
                   const uint8_t* finished, int eos, int batch, int beams, int vocab, int count, float* out_scores,
                   int32_t* out_parents, int32_t* out_tokens, void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_select(batch, beams, vocab, count);
        require(!finished || (eos >= 0 && eos < vocab), "beam selection: eos must be in the vocabulary");
        if (batch == 0) return;
        require(logits && scores && out_scores && out_parents && out_tokens, "beam selection: null argument");
        require(multiple(scores, 4) && multiple(out_scores, 4) && multiple(out_parents, 4) && multiple(out_tokens, 4),
                "beam selection: argument not aligned to its elements");
        with_type(dtype, [&](auto t) {
            require(multiple(logits, sizeof(typename decltype(t)::type)), "beam selection: logits not aligned to their elements");
        });
        const SelectPlan r = select_plan(batch, beams, vocab);
        require(r.bytes == 0 || (workspace && multiple(workspace, 16) && workspace_bytes >= static_cast<size_t>(r.bytes)),
                "beam selection: workspace too small or not 16-byte aligned");
        mm::beam::Pair* best = static_cast<mm::beam::Pair*>(workspace);
        const mm::beam::Select a{logits, batch_stride, beam_stride, scores, finished, eos, batch, beams, vocab, count, r.parts,
                                 out_scores, out_parents, out_tokens, best,
                                 reinterpret_cast<float2*>(best + static_cast<int64_t>(batch) * beams * r.parts * 32)};
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        with_type(dtype, [&](auto t) {
            using T = typename decltype(t)::type;
            const int64_t e = 16 / sizeof(T);  // whether every row begins at a multiple of 16 bytes
            if (multiple(logits, 16) && batch_stride % e == 0 && beam_stride % e == 0) launch_select<T, false>(a, r, s);
            else launch_select<T, true>(a, r, s);
        });
    });
}

int mm_beam_reorder(const mm_paged_cache* cache, int layers, const int64_t layer_strides[3], const int32_t* spare,
                    const int32_t* lengths, const int32_t* parents, int32_t* out_table, int32_t* out_spare,
                    int32_t* out_lengths, void* stream) {
    return guarded([&] {
        check_paged(cache);
        require(layers >= 0 && layer_strides, "beam reorder: invalid layers");
        const mm_latent_cache& c = cache->pool;
        const int rows = cache->table_rows;
        if (rows == 0) return;
        require(cache->table_columns >= 1, "beam reorder: a table of no pages");
        require(spare && lengths && parents && out_table && out_spare && out_lengths, "beam reorder: null argument");
        for (const int32_t* x : {spare, lengths, parents, const_cast<const int32_t*>(out_table), const_cast<const int32_t*>(out_spare),
                                 const_cast<const int32_t*>(out_lengths)})
            require(multiple(x, 4), "beam reorder: argument not aligned to its elements");
        const bool q8 = c.kind == MM_E4M3;
        mm::paged::Reorder a{table_of(cache), spare, lengths, parents, out_table, out_spare, out_lengths, c.positions,
                             c.rows, layers, {}};
        auto plane = [](void* data, int64_t layer, int64_t page, int64_t position, int n, int size) {
            mm::paged::Plane r{static_cast<uint8_t*>(data), static_cast<long long>(layer * size),
                               static_cast<long long>(page * size), static_cast<long long>(position * size), n * size, 1};
            // positions in line are copied as one row, whose end need not be a whole access of 16 bytes
            for (int v : {4, 16})
                if (multiple(data, v) && r.layer % v == 0 && r.page % v == 0 && r.position % v == 0 && r.bytes % v == 0) r.vec = v;
            return r;
        };
        if (q8) {
            a.plane[0] = plane(c.latent, layer_strides[0], c.row_stride, c.pos_stride, c.kv, 1);
            if (c.rope_dim > 0) a.plane[1] = plane(c.rope, layer_strides[1], c.rope_row_stride, c.rope_pos_stride, c.rope_dim, 2);
            a.plane[2] = plane(c.scale, layer_strides[2], c.scale_row_stride, 1, 1, 4);
        } else {
            a.plane[0] = plane(c.latent, layer_strides[0], c.row_stride, c.pos_stride, c.kv + c.rope_dim, 2);
        }
        launch(static_cast<cudaStream_t>(stream), mm::paged::reorder_kernel,
               dim3(static_cast<unsigned>(rows), static_cast<unsigned>(std::min(std::max(layers, 1), 64))), dim3(256), 0, a);
    });
}

}  // extern "C"
