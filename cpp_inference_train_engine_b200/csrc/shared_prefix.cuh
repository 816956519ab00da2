// Absorbed latent attention of a batch whose rows share stored prefixes: a query attends over
// its group's prefix and its row's own suffix (mm_shared_prefix_attention).
#pragma once
#include "latent_cache.cuh"

namespace mm {
namespace spa {

using lat::CacheView;

// What every kernel of the call needs. A query row is (row b, token t, head h), numbered
// (b * T + t) * H + h.
struct Problem {
    const void* q;
    long long q_row, q_tok, q_head;  // strides in elements
    int B, T, H;
    CacheView prefix, suffix;
    const int* group_start;
    const int* prefix_len;
    const int* suffix_len;
    int G, max_group, max_prefix, max_suffix;
    int kv, rd;
    float scale;
    void* out;
    float* lse;
};

// The group of row b, or -1: the last g with group_start[g] <= b, when b is also below its end
// and among its first max_group rows.
__device__ __forceinline__ int group_of(const Problem& p, int b) {
    int lo = 0, hi = p.G;  // group_start is non-decreasing
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (p.group_start[mid] <= b) lo = mid + 1;
        else hi = mid;
    }
    const int g = lo - 1;
    if (g < 0 || b >= p.group_start[g + 1] || b - p.group_start[g] >= p.max_group) return -1;
    return g;
}
__device__ __forceinline__ int prefix_length(const Problem& p, int g) {
    return g < 0 ? 0 : min(max(p.prefix_len[g], 0), p.max_prefix);
}
__device__ __forceinline__ int suffix_length(const Problem& p, int b) {
    return p.max_suffix > 0 ? min(max(p.suffix_len[b], 0), p.max_suffix) : 0;
}

// ------------------------------------------------------------------ any width
// One warp per query row, keys in tiles of 32: lane j scores key j of the tile (its own cache
// row), the tile's softmax is one warp reduction with the running maximum and sum, then every
// lane adds p_j * value for its columns. The query (fp32, pre-scaled) and the output row live
// in shared memory, so any kv and rope width works. Used for the widths that have no
// tensor-core form; bound by its scalar loads and the row by row walk (8 rows of 8 heads over a prompt
// of 128, 128 + 16 wide: 57 us where the tensor-core form takes 12).
constexpr int kAnyWarps = 4;
template <typename T, bool Q8P, bool Q8S>
__global__ void __launch_bounds__(32 * kAnyWarps) any_width_kernel(const Problem p) {
    MM_PDL_ENTRY();
    extern __shared__ float any_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long r = static_cast<long long>(blockIdx.x) * kAnyWarps + warp;
    if (r >= static_cast<long long>(p.B) * p.T * p.H) return;
    const int W = p.kv + p.rd;
    float* q = any_smem + warp * (W + p.kv);
    float* acc = q + W;
    const int h = static_cast<int>(r % p.H);
    const long long bt = r / p.H;
    const int t = static_cast<int>(bt % p.T), b = static_cast<int>(bt / p.T);
    const T* qp = static_cast<const T*>(p.q) + b * p.q_row + t * p.q_tok + h * p.q_head;
    for (int c = lane; c < W; c += 32) q[c] = lat::to_f32(qp[c]) * p.scale;
    for (int c = lane; c < p.kv; c += 32) acc[c] = 0.f;
    __syncwarp();
    float m = -INFINITY, l = 0.f;
    auto segment = [&](const CacheView& c, int row, int n, auto q8) {
        constexpr bool Q8 = decltype(q8)::value;
        const uint8_t* base = c.latent + row * c.row_stride * (Q8 ? 1 : 2);
        const T* rbase = Q8 ? reinterpret_cast<const T*>(c.rope) + row * c.rope_row_stride : nullptr;
        for (int j0 = 0; j0 < n; j0 += 32) {
            const int j = j0 + lane;
            float s = -INFINITY, ks = 1.f;
            if (j < n) {
                float a = 0.f;
                if (Q8) {
                    const uint8_t* k = base + j * c.pos_stride;
                    for (int i = 0; i < p.kv; ++i) a = fmaf(q[i], lat::e4m3_to_f32(k[i]), a);
                    ks = c.scale[row * c.scale_row_stride + j];
                    a *= ks;
                    const T* kr = rbase + j * c.rope_pos_stride;
                    for (int i = 0; i < p.rd; ++i) a = fmaf(q[p.kv + i], lat::to_f32(kr[i]), a);
                } else {
                    const T* k = reinterpret_cast<const T*>(base) + j * c.pos_stride;
                    for (int i = 0; i < W; ++i) a = fmaf(q[i], lat::to_f32(k[i]), a);
                }
                s = a;
            }
            const float mn = fmaxf(m, warp_max(s));
            const float at = mn == -INFINITY ? 0.f : mn;
            const float corr = expf(m - at);
            const float e = j < n ? expf(s - at) : 0.f;
            l = l * corr + warp_sum(e);
            m = mn;
            const float w = e * ks;
            const int cnt = min(32, n - j0);
            for (int c0 = lane; c0 < p.kv; c0 += 32) acc[c0] *= corr;
            for (int i = 0; i < cnt; ++i) {
                const float wi = __shfl_sync(0xffffffffu, w, i);
                if (Q8) {
                    const uint8_t* k = base + (j0 + i) * c.pos_stride;
                    for (int c0 = lane; c0 < p.kv; c0 += 32) acc[c0] = fmaf(wi, lat::e4m3_to_f32(k[c0]), acc[c0]);
                } else {
                    const T* k = reinterpret_cast<const T*>(base) + (j0 + i) * c.pos_stride;
                    for (int c0 = lane; c0 < p.kv; c0 += 32) acc[c0] = fmaf(wi, lat::to_f32(k[c0]), acc[c0]);
                }
            }
        }
    };
    const int g = p.G > 0 ? group_of(p, b) : -1;
    segment(p.prefix, g < 0 ? 0 : g, prefix_length(p, g), std::integral_constant<bool, Q8P>());
    segment(p.suffix, b, suffix_length(p, b) - (p.T - 1 - t), std::integral_constant<bool, Q8S>());
    const float inv = l > 0.f ? 1.f / l : 0.f;
    T* o = static_cast<T*>(p.out) + r * p.kv;
    for (int c = lane; c < p.kv; c += 32) o[c] = lat::from_f32<T>(l == 0.f ? 0.f : acc[c] * inv);
    if (p.lse && lane == 0) p.lse[r] = l == 0.f ? -INFINITY : m + logf(l);
}

}  // namespace spa
}  // namespace mm
