// Absorbed latent attention of one query token per row over a paged cache (mm_paged_attention).
#pragma once
#include "paged_cache.cuh"

namespace mm {
namespace paged {

__device__ int paged_status;  // DeviceError bits since they were last read (mm_paged_status)

struct Attention {
    const void* q;
    long long q_row, q_head;  // strides in elements
    int B, H;
    lat::CacheView pool;      // rows: pages, positions: entries of a page
    Table table;
    const int* lengths;
    int max_length, window, sinks;
    int kv, rd;
    float scale;
    void* out;
    float* lse;
};

__device__ __forceinline__ int length_of(const Attention& p, int b) { return min(max(__ldg(p.lengths + b), 0), p.max_length); }
// First position of the window.
__device__ __forceinline__ int window_start(const Attention& p, int len) { return p.window > 0 ? max(len - p.window, 0) : 0; }

// ------------------------------------------------------------------ any width
// One warp per (row, head), positions in tiles of 32: lane j scores position j of the tile, the tile's softmax
// is one warp reduction with the running maximum and sum, then every lane adds p_j * value for its
// columns. The query (fp32, scaled) and the output row live in shared memory. For the widths, page
// sizes and alignments that have no tensor-core form; bound by its scalar loads, a position's by one lane, and one
// warp's chain a row and head (120 + 16 wide, 8 heads: 4 rows of 197 positions 95 us where 128 + 16 take 7, 64 of 1,024 581).
constexpr int kAnyWarps = 4;
template <typename T, bool Q8>
__global__ void __launch_bounds__(32 * kAnyWarps) any_width_kernel(const Attention p) {
    MM_PDL_ENTRY();
    extern __shared__ float any_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long r = static_cast<long long>(blockIdx.x) * kAnyWarps + warp;
    if (r >= static_cast<long long>(p.B) * p.H) return;
    const int W = p.kv + p.rd;
    float* q = any_smem + warp * (W + p.kv);
    float* acc = q + W;
    const int b = static_cast<int>(r / p.H), h = static_cast<int>(r - static_cast<long long>(b) * p.H);
    const T* qp = static_cast<const T*>(p.q) + b * p.q_row + h * p.q_head;
    for (int c = lane; c < W; c += 32) q[c] = lat::to_f32(qp[c]) * p.scale;
    for (int c = lane; c < p.kv; c += 32) acc[c] = 0.f;
    __syncwarp();
    const int len = length_of(p, b), start = window_start(p, len);
    float m = -INFINITY, l = 0.f;
    const int sinks = min(p.sinks, start);  // positions [0, sinks) and [start, len) are seen
    for (long long i0 = 0; i0 < sinks + len - start; i0 += 32) {
        const long long i = i0 + lane, j = i < sinks ? i : start + i - sinks;
        int at = 0;
        const long long page = j < len ? page_of(p.table, p.pool.rows, p.pool.positions, b, static_cast<int>(j), at) : -1;
        float s = -INFINITY, ks = 1.f;
        const uint8_t* k = p.pool.latent + (page * p.pool.row_stride + at * p.pool.pos_stride) * (Q8 ? 1 : 2);
        if (page >= 0) {
            float a = 0.f;
            if (Q8) {
                for (int c = 0; c < p.kv; ++c) a = fmaf(q[c], lat::e4m3_to_f32(k[c]), a);
                ks = p.pool.scale[page * p.pool.scale_row_stride + at];
                a *= ks;
                const T* kr = reinterpret_cast<const T*>(p.pool.rope) + page * p.pool.rope_row_stride + at * p.pool.rope_pos_stride;
                for (int c = 0; c < p.rd; ++c) a = fmaf(q[p.kv + c], lat::to_f32(kr[c]), a);
            } else {
                for (int c = 0; c < W; ++c) a = fmaf(q[c], lat::to_f32(reinterpret_cast<const T*>(k)[c]), a);
            }
            s = a;
        }
        const float mn = fmaxf(m, warp_max(s));
        const float ref = mn == -INFINITY ? 0.f : mn;
        const float corr = expf(m - ref);
        const float e = page >= 0 ? expf(s - ref) : 0.f;
        l = l * corr + warp_sum(e);
        m = mn;
        const float w = e * ks;
        for (int c = lane; c < p.kv; c += 32) acc[c] *= corr;
        for (int t = 0; t < 32; ++t) {
            const float wt = __shfl_sync(0xffffffffu, w, t);
            const uint8_t* kt = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(k), t));
            if (!__shfl_sync(0xffffffffu, static_cast<int>(page >= 0), t)) continue;
            for (int c = lane; c < p.kv; c += 32)
                acc[c] = fmaf(wt, Q8 ? lat::e4m3_to_f32(kt[c]) : lat::to_f32(reinterpret_cast<const T*>(kt)[c]), acc[c]);
        }
    }
    const float inv = 1.f / l;
    T* o = static_cast<T*>(p.out) + r * p.kv;
    for (int c = lane; c < p.kv; c += 32) o[c] = lat::from_f32<T>(l == 0.f ? 0.f : acc[c] * inv);
    if (p.lse && lane == 0) p.lse[r] = l == 0.f ? -INFINITY : m + logf(l);
}

}  // namespace paged
}  // namespace mm
