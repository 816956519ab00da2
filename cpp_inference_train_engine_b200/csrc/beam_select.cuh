// Beam search's selection over beams and vocabulary (mm_beam_select).
//
// One pass over the logits: a warp takes a part of a beam's tokens and keeps their maximum, the sum of
// exponentials below it, and the best `count` of them (rank r in lane r); a second kernel joins the parts of a
// beam and then the beams. A token enters the list by a vote against its last entry, which after the first few
// hundred tokens almost never happens, so the pass is bound by its loads.
#pragma once
#include "latent_cache.cuh"

namespace mm {
namespace beam {

constexpr int kMaxBeams = 32;
constexpr int kMaxVocab = 1 << 20;  // flat candidates k * vocab + v stay below 2^25
constexpr int kMaxParts = 64;       // of a beam's tokens

struct Select {
    const void* logits;
    long long batch_stride, beam_stride;
    const float* scores;
    const uint8_t* finished;
    int eos, batch, beams, vocab, count, parts;
    float* out_scores;
    int* out_parents;
    int* out_tokens;
    // a part's best values and tokens, maximum and sum: [batch * beams * parts][count], [batch * beams * parts]
    float* best;
    int* token;
    float2* sum;
};

// The best `count` candidates so far, rank r in lane r; lanes behind the last hold (-infinity, kNobody).
constexpr int kNobody = 0x7fffffff;
template <typename V> struct Best {
    V value;
    int at;
    V last;     // of rank count - 1
    int last_at;
    __device__ __forceinline__ Best() : value(-INFINITY), at(kNobody), last(-INFINITY), last_at(kNobody) {}
    __device__ __forceinline__ bool enters(V v, int i) const { return (v > last || (v == last && i < last_at)) && v > -INFINITY; }
    // Offers every lane's candidate.
    __device__ __forceinline__ void offer(V v, int i, int count) {
        const int lane = threadIdx.x & 31;
        unsigned todo = __ballot_sync(0xffffffffu, enters(v, i));
        while (todo) {
            const int from = __ffs(todo) - 1;
            const V cv = __shfl_sync(0xffffffffu, v, from);
            const int ci = __shfl_sync(0xffffffffu, i, from);
            const int rank = __popc(__ballot_sync(0xffffffffu, value > cv || (value == cv && at < ci)));
            const V uv = __shfl_up_sync(0xffffffffu, value, 1);
            const int ui = __shfl_up_sync(0xffffffffu, at, 1);
            if (lane >= rank) {
                value = lane == rank ? cv : uv;
                at = lane == rank ? ci : ui;
            }
            if (lane >= count) {
                value = -INFINITY;
                at = kNobody;
            }
            last = __shfl_sync(0xffffffffu, value, count - 1);
            last_at = __shfl_sync(0xffffffffu, at, count - 1);
            todo &= todo - 1;
            todo &= __ballot_sync(0xffffffffu, enters(v, i));
        }
    }
};

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < INFINITY; }

// Warp: part `part` of beam row `row`. E values of 16 bytes a load; a row's first and last tokens that are
// not in a whole aligned load are taken one a lane.
template <typename T>
__global__ void __launch_bounds__(128) select_parts_kernel(const Select a) {
    MM_PDL_ENTRY();
    constexpr int E = 16 / sizeof(T), U = 4;  // values per load, loads per step
    const int lane = threadIdx.x & 31;
    const long long w = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    if (w >= static_cast<long long>(a.batch) * a.beams * a.parts) return;
    const int row = static_cast<int>(w / a.parts), part = static_cast<int>(w - static_cast<long long>(row) * a.parts);
    if (!finite(__ldg(a.scores + row)) || (a.finished && a.finished[row])) return;  // the join does not read it either
    const int b = row / a.beams;
    const T* x = static_cast<const T*>(a.logits) + b * a.batch_stride + (row - b * a.beams) * a.beam_stride;
    // whole loads begin at token `head`, which is where the address is a multiple of 16
    const int head = min(a.vocab, static_cast<int>((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T)));
    const int loads = (a.vocab - head) / E;
    const int per = (loads + a.parts - 1) / a.parts, l0 = min(part * per, loads), l1 = min(l0 + per, loads);
    Best<float> best;
    float m = -INFINITY, s = 0.f;
    auto add = [&](const float* v, int n, float top) {  // n values of this lane into its sum
        if (top > m) {
            s *= m == -INFINITY ? 0.f : fast_exp2((m - top) * 1.4426950408889634f);
            m = top;
        }
        const float ref = m == -INFINITY ? 0.f : m;
        for (int e = 0; e < n; ++e) s += fast_exp2((v[e] - ref) * 1.4426950408889634f);
    };
    for (int i0 = l0; i0 < l1; i0 += 32 * U) {
        uint4 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * 32 + lane;
            if (i < l1) raw[u] = __ldcs(reinterpret_cast<const uint4*>(x + head) + i);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * 32 + lane;
            if (i0 + u * 32 >= l1) break;
            float v[E];
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = i < l1 ? lat::to_f32(reinterpret_cast<const T*>(&raw[u])[e]) : -INFINITY;
            float top = v[0];
#pragma unroll
            for (int e = 1; e < E; ++e) top = fmaxf(top, v[e]);
            if (top > m) {
                s *= m == -INFINITY ? 0.f : fast_exp2((m - top) * 1.4426950408889634f);
                m = top;
            }
            const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int e = 0; e < E; ++e) s += fast_exp2((v[e] - ref) * 1.4426950408889634f);
            if (__any_sync(0xffffffffu, top >= best.last && top > -INFINITY)) {
#pragma unroll
                for (int e = 0; e < E; ++e) best.offer(v[e], head + i * E + e, a.count);
            }
        }
    }
    if (part == 0) {  // the ends, at most 2 (E - 1) <= 14 tokens
        const int tail = head + loads * E;
        const int t = lane < head ? lane : tail + lane - head;
        const float v = t < a.vocab ? lat::to_f32(x[t]) : -INFINITY;
        add(&v, 1, v);
        best.offer(v, t, a.count);
    }
    // the lanes' sums below one maximum (a NaN or +infinity anywhere makes the sum a NaN)
    const float top = warp_max(m);
    s *= m == -INFINITY ? 0.f : fast_exp2((m - top) * 1.4426950408889634f);
    s = warp_sum(m == -INFINITY && s == 0.f ? 0.f : s);
    if (lane < a.count) {
        a.best[w * a.count + lane] = best.value;
        a.token[w * a.count + lane] = best.at;
    }
    if (lane == 0) a.sum[w] = make_float2(top, s);
}

// Block per batch entry, a warp per beam: its log-sum-exp and its best tokens' scores; then the first warp
// takes the best of the beams' lists.
static __global__ void __launch_bounds__(1024) select_join_kernel(const Select a) {
    MM_PDL_ENTRY();
    __shared__ double score_s[kMaxBeams * kMaxBeams];
    __shared__ int at_s[kMaxBeams * kMaxBeams];
    const int b = blockIdx.x, k = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = b * a.beams + k;
    const float score = __ldg(a.scores + row);
    double cand = -INFINITY;
    int at = kNobody;
    if (finite(score)) {
        if (a.finished && a.finished[row]) {
            if (lane == 0) {
                cand = score;
                at = k * a.vocab + a.eos;
            }
        } else {
            const long long p0 = static_cast<long long>(row) * a.parts;
            float top = -INFINITY;
            for (int p = lane; p < a.parts; p += 32) top = fmaxf(top, a.sum[p0 + p].x);
            top = warp_max(top);
            double s = 0;
            for (int p = lane; p < a.parts; p += 32) {
                const float2 v = a.sum[p0 + p];
                s += v.x == -INFINITY ? static_cast<double>(v.y) : static_cast<double>(v.y) * exp(static_cast<double>(v.x) - top);
            }
            s = warp_sum(s);
            const double lse = top + log(s);
            Best<float> best;
            const int n = a.parts * a.count;
            for (int i = lane; i < (n + 31) / 32 * 32; i += 32) {
                const float v = i < n ? a.best[p0 * a.count + i] : -INFINITY;
                best.offer(v, i < n ? a.token[p0 * a.count + i] : kNobody, a.count);
            }
            // not a number where the log-sum-exp is not finite
            if (best.at != kNobody && fabs(lse) < INFINITY) {
                cand = score + (static_cast<double>(best.value) - lse);
                at = k * a.vocab + best.at;
            }
        }
    }
    if (!(static_cast<float>(cand) > -INFINITY)) {  // what fp32 cannot hold is no score
        cand = -INFINITY;
        at = kNobody;
    }
    if (lane < a.count) {
        score_s[k * a.count + lane] = cand;
        at_s[k * a.count + lane] = at;
    }
    __syncthreads();
    if (k) return;
    Best<double> best;
    const int n = a.beams * a.count;
    for (int i = lane; i < (n + 31) / 32 * 32; i += 32) best.offer(i < n ? score_s[i] : -INFINITY, i < n ? at_s[i] : kNobody, a.count);
    if (lane < a.count) {
        const bool none = best.at == kNobody;
        const long long o = static_cast<long long>(b) * a.count + lane;
        a.out_scores[o] = static_cast<float>(best.value);
        a.out_parents[o] = none ? min(lane, a.beams - 1) : best.at / a.vocab;
        a.out_tokens[o] = none ? -1 : best.at % a.vocab;
    }
}

}  // namespace beam
}  // namespace mm
