// Beam search's selection over beams and vocabulary (mm_beam_select).
//
// One pass over the logits: a block takes a part of a beam's tokens, each of its warps a quarter, and keeps
// their maximum, the sum of exponentials below it and the best `count` of them (rank r in lane r); a second kernel
// joins the parts of a beam and then the beams. The pass itself keeps one maximum per lane and step: of the 32
// lanes' maxima over a stretch of steps the count-th largest bounds the list from below, so that only the few (lane,
// step) pairs that reach it are looked at again, from the cache.
#pragma once
#include "latent_cache.cuh"

namespace mm {
namespace beam {

constexpr int kMaxBeams = 32;
constexpr int kMaxVocab = 1 << 20;  // flat candidates k * vocab + v stay below 2^25
constexpr float kLowest = -3.402823466e38f;
constexpr int kMaxParts = 32;       // of a beam's tokens

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

// Candidates in order: by value, then by the lower index. Nobody: (-infinity, kNobody).
constexpr int kNobody = 0x7fffffff;
struct Pair {
    float value;
    int at;
};
__device__ __forceinline__ bool ahead(Pair a, Pair b) { return a.value > b.value || (a.value == b.value && a.at < b.at); }
__device__ __forceinline__ Pair from_lane(Pair p, int lane_xor) {
    return {__shfl_xor_sync(0xffffffffu, p.value, lane_xor), __shfl_xor_sync(0xffffffffu, p.at, lane_xor)};
}
// One step of a bitonic network over the lanes; `down`: the better of the two goes to the lower lane.
__device__ __forceinline__ void exchange(Pair& p, int o, bool down) {
    const Pair q = from_lane(p, o);
    const bool lower = (threadIdx.x & o) == 0;
    if (ahead(q, p) == (lower == down)) p = q;
}
// The best 32 candidates so far, rank r in lane r.
struct Best {
    Pair p{-INFINITY, kNobody};
    // Joins 32 more, one a lane, in any order.
    __device__ __forceinline__ void join(Pair q) {
#pragma unroll
        for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
            for (int o = size >> 1; o > 0; o >>= 1) exchange(q, o, (threadIdx.x & size) == 0 || size == 32);
        join_sorted(q);
    }
    // The same, from the best to the last.
    __device__ __forceinline__ void join_sorted(Pair q) {
        // the better of rank r and rank 31 - r are the best 32, rising and falling once
        q = from_lane(q, 31);
        if (ahead(q, p)) p = q;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) exchange(p, o, true);
    }
    __device__ __forceinline__ Pair rank(int r) const {
        return {__shfl_sync(0xffffffffu, p.value, r), __shfl_sync(0xffffffffu, p.at, r)};
    }
};

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < INFINITY; }

// Two fp32 values in one register pair: sums and products of both in one instruction.
struct Two {
    unsigned long long v;
    __device__ __forceinline__ Two(unsigned long long x) : v(x) {}
    __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
    __device__ __forceinline__ float lo() const { return __uint_as_float(static_cast<uint32_t>(v)); }
    __device__ __forceinline__ float hi() const { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
};
__device__ __forceinline__ Two operator+(Two a, Two b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Two operator*(Two a, Two b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a.v), "l"(b.v));
    return r;
}

// Block (part, beam row). E values of 16 bytes a load; a row's first and last tokens that are not in a whole
// aligned load are taken one a lane.
template <typename T>
__global__ void __launch_bounds__(128, 8) select_parts_kernel(const Select a) {
    MM_PDL_ENTRY();
    constexpr int E = 16 / sizeof(T), U = 4, kSteps = 8;  // values per load, loads per step, steps per stretch
    __shared__ Pair wait_s[4][64];
    __shared__ float2 sum_s[4];
    __shared__ uint8_t pairs_s[4][32 * kSteps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
    if (!finite(__ldg(a.scores + row)) || (a.finished && a.finished[row])) return;  // the join does not read it either
    const int b = row / a.beams;
    const T* x = static_cast<const T*>(a.logits) + b * a.batch_stride + (row - b * a.beams) * a.beam_stride;
    // whole loads begin at token `head`, which is where the address is a multiple of 16
    const int head = min(a.vocab, static_cast<int>((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T)));
    const int loads = (a.vocab - head) / E;
    const int per = (loads + 4 * a.parts - 1) / (4 * a.parts), l0 = min((part * 4 + warp) * per, loads), l1 = min(l0 + per, loads);
    // Candidates wait in shared memory until there are 32 (or no more): joining the list costs a sort. What is
    // behind the list's last entry does not wait.
    Pair* wait = wait_s[warp];
    int waiting = 0;
    Best best;
    Pair last{-INFINITY, kNobody};
    auto join = [&] {
        __syncwarp();
        best.join(lane < waiting ? wait[lane] : Pair{-INFINITY, kNobody});
        const Pair l = best.rank(a.count - 1);
        if (l.at != kNobody) last = l;  // (a list that is not full keeps its floor)
        const Pair rest = wait[32 + lane];
        __syncwarp();
        wait[lane] = rest;
        waiting = max(waiting - 32, 0);
    };
    auto offer = [&](float v, int i) {
        const bool in = v > -INFINITY && ahead({v, i}, last);
        const unsigned who = __ballot_sync(0xffffffffu, in);
        if (in) wait[waiting + __popc(who & ((1u << lane) - 1))] = {v, i};
        waiting += __popc(who);
        if (waiting >= 32) join();
    };
    constexpr float kLog2e = 1.4426950408889634f;
    float m = kLowest, s = 0.f;  // (a finite maximum of nothing: differences from it are no NaN)
    uint4 raw[U];  // a step ahead
    auto fetch = [&](int i0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * 32 + lane;
            if (i < l1) raw[u] = __ldg(reinterpret_cast<const uint4*>(x + head) + i);
        }
    };
    fetch(l0);
    for (int base = l0; base < l1; base += 32 * U * kSteps) {
        float tops[kSteps], most = -INFINITY;
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
            const int i0 = base + st * 32 * U;
            tops[st] = -INFINITY;
            if (i0 >= l1) continue;
            float v[U][E];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < E; ++e) v[u][e] = lat::to_f32(reinterpret_cast<const T*>(&raw[u])[e]);
            if (i0 + 32 * U > l1) {
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (i0 + u * 32 + lane >= l1) {
#pragma unroll
                        for (int e = 0; e < E; ++e) v[u][e] = -INFINITY;
                    }
            }
            fetch(i0 + 32 * U);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < E; ++e) tops[st] = fmaxf(tops[st], v[u][e]);
            const float mn = fmaxf(m, tops[st]);
            s *= fast_exp2((m - mn) * kLog2e);
            m = mn;
            const Two ref(-m, -m), by(kLog2e, kLog2e);
            Two sums[2] = {Two(0.f, 0.f), Two(0.f, 0.f)};
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    const Two z = (Two(v[u][e], v[u][e + 1]) + ref) * by;
                    sums[u & 1] = sums[u & 1] + Two(fast_exp2(z.lo()), fast_exp2(z.hi()));
                }
            sums[0] = sums[0] + sums[1];
            s += sums[0].lo() + sums[0].hi();
            most = fmaxf(most, tops[st]);
        }
        // `count` of the lanes' largest are `count` candidates: nothing below the least of them enters
        {
            Best all;
            all.join({most, lane});
            const float floor = all.rank(a.count - 1).value;
            if (floor > last.value) last = {floor, kNobody};
        }
        // the steps and lanes that reach it, in line; their values from the cache, kAtOnce pairs' at a time
        int pairs = 0;
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
            const bool in = tops[st] >= last.value && tops[st] > -INFINITY;
            const unsigned who = __ballot_sync(0xffffffffu, in);
            if (in) pairs_s[warp][pairs + __popc(who & ((1u << lane) - 1))] = static_cast<uint8_t>(st * 32 + lane);
            pairs += __popc(who);
        }
        __syncwarp();
        constexpr int kSide = 32 / (U * E), kAtOnce = 4 * kSide;  // pairs side by side in a warp: 2 for 16 values
        const int place = lane % (U * E);
        for (int j0 = 0; j0 < pairs; j0 += kAtOnce) {
            float v[4];
            int t[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int pair = j0 + j * kSide + lane / (U * E), code = pair < pairs ? pairs_s[warp][pair] : 0;
                const int i = base + (code >> 5) * 32 * U + place / E * 32 + (code & 31);
                t[j] = head + i * E + place % E;
                v[j] = pair < pairs && i < l1 ? lat::to_f32(x[t[j]]) : -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) offer(v[j], t[j]);
        }
        __syncwarp();
    }
    if (part == 0 && warp == 0) {  // the ends, at most 2 (E - 1) <= 14 tokens
        const int tail = head + loads * E;
        const int t = lane < head ? lane : tail + lane - head;
        const float v = t < a.vocab ? lat::to_f32(x[t]) : -INFINITY;
        const float mn = fmaxf(m, v);
        s = s * fast_exp2((m - mn) * kLog2e) + fast_exp2((v - mn) * kLog2e);
        m = mn;
        offer(v, t);
    }
    join();
    // the lanes' sums below one maximum (a NaN or +infinity anywhere makes the sum a NaN), then the warps'
    auto scaled = [&](float2 v, float top) { return v.y * fast_exp2((v.x - top) * kLog2e); };
    float top = warp_max(m);
    s = warp_sum(scaled({m, s}, top));
    if (lane == 0) sum_s[warp] = make_float2(top, s);
    wait[lane] = best.p;
    __syncthreads();
    if (warp) return;
    for (int w = 1; w < 4; ++w) best.join_sorted(wait_s[w][lane]);
    const long long o = static_cast<long long>(blockIdx.x) * a.count + lane;
    if (lane < a.count) {
        a.best[o] = best.p.value;
        a.token[o] = best.p.at;
    }
    if (lane == 0) {
        top = fmaxf(fmaxf(sum_s[0].x, sum_s[1].x), fmaxf(sum_s[2].x, sum_s[3].x));
        a.sum[blockIdx.x] = make_float2(top, (scaled(sum_s[0], top) + scaled(sum_s[1], top)) + (scaled(sum_s[2], top) + scaled(sum_s[3], top)));
    }
}

// Block per batch entry, a warp per beam: its log-sum-exp and the best of its parts' lists; then the rank of
// every beam's candidates among all of them, counted by a thread each.
static __global__ void __launch_bounds__(1024) select_join_kernel(const Select a) {
    MM_PDL_ENTRY();
    __shared__ double score_s[kMaxBeams * kMaxBeams];
    __shared__ int at_s[kMaxBeams * kMaxBeams];
    const int b = blockIdx.x, k = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = b * a.beams + k, n = a.parts * a.count;
    // everything asked for at once: what the parts of a finished or dead beam hold is not used
    const long long p0 = static_cast<long long>(row) * a.parts;
    auto entry = [&](int i) { return i < n ? Pair{__ldcg(a.best + p0 * a.count + i), __ldcg(a.token + p0 * a.count + i)} : Pair{-INFINITY, kNobody}; };
    Pair next = entry(lane);
    const float2 sum = lane < a.parts ? __ldcg(a.sum + p0 + lane) : make_float2(kLowest, 0.f);
    const float score = __ldg(a.scores + row);
    const bool ended = a.finished && __ldg(a.finished + row);
    double cand = -INFINITY;
    int at = kNobody;
    if (finite(score)) {
        if (ended) {
            if (lane == 0) {
                cand = score;
                at = k * a.vocab + a.eos;
            }
        } else {
            const float top = warp_max(sum.x);
            const double s = static_cast<double>(sum.y) * exp(static_cast<double>(sum.x) - top);
            const double lse = top + log(warp_sum(s));
            Best best;
#pragma unroll 1
            for (int i = 32; i < n + 32; i += 32) {
                const Pair q = next;
                next = entry(i + lane);
                best.join(q);
            }
            // a log-sum-exp that is not finite makes no candidate; what fp32 cannot hold is no score
            cand = score + (static_cast<double>(best.p.value) - lse);
            if (best.p.at != kNobody && fabs(lse) < INFINITY && static_cast<float>(cand) > -INFINITY) at = k * a.vocab + best.p.at;
        }
    }
    if (lane < a.count) {
        score_s[k * a.count + lane] = cand;
        at_s[k * a.count + lane] = at;
    }
    const int all = a.beams * a.count, i = threadIdx.x;
    const long long o = static_cast<long long>(b) * a.count;
    const int candidates = __syncthreads_count(lane < a.count && at != kNobody);
    // 2^side threads a candidate, which fit: the block has 32 threads a beam
    const int side = 31 - __clz(32 / a.count), mine = i >> side;
    double c = 0;
    int t = kNobody, rank = 0;
    if (mine < all && at_s[mine] != kNobody) {
        c = score_s[mine];
        t = at_s[mine];
#pragma unroll 4
        for (int j = i & ((1 << side) - 1); j < all; j += 1 << side)
            rank += at_s[j] != kNobody && (score_s[j] > c || (score_s[j] == c && at_s[j] < t));
    }
    for (int d = 1; d < 1 << side; d <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, d);
    if (t != kNobody && rank < a.count && (i & ((1 << side) - 1)) == 0) {
        a.out_scores[o + rank] = static_cast<float>(c);
        a.out_parents[o + rank] = t / a.vocab;
        a.out_tokens[o + rank] = t % a.vocab;
    }
    if (i >= candidates && i < a.count) {  // left over
        a.out_scores[o + i] = -INFINITY;
        a.out_parents[o + i] = min(i, a.beams - 1);
        a.out_tokens[o + i] = -1;
    }
}

}  // namespace beam
}  // namespace mm
