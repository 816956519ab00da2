// Beam search's selection over beams and vocabulary (mm_beam_select).
//
// One pass over the logits: a block takes a part of a beam's tokens, its warps divide them, and keeps their
// maximum, the sum of exponentials below it and the best 32 of them (rank r in lane r); then the parts of a beam are
// joined, and the beams. The pass itself keeps one maximum per lane and step: of the 32 lanes' maxima over a
// stretch of steps the count-th largest bounds the list from below, so that only the few (lane, step) pairs that
// reach it are looked at again, from the cache. Where a batch entry's blocks fit a cluster (16) its first block joins
// them from their shared memory, else a second kernel from the workspace.
//
// Measured on one B200: 64 x 8 beams of 32,768 fp32 tokens 21 us (3.1 TB/s; the pass 16 and the joins 5), bound by the
// phases of the pass, whose warps all load first and then all sort; 1 x 4 of 16,384 8.4 us, bound by the chain of a load,
// two sorts and the joins.
#pragma once
#include "paged_cache.cuh"

namespace mm {
namespace beam {

using paged::Two;

constexpr int kMaxBeams = 32;
constexpr int kMaxVocab = 1 << 20;  // flat candidates k * vocab + v stay below 2^25
constexpr float kLowest = -3.402823466e38f;
constexpr int kMaxParts = 32;       // of a beam's tokens, a block each
constexpr int kMaxCluster = 16;

// Candidates in order: by value, then by the lower index. Nobody: (-infinity, kNobody).
constexpr int kNobody = 0x7fffffff;
struct alignas(8) Pair {
    float value;
    int at;
};
struct Select {
    const void* logits;
    long long batch_stride, beam_stride;
    const float* scores;
    const uint8_t* finished;
    int eos, batch, beams, vocab, count, parts;
    float* out_scores;
    int* out_parents;
    int* out_tokens;
    // without a cluster, of each part [batch * beams * parts]: its best tokens [32], maximum and sum
    Pair* best;
    float2* sum;
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
// The lanes' candidates in order, the best in lane 0. A function of its own: it is called from several places, once or
// twice a warp, and its instructions come from memory the first time.
static __device__ __noinline__ Pair sorted(Pair q) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size >> 1; o > 0; o >>= 1) exchange(q, o, (threadIdx.x & size) == 0 || size == 32);
    return q;
}
// The best 32 candidates so far, rank r in lane r.
struct Best {
    Pair p{-INFINITY, kNobody};
    // Joins 32 more, in order.
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
// The k-th largest (from 1) of the lanes' values.
__device__ __forceinline__ float kth_largest(float v, int k) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size >> 1; o > 0; o >>= 1) {
            const float u = __shfl_xor_sync(0xffffffffu, v, o);
            v = ((threadIdx.x & o) == 0) == ((threadIdx.x & size) == 0 || size == 32) ? fmaxf(u, v) : fminf(u, v);
        }
    return __shfl_sync(0xffffffffu, v, k - 1);
}

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < INFINITY; }

// Candidates of several beams: scores in fp64, k * vocab + v.
struct Scored {
    double value;
    int at;
};
__device__ __forceinline__ Scored from_lane(Scored p, int lane_xor) {
    return {__shfl_xor_sync(0xffffffffu, p.value, lane_xor), __shfl_xor_sync(0xffffffffu, p.at, lane_xor)};
}
__device__ __forceinline__ bool ahead(Scored a, Scored b) { return a.value > b.value || (a.value == b.value && a.at < b.at); }
// Best::join_sorted of these: p's lanes become the best 32 of both lists, in order.
__device__ __forceinline__ void join_sorted(Scored& p, Scored q) {
    q = from_lane(q, 31);
    if (ahead(q, p)) p = q;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Scored u = from_lane(p, o);
        if (ahead(u, p) == ((threadIdx.x & o) == 0)) p = u;
    }
}

// Joins a batch entry's parts and beams with `warps` warps, which all come here. list(k, part) is the lane's entry
// of a part's list, sum(k, part) its maximum and sum. scratch: 512 bytes for each warp.
template <class List, class Sum>
__device__ __forceinline__ void finish(const Select& a, int b, int warps, uint8_t* scratch, List list, Sum sum) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Scored all{-INFINITY, kNobody};
    for (int k = warp; k < a.beams; k += warps) {
        const int row = b * a.beams + k;
        // asked for together: what the parts of a finished or dead beam hold is not used
        Pair next = list(k, 0);
        const float2 part = lane < a.parts ? sum(k, lane) : make_float2(kLowest, 0.f);
        const float score = __ldg(a.scores + row);
        const bool ended = a.finished && __ldg(a.finished + row);
        Scored mine{-INFINITY, kNobody};
        if (finite(score) && ended) {
            if (lane == 0) mine = {score, k * a.vocab + a.eos};
        } else if (finite(score)) {
            const float top = warp_max(part.x);
            const double s = static_cast<double>(part.y) * exp(static_cast<double>(part.x) - top);
            const double lse = top + log(warp_sum(s));
            Best best;
#pragma unroll 1
            for (int i = 1; i <= a.parts; ++i) {
                const Pair q = next;
                if (i < a.parts) next = list(k, i);
                best.join_sorted(q);
            }
            // a log-sum-exp that is not finite makes no candidate; what fp32 cannot hold is no score
            const double c = score + (static_cast<double>(best.p.value) - lse);
            if (best.p.at != kNobody && fabs(lse) < INFINITY && static_cast<float>(c) > -INFINITY) mine = {c, k * a.vocab + best.p.at};
        }
        join_sorted(all, mine);
    }
    // the warps' lists two by two
    double* value_s = reinterpret_cast<double*>(scratch);
    int* at_s = reinterpret_cast<int*>(value_s + warps * 32);
    for (int d = 1; d < warps; d <<= 1) {
        if (warp % (2 * d) == d) {
            value_s[warp * 32 + lane] = all.value;
            at_s[warp * 32 + lane] = all.at;
        }
        __syncthreads();
        if (warp % (2 * d) == 0 && warp + d < warps) join_sorted(all, {value_s[(warp + d) * 32 + lane], at_s[(warp + d) * 32 + lane]});
    }
    if (warp == 0 && lane < a.count) {
        const bool none = all.at == kNobody;
        const long long o = static_cast<long long>(b) * a.count + lane;
        a.out_scores[o] = static_cast<float>(all.value);
        a.out_parents[o] = none ? min(lane, a.beams - 1) : all.at / a.vocab;
        a.out_tokens[o] = none ? -1 : all.at % a.vocab;
    }
}

__device__ __forceinline__ unsigned long long load_cluster64(uint32_t cluster_addr) {
    unsigned long long v;
    asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(v) : "r"(cluster_addr) : "memory");
    return v;
}

// `n` bytes (0 to 16) of a 16-byte piece, the others as zeros.
__device__ __forceinline__ void copy_piece(void* dst, const void* src, int n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(n) : "memory");
}

// Block (part, beam row). A load is E values, counted from the row's first token, so that equal rows have equal sums
// wherever they stand (a beam's continuations tie with those of an equal one). The memory comes in aligned pieces of
// 16 bytes, two steps ahead, through shared memory; of a row that begins inside a piece (by `shift` values) a load is the
// end of one piece and the beginning of the next.
constexpr int kLoads = 4, kStages = 3;
constexpr int kPieces = kStages * kLoads * 33;  // a warp's: each 32 loads and one piece more
constexpr int ring_bytes(int warps) { return warps * kPieces * 16; }  // 198 KB an SM
template <typename T, int kWarps, bool CLUSTER, bool SHIFTED>
__global__ void __launch_bounds__(32 * kWarps, 32 / kWarps) select_parts_kernel(const Select a) {
    MM_PDL_ENTRY();
    constexpr int E = 16 / sizeof(T), U = kLoads, kSteps = 8;  // values per load, loads per step, steps per stretch
    extern __shared__ uint4 ring_s[];
    __shared__ Pair list_s[32];
    __shared__ float2 total_s;
    __shared__ Pair wait_s[kWarps][64];
    __shared__ float2 sum_s[kWarps];
    __shared__ uint8_t pairs_s[kWarps][32 * kSteps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
    const int b = row / a.beams;
    const bool dead = !finite(__ldg(a.scores + row)) || (a.finished && a.finished[row]);
    if (!CLUSTER && dead) return;  // the join does not use it either
    const T* x = static_cast<const T*>(a.logits) + b * a.batch_stride + (row - b * a.beams) * a.beam_stride;
    const int shift = SHIFTED ? static_cast<int>(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T)) : 0;
    const uint8_t* pieces = reinterpret_cast<const uint8_t*>(x - shift);
    const int loads = dead ? 0 : (a.vocab + E - 1) / E;
    const int per = (loads + kWarps * a.parts - 1) / (kWarps * a.parts), l0 = min((part * kWarps + warp) * per, loads), l1 = min(l0 + per, loads);
    // Candidates wait in shared memory until there are 32 (or no more): joining the list costs a sort. What is
    // behind the list's last entry does not wait.
    Pair* wait = wait_s[warp];
    int waiting = 0;
    Best best;
    Pair last{-INFINITY, kNobody};
    auto join = [&] {
        __syncwarp();
        best.join_sorted(sorted(lane < waiting ? wait[lane] : Pair{-INFINITY, kNobody}));
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
    uint4* ring = ring_s + warp * kPieces + lane;
    int stage = 0, filled = 0;
    auto bring = [&](uint4* dst, int piece) {
        const int n = (a.vocab + shift - piece * E) * static_cast<int>(sizeof(T));  // up to the row's end
        if (SHIFTED && piece == 0) {  // what is before the row is not read
            for (int e = shift; e < min(E, a.vocab + shift); ++e) reinterpret_cast<T*>(dst)[e] = x[e - shift];
        } else if (n > 0) {
            copy_piece(dst, pieces + static_cast<long long>(piece) * 16, min(n, 16));
        }
    };
    auto fetch = [&](int i0) {
        uint4* to = ring + filled * U * 33;
        const int i = i0 + lane;
        if (i0 + U * 32 <= l1 && (i0 + U * 32 + 1) * E <= a.vocab && (!SHIFTED || i0 > 0)) {  // whole pieces all
            const uint8_t* from = pieces + static_cast<long long>(i) * 16;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                cp_async16(to + u * 33, from + u * 512, true);
                if (SHIFTED && lane == 0) cp_async16(to + u * 33 + 32, from + u * 512 + 512, true);
            }
        } else if (i0 < l1) {  // (nothing is written behind the last step)
#pragma unroll 1
            for (int u = 0; u < U; ++u) {
                if (i + u * 32 < l1 + (SHIFTED ? 1 : 0)) bring(to + u * 33, i + u * 32);
                if (SHIFTED && lane == 0 && i + u * 32 + 32 <= l1) bring(to + u * 33 + 32, i + u * 32 + 32);
            }
        }
        cp_async_commit();
        filled = filled == kStages - 1 ? 0 : filled + 1;
    };
    // The load in pieces p[0] and p[1], as 32-bit words.
    auto words = [&](const uint4* p, uint32_t (&w)[4]) {
        const uint4 first = p[0];
        w[0] = first.x;
        w[1] = first.y;
        w[2] = first.z;
        w[3] = first.w;
        if constexpr (SHIFTED) {
            const uint4 second = p[1];
            uint32_t v[8] = {w[0], w[1], w[2], w[3], second.x, second.y, second.z, second.w};
            const int whole = shift * static_cast<int>(sizeof(T)) / 4;
#pragma unroll
            for (int j = 0; j < 7; ++j) v[j] = whole & 1 ? v[j + 1] : v[j];
#pragma unroll
            for (int j = 0; j < 5; ++j) v[j] = whole & 2 ? v[j + 2] : v[j];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = sizeof(T) == 2 && (shift & 1) ? __funnelshift_r(v[j], v[j + 1], 16) : v[j];
        }
    };
    fetch(l0);
    fetch(l0 + 32 * U);
    for (int base = l0; base < l1; base += 32 * U * kSteps) {
        float tops[kSteps], most = -INFINITY;
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
            const int i0 = base + st * 32 * U;
            tops[st] = -INFINITY;
            if (i0 >= l1) continue;
            float v[U][E];
            cp_async_wait<kStages - 2>();
            if constexpr (SHIFTED) __syncwarp();  // (a lane's second piece is its neighbour's first)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                uint32_t raw[4];
                words(ring + (stage * U + u) * 33, raw);
#pragma unroll
                for (int e = 0; e < E; ++e) v[u][e] = lat::to_f32(reinterpret_cast<const T*>(raw)[e]);
            }
            stage = stage == kStages - 1 ? 0 : stage + 1;
            if (i0 + 32 * U > l1 || (i0 + 32 * U) * E > a.vocab) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int i = i0 + u * 32 + lane, n = i < l1 ? a.vocab - i * E : 0;  // values of the load
#pragma unroll
                    for (int e = 0; e < E; ++e) v[u][e] = e < n ? v[u][e] : -INFINITY;
                }
            }
            fetch(i0 + 2 * 32 * U);
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
            const float floor = kth_largest(most, a.count);
            if (floor > last.value) last = {floor, kNobody};
        }
        // the steps and lanes that reach it, in line; their values from the ring or the cache, kAtOnce pairs' at a time
        int pairs = 0;
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
            const bool in = tops[st] >= last.value && tops[st] > -INFINITY;
            const unsigned who = __ballot_sync(0xffffffffu, in);
            if (in) pairs_s[warp][pairs + __popc(who & ((1u << lane) - 1))] = static_cast<uint8_t>(st * 32 + lane);
            pairs += __popc(who);
        }
        __syncwarp();
        const bool held = l1 - l0 <= 32 * U * kStages;  // in the ring: no step has been overwritten
        constexpr int kSide = 32 / (U * E), kAtOnce = 4 * kSide;  // pairs side by side in a warp: 2 for 16 values
        const int place = lane % (U * E);
        for (int j0 = 0; j0 < pairs; j0 += kAtOnce) {
            float v[4];
            int t[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int pair = j0 + j * kSide + lane / (U * E), code = pair < pairs ? pairs_s[warp][pair] : 0;
                const int i = base + (code >> 5) * 32 * U + place / E * 32 + (code & 31);
                t[j] = i * E + place % E;
                const T* from = held ? reinterpret_cast<const T*>(ring_s + warp * kPieces + ((code >> 5) * U + place / E) * 33 + (code & 31)) + shift + place % E
                                     : x + t[j];
                v[j] = pair < pairs && i < l1 && t[j] < a.vocab ? lat::to_f32(*from) : -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) offer(v[j], t[j]);
        }
        __syncwarp();
    }
    cp_async_wait<0>();
    join();
    // the lanes' sums below one maximum (a NaN or +infinity anywhere makes the sum a NaN), then the warps'
    auto scaled = [&](float2 v, float top) { return v.y * fast_exp2((v.x - top) * kLog2e); };
    float top = warp_max(m);
    s = warp_sum(scaled({m, s}, top));
    if (lane == 0) sum_s[warp] = make_float2(top, s);
    // the warps' lists two by two
    wait[lane] = best.p;
    for (int d = 1; d < kWarps; d <<= 1) {
        __syncthreads();
        if (warp % (2 * d) == 0) {
            best.join_sorted(wait_s[warp + d][lane]);
            wait[lane] = best.p;
        }
    }
    if (warp == 0) {
        const float2 mine = lane < kWarps ? sum_s[lane] : make_float2(kLowest, 0.f);
        top = warp_max(mine.x);
        s = warp_sum(scaled(mine, top));
        if constexpr (CLUSTER) {
            list_s[lane] = best.p;
            if (lane == 0) total_s = make_float2(top, s);
        } else {
            a.best[static_cast<long long>(blockIdx.x) * 32 + lane] = best.p;
            if (lane == 0) a.sum[blockIdx.x] = make_float2(top, s);
        }
    }
    if constexpr (CLUSTER) {
        cluster_sync_all();
        if (cluster_ctarank() == 0) {
            const uint32_t lists = smem_u32(list_s), totals = smem_u32(&total_s);
            finish(a, b, kWarps, reinterpret_cast<uint8_t*>(ring_s),
                   [&](int k, int p) {
                       const unsigned long long v = load_cluster64(mapa_shared(lists + lane * 8, k * a.parts + p));
                       return Pair{__uint_as_float(static_cast<uint32_t>(v)), static_cast<int>(v >> 32)};
                   },
                   [&](int k, int p) {
                       const unsigned long long v = load_cluster64(mapa_shared(totals, k * a.parts + p));
                       return make_float2(__uint_as_float(static_cast<uint32_t>(v)), __uint_as_float(static_cast<uint32_t>(v >> 32)));
                   });
        }
        cluster_sync_all();  // no block's shared memory goes before it has been read
    }
}

// Block per batch entry, a warp per beam.
static __global__ void __launch_bounds__(1024) select_join_kernel(const Select a) {
    MM_PDL_ENTRY();
    extern __shared__ uint4 join_s[];
    const int b = blockIdx.x, lane = threadIdx.x & 31;
    finish(a, b, a.beams, reinterpret_cast<uint8_t*>(join_s),
           [&](int k, int p) {
               const float2 v = __ldcg(reinterpret_cast<const float2*>(a.best + (static_cast<long long>(b * a.beams + k) * a.parts + p) * 32 + lane));
               return Pair{v.x, __float_as_int(v.y)};
           },
           [&](int k, int p) { return __ldcg(a.sum + static_cast<long long>(b * a.beams + k) * a.parts + p); });
}

}  // namespace beam
}  // namespace mm
