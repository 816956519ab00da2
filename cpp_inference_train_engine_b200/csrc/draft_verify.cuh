// Verification of drafted tokens: acceptance against the target's probabilities and one draw
// from the residual (or the bonus) distribution, from given random numbers.
#pragma once
#include "latent_cache.cuh"

namespace mm {
namespace ver {

constexpr int kChunk = 512;                       // vocabulary entries one warp sums at a time
constexpr int kMaxVocab = 262144;
constexpr int kMaxChunks = kMaxVocab / kChunk;

using i64 = long long;

// floor(2^38 clamp(r, 0, 1)); NaN gives 0. Scaling by a power of two is exact.
__device__ __forceinline__ i64 weight(float r) {
    return __float2ll_rz(fminf(fmaxf(r, 0.f), 1.f) * 274877906944.f);
}

// Adds floor(2^38 clamp(r, 0, 1)) = 2^16 hi + lo to two 32-bit sums: hi = floor(x), x = 2^22 r, and lo the
// next 16 bits. Adding 2^23 towards zero leaves the floor in the low mantissa bits (x < 2^23), the
// difference of x and its floor is exact, and the sums count kWeightBias too much per value.
constexpr uint32_t kWeightBias = 0x4B000000u;  // the bits of 2^23
__device__ __forceinline__ void add_weight(float r, uint32_t& hi, uint32_t& lo) {
    const float x = __saturatef(r) * 4194304.f;  // NaN: 0
    const float h = __fadd_rz(x, 8388608.f);
    hi += __float_as_uint(h);
    lo += __float_as_uint(__fmaf_rz(x - (h - 8388608.f), 65536.f, 8388608.f));
}

__device__ __forceinline__ i64 warp_sum_i64(i64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Four consecutive values of a row from entry x (zeros past the vocabulary). ALIGNED: every row
// starts on a 4-value boundary and vocab is a multiple of 4, so they are one vector load.
template <typename T, bool ALIGNED>
__device__ __forceinline__ void load4(const T* __restrict__ row, int x, int vocab, float (&v)[4]) {
    if (ALIGNED) {
        if (x < vocab) {
            if constexpr (sizeof(T) == 4) {
                const float4 f = __ldg(reinterpret_cast<const float4*>(row + x));
                v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
            } else {
                const uint2 u = __ldg(reinterpret_cast<const uint2*>(row + x));
                const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = lat::to_f32(t[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = 0.f;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = x + i < vocab ? lat::to_f32(row[x + i]) : 0.f;
    }
}

// A lane's 8 entries of the 256 from entry x0 on: entry i, and all of them (zeros past the
// vocabulary). ALIGNED: two vector loads; else the warp's lanes load neighbours.
template <bool ALIGNED> __device__ __forceinline__ int entry_of(int x0, int lane, int i) {
    return ALIGNED ? x0 + (i >> 2) * 128 + lane * 4 + (i & 3) : x0 + i * 32 + lane;
}
template <typename T, bool ALIGNED>
__device__ __forceinline__ void load_entries(const T* __restrict__ row, int x0, int lane, int vocab, float (&v)[8]) {
    if constexpr (ALIGNED) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float f[4];
            load4<T, true>(row, x0 + k * 128 + lane * 4, vocab, f);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * k + i] = f[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int at = x0 + i * 32 + lane;
            v[i] = at < vocab ? lat::to_f32(row[at]) : 0.f;
        }
    }
}

// One block per row. Acceptance is one gather per draft; then one pass over one row of p (and
// q) sums the weights of 512-entry chunks, warp 0 finds the chunk that holds the draw from the
// chunk sums, and the chunk alone is read again to find the entry. Bound by the p (and q)
// row's bytes at large batches and by that chain's latency at small ones. 32 registers keep every
// warp slot taken. THREADS: 1024 spreads a row over more warps, 512 runs four rows beside each other on
// an SM, whose chains overlap: 512 where the rows do not fit at once with 1024, two to an SM. Both, in us
// (1024 / 512), probabilities read from memory, with draft probabilities:
//   rows                      64           148          296          370          592          600          1024
//   16,384 tokens, fp32    8.0 / 9.6    8.8 / 10.0  11.0 / 11.9  15.6 / 13.1  19.0 / 16.0  20.2 / 19.0  31.0 / 26.0
//   32,768 tokens, fp32   11.1 / 14.9  12.6 / 15.6  16.8 / 18.9  23.3 / 21.1  29.8 / 28.1  31.0 / 31.9  47.6 / 43.5
//   32,768 tokens, bf16   11.9 / 17.4  12.2 / 17.6  14.2 / 19.1  21.6 / 22.1  26.6 / 23.2  27.9 / 28.9  44.3 / 40.1
// (at 600 the second wave of 512 is nearly empty). 1,024 fp32 rows of 32,768 run at 5.5 TB/s.
template <typename T, bool ALIGNED, int THREADS>
__global__ void __launch_bounds__(THREADS, 2048 / THREADS) verify_drafts_kernel(
    const T* __restrict__ target, const T* __restrict__ draft, const int* __restrict__ tokens,
    const int* __restrict__ lens, const float* __restrict__ u_accept, const float* __restrict__ u_sample, int K, int V,
    int* __restrict__ out_tokens, int* __restrict__ accepted) {
    MM_PDL_ENTRY();
    __shared__ i64 sums[kMaxChunks];
    __shared__ int s_n;
    __shared__ i64 s_total;
    const int b = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const T* p0 = target + static_cast<i64>(b) * (K + 1) * V;
    const T* q0 = draft ? draft + static_cast<i64>(b) * K * V : nullptr;
    const int* x = tokens + static_cast<i64>(b) * K;
    const int len = min(max(lens[b], 0), K);
    if (warp == 0) {
        int n = 0;
        for (int i0 = 0; i0 < len; i0 += 32) {
            const int i = i0 + lane;
            bool ok = i < len;
            if (ok) {
                const int t = x[i];
                ok = t >= 0 && t < V;
                if (ok) {
                    const float p = lat::to_f32(p0[static_cast<i64>(i) * V + t]);
                    const float q = q0 ? lat::to_f32(q0[static_cast<i64>(i) * V + t]) : 1.f;
                    ok = __fmul_rn(u_accept[static_cast<i64>(b) * K + i], q) < p;
                }
            }
            const unsigned m = __ballot_sync(0xffffffffu, ok);
            const int run = m == 0xffffffffu ? 32 : __ffs(~m) - 1;
            n += run;
            if (run < 32) break;
        }
        if (lane == 0) s_n = min(n, len);
    }
    __syncthreads();
    const int n = s_n;
    const T* p = p0 + static_cast<i64>(n) * V;
    const bool rejected = n < len;
    const T* q = rejected && q0 ? q0 + static_cast<i64>(n) * V : nullptr;
    const int hole = rejected && !q0 ? x[n] : -1;  // deterministic drafts: q = 1 at one token
    const int chunks = (V + kChunk - 1) / kChunk;
    bool residual = rejected;

    auto weights4 = [&](int at, i64 (&w)[4]) {
        float pv[4];
        load4<T, ALIGNED>(p, at, V, pv);
        if (residual) {
            if (q) {
                float qv[4];
                load4<T, ALIGNED>(q, at, V, qv);
#pragma unroll
                for (int i = 0; i < 4; ++i) pv[i] -= qv[i];
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (at + i == hole) pv[i] -= 1.f;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = weight(pv[i]);
    };

    for (int pass = 0; pass < 2; ++pass) {
        for (int c = warp; c < chunks; c += THREADS / 32) {
            // 8 entries a lane at a time, all loads first; any order: the sums are exact
            uint32_t hi = 0, lo = 0;
#pragma unroll 1
            for (int x0 = c * kChunk; x0 < (c + 1) * kChunk; x0 += 256) {
                float pv[8];
                load_entries<T, ALIGNED>(p, x0, lane, V, pv);
                if (residual && q) {
                    float qv[8];
                    load_entries<T, ALIGNED>(q, x0, lane, V, qv);
#pragma unroll
                    for (int i = 0; i < 8; ++i) pv[i] -= qv[i];
                } else if (residual && hole >= x0 && hole < x0 + 256) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (entry_of<ALIGNED>(x0, lane, i) == hole) pv[i] -= 1.f;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) add_weight(pv[i], hi, lo);
            }
            // at most 2^31 and 2^25 in a chunk
            hi = __reduce_add_sync(0xffffffffu, hi - kChunk / 32 * kWeightBias);
            lo = __reduce_add_sync(0xffffffffu, lo - kChunk / 32 * kWeightBias);
            const i64 s = (static_cast<i64>(hi) << 16) + lo;
            if (lane == 0) sums[c] = s;
        }
        __syncthreads();
        if (warp == 0) {
            i64 t = 0;
            for (int c = lane; c < chunks; c += 32) t += sums[c];
            t = warp_sum_i64(t);
            if (lane == 0) s_total = t;
        }
        __syncthreads();
        if (s_total > 0 || !residual) break;
        residual = false;  // the residual is all zeros: draw from p itself
        __syncthreads();
    }
    if (warp != 0) return;
    const i64 total = s_total;
    int y = -1;
    if (total > 0) {
        const float u = u_sample[b];
        const i64 k = min(max(__float2ll_rz(u * 16777216.f), 0LL), 16777215LL);  // NaN: 0 after the clamp
        const i64 t = (total >> 24) * k + (((total & 16777215LL) * k) >> 24);   // floor(total k / 2^24)
        // chunk holding the draw
        i64 before = 0;
        int chunk = 0;
        for (int c0 = 0; c0 < chunks; c0 += 32) {
            i64 s = c0 + lane < chunks ? sums[c0 + lane] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const i64 v = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += v;
            }
            const unsigned m = __ballot_sync(0xffffffffu, before + s > t);
            if (m) {
                const int l = __ffs(m) - 1;
                chunk = c0 + l;
                if (l > 0) before += __shfl_sync(0xffffffffu, s, l - 1);
                break;
            }
            before += __shfl_sync(0xffffffffu, s, 31);
        }
        // entry within the chunk
        for (int kk = 0; kk < kChunk / 128; ++kk) {
            const int at = chunk * kChunk + kk * 128 + lane * 4;
            i64 w[4];
            weights4(at, w);
            const i64 own = (w[0] + w[1]) + (w[2] + w[3]);
            i64 s = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const i64 v = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += v;
            }
            const unsigned m = __ballot_sync(0xffffffffu, before + s > t);
            if (m) {
                const int l = __ffs(m) - 1;
                i64 run = before + s - own;
                int e = 0;
                for (; e < 3; ++e) {
                    run += w[e];
                    if (run > t) break;
                }
                y = __shfl_sync(0xffffffffu, at + e, l);
                break;
            }
            before += __shfl_sync(0xffffffffu, s, 31);
        }
    }
    int* out = out_tokens + static_cast<i64>(b) * (K + 1);
    for (int i = lane; i <= K; i += 32) out[i] = i < n ? x[i] : (i == n ? y : -1);
    if (lane == 0) accepted[b] = n;
}

}  // namespace ver
}  // namespace mm
