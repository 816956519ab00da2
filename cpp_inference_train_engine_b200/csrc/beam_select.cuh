// Beam search's selection over beams and vocabulary (mm_beam_select).
#pragma once
#include "latent_cache.cuh"

namespace mm {
namespace beam {

constexpr int kMaxBeams = 32;
constexpr int kMaxVocab = 1 << 20;  // flat candidates k * vocab + v stay below 2^25

struct Select {
    const void* logits;
    long long batch_stride, beam_stride;
    const float* scores;
    const uint8_t* finished;
    int eos, batch, beams, vocab, count;
    float* out_scores;
    int* out_parents;
    int* out_tokens;
};

// One block per batch entry: the beams' log-sum-exp, then the best candidate behind the last one, count times.
template <typename T>
__global__ void __launch_bounds__(256) select_kernel(const Select a) {
    MM_PDL_ENTRY();
    __shared__ double base_s[kMaxBeams];
    __shared__ double best_s[8];
    __shared__ int at_s[8];
    __shared__ float part_s[8];
    __shared__ double sum_s[8];
    const int b = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const T* x0 = static_cast<const T*>(a.logits) + b * a.batch_stride;
    for (int k = 0; k < a.beams; ++k) {
        const T* x = x0 + k * a.beam_stride;
        float m = -INFINITY;
        bool bad = false;
        for (int v = tid; v < a.vocab; v += 256) {
            const float f = lat::to_f32(x[v]);
            bad |= f != f;
            m = fmaxf(m, f);
        }
        m = warp_max(m);
        if (lane == 0) part_s[warp] = m;
        bad = __syncthreads_or(bad);
        for (int w = 0; w < 8; ++w) m = fmaxf(m, part_s[w]);
        double s = 0;
        for (int v = tid; v < a.vocab; v += 256) s += expf(lat::to_f32(x[v]) - m);
        s = warp_sum(s);
        if (lane == 0) sum_s[warp] = s;
        __syncthreads();
        if (tid == 0) {
            s = 0;
            for (int w = 0; w < 8; ++w) s += sum_s[w];
            base_s[k] = bad ? nan("") : m + log(s);
        }
        __syncthreads();
    }
    double last = INFINITY;
    int last_at = -1;
    for (int r = 0; r < a.count; ++r) {
        double best = -INFINITY;
        int at = 0x7fffffff;
        auto offer = [&](double c, int i) {  // (NaN compares false; what fp32 cannot hold is no score)
            if ((c < last || (c == last && i > last_at)) && (c > best || (c == best && i < at)) && static_cast<float>(c) > -INFINITY) {
                best = c;
                at = i;
            }
        };
        for (int k = 0; k < a.beams; ++k) {
            const float sc = a.scores[b * a.beams + k];
            if (!(fabsf(sc) < INFINITY)) continue;
            if (a.finished && a.finished[b * a.beams + k]) {
                if (tid == 0) offer(sc, k * a.vocab + a.eos);
            } else if (fabs(base_s[k]) < INFINITY) {
                for (int v = tid; v < a.vocab; v += 256)
                    offer(sc + (static_cast<double>(lat::to_f32(x0[k * a.beam_stride + v])) - base_s[k]), k * a.vocab + v);
            }
        }
        for (int o = 16; o > 0; o >>= 1) {
            const double c = __shfl_xor_sync(0xffffffffu, best, o);
            const int i = __shfl_xor_sync(0xffffffffu, at, o);
            if (c > best || (c == best && i < at)) {
                best = c;
                at = i;
            }
        }
        if (lane == 0) {
            best_s[warp] = best;
            at_s[warp] = at;
        }
        __syncthreads();
        for (int w = 0; w < 8; ++w)
            if (best_s[w] > best || (best_s[w] == best && at_s[w] < at)) {
                best = best_s[w];
                at = at_s[w];
            }
        __syncthreads();
        last = best;
        last_at = at;
        if (tid == 0) {
            const bool none = !(best > -INFINITY);
            const long long o = static_cast<long long>(b) * a.count + r;
            a.out_scores[o] = static_cast<float>(best);
            a.out_parents[o] = none ? min(r, a.beams - 1) : at / a.vocab;
            a.out_tokens[o] = none ? -1 : at % a.vocab;
        }
    }
}

}  // namespace beam
}  // namespace mm
