// A latent cache in pages: appending positions through a page table (normalised, rotated, in 8 or 16
// bits) and page tables that follow a beam search's parents.
#pragma once
#include "latent_cache.cuh"

namespace mm {
namespace paged {

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
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

struct Table {
    const int* entry;
    long long stride;
    int rows, columns;
    int shift;  // log2 of the page size, -1 where it is no power of two
};

// The pool's page of position t of table row r, or -1 (a position or a page that is not there); at: the entry.
__device__ __forceinline__ int page_of(const Table& t, int pages, int page, int row, int position, int& at) {
    if (row < 0 || row >= t.rows || position < 0) return -1;
    const int column = t.shift >= 0 ? position >> t.shift : position / page;
    if (column >= t.columns) return -1;
    at = position - column * page;
    const int p = __ldg(t.entry + row * t.stride + column);
    return p >= 0 && p < pages ? p : -1;
}

// Pair j's angle at `position` in turns: f = theta^(-2 j / width) / (2 pi) in fp64, whose product with any
// 31-bit position is off by 2^31 * 2^-53 turns at most; the fraction, within half a turn, goes on in fp32, where
// the fast sine and cosine are off by 2^-21, far below a 16-bit key's rounding. (sincospif: 40 instructions more
// a token, 63 us instead of 57 for 131,072 tokens when that was measured.)
__device__ __forceinline__ void rotation(double f, int position, float& sin_t, float& cos_t) {
    const double turns = f * position;
    __sincosf(6.283185307f * static_cast<float>(turns - rint(turns)), &sin_t, &cos_t);
}

constexpr int kMaxPairs = 128;  // of a rope key of 256
struct Rotation {
    double f[kMaxPairs];
};

// ------------------------------------------------------------------ append
// Any width, stride and alignment: one warp per token. The widths of the framework's models run on
// append_vec_kernel. Bound by its scalar loads, of each value two or three times: 131,072 fp16 tokens of 504 + 32 take 153 us
// into 8-bit pages (1.4 TB/s), 103 into 16-bit ones; 61 of 120 + 16 3.8, a launch.
template <typename T, typename T16, bool Q8>
__global__ void __launch_bounds__(256) append_kernel(lat::CacheOut c, Table table, const T* __restrict__ values,
                                                     long long stride, const int* __restrict__ rows,
                                                     const int* __restrict__ positions, long long n, int kv, int rd,
                                                     const float* __restrict__ norm, float eps,
                                                     const __grid_constant__ Rotation rot) {
    MM_PDL_ENTRY();
    const long long i = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (i >= n) return;
    const int position = positions[i];
    int at = 0;
    const long long p = page_of(table, c.rows, c.positions, rows ? rows[i] : static_cast<int>(i), position, at);
    if (p < 0) return;
    const T* x = values + i * stride;
    float inv = 1.f;
    if (norm) {
        float sum = 0.f;
        for (int k = lane; k < kv; k += 32) {
            const float v = lat::to_f32(x[k]);
            sum = fmaf(v, v, sum);
        }
        inv = rsqrtf(warp_sum(sum) / kv + eps);
    }
    auto value = [&](int k) { return norm ? lat::to_f32(x[k]) * inv * norm[k] : lat::to_f32(x[k]); };
    T16* key;
    if constexpr (Q8) {
        float mx = 0.f;
        for (int k = lane; k < kv; k += 32) mx = fmaxf(mx, fabsf(value(k)));
        const float s = fmaxf(__fdiv_rn(warp_max(mx), lat::kE4m3Max), lat::kScaleFloor);
        uint8_t* dst = c.latent + p * c.row_stride + at * c.pos_stride;
        for (int k = lane; k < kv; k += 32) dst[k] = __nv_cvt_float_to_fp8(__fdiv_rn(value(k), s), __NV_SATFINITE, __NV_E4M3);
        if (lane == 0) c.scale[p * c.scale_row_stride + at] = s;
        key = reinterpret_cast<T16*>(c.rope) + p * c.rope_row_stride + at * c.rope_pos_stride;
    } else {
        T16* dst = reinterpret_cast<T16*>(c.latent) + p * c.row_stride + at * c.pos_stride;
        for (int k = lane; k < kv; k += 32) dst[k] = lat::from_f32<T16>(value(k));
        key = dst + kv;
    }
    for (int j = lane; j < rd / 2; j += 32) {
        float sn, cs;
        rotation(rot.f[j], position, sn, cs);
        const float a = lat::to_f32(x[kv + 2 * j]), b = lat::to_f32(x[kv + 2 * j + 1]);
        key[2 * j] = lat::from_f32<T16>(a * cs - b * sn);
        key[2 * j + 1] = lat::from_f32<T16>(a * sn + b * cs);
    }
}

// KV = 128 or 512, 16-byte accesses: KV / 16 lanes take a token, 16 latent values and (the first R / 2 of them)
// one pair of the key each; sums and maxima are shuffle reductions over the lane group. The CTAs that fit walk
// the tokens, the next ones already on their way to shared memory, where a lane finds what it asked for itself (no
// barrier); where they go each lane looks up for one of the group's next tokens (a lookup a token, by all of its lanes,
// took 51.8 us for the first of the following, and what was on its way in registers 50.5). 131,072 fp16 tokens of 512 + 32
// take 41 us into 8-bit pages (5.3 TB/s; 44 to 46 us where other inputs come in between; bound by instructions, without the
// rotation it is 1 less), without a norm, whose codes are the quotients', 45; 51 into 16-bit ones (5.6 TB/s of reads and
// writes mixed).
//
// Slots of a warp (the token at hand and those on their way) and CTAs per SM: more are not better where the bytes are
// the bound. us of the above into 8-bit pages, into 16-bit ones, of 65,536 fp32 tokens into 8-bit ones, and of 300,000
// bf16 ones of 128 + 16 into 16-bit ones: 2 slots and 3 CTAs 44.2, 51.1, 31.2, 32.0; 3 and 4 41.1, 56.2, 32.9 (with 2
// slots), 31.7; 4 and 4 42.3, 56.5, -, 35.1.
template <typename T, bool Q8> struct AppendRing {
    static constexpr bool kMore = Q8 && sizeof(T) == 2;
    static constexpr int kSlots = kMore ? 3 : 2, kCtas = kMore ? 4 : 3;
    static constexpr int kKey = 512 * static_cast<int>(sizeof(T));  // [chunk][lane] 16 bytes, then [lane] a pair
    static constexpr int kSlot = kKey + 32 * 2 * static_cast<int>(sizeof(T));
};
template <int BYTES> __device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
template <typename T, typename T16, int KV, int R, bool Q8, bool NORM>
__global__ void __launch_bounds__(256, AppendRing<T, Q8>::kCtas) append_vec_kernel(
    lat::CacheOut c, Table table, const T* __restrict__ values, long long stride, const int* __restrict__ rows,
    const int* __restrict__ positions, long long n, const float* __restrict__ norm, float eps, const __grid_constant__ Rotation rot) {
    using Ring = AppendRing<T, Q8>;
    const bool normed = Q8 ? NORM : norm != nullptr;
    constexpr int L = KV / 16, P = 32 / L;                              // lanes per token, tokens side by side in a warp
    constexpr int E = 16 / static_cast<int>(sizeof(T)), NC = 16 / E;    // values of a chunk, chunks of a lane: every L-th
    __shared__ float4 norm_s[KV / 4];
    __shared__ alignas(16) uint8_t ring_s[8][Ring::kSlots][Ring::kSlot];
    const int lane = threadIdx.x & 31, sub = lane % L, mine = lane / L;
    const double f = sub < R / 2 ? rot.f[sub] : 0.0;
    uint8_t* ring = ring_s[threadIdx.x >> 5][0];
    const uint32_t chunks = smem_u32(ring) + lane * 16, keys = smem_u32(ring) + Ring::kKey + lane * 2 * static_cast<int>(sizeof(T));
    MM_PDL_ENTRY();
    // (quarter q of every lane's 16 in line: no bank is asked twice)
    if (normed && threadIdx.x < KV / 4) {
        const int q = threadIdx.x / L, l = threadIdx.x % L;  // 4 values of chunk q * 4 / E
        norm_s[threadIdx.x] = __ldg(reinterpret_cast<const float4*>(norm + q * 4 / E * (KV / NC) + l * E + q * 4 % E));
    }
    __syncthreads();
    const long long step = static_cast<long long>(gridDim.x) * 8 * P;
    const long long first = (static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5)) * P;
    long long i = first + mine;  // this lane group's token
    const T* x = values + i * stride + sub * E;
    auto ask = [&](long long j, const T* from, int slot) {
        if (j < n) {
#pragma unroll
            for (int q = 0; q < NC; ++q) copy_async<16>(chunks + slot + q * 512, from + q * (KV / NC));
            if (sub < R / 2) copy_async<2 * sizeof(T)>(keys + slot, from + (KV - (E - 2) * sub));
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const long long stride_step = step * stride;
    // Where the group's next L tokens go, a token a lane.
    long long latent_at = 0, rope_at = 0, scale_at = 0;
    int position = -1;
    auto look_up = [&](long long j) {
        int at = 0;
        position = j < n ? __ldg(positions + j) : -1;
        const int p = page_of(table, c.rows, c.positions, rows && j < n ? __ldg(rows + j) : static_cast<int>(j), position, at);
        if (p < 0) position = -1;
        latent_at = p * c.row_stride + at * c.pos_stride;
        if (Q8) {
            rope_at = p * c.rope_row_stride + at * c.rope_pos_stride;
            scale_at = p * c.scale_row_stride + at;
        }
    };
    look_up(i + sub * step);
#pragma unroll
    for (int k = 0; k + 1 < Ring::kSlots; ++k, x += stride_step) ask(i + k * step, x, k * Ring::kSlot);
    int slot = 0, turn = 0;
    for (long long i0 = first; i0 < n; i0 += step, i += step, x += stride_step) {  // whole warps walk together (their shuffles)
        ask(i + (Ring::kSlots - 1) * step, x, slot == 0 ? (Ring::kSlots - 1) * Ring::kSlot : slot - Ring::kSlot);
        if (turn == 0 && i0 != first) look_up(i + sub * step);
        const int now = __shfl_sync(0xffffffffu, position, turn, L);
        const long long to = __shfl_sync(0xffffffffu, latent_at, turn, L);
        long long rope_to = 0, scale_to = 0;
        if (Q8) {
            rope_to = __shfl_sync(0xffffffffu, rope_at, turn, L);
            scale_to = __shfl_sync(0xffffffffu, scale_at, turn, L);
        }
        turn = (turn + 1) % L;
        asm volatile("cp.async.wait_group %0;" ::"n"(Ring::kSlots - 1) : "memory");
        float v[16];
#pragma unroll
        for (int q = 0; q < NC; ++q) {
            const uint4 x = *reinterpret_cast<const uint4*>(ring + slot + q * 512 + lane * 16);
#pragma unroll
            for (int e = 0; e < E; ++e) v[q * E + e] = lat::to_f32(reinterpret_cast<const T*>(&x)[e]);
        }
        T pair[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) pair[e] = reinterpret_cast<const T*>(ring + slot + Ring::kKey)[2 * lane + e];
        slot = slot == (Ring::kSlots - 1) * Ring::kSlot ? 0 : slot + Ring::kSlot;
        float inv = 1.f;  // what the values below are still to be multiplied by
        if (normed) {
            Two sums[2] = {Two(0.f, 0.f), Two(0.f, 0.f)};
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const float4 w = norm_s[e / 4 * L + sub];
                const Two x(v[e], v[e + 1]), y(v[e + 2], v[e + 3]), a = x * Two(w.x, w.y), b = y * Two(w.z, w.w);
                sums[0] = fma2(x, x, sums[0]);
                sums[1] = fma2(y, y, sums[1]);
                v[e] = a.lo();
                v[e + 1] = a.hi();
                v[e + 2] = b.lo();
                v[e + 3] = b.hi();
            }
            sums[0] = sums[0] + sums[1];
            float sum = sums[0].lo() + sums[0].hi();
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            inv = rsqrtf(sum * (1.f / KV) + eps);
        }
        float s = 0.f;
        if constexpr (Q8) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s = fmaxf(s, fabsf(v[e]));
            if constexpr (L == 32) {  // (of values that are not negative their bits have the same order)
                s = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(s)));
            } else {
#pragma unroll
                for (int o = L / 2; o > 0; o >>= 1) s = fmaxf(s, __shfl_xor_sync(0xffffffffu, s, o));
            }
            s = fmaxf(__fdiv_rn(s * inv, lat::kE4m3Max), lat::kScaleFloor);
        }
        if (now < 0) continue;
        T16* key;
        if constexpr (Q8) {
            auto codes4 = [](float a, float b, float c, float d) {
                return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3)) |
                       (static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3)) << 16);
            };
            auto codes = [&](int e, float by) {
                const Two f(by, by), x = Two(v[4 * e], v[4 * e + 1]) * f, y = Two(v[4 * e + 2], v[4 * e + 3]) * f;
                return codes4(x.lo(), x.hi(), y.lo(), y.hi());
            };
            const float r = __frcp_rn(s);
            uint32_t q[4];
            if (normed) {
                // by the reciprocal: within 3 ulp of the quotient, as the normalised values are of theirs (the quotients' own
                // codes, as below, take 7 us more for the first of the tokens above)
                float by = inv * r;
                if (by > 3.402823466e38f) {  // (zero weights over tiny values: not 0 times an infinity)
                    by = r;
#pragma unroll
                    for (int e = 0; e < 16; ++e) v[e] *= inv;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) q[e] = codes(e, by);
            } else {
                // The codes of the quotients. The product with the reciprocal is within 2 ulp of the quotient, and rounding is
                // monotonic: where the products with one 2^-21 lower and higher have the same code, so has the quotient. A
                // lane in which they differ anywhere (a quotient that close to the middle of two codes) divides.
                const float below = r * (1.f - 4.76837158e-7f), above = r * (1.f + 4.76837158e-7f);
                uint32_t differ = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    q[e] = codes(e, below);
                    differ |= q[e] ^ codes(e, above);
                }
                if (differ) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        q[e] = codes4(__fdiv_rn(v[4 * e], s), __fdiv_rn(v[4 * e + 1], s), __fdiv_rn(v[4 * e + 2], s), __fdiv_rn(v[4 * e + 3], s));
                }
            }
            uint8_t* dst = c.latent + to + sub * E;
#pragma unroll
            for (int x = 0; x < NC; ++x) {
                if constexpr (E == 8) *reinterpret_cast<uint2*>(dst + x * (KV / NC)) = make_uint2(q[2 * x], q[2 * x + 1]);
                else *reinterpret_cast<uint32_t*>(dst + x * (KV / NC)) = q[x];
            }
            if (sub == 0) c.scale[scale_to] = s;
            key = reinterpret_cast<T16*>(c.rope) + rope_to;
        } else {
            T16* dst = reinterpret_cast<T16*>(c.latent) + to;
            if (normed) {
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] *= inv;
            }
#pragma unroll
            for (int x = 0; x < NC; ++x) {
                uint32_t w[E / 2];
#pragma unroll
                for (int e = 0; e < E; e += 2) w[e / 2] = lat::pack2<T16>(v[x * E + e], v[x * E + e + 1]);
                T16* to = dst + x * (KV / NC) + sub * E;
                if constexpr (E == 8) *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
                else *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
            }
            key = dst + KV;
        }
        if (sub < R / 2) {
            float sn, cs;
            rotation(f, now, sn, cs);
            const float a = lat::to_f32(pair[0]), b = lat::to_f32(pair[1]);
            *reinterpret_cast<uint32_t*>(key + 2 * sub) = lat::pack2<T16>(a * cs - b * sn, a * sn + b * cs);
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ------------------------------------------------------------------ reorder
// One array of the pool (latent, rope keys or scales) as bytes.
struct Plane {
    uint8_t* data;
    long long layer, page, position;  // strides in bytes
    int bytes;                        // of a position
    int vec;                          // bytes an access may take: 16, 4 or 1
};
struct Reorder {
    Table table;
    const int* spare;
    const int* lengths;
    const int* parents;
    int* out_table;
    int* out_spare;
    int* out_lengths;
    int page, pages, layers;
    Plane plane[3];
};

struct Move {
    int parent, length, full;  // the parent, its positions and its full pages
    bool swap;                 // the row's spare page becomes its entry `full`, its own page its spare one
    int part;                  // positions to copy into it
    int from, to;              // from this page of the pool, to that
};
__device__ __forceinline__ int length_of(const Reorder& a, int row) {
    return static_cast<int>(min(max(static_cast<long long>(a.lengths[row]), 0LL), static_cast<long long>(a.table.columns) * a.page));
}
// A row that takes over another one needs a page of its own behind the full ones. Its entry there is one where both
// have the same whole number of pages (it is still to be filled); a row of another length may hold a page there
// that others share, so that it takes its spare page even where there is nothing to copy.
__device__ __forceinline__ Move move_of(const Reorder& a, int row) {
    Move m;
    m.parent = a.parents[row];
    if (m.parent < 0 || m.parent >= a.table.rows) m.parent = row;
    m.length = length_of(a, m.parent);
    m.full = m.length / a.page;
    const int part = m.length - m.full * a.page;
    m.swap = m.parent != row && m.full < a.table.columns && (part > 0 || m.length != length_of(a, row));
    m.part = m.swap ? part : 0;
    m.from = m.to = -1;
    if (m.swap) {
        m.from = a.table.entry[m.parent * a.table.stride + m.full];
        m.to = a.spare[row];
    }
    return m;
}

// Whether another row has the page that `row` has in column j (rows share pages in one column); looks at every `step`-th.
__device__ __forceinline__ bool shared_at(const Reorder& a, int row, int j, int first, int step) {
    const int* column = a.table.entry + j;
    const int page = column[row * a.table.stride];
    for (int r = first; r < a.table.rows; r += step)
        if (r != row && column[r * a.table.stride] == page) return true;
    return false;
}

// `n` elements of type V per position, `positions` of them; all loads of a step ahead of its stores.
template <typename V>
__device__ __forceinline__ void copy_tail(const Plane& p, const uint8_t* src, uint8_t* dst, int positions) {
    constexpr int U = 4;
    int rows = positions, n = p.bytes / static_cast<int>(sizeof(V));
    if (p.position == p.bytes) {  // positions in line: one row
        n *= rows;
        rows = 1;
    }
    const int width = rows == 1 ? 256 : 32, lanes = threadIdx.x % width;  // threads along a row
    for (int r = threadIdx.x / width; r < rows; r += 256 / width) {
        const V* s = reinterpret_cast<const V*>(src + r * p.position);
        V* d = reinterpret_cast<V*>(dst + r * p.position);
        for (int e = lanes; e < n; e += U * width) {
            V v[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (e + u * width < n) v[u] = __ldcs(s + e + u * width);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (e + u * width < n) d[e + u * width] = v[u];
        }
    }
}

// Block (row, layer group): copies the row's tail in the layers blockIdx.y, blockIdx.y + gridDim.y, ...;
// the first group's block writes the row's table entries. Bound by the bytes read and written (256 rows of 23 positions,
// 512 + 32 wide, in 24 layers: 40 us, 6.2 TB/s), and for few rows by the chain parent, its length, its page, the copy.
static __global__ void __launch_bounds__(256) reorder_kernel(const __grid_constant__ Reorder a) {
    MM_PDL_ENTRY();
    const int row = blockIdx.x, tid = threadIdx.x;
    const Move m = move_of(a, row);
    if (blockIdx.y == 0) {
        const int length = length_of(a, row), own = length / a.page;  // (a row that fills its table has no page of its own left)
        // The page that the row begins, or lays aside unwritten: its own, but for a row that took over one shorter by a page
        // or more, whose entries up to its old length are pages that others may have, the last of them its spare one.
        const int begun = m.swap ? (length % a.page ? a.table.columns : own) : m.length % a.page ? a.table.columns : m.full;
        int kept = -1;
        if (begun < a.table.columns) {
            const int page = a.table.entry[row * a.table.stride + begun];
            if (!__syncthreads_or(page == a.spare[row] || shared_at(a, row, begun, tid, blockDim.x))) kept = page;
        }
        for (int j = tid; j < a.table.columns; j += blockDim.x) {
            int page = a.table.entry[(j < m.full ? m.parent : row) * a.table.stride + j];
            if (j == m.full && m.swap) page = m.to;
            else if (j == m.full && j == begun) page = kept;
            else if (j > m.full && m.swap && (page == m.to || (j < own && shared_at(a, row, j, 0, 1)))) page = -1;
            a.out_table[static_cast<long long>(row) * a.table.columns + j] = page;
        }
        if (tid == 0) {
            a.out_spare[row] = !m.swap ? a.spare[row] : own >= a.table.columns ? -1 : own == begun ? kept : a.table.entry[row * a.table.stride + own];
            a.out_lengths[row] = m.length;
        }
    }
    if (m.part == 0 || m.from < 0 || m.from >= a.pages || m.to < 0 || m.to >= a.pages || m.from == m.to) return;
    for (int l = blockIdx.y; l < a.layers; l += gridDim.y)
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            const Plane& p = a.plane[q];
            if (!p.data) continue;
            const uint8_t* src = p.data + l * p.layer + m.from * p.page;
            uint8_t* dst = p.data + l * p.layer + m.to * p.page;
            if (p.vec == 16) copy_tail<uint4>(p, src, dst, m.part);
            else if (p.vec == 4) copy_tail<uint32_t>(p, src, dst, m.part);
            else copy_tail<uint8_t>(p, src, dst, m.part);
        }
}

}  // namespace paged
}  // namespace mm
