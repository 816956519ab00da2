// The 8-bit latent cache: element types, quantisation of new positions and reading back.
#pragma once
#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"

namespace mm {
namespace lat {

// ------------------------------------------------------------------ element types
template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }

// Two values as one 32-bit register of the 16-bit type (lo in the low half).
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float e4m3_to_f32(uint8_t c) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}
// Two e4m3 codes (low byte first) as two 16-bit values: exact in fp16 and in bf16 (4
// significant bits, exponents -9..8 both hold).
template <typename T> __device__ __forceinline__ uint32_t e4m3x2_to(uint16_t c);
template <> __device__ __forceinline__ uint32_t e4m3x2_to<__half>(uint16_t c) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(c, __NV_E4M3);
    return static_cast<uint32_t>(h.x) | (static_cast<uint32_t>(h.y) << 16);
}
template <> __device__ __forceinline__ uint32_t e4m3x2_to<__nv_bfloat16>(uint16_t c) {
    const __half2 h(__nv_cvt_fp8x2_to_halfraw2(c, __NV_E4M3));
    const float2 f = __half22float2(h);
    return pack2<__nv_bfloat16>(f.x, f.y);
}

constexpr float kE4m3Max = 448.f;
constexpr float kScaleFloor = 7.888609052210118e-31f;  // 2^-100: keeps x / scale finite for tiny rows

// Device view of a latent cache (mm_latent_cache without its host-only fields).
struct CacheView {
    const uint8_t* latent;  // e4m3 codes, or the 16-bit [kv | rope] rows
    const uint8_t* rope;    // 16-bit rope rows (e4m3 caches)
    const float* scale;
    long long row_stride, pos_stride;            // elements
    long long rope_row_stride, rope_pos_stride;
    long long scale_row_stride;
    int rows, positions;
};

struct CacheOut {
    uint8_t* latent;
    uint8_t* rope;
    float* scale;
    long long row_stride, pos_stride, rope_row_stride, rope_pos_stride, scale_row_stride;
    int rows, positions;
};

// ------------------------------------------------------------------ write
// Any width, stride and alignment: one warp per position, the row maximum and then the codes in
// 32-value steps. The widths of the framework's models run on latent_write_vec_kernel.
template <typename T, typename T16>
__global__ void latent_write_kernel(CacheOut c, const T* __restrict__ latent, long long latent_stride,
                                    const T* __restrict__ rope, long long rope_stride, const long long* __restrict__ slots,
                                    long long n, int kv, int rd) {
    MM_PDL_ENTRY();
    const long long i = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (i >= n) return;
    const long long slot = slots[i];
    if (slot < 0 || slot >= static_cast<long long>(c.rows) * c.positions) return;
    const long long row = slot / c.positions, pos = slot - row * c.positions;
    const T* x = latent + i * latent_stride;
    float mx = 0.f;
    for (int k = lane; k < kv; k += 32) mx = fmaxf(mx, fabsf(to_f32(x[k])));
    const float s = fmaxf(__fdiv_rn(warp_max(mx), kE4m3Max), kScaleFloor);
    uint8_t* dst = c.latent + row * c.row_stride + pos * c.pos_stride;
    for (int k = lane; k < kv; k += 32)
        dst[k] = __nv_cvt_float_to_fp8(__fdiv_rn(to_f32(x[k]), s), __NV_SATFINITE, __NV_E4M3);
    if (lane == 0) c.scale[row * c.scale_row_stride + pos] = s;
    T16* rdst = reinterpret_cast<T16*>(c.rope) + row * c.rope_row_stride + pos * c.rope_pos_stride;
    for (int k = lane; k < rd; k += 32) rdst[k] = from_f32<T16>(to_f32(rope[i * rope_stride + k]));
}

template <typename T> __device__ __forceinline__ void store16(T* __restrict__ p, const float (&v)[16]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            reinterpret_cast<float4*>(p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            reinterpret_cast<uint4*>(p)[i] =
                make_uint4(pack2<T>(v[8 * i], v[8 * i + 1]), pack2<T>(v[8 * i + 2], v[8 * i + 3]),
                           pack2<T>(v[8 * i + 4], v[8 * i + 5]), pack2<T>(v[8 * i + 6], v[8 * i + 7]));
    }
}
// Eight values of one type to eight of a 16-bit one.
template <typename T, typename T16> __device__ __forceinline__ uint4 rope8(const uint4 (&r)[sizeof(T) / 2]) {
    if constexpr (std::is_same<T, T16>::value) {
        return r[0];
    } else {
        const T* t = reinterpret_cast<const T*>(r);
        return make_uint4(pack2<T16>(to_f32(t[0]), to_f32(t[1])), pack2<T16>(to_f32(t[2]), to_f32(t[3])),
                          pack2<T16>(to_f32(t[4]), to_f32(t[5])), pack2<T16>(to_f32(t[6]), to_f32(t[7])));
    }
}

// The e4m3 codes of v[i] / s (IEEE quotients), 16 of them. The product with the reciprocal is
// within 2 ulp of the quotient, and rounding is monotonic: where the products with a reciprocal
// 2^-21 lower and higher round to the same code, so does the quotient. A lane in which they differ
// anywhere (a quotient that close to the middle of two codes) divides.
template <typename T> __device__ __forceinline__ uint4 e4m3_quotients(const uint4 (&x)[sizeof(T)], float s) {
    float v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = to_f32(reinterpret_cast<const T*>(x)[e]);
    const float inv = __frcp_rn(s), below = inv * (1.f - 4.76837158e-7f), above = inv * (1.f + 4.76837158e-7f);
    auto codes4 = [](float a, float b, float c, float d) {
        return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3)) |
               (static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3)) << 16);
    };
    uint32_t w[4], differ = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        w[e] = codes4(v[4 * e] * below, v[4 * e + 1] * below, v[4 * e + 2] * below, v[4 * e + 3] * below);
        differ |= w[e] ^ codes4(v[4 * e] * above, v[4 * e + 1] * above, v[4 * e + 2] * above, v[4 * e + 3] * above);
    }
    if (differ) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            w[e] = codes4(__fdiv_rn(v[4 * e], s), __fdiv_rn(v[4 * e + 1], s), __fdiv_rn(v[4 * e + 2], s), __fdiv_rn(v[4 * e + 3], s));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Slot -> (row, position); 32-bit division where the cache has fewer than 2^31 positions.
__device__ __forceinline__ void split_slot(long long slot, long long total, int positions, long long& row, long long& pos) {
    if (total <= 0x7fffffffLL) {
        const uint32_t r = static_cast<uint32_t>(slot) / static_cast<uint32_t>(positions);
        row = r;
        pos = static_cast<uint32_t>(slot) - r * static_cast<uint32_t>(positions);
    } else {
        row = slot / positions;
        pos = slot - row * positions;
    }
}

// The largest magnitude of 16 values held as uint4s of T (NaN is passed over).
template <typename T> __device__ __forceinline__ float amax16(const uint4 (&x)[sizeof(T)]) {
    float mx = 0.f;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 f = *reinterpret_cast<const float4*>(&x[i]);
            mx = fmaxf(fmaxf(mx, fmaxf(fabsf(f.x), fabsf(f.y))), fmaxf(fabsf(f.z), fabsf(f.w)));
        }
    } else {
        using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
        const T2* t = reinterpret_cast<const T2*>(x);
        T2 m = __habs2(t[0]);
#pragma unroll
        for (int i = 1; i < 8; ++i) m = __hmax2(m, __habs2(t[i]));
        const T* e = reinterpret_cast<const T*>(&m);
        mx = fmaxf(fmaxf(mx, to_f32(e[0])), to_f32(e[1]));
    }
    return mx;
}

// A lane's share of a position to write, as it was loaded.
template <typename T> struct WriteRow {
    uint4 x[sizeof(T)], r[sizeof(T) / 2];
    long long slot;
};

// KV = 128 or 512, 16-byte accesses: a lane takes 16 values of a position (KV / 16 lanes each), the
// maximum is a shuffle reduction over the lane group. The CTAs that fit walk the positions with the
// next ones already loaded, as they are (14 registers for 16-bit rows). Bound by the bytes in and out
// that so few positions ahead keep in flight: 196,608 x (512 + 32) fp16 values, 330 MB in 67 us back to back
// (4.9 TB/s), to random slots and to neighbouring ones alike, 70 among other work (a CTA per eight positions
// 79.9; two positions ahead, or five and six CTAs an SM, 77 to 97: spills or fewer CTAs); 50,001 fp32 rows
// 24.4 us (5.6 TB/s).
template <typename T> constexpr int kWriteCtas = sizeof(T) == 4 ? 3 : 4;  // CTAs per SM
template <typename T, typename T16, int KV, int R>
__global__ void __launch_bounds__(256, kWriteCtas<T>) latent_write_vec_kernel(
    CacheOut c, const T* __restrict__ latent, long long latent_stride, const T* __restrict__ rope, long long rope_stride,
    const long long* __restrict__ slots, long long n) {
    MM_PDL_ENTRY();
    constexpr int L = KV / 16, P = 32 / L;  // lanes per position, positions side by side in a warp
    const int lane = threadIdx.x & 31, sub = lane % L;
    const long long step = static_cast<long long>(gridDim.x) * 8 * P, total = static_cast<long long>(c.rows) * c.positions;
    auto fetch = [&](long long i) {
        WriteRow<T> w;
        w.slot = -1;
        if (i < n) {
            w.slot = slots[i];
            const uint4* x = reinterpret_cast<const uint4*>(latent + i * latent_stride + sub * 16);
#pragma unroll
            for (int e = 0; e < static_cast<int>(sizeof(T)); ++e) w.x[e] = __ldcs(x + e);
            if (sub < R / 8) {
                const uint4* r = reinterpret_cast<const uint4*>(rope + i * rope_stride + sub * 8);
#pragma unroll
                for (int e = 0; e < static_cast<int>(sizeof(T)) / 2; ++e) w.r[e] = __ldcs(r + e);
            }
        } else {
#pragma unroll
            for (int e = 0; e < static_cast<int>(sizeof(T)); ++e) w.x[e] = make_uint4(0, 0, 0, 0);
        }
        return w;
    };
    // whole warps walk together (the reduction's shuffles); lane groups past n hold nothing
    long long i0 = (static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5)) * P;
    const int mine = lane / L;
    WriteRow<T> next = fetch(i0 + mine);
    for (; i0 < n; i0 += step) {
        const WriteRow<T> w = next;
        next = fetch(i0 + mine + step);
        float mx = amax16<T>(w.x);
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float s = fmaxf(__fdiv_rn(mx, kE4m3Max), kScaleFloor);
        const uint4 codes = e4m3_quotients<T>(w.x, s);
        if (w.slot < 0 || w.slot >= total) continue;
        long long row, pos;
        split_slot(w.slot, total, c.positions, row, pos);
        *reinterpret_cast<uint4*>(c.latent + row * c.row_stride + pos * c.pos_stride + sub * 16) = codes;
        if (sub < R / 8)
            *reinterpret_cast<uint4*>(c.rope + 2 * (row * c.rope_row_stride + pos * c.rope_pos_stride) + sub * 16) =
                rope8<T, T16>(w.r);
        if (sub == 0) c.scale[row * c.scale_row_stride + pos] = s;
    }
}

// ------------------------------------------------------------------ read
// KV = 128 or 512, 16-byte accesses: 16 codes of a position per lane, U positions per lane
// group with all loads first. Bound by the bytes in and out: 131,072 scattered positions, 512 + 32 wide,
// to bf16 rows, 220 MB in 41 us (5.3 TB/s).
template <typename T16, typename TO, int KV, int R, int U>
__global__ void __launch_bounds__(256) latent_read_vec_kernel(CacheView c, const long long* __restrict__ slots, long long n,
                                                              TO* __restrict__ out, long long out_stride) {
    MM_PDL_ENTRY();
    constexpr int L = KV / 16, P = 32 / L;
    const int lane = threadIdx.x & 31, sub = lane % L;
    const long long first = ((static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5)) * U) * P + lane / L;
    const long long total = static_cast<long long>(c.rows) * c.positions;
    uint4 code[U], rv[U];
    float s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long i = first + u * P, slot = i < n ? slots[i] : -1;
        code[u] = rv[u] = make_uint4(0, 0, 0, 0);
        s[u] = 0.f;
        if (slot >= 0 && slot < total) {
            long long row, pos;
            split_slot(slot, total, c.positions, row, pos);
            code[u] = __ldg(reinterpret_cast<const uint4*>(c.latent + row * c.row_stride + pos * c.pos_stride + sub * 16));
            s[u] = __ldg(c.scale + row * c.scale_row_stride + pos);
            if (sub < R / 8)
                rv[u] = __ldg(reinterpret_cast<const uint4*>(c.rope + 2 * (row * c.rope_row_stride + pos * c.rope_pos_stride) + sub * 16));
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long i = first + u * P;
        if (i >= n) return;
        TO* o = out + i * out_stride;
        float v[16];
        const uint32_t w[4] = {code[u].x, code[u].y, code[u].z, code[u].w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(
                static_cast<__nv_fp8x2_storage_t>(w[e >> 1] >> (16 * (e & 1))), __NV_E4M3)));
            v[2 * e] = f.x * s[u];
            v[2 * e + 1] = f.y * s[u];
        }
        store16(o + sub * 16, v);
        if (sub < R / 8) {
            const T16* t = reinterpret_cast<const T16*>(&rv[u]);
            float q[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) q[e] = to_f32(t[e]);
            if constexpr (sizeof(TO) == 4) {
                reinterpret_cast<float4*>(o + KV + sub * 8)[0] = make_float4(q[0], q[1], q[2], q[3]);
                reinterpret_cast<float4*>(o + KV + sub * 8)[1] = make_float4(q[4], q[5], q[6], q[7]);
            } else {
                *reinterpret_cast<uint4*>(o + KV + sub * 8) =
                    make_uint4(pack2<TO>(q[0], q[1]), pack2<TO>(q[2], q[3]), pack2<TO>(q[4], q[5]), pack2<TO>(q[6], q[7]));
            }
        }
    }
}

// Any width, stride and alignment: one warp per position.
template <typename T16, typename TO>
__global__ void latent_read_kernel(CacheView c, const long long* __restrict__ slots, long long n, TO* __restrict__ out,
                                   long long out_stride, int kv, int rd) {
    MM_PDL_ENTRY();
    const long long i = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (i >= n) return;
    const long long slot = slots[i];
    TO* o = out + i * out_stride;
    if (slot < 0 || slot >= static_cast<long long>(c.rows) * c.positions) {
        for (int k = lane; k < kv + rd; k += 32) o[k] = from_f32<TO>(0.f);
        return;
    }
    const long long row = slot / c.positions, pos = slot - row * c.positions;
    const uint8_t* src = c.latent + row * c.row_stride + pos * c.pos_stride;
    const float s = c.scale[row * c.scale_row_stride + pos];
    for (int k = lane; k < kv; k += 32) o[k] = from_f32<TO>(e4m3_to_f32(src[k]) * s);
    const T16* rsrc = reinterpret_cast<const T16*>(c.rope) + row * c.rope_row_stride + pos * c.rope_pos_stride;
    for (int k = lane; k < rd; k += 32) o[kv + k] = from_f32<TO>(to_f32(rsrc[k]));
}

}  // namespace lat
}  // namespace mm
