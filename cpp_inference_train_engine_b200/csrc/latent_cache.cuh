// The 8-bit latent cache: element types, quantisation of new positions and reading back.
#pragma once
#include <cuda_fp8.h>

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
// One warp per position: the row maximum in one pass held in registers (up to 1024 latent
// values, 32 per lane), the scale, then the codes. Any width, stride and alignment.
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

// ------------------------------------------------------------------ read
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
