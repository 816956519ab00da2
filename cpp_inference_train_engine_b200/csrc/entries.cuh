// What the C entries on device pointers (include/mm_latent.h, mm_paged.h) share: errors, launches,
// argument checks and dispatch on element types.
#pragma once
#include <cudaTypedefs.h>

#include <atomic>
#include <exception>
#include <string>
#include <type_traits>

#include "latent_cache.cuh"

#include "../../include/mm_latent.h"

namespace mm {
namespace entry {

inline thread_local std::string g_error;  // the calling thread's last message

struct Refusal {
    int code;
    const char* what;
};

[[noreturn]] inline void refuse(int code, const char* what) { throw Refusal{code, what}; }
inline void require(bool ok, const char* what) {
    if (!ok) refuse(MM_INVALID_ARGUMENT, what);
}
inline void check(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return;
    g_error = std::string(what) + ": " + cudaGetErrorString(e);
    throw Refusal{e == cudaErrorMemoryAllocation ? MM_OUT_OF_MEMORY : MM_GPU_ERROR, nullptr};
}

// Runs f; failures become 1 + ErrorCode with a message.
template <class F> int guarded(F&& f) {
    try {
        f();
        return MM_OK;
    } catch (const Refusal& r) {
        try {
            if (r.what) g_error = r.what;
        } catch (...) {
        }
        return r.code;
    } catch (...) {
        return MM_OUT_OF_MEMORY;
    }
}

// Launch with programmatic stream serialization (every kernel enters through MM_PDL_ENTRY or
// waits itself before it touches memory). The error is taken from the launch itself.
template <typename... KArgs, typename... Args>
void launch(cudaStream_t s, void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    check(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...), "kernel launch");
}

// cudaFuncSetAttribute(MaxDynamicSharedMemorySize) for a kernel, once per device.
template <auto Kernel> void set_dynamic_smem(int bytes) {
    static std::atomic<unsigned long long> done{0};
    int dev = 0;
    check(cudaGetDevice(&dev), "cudaGetDevice");
    const unsigned long long bit = 1ull << (dev & 63);
    if (dev < 64 && (done.load() & bit)) return;
    check(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "shared memory attribute");
    done.fetch_or(bit);
}

// Whether p is a multiple of n bytes.
inline bool multiple(const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

inline void check_cache(const mm_latent_cache* c) {
    require(c->rows >= 0 && c->positions >= 0, "latent cache: negative size");
    require(c->kv >= 1 && c->kv <= 1024 && c->rope_dim >= 0 && c->rope_dim <= 256,
            "latent cache: kv must be in [1, 1024] and rope_dim in [0, 256]");
    require(c->kind == MM_F16 || c->kind == MM_BF16 || c->kind == MM_E4M3, "latent cache: unknown kind");
    const bool empty = c->rows == 0 || c->positions == 0;
    require(c->latent || empty, "latent cache: null storage");
    if (c->kind == MM_E4M3) {
        require(c->rope_kind == MM_F16 || c->rope_kind == MM_BF16, "latent cache: rope must be fp16 or bf16");
        require(empty || (c->scale && (c->rope || c->rope_dim == 0)), "latent cache: null storage");
    }
    require(multiple(c->latent, c->kind == MM_E4M3 ? 1 : 2) && (c->kind != MM_E4M3 || (multiple(c->rope, 2) && multiple(c->scale, 4))),
            "latent cache: storage not aligned to its elements");
}

inline lat::CacheView view(const mm_latent_cache* c) {
    lat::CacheView v{};
    if (!c) return v;
    v.latent = static_cast<const uint8_t*>(c->latent);
    v.rope = static_cast<const uint8_t*>(c->rope);
    v.scale = c->scale;
    v.row_stride = c->row_stride;
    v.pos_stride = c->pos_stride;
    v.rope_row_stride = c->rope_row_stride;
    v.rope_pos_stride = c->rope_pos_stride;
    v.scale_row_stride = c->scale_row_stride;
    v.rows = c->rows;
    v.positions = c->positions;
    return v;
}

constexpr long long kMaxBlocks = 2147483647LL;

inline unsigned blocks(long long n, int per) {
    const long long b = (n + per - 1) / per;
    if (b > kMaxBlocks) refuse(MM_UNSUPPORTED, "too many rows for one launch");
    return static_cast<unsigned>(b);
}

// Calls f(std::type_identity-like tag) for a 16-bit or 32-bit element type.
template <typename T> struct Tag {
    using type = T;
};
template <class F> void with_type(int dtype, F&& f) {
    if (dtype == MM_F16) f(Tag<__half>{});
    else if (dtype == MM_BF16) f(Tag<__nv_bfloat16>{});
    else if (dtype == MM_F32) f(Tag<float>{});
    else refuse(MM_INVALID_ARGUMENT, "unsupported element type");
}
template <class F> void with_half(int dtype, F&& f) {
    if (dtype == MM_F16) f(Tag<__half>{});
    else if (dtype == MM_BF16) f(Tag<__nv_bfloat16>{});
    else refuse(MM_INVALID_ARGUMENT, "unsupported element type");
}

// Whether the rows of an e4m3 cache can be accessed 16 bytes at a time.
inline bool aligned_e4m3(const mm_latent_cache* c) {
    auto ok = [](const void* p, long long a, long long b, int size) {
        return reinterpret_cast<uintptr_t>(p) % 16 == 0 && a * size % 16 == 0 && b * size % 16 == 0;
    };
    return ok(c->latent, c->row_stride, c->pos_stride, 1) && ok(c->rope, c->rope_row_stride, c->rope_pos_stride, 2);
}

inline int sm_count() {
    static std::atomic<int> count{0};
    int n = count.load();
    if (!n) {
        int dev = 0;
        check(cudaGetDevice(&dev), "cudaGetDevice");
        check(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev), "multiprocessor count");
        count.store(n);
    }
    return n;
}

inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
    static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> fn{nullptr};
    PFN_cuTensorMapEncodeTiled_v12000 f = fn.load();
    if (!f) {
        cudaDriverEntryPointQueryResult found;
        void* p = nullptr;
        check(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found), "cuTensorMapEncodeTiled");
        if (found != cudaDriverEntryPointSuccess || !p) refuse(MM_GPU_ERROR, "cuTensorMapEncodeTiled unavailable");
        f = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
        fn.store(f);
    }
    return f;
}

}  // namespace entry
}  // namespace mm
