// Paged latent attention for [128 latent | 16 rope] and [512 latent | 32 rope] caches: tiles of 32 positions by
// TMA through the page table, products by mma.sync.
//
// One query token per row is 8 or 16 heads against every position: 15 to 31 flops a byte, far below what the
// tensor cores need to be the bound, so the kernel is built to keep loads in flight. A CTA takes 16 query rows
// (heads of one row) over a run of the row's tiles. Heads are the M = 16 side of both products, S = Q K^T and
// O += P V with V = K's latent columns, so P's accumulator layout is its operand layout and nothing but
// scores crosses threads. Warps:
//   products   4. Each owns 128 latent columns of the tiles it reads, in both products: its share of Q and
//              its O [16 x 128] stay in registers, and it alone reads (and clears) those columns. 512 wide: the
//              four take a tile together and add their shares of S through shared memory; 128 wide: each has
//              tiles of its own (every fourth) and the four results are joined at the row's end.
//   loads      1, which walks the same runs ahead of them: page numbers 32 boxes at a time, a box a lane.
// Positions that a row does not see are masked in S and cleared in the tile (a probability of zero times a NaN
// would be one). Two CTAs an SM, each with a ring of its own; the row's sums and maxima are fp32, the weights of
// the second product are rounded to 16 bits once, as its operand has to be.
//
// The tiles of all rows, in line, are divided evenly over the CTAs (a row costs kRowCost tiles more); a row
// that is cut leaves partial results to the join kernel.
#pragma once
#include <type_traits>

#include "paged_attention.cuh"

namespace mm {
namespace paged {

struct MmaArgs {
    Attention p;
    int box;           // positions per TMA box: 32, or 16 where pages are not a multiple of 32
    int blocks;        // blocks of 16 heads per row
    int shares;        // even shares of all tiles (else a CTA takes whole rows in turn)
    int by_unit;       // the cut list is indexed by unit (no more units than CTAs), else by CTA
    float* part_o;     // [2 CTAs][16][kv], unnormalised
    float2* part_ml;   // [2 CTAs][16] maximum and sum, base 2
    int4* cut;         // (unit, parts, first CTA): a unit cut at the end of the share it begins in; no parts: none
};

constexpr int kTile = 32;       // positions
constexpr int kRowCost = 2;     // tiles that a row's queries and results cost
constexpr int kMinShare = 6;    // tiles of a CTA at least
constexpr int kMmaThreads = 160;
constexpr float kNone = -3.402823466e38f;  // maximum of nothing (finite: its exp2 is 0, never NaN)

template <int KV, int R, bool Q8> struct MmaCfg {
    static constexpr int CW = KV / 128;      // warps that share a tile
    static constexpr int KG = 4 / CW;        // groups with tiles of their own
    static constexpr int kBoxes = Q8 ? KV / 128 : KV / 64;  // latent boxes of 128-byte rows
    static constexpr int kLatent = kBoxes * kTile * 128;
    static constexpr int kRope = kTile * R * 2;
    static constexpr int kScale = Q8 ? 256 : 0;             // two boxes of 16 at 128-byte addresses
    static constexpr int kSlot = (kLatent + kRope + kScale + 1023) / 1024 * 1024;
    static constexpr int kBytes = kLatent + kRope + (Q8 ? kTile * 4 : 0);  // that TMA brings
    static constexpr int SG = KV == 512 ? (Q8 ? 5 : 3) : (Q8 ? 3 : 2);     // slots of a group
    static constexpr int SLOTS = KG * SG;
    // 512: the four shares of S; 128: the four results of a row
    static constexpr int kShare = KV == 512 ? 4 * 16 * kTile * 4 : 4 * 16 * 128 * 4;
    static constexpr int oShare = SLOTS * kSlot;
    static constexpr int oStat = oShare + kShare;           // [4][16] maxima and sums (128 wide)
    static constexpr int oBar = oStat + 4 * 16 * 8;
    static constexpr int oMeta = oBar + 2 * SLOTS * 8;
    static constexpr int oPlan = (oMeta + SLOTS * 4 + 15) / 16 * 16;
    static constexpr int kSmem = oPlan + 64 + 1024;         // + alignment of the base
    static_assert(oBar % 8 == 0 && oStat % 8 == 0 && oShare % 1024 == 0 && kSlot % 1024 == 0, "alignment");
    static_assert(2 * (kSmem + 1024) <= 228 * 1024, "two CTAs an SM");
};

// What a CTA does next: tiles [from, to) of a unit (16 heads of a row). Tile i stands at position 32 i below
// `sinks` tiles, behind them `skip` tiles further.
struct Run {
    int row, block, unit, len, n, sinks, skip, from, to, part;  // part: slot of partial results, -1: the whole unit
    __device__ __forceinline__ int position(int i) const { return kTile * (i < sinks ? i : i + skip); }
};

// Tiles of row b: those with one of the first `sinks` positions, then those from the window's on.
__device__ __forceinline__ int row_tiles(const Attention& p, int len, int& sink_tiles, int& skip) {
    const int start = window_start(p, len), all = (len + kTile - 1) / kTile;
    sink_tiles = (min(p.sinks, start) + kTile - 1) / kTile;
    const int first = max(start / kTile, sink_tiles);
    skip = first - sink_tiles;
    return all - skip;
}

// The runs of a CTA, the same in every warp.
struct Runs {
    const MmaArgs& a;
    long long w0, w1, span, before;  // the share, and the weight ahead of row `row`
    int row, block, len;
    __device__ __forceinline__ Runs(const MmaArgs& args, long long span_, int row0, long long before0) : a(args), span(span_) {
        if (a.shares) {
            w0 = static_cast<long long>(blockIdx.x) * span;
            w1 = w0 + span;
            row = row0;
            before = before0;
            block = 0;
        } else {
            row = static_cast<int>(blockIdx.x) / a.blocks;
            block = static_cast<int>(blockIdx.x) - row * a.blocks;
        }
        len = row < a.p.B ? length_of(a.p, row) : 0;
    }
    __device__ __forceinline__ bool next(Run& r) {
        while (row < a.p.B) {
            r.row = row;
            r.block = block;
            r.len = len;
            r.unit = row * a.blocks + block;
            r.n = row_tiles(a.p, len, r.sinks, r.skip);
            if (!a.shares) {
                r.from = 0;
                r.to = r.n;
                r.part = -1;
                const int u = r.unit + static_cast<int>(gridDim.x);
                row = u / a.blocks;
                block = u - row * a.blocks;
                if (row < a.p.B) len = length_of(a.p, row);
                return true;
            }
            const long long weight = r.n + kRowCost, at = before + block * weight;
            if (at >= w1) return false;
            r.from = static_cast<int>(min(max(w0 - at, 0LL), static_cast<long long>(r.n)));
            r.to = static_cast<int>(min(w1 - at, static_cast<long long>(r.n)));
            const bool begins = at >= w0;
            r.part = begins && r.to == r.n ? -1 : 2 * static_cast<int>(blockIdx.x) + (begins ? 1 : 0);
            if (++block == a.blocks) {
                block = 0;
                before += a.blocks * weight;
                if (++row < a.p.B) len = length_of(a.p, row);
            }
            if (begins || r.from < r.to) return true;
        }
        return false;
    }
    // Parts of a unit that begins here and does not end here.
    __device__ __forceinline__ int parts(const Run& r) const {
        // its first tile's weight is w1 - to, so its last tile lies this many shares further
        return static_cast<int>((w1 - r.to + r.n - 1) / span) - static_cast<int>(blockIdx.x) + 1;
    }
};

__device__ __forceinline__ void tma_load_box(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <typename T> __device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Byte offset of 16-byte chunk c of row r in a box of 128-, 64- or 32-byte rows, as TMA swizzles it.
__device__ __forceinline__ uint32_t swizzled(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }
template <int R> __device__ __forceinline__ uint32_t swizzled_rope(int r, int c) {
    return R == 32 ? r * 64 + ((c ^ ((r >> 1) & 3)) << 4) : r * 32 + ((c ^ ((r >> 2) & 1)) << 4);
}
__device__ __forceinline__ uint32_t codes2(uint32_t two) {  // two e4m3 codes as two fp16 values (exact)
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xffff), __NV_E4M3);
    return static_cast<uint32_t>(h.x) | (static_cast<uint32_t>(h.y) << 16);
}
__device__ __forceinline__ void products_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
// floor(log2 |s|) of a key's scale, kept within what fp32 probabilities take: below 2^-40 a value is less than
// any 16-bit result can show beside others.
__device__ __forceinline__ float exponent_of(float s) {
    return static_cast<float>(min(max(static_cast<int>((__float_as_uint(s) >> 23) & 255) - 127, -40), 100));
}

template <int KV, int R, typename T, bool Q8>
__global__ void __launch_bounds__(kMmaThreads, 2)
    paged_mma_kernel(const __grid_constant__ MmaArgs a, const __grid_constant__ CUtensorMap map_latent,
                     const __grid_constant__ CUtensorMap map_rope, const __grid_constant__ CUtensorMap map_scale) {
    using C = MmaCfg<KV, R, Q8>;
    using TP = std::conditional_t<Q8, __half, T>;  // the second product's type (codes are exact in fp16)
    constexpr float kLift = std::is_same<TP, __half>::value ? 10.f : 0.f;  // log2 of the largest weight: small ones stay normal
    extern __shared__ uint8_t mma_smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(mma_smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::oBar);
    uint64_t* empty = full + C::SLOTS;
    volatile uint32_t* meta = reinterpret_cast<volatile uint32_t*>(smem + C::oMeta);
    long long* plan = reinterpret_cast<long long*>(smem + C::oPlan);  // span, before, row; then a flag
    volatile int* bad = reinterpret_cast<volatile int*>(smem + C::oPlan + 24);
    const Attention& p = a.p;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < C::SLOTS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], C::CW);
        }
        fence_mbar_init();
        *bad = 0;
    }
    if (warp == 4 && lane == 0) {
        prefetch_tmap(&map_latent);
        prefetch_tmap(&map_rope);
        if (Q8) prefetch_tmap(&map_scale);
    }
    MM_PDL_ENTRY();
    if (a.shares) {
        // the weight of all rows, and the row that this CTA's share begins in
        long long* sums = reinterpret_cast<long long*>(smem);  // free until the first tile
        const int per = (p.B + kMmaThreads - 1) / kMmaThreads, b0 = tid * per, b1 = min(b0 + per, p.B);
        auto weight = [&](int b) {
            int st, skip;
            return static_cast<long long>(row_tiles(p, length_of(p, b), st, skip) + kRowCost) * a.blocks;
        };
        long long mine = 0;
        for (int b = b0; b < b1; ++b) mine += weight(b);
        sums[tid] = mine;
        __syncthreads();
        long long ahead = 0, total = 0;
        for (int i = 0; i < kMmaThreads; ++i) {
            const long long s = sums[i];
            ahead += i < tid ? s : 0;
            total += s;
        }
        const long long span = max((total + gridDim.x - 1) / gridDim.x, static_cast<long long>(kMinShare));
        const long long w0 = static_cast<long long>(blockIdx.x) * span;
        if (tid == 0) {
            plan[0] = span;
            if (w0 >= total) plan[2] = p.B;
        }
        if (w0 >= ahead && w0 < ahead + mine) {
            int b = b0;
            for (long long w; ahead + (w = weight(b)) <= w0; ++b) ahead += w;
            plan[1] = ahead;
            plan[2] = b;
        }
        if (!a.by_unit && tid == 0) a.cut[blockIdx.x] = make_int4(0, 0, 0, 0);
        fence_proxy_async_smem();  // `sums`, before a tile lands there
    }
    __syncthreads();
    Runs runs(a, a.shares ? plan[0] : 0, static_cast<int>(a.shares ? plan[2] : 0), a.shares ? plan[1] : 0);
    Run run;
    bool ok = true;
    // a wait that ran out is recorded once; later waits of this thread are skipped
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (ok && !mbar_wait_bounded(bar, parity, &paged_status)) {
            ok = false;
            *bad = 1;
        }
    };

    if (warp == 4) {
        // ------------------------------------------------------------ loads
        int slot[C::KG];  // position in each group's ring
        uint32_t phase = 0;  // bit g: parity of group g's round
#pragma unroll
        for (int g = 0; g < C::KG; ++g) slot[g] = 0;
        const int per = kTile / a.box, page = p.pool.positions;
        const int each = C::kBoxes + 1 + (Q8 ? 1 : 0);  // boxes of one stretch of `box` positions
        // this lane's boxes of a tile: which stretch, which box of it (at most 18 of them)
        const int stretch = lane / each, which = lane - stretch * each;
        while (runs.next(run)) {
            if (lane == 0 && a.shares && run.from == 0) {
                const int parts = run.part < 0 ? 0 : runs.parts(run);
                if (a.by_unit || parts) a.cut[a.by_unit ? run.unit : blockIdx.x] = make_int4(run.unit, parts, blockIdx.x, 0);
            }
            // lane l holds the page of stretch l of the 32 from `base` on, and of the next 32
            auto pages_from = [&](int s) {
                const int i = run.from + (s + lane) / per;
                if (i >= run.to) return -1;
                const int at = run.position(i) + (s + lane) % per * a.box;
                if (at >= run.len) return -1;
                const int id = __ldg(p.table.entry + run.row * p.table.stride + at / page);
                return id >= 0 && id < p.pool.rows ? id : -1;
            };
            int base = 0, ids = pages_from(0), ids_next = pages_from(32);
            for (int i = run.from; i < run.to; ++i) {
                const int g = C::KG == 1 ? 0 : (i - run.from) % C::KG;
                int s_of = 0;
#pragma unroll
                for (int x = 0; x < C::KG; ++x) s_of = x == g ? slot[x] : s_of;
                const int s = g * C::SG + s_of;
                const int first = (i - run.from) * per;
                if (first - base == 32) {
                    base = first;
                    ids = ids_next;
                    ids_next = pages_from(base + 32);
                }
                const int id0 = __shfl_sync(0xffffffffu, ids, first - base), id1 = __shfl_sync(0xffffffffu, ids, first - base + per - 1);
                const int id = stretch == 0 ? id0 : id1;
                wait(&empty[s], ((phase >> g) & 1) ^ 1);
                if (__any_sync(0xffffffffu, !ok)) break;
                if (lane == 0) {
                    meta[s] = (id0 >= 0 ? 0xffffu : 0u) | (id1 >= 0 ? 0xffff0000u : 0u);
                    mbar_arrive_expect_tx(&full[s], C::kBytes);
                }
                __syncwarp();
                if (stretch < per) {
                    // a page outside the pool (or behind the row) is asked for behind the last one: zeros
                    const int at = (run.position(i) + stretch * a.box) % page, z = id >= 0 ? id : p.pool.rows;
                    uint8_t* dst = smem + s * C::kSlot;
                    if (which < C::kBoxes)
                        tma_load_box(dst + which * kTile * 128 + stretch * a.box * 128, &map_latent, &full[s], which * (Q8 ? 128 : 64), at, z);
                    else if (which == C::kBoxes)
                        tma_load_box(dst + C::kLatent + stretch * a.box * R * 2, &map_rope, &full[s], Q8 ? 0 : KV, at, z);
                    else
                        tma_load_2d(dst + C::kLatent + C::kRope + stretch * 128, &map_scale, &full[s], at, z);
                }
#pragma unroll
                for (int x = 0; x < C::KG; ++x)
                    if (x == g && ++slot[x] == C::SG) {
                        slot[x] = 0;
                        phase ^= 1u << x;
                    }
            }
            if (!ok) break;
        }
    } else {
        // ------------------------------------------------------------ products
        const int cw = warp % C::CW, group = warp / C::CW;
        const int g = lane >> 2, t4 = lane & 3;  // row of the fragments, place in its quad
        const uint32_t ring = smem_u32(smem) + group * C::SG * C::kSlot;
        // this lane's rows of the matrices that ldmatrix reads
        const int mrow = lane & 7, msel = lane >> 3;
        float* share = reinterpret_cast<float*>(smem + C::oShare);
        const float cs = p.scale * 1.4426950408889634f;
        int slot = 0;
        uint32_t phase = 0;
        while (runs.next(run)) {
            const int h0 = run.block * 16;
            const int heads = min(16, p.H - h0);
            uint32_t q[8][4], qr[4];
            float qf[2] = {1.f, 1.f};  // what the scores of codes are multiplied by (bf16 queries as fp16)
            {
                const T* base = static_cast<const T*>(p.q) + run.row * p.q_row + h0 * p.q_head;
                const T* lo = base + min(g, heads - 1) * p.q_head;
                const T* hi = base + min(g + 8, heads - 1) * p.q_head;
                if constexpr (!Q8) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int c = cw * 128 + k * 16 + t4 * 2;
                        q[k][0] = __ldg(reinterpret_cast<const uint32_t*>(lo + c));
                        q[k][1] = __ldg(reinterpret_cast<const uint32_t*>(hi + c));
                        q[k][2] = __ldg(reinterpret_cast<const uint32_t*>(lo + c + 8));
                        q[k][3] = __ldg(reinterpret_cast<const uint32_t*>(hi + c + 8));
                    }
                } else {
                    // ldmatrix gives a lane four neighbouring codes of a position: the product's k order is
                    // permuted to match
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int c = cw * 128 + k * 16 + t4 * 4;
                        const uint2 x = __ldg(reinterpret_cast<const uint2*>(lo + c)), y = __ldg(reinterpret_cast<const uint2*>(hi + c));
                        q[k][0] = x.x;
                        q[k][1] = y.x;
                        q[k][2] = x.y;
                        q[k][3] = y.y;
                    }
                    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                        // to fp16 with the row's largest value of these columns at 2^8: what falls out of the normal
                        // range is below 2^-22 of it
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float mx = 0.f;
#pragma unroll
                            for (int k = 0; k < 8; ++k)
#pragma unroll
                                for (int e = h; e < 4; e += 2) {
                                    const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&q[k][e]);
                                    mx = fmaxf(mx, fmaxf(fabsf(__low2float(v)), fabsf(__high2float(v))));
                                }
                            mx = quad_max(mx);
                            int e2 = static_cast<int>(__float_as_uint(mx) >> 23) - 127;
                            e2 = e2 > 127 ? 8 : min(max(e2, -110), 118);
                            const float up = __uint_as_float(static_cast<uint32_t>(8 - e2 + 127) << 23);
                            qf[h] = __uint_as_float(static_cast<uint32_t>(e2 - 8 + 127) << 23);
#pragma unroll
                            for (int k = 0; k < 8; ++k)
#pragma unroll
                                for (int e = h; e < 4; e += 2) {
                                    const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&q[k][e]);
                                    q[k][e] = lat::pack2<__half>(__low2float(v) * up, __high2float(v) * up);
                                }
                        }
                    }
                }
                if (cw < R / 16) {
                    const int c = KV + cw * 16 + t4 * 2;
                    qr[0] = __ldg(reinterpret_cast<const uint32_t*>(lo + c));
                    qr[1] = __ldg(reinterpret_cast<const uint32_t*>(hi + c));
                    qr[2] = __ldg(reinterpret_cast<const uint32_t*>(lo + c + 8));
                    qr[3] = __ldg(reinterpret_cast<const uint32_t*>(hi + c + 8));
                }
            }
            float o[16][4];
#pragma unroll
            for (int n = 0; n < 16; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
            float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
            const int start = window_start(p, run.len), sinks = min(p.sinks, start);
            for (int i = run.from + group; i < run.to; i += C::KG) {
                const uint32_t sp = ring + slot * C::kSlot;
                wait(&full[group * C::SG + slot], phase);
                // positions of the tile that the row sees
                uint32_t seen = meta[group * C::SG + slot];
                {
                    const int p0 = run.position(i);
                    auto below = [&](int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; };
                    seen &= below(run.len - p0) & (below(sinks - p0) | ~below(start - p0));
                }
                // ---- S
                float s[4][4];
#pragma unroll
                for (int n = 0; n < 4; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
                if constexpr (!Q8) {
                    const uint32_t box = sp + cw * 2 * (kTile * 128);
#pragma unroll
                    for (int k = 0; k < 8; ++k)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            uint32_t b[4];
                            ldsm4(b, box + (k >> 2) * (kTile * 128) + swizzled(h * 16 + (msel >> 1) * 8 + mrow, (k & 3) * 2 + (msel & 1)));
                            mma16<T>(s[2 * h], q[k], b[0], b[1]);
                            mma16<T>(s[2 * h + 1], q[k], b[2], b[3]);
                        }
                } else {
                    const uint32_t box = sp + cw * (kTile * 128);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        uint32_t b[4];
                        ldsm4(b, box + swizzled(msel * 8 + mrow, k));
#pragma unroll
                        for (int n = 0; n < 4; ++n) mma16<__half>(s[n], q[k], codes2(b[n]), codes2(b[n] >> 16));
                    }
                }
                float ks[8];  // scales of the lane's positions: 8 n + 2 t4 + e
                if constexpr (Q8) {
                    const float* sc = reinterpret_cast<const float*>(smem + (group * C::SG + slot) * C::kSlot + C::kLatent + C::kRope);
                    const int gap = a.box == 16 ? 16 : 0;  // a second box of 16 starts 128 bytes on
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const float2 v = *reinterpret_cast<const float2*>(sc + n * 8 + t4 * 2 + (n >= 2 ? gap : 0));
                        ks[2 * n] = v.x;
                        ks[2 * n + 1] = v.y;
                        s[n][0] *= qf[0] * v.x;
                        s[n][1] *= qf[0] * v.y;
                        s[n][2] *= qf[1] * v.x;
                        s[n][3] *= qf[1] * v.y;
                    }
                }
                if (cw < R / 16) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t b[4];
                        ldsm4(b, sp + C::kLatent + swizzled_rope<R>(h * 16 + (msel >> 1) * 8 + mrow, cw * 2 + (msel & 1)));
                        mma16<T>(s[2 * h], qr, b[0], b[1]);
                        mma16<T>(s[2 * h + 1], qr, b[2], b[3]);
                    }
                }
                if constexpr (C::CW > 1) {
                    // the four warps' shares, added in the same order by each
                    float4* mine = reinterpret_cast<float4*>(share) + cw * 128 + lane;
#pragma unroll
                    for (int n = 0; n < 4; ++n) mine[n * 32] = make_float4(s[n][0], s[n][1], s[n][2], s[n][3]);
                    products_sync();
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const float4* v = reinterpret_cast<const float4*>(share) + n * 32 + lane;
                        const float4 x = v[0], y = v[128], z = v[256], w = v[384];
                        s[n][0] = (x.x + y.x) + (z.x + w.x);
                        s[n][1] = (x.y + y.y) + (z.y + w.y);
                        s[n][2] = (x.z + y.z) + (z.z + w.z);
                        s[n][3] = (x.w + y.w) + (z.w + w.w);
                    }
                    products_sync();
                }
                // ---- softmax
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[n][e] *= cs;
                        const int key = n * 8 + t4 * 2 + (e & 1);
                        if (seen != ~0u && !((seen >> key) & 1)) s[n][e] = -INFINITY;
                        top[e >> 1] = fmaxf(top[e >> 1], Q8 ? s[n][e] + exponent_of(ks[2 * n + (e & 1)]) : s[n][e]);
                    }
                float corr[2], ref[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float mn = fmaxf(m[h], quad_max(top[h]));
                    const float at = mn == -INFINITY ? 0.f : mn;
                    corr[h] = m[h] == mn ? 1.f : fast_exp2(m[h] - at);
                    m[h] = mn;
                    ref[h] = at - kLift;
                }
                if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
                    for (int n = 0; n < 16; ++n) {
                        o[n][0] *= corr[0];
                        o[n][1] *= corr[0];
                        o[n][2] *= corr[1];
                        o[n][3] *= corr[1];
                    }
                    l[0] *= corr[0];
                    l[1] *= corr[1];
                }
                uint32_t w[2][4];  // the weights as the second product's operand: 16 positions each
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    float e[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        e[x] = fast_exp2(s[n][x] - ref[x >> 1]);
                        l[x >> 1] += e[x];
                        if (Q8) e[x] = seen == ~0u || ((seen >> (n * 8 + t4 * 2 + (x & 1))) & 1) ? e[x] * ks[2 * n + (x & 1)] : 0.f;
                    }
                    w[n >> 1][(n & 1) * 2] = lat::pack2<TP>(e[0], e[1]);
                    w[n >> 1][(n & 1) * 2 + 1] = lat::pack2<TP>(e[2], e[3]);
                }
                // ---- positions that are not seen hold anything
                if (seen != ~0u) {
                    __syncwarp();
                    uint8_t* boxes = smem + (group * C::SG + slot) * C::kSlot + cw * (Q8 ? 1 : 2) * (kTile * 128);
                    for (uint32_t hide = ~seen; hide; hide &= hide - 1) {
                        const int r = __ffs(hide) - 1;
                        if (lane < (Q8 ? 8 : 16))
                            *reinterpret_cast<uint4*>(boxes + (lane >> 3) * (kTile * 128) + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    __syncwarp();
                }
                // ---- O
                if constexpr (!Q8) {
                    const uint32_t box = sp + cw * 2 * (kTile * 128);
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            uint32_t b[4];
                            ldsm4_t(b, box + (c >> 2) * (kTile * 128) + swizzled(k * 16 + (msel & 1) * 8 + mrow, (c & 3) * 2 + (msel >> 1)));
                            mma16<T>(o[2 * c], w[k], b[0], b[1]);
                            mma16<T>(o[2 * c + 1], w[k], b[2], b[3]);
                        }
                } else {
                    // a transposed pair of codes is two neighbouring columns of one position: the even columns of 16
                    // make one tile of the product, the odd ones another
                    const uint32_t box = sp + cw * (kTile * 128);
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            uint32_t b[4];
                            ldsm4_t(b, box + swizzled(k * 16 + (msel & 1) * 8 + mrow, c * 2 + (msel >> 1)));
#pragma unroll
                            for (int x = 0; x < 4; ++x) b[x] = __byte_perm(b[x], 0, 0x3120);
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                mma16<__half>(o[4 * c + 2 * x], w[k], codes2(b[2 * x]), codes2(b[2 * x + 1]));
                                mma16<__half>(o[4 * c + 2 * x + 1], w[k], codes2(b[2 * x] >> 16), codes2(b[2 * x + 1] >> 16));
                            }
                        }
                }
                if (seen != ~0u) fence_proxy_async_smem();  // the cleared rows, before the next tile lands on them
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[group * C::SG + slot]);
                if (++slot == C::SG) {
                    slot = 0;
                    phase ^= 1;
                }
            }
            // ------------------------------------------------------------ results
            l[0] = quad_sum(l[0]);
            l[1] = quad_sum(l[1]);
            if (!ok || *bad) l[0] = l[1] = __int_as_float(0x7fc00000);
            const bool whole = run.part < 0;
            const long long first = static_cast<long long>(run.row) * p.H + h0;  // query row
            // column of o[n][e]: n-tiles of 8 (codes: 16 columns are two tiles, even and odd)
            if constexpr (C::KG == 1) {
                float f[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    f[h] = !whole ? 1.f : l[h] == 0.f ? 0.f : 1.f / l[h];
                    const int row = g + 8 * h;
                    if (cw == 0 && t4 == 0 && row < heads) {
                        if (!whole) a.part_ml[run.part * 16 + row] = make_float2(l[h] == 0.f ? kNone : m[h] - kLift, l[h]);
                        else if (p.lse) p.lse[first + row] = l[h] == 0.f ? -INFINITY : (m[h] - kLift + log2f(l[h])) * 0.6931471805599453f;
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = g + 8 * h;
                    if (row >= heads) continue;
#pragma unroll
                    for (int n = 0; n < 16; n += 2) {
                        if constexpr (!Q8) {
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                const int c = cw * 128 + (n + x) * 8 + t4 * 2;
                                if (whole)
                                    *reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + (first + row) * KV + c) =
                                        lat::pack2<T>(o[n + x][2 * h] * f[h], o[n + x][2 * h + 1] * f[h]);
                                else
                                    *reinterpret_cast<float2*>(a.part_o + (static_cast<long long>(run.part) * 16 + row) * KV + c) =
                                        make_float2(o[n + x][2 * h], o[n + x][2 * h + 1]);
                            }
                        } else {
                            const int c = cw * 128 + n * 8 + t4 * 4;
                            const float4 v = make_float4(o[n][2 * h] * f[h], o[n + 1][2 * h] * f[h], o[n][2 * h + 1] * f[h], o[n + 1][2 * h + 1] * f[h]);
                            if (whole)
                                *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + (first + row) * KV + c) =
                                    make_uint2(lat::pack2<T>(v.x, v.y), lat::pack2<T>(v.z, v.w));
                            else
                                *reinterpret_cast<float4*>(a.part_o + (static_cast<long long>(run.part) * 16 + row) * KV + c) = v;
                        }
                    }
                }
            } else {
                // the four warps' results: each to shared memory relative to its own maximum, joined by all
                float2* stat = reinterpret_cast<float2*>(smem + C::oStat);
                products_sync();  // the last row's have been read
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = g + 8 * h;
                    float* dst = share + (warp * 16 + row) * 128;
#pragma unroll
                    for (int n = 0; n < 16; n += 2) {
                        if constexpr (!Q8) {
#pragma unroll
                            for (int x = 0; x < 2; ++x)
                                *reinterpret_cast<float2*>(dst + (n + x) * 8 + t4 * 2) = make_float2(o[n + x][2 * h], o[n + x][2 * h + 1]);
                        } else {
                            *reinterpret_cast<float4*>(dst + n * 8 + t4 * 4) =
                                make_float4(o[n][2 * h], o[n + 1][2 * h], o[n][2 * h + 1], o[n + 1][2 * h + 1]);
                        }
                    }
                    if (t4 == 0) stat[warp * 16 + row] = make_float2(l[h] == 0.f ? kNone : m[h] - kLift, l[h]);
                }
                products_sync();
                // a warp takes four query rows, a lane four columns
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = warp * 4 + r;
                    if (row >= heads) break;
                    float2 st[4];
                    float M = kNone;
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        st[x] = stat[x * 16 + row];
                        M = fmaxf(M, st[x].x);
                    }
                    float L = 0.f;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const float fx = fast_exp2(st[x].x - M);
                        L = fmaf(st[x].y, fx, L);
                        const float4 y = *reinterpret_cast<const float4*>(share + (x * 16 + row) * 128 + lane * 4);
                        v.x = fmaf(y.x, fx, v.x);
                        v.y = fmaf(y.y, fx, v.y);
                        v.z = fmaf(y.z, fx, v.z);
                        v.w = fmaf(y.w, fx, v.w);
                    }
                    if (!whole) {
                        *reinterpret_cast<float4*>(a.part_o + (static_cast<long long>(run.part) * 16 + row) * KV + lane * 4) = v;
                        if (lane == 0) a.part_ml[run.part * 16 + row] = make_float2(L == 0.f ? kNone : M, L);
                    } else {
                        const float inv = L == 0.f ? 0.f : 1.f / L;
                        *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + (first + row) * KV + lane * 4) =
                            make_uint2(lat::pack2<T>(v.x * inv, v.y * inv), lat::pack2<T>(v.z * inv, v.w * inv));
                        if (p.lse && lane == 0) p.lse[first + row] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
                    }
                }
            }
        }
    }
    __syncthreads();
    if (*bad && tid < C::SLOTS) {
        // what was asked for lands (or a limit runs out) before the shared memory is another CTA's
        const uint32_t open = mbar_try_wait(&full[tid], 0) ? 1 : 0;
        for (int k = 0; k < 1 << 16 && !mbar_try_wait(&full[tid], open); ++k) __nanosleep(256);
    }
}

// Joins the parts of the units that were cut. Block (entry of the cut list, y) of 8 warps; a task is 128
// columns of a head. Few parts: a warp a task; many: the warps divide the parts.
template <int KV, typename T>
__global__ void __launch_bounds__(256) paged_join_kernel(const MmaArgs a) {
    MM_PDL_ENTRY();
    constexpr int NS = KV / 128;
    __shared__ float4 sum_s[8][32];
    const int4 cut = __ldcg(&a.cut[blockIdx.x]);
    if (cut.y == 0) return;
    const Attention& p = a.p;
    const int row = cut.x / a.blocks, h0 = (cut.x - row * a.blocks) * 16, heads = min(16, p.H - h0);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, parts = cut.y;
    auto slot = [&](int i) { return i == 0 ? 2 * cut.z + 1 : 2 * (cut.z + i); };
    const bool many = parts > 16;
    for (int task = many ? blockIdx.y : blockIdx.y * 8 + warp; task < heads * NS; task += gridDim.y * (many ? 1 : 8)) {
        const int h = task / NS, c = (task - h * NS) * 128 + lane * 4;
        float M = kNone, L = 0.f;
        for (int i = lane; i < parts; i += 32) M = fmaxf(M, __ldcg(&a.part_ml[slot(i) * 16 + h]).x);
        M = warp_max(M);
        for (int i = lane; i < parts; i += 32) {
            const float2 v = __ldcg(&a.part_ml[slot(i) * 16 + h]);
            L += v.y * fast_exp2(v.x - M);
        }
        L = warp_sum(L);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int i = many ? warp : 0; i < parts; i += many ? 8 : 1) {
            const float f = fast_exp2(__ldcg(&a.part_ml[slot(i) * 16 + h]).x - M);
            const float4 v = __ldcg(reinterpret_cast<const float4*>(a.part_o + (static_cast<long long>(slot(i)) * 16 + h) * KV + c));
            acc.x = fmaf(v.x, f, acc.x);
            acc.y = fmaf(v.y, f, acc.y);
            acc.z = fmaf(v.z, f, acc.z);
            acc.w = fmaf(v.w, f, acc.w);
        }
        if (many) {
            __syncthreads();
            sum_s[warp][lane] = acc;
            __syncthreads();
            if (warp) continue;
            for (int w = 1; w < 8; ++w) {
                const float4 v = sum_s[w][lane];
                acc.x += v.x;
                acc.y += v.y;
                acc.z += v.z;
                acc.w += v.w;
            }
        }
        const float inv = L == 0.f ? 0.f : 1.f / L;
        const long long r = static_cast<long long>(row) * p.H + h0 + h;
        *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + r * KV + c) =
            make_uint2(lat::pack2<T>(acc.x * inv, acc.y * inv), lat::pack2<T>(acc.z * inv, acc.w * inv));
        if (p.lse && lane == 0 && c == 0) p.lse[r] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
    }
}

}  // namespace paged
}  // namespace mm
