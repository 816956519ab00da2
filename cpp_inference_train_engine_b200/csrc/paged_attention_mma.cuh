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
//              four take a tile (8-bit ones: two) together and add their shares of S through shared memory; 128 wide: each has
//              tiles of its own (every fourth) and the four results are joined at the row's end.
//   loads      1, which walks the CTA's runs ahead of them and queues what they need to know of each: a box a
//              lane, its page number asked for a step ahead.
// Positions that a row does not see are masked in S and cleared in the tile (a probability of zero times a NaN
// would be one). Two CTAs an SM, each with a ring of its own; the row's sums and maxima are fp32, the weights of
// the second product are rounded to 16 bits once, as its operand has to be.
//
// The tiles of all rows, in line, are divided evenly over the CTAs (a row costs row_cost() tiles more); a row
// that is cut leaves partial results to the join kernel.
//
// Measured on one B200, back to back. 296 rows of 1,312 positions, 512 + 32 wide, bf16, take 72.9 us (5.8 TB/s), as an
// earlier form of the loads alone did (73.8). Why mma.sync and not tcgen05: with so few rows it needs no
// tensor memory, no descriptors and no proxy fence between the loads and the products, and its tensor pipe is 36 %
// busy. The tcgen05 kernel of contiguous caches (shared_prefix_tc.cuh) takes 84.0 us for the same rows, 98.3 against
// 63.9 with e4m3 caches; 512 rows of 1,024, 128 + 16 wide, 36.1 against 33.6; one row of 131,072 187 against 42. 8-bit
// rows are bound by the chain of a tile's steps (40 % of the issue slots) and by the unpacking of the codes, once for
// each product; products of e4m3 operands (queries in 2 or 3 parts) were slower, 110 us.
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
    int give_up;       // -1; the self-test: steps of a run after which the loads of every other CTA end as after a wait that ran out
    float* part_o;     // [2 CTAs][16][kv], unnormalised
    float2* part_ml;   // [2 CTAs][16] maximum and sum, base 2
    int4* cut;         // (unit, parts, first CTA): a unit cut at the end of the share it begins in; no parts: none
};

constexpr int kTile = 32;       // positions
// Tiles that a row's queries and results cost: by 512 rows of up to 2,048, 128 wide (2: 36.4 us, 6: 35.0, 10: 35.5, 20:
// 36.7, 40: 40.4), and 96 of up to 8,192 and 400 of up to 700, 512 wide (2: 79.4 and 46.5, 4: 79.2 and 43.8, 6: 79.5 and
// 44.3, 10: 80.2 and 45.0).
constexpr int row_cost(int kv) { return kv == 128 ? 10 : 4; }
// Tiles of a CTA at least, so that few rows make no more partial results than they gain: 512 wide, 8 rows of up to
// 4,096 take 25.8 us with 12, 19.9 with 6, 18.4 with 4, 18.0 with 2, one of 300 16.3, 13.7, 12.1 to 13.5 and 13.7. 128
// wide a tile is a quarter of the bytes and each of the four warps has its own: 5 rows of up to 900 take 9.3 us with 8, 11
// to 13.5 with 16 and 9.3, without a join, with 24.
constexpr int min_share(int kv) { return kv == 128 ? 24 : 4; }
constexpr int kMmaThreads = 160;
constexpr int kQueue = 4;       // runs queued for the warps of the products
constexpr uint32_t kPolls = 1u << 18;  // of a wait until it has run out: about a second
constexpr float kNone = -3.402823466e38f;  // maximum of nothing (finite: its exp2 is 0, never NaN)

template <int KV, int R, bool Q8> struct MmaCfg {
    static constexpr int CW = KV / 128;      // warps that share a tile
    static constexpr int KG = 4 / CW;        // groups with tiles of their own
    static constexpr int kBoxes = Q8 ? KV / 128 : KV / 64;  // latent boxes of 128-byte rows
    static constexpr int kLatent = kBoxes * kTile * 128;
    static constexpr int kRope = kTile * R * 2;
    static constexpr int kScale = Q8 ? 256 : 0;             // two boxes of 16 at 128-byte addresses
    static constexpr int kSlot = (kLatent + kRope + 1023) / 1024 * 1024;
    static constexpr int kBytes = kLatent + kRope + (Q8 ? kTile * 4 : 0);  // that TMA brings
    static constexpr int SG = KV == 512 ? (Q8 ? 5 : 3) : (Q8 ? 3 : 2);     // slots of a group
    static constexpr int SLOTS = KG * SG;
    // Tiles that warps who share them weigh at a time. 8-bit ones, of which an SM has to do more in the same time, two:
    // the exchange costs as much (120 rows of up to 6,001 positions 79.0 -> 75.7 us); the others' ring has no room for it.
    static constexpr int TW = CW > 1 && Q8 ? 2 : 1;
    // 512: the four shares of S; 128: the four results of a row
    static constexpr int kShareRow = 136;  // (128 columns and 8 more, which spread eight rows over all banks)
    static constexpr int kShare = KV == 512 ? TW * 4 * 16 * kTile * 4 : 4 * 16 * kShareRow * 4;
    static constexpr int oShare = SLOTS * kSlot;
    static constexpr int oScale = oShare + kShare;          // of the slots' positions
    static constexpr int oStat = oScale + SLOTS * kScale;   // [4][16] maxima and sums (128 wide)
    static constexpr int oTops = oStat;                     // [4][16] maxima, sums (512 wide)
    static constexpr int oHand = oStat + 4 * 16 * 8;        // [TW][4][32] weights, 8 positions from each warp (512 wide)
    static constexpr int oRuns = oHand + (KV == 512 ? TW * 1024 : 0);
    static constexpr int oPlan = oRuns + kQueue * 32;
    static constexpr int oBar = oPlan + 48;
    static constexpr int oMeta = oBar + (2 * SLOTS + 2 * kQueue) * 8;
    static constexpr int kSmem = oMeta + SLOTS * 4 + 1024;  // + alignment of the base
    static_assert(oBar % 8 == 0 && oRuns % 16 == 0 && oStat % 8 == 0 && oShare % 1024 == 0 && oScale % 128 == 0 && kSlot % 1024 == 0, "alignment");
    static_assert(2 * (kSmem + 1024) <= 228 * 1024, "two CTAs an SM");
};

// What a CTA does next: tiles [from, to) of 16 heads of a row, from h0 on. Tile i stands at position 32 i below
// `sinks` tiles, behind them `skip` tiles further.
struct alignas(16) Run {
    int row, h0, len, sinks, skip, from, to;
    int part;  // slot of partial results, -1: the whole row
    // (unsigned: a step past a row of 2^31 positions wraps around, and is not used)
    __device__ __forceinline__ int position(int i) const { return static_cast<int>(32u * static_cast<unsigned>(i < sinks ? i : i + skip)); }
};

// Tiles of row b: those with one of the first `sinks` positions, then those from the window's on.
__device__ __forceinline__ int row_tiles(const Attention& p, int len, int& sink_tiles, int& skip) {
    auto tiles = [](int n) { return n / kTile + (n % kTile > 0); };  // (n + kTile - 1 may pass 32 bits)
    const int start = window_start(p, len);
    sink_tiles = tiles(min(p.sinks, start));
    skip = max(start / kTile, sink_tiles) - sink_tiles;
    return tiles(len) - skip;
}

// The runs of a CTA. With even shares, the CTA's are the tiles of weight [w0, w1) of all rows in line, where a
// row's tiles are followed by its cost.
struct Runs {
    const MmaArgs& a;
    int w0, w1, span, before;  // the share, and the weight ahead of row `row`
    int cost;
    int row, block, len;
    __device__ __forceinline__ Runs(const MmaArgs& args, int cost_, int span_, int row0, int before0)
        : a(args), span(span_), cost(cost_) {
        if (a.shares) {
            w0 = static_cast<int>(blockIdx.x) * span;
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
    // cut: the unit's parts where it begins here (0: it is whole), else -1.
    __device__ __forceinline__ bool next(Run& r, int& cut) {
        while (row < a.p.B) {
            r.row = row;
            r.h0 = block * 16;
            r.len = len;
            const int n = row_tiles(a.p, len, r.sinks, r.skip);
            if (!a.shares) {
                r.from = 0;
                r.to = n;
                r.part = cut = -1;
                const int u = row * a.blocks + block + static_cast<int>(gridDim.x);
                row = u / a.blocks;
                block = u - row * a.blocks;
                if (row < a.p.B) len = length_of(a.p, row);
                return true;
            }
            const int at = before + block * (n + cost);
            if (at >= w1) return false;
            const bool begins = at >= w0;
            r.from = begins ? 0 : min(w0 - at, n);
            r.to = min(w1 - at, n);
            const bool whole = begins && r.to == n;
            r.part = whole ? -1 : 2 * static_cast<int>(blockIdx.x) + (begins ? 1 : 0);
            cut = !begins ? -1 : whole ? 0 : (at + n - 1) / span - static_cast<int>(blockIdx.x) + 1;
            if (++block == a.blocks) {
                block = 0;
                before += a.blocks * (n + cost);
                if (++row < a.p.B) len = length_of(a.p, row);
            }
            if (begins || r.from < r.to) return true;
        }
        return false;
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
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same from zero.
template <typename T> __device__ __forceinline__ void mma16_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// Byte offset of 16-byte chunk c of row r in a box of 128-, 64- or 32-byte rows, as TMA swizzles it.
__device__ __forceinline__ uint32_t swizzled(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }
template <int R> __device__ __forceinline__ uint32_t swizzled_rope(int r, int c) {
    return R == 32 ? r * 64 + ((c ^ ((r >> 1) & 3)) << 4) : r * 32 + ((c ^ ((r >> 2) & 1)) << 4);
}
// Four e4m3 codes as fp16 values (exact): the first two, the last two.
__device__ __forceinline__ void codes4(uint32_t four, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(four));
}
// The four warps of the products, all of their threads.
__device__ __forceinline__ void products_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool products_any(bool p) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbar.red.or.pred p, 1, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r)
        : "r"(static_cast<uint32_t>(p))
        : "memory");
    return r != 0;
}
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

// The end of a CTA in which a wait ran out. What it asked for lands (the phases of the slots' barriers that are open; one
// that nothing is in lasts its limit, a quarter of a second) before the shared memory is another CTA's. Its runs, walked once more
// from the start, get NaN for results, the parts of cut rows too, and the join gets every entry that it reads: nothing is left
// as the memory was. (As a function that is called it costs the product warps 32 bytes of spills.)
template <int KV, typename T>
__device__ __forceinline__ void end_after_timeout(const MmaArgs& a, const int* plan, uint64_t* full, int slots) {
    const Attention& p = a.p;
    const int tid = threadIdx.x;
    const float nan = __int_as_float(0x7fc00000);
    if (tid < slots) {
        const uint32_t open = mbar_try_wait(&full[tid], 0) ? 1 : 0;
        for (int k = 0; k < 1 << 16 && !mbar_try_wait(&full[tid], open); ++k) __nanosleep(256);
    }
    Runs runs(a, row_cost(KV), a.shares ? plan[5] : 0, a.shares ? plan[7] : 0, a.shares ? plan[6] : 0);
    Run run;
    int cut;
    while (runs.next(run, cut)) {
        const int heads = min(16, p.H - run.h0);
        const long long first = static_cast<long long>(run.row) * p.H + run.h0;
        if (run.part < 0) {
            for (int i = tid; i < heads * KV; i += kMmaThreads) static_cast<T*>(p.out)[first * KV + i] = lat::from_f32<T>(nan);
            if (p.lse && tid < heads) p.lse[first + tid] = nan;
        } else if (tid < 16) {
            a.part_ml[run.part * 16 + tid] = make_float2(0.f, nan);  // (whatever its values are: a sum of NaN divides them)
        }
        if (tid == 0 && (a.by_unit ? cut >= 0 : cut > 0)) {
            const int unit = run.row * a.blocks + run.h0 / 16;
            a.cut[a.by_unit ? unit : blockIdx.x] = make_int4(unit, cut, blockIdx.x, 0);
        }
    }
}

// HALF: at most 8 heads, whose rows are the first 8 of the products': nothing is done for the others.
template <int KV, int R, typename T, bool Q8, bool HALF>
__global__ void __launch_bounds__(kMmaThreads, 2)
    paged_mma_kernel(const __grid_constant__ MmaArgs a, const __grid_constant__ CUtensorMap map_latent,
                     const __grid_constant__ CUtensorMap map_rope, const __grid_constant__ CUtensorMap map_scale) {
    using C = MmaCfg<KV, R, Q8>;
    constexpr int RH = HALF ? 1 : 2;               // halves of the 16 rows
    using TP = std::conditional_t<Q8, __half, T>;  // the second product's type (codes are exact in fp16)
    // log2 of the largest weight when its reference is taken: small fp16 ones stay normal, large ones below 2^16
    constexpr float kGrowth = 8.f, kLift = !std::is_same<TP, __half>::value ? 0.f : C::CW > 1 ? 6.f : 10.f;
    extern __shared__ uint8_t mma_smem_raw[];
    // (an offset, not a rounded address: the compiler has to see that the pointers below are of shared memory)
    uint8_t* smem = mma_smem_raw + ((1024 - (smem_u32(mma_smem_raw) & 1023)) & 1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::oBar);
    uint64_t* empty = full + C::SLOTS;
    uint64_t* run_full = empty + C::SLOTS;
    uint64_t* run_empty = run_full + kQueue;
    Run* queue = reinterpret_cast<Run*>(smem + C::oRuns);
    // positions of the tile in a slot that the row sees, by halves of 16
    volatile uint16_t* meta = reinterpret_cast<volatile uint16_t*>(smem + C::oMeta);
    int* plan = reinterpret_cast<int*>(smem + C::oPlan);  // the warps' sums; span, weight ahead, row
    volatile int* bad = reinterpret_cast<volatile int*>(smem + C::oPlan + 44);
    const Attention& p = a.p;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < C::SLOTS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], C::CW);
        }
        for (int i = 0; i < kQueue; ++i) {
            mbar_init(&run_full[i], 1);
            mbar_init(&run_empty[i], 4);
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
        // the weight of all rows, and the row that this CTA's share begins in: a thread sums some rows in line
        const int per = (p.B + kMmaThreads - 1) / kMmaThreads, b0 = tid * per, b1 = min(b0 + per, p.B);
        auto weight = [&](int b) {
            int st, skip;
            return (row_tiles(p, length_of(p, b), st, skip) + row_cost(KV)) * a.blocks;
        };
        int mine = 0;
#pragma unroll 4
        for (int b = b0; b < b1; ++b) mine += weight(b);
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        if (lane == 31) plan[warp] = upto;
        __syncthreads();
        int ahead = upto - mine, total = 0;
#pragma unroll
        for (int i = 0; i < kMmaThreads / 32; ++i) {
            ahead += i < warp ? plan[i] : 0;
            total += plan[i];
        }
        const int span = max((total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x), min_share(KV));
        const int w0 = static_cast<int>(blockIdx.x) * span;  // below the grid's shares, which fit 32 bits
        if (tid == 0) {
            plan[5] = span;
            if (w0 >= total) plan[7] = p.B;
            if (!a.by_unit) a.cut[blockIdx.x] = make_int4(0, 0, 0, 0);
        }
        if (w0 >= ahead && w0 < ahead + mine) {
            int b = b0;
            for (int w; ahead + (w = weight(b)) <= w0; ++b) ahead += w;
            plan[6] = ahead;
            plan[7] = b;
        }
    }
    __syncthreads();
    bool ok = true;
    // a wait that ran out is recorded once; later waits of this thread are skipped
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (ok && !mbar_wait_bounded(bar, parity, &paged_status, kPolls)) {
            ok = false;
            *bad = 1;
        }
    };
    auto give_up = [&] {
        raise_error(&paged_status, kErrWaitTimeout);
        ok = false;
        *bad = 1;
    };

    if (warp == 4) {
        // ------------------------------------------------------------ loads
        Runs runs(a, row_cost(KV), a.shares ? plan[5] : 0, a.shares ? plan[7] : 0, a.shares ? plan[6] : 0);
        Run run;
        // A step is a tile for each group. This lane's box of its group's tile: which stretch of `box` positions,
        // which box of it (128 wide: 3 or 6 boxes for 8 lanes; 512 wide: at most 18 for 32).
        constexpr int kLanes = 32 / C::KG, kEach = C::kBoxes + 1 + (Q8 ? 1 : 0);
        const int group = lane / kLanes, sub = lane % kLanes, stretch = sub / kEach, which = sub % kEach;
        const bool loads = stretch * a.box < kTile;
        const int page = p.pool.positions;
        const uint32_t offset = which < C::kBoxes    ? which * kTile * 128 + stretch * a.box * 128
                                : which == C::kBoxes ? C::kLatent + stretch * a.box * R * 2
                                                     : C::oScale + stretch * 128;
        const int each = which <= C::kBoxes ? C::kSlot : C::kScale;  // from one slot's to the next one's
        const CUtensorMap* map = which < C::kBoxes ? &map_latent : which == C::kBoxes ? &map_rope : &map_scale;
        const int column = which < C::kBoxes ? which * (Q8 ? 128 : 64) : Q8 ? 0 : KV;
        int slot = 0, q = 0;
        uint32_t phase = 0, q_phase = 0;  // parity of the round in this group's ring, in the queue
        int cut;
        // page and entry of this lane's stretch of tile i
        int id = -1, at = 0;
        auto ask = [&](int i) {
            const int t = static_cast<int>(static_cast<unsigned>(run.position(i)) + static_cast<unsigned>(stretch * a.box));
            const int c = p.table.shift >= 0 ? t >> p.table.shift : t / page;
            at = t - c * page;
            id = -1;
            if (loads && i < run.to && t < run.len) id = __ldg(p.table.entry + run.row * p.table.stride + c);
        };
        while (ok) {
            const bool more = runs.next(run, cut);
            if (more) {
                ask(run.from + group);
                // its queries, for the warps of the products
                constexpr int kLines = ((KV + R) * 2 + 127) / 128;
                const T* heads = static_cast<const T*>(p.q) + run.row * p.q_row + run.h0 * p.q_head;
                const int n = min(16, p.H - run.h0) * kLines;
                for (int e = lane; e < n; e += 32) prefetch_l1(heads + e / kLines * p.q_head + min(e % kLines * 64, KV + R - 1));
            }
            wait(&run_empty[q], q_phase ^ 1);
            // (all lanes or none: the votes below are of whole warps, and a queue entry that is still read is not written)
            if (__any_sync(0xffffffffu, !ok)) break;
            if (lane == 0) {
                if (!more) run.row = -1;
                queue[q] = run;
                mbar_arrive(&run_full[q]);
                if (more && (a.by_unit ? cut >= 0 : cut > 0)) {
                    const int unit = run.row * a.blocks + run.h0 / 16;
                    a.cut[a.by_unit ? unit : blockIdx.x] = make_int4(unit, cut, blockIdx.x, 0);
                }
            }
            if (++q == kQueue) {
                q = 0;
                q_phase ^= 1;
            }
            if (!more) break;
            const int start = window_start(p, run.len), sinks = min(p.sinks, start);
            for (int i = run.from + group; i - group < run.to; i += C::KG) {
                // a page outside the pool (or behind the row) is asked for behind the last one: zeros
                const bool there = id >= 0 && id < p.pool.rows, mine = i < run.to;
                const int z = there ? id : p.pool.rows, y = at;
                ask(i + C::KG);
                const int s = group * C::SG + slot;
                if (mine) wait(&empty[s], phase ^ 1);
                if (i - group - run.from == a.give_up * C::KG && blockIdx.x & 1) give_up();
                if (__any_sync(0xffffffffu, !ok)) {
                    ok = false;
                    break;
                }
                if (mine && loads && which == 0) {
                    uint32_t seen = 0;
                    if (there) {
                        const int t = run.position(i);
                        auto below = [&](int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; };
                        seen = below(run.len - t) & (below(sinks - t) | ~below(start - t));
                    }
                    if (a.box == kTile) *reinterpret_cast<volatile uint32_t*>(meta + 2 * s) = seen;
                    else meta[2 * s + stretch] = static_cast<uint16_t>(seen >> (16 * stretch));
                }
                __syncwarp();
                if (mine && sub == 0) mbar_arrive_expect_tx(&full[s], C::kBytes);
                __syncwarp();
                if (mine) {
                    if (loads) {
                        uint8_t* dst = smem + s * each + offset;
                        if (Q8 && which > C::kBoxes) tma_load_2d(dst, map, &full[s], y, z);
                        else tma_load_box(dst, map, &full[s], column, y, z);
                    }
                    if (++slot == C::SG) {
                        slot = 0;
                        phase ^= 1;
                    }
                }
            }
        }
    } else {
        // ------------------------------------------------------------ products
        const int cw = warp % C::CW, group = warp / C::CW;
        const int g = lane >> 2, t4 = lane & 3;  // row of the fragments, place in its quad
        const uint32_t ring = smem_u32(smem) + group * C::SG * C::kSlot;
        // this lane's rows of the matrices that ldmatrix reads
        const int mrow = lane & 7, msel = lane >> 3;
        // offsets in a slot of its first matrices: the next columns are an exclusive or away (the swizzle's chunk is
        // chunk ^ row, and slots and rows of a box keep those bits free), the next 16 rows 2,048 bytes
        const uint32_t s_at = cw * (Q8 ? 1 : 2) * (kTile * 128) + (Q8 ? swizzled(msel * 8 + mrow, 0) : swizzled((msel >> 1) * 8 + mrow, msel & 1));
        const uint32_t o_at = cw * (Q8 ? 1 : 2) * (kTile * 128) + swizzled((msel & 1) * 8 + mrow, msel >> 1);
        const uint32_t rope_at = C::kLatent + swizzled_rope<R>((msel >> 1) * 8 + mrow, cw * 2 + (msel & 1));
        float* share = reinterpret_cast<float*>(smem + C::oShare);
        const float cs = p.scale * 1.4426950408889634f;
        // scales of the lane's positions 8 n + 2 t4 and the next (a second box of 16 starts 128 bytes on)
        auto scales_of = [&](int sl, int n) {
            const uint8_t* at = smem + C::oScale + (group * C::SG + sl) * C::kScale;
            return *reinterpret_cast<const float2*>(at + (n * 8 + t4 * 2) * 4 + (n >= 2 && a.box == 16 ? 64 : 0));
        };
        int slot = 0, turn = 0;
        uint32_t phase = 0, turn_phase = 0;
        auto warp_arrive = [&](uint64_t* bar) {
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        while (true) {
            wait(&run_full[turn], turn_phase);
            if (products_any(!ok)) break;  // the four warps meet at barriers of their own: they leave together
            const Run run = queue[turn];
            __syncwarp();
            if (lane == 0) mbar_arrive(&run_empty[turn]);
            if (++turn == kQueue) {
                turn = 0;
                turn_phase ^= 1;
            }
            if (run.row < 0) break;
            const int h0 = run.h0, heads = min(16, p.H - h0);
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
            // S of the tile in slot sl: this warp's columns of it
            auto scores = [&](int sl, float (&s)[4][4]) {
                const uint32_t sp = ring + sl * C::kSlot;
                if constexpr (!Q8) {
                    // (loads one step ahead of the products: issue is in order)
                    const uint32_t box = sp + s_at;
                    uint32_t b[2][2][4];
                    auto load = [&](int k, uint32_t (&d)[2][4]) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) ldsm4(d[h], (box ^ ((k & 3) * 32)) + (k >> 2) * (kTile * 128) + h * 2048);
                    };
                    load(0, b[0]);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        if (k < 7) load(k + 1, b[(k + 1) & 1]);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (k == 0) {
                                mma16_first<T>(s[2 * h], q[k], b[0][h][0], b[0][h][1]);
                                mma16_first<T>(s[2 * h + 1], q[k], b[0][h][2], b[0][h][3]);
                            } else {
                                mma16<T>(s[2 * h], q[k], b[k & 1][h][0], b[k & 1][h][1]);
                                mma16<T>(s[2 * h + 1], q[k], b[k & 1][h][2], b[k & 1][h][3]);
                            }
                        }
                    }
                } else {
                    const uint32_t box = sp + s_at;
                    uint32_t b[2][4];
                    ldsm4(b[0], box);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        if (k < 7) ldsm4(b[(k + 1) & 1], box ^ ((k + 1) * 16));
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            uint32_t lo, hi;
                            codes4(b[k & 1][n], lo, hi);
                            if (k == 0) mma16_first<__half>(s[n], q[k], lo, hi);
                            else mma16<__half>(s[n], q[k], lo, hi);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const float2 v = scales_of(sl, n);
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
                        ldsm4(b, sp + rope_at + h * 16 * R * 2);
                        mma16<T>(s[2 * h], qr, b[0], b[1]);
                        mma16<T>(s[2 * h + 1], qr, b[2], b[3]);
                    }
                }
            };
            // positions of the tile in slot sl that the row sees
            auto seen_of = [&](int sl) { return reinterpret_cast<volatile const uint32_t*>(meta)[group * C::SG + sl]; };
            // Weights of the tile in slot sl (the second product's operand, 16 positions each) from its scores.
            auto weigh = [&](int sl, float (&s)[4][4], uint32_t (&w)[2][4]) {
                const uint32_t seen = seen_of(sl);
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int e = 0; e < 2 * RH; ++e) s[n][e] *= cs;
                if (seen != ~0u) {
#pragma unroll
                    for (int n = 0; n < 4; ++n)
#pragma unroll
                        for (int e = 0; e < 2 * RH; ++e)
                            if (!((seen >> (n * 8 + t4 * 2 + (e & 1))) & 1)) s[n][e] = -INFINITY;
                }
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    float2 e2 = make_float2(0.f, 0.f);
                    if constexpr (Q8) {
                        const float2 v = scales_of(sl, n);
                        e2 = make_float2(exponent_of(v.x), exponent_of(v.y));
                    }
#pragma unroll
                    for (int e = 0; e < 2 * RH; ++e)
                        top[e >> 1] = fmaxf(top[e >> 1], Q8 ? s[n][e] + (e & 1 ? e2.y : e2.x) : s[n][e]);
                }
                float corr[2] = {1.f, 1.f}, ref[2];
#pragma unroll
                for (int h = 0; h < RH; ++h) {
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
                        if (RH == 2) {
                            o[n][2] *= corr[1];
                            o[n][3] *= corr[1];
                        }
                    }
                    l[0] *= corr[0];
                    l[1] *= corr[1];
                }
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    float2 v = make_float2(1.f, 1.f);
                    if constexpr (Q8) {
                        v = scales_of(sl, n);
                        if (seen != ~0u) {  // (0 times what an unseen position has for a scale may be a NaN)
                            if (!((seen >> (n * 8 + t4 * 2)) & 1)) v.x = 0.f;
                            if (!((seen >> (n * 8 + t4 * 2 + 1)) & 1)) v.y = 0.f;
                        }
                    }
                    float e[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int x = 0; x < 2 * RH; ++x) {
                        e[x] = fast_exp2(s[n][x] - ref[x >> 1]);
                        l[x >> 1] += e[x];
                        if (Q8) e[x] *= x & 1 ? v.y : v.x;
                    }
                    w[n >> 1][(n & 1) * 2] = lat::pack2<TP>(e[0], e[1]);
                    w[n >> 1][(n & 1) * 2 + 1] = lat::pack2<TP>(e[2], e[3]);
                }
                return seen;
            };
            // O += P V over this warp's columns, and the slot goes back
            auto values = [&](int sl, uint32_t seen, const uint32_t (&w)[2][4]) {
                const uint32_t sp = ring + sl * C::kSlot;
                if (seen != ~0u) {  // positions that are not seen hold anything
                    __syncwarp();
                    uint8_t* boxes = smem + (group * C::SG + sl) * C::kSlot + cw * (Q8 ? 1 : 2) * (kTile * 128);
                    for (uint32_t hide = ~seen; hide; hide &= hide - 1) {
                        const int r = __ffs(hide) - 1;
                        if (lane < (Q8 ? 8 : 16))
                            *reinterpret_cast<uint4*>(boxes + (lane >> 3) * (kTile * 128) + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    __syncwarp();
                }
                if constexpr (!Q8) {
                    // (16 positions after the other 16: a product follows the one that it adds to by 15 others)
                    const uint32_t box = sp + o_at;
                    uint32_t b[2][2][4];
                    auto load = [&](int j, uint32_t (&d)[2][4]) {
                        const int k = j >> 2, c = (j & 3) * 2;
#pragma unroll
                        for (int x = 0; x < 2; ++x) ldsm4_t(d[x], (box ^ (((c + x) & 3) * 32)) + (c >> 2) * (kTile * 128) + k * 2048);
                    };
                    load(0, b[0]);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int k = j >> 2, c = (j & 3) * 2;
                        if (j < 7) load(j + 1, b[(j + 1) & 1]);
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            mma16<T>(o[2 * (c + x)], w[k], b[j & 1][x][0], b[j & 1][x][1]);
                            mma16<T>(o[2 * (c + x) + 1], w[k], b[j & 1][x][2], b[j & 1][x][3]);
                        }
                    }
                } else {
                    // a transposed pair of codes is two neighbouring columns of one position: the even columns of 16
                    // make one tile of the product, the odd ones another
                    const uint32_t box = sp + o_at;
                    uint32_t b[2][4];
                    auto load = [&](int j, uint32_t (&d)[4]) { ldsm4_t(d, (box ^ ((j & 3) * 32)) + (j >> 2) * 2048); };
                    load(0, b[0]);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int k = j >> 2, c = j & 3;
                        if (j < 7) load(j + 1, b[(j + 1) & 1]);
                        uint32_t even[4], odd[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) codes4(__byte_perm(b[j & 1][x], 0, 0x3120), even[x], odd[x]);
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            mma16<__half>(o[4 * c + 2 * x], w[k], even[2 * x], even[2 * x + 1]);
                            mma16<__half>(o[4 * c + 2 * x + 1], w[k], odd[2 * x], odd[2 * x + 1]);
                        }
                    }
                }
                if (seen != ~0u) fence_proxy_async_smem();  // the cleared rows, before the next tile lands on them
                warp_arrive(&empty[group * C::SG + sl]);
            };
            uint32_t w[2][4];
            float s[4][4];
            if constexpr (C::CW == 1) {
                for (int i = run.from + group; i < run.to; i += C::KG) {
                    wait(&full[group * C::SG + slot], phase);
                    scores(slot, s);
                    const uint32_t seen = weigh(slot, s, w);
                    values(slot, seen, w);
                    if (++slot == C::SG) {
                        slot = 0;
                        phase ^= 1;
                    }
                }
            } else {
                // Each warp adds the four shares of S for 8 of the tile's positions and hands their weights to the
                // others. The reference of the weights is the running maximum when it last moved, which it does
                // only where a score passes it by 2^8 (or there was none): the warps vote on it with the barrier that
                // hands the weights over. The next tile's shares are made before this tile's O product, which hides
                // their exchange.
                constexpr int TW = C::TW;
                float4* mine = reinterpret_cast<float4*>(share) + cw * 128 + lane;
                uint2* hand = reinterpret_cast<uint2*>(smem + C::oHand) + lane;
                float* tops = reinterpret_cast<float*>(smem + C::oTops);
                float ref[2] = {-kLift, -kLift};  // what scores are taken from: m, or 0 where there is none, below the lift
                // waits for the next tile and makes its shares as tile x of a round (the last round's were read before
                // its weights were handed over)
                auto take = [&](int x) {
                    const int sl = slot;
                    wait(&full[sl], phase);
                    if (++slot == C::SG) {
                        slot = 0;
                        phase ^= 1;
                    }
                    scores(sl, s);
#pragma unroll
                    for (int n = 0; n < 4; ++n) mine[x * 512 + n * 32] = make_float4(s[n][0], s[n][1], s[n][2], s[n][3]);
                    return sl;
                };
                int at[TW] = {};  // the round's slots
#pragma unroll
                for (int x = 0; x < TW; ++x)
                    if (run.from + x < run.to) at[x] = take(x);
                for (int i = run.from; i < run.to; i += TW) {
                    products_sync();
                    float z[TW][4], top[2] = {-INFINITY, -INFINITY};
                    float2 ks[TW];
#pragma unroll
                    for (int x = 0; x < TW; ++x) {
                        ks[x] = make_float2(0.f, 0.f);
                        z[x][0] = z[x][1] = z[x][2] = z[x][3] = -INFINITY;
                        if (x > 0 && i + x >= run.to) continue;
                        const ulonglong2* v = reinterpret_cast<const ulonglong2*>(share) + x * 512 + cw * 32 + lane;
                        const ulonglong2 u0 = v[0], u1 = v[128], u2 = v[256], u3 = v[384];
                        const Two by(cs, cs), lo = ((Two(u0.x) + Two(u1.x)) + (Two(u2.x) + Two(u3.x))) * by,
                                  hi = ((Two(u0.y) + Two(u1.y)) + (Two(u2.y) + Two(u3.y))) * by;
                        z[x][0] = lo.lo();
                        z[x][1] = lo.hi();
                        z[x][2] = hi.lo();
                        z[x][3] = hi.hi();
                        const uint32_t seen = seen_of(at[x]);
                        float2 e2 = make_float2(0.f, 0.f);
                        if constexpr (Q8) {
                            ks[x] = scales_of(at[x], cw);
                            e2 = make_float2(exponent_of(ks[x].x), exponent_of(ks[x].y));
                        }
                        if (seen != ~0u) {
                            if (!((seen >> (cw * 8 + t4 * 2)) & 1)) {
                                z[x][0] = z[x][2] = -INFINITY;
                                ks[x].x = 0.f;  // (0 times what an unseen position has for a scale may be a NaN)
                            }
                            if (!((seen >> (cw * 8 + t4 * 2 + 1)) & 1)) {
                                z[x][1] = z[x][3] = -INFINITY;
                                ks[x].y = 0.f;
                            }
                        }
                        top[0] = fmaxf(top[0], fmaxf(z[x][0] + e2.x, z[x][1] + e2.y));
                        top[1] = fmaxf(top[1], fmaxf(z[x][2] + e2.x, z[x][3] + e2.y));
                    }
                    float add[2];
                    auto give = [&] {
                        add[0] = add[1] = 0.f;
#pragma unroll
                        for (int x = 0; x < TW; ++x) {
                            float e[4];
#pragma unroll
                            for (int y = 0; y < 4; ++y) e[y] = fast_exp2(z[x][y] - ref[y >> 1]);
                            add[0] += e[0] + e[1];
                            add[1] += e[2] + e[3];
                            if constexpr (Q8) {
                                e[0] *= ks[x].x;
                                e[1] *= ks[x].y;
                                e[2] *= ks[x].x;
                                e[3] *= ks[x].y;
                            }
                            hand[(x * 4 + cw) * 32] = make_uint2(lat::pack2<TP>(e[0], e[1]), lat::pack2<TP>(e[2], e[3]));
                        }
                    };
                    give();
                    if (products_any(top[0] > m[0] + kGrowth || top[1] > m[1] + kGrowth)) {
                        // the maximum over the tiles, and the sums and products so far below it
                        const float a0 = quad_max(top[0]), a1 = quad_max(top[1]);
                        if (t4 == 0) {
                            tops[cw * 16 + g] = a0;
                            tops[cw * 16 + g + 8] = a1;
                        }
                        products_sync();
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float* t = tops + g + 8 * h;
                            const float mn = fmaxf(fmaxf(m[h], fmaxf(t[0], t[16])), fmaxf(t[32], t[48]));
                            const float corr = m[h] == mn ? 1.f : fast_exp2(m[h] - mn);
                            m[h] = mn;
                            ref[h] = (mn == -INFINITY ? 0.f : mn) - kLift;
                            l[h] *= corr;
#pragma unroll
                            for (int n = 0; n < 16; ++n) {
                                o[n][2 * h] *= corr;
                                o[n][2 * h + 1] *= corr;
                            }
                        }
                        give();
                        products_sync();
                    }
                    l[0] += add[0];
                    l[1] += add[1];
                    // (a slot is given back before the next round's second tile is waited for)
#pragma unroll
                    for (int x = 0; x < TW; ++x) {
                        const int sl = at[x];
                        auto handed = [&] {
#pragma unroll
                            for (int n = 0; n < 4; ++n) {
                                const uint2 v = hand[(x * 4 + n) * 32];
                                w[n >> 1][(n & 1) * 2] = v.x;
                                w[n >> 1][(n & 1) * 2 + 1] = v.y;
                            }
                        };
                        if constexpr (TW == 1) handed();
                        if (i + TW + x < run.to) at[x] = take(x);
                        if constexpr (TW > 1) handed();
                        if (x == 0 || i + x < run.to) values(sl, seen_of(sl), w);
                    }
                }
            }
            // ------------------------------------------------------------ results
            l[0] = quad_sum(l[0]);
            l[1] = quad_sum(l[1]);
            if constexpr (C::CW > 1) {  // of the positions that each warp weighed
                float* sums = reinterpret_cast<float*>(smem + C::oTops);
                products_sync();
                if (t4 == 0) {
                    sums[cw * 16 + g] = l[0];
                    sums[cw * 16 + g + 8] = l[1];
                }
                products_sync();
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float* t = sums + g + 8 * h;
                    l[h] = (t[0] + t[16]) + (t[32] + t[48]);
                }
            }
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
                for (int h = 0; h < RH; ++h) {
                    const int row = g + 8 * h;
                    float* dst = share + (warp * 16 + row) * C::kShareRow;
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
                // a warp takes every fourth query row, a lane four columns
#pragma unroll
                for (int r = 0; r < 2 * RH; ++r) {
                    const int row = r * 4 + warp;
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
                        const float4 y = *reinterpret_cast<const float4*>(share + (x * 16 + row) * C::kShareRow + lane * 4);
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
    if (*bad) end_after_timeout<KV, T>(a, plan, full, C::SLOTS);
}

// Bound by the latency of two rounds of loads from L2 and by the launch: 5 us of the 80 that 96 wide rows of up to 8,192
// positions take.
//
// Joins the parts of the units that were cut. Block (entry of the cut list, y) of 8 warps. Up to kFew parts: a warp
// takes NG times 128 columns of a head, eight 16-byte loads a lane at a time; more: the warps of a block divide the
// parts of 128 columns of a head.
constexpr int kFew = 8;
struct Mean {  // a weighted mean in the making: maximum and sum of the weights
    float m = kNone, l = 0.f;
    // Factors of what there is and of a part that comes.
    __device__ __forceinline__ float2 add(float2 ml) {
        const float top = fmaxf(m, ml.x), f = fast_exp2(m - top), g = fast_exp2(ml.x - top);
        l = fmaf(ml.y, g, l * f);
        m = top;
        return make_float2(f, g);
    }
};
__device__ __forceinline__ void blend(float4& o, float4 v, float2 f) {
    o = make_float4(fmaf(v.x, f.y, o.x * f.x), fmaf(v.y, f.y, o.y * f.x), fmaf(v.z, f.y, o.z * f.x), fmaf(v.w, f.y, o.w * f.x));
}
template <int KV, int NG, typename T>
__global__ void __launch_bounds__(256) paged_join_kernel(const __grid_constant__ MmaArgs a) {
    MM_PDL_ENTRY();
    constexpr int NS = KV / 128, PER = 8 / NG;
    __shared__ float4 sum_s[8][32];
    __shared__ float2 ml_s[8];
    const int4 cut = __ldcg(&a.cut[blockIdx.x]);
    const int parts = cut.y;
    if (parts == 0) return;
    const Attention& p = a.p;
    const int row = cut.x / a.blocks, h0 = (cut.x - row * a.blocks) * 16, heads = min(16, p.H - h0);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto slot = [&](int i) { return i == 0 ? 2 * cut.z + 1 : 2 * (cut.z + i); };
    const long long first = static_cast<long long>(row) * p.H + h0;
    auto finish = [&](int h, int c, float4 o, const Mean& sum) {
        const float inv = sum.l == 0.f ? 0.f : 1.f / sum.l;
        *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + (first + h) * KV + c) =
            make_uint2(lat::pack2<T>(o.x * inv, o.y * inv), lat::pack2<T>(o.z * inv, o.w * inv));
        if (p.lse && c == 0) p.lse[first + h] = sum.l == 0.f ? -INFINITY : (sum.m + log2f(sum.l)) * 0.6931471805599453f;
    };
    if (parts <= kFew) {
        for (int task = blockIdx.y * 8 + warp; task < heads * (NS / NG); task += gridDim.y * 8) {
            const int h = task / (NS / NG), c = (task - h * (NS / NG)) * NG * 128 + lane * 4;
            Mean sum;
            float4 o[NG];
#pragma unroll
            for (int x = 0; x < NG; ++x) o[x] = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int i0 = 0; i0 < parts; i0 += PER) {
                float4 v[PER][NG];
                float2 ml[PER];
#pragma unroll
                for (int k = 0; k < PER; ++k) {
                    if (i0 + k >= parts) continue;
                    const int at = slot(i0 + k) * 16 + h;
                    ml[k] = __ldcg(&a.part_ml[at]);
#pragma unroll
                    for (int x = 0; x < NG; ++x)
                        v[k][x] = __ldcg(reinterpret_cast<const float4*>(a.part_o + static_cast<long long>(at) * KV + c + x * 128));
                }
#pragma unroll
                for (int k = 0; k < PER; ++k) {
                    if (i0 + k >= parts) continue;
                    const float2 f = sum.add(ml[k]);
#pragma unroll
                    for (int x = 0; x < NG; ++x) blend(o[x], v[k][x], f);
                }
            }
#pragma unroll
            for (int x = 0; x < NG; ++x) finish(h, c + x * 128, o[x], sum);
        }
        return;
    }
    for (int task = blockIdx.y; task < heads * NS; task += gridDim.y) {
        const int h = task / NS, c = (task - h * NS) * 128 + lane * 4;
        Mean sum;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i0 = warp; i0 < parts; i0 += 8 * 8) {
            float4 v[8];
            float2 ml[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (i0 + 8 * k >= parts) continue;
                const int at = slot(i0 + 8 * k) * 16 + h;
                ml[k] = __ldcg(&a.part_ml[at]);
                v[k] = __ldcg(reinterpret_cast<const float4*>(a.part_o + static_cast<long long>(at) * KV + c));
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (i0 + 8 * k < parts) blend(o, v[k], sum.add(ml[k]));
        }
        __syncthreads();  // the last task's sums have been read
        sum_s[warp][lane] = o;
        if (lane == 0) ml_s[warp] = make_float2(sum.m, sum.l);
        __syncthreads();
        if (warp) continue;
        for (int w = 1; w < 8; ++w) blend(o, sum_s[w][lane], sum.add(ml_s[w]));
        finish(h, c, o, sum);
    }
}

}  // namespace paged
}  // namespace mm
