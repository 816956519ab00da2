// Shared-prefix latent attention on the 5th-generation tensor cores, for [128 latent | 16 rope]
// and [512 latent | 32 rope] caches.
//
// Keys are the M side of both products, queries the N side:
//   S^T [128 keys x N queries] = K [128 x (kv + rope)] Q^T,     O^T [kv x N] += V^T [kv x keys] P^T,
// V being K's first kv columns, so one shared-memory tile of the cache is read by both products
// (K-major for S^T, MN-major for O^T) and a cache row crosses HBM once per block of N queries.
// A decode step has few queries per key (8 or 16 heads of a row; a group's rows x heads over its
// prefix): with queries on M, a 128-row tile would be mostly empty and the [M x kv] fp32
// accumulator would fill the whole tensor memory at kv = 512; with keys on M every tile is full
// and O^T takes kv / 128 x N columns (256 of 512 at N = 64).
//
// A work item is (block of N query rows, key range): one group's query rows over a range of its
// prefix, or one row's queries over a range of its suffix. CTAs are persistent and walk the items
// (tables of 32 at a time in shared memory, so no role waits for an item's lengths); barrier
// phases run on across items. Warps:
//   softmax    4 (N = 16) or 8 (N = 64, each four take 32 of the queries): thread = key
//              (tensor-memory lane). The running maximum is lazy: the first tile's maximum is the
//              reference, and a later tile whose weights stay below 2^8 times the largest of the first
//              uses it as it is, decided by one 4-warp vote; otherwise the column maxima are taken and
//              O^T and the sums are rescaled. Behind a reference of large magnitude (keys that are masked
//              by the lowest score) every tile looks at its maxima again, from its scores as they are.
//              A key's scale (e4m3) multiplies its latent scores and,
//              for the second product, its probabilities.
//              The second product takes the weights (probability, times the scale) as 16-bit values, each
//              rounded once, as the tensor cores' operand has to be; sums and statistics are fp32. So that
//              fp16 loses no weight to its range, the maximum is taken over the weights (score + log2 scale)
//              and stands at 2^6: small weights are in the normal range down to 2^-20 of the largest, large
//              ones reach 2^15.
//   producers  2 or 4: the item's queries, then per tile of KT keys the rope columns and kv / 128 pairs
//              of 64-column boxes (each pair its own warps) into rings of swizzled boxes. 16-bit caches come
//              by TMA; e4m3 codes are loaded D tiles ahead into registers and stored as 16-bit values
//              (exact). What the cache holds past the range is masked in S and never read by an O product.
//   fence      one warp passes each landed tile on to the asynchronous proxy: a proxy fence costs
//              about 100 ns, and in the loading threads it would wait for every load they have in
//              flight (measured: 1.7 instead of over 5 TB/s). It also takes a NaN or an infinity out of the
//              value rows that some tokens of a block see and others do not (drop_bad_rows).
//   results    4 (N = 16): an item's O^T and sums, joined with the prefix's share, to memory.
//   MMA        one thread issues tcgen05.mma. With KT = 64 the S^T product has M = 64, whose row r
//              is tensor-memory lane 32 (r / 16) + r % 16.
// Every mbarrier wait is bounded. After a wait that runs out the CTA asks for no more tiles and products and
// goes on without waiting (every loop is bounded, every access in bounds): its results are NaN, the wait is
// noted in latent_status, and the CTA ends once the copies and products that it had in flight have (waited for
// with a limit of their own).
//
// Measured on one B200. Cache loads: 296 rows of 1,024 positions, 512 + 32 wide, fp16, 68 us (4.8 TB/s of
// the 6.5 a copy reaches); one SM's ring holds ten pairs of boxes (160 KB). As e4m3 the same rows take 77 us
// for 55 % of the bytes: they are bound by the conversion. Products: 2,048 query rows over one prompt of
// 8,192, 75 us (472 TFLOP/s), the tensor pipe 34 % active over all SMs: the S product of a 64-key tile has
// M = 64, and two tiles fill the ring. (128 queries a block would fill the tensor memory at 512 columns with
// their fp32 O^T.)
#pragma once
#include <type_traits>

#include "shared_prefix.cuh"

namespace mm {
namespace spa {

__device__ int latent_status;  // DeviceError bits since they were last read (mm_latent_status)

// A CTA that gave up on a wait notes it and stays until the tiles that it asked for have landed (the phases
// of their barriers that are open; a phase that nothing is in lasts its limit, a quarter of a second): its shared memory
// is another CTA's after that. Out of line: the code is never run and costs the tile loops registers.
__device__ __noinline__ void end_after_timeout(uint64_t* tile_in, int n) {
    raise_error(&latent_status, kErrWaitTimeout);
    for (int i = 0; i < n; ++i) {
        const uint32_t open = mbar_try_wait(&tile_in[i], 0) ? 1 : 0;
        for (int k = 0; k < 1 << 16 && !mbar_try_wait(&tile_in[i], open); ++k) __nanosleep(256);
    }
}

// How a launch covers its items and where its partial results go.
struct TcArgs {
    Problem p;
    int suffix;        // 0: prefix items, 1: suffix items
    int splits, kps;   // key ranges per query block and keys per range (a multiple of 128)
    // partials of this launch: fp32 O [splits][query rows][kv] unnormalised, (max, sum) in base 2
    float* part_o;
    float2* part_ml;
    // a suffix launch writes the results of the rows whose suffix is one range (or empty) itself and
    // joins the prefix launch's partials (at most kMaxJoin ranges of prefix_kps keys) to them
    // (16-query blocks only: with 64 the registers are needed for the tiles)
    const float* pre_o;
    const float2* pre_ml;
    int prefix_kps;
    int overlap;       // the launch before this one is the call's own prefix launch: run beside it
    // a suffix launch of 16-query blocks, 512 wide, may divide the tiles of all its rows evenly over the
    // CTAs; a row cut where a CTA's share ends is left to the join kernel. Per row the first CTA and the number of
    // its parts (0: whole, the launch wrote its result); null: key ranges
    int2* pieces;
    int apart;         // the limits of a suffix block's tokens end at most this far apart
    int map_rows;      // 0: the cache's rows are one and the same (a row stride of zero), and so is the tensor maps'
};

constexpr int kTcMaxPlan = 512;   // entries of the shared plan (the items of runs of groups or rows)
constexpr int kTcTable = 32;      // items per shared table
constexpr int kMinSpan = 4;       // tiles of a CTA's share at least
constexpr int kMaxJoin = 4;       // prefix ranges a suffix launch joins itself
constexpr float kGrowth = 8.f;    // log2 of what a weight may grow over its reference
constexpr float kNear = 512.f;    // references up to here are subtracted with the scale's product
constexpr float kNoMax = -3.402823466e38f;  // running maximum before any key (finite: its exp2 is 0, never NaN)

// One work item.
struct Item {
    int q0, nq;       // query rows [q0, q0 + nq)
    int row;          // cache row
    int k0, nk, nt;   // first key, keys, tiles (0: nothing to attend)
    int split;        // key range (span: the CTA's slot of partials)
    int np;           // the prefix ranges to join to the result, -1: this item writes partials
};

template <int KV, int R, int N, bool Q8> struct TcCfg {
    static constexpr int NP = KV / 128;                    // 128-column pairs of boxes
    static constexpr int KT = KV == 512 ? 64 : 128;        // keys per tile
    static constexpr int kBox = KT * 128;                  // KT keys x 64 columns of 16 bits
    static constexpr int kPair = 2 * kBox;
    static constexpr int kRope = KT * R * 2;
    static constexpr int kRopeA = (kRope + 1023) / 1024 * 1024;
    static constexpr int kQBox = N * 128;
    static constexpr int kQ = 2 * NP * kQBox + N * R * 2;  // N query rows
    static constexpr int kQA = (kQ + 1023) / 1024 * 1024;
    // P^T: N = 64: one MN-major box [KT keys x 64 queries]; N = 16: K-major boxes of 64 keys
    static constexpr int kP = N == 64 ? KT * 128 : KT / 64 * 16 * 128;
    // CTAs per SM, and rings: queries, pairs, rope boxes, P buffers, O accumulators (what 227 KB
    // and 512 tensor memory columns hold)
    static constexpr int kCtas = KV == 128 && N == 16 ? 2 : 1;
    static constexpr int QB = KV == 512 && N == 64 ? 1 : 2;
    static constexpr int PS = KV == 512 ? (N == 64 ? 8 : 10) : (N == 64 ? 4 : 2);
    static constexpr int RS = KV == 512 ? (N == 64 ? 2 : 3) : PS;
    static constexpr int PB = 2;
    static constexpr int TS = 4;  // tiles announced: no fewer than the pair ring holds
    static constexpr int OB = KV == 512 && N == 64 ? 1 : 2;
    // tensor memory columns: two S buffers (e4m3: two more for the rope columns' share, which the
    // key's scale does not multiply), then the O accumulators
    static constexpr int kColS = 0, kColR = 2 * N, kColO = Q8 ? 4 * N : 2 * N;
    static constexpr int kCols = kColO + OB * NP * N;
    static constexpr int kTmem = kCols <= 64 ? 64 : kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
    // warps: softmax groups of four, producers, the MMA warp and the fence warp (N = 64: a whole
    // warpgroup for these two, so that registers can move between the roles)
    static constexpr int SG = N == 64 ? 2 : 1, NC = N / SG, SW = 4 * SG;
    static constexpr int PW = N == 64 || KV == 512 ? 4 : 2, PT = 32 * PW;
    // N = 16: four warps of their own write the results, while the softmax goes on with the next item
    // (N = 64: the softmax warps write them, the registers are needed there)
    static constexpr int EW = N == 16 ? 4 : 0;
    static constexpr int kThreads = 32 * (SW + PW + (N == 64 ? 4 : 2) + EW);
    // producer warps per pair of a tile
    static constexpr int WPP = PW / NP;
    // e4m3: 16-byte loads per tile and thread, tiles ahead in registers
    static constexpr int VPT = KT * 8 / (32 * WPP), D = KV == 128 && N == 64 ? 3 : 1;
    static constexpr int oPair = 0;
    static constexpr int oQ = oPair + PS * kPair;
    static constexpr int oRope = oQ + QB * kQA;
    static constexpr int oP = oRope + RS * kRopeA;
    static constexpr int oTab = oP + PB * kP;
    static constexpr int oF = oTab + kTcTable * 32;  // floats: m[N], corr[N], red[4][N], lim[N], up[N], base[N], mail[2][5][N], factor[5][N], limit[2] + 2
    static constexpr int oPlan = oF + (9 + (EW ? 15 : 0)) * N * 4 + 16;
    static constexpr int oBar = oPlan + (kTcMaxPlan + 1) * 4 + 12;
    static constexpr int kBars = QB + PS + 2 * TS + 4 + 2 * PB + 2 * OB + 4 + 1;
    static_assert(RS * NP >= PS && TS * NP >= PS, "the rope ring and the tile barriers outlast the pair ring");
    static constexpr int kSmem = oBar + kBars * 8 + 16 + 1024;  // + alignment of the base
    static_assert(kCtas * (kSmem + 1024) <= 228 * 1024 && kCols * kCtas <= 512, "shared and tensor memory");
};

// floor(log2 |s|) of an e4m3 key's scale, kept within what the weights' range needs: below 2^-40 a value is
// less than fp16 (and its share of a bf16 row) can show, above 2^100 probabilities would leave fp32.
__device__ __forceinline__ float scale_exponent(float s) {
    return static_cast<float>(min(max(static_cast<int>((__float_as_uint(s) >> 23) & 255) - 127, -40), 100));
}

// Swizzled byte offset of 16-byte chunk c of row r in a box of 128-, 64- or 32-byte rows.
__device__ __forceinline__ uint32_t sw128(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }
template <int R> __device__ __forceinline__ uint32_t sw_rope(int r, int c) {
    return R == 32 ? r * 64 + ((c ^ ((r >> 1) & 3)) << 4) : r * 32 + ((c ^ ((r >> 2) & 1)) << 4);
}
// Descriptor of a K-major rope box: 64-byte (R = 32) or 32-byte (R = 16) swizzle.
template <int R> __device__ __forceinline__ uint64_t rope_desc(uint32_t addr) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((addr >> 4) & 0x3FFF);
    d |= static_cast<uint64_t>(1) << 16;
    d |= static_cast<uint64_t>((8 * R * 2) >> 4) << 32;  // eight rows
    d |= 1ull << 46;
    d |= (R == 32 ? 4ull : 6ull) << 61;
    return d;
}

// One lane of the warp (the same one every time). Inside a branch on it the compiler knows that a
// single thread runs and keeps tcgen05.mma's descriptors in uniform registers; under lane == 0 it
// goes through the possible lanes for every instruction (about 95 cycles each, measured here).
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r));
    return r != 0;
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}

__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}

// The barrier counts this thread once its cp.async copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Barrier of the four warps of a softmax group, with and without an OR of a predicate.
__device__ __forceinline__ void soft_sync(int group) { asm volatile("bar.sync %0, 128;" ::"r"(group + 1) : "memory"); }
__device__ __forceinline__ bool soft_any(int group, bool p) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
        "bar.red.or.pred p, %2, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r)
        : "r"(static_cast<uint32_t>(p)), "r"(group + 1)
        : "memory");
    return r != 0;
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float (&v)[16]) {
    uint32_t r[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(v[i]);
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Column reductions over the 32 lanes (those that differ in the bits up to FIRST): each step folds half of
// the remaining columns into the other half's lane (31 shuffles for 32 values). Returns the column the lane
// ends up with; its result is v[0] (16 columns: both lanes of a pair hold it).
template <int FIRST = 16, int NC, class Op> __device__ __forceinline__ int fold_columns(float (&v)[NC], int lane, Op op) {
    int own = 0, w = NC;
#pragma unroll
    for (int o = FIRST; o > 0; o >>= 1) {
        if (w > 1) {
            w >>= 1;
            const bool up = lane & o;
#pragma unroll
            for (int i = 0; i < NC / 2; ++i)
                if (i < w) {
                    const float got = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + w], o);
                    v[i] = op(up ? v[i + w] : v[i], got);
                }
            if (up) own += w;
        } else {
            v[0] = op(v[0], __shfl_xor_sync(0xffffffffu, v[0], o));
        }
    }
    return own;
}

// The prefix ranges a suffix launch joins to row b's result, -1 when the row is left to the join
// kernel (several suffix ranges, or more than kMaxJoin prefix ranges).
__device__ __forceinline__ int direct_join(const Problem& p, int b, int suffix_kps, int prefix_kps) {
    if (suffix_length(p, b) > suffix_kps) return -1;
    const int np = (prefix_length(p, p.G > 0 ? group_of(p, b) : -1) + prefix_kps - 1) / prefix_kps;
    return np <= kMaxJoin ? np : -1;
}

// Keys of a row's suffix of `len` that its query row u (< T * H) sees.
__device__ __forceinline__ int seen_by(const Problem& p, int len, int u) { return max(len - (p.T - 1 - u / p.H), 0); }

// A launch's items come from units: groups (prefix) or rows (suffix). Unit u holds `blocks` blocks of
// N query rows from q0 on and attends over `len` keys in `ranges` key ranges (a suffix row of a
// direct result keeps one, however empty).
struct Unit {
    int q0, nq, len, blocks, ranges, np;
};
template <int N> __device__ __forceinline__ Unit get_unit(const TcArgs& a, int u) {
    const Problem& p = a.p;
    const int th = p.T * p.H;
    Unit r;
    r.np = -1;
    if (a.suffix) {
        r.q0 = u * th;
        r.nq = th;
        r.len = suffix_length(p, u);
        if (N == 16) r.np = direct_join(p, u, a.kps, a.prefix_kps);
    } else {
        const int b0 = min(max(p.group_start[u], 0), p.B), b1 = min(max(p.group_start[u + 1], b0), p.B);
        r.q0 = b0 * th;
        r.nq = min(b1 - b0, p.max_group) * th;
        r.len = r.nq > 0 ? prefix_length(p, u) : 0;
    }
    r.blocks = (r.nq + N - 1) / N;
    r.ranges = max((r.len + a.kps - 1) / a.kps, r.np >= 0 ? 1 : 0);
    return r;
}

template <int N> __device__ __forceinline__ int unit_items(const TcArgs& a, int u) {
    const Unit r = get_unit<N>(a, u);
    return r.blocks * r.ranges;
}

// Item idx of the launch. With a plan (shared: cumulative items of runs of `step` units) the items are
// dense, so that they spread evenly over the CTAs whatever the lengths; without one (a suffix launch
// of one range per row, where there is none to skip) every unit has `per` blocks.
template <int N, int KT, bool CAUSAL>
__device__ __forceinline__ Item get_item(const TcArgs& a, const int* plan, int units, int step, int per, int idx) {
    int u, local;
    if (plan) {
        int lo = 0, hi = (units + step - 1) / step;  // the run with plan[lo] <= idx < plan[lo + 1]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (plan[mid] <= idx) lo = mid;
            else hi = mid;
        }
        u = lo * step;
        local = idx - plan[lo];
        if (step > 1) {
            const int last = min(units, u + step) - 1;
#pragma unroll 1
            for (int n; u < last && local >= (n = unit_items<N>(a, u)); ++u) local -= n;
        }
    } else {
        u = idx / per;
        local = idx - u * per;
    }
    const Unit r = get_unit<N>(a, u);
    const int ranges = plan ? r.ranges : 1;
    const int block = local / ranges;
    Item it;
    it.split = local - block * ranges;
    it.row = u;
    it.q0 = r.q0 + block * N;
    it.nq = max(0, min(N, r.nq - block * N));
    it.k0 = it.split * a.kps;
    // a block ends at the last key that its last query sees (16-query blocks hold a row's last token)
    int len = r.len;
    if (N == 64 && CAUSAL && a.suffix && it.nq > 0) len = seen_by(a.p, len, block * N + it.nq - 1);
    it.nk = it.nq > 0 ? max(0, min(a.kps, len - it.k0)) : 0;
    it.nt = (it.nk + KT - 1) / KT;
    it.np = it.split == 0 ? r.np : -1;
    return it;
}

// Even shares of a suffix launch's work: a row weighs its tiles and one more (its queries and results),
// CTA c has the weights [c span, (c + 1) span) of the rows in line. What a share holds of a row is one
// item; a cut row's first part is its CTA's last item (slot 2 c + 1), a later part its CTA's first (slot 2 c).
template <int KT> __device__ __forceinline__ int row_weight(const Problem& p, int u) {
    return (suffix_length(p, u) + KT - 1) / KT + 1;
}
// The row that holds weight w; before: the weight of the rows ahead of it.
template <int KT>
__device__ __forceinline__ int row_at(const Problem& p, const int* plan, int units, int step, int w, int& before) {
    int lo = 0, hi = (units + step - 1) / step;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (plan[mid] <= w) lo = mid;
        else hi = mid;
    }
    int u = lo * step;
    before = plan[lo];
    const int last = min(units, u + step) - 1;
    for (int n; u < last && before + (n = row_weight<KT>(p, u)) <= w; ++u) before += n;
    return u;
}
template <int KT>
__device__ __forceinline__ Item span_item(const TcArgs& a, const int* plan, int step, int span, int u) {
    const Problem& p = a.p;
    int before = plan[u / step];
    for (int v = u / step * step; v < u; ++v) before += row_weight<KT>(p, v);
    const int th = p.T * p.H, len = suffix_length(p, u), nt = (len + KT - 1) / KT;
    const int w0 = static_cast<int>(blockIdx.x) * span, from = min(max(w0 - before, 0), nt), to = min(w0 + span - before, nt);
    const bool whole = before >= w0 && to == nt;
    if (whole || (to == nt && from < nt)) {  // the share that ends the row notes its parts
        const int first = before / span;
        a.pieces[u] = make_int2(first, whole ? 0 : static_cast<int>(blockIdx.x) - first + 1);
    }
    Item it;
    it.row = u;
    it.q0 = u * th;
    it.nq = th;
    it.k0 = from * KT;
    it.nt = to - from;
    it.nk = min(len - it.k0, it.nt * KT);
    it.split = 2 * static_cast<int>(blockIdx.x) + (from == 0 ? 1 : 0);
    it.np = whole ? (prefix_length(p, p.G > 0 ? group_of(p, u) : -1) + a.prefix_kps - 1) / a.prefix_kps : -1;
    return it;
}

// Position in a ring of S barriers: the slot and its phase parity.
template <int S> struct Ring {
    int i = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next() {
        if (++i == S) {
            i = 0;
            phase ^= 1;
        }
    }
    __device__ __forceinline__ void skip(int n) {
        if ((i += n) >= S) {
            i -= S;
            phase ^= 1;
        }
    }
};

// Cursor over the tiles of a table's items that have any.
struct Cursor {
    const Item* tab;
    int n, at, j, nt;
    __device__ __forceinline__ Cursor(const Item* t, int count) : tab(t), n(count), at(-1), j(0), nt(0) { next_item(); }
    __device__ __forceinline__ void next_item() {
        j = 0;
        do {
            if (++at >= n) return;
            nt = tab[at].nt;
        } while (nt == 0);
    }
    __device__ __forceinline__ bool valid() const { return at < n; }
    __device__ __forceinline__ bool last() const { return j == nt - 1; }
    __device__ __forceinline__ const Item& item() const { return tab[at]; }
    __device__ __forceinline__ void next() {
        if (++j == nt) next_item();
    }
};

// Value rows [from, to) of a landed tile are seen by some of the block's queries and masked for others, and a
// probability of zero times a NaN or an infinity is a NaN: a row that holds one becomes zeros, with a NaN in
// its rope columns, which only the scores read. So the queries that see it get NaN, and no other.
template <bool kBf16> __device__ __forceinline__ bool bad_chunk(const uint4& v) {  // 16-bit values of it
    constexpr uint32_t kExp = kBf16 ? 0x7F80u : 0x7C00u;
    auto odd = [](uint32_t w) { return (w & kExp) == kExp || (w >> 16 & kExp) == kExp; };
    return odd(v.x) || odd(v.y) || odd(v.z) || odd(v.w);
}
// 16-byte chunk e of value row r; the tile's pairs begin at first_pair of the ring.
template <class C> __device__ __forceinline__ uint4* value_chunk(uint8_t* pairs, int first_pair, int r, int e) {
    int pair = first_pair + (e >> 4);
    if (pair >= C::PS) pair -= C::PS;
    return reinterpret_cast<uint4*>(pairs + pair * C::kPair + ((e >> 3) & 1) * C::kBox + sw128(r, e & 7));
}
template <class C, int R, bool kBf16>
__device__ __forceinline__ void drop_bad_rows(uint8_t* pairs, int first_pair, uint8_t* rope, int from, int to, int lane) {
    for (int r = from; r < to; ++r) {
        bool bad = false;
        for (int e = lane; e < 16 * C::NP; e += 32) bad |= bad_chunk<kBf16>(*value_chunk<C>(pairs, first_pair, r, e));
        if (!__any_sync(0xffffffffu, bad)) continue;
        for (int e = lane; e < 16 * C::NP; e += 32) *value_chunk<C>(pairs, first_pair, r, e) = make_uint4(0, 0, 0, 0);
        if (lane < R / 8) *reinterpret_cast<uint4*>(rope + sw_rope<R>(r, lane)) = make_uint4(~0u, ~0u, ~0u, ~0u);
    }
}

// CAUSAL: a call of more than one token a row, whose last positions are masked for some of them in the suffix
// launch. A kernel of its own, because the others pay for code that they do not run (2,048 rows, 128 + 16 wide:
// 64.0 us in one kernel with it, 59.4 apart). Both launches of a call use the same one: two kernels that spill
// registers do not run beside each other (143 rows of 4 tokens, e4m3: 22.7 us with a prefix launch of the
// other one, 15.3).
template <int KV, int R, int N, typename T, bool Q8, bool CAUSAL>
__global__ void __launch_bounds__(TcCfg<KV, R, N, Q8>::kThreads, TcCfg<KV, R, N, Q8>::kCtas)
    shared_prefix_tc_kernel(const __grid_constant__ TcArgs a, const __grid_constant__ CUtensorMap map_tile,
                            const __grid_constant__ CUtensorMap map_block, const __grid_constant__ CUtensorMap map_rope) {
    using C = TcCfg<KV, R, N, Q8>;
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    constexpr int NC = C::NC, KT = C::KT;
    extern __shared__ uint8_t tc_smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(tc_smem_raw) + 1023) &
                                               ~static_cast<uintptr_t>(1023));
    Item* table = reinterpret_cast<Item*>(smem + C::oTab);
    float* m_s = reinterpret_cast<float*>(smem + C::oF);
    float* corr_s = m_s + N;
    float* red_s = corr_s + N;  // [4][N]
    int* lim_s = reinterpret_cast<int*>(red_s + 4 * N);
    float* up_s = red_s + 5 * N;
    float* base_s = up_s + N;        // the part of m that a tile's scores start from
    float* mail_s = base_s + N;      // [2][5][N] an item's sums (one row per softmax warp) and maxima
    float* fac_s = mail_s + 10 * N;  // [5][N]
    float* over_s = reinterpret_cast<float*>(smem + C::oPlan - 16);  // [2] scores above it make a group look at its maxima
    int* plan_s = reinterpret_cast<int*>(smem + C::oPlan);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::oBar);
    uint64_t* q_empty = bars;                    // [QB] the item's S products have read Q
    uint64_t* pair_empty = q_empty + C::QB;      // [PS] O products done with the pair
    uint64_t* tile_in = pair_empty + C::PS;      // [TS] the producer threads
    uint64_t* tile_full = tile_in + C::TS;       // [TS] the fence warp: the tile's boxes can be read
    uint64_t* s_full = tile_full + C::TS;        // [2]
    uint64_t* s_free = s_full + 2;               // [2] the softmax warps
    uint64_t* p_full = s_free + 2;               // [PB] the softmax warps
    uint64_t* p_free = p_full + C::PB;           // [PB] the tile's O products are complete
    uint64_t* o_full = p_free + C::PB;           // [OB]
    uint64_t* o_free = o_full + C::OB;           // [OB] the warps that write the results
    uint64_t* e_full = o_free + C::OB;           // [2] the softmax warps: an item's sums and maxima
    uint64_t* e_free = e_full + 2;               // [2] the result warps
    uint64_t* ended = e_free + 2;                // after a wait that ran out: the products in flight are complete
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kBars);
    int* bad_s = reinterpret_cast<int*>(tmem_slot + 1);
    const Problem& p = a.p;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int th = p.T * p.H;
    constexpr int kMmaWarp = C::SW + C::PW, kFenceWarp = kMmaWarp + 1, kResultWarp = kMmaWarp + (C::EW ? 2 : 4);

    if (warp == kMmaWarp) {
        if (lane == 0) {
            for (int i = 0; i < C::QB; ++i) mbar_init(&q_empty[i], 1);
            for (int i = 0; i < C::PS; ++i) mbar_init(&pair_empty[i], 1);
            for (int i = 0; i < C::TS; ++i) { mbar_init(&tile_in[i], C::PT + (Q8 ? C::PW : C::NP)); mbar_init(&tile_full[i], 1); }
            for (int i = 0; i < 2; ++i) { mbar_init(&s_full[i], 1); mbar_init(&s_free[i], C::SW); }
            for (int i = 0; i < C::PB; ++i) { mbar_init(&p_full[i], C::SW); mbar_init(&p_free[i], 1); }
            for (int i = 0; i < C::OB; ++i) { mbar_init(&o_full[i], 1); mbar_init(&o_free[i], C::EW ? C::EW : C::SW); }
            for (int i = 0; i < 2; ++i) { mbar_init(&e_full[i], C::SW); mbar_init(&e_free[i], 4); }
            mbar_init(ended, 1);
            *bad_s = 0;
            fence_mbar_init();
        }
        __syncwarp();
        tmem_alloc(tmem_slot, C::kTmem);
        tmem_relinquish();
    }
    // Beside its own prefix launch a suffix launch starts at once: that launch lets its dependents
    // begin only after it has itself waited for everything before it. Its partials are waited for
    // where they are read.
    if (!a.overlap) pdl_wait();
    pdl_launch_dependents();
    const int units = a.suffix ? p.B : p.G;
    const int per = ((a.suffix ? th : p.max_group * th) + N - 1) / N;
    constexpr bool kShares = KV == 512 && N == 16;  // (128 wide: the registers of two CTAs per SM are needed)
    const int* plan = nullptr;
    int items = units * per;
    const int step = (units + kTcMaxPlan - 1) / kTcMaxPlan;
    bool spans = kShares && a.pieces;
    if (spans || a.splits > 1 || !a.suffix) {
        plan = plan_s;
        const int runs = (units + step - 1) / step;
        for (int i = tid; i < runs; i += C::kThreads) {
            int n = 0;
            if (kShares && spans) {
                for (int u = i * step; u < min(units, (i + 1) * step); ++u) n += row_weight<KT>(p, u);
            } else {
                n = unit_items<N>(a, i * step);
#pragma unroll 1
                for (int u = i * step + 1; u < min(units, (i + 1) * step); ++u) n += unit_items<N>(a, u);
            }
            plan_s[i + 1] = n;
        }
        __syncthreads();
        if (warp == 0) {
            int base = 0;
            for (int u0 = 0; u0 < runs; u0 += 32) {
                int v = u0 + lane < runs ? plan_s[u0 + lane + 1] : 0;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int w = __shfl_up_sync(0xffffffffu, v, o);
                    if (lane >= o) v += w;
                }
                if (u0 + lane < runs) plan_s[u0 + lane + 1] = base + v;
                base += __shfl_sync(0xffffffffu, v, 31);
            }
            if (lane == 0) plan_s[0] = 0;
        }
        __syncthreads();
        items = plan_s[runs];
    }
    // Shares, or the rows one by one in turn, which needs no join and serves rows of like lengths: by the
    // fullest CTA's rows against the mean, shares from 1.25 on. 512 + 32 wide, us in turn / in shares, fp16
    // and e4m3:
    //   136 rows of about 1,000, spread (fullest over mean 1.06, 1.25, 1.44, 1.75, 2.06)
    //     38.4 / 44.6, 41.8 / 43.8, 44.6 / 43.6, 51.4 / 44.6, 56.1 / 44.0
    //     41.9 / 46.1, 47.6 / 46.4, 51.5 / 47.0, 60.9 / 47.7, 69.3 / 47.4
    //   250, 600, 340, 300, 170 rows of 700 (1.14, 1.22, 1.29, 1.44, 1.71)
    //     49.2 / 50.8, 105.4 / 98.4, 68.0 / 63.5, 65.6 / 58.5, 47.0 / 40.1
    //     57.4 / 57.6, 121.5 / 114.3, 79.3 / 72.0, 76.0 / 65.8, 52.4 / 41.8
    int span = 0;
    if (kShares && spans) {
        int* bins = reinterpret_cast<int*>(table);  // free until the first table
        const int grid = static_cast<int>(gridDim.x);
        int most = 0;
        if (grid <= kTcTable * 8) {
            for (int i = tid; i < grid; i += C::kThreads) bins[i] = 0;
            __syncthreads();
            for (int u = tid; u < units; u += C::kThreads) atomicAdd(&bins[u % grid], row_weight<KT>(p, u));
            __syncthreads();
            for (int i = lane; i < grid; i += 32) most = max(most, bins[i]);
            most = __reduce_max_sync(0xffffffffu, most);
        }
        span = max((items + grid - 1) / grid, kMinSpan);
        if (most > 0 && 4 * most < 5 * span) {
            spans = false;
            plan = nullptr;
            items = units;
        } else if (tid < 2) {
            // the first row of the share and the row after its last
            const int w = min((static_cast<int>(blockIdx.x) + tid) * span, items) - tid;
            int before, u = units;
            if (w >= 0 && w < items) u = row_at<KT>(p, plan, units, step, w, before) + tid;
            plan_s[kTcMaxPlan + 1 + tid] = u;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int mine = kShares && spans ? max(plan_s[kTcMaxPlan + 2] - plan_s[kTcMaxPlan + 1], 0)
                           : blockIdx.x < items ? (items - blockIdx.x + gridDim.x - 1) / gridDim.x : 0;
    const lat::CacheView& cv = a.suffix ? p.suffix : p.prefix;
    bool ok = true;
    // a wait that ran out is recorded once; later waits of this thread are skipped
    const bool causal = CAUSAL && a.suffix;  // the last positions are masked for some tokens
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (ok && !mbar_wait_bounded(bar, parity, nullptr)) {
            ok = false;
            *reinterpret_cast<volatile int*>(bad_s) = 1;
        }
    };
    // The next table of this CTA's items; every thread of the CTA comes here for each table. The first
    // softmax warp builds it (only its branch holds the code and the registers for it).
    auto next_table = [&](int base, auto builds) {
        if (base > 0) __syncthreads();
        if constexpr (decltype(builds)::value) {
            if (tid < kTcTable && base + tid < mine) {
                if (kShares && spans) {
                    table[tid] = span_item<KT>(a, plan, step, span, plan_s[kTcMaxPlan + 1] + base + tid);
                } else {
                    const Item it = get_item<N, KT, CAUSAL>(a, plan, units, step, per, blockIdx.x + (base + tid) * gridDim.x);
                    table[tid] = it;
                    if (kShares && a.pieces) a.pieces[it.row] = make_int2(0, 0);
                }
            }
        }
        __syncthreads();
        return min(kTcTable, mine - base);
    };

    if (warp >= C::SW && warp < kMmaWarp) {
        // ------------------------------------------------------------ producers
        if constexpr (Q8 && N == 64) asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
        const int pt = tid - 32 * C::SW;  // 0..PT - 1
        uint8_t* sQ = smem + C::oQ;
        uint8_t* sPair = smem + C::oPair;
        uint8_t* sRope = smem + C::oRope;
        // eight lanes per query row and 64-column box
        auto load_q = [&](const Item& it, int qb) {
            uint8_t* q = sQ + qb * C::kQA;
            const int c = pt & 7;
            // query rows one q_head apart (contiguous q, or one token per row with rows in line): no divisions
            const bool line = p.q_tok == p.H * p.q_head && p.q_row == th * p.q_head;
#pragma unroll 1
            for (int n = pt >> 3; n < N; n += C::PT / 8) {
                const bool in = n < it.nq;
                const int r = it.q0 + (in ? n : 0);
                long long off = r * p.q_head;
                if (!line) {
                    const int b = r / th, u = r - b * th, t = u / p.H;
                    off = b * p.q_row + t * p.q_tok + (u - t * p.H) * p.q_head;
                }
                const T* src = static_cast<const T*>(p.q) + off + c * 8;
                uint8_t* dst = q + sw128(n, c);
#pragma unroll
                for (int x = 0; x < 2 * C::NP; ++x) cp_async16(dst + x * C::kQBox, src + x * 64, in);
                if (c < R / 8) cp_async16(q + 2 * C::NP * C::kQBox + sw_rope<R>(n, c), src + KV, in);
            }
        };
        auto load_rope = [&](const Item& it, int j, int slot) {
            constexpr int kChunks = R / 8, kRows = C::PT / kChunks;
            const int c = pt % kChunks, r0 = pt / kChunks, left = it.nk - j * KT;
            uint8_t* d = sRope + slot * C::kRopeA;
            const long long ps = 2 * cv.rope_pos_stride;
            const uint8_t* src = cv.rope + 2 * (it.row * cv.rope_row_stride) + (it.k0 + j * KT) * ps + c * 16;
#pragma unroll
            for (int r = r0; r < KT; r += kRows) cp_async16(d + sw_rope<R>(r, c), src + (r < left ? r : 0) * ps, r < left);
        };
        // WPP warps per pair of a tile, so that the pairs' waits and copies run side by side; a tile
        // (and the item's queries with its first) is announced by one arrival per thread (e4m3: and warp). The rope
        // ring holds at least the tiles of the pair ring: its boxes are free when the pair's are.
        const int pw = warp - C::SW, own = pw / C::WPP, sub = pw % C::WPP;
        Ring<C::QB> rq;
        Ring<C::RS> rr;
        Ring<C::TS> rt;
        Ring<C::PS> rp;
        rp.i = own;
        auto begin_tile = [&](const Item& it, int j) {
            if (j == 0) {
                wait(&q_empty[rq.i], rq.phase ^ 1);
                load_q(it, rq.i);
                rq.next();
            }
            wait(&pair_empty[rp.i], rp.phase ^ 1);
        };
        auto end_tile = [&] {
            rr.next();
            cp_async_arrive(&tile_in[rt.i]);
            if (Q8) {  // the warp's converted codes
                __syncwarp();
                if (lane == 0) mbar_arrive(&tile_in[rt.i]);
            }
            rt.next();
            rp.skip(C::NP);
        };
        if constexpr (!Q8) {
            for (int base = 0; base < mine; base += kTcTable) {
                const int count = next_table(base, std::false_type());
                for (Cursor c(table, count); c.valid(); c.next()) {
                    const Item& it = c.item();
                    begin_tile(it, c.j);
                    const int left = it.nk - c.j * KT;
                    // one thread per pair asks for its two boxes, a range's last tile in the blocks of 32
                    // positions that the range reaches, and the first pair's for the rope columns
                    if (sub == 0 && elect_one() && ok) {
                        const int nb = min((left + 31) >> 5, KT / 32), pos = it.k0 + c.j * KT, row = it.row * a.map_rows;
                        uint64_t* bar = &tile_in[rt.i];
                        mbar_arrive_expect_tx(bar, nb * (2 * 4096 + (own == 0 ? 64 * R : 0)));
                        uint8_t* box = sPair + rp.i * C::kPair;
                        if (left >= KT) {
                            tma_load_3d(box, &map_tile, bar, own * 128, pos, row);
                            tma_load_3d(box + C::kBox, &map_tile, bar, own * 128 + 64, pos, row);
                        } else {
#pragma unroll 1
                            for (int k = 0; k < nb; ++k) {
                                tma_load_3d(box + k * 4096, &map_block, bar, own * 128, pos + 32 * k, row);
                                tma_load_3d(box + C::kBox + k * 4096, &map_block, bar, own * 128 + 64, pos + 32 * k, row);
                            }
                        }
                        if (own == 0) {
#pragma unroll 1
                            for (int k = 0; k < nb; ++k)
                                tma_load_3d(sRope + rr.i * C::kRopeA + k * 64 * R, &map_rope, bar, KV, pos + 32 * k, row);
                        }
                    }
                    if (__any_sync(0xffffffffu, !ok)) break;
                    end_tile();
                }
            }
        } else {
            // codes D tiles ahead in registers, asked for again as soon as they have been converted
            constexpr int D = C::D, kRows = 4 * C::WPP;
            uint4 v[D][C::VPT];
            const int cc = lane & 7, r0 = (lane >> 3) + 4 * sub;  // 16-byte chunk of the pair's 128 codes, first row
            const long long rstep = kRows * cv.pos_stride;
            auto fetch = [&](uint4 (&x)[C::VPT], const Cursor& c) {
                const Item& it = c.item();
                const int left = it.nk - c.j * KT - r0;
                const uint8_t* src = cv.latent + it.row * cv.row_stride + (it.k0 + c.j * KT + r0) * cv.pos_stride + own * 128 + cc * 16;
#pragma unroll
                for (int k = 0; k < C::VPT; ++k) {
                    x[k] = kRows * k < left ? __ldg(reinterpret_cast<const uint4*>(src)) : make_uint4(0, 0, 0, 0);
                    src += rstep;
                }
            };
            for (int base = 0; base < mine; base += kTcTable) {
                const int count = next_table(base, std::false_type());
                Cursor lc(table, count), sc(table, count);
#pragma unroll
                for (int d = 0; d < D; ++d)
                    if (lc.valid()) {
                        fetch(v[d], lc);
                        lc.next();
                    }
                while (sc.valid()) {
#pragma unroll
                    for (int d = 0; d < D; ++d) {
                        if (sc.valid()) {
                            begin_tile(sc.item(), sc.j);
                            load_rope(sc.item(), sc.j, rr.i);
                            uint8_t* dst = sPair + rp.i * C::kPair + (cc >> 2) * C::kBox;
#pragma unroll
                            for (int k = 0; k < C::VPT; ++k) {
                                const int r = r0 + kRows * k;
                                const uint32_t w[4] = {v[d][k].x, v[d][k].y, v[d][k].z, v[d][k].w};
                                uint32_t o[8];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    o[2 * e] = lat::e4m3x2_to<T>(static_cast<uint16_t>(w[e] & 0xffff));
                                    o[2 * e + 1] = lat::e4m3x2_to<T>(static_cast<uint16_t>(w[e] >> 16));
                                }
                                *reinterpret_cast<uint4*>(dst + sw128(r, (2 * cc) & 7)) = make_uint4(o[0], o[1], o[2], o[3]);
                                *reinterpret_cast<uint4*>(dst + sw128(r, (2 * cc + 1) & 7)) = make_uint4(o[4], o[5], o[6], o[7]);
                            }
                            end_tile();
                            if (lc.valid()) {
                                fetch(v[d], lc);
                                lc.next();
                            }
                            sc.next();
                        }
                    }
                }
            }
        }
        cp_async_wait<0>();
    } else if (warp >= kMmaWarp && warp < kResultWarp) {
        // ------------------------------------------------------------ tensor-core products
        if constexpr (Q8 && N == 64) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        const uint32_t id_s = umma_idesc_f16(kBf16, false, false, KT, N);
        const uint32_t id_o = umma_idesc_f16(kBf16, true, N == 64, 128, N);
        const uint32_t aPair = smem_u32(smem + C::oPair), aQ = smem_u32(smem + C::oQ), aR = smem_u32(smem + C::oRope),
                       aP = smem_u32(smem + C::oP);
        // descriptors advance by address / 16 (shared memory ends below 2^18, so no field overflows)
        const uint64_t kd = umma_desc_sw128(aPair, 16, 1024), vd = umma_desc_sw128(aPair, C::kBox, 1024);
        // positions of the S side and of the O side, and how many tiles S is ahead. This thread's
        // instructions are on the path of every tile: positions are kept instead of computed, and a
        // tile's boxes are waited for as one.
        Ring<C::PS> sp, op;
        Ring<C::RS> sr;
        Ring<C::TS> st;
        Ring<C::QB> sq;
        Ring<2> ss;
        Ring<C::PB> pb;
        Ring<C::OB> ob;
        int ahead = 0;
        auto issue_s = [&](Cursor& c) {
            const uint32_t q = aQ + sq.i * C::kQA, d = tmem + C::kColS + ss.i * N;
            tc_fence_after();
            {
                const uint64_t ka = rope_desc<R>(aR + sr.i * C::kRopeA), qa = rope_desc<R>(q + 2 * C::NP * C::kQBox);
                const uint32_t dr = Q8 ? tmem + C::kColR + ss.i * N : d;
#pragma unroll
                for (int k = 0; k < R / 16; ++k) tc_mma_f16(dr, ka + k * 2, qa + k * 2, id_s, k ? 1u : 0u);
            }
            sr.next();
            const uint64_t qd = umma_desc_sw128(q, 16, 1024);
#pragma unroll
            for (int i = 0; i < C::NP; ++i) {
                const uint64_t ka = kd + static_cast<uint32_t>(sp.i * (C::kPair >> 4));
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    tc_mma_f16(d, ka + ((k >> 2) * C::kBox + (k & 3) * 32) / 16,
                               qd + (2 * i * C::kQBox + (k >> 2) * C::kQBox + (k & 3) * 32) / 16, id_s,
                               Q8 && i == 0 && k == 0 ? 0u : 1u);
                sp.next();
            }
            tc_commit(&s_full[ss.i]);
            ss.next();
            st.next();
            if (c.last()) {
                tc_commit(&q_empty[sq.i]);
                sq.next();
            }
            ++ahead;
            c.next();
        };
        auto issue_o = [&](Cursor& c) {
            if (c.j == 0) wait(&o_free[ob.i], ob.phase ^ 1);
            tc_fence_after();
            const uint64_t pa = umma_desc_sw128(aP + pb.i * C::kP, N == 64 ? C::kBox : 16, 1024);
            const uint32_t d = tmem + C::kColO + ob.i * C::NP * N;
            const uint32_t first = c.j ? 1u : 0u;
            const int left = c.item().nk - c.j * KT;
#pragma unroll
            for (int i = 0; i < C::NP; ++i) {
                const uint64_t va = vd + static_cast<uint32_t>(op.i * (C::kPair >> 4));
#pragma unroll
                for (int k = 0; k < KT / 16; ++k) {
                    if (16 * k >= left) break;  // keys past the range
                    // V^T MN-major: 16 keys = 2,048 B down a box, the next 64 columns one box on
                    tc_mma_f16(d + i * N, va + k * 128, pa + (N == 64 ? k * 128 : ((k >> 2) * 2048 + (k & 3) * 32) / 16), id_o,
                               k ? 1u : first);
                }
                tc_commit(&pair_empty[op.i]);
                op.next();
            }
            tc_commit(&p_free[pb.i]);
            pb.next();
            if (c.last()) {
                tc_commit(&o_full[ob.i]);
                ob.next();
            }
            --ahead;
            c.next();
        };
        Ring<C::TS> ft;
        Ring<C::PS> fp;
        Ring<C::RS> fr;
        int shown = 0x7fffffff;  // keys of the item that all of its queries see
        for (int base = 0; base < mine; base += kTcTable) {
            const int count = next_table(base, std::false_type());
            if (warp == kFenceWarp) {
                // what has been written in the generic proxy (copies, converted codes) becomes readable by
                // the products. TMA brings whole blocks of positions, whatever lies past the range: the rows
                // that the O products still read are cleared first (a probability of zero times a NaN
                // would be one).
                for (Cursor c(table, count); c.valid(); c.next(), ft.next()) {
                    if (causal && c.j == 0) {
                        const Item& it = c.item();
                        shown = seen_by(p, suffix_length(p, it.row), it.q0 - it.row * th) - it.k0;
                    }
                    wait(&tile_in[ft.i], ft.phase);
                    const int left = c.item().nk - c.j * KT;
                    if (!Q8 && left < KT && (left & 15)) {
                        // the O products read whole steps of 16 keys: rows [left, next multiple of 16)
                        const int rows = 16 - (left & 15);
                        const uint4 zero = make_uint4(0, 0, 0, 0);
                        Ring<C::PS> z = fp;
#pragma unroll 1
                        for (int i = 0; i < 2 * C::NP; ++i) {
                            uint4* box = reinterpret_cast<uint4*>(smem + C::oPair + z.i * C::kPair + (i & 1) * C::kBox) + left * 8;
                            for (int e = lane; e < rows * 8; e += 32) box[e] = zero;
                            if (i & 1) z.next();
                        }
                    }
                    if constexpr (CAUSAL) {
                        const int to = min(left, KT), from = min(max(shown - c.j * KT, 0), to), chunks = (to - from) * 16 * C::NP;
                        bool bad = false;
                        __syncwarp();
                        for (int e = lane; e < chunks; e += 32)
                            bad |= bad_chunk<kBf16>(*value_chunk<C>(smem + C::oPair, fp.i, from + e / (16 * C::NP), e % (16 * C::NP)));
                        if (__any_sync(0xffffffffu, bad))
                            drop_bad_rows<C, R, kBf16>(smem + C::oPair, fp.i, smem + C::oRope + fr.i * C::kRopeA, from, to, lane);
                        fr.next();
                    }
                    fp.skip(C::NP);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&tile_full[ft.i]);
                }
            }
            if (warp == kMmaWarp && elect_one()) {
                Cursor cs(table, count), co(table, count);
                // a tile's O when its probabilities are there, else the next tile's S when its boxes are:
                // neither waits behind the other
                int polls = 0;
                while (ok && co.valid()) {
                    if (ahead > 0 && mbar_test(&p_full[pb.i], pb.phase)) {
                        issue_o(co);
                        polls = 0;
                    } else if (ahead < 2 && cs.valid() && mbar_test(&tile_full[st.i], st.phase) &&
                               mbar_test(&s_free[ss.i], ss.phase ^ 1)) {
                        issue_s(cs);
                        polls = 0;
                    } else if (++polls > (1 << 24)) {
                        ok = false;
                        *reinterpret_cast<volatile int*>(bad_s) = 1;
                    }
                }
                if (!ok) {  // the products in flight end before the CTA does
                    tc_commit(ended);
                    mbar_wait_bounded(ended, 0, nullptr);
                }
            }
            __syncwarp();
        }
    } else if (warp < C::SW) {
        // ------------------------------------------------------------ softmax (N = 64: and results)
        const int group = warp >> 2, gw = warp & 3, gt = tid & 127;  // gt: tensor-memory lane
        const int c0 = group * NC;                                   // first query column of the group
        // the key this lane's scores belong to (64-key tiles: the lower half of each warp)
        const int kt = KT == 128 ? gt : gw * 16 + lane;
        const bool live = KT == 128 || lane < 16;
        const uint32_t lane_base = tmem + (static_cast<uint32_t>(gw * 32) << 16);
        const float cs = p.scale * 1.4426950408889634f;
        const long long rows = static_cast<long long>(p.B) * th;
        const float* base_c = base_s + c0;
        // log2 of the largest weight when its reference is taken
        constexpr float kLift = kBf16 ? 0.f : 6.f;
        int tile = 0, item = 0;
        Ring<2> eb;
        for (int base = 0; base < mine; base += kTcTable) {
            const int count = next_table(base, std::true_type());
            for (int e0 = 0; e0 < count; ++e0) {
                const Item it = table[e0];
                if (it.nt == 0 && (N != 16 || it.np < 0)) continue;
                const int nq = min(it.nq - c0, NC);  // the group's queries (none: <= 0)
                float l[NC];
#pragma unroll
                for (int n = 0; n < NC; ++n) l[n] = 0.f;
                // keys of the item each query sees; the tokens of a suffix end one position apart
                soft_sync(group);  // the previous item's readers of m_s, lim_s and red_s are done
                if (gt == 0) over_s[group] = kLift + kGrowth;
                if (gt < NC) {
                    m_s[c0 + gt] = base_s[c0 + gt] = 0.f;
                    if (causal) {
                        const int t = min((it.q0 + c0 + gt - it.row * th) / p.H, p.T - 1);
                        lim_s[c0 + gt] = min(it.nk, suffix_length(p, it.row) - (p.T - 1 - t) - it.k0);
                    }
                }
                soft_sync(group);
                const int lim_min = causal ? it.nk - a.apart : it.nk;
                const float* ks_row = Q8 ? cv.scale + it.row * cv.scale_row_stride + it.k0 : nullptr;
                float ks_next = 1.f;
                if (Q8 && live && kt < it.nk) ks_next = __ldg(ks_row + kt);
                for (int j = 0; j < it.nt; ++j, ++tile) {
                    const int key = j * KT + kt;
                    // an infinite scale is no number either (it would be one for scores of one sign)
                    const float ks = !Q8 || fabsf(ks_next) <= 3.402823466e38f ? ks_next : __int_as_float(0x7fc00000);
                    const float kw = ks == ks ? ks : 1.f;  // a masked probability of zero stays zero
                    if (Q8) ks_next = live && key + KT < it.nk ? __ldg(ks_row + key + KT) : 1.f;
                    const int sb = tile & 1;
                    wait(&s_full[sb], (tile >> 1) & 1);
                    tc_fence_after();
                    float z[NC];
                    if constexpr (NC == 32) {
                        tmem_ld32_nowait(lane_base + C::kColS + sb * N + c0, z);
                        tmem_wait_ld();
                    } else {
                        tmem_ld16(lane_base + C::kColS + sb * N, z);
                    }
                    if constexpr (Q8) {
#pragma unroll
                        for (int n = 0; n < NC; n += 16) {
                            float r[16];
                            tmem_ld16(lane_base + C::kColR + sb * N + c0 + n, r);
#pragma unroll
                            for (int e = 0; e < 16; ++e) z[n + e] = fmaf(z[n + e], ks, r[e]);
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s_free[sb]);
                    // scores relative to the column's reference, base 2; the first tile's reference is 0
                    bool over = j == 0;
                    float top = -INFINITY;
#pragma unroll
                    for (int n = 0; n < NC; n += 4) {
                        const float4 m = *reinterpret_cast<const float4*>(base_c + n);
                        z[n] = fmaf(z[n], cs, -m.x);
                        z[n + 1] = fmaf(z[n + 1], cs, -m.y);
                        z[n + 2] = fmaf(z[n + 2], cs, -m.z);
                        z[n + 3] = fmaf(z[n + 3], cs, -m.w);
                    }
                    if ((j + 1) * KT > lim_min) {  // the last tile(s): keys past a query's limit
                        if (causal) {
#pragma unroll
                            for (int n = 0; n < NC; ++n)
                                if (key >= lim_s[c0 + n]) z[n] = -INFINITY;
                        } else if (key >= it.nk) {
#pragma unroll
                            for (int n = 0; n < NC; ++n) z[n] = -INFINITY;
                        }
                    }
                    if (KT == 64 && !live) {
#pragma unroll
                        for (int n = 0; n < NC; ++n) z[n] = -INFINITY;
                    }
#pragma unroll
                    for (int n = 0; n < NC; ++n) top = fmaxf(top, z[n]);
                    if (Q8) top += scale_exponent(ks);
                    over |= top > over_s[group];
                    if (soft_any(group, over)) {
                        auto larger = [](float u, float w) { return fmaxf(u, w); };
                        int own;
                        float most;
                        if constexpr (Q8) {
                            // the first step here: its lanes have exponents of their own, and values with
                            // them beside the scores would not fit the registers
                            float x[NC / 2];
                            const bool up = lane & 16;
                            const float te = scale_exponent(ks), to = __shfl_xor_sync(0xffffffffu, te, 16);
#pragma unroll
                            for (int n = 0; n < NC / 2; ++n) {
                                const float got = __shfl_xor_sync(0xffffffffu, up ? z[n] : z[n + NC / 2], 16);
                                x[n] = fmaxf((up ? z[n + NC / 2] : z[n]) + te, got + to);
                            }
                            own = (up ? NC / 2 : 0) + fold_columns<8>(x, lane, larger);
                            most = x[0];
                        } else {
                            float x[NC];
#pragma unroll
                            for (int n = 0; n < NC; ++n) x[n] = z[n];
                            own = fold_columns(x, lane, larger);
                            most = x[0];
                        }
                        if (NC == 32 || (lane & 1) == 0) red_s[gw * N + c0 + own] = most;
                        soft_sync(group);
                        if (gt < NC) {
                            // every column that sees a key of the item sees one in its first tile: there
                            // the reference becomes the tile's maximum, later it moves only by more than the
                            // growth. A column whose keys so far score -infinity keeps kNoMax.
                            const int n = c0 + gt;
                            const float top_n = fmaxf(fmaxf(red_s[n], red_s[N + n]), fmaxf(red_s[2 * N + n], red_s[3 * N + n]));
                            const float old = m_s[n], from = base_s[n];
                            float m = old;
                            if (j == 0 ? top_n > -INFINITY : (from - old) + top_n > kLift + kGrowth) m = from + (top_n - kLift);
                            else if (j == 0 && !(causal && lim_s[n] <= 0)) m = kNoMax;
                            corr_s[n] = fast_exp2(old - m);
                            up_s[n] = m - from;
                            m_s[n] = m;
                            // scores relative to a large reference (keys masked by the lowest value, say) would
                            // lose the digits of what comes after it: from there on every tile starts from 0
                            const bool near = fabsf(m) <= kNear;
                            base_s[n] = near ? m : 0.f;
                            if (!near) over_s[group] = -INFINITY;
                        }
                        soft_sync(group);
#pragma unroll
                        for (int n = 0; n < NC; ++n) z[n] -= up_s[c0 + n];
                        if (j > 0) {
#pragma unroll
                            for (int n = 0; n < NC; ++n) l[n] *= corr_s[c0 + n];
                            // the previous tile's products have landed: rescale the accumulator
                            const int pt = tile - 1;
                            wait(&p_free[pt % C::PB], (pt / C::PB) & 1);
                            tc_fence_after();
                            const uint32_t o = lane_base + C::kColO + (item % C::OB) * C::NP * N + c0;
#pragma unroll 1
                            for (int i = 0; i < C::NP; ++i)
#pragma unroll 1
                                for (int c = 0; c < NC; c += 16) {
                                    float v[16];
                                    tmem_ld16(o + i * N + c, v);
#pragma unroll
                                    for (int e = 0; e < 16; ++e) v[e] *= corr_s[c0 + c + e];
                                    tmem_st16(o + i * N + c, v);
                                }
                            tmem_wait_st();
                        }
                    }
                    const int pb = tile % C::PB;
                    wait(&p_free[pb], ((tile / C::PB) & 1) ^ 1);
                    if (live) {
                        uint8_t* P = smem + C::oP + pb * C::kP;
#pragma unroll
                        for (int n0 = 0; n0 < NC; n0 += 8) {
                            if (n0 >= nq) break;  // columns past the block's queries feed results nobody reads
                            float e[8];
#pragma unroll
                            for (int q = 0; q < 8; ++q) {
                                e[q] = fast_exp2(z[n0 + q]);
                                l[n0 + q] += e[q];
                                if (Q8) e[q] *= kw;
                            }
                            if constexpr (N == 64) {
                                *reinterpret_cast<uint4*>(P + sw128(kt, (c0 + n0) >> 3)) =
                                    make_uint4(lat::pack2<T>(e[0], e[1]), lat::pack2<T>(e[2], e[3]),
                                               lat::pack2<T>(e[4], e[5]), lat::pack2<T>(e[6], e[7]));
                            } else {
                                // K-major: query row n, key kt of the 64-key box kt / 64
#pragma unroll
                                for (int q = 0; q < 8; ++q)
                                    *reinterpret_cast<T*>(P + (kt >> 6) * 2048 + sw128(n0 + q, (kt & 63) >> 3) + (kt & 7) * 2) =
                                        lat::from_f32<T>(e[q]);
                            }
                        }
                        fence_proxy_async_smem();
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[pb]);
                }
                // the sums over the item's keys
                const int own = fold_columns(l, lane, [](float u, float w) { return u + w; });
                if constexpr (C::EW > 0) {
                    float* mail = mail_s + eb.i * 5 * N;
                    wait(&e_free[eb.i], eb.phase ^ 1);
                    if ((lane & 1) == 0) mail[gw * N + own] = l[0];
                    if (gt < N) mail[4 * N + gt] = m_s[gt];
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&e_full[eb.i]);
                    eb.next();
                    if (it.nt > 0) ++item;
                } else {
                    const long long as = it.split * rows + it.q0 + c0;
                    const int ob = item % C::OB;
                    red_s[gw * N + c0 + own] = l[0];
                    soft_sync(group);
                    if (gt < nq) {
                        const int n = c0 + gt;
                        float l_own = (red_s[n] + red_s[N + n]) + (red_s[2 * N + n] + red_s[3 * N + n]);
                        if (*reinterpret_cast<volatile int*>(bad_s)) l_own = __int_as_float(0x7fc00000);
                        a.part_ml[as + gt] = make_float2(l_own == 0.f ? kNoMax : m_s[n], l_own);
                    }
                    wait(&o_full[ob], (item / C::OB) & 1);
                    tc_fence_after();
                    const uint32_t o = lane_base + C::kColO + ob * C::NP * N + c0;
#pragma unroll 1
                    for (int i = 0; i < C::NP; ++i)
#pragma unroll 1
                        for (int c = 0; c < nq; c += 16) {
                            float v[16];
                            tmem_ld16(o + i * N + c, v);
                            float* dst = a.part_o + (as + c) * KV + i * 128 + gt;
#pragma unroll
                            for (int e = 0; e < 16; ++e)
                                if (c + e < nq) dst[static_cast<long long>(e) * KV] = v[e];
                        }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&o_free[ob]);
                    ++item;
                }
            }
        }
    } else if constexpr (C::EW > 0) {
        // ------------------------------------------------------------ results (N = 16)
        // thread = latent dimension (tensor-memory lane) of a 128-column pair, 16 query columns
        const int quad = warp & 3, dim = quad * 32 + lane;
        const int n = tid - 32 * kResultWarp;  // < N: the query whose factors this thread works out
        const long long rows = static_cast<long long>(p.B) * th;
        Ring<C::OB> ob;
        Ring<2> eb;
        bool waited = !a.overlap;
        for (int base = 0; base < mine; base += kTcTable) {
            const int count = next_table(base, std::false_type());
            for (int e0 = 0; e0 < count; ++e0) {
                const Item it = table[e0];
                const bool direct = it.np >= 0;
                if (it.nt == 0 && !direct) continue;
                const long long at = it.q0;  // first query row
                const long long part = kShares && spans ? it.split * static_cast<long long>(N) : it.split * rows + at;
                // The prefix's share of a direct result: unit u = (pair, prefix range) of the partials. The
                // first is asked for before the item's tiles are done: a load issued behind a full ring
                // of cache tiles waits its turn (2 to 4 us).
                const bool joins = it.np > 0;
                float x0[16];
                float2 ml[kMaxJoin];
                auto ask = [&](int u, float (&x)[16]) {
                    const int s = u % it.np, i = u / it.np;
                    const float* src = a.pre_o + (s * rows + at) * KV + i * 128 + dim;
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[e] = e < it.nq ? __ldcg(src + static_cast<long long>(e) * KV) : 0.f;
                };
                if (joins) {
                    if (!waited) {
                        pdl_wait();
                        waited = true;
                    }
                    ask(0, x0);
                }
#pragma unroll
                for (int s = 0; s < kMaxJoin; ++s)
                    ml[s] = s < it.np && n < it.nq ? __ldcg(&a.pre_ml[s * rows + at + n]) : make_float2(kNoMax, 0.f);
                wait(&e_full[eb.i], eb.phase);
                const float* mail = mail_s + eb.i * 5 * N;
                if (n < it.nq) {
                    float l_own = (mail[n] + mail[N + n]) + (mail[2 * N + n] + mail[3 * N + n]);
                    if (*reinterpret_cast<volatile int*>(bad_s)) l_own = __int_as_float(0x7fc00000);
                    const float m_own = l_own == 0.f ? kNoMax : mail[4 * N + n];
                    if (!direct) {
                        a.part_ml[part + n] = make_float2(m_own, l_own);
                    } else {
                        // joint maximum and sum with the prefix's ranges (at most kMaxJoin); each part's
                        // factor, the division by the sum included
                        float M = m_own;
#pragma unroll
                        for (int s = 0; s < kMaxJoin; ++s) M = fmaxf(M, ml[s].x);
                        const float f = fast_exp2(m_own - M);
                        float L = l_own * f;
#pragma unroll
                        for (int s = 0; s < kMaxJoin; ++s) L += ml[s].y * fast_exp2(ml[s].x - M);
                        const float inv = L == 0.f ? 0.f : 1.f / L;
                        fac_s[n] = f * inv;
#pragma unroll
                        for (int s = 0; s < kMaxJoin; ++s) fac_s[(1 + s) * N + n] = fast_exp2(ml[s].x - M) * inv;
                        if (p.lse) p.lse[at + n] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
                    }
                }
                soft_sync(2);
                if (lane == 0) mbar_arrive(&e_free[eb.i]);
                eb.next();
                if (it.nt > 0) {
                    wait(&o_full[ob.i], ob.phase);
                    tc_fence_after();
                }
                const uint32_t o = tmem + (static_cast<uint32_t>(quad * 32) << 16) + C::kColO + ob.i * C::NP * N;
                int u = 0;
#pragma unroll 1
                for (int i = 0; i < C::NP; ++i) {
                    float v[16];
                    if (it.nt > 0) tmem_ld16(o + i * N, v);
                    if (!direct) {
                        float* dst = a.part_o + part * KV + i * 128 + dim;
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (e < it.nq) dst[static_cast<long long>(e) * KV] = v[e];
                        continue;
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) v[e] = it.nt > 0 ? v[e] * fac_s[e] : 0.f;
#pragma unroll 1
                    for (int s = 0; s < it.np; ++s, ++u) {
                        float xn[16];
                        if (u + 1 < it.np * C::NP) ask(u + 1, xn);
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (e < it.nq) v[e] = fmaf(x0[e], fac_s[(1 + s) * N + e], v[e]);
#pragma unroll
                        for (int e = 0; e < 16; ++e) x0[e] = xn[e];
                    }
                    T* dst = static_cast<T*>(p.out) + at * KV + i * 128 + dim;
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (e < it.nq) dst[static_cast<long long>(e) * KV] = lat::from_f32<T>(v[e]);
                }
                soft_sync(2);  // fac_s may be written again
                if (it.nt > 0) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&o_free[ob.i]);
                    ob.next();
                }
            }
        }
        // this launch must not end before the one it ran beside
        if (!waited) pdl_wait();
    }
    if (C::EW == 0 && a.overlap) pdl_wait();  // nor with 64-query blocks
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && *reinterpret_cast<volatile int*>(bad_s)) end_after_timeout(tile_in, C::TS);
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, C::kTmem);
    }
}

// Joins the partials of a query row: its group's prefix ranges and its suffix ranges. One warp
// per query row, kv / 32 columns per lane.
template <int KV, typename T, bool PIECES>
__global__ void __launch_bounds__(256) shared_prefix_join_kernel(const Problem p, const float* __restrict__ pre_o,
                                                                 const float2* __restrict__ pre_ml, int pre_kps,
                                                                 const float* __restrict__ suf_o,
                                                                 const float2* __restrict__ suf_ml, int suf_kps,
                                                                 int direct, const int2* __restrict__ pieces) {
    MM_PDL_ENTRY();
    const int th = p.T * p.H, lane = threadIdx.x & 31;
    const long long rows = static_cast<long long>(p.B) * th;  // below 2^31
    const long long r = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    if (r >= rows) return;
    const int b = static_cast<int>(r) / th, u = static_cast<int>(r) - b * th;
    int first = 0, ns;
    if constexpr (PIECES) {  // the parts of a row cut between CTAs
        const int2 v = __ldcg(&pieces[b]);
        if (v.y == 0) return;  // the suffix launch wrote it
        first = v.x;
        ns = v.y;
    } else {
        if (direct && direct_join(p, b, suf_kps, pre_kps) >= 0) return;  // the suffix launch wrote it
        int len = suffix_length(p, b);
        if (!direct) {  // blocks of 64 queries end where their last one does
            len = seen_by(p, len, min((u / 64 + 1) * 64, th) - 1);
        }
        ns = (len + suf_kps - 1) / suf_kps;
    }
    const int g = p.G > 0 ? group_of(p, b) : -1;
    const int np = (prefix_length(p, g) + pre_kps - 1) / pre_kps;
    auto suf_at = [&](int s) {  // the query row of suffix part s among the partials
        if constexpr (PIECES) return (2LL * (first + s) + (s == 0)) * 16 + u;
        else return s * rows + r;
    };
    auto ml = [&](int s) { return s < np ? __ldcg(&pre_ml[s * rows + r]) : __ldcg(&suf_ml[suf_at(s - np)]); };
    float M = kNoMax;
    for (int s = lane; s < np + ns; s += 32) M = fmaxf(M, ml(s).x);
    M = warp_max(M);
    float L = 0.f;
    for (int s = lane; s < np + ns; s += 32) {
        const float2 v = ml(s);
        L += v.y * fast_exp2(v.x - M);
    }
    L = warp_sum(L);
    const float inv = L == 0.f ? 0.f : 1.f / L;
    constexpr int C = KV / 128;  // float4s per lane
    float4 acc[C];
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = 0; s < np + ns; ++s) {
        const float f = fast_exp2(ml(s).x - M);
        const float4* o = reinterpret_cast<const float4*>((s < np ? pre_o + (s * rows + r) * KV : suf_o + suf_at(s - np) * KV)) + lane;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const float4 v = __ldcg(o + 32 * c);
            acc[c].x += f * v.x;
            acc[c].y += f * v.y;
            acc[c].z += f * v.z;
            acc[c].w += f * v.w;
        }
    }
    uint2* out = reinterpret_cast<uint2*>(static_cast<T*>(p.out) + r * KV) + lane;
#pragma unroll
    for (int c = 0; c < C; ++c)
        out[32 * c] = make_uint2(lat::pack2<T>(acc[c].x * inv, acc[c].y * inv), lat::pack2<T>(acc[c].z * inv, acc[c].w * inv));
    if (p.lse && lane == 0) p.lse[r] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
}

}  // namespace spa
}  // namespace mm
