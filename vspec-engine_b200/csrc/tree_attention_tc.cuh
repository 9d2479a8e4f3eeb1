// tree_attention_tc.cuh -- tree attention on the 5th-generation tensor cores:
// many query rows a (sequence, KV head) pair (wide trees, large groups).
//
// With R rows a pair, every cached token costs 4 R d operations for 4 d bytes of
// fp16: from a few dozen rows on, warp-level MMA (576 TFLOP/s here) and not DRAM
// is the bound.  Here one thread issues tcgen05.mma for tiles of 128 rows x 128
// tokens, with S = Q K^T and O = P V in tensor memory:
//   warps 0-3, 4-7   softmax, a row (TMEM lane) a thread: maximum and
//                    exponentials of S, P back over S as fp16, the step's O
//                    added to fp32 registers (a step's product starts from 0:
//                    the tensor cores truncate, see tree_attention_mma.cuh)
//   warp 8           one lane issues the products
//   warps 9-11       K and V pages into a ring of swizzled 128-token tiles by
//   (9-15 for 8-bit) TMA boxes (page_tokens a multiple of 8); 8-bit codes land
//                    in a raw ring and are widened to fp16 into the tiles
// Two tiles are in flight so that the tensor cores work on one while the other
// is in its softmax: two row tiles sharing each K and V tile when a pair has
// more than 128 rows (TILES = 2), else alternate steps of one row tile, with the
// two softmax groups sharing out a step's tokens and the dims (TILES = 1).
//
// The grid is persistent: all pairs' steps, laid out in a row, are cut into
// equal runs, one a CTA, so that sequences of any lengths balance to one step.
// A run that cuts a pair writes that part's (O, m, l); a second kernel joins
// the parts of such pairs in order.  fp32 q, weights and 8-bit pages are split
// and scaled as in the warp-MMA kernels.
//
// Measured, 8 KV heads of 128, 16-token pages, 4 query heads a KV head: 32 x 64
// drafted tokens over 512..8192, fp32 q and fp16 pages, 310 us replayed in a graph,
// 352 to 362 us a call with other inputs in between: 950 and 820 TFLOP/s of issued
// products (two parts of q, two of the weights), 58 and 50 % of a cuBLAS GEMM's
// rate; with fp16 q 260 us.  A step takes 3.6 us with fp32 q, of which the products
// need 3.0; a change of pairs (q rows, rows out, an empty pipeline) about 20 us, 2.7
// of them a CTA.  8 x 16 drafted tokens on fp8 pages, fp16 q, 1024..6144: 62 us.  8 x
// 32768 tokens, 64 rows a pair, fp16 q: 3.8 TB/s of fp16 pages (279 us) and 1.6 TB/s
// of fp8 pages (353 us), bound by the latency of the softmax's steps and, for
// 8-bit pages, by the instructions of the widening beside them.
#pragma once

#include <stddef.h>

#include "tma_map.cuh"
#include "tree_attention_mma.cuh"

namespace vb200 {

constexpr int kTcMmaWarp = 8, kTcFirstProducer = 9;
constexpr int kTcStep = 128;
constexpr long long kTcWaitCycles = 4000000000ll;  // about two seconds
constexpr uint32_t kTcDrainPolls = 1000000u;       // of about a microsecond
constexpr uint32_t kTcHalf = 128u * 128u;          // 128 rows x 64 fp16
constexpr int kTcRawSlots = 3;
constexpr uint32_t kTcSmemMax = 232448u;

struct TcParams {
    TreeParams t;
    CUtensorMap k_map, v_map;   // [pool rows][KV heads][d], boxes of box_rows x 1 x 64 values (8-bit: x d)
    int box_rows;               // divides page_tokens and kTcStep
    int* timeout;
    long long wait_cycles;      // after which a wait gives up
};

template <int D, int TILES, int QS, int KV>
struct TcShape {
    static constexpr int kProducers = KV == kTreeF16 ? 3 : 7;
    static constexpr int kFillers = KV == kTreeF16 ? 3 : 6;   // warps that hand a tile over
    static constexpr int kThreads = (kTcFirstProducer + kProducers) * 32;
    // registers a thread of the softmax warps (256 threads) and of the others: together what the CTA is launched
    // with, 384 x 168 or 512 x 128
    static constexpr int kSoftmaxRegs = KV == kTreeF16 ? (TILES == 2 ? 216 : 184) : (TILES == 2 ? 176 : 152);
    static constexpr int kOtherRegs = KV == kTreeF16 ? (TILES == 2 ? 72 : 136) : (TILES == 2 ? 80 : 104);
    static_assert(256 * kSoftmaxRegs + (kThreads - 256) * kOtherRegs <= kThreads * (65536 / kThreads / 8 * 8), "register split");
    static constexpr uint32_t kSlot = kTcStep * D * 2;
    static constexpr uint32_t kQ = TILES * QS * kSlot;
    static constexpr uint32_t kRaw = KV == kTreeF16 ? 0 : kTcRawSlots * kTcStep * D;
    static constexpr uint32_t kMisc = KV == kTreeF16 ? (TILES == 2 ? 3072 : 4096) : (TILES == 2 ? 8192 : 10240);
    static constexpr int kFit = (int)((kTcSmemMax - kMisc - kQ - kRaw) / kSlot);
    static constexpr int kMost = 6;
    static constexpr int kSlots = kFit < kMost ? kFit : kMost;
    static constexpr uint32_t kRingAt = kQ, kRawAt = kQ + kSlots * kSlot, kMiscAt = kRawAt + kRaw;
    static constexpr uint32_t kTotal = kMiscAt + kMisc;
    static_assert(kSlots >= 3, "ring");
};

// misc area
struct alignas(16) TcMisc {
    float mul[256];             // score multiplier of each row
    uint64_t full[6], empty[6], raw_full[kTcRawSlots], raw_empty[kTcRawSlots], sc_full[4], sc_empty[4], s_full[2], p_half[2], p_full[2], q_full, pair, staged[2], drain;
    uint32_t tmem;
    int abort;
    int start_b;
    long long start_off, total;
    int odd[8];                 // step + 1 where V held infinities or NaN
    alignas(16) float row[2][2][128];       // maxima, at last sums, of the two softmax groups (TILES = 1), in turn
    int v_exp[2][2][128];       // exponents of the largest V scales that the groups' rows see (8-bit pages), in turn
};
struct alignas(16) TcScales {   // 8-bit pages: scales of four steps, read four at a time
    float k[4][kTcStep], v[4][kTcStep];
    float one[kTcStep];
    int v_exp[4];
};
__device__ __forceinline__ void tc_tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void tc_st_x16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n"
        ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
          "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tc_st_x8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n"
                 ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
// Shared-memory operands, 128-byte swizzle, as the two words of their
// descriptors: low = address >> 4 (14 bits) | leading offset >> 4 << 16, high =
// stride offset 1024 >> 4 | version 1 << 14 | swizzle 2 << 29.
//   K-major (Q, K): rows of 64 values, 8-row groups 1024 bytes apart.
//   N-major (V: tokens are K, dims N): 64 dims a 128-byte row, 8 tokens 1024
//   bytes, the next 64 dims kTcHalf bytes on (the leading offset).
constexpr uint32_t kTcDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
constexpr uint32_t kTcLeadK = 1u << 16, kTcLeadV = (kTcHalf >> 4) << 16;
// D[tmem] (+)= A[smem] * B[smem], issued by one thread.
__device__ __forceinline__ void tc_mma_ss(uint32_t d_taddr, uint32_t a_low, uint32_t b_low, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n.reg .pred p;\n.reg .b64 da, db;\nsetp.ne.u32 p, %4, 0;\nmov.b64 da, {%1, %5};\nmov.b64 db, {%2, %5};\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n"
        ::"r"(d_taddr), "r"(a_low), "r"(b_low), "r"(idesc), "r"(acc), "r"(kTcDescHigh) : "memory");
}
// The same with A in tensor memory.
__device__ __forceinline__ void tc_mma_ts(uint32_t d_taddr, uint32_t a_taddr, uint32_t b_low, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n.reg .pred p;\n.reg .b64 db;\nsetp.ne.u32 p, %4, 0;\nmov.b64 db, {%2, %5};\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}\n"
        ::"r"(d_taddr), "r"(a_taddr), "r"(b_low), "r"(idesc), "r"(acc), "r"(kTcDescHigh) : "memory");
}
template <int N>
__device__ __forceinline__ void tc_regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void tc_regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(N)); }

// Waits for this warp's TMEM loads; v is what one of them returned, so that no
// use of it can be moved in front of the wait.
__device__ __forceinline__ void tc_landed(float (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                   "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
                 :: "memory");
}
// f(c, v) for N chunks of 16 TMEM columns of this thread's lane, the next
// chunk's load in flight.  UNROLL: c is a constant in f (it indexes registers);
// else a loop of two chunks, which keeps the code of a step in the instruction
// cache.
template <int N, bool UNROLL, typename F>
__device__ __forceinline__ void tc_sweep(uint32_t taddr, F f) {
    static_assert(N % 2 == 0, "pairs of chunks");
    float a[16], b[16];
    tmem_ld_x16(taddr, a);
#pragma unroll (UNROLL ? N / 2 : 1)
    for (int c = 0; c < N; c += 2) {
        tc_landed(a);
        tmem_ld_x16(taddr + 16u * (c + 1), b);
        f(c, a);
        tc_landed(b);
        if (c + 2 < N) tmem_ld_x16(taddr + 16u * (c + 2), a);
        f(c + 1, b);
    }
}
template <bool ON>
__device__ __forceinline__ void tc_scale(float (&v)[16], const float* s) {
#pragma unroll
    for (int x = 0; ON && x < 16; x += 4) {
        const float4 k = *reinterpret_cast<const float4*>(s + x);
        unpack2(mul2(pack2(v[x], v[x + 1]), pack2(k.x, k.y)), v[x], v[x + 1]);
        unpack2(mul2(pack2(v[x + 2], v[x + 3]), pack2(k.z, k.w)), v[x + 2], v[x + 3]);
    }
}

// When a wait gives up: the CTA's flag is set, or a number of cycles have passed.
struct TcGiveUp {
    volatile int* flag;
    long long cycles;
};
__device__ __forceinline__ bool tc_wait_one(uint64_t* bar, uint32_t parity, const TcGiveUp& up) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long start = clock64();
    while (!mbar_try_wait(bar, parity))
        if (*up.flag || clock64() - start > up.cycles) return false;
    return true;
}
// The same for a whole warp, with one answer for all its lanes.
__device__ __forceinline__ bool tc_wait(uint64_t* bar, uint32_t parity, const TcGiveUp& up) {
    return __all_sync(0xffffffffu, tc_wait_one(bar, parity, up));
}

// ---- the work: sequence b has pairs (KV head, row tile) of n steps each.  A pair also costs its q rows, its
//      output and the filling of the pipeline, about p.pair_cost steps: runs are equal in steps and those ----
template <int RT>
__device__ __forceinline__ long long tc_work(const TreeParams& p, int b, int& n, int& tiles) {
    int row0;
    const int drafted = tree_rows(p, b, row0);
    const int total = tree_ctx(p, b) + drafted;
    n = (total + kTcStep - 1) / kTcStep;
    tiles = (drafted * p.group + RT - 1) / RT;
    return drafted ? (long long)(n + p.pair_cost) * p.hkv * tiles : 0;
}
// CTAs that take part: at least three units each.
__device__ __forceinline__ int tc_ctas(long long total, int most) {
    const long long g = (total + 2) / 3;
    return (int)(g < 1 ? 1 : (g < most ? g : most));
}

// A run of steps within one pair.
struct TcSegment {
    int b, row0, drafted, ctx, kvh, rt, n, step0, steps;
};
template <int RT>
struct TcWalk {
    int b;
    long long off, left;
    // the next segment of the CTA's run, or false
    __device__ __forceinline__ bool next(const TreeParams& p, TcSegment& s) {
        while (left > 0) {
            int n, tiles;
            const long long w = tc_work<RT>(p, b, n, tiles);
            if (off >= w) { off -= w; ++b; continue; }
            // a pair's units: p.pair_cost, then its steps
            const int units = n + p.pair_cost;
            const long long pair = off >> 31 ? off / units : (long long)((unsigned)off / (unsigned)units);
            const int u0 = (int)(off - pair * units), u1 = (int)min((long long)units, u0 + left);
            off += u1 - u0;
            left -= u1 - u0;
            s.step0 = max(u0 - p.pair_cost, 0);
            s.steps = max(u1 - p.pair_cost, 0) - s.step0;
            if (s.steps == 0) continue;        // only the pair's cost: the next CTA begins its first step
            s.b = b;
            s.drafted = tree_rows(p, b, s.row0);
            s.ctx = tree_ctx(p, b);
            s.n = n;
            s.kvh = (int)pair / tiles;         // pairs of a sequence: at most 65535
            s.rt = (int)pair - s.kvh * tiles;
            return true;
        }
        return false;
    }
};

// Eight fp16 values with infinities and NaN replaced by 0.
__device__ __forceinline__ void tc_clear_odd(uint4& v) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if ((w[e] & 0x7C00u) == 0x7C00u) w[e] &= 0xFFFF0000u;
        if ((w[e] & 0x7C000000u) == 0x7C000000u) w[e] &= 0x0000FFFFu;
    }
}

// Bits of the drafted tokens j0 .. j0 + 31 (j0 < 0: committed ones) that token i of the tree sees.
__device__ __forceinline__ uint32_t tc_sees32(const TreeParams& p, int row0, int i, int drafted, int j0) {
    auto word = [&](int k) -> uint32_t {
        if (k < 0) return 0xffffffffu;
        const int left = drafted - 32 * k;
        if (left <= 0) return 0u;
        uint32_t v;
        if (p.mask) v = __ldg(p.mask + (size_t)(row0 + i) * p.mask_words + k);
        else v = i - 32 * k >= 31 ? 0xffffffffu : (i < 32 * k ? 0u : (2u << (i - 32 * k)) - 1u);
        return left < 32 ? v & ((1u << left) - 1u) : v;
    };
    const int k = j0 >> 5, sh = j0 & 31;
    return sh ? (word(k) >> sh) | (word(k + 1) << (32 - sh)) : word(k);
}

template <int D, int TILES, int QS, int KV>
__global__ void __launch_bounds__(TcShape<D, TILES, QS, KV>::kThreads, 1) tree_tc_kernel(const __grid_constant__ TcParams pp) {
    const TreeParams& p = pp.t;
    using S = TcShape<D, TILES, QS, KV>;
    constexpr int RT = 128 * TILES, NS = S::kSlots, kTcProducers = S::kProducers;
    extern __shared__ __align__(1024) unsigned char tc_smem[];
    unsigned char* const smem = tc_smem;
    TcMisc& sm = *reinterpret_cast<TcMisc*>(smem + S::kMiscAt);
    // what lies behind `row` (TILES = 2) or `v_exp` (fp16 pages) is not there
    constexpr uint32_t kMiscUsed = TILES == 2 ? offsetof(TcMisc, row) : KV == kTreeF16 ? offsetof(TcMisc, v_exp) : sizeof(TcMisc);
    static_assert(kMiscUsed % 16 == 0 && kMiscUsed + (KV == kTreeF16 ? 0 : sizeof(TcScales)) <= S::kMisc, "misc area");
    static_assert(S::kMiscAt % 16 == 0, "vector reads of the scales");
    TcScales& sc = *reinterpret_cast<TcScales*>(smem + S::kMiscAt + kMiscUsed);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const TcGiveUp give_up = {&sm.abort, pp.wait_cycles};

    if (tid == 0) {
        sm.abort = 0;
        for (int i = 0; i < 6; ++i) { mbar_init(&sm.full[i], S::kFillers); mbar_init(&sm.empty[i], 1); }
        for (int i = 0; i < kTcRawSlots; ++i) { mbar_init(&sm.raw_full[i], 1); mbar_init(&sm.raw_empty[i], S::kFillers); }
        for (int i = 0; i < 4; ++i) { mbar_init(&sm.sc_full[i], 1); mbar_init(&sm.sc_empty[i], 8); }
        for (int i = 0; i < 2; ++i) { mbar_init(&sm.s_full[i], 1); mbar_init(&sm.p_half[i], 128); mbar_init(&sm.p_full[i], 128); }
        mbar_init(&sm.q_full, 256);
        mbar_init(&sm.pair, 256);
        for (int i = 0; i < 2; ++i) mbar_init(&sm.staged[i], 128);
        mbar_init(&sm.drain, 1);
        mbar_fence_init();
        for (int i = 0; i < 8; ++i) sm.odd[i] = 0;
        tma_prefetch_desc(&pp.k_map);
        tma_prefetch_desc(&pp.v_map);
    }
    if (KV != kTreeF16 && tid < kTcStep) sc.one[tid] = 1.0f;
    pdl_wait();
    pdl_trigger();

    // ---- this CTA's run ----
    long long lo = 0, hi = 0;
    if (warp == 0) {
        long long total = 0;
        for (int b0 = 0; b0 < p.batch; b0 += 32) {
            int n, tiles;
            long long w = b0 + lane < p.batch ? tc_work<RT>(p, b0 + lane, n, tiles) : 0;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
            total += w;
        }
        const int g = tc_ctas(total, gridDim.x);
        lo = (int)blockIdx.x < g ? total * (int)blockIdx.x / g : total;
        long long before = 0;
        int found = -1;
        for (int b0 = 0; b0 < p.batch && found < 0 && lo < total; b0 += 32) {
            int n, tiles;
            const long long w = b0 + lane < p.batch ? tc_work<RT>(p, b0 + lane, n, tiles) : 0;
            long long incl = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long u = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += u;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, before + incl > lo);
            if (hit) {
                const int at = __ffs(hit) - 1;
                found = b0 + at;
                const long long start = before + __shfl_sync(0xffffffffu, incl - w, at);
                if (lane == 0) { sm.start_b = found; sm.start_off = lo - start; }
            }
            before += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) sm.total = total;
    }
    if (warp == kTcMmaWarp) {
        tmem_alloc(&sm.tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem;
    TcWalk<RT> walk;
    {
        const long long total = sm.total;
        const int g = tc_ctas(total, gridDim.x);
        lo = (int)blockIdx.x < g ? total * (int)blockIdx.x / g : total;
        hi = (int)blockIdx.x < g ? total * ((int)blockIdx.x + 1) / g : total;
        walk.left = hi - lo;
        walk.b = walk.left > 0 ? sm.start_b : 0;
        walk.off = walk.left > 0 ? sm.start_off : 0;
    }
    // TMEM columns: S (and P over it) of softmax group w at 128 w, its O at 256 + 128 w
    TcSegment seg;
    bool ok = true;
    if (warp >= kTcMmaWarp) {
    tc_regs_dec<S::kOtherRegs>();
    if (warp >= kTcFirstProducer) {
        // ============================ producers ============================
        const int pw = warp - kTcFirstProducer;
        const int br = pp.box_rows, boxes = kTcStep / br;      // boxes of a whole tile: 1 to 16
        int slot = 0, raw = 0;
        uint32_t phase = 0, raw_phase = 0;   // of the slot's next use
        bool wrapped = false;                // the ring has been filled once
        int k_steps = 0;                     // steps of the CTA's run before this segment
        // the first warp's copies, for their end after a wait that gave up: barriers with copies (a bit each) and the
        // parity of the last of them
        uint32_t armed = 0, armed_phase = 0, raw_armed = 0, raw_armed_phase = 0;
        auto advance = [&]() {
            if (++slot == NS) { slot = 0; phase ^= 1u; wrapped = true; }
        };
        auto wait_slot = [&]() -> bool { return !wrapped || tc_wait(&sm.empty[slot], phase ^ 1u, give_up); };
        // load li of a segment: K or V of its step j, in the order in which the products need them
        auto decode = [&](int li, bool& is_v, int& j) {
            if (TILES == 2) { is_v = li & 1; j = li >> 1; }
            else if (li == 0) { is_v = false; j = 0; }
            else { is_v = (li & 1) == 0; j = is_v ? (li - 2) >> 1 : (li + 1) >> 1; }
        };
        while (ok && walk.next(p, seg)) {
            const int32_t* table = p.table + (size_t)seg.b * p.max_pages;
            const int total = seg.ctx + seg.drafted, t_first = seg.step0 * kTcStep;
            const int loads = TILES == 2 ? 2 * seg.steps : 2 * seg.steps + 1;
            // page of box `lane` of step j, loaded two steps ahead of its use and looked at only then
            auto find = [&](int j) -> int {
                const int t = min(t_first + j * kTcStep + lane * br, total - 1);
                return __ldg(table + min(t / p.page_tokens, p.max_pages - 1));
            };
            int page_even = find(0), page_odd = find(1);
            // the boxes of K or V of step j
            auto issue = [&](bool is_v, int j, uint32_t dst, uint64_t* bar) {
                const int left = total - (t_first + j * kTcStep);
                const int nb = left >= kTcStep ? boxes : (left + br - 1) / br;
                constexpr uint32_t kRowBytes = KV == kTreeF16 ? D * 2 : D;
                if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(nb * br) * kRowBytes);
                __syncwarp();
                const int t = min(t_first + j * kTcStep + lane * br, total - 1), at = t / p.page_tokens;
                int page = (j & 1) ? page_odd : page_even;
                if (at >= p.max_pages || page < 0 || page >= p.num_pages) {
                    if (lane < nb) atomicOr(p.fault, 1);
                    page = 0;
                }
                const int row = page * p.page_tokens + (t - at * p.page_tokens);
                const CUtensorMap* map = is_v ? &pp.v_map : &pp.k_map;
                if (lane < nb) {
                    if (KV == kTreeF16) {
#pragma unroll
                        for (int h = 0; h < D / 64; ++h)
                            tc_tma_3d(dst + h * kTcHalf + (uint32_t)(lane * br) * 128u, map, 64 * h, seg.kvh, row, bar);
                    } else {
                        tc_tma_3d(dst + (uint32_t)(lane * br) * D, map, 0, seg.kvh, row, bar);
                    }
                }
                // K and V of a step share its pages: after V they are those of the step after next
                if (is_v) {
                    if (j & 1) page_odd = find(j + 2); else page_even = find(j + 2);
                }
            };
            const uint32_t ring = smem_u32(smem) + S::kRingAt;
            if constexpr (KV == kTreeF16) {
                for (int li = 0; li < loads && ok; ++li) {
                    bool is_v;
                    int j;
                    decode(li, is_v, j);
                    if (j >= seg.steps) continue;
                    const bool drafted = t_first + (j + 1) * kTcStep > seg.ctx;
                    if (pw == 0 && !wait_slot()) { ok = false; break; }
                    if (!(is_v && drafted)) {
                        // the first warp arrives for all, so that the phase ends with its copies, whatever the others do
                        if (pw == 0) {
                            if (lane == 0) mbar_arrive_n(&sm.full[slot], S::kFillers - 1);
                            issue(is_v, j, ring + (uint32_t)slot * S::kSlot, &sm.full[slot]);
                            armed |= 1u << slot;
                            armed_phase = (armed_phase & ~(1u << slot)) | (phase << slot);
                        }
                    } else {
                        // V of a step with drafted tokens: what is past the last token becomes 0, and so do infinities and
                        // NaN, which are noted.  The barrier is armed again when all three warps have seen its last phase:
                        // one that missed a phase would wait for the wrong parity.
                        if (pw == 0) {
                            if (!tc_wait(&sm.raw_empty[0], raw_phase ^ 1u, give_up)) { ok = false; break; }
                            issue(true, j, ring + (uint32_t)slot * S::kSlot, &sm.raw_full[0]);
                            raw_armed = 1u;
                            raw_armed_phase = raw_phase;
                            armed &= ~(1u << slot);     // the slot's last copies are these
                        }
                        if (!tc_wait(&sm.raw_full[0], raw_phase, give_up)) { ok = false; break; }
                        if (lane == 0) mbar_arrive(&sm.raw_empty[0]);
                        raw_phase ^= 1u;
                        unsigned char* st = smem + S::kRingAt + (uint32_t)slot * S::kSlot;
                        const int there = min(total - (t_first + j * kTcStep), kTcStep);
                        bool odd = false;
#pragma unroll 4
                        for (int i = pw * 32 + lane; i < kTcStep * (D / 8); i += kTcProducers * 32) {
                            uint4* at = reinterpret_cast<uint4*>(st) + i;
                            const int r = (i >> 3) & (kTcStep - 1);     // 8 chunks a row of each half
                            if (r >= there) {
                                *at = make_uint4(0, 0, 0, 0);
                            } else if (tree_odd_chunk(*at)) {
                                odd = true;
                                uint4 v = *at;
                                tc_clear_odd(v);
                                *at = v;
                            }
                        }
                        if (odd) sm.odd[(k_steps + j) & 7] = k_steps + j + 1;
                        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sm.full[slot]);
                    }
                    advance();
                }
            } else {
                // The first warp has codes land in the raw ring, as far ahead as it reaches, and fetches the scales; the
                // others widen the codes.  (With page lookups and scales on a widening warp, that warp was the step's
                // longest path.)
                if (pw == 0) {
                    // Scales of K and V of a step's tokens, four a lane, in registers a step ahead and then in a ring of
                    // their own.  Every load is issued whatever its token, so that all are in flight at once.
                    float ks[4], vs[4];
                    int spage[4];                            // pages of the step after
                    auto token = [&](int j, int q) { return t_first + j * kTcStep + 32 * q + lane; };
                    auto fetch_pages = [&](int j) {
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            spage[q] = __ldg(table + min(min(token(j, q), total - 1) / p.page_tokens, p.max_pages - 1));
                    };
                    auto fetch_scales = [&](int j) {         // from spage
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const int t = min(token(j, q), total - 1), at = t / p.page_tokens;
                            const bool bad = at >= p.max_pages || spage[q] < 0 || spage[q] >= p.num_pages;   // noted with the boxes
                            const size_t r = (size_t)((bad ? 0 : spage[q]) * p.page_tokens + (t - at * p.page_tokens)) * p.hkv + seg.kvh;
                            ks[q] = __ldg(p.k_scales + r);
                            vs[q] = __ldg(p.v_scales + r);
                        }
                    };
                    fetch_pages(0);
                    fetch_scales(0);
                    fetch_pages(1);
                    for (int li = 0; li < loads && ok; ++li) {
                        bool is_v;
                        int j;
                        decode(li, is_v, j);
                        if (j >= seg.steps) continue;
                        if (wrapped && !tc_wait(&sm.raw_empty[raw], raw_phase ^ 1u, give_up)) { ok = false; break; }
                        issue(is_v, j, smem_u32(smem) + S::kRawAt + (uint32_t)raw * (kTcStep * D), &sm.raw_full[raw]);
                        raw_armed |= 1u << raw;
                        raw_armed_phase = (raw_armed_phase & ~(1u << raw)) | (raw_phase << raw);
                        if (++raw == kTcRawSlots) { raw = 0; raw_phase ^= 1u; wrapped = true; }
                        if (is_v) continue;
                        const int k = k_steps + j, e = k & 3;
                        if (k >= 4 && !tc_wait(&sm.sc_empty[e], (uint32_t)((k >> 2) - 1) & 1u, give_up)) { ok = false; break; }
                        const bool drafted = t_first + (j + 1) * kTcStep > seg.ctx;
                        float top = 0.f;
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            if (token(j, q) >= total) ks[q] = vs[q] = 0.f;
                            // a V scale that is not finite reaches the rows that see its token as its values do
                            if (!(vs[q] <= 3.402823466e+38f) && drafted) { sm.odd[k & 7] = k + 1; vs[q] = 0.f; }
                            sc.k[e][32 * q + lane] = ks[q];
                            sc.v[e][32 * q + lane] = vs[q];
                            if (vs[q] <= 3.402823466e+38f) top = fmaxf(top, vs[q]);
                        }
                        top = warp_max(top);
                        int ex = -100;
                        if (top > 0.f) (void)frexpf(top, &ex);
                        if (lane == 0) sc.v_exp[e] = max(ex, -100);
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sm.sc_full[e]);
                        fetch_scales(j + 1);
                        fetch_pages(j + 2);
                    }
                    k_steps += seg.steps;
                    continue;
                }
                for (int li = 0; li < loads && ok; ++li) {
                    bool is_v;
                    int j;
                    decode(li, is_v, j);
                    if (j >= seg.steps) continue;
                    const int t0 = t_first + j * kTcStep;
                    const bool drafted = t0 + kTcStep > seg.ctx;
                    if (!tc_wait(&sm.raw_full[raw], raw_phase, give_up) || !wait_slot()) { ok = false; break; }
                    unsigned char* st = smem + S::kRingAt + (uint32_t)slot * S::kSlot;
                    const unsigned char* rs = smem + S::kRawAt + raw * (kTcStep * D);
                    const int there = min(total - t0, kTcStep);
                    bool odd = false;
                    // Pieces of 16 codes, piece i0 + x LANES to this lane: its place in the row and in the swizzle is the
                    // same for every x.  The two halves of 64 dims lie in the same banks: lanes of the second store their
                    // chunks in the other order, so that eight lanes cover all banks.
                    constexpr int PIECES = kTcStep * (D / 16), LANES = S::kFillers * 32, MINE = (PIECES + LANES - 1) / LANES;
                    constexpr int ROWS = LANES / (D / 16);   // from x to x + 1
                    static_assert(LANES % (D / 16) == 0 && ROWS % 8 == 0, "the same place in every round");
                    const int i0 = (pw - 1) * 32 + lane, r0 = i0 / (D / 16), pc = i0 % (D / 16);
                    const int h = pc >> 2, ch = (2 * pc) & 7;
                    const unsigned char* from = rs + i0 * 16;
                    unsigned char* first = st + h * kTcHalf + r0 * 128 + (((ch + h) ^ (r0 & 7)) << 4);
                    unsigned char* second = st + h * kTcHalf + r0 * 128 + (((ch + 1 - h) ^ (r0 & 7)) << 4);
                    auto widen = [&](const uint4 c, uint4& a, uint4& b) {
                        tree_widen<KV>(h ? c.z : c.x, a.x, a.y);
                        tree_widen<KV>(h ? c.w : c.y, a.z, a.w);
                        tree_widen<KV>(h ? c.x : c.z, b.x, b.y);
                        tree_widen<KV>(h ? c.y : c.w, b.z, b.w);
                    };
                    if (!drafted) {
                        uint4 code[MINE];
#pragma unroll
                        for (int x = 0; x < MINE; ++x)
                            if ((x + 1) * LANES <= PIECES || i0 + x * LANES < PIECES)
                                code[x] = *reinterpret_cast<const uint4*>(from + x * LANES * 16);
#pragma unroll
                        for (int x = 0; x < MINE; ++x) {
                            if ((x + 1) * LANES > PIECES && i0 + x * LANES >= PIECES) break;
                            uint4 a, b;
                            widen(code[x], a, b);
                            *reinterpret_cast<uint4*>(first + x * ROWS * 128) = a;
                            *reinterpret_cast<uint4*>(second + x * ROWS * 128) = b;
                        }
                    } else {
                        // the few steps with drafted tokens: what is past the last token becomes 0, and so do V's infinities
                        // and NaN, which are noted
#pragma unroll 1
                        for (int x = 0; i0 + x * LANES < PIECES; ++x) {
                            uint4 c = *reinterpret_cast<const uint4*>(from + x * LANES * 16), a, b;
                            if (r0 + x * ROWS >= there) c = make_uint4(0, 0, 0, 0);
                            widen(c, a, b);
                            if (KV == kTreeFp8 && is_v && (tree_odd_chunk(a) || tree_odd_chunk(b))) {
                                odd = true;
                                tc_clear_odd(a);
                                tc_clear_odd(b);
                            }
                            *reinterpret_cast<uint4*>(first + x * ROWS * 128) = a;
                            *reinterpret_cast<uint4*>(second + x * ROWS * 128) = b;
                        }
                    }
                    if (odd) sm.odd[(k_steps + j) & 7] = k_steps + j + 1;
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                    __syncwarp();
                    if (lane == 0) { mbar_arrive(&sm.full[slot]); mbar_arrive(&sm.raw_empty[raw]); }
                    advance();
                    if (++raw == kTcRawSlots) { raw = 0; raw_phase ^= 1u; }
                }
            }
            k_steps += seg.steps;
        }
        if (!ok) { *give_up.flag = 1; atomicOr(pp.timeout, 1); }
        // every copy lands before shared memory is released, also where a wait gave up
        if (pw == 0 && lane == 0) {
            for (int i = 0; i < NS; ++i)
                if ((armed >> i) & 1u) (void)mbar_wait_drain(&sm.full[i], (armed_phase >> i) & 1u, kTcDrainPolls);
            for (int i = 0; i < kTcRawSlots; ++i)
                if ((raw_armed >> i) & 1u) (void)mbar_wait_drain(&sm.raw_full[i], (raw_armed_phase >> i) & 1u, kTcDrainPolls);
        }
        __syncwarp();
    } else {
        // ============================ tensor cores =========================
        if (lane == 0) {
            constexpr uint32_t idesc_s = (1u << 4) | ((uint32_t)(kTcStep >> 3) << 17) | ((128u >> 4) << 24);
            constexpr uint32_t idesc_o = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((128u >> 4) << 24);
            const uint32_t q_base = smem_u32(smem), ring = q_base + S::kRingAt;
            int slot = 0;
            uint32_t phase = 0;
            uint32_t q_phase = 0, p_phase[2] = {0, 0};
            auto take = [&](int& s) -> bool {   // next tile of the ring
                if (!tc_wait_one(&sm.full[slot], phase, give_up)) return false;
                s = slot;
                if (++slot == NS) { slot = 0; phase ^= 1u; }
                return true;
            };
            // addresses >> 4: a tile's second half of 64 dims, a step of 16 dims, 16 tokens
            constexpr uint32_t HALF = kTcHalf >> 4, DIMS = 32u >> 4, TOKENS = 2048u >> 4;
            auto issue_s = [&](int w, int s) {
                tc_fence_after();
                const uint32_t kb = ((ring + (uint32_t)s * S::kSlot) >> 4) | kTcLeadK;
                const uint32_t qa = ((q_base + (TILES == 2 ? w * QS : 0) * S::kSlot) >> 4) | kTcLeadK;
                const uint32_t d = tmem + 128u * w;
#pragma unroll 1
                for (int q = 0; q < QS; ++q)
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint32_t in = (uint32_t)(kk >> 2) * HALF + (uint32_t)(kk & 3) * DIMS;
                        tc_mma_ss(d, qa + (uint32_t)q * (S::kSlot >> 4) + in, kb + in, idesc_s, q || kk);
                    }
            };
            auto issue_o = [&](int w, int s, int half) {   // over half of the step's tokens
                const uint32_t vb = ((ring + (uint32_t)s * S::kSlot) >> 4) | kTcLeadV;
                const uint32_t a = tmem + 128u * w, d = tmem + 256u + 128u * w;
#pragma unroll 1
                for (int k2 = 2 * half; k2 < 2 * half + 2; ++k2)
#pragma unroll
                    for (int k1 = 0; k1 < 2; ++k1)
#pragma unroll
                        for (int q = 0; q < kTreeParts; ++q)
                            tc_mma_ts(d, a + 64u * half + 8u * (kTreeParts * (2 * (k2 & 1) + k1) + q), vb + (uint32_t)(2 * k2 + k1) * TOKENS, idesc_o, k2 || k1 || q);
            };
            // the two halves of a step's weights have a barrier each: one barrier's second completion would hide the first
            auto wait_p = [&](int w, int half) -> bool {
                if (!tc_wait_one(half ? &sm.p_full[w] : &sm.p_half[w], p_phase[w], give_up)) return false;
                if (half) p_phase[w] ^= 1u;
                tc_fence_after();
                return true;
            };
            while (ok && walk.next(p, seg)) {
                if (!tc_wait_one(&sm.q_full, q_phase, give_up)) { ok = false; break; }
                q_phase ^= 1u;
                int ks = 0, vs = 0;
                if (TILES == 2) {
                    if (!take(ks)) { ok = false; break; }
                    issue_s(0, ks);
                    umma_commit(&sm.s_full[0]);
                    issue_s(1, ks);
                    umma_commit(&sm.s_full[1]);
                    umma_commit(&sm.empty[ks]);
                    for (int j = 0; j < seg.steps && ok; ++j)
                        for (int w = 0; w < 2; ++w) {
                            if ((w == 0 && !take(vs)) || !wait_p(w, 0)) { ok = false; break; }
                            issue_o(w, vs, 0);
                            if (!wait_p(w, 1)) { ok = false; break; }
                            issue_o(w, vs, 1);
                            if (w == 1) umma_commit(&sm.empty[vs]);
                            if (j + 1 < seg.steps) {
                                if (w == 0 && !take(ks)) { ok = false; break; }
                                issue_s(w, ks);
                            }
                            umma_commit(&sm.s_full[w]);
                            if (w == 1 && j + 1 < seg.steps) umma_commit(&sm.empty[ks]);
                        }
                } else {
                    for (int w = 0; w < 2 && w < seg.steps && ok; ++w) {
                        if (!take(ks)) { ok = false; break; }
                        issue_s(w, ks);
                        umma_commit(&sm.s_full[w]);
                        umma_commit(&sm.empty[ks]);
                    }
                    for (int j = 0; j < seg.steps && ok; ++j) {
                        const int w = j & 1;
                        if (!take(vs) || !wait_p(w, 0)) { ok = false; break; }
                        issue_o(w, vs, 0);
                        if (!wait_p(w, 1)) { ok = false; break; }
                        issue_o(w, vs, 1);
                        umma_commit(&sm.empty[vs]);
                        if (j + 2 < seg.steps) {
                            if (!take(ks)) { ok = false; break; }
                            issue_s(w, ks);
                            umma_commit(&sm.empty[ks]);
                        }
                        umma_commit(&sm.s_full[w]);
                    }
                }
            }
            if (!ok) { *give_up.flag = 1; atomicOr(pp.timeout, 1); }
            // every product completes before tensor memory is released
            umma_commit(&sm.drain);
            (void)mbar_wait_drain(&sm.drain, 0u, kTcDrainPolls);
        }
        __syncwarp();
    }
    } else {
        // ============================ softmax ==============================
        tc_regs_inc<S::kSoftmaxRegs>();
        const int w = warp >> 2, quad = warp & 3, row = 32 * quad + lane;
        const uint32_t lanes = (uint32_t)(32 * quad) << 16;
        uint32_t q_phase = 0, s_phase = 0, pair_phase = 0, staged_phase = 0;
        int k_steps = 0;
        TcSegment ahead;
        bool more = walk.next(p, seg);
        for (; ok && more; seg = ahead) {
            const int rows = seg.drafted * p.group;
            // ---- q rows of the segment's tile: power-of-two scale, fp16 parts; eight lanes a row, each with every
            //      eighth group of four values ----
            {
                constexpr int G = D / 32, B = 2;                    // groups a lane; rows with loads in flight
                constexpr int NW = TILES == 2 ? 4 : 8;              // warps that share a tile's rows
                const int tile = TILES == 2 ? w : 0, mine = TILES == 2 ? quad : warp;
                unsigned char* qt = smem + tile * QS * S::kSlot;
                const float sign = p.scale < 0.f ? -1.f : 1.f;      // a row's multiplier is not negative
                const int l8 = lane & 7;
#pragma unroll 1
                for (int r0 = mine * 4 + (lane >> 3); r0 < 128; r0 += NW * 4 * B) {
                    float q[B * G][4];
                    size_t at[B * G];
#pragma unroll
                    for (int x = 0; x < B; ++x) {
                        const int pr = seg.rt * RT + tile * 128 + r0 + NW * 4 * x;
                        const bool there = pr < rows;
                        const int i = there ? pr / p.group : 0;
                        const size_t row = (size_t)(seg.row0 + i) * p.q_stride + (size_t)(seg.kvh * p.group + (there ? pr - i * p.group : 0)) * p.d;
#pragma unroll
                        for (int g = 0; g < G; ++g) {
                            const int e = 4 * (l8 + 8 * g);
                            at[x * G + g] = there && e < p.d ? row + e : kTreeNone;
                        }
                    }
                    tree_load<4, B * G>(p.q, p.q_type, at, q);
#pragma unroll
                    for (int i = 0; i < B * G; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) q[i][e] *= sign;
#pragma unroll
                    for (int x = 0; x < B; ++x) {
                        const int r = r0 + NW * 4 * x;
                        float mul = 1.0f;
                        if (p.q_type != VSPEC_B200_T_F16) {
                            float top = 0.f;
#pragma unroll
                            for (int e = 0; e < 4 * G; ++e) top = fmaxf(top, fabsf(q[x * G + e / 4][e % 4]));
#pragma unroll
                            for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                            // 2^ex with the row's largest value in [2^13, 2^14), as far as normal numbers reach
                            int ex = (int)(__float_as_uint(top) >> 23) - 126 - 14;
                            ex = top > 0.f && top <= 3.402823466e+38f ? max(-126, ex) : 0;   // at most 114
                            mul = __uint_as_float((uint32_t)(127 + ex) << 23);
                            const float inv = __uint_as_float((uint32_t)(127 - ex) << 23);
#pragma unroll
                            for (int e = 0; e < 4 * G; ++e) q[x * G + e / 4][e % 4] *= inv;
                        }
                        // a scale of 0: scores of 0 from products of any size, and -inf stays -inf
                        if (l8 == 0) sm.mul[tile * 128 + r] = fmaxf(mul * fabsf(p.scale) * kTreeLog2e, 1e-38f);
#pragma unroll
                        for (int g = 0; g < G; ++g) {
                            const int el = 4 * (l8 + 8 * g), ch = el >> 3;
                            unsigned char* at = qt + (ch >> 3) * kTcHalf + r * 128 + (((ch & 7) ^ (r & 7)) << 4) + (el & 4) * 2;
                            float (&v)[4] = q[x * G + g];
#pragma unroll
                            for (int s = 0; s < QS; ++s) {
                                const uint32_t h0 = tree_pack(v[0], v[1]), h1 = tree_pack(v[2], v[3]);
                                const float2 u0 = tree_unpack(h0), u1 = tree_unpack(h1);
                                v[0] -= u0.x; v[1] -= u0.y; v[2] -= u1.x; v[3] -= u1.y;
                                *reinterpret_cast<uint2*>(at + s * S::kSlot) = make_uint2(h0, h1);
                            }
                        }
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                mbar_arrive(&sm.q_full);
                // the next segment, and its q rows into L2, while this one's products begin
                more = walk.next(p, ahead);
                if (more) {
                    const int pr = ahead.rt * RT + (TILES == 2 ? 128 * w : 0) + row;
                    if ((TILES == 2 || w == 0) && pr < ahead.drafted * p.group) {
                        const int i = pr / p.group, es = p.q_type == VSPEC_B200_T_F32 ? 4 : 2;
                        const char* at = (const char*)p.q + ((size_t)(ahead.row0 + i) * p.q_stride + (size_t)(ahead.kvh * p.group + pr - i * p.group) * p.d) * es;
                        for (int x = 0; x < p.d * es; x += 128) asm volatile("prefetch.global.L2 [%0];\n" ::"l"(at + x));
                    }
                }
                if (!tc_wait(&sm.q_full, q_phase, give_up)) { ok = false; break; }
                q_phase ^= 1u;
            }
            const int local = (TILES == 2 ? 128 * w : 0) + row;     // row of the tile pair
            const int pr = seg.rt * RT + local;
            const bool in = pr < rows;
            const int ti = in ? pr / p.group : 0;
            const float mul = sm.mul[local];
            // TILES = 2: this thread has its row's 128 tokens of a step and all dims.  TILES = 1: 64 of the tokens and half
            // of the dims, the other group the rest; the two agree on a step's maximum, and steps alternate between the two
            // S and O buffers, whose products are a step ahead.
            constexpr int OD = TILES == 2 ? D : D / 2, NC = TILES == 2 ? 8 : 4, LAG = TILES == 2 ? 1 : 2;
            const int col0 = TILES == 2 ? 0 : 64 * w, dim0 = TILES == 2 ? 0 : OD * w;
            float o[OD];
#pragma unroll
            for (int i = 0; i < OD; ++i) o[i] = 0.f;
            float m = kTreeLowest, l = 0.f, f_even = 1.f, f_odd = 1.f;
            int v_exp = -100;
            // the product of step j: o = o f + P V
            auto add_o = [&](int j, int u, float f) {
                const int tag = k_steps + j + 1;
                tc_sweep<OD / 16, true>(tmem + lanes + 256u + 128u * u + (uint32_t)dim0, [&](int c, float (&v)[16]) {
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        float* a = o + 16 * c + i;
                        unpack2(fma2(pack2(a[0], a[1]), pack2(f, f), pack2(v[i], v[i + 1])), a[0], a[1]);
                    }
                });
                if (sm.odd[(tag - 1) & 7] == tag) {
                    // infinities and NaN that the producers took out of the step's V, for the rows that see them (committed
                    // tokens: all)
                    const int32_t* table = p.table + (size_t)seg.b * p.max_pages;
                    const int t0 = (seg.step0 + j) * kTcStep;
                    for (int t = t0; t < min(t0 + kTcStep, seg.ctx + seg.drafted); ++t) {
                        if (!in || !tree_sees(p, seg.row0, ti, seg.ctx, seg.drafted, t)) continue;
                        const size_t head = (size_t)tree_pool_row(p, table, t) * p.hkv + seg.kvh, at = head * p.d + dim0;
                        const float vs = KV == kTreeF16 ? 1.f : __ldg(p.v_scales + head);
#pragma unroll
                        for (int i = 0; i < OD; ++i) {
                            if (dim0 + i >= p.d) continue;
                            float v;
                            if (KV == kTreeF16) {
                                v = __half2float(reinterpret_cast<const __half*>(p.v_pages)[at + i]);
                            } else {
                                const uint8_t code = reinterpret_cast<const uint8_t*>(p.v_pages)[at + i];
                                v = KV == kTreeFp8 ? __half2float(__half(__nv_cvt_fp8_to_halfraw(code, __NV_E4M3))) : (float)(int8_t)code;
                                v *= vs;
                            }
                            if (!isfinite(v)) o[i] += v;
                        }
                    }
                }
            };
            const int n = seg.steps;
            // LAG passes more than steps: they add the last products
            for (int i = 0; i < n + LAG; ++i) {
                const int u = TILES == 2 ? w : i & 1;
                if (i < n || i >= LAG) {
                    if (!tc_wait(&sm.s_full[u], (s_phase >> u) & 1u, give_up)) { ok = false; break; }
                    s_phase ^= 1u << u;
                    tc_fence_after();
                }
                const bool even = TILES == 2 || u == 0;
                if (i >= LAG) add_o(i - LAG, u, even ? f_even : f_odd);
                if (i >= n) continue;
                const uint32_t s_addr = tmem + lanes + 128u * u + (uint32_t)col0;
                const int t0 = (seg.step0 + i) * kTcStep + col0, e4 = (k_steps + i) & 3;
                const bool masked = (seg.step0 + i + 1) * kTcStep > seg.ctx;
                if (KV != kTreeF16 && !tc_wait(&sm.sc_full[e4], (uint32_t)((k_steps + i) >> 2) & 1u, give_up)) { ok = false; break; }
                const float* ks = KV == kTreeF16 ? nullptr : sc.k[e4] + col0;
                if (masked) {
                    // what the row does not see becomes -inf in S; the scales of K are applied on the way
#pragma unroll 1
                    for (int c = 0; c < NC; ++c) {
                        float v[16];
                        tmem_ld_x16(s_addr + 16u * c, v);
                        const uint32_t see = in ? tc_sees32(p, seg.row0, ti, seg.drafted, t0 + 16 * c - seg.ctx) : 0u;
                        tc_landed(v);
                        uint32_t h[16];
#pragma unroll
                        for (int x = 0; x < 16; ++x) {
                            if (KV != kTreeF16) v[x] *= ks[16 * c + x];
                            h[x] = (see >> x) & 1u ? __float_as_uint(v[x]) : 0xFF800000u;
                        }
                        tc_st_x16(s_addr + 16u * c, h);
                    }
                    tmem_wait_st();
                    ks = sc.one;
                }
                // ---- the step's unit: the largest V scale, where drafted tokens are among them the largest that the row
                //      sees (a larger one beside it would push its weights below fp16), looked up if it can matter ----
                int ex = -100;
                bool own_unit = false;
                if (KV != kTreeF16) {
                    ex = sc.v_exp[e4];
                    own_unit = masked && __any_sync(0xffffffffu, ex > v_exp);
                    if (own_unit) {
                        float v_top = 0.f;
#pragma unroll 1
                        for (int c = 0; c < 16 * NC; c += 16) {
                            const uint32_t see = in ? tc_sees32(p, seg.row0, ti, seg.drafted, t0 + c - seg.ctx) : 0u;
#pragma unroll
                            for (int x = 0; x < 16; x += 4) {
                                const float4 k = *reinterpret_cast<const float4*>(&sc.v[e4][col0 + c + x]);
                                v_top = fmaxf(v_top, fmaxf(fmaxf((see >> x) & 1u ? k.x : 0.f, (see >> (x + 1)) & 1u ? k.y : 0.f),
                                                           fmaxf((see >> (x + 2)) & 1u ? k.z : 0.f, (see >> (x + 3)) & 1u ? k.w : 0.f)));
                            }
                        }
                        ex = max((int)(__float_as_uint(v_top) >> 23) - 126, -100);
                    }
                }
                // ---- maximum ----
                float tops[2] = {-INFINITY, -INFINITY};
                tc_sweep<NC, false>(s_addr, [&](int c, float (&v)[16]) {
                    tc_scale<KV != kTreeF16>(v, ks + 16 * c);
#pragma unroll
                    for (int x = 0; x < 16; ++x) tops[x & 1] = fmaxf(tops[x & 1], v[x]);
                });
                float top = fmaxf(tops[0], tops[1]);
                if (TILES == 1) {
                    // behind this wait the other group has read its part of the O buffer, too
                    sm.row[i & 1][w][row] = top;
                    if (KV != kTreeF16 && own_unit) sm.v_exp[i & 1][w][row] = ex;
                    tc_fence_before();
                    mbar_arrive(&sm.pair);
                    if (!tc_wait(&sm.pair, pair_phase, give_up)) { ok = false; break; }
                    pair_phase ^= 1u;
                    tc_fence_after();
                    top = fmaxf(top, sm.row[i & 1][w ^ 1][row]);
                    if (KV != kTreeF16 && own_unit) ex = max(ex, sm.v_exp[i & 1][w ^ 1][row]);
                }
                const float m_new = top == -INFINITY ? m : fmaxf(m, top * mul);
                const float f = tree_ex2(m - m_new);
                float fo = f;                // O is kept in units of 2^v_exp, l is not
                m = m_new;
                if (KV != kTreeF16) {
                    if (ex > v_exp) {
                        fo *= ldexpf(1.0f, max(v_exp - ex, -126));
                        v_exp = ex;
                    }
                }
                if (even) f_even = fo; else f_odd = fo;
                // ---- weights 2^(s - m + 14 - v_exp), over S: 16 tokens at a time ----
                const float bias = (KV == kTreeF16 ? 14.f : (float)(14 - v_exp)) - m_new;
                pair32 ls[2] = {0, 0};
                tc_sweep<NC, false>(s_addr, [&](int c, float (&v)[16]) {
                    tc_scale<KV != kTreeF16>(v, ks + 16 * c);
#pragma unroll
                    for (int x = 0; x < 16; x += 2) {
                        float a, b;
                        unpack2(fma2(pack2(v[x], v[x + 1]), pack2(mul, mul), pack2(bias, bias)), a, b);
                        v[x] = tree_ex2(a);
                        v[x + 1] = tree_ex2(b);
                        ls[(x >> 1) & 1] = add2(ls[(x >> 1) & 1], pack2(v[x], v[x + 1]));
                    }
                    tc_scale<KV != kTreeF16>(v, &sc.v[e4][col0 + 16 * c]);
                    uint32_t h[8];
#pragma unroll
                    for (int x = 0; x < 8; ++x) h[x] = tree_pack(v[2 * x], v[2 * x + 1]);
                    // 8 columns of high parts, then 8 of low parts, where the 16 scores were
                    const uint32_t to = s_addr + 16u * c;
                    tc_st_x8(to, h);
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const float2 y = tree_unpack(h[x]);
                        float a, b;
                        unpack2(add2(pack2(v[2 * x], v[2 * x + 1]), pack2(-y.x, -y.y)), a, b);
                        h[x] = tree_pack(a, b);
                    }
                    tc_st_x8(to + 8u, h);
                    if ((c & 3) == 3) {      // half of the step's weights are there
                        tmem_wait_st();
                        tc_fence_before();
                        mbar_arrive((TILES == 2 ? c == 3 : w == 0) ? &sm.p_half[u] : &sm.p_full[u]);
                    }
                });
                const float sum = (low2(ls[0]) + high2(ls[0])) + (low2(ls[1]) + high2(ls[1]));
                l = fmaf(l, f, sum * (KV == kTreeF16 ? 1.0f / kTreePScale : __uint_as_float((uint32_t)(127 + v_exp - 14) << 23)));
                if (KV != kTreeF16) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sm.sc_empty[e4]);
                }
            }
            if (!ok) break;
            k_steps += n;
            // ---- the rows: natural scale, out ----
            const float unit = ldexpf(1.0f / kTreePScale, KV == kTreeF16 ? 0 : v_exp);
#pragma unroll
            for (int i = 0; i < OD; ++i) o[i] *= unit;
            if (TILES == 1) {
                // the weights of the other group's tokens
                sm.row[n & 1][w][row] = l;
                mbar_arrive(&sm.pair);
                if (!tc_wait(&sm.pair, pair_phase, give_up)) { ok = false; break; }
                pair_phase ^= 1u;
                l += sm.row[n & 1][w ^ 1][row];
            }
            // rows out through this warp's part of the q tile, whose products are done, CW values of each at a time: a
            // lane puts its row in, then lanes side by side store pieces of one row
            constexpr int kStageWarps = TILES == 2 ? 4 : 8;
            constexpr int CW = QS * S::kSlot / (kStageWarps * 128) < 64 ? QS * S::kSlot / (kStageWarps * 128) : 64, LPR = CW / 4;
            const bool whole = seg.steps == seg.n;
            const size_t part = (size_t)(2 * blockIdx.x + (seg.step0 == 0 ? 1 : 0)) * RT + local;
            const float inv = !whole ? 1.f : (l == 0.f ? 0.f : 1.0f / l);
            // where this lane's row goes
            const size_t out_at = !in ? kTreeNone : !whole ? part * p.d
                : ((size_t)(seg.row0 + ti) * p.hq + (size_t)seg.kvh * p.group + (pr - ti * p.group)) * p.d;
            const uint32_t mine_lo = (uint32_t)out_at, mine_hi = (uint32_t)(out_at >> 32);
            float4* stage = reinterpret_cast<float4*>(smem + (TILES == 2 ? w * QS : 0) * S::kSlot + (TILES == 2 ? quad : warp) * (32 * CW * 4));
            constexpr int SW = LPR < 8 ? LPR - 1 : 7;
#pragma unroll
            for (int c = 0; c < OD / CW; ++c) {
                __syncwarp();
#pragma unroll
                for (int i = 0; i < LPR; ++i) {
                    const float* v = o + CW * c + 4 * i;
                    stage[lane * LPR + (i ^ (lane & SW))] = whole && l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                        : make_float4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
                }
                __syncwarp();
                const int piece = lane % LPR, e = dim0 + CW * c + 4 * piece;
#pragma unroll 4
                for (int i = 0; i < 32; i += 32 / LPR) {
                    const int r = i + lane / LPR;
                    const float4 v = stage[r * LPR + (piece ^ (r & SW))];
                    const size_t at = __shfl_sync(0xffffffffu, mine_lo, r) | (size_t)__shfl_sync(0xffffffffu, mine_hi, r) << 32;
                    if (at != kTreeNone && e < p.d) {
                        if (whole) tree_store4(p.out, p.q_type, at + e, v, 1.f, false);
                        else *reinterpret_cast<float4*>(p.part_o + at + e) = v;
                    }
                }
            }
            if (!whole && in && (TILES == 2 || w == 0)) *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(m, l);
            // every warp's stage has been read before any writes the next segment's q there
            uint64_t* read = TILES == 1 ? &sm.pair : &sm.staged[w];
            mbar_arrive(read);
            if (!tc_wait(read, TILES == 1 ? pair_phase : staged_phase, give_up)) { ok = false; break; }
            if (TILES == 1) pair_phase ^= 1u; else staged_phase ^= 1u;
            tc_fence_after();
        }
        if (!ok) { *give_up.flag = 1; atomicOr(pp.timeout, 1); }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kTcMmaWarp) tmem_dealloc(tmem, 512);
}

// Joins the parts of the pairs that were cut.  Block column x stands for the cut
// between CTAs x and x + 1; the first cut within a pair joins all its parts, in
// order: the first is in the second part slot of its CTA, the others in the
// first of theirs.
template <int RT>
__global__ void __launch_bounds__(256) tree_tc_combine_kernel(const TreeParams p) {
    pdl_trigger();
    // lengths come from before the attention kernel, which has waited for them: where the cut lies is found while it
    // still runs
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, most = gridDim.x + 1, cut = blockIdx.x + 1;
    long long total = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
        int n, tiles;
        long long w = b0 + lane < p.batch ? tc_work<RT>(p, b0 + lane, n, tiles) : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
        total += w;
    }
    const int g = tc_ctas(total, most);
    // one block waits whatever its cut, so that this grid never completes before the attention kernel
    if (cut == 1 && blockIdx.y == 0) pdl_wait();
    if (cut >= g) return;
    const long long at = total * cut / g;      // first step behind the cut
    // its sequence
    long long before = 0;
    int b = -1;
    for (int b0 = 0; b0 < p.batch && b < 0; b0 += 32) {
        int n, tiles;
        const long long w = b0 + lane < p.batch ? tc_work<RT>(p, b0 + lane, n, tiles) : 0;
        long long incl = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += u;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + incl > at);
        if (hit) {
            const int x = __ffs(hit) - 1;
            b = b0 + x;
            before += __shfl_sync(0xffffffffu, incl - w, x);
        } else {
            before += __shfl_sync(0xffffffffu, incl, 31);
        }
    }
    int n, tiles, row0;
    (void)tc_work<RT>(p, b, n, tiles);
    const int drafted = tree_rows(p, b, row0), rows = drafted * p.group;
    const int units = n + p.pair_cost, pair = (int)((at - before) / units);
    const long long start = before + (long long)pair * units + p.pair_cost;   // the pair's first step
    if (at <= start) return;                   // between two pairs
    // the CTA of unit s: the largest c with total c / g <= s
    const int first = (int)(((start + 1) * g + total - 1) / total) - 1;
    const int last = (int)(((start + n) * g + total - 1) / total) - 1;
    if (first != cut - 1) return;              // not the pair's first cut
    pdl_wait();
    const int kvh = pair / tiles, rt = pair - kvh * tiles;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml);
    // four rows a warp, their loads in flight together
    constexpr int R = 4;
    const int local0 = (blockIdx.y * 8 + warp) * R, e = lane * 4;
    if (rt * RT + local0 >= rows) return;
    float M[R], L[R];
    float4 acc[R];
#pragma unroll
    for (int r = 0; r < R; ++r) { M[r] = kTreeLowest; L[r] = 0.f; acc[r] = make_float4(0.f, 0.f, 0.f, 0.f); }
    for (int c0 = first; c0 <= last; c0 += 32) {   // a lane a part
        const bool there = c0 + lane <= last;
        const size_t at = (size_t)(2 * (c0 + lane) + (c0 + lane == first ? 1 : 0)) * RT + local0;
#pragma unroll
        for (int r = 0; r < R; ++r) M[r] = fmaxf(M[r], there ? ml[at + r].x : kTreeLowest);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) M[r] = warp_max(M[r]);
    for (int c0 = first; c0 <= last; c0 += 32) {
        const bool there = c0 + lane <= last;
        const size_t at = (size_t)(2 * (c0 + lane) + (c0 + lane == first ? 1 : 0)) * RT + local0;
        float w[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float2 x = there ? ml[at + r] : make_float2(kTreeLowest, 0.f);
            w[r] = tree_ex2(x.x - M[r]);
            L[r] += warp_sum(x.y * w[r]);
        }
        const int k = min(32, last - c0 + 1);
#pragma unroll 2
        for (int i = 0; i < k; ++i) {
            const size_t from = ((size_t)(2 * (c0 + i) + (c0 + i == first ? 1 : 0)) * RT + local0) * p.d + e;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float f = __shfl_sync(0xffffffffu, w[r], i);
                if (e < p.d) {
                    const float4 v = *reinterpret_cast<const float4*>(p.part_o + from + (size_t)r * p.d);
                    // a row past the pair's last holds what an earlier call left: its sums are not stored
                    acc[r].x += v.x * f; acc[r].y += v.y * f; acc[r].z += v.z * f; acc[r].w += v.w * f;
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int pr = rt * RT + local0 + r, i = pr / p.group;
        if (pr < rows && e < p.d)
            tree_store4(p.out, p.q_type, ((size_t)(row0 + i) * p.hq + (size_t)kvh * p.group + (pr - i * p.group)) * p.d + e, acc[r],
                        L[r] == 0.f ? 0.f : 1.0f / L[r], L[r] == 0.f);
    }
}

template <int D, int TILES, int QS, int KV>
cudaError_t tree_tc_launch_one(const TcParams& pp, int ctas, cudaStream_t st) {
    static int configured[64] = {0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    constexpr uint32_t bytes = TcShape<D, TILES, QS, KV>::kTotal;
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        e = cudaFuncSetAttribute(tree_tc_kernel<D, TILES, QS, KV>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) configured[dev] = 1;
    }
    e = launch_pdl(tree_tc_kernel<D, TILES, QS, KV>, dim3(ctas), dim3(TcShape<D, TILES, QS, KV>::kThreads), bytes, st, pp);
    if (e != cudaSuccess) return e;
    if (ctas == 1) return cudaSuccess;
    return launch_pdl(tree_tc_combine_kernel<128 * TILES>, dim3(ctas - 1, 4 * TILES), dim3(256), 0, st, pp.t);
}

// Row tiles a CTA: two for pairs of more than 128 rows; over 8-bit pages only for
// heads of at most 64 and 16-bit q.  Heads of 128 need 128 registers for a row's
// output, which beside the widening warps' share spill (one tile / two, fp16 q,
// fp8 pages of 512..8192 tokens, us: 16 x 256 rows 216 / 264, 4 x 132 rows 69 /
// 91; heads of 64: 199 / 166, 64 / 62), and two tiles' two-part q has no room.
constexpr bool tree_tc_two_tiles(int d, bool f16_pages, bool f32_q) { return f16_pages || (d <= 64 && !f32_q); }

template <int D, int KV>
cudaError_t tree_tc_pick(const TcParams& pp, int ctas, cudaStream_t st) {
    constexpr bool f16 = KV == kTreeF16;
    const bool two = pp.t.q_type == VSPEC_B200_T_F32, many = pp.t.max_q * pp.t.group > 128;
    if constexpr (tree_tc_two_tiles(D, f16, true))
        if (many && two) return tree_tc_launch_one<D, 2, 2, KV>(pp, ctas, st);
    if constexpr (tree_tc_two_tiles(D, f16, false))
        if (many && !two) return tree_tc_launch_one<D, 2, 1, KV>(pp, ctas, st);
    return two ? tree_tc_launch_one<D, 1, 2, KV>(pp, ctas, st) : tree_tc_launch_one<D, 1, 1, KV>(pp, ctas, st);
}

// Boxes of box_rows pool rows x one KV head x 64 fp16 values or a whole row of D codes.
inline int tree_tc_map(CUtensorMap* map, const void* pages, const TreeParams& p, bool f16, int box_rows) {
    PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
    if (!enc) { set_error("cuTensorMapEncodeTiled unavailable"); return VSPEC_B200_ERR_CUDA; }
    const cuuint64_t es = f16 ? 2 : 1;
    cuuint64_t dims[3] = {(cuuint64_t)p.d, (cuuint64_t)p.hkv, (cuuint64_t)p.num_pages * (cuuint64_t)p.page_tokens};
    cuuint64_t strides[2] = {(cuuint64_t)p.d * es, (cuuint64_t)p.hkv * p.d * es};
    cuuint32_t box[3] = {f16 ? 64u : (p.d <= 64 ? 64u : 128u), 1u, (cuuint32_t)box_rows};
    cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = enc(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 3,
                           const_cast<void*>(pages), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           f16 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) { set_error("cuTensorMapEncodeTiled failed (%d)", (int)r); return VSPEC_B200_ERR_CUDA; }
    return VSPEC_B200_OK;
}

template <int KV>
cudaError_t tree_tc_launch(const TcParams& pp, int ctas, cudaStream_t st) {
    return pp.t.d <= 64 ? tree_tc_pick<64, KV>(pp, ctas, st) : tree_tc_pick<128, KV>(pp, ctas, st);
}

// one translation unit per page type
extern template cudaError_t tree_tc_launch<kTreeF16>(const TcParams&, int, cudaStream_t);
extern template cudaError_t tree_tc_launch<kTreeFp8>(const TcParams&, int, cudaStream_t);
extern template cudaError_t tree_tc_launch<kTreeInt8>(const TcParams&, int, cudaStream_t);

}  // namespace vb200
