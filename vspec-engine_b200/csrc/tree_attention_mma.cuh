// tree_attention_mma.cuh -- tree attention on warp-level tensor-core MMA: few
// query rows, any head size.
//
// The rows of a (sequence, KV head) pair are its drafted tokens times the query
// heads of the group (row r = token r / group, head r % group).  A CTA takes
// 16 * WR of them and a piece of the context, 64 tokens at a time; its four
// warps are WR row warps x 4/WR token warps, so that a small tree still has
// every warp at work on tokens.  Softmax runs online in fp32 registers
//   m' = max(m, s),  l' = l 2^(m-m') + sum 2^(s-m'),  O' = O 2^(m-m') + P V,
// token warps join in shared memory, context pieces in a second kernel in piece
// order.
//
// Products are fp16 with fp32 accumulation.  K and V codes of every page type
// are exact in fp16; their scales multiply scores and weights, not codes.  An
// fp32 q row is scaled by a power of two and split into hi + lo fp16 parts (22
// bits, two MMAs), and so are the weights P for every type: one part's rounding,
// 2^-12, would show beside that of an fp16 result (error 2.9e-4 of the result in
// place of 2.1e-4).  P is kept times 2^14 (and, over 8-bit pages, times the V
// scale over a running power of two), so that small weights stay normal.
//
// Bound by the latency of a short chain of loads when there is little to read:
// 8 drafted tokens over 768, 4 heads a KV head, 15.3 us in a graph with the joining
// kernel.  8 x 32768 tokens, 4 rows a pair: 203 us with fp16 q, 5.3 TB/s of fp16
// pages, 258 us with fp32 q.  32 x 1 tokens over 2048..6144: 118 us of fp16 pages
// (5.5 TB/s), 170 of fp8 (twice the steps a byte).
#pragma once

#include "tc_primitives.cuh"
#include "tree_attention.cuh"

#include <cuda_fp8.h>

namespace vb200 {

constexpr int kTreeThreads = 128;
constexpr int kTreeTile = 64;                      // tokens a step
constexpr int kTreeF16 = 0, kTreeFp8 = 1, kTreeInt8 = 2;
constexpr int kTreeParts = 2;                      // fp16 parts of a weight

__device__ __forceinline__ float tree_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void tree_cp16(uint32_t dst, const void* src, uint32_t src_bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ void tree_ldsm(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tree_ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t tree_pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 tree_unpack(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// Whether any of eight fp16 values is an infinity or NaN.
__device__ __forceinline__ int tree_odd_chunk(const uint4 v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    int odd = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) odd |= (w[e] & 0x7C00u) == 0x7C00u || (w[e] & 0x7C000000u) == 0x7C000000u;
    return odd;
}

// Four 8-bit codes to four exact fp16 values.
template <int KV>
__device__ __forceinline__ void tree_widen(uint32_t w, uint32_t& a, uint32_t& b) {
    if (KV == kTreeFp8) {
        asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %2;\ncvt.rn.f16x2.e4m3x2 %0, lo;\ncvt.rn.f16x2.e4m3x2 %1, hi;\n}"
            : "=r"(a), "=r"(b) : "r"(w));
    } else {
        // 0x64uu is 1024 + u; u = code + 128, so subtracting 1152 leaves the code
        const uint32_t u = w ^ 0x80808080u;
        const uint32_t m1152 = f16x2_bits(1152.0, 1152.0);
        a = hsub2_bits(__byte_perm(u, 0x64646464u, 0x4140), m1152);
        b = hsub2_bits(__byte_perm(u, 0x64646464u, 0x4342), m1152);
    }
}

template <int D, int WR, int QS>
struct TreeSmem {
    static constexpr uint32_t kRows = 16 * WR;
    static constexpr uint32_t kQ = QS * kRows * D * 2;
    static constexpr uint32_t kTileBytes = kTreeTile * D * 2;      // K or V of a step
    static constexpr uint32_t kTotal = kQ + 4 * kTileBytes;        // two stages of K and V
};

template <int D, int WR, int QS, int KV>
__global__ void __launch_bounds__(kTreeThreads) tree_mma_kernel(const TreeParams p) {
    pdl_wait();
    pdl_trigger();
    using S = TreeSmem<D, WR, QS>;
    constexpr int MT = 16 * WR, WT = 4 / WR, NT = kTreeTile / WT;
    constexpr int CH = D / 8;                       // 16-byte chunks a row of fp16
    const int split = blockIdx.x;
    const int kvh = blockIdx.y / p.row_tiles, rt = blockIdx.y % p.row_tiles;
    const int b = blockIdx.z;
    int row0;
    const int drafted = tree_rows(p, b, row0);
    const int rows = drafted * p.group;             // of this pair
    if (rt * MT >= rows) return;
    const int ctx = tree_ctx(p, b);
    const int total = ctx + drafted;
    const int t_begin = split * p.split_tokens;
    if (t_begin >= total) return;                   // gridDim.x is max_splits
    const int nsplit = tree_pieces(p, total);
    const int t_end = split + 1 == nsplit ? total : t_begin + p.split_tokens;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int g = lane >> 2, c = lane & 3;
    const int wr = warp % WR, wt = warp / WR;
    const int32_t* table = p.table + (size_t)b * p.max_pages;

    extern __shared__ __align__(128) unsigned char smem[];
    const uint32_t q_base = smem_u32(smem), kv_base = q_base + S::kQ;
    __shared__ int sm_row[2][kTreeTile];            // pool rows of a step's tokens
    __shared__ float sm_scale[2][2][kTreeTile];     // K and V scales of a step's tokens (8-bit pages)
    __shared__ float sm_mul[MT];                    // score multiplier of each row
    __shared__ float sm_ml[WT][MT][2];

    const int ntiles = (t_end - t_begin + kTreeTile - 1) / kTreeTile;
    auto find_rows = [&](int it) {                  // threads 0..63: pool row of token `tid` of step it
        const int t = t_begin + it * kTreeTile + tid;
        return t < t_end ? tree_pool_row(p, table, t) : -1;
    };
    if (tid < kTreeTile) {
        sm_row[0][tid] = find_rows(0);
        if (ntiles > 1) sm_row[1][tid] = find_rows(1);
    }

    // ---- q rows: power-of-two scale, fp16 parts, swizzled (chunk x of row r at x ^ (r & 7)) ----
    {
        constexpr int E = D / 32, B = 4;             // values a lane and row; rows with loads in flight
        float q[B][E];
#pragma unroll 1
        for (int r0 = warp; r0 < MT; r0 += 4 * B) {
        size_t at[B];
#pragma unroll
        for (int x = 0; x < B; ++x) {
            const int pr = rt * MT + r0 + 4 * x;
            at[x] = pr < rows && lane * E < p.d ? (size_t)(row0 + pr / p.group) * p.q_stride +
                                                      (size_t)(kvh * p.group + pr % p.group) * p.d + lane * E
                                                : kTreeNone;
        }
        tree_load<E, B>(p.q, p.q_type, at, q);
#pragma unroll
        for (int x = 0; x < B; ++x) {
            const int r = r0 + 4 * x;
            float (&v)[E] = q[x];
            float top = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) top = fmaxf(top, fabsf(v[e]));
            float mul = 1.0f;
            if (p.q_type != VSPEC_B200_T_F16) {
                top = warp_max(top);
                int ex = 14;
                if (top > 0.f && top <= 3.402823466e+38f) (void)frexpf(top, &ex);
                ex = max(-126, ex - 14);             // at most 114
                mul = ldexpf(1.0f, ex);
                const float inv = ldexpf(1.0f, -ex);
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] *= inv;
            }
            if (lane == 0) sm_mul[r] = mul * p.scale * kTreeLog2e;
            const uint32_t at = (uint32_t)r * (D * 2) + ((uint32_t)(((lane * E) / 8) ^ (r & 7)) << 4) + ((lane * E) % 8) * 2;
#pragma unroll
            for (int s = 0; s < QS; ++s) {
                uint32_t w[E / 2];
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    w[e / 2] = tree_pack(v[e], v[e + 1]);
                    const float2 hi = tree_unpack(w[e / 2]);
                    v[e] -= hi.x;
                    v[e + 1] -= hi.y;
                }
                unsigned char* dst = smem + s * (MT * D * 2) + at;
#pragma unroll
                for (int e = 0; e < E / 2; ++e) reinterpret_cast<uint32_t*>(dst)[e] = w[e];
            }
        }
        }
    }
    __syncthreads();

    // ---- K and V of a step into its stage ----
    const size_t pool_stride = (size_t)p.hkv * p.d;
    auto stage_addr = [&](int it) { return kv_base + (uint32_t)(it & 1) * 2u * S::kTileBytes; };
    auto issue_f16 = [&](int it) {
        const uint32_t st = stage_addr(it);
        const __half* kp = reinterpret_cast<const __half*>(p.k_pages) + (size_t)kvh * p.d;
        const __half* vp = reinterpret_cast<const __half*>(p.v_pages) + (size_t)kvh * p.d;
#pragma unroll
        for (int i = 0; i < kTreeTile * CH / kTreeThreads; ++i) {
            const int idx = i * kTreeThreads + tid, r = idx / CH, ch = idx % CH;
            const int pool = sm_row[it & 1][r];
            const bool ok = pool >= 0 && ch * 8 < p.d;
            const size_t from = ok ? (size_t)pool * pool_stride + ch * 8 : 0;
            const uint32_t to = st + (uint32_t)r * (D * 2) + ((uint32_t)(ch ^ (r & 7)) << 4);
            tree_cp16(to, kp + from, ok ? 16u : 0u);
            tree_cp16(to + S::kTileBytes, vp + from, ok ? 16u : 0u);
        }
    };
    constexpr int PC = D / 16;                       // 16-byte pieces a row of codes
    constexpr int NP = kTreeTile * PC / kTreeThreads;
    uint4 codes[KV == kTreeF16 ? 1 : 2 * NP];
    float my_scale = 0.f;
    auto fetch_codes = [&](int it) {
        if (KV == kTreeF16) return;
        const uint8_t* kp = reinterpret_cast<const uint8_t*>(p.k_pages) + (size_t)kvh * p.d;
        const uint8_t* vp = reinterpret_cast<const uint8_t*>(p.v_pages) + (size_t)kvh * p.d;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int idx = i * kTreeThreads + tid, r = idx / PC, pc = idx % PC;
            const int pool = sm_row[it & 1][r];
            const bool ok = pool >= 0 && pc * 16 < p.d;
            const size_t from = ok ? (size_t)pool * pool_stride + pc * 16 : 0;
            codes[i] = ok ? ldg_stream_v4(kp + from) : make_uint4(0, 0, 0, 0);
            codes[NP + i] = ok ? ldg_stream_v4(vp + from) : make_uint4(0, 0, 0, 0);
        }
        const int pool = sm_row[it & 1][tid & 63];
        my_scale = pool < 0 ? 0.f : __ldg((tid < 64 ? p.k_scales : p.v_scales) + (size_t)pool * p.hkv + kvh);
    };
    auto store_codes = [&](int it) {
        if (KV == kTreeF16) return;
        unsigned char* st = smem + S::kQ + (uint32_t)(it & 1) * 2u * S::kTileBytes;
#pragma unroll
        for (int i = 0; i < 2 * NP; ++i) {
            const int idx = (i % NP) * kTreeThreads + tid, r = idx / PC, pc = idx % PC;
            unsigned char* row = st + (i / NP) * S::kTileBytes + r * (D * 2);
            uint4 lo, hi;
            tree_widen<KV>(codes[i].x, lo.x, lo.y);
            tree_widen<KV>(codes[i].y, lo.z, lo.w);
            tree_widen<KV>(codes[i].z, hi.x, hi.y);
            tree_widen<KV>(codes[i].w, hi.z, hi.w);
            *reinterpret_cast<uint4*>(row + (((2 * pc) ^ (r & 7)) << 4)) = lo;
            *reinterpret_cast<uint4*>(row + (((2 * pc + 1) ^ (r & 7)) << 4)) = hi;
        }
        sm_scale[it & 1][tid >> 6][tid & 63] = my_scale;
    };
    if (KV == kTreeF16) {
        issue_f16(0);
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    } else {
        fetch_codes(0);
        store_codes(0);
    }

    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m_run[2] = {kTreeLowest, kTreeLowest}, l_run[2] = {0.f, 0.f};
    int v_exp[2] = {-100, -100};                     // 8-bit pages: a row's weights carry V scale / 2^v_exp
    float v_mul[2];                                  // 2^(14 - v_exp)
    v_mul[0] = v_mul[1] = KV == kTreeF16 ? kTreePScale : __uint_as_float((127u + 114u) << 23);
    const float mul0 = sm_mul[wr * 16 + g], mul1 = sm_mul[wr * 16 + g + 8];
    const int pr0 = rt * MT + wr * 16 + g, pr1 = pr0 + 8;   // rows of the pair
    const int a_row = wr * 16 + (lane & 15), a_hi = lane >> 4;
    const int k_row = (lane & 7) + 8 * (lane >> 4), k_hi = (lane >> 3) & 1;
    const int v_row = lane & 15, v_hi = lane >> 4;

    for (int it = 0; it < ntiles; ++it) {
        const int t0 = t_begin + it * kTreeTile;
        int next_row = -1;
        if (it + 1 < ntiles) {
            if (KV == kTreeF16) issue_f16(it + 1); else fetch_codes(it + 1);
        }
        if (KV == kTreeF16) asm volatile("cp.async.commit_group;\n" ::: "memory");
        if (it + 2 < ntiles && tid < kTreeTile) next_row = find_rows(it + 2);
        if (KV == kTreeF16) asm volatile("cp.async.wait_group 1;\n" ::: "memory");
        __syncthreads();                             // step it has landed for every thread
        const uint32_t st_k = stage_addr(it), st_v = st_k + S::kTileBytes;
        const bool masked = t0 + kTreeTile > ctx;    // drafted tokens or the end inside

        // ---- S = Q K^T ----
        float s[NT / 8][4];
#pragma unroll
        for (int n = 0; n < NT / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            uint32_t a[QS][4];
#pragma unroll
            for (int q = 0; q < QS; ++q)
                tree_ldsm(q_base + (uint32_t)(q * MT + a_row) * (D * 2) +
                              ((uint32_t)((2 * kk + a_hi) ^ (a_row & 7)) << 4), a[q]);
#pragma unroll
            for (int n2 = 0; n2 < NT / 16; ++n2) {
                const int r = wt * NT + n2 * 16 + k_row;
                uint32_t kb[4];
                tree_ldsm(st_k + (uint32_t)r * (D * 2) + ((uint32_t)((2 * kk + k_hi) ^ (r & 7)) << 4), kb);
#pragma unroll
                for (int q = 0; q < QS; ++q) {
                    mma_16816_f16_acc(s[2 * n2], a[q], kb[0], kb[1]);
                    mma_16816_f16_acc(s[2 * n2 + 1], a[q], kb[2], kb[3]);
                }
            }
        }
        // ---- scores, mask, running maximum ----
        uint32_t seen = 0xffffffffu;                 // bit 4n + e: s[n][e]
        if (masked) {
            seen = 0u;
            const int i0 = pr0 / p.group, i1 = pr1 / p.group;
#pragma unroll
            for (int n = 0; n < NT / 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int t = t0 + wt * NT + n * 8 + 2 * c + (e & 1);
                    const bool ok = t < t_end && (e < 2 ? pr0 : pr1) < rows &&
                                    tree_sees(p, row0, e < 2 ? i0 : i1, ctx, drafted, t);
                    seen |= (ok ? 1u : 0u) << (4 * n + e);
                }
        }
        float top0 = kTreeLowest, top1 = kTreeLowest;
#pragma unroll
        for (int n = 0; n < NT / 8; ++n) {
            float k0 = 1.f, k1 = 1.f;
            if (KV != kTreeF16) {
                const float2 ks = *reinterpret_cast<const float2*>(&sm_scale[it & 1][0][wt * NT + n * 8 + 2 * c]);
                k0 = ks.x; k1 = ks.y;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x = s[n][e] * (e < 2 ? mul0 : mul1);
                if (KV != kTreeF16) x *= (e & 1) ? k1 : k0;
                s[n][e] = (seen >> (4 * n + e)) & 1u ? x : -INFINITY;
            }
            top0 = fmaxf(top0, fmaxf(s[n][0], s[n][1]));
            top1 = fmaxf(top1, fmaxf(s[n][2], s[n][3]));
        }
#pragma unroll
        for (int x = 1; x <= 2; x <<= 1) {
            top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, x));
            top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, x));
        }
        const float n0 = fmaxf(m_run[0], top0), n1 = fmaxf(m_run[1], top1);
        float f0 = tree_ex2(m_run[0] - n0), f1 = tree_ex2(m_run[1] - n1);
        m_run[0] = n0; m_run[1] = n1;
        l_run[0] *= f0; l_run[1] *= f1;
        if (KV != kTreeF16) {
            // the unit goes by what the row sees: a larger scale beside it would push its weights below fp16
            float top[2] = {0.f, 0.f};
            if (!masked) {
                const float2 vs = *reinterpret_cast<const float2*>(&sm_scale[it & 1][1][2 * lane]);
                if (vs.x <= 3.402823466e+38f) top[0] = vs.x;
                if (vs.y <= 3.402823466e+38f) top[0] = fmaxf(top[0], vs.y);
                top[0] = top[1] = warp_max(top[0]);
            } else {
#pragma unroll
                for (int n = 0; n < NT / 8; ++n) {
                    const float2 vs = *reinterpret_cast<const float2*>(&sm_scale[it & 1][1][wt * NT + n * 8 + 2 * c]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float v = (e & 1) ? vs.y : vs.x;
                        if (((seen >> (4 * n + e)) & 1u) && v <= 3.402823466e+38f) top[e >> 1] = fmaxf(top[e >> 1], v);
                    }
                }
#pragma unroll
                for (int x = 1; x <= 2; x <<= 1) {
                    top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], x));
                    top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], x));
                }
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int ex = max((int)(__float_as_uint(top[x]) >> 23) - 126, -100);
                if (ex > v_exp[x]) {
                    (x ? f1 : f0) *= __uint_as_float((uint32_t)(127 + max(v_exp[x] - ex, -126)) << 23);
                    v_mul[x] = __uint_as_float((uint32_t)(127 + 14 - ex) << 23);
                    v_exp[x] = ex;
                }
            }
        }
        // ---- weights ----
#pragma unroll
        for (int n = 0; n < NT / 8; ++n) {
            float2 vs = {1.f, 1.f};
            if (KV != kTreeF16) vs = *reinterpret_cast<const float2*>(&sm_scale[it & 1][1][wt * NT + n * 8 + 2 * c]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = tree_ex2(s[n][e] - (e < 2 ? n0 : n1));
                l_run[e >> 1] += x;
                // a weight of 0 must not meet the V scale of a token that the row does not see
                s[n][e] = KV == kTreeF16 || ((seen >> (4 * n + e)) & 1u) ? x * (v_mul[e >> 1] * ((e & 1) ? vs.y : vs.x)) : 0.f;
            }
        }
        // ---- a non-finite V among drafted tokens: its product goes to the rows that see it, and the value is
        //      replaced by 0, so that the weight 0 of every other row leaves nothing ----
        if (masked && KV != kTreeInt8) {
            unsigned char* vt = smem + (st_v - q_base);
            int odd = 0;
            for (int i = tid; i < kTreeTile * CH; i += kTreeThreads) odd |= tree_odd_chunk(*reinterpret_cast<const uint4*>(vt + i * 16));
            if (__syncthreads_or(odd)) {
                // an infinity must not meet a factor of 0 below
                const float z0 = f0 == 0.f ? 0.f : 1.f, z1 = f1 == 0.f ? 0.f : 1.f;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) { o[i][0] *= z0; o[i][1] *= z0; o[i][2] *= z1; o[i][3] *= z1; }
                if (f0 == 0.f) f0 = 1.f;
                if (f1 == 0.f) f1 = 1.f;
#pragma unroll
                for (int n = 0; n < NT / 8; ++n)
                    for (int j = 0; j < 8; ++j) {
                        const int from = (lane & 28) | (j >> 1);
                        const uint32_t sb = __shfl_sync(0xffffffffu, seen, from) >> (4 * n + (j & 1));
                        const float x0 = __shfl_sync(0xffffffffu, s[n][0], from), x1 = __shfl_sync(0xffffffffu, s[n][1], from);
                        const float y0 = __shfl_sync(0xffffffffu, s[n][2], from), y1 = __shfl_sync(0xffffffffu, s[n][3], from);
                        const float w0 = (j & 1) ? x1 : x0, w1 = (j & 1) ? y1 : y0;
                        const int r = wt * NT + n * 8 + j;
#pragma unroll
                        for (int i = 0; i < D / 8; ++i) {
                            const float2 v = tree_unpack(*reinterpret_cast<const uint32_t*>(vt + r * (D * 2) + ((i ^ (r & 7)) << 4) + 4 * c));
                            const float zx = isfinite(v.x) ? 0.f : v.x, zy = isfinite(v.y) ? 0.f : v.y;
                            if ((sb & 1u) && zx != 0.f) o[i][0] = fmaf(w0, zx, o[i][0]);
                            if ((sb & 1u) && zy != 0.f) o[i][1] = fmaf(w0, zy, o[i][1]);
                            if ((sb & 4u) && zx != 0.f) o[i][2] = fmaf(w1, zx, o[i][2]);
                            if ((sb & 4u) && zy != 0.f) o[i][3] = fmaf(w1, zy, o[i][3]);
                        }
                    }
                __syncthreads();
                for (int i = tid; i < kTreeTile * CH * 8; i += kTreeThreads) {
                    uint16_t* h = reinterpret_cast<uint16_t*>(vt) + i;
                    if ((*h & 0x7C00u) == 0x7C00u) *h = 0;
                }
                __syncthreads();
            }
        }
        // ---- O = O 2^(m-m') + P V.  A step's product starts from 0 and is added in fp32: the tensor cores cut
        //      off what their accumulator cannot hold, which over thousands of tokens would add up (6e-6 of the
        //      result at 8192 tokens, against 1e-6 this way) ----
        uint32_t a[NT / 16][kTreeParts][4];
#pragma unroll
        for (int k2 = 0; k2 < NT / 16; ++k2)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float lo = s[2 * k2 + (x >> 1)][(x & 1) * 2], hi = s[2 * k2 + (x >> 1)][(x & 1) * 2 + 1];
                a[k2][0][x] = tree_pack(lo, hi);
                const float2 h = tree_unpack(a[k2][0][x]);
                a[k2][1][x] = tree_pack(lo - h.x, hi - h.y);
            }
#pragma unroll
        for (int i2 = 0; i2 < D / 16; ++i2) {
            float d0[4] = {0.f, 0.f, 0.f, 0.f}, d1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k2 = 0; k2 < NT / 16; ++k2) {
                const int r = wt * NT + k2 * 16 + v_row;
                uint32_t vb[4];
                tree_ldsm_t(st_v + (uint32_t)r * (D * 2) + ((uint32_t)((2 * i2 + v_hi) ^ (r & 7)) << 4), vb);
#pragma unroll
                for (int q = 0; q < kTreeParts; ++q) {
                    mma_16816_f16_acc(d0, a[k2][q], vb[0], vb[1]);
                    mma_16816_f16_acc(d1, a[k2][q], vb[2], vb[3]);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float f = e < 2 ? f0 : f1;
                o[2 * i2][e] = fmaf(o[2 * i2][e], f, d0[e]);
                o[2 * i2 + 1][e] = fmaf(o[2 * i2 + 1][e], f, d1[e]);
            }
        }
        if (KV != kTreeF16 && it + 1 < ntiles) store_codes(it + 1);
        if (it + 2 < ntiles && tid < kTreeTile) sm_row[it & 1][tid] = next_row;
        __syncthreads();                             // every thread is done with step it and its rows
    }

    // ---- join the token warps, write ----
    float unit[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) unit[x] = KV == kTreeF16 ? 1.0f / kTreePScale : ldexpf(1.0f / kTreePScale, v_exp[x]);
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
        l_run[0] += __shfl_xor_sync(0xffffffffu, l_run[0], x);
        l_run[1] += __shfl_xor_sync(0xffffffffu, l_run[1], x);
    }
    float* sm_o = reinterpret_cast<float*>(smem + S::kQ);   // [WT][MT][D]
    if (c == 0) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            sm_ml[wt][wr * 16 + g + 8 * x][0] = m_run[x];
            sm_ml[wt][wr * 16 + g + 8 * x][1] = l_run[x];
        }
    }
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            float2 v = {o[i][2 * x] * unit[x], o[i][2 * x + 1] * unit[x]};
            *reinterpret_cast<float2*>(sm_o + ((size_t)wt * MT + wr * 16 + g + 8 * x) * D + i * 8 + 2 * c) = v;
        }
    __syncthreads();
    for (int z = tid; z < MT * (D / 4); z += kTreeThreads) {
        const int r = z / (D / 4), e = (z % (D / 4)) * 4;
        const int pr = rt * MT + r;
        if (pr >= rows || e >= p.d) continue;
        float M = sm_ml[0][r][0];
#pragma unroll
        for (int w = 1; w < WT; ++w) M = fmaxf(M, sm_ml[w][r][0]);
        float L = 0.f;
        float4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < WT; ++w) {
            const float f = tree_ex2(sm_ml[w][r][0] - M);
            const float4 v = *reinterpret_cast<const float4*>(sm_o + ((size_t)w * MT + r) * D + e);
            L += sm_ml[w][r][1] * f;
            acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
        }
        const size_t orow = (size_t)(row0 + pr / p.group) * p.hq + (size_t)kvh * p.group + pr % p.group;
        if (nsplit == 1) {
            tree_store4(p.out, p.q_type, orow * p.d + e, acc, L == 0.f ? 0.f : 1.0f / L, L == 0.f);
        } else {
            const size_t at = orow * p.max_splits + split;
            *reinterpret_cast<float4*>(p.part_o + at * p.d + e) = acc;
            if (e == 0) { p.part_ml[at * 2] = M; p.part_ml[at * 2 + 1] = L; }
        }
    }
}

template <int D, int WR, int QS, int KV>
cudaError_t tree_mma_launch_one(const TreeParams& p, cudaStream_t st) {
    static int configured[64] = {0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    constexpr uint32_t bytes = TreeSmem<D, WR, QS>::kTotal;
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        e = cudaFuncSetAttribute(tree_mma_kernel<D, WR, QS, KV>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) configured[dev] = 1;
    }
    return launch_pdl(tree_mma_kernel<D, WR, QS, KV>, dim3(p.max_splits, p.hkv * p.row_tiles, p.batch),
                      dim3(kTreeThreads), bytes, st, p);
}

template <int D, int KV>
cudaError_t tree_mma_pick(const TreeParams& p, int wr, cudaStream_t st) {
    const bool two = p.q_type == VSPEC_B200_T_F32;
    if (wr == 1) return two ? tree_mma_launch_one<D, 1, 2, KV>(p, st) : tree_mma_launch_one<D, 1, 1, KV>(p, st);
    if (wr == 2) return two ? tree_mma_launch_one<D, 2, 2, KV>(p, st) : tree_mma_launch_one<D, 2, 1, KV>(p, st);
    return two ? tree_mma_launch_one<D, 4, 2, KV>(p, st) : tree_mma_launch_one<D, 4, 1, KV>(p, st);
}

template <int KV>
cudaError_t tree_mma_launch(const TreeParams& p, int wr, cudaStream_t st) {
    return p.d <= 64 ? tree_mma_pick<64, KV>(p, wr, st)
         : p.d <= 128 ? tree_mma_pick<128, KV>(p, wr, st)
                      : tree_mma_pick<256, KV>(p, wr, st);
}

// one translation unit per page type
extern template cudaError_t tree_mma_launch<kTreeF16>(const TreeParams&, int, cudaStream_t);
extern template cudaError_t tree_mma_launch<kTreeFp8>(const TreeParams&, int, cudaStream_t);
extern template cudaError_t tree_mma_launch<kTreeInt8>(const TreeParams&, int, cudaStream_t);

}  // namespace vb200
