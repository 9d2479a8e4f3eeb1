// tree_attention.cuh -- internal interface of the tree attention kernels.
#pragma once

#include "elem_types.cuh"

namespace vb200 {

constexpr float kTreeLog2e = 1.4426950408889634f;
constexpr float kTreeLowest = -3.402823466e+38f;   // running maximum of a row that has seen nothing
constexpr float kTreePScale = 16384.0f;            // weights are rounded to fp16 as p * 2^14: no part underflows

struct TreeParams {
    const void* q;
    const void *k_pages, *v_pages;
    const float *k_scales, *v_scales;
    const int32_t *table, *ctx_len, *cu_q;
    const uint32_t* mask;
    void* out;
    float* part_o;    // [total_q * hq][max_splits][d], not normalised
    float* part_ml;   // [total_q * hq][max_splits][2]
    size_t q_stride;
    float scale;
    int batch, total_q, max_q, hq, hkv, group, d;
    int page_tokens, max_pages, num_pages, mask_words;
    int table_tokens;   // of a sequence's row of the table, at most what keeps positions in 32 bits
    int split_tokens, max_splits, row_tiles;   // warp-MMA kernel
    int pair_cost;                             // tcgen05 kernel: steps' worth of time a pair takes besides its steps
    int q_type;
    int* fault;
};

// Pool row of cached token t, or of page 0 with the fault flag raised where the table has none.
__device__ __forceinline__ int tree_pool_row(const TreeParams& p, const int32_t* table, int t) {
    const int at = t / p.page_tokens;
    int page = at < p.max_pages ? __ldg(table + at) : -1;
    if (page < 0 || page >= p.num_pages) {
        atomicOr(p.fault, 1);
        page = 0;
    }
    return page * p.page_tokens + (t - at * p.page_tokens);
}

// First query row of sequence b and its drafted tokens (0 for a d_cu_q that leaves [0, total_q]).
__device__ __forceinline__ int tree_rows(const TreeParams& p, int b, int& row0) {
    if (!p.cu_q) {
        row0 = b * p.max_q;
        return p.max_q;
    }
    row0 = p.cu_q[b];
    const int end = min(p.cu_q[b + 1], p.total_q);
    return row0 < 0 || row0 >= end ? 0 : min(end - row0, p.max_q);
}

// Committed tokens of sequence b.  A length past the page table is cut to it, which bounds positions and work whatever
// the length is; the drafted tokens behind have no page then, and their lookups raise the fault flag.
__device__ __forceinline__ int tree_ctx(const TreeParams& p, int b) { return min(max(p.ctx_len[b], 0), p.table_tokens); }

// Context pieces of a sequence (warp-MMA kernel); the last takes what is left, also past the caller's max_ctx.
__device__ __forceinline__ int tree_pieces(const TreeParams& p, int total) {
    return min((total + p.split_tokens - 1) / p.split_tokens, p.max_splits);
}

// N (2, 4 or 8) consecutive values of q from each of R places (multiples of N), 0
// where at[r] is kTreeNone.  Every load is issued whatever its place, so that all
// of them are in flight at once: a branch around each made them wait for one
// another (6300 cycles for eight loads against 900).
constexpr size_t kTreeNone = ~(size_t)0;
template <typename T, int N, int R>
__device__ __forceinline__ void tree_load_as(const void* p, const size_t (&at)[R], float (&v)[R][N]) {
    constexpr int M = N * sizeof(T) > 16 ? 16 / sizeof(T) : N;
    Vec<T, M> w[R][N / M];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int x = 0; x < N / M; ++x)
            w[r][x] = *reinterpret_cast<const Vec<T, M>*>(reinterpret_cast<const T*>(p) + (at[r] == kTreeNone ? 0 : at[r]) + x * M);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < N; ++e) v[r][e] = at[r] == kTreeNone ? 0.f : elem_to_f32<T>(w[r][e / M].e[e % M]);
}
template <int N, int R>
__device__ __forceinline__ void tree_load(const void* p, int type, const size_t (&at)[R], float (&v)[R][N]) {
    if (type == VSPEC_B200_T_F32) tree_load_as<float>(p, at, v);
    else if (type == VSPEC_B200_T_F16) tree_load_as<__half>(p, at, v);
    else tree_load_as<__nv_bfloat16>(p, at, v);
}

// Four values v * inv in a row (0 for a row that saw nothing), rounded once.
__device__ __forceinline__ void tree_store4(void* p, int type, size_t i, float4 v, float inv, bool empty) {
    v = empty ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    if (type == VSPEC_B200_T_F32) {
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i) = v;
    } else if (type == VSPEC_B200_T_F16) {
        Vec<__half, 4> w = {{__float2half_rn(v.x), __float2half_rn(v.y), __float2half_rn(v.z), __float2half_rn(v.w)}};
        *reinterpret_cast<Vec<__half, 4>*>(reinterpret_cast<__half*>(p) + i) = w;
    } else {
        Vec<__nv_bfloat16, 4> w = {{__float2bfloat16_rn(v.x), __float2bfloat16_rn(v.y), __float2bfloat16_rn(v.z), __float2bfloat16_rn(v.w)}};
        *reinterpret_cast<Vec<__nv_bfloat16, 4>*>(reinterpret_cast<__nv_bfloat16*>(p) + i) = w;
    }
}

// Whether row i of the tree (first mask row of the sequence: row0) sees the cached token at position t.
__device__ __forceinline__ bool tree_sees(const TreeParams& p, int row0, int i, int ctx, int drafted, int t) {
    if (t < ctx) return true;
    const int j = t - ctx;
    if (j >= drafted) return false;
    if (!p.mask) return j <= i;
    return (__ldg(p.mask + (size_t)(row0 + i) * p.mask_words + (j >> 5)) >> (j & 31)) & 1u;
}

}  // namespace vb200
