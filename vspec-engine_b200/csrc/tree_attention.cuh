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
    int split_tokens, max_splits, row_tiles;
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

__device__ __forceinline__ float tree_load(const void* p, int type, size_t i) {
    if (type == VSPEC_B200_T_F32) return reinterpret_cast<const float*>(p)[i];
    if (type == VSPEC_B200_T_F16) return __half2float(reinterpret_cast<const __half*>(p)[i]);
    return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void tree_store(void* p, int type, size_t i, float v) {
    if (type == VSPEC_B200_T_F32) reinterpret_cast<float*>(p)[i] = v;
    else if (type == VSPEC_B200_T_F16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
    else reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
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
