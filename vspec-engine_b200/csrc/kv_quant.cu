// kv_quant.cu -- 8-bit KV pages: rows quantised as they are appended, and
// whole sequences read back in token order.
//
//   scale = absmax / M,  code = round_to_even(x * (M / absmax)),  M = 448 (e4m3) or 127 (int8)
//
// one scale a row of head_dim values.  Both are memory-bound: a row is read
// once, held in registers between the maximum and the rounding, and its codes
// written once.
#include "elem_types.cuh"
#include "attention_kernels.cuh"

#include <cuda_fp8.h>
#include <string.h>

namespace vb200 {

constexpr int kQuantThreads = 256;
constexpr int kQuantMaxDim = 512;

struct QuantParams {
    const void *k, *v;
    const int32_t* slots;
    size_t rows, k_stride, v_stride, pool_rows;
    int heads, d;
    uint8_t *k_codes, *v_codes;
    float *k_scales, *v_scales;
    int* fault;
};

template <bool FP8>
__device__ __forceinline__ uint8_t quant_code(float x, float inv) {
    constexpr float M = FP8 ? 448.0f : 127.0f;
    float c = x * inv;
    // 0 * inf (a row of zeros) and NaN inputs store 0; what passes M saturates
    c = c == c ? fminf(fmaxf(c, -M), M) : 0.0f;
    if (FP8) return (uint8_t)__nv_cvt_float_to_fp8(c, __NV_SATFINITE, __NV_E4M3);
    return (uint8_t)(int8_t)__float2int_rn(c);
}

// L lanes a row, each with C vectors of V elements (lane l: vectors l, l + L,
// ...): 16-byte loads where alignment allows.  A lane group works on the K and
// the V row of one (row, head), so two loads are in flight per vector.
template <typename T, bool FP8, int V, int C>
__global__ void __launch_bounds__(kQuantThreads) kv_quant_append_kernel(const QuantParams p, int lanes) {
    pdl_wait();
    pdl_trigger();
    const size_t item = ((size_t)blockIdx.x * kQuantThreads + threadIdx.x) / lanes;
    const int l = threadIdx.x % lanes;
    const size_t items = p.rows * p.heads;
    const bool inside = item < items;
    const size_t r = inside ? item / p.heads : 0;
    const int h = inside ? (int)(item % p.heads) : 0;
    float x[2][C * V];
    float top[2] = {0.f, 0.f};
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        const T* src = (side ? (const T*)p.v + r * p.v_stride : (const T*)p.k + r * p.k_stride) + (size_t)h * p.d;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int at = (c * lanes + l) * V;
            if (inside && at < p.d) {
                const Vec<T, V> w = *reinterpret_cast<const Vec<T, V>*>(src + at);
#pragma unroll
                for (int j = 0; j < V; ++j) x[side][c * V + j] = elem_to_f32<T>(w.e[j]);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) x[side][c * V + j] = 0.f;
            }
        }
    }
    const long long slot = p.slots ? (long long)p.slots[r] : (long long)r;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
#pragma unroll
        for (int j = 0; j < C * V; ++j) {
            const float a = fabsf(x[side][j]);
            if (a <= 3.402823466e+38f) top[side] = fmaxf(top[side], a);   // finite values only
        }
        for (int o = lanes >> 1; o > 0; o >>= 1) top[side] = fmaxf(top[side], __shfl_xor_sync(0xffffffffu, top[side], o));
    }
    if (!inside || slot < 0) return;
    if ((size_t)slot >= p.pool_rows) {
        if (l == 0) atomicOr(p.fault, 1);
        return;
    }
    constexpr float M = FP8 ? 448.0f : 127.0f;
    const size_t out_row = (size_t)slot * p.heads + h;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        uint8_t* dst = (side ? p.v_codes : p.k_codes) + out_row * p.d;
        const float inv = __fdiv_rn(M, top[side]);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int at = (c * lanes + l) * V;
            if (at < p.d) {
                Vec<uint8_t, V> w;
#pragma unroll
                for (int j = 0; j < V; ++j) w.e[j] = quant_code<FP8>(x[side][c * V + j], inv);
                *reinterpret_cast<Vec<uint8_t, V>*>(dst + at) = w;
            }
        }
        if (l == 0) (side ? p.v_scales : p.k_scales)[out_row] = __fdiv_rn(top[side], M);
    }
}

struct GatherParams {
    const uint8_t *k_codes, *v_codes;
    const float *k_scales, *v_scales;
    const int32_t *table, *cu;
    size_t total;
    int batch, heads, d, page_tokens, max_pages, num_pages;
    void *k_out, *v_out;
    int* fault;
};

template <bool FP8>
__device__ __forceinline__ float dequant_code(uint8_t c) {
    if (FP8) return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3)));
    return (float)(int8_t)c;
}

// One warp a token: it finds its sequence and pool row once and converts every
// head's K and V codes, which are contiguous in the pool and in the output.
template <typename T, bool FP8, int V>
__global__ void __launch_bounds__(256) kv_quant_gather_kernel(const GatherParams p) {
    pdl_wait();
    pdl_trigger();
    const size_t r = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (r >= p.total || (long long)r >= (long long)p.cu[p.batch]) return;
    int lo = 0, hi = p.batch - 1;              // last sequence whose first row is <= r
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if ((long long)p.cu[mid] <= (long long)r) lo = mid; else hi = mid - 1;
    }
    const long long t = (long long)r - p.cu[lo];
    if (t < 0) return;
    const long long at_page = t / p.page_tokens;
    int page = at_page < p.max_pages ? p.table[(size_t)lo * p.max_pages + at_page] : -1;
    if (page < 0 || page >= p.num_pages) {
        if (lane == 0) atomicOr(p.fault, 1);
        page = 0;
    }
    const size_t row = ((size_t)page * p.page_tokens + (size_t)(t % p.page_tokens)) * p.heads;
    const int units = p.heads * p.d / V;
#pragma unroll 2
    for (int u = lane; u < units; u += 32) {
        const int h = u * V / p.d;
        const size_t from = row * p.d + (size_t)u * V, to = r * p.heads * p.d + (size_t)u * V;
        const Vec<uint8_t, V> kc = *reinterpret_cast<const Vec<uint8_t, V>*>(p.k_codes + from);
        const Vec<uint8_t, V> vc = *reinterpret_cast<const Vec<uint8_t, V>*>(p.v_codes + from);
        const float ks = p.k_scales[row + h], vs = p.v_scales[row + h];
        Vec<T, V> ko, vo;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            ko.e[j] = elem_from_f32<T>(dequant_code<FP8>(kc.e[j]) * ks);
            vo.e[j] = elem_from_f32<T>(dequant_code<FP8>(vc.e[j]) * vs);
        }
        *reinterpret_cast<Vec<T, V>*>((T*)p.k_out + to) = ko;
        *reinterpret_cast<Vec<T, V>*>((T*)p.v_out + to) = vo;
    }
}

template <typename T, bool FP8, int V, int C>
static cudaError_t append_launch(const QuantParams& p, int lanes, cudaStream_t st) {
    const size_t items = p.rows * p.heads, per = kQuantThreads / lanes;
    return launch_pdl(kv_quant_append_kernel<T, FP8, V, C>, dim3((unsigned)((items + per - 1) / per)),
                      dim3(kQuantThreads), 0, st, p, lanes);
}

template <typename T, bool FP8>
static cudaError_t append_pick(const QuantParams& p, bool aligned, cudaStream_t st) {
    constexpr int F = 16 / (int)sizeof(T);
    if (aligned) {
        // the fewest lanes that hold a row in one vector each, up to a warp
        const int vecs = p.d / F;
        int lanes = 1;
        while (lanes < vecs && lanes < 32) lanes <<= 1;
        if (vecs <= lanes) return append_launch<T, FP8, F, 1>(p, lanes, st);
        return append_launch<T, FP8, F, kQuantMaxDim / F / 32>(p, 32, st);
    }
    return append_launch<T, FP8, 1, kQuantMaxDim / 32>(p, 32, st);
}

template <typename T, bool FP8>
static cudaError_t gather_pick(const GatherParams& p, uintptr_t addresses, cudaStream_t st) {
    constexpr int F = 16 / (int)sizeof(T);
    const dim3 grid((unsigned)((p.total + 7) / 8)), block(256);
    if (p.d % F == 0 && addresses % 16 == 0) return launch_pdl(kv_quant_gather_kernel<T, FP8, F>, grid, block, 0, st, p);
    return launch_pdl(kv_quant_gather_kernel<T, FP8, 1>, grid, block, 0, st, p);
}

}  // namespace vb200

using namespace vb200;

extern "C" int vspec_b200_kv_quant_append(const VspecB200KvQuantArgs* a, void* stream) {
    if (!a) { set_error("args is NULL"); return VSPEC_B200_ERR_ARG; }
    if (!elem_type_known(a->src_dtype)) { set_error("bad src_dtype %d", a->src_dtype); return VSPEC_B200_ERR_ARG; }
    if (a->kv_dtype != VSPEC_B200_KV_FP8 && a->kv_dtype != VSPEC_B200_KV_INT8) { set_error("kv_dtype must be KV_FP8 or KV_INT8"); return VSPEC_B200_ERR_ARG; }
    if (!a->d_k || !a->d_v || !a->d_k_codes || !a->d_v_codes || !a->d_k_scales || !a->d_v_scales) { set_error("NULL pointer argument"); return VSPEC_B200_ERR_ARG; }
    if (a->num_kv_heads == 0 || a->head_dim == 0 || a->pool_rows == 0) { set_error("zero dimension"); return VSPEC_B200_ERR_ARG; }
    if (a->head_dim > kQuantMaxDim) { set_error("head_dim %zu is above %d", a->head_dim, kQuantMaxDim); return VSPEC_B200_ERR_UNSUPPORTED; }
    if (a->num_kv_heads > 65535 || a->rows > 0x7fffffffu / a->num_kv_heads) { set_error("too many rows"); return VSPEC_B200_ERR_ARG; }
    const size_t hd = a->num_kv_heads * a->head_dim;
    QuantParams p;
    memset(&p, 0, sizeof(p));
    p.k = a->d_k; p.v = a->d_v;
    p.slots = a->d_slots;
    p.rows = a->rows;
    p.k_stride = a->k_stride ? a->k_stride : hd;
    p.v_stride = a->v_stride ? a->v_stride : hd;
    if (p.k_stride < hd || p.v_stride < hd) { set_error("a row stride is smaller than its heads"); return VSPEC_B200_ERR_ARG; }
    if (a->rows == 0) return VSPEC_B200_OK;
    p.pool_rows = a->pool_rows;
    p.heads = (int)a->num_kv_heads;
    p.d = (int)a->head_dim;
    p.k_codes = (uint8_t*)a->d_k_codes; p.v_codes = (uint8_t*)a->d_v_codes;
    p.k_scales = a->d_k_scales; p.v_scales = a->d_v_scales;
    p.fault = attn_page_fault_device_ptr();
    if (!p.fault) return cuda_status(cudaGetLastError(), "page fault flag");
    const bool f32 = a->src_dtype == VSPEC_B200_T_F32;
    const size_t vec = f32 ? 4 : 8;   // 16-byte loads, code vectors of as many bytes
    const bool aligned = (p.k_stride | p.v_stride | a->head_dim) % vec == 0 &&
                         ((uintptr_t)p.k | (uintptr_t)p.v) % 16 == 0 &&
                         ((uintptr_t)p.k_codes | (uintptr_t)p.v_codes) % vec == 0;
    const bool fp8 = a->kv_dtype == VSPEC_B200_KV_FP8;
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e;
    if (f32) e = fp8 ? append_pick<float, true>(p, aligned, st) : append_pick<float, false>(p, aligned, st);
    else if (a->src_dtype == VSPEC_B200_T_F16)
        e = fp8 ? append_pick<__half, true>(p, aligned, st) : append_pick<__half, false>(p, aligned, st);
    else e = fp8 ? append_pick<__nv_bfloat16, true>(p, aligned, st) : append_pick<__nv_bfloat16, false>(p, aligned, st);
    return e == cudaSuccess ? VSPEC_B200_OK : cuda_status(e, "kv_quant_append_kernel launch");
}

extern "C" int vspec_b200_kv_quant_gather(const VspecB200KvGatherArgs* a, void* stream) {
    if (!a) { set_error("args is NULL"); return VSPEC_B200_ERR_ARG; }
    if (!elem_type_known(a->out_dtype)) { set_error("bad out_dtype %d", a->out_dtype); return VSPEC_B200_ERR_ARG; }
    if (a->kv_dtype != VSPEC_B200_KV_FP8 && a->kv_dtype != VSPEC_B200_KV_INT8) { set_error("kv_dtype must be KV_FP8 or KV_INT8"); return VSPEC_B200_ERR_ARG; }
    if (!a->d_k_codes || !a->d_v_codes || !a->d_k_scales || !a->d_v_scales || !a->d_page_table || !a->d_cu_tokens ||
        !a->d_k_out || !a->d_v_out) {
        set_error("NULL pointer argument"); return VSPEC_B200_ERR_ARG;
    }
    if (a->batch == 0 || a->num_kv_heads == 0 || a->head_dim == 0 || a->page_tokens == 0 ||
        a->max_pages_per_seq == 0 || a->num_pages == 0) {
        set_error("zero dimension"); return VSPEC_B200_ERR_ARG;
    }
    const size_t lim = 0x7fffffffu;
    if (a->batch > lim || a->num_pages > lim || a->page_tokens > lim || a->max_pages_per_seq > lim ||
        a->total_tokens > lim || a->num_kv_heads > 65535 || a->head_dim > kQuantMaxDim) {
        set_error("a size is too large"); return VSPEC_B200_ERR_ARG;
    }
    if (a->total_tokens == 0) return VSPEC_B200_OK;
    GatherParams p;
    memset(&p, 0, sizeof(p));
    p.k_codes = (const uint8_t*)a->d_k_codes; p.v_codes = (const uint8_t*)a->d_v_codes;
    p.k_scales = a->d_k_scales; p.v_scales = a->d_v_scales;
    p.table = a->d_page_table; p.cu = a->d_cu_tokens;
    p.total = a->total_tokens;
    p.batch = (int)a->batch; p.heads = (int)a->num_kv_heads; p.d = (int)a->head_dim;
    p.page_tokens = (int)a->page_tokens; p.max_pages = (int)a->max_pages_per_seq; p.num_pages = (int)a->num_pages;
    p.k_out = a->d_k_out; p.v_out = a->d_v_out;
    p.fault = attn_page_fault_device_ptr();
    if (!p.fault) return cuda_status(cudaGetLastError(), "page fault flag");
    const uintptr_t addr = (uintptr_t)p.k_codes | (uintptr_t)p.v_codes | (uintptr_t)p.k_out | (uintptr_t)p.v_out;
    const bool fp8 = a->kv_dtype == VSPEC_B200_KV_FP8;
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e;
    if (a->out_dtype == VSPEC_B200_T_F32) e = fp8 ? gather_pick<float, true>(p, addr, st) : gather_pick<float, false>(p, addr, st);
    else if (a->out_dtype == VSPEC_B200_T_F16) e = fp8 ? gather_pick<__half, true>(p, addr, st) : gather_pick<__half, false>(p, addr, st);
    else e = fp8 ? gather_pick<__nv_bfloat16, true>(p, addr, st) : gather_pick<__nv_bfloat16, false>(p, addr, st);
    return e == cudaSuccess ? VSPEC_B200_OK : cuda_status(e, "kv_quant_gather_kernel launch");
}
