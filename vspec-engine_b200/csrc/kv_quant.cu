// kv_quant.cu -- 8-bit KV pages: rows quantised as they are appended, and
// whole sequences read back in token order.
//
//   scale = absmax / M,  code = round_to_even(x * (M / absmax)),  M = 448 (e4m3) or 127 (int8)
//
// one scale a row of head_dim values.  Both are memory-bound: a row is read
// once, held in registers between the maximum and the rounding, and its codes
// written once.  Measured, 8 heads of 128, replayed in a graph: 16384 rows of fp16
// to int8 20.3 us, 5.0 TB/s (77 % of a copy's rate; the SMs issue 82 % of the
// time), 512 rows of fp32 to fp8 2.4 us; 16384 tokens of fp8 pages to fp16 22.6
// us, 4.5 TB/s (69 %: the SMs issue 46 % of the time, warps wait for a token's page
// and then for its codes), 777 tokens 4.0 us.
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
    size_t k_stride, v_stride, pool_rows;
    int items, heads, d;   // items: rows * heads
    uint8_t *k_codes, *v_codes;
    float *k_scales, *v_scales;
    int* fault;
};

// Largest absolute value of a vector as fp32 bits with the sign off: ordered as unsigned, and at or above
// kInfBits when a value is not finite.
constexpr uint32_t kInfBits = 0x7F800000u;
template <typename T, int V>
__device__ __forceinline__ uint32_t abs_max_bits(const Vec<T, V>& w) {
    uint32_t m = 0;
    if constexpr (sizeof(T) == 2 && V % 2 == 0) {
        // 16-bit patterns without their signs order as unsigned halves
        const uint32_t* p = reinterpret_cast<const uint32_t*>(&w);
        uint32_t h = p[0] & 0x7FFF7FFFu;
#pragma unroll
        for (int i = 1; i < V / 2; ++i) h = __vmaxu2(h, p[i] & 0x7FFF7FFFu);
        const uint16_t top = (uint16_t)max(h & 0xFFFFu, h >> 16);
        T t;
        memcpy(&t, &top, 2);
        m = __float_as_uint(elem_to_f32<T>(t));
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) m = max(m, __float_as_uint(elem_to_f32<T>(w.e[i])) & 0x7FFFFFFFu);
    }
    return m;
}

// V codes of values times inv.  Fast: every value finite and |x * inv| at most
// M but for its rounding, so that nothing has to be caught: e4m3 by the packed
// conversion; int8 by adding 1.5 * 2^23, which leaves the integer, rounded to
// even, in the low byte of the sum.
template <bool FP8, int V>
__device__ __forceinline__ void quant_fast(const float (&x)[V], float inv, Vec<uint8_t, V>& out) {
    static_assert(V % 4 == 0, "whole words");
    uint32_t* w = reinterpret_cast<uint32_t*>(&out);
#pragma unroll
    for (int i = 0; i < V; i += 4) {
        if (FP8) {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[i] * inv, x[i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[i + 2] * inv, x[i + 3] * inv), __NV_SATFINITE, __NV_E4M3);
            w[i / 4] = lo | (hi << 16);
        } else {
            uint32_t u[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) u[e] = __float_as_uint(__fadd_rn(__fmul_rn(x[i + e], inv), 12582912.0f));
            w[i / 4] = __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
        }
    }
}
template <bool FP8>
__device__ __forceinline__ uint8_t quant_code(float x, float inv) {
    constexpr float M = FP8 ? 448.0f : 127.0f;
    float c = __fmul_rn(x, inv);
    // 0 * inf (a row of zeros) and NaN inputs store 0; what passes M saturates
    c = c == c ? fminf(fmaxf(c, -M), M) : 0.0f;
    if (FP8) return (uint8_t)__nv_cvt_float_to_fp8(c, __NV_SATFINITE, __NV_E4M3);
    return (uint8_t)(int8_t)__float2int_rn(c);
}

// 2^LL lanes a row, each with C vectors of V elements (lane l: vectors l, l +
// lanes, ...): 16-byte loads where alignment allows.  A lane group works on the
// K and the V row of one (row, head), so two loads are in flight per vector.
template <typename T, bool FP8, int V, int C, int LL>
__global__ void __launch_bounds__(kQuantThreads) kv_quant_append_kernel(const QuantParams p) {
    pdl_wait();
    pdl_trigger();
    constexpr int lanes = 1 << LL;
    const unsigned item = blockIdx.x * (kQuantThreads >> LL) + (threadIdx.x >> LL);   // < 2^31
    const int l = threadIdx.x & (lanes - 1);
    const bool inside = item < (unsigned)p.items;
    const unsigned r = inside ? item / (unsigned)p.heads : 0;
    const unsigned h = inside ? item - r * p.heads : 0;
    Vec<T, V> x[2][C];
    const int slot = !p.slots ? (int)r : p.slots[r];
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        const T* src = (side ? (const T*)p.v + r * p.v_stride : (const T*)p.k + r * p.k_stride) + h * (unsigned)p.d;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int at = (c * lanes + l) * V;
            if (inside && at < p.d) {
                x[side][c] = *reinterpret_cast<const Vec<T, V>*>(src + at);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) x[side][c].e[j] = elem_from_f32<T>(0.f);
            }
        }
    }
    uint32_t top[2] = {0u, 0u};
#pragma unroll
    for (int side = 0; side < 2; ++side) {
#pragma unroll
        for (int c = 0; c < C; ++c) top[side] = max(top[side], abs_max_bits<T, V>(x[side][c]));
#pragma unroll
        for (int o = lanes >> 1; o > 0; o >>= 1) top[side] = max(top[side], __shfl_xor_sync(0xffffffffu, top[side], o));
    }
    bool odd[2] = {false, false};   // not all values are finite
    if (__any_sync(0xffffffffu, top[0] >= kInfBits || top[1] >= kInfBits)) {
        // rare: the maximum over finite values alone
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            odd[side] = top[side] >= kInfBits;
            uint32_t m = 0;
            for (int c = 0; c < C; ++c)
                for (int j = 0; j < V; ++j) {
                    const uint32_t u = __float_as_uint(elem_to_f32<T>(x[side][c].e[j])) & 0x7FFFFFFFu;
                    if (u < kInfBits) m = max(m, u);
                }
            for (int o = lanes >> 1; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            top[side] = m;
        }
    }
    // the four quotients M / top and top / M of K and V, one a lane (LL >= 2); where M / top would leave fp32, values
    // and top are taken times 2^100
    constexpr float M = FP8 ? 448.0f : 127.0f;
    constexpr float kTiny = 1e-35f, kUp = 1.2676506002282294e30f;
    const float mine = __uint_as_float((l & 1) ? top[1] : top[0]);
    const float quot = __fdiv_rn((l & 2) ? mine : M, (l & 2) ? M : (mine > kTiny ? mine : mine * kUp));
    const float inv[2] = {__shfl_sync(0xffffffffu, quot, 0, lanes), __shfl_sync(0xffffffffu, quot, 1, lanes)};
    if (!inside || slot < 0) return;
    if ((size_t)slot >= p.pool_rows) {
        if (l == 0) atomicOr(p.fault, 1);
        return;
    }
    const size_t out_row = (size_t)slot * p.heads + h;
    if (l == 2 || l == 3) (l == 3 ? p.v_scales : p.k_scales)[out_row] = quot;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        uint8_t* dst = (side ? p.v_codes : p.k_codes) + out_row * p.d;
        const bool tiny = __uint_as_float(top[side]) <= kTiny;
        const bool fast = V % 4 == 0 && !odd[side] && !tiny;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int at = (c * lanes + l) * V;
            if (at < p.d) {
                Vec<uint8_t, V> w;
                float v[V];
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = elem_to_f32<T>(x[side][c].e[j]);
                if (fast) {
                    if constexpr (V % 4 == 0) quant_fast<FP8, V>(v, inv[side], w);
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j) w.e[j] = quant_code<FP8>(tiny ? v[j] * kUp : v[j], inv[side]);
                }
                *reinterpret_cast<Vec<uint8_t, V>*>(dst + at) = w;
            }
        }
    }
}

struct GatherParams {
    const uint8_t *k_codes, *v_codes;
    const float *k_scales, *v_scales;
    const int32_t *table, *cu;
    int total, batch, heads, d, page_tokens, max_pages, num_pages;
    unsigned head_magic;
    void *k_out, *v_out;
    int* fault;
};

// Two values rounded to T, in one word for the 16-bit types.
template <typename T> __device__ __forceinline__ Vec<T, 2> round2(float a, float b);
template <> __device__ __forceinline__ Vec<float, 2> round2<float>(float a, float b) { return {{a, b}}; }
template <> __device__ __forceinline__ Vec<__half, 2> round2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return {{h.x, h.y}};
}
template <> __device__ __forceinline__ Vec<__nv_bfloat16, 2> round2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return {{h.x, h.y}};
}

// V codes times a scale, rounded to T once.
template <typename T, bool FP8, int V>
__device__ __forceinline__ Vec<T, V> dequant(const Vec<uint8_t, V>& c, float scale) {
    Vec<T, V> out;
    if constexpr (V % 2 == 0) {
        const uint16_t* two = reinterpret_cast<const uint16_t*>(&c);
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            float2 v;
            if (FP8) {
                v = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two[j / 2], __NV_E4M3)));
            } else {
                v = make_float2((float)(int8_t)c.e[j], (float)(int8_t)c.e[j + 1]);
            }
            const Vec<T, 2> w = round2<T>(v.x * scale, v.y * scale);
            out.e[j] = w.e[0];
            out.e[j + 1] = w.e[1];
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float v = FP8 ? __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c.e[j], __NV_E4M3)))
                                : (float)(int8_t)c.e[j];
            out.e[j] = elem_from_f32<T>(v * scale);
        }
    }
    return out;
}

// One warp a token: it finds its sequence and pool row once and converts every
// head's K and V codes, which are contiguous in the pool and in the output.
template <typename T, bool FP8, int V>
__global__ void __launch_bounds__(256) kv_quant_gather_kernel(const GatherParams p) {
    pdl_wait();
    pdl_trigger();
    const int r = blockIdx.x * 8 + (threadIdx.x >> 5);   // < 2^31
    const int lane = threadIdx.x & 31;
    if (r >= p.total || r >= p.cu[p.batch]) return;
    int lo = 0, hi = p.batch - 1;              // last sequence whose first row is <= r
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.cu[mid] <= r) lo = mid; else hi = mid - 1;
    }
    const int t = r - p.cu[lo];
    if (t < 0) return;
    const int at_page = t / p.page_tokens;
    int page = at_page < p.max_pages ? p.table[(size_t)lo * p.max_pages + at_page] : -1;
    if (page < 0 || page >= p.num_pages) {
        if (lane == 0) atomicOr(p.fault, 1);
        page = 0;
    }
    const size_t row = ((size_t)page * p.page_tokens + (size_t)(t % p.page_tokens)) * p.heads;
    const int units = p.heads * p.d / V;
#pragma unroll 4
    for (int u = lane; u < units; u += 32) {
        const int h = p.head_magic ? (int)__umulhi((unsigned)u, p.head_magic) : u;   // u / (d / V)
        const size_t from = row * p.d + (size_t)u * V, to = (size_t)r * p.heads * p.d + (size_t)u * V;
        const Vec<uint8_t, V> kc = *reinterpret_cast<const Vec<uint8_t, V>*>(p.k_codes + from);
        const Vec<uint8_t, V> vc = *reinterpret_cast<const Vec<uint8_t, V>*>(p.v_codes + from);
        const float ks = p.k_scales[row + h], vs = p.v_scales[row + h];
        *reinterpret_cast<Vec<T, V>*>((T*)p.k_out + to) = dequant<T, FP8, V>(kc, ks);
        *reinterpret_cast<Vec<T, V>*>((T*)p.v_out + to) = dequant<T, FP8, V>(vc, vs);
    }
}

template <typename T, bool FP8, int V, int C, int LL>
static cudaError_t append_launch(const QuantParams& p, cudaStream_t st) {
    constexpr unsigned per = kQuantThreads >> LL;
    return launch_pdl(kv_quant_append_kernel<T, FP8, V, C, LL>, dim3(((unsigned)p.items + per - 1) / per),
                      dim3(kQuantThreads), 0, st, p);
}

// Lanes a row: 8, 16 or 32, the fewest that hold it in one vector each; longer and unaligned rows a warp.
template <typename T, bool FP8>
static cudaError_t append_pick(const QuantParams& p, bool aligned, cudaStream_t st) {
    constexpr int F = 16 / (int)sizeof(T);
    if (aligned) {
        if (p.d <= 8 * F) return append_launch<T, FP8, F, 1, 3>(p, st);
        if (p.d <= 16 * F) return append_launch<T, FP8, F, 1, 4>(p, st);
        if (p.d <= 32 * F) return append_launch<T, FP8, F, 1, 5>(p, st);
        return append_launch<T, FP8, F, kQuantMaxDim / F / 32, 5>(p, st);
    }
    return append_launch<T, FP8, 1, kQuantMaxDim / 32, 5>(p, st);
}

template <typename T, bool FP8>
static cudaError_t gather_pick(GatherParams p, uintptr_t addresses, cudaStream_t st) {
    constexpr int F = 16 / (int)sizeof(T);
    const dim3 grid((unsigned)((p.total + 7) / 8)), block(256);
    const bool wide = p.d % F == 0 && addresses % 16 == 0;
    // ceil(2^32 / n): its high product with u is u / n while u * n < 2^32 (heads * d units of n <= 512); n = 1 apart
    const unsigned n = (unsigned)(wide ? p.d / F : p.d);
    p.head_magic = n > 1 ? (unsigned)((((uint64_t)1 << 32) + n - 1) / n) : 0u;
    if (wide) return launch_pdl(kv_quant_gather_kernel<T, FP8, F>, grid, block, 0, st, p);
    return launch_pdl(kv_quant_gather_kernel<T, FP8, 1>, grid, block, 0, st, p);
}

}  // namespace vb200

using namespace vb200;

extern "C" int vspec_b200_kv_quant_append(const VspecB200KvQuantArgs* a, void* stream) {
    if (!a) { set_error("args is NULL"); return VSPEC_B200_ERR_ARG; }
    if (!elem_type_known(a->src_dtype)) { set_error("bad src_dtype %d", a->src_dtype); return VSPEC_B200_ERR_ARG; }
    if (a->kv_dtype != VSPEC_B200_KV_FP8 && a->kv_dtype != VSPEC_B200_KV_INT8) { set_error("kv_dtype must be KV_FP8 or KV_INT8"); return VSPEC_B200_ERR_ARG; }
    if (!a->d_k || !a->d_v || !a->d_k_codes || !a->d_v_codes || !a->d_k_scales || !a->d_v_scales) { set_error("NULL pointer argument"); return VSPEC_B200_ERR_ARG; }
    if (off_type(elem_bytes(a->src_dtype), {a->d_k, a->d_v}) || off_type(4, {a->d_slots, a->d_k_scales, a->d_v_scales})) {
        set_error("rows, slots and scales must be aligned to their types"); return VSPEC_B200_ERR_ARG;
    }
    if (a->num_kv_heads == 0 || a->head_dim == 0 || a->pool_rows == 0) { set_error("zero dimension"); return VSPEC_B200_ERR_ARG; }
    if (a->head_dim > kQuantMaxDim) { set_error("head_dim %zu is above %d", a->head_dim, kQuantMaxDim); return VSPEC_B200_ERR_UNSUPPORTED; }
    if (a->num_kv_heads > 8192 || a->rows > 0x7ffffff0u / a->num_kv_heads) { set_error("too many rows"); return VSPEC_B200_ERR_ARG; }
    const size_t hd = a->num_kv_heads * a->head_dim;
    QuantParams p;
    memset(&p, 0, sizeof(p));
    p.k = a->d_k; p.v = a->d_v;
    p.slots = a->d_slots;
    p.k_stride = a->k_stride ? a->k_stride : hd;
    p.v_stride = a->v_stride ? a->v_stride : hd;
    if (p.k_stride < hd || p.v_stride < hd) { set_error("a row stride is smaller than its heads"); return VSPEC_B200_ERR_ARG; }
    if (a->rows == 0) return VSPEC_B200_OK;
    p.pool_rows = a->pool_rows;
    p.heads = (int)a->num_kv_heads;
    p.items = (int)(a->rows * a->num_kv_heads);
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
    if (off_type(elem_bytes(a->out_dtype), {a->d_k_out, a->d_v_out}) ||
        off_type(4, {a->d_k_scales, a->d_v_scales, a->d_page_table, a->d_cu_tokens})) {
        set_error("scales, table, d_cu_tokens and outputs must be aligned to their types"); return VSPEC_B200_ERR_ARG;
    }
    if (a->batch == 0 || a->num_kv_heads == 0 || a->head_dim == 0 || a->page_tokens == 0 ||
        a->max_pages_per_seq == 0 || a->num_pages == 0) {
        set_error("zero dimension"); return VSPEC_B200_ERR_ARG;
    }
    const size_t lim = 0x7fffffffu;
    if (a->batch > lim || a->num_pages > lim || a->page_tokens > lim || a->max_pages_per_seq > lim ||
        a->total_tokens > lim - 8 || a->num_kv_heads > 8192 || a->head_dim > kQuantMaxDim) {
        set_error("a size is too large"); return VSPEC_B200_ERR_ARG;
    }
    if (a->total_tokens == 0) return VSPEC_B200_OK;
    GatherParams p;
    memset(&p, 0, sizeof(p));
    p.k_codes = (const uint8_t*)a->d_k_codes; p.v_codes = (const uint8_t*)a->d_v_codes;
    p.k_scales = a->d_k_scales; p.v_scales = a->d_v_scales;
    p.table = a->d_page_table; p.cu = a->d_cu_tokens;
    p.total = (int)a->total_tokens;
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
