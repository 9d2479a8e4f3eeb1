// tree_attention.cu -- entry point of the tree attention: argument checks, the
// plan (rows and context of a CTA) and the kernel that joins context pieces.
#include "attention_kernels.cuh"
#include "thread_scratch.cuh"
#include "tree_attention_tc.cuh"

#include <limits.h>
#include <string.h>

#include <atomic>

namespace vb200 {

// WARPS warps a (drafted token, head): out = sum_s O_s 2^(m_s - M) / sum_s l_s 2^(m_s - M), warp w
// taking the pieces w, w + WARPS, ... in order, the warps' sums added in theirs.
template <int WARPS>
__global__ void __launch_bounds__(256) tree_combine_kernel(const TreeParams p) {
    __shared__ float4 sums[WARPS > 1 ? WARPS : 1][WARPS > 1 ? 64 : 1];
    __shared__ float lsum[WARPS];
    pdl_wait();
    pdl_trigger();
    const int b = blockIdx.y;
    int row0;
    const int drafted = tree_rows(p, b, row0);
    const int lane = threadIdx.x & 31, w = WARPS > 1 ? (int)threadIdx.x >> 5 : 0;
    const long long r = WARPS > 1 ? (long long)blockIdx.x : (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (r >= (long long)drafted * p.hq) return;   // the same for all warps of a row
    const int total = tree_ctx(p, b) + drafted;
    const int n = tree_pieces(p, total);
    if (n <= 1) return;
    const size_t row = (size_t)row0 * p.hq + (size_t)r;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + row * p.max_splits;
    float M = kTreeLowest;
#pragma unroll 4
    for (int s = lane; s < n; s += 32) M = fmaxf(M, ml[s].x);
    M = warp_max(M);
    const float* part = p.part_o + row * p.max_splits * p.d;
    // 32 of the warp's pieces at a time, a lane holding the weight of one; eight pieces' loads in flight
    const int mine = (n - w + WARPS - 1) / WARPS;   // pieces of this warp
    float L = 0.f;
    float4 acc[2] = {};
    for (int i0 = 0; i0 < mine; i0 += 32) {
        const float2 one = i0 + lane < mine ? ml[w + (i0 + lane) * WARPS] : make_float2(kTreeLowest, 0.f);
        const float f_own = tree_ex2(one.x - M);
        L += warp_sum(one.y * f_own);
        const int k = min(32, mine - i0);
#pragma unroll 8
        for (int i = 0; i < k; ++i) {
            const float f = __shfl_sync(0xffffffffu, f_own, i);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int e = lane * 4 + 128 * x;
                if (e < p.d) {
                    const float4 v = *reinterpret_cast<const float4*>(part + (size_t)(w + (i0 + i) * WARPS) * p.d + e);
                    acc[x].x += v.x * f; acc[x].y += v.y * f; acc[x].z += v.z * f; acc[x].w += v.w * f;
                }
            }
        }
    }
    if constexpr (WARPS > 1) {
        sums[w][lane] = acc[0];
        sums[w][32 + lane] = acc[1];
        if (lane == 0) lsum[w] = L;
        __syncthreads();
        if (w != 0) return;
#pragma unroll
        for (int v = 1; v < WARPS; ++v) {
            L += lsum[v];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const float4 o = sums[v][32 * x + lane];
                acc[x].x += o.x; acc[x].y += o.y; acc[x].z += o.z; acc[x].w += o.w;
            }
        }
    }
    const float inv = L == 0.f ? 0.f : 1.0f / L;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int e = lane * 4 + 128 * x;
        if (e < p.d) tree_store4(p.out, p.q_type, row * p.d + e, acc[x], inv, L == 0.f);
    }
}

__device__ int g_tree_timeout = 0;

static int* tree_timeout_ptr() {
    static int* ptr[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
    if (!ptr[dev]) {
        void* p = nullptr;
        if (cudaGetSymbolAddress(&p, g_tree_timeout) != cudaSuccess) return nullptr;
        ptr[dev] = reinterpret_cast<int*>(p);
    }
    return ptr[dev];
}

// Above this many pieces eight warps join a row, else one.  4 rows a pair, 8 KV heads, one warp / eight,
// us: 19 pieces (8 x 2048 tokens) 32 / 29, 64 pieces (1 x 8192) 35 / 20, 128 (1 x 32768) 108 / 54.
constexpr int kCombineWide = 8;

struct TreePlan {
    bool tc;
    int ctas, pair_cost;                               // tcgen05 kernel
    int wr, row_tiles, split_tokens, max_splits;       // warp-MMA kernel
};

// Which kernel: rows are a pair's at most, its drafted tokens times the group's
// heads.  The warp-MMA kernel's time grows with a pair's 16-row tiles, the tcgen05
// kernel's, whose tile is 128 rows, does not, but its first result comes later
// (22 us a call with next to nothing to read, against 13 to 20).  So tcgen05 from
// 17 rows on if tiles * tokens of all pairs reach 2^18, and above 64 rows, where
// the other kernel reads the cache more than once, always.  Warp-MMA / tcgen05, us,
// f16 queries, heads of 128, 8 KV heads, f16 pages, fp8 pages:
//   16 rows:  1 x 8192 tokens  25 /  41,  26 /  46,  16 x 2048  55 /  56,  65 /  71,  16 x 8192 122 / 154, 181 / 188
//   32 rows:  1 x 8192         31 /  42,  33 /  47,   4 x 2048  30 /  30,  32 /  35,  16 x 1024  60 /  38,  63 /  52
//   64 rows:  1 x 2048         19 /  26,  24 /  29,   4 x  512  21 /  22,  24 /  26,  16 x 2048 121 /  58, 144 /  72
//  128 rows:  1 x  256         19 /  22,  20 /  22,   4 x 1024  49 /  26,  52 /  29,  16 x 2048 170 /  59, 218 /  74
// fp32 queries move both sides by about a fifth (32 rows, 4 x 2048: 34 / 32).  Other
// heads and numbers of KV heads go by the same rule; they were not timed.
// Heads above 128 do not fit the tcgen05 kernel's registers (a row's output a
// thread), pages of other than 8 k tokens its TMA boxes.
static bool tree_uses_tc(long long rows, double tokens, size_t d, size_t page_tokens) {
    return d <= 128 && page_tokens % 8 == 0 &&
           (rows > 64 || (rows > 16 && (double)((rows + 15) / 16) * tokens >= (double)(1 << 18)));
}

// What a change of pairs costs the tcgen05 kernel in its steps (q rows in, rows
// out, an empty pipeline).  Sequences of 512..8192 tokens, 8 KV heads, us with 2 /
// 3 / 4 / 6 / 8: 32 of 256 rows, fp32 q and fp16 pages 377 / 346 / 334 / 314 / 313,
// fp16 q (one part a weight then) 267 / - / 241 / 226; 32 of 96 rows 196 / 185 /
// 179 / 179.  Steps on 8-bit pages take longer, fp16 q with 3 / 4: 32 of 256 rows
// 430 / 417, 16 of 256 218 / 216, heads of 64 162 / 165; with 2 / 3 / 4 / 6 (one
// part a weight) 8 of 64 rows (1024..6144 tokens) 59.1 / 57.8 / 61.2 / 60.7.
static int tree_pair_cost(long long rows, bool f16) { return f16 ? (rows > 128 ? 6 : 4) : (rows > 128 ? 4 : 3); }

// Warp-MMA: rows a CTA 16, 32 or 64, the fewest that hold a pair's rows; context
// pieces: about four CTAs for each that is resident at once (sequences differ
// in length), at least 128 tokens each.
static TreePlan tree_plan(size_t batch, size_t max_q, size_t hq, size_t hkv, size_t d, size_t page_tokens, size_t max_ctx,
                          bool f16) {
    TreePlan t = {};
    const long long rows = (long long)max_q * (long long)(hq / hkv);
    t.tc = tree_uses_tc(rows, (double)batch * (double)hkv * (double)max_ctx, d, page_tokens);
    if (t.tc) {
        t.pair_cost = tree_pair_cost(rows, f16);
        const double units = (double)batch * (double)hkv * (double)((rows + 127) / 128) *
                             (double)(((long long)max_ctx + kTcStep - 1) / kTcStep + t.pair_cost);
        const int most = device_sm_count();
        t.ctas = units < 3.0 * most ? (int)((units + 2) / 3) : most;
        t.max_splits = 1;
        return t;
    }
    t.wr = rows <= 16 ? 1 : (rows <= 32 ? 2 : 4);
    t.row_tiles = (int)((rows + 16 * t.wr - 1) / (16 * t.wr));
    const long long pairs = (long long)batch * hkv * t.row_tiles;
    const long long want = 4LL * 2 * device_sm_count();
    const long long pieces = pairs >= want ? 1 : (want + pairs - 1) / pairs;
    long long s = (((long long)max_ctx + pieces - 1) / pieces + kTreeTile - 1) / kTreeTile * kTreeTile;
    if (s < 128) s = 128;
    t.split_tokens = (int)s;
    t.max_splits = (int)(((long long)max_ctx + s - 1) / s);
    if (t.max_splits < 1) t.max_splits = 1;
    return t;
}

// Part slots of the plan: (O, m, l) each.
static size_t tree_parts(const TreePlan& t, size_t total_q, size_t max_q, size_t hq, size_t hkv) {
    if (t.tc) return (size_t)2 * t.ctas * (max_q * (hq / hkv) > 128 ? 256 : 128);
    return t.max_splits > 1 ? total_q * hq * (size_t)t.max_splits : 0;
}

static std::atomic<long long> g_tree_wait_cycles{kTcWaitCycles};

static thread_local ThreadScratch g_tree_scratch;

}  // namespace vb200

using namespace vb200;

extern "C" int vspec_b200_tree_attention_timeout_flag(int* out_flag) {
    if (!out_flag) { set_error("NULL out_flag"); return VSPEC_B200_ERR_ARG; }
    int v = 0, zero = 0;
    VB_CHECK_CUDA(cudaMemcpyFromSymbol(&v, g_tree_timeout, sizeof(int)));
    VB_CHECK_CUDA(cudaMemcpyToSymbol(g_tree_timeout, &zero, sizeof(int)));
    *out_flag = v;
    return VSPEC_B200_OK;
}

// Test hook: cycles after which a wait of the tcgen05 kernel gives up (negative: the default).
extern "C" int vspec_b200_debug_tree_wait_cycles(long long cycles) {
    g_tree_wait_cycles = cycles < 0 ? kTcWaitCycles : cycles;
    return VSPEC_B200_OK;
}

extern "C" size_t vspec_b200_tree_attention_workspace_bytes(size_t batch, size_t total_q, size_t max_q, size_t hq,
                                                            size_t hkv, size_t d, size_t max_ctx) {
    if (batch == 0 || max_q == 0 || hq == 0 || hkv == 0 || hq % hkv != 0 || d == 0 || max_ctx == 0 ||
        max_ctx > (size_t)INT_MAX || batch > 65535 || max_q > (size_t)INT_MAX / hq)
        return 0;
    // the larger of the two kernels' (the page size decides between them; fp16 pages take the most CTAs)
    const size_t a = tree_parts(tree_plan(batch, max_q, hq, hkv, d, 8, max_ctx, true), total_q, max_q, hq, hkv);
    const size_t b = tree_parts(tree_plan(batch, max_q, hq, hkv, d, 1, max_ctx, true), total_q, max_q, hq, hkv);
    return (a > b ? a : b) * (d + 2) * sizeof(float);
}

extern "C" int vspec_b200_tree_attention(const VspecB200TreeAttnArgs* a, void* stream) {
    if (!a) { set_error("args is NULL"); return VSPEC_B200_ERR_ARG; }
    if (!elem_type_known(a->q_dtype)) { set_error("bad q_dtype %d", a->q_dtype); return VSPEC_B200_ERR_ARG; }
    const bool f16 = a->kv_dtype == VSPEC_B200_KV_F16;
    if (!f16 && a->kv_dtype != VSPEC_B200_KV_FP8 && a->kv_dtype != VSPEC_B200_KV_INT8) {
        set_error("kv_dtype must be KV_F16, KV_FP8 or KV_INT8"); return VSPEC_B200_ERR_ARG;
    }
    if (!a->d_q || !a->d_k_pages || !a->d_v_pages || !a->d_page_table || !a->d_ctx_len || !a->d_out ||
        (!f16 && (!a->d_k_scales || !a->d_v_scales))) {
        set_error("NULL pointer argument"); return VSPEC_B200_ERR_ARG;
    }
    if (a->batch == 0 || a->max_q == 0 || a->num_q_heads == 0 || a->num_kv_heads == 0 || a->head_dim == 0 ||
        a->page_tokens == 0 || a->max_pages_per_seq == 0 || a->num_pages == 0) {
        set_error("zero dimension"); return VSPEC_B200_ERR_ARG;
    }
    if (a->num_q_heads % a->num_kv_heads != 0) { set_error("num_q_heads must be a multiple of num_kv_heads"); return VSPEC_B200_ERR_ARG; }
    if (a->head_dim > 256 || a->head_dim % (f16 ? 8 : 16) != 0) {
        set_error("head_dim must be a multiple of %d, at most 256", f16 ? 8 : 16); return VSPEC_B200_ERR_UNSUPPORTED;
    }
    const size_t lim = (size_t)INT_MAX;
    if (a->batch > 65535 || a->num_q_heads > 65535 || a->max_q > lim / a->num_q_heads / 4 || a->total_q > lim ||
        a->page_tokens > lim || a->num_pages > lim / a->page_tokens || a->max_pages_per_seq > lim) {
        set_error("a size is too large"); return VSPEC_B200_ERR_ARG;
    }
    const size_t cap = a->max_pages_per_seq * a->page_tokens;
    if (a->max_ctx > cap) { set_error("max_ctx %zu exceeds the page table capacity %zu", a->max_ctx, cap); return VSPEC_B200_ERR_ARG; }
    const size_t max_ctx = a->max_ctx ? a->max_ctx : cap;
    if (max_ctx > lim - 1024) { set_error("a size is too large"); return VSPEC_B200_ERR_ARG; }
    if (a->d_mask && a->mask_words < (a->max_q + 31) / 32) { set_error("mask_words %zu is below ceil(max_q / 32)", a->mask_words); return VSPEC_B200_ERR_ARG; }
    if (a->mask_words > lim) { set_error("a size is too large"); return VSPEC_B200_ERR_ARG; }
    if (!a->d_cu_q && a->total_q != a->batch * a->max_q) { set_error("without d_cu_q total_q is batch * max_q"); return VSPEC_B200_ERR_ARG; }
    const size_t qd = a->num_q_heads * a->head_dim;
    if (a->q_stride && (a->q_stride < qd || a->q_stride % 8 != 0)) { set_error("q_stride must be a multiple of 8 and at least heads * head_dim"); return VSPEC_B200_ERR_ARG; }
    const uintptr_t al = (uintptr_t)a->d_q | (uintptr_t)a->d_k_pages | (uintptr_t)a->d_v_pages | (uintptr_t)a->d_out |
                         (f16 ? 0 : (uintptr_t)a->d_k_scales | (uintptr_t)a->d_v_scales);
    if (al % 16 != 0) { set_error("q, out, pages and scales must be 16-byte aligned"); return VSPEC_B200_ERR_ARG; }
    if (off_type(4, {a->d_page_table, a->d_ctx_len, a->d_cu_q, a->d_mask})) { set_error("table, d_ctx_len, d_cu_q and d_mask must be aligned to 4 bytes"); return VSPEC_B200_ERR_ARG; }
    if (a->total_q == 0) return VSPEC_B200_OK;

    const TreePlan plan = tree_plan(a->batch, a->max_q, a->num_q_heads, a->num_kv_heads, a->head_dim, a->page_tokens, max_ctx, f16);
    TreeParams p;
    memset(&p, 0, sizeof(p));
    p.q = a->d_q;
    p.k_pages = a->d_k_pages; p.v_pages = a->d_v_pages;
    p.k_scales = a->d_k_scales; p.v_scales = a->d_v_scales;
    p.table = a->d_page_table;
    p.ctx_len = a->d_ctx_len;
    p.cu_q = a->d_cu_q;
    p.mask = a->d_mask;
    p.out = a->d_out;
    p.q_stride = a->q_stride ? a->q_stride : qd;
    p.scale = a->scale;
    p.batch = (int)a->batch; p.total_q = (int)a->total_q; p.max_q = (int)a->max_q;
    p.hq = (int)a->num_q_heads; p.hkv = (int)a->num_kv_heads; p.group = p.hq / p.hkv; p.d = (int)a->head_dim;
    p.page_tokens = (int)a->page_tokens; p.max_pages = (int)a->max_pages_per_seq; p.num_pages = (int)a->num_pages;
    p.mask_words = (int)a->mask_words;
    const size_t most = lim - 4096 - a->max_q;
    p.table_tokens = (int)(cap < most ? cap : most);
    p.split_tokens = plan.split_tokens; p.max_splits = plan.max_splits; p.row_tiles = plan.row_tiles;
    p.pair_cost = plan.pair_cost;
    p.q_type = a->q_dtype;
    if ((size_t)p.hkv * p.row_tiles > 65535) { set_error("a size is too large"); return VSPEC_B200_ERR_ARG; }
    p.fault = attn_page_fault_device_ptr();
    if (!p.fault) return cuda_status(cudaGetLastError(), "page fault flag");
    const size_t parts = tree_parts(plan, a->total_q, a->max_q, a->num_q_heads, a->num_kv_heads);
    const size_t need = parts * (a->head_dim + 2) * sizeof(float);
    if (need) {
        void* ws = a->d_workspace;
        if (ws) {
            if (a->workspace_bytes < need) { set_error("workspace too small (%zu < %zu)", a->workspace_bytes, need); return VSPEC_B200_ERR_ARG; }
            if ((uintptr_t)ws % 16 != 0) { set_error("workspace must be 16-byte aligned"); return VSPEC_B200_ERR_ARG; }
        } else {
            const int rc = g_tree_scratch.get(need, 0, (cudaStream_t)stream, &ws);
            if (rc != VSPEC_B200_OK) return rc;
        }
        p.part_o = (float*)ws;
        p.part_ml = p.part_o + parts * a->head_dim;
    }
    cudaStream_t st = (cudaStream_t)stream;
    if (plan.tc) {
        TcParams pp;
        memset(&pp, 0, sizeof(pp));
        pp.t = p;
        pp.timeout = tree_timeout_ptr();
        if (!pp.timeout) return cuda_status(cudaGetLastError(), "timeout flag");
        pp.wait_cycles = g_tree_wait_cycles;
        pp.box_rows = 8;   // the largest power of two that divides the page, up to a whole step
        while (pp.box_rows < kTcStep && p.page_tokens % (2 * pp.box_rows) == 0) pp.box_rows *= 2;
        int rc = tree_tc_map(&pp.k_map, p.k_pages, p, f16, pp.box_rows);
        if (rc == VSPEC_B200_OK) rc = tree_tc_map(&pp.v_map, p.v_pages, p, f16, pp.box_rows);
        if (rc != VSPEC_B200_OK) return rc;
        const cudaError_t e = f16 ? tree_tc_launch<kTreeF16>(pp, plan.ctas, st)
                            : a->kv_dtype == VSPEC_B200_KV_FP8 ? tree_tc_launch<kTreeFp8>(pp, plan.ctas, st)
                                                               : tree_tc_launch<kTreeInt8>(pp, plan.ctas, st);
        return e == cudaSuccess ? VSPEC_B200_OK : cuda_status(e, "tree attention launch");
    }
    cudaError_t e = f16 ? tree_mma_launch<kTreeF16>(p, plan.wr, st)
                  : a->kv_dtype == VSPEC_B200_KV_FP8 ? tree_mma_launch<kTreeFp8>(p, plan.wr, st)
                                                     : tree_mma_launch<kTreeInt8>(p, plan.wr, st);
    if (e != cudaSuccess) return cuda_status(e, "tree attention launch");
    if (p.max_splits > 1) {
        const size_t per = (size_t)p.max_q * p.hq;
        e = p.max_splits > kCombineWide
                ? launch_pdl(tree_combine_kernel<8>, dim3((unsigned)per, p.batch), dim3(256), 0, st, p)
                : launch_pdl(tree_combine_kernel<1>, dim3((unsigned)((per + 7) / 8), p.batch), dim3(256), 0, st, p);
        if (e != cudaSuccess) return cuda_status(e, "tree attention combine launch");
    }
    return VSPEC_B200_OK;
}
