// logprobs.cu -- log probabilities of given tokens, entropy and the best
// alternatives, in one pass over the logits.
//
// With m the row's maximum, S = sum exp((x - m)/T) and U = sum exp((x - m)/T) (x - m):
//   log p(v) = (x_v - m)/T - ln S,   entropy = ln S - U / (T S).
// A thread keeps (m, S, U) of what it has read and rescales when its maximum
// grows; lanes, warps and the CTAs of a row join with the same rule.  The list
// of the best is kept by each warp, one 64-bit key a lane in order (ordered
// bits of the logit, then the complement of the id, so that ties go to the
// lowest id); a value enters it only when it passes the CTA's threshold, the
// best k-th key that any of its warps holds, so after the first few thousand
// values almost none do.
// Bound by memory: a logit is read once.  Few rows: several CTAs share a row
// and the last one to finish joins their parts in CTA order (no result depends
// on the order of arrival).
#include "elem_types.cuh"

#include <math.h>
#include <string.h>

namespace vb200 {

constexpr int kLpThreads = 512;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpMaxTop = 32;
constexpr int kLpMaxSplitRows = 2048;              // rows above this are never split
constexpr size_t kLpCounterBytes = kLpMaxSplitRows * sizeof(unsigned);
constexpr float kLpLowest = -3.402823466e+38f;

struct LpParams {
    const void* logits;
    const uint32_t* allowed;
    const int32_t* tokens;
    float *token_lp, *entropy, *top_lp;
    int32_t* top_ids;
    size_t row_stride;
    int vocab, words, num_tokens, top_k, splits, chunk;   // chunk: values a CTA
    float inv_t;
    unsigned* counters;             // [rows] with splits > 1, zero between calls
    float* part_stats;              // [rows][splits][4]
    unsigned long long* part_keys;  // [rows][splits][top_k]
};

__device__ __forceinline__ float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// max that keeps NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// 0 is the key of nothing: -inf and NaN have no key.
__device__ __forceinline__ unsigned long long lp_key(float v, int id) {
    const uint32_t u = __float_as_uint(v + 0.0f);   // -0 and +0 tie
    const uint32_t o = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((unsigned long long)o << 32) | (0xFFFFFFFFu - (uint32_t)id);
}
__device__ __forceinline__ float lp_key_value(unsigned long long k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
__device__ __forceinline__ int lp_key_id(unsigned long long k) { return (int)(0xFFFFFFFFu - (uint32_t)k); }

struct LpStats {
    float m, s, u;
};
// u of a part whose maximum grows by -d, f = 2^(d c).  Where f is 0 the product d * s may be infinite: what is left
// is 0, or the NaN that s holds.
__device__ __forceinline__ float lp_rescale_u(const LpStats& a, float d, float f) {
    return f == 0.f ? a.s * f : (a.u + d * a.s) * f;
}
// c = log2(e)/T.  A part without values has s = 0 and the lowest m.
__device__ __forceinline__ LpStats lp_join(const LpStats a, const LpStats b, float c) {
    LpStats r;
    r.m = fmaxf(a.m, b.m);
    const float da = a.m - r.m, db = b.m - r.m;
    const float fa = ex2_approx(da * c), fb = ex2_approx(db * c);
    r.s = a.s * fa + b.s * fb;
    r.u = lp_rescale_u(a, da, fa) + lp_rescale_u(b, db, fb);
    return r;
}

// A warp's best keys, lane l holding the l-th largest.
__device__ __forceinline__ void lp_insert(unsigned long long& best, unsigned long long key, int lane) {
    const int at = __popc(__ballot_sync(0xffffffffu, best > key));
    const unsigned long long up = __shfl_up_sync(0xffffffffu, best, 1);
    best = lane < at ? best : (lane == at ? key : up);
}

template <typename T, int V, bool ALLOWED, bool TOP>
__global__ void __launch_bounds__(kLpThreads) logprobs_kernel(const LpParams p) {
    pdl_wait();
    pdl_trigger();
    const size_t row = blockIdx.y;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const T* x = (const T*)p.logits + row * p.row_stride;
    const uint32_t* bits = ALLOWED ? p.allowed + row * p.words : nullptr;
    __shared__ unsigned long long sm_thr;
    __shared__ unsigned long long sm_keys[kLpWarps][kLpMaxTop];
    __shared__ LpStats sm_stats[kLpWarps];
    __shared__ unsigned sm_last;
    if (TOP && tid == 0) sm_thr = 0;
    if (TOP) __syncthreads();

    const float c = p.inv_t * 1.4426950408889634f;
    LpStats st = {kLpLowest, 0.f, 0.f};
    unsigned long long best = 0, thr = 0;
    float thr_v = -INFINITY;

    // one vector of values starting at id j; n of them count
    auto take = [&](const float (&v)[V], int j, int n) {
        uint32_t ok = n >= V ? 0xffffffffu : (n > 0 ? (1u << n) - 1u : 0u);
        if (ALLOWED && n > 0) {
            uint32_t b = bits[j >> 5] >> (j & 31);
            if ((j & 31) + (n < V ? n : V) > 32) b |= bits[(j >> 5) + 1] << (32 - (j & 31));
            ok &= b;
        }
        float w[V], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            w[i] = (ok >> i) & 1u ? v[i] : -INFINITY;
            top = fmaxf(top, w[i]);
        }
        if (top > st.m) {
            const float d = st.m - top, f = ex2_approx(d * c);
            st.u = lp_rescale_u(st, d, f);
            st.s *= f;
            st.m = top;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float d = max_nan(w[i] - st.m, kLpLowest);   // -inf - m stays finite, so that 0 * d is 0
            const float e = ex2_approx(d * c);
            st.s += e;
            st.u = fmaf(e, d, st.u);
        }
        if (TOP) {
            if (__any_sync(0xffffffffu, top >= thr_v && top > -INFINITY)) {
                const unsigned long long shared_thr = *(volatile unsigned long long*)&sm_thr;
                if (shared_thr > thr) thr = shared_thr;
                const unsigned long long before = thr;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    // NaN fails the comparison; -inf has no place in the list
                    const unsigned long long key = w[i] > -INFINITY ? lp_key(w[i], j + i) : 0ull;
                    unsigned in = __ballot_sync(0xffffffffu, key > thr);
                    while (in) {
                        const int from = __ffs(in) - 1;
                        in &= in - 1;
                        const unsigned long long k = __shfl_sync(0xffffffffu, key, from);
                        if (k > thr) {
                            lp_insert(best, k, lane);
                            const unsigned long long mine = __shfl_sync(0xffffffffu, best, p.top_k - 1);
                            if (mine > thr) thr = mine;
                        }
                    }
                }
                if (lane == 0 && thr > before) atomicMax(&sm_thr, thr);
                thr_v = thr ? lp_key_value(thr) : -INFINITY;
            }
        }
    };

    const int j0 = blockIdx.x * p.chunk, j1 = min(p.vocab, j0 + p.chunk);
    // values before the first 16-byte boundary, whole vectors, values after the last
    const int off = (int)(((uintptr_t)(x + j0) % (V * sizeof(T))) / sizeof(T));
    const int head = off ? min(V - off, j1 - j0) : 0;
    const int vecs = j1 > j0 + head ? (j1 - j0 - head) / V : 0;
    const int body = j0 + head;
    constexpr int U = 4;   // vectors in flight a thread
    using W = Vec<T, V>;
    for (int g0 = 0; g0 < vecs; g0 += kLpThreads * U) {
        W w[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int g = g0 + i * kLpThreads + tid;
            if (g < vecs) w[i] = *reinterpret_cast<const W*>(x + body + (size_t)g * V);
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int g = g0 + i * kLpThreads + tid;
            if (g0 + i * kLpThreads + warp * 32 >= vecs) break;   // the whole warp is past the end
            float v[V];
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = g < vecs ? elem_to_f32<T>(w[i].e[e]) : 0.f;
            take(v, body + g * V, g < vecs ? V : 0);
        }
    }
    // the ends, a value a lane of warp 0: lanes 0-15 the head, 16-31 the tail
    if (warp == 0) {
        const int j = lane < 16 ? j0 + lane : body + vecs * V + lane - 16;
        const bool in = lane < 16 ? lane < head : j < j1;
        float v[V];
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = 0.f;
        if (in) v[0] = elem_to_f32<T>(x[j]);
        take(v, j, in ? 1 : 0);
    }

    // ---- join the warps ----
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        LpStats q;
        q.m = __shfl_xor_sync(0xffffffffu, st.m, o);
        q.s = __shfl_xor_sync(0xffffffffu, st.s, o);
        q.u = __shfl_xor_sync(0xffffffffu, st.u, o);
        // one order for both lanes of a pair
        st = (lane & o) ? lp_join(q, st, c) : lp_join(st, q, c);
    }
    if (lane == 0) sm_stats[warp] = st;
    if (TOP) sm_keys[warp][lane] = lane < p.top_k ? best : 0ull;
    __syncthreads();
    if (warp != 0) return;
    st = sm_stats[0];
    for (int w = 1; w < kLpWarps; ++w) st = lp_join(st, sm_stats[w], c);
    if (TOP) {
        for (int w = 1; w < kLpWarps; ++w) {
            for (int i = 0; i < p.top_k; ++i) {
                const unsigned long long k = sm_keys[w][i];
                if (k <= __shfl_sync(0xffffffffu, best, p.top_k - 1)) break;   // the rest are smaller
                lp_insert(best, k, lane);
            }
        }
    }

    if (p.splits > 1) {
        const size_t at = row * p.splits + blockIdx.x;
        if (TOP && lane < p.top_k) p.part_keys[at * p.top_k + lane] = best;
        if (lane == 0) {
            p.part_stats[at * 4 + 0] = st.m;
            p.part_stats[at * 4 + 1] = st.s;
            p.part_stats[at * 4 + 2] = st.u;
        }
        __threadfence();
        __syncwarp();
        if (lane == 0) {
            sm_last = atomicAdd(&p.counters[row], 1u) == (unsigned)p.splits - 1;
            if (sm_last) p.counters[row] = 0;
        }
        __syncwarp();
        if (!sm_last) return;
        __threadfence();
        const volatile float* ps = p.part_stats + row * p.splits * 4;
        const volatile unsigned long long* pk = p.part_keys + row * p.splits * (size_t)p.top_k;
        st = {ps[0], ps[1], ps[2]};
        if (TOP) best = lane < p.top_k ? pk[lane] : 0ull;
        for (int i = 1; i < p.splits; ++i) {
            st = lp_join(st, LpStats{ps[i * 4], ps[i * 4 + 1], ps[i * 4 + 2]}, c);
            if (TOP) {
                const unsigned long long mine = lane < p.top_k ? pk[(size_t)i * p.top_k + lane] : 0ull;
                for (int e = 0; e < p.top_k; ++e) {
                    const unsigned long long k = __shfl_sync(0xffffffffu, mine, e);
                    if (k <= __shfl_sync(0xffffffffu, best, p.top_k - 1)) break;
                    lp_insert(best, k, lane);
                }
            }
        }
    }

    // ---- results ----
    const bool none = st.s == 0.f;
    const float ln_s = logf(st.s);
    if (lane == 0 && p.entropy) p.entropy[row] = none ? 0.f : ln_s - st.u * p.inv_t / st.s;
    if (TOP && lane < p.top_k) {
        const size_t at = row * p.top_k + lane;
        p.top_ids[at] = best ? lp_key_id(best) : -1;
        p.top_lp[at] = best ? (lp_key_value(best) - st.m) * p.inv_t - ln_s : -INFINITY;
    }
    for (int g = lane; g < p.num_tokens; g += 32) {
        const int id = p.tokens[row * p.num_tokens + g];
        float lp = -INFINITY;
        if (id >= 0 && id < p.vocab && (!ALLOWED || (bits[id >> 5] >> (id & 31)) & 1u)) {
            const float v = elem_to_f32<T>(x[id]);
            if (!none && v != -INFINITY) lp = (v - st.m) * p.inv_t - ln_s;
        }
        p.token_lp[row * p.num_tokens + g] = lp;
    }
}

// CTAs a row: enough for about four on every SM together, each with at least 4096 values.
static int lp_splits(size_t rows, size_t vocab) {
    if (rows >= (size_t)kLpMaxSplitRows) return 1;
    size_t s = (4 * (size_t)device_sm_count() + rows - 1) / rows;
    const size_t most = vocab / 4096;
    if (s > most) s = most;
    return s < 1 ? 1 : (int)s;
}

static size_t lp_workspace(size_t rows, size_t vocab, size_t top_k) {
    const size_t s = (size_t)lp_splits(rows, vocab);
    return s > 1 ? kLpCounterBytes + rows * s * (4 * sizeof(float) + top_k * sizeof(unsigned long long)) : 0;
}

// Library-managed scratch, one grow-only buffer per device and host thread;
// its counters are zero between calls.
struct LpScratch {
    void* ptr;
    size_t cap;
};
static thread_local LpScratch g_lp_scratch[64];

static void* lp_scratch(size_t bytes, cudaStream_t st) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
    LpScratch& s = g_lp_scratch[dev];
    if (s.cap < bytes) {
        if (s.ptr) cudaFree(s.ptr);
        s.ptr = nullptr;
        s.cap = 0;
        if (cudaMalloc(&s.ptr, bytes) != cudaSuccess) { s.ptr = nullptr; return nullptr; }
        if (cudaMemsetAsync(s.ptr, 0, kLpCounterBytes, st) != cudaSuccess) { cudaFree(s.ptr); s.ptr = nullptr; return nullptr; }
        s.cap = bytes;
    }
    return s.ptr;
}

template <typename T>
static cudaError_t lp_launch(const LpParams& p, size_t rows, cudaStream_t st) {
    constexpr int F = 16 / (int)sizeof(T);
    const dim3 grid((unsigned)p.splits, (unsigned)rows), block(kLpThreads);
    const bool top = p.top_k > 0;
    if (p.allowed)
        return top ? launch_pdl(logprobs_kernel<T, F, true, true>, grid, block, 0, st, p)
                   : launch_pdl(logprobs_kernel<T, F, true, false>, grid, block, 0, st, p);
    return top ? launch_pdl(logprobs_kernel<T, F, false, true>, grid, block, 0, st, p)
               : launch_pdl(logprobs_kernel<T, F, false, false>, grid, block, 0, st, p);
}

}  // namespace vb200

using namespace vb200;

extern "C" size_t vspec_b200_logprobs_workspace_bytes(size_t rows, size_t vocab, size_t top_k) {
    if (rows == 0 || vocab == 0 || top_k > (size_t)kLpMaxTop) return 0;
    return lp_workspace(rows, vocab, top_k);
}

extern "C" int vspec_b200_logprobs(const VspecB200LogprobsArgs* a, void* stream) {
    if (!a) { set_error("args is NULL"); return VSPEC_B200_ERR_ARG; }
    if (!elem_type_known(a->dtype)) { set_error("bad dtype %d", a->dtype); return VSPEC_B200_ERR_ARG; }
    if (!a->d_logits) { set_error("NULL pointer argument"); return VSPEC_B200_ERR_ARG; }
    if (a->vocab == 0 || a->vocab > (size_t)1 << 30) { set_error("vocab must be from 1 to 2^30"); return VSPEC_B200_ERR_ARG; }
    if (a->row_stride && a->row_stride < a->vocab) { set_error("row_stride is smaller than vocab"); return VSPEC_B200_ERR_ARG; }
    if (a->num_tokens > (size_t)1 << 20) { set_error("too many tokens a row"); return VSPEC_B200_ERR_ARG; }
    if (a->num_tokens && (!a->d_tokens || !a->d_token_logprobs)) { set_error("num_tokens needs d_tokens and d_token_logprobs"); return VSPEC_B200_ERR_ARG; }
    if (a->top_k > (size_t)kLpMaxTop) { set_error("top_k %zu is above %d", a->top_k, kLpMaxTop); return VSPEC_B200_ERR_UNSUPPORTED; }
    if (a->top_k && (!a->d_top_logprobs || !a->d_top_ids)) { set_error("top_k needs d_top_logprobs and d_top_ids"); return VSPEC_B200_ERR_ARG; }
    if (!(a->inv_temperature >= 1e-30f) || isinf(a->inv_temperature)) { set_error("inv_temperature must be finite and at least 1e-30"); return VSPEC_B200_ERR_ARG; }
    if (!a->num_tokens && !a->d_entropy && !a->top_k) { set_error("no output is asked for"); return VSPEC_B200_ERR_ARG; }
    if (a->rows > 65535) { set_error("at most 65535 rows a call"); return VSPEC_B200_ERR_UNSUPPORTED; }
    const size_t elem = a->dtype == VSPEC_B200_T_F32 ? 4 : 2;
    if ((uintptr_t)a->d_logits % elem != 0) { set_error("logits are not aligned to their type"); return VSPEC_B200_ERR_ARG; }
    if (a->rows == 0) return VSPEC_B200_OK;
    LpParams p;
    memset(&p, 0, sizeof(p));
    p.logits = a->d_logits;
    p.allowed = a->d_allowed;
    p.tokens = a->d_tokens;
    p.token_lp = a->d_token_logprobs;
    p.entropy = a->d_entropy;
    p.top_lp = a->d_top_logprobs;
    p.top_ids = a->d_top_ids;
    p.row_stride = a->row_stride ? a->row_stride : a->vocab;
    p.vocab = (int)a->vocab;
    p.words = (int)((a->vocab + 31) / 32);
    p.num_tokens = (int)a->num_tokens;
    p.top_k = (int)a->top_k;
    p.inv_t = a->inv_temperature;
    p.splits = lp_splits(a->rows, a->vocab);
    p.chunk = (int)(((a->vocab + p.splits - 1) / p.splits + 63) / 64 * 64);
    p.splits = (int)((a->vocab + p.chunk - 1) / p.chunk);
    cudaStream_t st = (cudaStream_t)stream;
    const size_t need = lp_workspace(a->rows, a->vocab, a->top_k);
    if (p.splits > 1) {
        void* ws = a->d_workspace;
        if (ws) {
            if (a->workspace_bytes < need) { set_error("workspace too small (%zu < %zu)", a->workspace_bytes, need); return VSPEC_B200_ERR_ARG; }
            if ((uintptr_t)ws % 16 != 0) { set_error("workspace must be 16-byte aligned"); return VSPEC_B200_ERR_ARG; }
        } else {
            ws = lp_scratch(need, st);
            if (!ws) { set_error("cannot allocate %zu bytes of scratch", need); return VSPEC_B200_ERR_NOMEM; }
        }
        p.counters = (unsigned*)ws;
        p.part_keys = (unsigned long long*)((char*)ws + kLpCounterBytes);
        p.part_stats = (float*)(p.part_keys + a->rows * p.splits * a->top_k);
    }
    const cudaError_t e = a->dtype == VSPEC_B200_T_F32   ? lp_launch<float>(p, a->rows, st)
                          : a->dtype == VSPEC_B200_T_F16 ? lp_launch<__half>(p, a->rows, st)
                                                         : lp_launch<__nv_bfloat16>(p, a->rows, st);
    return e == cudaSuccess ? VSPEC_B200_OK : cuda_status(e, "logprobs_kernel launch");
}
