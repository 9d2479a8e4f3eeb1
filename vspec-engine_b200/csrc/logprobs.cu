// logprobs.cu -- log probabilities of given tokens, entropy and the best
// alternatives, in one pass over the logits.
//
// With m the row's maximum, S = sum exp((x - m)/T) and U = sum exp((x - m)/T) (x - m):
//   log p(v) = (x_v - m)/T - ln S,   entropy = ln S - U / (T S).
// A thread keeps (m, S, U) of what it has read and rescales when its maximum
// grows; lanes, warps and the CTAs of a row join with the same rule.  The best
// are 64-bit keys (ordered bits of the logit, then the complement of the id, so
// that ties go to the lowest id); only values that pass a threshold are looked
// at again, which after a row's first block almost none do.
// Bound by memory: a logit is read once.  Few rows: several CTAs share a row
// and the last one to finish joins their parts in CTA order (no result depends
// on the order of arrival).  Measured, fp32 logits of 151936 tokens: 512 rows,
// top 20, 62 us, 5.0 TB/s (76 % of a copy's rate; 512 rows are 3.5 a SM, so some
// have 4 and some 3); 8 rows, top 5, 14.6 us, most of it the chain of the first
// block's selection, the parts' way to the last CTA and its join (24 us for the top
// 20).  bf16 logits meet the same instructions a value: 512 rows 73 us; a mask
// takes the path that guards every value: 105 us bf16, 128 us fp32.
#include "elem_types.cuh"
#include "thread_scratch.cuh"

#include <math.h>
#include <string.h>

namespace vb200 {

constexpr int kLpThreads = 256;
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

// Sorts 32 keys over a warp's lanes, the largest in lane 0.
__device__ __forceinline__ unsigned long long lp_warp_sort(unsigned long long k, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size >> 1; o > 0; o >>= 1) {
            const unsigned long long q = __shfl_xor_sync(0xffffffffu, k, o);
            const bool larger = ((lane & o) == 0) == ((lane & size) == 0);   // this lane keeps the larger one
            k = (q > k) == larger ? q : k;
        }
    return k;
}

struct LpShared {
    unsigned long long lists[kLpWarps][32];   // the warps' sorted keys of a selection
    unsigned long long top[kLpMaxTop];        // the best so far, in order
    LpStats stats[kLpWarps];
    unsigned jth[kLpWarps];                   // ordered bits of each warp's j-th best so far, 0 = fewer
    int last;
};

// The larger half of two ordered lists of 32, in order again: the pairs (i, 31 - i) leave a bitonic sequence.
__device__ __forceinline__ unsigned long long lp_warp_merge(unsigned long long a, unsigned long long b_reversed, int lane) {
    unsigned long long k = a > b_reversed ? a : b_reversed;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long q = __shfl_xor_sync(0xffffffffu, k, o);
        k = (q > k) == ((lane & o) == 0) ? q : k;
    }
    return k;
}

// Lane i's key of the 32 largest of an ordered list and the keys of the lanes in `has`.
constexpr int kLpOneByOne = 6;   // an insertion is about 15 instructions, a sort with its merge about 160
__device__ __forceinline__ unsigned long long lp_insert(unsigned long long best, unsigned long long key, unsigned has, int lane) {
    if (__popc(has) > kLpOneByOne) {
        key = lp_warp_sort((has >> lane) & 1u ? key : 0ull, lane);
        return lp_warp_merge(best, __shfl_sync(0xffffffffu, key, 31 - lane), lane);
    }
    for (; has; has &= has - 1) {
        const unsigned long long k = __shfl_sync(0xffffffffu, key, __ffs(has) - 1);
        const unsigned long long up = __shfl_up_sync(0xffffffffu, best, 1);
        best = best > k ? best : (lane == 0 || up > k ? k : up);
    }
    return best;
}

// out[0..32) = the 32 largest of the warps' ordered lists (a key a lane), in
// order; the lists join in pairs.  Called by all threads; 1 + log2(warps)
// barriers.
__device__ __noinline__ void lp_join_lists(LpShared& sm, unsigned long long key, unsigned long long* out) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    sm.lists[warp][lane] = key;
#pragma unroll 1
    for (int n = kLpWarps / 2; n > 0; n >>= 1) {
        __syncthreads();
        if (warp < n) {
            key = lp_warp_merge(key, sm.lists[warp + n][31 - lane], lane);
            sm.lists[warp][lane] = key;
        }
    }
    if (warp == 0) out[lane] = key;
    __syncthreads();
}

// sm.top = the best of itself and n keys.
template <typename Load>
__device__ __forceinline__ void lp_take_keys(LpShared& sm, int n, Load load) {
    constexpr int kFresh = kLpThreads - kLpMaxTop;
    for (int at = 0; at < n; at += kFresh) {
        const int i = at + (int)threadIdx.x - kLpMaxTop;
        const unsigned long long key = threadIdx.x < kLpMaxTop ? sm.top[threadIdx.x] : (i < n ? load(i) : 0ull);
        lp_join_lists(sm, lp_warp_sort(key, threadIdx.x & 31), sm.top);
    }
}

// Statistics of the CTA in every thread of warp 0 (one order of joining, whatever ran first).
__device__ __forceinline__ LpStats lp_join_cta(LpShared& sm, LpStats st, float c) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto join_lanes = [&](int from) {
        for (int o = from; o > 0; o >>= 1) {
            LpStats q;
            q.m = __shfl_xor_sync(0xffffffffu, st.m, o);
            q.s = __shfl_xor_sync(0xffffffffu, st.s, o);
            q.u = __shfl_xor_sync(0xffffffffu, st.u, o);
            st = (lane & o) ? lp_join(q, st, c) : lp_join(st, q, c);
        }
    };
    join_lanes(16);
    __syncthreads();
    if (lane == 0) sm.stats[warp] = st;
    __syncthreads();
    if (warp == 0) {
        st = sm.stats[lane % kLpWarps];
        join_lanes(kLpWarps / 2);
    }
    return st;
}

// A CTA walks over its part of a row in blocks of kLpThreads * U vectors, with
// the next block's loads in flight.  No warp waits for another on the way: each
// keeps the 32 best of its own values, ordered over its lanes, and looks again
// only at those that reach its threshold: the top_k-th of them (before there are
// that many, the top_k-th of its lanes' maxima) or, if higher, the lowest of the
// warps' j-th best with j * warps >= top_k.  What a warp sees of the others
// changes its work, not what is among the best.
template <typename T, int V, bool ALLOWED, bool TOP>
__global__ void __launch_bounds__(kLpThreads, 4) logprobs_kernel(const LpParams p) {
    pdl_wait();
    pdl_trigger();
    constexpr int U = 16 / V;   // vectors a thread and block (16 values: more spill)
    const size_t row = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 31;
    const T* x = (const T*)p.logits + row * p.row_stride;
    const uint32_t* bits = ALLOWED ? p.allowed + row * p.words : nullptr;
    __shared__ LpShared sm;
    if (TOP) {
        if (tid < kLpWarps) sm.jth[tid] = 0;
        __syncthreads();
    }

    const float c = fminf(p.inv_t * 1.4426950408889634f, -kLpLowest);   // finite, so that 0 * c is 0
    LpStats st = {kLpLowest, 0.f, 0.f};
    unsigned long long best = 0;   // the warp's best, in order over its lanes
    const int j_lane = (p.top_k + kLpWarps - 1) / kLpWarps - 1;
    float thr = kLpLowest;         // no lower value is among the row's best, the same in the warp's lanes

    const int j0 = blockIdx.x * p.chunk, j1 = min(p.vocab, j0 + p.chunk);
    // values before the first 16-byte boundary, whole vectors, values after the last
    const int off = (int)(((uintptr_t)(x + j0) % (V * sizeof(T))) / sizeof(T));
    const int head = off ? min(V - off, j1 - j0) : 0;
    const int vecs = j1 > j0 + head ? (j1 - j0 - head) / V : 0;
    const int body = j0 + head, tail = body + vecs * V;
    using W = Vec<T, V>;

    // value e of a vector, -inf where it is not allowed (a vector past the end is all -inf)
    auto value = [&](const W& w, int e, uint32_t ok) {
        const float v = elem_to_f32<T>(w.e[e]);
        return !ALLOWED || ((ok >> e) & 1u) ? v : -INFINITY;
    };
    auto allowed_bits = [&](int j, int n) -> uint32_t {   // bits of ids j .. j + n - 1
        uint32_t ok = (1u << n) - 1u;
        if (ALLOWED) {
            uint32_t b = bits[j >> 5] >> (j & 31);
            if ((j & 31) + n > 32) b |= bits[(j >> 5) + 1] << (32 - (j & 31));
            ok &= b;
        }
        return ok;
    };
    auto add = [&](float v) {
        const float d = max_nan(v - st.m, kLpLowest);   // -inf - m stays finite, so that 0 * d is 0
        const float e = ex2_approx(d * c);
        st.s += e;
        st.u = fmaf(e, d, st.u);
    };
    auto grow = [&](float top) {
        if (top > st.m) {
            const float d = st.m - top, f = ex2_approx(d * c);
            st.u = lp_rescale_u(st, d, f);
            st.s *= f;
            st.m = top;
        }
    };
    auto keep = [&](float v, int id, bool want) {   // called by whole warps
        const unsigned has = __ballot_sync(0xffffffffu, want && v >= thr);   // false for -inf and NaN
        best = lp_insert(best, lp_key(v, id), has, lane);
        const unsigned long long k = __shfl_sync(0xffffffffu, best, p.top_k - 1);
        if (k) thr = fmaxf(thr, lp_key_value(k));
    };

    W cur[U], nxt[U];
    auto fetch = [&](int g0, W (&w)[U]) {
        if (g0 + kLpThreads * U <= vecs) {   // no branch between the loads: all of them in flight
#pragma unroll
            for (int i = 0; i < U; ++i) w[i] = *reinterpret_cast<const W*>(x + body + (size_t)(g0 + i * kLpThreads + tid) * V);
            return;
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int g = g0 + i * kLpThreads + tid;
            if (g < vecs) {
                w[i] = *reinterpret_cast<const W*>(x + body + (size_t)g * V);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) w[i].e[e] = elem_from_f32<T>(-INFINITY);
            }
        }
    };
    fetch(0, cur);
    // the ends, a value a thread: threads 0-15 the head, 16-31 the tail
    {
        const int j = tid < 16 ? j0 + tid : tail + tid - 16;
        const bool in = tid < 16 ? tid < head : tid < 32 && j < j1;
        float v = -INFINITY;
        if (in && (allowed_bits(j, 1) & 1u)) v = elem_to_f32<T>(x[j]);
        grow(v);
        add(v);
        if (TOP && tid < 32) keep(v, j, in);
    }
    for (int g0 = 0; g0 < vecs; g0 += kLpThreads * U) {
        fetch(g0 + kLpThreads * U, nxt);
        uint32_t ok[U];
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int g = g0 + i * kLpThreads + tid;
            ok[i] = ALLOWED && g < vecs ? allowed_bits(body + g * V, V) : 0u;
#pragma unroll
            for (int e = 0; e < V; ++e) top = fmaxf(top, value(cur[i], e, ok[i]));
        }
        grow(top);
        // in pairs and without add's guard for -inf, which shows as 0 * inf in the sum; then once more with it (masks
        // are full of -inf: at once)
        bool guard = ALLOWED;
        if (!ALLOWED) {
            const pair32 m2 = pack2(-st.m, -st.m), c2 = pack2(c, c);
            pair32 s2 = 0, u2 = 0;
#pragma unroll
            for (int i = 0; i < U; ++i)
#pragma unroll
                for (int e = 0; e < V; e += 2) {
                    const pair32 d = add2(pack2(value(cur[i], e, 0), value(cur[i], e + 1, 0)), m2), t = mul2(d, c2);
                    const pair32 w = pack2(ex2_approx(low2(t)), ex2_approx(high2(t)));
                    s2 = add2(s2, w);
                    u2 = fma2(w, d, u2);
                }
            const float u = low2(u2) + high2(u2);
            guard = u != u;
            if (!guard) {
                st.s += low2(s2) + high2(s2);
                st.u += u;
            }
        }
        if (guard) {
#pragma unroll
            for (int i = 0; i < U; ++i)
#pragma unroll
                for (int e = 0; e < V; ++e) add(value(cur[i], e, ok[i]));
        }
        if (TOP) {
            const unsigned seen = __reduce_min_sync(0xffffffffu, *(volatile unsigned*)&sm.jth[lane % kLpWarps]);
            if (seen) thr = fmaxf(thr, lp_key_value((unsigned long long)seen << 32));
            const int n = __popc(__ballot_sync(0xffffffffu, top >= thr));
            if (n) {
                if (n > p.top_k && n > kLpOneByOne) {
                    float t = top;
#pragma unroll
                    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
                        for (int o = size >> 1; o > 0; o >>= 1) {
                            const float q = __shfl_xor_sync(0xffffffffu, t, o);
                            t = ((lane & o) == 0) == ((lane & size) == 0) ? fmaxf(t, q) : fminf(t, q);
                        }
                    thr = fmaxf(thr, __shfl_sync(0xffffffffu, t, p.top_k - 1));
                }
                uint32_t mine = 0;
#pragma unroll
                for (int i = 0; i < U; ++i)
#pragma unroll
                    for (int e = 0; e < V; ++e) mine |= (value(cur[i], e, ok[i]) >= thr ? 1u : 0u) << (i * V + e);
                while (__any_sync(0xffffffffu, mine != 0)) {
                    const int at = __ffs(mine) - 1;   // -1: this lane has none left
                    float v = 0.f;
#pragma unroll
                    for (int i = 0; i < U; ++i)
#pragma unroll
                        for (int e = 0; e < V; ++e) v = at == i * V + e ? elem_to_f32<T>(cur[i].e[e]) : v;
                    keep(v, body + (g0 + (at / V) * kLpThreads + tid) * V + at % V, mine != 0);
                    mine &= mine - 1;
                }
                if (lane == j_lane) *(volatile unsigned*)&sm.jth[tid >> 5] = (unsigned)(best >> 32);
            }
        }
#pragma unroll
        for (int i = 0; i < U; ++i) cur[i] = nxt[i];
    }

    st = lp_join_cta(sm, st, c);
    if (TOP) lp_join_lists(sm, best, sm.top);

    if (p.splits > 1) {
        const size_t at = row * p.splits + blockIdx.x;
        if (TOP && tid < p.top_k) p.part_keys[at * p.top_k + tid] = sm.top[tid];
        if (tid == 0) {
            p.part_stats[at * 4 + 0] = st.m;
            p.part_stats[at * 4 + 1] = st.s;
            p.part_stats[at * 4 + 2] = st.u;
        }
        __threadfence();
        __syncthreads();
        if (tid == 0) {
            sm.last = atomicAdd(&p.counters[row], 1u) == (unsigned)p.splits - 1;
            if (sm.last) p.counters[row] = 0;
        }
        __syncthreads();
        if (!sm.last) return;
        __threadfence();
        st = {kLpLowest, 0.f, 0.f};
        const float* ps = p.part_stats + row * p.splits * 4;
        for (int i = tid; i < p.splits; i += kLpThreads)
            st = lp_join(st, LpStats{__ldcg(ps + i * 4), __ldcg(ps + i * 4 + 1), __ldcg(ps + i * 4 + 2)}, c);
        st = lp_join_cta(sm, st, c);
        if (TOP) {
            const unsigned long long* pk = p.part_keys + row * p.splits * (size_t)p.top_k;
            if (tid < kLpMaxTop) sm.top[tid] = 0;
            __syncthreads();
            lp_take_keys(sm, p.splits * p.top_k, [&](int i) { return __ldcg(pk + i); });
        }
    }
    if (tid >= 32) return;

    // ---- results ----
    const bool none = st.s == 0.f;
    const float ln_s = logf(st.s);
    if (lane == 0 && p.entropy) p.entropy[row] = none ? 0.f : ln_s - st.u * p.inv_t / st.s;
    if (TOP && lane < p.top_k) {
        const size_t at = row * p.top_k + lane;
        const unsigned long long best = sm.top[lane];
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

// CTAs a row: what fills the four resident on every SM, each with at least 2048
// values. A part's fixed cost (its selection and the join) is why rows that fill
// the SMs are not split for a better balance. 151936 fp32 values, top 20, us with
// 1 / 2 / 4 / 8 CTAs a row: 512 rows (rule: 1) 63 / 78 / 93 / 124, 160 rows (rule:
// 3, 38.7) 38 / 45 / 40 / 48, 64 rows (rule: 9, 26.4) 29 / 25 / 25 / 27: the rule is
// within 2 and 6 % of the best there.
static int lp_splits(size_t rows, size_t vocab) {
    if (rows >= (size_t)kLpMaxSplitRows) return 1;
    size_t s = 4 * (size_t)device_sm_count() / rows;
    const size_t most = vocab / 2048;
    if (s > most) s = most;
    return s < 1 ? 1 : (int)s;
}

static size_t lp_workspace(size_t rows, size_t vocab, size_t top_k) {
    const size_t s = (size_t)lp_splits(rows, vocab);
    return s > 1 ? kLpCounterBytes + rows * s * (4 * sizeof(float) + top_k * sizeof(unsigned long long)) : 0;
}

// The counters in front of it are zero between calls.
static thread_local ThreadScratch g_lp_scratch;

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
    if (off_type(elem_bytes(a->dtype), {a->d_logits})) { set_error("logits are not aligned to their type"); return VSPEC_B200_ERR_ARG; }
    if (off_type(4, {a->d_allowed, a->d_tokens, a->d_token_logprobs, a->d_entropy, a->d_top_logprobs, a->d_top_ids})) {
        set_error("tokens, allowed bits and results must be aligned to 4 bytes");
        return VSPEC_B200_ERR_ARG;
    }
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
            // whatever used it before
            VB_CHECK_CUDA(cudaMemsetAsync(ws, 0, a->rows * sizeof(unsigned), st));
        } else {
            const int rc = g_lp_scratch.get(need, kLpCounterBytes, st, &ws);
            if (rc != VSPEC_B200_OK) return rc;
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
