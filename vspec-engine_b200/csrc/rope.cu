// rope.cu -- rotary positions of q and k rows (any token stride, in place or
// not), pairs interleaved or in halves, part of the head, and the host side of
// the frequencies (plain, linear, NTK, YaRN: "YaRN: Efficient Context Window
// Extension of Large Language Models", Peng et al. 2023, section 3).
//
// (a, b) -> (a cos - b sin, a sin + b cos) * attn_factor, angle = pos * f.
// f is kept in turns as a 64-bit fraction, so pos * turns mod 2^64 is the exact
// place in the turn (an integer product that drops whole turns); its top 32
// bits, as a signed fraction of a half turn, go to sincospif, which then needs
// no range reduction and holds 24 bits at any position.
//
// Memory-bound: every value is read and written once.  A CTA works on up to
// four tokens: its threads share out the tokens' angles (one sincospif a pair
// and token, kept in shared memory) while the first rows are on their way, then
// every thread walks over the heads of each token with a fixed place in the
// head.  Without the sharing, 16 threads with the same place computed the same
// sines and those took longer than the rows (75 us).  Measured in a graph: 8192
// tokens of 32 + 8 heads of 128 in bf16, half of the dims rotated, 35.9 us, 4.7
// TB/s read and written (26 us at the rate of a copy).  What is left is latency: 42
// % of the warps are active and wait for their rows, and the angles, a third of a
// warp's time, lie between its loads and stores.  8 tokens 1.9 us.
#include "elem_types.cuh"

#include <math.h>
#include <string.h>

namespace vb200 {

constexpr int kRopeThreads = 256;
constexpr int kRopePairs = 256;   // angles of a token group

struct RopeParams {
    const void *q, *k;
    void *q_out, *k_out;
    const int32_t* pos;
    const uint64_t* turns;
    size_t q_stride, k_stride, q_out_stride, k_out_stride;
    int hq, heads, d, rot;     // heads = hq + hk
    int units, rot_units;      // units of 2V elements a head (the rotated ones first)
    int group;                 // tokens a CTA
    size_t tokens;
    float mult, sign;          // attn_factor; -1 for the inverse rotation
};

// Grid (token groups, head slices).  A unit is 2V elements: V pairs (for
// halves, V elements at i and V at i + rot/2; interleaved, 2V in a row), or 2V
// elements of the copied tail.
template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(kRopeThreads, 4) rope_kernel(const RopeParams p) {
    pdl_wait();
    pdl_trigger();
    __shared__ __align__(16) float sm_cos[kRopePairs], sm_sin[kRopePairs];   // [token of the group][pair]
    const int pairs = p.rot / 2, per = kRopeThreads / p.units;
    const size_t t0 = (size_t)blockIdx.x * p.group;
    const int tokens = (int)min((size_t)p.group, p.tokens - t0);
    const int u = threadIdx.x % p.units;
    const int step = per * gridDim.y, w0 = (int)threadIdx.x / p.units + per * blockIdx.y;
    const bool turn = u < p.rot_units;
    const int i0 = INTER || !turn ? 2 * V * u : V * u;                    // first element of the unit
    const int i1 = INTER || !turn ? i0 + V : i0 + pairs;                  // its second vector
    const int rows = (int)threadIdx.x < per * p.units ? tokens * p.heads : 0;   // (token, head) rows to walk over
    using W = Vec<T, V>;
    constexpr int H = 2;   // rows with loads in flight
    W a[H], b[H];
    T* dst[H];
    int at[H];             // first angle of the row's token
    auto fetch = [&](int w) {
#pragma unroll
        for (int i = 0; i < H; ++i) {
            dst[i] = nullptr;
            if (w + i * step >= rows) continue;
            const int t = (w + i * step) / p.heads, h = w + i * step - t * p.heads;
            const bool is_q = h < p.hq;
            const T* src = is_q ? (const T*)p.q + (t0 + t) * p.q_stride + (size_t)h * p.d
                                : (const T*)p.k + (t0 + t) * p.k_stride + (size_t)(h - p.hq) * p.d;
            T* to = is_q ? (T*)p.q_out + (t0 + t) * p.q_out_stride + (size_t)h * p.d
                         : (T*)p.k_out + (t0 + t) * p.k_out_stride + (size_t)(h - p.hq) * p.d;
            if (!turn && src == to) continue;
            dst[i] = to;
            at[i] = t * pairs;
            a[i] = *reinterpret_cast<const W*>(src + i0);
            b[i] = *reinterpret_cast<const W*>(src + i1);
        }
    };
    fetch(w0);
    for (int i = threadIdx.x; i < tokens * pairs; i += kRopeThreads) {
        const int t = i / pairs;
        const uint64_t pos = (uint64_t)(int64_t)p.pos[t0 + t];
        const int32_t part = (int32_t)((pos * p.turns[i - t * pairs]) >> 32);
        float s, c;
        sincospif((float)part * (1.0f / 2147483648.0f), &s, &c);
        sm_cos[i] = c * p.mult;
        sm_sin[i] = s * p.sign * p.mult;
    }
    __syncthreads();
    for (int w = w0; w < rows; w += H * step) {
        if (w > w0) fetch(w);
#pragma unroll
        for (int i = 0; i < H; ++i) {
            if (!dst[i]) continue;
            if (turn) {
                constexpr int F = V < 4 ? V : 4;
                float cs[V], sn[V];
#pragma unroll
                for (int j = 0; j < V; j += F) {
                    const Vec<float, F> vc = *reinterpret_cast<const Vec<float, F>*>(sm_cos + at[i] + V * u + j);
                    const Vec<float, F> vs = *reinterpret_cast<const Vec<float, F>*>(sm_sin + at[i] + V * u + j);
#pragma unroll
                    for (int e = 0; e < F; ++e) { cs[j + e] = vc.e[e]; sn[j + e] = vs.e[e]; }
                }
                T v[2 * V];
#pragma unroll
                for (int j = 0; j < V; ++j) { v[j] = a[i].e[j]; v[V + j] = b[i].e[j]; }
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    T& lo = INTER ? v[2 * j] : v[j];
                    T& hi = INTER ? v[2 * j + 1] : v[V + j];
                    const float x = elem_to_f32<T>(lo), y = elem_to_f32<T>(hi);
                    lo = elem_from_f32<T>(x * cs[j] - y * sn[j]);
                    hi = elem_from_f32<T>(x * sn[j] + y * cs[j]);
                }
#pragma unroll
                for (int j = 0; j < V; ++j) { a[i].e[j] = v[j]; b[i].e[j] = v[V + j]; }
            }
            *reinterpret_cast<W*>(dst[i] + i0) = a[i];
            *reinterpret_cast<W*>(dst[i] + i1) = b[i];
        }
    }
}

template <typename T>
static cudaError_t rope_launch(RopeParams p, size_t tokens, bool inter, uintptr_t addresses, size_t counts,
                               cudaStream_t st) {
    // a unit is two vectors of a head's rotated part or of its tail
    const size_t pairs = (size_t)p.rot / 2;
    int v = elem_vec<T>(addresses, counts | pairs);
    if ((inter || p.d > p.rot) && (p.rot % (2 * v) != 0 || (p.d - p.rot) % (2 * v) != 0))
        v = p.rot % 4 == 0 && (p.d - p.rot) % 4 == 0 && v >= 2 ? 2 : 1;
    p.units = p.d / (2 * v);
    p.rot_units = p.rot / (2 * v);
    // four tokens a CTA, as far as their angles fit and every SM still gets eight CTAs; with fewer
    // tokens than that, slices of the heads
    const size_t want = 8 * (size_t)device_sm_count();
    p.tokens = tokens;
    p.group = 1;
    while (p.group < 4 && 2 * p.group * (p.rot / 2) <= kRopePairs && tokens / (2 * p.group) >= want) p.group *= 2;
    const int per = kRopeThreads / p.units;
    const int most = (p.heads + per - 1) / per;
    size_t slices = tokens >= want ? 1 : (want + tokens - 1) / tokens;
    if (slices > (size_t)most) slices = most;
    const dim3 grid((unsigned)((tokens + p.group - 1) / p.group), (unsigned)slices);
    constexpr int threads = kRopeThreads;
    constexpr int F = 16 / (int)sizeof(T);
    if (inter)
        return v == F ? launch_pdl(rope_kernel<T, F, true>, grid, dim3(threads), 0, st, p)
             : v == 2 ? launch_pdl(rope_kernel<T, 2, true>, grid, dim3(threads), 0, st, p)
                      : launch_pdl(rope_kernel<T, 1, true>, grid, dim3(threads), 0, st, p);
    return v == F ? launch_pdl(rope_kernel<T, F, false>, grid, dim3(threads), 0, st, p)
         : v == 2 ? launch_pdl(rope_kernel<T, 2, false>, grid, dim3(threads), 0, st, p)
                  : launch_pdl(rope_kernel<T, 1, false>, grid, dim3(threads), 0, st, p);
}

}  // namespace vb200

using namespace vb200;

extern "C" int vspec_b200_rope(const VspecB200RopeArgs* a, void* stream) {
    if (!a) { set_error("args is NULL"); return VSPEC_B200_ERR_ARG; }
    if (!elem_type_known(a->dtype)) { set_error("bad dtype %d", a->dtype); return VSPEC_B200_ERR_ARG; }
    if (a->flags & ~(VSPEC_B200_ROPE_INTERLEAVED | VSPEC_B200_ROPE_INVERSE)) { set_error("unknown rope flags 0x%x", a->flags); return VSPEC_B200_ERR_ARG; }
    if (!a->d_q || !a->d_q_out || !a->d_pos || !a->d_turns) { set_error("NULL pointer argument"); return VSPEC_B200_ERR_ARG; }
    if ((a->d_k == nullptr) != (a->d_k_out == nullptr)) { set_error("d_k and d_k_out go together"); return VSPEC_B200_ERR_ARG; }
    if (off_type(elem_bytes(a->dtype), {a->d_q, a->d_k, a->d_q_out, a->d_k_out}) || off_type(4, {a->d_pos}) || off_type(8, {a->d_turns})) {
        set_error("q, k, outputs, d_pos and d_turns must be aligned to their types");
        return VSPEC_B200_ERR_ARG;
    }
    const size_t hk = a->d_k ? a->num_k_heads : 0;
    if (a->num_q_heads == 0 || a->head_dim == 0 || (a->d_k && hk == 0)) { set_error("zero dimension"); return VSPEC_B200_ERR_ARG; }
    if (a->rot_dim == 0 || a->rot_dim % 2 != 0 || a->rot_dim > a->head_dim || a->head_dim > 512 || a->head_dim % 2 != 0) {
        set_error("rot_dim must be even, from 2 to head_dim, head_dim even and at most 512");
        return VSPEC_B200_ERR_ARG;
    }
    if (a->num_q_heads > 65535 || hk > 65535) { set_error("too many heads"); return VSPEC_B200_ERR_ARG; }
    if (a->tokens > 0x7fffffffu) { set_error("too many tokens"); return VSPEC_B200_ERR_ARG; }
    const size_t qd = a->num_q_heads * a->head_dim, kd = hk * a->head_dim;
    RopeParams p;
    memset(&p, 0, sizeof(p));
    p.q = a->d_q; p.k = a->d_k; p.q_out = a->d_q_out; p.k_out = a->d_k_out;
    p.pos = a->d_pos;
    p.turns = a->d_turns;
    p.q_stride = a->q_stride ? a->q_stride : qd;
    p.k_stride = a->k_stride ? a->k_stride : kd;
    p.q_out_stride = a->q_out_stride ? a->q_out_stride : qd;
    p.k_out_stride = a->k_out_stride ? a->k_out_stride : kd;
    if (p.q_stride < qd || p.q_out_stride < qd || p.k_stride < kd || p.k_out_stride < kd) {
        set_error("a token stride is smaller than its heads");
        return VSPEC_B200_ERR_ARG;
    }
    if ((a->d_q == a->d_q_out && p.q_stride != p.q_out_stride) ||
        (a->d_k && a->d_k == a->d_k_out && p.k_stride != p.k_out_stride)) {
        set_error("in place needs one stride for input and output");
        return VSPEC_B200_ERR_ARG;
    }
    if (a->tokens == 0) return VSPEC_B200_OK;
    p.hq = (int)a->num_q_heads;
    p.heads = (int)(a->num_q_heads + hk);
    p.d = (int)a->head_dim;
    p.rot = (int)a->rot_dim;
    p.mult = a->attn_factor;
    p.sign = (a->flags & VSPEC_B200_ROPE_INVERSE) ? -1.0f : 1.0f;
    const bool inter = (a->flags & VSPEC_B200_ROPE_INTERLEAVED) != 0;
    const uintptr_t addr = (uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.q_out | (uintptr_t)p.k_out;
    size_t counts = p.q_stride | p.q_out_stride | a->head_dim;
    if (a->d_k) counts |= p.k_stride | p.k_out_stride;
    cudaStream_t st = (cudaStream_t)stream;
    const cudaError_t e = a->dtype == VSPEC_B200_T_F32   ? rope_launch<float>(p, a->tokens, inter, addr, counts, st)
                          : a->dtype == VSPEC_B200_T_F16 ? rope_launch<__half>(p, a->tokens, inter, addr, counts, st)
                                                         : rope_launch<__nv_bfloat16>(p, a->tokens, inter, addr, counts, st);
    return e == cudaSuccess ? VSPEC_B200_OK : cuda_status(e, "rope_kernel launch");
}

extern "C" int vspec_b200_rope_turns(size_t rot_dim, double theta, int scaling, double factor, double original_ctx,
                                     double beta_fast, double beta_slow, uint64_t* turns, float* attn_factor) {
    if (!turns || !attn_factor) { set_error("NULL pointer argument"); return VSPEC_B200_ERR_ARG; }
    if (rot_dim < 2 || rot_dim % 2 != 0 || rot_dim > 512) { set_error("rot_dim must be even, from 2 to 512"); return VSPEC_B200_ERR_ARG; }
    if (!(theta > 1.0) || !isfinite(theta)) { set_error("theta must be finite and above 1"); return VSPEC_B200_ERR_ARG; }
    if (scaling < VSPEC_B200_ROPE_PLAIN || scaling > VSPEC_B200_ROPE_YARN) { set_error("unknown scaling %d", scaling); return VSPEC_B200_ERR_ARG; }
    if (scaling != VSPEC_B200_ROPE_PLAIN && (!(factor >= 1.0) || !isfinite(factor))) { set_error("factor must be finite and at least 1"); return VSPEC_B200_ERR_ARG; }
    const double two_pi = 6.283185307179586476925286766559;
    const double n = (double)rot_dim;
    double lo = 0.0, hi = 0.0;
    if (scaling == VSPEC_B200_ROPE_YARN) {
        if (!(original_ctx > 0.0) || !(beta_slow > 0.0) || !(beta_fast >= beta_slow)) {
            set_error("YaRN needs original_ctx > 0 and beta_fast >= beta_slow > 0");
            return VSPEC_B200_ERR_ARG;
        }
        // the pair that makes beta turns in original_ctx positions
        lo = floor(n * log(original_ctx / (beta_fast * two_pi)) / (2.0 * log(theta)));
        hi = ceil(n * log(original_ctx / (beta_slow * two_pi)) / (2.0 * log(theta)));
        if (lo < 0.0) lo = 0.0;
        if (hi > n - 1.0) hi = n - 1.0;
    }
    if (scaling == VSPEC_B200_ROPE_NTK) theta *= pow(factor, n / (n > 3.0 ? n - 2.0 : 1.0));
    for (size_t i = 0; i < rot_dim / 2; ++i) {
        double f = pow(theta, -2.0 * (double)i / n);
        if (scaling == VSPEC_B200_ROPE_LINEAR) f /= factor;
        if (scaling == VSPEC_B200_ROPE_YARN) {
            double ramp = ((double)i - lo) / (hi - lo > 0.001 ? hi - lo : 0.001);
            ramp = ramp < 0.0 ? 0.0 : (ramp > 1.0 ? 1.0 : ramp);
            f = f * (1.0 - ramp) + f / factor * ramp;
        }
        turns[i] = (uint64_t)(f / two_pi * 18446744073709551616.0);
    }
    *attn_factor = scaling == VSPEC_B200_ROPE_YARN ? (float)(0.1 * log(factor) + 1.0) : 1.0f;
    return VSPEC_B200_OK;
}
