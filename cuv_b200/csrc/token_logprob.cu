// Log probabilities of given tokens under softmax(scale * logits), column by column, with the log-sum-exp, the entropy
// and the likeliest tokens; and the gradient with respect to the logits.
//
// Everything is held in 32 bits in powers of two: with c = scale * log2(e), the largest logit M of a column and
// d_v = (logit_v - M) * c (the difference first, so that logits far from zero and masks of the type's lowest value do no harm),
//   s = sum_v 2^d_v        t = sum_v 2^d_v * d_v
//   lse = scale * M + ln 2 * log2 s      entropy = ln 2 * (log2 s - t / s)      logp_v = scale * (logit_v - M) - ln 2 * log2 s
// M, s and t come from one pass: a running maximum, and sums that are rescaled by 2^(c * (old M - new M)) when it grows.
#include "typed.cuh"

namespace cuvdia {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int TOP_MAX = 32;
constexpr float LEAST = -1000.f;        // 2^-1000 is zero: exponents are cut here before they multiply a power, 0 * -inf being NaN

__device__ __forceinline__ float exp2_approx(float x) {         // relative error 2^-22, results below 2^-126 are zero
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Running softmax statistics: the largest logit met so far, and the sums relative to it.
struct Stat { float m, s, t; };

// what to subtract from a logit: the maximum, or zero while every logit met is -inf
__device__ __forceinline__ float shift(float m) { return m == -INFINITY ? 0.f : m; }

// expresses the sums of `a` relative to the larger maximum m
__device__ __forceinline__ void rescale(Stat& a, float m, float c) {
    if (a.m != -INFINITY) {                                     // else nothing is summed yet (or NaN, which stays)
        const float by = (a.m - m) * c, f = exp2_approx(by);
        a.t = f * fmaf(a.s, fmaxf(by, LEAST), a.t);
        a.s *= f;
    }
    a.m = m;
}

__device__ __forceinline__ Stat merge(Stat a, Stat b, float c) {
    const float m = fmaxf(a.m, b.m);
    if (a.m != m) rescale(a, m, c);
    if (b.m != m) rescale(b, m, c);
    a.s += b.s; a.t += b.t;
    return a;
}

// The k largest logits a warp has met, one a lane, in order (ties: the lower index first).  Lane k-1 is the bar a new one
// has to pass.  NaN and -inf never enter; a place that stays empty has index -1.
struct Top {
    float v, bar_v;
    int i, bar_i;
    __device__ __forceinline__ void clear() { v = bar_v = -INFINITY; i = bar_i = -1; }
    __device__ __forceinline__ bool passes(float x, int at) const { return x > bar_v || (x == bar_v && at < bar_i); }
    __device__ __forceinline__ void insert(float x, int at, int k) {                  // x, at: the same in all lanes
        const int lane = threadIdx.x & 31;
        const int before = __popc(__ballot_sync(0xffffffffu, v > x || (v == x && i < at)));
        const float pv = __shfl_up_sync(0xffffffffu, v, 1);
        const int pi = __shfl_up_sync(0xffffffffu, i, 1);
        if (lane == before) { v = x; i = at; }
        else if (lane > before) { v = pv; i = pi; }
        bar_v = __shfl_sync(0xffffffffu, v, k - 1);
        bar_i = __shfl_sync(0xffffffffu, i, k - 1);
    }
    // one candidate per lane, for those with `there`
    __device__ __forceinline__ void offer(float x, int at, bool there, int k) {
        unsigned todo = __ballot_sync(0xffffffffu, there && passes(x, at));
        while (todo) {
            const int from = __ffs(todo) - 1;
            todo &= todo - 1;
            const float y = __shfl_sync(0xffffffffu, x, from);
            const int a = __shfl_sync(0xffffffffu, at, from);
            if (passes(y, a)) insert(y, a, k);
        }
    }
};

// One block per column.  A column's elements are walked as 16-byte vectors of the memory they lie in, so a column that
// does not start on a 16-byte boundary costs element-wise loads at its two ends only.
template <class T, class I, bool TOP>
__global__ void __launch_bounds__(256)
token_logprob_kernel(const T* __restrict__ logits, long long ld, int vocab, int ncols, const I* __restrict__ tokens, float scale,
                     float* __restrict__ logp, float* __restrict__ lse, float* __restrict__ entropy, int top,
                     float* __restrict__ top_logp, int* __restrict__ top_index) {
    constexpr int V = Vec16<T>::N, U = 4;
    __shared__ Stat stats[8];
    __shared__ float top_v[8][TOP_MAX];
    __shared__ int top_i[8][TOP_MAX];
    const long long col = blockIdx.x;
    const T* x0 = logits + col * ld;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float c = scale * LOG2E;
    const int head = (int)((reinterpret_cast<uintptr_t>(x0) & 15) / sizeof(T));      // elements before x0 in its first vector
    const int nvec = (int)(((long long)vocab + head + V - 1) / V);
    Stat a = {-INFINITY, 0.f, 0.f};
    Top best;
    best.clear();
    for (int i0 = 0; i0 < nvec; i0 += 256 * U) {
        float x[U][V];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = i0 + u * 256 + threadIdx.x;
            const long long e0 = (long long)i * V - head;
            if (e0 >= 0 && e0 + V <= vocab) {
                unpack16<T>(*reinterpret_cast<const uint4*>(x0 + e0), x[u]);
            } else {
#pragma unroll
                for (int e = 0; e < V; e++) x[u][e] = e0 + e >= 0 && e0 + e < vocab ? to_f32(x0[e0 + e]) : -INFINITY;
            }
        }
        float m = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < V; e++) m = fmaxf(m, x[u][e]);
        if (m > a.m) rescale(a, m, c);
        const float m0 = shift(a.m);
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < V; e++) {
                const float d = (x[u][e] - m0) * c, p = exp2_approx(d);
                a.s += p;
                a.t = fmaf(p, fmaxf(d, LEAST), a.t);
            }
        if (TOP && __any_sync(0xffffffffu, m >= best.bar_v && m > -INFINITY)) {
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int e = 0; e < V; e++)
                    best.offer(x[u][e], (i0 + u * 256 + (int)threadIdx.x) * V - head + e, x[u][e] > -INFINITY, top);
        }
    }
#pragma unroll
    for (int s = 16; s > 0; s /= 2) {
        Stat b;
        b.m = __shfl_xor_sync(0xffffffffu, a.m, s); b.s = __shfl_xor_sync(0xffffffffu, a.s, s); b.t = __shfl_xor_sync(0xffffffffu, a.t, s);
        a = merge(a, b, c);
    }
    if (lane == 0) stats[warp] = a;
    if (TOP) { top_v[warp][lane] = best.v; top_i[warp][lane] = best.i; }
    __syncthreads();
    if (warp != 0) return;
    a = stats[0];
    for (int w = 1; w < 8; w++) a = merge(a, stats[w], c);
    const bool none = a.m == -INFINITY && a.s == 0.f;
    const float m0 = shift(a.m), l2s = log2f(a.s);
    if (lane == 0) {
        if (lse) lse[col] = fmaf(m0, scale, l2s * LN2);
        if (entropy) { const float h = (l2s - a.t / a.s) * LN2; entropy[col] = none || h < 0.f ? 0.f : h; }
        if (logp) {
            const long long t = (long long)tokens[col];
            float r = 0.f;
            if (t >= 0 && t < vocab) r = none ? -INFINITY : fmaf(to_f32(x0[t]) - m0, scale, -l2s * LN2);
            logp[col] = r;
        }
    }
    if (TOP) {
        for (int w = 1; w < 8; w++) best.offer(top_v[w][lane], top_i[w][lane], lane < top && top_i[w][lane] >= 0, top);
        if (lane < top) {
            top_logp[col * top + lane] = best.i < 0 ? -INFINITY : fmaf(best.v - m0, scale, -l2s * LN2);
            top_index[col * top + lane] = best.i;
        }
    }
}

int launch_token_logprob(const void* logits, int ld, int type, int vocab, int ncols, const void* tokens, int token_type,
                         float scale, float* logp, float* lse, float* entropy, int top, float* top_logp, int* top_index,
                         cudaStream_t st) {
#define LP_GO(I, K) token_logprob_kernel<T, I, K><<<ncols, 256, 0, st>>>((const T*)logits, ld, vocab, ncols, (const I*)tokens, \
    scale, logp, lse, entropy, top, top_logp, top_index)
    CUVDIA_FLOAT_TYPE(type, {
        if (token_type == CUVDIA_T_I32) { if (top) LP_GO(int, true); else LP_GO(int, false); }
        else { if (top) LP_GO(long long, true); else LP_GO(long long, false); }
    });
#undef LP_GO
    count_launch();
    return check_launch("token_logprob_kernel");
}

// ---- gradient ------------------------------------------------------------------------------------------------------
//   dlogits_v = scale * (dlogp * ([v = token] - p_v) - dentropy * p_v * (log p_v + entropy)),   p_v = exp(scale * logit_v - lse)
// Element-wise once lse and entropy are known: a block owns up to 1024 vectors of one column.  Vectors are those of the
// logits' memory; the stores are vectors too where dlogits lies alike (VEC), else element by element.  In place is fine:
// a thread reads its elements before it writes them.
template <class T, class I>
__global__ void __launch_bounds__(256)
token_logprob_grad_kernel(T* dlogits, long long ldd, const T* logits, long long ld, int vocab, int ncols,
                          const I* __restrict__ tokens, float scale, const float* __restrict__ lse,
                          const float* __restrict__ dlogp, const float* __restrict__ entropy,
                          const float* __restrict__ dentropy, int chunks) {
    constexpr int V = Vec16<T>::N, U = 4;
    const long long col = blockIdx.x / (unsigned)chunks;
    const int chunk = blockIdx.x - (unsigned)col * (unsigned)chunks;
    const T* x0 = logits + col * ld;
    T* y0 = dlogits + col * ldd;
    const int head = (int)((reinterpret_cast<uintptr_t>(x0) & 15) / sizeof(T));
    const bool alike = ((reinterpret_cast<uintptr_t>(x0) ^ reinterpret_cast<uintptr_t>(y0)) & 15) == 0;
    long long t = tokens ? (long long)tokens[col] : -1;
    if (t < 0 || t >= vocab || dlogp == nullptr) t = -1;
    const float g = t >= 0 ? dlogp[col] : 0.f, h = dentropy ? dentropy[col] : 0.f, l = lse[col];
    const float ent = dentropy ? entropy[col] : 0.f;
    // A padded column without an entropy term is zero without a look at its logits, and so is a column that has no
    // finite logit.
    const bool zero = (t < 0 && dentropy == nullptr) || l == -INFINITY;
    const int i0 = chunk * 256 * U + threadIdx.x;
    float x[U][V];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const long long e0 = ((long long)i0 + u * 256) * V - head;
        if (zero) {
#pragma unroll
            for (int e = 0; e < V; e++) x[u][e] = 0.f;
        } else if (e0 >= 0 && e0 + V <= vocab) {
            unpack16<T>(*reinterpret_cast<const uint4*>(x0 + e0), x[u]);
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) x[u][e] = e0 + e >= 0 && e0 + e < vocab ? to_f32(x0[e0 + e]) : 0.f;
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const long long e0 = ((long long)i0 + u * 256) * V - head;
        if (e0 >= vocab) break;
        if (!zero) {
#pragma unroll
            for (int e = 0; e < V; e++) {
                const float d = fmaf(x[u][e], scale, -l), p = exp2_approx(d * LOG2E);
                const float w = dentropy ? fmaf(h, fmaxf(d, LEAST) + ent, g) : g;
                const float hot = e0 + e == t ? g : 0.f;
                x[u][e] = scale * fmaf(-p, w, hot);
            }
        }
        if (alike && e0 >= 0 && e0 + V <= vocab) {
            *reinterpret_cast<uint4*>(y0 + e0) = pack16<T>(x[u]);
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) if (e0 + e >= 0 && e0 + e < vocab) y0[e0 + e] = from_f32<T>(x[u][e]);
        }
    }
}

int launch_token_logprob_grad(void* dlogits, int ldd, const void* logits, int ld, int type, int vocab, int ncols,
                              const void* tokens, int token_type, float scale, const float* lse, const float* dlogp,
                              const float* entropy, const float* dentropy, cudaStream_t st) {
    const int v = 16 / type_size(type);
    const long long chunks = ((long long)vocab + v - 1 + 1024 * v - 1) / (1024 * v);       // up to v - 1 elements of offset
    const long long blocks = chunks * ncols;
    if (blocks > 2147483647LL) { set_last_error("token_logprob_grad: %lld blocks", blocks); return CUVDIA_ERR_UNSUPPORTED; }
#define LG_GO(I) token_logprob_grad_kernel<T, I><<<(unsigned)blocks, 256, 0, st>>>((T*)dlogits, ldd, (const T*)logits, ld, vocab, \
    ncols, (const I*)tokens, scale, lse, dlogp, entropy, dentropy, (int)chunks)
    CUVDIA_FLOAT_TYPE(type, { if (token_type == CUVDIA_T_I32) LG_GO(int); else LG_GO(long long); });
#undef LG_GO
    count_launch();
    return check_launch("token_logprob_grad_kernel");
}

}  // namespace cuvdia
