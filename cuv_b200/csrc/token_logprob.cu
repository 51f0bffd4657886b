// Log probabilities of given tokens under softmax(scale * logits), column by column, with the log-sum-exp, the entropy
// and the likeliest tokens; and the gradient with respect to the logits.
//
// Everything is held in 32 bits in powers of two: with c = scale * log2(e), the largest logit M of a column and
// d_v = (logit_v - M) * c (the difference first, so that logits far from zero and masks of the type's lowest value do no harm),
//   s = sum_v 2^d_v        t = sum_v 2^d_v * d_v
//   lse = scale * M + ln 2 * log2 s      entropy = ln 2 * (log2 s - t / s)      logp_v = scale * (logit_v - M) - ln 2 * log2 s
// M, s and t come from one pass: a running maximum, and sums that are rescaled by 2^(c * (old M - new M)) when it grows.
#include <type_traits>

#include "typed.cuh"

namespace cuvdia {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
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

// ---- the likeliest tokens ------------------------------------------------------------------------------------------
// A candidate is one 64-bit number that orders like (logit descending, index ascending): the larger, the better; 0 = none.
// NaN and -inf are never candidates.
typedef unsigned long long Key;

__device__ __forceinline__ Key make_key(float x, int at) {
    const unsigned u = __float_as_uint(x + 0.f);                // -0 becomes +0: the two tie
    return ((Key)(u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u)) << 32) | (unsigned)~at;
}
__device__ __forceinline__ float key_value(Key k) {             // -inf for "none"
    const unsigned u = (unsigned)(k >> 32);
    return k == 0 ? -INFINITY : __uint_as_float(u ^ ((u >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ int key_index(Key k) { return k == 0 ? -1 : (int)~(unsigned)k; }

// 32 candidates, one a lane, put in descending order (bitonic network)
__device__ __forceinline__ Key sort_desc(Key k) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int n = 2; n <= 32; n *= 2)
#pragma unroll
        for (int s = n / 2; s > 0; s /= 2) {
            const Key o = __shfl_xor_sync(0xffffffffu, k, s);
            const bool upper = (lane & s) != 0, descending = (lane & n) == 0 || n == 32;
            k = (o > k) == (upper != descending) ? o : k;
        }
    return k;
}

// the best 32 of two descending lists, in descending order
__device__ __forceinline__ Key merge_desc(Key a, Key b) {
    const int lane = threadIdx.x & 31;
    const Key r = __shfl_sync(0xffffffffu, b, 31 - lane);
    a = r > a ? r : a;
#pragma unroll
    for (int s = 16; s > 0; s /= 2) {
        const Key o = __shfl_xor_sync(0xffffffffu, a, s);
        a = (o > a) == ((lane & s) == 0) ? o : a;
    }
    return a;
}

// A warp's best candidates so far: a descending list (one a lane), and up to 63 more in shared memory that wait to be sorted
// in, 32 at a time.  `bar` is the k-th best of the list: what a new one has to beat.  `floor` is a lower bound on the
// column's k-th best logit that the warps of the block raise together.
struct Top {
    Key list, bar;
    float bar_v;
    int waiting;
    __device__ __forceinline__ void clear() { list = bar = 0; bar_v = -INFINITY; waiting = 0; }
    __device__ __forceinline__ void absorb(Key batch, int k) {
        list = merge_desc(list, sort_desc(batch));
        bar = __shfl_sync(0xffffffffu, list, k - 1);
        bar_v = key_value(bar);
    }
    // at most one candidate per lane (0: none)
    __device__ __forceinline__ void push(Key key, Key* buffer, int k) {
        const int lane = threadIdx.x & 31;
        const unsigned there = __ballot_sync(0xffffffffu, key > bar);
        if (key > bar) buffer[waiting + __popc(there & ((1u << lane) - 1))] = key;
        waiting += __popc(there);
        if (waiting >= 32) {
            __syncwarp();
            const Key batch = buffer[lane], rest = buffer[32 + lane];
            __syncwarp();
            buffer[lane] = rest;
            waiting -= 32;
            absorb(batch, k);
        }
        __syncwarp();
    }
    __device__ __forceinline__ void finish(const Key* buffer, int k) {
        const int lane = threadIdx.x & 31;
        if (waiting > 0) absorb(lane < waiting ? buffer[lane] : 0, k);
        waiting = 0;
    }
};

// ---- one pass over a column -------------------------------------------------------------------------------------------
__device__ __forceinline__ float max_raw(const uint4& r, float) {
    return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
}
__device__ __forceinline__ float min_raw(const uint4& r, float) {
    return fminf(fminf(__uint_as_float(r.x), __uint_as_float(r.y)), fminf(__uint_as_float(r.z), __uint_as_float(r.w)));
}
#define CUVDIA_RAW16(H, H2)                                                                                                    \
    __device__ __forceinline__ float max_raw(const uint4& r, H) {                                                              \
        const H2* h = reinterpret_cast<const H2*>(&r);                                                                         \
        const H2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));                                                        \
        return fmaxf(to_f32(m.x), to_f32(m.y));                                                                                \
    }                                                                                                                          \
    __device__ __forceinline__ float min_raw(const uint4& r, H) {                                                              \
        const H2* h = reinterpret_cast<const H2*>(&r);                                                                         \
        const H2 m = __hmin2(__hmin2(h[0], h[1]), __hmin2(h[2], h[3]));                                                        \
        return fminf(to_f32(m.x), to_f32(m.y));                                                                                \
    }
CUVDIA_RAW16(__half, __half2)
CUVDIA_RAW16(__nv_bfloat16, __nv_bfloat162)
#undef CUVDIA_RAW16

template <class T> __device__ __forceinline__ unsigned minus_inf_word();
template <> __device__ __forceinline__ unsigned minus_inf_word<float>() { return 0xff800000u; }
template <> __device__ __forceinline__ unsigned minus_inf_word<__half>() { return 0xfc00fc00u; }
template <> __device__ __forceinline__ unsigned minus_inf_word<__nv_bfloat16>() { return 0xff80ff80u; }

// The sums of a thread as pairs, so that two elements share an instruction.
struct Sums { float m; float2 s, t; };

template <bool ENT>
__device__ __forceinline__ Stat fold(const Sums& a) {
    return {a.m, a.s.x + a.s.y, ENT ? a.t.x + a.t.y : 0.f};
}

// Adds U vectors to a thread's sums.  The exponents of an ordinary chunk are not cut (see LEAST): a chunk is cut only if its
// smallest logit is so far below the maximum that an exponent times its power could be 0 * -inf.
template <class T, bool ENT, int U>
__device__ __forceinline__ void add_chunk(Sums& a, float m, const uint4 (&raw)[U], float c) {
    constexpr int V = Vec16<T>::N;
    if (m > a.m) {
        if (a.m != -INFINITY) {
            const float by = (a.m - m) * c, f = exp2_approx(by), cut = fmaxf(by, LEAST);
            if (ENT) { a.t.x = f * fmaf(a.s.x, cut, a.t.x); a.t.y = f * fmaf(a.s.y, cut, a.t.y); }
            a.s.x *= f; a.s.y *= f;
        }
        a.m = m;
    }
    const float m0 = shift(a.m);
    const float2 minus = make_float2(-m0, -m0), by = make_float2(c, c);
    bool cut = false;
    if (ENT) {
        float low = min_raw(raw[0], T());
#pragma unroll
        for (int u = 1; u < U; u++) low = fminf(low, min_raw(raw[u], T()));
        cut = (low - m0) * c < LEAST;
    }
    auto sum = [&](auto with_cut) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            float x[V];
            unpack16<T>(raw[u], x);
#pragma unroll
            for (int e = 0; e < V; e += 2) {
                float2 d = __fmul2_rn(__fadd2_rn(make_float2(x[e], x[e + 1]), minus), by);
                const float2 p = make_float2(exp2_approx(d.x), exp2_approx(d.y));
                a.s = __fadd2_rn(a.s, p);
                if (ENT) {
                    if (decltype(with_cut)::value) d = make_float2(fmaxf(d.x, LEAST), fmaxf(d.y, LEAST));
                    a.t = __ffma2_rn(p, d, a.t);
                }
            }
        }
    };
    if (ENT && cut) sum(std::true_type()); else sum(std::false_type());
}

// Offers a chunk's elements to the warp's list.  x0: the column; first: the thread's first whole vector, later ones `step`
// vectors apart; v1: the first vector behind the part.
template <class T, int U>
__device__ __forceinline__ void offer_chunk(Top& top, int k, Key* buffer, unsigned* floor, float m, const uint4 (&raw)[U],
                                            const T* x0, long long first, int step, int head) {
    constexpr int V = Vec16<T>::N;
    if (top.bar == 0 && top.waiting == 0) {
        // Nothing met yet: the k-th largest of the 32 lanes' maxima bounds the k-th best from below.
        const Key sorted = sort_desc(m > -INFINITY ? make_key(m, 0) : 0);
        const float kth = key_value(__shfl_sync(0xffffffffu, sorted, k - 1));
        if ((threadIdx.x & 31) == 0 && kth > -INFINITY) atomicMax(floor, (unsigned)(make_key(kth, 0) >> 32));
        __syncwarp();
    }
    const unsigned fl = *(volatile unsigned*)floor;
    const float least = fmaxf(top.bar_v, fl ? key_value((Key)fl << 32) : -INFINITY);
    unsigned hits = 0;
    if (m >= least) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            float x[V];
            unpack16<T>(raw[u], x);
#pragma unroll
            for (int e = 0; e < V; e++) hits |= (x[e] >= least && x[e] > -INFINITY) ? 1u << (u * V + e) : 0u;
        }
    }
    const Key before = top.bar;
    while (__any_sync(0xffffffffu, hits != 0)) {
        Key key = 0;
        if (hits) {
            const int slot = __ffs(hits) - 1;
            hits &= hits - 1;
            const int at = (int)((first + (long long)(slot / V) * step) * V) + head + slot % V;
            key = make_key(to_f32(x0[at]), at);                 // a second look: the registers cannot be indexed
        }
        top.push(key, buffer, k);
    }
    if (top.bar != before && (threadIdx.x & 31) == 0) atomicMax(floor, (unsigned)(top.bar >> 32));
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// the address, in the cluster's first block, of the variable that this block sees at p
__device__ __forceinline__ unsigned in_first_block(const void* p) {
    unsigned a = (unsigned)__cvta_generic_to_shared(p), r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(a));
    return r;
}
__device__ __forceinline__ void store_remote(unsigned to, unsigned v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(v) : "memory");
}
__device__ __forceinline__ void store_remote(unsigned to, Key v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(v) : "memory");
}

struct LogprobArgs {
    const void* logits; long long ld; int vocab, ncols;
    Tokens tokens;
    float scale;
    float *logp, *lse, *entropy;
    int top;
    float* top_logp; int* top_index;
};

// The results of a column from its statistics and its descending list: one warp.
template <class T, bool ENT, bool TOP>
__device__ __forceinline__ void write_column(const LogprobArgs& q, long long col, const T* x0, const Stat& a, Key list) {
    const int lane = threadIdx.x & 31;
    const bool none = a.m == -INFINITY && a.s == 0.f;
    const float m0 = shift(a.m), l2s = log2f(a.s);
    if (lane == 0) {
        if (q.lse) q.lse[col] = fmaf(m0, q.scale, l2s * LN2);
        if (ENT) { const float h = (l2s - a.t / a.s) * LN2; q.entropy[col] = none || h < 0.f ? 0.f : h; }
        if (q.logp) {
            const long long t = q.tokens[col];
            float r = 0.f;
            if (t >= 0 && t < q.vocab) r = none ? -INFINITY : fmaf(to_f32(x0[t]) - m0, q.scale, -l2s * LN2);
            q.logp[col] = r;
        }
    }
    if (TOP && lane < q.top) {
        q.top_logp[col * q.top + lane] = list == 0 ? -INFINITY : fmaf(key_value(list) - m0, q.scale, -l2s * LN2);
        q.top_index[col * q.top + lane] = key_index(list);
    }
}

// TEAM threads share a column's part: a whole block of 256, or a warp (eight columns a block) where a column is so short
// that a block's joins would cost more than its elements.  A cluster of `parts` blocks shares a column where the columns
// alone are too few to fill the GPU: its blocks leave their sums and lists in the first block's shared memory, which joins
// them, so that there is one launch and no scratch memory.
template <class T, bool ENT, bool TOP, int TEAM>
__global__ void __launch_bounds__(256)
token_logprob_kernel(const LogprobArgs q, int parts) {
    constexpr int V = Vec16<T>::N, U = 4, WARPS = 8, STEP = TEAM;
    __shared__ Stat stats[WARPS], part_stats[WARPS];
    __shared__ Key lists[TOP ? WARPS : 1][32], part_lists[TOP ? WARPS : 1][32], buffers[TOP ? WARPS : 1][64];
    __shared__ unsigned floors[TOP ? WARPS : 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int part = TEAM == 256 ? blockIdx.x % (unsigned)parts : 0;
    const long long col = TEAM == 256 ? blockIdx.x / (unsigned)parts : (long long)blockIdx.x * WARPS + warp;
    if (TEAM == 256 && parts > 1) cluster_arrive();             // waited for before the first remote store: all blocks run then
    if (TOP) {
        if (threadIdx.x < WARPS) floors[threadIdx.x] = 0;
        __syncthreads();
    }
    if (col >= q.ncols) return;
    const T* x0 = (const T*)q.logits + col * q.ld;
    const float c = q.scale * LOG2E;
    const int tid = TEAM == 256 ? threadIdx.x : lane;
    unsigned* floor = &floors[TOP ? (TEAM == 256 ? 0 : warp) : 0];
    Key* buffer = buffers[TOP ? warp : 0];
    // whole 16-byte vectors of the column, behind `head` elements and before the rest
    const int head = min(q.vocab, (int)((16 - (reinterpret_cast<uintptr_t>(x0) & 15)) % 16 / sizeof(T)));
    const int nvec = (q.vocab - head) / V, rest = q.vocab - head - nvec * V;
    const uint4* xv = reinterpret_cast<const uint4*>(x0 + head);
    const int v0 = (int)((long long)nvec * part / parts), v1 = (int)((long long)nvec * (part + 1) / parts);
    Sums a = {-INFINITY, {0.f, 0.f}, {0.f, 0.f}};
    Top best;
    best.clear();
    const unsigned nothing = minus_inf_word<T>();
    uint4 next[U];
    auto fetch = [&](int i) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int v = i + u * STEP + tid;
            next[u] = v < v1 ? __ldg(xv + v) : make_uint4(nothing, nothing, nothing, nothing);
        }
    };
    fetch(v0);
    for (int i = v0; i < v1; i += STEP * U) {
        uint4 raw[U];
#pragma unroll
        for (int u = 0; u < U; u++) raw[u] = next[u];
        if (i + STEP * U < v1) fetch(i + STEP * U);
        float m = max_raw(raw[0], T());
#pragma unroll
        for (int u = 1; u < U; u++) m = fmaxf(m, max_raw(raw[u], T()));
        add_chunk<T, ENT, U>(a, m, raw, c);
        // later elements have higher indices, so a tie with the bar is not a candidate
        if (TOP && __any_sync(0xffffffffu, m > best.bar_v)) offer_chunk<T, U>(best, q.top, buffer, floor, m, raw, x0, i + tid, STEP, head);
    }
    if (part == 0 && (TEAM == 32 || warp == 0) && head + rest > 0) {       // the ends, element by element
        const int at = lane < head ? lane : lane >= 16 && lane - 16 < rest ? head + nvec * V + lane - 16 : -1;
        const float x = at >= 0 ? to_f32(x0[at]) : -INFINITY;
        Stat b = {fmaxf(x, -INFINITY), 0.f, 0.f};               // NaN: leaves the maximum to the others
        const float d = (x - shift(b.m)) * c;
        b.s = exp2_approx(d);
        b.t = b.s * fmaxf(d, LEAST);
        const Stat joined = merge(fold<ENT>(a), b, c);
        a = {joined.m, {joined.s, 0.f}, {joined.t, 0.f}};
        if (TOP) best.push(x > -INFINITY ? make_key(x, at) : 0, buffer, q.top);
    }
    if (TOP) best.finish(buffer, q.top);
    Stat st = fold<ENT>(a);
#pragma unroll
    for (int s = 16; s > 0; s /= 2) {
        Stat b;
        b.m = __shfl_xor_sync(0xffffffffu, st.m, s); b.s = __shfl_xor_sync(0xffffffffu, st.s, s);
        b.t = ENT ? __shfl_xor_sync(0xffffffffu, st.t, s) : 0.f;
        st = merge(st, b, c);
    }
    if (TEAM == 32) { write_column<T, ENT, TOP>(q, col, x0, st, best.list); return; }

    // the block's warps, pairwise
    auto join = [&](Stat* ss, Key (*ls)[32], int n) {
        if (lane == 0) ss[warp] = st;
        if (TOP) ls[warp][lane] = best.list;
        __syncthreads();
        if (TOP) {
            for (int half = n / 2; half > 0; half /= 2) {
                if (warp < half) {
                    best.list = merge_desc(best.list, ls[warp + half][lane]);
                    ls[warp][lane] = best.list;
                }
                __syncthreads();
            }
        }
        if (warp == 0) {
            st = ss[0];
            for (int w = 1; w < n; w++) st = merge(st, ss[w], c);
        }
    };
    join(stats, lists, WARPS);
    if (parts > 1) {
        cluster_wait();
        if (warp == 0) {
            if (lane == 0) {
                const unsigned to = in_first_block(&part_stats[part]);
                store_remote(to, __float_as_uint(st.m)); store_remote(to + 4, __float_as_uint(st.s)); store_remote(to + 8, __float_as_uint(st.t));
            }
            if (TOP) store_remote(in_first_block(&part_lists[part][lane]), best.list);
        }
        cluster_arrive();
        cluster_wait();
        if (part != 0) return;
        const Stat mine = part_stats[min(warp, parts - 1)];
        st = mine;
        if (TOP) best.list = part_lists[min(warp, parts - 1)][lane];
        __syncthreads();
        join(stats, lists, parts);
    }
    if (warp == 0) write_column<T, ENT, TOP>(q, col, x0, st, best.list);
}

template <class T, bool ENT, bool TOP>
static int logprob_go(const LogprobArgs& q, cudaStream_t st) {
    const int nvec = q.vocab / Vec16<T>::N;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    if (nvec <= 512 && q.ncols >= 4 * sm_count()) {
        cfg.gridDim = dim3((q.ncols + 7) / 8);
        CUVDIA_CUDA(cudaLaunchKernelEx(&cfg, token_logprob_kernel<T, ENT, TOP, 32>, q, 1));
        return CUVDIA_OK;
    }
    int parts = 1;
    while (parts < 8 && (long long)q.ncols * parts < 16 * sm_count() && nvec / (2 * parts) >= 1024) parts *= 2;
    if ((long long)q.ncols * parts > 2147483647LL) { set_last_error("token_logprob: too many columns"); return CUVDIA_ERR_UNSUPPORTED; }
    cfg.gridDim = dim3((unsigned)(q.ncols * parts));
    cudaLaunchAttribute cluster;
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = parts; cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    cfg.attrs = &cluster;
    cfg.numAttrs = 1;
    CUVDIA_CUDA(cudaLaunchKernelEx(&cfg, token_logprob_kernel<T, ENT, TOP, 256>, q, parts));
    return CUVDIA_OK;
}

template <class T>
static int logprob_pick(const LogprobArgs& q, cudaStream_t st) {
    if (q.entropy) return q.top ? logprob_go<T, true, true>(q, st) : logprob_go<T, true, false>(q, st);
    return q.top ? logprob_go<T, false, true>(q, st) : logprob_go<T, false, false>(q, st);
}

int launch_token_logprob(const void* logits, int ld, int type, int vocab, int ncols, const void* tokens, int token_type,
                         float scale, float* logp, float* lse, float* entropy, int top, float* top_logp, int* top_index,
                         cudaStream_t st) {
    int rc = CUVDIA_OK;
    const LogprobArgs q = {logits, ld, vocab, ncols, make_tokens(tokens, token_type), scale, logp, lse, entropy, top, top_logp, top_index};
    CUVDIA_FLOAT_TYPE(type, rc = logprob_pick<T>(q, st));
    if (rc) return rc;
    count_launch();
    return check_launch("token_logprob_kernel");
}

// ---- gradient ------------------------------------------------------------------------------------------------------
//   dlogits_v = scale * (dlogp * ([v = token] - p_v) - dentropy * p_v * (log p_v + entropy)),   p_v = exp(scale * logit_v - lse)
// Element-wise once lse and entropy are known: a block owns up to 1024 vectors of one column.  Vectors are those of the
// logits' memory; the stores are vectors too where dlogits lies alike (VEC), else element by element.  In place is fine:
// a thread reads its elements before it writes them.
template <class T>
__global__ void __launch_bounds__(256)
token_logprob_grad_kernel(T* dlogits, long long ldd, const T* logits, long long ld, int vocab, int ncols,
                          const Tokens tokens, float scale, const float* __restrict__ lse,
                          const float* __restrict__ dlogp, const float* __restrict__ entropy,
                          const float* __restrict__ dentropy, int chunks) {
    constexpr int V = Vec16<T>::N, U = 4;
    const long long col = blockIdx.x / (unsigned)chunks;
    const int chunk = blockIdx.x - (unsigned)col * (unsigned)chunks;
    const T* x0 = logits + col * ld;
    T* y0 = dlogits + col * ldd;
    const int head = (int)((reinterpret_cast<uintptr_t>(x0) & 15) / sizeof(T));
    const bool alike = ((reinterpret_cast<uintptr_t>(x0) ^ reinterpret_cast<uintptr_t>(y0)) & 15) == 0;
    long long t = dlogp ? tokens[col] : -1;
    if (t < 0 || t >= vocab) t = -1;
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
    CUVDIA_FLOAT_TYPE(type, (token_logprob_grad_kernel<T><<<(unsigned)blocks, 256, 0, st>>>((T*)dlogits, ldd, (const T*)logits, ld,
        vocab, ncols, make_tokens(tokens, token_type), scale, lse, dlogp, entropy, dentropy, (int)chunks)));
    count_launch();
    return check_launch("token_logprob_grad_kernel");
}

}  // namespace cuvdia
