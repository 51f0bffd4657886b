// Log probabilities of given tokens under softmax(scale * logits), column by column, with the log-sum-exp, the entropy
// and the likeliest tokens; and the gradient with respect to the logits.
//
// Everything is held in 32 bits in powers of two: with c = scale * log2(e), R one of the column's largest logits (below) and
// d_v = (logit_v - R) * c (the difference first, so that logits far from zero and masks of the type's lowest value do no harm),
//   s = sum_v 2^d_v        t = sum_v 2^d_v * d_v
//   lse = scale * R + ln 2 * log2 s      entropy = ln 2 * (log2 s - t / s)      logp_v = scale * (logit_v - R) - ln 2 * log2 s
// R, s and t come from one pass.  A thread's sums are relative to a logit it has met, and are rescaled by 2^(c * (old R - new R))
// when that is left behind: at once where alternatives are asked for, so that R is the column's largest logit M; else only when a
// chunk's sum exceeds 2^24, so that R lies at most 24 powers of two below M.  That bounds what log2 s - t / s and logit_v - R
// against log2 s lose to cancellation: numbers below 32 have a spacing of 2^-19 at most, some 1e-6 in the results.
#include <type_traits>

#include "cluster.cuh"
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

// the largest and the smallest of a vector's elements, NaN left out
__device__ __forceinline__ float max_raw(const uint4& r, float) {
    return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
}
__device__ __forceinline__ float min_raw(const uint4& r, float) {
    return fminf(fminf(__uint_as_float(r.x), __uint_as_float(r.y)), fminf(__uint_as_float(r.z), __uint_as_float(r.w)));
}
#define CUVDIA_RAW16(H, H2, NAME, PAIRS, SINGLE)                                \
    __device__ __forceinline__ float NAME(const uint4& r, H) {                  \
        const H2* h = reinterpret_cast<const H2*>(&r);                          \
        const H2 m = PAIRS(PAIRS(h[0], h[1]), PAIRS(h[2], h[3]));               \
        return SINGLE(to_f32(m.x), to_f32(m.y));                                \
    }
CUVDIA_RAW16(__half, __half2, max_raw, __hmax2, fmaxf)
CUVDIA_RAW16(__half, __half2, min_raw, __hmin2, fminf)
CUVDIA_RAW16(__nv_bfloat16, __nv_bfloat162, max_raw, __hmax2, fmaxf)
CUVDIA_RAW16(__nv_bfloat16, __nv_bfloat162, min_raw, __hmin2, fminf)
#undef CUVDIA_RAW16

template <class T> __device__ __forceinline__ unsigned minus_inf_word();
template <> __device__ __forceinline__ unsigned minus_inf_word<float>() { return 0xff800000u; }
template <> __device__ __forceinline__ unsigned minus_inf_word<__half>() { return 0xfc00fc00u; }
template <> __device__ __forceinline__ unsigned minus_inf_word<__nv_bfloat16>() { return 0xff80ff80u; }

constexpr int U = 4;                    // vectors a thread takes at a time: a chunk

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

// 32 numbers, one a lane, put in descending order (bitonic network); K is Key, or the upper word of one
template <class K>
__device__ __forceinline__ K sort_desc(K k) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int n = 2; n <= 32; n *= 2)
#pragma unroll
        for (int s = n / 2; s > 0; s /= 2) {
            const K o = __shfl_xor_sync(0xffffffffu, k, s);
            const bool upper = (lane & s) != 0, descending = (lane & n) == 0 || n == 32;
            k = (o > k) == (upper != descending) ? o : k;
        }
    return k;
}

// the best 32 of two descending lists, in descending order
template <class K>
__device__ __forceinline__ K merge_desc(K a, K b) {
    const int lane = threadIdx.x & 31;
    const K r = __shfl_sync(0xffffffffu, b, 31 - lane);
    a = r > a ? r : a;
#pragma unroll
    for (int s = 16; s > 0; s /= 2) {
        const K o = __shfl_xor_sync(0xffffffffu, a, s);
        a = (o > a) == ((lane & s) == 0) ? o : a;
    }
    return a;
}

// the best 32 of the descending lists of n warps, pairwise through shared memory: the result is warp 0's
template <class K>
__device__ __forceinline__ K merge_warps(K mine, K (*lists)[32], int n) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    lists[warp][lane] = mine;
    __syncthreads();
    for (int half = n / 2; half > 0; half /= 2) {
        if (warp < half) lists[warp][lane] = mine = merge_desc(mine, lists[warp + half][lane]);
        __syncthreads();
    }
    return mine;
}

// The best 32 of a descending list and 32 candidates in any order.  Called, not inlined: it is rare and long, and copies of it
// cost more in instruction fetches than the calls.
__device__ __noinline__ Key absorb32(Key list, Key batch) { return merge_desc(list, sort_desc(batch)); }
__device__ __noinline__ unsigned sort_upper(unsigned k) { return sort_desc(k); }
__device__ __noinline__ Key sort_keys(Key k) { return sort_desc(k); }

// A warp's best candidates: a descending list (one a lane), and up to 63 more in shared memory that wait to be sorted in,
// 32 at a time.  `bar` is the k-th best of the list: what a new one has to beat.
struct Top {
    Key list, bar;
    int waiting;
    __device__ __forceinline__ void clear() { list = bar = 0; waiting = 0; }
    __device__ __forceinline__ void absorb(Key batch, int k) {
        list = absorb32(list, batch);
        bar = __shfl_sync(0xffffffffu, list, k - 1);
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

// What a thread remembers of its chunks for `collect`: the vector index at which the chunk with its largest logit begins, and
// the largest logit of its other chunks.
struct Where { int chunk; float second; };

// The candidates among a warp's vectors, looked at a second time once `least` is known, a lower bound on the k-th best logit of
// all: only the few threads whose largest logit reaches it own any, nearly always in the one chunk they remember, and what is
// read again lies in L2.  The warp looks at the U vectors of 32 / U such chunks at once; the vectors of a thread with
// candidates in several chunks it goes through 64 at a time.  xv: the column's whole vectors; the warp's own are
// start + lane, start + lane + step, .. below last.
// take(key): one candidate per lane at most (0: none), called by the whole warp.
template <class T, class F>
__device__ __forceinline__ void collect(F&& take, float least, float largest, const Where& w, const uint4* xv, int start, int last,
                                        int step, int head) {
    constexpr int V = Vec16<T>::N, G = 4, W = 2;
    const unsigned nothing = minus_inf_word<T>();
    const int lane = threadIdx.x & 31;
    const bool any = largest >= least && largest > -INFINITY;
    unsigned owners = __ballot_sync(0xffffffffu, any && !(w.second >= least));
    while (owners) {
        int v = last;
#pragma unroll
        for (int g = 0; g < 32 / U; g++) {
            const int from = owners ? __ffs(owners) - 1 : 0;
            const int chunk = __shfl_sync(0xffffffffu, w.chunk, from);
            if (owners && lane / U == g) v = chunk + from + lane % U * step;
            owners &= owners - 1;
        }
        const uint4 raw = v < last ? xv[v] : make_uint4(nothing, nothing, nothing, nothing);
        float x[V];
        unpack16<T>(raw, x);
        unsigned hits = 0;
#pragma unroll
        for (int e = 0; e < V; e++) hits |= x[e] >= least && x[e] > -INFINITY ? 1u << e : 0u;
        while (__any_sync(0xffffffffu, hits != 0)) {
            Key key = 0;
#pragma unroll
            for (int e = V - 1; e >= 0; e--) if (hits >> e & 1) key = make_key(x[e], v * V + e + head);
            hits &= hits - 1;
            take(key);
        }
    }
    owners = __ballot_sync(0xffffffffu, any && w.second >= least);
    while (owners) {
        int first[G];                                           // four threads' vectors are in flight at a time
#pragma unroll
        for (int g = 0; g < G; g++) {
            first[g] = owners ? start + __ffs(owners) - 1 : last;
            owners &= owners - 1;
        }
        for (int r = 0; first[0] + r * step < last; r += 32 * W) {
            uint4 raw[G][W];
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int u = 0; u < W; u++) {
                    const long long v = first[g] + (long long)(r + u * 32 + lane) * step;
                    raw[g][u] = v < last ? xv[v] : make_uint4(nothing, nothing, nothing, nothing);
                }
            unsigned long long hits = 0;                        // bit (g * W + u) * V + e: element e of vector u of thread g
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int u = 0; u < W; u++) {
                    const float m = max_raw(raw[g][u], T());
                    if (m >= least && m > -INFINITY) {
                        float x[V];
                        unpack16<T>(raw[g][u], x);
                        unsigned h = 0;
#pragma unroll
                        for (int e = 0; e < V; e++) h |= x[e] >= least && x[e] > -INFINITY ? 1u << e : 0u;
                        hits |= (unsigned long long)h << ((g * W + u) * V);
                    }
                }
            while (__any_sync(0xffffffffu, hits != 0)) {
                Key key = 0;
                if (hits) {
                    const int slot = __ffsll(hits) - 1, g = slot / (W * V), u = slot / V % W;
                    hits &= hits - 1;
                    const int f = g == 0 ? first[0] : g == 1 ? first[1] : g == 2 ? first[2] : first[3];
                    const int at = (f + (r + u * 32 + lane) * step) * V + slot % V;
                    key = make_key(to_f32(reinterpret_cast<const T*>(xv)[at]), at + head);     // the registers cannot be indexed
                }
                take(key);
            }
        }
    }
}

// ---- one pass over a column -------------------------------------------------------------------------------------------
// The sums of a thread as pairs, so that two elements share an instruction.
struct Sums { float m; float2 s, t; };

// The sums of LANES neighbouring lanes as one, in all of them: relative to their maximum first, so that only one rescaling each
// is needed.
template <bool ENT, int LANES>
__device__ __forceinline__ Stat join_lanes(Stat r, float c) {
    float m = r.m;
    if (LANES == 32) {
        asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(r.m));
    } else {
#pragma unroll
        for (int s = LANES / 2; s > 0; s /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
    }
    if (r.m != m) rescale(r, m, c);
#pragma unroll
    for (int s = LANES / 2; s > 0; s /= 2) {
        r.s += __shfl_xor_sync(0xffffffffu, r.s, s);
        if (ENT) r.t += __shfl_xor_sync(0xffffffffu, r.t, s);
    }
    return r;
}

// The vectors of a column on their way through shared memory: a thread copies its own vectors in asynchronously, some chunks
// ahead, and reads back what it copied itself, so that no barrier is involved and vectors in flight hold no registers.

template <class T>
__device__ __forceinline__ float max_chunk(const uint4* v, int step) {
    float m = max_raw(v[0], T());
#pragma unroll
    for (int u = 1; u < U; u++) m = fmaxf(m, max_raw(v[u * step], T()));
    return m;
}

template <bool ENT>
__device__ __forceinline__ void raise(Sums& a, float m, float c) {
    if (!(m > a.m)) return;
    if (a.m != -INFINITY) {
        const float by = (a.m - m) * c, f = exp2_approx(by), cut = fmaxf(by, LEAST);
        if (ENT) { a.t.x = f * fmaf(a.s.x, cut, a.t.x); a.t.y = f * fmaf(a.s.y, cut, a.t.y); }
        a.s.x *= f; a.s.y *= f;
    }
    a.m = m;
}

// The sums of a chunk, the U vectors v, v + step, .., relative to the logit m0, two elements an instruction.  CUT: exponents are
// cut, see LEAST.
template <class T, bool ENT, bool CUT>
__device__ __forceinline__ void sum_chunk(const uint4* v, int step, float m0, float c, float2& s, float2& t) {
    constexpr int V = Vec16<T>::N;
    const float2 minus = make_float2(-m0, -m0), by = make_float2(c, c);
    s = t = make_float2(0.f, 0.f);
#pragma unroll
    for (int u = 0; u < U; u++) {
        float x[V];
        unpack16<T>(v[u * step], x);
#pragma unroll
        for (int e = 0; e < V; e += 2) {
            float2 d = __fmul2_rn(__fadd2_rn(make_float2(x[e], x[e + 1]), minus), by);
            const float2 p = make_float2(exp2_approx(d.x), exp2_approx(d.y));
            s = __fadd2_rn(s, p);
            if (ENT) {
                if (CUT) d = make_float2(fmaxf(d.x, LEAST), fmaxf(d.y, LEAST));
                t = __ffma2_rn(p, d, t);
            }
        }
    }
}

// A chunk's sum beyond this has left its reference behind: 2^24, of exponents of up to 24 times the powers with ENT.  (At 2^16 the
// logits of a normal distribution with a deviation of 5 exceeded it often enough to cost a tenth of the time, at 2^24 next to never.)
template <bool ENT> constexpr float OVER = ENT ? 16.f * 16777216.f : 16777216.f;

// Adds a chunk to a thread's sums.  The sums may be relative to any logit not far below the largest, so the maximum is only looked
// for in a thread's first chunk (MAX: in every chunk, for callers that want the maximum itself).  A chunk whose sum exceeds OVER - a
// logit far above the reference - or come out NaN - an exponent of -inf (a forbidden token, or the empty end of a column's last
// chunk) times its power of zero - is summed once more, relative to its maximum and with its exponents cut; after a NaN so are the
// thread's later chunks at once (careful).  The other threads need no test per element.
template <class T, bool ENT, bool MAX>
__device__ __forceinline__ void add_chunk(Sums& a, const uint4* v, int step, float c, Where& w, int at, bool& careful) {
    if (MAX) {
        const float m = max_chunk<T>(v, step), before = a.m;
        if (m > before) w.chunk = at;
        w.second = fmaxf(w.second, fminf(m, before));
        raise<ENT>(a, m, c);
    } else if (a.m == -INFINITY || careful) {
        raise<ENT>(a, max_chunk<T>(v, step), c);
    }
    float2 s, t;
    bool again = careful;
    if (!careful) {
        sum_chunk<T, ENT, false>(v, step, shift(a.m), c, s, t);
        const float sum = ENT ? t.x + t.y : s.x + s.y;
        again = !(sum < OVER<ENT>);
        careful = sum != sum;
        if (again && !MAX) raise<ENT>(a, max_chunk<T>(v, step), c);
    }
    if (again) sum_chunk<T, ENT, ENT>(v, step, shift(a.m), c, s, t);
    a.s = __fadd2_rn(a.s, s);
    if (ENT) a.t = __fadd2_rn(a.t, t);
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

// The results of a column from its statistics and its descending list: LANES neighbouring lanes.  given: the column's token is
// one of the vocabulary; given_logit is its logit then.
template <class T, bool ENT, bool TOP, int LANES>
__device__ __forceinline__ void write_column(const LogprobArgs& q, long long col, bool given, float given_logit, const Stat& a,
                                             Key list) {
    const int lane = threadIdx.x % LANES;
    const bool none = a.m == -INFINITY && a.s == 0.f;
    const float m0 = shift(a.m), l2s = log2f(a.s);
    if (lane == 0) {
        if (q.lse) q.lse[col] = fmaf(m0, q.scale, l2s * LN2);
        if (ENT) { const float h = (l2s - a.t / a.s) * LN2; q.entropy[col] = none || h < 0.f ? 0.f : h; }
        if (q.logp) q.logp[col] = !given ? 0.f : none ? -INFINITY : fmaf(given_logit - m0, q.scale, -l2s * LN2);
    }
    if (TOP && lane < q.top) {
        q.top_logp[col * q.top + lane] = list == 0 ? -INFINITY : fmaf(key_value(list) - m0, q.scale, -l2s * LN2);
        q.top_index[col * q.top + lane] = key_index(list);
    }
}

// TEAM threads share a column's part: a whole block, or a warp or eight lanes (8 or 32 columns a block of 256) where a column
// is so short that a block's joins, or a warp's, would cost more than its elements.  A cluster of `parts` blocks shares a column where the columns
// alone are too few to fill the GPU: its blocks leave their sums and lists in the first block's shared memory, which joins
// them, so that there is one launch and no scratch memory.
//
// Bound by memory where columns are many: 32768 x 8192 bf16 with entropies 82 us (6.5 TB/s; the exponential unit is 80 % busy; in
// short bursts, under a sustained load at a lower clock 89 to 96 us), 32767 x 8192 90 us, whose last chunks have empty places,
// 50021 x 1000 f32 39 us (5.1 TB/s: 7 blocks on most SMs, 6 on the others, and their common start and end), with 20 alternatives
// and a third of the tokens forbidden 45 us.  A few columns are bound by latency: 131072 x 4 bf16 6 us, 8.5 us with alternatives.
template <class T, bool ENT, bool TOP, int TEAM>
__global__ void __launch_bounds__(TEAM < 128 ? 256 : TEAM, TEAM == 128 ? 8 : 4)
token_logprob_kernel(const LogprobArgs q, int parts) {
    constexpr int V = Vec16<T>::N, THREADS = TEAM < 128 ? 256 : TEAM, WARPS = THREADS / 32, LANES = TEAM < 32 ? TEAM : 32, STEP = TEAM;
    constexpr int STAGES = TEAM == 128 && !TOP ? 3 : 2;          // three would not leave room for a list's arrays in as many blocks
    constexpr bool BLOCK = TEAM >= 128;
    static_assert(TEAM >= 32 || (TEAM >= V - 1 && !TOP), "lists and ends");
    __shared__ uint4 ring[STAGES * U * THREADS];
    __shared__ Stat stats[WARPS], part_stats[8];
    __shared__ Key lists[TOP ? WARPS : 1][32], part_lists[TOP ? 8 : 1][32], buffers[TOP ? WARPS : 1][64];
    __shared__ unsigned maxima[TOP ? 32 : 1];
    __shared__ int found;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int part = BLOCK ? blockIdx.x % (unsigned)parts : 0;
    long long col = BLOCK ? blockIdx.x / (unsigned)parts : (long long)blockIdx.x * (THREADS / TEAM) + threadIdx.x / TEAM;
    if (BLOCK && parts > 1) cluster_arrive();             // waited for before the first remote store: all blocks run then
    const bool beyond = col >= q.ncols;
    if (beyond && TEAM >= 32) return;
    if (beyond) col = q.ncols - 1;                              // for the other lanes' shuffles; nothing is written
    const T* x0 = (const T*)q.logits + col * q.ld;
    const float c = q.scale * LOG2E;
    const int tid = threadIdx.x % TEAM;
    // whole 16-byte vectors of the column, behind `head` elements and before the rest
    const int head = min(q.vocab, (int)((16 - (reinterpret_cast<uintptr_t>(x0) & 15)) % 16 / sizeof(T)));
    const int nvec = (q.vocab - head) / V, rest = q.vocab - head - nvec * V;
    const uint4* xv = reinterpret_cast<const uint4*>(x0 + head);
    const int v0 = (int)((long long)nvec * part / parts), v1 = (int)((long long)nvec * (part + 1) / parts);
    Sums a = {-INFINITY, {0.f, 0.f}, {0.f, 0.f}};
    Where where = {0, -INFINITY};
    bool careful = false;
    // the given token's logit, fetched here so that it need not be waited for at the end
    bool given = false;
    float given_logit = 0.f;
    if (q.logp && tid == 0 && part == 0) {
        const long long t = q.tokens[col];
        given = t >= 0 && t < q.vocab;
        if (given) given_logit = to_f32(x0[t]);
    }
    const unsigned nothing = minus_inf_word<T>();
    uint4* mine = ring + threadIdx.x;                            // [stage][u][thread]
    const uint4* from = xv + v0 + tid;                          // the chunk to fetch next
    int ahead = v0, stage = 0;
    auto fetch = [&](int to) {
        uint4* slot = mine + to * (U * THREADS);
        if (ahead + STEP * U <= v1) {
#pragma unroll
            for (int u = 0; u < U; u++) copy_async16(slot + u * THREADS, from + u * STEP);
        } else if (ahead < v1) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (ahead + u * STEP + tid < v1) copy_async16(slot + u * THREADS, from + u * STEP);
                else slot[u * THREADS] = make_uint4(nothing, nothing, nothing, nothing);
            }
        }
        copies_commit();
        ahead += STEP * U;
        from += STEP * U;
    };
#pragma unroll
    for (int k = 0; k < STAGES; k++) fetch(k);
    for (int i = v0; i < v1; i += STEP * U) {
        copies_wait<STAGES - 1>();
        add_chunk<T, ENT, TOP>(a, mine + stage * (U * THREADS), THREADS, c, where, i + tid - lane, careful);
        fetch(stage);
        stage = stage + 1 == STAGES ? 0 : stage + 1;
    }
    const float largest = a.m;
    float edge = -INFINITY;                                     // of the ends: one element a lane at most
    int edge_at = -1;
    auto add_edge = [&](int at) {
        edge_at = at;
        edge = at >= 0 ? to_f32(x0[at]) : -INFINITY;
        Stat b = {fmaxf(edge, -INFINITY), 0.f, 0.f};            // NaN: leaves the maximum to the others
        const float d = (edge - shift(b.m)) * c;
        b.s = exp2_approx(d);
        b.t = b.s * fmaxf(d, LEAST);
        const Stat joined = merge({a.m, a.s.x + a.s.y, a.t.x + a.t.y}, b, c);
        a = {joined.m, {joined.s, 0.f}, {joined.t, 0.f}};
    };
    if (part == 0 && (!BLOCK || warp == 0) && head + rest > 0) {       // the ends, element by element
        if (TEAM >= 32) {
            add_edge(lane < head ? lane : lane >= 16 && lane - 16 < rest ? head + nvec * V + lane - 16 : -1);
        } else {
            add_edge(tid < head ? tid : -1);
            add_edge(tid < rest ? head + nvec * V + tid : -1);
        }
    }
    Key list = 0;
    if (TOP) {
        // The k-th largest of some of the threads' largest logits bounds the k-th best from below, and few logits reach it.
        unsigned own = a.m > -INFINITY ? (unsigned)(make_key(a.m, 0) >> 32) : 0;
        if (BLOCK) {                                            // 32 of them, the same number from each warp
            for (int j = 0; j < 32 / WARPS; j++) {
                const unsigned m = __reduce_max_sync(0xffffffffu, own);
                const int from = __ffs(__ballot_sync(0xffffffffu, own == m)) - 1;
                if (lane == from) own = 0;
                if (lane == 0) maxima[warp * (32 / WARPS) + j] = m;
            }
            if (threadIdx.x == 0) found = 0;
            __syncthreads();
            own = maxima[lane];
        }
        const float least = key_value((Key)__shfl_sync(0xffffffffu, sort_upper(own), q.top - 1) << 32);
        const bool at_edge = edge >= least && edge > -INFINITY;
        // A block gathers its candidates in shared memory; a warp on its own, and a block with more of them than fit there
        // (many ties), sorts them into lists of its warps as they come.
        if (BLOCK) {
            auto take = [&](Key key) {
                const unsigned there = __ballot_sync(0xffffffffu, key != 0);
                int at = 0;
                if (lane == 0) at = atomicAdd(&found, __popc(there));
                at = __shfl_sync(0xffffffffu, at, 0) + __popc(there & ((1u << lane) - 1));
                if (key != 0 && at < WARPS * 32) (&lists[0][0])[at] = key;
            };
            collect<T>(take, least, largest, where, xv, v0 + tid - lane, v1, STEP, head);
            if (__any_sync(0xffffffffu, at_edge)) take(at_edge ? make_key(edge, edge_at) : 0);
            __syncthreads();
        }
        const int n = BLOCK ? found : WARPS * 32 + 1;
        if (n <= WARPS * 32) {
            if (warp * 32 < n) list = sort_keys(warp * 32 + lane < n ? lists[warp][lane] : 0);
            __syncthreads();
            if (n > 32) list = merge_warps(list, lists, WARPS);
        } else {
            Top best;
            best.clear();
            auto take = [&](Key key) { best.push(key, buffers[warp], q.top); };
            collect<T>(take, least, largest, where, xv, v0 + tid - lane, v1, STEP, head);
            if (__any_sync(0xffffffffu, at_edge)) take(at_edge ? make_key(edge, edge_at) : 0);
            best.finish(buffers[warp], q.top);
            list = best.list;
            if (BLOCK) {
                __syncthreads();
                list = merge_warps(list, lists, WARPS);
            }
        }
    }
    Stat st = join_lanes<ENT, LANES>({a.m, a.s.x + a.s.y, ENT ? a.t.x + a.t.y : 0.f}, c);
    if (!BLOCK) {
        if (!beyond) write_column<T, ENT, TOP, LANES>(q, col, given, given_logit, st, list);
        return;
    }

    if (lane == 0) stats[warp] = st;
    __syncthreads();
    if (warp == 0) st = join_lanes<ENT, WARPS>(stats[lane % WARPS], c);
    if (parts > 1) {
        cluster_wait();
        if (warp == 0) {
            if (lane == 0) {
                const unsigned to = in_block(&part_stats[part], 0);
                store_remote(to, __float_as_uint(st.m)); store_remote(to + 4, __float_as_uint(st.s)); store_remote(to + 8, __float_as_uint(st.t));
            }
            if (TOP) store_remote(in_block(&part_lists[part][lane], 0), list);
        }
        cluster_arrive();
        cluster_wait();
        if (part != 0) return;
        if (warp == 0) st = join_lanes<ENT, 8>(lane % 8 < parts ? part_stats[lane % 8] : Stat{-INFINITY, 0.f, 0.f}, c);
        if (TOP) {
            list = part_lists[min(warp, parts - 1)][lane];
            __syncthreads();                                    // `lists` is read above
            list = merge_warps(list, lists, parts);
        }
    }
    if (warp == 0) write_column<T, ENT, TOP, LANES>(q, col, given, given_logit, st, list);
}

template <class T, bool ENT, bool TOP>
static int logprob_go(const LogprobArgs& q, cudaStream_t st) {
    const int nvec = q.vocab / Vec16<T>::N;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    // eight lanes a column where it is short (304 x 20000 bf16: 10.3 us, by warps 20 us; 1024 x 20000: 14.5 and 19 us, but
    // 2048 x 4000: 10.2 and 8.2 us), if there are enough of them (304 x 1000: 5.6 us, by blocks 7.4 us)
    if (!TOP && nvec <= 128 && q.ncols >= 4 * sm_count()) {
        cfg.gridDim = dim3((unsigned)(((long long)q.ncols + 31) / 32));
        CUVDIA_CUDA(cudaLaunchKernelEx(&cfg, token_logprob_kernel<T, ENT, false, 8>, q, 1));
        return CUVDIA_OK;
    }
    // a warp a column (8000 x 8000 bf16: 29 us, by blocks 35 us), if there are enough of them (8000 x 700: 8.2 us, by blocks 7.1 us)
    if (nvec <= 1024 && q.ncols >= 8 * sm_count()) {
        cfg.gridDim = dim3(((unsigned)q.ncols + 7) / 8);
        CUVDIA_CUDA(cudaLaunchKernelEx(&cfg, token_logprob_kernel<T, ENT, TOP, 32>, q, 1));
        return CUVDIA_OK;
    }
    // What a call takes, in fifths of the time an SM needs to bring in a chunk of 16 KB (0.37 us): a block's chunks, each at the
    // rate its SM's blocks leave it but no faster than a round trip to memory allows; and for clusters 2 us and 0.7 us a block of
    // an SM (131072 x 200 bf16 in 1, 2, 4, 8 parts: 16.5, 16.7, 20.5, 22.5 us; 131072 x 4: 14.2 us in one, 8.5 us in 8).
    int parts = 1;
    long long best = 0;
    for (int p = 1; p <= 8; p *= 2) {
        const long long chunks = (nvec + 1024 * p - 1) / (1024 * p), per_sm = ((long long)q.ncols * p + sm_count() - 1) / sm_count();
        const long long cost = chunks * std::max(5 * per_sm, 6LL) + (p > 1 ? 27 + 9 * per_sm : 0);
        if (p == 1 || cost < best) { parts = p; best = cost; }
    }
    // Many columns: smaller blocks, of which a thread's share of the joins is smaller (32768 x 8192 bf16: 82 us, blocks of 256 90 us)
    if (parts == 1 && q.ncols >= 4 * sm_count()) {
        cfg.blockDim = dim3(128);
        cfg.gridDim = dim3(q.ncols);
        CUVDIA_CUDA(cudaLaunchKernelEx(&cfg, token_logprob_kernel<T, ENT, TOP, 128>, q, 1));
        return CUVDIA_OK;
    }
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
// Element-wise once lse and entropy are known: with d = scale * logit - lse,
//   dlogits_v = 2^(d log2 e) * (A d + B) (+ scale * dlogp at the token),   A = -scale dentropy,  B = -scale (dlogp + dentropy entropy)
// two elements an instruction.  A block owns up to 1024 vectors of one column, those of the logits' memory; 16 lanes own all of
// a column of up to 64.  The stores are vectors too where dlogits lies alike, else element by element.  In place is fine: a
// thread reads its elements before it writes them.
// Bound by memory: 32768 x 8192 bf16 with or without entropies 158 us (6.8 TB/s), 32768 x 4096 f32 160 us.  The straight-line path
// for blocks that lie inside a column is what that took (one path with tests per vector: 176 us).  A result that lies otherwise than
// the logits on the 16-byte grid is stored element by element: 32768 x 8192 bf16 520 to 600 us, 32768 x 4096 f32 184 us.
struct GradFactors { float scale, minus_lse, a, b; };

// two gradients but for the token's own term; CUT: exponents are cut, see LEAST
template <bool ENT, bool CUT>
__device__ __forceinline__ void grad_pair(float& x, float& y, const GradFactors& f) {
    float2 d = __ffma2_rn(make_float2(x, y), make_float2(f.scale, f.scale), make_float2(f.minus_lse, f.minus_lse));
    const float2 q = __fmul2_rn(d, make_float2(LOG2E, LOG2E));
    const float2 p = make_float2(exp2_approx(q.x), exp2_approx(q.y));
    if (ENT && CUT) d = make_float2(fmaxf(d.x, LEAST), fmaxf(d.y, LEAST));
    const float2 b = make_float2(f.b, f.b);
    const float2 r = __fmul2_rn(p, ENT ? __ffma2_rn(d, make_float2(f.a, f.a), b) : b);
    x = r.x; y = r.y;
}

template <class T, bool ENT, bool CUT>
__device__ __forceinline__ void grad_vector(float (&x)[Vec16<T>::N], const GradFactors& f) {
#pragma unroll
    for (int e = 0; e < Vec16<T>::N; e += 2) grad_pair<ENT, CUT>(x[e], x[e + 1], f);
}

template <class T, bool ENT, int TEAM>
__global__ void __launch_bounds__(TEAM < 64 ? 256 : TEAM)
token_logprob_grad_kernel(T* dlogits, long long ldd, const T* logits, long long ld, int vocab, int ncols, const Tokens tokens, float scale,
                          const float* __restrict__ lse, const float* __restrict__ dlogp, const float* __restrict__ entropy,
                          const float* __restrict__ dentropy, int chunks) {
    constexpr int V = Vec16<T>::N;
    constexpr bool SHORT = TEAM < 64;                           // several columns a block
    const int tid = threadIdx.x % TEAM;
    const long long col = SHORT ? (long long)blockIdx.x * (256 / TEAM) + threadIdx.x / TEAM : blockIdx.x / (unsigned)chunks;
    const int chunk = SHORT ? 0 : blockIdx.x - (unsigned)col * (unsigned)chunks;
    if (SHORT && col >= ncols) return;
    const T* x0 = logits + col * ld;
    T* y0 = dlogits + col * ldd;
    // whole vectors of the column, behind `head` elements and before the rest
    const int head = min(vocab, (int)((16 - (reinterpret_cast<uintptr_t>(x0) & 15)) % 16 / sizeof(T)));
    const int nvec = (vocab - head) / V, rest = vocab - head - nvec * V;
    const bool alike = ((reinterpret_cast<uintptr_t>(x0) ^ reinterpret_cast<uintptr_t>(y0)) & 15) == 0;
    const float l = lse[col];
    long long t = dlogp ? tokens[col] : -1;
    if (t < 0 || t >= vocab) t = -1;
    // A padded column without an entropy term is zero without a look at its logits, and so is a column that has no
    // finite logit.
    const bool zero = (t < 0 && !ENT) || l == -INFINITY;
    const uint4* from = reinterpret_cast<const uint4*>(x0 + head);
    T* to = y0 + head;
    const int v0 = chunk * (TEAM * U) + tid;
    const bool plain = !SHORT && alike && !zero && (chunk + 1) * (TEAM * U) <= nvec;    // as most blocks are
    uint4 raw[U];
    if (plain) {
#pragma unroll
        for (int u = 0; u < U; u++) raw[u] = from[v0 + u * TEAM];
    }
    const float g = t >= 0 ? dlogp[col] : 0.f, h = ENT ? dentropy[col] : 0.f, hot = scale * g;
    const GradFactors f = {scale, -l, -scale * h, -scale * (ENT ? fmaf(h, entropy[col], g) : g)};
    const int token = t >= 0 ? (int)t - head : -1;              // the token's place behind the whole vectors' start
    // a whole vector's gradients; 0 * -inf comes up only where the least exponent is out of all proportion (a forbidden token)
    auto whole_vector = [&](const uint4& r, int v) {
        float x[V];
        unpack16<T>(r, x);
        if (ENT && fmaf(min_raw(r, T()), scale, -l) < LEAST) grad_vector<T, ENT, true>(x, f);
        else grad_vector<T, ENT, false>(x, f);
        const unsigned at = (unsigned)(token - v * V);
        if (at < V && token >= 0) {
#pragma unroll
            for (int e = 0; e < V; e++) if (e == (int)at) x[e] += hot;
        }
        return pack16<T>(x);
    };
    if (plain) {
#pragma unroll
        for (int u = 0; u < U; u++) reinterpret_cast<uint4*>(to)[v0 + u * TEAM] = whole_vector(raw[u], v0 + u * TEAM);
    } else if (SHORT && alike && !zero) {
#pragma unroll
        for (int u = 0; u < U; u++) if (v0 + u * TEAM < nvec) raw[u] = from[v0 + u * TEAM];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (v0 + u * TEAM < nvec) reinterpret_cast<uint4*>(to)[v0 + u * TEAM] = whole_vector(raw[u], v0 + u * TEAM);
    } else {
#pragma unroll 1
        for (int v = v0; v < min(nvec, (chunk + 1) * (TEAM * U)); v += TEAM) {
            const uint4 r = zero ? make_uint4(0, 0, 0, 0) : whole_vector(from[v], v);
            if (alike) { reinterpret_cast<uint4*>(to)[v] = r; continue; }
            float x[V];
            unpack16<T>(r, x);
#pragma unroll
            for (int e = 0; e < V; e++) to[v * V + e] = from_f32<T>(x[e]);
        }
    }
    static_assert(TEAM >= 2 * (V - 1), "ends");
    if (chunk == 0 && tid < head + rest) {                      // the ends, one element a thread
        const int i = tid < head ? tid : nvec * V + tid;
        float x[2] = {zero ? 0.f : to_f32(x0[i]), 0.f};
        if (!zero) grad_pair<ENT, true>(x[0], x[1], f);
        y0[i] = from_f32<T>(zero ? 0.f : t == i ? x[0] + hot : x[0]);
    }
}

int launch_token_logprob_grad(void* dlogits, int ldd, const void* logits, int ld, int type, int vocab, int ncols,
                              const void* tokens, int token_type, float scale, const float* lse, const float* dlogp,
                              const float* entropy, const float* dentropy, cudaStream_t st) {
    const int v = 16 / type_size(type);
    // blocks of 1024 vectors, of 256 where a column has no more (1000 x 4000 bf16: 8.2 us, with large blocks 12.3 us); 16 lanes a
    // column where columns are short (305 x 100000 bf16: 31 us, by blocks 59 us; 512 x 20000: 12.3 and 16.4 us, but 1024 x 1000:
    // 5.3 and 4.4 us) and more than the SMs hold at a time (below that the two take the same)
    const int team = vocab > 256 * v ? 256 : vocab > 64 * v || ncols < 4 * sm_count() ? 64 : 16;
    const long long chunks = std::max(1LL, ((long long)vocab / v + team * U - 1) / (team * U));
    const long long blocks = team == 16 ? ((long long)ncols + 15) / 16 : chunks * ncols;
    if (blocks > 2147483647LL) { set_last_error("token_logprob_grad: %lld blocks", blocks); return CUVDIA_ERR_UNSUPPORTED; }
#define LG_GO(E, N) token_logprob_grad_kernel<T, E, N><<<(unsigned)blocks, N < 64 ? 256 : N, 0, st>>>((T*)dlogits, ldd, (const T*)logits, ld, \
    vocab, ncols, make_tokens(tokens, token_type), scale, lse, dlogp, entropy, dentropy, (int)chunks)
    CUVDIA_FLOAT_TYPE(type, {
        if (team == 256)     { if (dentropy) LG_GO(true, 256); else LG_GO(false, 256); }
        else if (team == 64) { if (dentropy) LG_GO(true, 64); else LG_GO(false, 64); }
        else                 { if (dentropy) LG_GO(true, 16); else LG_GO(false, 16); }
    });
#undef LG_GO
    count_launch();
    return check_launch("token_logprob_grad_kernel");
}

}  // namespace cuvdia
