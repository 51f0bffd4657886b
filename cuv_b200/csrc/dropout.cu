// Dropout with the uniform numbers of philox.cuh, drawn in registers:
//   dst = (u >= p ? src / (1 - p) : 0) + residual
// with u the number cuvdia_uniform_f32 gives for the element, so no mask is ever stored: the backward pass is the same
// pass over the gradient, and it draws the same numbers.  u >= p is decided on the generator's words: u = (word >> 8)
// * 2^-24, hence u >= p exactly if word >= ceil(p * 2^24) * 2^8.
#include <cmath>

#include "philox.cuh"
#include "typed.cuh"

namespace cuvdia {

// What a call's threads share: the round keys of the generator (added up on the host: a thread would spend a third of the
// generator's instructions on them), and the second and third word of the counter but for the column.
struct DropoutArgs {
    unsigned key0[10], key1[10], which, step;
    long long col0;
    unsigned least;                     // the smallest word that keeps its element
    float scale;
};

constexpr unsigned M0 = 0xD2511F53u, M1 = 0xCD9E8D57u;

// The four words of a group of rows; first = M0 * group, the first round's product, which a caller that walks through a column
// adds up instead of multiplying.
__device__ __forceinline__ uint4 draw_words(const DropoutArgs& a, unsigned long long first, long long gcol) {
    const unsigned long long second = (unsigned long long)M1 * (a.which + 65536u * (unsigned)(gcol >> 32));
    uint4 c = make_uint4((unsigned)(second >> 32) ^ (unsigned)gcol ^ a.key0[0], (unsigned)second,
                         (unsigned)(first >> 32) ^ a.step ^ a.key1[0], (unsigned)first);
#pragma unroll
    for (int r = 1; r < 10; r++) {
        const unsigned long long p0 = (unsigned long long)M0 * c.x, p1 = (unsigned long long)M1 * c.z;
        c = make_uint4((unsigned)(p1 >> 32) ^ c.y ^ a.key0[r], (unsigned)p1, (unsigned)(p0 >> 32) ^ c.w ^ a.key1[r], (unsigned)p0);
    }
    return c;
}

// One word per element for the rows from a group of four on
template <int WORDS>
__device__ __forceinline__ void draw(const DropoutArgs& a, unsigned long long first, long long gcol, unsigned (&word)[WORDS]) {
#pragma unroll
    for (int q = 0; q < WORDS / 4; q++) {
        const uint4 w = draw_words(a, first + (unsigned long long)M0 * q, gcol);
        word[4 * q] = w.x; word[4 * q + 1] = w.y; word[4 * q + 2] = w.z; word[4 * q + 3] = w.w;
    }
}

template <class T> struct Streams { T* dst; const T* src; const T* residual; long long ldd, lds, ldr; };

// ---- matrices whose columns lie alike --------------------------------------------------------------------------------
// A column is walked as the 16-byte vectors of the memory it lies in, E elements each.  Where every column starts on such a
// vector (SHIFTED = false) a vector's rows are whole groups of the generator.  Where columns start h elements into one (the
// same h in all matrices), the rows of vector k are E*k - h ..: a lane draws for the rows E*k .. and takes the other h
// decisions from the lane before it, so nothing is drawn twice but one lane's share of a part.
// `lanes` threads (a power of two; of one warp if SHIFTED) take a part of a column, U vectors each, `lanes` vectors apart: all
// loads are in flight before the first number is drawn.  WIDE: a part is a block's.  NONE: p = 1, every element is dropped.
//
// Bound by memory where an element is at least six bytes of traffic: 16384 x 8192 bf16 with residual 117 us (6.9 TB/s), 16384 x 4096
// f32 80 us (6.7 TB/s), in short bursts of calls (under a sustained load, at a lower clock, the first takes 128 to 136 us).  A 16-bit pass
// without residual (four bytes) is bound by the generator's 17 wide products per four elements: 103 to 107 us at 16384 x 8192 for
// 82 us of traffic, its warps waiting for arithmetic and dispatch and hardly for memory; taking the products' high words from the
// double units instead gained nothing, the register moves around them costing as much.  Columns that do not start on vectors:
// 16383 x 8191 168 us with residual (element by element 315 us), 154 us without.
template <class T, bool RESIDUAL, bool SHIFTED, bool NONE, int U, bool WIDE>
__global__ void __launch_bounds__(256, 4)
dropout_kernel(const Streams<T> m, int rows, int ncols, int log_lanes, int parts, const DropoutArgs a) {
    constexpr int E = Vec16<T>::N;
    const int lanes = WIDE ? 256 : 1 << log_lanes, l = threadIdx.x & (lanes - 1), span = lanes * U - (SHIFTED ? 1 : 0);
    long long col;
    int part;
    if (WIDE) {                                                 // one part a block
        col = (long long)blockIdx.z * gridDim.y + blockIdx.y;
        part = blockIdx.x;
    } else {
        const unsigned team = blockIdx.x * (256u >> log_lanes) + (threadIdx.x >> log_lanes);
        col = team / (unsigned)parts;
        part = (int)(team - (unsigned)col * (unsigned)parts);
    }
    const bool idle = col >= ncols;
    if (!SHIFTED && idle) return;
    if (idle) col = 0;
    const T* s = m.src + col * m.lds;
    const T* r = RESIDUAL ? m.residual + col * m.ldr : nullptr;
    T* d = m.dst + col * m.ldd;
    const int h = SHIFTED ? (int)((reinterpret_cast<uintptr_t>(d) & 15) / sizeof(T)) : 0;
    const int w0 = part * span + l, i0 = w0 * E - h;
    const long long gcol = a.col0 + col;
    unsigned long long first = (unsigned long long)M0 * (unsigned)(w0 * (E / 4));
    const unsigned long long first_step = (unsigned long long)M0 * (unsigned)(lanes * (E / 4));
    unsigned before = 0;
    // the decisions for vector u, which comes after u - 1: words, or (SHIFTED) bits
    auto decide = [&](int u, unsigned (&word)[E]) {
        unsigned mask = 0;
        if (!NONE) draw<E>(a, first, gcol, word);
        first += first_step;
        if (SHIFTED) {
            if (!NONE) {
#pragma unroll
                for (int e = 0; e < E; e++) mask |= word[e] >= a.least ? 1u << e : 0u;
            }
            unsigned prev = __shfl_up_sync(0xffffffffu, mask, 1, lanes);
            const unsigned last = __shfl_sync(0xffffffffu, before, lanes - 1, lanes);
            if (u > 0 && l == 0) prev = last;
            before = mask;
            mask = (prev | mask << E) >> (E - h);
        }
        return mask;
    };
    auto apply = [&](float (&x)[E], const float (&y)[E], const unsigned (&word)[E], unsigned mask) {
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const float2 scaled = __fmul2_rn(make_float2(x[e], x[e + 1]), make_float2(a.scale, a.scale));
            const bool keep0 = SHIFTED ? mask >> e & 1 : !NONE && word[e] >= a.least;
            const bool keep1 = SHIFTED ? mask >> (e + 1) & 1 : !NONE && word[e + 1] >= a.least;
            const float2 kept = make_float2(keep0 ? scaled.x : 0.f, keep1 ? scaled.y : 0.f);
            const float2 sum = RESIDUAL ? __fadd2_rn(kept, make_float2(y[e], y[e + 1])) : kept;
            x[e] = sum.x; x[e + 1] = sum.y;
        }
    };
    const bool ghost = SHIFTED && part > 0 && l == 0;           // whose first vector is the lane's before: drawn, not written
    // threads whose vectors all lie inside the column, as most do, take a straight line; shifted columns have ends enough to be
    // left to one path, which loads ahead too
    const bool plain = !SHIFTED && i0 + ((U - 1) * lanes + 1) * E <= rows;
    uint4 xs[U], ys[U];
    if (plain || SHIFTED) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = i0 + u * lanes * E;
            if (SHIFTED && (idle || i < 0 || i + E > rows)) continue;
            xs[u] = *reinterpret_cast<const uint4*>(s + i);
            if (RESIDUAL) ys[u] = *reinterpret_cast<const uint4*>(r + i);
        }
    }
    if (plain) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            unsigned word[E];
            const unsigned mask = decide(u, word);
            float x[E], y[E];
            unpack16<T>(xs[u], x);
            if (RESIDUAL) unpack16<T>(ys[u], y);
            apply(x, y, word, mask);
            *reinterpret_cast<uint4*>(d + i0 + u * lanes * E) = pack16<T>(x);
        }
        return;
    }
#pragma unroll (SHIFTED ? U : 1)
    for (int u = 0; u < U; u++) {
        const int i = i0 + u * lanes * E;
        unsigned word[E];
        const unsigned mask = decide(u, word);
        if (idle || i >= rows || (u == 0 && ghost)) continue;
        const bool whole = i >= 0 && i + E <= rows;
        float x[E], y[E];
        if (whole) {
            unpack16<T>(SHIFTED ? xs[u] : *reinterpret_cast<const uint4*>(s + i), x);
            if (RESIDUAL) unpack16<T>(SHIFTED ? ys[u] : *reinterpret_cast<const uint4*>(r + i), y);
        } else {
#pragma unroll
            for (int e = 0; e < E; e++) {
                const bool in = i + e >= 0 && i + e < rows;
                x[e] = in ? to_f32(s[i + e]) : 0.f;
                if (RESIDUAL) y[e] = in ? to_f32(r[i + e]) : 0.f;
            }
        }
        apply(x, y, word, mask);
        if (whole) {
            *reinterpret_cast<uint4*>(d + i) = pack16<T>(x);
        } else {
#pragma unroll
            for (int e = 0; e < E; e++) if (i + e >= 0 && i + e < rows) d[i + e] = from_f32<T>(x[e]);
        }
    }
}

// ---- any layout --------------------------------------------------------------------------------------------------------
// Matrices that lie differently: four rows, one group of the generator, a thread, element by element (16383 x 8191 bf16 221 us with
// residual, 197 us without; 16383 x 4096 f32 102 us).
template <class T, bool RESIDUAL>
__global__ void __launch_bounds__(256)
dropout_any_kernel(const Streams<T> m, int rows, int ncols, long long groups, bool none, const DropoutArgs a) {
    const long long t = (long long)blockIdx.x * 256 + threadIdx.x, col = t / groups;
    if (col >= ncols) return;
    const int i = (int)(t - col * groups) * 4;
    unsigned word[4];
    draw<4>(a, (unsigned long long)M0 * (unsigned)(i >> 2), a.col0 + col, word);
    const T* src = m.src + col * m.lds + i;
    const T* residual = RESIDUAL ? m.residual + col * m.ldr + i : nullptr;
    float x[4], r[4];
    load_run<T, 4>(src, rows - i, x);
    if (RESIDUAL) load_run<T, 4>(residual, rows - i, r);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float kept = !none && word[e] >= a.least ? x[e] * a.scale : 0.f;
        x[e] = RESIDUAL ? kept + r[e] : kept;
    }
    store_run<T, 4>(m.dst + col * m.ldd + i, rows - i, x);
}

template <class T, bool RESIDUAL>
static int dropout_go(const Streams<T>& m, int rows, int ncols, bool none, const DropoutArgs& a, cudaStream_t st) {
    const auto alike = [&](const T* p, long long ld) {
        return ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(m.dst)) & 15) == 0 && ((ld - m.ldd) * (long long)sizeof(T)) % 16 == 0;
    };
    if (!alike(m.src, m.lds) || (RESIDUAL && !alike(m.residual, m.ldr))) {
        const long long groups = (rows + 3) / 4, blocks = (groups * ncols + 255) / 256;
        if (blocks > 2147483647LL) { set_last_error("dropout: %lld blocks", blocks); return CUVDIA_ERR_UNSUPPORTED; }
        dropout_any_kernel<T, RESIDUAL><<<(unsigned)blocks, 256, 0, st>>>(m, rows, ncols, groups, none, a);
        count_launch();
        return check_launch("dropout_any_kernel");
    }
    constexpr int E = Vec16<T>::N;
    const bool shifted = !columns16(m.dst, m.ldd, sizeof(T));
    const long long vectors = ((long long)rows + E - 1 + (shifted ? E - 1 : 0)) / E, per = shifted ? 3 : 4;
    // As many lanes a part as leave at most an eighth of a column's parts empty, a whole block at best: its vectors lie
    // together and its column is known without a division (16384 x 8192 bf16 with residual: 125 us when this was
    // chosen, parts of a warp each 150 us).  Four vectors a thread (two: 146 us), three where columns are shifted (16383 x 8191:
    // 171 us; two 178, four 195).
    int log_lanes = 0;
    while (log_lanes < 5 && (per << log_lanes) < vectors) log_lanes++;
    if (!shifted)
        for (int k = 6; k <= 8; k++) {
            const long long block = per << k;
            if ((vectors + block - 1) / block * block - vectors <= vectors / 8) log_lanes = k;
        }
    const long long span = (per << log_lanes) - (shifted ? 1 : 0);
    const long long parts = vectors <= per << log_lanes ? 1 : (vectors + span - 1) / span, teams = parts * ncols;
    const long long y = std::min((long long)ncols, 32768LL);
    const long long blocks = log_lanes == 8 ? parts : (teams + (256 >> log_lanes) - 1) >> (8 - log_lanes);
    if (teams > 4294967295LL || blocks > 2147483647LL) { set_last_error("dropout: %lld blocks", blocks); return CUVDIA_ERR_UNSUPPORTED; }
    const dim3 grid((unsigned)blocks, log_lanes == 8 ? (unsigned)y : 1, log_lanes == 8 ? (unsigned)((ncols + y - 1) / y) : 1);
#define DROP_GO(SH, U, W) do {                                                                                                     \
        if (none) dropout_kernel<T, RESIDUAL, SH, true, U, W><<<grid, 256, 0, st>>>(m, rows, ncols, log_lanes, (int)parts, a);      \
        else dropout_kernel<T, RESIDUAL, SH, false, U, W><<<grid, 256, 0, st>>>(m, rows, ncols, log_lanes, (int)parts, a);          \
    } while (0)
    if (shifted) DROP_GO(true, 3, false);
    else if (log_lanes == 8) DROP_GO(false, 4, true);
    else DROP_GO(false, 4, false);
#undef DROP_GO
    count_launch();
    return check_launch("dropout_kernel");
}

int launch_dropout(void* dst, int ldd, const void* src, int lds, const void* residual, int ldr, int type, int rows,
                   int ncols, float p, const DrawParams& d, cudaStream_t st) {
    DropoutArgs a;
    for (int r = 0; r < 10; r++) { a.key0[r] = d.k0 + r * 0x9E3779B9u; a.key1[r] = d.k1 + r * 0xBB67AE85u; }
    a.which = d.which; a.step = d.step; a.col0 = d.col0;
    const bool none = p >= 1.f;
    a.least = none ? 0 : (unsigned)std::ceil((double)p * 16777216.0) << 8;
    a.scale = none ? 0.f : (float)(1.0 / (1.0 - (double)p));
    int rc = CUVDIA_OK;
    CUVDIA_FLOAT_TYPE(type, {
        const Streams<T> m = {(T*)dst, (const T*)src, (const T*)residual, ldd, lds, ldr};
        rc = residual ? dropout_go<T, true>(m, rows, ncols, none, a, st) : dropout_go<T, false>(m, rows, ncols, none, a, st);
    });
    return rc;
}

}  // namespace cuvdia
