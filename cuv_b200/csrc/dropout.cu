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

__device__ __forceinline__ uint4 draw_words(const DropoutArgs& a, unsigned group, long long gcol) {
    uint4 c = make_uint4(group, (unsigned)gcol, a.which + 65536u * (unsigned)(gcol >> 32), a.step);
#pragma unroll
    for (int r = 0; r < 10; r++) {
        const unsigned long long p0 = (unsigned long long)0xD2511F53u * c.x, p1 = (unsigned long long)0xCD9E8D57u * c.z;
        c = make_uint4((unsigned)(p1 >> 32) ^ c.y ^ a.key0[r], (unsigned)p1, (unsigned)(p0 >> 32) ^ c.w ^ a.key1[r], (unsigned)p0);
    }
    return c;
}

// A thread owns U runs of N = 8 consecutive rows of one column, `lanes` runs apart (`lanes` threads, a power of two, work on one
// column of the block, 256 / lanes columns on one block); all of its loads are in flight before the first number is drawn.
// NONE: p = 1, every element is dropped.
template <class T, bool RESIDUAL, bool ALIGNED, bool NONE>
__global__ void __launch_bounds__(256)
dropout_kernel(T* dst, long long ldd, const T* src, long long lds, const T* residual, long long ldr, int rows, int ncols,
               int lanes, int chunks, const DropoutArgs a) {
    constexpr int N = 8, U = 2, W = N / Vec16<T>::N;
    const unsigned group = blockIdx.x / (unsigned)chunks, chunk = blockIdx.x - group * (unsigned)chunks;
    const int sub = threadIdx.x / lanes, lane = threadIdx.x - sub * lanes;
    const long long col = (long long)group * (256 / lanes) + sub;
    if (col >= ncols) return;
    const long long gcol = a.col0 + col;
    const T* s = src + col * lds;
    const T* r = RESIDUAL ? residual + col * ldr : nullptr;
    T* d = dst + col * ldd;
    const int i0 = ((int)chunk * U * lanes + lane) * N;
    uint4 xs[U][W], rs[U][W];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int i = i0 + u * lanes * N;
        if (ALIGNED && i + N <= rows) {
#pragma unroll
            for (int w = 0; w < W; w++) {
                xs[u][w] = reinterpret_cast<const uint4*>(s + i)[w];
                if (RESIDUAL) rs[u][w] = reinterpret_cast<const uint4*>(r + i)[w];
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int i = i0 + u * lanes * N;
        if (i >= rows) break;
        const bool whole = ALIGNED && i + N <= rows;
        float x[N], y[N];
        if (whole) {
#pragma unroll
            for (int w = 0; w < W; w++) {
                float v[Vec16<T>::N];
                unpack16<T>(xs[u][w], v);
#pragma unroll
                for (int e = 0; e < Vec16<T>::N; e++) x[w * Vec16<T>::N + e] = v[e];
                if (RESIDUAL) {
                    unpack16<T>(rs[u][w], v);
#pragma unroll
                    for (int e = 0; e < Vec16<T>::N; e++) y[w * Vec16<T>::N + e] = v[e];
                }
            }
        } else {
            load_run<T, N, false>(s + i, rows - i, x);
            if (RESIDUAL) load_run<T, N, false>(r + i, rows - i, y);
        }
#pragma unroll
        for (int q = 0; q < N / 4; q++) {
            const uint4 w = draw_words(a, (unsigned)(i >> 2) + q, gcol);
            const unsigned word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float kept = !NONE && word[e] >= a.least ? x[4 * q + e] * a.scale : 0.f;
                x[4 * q + e] = RESIDUAL ? kept + y[4 * q + e] : kept;
            }
        }
        if (whole) store_run<T, N, true>(d + i, N, x);
        else store_run<T, N, false>(d + i, rows - i, x);
    }
}

template <class T, bool RESIDUAL, bool ALIGNED>
static int dropout_go(void* dst, int ldd, const void* src, int lds, const void* residual, int ldr, int rows, int ncols, bool none,
                      const DropoutArgs& a, cudaStream_t st) {
    constexpr int N = 8, U = 2;
    const long long items = ((long long)rows + U * N - 1) / (U * N);
    int lanes = 1;
    while (lanes < 256 && lanes < items) lanes *= 2;
    const long long chunks = (items + lanes - 1) / lanes, per = 256 / lanes, blocks = (ncols + per - 1) / per * chunks;
    if (blocks > 2147483647LL) { set_last_error("dropout: %lld blocks", blocks); return CUVDIA_ERR_UNSUPPORTED; }
#define DROP_GO(Z) dropout_kernel<T, RESIDUAL, ALIGNED, Z><<<(unsigned)blocks, 256, 0, st>>>((T*)dst, ldd, (const T*)src, lds, \
    (const T*)residual, ldr, rows, ncols, lanes, (int)chunks, a)
    if (none) DROP_GO(true); else DROP_GO(false);
#undef DROP_GO
    count_launch();
    return check_launch("dropout_kernel");
}

int launch_dropout(void* dst, int ldd, const void* src, int lds, const void* residual, int ldr, int type, int rows,
                   int ncols, float p, const DrawParams& d, cudaStream_t st) {
    const int size = type_size(type);
    const bool aligned = columns16(dst, ldd, size) && columns16(src, lds, size) && (!residual || columns16(residual, ldr, size));
    DropoutArgs a;
    for (int r = 0; r < 10; r++) { a.key0[r] = d.k0 + r * 0x9E3779B9u; a.key1[r] = d.k1 + r * 0xBB67AE85u; }
    a.which = d.which; a.step = d.step; a.col0 = d.col0;
    const bool none = p >= 1.f;
    a.least = none ? 0 : (unsigned)std::ceil((double)p * 16777216.0) << 8;
    a.scale = none ? 0.f : (float)(1.0 / (1.0 - (double)p));
    int rc = CUVDIA_OK;
    CUVDIA_FLOAT_TYPE(type, {
        if (residual) rc = aligned ? dropout_go<T, true, true>(dst, ldd, src, lds, residual, ldr, rows, ncols, none, a, st)
                                   : dropout_go<T, true, false>(dst, ldd, src, lds, residual, ldr, rows, ncols, none, a, st);
        else rc = aligned ? dropout_go<T, false, true>(dst, ldd, src, lds, residual, ldr, rows, ncols, none, a, st)
                          : dropout_go<T, false, false>(dst, ldd, src, lds, residual, ldr, rows, ncols, none, a, st);
    });
    return rc;
}

}  // namespace cuvdia
