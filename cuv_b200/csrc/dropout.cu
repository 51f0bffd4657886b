// Dropout with the uniform numbers of philox.cuh, drawn in registers:
//   dst = (u >= p ? src / (1 - p) : 0) + residual
// with u the number cuvdia_uniform_f32 gives for the element, so no mask is ever stored: the backward pass is the same
// pass over the gradient, and it draws the same numbers.  u >= p is decided on the generator's 24 bits: u = (word >> 8)
// * 2^-24, hence u >= p exactly if (word >> 8) >= ceil(p * 2^24).
#include <cmath>

#include "philox.cuh"
#include "typed.cuh"

namespace cuvdia {

// A thread owns N consecutive rows, starting at a multiple of four, of one column; `lanes` threads (a power of two) work
// on one column of the block, 256 / lanes columns on one block.
template <class T, int N, bool ALIGNED>
__global__ void __launch_bounds__(256)
dropout_kernel(T* dst, long long ldd, const T* src, long long lds, const T* residual, long long ldr, int rows, int ncols,
               unsigned least, float scale, int lanes, int chunks, const DrawParams d) {
    const unsigned group = blockIdx.x / (unsigned)chunks, chunk = blockIdx.x - group * (unsigned)chunks;
    const int sub = threadIdx.x / lanes, lane = threadIdx.x - sub * lanes;
    const long long col = (long long)group * (256 / lanes) + sub;
    const long long i = ((long long)chunk * lanes + lane) * N;
    if (col >= ncols || i >= rows) return;
    const int n = (int)min((long long)N, rows - i);
    float x[N], r[N];
    load_run<T, N, ALIGNED>(src + col * lds + i, n, x);
    if (residual) load_run<T, N, ALIGNED>(residual + col * ldr + i, n, r);
    const long long gcol = d.col0 + col;
#pragma unroll
    for (int q = 0; q < N / 4; q++) {
        const uint4 w = philox4x32_10(make_uint4((unsigned)(i >> 2) + q, (unsigned)gcol,
                                                 d.which + 65536u * (unsigned)(gcol >> 32), d.step), make_uint2(d.k0, d.k1));
        const unsigned word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float kept = (word[e] >> 8) >= least ? x[4 * q + e] * scale : 0.f;
            x[4 * q + e] = residual ? kept + r[4 * q + e] : kept;
        }
    }
    store_run<T, N, ALIGNED>(dst + col * ldd + i, n, x);
}

int launch_dropout(void* dst, int ldd, const void* src, int lds, const void* residual, int ldr, int type, int rows,
                   int ncols, float p, const DrawParams& d, cudaStream_t st) {
    const int size = type_size(type);
    const bool aligned = columns16(dst, ldd, size) && columns16(src, lds, size) && (!residual || columns16(residual, ldr, size));
    const unsigned least = (unsigned)std::ceil((double)p * 16777216.0);
    const float scale = p < 1.f ? (float)(1.0 / (1.0 - (double)p)) : 0.f;
    const int n = 8;
    const long long items = (rows + n - 1) / n;
    int lanes = 1;
    while (lanes < 256 && lanes < items) lanes *= 2;
    const long long chunks = (items + lanes - 1) / lanes, per = 256 / lanes;
    const long long blocks = (ncols + per - 1) / per * chunks;
    if (blocks > 2147483647LL) { set_last_error("dropout: %lld blocks", blocks); return CUVDIA_ERR_UNSUPPORTED; }
#define DROP_GO(A) CUVDIA_FLOAT_TYPE(type, (dropout_kernel<T, 8, A><<<(unsigned)blocks, 256, 0, st>>>((T*)dst, ldd, (const T*)src, \
    lds, (const T*)residual, ldr, rows, ncols, least, scale, lanes, (int)chunks, d)))
    if (aligned) { DROP_GO(true); } else { DROP_GO(false); }
#undef DROP_GO
    count_launch();
    return check_launch("dropout_kernel");
}

}  // namespace cuvdia
