// Column lookup by token and the gradient of the table it reads from.
//   lookup    dst[:, j] = scale * table[:, tok_j]
//   gradient  dtable[:, v] = factOld * dtable[:, v] + factNew * sum over the j with tok_j = v, ascending, of dout[:, j]
// A token outside [0, vocab) names no column: the lookup writes zeros for it and the gradient passes over it.
#include "typed.cuh"

namespace cuvdia {

// ---- lookup -----------------------------------------------------------------------------------------------------
// `lanes` threads (a power of two) take a part of a column of dst, U of the 16-byte vectors of the memory it lies in each, `lanes`
// vectors apart, and keep them as they are until they are stored: all loads are in flight before the first store.  Where columns
// do not start on such vectors (ALIGNED = false) a vector's elements straddle two vectors of the table, which are loaded both
// and shifted into place, so that only the ends of a column are moved element by element.
template <class T, bool ALIGNED, bool WIDE>
__global__ void __launch_bounds__(256)
embedding_kernel(T* __restrict__ dst, long long ldd, const T* __restrict__ table, long long ldt, int units, int vocab,
                 const Tokens tokens, int ncols, float scale, int log_lanes, int parts) {
    constexpr int U = ALIGNED ? 4 : 2, E = Vec16<T>::N;
    const int lanes = WIDE ? 256 : 1 << log_lanes, l = threadIdx.x & (lanes - 1);
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
    if (col >= ncols) return;
    const long long tok = tokens[col];
    const bool there = tok >= 0 && tok < vocab;
    const T* from = table + (there ? tok : 0) * ldt;
    T* to = dst + col * ldd;
    const int i0 = (part * lanes * U + l) * E - (ALIGNED ? 0 : behind16(to));
    const int r = ALIGNED ? 0 : behind16(from + i0);            // the same for all of a column's vectors
    uint4 raw[U], more[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int i = i0 + u * lanes * E;
        raw[u] = more[u] = make_uint4(0, 0, 0, 0);
        if (there && i - r >= 0 && i - r + (r ? 2 : 1) * E <= units) {
            raw[u] = __ldg(reinterpret_cast<const uint4*>(from + i - r));
            if (!ALIGNED && r) more[u] = __ldg(reinterpret_cast<const uint4*>(from + i - r) + 1);
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int i = i0 + u * lanes * E;
        if (i >= units) break;
        if (i >= 0 && i + E <= units && (!there || (i - r >= 0 && i - r + (r ? 2 : 1) * E <= units))) {
            if (!ALIGNED) raw[u] = shift16(raw[u], more[u], r * (int)sizeof(T));
            if (scale != 1.f && there) {
                float x[E];
                unpack16<T>(raw[u], x);
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    const float2 y = __fmul2_rn(make_float2(x[e], x[e + 1]), make_float2(scale, scale));
                    x[e] = y.x; x[e + 1] = y.y;
                }
                raw[u] = pack16<T>(x);
            }
            *reinterpret_cast<uint4*>(to + i) = raw[u];
        } else {
#pragma unroll
            for (int e = 0; e < E; e++)
                if (i + e >= 0 && i + e < units) to[i + e] = from_f32<T>(there ? to_f32(from[i + e]) * scale : 0.f);
        }
    }
}

template <class T, bool ALIGNED>
static int embedding_go(T* dst, int ldd, const T* table, int ldt, int units, int vocab, const Tokens& tokens, int ncols,
                        float scale, cudaStream_t st) {
    constexpr long long U = ALIGNED ? 4 : 2;
    const long long e = Vec16<T>::N, runs = ((long long)units + e - 1 + (ALIGNED ? 0 : e - 1)) / e;
    // as in dropout.cu: as many lanes a part as leave at most an eighth of a column's parts empty
    int log_lanes = 0;
    while (log_lanes < 5 && (U << log_lanes) < runs) log_lanes++;
    for (int k = 6; k <= 8; k++) {
        const long long block = U << k;
        if ((runs + block - 1) / block * block - runs <= runs / 8) log_lanes = k;
    }
    const long long span = U << log_lanes, parts = (runs + span - 1) / span, teams = parts * ncols;
    const long long y = std::min((long long)ncols, 32768LL);
    const long long blocks = log_lanes == 8 ? parts : (teams + (256 >> log_lanes) - 1) >> (8 - log_lanes);
    if (teams > 4294967295LL || blocks > 2147483647LL) { set_last_error("embedding: %lld blocks", blocks); return CUVDIA_ERR_UNSUPPORTED; }
    const dim3 grid((unsigned)blocks, log_lanes == 8 ? (unsigned)y : 1, log_lanes == 8 ? (unsigned)((ncols + y - 1) / y) : 1);
    if (log_lanes == 8) embedding_kernel<T, ALIGNED, true><<<grid, 256, 0, st>>>(dst, ldd, table, ldt, units, vocab, tokens, ncols, scale, log_lanes, (int)parts);
    else embedding_kernel<T, ALIGNED, false><<<grid, 256, 0, st>>>(dst, ldd, table, ldt, units, vocab, tokens, ncols, scale, log_lanes, (int)parts);
    count_launch();
    return check_launch("embedding_kernel");
}

int launch_embedding(void* dst, int ldd, const void* table, int ldt, int type, int units, int vocab, const void* tokens,
                     int token_type, int ncols, float scale, cudaStream_t st) {
    const int size = type_size(type);
    const bool aligned = columns16(dst, ldd, size) && columns16(table, ldt, size);
    const Tokens toks = make_tokens(tokens, token_type);
    int rc = CUVDIA_OK;
    CUVDIA_FLOAT_TYPE(type, {
        rc = aligned ? embedding_go<T, true>((T*)dst, ldd, (const T*)table, ldt, units, vocab, toks, ncols, scale, st)
                     : embedding_go<T, false>((T*)dst, ldd, (const T*)table, ldt, units, vocab, toks, ncols, scale, st);
    });
    return rc;
}

// ---- positions sorted by token -----------------------------------------------------------------------------------
// A stable least-significant-digit radix sort of the pairs (token, position), a token that names no column becoming
// `vocab`, the largest key.  Digits of up to 9 bits: two passes for any vocabulary below 2^18.  A pass is three kernels:
// digit counts of every tile of 4096 pairs, one scan over (digit, tile), and the move of each pair to its place.  Equal
// tokens stay in ascending position, so the sums below are taken in the same order on every run.
constexpr int SORT_TILE = 4096, SORT_DIGITS = 512, SORT_THREADS = 256;

__device__ __forceinline__ int sort_key(const Tokens& tokens, long long j, int vocab) {
    const long long t = tokens[j];
    return t >= 0 && t < vocab ? (int)t : vocab;
}

// the pair at place j of the pass's input: the tokens themselves in the first pass
template <bool FIRST>
__device__ __forceinline__ void sort_pair(const Tokens& tokens, const int* keys, const int* pos, int j, int vocab, int& key, int& at) {
    if (FIRST) { key = sort_key(tokens, j, vocab); at = j; }
    else       { key = keys[j]; at = pos[j]; }
}

template <bool FIRST>
__global__ void __launch_bounds__(SORT_THREADS)
sort_count_kernel(const Tokens tokens, const int* __restrict__ keys, int n, int vocab, int shift, int digits,
                  int tiles, int* __restrict__ counts) {
    __shared__ int hist[SORT_DIGITS];
    for (int d = threadIdx.x; d < digits; d += SORT_THREADS) hist[d] = 0;
    __syncthreads();
    const int first = blockIdx.x * SORT_TILE;
    for (int k = threadIdx.x; k < SORT_TILE && k < n - first; k += SORT_THREADS) {
        const int key = FIRST ? sort_key(tokens, first + k, vocab) : keys[first + k];
        atomicAdd(&hist[(key >> shift) & (digits - 1)], 1);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += SORT_THREADS) counts[(long long)d * tiles + blockIdx.x] = hist[d];
}

// exclusive scan of `n` counts in place, one block
__global__ void __launch_bounds__(1024) sort_scan_kernel(int* __restrict__ counts, long long n) {
    __shared__ int warp_sum[32];
    const long long per = (n + 1023) / 1024, first = per * threadIdx.x, last = min(n, first + per);
    int sum = 0;
    for (long long k = first; k < last; k++) sum += counts[k];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int run = sum;
#pragma unroll
    for (int s = 1; s < 32; s *= 2) { const int o = __shfl_up_sync(0xffffffffu, run, s); if (lane >= s) run += o; }
    if (lane == 31) warp_sum[warp] = run;
    __syncthreads();
    if (warp == 0) {
        const int v = warp_sum[lane];
        int r = v;
#pragma unroll
        for (int s = 1; s < 32; s *= 2) { const int o = __shfl_up_sync(0xffffffffu, r, s); if (lane >= s) r += o; }
        warp_sum[lane] = r - v;
    }
    __syncthreads();
    run += warp_sum[warp] - sum;
    for (long long k = first; k < last; k++) { const int v = counts[k]; counts[k] = run; run += v; }
}

template <bool FIRST>
__global__ void __launch_bounds__(SORT_THREADS)
sort_move_kernel(const Tokens tokens, const int* __restrict__ keys, const int* __restrict__ pos, int n, int vocab,
                 int shift, int digits, int tiles, const int* __restrict__ counts, int* __restrict__ keys_out,
                 int* __restrict__ pos_out) {
    constexpr int WARPS = SORT_THREADS / 32, PER = SORT_TILE / SORT_THREADS;
    __shared__ int hist[WARPS][SORT_DIGITS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int d = threadIdx.x; d < WARPS * SORT_DIGITS; d += SORT_THREADS) (&hist[0][0])[d] = 0;
    __syncthreads();
    // each warp ranks its own consecutive pairs, 32 at a time, among the earlier ones of the warp with the same digit
    const int first = blockIdx.x * SORT_TILE + warp * (PER * 32) + lane;
    int key[PER], at[PER], rank[PER];
#pragma unroll
    for (int r = 0; r < PER; r++) {
        const int j = first + r * 32;
        key[r] = at[r] = 0;
        if (j < n) sort_pair<FIRST>(tokens, keys, pos, j, vocab, key[r], at[r]);
    }
#pragma unroll
    for (int r = 0; r < PER; r++) {
        const bool valid = first + r * 32 < n;
        const int digit = valid ? (key[r] >> shift) & (digits - 1) : -1;
        const unsigned peers = __match_any_sync(0xffffffffu, digit);
        rank[r] = valid ? hist[warp][digit] + __popc(peers & ((1u << lane) - 1)) : 0;
        __syncwarp();
        if (valid && (peers >> lane) == 1u) hist[warp][digit] += __popc(peers);       // the highest lane of the digit
        __syncwarp();
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += SORT_THREADS) {
        int run = counts[(long long)d * tiles + blockIdx.x];
#pragma unroll
        for (int w = 0; w < WARPS; w++) { const int v = hist[w][d]; hist[w][d] = run; run += v; }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < PER; r++) {
        if (first + r * 32 >= n) continue;
        const int to = hist[warp][(key[r] >> shift) & (digits - 1)] + rank[r];
        keys_out[to] = key[r];
        pos_out[to] = at[r];
    }
}

// ---- gradient ------------------------------------------------------------------------------------------------------
// The sorted positions are cut into chunks of `len`; a block sums one chunk for one tile of units, in 32 bits and in
// ascending position.  A token whose positions lie inside the chunk is finished here.  One that reaches over a chunk's
// border leaves a partial sum: slot 0 of the chunk if the token began in an earlier one, else slot 1; the second kernel
// adds a token's partial sums in the order of the chunks.
template <class T, class G, int N, bool ALIGNED>
__global__ void __launch_bounds__(256)
embedding_sum_kernel(G* __restrict__ dtable, long long ldt, const T* __restrict__ dout, long long ldo, int units, int vocab,
                     const int* __restrict__ keys, const int* __restrict__ pos, int n, int len, int tiles,
                     float* __restrict__ partial, float fnew, float fold) {
    constexpr int B = 8;                                        // columns in flight
    __shared__ int skey[130], spos[128];
    const long long chunk = blockIdx.x / (unsigned)tiles;
    const int tile = blockIdx.x - (unsigned)chunk * (unsigned)tiles;
    const long long first = chunk * len;
    const int count = (int)min((long long)len, n - first);
    for (int k = threadIdx.x; k < count + 2; k += 256) {        // with the key before and the key after the chunk
        const long long j = first + k - 1;
        skey[k] = j >= 0 && j < n ? keys[j] : -1;
    }
    for (int k = threadIdx.x; k < count; k += 256) spos[k] = pos[first + k];
    __syncthreads();
    const long long u = ((long long)tile * 256 + threadIdx.x) * N;
    const int nu = (int)max(0LL, min((long long)N, units - u));
    float acc[N];
#pragma unroll
    for (int e = 0; e < N; e++) acc[e] = 0.f;
    bool begun_before = skey[1] == skey[0];
    for (int k0 = 0; k0 < count; k0 += B) {
        float x[B][N];
#pragma unroll
        for (int b = 0; b < B; b++) {
            const bool there = k0 + b < count && skey[min(k0 + b, count - 1) + 1] < vocab;
            load_run<T, N, ALIGNED>(dout + (long long)spos[there ? k0 + b : 0] * ldo + u, there ? nu : 0, x[b]);
        }
#pragma unroll
        for (int b = 0; b < B; b++) {
            const int k = k0 + b;
            if (k >= count || skey[k + 1] >= vocab) return;     // the rest names no column
#pragma unroll
            for (int e = 0; e < N; e++) acc[e] += x[b][e];
            const int key = skey[k + 1];
            const bool goes_on = k + 1 == count && skey[k + 2] == key;
            if (skey[k + 2] == key && !goes_on) continue;
            if (!begun_before && !goes_on) {
                G* to = dtable + (long long)key * ldt + u;
                float old[N];
                if (fold != 0.f) load_run<G, N, ALIGNED>(to, nu, old);
#pragma unroll
                for (int e = 0; e < N; e++) acc[e] = fold != 0.f ? fold * old[e] + fnew * acc[e] : fnew * acc[e];
                store_run<G, N, ALIGNED>(to, nu, acc);
            } else {
                float* to = partial + (chunk * 2 + (begun_before ? 0 : 1)) * units + u;
                store_run<float, N, false>(to, nu, acc);
            }
            begun_before = false;
#pragma unroll
            for (int e = 0; e < N; e++) acc[e] = 0.f;
        }
    }
}

template <class G>
__global__ void __launch_bounds__(256)
embedding_join_kernel(G* __restrict__ dtable, long long ldt, int units, int vocab, const int* __restrict__ keys, int n, int len,
                      int tiles, const float* __restrict__ partial, float fnew, float fold) {
    const long long chunk = blockIdx.x / (unsigned)tiles;
    const int tile = blockIdx.x - (unsigned)chunk * (unsigned)tiles;
    const long long first = chunk * len, next = first + len;
    if (next >= n) return;
    const int key = keys[next - 1];
    if (key >= vocab || keys[next] != key) return;                                        // no token reaches over
    if (first > 0 && keys[first] == key && keys[first - 1] == key) return;                // it began in an earlier chunk
    const long long u = (long long)tile * 256 + threadIdx.x;
    if (u >= units) return;
    float acc = partial[(chunk * 2 + 1) * units + u];
    for (long long c = chunk + 1; c * len < n && keys[c * len] == key; c++) acc += partial[c * 2 * units + u];
    G* to = dtable + (long long)key * ldt + u;
    *to = from_f32<G>(fold != 0.f ? fold * to_f32(*to) + fnew * acc : fnew * acc);
}

// The columns of tokens that do not occur: 32 columns a block.
template <class G>
__global__ void __launch_bounds__(256)
embedding_rest_kernel(G* __restrict__ dtable, long long ldt, int units, int vocab, const int* __restrict__ keys, int n,
                      float fold) {
    __shared__ int occurs[32];
    const long long v0 = (long long)blockIdx.x * 32;
    if (threadIdx.x < 32) {
        const long long v = v0 + threadIdx.x;
        int lo = 0, hi = n;                                     // the first place whose key is not below v
        while (lo < hi) { const int mid = lo + (hi - lo) / 2; if (keys[mid] < v) lo = mid + 1; else hi = mid; }
        occurs[threadIdx.x] = v >= vocab || (lo < n && keys[lo] == v);
    }
    __syncthreads();
    for (int c = 0; c < 32; c++) {
        if (occurs[c]) continue;
        G* to = dtable + (v0 + c) * ldt;
        for (long long u = threadIdx.x; u < units; u += 256) to[u] = from_f32<G>(fold == 0.f ? 0.f : fold * to_f32(to[u]));
    }
}

// How the gradient's workspace is laid out, from the sizes alone.
struct GradLayout {
    int bits, passes, digit_bits, tiles, len;
    long long chunks;
    long long keys[2], pos[2], counts, partial, bytes;          // byte offsets
};

static GradLayout grad_layout(int units, int vocab, int ncols) {
    GradLayout g = {};
    while (g.bits < 31 && (vocab >> g.bits) != 0) g.bits++;     // keys 0 .. vocab
    g.passes = (g.bits + 8) / 9;
    g.digit_bits = (g.bits + g.passes - 1) / g.passes;
    g.tiles = (ncols + SORT_TILE - 1) / SORT_TILE;
    // Chunks as long as still leave several blocks for each of the GPU's SMs (a longer chunk leaves fewer partial sums).
    const long long unit_tiles = (units + 1023) / 1024;
    g.len = 128;
    while (g.len > 16 && (ncols / g.len) * unit_tiles < 1024) g.len /= 2;
    g.chunks = ((long long)ncols + g.len - 1) / g.len;
    long long at = 0;
    auto take = [&](long long bytes) { const long long o = at; at += (bytes + 255) / 256 * 256; return o; };
    for (int b = 0; b < 2; b++) { g.keys[b] = take(4LL * ncols); g.pos[b] = take(4LL * ncols); }
    g.counts = take(4LL * SORT_DIGITS * g.tiles);
    g.partial = take(4LL * 2 * g.chunks * units);
    g.bytes = at;
    return g;
}

long long embedding_grad_bytes(int units, int vocab, int ncols) { return ncols > 0 ? grad_layout(units, vocab, ncols).bytes : 0; }

int launch_embedding_grad(void* dtable, int ldt, int grad_type, const void* dout, int ldo, int type, int units, int vocab,
                          const void* tokens, int token_type, int ncols, float fnew, float fold, void* workspace,
                          cudaStream_t st) {
    const GradLayout g = grad_layout(units, vocab, ncols);
    char* ws = (char*)workspace;
    int* keys[2] = {(int*)(ws + g.keys[0]), (int*)(ws + g.keys[1])};
    int* pos[2] = {(int*)(ws + g.pos[0]), (int*)(ws + g.pos[1])};
    int* counts = (int*)(ws + g.counts);
    float* partial = (float*)(ws + g.partial);
    const Tokens toks = make_tokens(tokens, token_type);
    int src = 0;
    for (int p = 0; p < g.passes && ncols > 0; p++) {
        const int shift = p * g.digit_bits, digits = 1 << g.digit_bits;
#define SORT_GO(F) do {                                                                                                  \
        sort_count_kernel<F><<<g.tiles, SORT_THREADS, 0, st>>>(toks, keys[src], ncols, vocab, shift, digits, g.tiles, counts); \
        sort_scan_kernel<<<1, 1024, 0, st>>>(counts, (long long)digits * g.tiles);                                       \
        sort_move_kernel<F><<<g.tiles, SORT_THREADS, 0, st>>>(toks, keys[src], pos[src], ncols, vocab, shift, digits,    \
                                                              g.tiles, counts, keys[1 - src], pos[1 - src]);             \
    } while (0)
        if (p == 0) SORT_GO(true); else SORT_GO(false);
#undef SORT_GO
        count_launch(3);
        int rc = check_launch("sort kernels of embedding_grad");
        if (rc) return rc;
        src = 1 - src;
    }
    if (fold != 1.f) {
        const unsigned blocks = (unsigned)(((long long)vocab + 31) / 32);
        CUVDIA_FLOAT_TYPE(grad_type, (embedding_rest_kernel<T><<<blocks, 256, 0, st>>>((T*)dtable, ldt, units, vocab, keys[src], ncols, fold)));
        count_launch();
        int rc = check_launch("embedding_rest_kernel");
        if (rc) return rc;
    }
    if (ncols == 0) return CUVDIA_OK;
    const bool aligned = columns16(dout, ldo, type_size(type)) && columns16(dtable, ldt, type_size(grad_type));
    const int n = aligned ? 16 / type_size(type) : 1;
    const long long tiles = ((long long)units + 256 * n - 1) / (256 * n), blocks = g.chunks * tiles;
    const long long jtiles = ((long long)units + 255) / 256, jblocks = g.chunks * jtiles;
    if (jblocks > 2147483647LL || blocks > 2147483647LL) { set_last_error("embedding_grad: %lld blocks", jblocks); return CUVDIA_ERR_UNSUPPORTED; }
#define SUM_GO(G, N, A) embedding_sum_kernel<T, G, N, A><<<(unsigned)blocks, 256, 0, st>>>((G*)dtable, ldt, (const T*)dout, ldo, \
    units, vocab, keys[src], pos[src], ncols, g.len, (int)tiles, partial, fnew, fold)
    CUVDIA_FLOAT_TYPE(type, {
        if (grad_type == type) { if (aligned) SUM_GO(T, Vec16<T>::N, true); else SUM_GO(T, 1, false); }
        else { if (aligned) SUM_GO(float, Vec16<T>::N, true); else SUM_GO(float, 1, false); }
    });
#undef SUM_GO
    CUVDIA_FLOAT_TYPE(grad_type, (embedding_join_kernel<T><<<(unsigned)jblocks, 256, 0, st>>>((T*)dtable, ldt, units, vocab,
        keys[src], ncols, g.len, (int)jtiles, partial, fnew, fold)));
    count_launch(2);
    return check_launch("embedding_sum_kernel");
}

}  // namespace cuvdia
