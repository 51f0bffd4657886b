// Column lookup by token and the gradient of the table it reads from.
//   lookup    dst[:, j] = scale * table[:, tok_j]
//   gradient  dtable[:, v] = factOld * dtable[:, v] + factNew * sum over the j with tok_j = v of dout[:, j]
// A token outside [0, vocab) names no column: the lookup writes zeros for it and the gradient passes over it.
#include "cluster.cuh"
#include "typed.cuh"

namespace cuvdia {

// ---- lookup -----------------------------------------------------------------------------------------------------
// `lanes` threads (a power of two) take a part of a column of dst, U of the 16-byte vectors of the memory it lies in each, `lanes`
// vectors apart, and keep them as they are until they are stored: all loads are in flight before the first store.  Where columns
// do not start on such vectors (ALIGNED = false) a vector's elements straddle two vectors of the table, which are loaded both
// and shifted into place, so that only the ends of a column are moved element by element.  Bound by memory: 4096 x 32768 bf16 from
// a table of 65536 tokens, text-like frequencies, 61 us (5.8 TB/s of columns read once and written); 4095 x 32768 84 us (element
// by element 145 us).  Four vectors a thread (two: 64 us), two where they are shifted (four: 90 us).
template <class T, bool ALIGNED, bool WIDE, bool SPREAD>
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
    // SPREAD: the elements below `front` and from `back` on, which no vector moves, fewer than 4 E, are moved by the last part's
    // threads, one each where there are 32.
    int front = 0, back = 0, ends = 0;
    T end;
    if (SPREAD) {
        const int low = there ? r : 0, high = units - E - (there && r ? E - r : 0), behind = behind16(to);  // first vectors' places
        front = min(units, (low + behind + E - 1) / E * E - behind);
        back = high >= front ? front + ((high - front) / E + 1) * E : front;
        if (part == parts - 1) ends = front + units - back;
        if (l < ends && there) end = from[l < front ? l : back + l - front];
    }
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
        } else if (!SPREAD) {
#pragma unroll
            for (int e = 0; e < E; e++)
                if (i + e >= 0 && i + e < units) to[i + e] = from_f32<T>(there ? to_f32(from[i + e]) * scale : 0.f);
        }
    }
    if (SPREAD) {
        if (l < ends) to[l < front ? l : back + l - front] = from_f32<T>(there ? to_f32(end) * scale : 0.f);
        for (int k = l + lanes; k < ends; k += lanes) {
            const int i = k < front ? k : back + k - front;
            to[i] = from_f32<T>(there ? to_f32(from[i]) * scale : 0.f);
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
#define LOOKUP_GO(W, S) \
    embedding_kernel<T, ALIGNED, W, S><<<grid, 256, 0, st>>>(dst, ldd, table, ldt, units, vocab, tokens, ncols, scale, log_lanes, (int)parts)
    // Shorter 16-bit columns have their ends spread over the threads (333 x 32000 bf16: 14 us, each vector by its own thread
    // 22 us; 1023: 31 and 35 us), which the others do better without (5001 x 32000 bf16: 92 us, spread 100 us; 1023 x 32000 f32:
    // 41 and 45 us).
    constexpr bool ENDS = !ALIGNED && sizeof(T) == 2;
    if (log_lanes == 8) LOOKUP_GO(true, false);
    else if (ENDS && units < 2048) LOOKUP_GO(false, ENDS);
    else LOOKUP_GO(false, false);
#undef LOOKUP_GO
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
// `vocab`, the largest key.  Digits of up to 9 bits: two passes for any vocabulary below 2^18.  Equal tokens stay in
// ascending position, so the sums below are taken in the same order on every run.

__device__ __forceinline__ int sort_key(const Tokens& tokens, long long j, int vocab) {
    const long long t = tokens[j];
    return t >= 0 && t < vocab ? (int)t : vocab;
}

constexpr int SORT_DIGITS = 512;

// the lanes of the warp whose digit is the same, from one vote a bit (65536 positions: 28 us for the sort, 33 us with
// match.any)
__device__ __forceinline__ unsigned same_digit(int digit, int bits) {
    unsigned peers = 0xffffffffu;
#pragma unroll
    for (int b = 0; b < 10; b++) {
        if (b >= bits) break;
        const bool set = digit >> b & 1;
        const unsigned votes = __ballot_sync(0xffffffffu, set);
        peers &= set ? votes : ~votes;
    }
    return peers;
}

// Up to 2^17 positions: one cluster of blocks holds all pairs in registers, 32 R consecutive ones a warp, R a lane, and moves
// them to their places in the blocks' shared memory: one launch, no traffic but tokens in and pairs out.  Per pass a warp ranks
// its pairs among its earlier ones of the same digit; then come the warps before it in the block, the blocks before it in the
// cluster, and the smaller digits.  Bound by latency (barriers, and the scattered stores of the moves): 8 us for up to 8192
// positions, 12 us for 16384, 27 us for 65536, where the three kernels a pass below took 57 us for 16384.
template <int R>
__global__ void __launch_bounds__(1024, 1)
sort_cluster_kernel(const Tokens tokens, int n, int vocab, int passes, int digit_bits, int* __restrict__ keys_out,
                    int* __restrict__ pos_out, int4* __restrict__ joins) {
    constexpr int M = 1024 * R;
    launch_dependents();                                        // whose first blocks need nothing from here
    extern __shared__ unsigned long long pairs[];               // M pairs, then the warps' digit counts, then two rows of digits
    unsigned short (*hist)[SORT_DIGITS] = reinterpret_cast<unsigned short (*)[SORT_DIGITS]>(pairs + M);
    int* total = reinterpret_cast<int*>(hist + 32);
    int* base = total + SORT_DIGITS;
    __shared__ int warp_sum[16];
    unsigned rank_in, ranks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank_in));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, digits = 1 << digit_bits;
    const int g0 = (int)rank_in * M + warp * (32 * R) + lane;
    if (rank_in == 0 && threadIdx.x == 0) joins[0] = make_int4(0, 0, 0, 0);
    int key[R], pos[R], place[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        pos[r] = g0 + r * 32;
        key[r] = pos[r] < n ? sort_key(tokens, pos[r], vocab) : vocab;          // what fills up the last block stays behind
    }
    for (int pass = 0; pass < passes; pass++) {
        const int shift = pass * digit_bits;
        for (int d = lane; d < SORT_DIGITS / 2; d += 32) reinterpret_cast<unsigned*>(hist[warp])[d] = 0;
        __syncwarp();
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int digit = (key[r] >> shift) & (digits - 1);
            const unsigned peers = same_digit(digit, digit_bits);
            const int before = hist[warp][digit];
            place[r] = before + __popc(peers & ((1u << lane) - 1));
            __syncwarp();
            if ((peers >> lane) == 1u) hist[warp][digit] = (unsigned short)(before + __popc(peers));     // its highest lane
            __syncwarp();
        }
        __syncthreads();
        if ((int)threadIdx.x < digits) {
            int run = 0;
#pragma unroll 8
            for (int w = 0; w < 32; w++) { const int v = hist[w][threadIdx.x]; hist[w][threadIdx.x] = (unsigned short)run; run += v; }
            total[threadIdx.x] = run;
        }
        cluster_arrive();
        cluster_wait();
        int all = 0, below = 0;
        if ((int)threadIdx.x < digits) {
            int v[8];                                           // all on their way before the first is added
#pragma unroll
            for (unsigned c = 0; c < 8; c++) {
                v[c] = 0;
                if (c < ranks) asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v[c]) : "r"(in_block(total + threadIdx.x, c)) : "memory");
            }
#pragma unroll
            for (unsigned c = 0; c < 8; c++) { all += v[c]; if (c < rank_in) below += v[c]; }
        }
        const bool last = pass + 1 == passes;
        if (last) cluster_arrive();                             // this block's reads of the others' counts are done: they may leave
        if (warp < 16) {                                        // exclusive scan over the digits
            int run = all;
#pragma unroll
            for (int s = 1; s < 32; s *= 2) { const int o = __shfl_up_sync(0xffffffffu, run, s); if (lane >= s) run += o; }
            if (lane == 31) warp_sum[warp] = run;
            all = run - all;
        }
        __syncthreads();
        if ((int)threadIdx.x < digits) {
            for (int w = 0; w < warp; w++) all += warp_sum[w];
            base[threadIdx.x] = all + below;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int digit = (key[r] >> shift) & (digits - 1), to = base[digit] + hist[warp][digit] + place[r];
            if (!last) {
                asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(in_block(pairs + to % M, to / M)),
                             "l"((unsigned long long)(unsigned)key[r] << 32 | (unsigned)pos[r]) : "memory");
            } else if (to < n) {
                keys_out[to] = key[r];
                pos_out[to] = pos[r];
            }
        }
        if (last) break;
        cluster_arrive();
        cluster_wait();
#pragma unroll
        for (int r = 0; r < R; r++) {
            const unsigned long long p = pairs[warp * (32 * R) + r * 32 + lane];
            key[r] = (int)(p >> 32); pos[r] = (int)(unsigned)p;
        }
    }
    cluster_wait();                                             // a block's counts stay until the others have read them
}

template <int R>
static int sort_cluster(int blocks, const Tokens& tokens, int n, int vocab, int passes, int digit_bits, int* keys, int* pos,
                        int4* joins, cudaStream_t st) {
    static bool done[64] = {false};
    const size_t bytes = 1024 * R * 8 + 32 * SORT_DIGITS * 2 + 2 * SORT_DIGITS * 4;
    int rc = allow_dynamic_smem(sort_cluster_kernel<R>, bytes, done);
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(1024);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = st;
    cudaLaunchAttribute cluster;
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = blocks; cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    cfg.attrs = &cluster;
    cfg.numAttrs = 1;
    CUVDIA_CUDA(cudaLaunchKernelEx(&cfg, sort_cluster_kernel<R>, tokens, n, vocab, passes, digit_bits, keys, pos, joins));
    count_launch();
    return check_launch("sort_cluster_kernel");
}

// More positions: a pass is three kernels - digit counts of every tile of 4096 pairs, one scan over (digit, tile), and the
// move of each pair to its place.
constexpr int SORT_TILE = 4096, SORT_THREADS = 256;

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
__global__ void __launch_bounds__(1024) sort_scan_kernel(int* __restrict__ counts, long long n, int4* __restrict__ joins) {
    __shared__ int warp_sum[32];
    if (threadIdx.x == 0) joins[0] = make_int4(0, 0, 0, 0);
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
                 int shift, int digit_bits, int tiles, const int* __restrict__ counts, int* __restrict__ keys_out,
                 int* __restrict__ pos_out) {
    const int digits = 1 << digit_bits;
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
        const unsigned peers = same_digit(valid ? digit : digits, digit_bits + 1);       // a digit of its own for what is not there
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
// The sorted positions are cut into chunks of 32; a warp sums one chunk for 256 units, in 32 bits and in ascending position,
// eight columns in flight.  A token whose positions lie inside the chunk is finished here.  One that reaches over a chunk's
// border leaves a partial sum: slot 0 of the chunk if the token began in an earlier one, else slot 1; the second kernel adds a
// token's partial sums, in the order of the chunks or of a fixed split of them.  Behind the blocks that sum come those that
// write the columns of tokens that do not occur, 32 columns each: stores that fill the memory's time between the loads.
// Bound by memory but for the joins and what the sums' launch does not hide of the sort: 4096 x 32768 f32 from 16384 bf16 columns
// 129 us (103 us of traffic), 1024 x 131072 from 8192 bf16 57 us (44 us).  Columns off 16-byte boundaries go element by element:
// 4095 x 32768 149 us.  factOld = 1 saves the absent columns and reads the others, in the middle of the sums: 96 us (47 us of
// traffic), but 1023 x 50021 from 8191 f32 132 us (with factOld = 0 59 us).  Longer chunks leave fewer partial sums but too few
// warps: with blocks that sum 64 columns each the first took 237 us.

constexpr int LONG_JOIN = 8;            // more partial sums than this are shared out among a block's warps

// the eight units of a lane: two runs of four consecutive ones, one of eight, or single ones 32 apart
template <class T, bool ALIGNED>
__device__ __forceinline__ int lane_unit(int slice, int e) {
    const int lane = threadIdx.x & 31;
    return slice * 256 + (!ALIGNED ? e * 32 + lane : sizeof(T) == 4 ? (e / 4) * 128 + lane * 4 + e % 4 : lane * 8 + e);
}

// x[e] of the units of a lane to or from a column of C; `units` of them exist.  T lays the lane's units out (see above).
template <class T, class C, bool ALIGNED>
__device__ __forceinline__ void store_units(C* to, int slice, int units, const float (&x)[8]) {
    if constexpr (ALIGNED) {
#pragma unroll
        for (int g = 0; g < 2; g++) {
            const int u = lane_unit<T, true>(slice, 4 * g);
            if (u + 4 <= units) {
                if constexpr (sizeof(C) == 4) *reinterpret_cast<float4*>(to + u) = make_float4(x[4 * g], x[4 * g + 1], x[4 * g + 2], x[4 * g + 3]);
                else *reinterpret_cast<uint2*>(to + u) = make_uint2(pack2<C>(x[4 * g], x[4 * g + 1]), pack2<C>(x[4 * g + 2], x[4 * g + 3]));
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) if (u + e < units) to[u + e] = from_f32<C>(x[4 * g + e]);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int u = lane_unit<T, false>(slice, e);
            if (u < units) to[u] = from_f32<C>(x[e]);
        }
    }
}

// A lane's part of a column on its way: as it is in memory (16-byte vectors), or converted (single elements)
template <class T, bool ALIGNED> struct Part;
template <class T> struct Part<T, true> {
    uint4 v[sizeof(T) == 4 ? 2 : 1];
    __device__ __forceinline__ void load(const T* from, int slice, int units) {
        constexpr int E = Vec16<T>::N;
#pragma unroll
        for (int g = 0; g < 8 / E; g++) {
            const int u = lane_unit<T, true>(slice, g * E);
            if (u + E <= units) v[g] = __ldg(reinterpret_cast<const uint4*>(from + u));
            else {
                float x[E];
                load_run<T, E>(from + u, max(0, units - u), x);
                v[g] = pack16<T>(x);
            }
        }
    }
    __device__ __forceinline__ void add_to(float (&acc)[8]) const {
        constexpr int E = Vec16<T>::N;
#pragma unroll
        for (int g = 0; g < 8 / E; g++) {
            float x[E];
            unpack16<T>(v[g], x);
#pragma unroll
            for (int e = 0; e < E; e++) acc[g * E + e] += x[e];
        }
    }
};
template <class T> struct Part<T, false> {
    T v[8];
    __device__ __forceinline__ void load(const T* from, int slice, int units) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int u = lane_unit<T, false>(slice, e);
            v[e] = u < units ? from[u] : from_f32<T>(0.f);
        }
    }
    __device__ __forceinline__ void add_to(float (&acc)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; e++) acc[e] += to_f32(v[e]);
    }
};

template <class G>
struct GradOut {
    G* dtable; long long ldt;
    int units, vocab;
    const int* keys; const int* pos; int n;
    Tokens tokens;
    float* partial; int pitch;                                  // two rows of `pitch` floats a chunk
    int4* joins; int chunks;                                    // {numbers of short and long joins}, then {chunk, token, chunks after
                                                                // this one that begin with the token} from both ends
    float fnew, fold;
};

template <class T, class G, bool ALIGNED>
__device__ __forceinline__ void finish_column(const GradOut<G>& o, int key, int slice, float (&acc)[8]) {
    G* to = o.dtable + key * o.ldt;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int u = lane_unit<T, ALIGNED>(slice, e);
        acc[e] *= o.fnew;
        if (o.fold != 0.f && u < o.units) acc[e] = o.fold * to_f32(to[u]) + acc[e];
    }
    store_units<T, G, ALIGNED>(to, slice, o.units, acc);
}

// The columns of 32 tokens that do not occur: zeroed or scaled by a block.  Which ones these are it finds in the sorted keys, or,
// while they are still being sorted (LOOK), by a look through all tokens.
template <bool LOOK, class G>
__device__ __forceinline__ void rest_columns(const GradOut<G>& o, long long v0, int* occurs) {
    if (threadIdx.x < 32) {
        const long long v = v0 + threadIdx.x;
        bool there = v >= o.vocab;
        if (!LOOK) {
            int lo = 0, hi = o.n;                               // the first place whose key is not below v
            while (lo < hi) { const int mid = lo + (hi - lo) / 2; if (o.keys[mid] < v) lo = mid + 1; else hi = mid; }
            there = there || (lo < o.n && o.keys[lo] == v);
        }
        occurs[threadIdx.x] = there;
    }
    if (LOOK) {
        __syncthreads();
#pragma unroll 8
        for (int j = threadIdx.x; j < o.n; j += 256) {
            const long long t = o.tokens[j] - v0;
            if (t >= 0 && t < 32) occurs[t] = 1;
        }
    }
    __syncthreads();
    // a warp a column: a whole block would be half empty on short ones
    const int lane = threadIdx.x & 31;
    for (int c = threadIdx.x >> 5; c < 32; c += 8) {
        if (occurs[c]) continue;
        G* to = o.dtable + (v0 + c) * o.ldt;
        if (o.fold != 0.f) {
#pragma unroll 4
            for (int u = lane; u < o.units; u += 32) to[u] = from_f32<G>(o.fold * to_f32(to[u]));
            continue;
        }
        const int head = min(o.units, (int)((16 - (reinterpret_cast<uintptr_t>(to) & 15)) % 16 / sizeof(G)));
        const int nvec = (o.units - head) / Vec16<G>::N, tail = head + nvec * Vec16<G>::N;
        uint4* v = reinterpret_cast<uint4*>(to + head);
#pragma unroll 4
        for (int k = lane; k < nvec; k += 32) v[k] = make_uint4(0, 0, 0, 0);
        if (lane < head) to[lane] = from_f32<G>(0.f);
        if (lane < o.units - tail) to[tail + lane] = from_f32<G>(0.f);
    }
}

template <class T, class G, bool ALIGNED>
__global__ void __launch_bounds__(256)
embedding_sum_kernel(const GradOut<G> o, const T* __restrict__ dout, long long ldo, unsigned look_blocks, unsigned sum_blocks,
                     int slices) {
    constexpr int B = 8;
    __shared__ int occurs[32];
    if (blockIdx.x < look_blocks) { rest_columns<true>(o, (long long)blockIdx.x * 32, occurs); return; }
    wait_for_dependencies();
    if (blockIdx.x >= look_blocks + sum_blocks) { rest_columns<false>(o, (long long)(blockIdx.x - sum_blocks) * 32, occurs); return; }
    const long long item = (long long)(blockIdx.x - look_blocks) * 8 + (threadIdx.x >> 5);
    const long long chunk = item / slices;
    const int slice = (int)(item - chunk * slices), lane = threadIdx.x & 31;
    const long long first = chunk * 32;
    if (first >= o.n) return;
    const int key = first + lane < o.n ? o.keys[first + lane] : o.vocab, at = first + lane < o.n ? o.pos[first + lane] : 0;
    const int count = __popc(__ballot_sync(0xffffffffu, key < o.vocab));          // the rest names no column
    if (count == 0) return;
    int after = __shfl_down_sync(0xffffffffu, key, 1);
    if (lane == 31) after = first + 32 < o.n ? o.keys[first + 32] : o.vocab;
    const unsigned ends = __ballot_sync(0xffffffffu, key != after);
    bool begun_before = first > 0 && __shfl_sync(0xffffffffu, key, 0) == o.keys[first - 1];
    float acc[8];
#pragma unroll
    for (int e = 0; e < 8; e++) acc[e] = 0.f;
    for (int k0 = 0; k0 < count; k0 += B) {
        Part<T, ALIGNED> part[B];
#pragma unroll
        for (int b = 0; b < B; b++) {
            const long long j = __shfl_sync(0xffffffffu, at, (k0 + b) & 31);
            if (k0 + b < count) part[b].load(dout + j * ldo, slice, o.units);
        }
#pragma unroll
        for (int b = 0; b < B; b++) {
            if (k0 + b >= count) break;
            part[b].add_to(acc);
            if (!(ends >> (k0 + b) & 1)) continue;
            if (begun_before) store_units<T, float, ALIGNED>(o.partial + chunk * 2 * o.pitch, slice, o.units, acc);
            else finish_column<T, G, ALIGNED>(o, __shfl_sync(0xffffffffu, key, k0 + b), slice, acc);
            begun_before = false;
#pragma unroll
            for (int e = 0; e < 8; e++) acc[e] = 0.f;
        }
    }
    if (ends >> (count - 1) & 1) return;
    store_units<T, float, ALIGNED>(o.partial + (chunk * 2 + (begun_before ? 0 : 1)) * o.pitch, slice, o.units, acc);
    if (begun_before || slice != 0) return;
    const int token = __shfl_sync(0xffffffffu, key, 31);        // this chunk's last token is to be joined
    int more = 0;
    for (;;) {
        const long long c = (chunk + 1 + more + lane) * 32;
        const unsigned same = __ballot_sync(0xffffffffu, c < o.n && o.keys[c] == token);
        if (same != 0xffffffffu) { more += __ffs(~same) - 1; break; }
        more += 32;
    }
    if (lane == 0) {
        const bool is_long = more > LONG_JOIN;
        const int place = atomicAdd(reinterpret_cast<int*>(o.joins) + is_long, 1);
        o.joins[1 + (is_long ? o.chunks - 1 - place : place)] = make_int4((int)chunk, token, more, 0);
    }
}

// Adds up the partial sums of the tokens that reach over a chunk's end, from the list of the chunks where they begin (the list's
// order changes nothing: every sum has its own place).  128 units at a time, by one warp, or by a block whose warps share out the
// partial sums where they are many.
template <class G>
__global__ void __launch_bounds__(256)
embedding_join_kernel(const GradOut<G> o) {
    __shared__ float4 shares[8][32];
    wait_for_dependencies();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, slices = (o.units + 127) / 128;
    auto add = [](float4& acc, const float4& x) { acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w; };
    auto finish = [&](int key, int u, const float4& acc) {
        G* to = o.dtable + key * o.ldt;
        const float x[4] = {acc.x, acc.y, acc.z, acc.w};
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (u + e < o.units) to[u + e] = from_f32<G>(o.fold != 0.f ? o.fold * to_f32(to[u + e]) + o.fnew * x[e] : o.fnew * x[e]);
    };
    const int4 numbers = o.joins[0];
    const long long n_long = (long long)numbers.y * slices, n_short = (long long)numbers.x * slices;
    for (long long item = blockIdx.x; item < n_long; item += gridDim.x) {
        const int4 join = o.joins[o.chunks - (int)(item / slices)];
        const int u = (int)(item % slices) * 128 + lane * 4, more = join.z;
        const float* row = o.partial + ((long long)join.x * 2 + 2) * o.pitch + u;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        if (u < o.pitch) {
            if (warp == 0) add(acc, *reinterpret_cast<const float4*>(row - o.pitch));
            const int end = (int)((long long)more * (warp + 1) / 8);
#pragma unroll 8
            for (int c = (int)((long long)more * warp / 8); c < end; c++) add(acc, *reinterpret_cast<const float4*>(row + (long long)c * 2 * o.pitch));
        }
        __syncthreads();
        shares[warp][lane] = acc;
        __syncthreads();
        if (warp == 0) {
            for (int w = 1; w < 8; w++) add(acc, shares[w][lane]);
            finish(join.y, u, acc);
        }
    }
    for (long long item = (long long)blockIdx.x * 8 + warp; item < n_short; item += (long long)gridDim.x * 8) {
        const int4 join = o.joins[1 + (int)(item / slices)];
        const int u = (int)(item % slices) * 128 + lane * 4, more = join.z;
        const float* row = o.partial + ((long long)join.x * 2 + 2) * o.pitch + u;
        if (u >= o.pitch) continue;
        float4 acc = *reinterpret_cast<const float4*>(row - o.pitch);
#pragma unroll 8
        for (int c = 0; c < more; c++) add(acc, *reinterpret_cast<const float4*>(row + (long long)c * 2 * o.pitch));
        finish(join.y, u, acc);
    }
}

// ---- few positions ---------------------------------------------------------------------------------------------------------
// With at most SMALL positions nothing is sorted: a warp takes one position for 256 units, leaves if its token occurs earlier too,
// and else adds up the columns of all positions of that token, in ascending order; the absent columns are written beside it.  One
// launch and no workspace, bound by latency or by the absent columns' stores: 256 x 1000 from 64 f32 columns 6 us (sorted 18.5 us),
// 512 x 1000 from 200 bf16 columns 9 us (21 us), 1023 x 50021 from 200 f32 columns 35 us (45 us); 256 positions of one and the same
// token, which a single warp adds up, 35 us (14 us), hence no more than that.
constexpr int SMALL = 256;

template <class T, class G, bool ALIGNED>
__global__ void __launch_bounds__(256)
embedding_small_kernel(const GradOut<G> o, const T* __restrict__ dout, long long ldo, unsigned sum_blocks, int slices) {
    constexpr int B = 8;
    __shared__ int occurs[32];
    if (blockIdx.x >= sum_blocks) { rest_columns<true>(o, (long long)(blockIdx.x - sum_blocks) * 32, occurs); return; }
    const unsigned item = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int j = (int)(item / (unsigned)slices), slice = (int)(item - (unsigned)j * (unsigned)slices);
    if (j >= o.n) return;
    const long long token = o.tokens[j];
    if (token < 0 || token >= o.vocab) return;
    unsigned same[SMALL / 32], earlier = 0;
#pragma unroll
    for (int k = 0; k < SMALL / 32; k++) {
        const int i = k * 32 + (int)lane;
        same[k] = __ballot_sync(0xffffffffu, i < o.n && o.tokens[i] == token);
        earlier |= k < j / 32 ? same[k] : k == j / 32 ? same[k] & ((1u << j % 32) - 1) : 0;
    }
    if (earlier) return;
    float acc[8];
#pragma unroll
    for (int e = 0; e < 8; e++) acc[e] = 0.f;
#pragma unroll
    for (int k = 0; k < SMALL / 32; k++) {
        unsigned mine = same[k];
        while (mine) {
            Part<T, ALIGNED> part[B];
            const int count = min(B, __popc(mine));
#pragma unroll
            for (int b = 0; b < B; b++)
                if (b < count) {
                    part[b].load(dout + (long long)(k * 32 + __ffs(mine) - 1) * ldo, slice, o.units);
                    mine &= mine - 1;
                }
#pragma unroll
            for (int b = 0; b < B; b++) if (b < count) part[b].add_to(acc);
        }
    }
    finish_column<T, G, ALIGNED>(o, (int)token, slice, acc);
}

// How the gradient's workspace is laid out, from the sizes alone.
struct GradLayout {
    int bits, passes, digit_bits, tiles, pitch;
    bool cluster;
    long long chunks;
    long long keys[2], pos[2], counts, joins, partial, bytes;          // byte offsets
};

static GradLayout grad_layout(int units, int vocab, int ncols) {
    GradLayout g = {};
    while (g.bits < 31 && (vocab >> g.bits) != 0) g.bits++;     // keys 0 .. vocab
    g.passes = (g.bits + 8) / 9;
    g.digit_bits = (g.bits + g.passes - 1) / g.passes;
    g.tiles = (ncols + SORT_TILE - 1) / SORT_TILE;
    g.cluster = ncols <= 131072;
    g.chunks = ((long long)ncols + 31) / 32;
    g.pitch = (int)std::min((units + 3LL) / 4 * 4, 2147483644LL);
    long long at = 0;
    auto take = [&](long long bytes) { const long long o = at; at += (bytes + 255) / 256 * 256; return o; };
    g.keys[0] = take(4LL * ncols);
    g.pos[0] = take(4LL * ncols);
    if (!g.cluster) {
        g.keys[1] = take(4LL * ncols);
        g.pos[1] = take(4LL * ncols);
        g.counts = take(4LL * SORT_DIGITS * g.tiles);
    }
    g.joins = take(16LL * (1 + g.chunks));
    g.partial = take(4LL * 2 * g.chunks * g.pitch);
    g.bytes = at;
    return g;
}

long long embedding_grad_bytes(int units, int vocab, int ncols) { return ncols > SMALL ? grad_layout(units, vocab, ncols).bytes : 0; }

int launch_embedding_grad(void* dtable, int ldt, int grad_type, const void* dout, int ldo, int type, int units, int vocab,
                          const void* tokens, int token_type, int ncols, float fnew, float fold, void* workspace,
                          cudaStream_t st) {
    const bool aligned = (ncols == 0 || columns16(dout, ldo, type_size(type))) && columns16(dtable, ldt, type_size(grad_type));
    const Tokens toks = make_tokens(tokens, token_type);
    const long long slices = ((long long)units + 255) / 256;
    if (ncols <= SMALL) {
        const long long sums = (ncols * slices + 7) / 8, blocks = sums + (fold != 1.f ? ((long long)vocab + 31) / 32 : 0);
        if (blocks > 2147483647LL) { set_last_error("embedding_grad: %lld blocks", blocks); return CUVDIA_ERR_UNSUPPORTED; }
        if (blocks == 0) return CUVDIA_OK;
#define SMALL_GO(G, A) do {                                                                                              \
        const GradOut<G> o = {(G*)dtable, ldt, units, vocab, nullptr, nullptr, ncols, toks, nullptr, 0, nullptr, 0, fnew, fold}; \
        embedding_small_kernel<T, G, A><<<(unsigned)blocks, 256, 0, st>>>(o, (const T*)dout, ldo, (unsigned)sums, (int)slices); \
    } while (0)
        CUVDIA_FLOAT_TYPE(type, {
            if (grad_type == type) { if (aligned) SMALL_GO(T, true); else SMALL_GO(T, false); }
            else { if (aligned) SMALL_GO(float, true); else SMALL_GO(float, false); }
        });
#undef SMALL_GO
        count_launch();
        return check_launch("embedding_small_kernel");
    }
    const GradLayout g = grad_layout(units, vocab, ncols);
    char* ws = (char*)workspace;
    int* keys[2] = {(int*)(ws + g.keys[0]), (int*)(ws + g.keys[1])};
    int* pos[2] = {(int*)(ws + g.pos[0]), (int*)(ws + g.pos[1])};
    int* counts = (int*)(ws + g.counts);
    int4* joins = (int4*)(ws + g.joins);
    int src = 0, rc = CUVDIA_OK;
    if (g.cluster) {
        int blocks = 1, r = 1;
        while (blocks < 8 && blocks * 1024 < ncols) blocks *= 2;
        while (blocks * 1024 * r < ncols) r *= 2;
        switch (r) {
            case 1: rc = sort_cluster<1>(blocks, toks, ncols, vocab, g.passes, g.digit_bits, keys[0], pos[0], joins, st); break;
            case 2: rc = sort_cluster<2>(blocks, toks, ncols, vocab, g.passes, g.digit_bits, keys[0], pos[0], joins, st); break;
            case 4: rc = sort_cluster<4>(blocks, toks, ncols, vocab, g.passes, g.digit_bits, keys[0], pos[0], joins, st); break;
            case 8: rc = sort_cluster<8>(blocks, toks, ncols, vocab, g.passes, g.digit_bits, keys[0], pos[0], joins, st); break;
            default: rc = sort_cluster<16>(blocks, toks, ncols, vocab, g.passes, g.digit_bits, keys[0], pos[0], joins, st); break;
        }
        if (rc) return rc;
    }
    for (int p = 0; p < g.passes && !g.cluster; p++) {
        const int shift = p * g.digit_bits, digits = 1 << g.digit_bits;
#define SORT_GO(F) do {                                                                                                  \
        sort_count_kernel<F><<<g.tiles, SORT_THREADS, 0, st>>>(toks, keys[src], ncols, vocab, shift, digits, g.tiles, counts); \
        sort_scan_kernel<<<1, 1024, 0, st>>>(counts, (long long)digits * g.tiles, joins);                                \
        sort_move_kernel<F><<<g.tiles, SORT_THREADS, 0, st>>>(toks, keys[src], pos[src], ncols, vocab, shift, g.digit_bits, \
                                                              g.tiles, counts, keys[1 - src], pos[1 - src]);             \
    } while (0)
        if (p == 0) SORT_GO(true); else SORT_GO(false);
#undef SORT_GO
        count_launch(3);
        rc = check_launch("sort kernels of embedding_grad");
        if (rc) return rc;
        src = 1 - src;
    }
    const long long sum_blocks = (g.chunks * slices + 7) / 8;
    const long long rest_blocks = fold != 1.f ? ((long long)vocab + 31) / 32 : 0, column = (long long)units * type_size(grad_type);
    // The first columns of absent tokens are written while the tokens are still being sorted, as many as that takes (some 128 MB), by
    // blocks that look through the tokens themselves where that is little against what they write.  (Only the sort may still be
    // running then: it is an ordinary launch, so what came before it in the stream has ended.)
    const long long look_blocks = g.cluster && 8LL * ncols <= 64 * column ? std::min(rest_blocks, (128LL << 20) / (32 * column)) : 0;
    if (sum_blocks + rest_blocks > 2147483647LL) { set_last_error("embedding_grad: %lld blocks", sum_blocks + rest_blocks); return CUVDIA_ERR_UNSUPPORTED; }
#define GRAD_OUT(G) {(G*)dtable, ldt, units, vocab, keys[src], pos[src], ncols, toks, (float*)(ws + g.partial), g.pitch, joins, (int)g.chunks, fnew, fold}
#define SUM_GO(G, A) do {                                                                                                \
        const GradOut<G> o = GRAD_OUT(G);                                                                                \
        rc = launch_dependent(embedding_sum_kernel<T, G, A>, (unsigned)(sum_blocks + rest_blocks), 256, st, o, (const T*)dout, \
                              (long long)ldo, (unsigned)look_blocks, (unsigned)sum_blocks, (int)slices);                 \
    } while (0)
    CUVDIA_FLOAT_TYPE(type, {
        if (grad_type == type) { if (aligned) SUM_GO(T, true); else SUM_GO(T, false); }
        else { if (aligned) SUM_GO(float, true); else SUM_GO(float, false); }
    });
    if (rc) return rc;
    count_launch();
    rc = check_launch("embedding_sum_kernel");
    if (rc) return rc;
    const unsigned join_blocks = (unsigned)std::min((g.chunks - 1) * (((long long)units + 127) / 128), 6LL * sm_count());
    CUVDIA_FLOAT_TYPE(grad_type, {
        const GradOut<T> o = GRAD_OUT(T);
        rc = launch_dependent(embedding_join_kernel<T>, join_blocks, 256, st, o);
    });
#undef SUM_GO
#undef GRAD_OUT
    if (rc) return rc;
    count_launch();
    return check_launch("embedding_join_kernel");
}

}  // namespace cuvdia
