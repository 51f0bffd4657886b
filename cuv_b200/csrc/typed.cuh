// Element types of the token-model operators (fp32, fp16, bf16): conversion to and from the fp32 that everything is
// computed in, and 16-byte vectors of them.  A store rounds once, to nearest even.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "cuvdia_internal.cuh"

namespace cuvdia {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

template <class T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// two packed 16-bit elements <-> two floats
template <class T> __device__ __forceinline__ float2 unpack2(unsigned w);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(unsigned w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(unsigned w) {
    __half2 h;
    *reinterpret_cast<unsigned*>(&h) = w;
    return __half22float2(h);
}
template <class T> __device__ __forceinline__ unsigned pack2(float a, float b);
template <> __device__ __forceinline__ unsigned pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&h);
}
template <> __device__ __forceinline__ unsigned pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&h);
}

// 16 bytes of T
template <class T> struct Vec16 { static constexpr int N = 16 / (int)sizeof(T); };

template <class T>
__device__ __forceinline__ void unpack16(const uint4& r, float (&x)[Vec16<T>::N]) {
    if constexpr (sizeof(T) == 4) {
        x[0] = __uint_as_float(r.x); x[1] = __uint_as_float(r.y); x[2] = __uint_as_float(r.z); x[3] = __uint_as_float(r.w);
    } else {
        const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const float2 f = unpack2<T>(w[q]);
            x[2 * q] = f.x; x[2 * q + 1] = f.y;
        }
    }
}

template <class T>
__device__ __forceinline__ uint4 pack16(const float (&x)[Vec16<T>::N]) {
    if constexpr (sizeof(T) == 4) {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    } else {
        return make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
    }
}

// 16 bytes into shared memory without a register on the way (both addresses 16-byte aligned).  A thread may read what it
// copied itself once copies_wait<n> has returned: all of its groups of copies but the n youngest are complete then.
__device__ __forceinline__ void copy_async16(void* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }

// up to N consecutive elements at p, element by element: the first n of them, zero for the rest
template <class T, int N>
__device__ __forceinline__ void load_run(const T* p, int n, float (&x)[N]) {
#pragma unroll
    for (int e = 0; e < N; e++) x[e] = e < n ? to_f32(p[e]) : 0.f;
}

template <class T, int N>
__device__ __forceinline__ void store_run(T* p, int n, const float (&x)[N]) {
#pragma unroll
    for (int e = 0; e < N; e++) if (e < n) p[e] = from_f32<T>(x[e]);
}

// The 16 bytes that begin `bytes` (0 .. 15, whole elements) behind the start of a, where b follows a in memory.
__device__ __forceinline__ uint4 shift16(const uint4& a, const uint4& b, int bytes) {
    const unsigned w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    unsigned t[6], u[5];
#pragma unroll
    for (int k = 0; k < 6; k++) t[k] = bytes & 8 ? w[k + 2] : w[k];
#pragma unroll
    for (int k = 0; k < 5; k++) u[k] = bytes & 4 ? t[k + 1] : t[k];
    const int bits = (bytes & 3) * 8;
    return make_uint4(__funnelshift_r(u[0], u[1], bits), __funnelshift_r(u[1], u[2], bits), __funnelshift_r(u[2], u[3], bits),
                      __funnelshift_r(u[3], u[4], bits));
}

// elements of T between the last 16-byte boundary and p
template <class T>
__device__ __forceinline__ int behind16(const T* p) { return (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T)); }

// every column of a matrix starts on a 16-byte boundary
inline bool columns16(const void* p, long long ld, int size) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * size) % 16 == 0;
}

inline int type_size(int type) {
    return type == CUVDIA_T_F32 ? 4 : (type == CUVDIA_T_F16 || type == CUVDIA_T_BF16) ? 2 : 0;
}

// token j of a vector of 32- or 64-bit integers
struct Tokens {
    const void* p;
    bool wide;
    __device__ __forceinline__ long long operator[](long long j) const {
        return wide ? static_cast<const long long*>(p)[j] : static_cast<const int*>(p)[j];
    }
};
inline Tokens make_tokens(const void* p, int token_type) { return {p, token_type == CUVDIA_T_I64}; }

// the statements, with T the element type `type` (checked by the caller)
#define CUVDIA_FLOAT_TYPE(type, ...) \
    switch (type) { \
        case CUVDIA_T_F32: { typedef float T; __VA_ARGS__; break; } \
        case CUVDIA_T_F16: { typedef __half T; __VA_ARGS__; break; } \
        default: { typedef __nv_bfloat16 T; __VA_ARGS__; break; } \
    }

}  // namespace cuvdia
