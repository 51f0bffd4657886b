// The counter-based generator of the element-wise passes.
#pragma once
#include "cuvdia_internal.cuh"

namespace cuvdia {

// ---- uniform numbers drawn where they are used -------------------------------------------------------------------
// CUV binarises an activation by comparing it with a uniform number drawn on the device (rnd_binarize,
// random/random.cu:86-91,139-156: one generator state per thread).  Here the number of element (row, column) of draw
// `which` in step `step` is a pure function of those four and a 64-bit seed - the counter-based generator
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011) - so a pass can
// draw it in registers instead of reading it from memory, any sharding of the batch columns draws the same numbers
// as the unsharded run, and a CPU restatement reproduces them bit for bit.  One call gives four 32-bit words: the
// numbers of rows 4q .. 4q+3 of one column; counter = (q, column, which + 65536 * (column >> 32), step), key = seed.
// A word x becomes the float (x >> 8) * 2^-24 in [0, 1): exact, and P(u < p) = p to within 2^-24.
__device__ __forceinline__ uint4 philox4x32_10(uint4 c, uint2 k) {
#pragma unroll
    for (int r = 0; r < 10; r++) {
        const unsigned long long p0 = (unsigned long long)0xD2511F53u * c.x;      // one wide multiply gives both halves
        const unsigned long long p1 = (unsigned long long)0xCD9E8D57u * c.z;
        c = make_uint4((unsigned)(p1 >> 32) ^ c.y ^ k.x, (unsigned)p1, (unsigned)(p0 >> 32) ^ c.w ^ k.y, (unsigned)p0);
        k.x += 0x9E3779B9u; k.y += 0xBB67AE85u;
    }
    return c;
}

__device__ __forceinline__ float u01(unsigned x) { return (float)(x >> 8) * (1.f / 16777216.f); }

// the four uniform numbers of rows 4q .. 4q+3 of global column gcol
__device__ __forceinline__ float4 draw4(const DrawParams& d, int q, long long gcol) {
    const uint4 r = philox4x32_10(make_uint4((unsigned)q, (unsigned)gcol, d.which + 65536u * (unsigned)(gcol >> 32), d.step),
                                  make_uint2(d.k0, d.k1));
    return make_float4(u01(r.x), u01(r.y), u01(r.z), u01(r.w));
}

}  // namespace cuvdia
