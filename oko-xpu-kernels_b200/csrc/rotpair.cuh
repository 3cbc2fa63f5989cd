// The ConvRot rotation of a pair of 256-groups by one half-warp ("slot"), as packed
// fp32x2 values: shared by the int8 rotation kernels and the MXFP4 quantizer, so both
// produce the same bits.
#pragma once

#include "common.cuh"

namespace xpuint8 {

// accumulation-chain radix-4 butterfly (unscaled) on fp32x2 lanes
__device__ __forceinline__ void seq2(f2 &a0, f2 &a1, f2 &a2, f2 &a3) {
    const f2 p = add2(a0, a1), m = sub2(a0, a1);
    const f2 o0 = sub2(add2(p, a2), a3);
    const f2 o1 = add2(sub2(p, a2), a3);
    const f2 o2 = add2(add2(m, a2), a3);
    const f2 o3 = add2(sub2(a2, m), a3);
    a0 = o0; a1 = o1; a2 = o2; a3 = o3;
}
// butterfly-association radix-4 butterfly (unscaled) on fp32x2 lanes
__device__ __forceinline__ void bfly2(f2 &a0, f2 &a1, f2 &a2, f2 &a3) {
    const f2 p = add2(a0, a1), m = sub2(a0, a1);
    const f2 q = add2(a2, a3), n = sub2(a2, a3);
    a0 = add2(p, n); a1 = sub2(p, n); a2 = add2(m, q); a3 = sub2(q, m);
}

// Rotate a pair of groups.  In: P[q] = (A[16l+q], B[16l+q]).  Out: P[w] =
// (A[16w+l], B[16w+l]), unscaled (x16).  `tile` is the slot's 2 KB tile.
__device__ __forceinline__ void rotate_pair(f2 (&P)[16], uint32_t tile, int l) {
#pragma unroll
    for (int j = 0; j < 4; ++j) seq2(P[4 * j], P[4 * j + 1], P[4 * j + 2], P[4 * j + 3]);
#pragma unroll
    for (int j = 0; j < 4; ++j) seq2(P[j], P[j + 4], P[j + 8], P[j + 12]);
    // row l <- P (128 bytes, 16-byte chunk c at c ^ (l & 7)); then read column l
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        float a0, b0, a1, b1;
        un2(P[2 * c], a0, b0);
        un2(P[2 * c + 1], a1, b1);
        st_shared_v4(tile + l * 128 + ((c ^ (l & 7)) << 4), __float_as_uint(a0), __float_as_uint(b0),
                     __float_as_uint(a1), __float_as_uint(b1));
    }
    __syncwarp();
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        const uint32_t addr = tile + w * 128 + ((((l >> 1) ^ w) & 7) << 4) + ((l & 1) << 3);
        asm volatile("ld.shared.b64 %0, [%1];" : "=l"(P[w].v) : "r"(addr));
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; ++j) bfly2(P[4 * j], P[4 * j + 1], P[4 * j + 2], P[4 * j + 3]);
#pragma unroll
    for (int j = 0; j < 4; ++j) bfly2(P[j], P[j + 4], P[j + 8], P[j + 12]);
}

}  // namespace xpuint8
