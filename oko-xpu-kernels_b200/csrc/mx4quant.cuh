// MXFP4 quantization on a half-warp: what the quantizers and the few-row product share.
#pragma once

#include "mx4.cuh"
#include "rotpair.cuh"

namespace xpuint8 {

// A lane's run of 16 consecutive values of a row, as loaded: 8 words of two 16-bit values, or 16 words
// of fp32.
template <int T>
struct Run {
    static constexpr int kWords = 4 * mx_size(T);
    uint32_t w[kWords];
};

// from column c on, zero past `cols`
template <int T, bool VEC>
__device__ __forceinline__ Run<T> load_run(const void *row, uint32_t c, uint32_t cols) {
    Run<T> r;
    if (VEC && c + 16 <= cols) {
        const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(row) + static_cast<int64_t>(c) * mx_size(T));
#pragma unroll
        for (int j = 0; j < Run<T>::kWords / 4; ++j) {
            const uint4 q = __ldg(p + j);
            r.w[4 * j] = q.x;
            r.w[4 * j + 1] = q.y;
            r.w[4 * j + 2] = q.z;
            r.w[4 * j + 3] = q.w;
        }
    } else if constexpr (T == kMxF32) {
#pragma unroll
        for (int t = 0; t < 16; ++t) r.w[t] = c + t < cols ? __ldg(static_cast<const uint32_t *>(row) + c + t) : 0u;
    } else {
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            const uint32_t lo = c + 2 * t < cols ? __ldg(static_cast<const uint16_t *>(row) + c + 2 * t) : 0u;
            const uint32_t hi = c + 2 * t + 1 < cols ? __ldg(static_cast<const uint16_t *>(row) + c + 2 * t + 1) : 0u;
            r.w[t] = lo | (hi << 16);
        }
    }
    return r;
}
template <int T>
__device__ __forceinline__ Run<T> zero_run() {
    Run<T> r;
#pragma unroll
    for (int j = 0; j < Run<T>::kWords; ++j) r.w[j] = 0u;
    return r;
}

// per half, the maximum of two unsigned 16-bit values
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// the fp32 bits of a 16-bit magnitude
template <int T>
__device__ __forceinline__ uint32_t widen_bits(uint32_t h) {
    if constexpr (T == kMxBf16) return h << 16;
    float lo, hi;
    mx_split<T>(h, lo, hi);
    return __float_as_uint(lo);
}

// the pair (v0, v1) times (s0, s1)
__device__ __forceinline__ void scale2(float &v0, float &v1, f2 s) { un2(mul2(mk2(v0, v1), s), v0, v1); }

// Codes of a lane's 16 values, its neighbour (lane ^ 1) holding the block's other 16: 8 bytes, and
// the block's scale byte.
template <int T>
__device__ __forceinline__ uint2 quantize_run(const Run<T> &r, uint32_t &e) {
    uint32_t m = 0;
    if constexpr (T == kMxF32) {
#pragma unroll
        for (int t = 0; t < 16; ++t) m = max(m, r.w[t] & 0x7FFFFFFFu);
        m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
    } else {
#pragma unroll
        for (int t = 0; t < 8; ++t) m = max_u16x2(m, r.w[t] & 0x7FFF7FFFu);
        m = max_u16x2(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
        m = widen_bits<T>(max(m & 0xFFFFu, m >> 16));
    }
    e = mx_exponent(m);
    const float inv = mx_inverse(e);
    const f2 s = mk2(inv, inv);
    float v[16];
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        if constexpr (T == kMxF32) {
            v[2 * t] = __uint_as_float(r.w[2 * t]);
            v[2 * t + 1] = __uint_as_float(r.w[2 * t + 1]);
        } else {
            mx_split<T>(r.w[t], v[2 * t], v[2 * t + 1]);
        }
        scale2(v[2 * t], v[2 * t + 1], s);
    }
    return make_uint2(mx_pack8(v), mx_pack8(v + 8));
}

// Lanes 0, 2, 4, 6 (8, 10, 12, 14) of a half-warp hold the scale bytes of a tile's four blocks: the
// word of them, on lanes 0 and 8.
__device__ __forceinline__ uint32_t join_scales(uint32_t e) {
    const uint32_t two = e | (__shfl_down_sync(0xFFFFFFFFu, e, 2) << 8);
    return two | (__shfl_down_sync(0xFFFFFFFFu, two, 4) << 16);
}

// A pair of 256-value groups A and B on a half-warp's lanes, turned to pairs: value c of both at
// pair_at(c) of the slot's shared memory, as a word (16-bit types) or two (fp32).  The pitches put
// the words of a column and those of a run into different banks, with every address a base and a
// constant.
constexpr int kSlotBytes = 16 * 144;
template <int T>
__device__ __forceinline__ constexpr uint32_t pair_at(int w, int l) { return T == kMxF32 ? w * 144 + l * 8 : w * 80 + l * 4; }

// The rotation of the pair, scaled and rounded to the type, left in shared memory.  Lane l brings
// values 16 l .. 16 l + 15 of both groups: two radix-4 steps in registers (accumulation chains), the
// turn through shared memory, two more (butterflies): the association of rotate(), so the same bits.
template <int T>
__device__ __forceinline__ void rotate_to_shared(const Run<T> &A, const Run<T> &B, uint32_t slot, int l) {
    f2 P[16];
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        float a0, a1, b0, b1;
        if constexpr (T == kMxF32) {
            a0 = __uint_as_float(A.w[2 * t]);
            a1 = __uint_as_float(A.w[2 * t + 1]);
            b0 = __uint_as_float(B.w[2 * t]);
            b1 = __uint_as_float(B.w[2 * t + 1]);
        } else {
            mx_split<T>(A.w[t], a0, a1);
            mx_split<T>(B.w[t], b0, b1);
        }
        P[2 * t] = mk2(a0, b0);
        P[2 * t + 1] = mk2(a1, b1);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) seq2(P[4 * j], P[4 * j + 1], P[4 * j + 2], P[4 * j + 3]);
#pragma unroll
    for (int j = 0; j < 4; ++j) seq2(P[j], P[j + 4], P[j + 8], P[j + 12]);
    const uint32_t mine = slot + l * 144, column = slot + l * 8;
#pragma unroll
    for (int c = 0; c < 8; ++c)
        asm volatile("st.shared.v2.b64 [%0], {%1, %2};" ::"r"(mine + c * 16), "l"(P[2 * c].v), "l"(P[2 * c + 1].v) : "memory");
    __syncwarp();
#pragma unroll
    for (int w = 0; w < 16; ++w) asm volatile("ld.shared.b64 %0, [%1];" : "=l"(P[w].v) : "r"(column + w * 144));
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; ++j) bfly2(P[4 * j], P[4 * j + 1], P[4 * j + 2], P[4 * j + 3]);
#pragma unroll
    for (int j = 0; j < 4; ++j) bfly2(P[j], P[j + 4], P[j + 8], P[j + 12]);
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        const f2 s = mul2(P[w], mk2(0.0625f, 0.0625f));
        if constexpr (T == kMxF32) {
            asm volatile("st.shared.b64 [%0], %1;" ::"r"(slot + pair_at<T>(w, 0) + l * 8), "l"(s.v) : "memory");
        } else {
            float p, q;
            un2(s, p, q);
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(slot + pair_at<T>(w, 0) + l * 4), "r"(mx_join<T>(p, q)) : "memory");
        }
    }
    __syncwarp();
}

// both runs of lane l to the pairs
template <int T>
__device__ __forceinline__ void runs_to_shared(const Run<T> &A, const Run<T> &B, uint32_t slot, int l) {
    const uint32_t at = slot + pair_at<T>(1, 0) * l;
    if constexpr (T == kMxF32) {
#pragma unroll
        for (int c = 0; c < 8; ++c) st_shared_v4(at + c * 16, A.w[2 * c], B.w[2 * c], A.w[2 * c + 1], B.w[2 * c + 1]);
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            st_shared_v4(at + c * 16, __byte_perm(A.w[2 * c], B.w[2 * c], 0x5410), __byte_perm(A.w[2 * c], B.w[2 * c], 0x7632),
                         __byte_perm(A.w[2 * c + 1], B.w[2 * c + 1], 0x5410), __byte_perm(A.w[2 * c + 1], B.w[2 * c + 1], 0x7632));
    }
}

// both runs of lane l back from the pairs
template <int T>
__device__ __forceinline__ void runs_from_shared(Run<T> &A, Run<T> &B, uint32_t slot, int l) {
    const uint32_t at = slot + pair_at<T>(1, 0) * l;
    if constexpr (T == kMxF32) {
#pragma unroll
        for (int c = 0; c < 8; ++c)
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(A.w[2 * c]), "=r"(B.w[2 * c]), "=r"(A.w[2 * c + 1]), "=r"(B.w[2 * c + 1]) : "r"(at + c * 16));
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            uint32_t w[4];
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at + c * 16));
            A.w[2 * c] = __byte_perm(w[0], w[1], 0x5410);
            B.w[2 * c] = __byte_perm(w[0], w[1], 0x7632);
            A.w[2 * c + 1] = __byte_perm(w[2], w[3], 0x5410);
            B.w[2 * c + 1] = __byte_perm(w[2], w[3], 0x7632);
        }
    }
}

}  // namespace xpuint8
