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

// eight words by one 32-byte access
__device__ __forceinline__ void load_v8(const void *p, uint32_t *w) {
    asm("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
        : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
        : "l"(p));
}
__device__ __forceinline__ void store_v8(void *p, const uint32_t *w) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                 "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// from column c on, zero past `cols`.  VEC: rows are 16-byte aligned; wide: 32-byte, so that a lane's
// run of a 16-bit type is one access and a warp's are whole lines (as two of 16 bytes they take twice
// the shared-memory pipe's time, which bounds the rotated quantizer)
template <int T, bool VEC>
__device__ __forceinline__ Run<T> load_run(const void *row, uint32_t c, uint32_t cols, bool wide) {
    Run<T> r;
    if (VEC && c + 16 <= cols) {
        const uint8_t *q = static_cast<const uint8_t *>(row) + static_cast<int64_t>(c) * mx_size(T);
        if (wide) {
#pragma unroll
            for (int j = 0; j < Run<T>::kWords / 8; ++j) load_v8(q + 32 * j, r.w + 8 * j);
            return r;
        }
        const uint4 *p = reinterpret_cast<const uint4 *>(q);
#pragma unroll
        for (int j = 0; j < Run<T>::kWords / 4; ++j) {
            const uint4 q = __ldg(p + j);
            r.w[4 * j] = q.x;
            r.w[4 * j + 1] = q.y;
            r.w[4 * j + 2] = q.z;
            r.w[4 * j + 3] = q.w;
        }
    } else if (!VEC && c >= 8 && c + 24 <= cols) {
        // the aligned 16-byte words around the run, all inside the row, moved into place ([9001, 4001] bf16
        // quantised in 18.4 us; value by value 39)
        constexpr int N = Run<T>::kWords + 4;
        const uint8_t *q = static_cast<const uint8_t *>(row) + static_cast<int64_t>(c) * mx_size(T);
        const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(q)) & 15;
        const uint4 *p = reinterpret_cast<const uint4 *>(q - off);
        uint32_t w[N];
#pragma unroll
        for (int j = 0; j < N / 4; ++j) {
            const uint4 v = __ldg(p + j);
            w[4 * j] = v.x;
            w[4 * j + 1] = v.y;
            w[4 * j + 2] = v.z;
            w[4 * j + 3] = v.w;
        }
#pragma unroll
        for (int j = 0; j < N - 2; ++j) w[j] = off & 8 ? w[j + 2] : w[j];
#pragma unroll
        for (int j = 0; j < N - 3; ++j) w[j] = off & 4 ? w[j + 1] : w[j];
#pragma unroll
        for (int j = 0; j < Run<T>::kWords; ++j) r.w[j] = T == kMxF32 ? w[j] : __funnelshift_r(w[j], w[j + 1], (off & 2) * 8);
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

// per half, the larger magnitude of two 16-bit values, its sign anything; a NaN is the largest
template <int T>
__device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (T == kMxBf16) asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// the largest of m and two magnitudes; a NaN is the largest
__device__ __forceinline__ float max_abs3(float m, uint32_t a, uint32_t b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(fabsf(__uint_as_float(a))), "f"(fabsf(__uint_as_float(b))));
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

// What a lane makes of its 16 values of two rows: 8 bytes of codes each and, on lanes 0 and 8 of the
// half-warp, the words of four scales that start there.
struct PairCodes {
    uint2 c0, c1;
    uint32_t w0, w1;
};

// the scale words of both rows from the lanes' scale bytes (lanes 0, 2, 4, 6 and 8, 10, 12, 14 hold a
// tile's four blocks)
__device__ __forceinline__ void join_scales(uint32_t e0, uint32_t e1, uint32_t &w0, uint32_t &w1) {
    const uint32_t both = e0 | (e1 << 16);
    const uint32_t two = both | (__shfl_down_sync(0xFFFFFFFFu, both, 2) << 8);
    const uint32_t next = __shfl_down_sync(0xFFFFFFFFu, two, 4);
    w0 = __byte_perm(two, next, 0x5410);
    w1 = __byte_perm(two, next, 0x7632);
}

// Two runs of 16, the neighbouring lane (lane ^ 1) holding each block's other 16 values.
template <int T>
__device__ __forceinline__ PairCodes quantize_runs(const Run<T> &A, const Run<T> &B) {
    uint32_t mA = 0, mB = 0;
    if constexpr (T == kMxF32) {
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int t = 0; t < 16; t += 2) {
            a = max_abs3(a, A.w[t], A.w[t + 1]);
            b = max_abs3(b, B.w[t], B.w[t + 1]);
        }
        mA = __float_as_uint(a);
        mB = __float_as_uint(b);
        mA = max(mA, __shfl_xor_sync(0xFFFFFFFFu, mA, 1));
        mB = max(mB, __shfl_xor_sync(0xFFFFFFFFu, mB, 1));
    } else {
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            mA = max_abs2<T>(mA, A.w[t]);
            mB = max_abs2<T>(mB, B.w[t]);
        }
        uint32_t m = max_abs2<T>(__byte_perm(mA, mB, 0x5410), __byte_perm(mA, mB, 0x7632));  // (A, B)
        m = max_abs2<T>(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1)) & 0x7FFF7FFFu;
        mA = widen_bits<T>(m & 0xFFFFu);
        mB = widen_bits<T>(m >> 16);
    }
    const uint32_t e0 = mx_exponent(mA), e1 = mx_exponent(mB);
    const f2 s0 = mk2(mx_inverse(e0), mx_inverse(e0)), s1 = mk2(mx_inverse(e1), mx_inverse(e1));
    float a[16], b[16];
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        if constexpr (T == kMxF32) {
            a[2 * t] = __uint_as_float(A.w[2 * t]);
            a[2 * t + 1] = __uint_as_float(A.w[2 * t + 1]);
            b[2 * t] = __uint_as_float(B.w[2 * t]);
            b[2 * t + 1] = __uint_as_float(B.w[2 * t + 1]);
        } else {
            mx_split<T>(A.w[t], a[2 * t], a[2 * t + 1]);
            mx_split<T>(B.w[t], b[2 * t], b[2 * t + 1]);
        }
        scale2(a[2 * t], a[2 * t + 1], s0);
        scale2(b[2 * t], b[2 * t + 1], s1);
    }
    PairCodes p;
    p.c0 = make_uint2(mx_pack8(a), mx_pack8(a + 8));
    p.c1 = make_uint2(mx_pack8(b), mx_pack8(b + 8));
    join_scales(e0, e1, p.w0, p.w1);
    return p;
}

// A pair of 256-value groups A and B on a half-warp's lanes, turned to pairs: value c of both at
// pair_at(c) of the slot's shared memory, as a word (16-bit types) or two (fp32).  The pitches put
// the words of a column and those of a run into different banks, with every address a base and a
// constant; the slots of a warp's two halves lie 16 banks apart.
constexpr int kSlotBytes = 16 * 144 + 64;
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

// lane l's 16 values of both groups from the pairs, as they lie there: words (A, B) of a 16-bit type,
// or fp32 pairs
template <int T>
struct Pairs {
    static constexpr int kWords = 8 * mx_size(T);
    uint32_t w[kWords];
};
template <int T>
__device__ __forceinline__ Pairs<T> pairs_from_shared(uint32_t slot, int l) {
    Pairs<T> p;
    const uint32_t at = slot + pair_at<T>(1, 0) * l;
#pragma unroll
    for (int c = 0; c < Pairs<T>::kWords / 4; ++c)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(p.w[4 * c]), "=r"(p.w[4 * c + 1]), "=r"(p.w[4 * c + 2]), "=r"(p.w[4 * c + 3]) : "r"(at + c * 16));
    return p;
}
// as two runs
template <int T>
__device__ __forceinline__ void split_pairs(const Pairs<T> &p, Run<T> &A, Run<T> &B) {
    if constexpr (T == kMxF32) {
#pragma unroll
        for (int t = 0; t < 16; ++t) {
            A.w[t] = p.w[2 * t];
            B.w[t] = p.w[2 * t + 1];
        }
    } else {
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            A.w[t] = __byte_perm(p.w[2 * t], p.w[2 * t + 1], 0x5410);
            B.w[t] = __byte_perm(p.w[2 * t], p.w[2 * t + 1], 0x7632);
        }
    }
}
// quantize_runs on the pairs: one maximum and one scaling serve both groups
template <int T>
__device__ __forceinline__ PairCodes quantize_pairs(const Pairs<T> &p) {
    uint32_t mA = 0, mB = 0;
    if constexpr (T == kMxF32) {
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int t = 0; t < 16; t += 2) {
            a = max_abs3(a, p.w[2 * t], p.w[2 * t + 2]);
            b = max_abs3(b, p.w[2 * t + 1], p.w[2 * t + 3]);
        }
        mA = __float_as_uint(a);
        mB = __float_as_uint(b);
        mA = max(mA, __shfl_xor_sync(0xFFFFFFFFu, mA, 1));
        mB = max(mB, __shfl_xor_sync(0xFFFFFFFFu, mB, 1));
    } else {
        uint32_t m = 0;
#pragma unroll
        for (int t = 0; t < 16; ++t) m = max_abs2<T>(m, p.w[t]);
        m = max_abs2<T>(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1)) & 0x7FFF7FFFu;
        mA = widen_bits<T>(m & 0xFFFFu);
        mB = widen_bits<T>(m >> 16);
    }
    const uint32_t e0 = mx_exponent(mA), e1 = mx_exponent(mB);
    const f2 s = mk2(mx_inverse(e0), mx_inverse(e1));
    float a[16], b[16];
#pragma unroll
    for (int t = 0; t < 16; ++t) {
        if constexpr (T == kMxF32) {
            a[t] = __uint_as_float(p.w[2 * t]);
            b[t] = __uint_as_float(p.w[2 * t + 1]);
        } else {
            mx_split<T>(p.w[t], a[t], b[t]);
        }
        scale2(a[t], b[t], s);
    }
    PairCodes r;
    r.c0 = make_uint2(mx_pack8(a), mx_pack8(a + 8));
    r.c1 = make_uint2(mx_pack8(b), mx_pack8(b + 8));
    join_scales(e0, e1, r.w0, r.w1);
    return r;
}

// n / d for 0 <= n < 2^31 by one high multiply, an add and a shift: the invariant-divisor method of
// Granlund & Montgomery (PLDI 1994, section 4), l = ceil(log2 d), m = floor(2^32 (2^l - d) / d) + 1
struct Divisor {
    uint32_t d, m, l;
    static Divisor of(uint32_t d) {
        uint32_t l = 0;
        while ((uint64_t{1} << l) < d) ++l;
        return {d, static_cast<uint32_t>(((uint64_t{1} << 32) * ((uint64_t{1} << l) - d)) / d + 1), l};
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (__umulhi(n, m) + n) >> l; }
};

}  // namespace xpuint8
