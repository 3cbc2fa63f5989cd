// MXFP4: what the quantizers, the products and the experts' kernels share.
//
// A row of K values is held as blocks of 32 values of 4 bits (E2M1: 0, 0.5, 1, 1.5, 2, 3, 4, 6
// and a sign) with one power-of-two scale a block (E8M0: byte e stands for 2^(e - 127), 255 for
// NaN), the OCP Microscaling format of 4 bits:
//
//   e    = max(floor(log2 max|v|) - 2 + 127, 0)         (2: the exponent of the largest code, 4..6)
//   code = the E2M1 value nearest to v / 2^(e - 127), ties to the even code, above 6 to 6
//
// Both steps are exact but for the last rounding: e is read from the maximum's exponent bits
// and the division is by a power of two.  A block that holds a NaN or an infinity gets e = 255,
// so every sum that reads it is NaN.
//
// Storage of a matrix of R rows: codes [R, ceil(K / 32) * 16] bytes, the earlier value of a byte
// in its low half, values past K zero; scales in tiles of 128 rows x 4 blocks, 512 bytes, the
// order in which the tensor cores take them from tensor memory: row 32 j + l of a tile and its
// block b at byte 16 l + 4 j + b, tiles [ceil(R / 128)][ceil(K / 128)].  Scales of blocks past K
// in a tile are 0 (2^-127); rows past R hold anything.
#pragma once

#include <stdint.h>

#include "common.cuh"

namespace xpuint8 {

constexpr int kMxTileBytes = 512;

// element types of the entry points
enum MxType { kMxBf16 = 0, kMxF16 = 1, kMxF32 = 2 };
__host__ __device__ constexpr int mx_size(int type) { return type == kMxF32 ? 4 : 2; }

// byte offset of the 4-byte word that holds row r's scales of 128-wide tile kt
__device__ __forceinline__ int64_t mx_scale_word(int64_t r, int kt, int KT) {
    return ((r >> 7) * KT + kt) * kMxTileBytes + (r & 31) * 16 + ((r >> 5) & 3) * 4;
}
// the scale byte of a block from the bits of its largest magnitude (an integer maximum, so a NaN
// is the largest of all)
__device__ __forceinline__ uint32_t mx_exponent(uint32_t amax_bits) {
    const int e = static_cast<int>(amax_bits >> 23);
    return e == 255 ? 255u : static_cast<uint32_t>(max(e - 2, 0));
}
// 1 / scale: 2^(127 - e), a normal number for every e below 254
__device__ __forceinline__ float mx_inverse(uint32_t e) {
    return e == 255u ? 0.f : __uint_as_float((254u - e) << 23);
}
__device__ __forceinline__ float mx_scale(uint32_t e) {
    return e == 255u ? __uint_as_float(0x7FC00000u) : e == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(e << 23);
}
// eight values, already divided by the scale, to four bytes of codes
__device__ __forceinline__ uint32_t mx_pack8(const float *v) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
// the value of a code in the low four bits: its exponent and mantissa bits at those of an fp32 number
// are the value times 2^-126, the smallest step (0.5) a subnormal number
__device__ __forceinline__ float mx_value(uint32_t code) {
    return __fmul_rn(__uint_as_float(((code & 7u) << 22) | ((code & 8u) << 28)), 8.507059173023462e37f);
}
// the two values of a byte of codes
__device__ __forceinline__ void mx_unpack2(uint32_t byte, float &lo, float &hi) {
    uint32_t h;
    asm("{\n\t.reg .b8 a, x, y, z;\n\tmov.b32 {a, x, y, z}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t}" : "=r"(h) : "r"(byte));
    asm("{\n\t.reg .f16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}"
        : "=f"(lo), "=f"(hi) : "r"(h));
}

// the two values of a 32-bit word of a 16-bit type
template <int T>
__device__ __forceinline__ void mx_split(uint32_t w, float &lo, float &hi) {
    if constexpr (T == kMxBf16) {
        lo = bf16_lo(w);
        hi = bf16_hi(w);
    } else {
        asm("{\n\t.reg .f16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}"
            : "=f"(lo), "=f"(hi) : "r"(w));
    }
}
// two values to a word of a 16-bit type, round to nearest even
template <int T>
__device__ __forceinline__ uint32_t mx_join(float lo, float hi) {
    if constexpr (T == kMxBf16) return cvt_bf16x2(lo, hi);
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <int T>
__device__ __forceinline__ void mx_store1(void *p, int64_t i, float v) {
    if constexpr (T == kMxF32) static_cast<float *>(p)[i] = v;
    else static_cast<uint16_t *>(p)[i] = static_cast<uint16_t>(mx_join<T>(v, 0.f));
}

}  // namespace xpuint8
