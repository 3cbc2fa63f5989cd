// MXFP4 quantization and reading back (the format: mx4.cuh).
//
//   rows     x [R, K] -> codes and scales along K, behind the group-256 rotation or not, of a
//            matrix, of a stack of matrices, or of tokens in the order of their experts
//   columns  x [R, C] -> codes and scales of x^T, along R
//   values   codes and scales -> values
//
// All three move bytes and compute little: 2 (4 for fp32) bytes a value one way, 17/32 of a byte
// the other.
#include <cuda_runtime.h>

#include <string>
#include <type_traits>

#include "internal.h"
#include "mx4.cuh"
#include "rotpair.cuh"
#include "xpu_kernels/convrot.h"

namespace xpuint8 {
namespace {

struct RowArgs {
    const void *x;
    int64_t ldx;                 // elements between rows of x
    uint8_t *codes, *scales;     // codes may be null: only the rotated values are wanted
    void *rotated;               // [rows, K] of x's type, or null
    uint32_t groups;             // rows * G
    uint32_t K, G, KB, KT;       // 256-groups, 32-blocks and 128-tiles of a row
    uint32_t matrix_rows;        // rows of each matrix of a stack
    uint32_t matrix_tiles;       // its 128-row tiles (0: one matrix)
    const int32_t *order;        // sorted rows: row r of x is the slot order[r]
    const int32_t *positions;    // [slots] the row of codes that a slot's row goes to
    const int32_t *scale_rows;   // [slots] the row of scales; negative: no expert takes it
    uint32_t fan;                // slots of a token
};

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

template <int T>
__device__ __forceinline__ void store_run(void *row, uint32_t c, const Run<T> &r) {
    uint4 *p = reinterpret_cast<uint4 *>(static_cast<uint8_t *>(row) + static_cast<int64_t>(c) * mx_size(T));
#pragma unroll
    for (int j = 0; j < Run<T>::kWords / 4; ++j) p[j] = make_uint4(r.w[4 * j], r.w[4 * j + 1], r.w[4 * j + 2], r.w[4 * j + 3]);
}

// One half-warp ("slot") quantizes a pair of 256-value groups: a lane holds 16 consecutive values
// of each, so a block of 32 is two lanes, codes leave as 8 bytes a lane (128 consecutive bytes a
// group) and scales as one 4-byte word a 128-wide tile.  Instructions bound it before memory does:
// 16-bit values stay packed up to the conversion (the maximum is an integer one of two at a time),
// the rotation and the scaling are packed fp32x2.
template <int T, bool ROT, bool VEC>
__global__ void __launch_bounds__(128) quantize_rows_kernel(const RowArgs a) {
    __shared__ __align__(128) uint8_t tiles[ROT ? 8 * kSlotBytes : 16];
    const int slot = threadIdx.x >> 4, l = threadIdx.x & 15;
    const uint32_t f0 = (blockIdx.x * 8u + slot) * 2u;
    const uint32_t r0 = f0 / a.G, g0 = f0 - r0 * a.G;
    const uint32_t r1 = g0 + 1 == a.G ? r0 + 1 : r0, g1 = g0 + 1 == a.G ? 0 : g0 + 1;
    const bool ok0 = f0 < a.groups, ok1 = f0 + 1 < a.groups;
    const uint8_t *base = static_cast<const uint8_t *>(a.x);
    Run<T> A = zero_run<T>(), B = zero_run<T>();
    if (ok0) A = load_run<T, VEC>(base + r0 * a.ldx * mx_size(T), g0 * 256 + l * 16, a.K);
    if (ok1) B = load_run<T, VEC>(base + r1 * a.ldx * mx_size(T), g1 * 256 + l * 16, a.K);
    if constexpr (ROT) {
        const uint32_t tile = smem_u32(tiles) + slot * kSlotBytes;
        rotate_to_shared<T>(A, B, tile, l);
        runs_from_shared<T>(A, B, tile, l);
        if (a.rotated) {
            uint8_t *out = static_cast<uint8_t *>(a.rotated);
            if (ok0) store_run<T>(out + static_cast<int64_t>(r0) * a.K * mx_size(T), g0 * 256 + l * 16, A);
            if (ok1) store_run<T>(out + static_cast<int64_t>(r1) * a.K * mx_size(T), g1 * 256 + l * 16, B);
        }
        if (!a.codes) return;
    }
    uint32_t e0, e1;
    const uint2 c0 = quantize_run<T>(A, e0), c1 = quantize_run<T>(B, e1);
    const uint32_t w0 = join_scales(e0), w1 = join_scales(e1);
    auto put = [&](uint32_t r, uint32_t g, const uint2 &code, uint32_t word) {
        const uint32_t c = g * 256 + l * 16, kt = g * 2 + (l >> 3);
        const bool has_code = c < a.KB * 32, has_word = (l & 7) == 0 && kt < a.KT;
        for (uint32_t j = 0; j < a.fan; ++j) {
            int64_t cr = r, sr;
            if (a.scale_rows) {
                const uint32_t at = a.order ? static_cast<uint32_t>(__ldg(a.order + r)) : r * a.fan + j;
                sr = __ldg(a.scale_rows + at);
                if (sr < 0) continue;
                if (!a.order) cr = __ldg(a.positions + at);
            } else if (a.matrix_tiles == 0) {
                sr = r;
            } else {
                const uint32_t b = r / a.matrix_rows;
                sr = static_cast<int64_t>(b) * a.matrix_tiles * 128 + (r - b * a.matrix_rows);
            }
            if (has_code) *reinterpret_cast<uint2 *>(a.codes + cr * a.KB * 16 + c / 2) = code;
            if (has_word) *reinterpret_cast<uint32_t *>(a.scales + mx_scale_word(sr, kt, a.KT)) = word;
        }
    };
    if (ok0) put(r0, g0, c0, w0);
    if (ok1) put(r1, g1, c1, w1);
}

struct ColumnArgs {
    const void *x;
    int64_t ldx, matrix_stride;   // elements
    uint8_t *codes, *scales;
    uint32_t rows, cols;          // of x, each matrix
    int64_t pitch;                // bytes of a row of codes
    int64_t matrix_codes, matrix_scales;  // bytes of each matrix's
    uint32_t KT;                  // 128-tiles along the rows
    uint32_t code_blocks;         // 32-blocks that a row of codes holds
    const int32_t *offsets, *tiles;  // experts: where rows and 128-tiles begin, or null
    int experts;
};

// The group of rows that padded 128-tile t holds: the last e with tiles[e] <= t.
__device__ __forceinline__ int find_tile(const int32_t *tiles, int experts, int t) {
    int lo = 0, hi = experts;  // tiles[lo] <= t < tiles[hi], where there is such
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(tiles + mid) <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

// One CTA: 128 rows of x (a tile of scales along the contraction) x 64 columns.  Warp w takes the
// block of rows 32 w .. 32 w + 31, a lane two neighbouring columns: 32 loads in flight of 128
// consecutive bytes a warp, the block's maximum in registers.  Codes are turned in shared memory
// so that each column's 64 bytes leave together.
template <int T, bool VEC>
__global__ void __launch_bounds__(128) quantize_columns_kernel(const ColumnArgs a) {
    __shared__ __align__(16) uint32_t s_code[64][20];  // 64 bytes a column, padded to 80
    __shared__ __align__(4) uint8_t s_scale[64][4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kt = blockIdx.y;
    uint32_t begin = kt * 128u, end = a.rows;
    if (a.offsets) {
        if (kt >= __ldg(a.tiles + a.experts)) return;  // no expert's: the whole CTA leaves
        const int e = find_tile(a.tiles, a.experts, kt);
        begin = __ldg(a.offsets + e) + (kt - __ldg(a.tiles + e)) * 128;
        end = __ldg(a.offsets + e + 1);
    }
    const uint32_t c = blockIdx.x * 64 + lane * 2;
    const uint32_t r0 = begin + warp * 32;
    const uint8_t *x = static_cast<const uint8_t *>(a.x) + blockIdx.z * a.matrix_stride * mx_size(T);
    // all loads before the first use; the two columns of a 16-bit type are one word
    using Word = typename std::conditional<T == kMxF32, float2, uint32_t>::type;
    Word w[32];
    if (VEC && c + 1 < a.cols) {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            w[i] = Word{};
            if (r0 + i < end) w[i] = __ldg(reinterpret_cast<const Word *>(x + (static_cast<int64_t>(r0 + i) * a.ldx + c) * mx_size(T)));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const int64_t at = static_cast<int64_t>(r0 + i) * a.ldx + c;
            const bool in0 = r0 + i < end && c < a.cols, in1 = r0 + i < end && c + 1 < a.cols;
            if constexpr (T == kMxF32) {
                const float *p = reinterpret_cast<const float *>(x);
                w[i] = make_float2(in0 ? __ldg(p + at) : 0.f, in1 ? __ldg(p + at + 1) : 0.f);
            } else {
                const uint16_t *p = reinterpret_cast<const uint16_t *>(x);
                w[i] = (in0 ? __ldg(p + at) : 0u) | (static_cast<uint32_t>(in1 ? __ldg(p + at + 1) : 0u) << 16);
            }
        }
    }
    uint32_t m0 = 0, m1 = 0;
    if constexpr (T == kMxF32) {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            m0 = max(m0, __float_as_uint(w[i].x) & 0x7FFFFFFFu);
            m1 = max(m1, __float_as_uint(w[i].y) & 0x7FFFFFFFu);
        }
    } else {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) m = max_u16x2(m, w[i] & 0x7FFF7FFFu);
        m0 = widen_bits<T>(m & 0xFFFFu);
        m1 = widen_bits<T>(m >> 16);
    }
    const uint32_t e0 = mx_exponent(m0), e1 = mx_exponent(m1);
    const f2 inv = mk2(mx_inverse(e0), mx_inverse(e1));
    uint32_t code[2][4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        float v0[8], v1[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (T == kMxF32) {
                v0[i] = w[8 * q + i].x;
                v1[i] = w[8 * q + i].y;
            } else {
                mx_split<T>(w[8 * q + i], v0[i], v1[i]);
            }
            scale2(v0[i], v1[i], inv);
        }
        code[0][q] = mx_pack8(v0);
        code[1][q] = mx_pack8(v1);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
        *reinterpret_cast<uint4 *>(&s_code[lane * 2 + h][warp * 4]) = make_uint4(code[h][0], code[h][1], code[h][2], code[h][3]);
    s_scale[lane * 2][warp] = static_cast<uint8_t>(e0);
    s_scale[lane * 2 + 1][warp] = static_cast<uint8_t>(e1);
    __syncthreads();
    uint8_t *codes = a.codes + blockIdx.z * a.matrix_codes;
    uint8_t *scales = a.scales + blockIdx.z * a.matrix_scales;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int col = (threadIdx.x >> 2) + 32 * i, part = threadIdx.x & 3;
        const uint32_t n = blockIdx.x * 64 + col;
        if (n < a.cols && kt * 4u + part < a.code_blocks)
            *reinterpret_cast<uint4 *>(codes + n * a.pitch + (kt * 4 + part) * 16) = *reinterpret_cast<const uint4 *>(&s_code[col][part * 4]);
    }
    if (threadIdx.x < 64) {
        const uint32_t n = blockIdx.x * 64 + threadIdx.x;
        if (n < a.cols)
            *reinterpret_cast<uint32_t *>(scales + mx_scale_word(n, kt, a.KT)) = *reinterpret_cast<const uint32_t *>(s_scale[threadIdx.x]);
    }
}

struct ValueArgs {
    const uint8_t *codes, *scales;
    void *out;
    uint32_t K, KB, KT, units;  // units: of a row, runs of 16 values or of eight blocks
    int64_t total;              // rows * units
    uint32_t matrix_rows, matrix_tiles;
};

// Rows that are 16-byte aligned: 16 values a thread, 8 bytes of codes, a scale byte, 32 (64) bytes out.
template <int T>
__global__ void __launch_bounds__(256) values_kernel(const ValueArgs a) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= a.total) return;
    const int64_t r = i / a.units;
    const uint32_t h = static_cast<uint32_t>(i - r * a.units);
    const int64_t b = r / a.matrix_rows;
    const int64_t sr = b * a.matrix_tiles * 128 + (r - b * a.matrix_rows);
    const uint2 code = __ldg(reinterpret_cast<const uint2 *>(a.codes + r * a.KB * 16 + h * 8));
    const float s = mx_scale(__ldg(a.scales + mx_scale_word(sr, h >> 3, a.KT) + ((h >> 1) & 3)));
    Run<T> out;
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        float v0, v1;
        mx_unpack2(((t < 4 ? code.x : code.y) >> (8 * (t & 3))) & 0xFFu, v0, v1);
        scale2(v0, v1, mk2(s, s));
        if constexpr (T == kMxF32) {
            out.w[2 * t] = __float_as_uint(v0);
            out.w[2 * t + 1] = __float_as_uint(v1);
        } else {
            out.w[t] = mx_join<T>(v0, v1);
        }
    }
    store_run<T>(static_cast<uint8_t *>(a.out) + r * a.K * mx_size(T), h * 16, out);
}

// Rows of any length: a warp reads eight blocks of a row one after another, a value a lane, so that
// neighbouring lanes write neighbouring values.
template <int T>
__global__ void __launch_bounds__(256) odd_values_kernel(const ValueArgs a) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (i >= a.total) return;
    const int64_t r = i / a.units;
    const uint32_t b0 = static_cast<uint32_t>(i - r * a.units) * 8;
    const int64_t m = r / a.matrix_rows;
    const int64_t sr = m * a.matrix_tiles * 128 + (r - m * a.matrix_rows);
    const uint8_t *codes = a.codes + r * a.KB * 16;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t b = b0 + j, c = b * 32 + lane;
        if (c < a.K) {
            const uint32_t byte = __ldg(codes + c / 2), code = lane & 1 ? byte >> 4 : byte & 15u;
            const float s = mx_scale(__ldg(a.scales + mx_scale_word(sr, b >> 2, a.KT) + (b & 3)));
            mx_store1<T>(a.out, r * a.K + c, __fmul_rn(mx_value(code), s));
        }
    }
}

bool aligned(const void *p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

template <int T>
void launch_rows(cudaStream_t s, const RowArgs &a, bool rotate, bool vec) {
    const uint32_t grid = (a.groups + 15) / 16;
    if (rotate) {
        if (vec) quantize_rows_kernel<T, true, true><<<grid, 128, 0, s>>>(a);
        else quantize_rows_kernel<T, true, false><<<grid, 128, 0, s>>>(a);
    } else {
        if (vec) quantize_rows_kernel<T, false, true><<<grid, 128, 0, s>>>(a);
        else quantize_rows_kernel<T, false, false><<<grid, 128, 0, s>>>(a);
    }
}

int quantize_rows(cudaStream_t s, RowArgs &a, int type, int64_t rows, int64_t K, int64_t ldx, bool rotate) {
    a.K = static_cast<uint32_t>(K);
    a.G = static_cast<uint32_t>((K + 255) / 256);
    a.KB = static_cast<uint32_t>((K + 31) / 32);
    a.KT = (a.KB + 3) / 4;
    a.ldx = ldx;
    if (rows * a.G > 0x7FFFFFF0ll) {
        set_error("mxfp4: rows x 256-groups must be below 2^31");
        return 2;
    }
    a.groups = static_cast<uint32_t>(rows * a.G);
    const int es = mx_size(type);
    const bool vec = aligned(a.x, 16) && (ldx * es) % 16 == 0;
    switch (type) {
        case kMxBf16: launch_rows<kMxBf16>(s, a, rotate, vec); break;
        case kMxF16: launch_rows<kMxF16>(s, a, rotate, vec); break;
        default: launch_rows<kMxF32>(s, a, rotate, vec); break;
    }
    return launch_status("mxfp4_quantize");
}

int check_type(int32_t type) {
    if (type >= 0 && type <= 2) return 0;
    set_error("mxfp4: the element type must be 0 (bf16), 1 (fp16) or 2 (fp32)");
    return 2;
}

int check_sizes(int64_t rows, int64_t K) {
    if (rows <= 0 || K <= 0) {
        set_error("mxfp4: rows and K must be positive");
        return 2;
    }
    if (rows > 0x7FFFFF00ll || K > 0x7FFFFF00ll) {
        set_error("mxfp4: rows and K must fit in 31 bits");
        return 2;
    }
    return 0;
}

// x: aligned to its elements; codes and scales: 16 bytes
int check_pointers(const void *x, int type, std::initializer_list<const void *> others) {
    if (!x || !aligned(x, mx_size(type))) {
        set_error("mxfp4: x is null or not aligned to its elements");
        return 2;
    }
    for (const void *p : others)
        if (!p || !aligned(p, 16)) {
            set_error("mxfp4: a required pointer is null or not 16-byte aligned");
            return 2;
        }
    return 0;
}

int check_rotate(int64_t K, int32_t rotate) {
    if (!rotate || K % 256 == 0) return 0;
    set_error("K must be divisible by the ConvRot group size (256)");
    return 3;
}

cudaStream_t as_stream(const void *s) { return static_cast<cudaStream_t>(const_cast<void *>(s)); }

}  // namespace
}  // namespace xpuint8

using namespace xpuint8;

extern "C" {

int xpuint8_mxfp4_quantize_stream(const void *stream, const void *x, int32_t type, int64_t ldx,
                                  uint8_t *codes, uint8_t *scales, void *rotated, int64_t rows,
                                  int64_t K, int64_t matrix_rows, int32_t rotate) {
    if (int rc = check_type(type)) return rc;
    if (int rc = check_sizes(rows, K)) return rc;
    if (int rc = check_rotate(K, rotate)) return rc;
    if (!codes && !scales && rotated && rotate) {
        if (int rc = check_pointers(x, type, {rotated})) return rc;
    } else {
        if (int rc = check_pointers(x, type, {codes, scales})) return rc;
        if (rotated && (!rotate || !aligned(rotated, 16))) {
            set_error("mxfp4: rotated values need rotate and a 16-byte aligned pointer");
            return 2;
        }
    }
    if (ldx < K || matrix_rows <= 0 || rows % matrix_rows) {
        set_error("mxfp4: ldx must be at least K and rows a multiple of matrix_rows");
        return 2;
    }
    RowArgs a{};
    a.x = x;
    a.codes = codes;
    a.scales = scales;
    a.rotated = rotated;
    a.matrix_rows = static_cast<uint32_t>(matrix_rows);
    a.matrix_tiles = matrix_rows == rows ? 0 : static_cast<uint32_t>((matrix_rows + 127) / 128);
    a.fan = 1;
    return quantize_rows(as_stream(stream), a, type, rows, K, ldx, rotate != 0);
}

int xpuint8_mxfp4_quantize_sorted_stream(const void *stream, const void *x, int32_t type,
                                         int64_t ldx, uint8_t *codes, uint8_t *scales,
                                         void *rotated, const int32_t *order,
                                         const int32_t *positions, const int32_t *scale_rows,
                                         int64_t rows, int64_t fan, int64_t K, int32_t rotate) {
    if (int rc = check_type(type)) return rc;
    if (int rc = check_sizes(rows, K)) return rc;
    if (int rc = check_rotate(K, rotate)) return rc;
    if (int rc = check_pointers(x, type, {codes, scales})) return rc;
    if (!positions || !scale_rows || fan <= 0 || (order && fan != 1) || ldx < K ||
        rows * fan > 0x7FFFFF00ll || (rotated && (!rotate || !aligned(rotated, 16)))) {
        set_error("mxfp4: sorted rows need positions, scale_rows, a positive fan (1 with order) and ldx >= K");
        return 2;
    }
    RowArgs a{};
    a.x = x;
    a.codes = codes;
    a.scales = scales;
    a.rotated = rotated;
    a.order = order;
    a.positions = positions;
    a.scale_rows = scale_rows;
    a.matrix_rows = a.matrix_tiles = 1;
    a.fan = static_cast<uint32_t>(fan);
    return quantize_rows(as_stream(stream), a, type, rows, K, ldx, rotate != 0);
}

int xpuint8_mxfp4_quantize_columns_stream(const void *stream, const void *x, int32_t type,
                                          int64_t ldx, uint8_t *codes, uint8_t *scales,
                                          int64_t rows, int64_t cols, int64_t matrices,
                                          const int32_t *offsets, const int32_t *tiles,
                                          int64_t experts, int64_t max_tiles) {
    if (int rc = check_type(type)) return rc;
    if (int rc = check_sizes(rows, cols)) return rc;
    if (int rc = check_pointers(x, type, {codes, scales})) return rc;
    const bool sorted = offsets != nullptr;
    if (ldx < cols || matrices <= 0 || matrices > 65535 ||
        (sorted && (!tiles || experts <= 0 || max_tiles <= 0 || matrices != 1))) {
        set_error("mxfp4: ldx must be at least cols, 1 to 65535 matrices, and experts need tiles");
        return 2;
    }
    ColumnArgs a{};
    a.x = x;
    a.ldx = ldx;
    a.matrix_stride = rows * ldx;
    a.codes = codes;
    a.scales = scales;
    a.rows = static_cast<uint32_t>(rows);
    a.cols = static_cast<uint32_t>(cols);
    a.code_blocks = static_cast<uint32_t>(sorted ? max_tiles * 4 : (rows + 31) / 32);
    a.KT = static_cast<uint32_t>(sorted ? max_tiles : (rows + 127) / 128);
    a.pitch = static_cast<int64_t>(a.code_blocks) * 16;
    a.matrix_codes = a.pitch * cols;
    a.matrix_scales = (cols + 127) / 128 * a.KT * static_cast<int64_t>(kMxTileBytes);
    a.offsets = offsets;
    a.tiles = tiles;
    a.experts = static_cast<int>(experts);
    if (a.KT > 65535u) {
        set_error("mxfp4: at most 8388480 rows along the contraction");
        return 2;
    }
    const int es = mx_size(type);
    const bool vec = aligned(x, 2 * es) && ldx % 2 == 0;
    const dim3 grid(static_cast<uint32_t>((cols + 63) / 64), a.KT, static_cast<uint32_t>(matrices));
    cudaStream_t s = as_stream(stream);
    switch (type * 2 + (vec ? 1 : 0)) {
        case 0: quantize_columns_kernel<kMxBf16, false><<<grid, 128, 0, s>>>(a); break;
        case 1: quantize_columns_kernel<kMxBf16, true><<<grid, 128, 0, s>>>(a); break;
        case 2: quantize_columns_kernel<kMxF16, false><<<grid, 128, 0, s>>>(a); break;
        case 3: quantize_columns_kernel<kMxF16, true><<<grid, 128, 0, s>>>(a); break;
        case 4: quantize_columns_kernel<kMxF32, false><<<grid, 128, 0, s>>>(a); break;
        default: quantize_columns_kernel<kMxF32, true><<<grid, 128, 0, s>>>(a); break;
    }
    return launch_status("mxfp4_quantize_columns");
}

int xpuint8_mxfp4_dequantize_stream(const void *stream, const uint8_t *codes,
                                    const uint8_t *scales, void *out, int32_t type, int64_t rows,
                                    int64_t K, int64_t matrix_rows) {
    if (int rc = check_type(type)) return rc;
    if (int rc = check_sizes(rows, K)) return rc;
    if (int rc = check_pointers(out, type, {codes, scales})) return rc;
    if (matrix_rows <= 0 || rows % matrix_rows) {
        set_error("mxfp4: rows must be a multiple of matrix_rows");
        return 2;
    }
    ValueArgs a{};
    a.codes = codes;
    a.scales = scales;
    a.out = out;
    a.K = static_cast<uint32_t>(K);
    a.KB = static_cast<uint32_t>((K + 31) / 32);
    a.KT = (a.KB + 3) / 4;
    a.matrix_rows = static_cast<uint32_t>(matrix_rows);
    a.matrix_tiles = static_cast<uint32_t>((matrix_rows + 127) / 128);
    const bool vec = aligned(out, 16) && (K * mx_size(type)) % 16 == 0 && K % 16 == 0;
    a.units = static_cast<uint32_t>(vec ? K / 16 : (K + 255) / 256);
    a.total = rows * a.units;
    const int64_t blocks = vec ? (a.total + 255) / 256 : (a.total + 7) / 8;
    if (blocks > 0x7FFFFFFFll) {
        set_error("mxfp4: too many values");
        return 2;
    }
    cudaStream_t s = as_stream(stream);
    const uint32_t grid = static_cast<uint32_t>(blocks);
    switch (type * 2 + (vec ? 1 : 0)) {
        case 0: odd_values_kernel<kMxBf16><<<grid, 256, 0, s>>>(a); break;
        case 1: values_kernel<kMxBf16><<<grid, 256, 0, s>>>(a); break;
        case 2: odd_values_kernel<kMxF16><<<grid, 256, 0, s>>>(a); break;
        case 3: values_kernel<kMxF16><<<grid, 256, 0, s>>>(a); break;
        case 4: odd_values_kernel<kMxF32><<<grid, 256, 0, s>>>(a); break;
        default: values_kernel<kMxF32><<<grid, 256, 0, s>>>(a); break;
    }
    return launch_status("mxfp4_dequantize");
}

}  // extern "C"
