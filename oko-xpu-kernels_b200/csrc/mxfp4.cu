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
    uint32_t matrix_tiles;       // its 128-row tiles
    const int32_t *order;        // sorted rows: row r of x is the slot order[r]
    const int32_t *positions;    // [slots] the row of codes that a slot's row goes to
    const int32_t *scale_rows;   // [slots] the row of scales; negative: no expert takes it
    uint32_t fan;                // slots of a token
};

// 16 consecutive values of a row from column c on, zero past K
template <int T, bool VEC>
__device__ __forceinline__ void load16(const RowArgs &a, const void *row, uint32_t c, float (&v)[16]) {
    if (VEC && c + 16 <= a.K) {
        const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(row) + static_cast<int64_t>(c) * mx_size(T));
        if constexpr (T == kMxF32) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint4 w = __ldg(p + j);
                v[4 * j] = __uint_as_float(w.x);
                v[4 * j + 1] = __uint_as_float(w.y);
                v[4 * j + 2] = __uint_as_float(w.z);
                v[4 * j + 3] = __uint_as_float(w.w);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint4 w = __ldg(p + j);
                mx_split<T>(w.x, v[8 * j], v[8 * j + 1]);
                mx_split<T>(w.y, v[8 * j + 2], v[8 * j + 3]);
                mx_split<T>(w.z, v[8 * j + 4], v[8 * j + 5]);
                mx_split<T>(w.w, v[8 * j + 6], v[8 * j + 7]);
            }
        }
        return;
    }
#pragma unroll
    for (int t = 0; t < 16; ++t) v[t] = c + t < a.K ? mx_load1<T>(row, c + t) : 0.f;
}

template <int T>
__device__ __forceinline__ void store16(void *row, uint32_t c, const float (&v)[16]) {
    uint4 *p = reinterpret_cast<uint4 *>(static_cast<uint8_t *>(row) + static_cast<int64_t>(c) * mx_size(T));
    if constexpr (T == kMxF32) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            p[j] = make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]),
                              __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3]));
    } else {
#pragma unroll
        for (int j = 0; j < 2; ++j)
            p[j] = make_uint4(mx_join<T>(v[8 * j], v[8 * j + 1]), mx_join<T>(v[8 * j + 2], v[8 * j + 3]),
                              mx_join<T>(v[8 * j + 4], v[8 * j + 5]), mx_join<T>(v[8 * j + 6], v[8 * j + 7]));
    }
}

// The rotated pair P[w] = (A[16 w + l], B[16 w + l]) (x16), scaled, rounded to the type, and
// turned so that lane l holds values 16 l .. 16 l + 15 of both groups.
template <int T>
__device__ __forceinline__ void settle_pair(f2 (&P)[16], uint32_t tile, int l, float (&A)[16], float (&B)[16]) {
    if constexpr (T == kMxF32) {
        // 8-byte words, row w of 128 bytes, 16-byte chunk c at c ^ (w & 7)
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            const f2 s = mul2(P[w], mk2(0.0625f, 0.0625f));
            asm volatile("st.shared.b64 [%0], %1;" ::"r"(tile + w * 128 + ((((l >> 1) ^ w) & 7) << 4) + ((l & 1) << 3)), "l"(s.v) : "memory");
        }
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            uint32_t x, y, z, u;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x), "=r"(y), "=r"(z), "=r"(u) : "r"(tile + l * 128 + ((c ^ (l & 7)) << 4)));
            A[2 * c] = __uint_as_float(x);
            B[2 * c] = __uint_as_float(y);
            A[2 * c + 1] = __uint_as_float(z);
            B[2 * c + 1] = __uint_as_float(u);
        }
    } else {
        // 4-byte words (A, B), row w of 64 bytes, 16-byte chunk c at c ^ ((w >> 1) & 3)
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            float p, q;
            un2(mul2(P[w], mk2(0.0625f, 0.0625f)), p, q);
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(tile + w * 64 + (((l >> 2) ^ ((w >> 1) & 3)) << 4) + ((l & 3) << 2)), "r"(mx_join<T>(p, q)) : "memory");
        }
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            uint32_t w[4];
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(tile + l * 64 + ((c ^ ((l >> 1) & 3)) << 4)));
#pragma unroll
            for (int t = 0; t < 4; ++t) mx_split<T>(w[t], A[4 * c + t], B[4 * c + t]);
        }
    }
}

// 16 values of this lane and the 16 of its neighbour (lane ^ 1) are a block: its codes (8 bytes a
// lane) and, on lanes 0 and 8 of the half-warp, the word of four scales that starts there.
__device__ __forceinline__ void quantize16(const float (&v)[16], int l, uint2 &code, uint32_t &word) {
    uint32_t m = 0;
#pragma unroll
    for (int t = 0; t < 16; ++t) m = max(m, __float_as_uint(v[t]) & 0x7FFFFFFFu);
    m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
    const uint32_t e = mx_exponent(m);
    const float inv = mx_inverse(e);
    float s[16];
#pragma unroll
    for (int t = 0; t < 16; ++t) s[t] = __fmul_rn(v[t], inv);
    code = make_uint2(mx_pack8(s), mx_pack8(s + 8));
    // lanes 0, 2, 4, 6 (8, 10, 12, 14) hold the bytes of a word
    const uint32_t two = e | (__shfl_down_sync(0xFFFFFFFFu, e, 2) << 8);
    word = two | (__shfl_down_sync(0xFFFFFFFFu, two, 4) << 16);
}

// One half-warp ("slot") quantizes a pair of 256-value groups: a lane holds 16 consecutive values
// of each, so a block of 32 is two lanes, codes leave as 8 bytes a lane (128 consecutive bytes a
// group) and scales as one 4-byte word a 128-wide tile.
template <int T, bool ROT, bool VEC>
__global__ void __launch_bounds__(128) quantize_rows_kernel(const RowArgs a) {
    __shared__ __align__(128) uint8_t tiles[ROT ? 8 * 2048 : 16];
    const int slot = threadIdx.x >> 4, l = threadIdx.x & 15;
    const uint32_t f0 = (blockIdx.x * 8u + slot) * 2u;
    const uint32_t r0 = f0 / a.G, g0 = f0 - r0 * a.G;
    const uint32_t r1 = g0 + 1 == a.G ? r0 + 1 : r0, g1 = g0 + 1 == a.G ? 0 : g0 + 1;
    const bool ok0 = f0 < a.groups, ok1 = f0 + 1 < a.groups;
    const uint8_t *base = static_cast<const uint8_t *>(a.x);
    float A[16] = {}, B[16] = {};
    if (ok0) load16<T, VEC>(a, base + r0 * a.ldx * mx_size(T), g0 * 256 + l * 16, A);
    if (ok1) load16<T, VEC>(a, base + r1 * a.ldx * mx_size(T), g1 * 256 + l * 16, B);
    if constexpr (ROT) {
        f2 P[16];
#pragma unroll
        for (int t = 0; t < 16; ++t) P[t] = mk2(A[t], B[t]);
        const uint32_t tile = smem_u32(tiles) + slot * 2048;
        rotate_pair(P, tile, l);
        settle_pair<T>(P, tile, l, A, B);
        if (a.rotated) {
            uint8_t *out = static_cast<uint8_t *>(a.rotated);
            if (ok0) store16<T>(out + static_cast<int64_t>(r0) * a.K * mx_size(T), g0 * 256 + l * 16, A);
            if (ok1) store16<T>(out + static_cast<int64_t>(r1) * a.K * mx_size(T), g1 * 256 + l * 16, B);
        }
        if (!a.codes) return;
    }
    uint2 c0, c1;
    uint32_t w0, w1;
    quantize16(A, l, c0, w0);
    quantize16(B, l, c1, w1);
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
    float v[2][32];
    if (VEC && c + 1 < a.cols) {
        // all loads before the first use: two columns of a 16-bit type are one word
        using Word = typename std::conditional<T == kMxF32, float2, uint32_t>::type;
        Word w[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            w[i] = Word{};
            if (r0 + i < end) w[i] = __ldg(reinterpret_cast<const Word *>(x + (static_cast<int64_t>(r0 + i) * a.ldx + c) * mx_size(T)));
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            if constexpr (T == kMxF32) {
                v[0][i] = w[i].x;
                v[1][i] = w[i].y;
            } else {
                mx_split<T>(w[i], v[0][i], v[1][i]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const int64_t at = static_cast<int64_t>(r0 + i) * a.ldx + c;
            v[0][i] = r0 + i < end && c < a.cols ? mx_load1<T>(x, at) : 0.f;
            v[1][i] = r0 + i < end && c + 1 < a.cols ? mx_load1<T>(x, at + 1) : 0.f;
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) m = max(m, __float_as_uint(v[h][i]) & 0x7FFFFFFFu);
        const uint32_t e = mx_exponent(m);
        const float inv = mx_inverse(e);
#pragma unroll
        for (int i = 0; i < 32; ++i) v[h][i] = __fmul_rn(v[h][i], inv);
        uint4 code = make_uint4(mx_pack8(v[h]), mx_pack8(v[h] + 8), mx_pack8(v[h] + 16), mx_pack8(v[h] + 24));
        *reinterpret_cast<uint4 *>(&s_code[lane * 2 + h][warp * 4]) = code;
        s_scale[lane * 2 + h][warp] = static_cast<uint8_t>(e);
    }
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
    uint32_t K, KB, KT, halves;  // halves: runs of 16 values of a row
    int64_t total;               // rows * halves
    uint32_t matrix_rows, matrix_tiles;
};

// 16 values a thread: 8 bytes of codes, a scale byte, 32 (64) bytes out
template <int T, bool VEC>
__global__ void __launch_bounds__(256) values_kernel(const ValueArgs a) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= a.total) return;
    const int64_t r = i / a.halves;
    const uint32_t h = static_cast<uint32_t>(i - r * a.halves);
    const int64_t b = r / a.matrix_rows;
    const int64_t sr = b * a.matrix_tiles * 128 + (r - b * a.matrix_rows);
    const uint2 code = __ldg(reinterpret_cast<const uint2 *>(a.codes + r * a.KB * 16 + h * 8));
    const float s = mx_scale(__ldg(a.scales + mx_scale_word(sr, h >> 3, a.KT) + ((h >> 1) & 3)));
    float v[16];
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        const uint32_t w = t < 4 ? code.x : code.y;
        mx_unpack2((w >> (8 * (t & 3))) & 0xFFu, v[2 * t], v[2 * t + 1]);
        v[2 * t] = __fmul_rn(v[2 * t], s);
        v[2 * t + 1] = __fmul_rn(v[2 * t + 1], s);
    }
    uint8_t *row = static_cast<uint8_t *>(a.out) + r * a.K * mx_size(T);
    const uint32_t c = h * 16;
    if (VEC && c + 16 <= a.K) {
        store16<T>(row, c, v);
    } else {
#pragma unroll
        for (int t = 0; t < 16; ++t)
            if (c + t < a.K) mx_store1<T>(row, c + t, v[t]);
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
    a.matrix_tiles = static_cast<uint32_t>((matrix_rows + 127) / 128);
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
    a.halves = static_cast<uint32_t>((K + 15) / 16);
    a.total = rows * a.halves;
    a.matrix_rows = static_cast<uint32_t>(matrix_rows);
    a.matrix_tiles = static_cast<uint32_t>((matrix_rows + 127) / 128);
    const int64_t blocks = (a.total + 255) / 256;
    if (blocks > 0x7FFFFFFFll) {
        set_error("mxfp4: too many values");
        return 2;
    }
    const bool vec = aligned(out, 16) && (K * mx_size(type)) % 16 == 0;
    cudaStream_t s = as_stream(stream);
    const uint32_t grid = static_cast<uint32_t>(blocks);
    switch (type * 2 + (vec ? 1 : 0)) {
        case 0: values_kernel<kMxBf16, false><<<grid, 256, 0, s>>>(a); break;
        case 1: values_kernel<kMxBf16, true><<<grid, 256, 0, s>>>(a); break;
        case 2: values_kernel<kMxF16, false><<<grid, 256, 0, s>>>(a); break;
        case 3: values_kernel<kMxF16, true><<<grid, 256, 0, s>>>(a); break;
        case 4: values_kernel<kMxF32, false><<<grid, 256, 0, s>>>(a); break;
        default: values_kernel<kMxF32, true><<<grid, 256, 0, s>>>(a); break;
    }
    return launch_status("mxfp4_dequantize");
}

}  // extern "C"
