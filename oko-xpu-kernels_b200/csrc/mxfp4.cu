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
#include "mx4.h"
#include "mx4quant.cuh"
#include "xpu_kernels/convrot.h"

namespace xpuint8 {
namespace {

struct RowArgs {
    const void *x;
    int64_t ldx;                 // elements between rows of x
    uint8_t *codes, *scales;     // codes may be null: only the rotated values are wanted
    void *rotated;               // [rows, K] of x's type, or null
    uint32_t tasks;              // row pairs * G
    uint32_t rows;
    uint32_t K, KB, KT;          // values, 32-blocks and 128-tiles of a row
    Divisor G;                   // 256-groups of a row
    uint32_t matrix_rows;        // rows of each matrix of a stack
    uint32_t matrix_tiles;       // its 128-row tiles (0: one matrix)
    const int32_t *order;        // sorted rows: row r of x is the slot order[r]
    const int32_t *positions;    // [slots] the row of codes that a slot's row goes to
    const int32_t *scale_rows;   // [slots] the row of scales; negative: no expert takes it
    uint32_t fan;                // slots of a token
    bool wide, wide_out;         // rows of x and of the rotated values are 32-byte aligned
};

// a run to a row that is 16-byte aligned (wide: 32)
template <int T>
__device__ __forceinline__ void store_run(void *row, uint32_t c, const Run<T> &r, bool wide) {
    uint8_t *q = static_cast<uint8_t *>(row) + static_cast<int64_t>(c) * mx_size(T);
    if (wide) {
#pragma unroll
        for (int j = 0; j < Run<T>::kWords / 8; ++j) store_v8(q + 32 * j, r.w + 8 * j);
        return;
    }
    uint4 *p = reinterpret_cast<uint4 *>(q);
#pragma unroll
    for (int j = 0; j < Run<T>::kWords / 4; ++j) p[j] = make_uint4(r.w[4 * j], r.w[4 * j + 1], r.w[4 * j + 2], r.w[4 * j + 3]);
}

enum Where { kOneMatrix = 0, kStack = 1, kExperts = 2 };

// One half-warp ("slot") quantizes the same 256-value group of two neighbouring rows: a lane holds 16
// consecutive values of each, so a block of 32 is two lanes, codes leave as 8 bytes a lane (128
// consecutive bytes a group) and scales as one 4-byte word a 128-wide tile.  Instructions bound it
// before memory does behind the rotation: 16-bit values stay packed up to the conversion (the maximum is
// of two at a time), the rotation and the scaling are packed fp32x2, and the second row's addresses are
// the first's and a constant.  bf16 [16384, 4096], 170 MB: 26.4 us (6.4 TB/s), behind the rotation 45 us,
// 68 % of the issue slots taken (a persistent loop that loads the next task early 48, scalar adds no
// faster); fp32, 304 MB, 45 and 60 us.
template <int T, bool ROT, bool VEC, int WHERE>
__global__ void __launch_bounds__(128) quantize_rows_kernel(const RowArgs a) {
    __shared__ __align__(128) uint8_t tiles[ROT ? 8 * kSlotBytes : 16];
    const int slot = threadIdx.x >> 4, l = threadIdx.x & 15;
    const uint32_t task = min(blockIdx.x * 8u + slot, a.tasks - 1);  // the last slots repeat a task: their warp's other half needs their lanes
    const uint32_t rp = a.G(task), g = task - rp * a.G.d, r = 2 * rp, c = g * 256 + l * 16;
    const bool two = r + 1 < a.rows;
    const uint8_t *row = static_cast<const uint8_t *>(a.x) + r * a.ldx * mx_size(T);
    const Run<T> A = load_run<T, VEC>(row, c, a.K, a.wide);
    const Run<T> B = two ? load_run<T, VEC>(row + a.ldx * mx_size(T), c, a.K, a.wide) : zero_run<T>();
    pdl_trigger();
    PairCodes q;
    if constexpr (ROT) {
        const uint32_t tile = smem_u32(tiles) + slot * kSlotBytes;
        rotate_to_shared<T>(A, B, tile, l);
        const Pairs<T> p = pairs_from_shared<T>(tile, l);
        if (a.rotated) {
            Run<T> u, v;
            split_pairs<T>(p, u, v);
            uint8_t *out = static_cast<uint8_t *>(a.rotated) + static_cast<int64_t>(r) * a.K * mx_size(T);
            store_run<T>(out, c, u, a.wide_out);
            if (two) store_run<T>(out + static_cast<int64_t>(a.K) * mx_size(T), c, v, a.wide_out);
        }
        if (!a.codes) return;
        q = quantize_pairs<T>(p);
    } else {
        q = quantize_runs<T>(A, B);
    }
    const uint32_t kt = g * 2 + (l >> 3);
    const bool has_code = c < a.KB * 32, has_word = (l & 7) == 0 && kt < a.KT;
    if constexpr (WHERE == kOneMatrix) {
        uint8_t *codes = a.codes + static_cast<int64_t>(r) * a.KB * 16 + c / 2;
        uint8_t *scales = a.scales + mx_scale_word(r, kt, a.KT);
        if (has_code) {
            *reinterpret_cast<uint2 *>(codes) = q.c0;
            if (two) *reinterpret_cast<uint2 *>(codes + a.KB * 16) = q.c1;
        }
        if (has_word) {  // r is even: the next row is the next 16 bytes of the tile
            *reinterpret_cast<uint32_t *>(scales) = q.w0;
            if (two) *reinterpret_cast<uint32_t *>(scales + 16) = q.w1;
        }
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (h && !two) break;
            for (uint32_t j = 0; j < (WHERE == kExperts ? a.fan : 1u); ++j) {
                int64_t cr = r + h, sr;
                if constexpr (WHERE == kExperts) {
                    const uint32_t at = a.order ? static_cast<uint32_t>(__ldg(a.order + r + h)) : (r + h) * a.fan + j;
                    sr = __ldg(a.scale_rows + at);
                    if (sr < 0) continue;
                    if (!a.order) cr = __ldg(a.positions + at);
                } else {
                    const uint32_t b = (r + h) / a.matrix_rows;
                    sr = static_cast<int64_t>(b) * a.matrix_tiles * 128 + (r + h - b * a.matrix_rows);
                }
                if (has_code) *reinterpret_cast<uint2 *>(a.codes + cr * a.KB * 16 + c / 2) = h ? q.c1 : q.c0;
                if (has_word) *reinterpret_cast<uint32_t *>(a.scales + mx_scale_word(sr, kt, a.KT)) = h ? q.w1 : q.w0;
            }
        }
    }
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
// so that each column's 64 bytes leave together.  Memory bounds it: bf16 [16384, 4096] 27.4 us, 6.2 TB/s;
// fp32 [4097, 5120], whose rows of the result are odd, 20 us.
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
    } else if (!VEC && T != kMxF32 && blockIdx.x * 64 + 66 <= a.cols && r0 + 32 <= end) {
        // a row that begins between two words: the words one value on, whose first the lane before has
        // (lane 0 reads its own): [9001, 4001] 22 us, 38 where each value is read by itself
        const uint8_t *p = x + (static_cast<int64_t>(r0) * a.ldx + c) * 2;
        const int64_t pitch = a.ldx * 2;
        const uint32_t o0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 2, o1 = (o0 + static_cast<uint32_t>(pitch)) & 2;
        uint32_t own[32], v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const uint8_t *q = p + i * pitch;
            v[i] = __ldg(reinterpret_cast<const uint32_t *>(q + (i & 1 ? o1 : o0)));
            own[i] = 0;
            if (lane == 0) own[i] = __ldg(reinterpret_cast<const uint16_t *>(q));
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            uint32_t up = __shfl_up_sync(0xFFFFFFFFu, v[i], 1);
            if (lane == 0) up = own[i] << 16;
            const uint32_t u = (i & 1 ? o1 : o0) ? __byte_perm(up, v[i], 0x5432) : v[i];
            if constexpr (T != kMxF32) w[i] = u;
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
        for (int i = 0; i < 32; i += 2) {
            m0 = __float_as_uint(max_abs3(__uint_as_float(m0), __float_as_uint(w[i].x), __float_as_uint(w[i + 1].x)));
            m1 = __float_as_uint(max_abs3(__uint_as_float(m1), __float_as_uint(w[i].y), __float_as_uint(w[i + 1].y)));
        }
    } else {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) m = max_abs2<T>(m, w[i]);
        m &= 0x7FFF7FFFu;
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

struct BothArgs {
    const void *x;
    int64_t ldx, matrix_stride;            // elements
    uint8_t *row_codes, *row_scales;       // null: not wanted
    uint8_t *col_codes, *col_scales;
    uint32_t rows, cols;                   // of a matrix
    uint32_t KB, KT;                       // blocks and tiles along the columns
    int64_t row_matrix_codes, row_matrix_scales;
    int64_t col_pitch, col_matrix_codes, col_matrix_scales;
    uint32_t col_blocks, col_KT;           // along the rows
    const int32_t *offsets, *tiles, *order;  // experts: rows are sorted rows, taken from slot order[row]'s token
    int experts;
    uint32_t fan;                          // slots of a token; 0: x's rows are sorted already
    int subs;                              // 32-row steps of a CTA: 4, or 2 or 1 where that fills the device
    bool wide;                             // rows of x are 32-byte aligned
};

constexpr int kBothThreads = 256, kBothSlots = 16;
// the columns' codes: the 16 bytes of 32 rows in a column's 64 bytes, by columns into different banks.
// Four CTAs an SM behind the rotation, whose arithmetic they hide; three without it, padded: four take
// 70 us for 16384 x 5632 bf16, three 67.
template <bool ROT>
constexpr int kBothSmem = kBothSlots * kSlotBytes + 256 * (ROT ? 64 : 80) + 256 * 4;
template <bool ROT>
__device__ __forceinline__ uint32_t code_at(uint32_t col, uint32_t part) {
    return ROT ? col * 64 + ((part ^ ((col >> 1) & 3)) << 4) : col * 80 + part * 16;
}

// Codes along the rows and along the columns in one read: a CTA takes 128 rows (a tile of scales
// along the rows) x 256 columns (a group of the rotation), 32 rows at a time.  A slot brings two
// neighbouring rows, rotates them, quantizes them along the columns and leaves them in shared memory
// as pairs; a thread a column then takes the 32 rows from there.  Against two kernels it saves one read
// of x (two thirds of the bytes' time at 16 bits).  No pipe is at its limit: with two barriers every 32 rows,
// 58 % of the issue slots are taken and 34 % of the warps there.  In a training step eight experts' bf16
// [5632, 2048], 282 MB, take 85 us rotated (3.3 TB/s); the next rows loaded before this step's barrier
// changed nothing.
template <int T, bool ROT, bool VEC>
__global__ void __launch_bounds__(kBothThreads, T == kMxF32 ? 2 : ROT ? 4 : 3) quantize_both_kernel(const BothArgs a) {
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t slots = smem_u32(smem);
    uint8_t *s_code = smem + kBothSlots * kSlotBytes;
    uint8_t *s_scale = s_code + 256 * (ROT ? 64 : 80);
    const int slot = threadIdx.x >> 4, l = threadIdx.x & 15;
    const int row0 = blockIdx.y * 32 * a.subs, kt = row0 >> 7, sub0 = (row0 >> 5) & 3;
    const uint32_t mine = slots + slot * kSlotBytes;
    pdl_trigger();
    uint32_t begin = kt * 128u, end = a.rows;
    if (a.offsets) {
        if (kt >= __ldg(a.tiles + a.experts)) return;
        const int e = find_tile(a.tiles, a.experts, kt);
        begin = __ldg(a.offsets + e) + (kt - __ldg(a.tiles + e)) * 128;
        end = __ldg(a.offsets + e + 1);
    }
    const uint32_t c = blockIdx.x * 256 + l * 16, tile = blockIdx.x * 2 + (l >> 3);
    const uint8_t *x = static_cast<const uint8_t *>(a.x) + blockIdx.z * a.matrix_stride * mx_size(T);
    const int64_t pitch = a.ldx * mx_size(T);
    // this slot's rows of a step are `row` and the next; they move on by 32 a step
    uint32_t row = begin + sub0 * 32 + 2 * slot;
    const uint8_t *at_x = x + row * pitch;
    uint8_t *codes = a.row_codes + blockIdx.z * a.row_matrix_codes + static_cast<int64_t>(row) * a.KB * 16 + c / 2;
    // row 2 slot of 32-row step j of the tile is at 32 slot + 4 j of its 512 bytes, the next 16 bytes on
    uint8_t *scales = a.row_scales + blockIdx.z * a.row_matrix_scales + (static_cast<int64_t>(kt) * a.KT + tile) * kMxTileBytes + slot * 32 + sub0 * 4;
    const bool has_code = c < a.KB * 32, has_word = (l & 7) == 0 && tile < a.KT;
    auto bring = [&](uint32_t r, const uint8_t *from) {
        if (r >= end) return zero_run<T>();
        if (a.fan) from = x + static_cast<uint32_t>(__ldg(a.order + r)) / a.fan * pitch;
        return load_run<T, VEC>(from, c, a.cols, a.wide);
    };
    Run<T> A = bring(row, at_x), B = bring(row + 1, at_x + pitch);
#pragma unroll 1
    for (int sub = sub0; sub < sub0 + a.subs; ++sub) {
        if constexpr (ROT) rotate_to_shared<T>(A, B, mine, l);
        else runs_to_shared<T>(A, B, mine, l);
        if (a.row_codes) {
            PairCodes q;
            if constexpr (ROT) q = quantize_pairs<T>(pairs_from_shared<T>(mine, l));
            else q = quantize_runs<T>(A, B);
            const bool one = row < end, two = row + 1 < end;
            if (has_code) {
                if (one) *reinterpret_cast<uint2 *>(codes) = q.c0;
                if (two) *reinterpret_cast<uint2 *>(codes + a.KB * 16) = q.c1;
            }
            if (has_word) {
                if (one) *reinterpret_cast<uint32_t *>(scales) = q.w0;
                if (two) *reinterpret_cast<uint32_t *>(scales + 16) = q.w1;
            }
            codes += static_cast<int64_t>(a.KB) * 512;
            scales += 4;
        }
        __syncwarp();
        row += 32;
        at_x += 32 * pitch;
        if (sub + 1 < sub0 + a.subs) {
            A = bring(row, at_x);
            B = bring(row + 1, at_x + pitch);
        }
        if (!a.col_codes) continue;
        __syncthreads();
        const uint32_t at = slots + pair_at<T>(1, 0) * (threadIdx.x >> 4) + (T == kMxF32 ? 8 : 4) * (threadIdx.x & 15);
        uint32_t e;
        float v[32];
        if constexpr (T == kMxF32) {
            uint32_t m = 0;
#pragma unroll
            for (int s = 0; s < 16; ++s) {
                asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v[2 * s]), "=f"(v[2 * s + 1]) : "r"(at + s * kSlotBytes));
                m = __float_as_uint(max_abs3(__uint_as_float(m), __float_as_uint(v[2 * s]), __float_as_uint(v[2 * s + 1])));
            }
            e = mx_exponent(m);
        } else {
            uint32_t w[16], m = 0;
#pragma unroll
            for (int s = 0; s < 16; ++s) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[s]) : "r"(at + s * kSlotBytes));
#pragma unroll
            for (int s = 0; s < 16; ++s) m = max_abs2<T>(m, w[s]);
            m &= 0x7FFF7FFFu;
            e = mx_exponent(widen_bits<T>(max(m & 0xFFFFu, m >> 16)));
#pragma unroll
            for (int s = 0; s < 16; ++s) mx_split<T>(w[s], v[2 * s], v[2 * s + 1]);
        }
        const float inv = mx_inverse(e);
#pragma unroll
        for (int s = 0; s < 16; ++s) scale2(v[2 * s], v[2 * s + 1], mk2(inv, inv));
        *reinterpret_cast<uint4 *>(s_code + code_at<ROT>(threadIdx.x, sub)) = make_uint4(mx_pack8(v), mx_pack8(v + 8), mx_pack8(v + 16), mx_pack8(v + 24));
        s_scale[threadIdx.x * 4 + sub] = static_cast<uint8_t>(e);
        __syncthreads();
    }
    if (!a.col_codes) return;
    uint8_t *col_codes = a.col_codes + blockIdx.z * a.col_matrix_codes;
    uint8_t *col_scales = a.col_scales + blockIdx.z * a.col_matrix_scales;
    const int shift = a.subs >> 1;  // log2
    for (int i = threadIdx.x; i < 256 << shift; i += kBothThreads) {
        const uint32_t col = i >> shift, part = sub0 + (i & (a.subs - 1)), n = blockIdx.x * 256 + col;
        if (n < a.cols && kt * 4u + part < a.col_blocks)
            *reinterpret_cast<uint4 *>(col_codes + n * a.col_pitch + (kt * 4 + part) * 16) = *reinterpret_cast<const uint4 *>(s_code + code_at<ROT>(col, part));
    }
    const uint32_t n = blockIdx.x * 256 + threadIdx.x;
    if (n < a.cols) {
        uint8_t *to = col_scales + mx_scale_word(n, kt, a.col_KT), *from = s_scale + threadIdx.x * 4;
        if (a.subs == 4) *reinterpret_cast<uint32_t *>(to) = *reinterpret_cast<const uint32_t *>(from);
        else
            for (int q = sub0; q < sub0 + a.subs; ++q) to[q] = from[q];
    }
}

struct TurnArgs {
    const float *x;              // [rows, K], or the experts' rows that are summed
    int64_t ldx;                 // sums: elements between x's rows, a multiple of 4
    void *out;                   // [rows, K]
    uint32_t groups, G, K;
    int64_t total;               // sums: rows * units
    Divisor units;               // sums: threads of a row
    const int32_t *positions, *scale_rows;  // experts: [rows, fan], or null
    uint32_t fan;
    bool wide, vec_out, wide_out;  // rows of x are 32-byte aligned, of out 16 and 32
};

// fp32 rows, or the sums of each token's rows, turned back by the rotation and rounded once.  8192 tokens,
// two rows of 2048 each, 168 MB: 34.5 us, 4.9 TB/s, by the rotation's instructions; eight experts' dW
// [5632, 2048] to bf16, 554 MB: 92 us, 6.0 TB/s.
template <int T>
__global__ void __launch_bounds__(128) turn_kernel(const TurnArgs a) {
    __shared__ __align__(128) uint8_t tiles[8 * kSlotBytes];
    const int slot = threadIdx.x >> 4, l = threadIdx.x & 15;
    const uint32_t f0 = (blockIdx.x * 8u + slot) * 2u;
    const uint32_t r0 = f0 / a.G, g0 = f0 - r0 * a.G;
    const uint32_t r1 = g0 + 1 == a.G ? r0 + 1 : r0, g1 = g0 + 1 == a.G ? 0 : g0 + 1;
    auto bring = [&](bool ok, uint32_t r, uint32_t g) {
        Run<kMxF32> v = zero_run<kMxF32>();
        if (!ok) return v;
        const uint32_t c = g * 256 + l * 16;
        if (!a.positions) return load_run<kMxF32, true>(a.x + static_cast<int64_t>(r) * a.K, c, a.K, a.wide);
#pragma unroll 2
        for (uint32_t j = 0; j < a.fan; ++j) {
            const int64_t at = static_cast<int64_t>(r) * a.fan + j;
            if (__ldg(a.scale_rows + at) < 0) continue;
            const Run<kMxF32> u = load_run<kMxF32, true>(a.x + static_cast<int64_t>(__ldg(a.positions + at)) * a.K, c, a.K, a.wide);
#pragma unroll
            for (int t = 0; t < 16; ++t) v.w[t] = __float_as_uint(__fadd_rn(__uint_as_float(v.w[t]), __uint_as_float(u.w[t])));
        }
        return v;
    };
    const bool ok0 = f0 < a.groups, ok1 = f0 + 1 < a.groups;
    Run<kMxF32> A = bring(ok0, r0, g0), B = bring(ok1, r1, g1);
    const uint32_t tile = smem_u32(tiles) + slot * kSlotBytes;
    rotate_to_shared<kMxF32>(A, B, tile, l);
    split_pairs<kMxF32>(pairs_from_shared<kMxF32>(tile, l), A, B);
    auto put = [&](uint32_t r, uint32_t g, const Run<kMxF32> &v) {
        uint8_t *row = static_cast<uint8_t *>(a.out) + static_cast<int64_t>(r) * a.K * mx_size(T);
        const uint32_t c = g * 256 + l * 16;
        if (!a.vec_out) {
#pragma unroll
            for (int t = 0; t < 16; ++t) mx_store1<T>(row, c + t, __uint_as_float(v.w[t]));
            return;
        }
        Run<T> o;
#pragma unroll
        for (int t = 0; t < Run<T>::kWords; ++t) {
            if constexpr (T == kMxF32) o.w[t] = v.w[t];
            else o.w[t] = mx_join<T>(__uint_as_float(v.w[2 * t]), __uint_as_float(v.w[2 * t + 1]));
        }
        store_run<T>(row, c, o, a.wide_out);
    };
    if (ok0) put(r0, g0, A);
    if (ok1) put(r1, g1, B);
}

// The sums of each token's fp32 rows, in the order of its choices, rounded once.  A thread takes two words of
// four values, a row's threads apart, so that lanes read neighbouring bytes; past K a word reads the
// rows' padding.  VEC: the output's rows take words of four values too; else they leave one by one, a
// fifth of the bytes.  Memory bounds it: 5778 tokens, 4 rows each of 2363, to bf16, 246 MB, 35 us (one value
// an access 99).
template <int T, bool VEC>
__global__ void __launch_bounds__(256) sum_kernel(const TurnArgs a) {
    constexpr int U = 2;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= a.total) return;
    const int64_t r = a.total < 0x7FFFFFFF ? a.units(static_cast<uint32_t>(i)) : i / a.units.d;
    const uint32_t step = a.units.d * 4, c = static_cast<uint32_t>(i - r * a.units.d) * 4;
    float sum[U][4] = {};
#pragma unroll 4
    for (uint32_t j = 0; j < a.fan; ++j) {
        const int64_t at = r * a.fan + j;
        if (__ldg(a.scale_rows + at) < 0) continue;
        const float *x = a.x + __ldg(a.positions + at) * a.ldx + c;
#pragma unroll
        for (int q = 0; q < U; ++q)
            if (c + q * step < a.K) {
                const float4 v = __ldcs(reinterpret_cast<const float4 *>(x + q * step));
                sum[q][0] = __fadd_rn(sum[q][0], v.x);
                sum[q][1] = __fadd_rn(sum[q][1], v.y);
                sum[q][2] = __fadd_rn(sum[q][2], v.z);
                sum[q][3] = __fadd_rn(sum[q][3], v.w);
            }
    }
    uint8_t *out = static_cast<uint8_t *>(a.out) + (r * a.K + c) * mx_size(T);
#pragma unroll
    for (int q = 0; q < U; ++q) {
        uint8_t *p = out + static_cast<int64_t>(q) * step * mx_size(T);
        if constexpr (VEC) {
            if (c + q * step >= a.K) break;
            if constexpr (T == kMxF32) *reinterpret_cast<float4 *>(p) = make_float4(sum[q][0], sum[q][1], sum[q][2], sum[q][3]);
            else *reinterpret_cast<uint2 *>(p) = make_uint2(mx_join<T>(sum[q][0], sum[q][1]), mx_join<T>(sum[q][2], sum[q][3]));
        } else {
#pragma unroll
            for (uint32_t t = 0; t < 4; ++t)
                if (c + q * step + t < a.K) mx_store1<T>(p, t, sum[q][t]);
        }
    }
}

struct ValueArgs {
    const uint8_t *codes, *scales;
    void *out;
    uint32_t K, KB, KT;
    Divisor units;              // of a row: runs of 16 values or a warp's steps
    uint32_t total;             // rows * units
    Divisor matrix_rows;
    uint32_t matrix_tiles;
    bool wide;                  // rows of out are 32-byte aligned
};

// Rows that are 16-byte aligned: 16 values a thread, 8 bytes of codes, a scale byte, 32 (64) bytes out.
// bf16 [16384, 4096], 170 MB: 27.1 us, 6.3 TB/s.
template <int T>
__global__ void __launch_bounds__(256) values_kernel(const ValueArgs a) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= a.total) return;
    const uint32_t row = a.units(i), h = i - row * a.units.d, b = a.matrix_rows(row);
    const int64_t r = row, sr = static_cast<int64_t>(b) * a.matrix_tiles * 128 + (row - b * a.matrix_rows.d);
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
    store_run<T>(static_cast<uint8_t *>(a.out) + r * a.K * mx_size(T), h * 16, out, a.wide);
}

// Rows of any length and alignment: a lane makes the values of one 16-byte word of the output, which
// begins anywhere in a row's blocks, so its codes come out of two words by a funnel shift and its scales
// from the lanes that hold the warp's blocks'; a row's first and last values leave one by one.
// [5120, 4097], 95 MB in fp32: 23 us, 4.1 TB/s (a value a lane 25; 32 blocks a warp in place of 16 34); bf16
// 17 us.  The two words, the shift and the shuffles of every 16 bytes bound it.
template <int T>
__global__ void __launch_bounds__(256) odd_values_kernel(const ValueArgs a) {
    constexpr int kPer = 16 / mx_size(T), kSteps = 4;
    const uint32_t i = blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (i >= a.total) return;
    const uint32_t unit_row = a.units(i), m = a.matrix_rows(unit_row);
    const int64_t r = unit_row, sr = static_cast<int64_t>(m) * a.matrix_tiles * 128 + (unit_row - m * a.matrix_rows.d);
    const uint8_t *codes = a.codes + r * a.KB * 16;
    uint8_t *row = static_cast<uint8_t *>(a.out) + r * a.K * mx_size(T);
    const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / mx_size(T));  // values of the first word that are the row before's
    const int K = static_cast<int>(a.K);
    int c = (static_cast<int>(i - unit_row * a.units.d) * kSteps * 32 + lane) * kPer - lead;
    // all steps' loads before the first is used
    uint32_t lo[kSteps], hi[kSteps], e[kSteps];
#pragma unroll
    for (int step = 0; step < kSteps; ++step) {
        const int at = c + step * 32 * kPer;
        const int first = max(__shfl_sync(0xFFFFFFFFu, at, 0), 0) >> 5;  // the warp's first block of the step; it has nine at most
        const uint32_t mine = min(static_cast<uint32_t>(first + lane), a.KB - 1), word = static_cast<uint32_t>(max(at, 0)) >> 3;
        e[step] = __ldg(a.scales + mx_scale_word(sr, mine >> 2, a.KT) + (mine & 3));
        lo[step] = __ldg(reinterpret_cast<const uint32_t *>(codes) + min(word, a.KB * 4 - 1));
        hi[step] = __ldg(reinterpret_cast<const uint32_t *>(codes) + min(word + 1, a.KB * 4 - 1));
    }
#pragma unroll
    for (int step = 0; step < kSteps; ++step, c += 32 * kPer) {
        const int first = max(__shfl_sync(0xFFFFFFFFu, c, 0), 0) >> 5;
        const float scale = mx_scale(e[step]);
        const float s0 = __shfl_sync(0xFFFFFFFFu, scale, (max(c, 0) >> 5) - first);
        const float s1 = __shfl_sync(0xFFFFFFFFu, scale, (max(c + kPer - 1, 0) >> 5) - first);
        if (c >= 0 && c + kPer <= K) {
            const uint32_t x = __funnelshift_r(lo[step], hi[step], (c & 7) * 4);
            const int other = 32 - (c & 31);  // values from here on are the next block's
            float v[kPer];
#pragma unroll
            for (int q = 0; q < kPer; ++q) v[q] = __fmul_rn(mx_value(x >> (4 * q)), q < other ? s0 : s1);
            uint4 o;
            if constexpr (T == kMxF32) o = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
            else o = make_uint4(mx_join<T>(v[0], v[1]), mx_join<T>(v[2], v[3]), mx_join<T>(v[4], v[5]), mx_join<T>(v[6], v[7]));
            *reinterpret_cast<uint4 *>(row + static_cast<int64_t>(c) * mx_size(T)) = o;
        } else {
            for (int q = max(c, 0); q < min(c + kPer, K); ++q) {
                const uint32_t byte = __ldg(codes + (q >> 1));
                mx_store1<T>(row, q, __fmul_rn(mx_value(q & 1 ? byte >> 4 : byte), (q >> 5) == (max(c, 0) >> 5) ? s0 : s1));
            }
        }
    }
}

bool aligned(const void *p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

template <int T, int WHERE>
void launch_rows(cudaStream_t s, const RowArgs &a, bool rotate, bool vec) {
    const uint32_t grid = (a.tasks + 7) / 8;
    if (rotate) {
        if (vec) quantize_rows_kernel<T, true, true, WHERE><<<grid, 128, 0, s>>>(a);
        else quantize_rows_kernel<T, true, false, WHERE><<<grid, 128, 0, s>>>(a);
    } else {
        if (vec) quantize_rows_kernel<T, false, true, WHERE><<<grid, 128, 0, s>>>(a);
        else quantize_rows_kernel<T, false, false, WHERE><<<grid, 128, 0, s>>>(a);
    }
}
template <int T>
void launch_rows(cudaStream_t s, const RowArgs &a, bool rotate, bool vec) {
    if (a.scale_rows) launch_rows<T, kExperts>(s, a, rotate, vec);
    else if (a.matrix_tiles) launch_rows<T, kStack>(s, a, rotate, vec);
    else launch_rows<T, kOneMatrix>(s, a, rotate, vec);
}

int quantize_rows(cudaStream_t s, RowArgs &a, int type, int64_t rows, int64_t K, int64_t ldx, bool rotate) {
    const int64_t G = (K + 255) / 256;
    if ((rows + 1) / 2 * G > 0x7FFFFFF0ll) {
        set_error("mxfp4: rows x 256-groups must be below 2^32");
        return 2;
    }
    a.rows = static_cast<uint32_t>(rows);
    a.K = static_cast<uint32_t>(K);
    a.G = Divisor::of(static_cast<uint32_t>(G));
    a.KB = static_cast<uint32_t>((K + 31) / 32);
    a.KT = (a.KB + 3) / 4;
    a.ldx = ldx;
    a.tasks = static_cast<uint32_t>((rows + 1) / 2 * G);
    const bool vec = aligned(a.x, 16) && (ldx * mx_size(type)) % 16 == 0;
    a.wide = aligned(a.x, 32) && (ldx * mx_size(type)) % 32 == 0;
    a.wide_out = aligned(a.rotated, 32);
    switch (type) {
        case kMxBf16: launch_rows<kMxBf16>(s, a, rotate, vec); break;
        case kMxF16: launch_rows<kMxF16>(s, a, rotate, vec); break;
        default: launch_rows<kMxF32>(s, a, rotate, vec); break;
    }
    return launch_status("mxfp4_quantize");
}

template <int T, bool ROT, bool VEC>
int launch_both(cudaStream_t s, const BothArgs &a, dim3 grid) {
    auto kern = quantize_both_kernel<T, ROT, VEC>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kBothSmem<ROT>) != cudaSuccess)
        return launch_status("mxfp4_quantize (shared memory attribute)");
    kern<<<grid, kBothThreads, kBothSmem<ROT>, s>>>(a);
    return launch_status("mxfp4_quantize");
}
template <int T>
int launch_both(cudaStream_t s, const BothArgs &a, dim3 grid, bool rotate, bool vec) {
    if (rotate) return vec ? launch_both<T, true, true>(s, a, grid) : launch_both<T, true, false>(s, a, grid);
    return vec ? launch_both<T, false, true>(s, a, grid) : launch_both<T, false, false>(s, a, grid);
}

template <int T>
void launch_turn(cudaStream_t s, const TurnArgs &a, bool rotate, bool vec) {
    const uint32_t sums = static_cast<uint32_t>((a.total + 255) / 256);
    if (rotate) turn_kernel<T><<<(a.groups + 15) / 16, 128, 0, s>>>(a);
    else if (vec) sum_kernel<T, true><<<sums, 256, 0, s>>>(a);
    else sum_kernel<T, false><<<sums, 256, 0, s>>>(a);
}

}  // namespace

int mx4_quantize_rows(cudaStream_t s, const void *x, int type, int64_t ldx, uint8_t *codes, uint8_t *scales, void *rotated, int64_t rows,
                      int64_t K, int64_t matrix_rows, bool rotate) {
    RowArgs a{};
    a.x = x;
    a.codes = codes;
    a.scales = scales;
    a.rotated = rotated;
    a.matrix_rows = static_cast<uint32_t>(matrix_rows);
    a.matrix_tiles = matrix_rows == rows ? 0 : static_cast<uint32_t>((matrix_rows + 127) / 128);
    a.fan = 1;
    return quantize_rows(s, a, type, rows, K, ldx, rotate);
}

int mx4_quantize_sorted(cudaStream_t s, const void *x, int type, int64_t ldx, uint8_t *codes, uint8_t *scales, void *rotated,
                        const int32_t *order, const int32_t *positions, const int32_t *scale_rows, int64_t rows, int64_t fan,
                        int64_t K, bool rotate) {
    RowArgs a{};
    a.x = x;
    a.codes = codes;
    a.scales = scales;
    a.rotated = rotated;
    a.order = order;
    a.positions = positions;
    a.scale_rows = scale_rows;
    a.matrix_rows = 1;
    a.fan = static_cast<uint32_t>(fan);
    return quantize_rows(s, a, type, rows, K, ldx, rotate);
}

int mx4_quantize_columns(cudaStream_t s, const void *x, int type, int64_t ldx, uint8_t *codes, uint8_t *scales, int64_t rows,
                         int64_t cols, int64_t matrices, const int32_t *offsets, const int32_t *tiles, int64_t experts, int64_t max_tiles) {
    const bool sorted = offsets != nullptr;
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

int mx4_quantize_both(cudaStream_t s, const Mx4Both &b) {
    const bool sorted = b.offsets != nullptr;
    // columns alone of what is not rotated nor gathered: the kernel made for them
    if (!b.row_codes && !b.rotate && !b.fan)
        return mx4_quantize_columns(s, b.x, b.type, b.ldx, b.col_codes, b.col_scales, b.rows, b.cols, b.matrices, b.offsets, b.tiles, b.experts, b.max_tiles);
    BothArgs a{};
    a.x = b.x;
    a.ldx = b.ldx;
    a.matrix_stride = b.rows * b.ldx;
    a.row_codes = b.row_codes;
    a.row_scales = b.row_scales;
    a.col_codes = b.col_codes;
    a.col_scales = b.col_scales;
    a.rows = static_cast<uint32_t>(b.rows);
    a.cols = static_cast<uint32_t>(b.cols);
    a.KB = static_cast<uint32_t>((b.cols + 31) / 32);
    a.KT = (a.KB + 3) / 4;
    a.row_matrix_codes = b.rows * a.KB * 16;
    a.row_matrix_scales = (b.rows + 127) / 128 * a.KT * static_cast<int64_t>(kMxTileBytes);
    a.col_blocks = static_cast<uint32_t>(sorted ? b.max_tiles * 4 : (b.rows + 31) / 32);
    a.col_KT = static_cast<uint32_t>(sorted ? b.max_tiles : (b.rows + 127) / 128);
    a.col_pitch = static_cast<int64_t>(a.col_blocks) * 16;
    a.col_matrix_codes = a.col_pitch * b.cols;
    a.col_matrix_scales = (b.cols + 127) / 128 * a.col_KT * static_cast<int64_t>(kMxTileBytes);
    a.offsets = b.offsets;
    a.tiles = b.tiles;
    a.order = b.order;
    a.experts = static_cast<int>(b.experts);
    a.fan = static_cast<uint32_t>(b.fan);
    if (a.col_KT > 65535u || b.matrices > 65535) {
        set_error("mxfp4: at most 8388480 rows along the contraction and 65535 matrices");
        return 2;
    }
    const bool vec = aligned(b.x, 16) && (b.ldx * mx_size(b.type)) % 16 == 0;
    a.wide = aligned(b.x, 32) && (b.ldx * mx_size(b.type)) % 32 == 0;
    // 128 rows a CTA write each column's 64 bytes together; fewer rows where the CTAs would not fill the
    // device twice (three or four fit an SM): [4096, 1280] takes 12.7 us in 160 CTAs of four steps, 10.5 in 640
    const int64_t ctas = (b.cols + 255) / 256 * a.col_KT * b.matrices;
    a.subs = 4;
    while (a.subs > 1 && ctas * (4 / a.subs) < 6 * num_sms() && a.col_KT * (8 / a.subs) <= 65535) a.subs /= 2;
    const dim3 grid(static_cast<uint32_t>((b.cols + 255) / 256), a.col_KT * (4 / a.subs), static_cast<uint32_t>(b.matrices));
    switch (b.type) {
        case kMxBf16: return launch_both<kMxBf16>(s, a, grid, b.rotate, vec);
        case kMxF16: return launch_both<kMxF16>(s, a, grid, b.rotate, vec);
        default: return launch_both<kMxF32>(s, a, grid, b.rotate, vec);
    }
}

int mx4_turn(cudaStream_t s, const float *x, int64_t ldx, void *out, int type, int64_t rows, int64_t K, const int32_t *positions,
             const int32_t *scale_rows, int64_t fan, bool rotate) {
    TurnArgs a{};
    a.x = x;
    a.ldx = ldx;
    a.out = out;
    a.G = static_cast<uint32_t>((K + 255) / 256);
    a.K = static_cast<uint32_t>(K);
    a.units = Divisor::of(static_cast<uint32_t>((K + 7) / 8));  // eight values a thread
    a.total = rows * a.units.d;
    if (rows * a.G > 0x7FFFFFF0ll || (a.total + 255) / 256 > 0x7FFFFFFFll) {
        set_error("mxfp4: rows x 256-groups must be below 2^31");
        return 2;
    }
    a.groups = static_cast<uint32_t>(rows * a.G);
    a.positions = positions;
    a.scale_rows = scale_rows;
    a.fan = static_cast<uint32_t>(fan);
    a.wide = aligned(x, 32);
    a.vec_out = aligned(out, 16);
    a.wide_out = aligned(out, 32);
    const bool vec = K % 4 == 0 && aligned(out, 4 * mx_size(type));
    switch (type) {
        case kMxBf16: launch_turn<kMxBf16>(s, a, rotate, vec); break;
        case kMxF16: launch_turn<kMxF16>(s, a, rotate, vec); break;
        default: launch_turn<kMxF32>(s, a, rotate, vec); break;
    }
    return launch_status("mxfp4_turn");
}

namespace {

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
    return mx4_quantize_rows(as_stream(stream), x, type, ldx, codes, scales, rotated, rows, K, matrix_rows, rotate != 0);
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
    return mx4_quantize_sorted(as_stream(stream), x, type, ldx, codes, scales, rotated, order, positions, scale_rows, rows, fan, K, rotate != 0);
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
    return mx4_quantize_columns(as_stream(stream), x, type, ldx, codes, scales, rows, cols, matrices, offsets, tiles, experts, max_tiles);
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
    a.matrix_rows = Divisor::of(static_cast<uint32_t>(matrix_rows));
    a.matrix_tiles = static_cast<uint32_t>((matrix_rows + 127) / 128);
    const bool vec = aligned(out, 16) && (K * mx_size(type)) % 16 == 0 && K % 16 == 0;
    a.wide = aligned(out, 32) && (K * mx_size(type)) % 32 == 0;
    const int64_t span = 4 * 32 * (16 / mx_size(type));  // values of a warp, and up to a word's more before the row
    const int64_t units = vec ? K / 16 : (K + 16 / mx_size(type) - 1 + span - 1) / span;
    if (rows * units > 0x7FFFFFF0ll) {
        set_error("mxfp4: rows x runs of 16 values must be below 2^31");
        return 2;
    }
    a.units = Divisor::of(static_cast<uint32_t>(units));
    a.total = static_cast<uint32_t>(rows * units);
    const int64_t blocks = vec ? (a.total + 255ll) / 256 : (a.total + 7ll) / 8;
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
