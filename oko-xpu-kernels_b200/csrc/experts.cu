// Tokens to their experts and back.
//
//   sort     expert ids [tokens, fan] -> the slots (token, choice) in the order of their experts,
//            a stable counting sort: equal ids keep their order, slots of no expert (an id outside
//            [0, experts)) come last
//   gather   x [tokens, W] -> rows in that order; a slot of no expert gives a zero row
//   combine  y[t] = sum_j w[t, j] rows[position[t, j]] over the slots that an expert took, in 32
//            bits, j ascending; without weights (w = 1) it is also the gradient of gather
//   combine's gradient: rows'[p] = w dy[t] and w'[t, j] = <dy[t], rows[position[t, j]]>
//
// Beside the order the sort gives each slot's row among rows padded to whole 128-row tiles an
// expert (the tiles of MXFP4 scales): tiles[e] is the first tile of expert e.
//
// Gather, combine and the gradient move bytes: each element is read and written once, 16 bytes a
// thread and access where the rows' alignment allows it.
#include <cuda_runtime.h>

#include <string>
#include <type_traits>

#include "internal.h"
#include "mx4quant.cuh"
#include "xpu_kernels/convrot.h"

namespace xpuint8 {
namespace {

// ------------------------------------------------------------------------------------------ sort

constexpr int kSortThreads = 256, kSortWarps = kSortThreads / 32;
constexpr int kMaxExperts = 1024;
constexpr int64_t kSortChunks = 128;  // CTAs of a large sort: each reads every chunk's counts
constexpr int64_t kSortOne = 4096;    // slots that one CTA sorts alone, in one launch

struct SortArgs {
    const void *ids;
    int wide;                   // 8-byte ids
    int64_t n, chunk;           // slots; slots of a CTA (a multiple of kSortThreads)
    int experts;
    int32_t *order, *positions, *scale_rows, *offsets, *tiles;
    int32_t *counts;            // [chunks][experts + 1]
};

__device__ __forceinline__ int sort_key(const SortArgs &a, int64_t i) {
    const int64_t id = a.wide ? __ldg(static_cast<const long long *>(a.ids) + i)
                              : static_cast<int64_t>(__ldg(static_cast<const int32_t *>(a.ids) + i));
    return id >= 0 && id < a.experts ? static_cast<int>(id) : a.experts;
}

// slots [begin, end) of warp w of this CTA's chunk
__device__ __forceinline__ void warp_range(const SortArgs &a, int w, int64_t &begin, int64_t &end) {
    const int64_t first = blockIdx.x * a.chunk, last = min(first + a.chunk, a.n);
    const int64_t each = a.chunk / kSortWarps;
    begin = min(first + w * each, last);
    end = min(begin + each, last);
}

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const SortArgs a) {
    extern __shared__ int32_t s_count[];  // [experts + 1]
    const int bins = a.experts + 1;
    pdl_trigger();
    for (int e = threadIdx.x; e < bins; e += kSortThreads) s_count[e] = 0;
    __syncthreads();
    const int64_t first = blockIdx.x * a.chunk, last = min(first + a.chunk, a.n);
    for (int64_t i = first + threadIdx.x; i < last; i += kSortThreads) atomicAdd(&s_count[sort_key(a, i)], 1);
    __syncthreads();
    for (int e = threadIdx.x; e < bins; e += kSortThreads) a.counts[blockIdx.x * static_cast<int64_t>(bins) + e] = s_count[e];
}

// exclusive sums of v over the CTA's threads (thread t gets the sum of threads before it)
__device__ __forceinline__ int exclusive_sum(int v, int *s_warp, int &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xFFFFFFFFu, x, d);
        if (lane >= d) x += y;
    }
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
        if (w < warp) before += s_warp[w];
        total += s_warp[w];
    }
    __syncthreads();
    return before + x - v;
}

// Every CTA counts its warps' slots by expert, adds the other chunks' counts (from the table, or
// none where one CTA holds all slots), and walks its slots in order: among 32 neighbours a slot's
// rank is the number of lower lanes with the same expert.  131072 slots by 128 experts: 3 and 9 us for the
// two kernels, the second's by the walk, one round trip through shared memory for 32 slots; up to 4096
// slots one CTA does all in one launch, 3.5 us for 64.
__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(const SortArgs a) {
    extern __shared__ int32_t smem[];
    const int bins = a.experts + 1;
    int32_t *s_next = smem;                          // [warps][bins]: the next row of each
    int32_t *s_offset = s_next + kSortWarps * bins;  // [bins + 1]
    int32_t *s_tile = s_offset + bins + 1;           // [bins]
    __shared__ int s_warp[kSortWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = threadIdx.x; i < kSortWarps * bins; i += kSortThreads) s_next[i] = 0;
    __syncthreads();
    int64_t begin, end;
    warp_range(a, warp, begin, end);
    for (int64_t i = begin + lane; i < end; i += 32) atomicAdd(&s_next[warp * bins + sort_key(a, i)], 1);
    __syncthreads();
    // totals of all chunks and counts of the earlier ones: the table's rows go around the warps, a
    // lane a column
    int32_t *s_total = s_offset, *s_before = s_tile;  // read into registers before those are written
    for (int e = threadIdx.x; e < bins; e += kSortThreads) s_total[e] = s_before[e] = 0;
    __syncthreads();
    if (gridDim.x == 1) {
        for (int e = threadIdx.x; e < bins; e += kSortThreads) {
            int sum = 0;
            for (int w = 0; w < kSortWarps; ++w) sum += s_next[w * bins + e];
            s_total[e] = sum;
        }
    } else {
        pdl_wait();
        for (int e = lane; e < bins; e += 32) {
            int sum = 0, early = 0;
#pragma unroll 16
            for (int c = warp; c < static_cast<int>(gridDim.x); c += kSortWarps) {
                const int v = a.counts[c * static_cast<int64_t>(bins) + e];
                sum += v;
                early += c < static_cast<int>(blockIdx.x) ? v : 0;
            }
            atomicAdd(&s_total[e], sum);
            atomicAdd(&s_before[e], early);
        }
    }
    __syncthreads();
    const int per = (bins + kSortThreads - 1) / kSortThreads;
    int sum = 0, tile_sum = 0;
    int total[(kMaxExperts + kSortThreads) / kSortThreads], before[(kMaxExperts + kSortThreads) / kSortThreads];
#pragma unroll
    for (int q = 0; q < (kMaxExperts + kSortThreads) / kSortThreads; ++q) {
        const int e = threadIdx.x * per + q;
        const bool in = q < per && e < bins;
        total[q] = in ? s_total[e] : 0;
        before[q] = in ? s_before[e] : 0;
        sum += total[q];
        if (in && e < a.experts) tile_sum += (total[q] + 127) / 128;
    }
    int all, all_tiles;
    int offset = exclusive_sum(sum, s_warp, all), tile = exclusive_sum(tile_sum, s_warp, all_tiles);
#pragma unroll
    for (int q = 0; q < (kMaxExperts + kSortThreads) / kSortThreads; ++q) {
        const int e = threadIdx.x * per + q;
        if (q < per && e < bins) {
            s_offset[e] = offset;
            s_tile[e] = tile;
            int at = offset + before[q];
            for (int w = 0; w < kSortWarps; ++w) {
                const int v = s_next[w * bins + e];
                s_next[w * bins + e] = at;
                at += v;
            }
            offset += total[q];
            tile += e < a.experts ? (total[q] + 127) / 128 : 0;
        }
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int e = threadIdx.x; e < bins; e += kSortThreads) {
            a.offsets[e] = s_offset[e];
            a.tiles[e] = s_tile[e];
        }
    for (int64_t i0 = begin; i0 < end; i0 += 32) {
        const int64_t i = i0 + lane;
        const bool in = i < end;
        const int key = in ? sort_key(a, i) : -1;
        const unsigned same = __match_any_sync(0xFFFFFFFFu, key);
        const int rank = __popc(same & ((1u << lane) - 1));
        int at = 0;
        if (in) at = s_next[warp * bins + key] + rank;
        __syncwarp();
        if (in && rank == 0) s_next[warp * bins + key] += __popc(same);
        __syncwarp();
        if (in) {
            a.positions[i] = at;
            a.order[at] = static_cast<int32_t>(i);
            a.scale_rows[i] = key < a.experts ? s_tile[key] * 128 + (at - s_offset[key]) : -1;
        }
    }
}

// ------------------------------------------------------------------------------ gather, combine

struct MoveArgs {
    const void *in;            // gather: x [tokens, W]; combine: rows [slots, W]
    int64_t ld_in;
    void *out;                 // contiguous
    const float *weights;      // combine: [tokens, fan] or null
    const int32_t *positions, *scale_rows;
    int64_t total;             // tokens * units
    Divisor units;             // vectors of a row
    uint32_t fan, W;
};

// vector i: its token and place in the row
__device__ __forceinline__ void place(const MoveArgs &a, int64_t i, int64_t &t, uint32_t &u) {
    t = a.total < 0x7FFFFFFF ? a.units(static_cast<uint32_t>(i)) : i / a.units.d;
    u = static_cast<uint32_t>(i - t * a.units.d);
}

// One thread: one vector of VEC elements of a token, read once and written to the token's rows.  Memory
// bounds it: 16384 tokens, 8 rows each of 2048 bf16, 604 MB in 97 us, 6.2 TB/s.
template <int T, int VEC>
__global__ void __launch_bounds__(256) gather_kernel(const MoveArgs a) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= a.total) return;
    int64_t t;
    uint32_t u;
    place(a, i, t, u);
    constexpr int kBytes = VEC * mx_size(T);
    using Word = typename std::conditional<kBytes == 16, uint4, typename std::conditional<kBytes == 4, uint32_t, uint16_t>::type>::type;
    const Word v = __ldg(reinterpret_cast<const Word *>(static_cast<const uint8_t *>(a.in) + (t * a.ld_in + static_cast<int64_t>(u) * VEC) * mx_size(T)));
    const Word zero{};
#pragma unroll 4
    for (uint32_t j = 0; j < a.fan; ++j) {
        const int64_t slot = t * a.fan + j;
        const int64_t row = __ldg(a.positions + slot);
        const bool taken = __ldg(a.scale_rows + slot) >= 0;
        *reinterpret_cast<Word *>(static_cast<uint8_t *>(a.out) + (row * a.W + static_cast<int64_t>(u) * VEC) * mx_size(T)) = taken ? v : zero;
    }
}

// VEC values as loaded (one, or 16 bytes of them), and in 32 bits
template <int T, int VEC>
struct VecWord {
    using type = uint4;
};
template <int T>
struct VecWord<T, 1> {
    using type = float;
};
template <int T, int VEC>
__device__ __forceinline__ typename VecWord<T, VEC>::type load_word(const void *p, int64_t at) {
    if constexpr (VEC == 1) return mx_load1<T>(p, at);
    else return __ldcs(reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(p) + at * mx_size(T)));
}
template <int T, int VEC>
__device__ __forceinline__ void spread(const typename VecWord<T, VEC>::type &w, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = w;
    } else {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if constexpr (T == kMxF32) v[q] = __uint_as_float(u[q]);
            else mx_split<T>(u[q], v[2 * q], v[2 * q + 1]);
        }
    }
}
template <int T, int VEC>
__device__ __forceinline__ void store_vec(void *p, int64_t at, const float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        mx_store1<T>(p, at, v[0]);
    } else {
        uint32_t u[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if constexpr (T == kMxF32) u[q] = __float_as_uint(v[q]);
            else u[q] = mx_join<T>(v[2 * q], v[2 * q + 1]);
        }
        __stcs(reinterpret_cast<uint4 *>(static_cast<uint8_t *>(p) + at * mx_size(T)), make_uint4(u[0], u[1], u[2], u[3]));
    }
}

constexpr int kFan = 8;   // choices whose products a gradient keeps at a time
constexpr int kRows = 4;  // rows whose loads are in flight together

// One thread: one vector of a token's sum.  Four rows' loads at a time and five CTAs an SM: with eight
// and three the same bytes take 119 us instead of 96 (16384 tokens, 8 rows each of 2048 bf16: 6.3 TB/s).
template <int T, int VEC>
__global__ void __launch_bounds__(256, 5) combine_kernel(const MoveArgs a) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= a.total) return;
    int64_t t;
    uint32_t u;
    place(a, i, t, u);
    const int64_t c = static_cast<int64_t>(u) * VEC;
    float sum[VEC] = {};
    for (uint32_t j0 = 0; j0 < a.fan; j0 += kRows) {
        float w[kRows];
        int32_t row[kRows];
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
            const int64_t slot = t * a.fan + j0 + j;
            row[j] = j0 + j < a.fan && __ldg(a.scale_rows + slot) >= 0 ? __ldg(a.positions + slot) : -1;
            w[j] = row[j] >= 0 && a.weights ? __ldg(a.weights + slot) : 1.f;
        }
        typename VecWord<T, VEC>::type v[kRows];
#pragma unroll
        for (int j = 0; j < kRows; ++j)
            if (row[j] >= 0) v[j] = load_word<T, VEC>(a.in, row[j] * a.ld_in + c);
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
            if (row[j] < 0) continue;
            float x[VEC];
            spread<T, VEC>(v[j], x);
#pragma unroll
            for (int q = 0; q < VEC; ++q) sum[q] = __fmaf_rn(w[j], x[q], sum[q]);
        }
    }
    store_vec<T, VEC>(a.out, t * a.W + c, sum);
}

struct GradArgs {
    const void *dy, *rows;   // [tokens, W], [slots, W]
    int64_t ld_dy, ld_rows;
    const float *weights;
    void *grad_rows;         // [slots, W] contiguous
    float *grad_weights;     // [tokens, fan]
    const int32_t *positions, *scale_rows;
    uint32_t fan, W;
};

constexpr int kGradThreads = 256;

// One CTA a token: its dy is read once for eight choices, whose rows are read once for the product
// and the sum's terms.  The sums go lane by lane, then warp by warp, in a fixed order.  Four CTAs an SM:
// 190 us for 16384 tokens, 8 rows each of 2048 bf16 (1.14 GB, 6.0 TB/s), 232 with two.
template <int T, int VEC>
__global__ void __launch_bounds__(kGradThreads, 4) combine_grad_kernel(const GradArgs a) {
    __shared__ float s_sum[kFan][kGradThreads / 32];
    const int64_t t = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (uint32_t j0 = 0; j0 < a.fan; j0 += kFan) {
        float dot[kFan], w[kFan];
        int32_t row[kFan];  // its row; ~row: of no expert, a zero gradient
        int n = 0;
#pragma unroll
        for (int j = 0; j < kFan; ++j) {
            dot[j] = 0.f;
            row[j] = 0;
            w[j] = 0.f;
            if (j0 + j < a.fan) {
                const int64_t slot = t * a.fan + j0 + j;
                row[j] = __ldg(a.positions + slot);
                if (__ldg(a.scale_rows + slot) < 0) row[j] = ~row[j];
                else w[j] = __ldg(a.weights + slot);
                n = j + 1;
            }
        }
        for (int64_t c = threadIdx.x * VEC; c < a.W; c += kGradThreads * VEC) {
            float d[VEC];
            spread<T, VEC>(load_word<T, VEC>(a.dy, t * a.ld_dy + c), d);
#pragma unroll
            for (int h = 0; h < kFan; h += kRows) {
                if (h >= n) break;
                typename VecWord<T, VEC>::type v[kRows];
#pragma unroll
                for (int j = 0; j < kRows; ++j)
                    if (h + j < n && row[h + j] >= 0) v[j] = load_word<T, VEC>(a.rows, row[h + j] * a.ld_rows + c);
#pragma unroll
                for (int j = 0; j < kRows; ++j) {
                    if (h + j >= n) break;
                    const bool taken = row[h + j] >= 0;
                    float u[VEC], g[VEC];
                    if (taken) {
                        spread<T, VEC>(v[j], u);
#pragma unroll
                        for (int q = 0; q < VEC; ++q) dot[h + j] = __fmaf_rn(d[q], u[q], dot[h + j]);
                    }
#pragma unroll
                    for (int q = 0; q < VEC; ++q) g[q] = taken ? __fmul_rn(w[h + j], d[q]) : 0.f;
                    store_vec<T, VEC>(a.grad_rows, static_cast<int64_t>(taken ? row[h + j] : ~row[h + j]) * a.W + c, g);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < kFan; ++j) {
#pragma unroll
            for (int m = 16; m >= 1; m >>= 1) dot[j] = __fadd_rn(dot[j], __shfl_xor_sync(0xFFFFFFFFu, dot[j], m));
            if (lane == 0) s_sum[j][warp] = dot[j];
        }
        __syncthreads();
        if (threadIdx.x < kFan && j0 + threadIdx.x < a.fan) {
            float sum = 0.f;
#pragma unroll
            for (int q = 0; q < kGradThreads / 32; ++q) sum = __fadd_rn(sum, s_sum[threadIdx.x][q]);
            a.grad_weights[t * a.fan + j0 + threadIdx.x] = sum;
        }
        __syncthreads();
    }
}

bool aligned(const void *p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
cudaStream_t as_stream(const void *s) { return static_cast<cudaStream_t>(const_cast<void *>(s)); }

int64_t sort_chunk(int64_t n) {
    if (n <= kSortOne) return (n + kSortThreads - 1) / kSortThreads * kSortThreads;
    const int64_t each = (n + kSortChunks - 1) / kSortChunks;
    const int64_t least = 1024;
    return (each > least ? each + kSortThreads - 1 : least) / kSortThreads * kSortThreads;
}

int check_move(const char *what, int32_t type, std::initializer_list<const void *> values,
               std::initializer_list<const void *> words, int64_t tokens, int64_t fan, int64_t width) {
    if (type < 0 || type > 2) {
        set_error(std::string(what) + ": the element type must be 0 (bf16), 1 (fp16) or 2 (fp32)");
        return 2;
    }
    if (tokens <= 0 || fan <= 0 || width <= 0 || tokens * fan > 0x7FFFFF00ll || width > 0x7FFFFF00ll) {
        set_error(std::string(what) + ": tokens, fan and width must be positive and fit in 31 bits");
        return 2;
    }
    for (const void *p : values)
        if (!p || !aligned(p, mx_size(type))) {
            set_error(std::string(what) + ": a required pointer is null or not aligned to its elements");
            return 2;
        }
    for (const void *p : words)
        if (!p || !aligned(p, 4)) {
            set_error(std::string(what) + ": a required pointer is null or not 4-byte aligned");
            return 2;
        }
    return 0;
}

int bad_stride(const char *what) {
    set_error(std::string(what) + ": the row stride must be at least the width");
    return 2;
}

template <int T>
int launch_move(cudaStream_t s, MoveArgs &a, bool gather, int64_t tokens, bool vec, const char *what) {
    constexpr int kVec = 16 / mx_size(T);
    a.units = Divisor::of(vec ? a.W / kVec : a.W);
    a.total = tokens * a.units.d;
    const int64_t blocks = (a.total + 255) / 256;
    if (blocks > 0x7FFFFFFFll) {
        set_error(std::string(what) + ": too many elements");
        return 2;
    }
    const uint32_t grid = static_cast<uint32_t>(blocks);
    if (gather) {
        if (vec) gather_kernel<T, kVec><<<grid, 256, 0, s>>>(a);
        else gather_kernel<T, 1><<<grid, 256, 0, s>>>(a);
    } else {
        if (vec) combine_kernel<T, kVec><<<grid, 256, 0, s>>>(a);
        else combine_kernel<T, 1><<<grid, 256, 0, s>>>(a);
    }
    return launch_status(what);
}

int move(cudaStream_t s, MoveArgs &a, int type, bool gather, int64_t tokens, const char *what) {
    const int es = mx_size(type);
    const bool vec = aligned(a.in, 16) && aligned(a.out, 16) && (a.ld_in * es) % 16 == 0 &&
                     (static_cast<int64_t>(a.W) * es) % 16 == 0;
    switch (type) {
        case kMxBf16: return launch_move<kMxBf16>(s, a, gather, tokens, vec, what);
        case kMxF16: return launch_move<kMxF16>(s, a, gather, tokens, vec, what);
        default: return launch_move<kMxF32>(s, a, gather, tokens, vec, what);
    }
}

template <int T>
void launch_grad(cudaStream_t s, const GradArgs &a, int64_t tokens, bool vec) {
    if (vec) combine_grad_kernel<T, 16 / mx_size(T)><<<static_cast<uint32_t>(tokens), kGradThreads, 0, s>>>(a);
    else combine_grad_kernel<T, 1><<<static_cast<uint32_t>(tokens), kGradThreads, 0, s>>>(a);
}

}  // namespace
}  // namespace xpuint8

using namespace xpuint8;

extern "C" {

int64_t xpuint8_expert_sort_workspace_bytes(int64_t slots, int64_t experts) {
    if (slots < 0 || slots > 0x7FFFFF00ll || experts <= 0 || experts > kMaxExperts) return -1;
    if (slots <= kSortOne) return 0;
    const int64_t chunk = sort_chunk(slots);
    return (slots + chunk - 1) / chunk * (experts + 1) * 4;
}

int xpuint8_expert_sort_stream(const void *stream, const void *ids, int32_t id_bytes,
                               int64_t slots, int64_t experts, int32_t *order,
                               int32_t *positions, int32_t *scale_rows, int32_t *offsets,
                               int32_t *tiles, void *workspace) {
    if (slots <= 0 || slots > 0x7FFFFF00ll || experts <= 0 || experts > kMaxExperts ||
        (id_bytes != 4 && id_bytes != 8)) {
        set_error("expert_sort: 1 to 2^31 - 256 slots, 1 to 1024 experts, ids of 4 or 8 bytes");
        return 2;
    }
    const bool one = slots <= kSortOne;
    if (!ids || !aligned(ids, id_bytes) || !order || !positions || !scale_rows || !offsets || !tiles ||
        (!one && (!workspace || !aligned(workspace, 4)))) {
        set_error("expert_sort: a required pointer is null or misaligned");
        return 2;
    }
    SortArgs a{};
    a.ids = ids;
    a.wide = id_bytes == 8;
    a.n = slots;
    a.chunk = sort_chunk(slots);
    a.experts = static_cast<int>(experts);
    a.order = order;
    a.positions = positions;
    a.scale_rows = scale_rows;
    a.offsets = offsets;
    a.tiles = tiles;
    a.counts = static_cast<int32_t *>(workspace);
    const int bins = a.experts + 1;
    const uint32_t chunks = static_cast<uint32_t>((slots + a.chunk - 1) / a.chunk);
    cudaStream_t s = as_stream(stream);
    if (chunks > 1) {
        sort_count_kernel<<<chunks, kSortThreads, bins * 4, s>>>(a);
        if (int rc = launch_status("expert_sort")) return rc;
    }
    const size_t smem = static_cast<size_t>(kSortWarps * bins + bins + 1 + bins) * 4;  // at most 41 KB
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(chunks);
    cfg.blockDim = dim3(kSortThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    // the counts are the only thing that the kernel before may still be writing: with one CTA the
    // launch is an ordinary one
    cfg.numAttrs = chunks > 1 ? 1 : 0;
    cudaLaunchKernelEx(&cfg, sort_place_kernel, a);
    return launch_status("expert_sort");
}

int xpuint8_expert_gather_stream(const void *stream, const void *x, int32_t type, int64_t ldx,
                                 void *out, const int32_t *positions, const int32_t *scale_rows,
                                 int64_t tokens, int64_t fan, int64_t width) {
    if (int rc = check_move("expert_gather", type, {x, out}, {positions, scale_rows}, tokens, fan, width)) return rc;
    if (ldx < width) return bad_stride("expert_gather");
    MoveArgs a{};
    a.in = x;
    a.ld_in = ldx;
    a.out = out;
    a.positions = positions;
    a.scale_rows = scale_rows;
    a.fan = static_cast<uint32_t>(fan);
    a.W = static_cast<uint32_t>(width);
    return move(as_stream(stream), a, type, true, tokens, "expert_gather");
}

int xpuint8_expert_combine_stream(const void *stream, const void *rows, int32_t type,
                                  int64_t ld_rows, const float *weights, void *out,
                                  const int32_t *positions, const int32_t *scale_rows,
                                  int64_t tokens, int64_t fan, int64_t width) {
    if (int rc = check_move("expert_combine", type, {rows, out}, {positions, scale_rows}, tokens, fan, width)) return rc;
    if (ld_rows < width) return bad_stride("expert_combine");
    if (!aligned(weights, 4)) {
        set_error("expert_combine: the weights are not 4-byte aligned");
        return 2;
    }
    MoveArgs a{};
    a.in = rows;
    a.ld_in = ld_rows;
    a.out = out;
    a.weights = weights;
    a.positions = positions;
    a.scale_rows = scale_rows;
    a.fan = static_cast<uint32_t>(fan);
    a.W = static_cast<uint32_t>(width);
    return move(as_stream(stream), a, type, false, tokens, "expert_combine");
}

int xpuint8_expert_combine_grad_stream(const void *stream, const void *dy, int32_t type,
                                       int64_t ld_dy, const void *rows, int64_t ld_rows,
                                       const float *weights, void *grad_rows, float *grad_weights,
                                       const int32_t *positions, const int32_t *scale_rows,
                                       int64_t tokens, int64_t fan, int64_t width) {
    if (int rc = check_move("expert_combine_grad", type, {dy, rows, grad_rows},
                            {weights, grad_weights, positions, scale_rows}, tokens, fan, width))
        return rc;
    if (ld_dy < width || ld_rows < width) return bad_stride("expert_combine_grad");
    GradArgs a{};
    a.dy = dy;
    a.rows = rows;
    a.ld_dy = ld_dy;
    a.ld_rows = ld_rows;
    a.weights = weights;
    a.grad_rows = grad_rows;
    a.grad_weights = grad_weights;
    a.positions = positions;
    a.scale_rows = scale_rows;
    a.fan = static_cast<uint32_t>(fan);
    a.W = static_cast<uint32_t>(width);
    const int es = mx_size(type);
    const bool vec = aligned(dy, 16) && aligned(rows, 16) && aligned(grad_rows, 16) &&
                     (ld_dy * es) % 16 == 0 && (ld_rows * es) % 16 == 0 && (width * es) % 16 == 0;
    cudaStream_t s = as_stream(stream);
    switch (type) {
        case kMxBf16: launch_grad<kMxBf16>(s, a, tokens, vec); break;
        case kMxF16: launch_grad<kMxF16>(s, a, tokens, vec); break;
        default: launch_grad<kMxF32>(s, a, tokens, vec); break;
    }
    return launch_status("expert_combine_grad");
}

}  // extern "C"
