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
// Gather, combine and the gradient move bytes: each element is read and written once.
#include <cuda_runtime.h>

#include <cstring>
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
    Divisor units;             // threads of a row
    uint32_t fan, W;
};

// A row is read and written in accesses of A bytes: 16 where the rows' alignment allows it, else 8, 4, or
// an element.  Of the narrow ones a thread takes several, which lie a row's threads apart, so that
// neighbouring lanes touch neighbouring bytes and a slot's place is looked up once for all of them
// (16384 tokens, 4 rows each of 2047 bf16: gather 87 us where one element a thread takes 143, combine
// 147 against 350, the gradient 170 against 353; rows of 2046 67, 71 and 129 us, of 2048 54, 53 and 115).
template <int T, int A>
struct Access {
    using Word = typename std::conditional<A == 16, uint4, typename std::conditional<A == 8, uint2, typename std::conditional<A == 4, uint32_t, uint16_t>::type>::type>::type;
    static constexpr int kValues = A / mx_size(T);
    static constexpr int kCount = A == 16 ? 1 : A == 8 ? 2 : 4;             // a thread's accesses
    static constexpr int kSums = A == 16 ? 1 : A == 8 ? 4 : A == 4 ? 8 : 4;  // in combine
};
template <int T, int A>
__device__ __forceinline__ typename Access<T, A>::Word load_word(const void *p, int64_t at) {
    return __ldcs(reinterpret_cast<const typename Access<T, A>::Word *>(static_cast<const uint8_t *>(p) + at * mx_size(T)));
}
template <int T, int A>
__device__ __forceinline__ void store_word(void *p, int64_t at, const typename Access<T, A>::Word &w) {
    __stcs(reinterpret_cast<typename Access<T, A>::Word *>(static_cast<uint8_t *>(p) + at * mx_size(T)), w);
}
// an access's values in 32 bits, and back
template <int T, int A>
__device__ __forceinline__ void spread(const typename Access<T, A>::Word &w, float *v) {
    if constexpr (A >= 8) {
        uint32_t u[A / 4];
        memcpy(u, &w, A);
#pragma unroll
        for (int q = 0; q < A / 4; ++q) {
            if constexpr (T == kMxF32) v[q] = __uint_as_float(u[q]);
            else mx_split<T>(u[q], v[2 * q], v[2 * q + 1]);
        }
    } else if constexpr (T == kMxF32) {
        v[0] = __uint_as_float(w);
    } else if constexpr (A == 4) {
        mx_split<T>(w, v[0], v[1]);
    } else {
        float none;
        mx_split<T>(w, v[0], none);
    }
}
template <int T, int A>
__device__ __forceinline__ typename Access<T, A>::Word join(const float *v) {
    if constexpr (A >= 8) {
        typename Access<T, A>::Word w;
        uint32_t u[A / 4];
#pragma unroll
        for (int q = 0; q < A / 4; ++q) {
            if constexpr (T == kMxF32) u[q] = __float_as_uint(v[q]);
            else u[q] = mx_join<T>(v[2 * q], v[2 * q + 1]);
        }
        memcpy(&w, u, A);
        return w;
    } else if constexpr (T == kMxF32) {
        return __float_as_uint(v[0]);
    } else if constexpr (A == 4) {
        return mx_join<T>(v[0], v[1]);
    } else {
        return static_cast<uint16_t>(mx_join<T>(v[0], 0.f));
    }
}

// thread i: its token and its place in the row
__device__ __forceinline__ void place(const MoveArgs &a, int64_t i, int64_t &t, uint32_t &u) {
    t = a.total < 0x7FFFFFFF ? a.units(static_cast<uint32_t>(i)) : i / a.units.d;
    u = static_cast<uint32_t>(i - t * a.units.d);
}

// One thread: its accesses of a token, read once and written to the token's rows.  Memory bounds it:
// 16384 tokens, 8 rows each of 2048 bf16, 604 MB in 97 us, 6.2 TB/s.
template <int T, int A>
__global__ void __launch_bounds__(256) gather_kernel(const MoveArgs a) {
    using C = Access<T, A>;
    constexpr int U = C::kCount;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= a.total) return;
    int64_t t;
    uint32_t u;
    place(a, i, t, u);
    const uint32_t step = a.units.d * C::kValues, c = u * C::kValues;
    typename C::Word v[U];
#pragma unroll
    for (int q = 0; q < U; ++q)
        if (U == 1 || c + q * step < a.W) v[q] = load_word<T, A>(a.in, t * a.ld_in + c + q * step);
    const typename C::Word zero{};
#pragma unroll 4
    for (uint32_t j = 0; j < a.fan; ++j) {
        const int64_t slot = t * a.fan + j;
        const int64_t row = __ldg(a.positions + slot);
        const bool taken = __ldg(a.scale_rows + slot) >= 0;
#pragma unroll
        for (int q = 0; q < U; ++q)
            if (U == 1 || c + q * step < a.W) store_word<T, A>(a.out, row * a.W + c + q * step, taken ? v[q] : zero);
    }
}

constexpr int kFan = 8;   // choices whose products a gradient keeps at a time
constexpr int kRows = 4;  // rows whose loads are in flight together

// One thread: its accesses of a token's sum.  Four rows' loads at a time and five CTAs an SM: with eight
// and three the same bytes take 119 us instead of 96 (16384 tokens, 8 rows each of 2048 bf16: 6.3 TB/s).
template <int T, int A>
__global__ void __launch_bounds__(256, A == 16 ? 5 : A == 2 ? 4 : 3) combine_kernel(const MoveArgs a) {
    using C = Access<T, A>;
    constexpr int U = C::kSums, E = C::kValues;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= a.total) return;
    int64_t t;
    uint32_t u;
    place(a, i, t, u);
    const uint32_t step = a.units.d * E, c = u * E;
    float sum[U * E] = {};
    for (uint32_t j0 = 0; j0 < a.fan; j0 += kRows) {
        float w[kRows];
        int32_t row[kRows];
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
            const int64_t slot = t * a.fan + j0 + j;
            row[j] = j0 + j < a.fan && __ldg(a.scale_rows + slot) >= 0 ? __ldg(a.positions + slot) : -1;
            w[j] = row[j] >= 0 && a.weights ? __ldg(a.weights + slot) : 1.f;
        }
        typename C::Word v[kRows][U];
#pragma unroll
        for (int j = 0; j < kRows; ++j)
#pragma unroll
            for (int q = 0; q < U; ++q)
                if (row[j] >= 0 && (U == 1 || c + q * step < a.W)) v[j][q] = load_word<T, A>(a.in, row[j] * a.ld_in + c + q * step);
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
            if (row[j] < 0) continue;
#pragma unroll
            for (int q = 0; q < U; ++q) {
                float x[E];
                spread<T, A>(v[j][q], x);
#pragma unroll
                for (int e = 0; e < E; ++e) sum[q * E + e] = __fmaf_rn(w[j], x[e], sum[q * E + e]);
            }
        }
    }
#pragma unroll
    for (int q = 0; q < U; ++q)
        if (U == 1 || c + q * step < a.W) store_word<T, A>(a.out, t * a.W + c + q * step, join<T, A>(sum + q * E));
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


// One CTA a token: its dy is read once for eight choices, whose rows are read once for the product
// and the sum's terms.  The sums go lane by lane, then warp by warp, in a fixed order.  Four CTAs of
// 256 threads an SM: 190 us for 16384 tokens, 8 rows each of 2048 bf16 (1.14 GB, 6.0 TB/s), 232 with two.
// Narrow rows go to CTAs of 64 threads (4 rows of 256 fp32 or 300 bf16 a token: below 48 us, the host's
// time, in place of 63 and 90).
template <int T, int A, int THREADS>
__global__ void __launch_bounds__(THREADS, (A == 16 ? 4 : 3) * 256 / THREADS) combine_grad_kernel(const GradArgs a) {
    using C = Access<T, A>;
    constexpr int U = C::kCount, E = C::kValues;
    __shared__ float s_sum[kFan][THREADS / 32];
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
        constexpr uint32_t step = THREADS * E;
        for (uint32_t c = threadIdx.x * E; c < a.W; c += step * U) {
            typename C::Word dw[U];
#pragma unroll
            for (int q = 0; q < U; ++q)
                if (U == 1 || c + q * step < a.W) dw[q] = load_word<T, A>(a.dy, t * a.ld_dy + c + q * step);
#pragma unroll
            for (int h = 0; h < kFan; h += kRows) {
                if (h >= n) break;
                typename C::Word v[kRows][U];
#pragma unroll
                for (int j = 0; j < kRows; ++j)
#pragma unroll
                    for (int q = 0; q < U; ++q)
                        if (h + j < n && row[h + j] >= 0 && (U == 1 || c + q * step < a.W)) v[j][q] = load_word<T, A>(a.rows, row[h + j] * a.ld_rows + c + q * step);
#pragma unroll
                for (int j = 0; j < kRows; ++j) {
                    if (h + j >= n) break;
                    const bool taken = row[h + j] >= 0;
                    const int64_t at = static_cast<int64_t>(taken ? row[h + j] : ~row[h + j]) * a.W + c;
#pragma unroll
                    for (int q = 0; q < U; ++q) {
                        if (U > 1 && c + q * step >= a.W) break;
                        float d[E], u[E], g[E];
                        spread<T, A>(dw[q], d);
                        if (taken) {
                            spread<T, A>(v[j][q], u);
#pragma unroll
                            for (int e = 0; e < E; ++e) dot[h + j] = __fmaf_rn(d[e], u[e], dot[h + j]);
                        }
#pragma unroll
                        for (int e = 0; e < E; ++e) g[e] = taken ? __fmul_rn(w[h + j], d[e]) : 0.f;
                        store_word<T, A>(a.grad_rows, at + q * step, join<T, A>(g));
                    }
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
            for (int q = 0; q < THREADS / 32; ++q) sum = __fadd_rn(sum, s_sum[threadIdx.x][q]);
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

// the widest access for these rows: 16 bytes, 8, 4, or an element's
int access(int type, std::initializer_list<const void *> values, std::initializer_list<int64_t> strides) {
    const int es = mx_size(type);
    for (const int n : {16, 8, 4}) {
        bool ok = true;
        for (const void *p : values) ok = ok && aligned(p, n);
        for (const int64_t ld : strides) ok = ok && ld * es % n == 0;
        if (ok) return n;
    }
    return es;
}

template <int T, int A>
int launch_move(cudaStream_t s, MoveArgs &a, bool gather, int64_t tokens, const char *what) {
    const int each = Access<T, A>::kValues * (gather ? Access<T, A>::kCount : Access<T, A>::kSums);
    a.units = Divisor::of((a.W + each - 1) / each);
    a.total = tokens * a.units.d;
    const int64_t blocks = (a.total + 255) / 256;
    if (blocks > 0x7FFFFFFFll) {
        set_error(std::string(what) + ": too many elements");
        return 2;
    }
    const uint32_t grid = static_cast<uint32_t>(blocks);
    if (gather) gather_kernel<T, A><<<grid, 256, 0, s>>>(a);
    else combine_kernel<T, A><<<grid, 256, 0, s>>>(a);
    return launch_status(what);
}
template <int T>
int launch_move(cudaStream_t s, MoveArgs &a, bool gather, int64_t tokens, int bytes, const char *what) {
    if (bytes == 16) return launch_move<T, 16>(s, a, gather, tokens, what);
    if (bytes == 8) return launch_move<T, 8>(s, a, gather, tokens, what);
    if constexpr (T != kMxF32)
        if (bytes == 2) return launch_move<T, 2>(s, a, gather, tokens, what);
    return launch_move<T, 4>(s, a, gather, tokens, what);
}

int move(cudaStream_t s, MoveArgs &a, int type, bool gather, int64_t tokens, const char *what) {
    const int bytes = access(type, {a.in, a.out}, {a.ld_in, a.W});
    switch (type) {
        case kMxBf16: return launch_move<kMxBf16>(s, a, gather, tokens, bytes, what);
        case kMxF16: return launch_move<kMxF16>(s, a, gather, tokens, bytes, what);
        default: return launch_move<kMxF32>(s, a, gather, tokens, bytes, what);
    }
}

template <int T, int A>
void launch_grad(cudaStream_t s, const GradArgs &a, int64_t tokens) {
    // rows that 64 threads take at once are left to them
    const uint32_t grid = static_cast<uint32_t>(tokens);
    if (a.W <= 64 * Access<T, A>::kValues * Access<T, A>::kCount) combine_grad_kernel<T, A, 64><<<grid, 64, 0, s>>>(a);
    else combine_grad_kernel<T, A, 256><<<grid, 256, 0, s>>>(a);
}
template <int T>
void launch_grad(cudaStream_t s, const GradArgs &a, int64_t tokens, int bytes) {
    if (bytes == 16) launch_grad<T, 16>(s, a, tokens);
    else if (bytes == 8) launch_grad<T, 8>(s, a, tokens);
    else if (bytes == 4) launch_grad<T, 4>(s, a, tokens);
    else if constexpr (T != kMxF32) launch_grad<T, 2>(s, a, tokens);
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
    const int bytes = access(type, {dy, rows, grad_rows}, {ld_dy, ld_rows, width});
    cudaStream_t s = as_stream(stream);
    switch (type) {
        case kMxBf16: launch_grad<kMxBf16>(s, a, tokens, bytes); break;
        case kMxF16: launch_grad<kMxF16>(s, a, tokens, bytes); break;
        default: launch_grad<kMxF32>(s, a, tokens, bytes); break;
    }
    return launch_status("expert_combine_grad");
}

}  // extern "C"
