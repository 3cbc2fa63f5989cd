// MXFP4 products on the 5th-generation tensor cores (tcgen05, kind::mxf4 with block scales).
//
//   D[m, n] = sum over blocks b of sa[m, b] sb[n, b] sum over k in b of a[m, k] b[n, k]  (+ bias[n])
//
// A [M, K] and B [N, K] in MXFP4 (mx4.cuh), the sums in 32 bits, one rounding to the output's type.
// The tensor cores multiply the codes and the scales exactly; what is rounded before the end is the
// 32-bit running sum.
//
//   dense        D = A B^T
//   rows         A's rows are grouped by expert (offsets), each expert has a B of its own
//                (its matrices follow one another): D's rows are A's rows
//   contraction  A and B hold all experts' contractions one after another, each padded to whole
//                128-value tiles (tiles): D is one matrix an expert
//
// Two kernels.  pair_kernel: CTA pairs (one CTA an SM) walk 256 x bn output tiles, for many rows:
// bound by the tensor cores.  few_kernel: for few rows a weight, where reading the weights counts:
// the weight's rows are the MMA's 128 lanes and the tokens its columns, a cluster of CTAs splits
// the contraction and adds its parts through distributed shared memory in a fixed order.
//
// Scales travel as stored: a TMA box of whole 512-byte tiles into shared memory, tcgen05.cp
// (32x128b, the four-fold copy) into tensor memory: 128 rows x 4 blocks are 4 columns of 4 bytes a
// lane.  An MMA takes 64 values of K, two blocks, whose scale bytes 0-1 or 2-3 of those columns its
// instruction descriptor names.
//
// Every mbarrier wait is bounded (common.cuh: mbar_wait); on a timeout the kernel records the site
// in g_mx4_fault and in the host's word, drains its own TMA loads and MMAs, frees its TMEM and returns;
// its output is not complete, and the next call is refused.  No load uses cluster multicast.
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <mutex>
#include <string>

#include "internal.h"
#include "mx4.h"
#include "mx4quant.cuh"
#include "tmap.h"
#include "xpu_kernels/convrot.h"

namespace xpuint8 {

__device__ int g_mx4_fault = 0;

namespace {

constexpr int kMaxExperts = 1024;
enum Mode { kDense = 0, kRows = 1, kContraction = 2 };

// -------------------------------------------------------------------- instructions and descriptors

// kind::mxf4 instruction descriptor: bits 4-5 B's scale bytes (0 or 2), 7-9 and 10-11 the types
// (1 = E2M1), 17-22 N >> 3, 23 the scales' type (1 = E8M0), 27-28 M >> 7, 29-30 A's scale bytes
__host__ __device__ constexpr uint32_t idesc_mx4(int M, int N, int half) {
    return (static_cast<uint32_t>(half * 2) << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(N >> 3) << 17) |
           (1u << 23) | (static_cast<uint32_t>(M >> 7) << 27) | (static_cast<uint32_t>(half * 2) << 29);
}
// shared-memory descriptor of a 512-byte scale tile: 32 rows of 16 bytes, no swizzle, 8-row groups
// 128 bytes apart
__device__ __forceinline__ uint64_t scale_desc(uint32_t saddr) {
    return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(128 >> 4) << 32) | (static_cast<uint64_t>(1) << 46);
}
template <int CTAS>
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
    if constexpr (CTAS == 2) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
    else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
template <int CTAS>
__device__ __forceinline__ void umma_mx4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if constexpr (CTAS == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
}

// Where a wait that gives up leaves its site (0: one that gave up because another had): the device's word,
// which makes the other waits give up too, and the host's, which the next call reads.  Not inlined: in the
// few-row kernel, whose CTAs are short, the code itself costs time (16 tokens, 4 of 64 experts 28.5 us, 29.9 inlined).
__device__ __noinline__ void record_fault(int *word, int *host, int site) {
    if (site) atomicCAS(word, 0, site);
    const int first = *reinterpret_cast<volatile int *>(word);
    *reinterpret_cast<volatile int *>(host) = first ? first : 196;
    __threadfence_system();
}
struct Fault {
    int *word, *host;
    __device__ __forceinline__ void at(int site) const { record_fault(word, host, site); }
};

// bounded wait that ignores other threads' faults: only to drain this CTA's own asynchronous work
__device__ __forceinline__ void drain_wait(uint32_t bar, uint32_t parity, const Fault &fault) {
    const uint64_t t0 = global_timer_ns();
    for (uint32_t it = 0; it < kWaitMaxIters; ++it) {
        if (mbar_try_wait(bar, parity)) return;
        if ((it & 255u) == 0u && global_timer_ns() - t0 > kWaitTimeoutNs) break;
    }
    fault.at(199);
}

// one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// mbar_wait by a whole warp: the same answer in every lane
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, const Fault &fault, int site, uint64_t timeout_ns = kWaitTimeoutNs) {
    if (__all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, fault.word, site, timeout_ns))) return true;
    fault.at(0);
    return false;
}

// ------------------------------------------------------------------------------------- pair kernel

constexpr int BK = 256;               // values of K a k-block: 128 bytes of codes a row
constexpr int kCodeRow = 128;         // bytes
constexpr int kScaleBlock = 1024;     // bytes of 128 rows' scales a k-block (two tiles)
constexpr int kGroupM = 16;

struct PairArgs {
    void *out;
    int64_t ldo;                      // elements
    const float *bias;
    int M, N;                         // of D, each matrix
    int num_m, num_n;                 // 256-row and bn-column tiles of a matrix (dense, contraction)
    int nk, last_steps;               // k-blocks; K = 64 steps in the last
    int mode;
    const int32_t *offsets, *tiles;   // experts
    int experts;
    int b_tiles;                      // rows: 128-row scale tiles of each expert's B
    int64_t rows;                     // rows: D's rows, the ones of no expert among them
    int tma_out;                      // D can be stored by the TMA unit
    int b_early;                      // B is not written by the kernel before this one
    int *host_fault;
};

template <int BN>
struct PairCfg {
    static constexpr int kABytes = 128 * kCodeRow;
    static constexpr int kBBytes = BN / 2 * kCodeRow;
    static constexpr int kSfbBytes = BN / 128 * kScaleBlock;
    static constexpr int kStageBytes = kABytes + kBBytes + kScaleBlock + kSfbBytes;
    static constexpr int kStages = BN == 256 ? 5 : 7;
    static constexpr int kEpiWarps = 8;
    static constexpr int kThreads = 64 + 32 * kEpiWarps;
    static constexpr int kEpiBytes = kEpiWarps * 4096;  // 32 rows of 128 bytes a warp
    static constexpr int kCumBytes = (kMaxExperts + 4) * 4;  // the experts' tiles, and up to 16 bytes
    static constexpr int kBarAt = kStages * kStageBytes + kEpiBytes + kCumBytes;
    static_assert(kBarAt % 16 == 0 && kStageBytes % 1024 == 0, "alignment of the barriers and tiles");
    static constexpr size_t kSmemBytes = kBarAt + 256;
    static_assert(kSmemBytes <= 232448, "over the 227 KB shared-memory limit of a CTA");
    // TMEM: two accumulators and the scales of a k-block, 24 columns.  Two of 256 columns do not fit
    // beside them, so the second begins 24 columns before the first ends; the drain of either takes
    // the shared columns first and hands them over by themselves (OVER)
    static constexpr int kScaleCol = 512 - 24;
    static constexpr int kAccCol1 = BN == 256 ? kScaleCol - BN : BN;
};

struct Tile {
    int a_row, a_sf, b_row, b_sf;  // first rows and scale tiles of A and B (the pair's)
    int k_code, k_sf;              // first byte of a row of codes; first 4-byte word of a row of scale tiles
    int nk, last_steps;
    int64_t out_row;
    int rows;                      // rows of D from out_row on that are this matrix's
    int n0;
};

// the last i with cum[i] <= t, 0 <= i < n
__device__ __forceinline__ int find_group(const int32_t *cum, int n, int t) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cum[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <int BN>
__device__ __forceinline__ Tile pair_tile(const PairArgs &a, const int32_t *s_cum, int tile) {
    Tile t;
    int mb, nb;
    if (a.mode == kRows) {
        const int e = find_group(s_cum, a.experts, tile / a.num_n);
        const int local = tile - s_cum[e] * a.num_n, mt = s_cum[e + 1] - s_cum[e];
        nb = local / mt;
        mb = local - nb * mt;
        const int begin = __ldg(a.offsets + e);
        t.a_row = begin + mb * 256;
        t.a_sf = __ldg(a.tiles + e) + mb * 2;
        t.rows = __ldg(a.offsets + e + 1) - t.a_row;
        t.out_row = t.a_row;
        t.b_row = e * a.N + nb * BN;
        t.b_sf = e * a.b_tiles + nb * (BN / 128);
        t.k_code = t.k_sf = 0;
        t.nk = a.nk;
        t.last_steps = a.last_steps;
        t.n0 = nb * BN;
        return t;
    }
    int e = 0;
    if (a.mode == kContraction) {
        e = tile / (a.num_m * a.num_n);
        tile -= e * a.num_m * a.num_n;
    }
    const int per_group = kGroupM * a.num_n;
    const int group = tile / per_group;
    const int first = group * kGroupM, size = min(kGroupM, a.num_m - first);
    const int local = tile - group * per_group;
    nb = local / size;
    mb = first + local - nb * size;
    t.a_row = mb * 256;
    t.a_sf = mb * 2;
    t.rows = a.M - t.a_row;
    t.out_row = static_cast<int64_t>(e) * a.M + t.a_row;
    t.b_row = nb * BN;
    t.b_sf = nb * (BN / 128);
    t.n0 = nb * BN;
    if (a.mode == kContraction) {
        const int k0 = __ldg(a.tiles + e), k1 = __ldg(a.tiles + e + 1);
        t.k_code = k0 * 64;
        t.k_sf = k0 * 128;
        t.nk = (k1 - k0 + 1) / 2;
        t.last_steps = ((k1 - k0) & 1) ? 2 : 4;
    } else {
        t.k_code = t.k_sf = 0;
        t.nk = a.nk;
        t.last_steps = a.last_steps;
    }
    return t;
}

__device__ __forceinline__ uint32_t stage_addr(uint32_t buf, int row, int c) { return buf + row * 128 + ((c ^ (row & 7)) << 4); }

// A box in shared memory (32 rows of 128 bytes, as the TMA store takes it) to `rows` rows of the output
// from column n on, where the TMA unit can't: rows that aren't 16-byte aligned, or strips that another
// matrix's rows follow.  A warp writes a row at a time, 4 bytes a lane; a 16-bit row that begins
// between two words goes one value on, its first and last by themselves.  The loops take rows of one
// parity, so that nothing in them branches: 4096 x 5122 x 1280 to bf16 takes 28 us so and 5121 columns
// 32, 41 where each row asks, 209 where each lane stores a row of its own, and 21 by TMA where N is
// 5120.
template <int T>
__device__ __forceinline__ void store_box(const PairArgs &a, uint32_t buf, int64_t row, int rows, int n, int lane) {
    const int left = a.N - n;  // columns that exist
    uint8_t *out = static_cast<uint8_t *>(a.out) + (row * a.ldo + n) * mx_size(T);
    const int64_t pitch = a.ldo * mx_size(T);
    auto word = [&](int r, int w) {  // 4-byte word w of row r
        uint32_t v;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(stage_addr(buf, r, w >> 2) + (w & 3) * 4));
        return v;
    };
    if (a.tma_out && left * mx_size(T) >= 128) {  // four rows at a time, 16 bytes a lane
#pragma unroll 1
        for (int r = lane >> 3; r < rows; r += 4) {
            uint32_t w[4];
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(stage_addr(buf, r, lane & 7)));
            *reinterpret_cast<uint4 *>(out + r * pitch + (lane & 7) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    } else if (T == kMxF32) {
        uint8_t *p = out + lane * 4;
        if (lane < left)
#pragma unroll 8
            for (int r = 0; r < rows; ++r, p += pitch) *reinterpret_cast<uint32_t *>(p) = word(r, lane);
    } else if (left < 64) {
#pragma unroll 1
        for (int r = 0; r < rows; ++r)
            for (int c = lane; c < left; c += 32) reinterpret_cast<uint16_t *>(out + r * pitch)[c] = static_cast<uint16_t>(word(r, c >> 1) >> (16 * (c & 1)));
    } else {
        // rows of one parity: all of them, or every other one
        const int by = pitch & 2 ? 2 : 1;
        const int64_t step = by * pitch;
#pragma unroll 1
        for (int first = 0; first < by; ++first) {
            const int count = (rows - first + by - 1) >> (by - 1);
            uint8_t *p = out + first * pitch + lane * 4;
            int r = first;
            if ((reinterpret_cast<uintptr_t>(p) & 2) == 0) {
                if (by == 1)
#pragma unroll 8
                    for (r = 0; r < rows; ++r, p += pitch) *reinterpret_cast<uint32_t *>(p) = word(r, lane);
                else
#pragma unroll 8
                    for (r = first; r < rows; r += 2, p += step) *reinterpret_cast<uint32_t *>(p) = word(r, lane);
            } else {
                const bool inner = lane < 31, edge = lane == 0 || lane == 31;
                uint8_t *e = p + (lane ? 2 : 0);
                int k = 0;  // eight rows' loads before their stores
#pragma unroll 1
                for (; k + 8 <= count; k += 8) {
                    uint32_t v[8], w[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = word(r + j * by, lane);
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j] = __byte_perm(v[j], __shfl_down_sync(0xFFFFFFFFu, v[j], 1), 0x5432);
                    if (inner) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) *reinterpret_cast<uint32_t *>(p + 2 + j * step) = w[j];
                    }
                    if (edge) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) *reinterpret_cast<uint16_t *>(e + j * step) = static_cast<uint16_t>(lane ? v[j] >> 16 : v[j]);
                    }
                    r += 8 * by;
                    p += 8 * step;
                    e += 8 * step;
                }
#pragma unroll 1
                for (; k < count; ++k, r += by, p += step, e += step) {
                    const uint32_t v = word(r, lane), next = __shfl_down_sync(0xFFFFFFFFu, v, 1);
                    if (inner) *reinterpret_cast<uint32_t *>(p + 2) = __byte_perm(v, next, 0x5432);
                    if (edge) *reinterpret_cast<uint16_t *>(e) = static_cast<uint16_t>(lane ? v >> 16 : v);
                }
            }
        }
    }
}

// A CTA pair: each CTA holds 128 of the tile's 256 rows of A, half of its BN rows of B, its own
// rows' scales and all of B's scales.
//   warp 0     TMA producer of its CTA; both CTAs' bytes complete on the leader's FULL barrier
//   warp 1     TMEM; in the leader the scale copies and MMAs of the pair
//   warps 2-9  drain: TMEM lanes 32 (w % 4) .., half of the tile's columns each
// The tensor cores bound it while the contraction is long: 8192 x 14336 x 4096 to bf16 takes 190 us alone
// (5.1 PFLOP/s; 0.32 us a k-block and 2.4 us a tile for the hand-over and the first chunk's drain),
// 223 us under a lasting load, where the 1 kW power limit holds the clock at 1.54 GHz.  Short ones
// are bound by that time a tile: 4096 x 5120 x 1280 21.2 us to bf16, 28 to fp32.
template <int BN, int T>
__global__ void __launch_bounds__(PairCfg<BN>::kThreads, 1)
    pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB,
                const __grid_constant__ CUtensorMap tmOut, const PairArgs args) {
    using C = PairCfg<BN>;
    constexpr int STAGES = C::kStages;
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {  // the 128-byte swizzle's alignment; the same in both CTAs
        if (threadIdx.x == 0) Fault{&g_mx4_fault, args.host_fault}.at(198);
        return;
    }
    const uint32_t sA = smem_u32(smem);
    const uint32_t sB = sA + STAGES * C::kABytes;
    const uint32_t sSA = sB + STAGES * C::kBBytes;
    const uint32_t sSB = sSA + STAGES * kScaleBlock;
    const uint32_t sEpi = sSB + STAGES * C::kSfbBytes;
    int32_t *s_cum = reinterpret_cast<int32_t *>(smem + STAGES * C::kStageBytes + C::kEpiBytes);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::kBarAt);
    const uint32_t bar0 = smem_u32(bars);
    auto FULL = [&](int s) { return bar0 + 8u * s; };
    auto EMPTY = [&](int s) { return bar0 + 8u * (STAGES + s); };
    auto TFULL = [&](int i) { return bar0 + 8u * (2 * STAGES + i); };
    auto TEMPTY = [&](int i) { return bar0 + 8u * (2 * STAGES + 2 + i); };
    auto OVER = [&](int i) { return bar0 + 8u * (2 * STAGES + 4 + i); };
    const uint32_t final_bar = bar0 + 8u * (2 * STAGES + 6);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * STAGES + 7);
    static_assert(8 * (2 * STAGES + 8) <= 256, "barriers");

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Fault fault{&g_mx4_fault, args.host_fault};
    const uint32_t rank = cluster_rank();
    const bool leader = rank == 0;
    const int pair = static_cast<int>(cluster_index()), npairs = static_cast<int>(cluster_count());

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(FULL(s), 1);   // leader: its expect_tx + both CTAs' bytes
            mbar_init(EMPTY(s), 1);  // the leader's commit
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(TFULL(i), 1);
            mbar_init(TEMPTY(i), 2 * C::kEpiWarps);
            mbar_init(OVER(i), C::kEpiWarps);  // the four warps of each CTA that hold the shared columns
        }
        mbar_init(final_bar, 1);
        fence_mbar_init();
        prefetch_tmap(&tmA);
        prefetch_tmap(&tmB);
        prefetch_tmap(&tmSA);
        prefetch_tmap(&tmSB);
        if (args.tma_out) prefetch_tmap(&tmOut);
    }
    cluster_sync();
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(tmem_slot), 512);
        tmem_relinquish_pair();
    }
    if (args.mode != kDense) pdl_wait();
    if (args.mode == kRows && warp == 2) {
        // s_cum[e]: 256-row tiles of the experts before e
        int sum = 0;
        for (int e0 = 0; e0 < args.experts; e0 += 32) {
            const int e = e0 + lane;
            const int v = e < args.experts ? (__ldg(args.offsets + e + 1) - __ldg(args.offsets + e) + 255) / 256 : 0;
            int x = v;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int y = __shfl_up_sync(0xFFFFFFFFu, x, d);
                if (lane >= d) x += y;
            }
            if (e < args.experts) s_cum[e] = sum + x - v;
            sum += __shfl_sync(0xFFFFFFFFu, x, 31);
        }
        if (lane == 0) s_cum[args.experts] = sum;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int num_tiles = args.mode == kRows ? s_cum[args.experts] * args.num_n
                          : args.num_m * args.num_n * (args.mode == kContraction ? args.experts : 1);

    if (warp == 0) {
        // ------------------------------------------------ TMA producer (both CTAs)
        int stage = 0;
        uint32_t ph = 0, issued = 0;
        constexpr uint32_t kTx = 2 * C::kStageBytes;
        if (!args.b_early) pdl_wait();
        // B's half and scales of k-block kb into stage st (one lane)
        auto load_b = [&](int st, int b_row, int b_sf, int k_code, int k_sf) {
            const uint32_t fb = peer_smem(FULL(st), 0);
            tma_load_2d_pair(sB + st * C::kBBytes, &tmB, fb, k_code, b_row);
            tma_load_2d_pair(sSB + st * C::kSfbBytes, &tmSB, fb, k_sf, b_sf);
        };
        // b_early: the first pass over the ring takes B before the kernel before is done
        uint32_t pre = 0;
        if (args.b_early) {
            int tile = pair, kb = 0;
            for (; pre < static_cast<uint32_t>(STAGES) && tile < num_tiles; ++pre) {
                const Tile t = pair_tile<BN>(args, s_cum, tile);
                if (lane == 0) load_b(static_cast<int>(pre), t.b_row + static_cast<int>(rank) * (BN / 2), t.b_sf, t.k_code + kb * kCodeRow, t.k_sf + kb * 256);
                if (++kb == t.nk) { kb = 0; tile += npairs; }
            }
            __syncwarp();
            pdl_wait();
        }
        bool ok = true;
        for (int tile = pair; ok && tile < num_tiles; tile += npairs) {
            const Tile t = pair_tile<BN>(args, s_cum, tile);
            const int nk = __shfl_sync(0xFFFFFFFFu, t.nk, 0);
            int k_code = __shfl_sync(0xFFFFFFFFu, t.k_code, 0), k_sf = __shfl_sync(0xFFFFFFFFu, t.k_sf, 0);
            const int a_row = __shfl_sync(0xFFFFFFFFu, t.a_row, 0) + static_cast<int>(rank) * 128, a_sf = __shfl_sync(0xFFFFFFFFu, t.a_sf, 0) + static_cast<int>(rank);
            const int b_row = __shfl_sync(0xFFFFFFFFu, t.b_row, 0) + static_cast<int>(rank) * (BN / 2), b_sf = __shfl_sync(0xFFFFFFFFu, t.b_sf, 0);
            for (int kb = 0; kb < nk; ++kb, k_code += kCodeRow, k_sf += 256) {
                if (!warp_wait(EMPTY(stage), ph ^ 1u, fault, 101)) { ok = false; break; }
                if (elect_one()) {
                    if (leader) mbar_expect_tx(FULL(stage), kTx);
                    const uint32_t fb = peer_smem(FULL(stage), 0);
                    tma_load_2d_pair(sA + stage * C::kABytes, &tmA, fb, k_code, a_row);
                    tma_load_2d_pair(sSA + stage * kScaleBlock, &tmSA, fb, k_sf, a_sf);
                    if (issued >= pre) load_b(stage, b_row, b_sf, k_code, k_sf);
                }
                __syncwarp();
                ++issued;
                if (++stage == STAGES) { stage = 0; ph ^= 1u; }
            }
        }
        pdl_trigger();
        // every load has landed once the MMAs that read it are done
        for (uint32_t s = 0; s < static_cast<uint32_t>(STAGES) && s < issued; ++s) {
            const uint32_t last = s + ((issued - 1 - s) / STAGES) * STAGES;
            drain_wait(EMPTY(s), (last / STAGES) & 1u, fault);
        }
    } else if (warp == 1) {
        if (leader) {
            // ------------------------------------------------ scale copies and MMAs (leader)
            // the whole warp walks the loop and one elected lane issues: the addresses and descriptors
            // then live in uniform registers, where these instructions take them from; in a branch of
            // one lane each operand is moved there first, and the issue itself bounds the main loop
            // (8192 x 14336 x 4096: 264 us so, 188 us this way)
            constexpr uint32_t kIdesc[2] = {idesc_mx4(256, BN, 0), idesc_mx4(256, BN, 1)};
            const uint32_t sfa = tmem_base + C::kScaleCol, sfb = sfa + 8;
            int stage = 0, count = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int tile = pair; ok && tile < num_tiles; tile += npairs) {
                const Tile t = pair_tile<BN>(args, s_cum, tile);
                const int nk = __shfl_sync(0xFFFFFFFFu, t.nk, 0), last_steps = __shfl_sync(0xFFFFFFFFu, t.last_steps, 0);
                if (nk == 0) continue;  // no contraction: the drain writes zeros
                const int acc = count & 1;
                if (!warp_wait(TEMPTY(acc), ((count >> 1) & 1) ^ 1u, fault, 102)) break;
                if (BN == 256 && count > 0 && !warp_wait(OVER(acc ^ 1), ((count - 1) >> 1) & 1, fault, 103)) break;
                tc_fence_after();
                const uint32_t d = tmem_base + static_cast<uint32_t>(acc ? C::kAccCol1 : 0);
                for (int kb = 0; kb < nk; ++kb) {
                    if (!warp_wait(FULL(stage), ph, fault, 104)) { ok = false; break; }
                    tc_fence_after();
                    const int steps = kb + 1 == nk ? last_steps : 4;
                    if (elect_one()) {
#pragma unroll
                        for (int kt = 0; kt < 2; ++kt) {
                            copy_scales<2>(sfa + 4 * kt, scale_desc(sSA + stage * kScaleBlock + kt * kMxTileBytes));
#pragma unroll
                            for (int rt = 0; rt < BN / 128; ++rt)
                                copy_scales<2>(sfb + kt * (BN / 32) + 4 * rt, scale_desc(sSB + stage * C::kSfbBytes + rt * kScaleBlock + kt * kMxTileBytes));
                        }
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) {
                            if (kk < steps)
                                umma_mx4<2>(d, umma_sdesc_sw128(sA + stage * C::kABytes + kk * 32, 16, 1024),
                                            umma_sdesc_sw128(sB + stage * C::kBBytes + kk * 32, 16, 1024), kIdesc[kk & 1],
                                            sfa + 4 * (kk >> 1), sfb + (kk >> 1) * (BN / 32), (kb | kk) != 0 ? 1u : 0u);
                        }
                        umma_commit_pair(EMPTY(stage));
                        umma_commit_pair(peer_smem(EMPTY(stage), 1));
                        if (kb + 1 == nk) {
                            umma_commit_pair(TFULL(acc));
                            umma_commit_pair(peer_smem(TFULL(acc), 1));
                        }
                    }
                    __syncwarp();
                    if (++stage == STAGES) { stage = 0; ph ^= 1u; }
                }
                if (!ok) break;
                ++count;
            }
            if (elect_one()) umma_commit_pair(final_bar);
            __syncwarp();
            drain_wait(final_bar, 0, fault);
        }
    } else {
        // ---------------------------------------------------------- drain (both CTAs)
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        // Columns of a box, 128 bytes a row: with rows of 64 bytes and two buffers a warp 8192 x 14336 x
        // 1024 takes 90.7 us against 87.0, and 191.2 against 190.3 at K 4096; two buffers of 128-byte rows
        // leave room for four stages only (85.1 and 192.9)
        constexpr int W = T == kMxF32 ? 32 : 64;
        constexpr int kChunks = BN / 2 / W;       // boxes of this warp's half
        const uint32_t buf = sEpi + (warp - 2) * 4096;
        const uint32_t tempty0 = peer_smem(TEMPTY(0), 0), over0 = peer_smem(OVER(0), 0);
        int count = 0;
        pdl_wait();
        auto hand_over = [&](uint32_t local, uint32_t remote) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (leader) mbar_arrive(local);
                else mbar_arrive_cluster(remote);
            }
        };
        for (int tile = pair; tile < num_tiles; tile += npairs) {
            const Tile t = pair_tile<BN>(args, s_cum, tile);
            const int row0 = static_cast<int>(rank) * 128 + quarter * 32;  // of the tile
            const int left = t.rows - row0;                                // rows of this warp that exist
            const int acc = count & 1;
            if (t.nk > 0) {
                // one answer for the warp: the TMEM loads and the cluster barrier below are .aligned
                if (!warp_wait(TFULL(acc), (count >> 1) & 1, fault, 105)) break;
                tc_fence_after();
            }
            const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc ? C::kAccCol1 : 0);
            // a whole 32-row strip (or dense, where the map ends with the matrix) leaves by TMA
            const bool tma = args.tma_out && (args.mode == kDense || left >= 32);
#pragma unroll 1
            for (int i = 0; i < kChunks; ++i) {
                // the columns that both accumulators use come first: the last of the first
                // accumulator, the first of the second
                const int c = half * (BN / 2) + W * (acc ? i : kChunks - 1 - i);
                const int n = t.n0 + c;
                float v[W];
                if (t.nk > 0) {
                    uint32_t r[W];
                    tmem_ld32(taddr + c, *reinterpret_cast<uint32_t(*)[32]>(r));
                    if constexpr (W == 64) tmem_ld32(taddr + c + 32, *reinterpret_cast<uint32_t(*)[32]>(r + W - 32));
                    tmem_wait_ld(*reinterpret_cast<uint32_t(*)[32]>(r));
                    if constexpr (W == 64) tmem_wait_ld(*reinterpret_cast<uint32_t(*)[32]>(r + W - 32));
                    if (BN == 256 && i == 0 && half == (acc ^ 1)) hand_over(OVER(acc), over0 + 8u * acc);
#pragma unroll
                    for (int j = 0; j < W; ++j) v[j] = __uint_as_float(r[j]);
                } else {
#pragma unroll
                    for (int j = 0; j < W; ++j) v[j] = 0.f;
                }
                if (n >= args.N || left <= 0) continue;
                if (args.bias) {
                    if (n + W <= args.N) {
#pragma unroll
                        for (int j = 0; j < W; j += 4) {
                            const float4 b = __ldg(reinterpret_cast<const float4 *>(args.bias + n + j));
                            v[j] += b.x;
                            v[j + 1] += b.y;
                            v[j + 2] += b.z;
                            v[j + 3] += b.w;
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < W; ++j)
                            if (n + j < args.N) v[j] += __ldg(args.bias + n + j);
                    }
                }
                if (lane == 0) bulk_wait_read<0>();  // the buffer's last store has read it
                __syncwarp();
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    if constexpr (T == kMxF32)
                        st_shared_v4(stage_addr(buf, lane, q), __float_as_uint(v[4 * q]), __float_as_uint(v[4 * q + 1]),
                                     __float_as_uint(v[4 * q + 2]), __float_as_uint(v[4 * q + 3]));
                    else
                        st_shared_v4(stage_addr(buf, lane, q), mx_join<T>(v[8 * q], v[8 * q + 1]), mx_join<T>(v[8 * q + 2], v[8 * q + 3]),
                                     mx_join<T>(v[8 * q + 4], v[8 * q + 5]), mx_join<T>(v[8 * q + 6], v[8 * q + 7]));
                }
                if (tma) fence_async_smem();
                __syncwarp();
                if (!tma) {
                    store_box<T>(args, buf, t.out_row + row0, min(left, 32), n, lane);
                    __syncwarp();
                } else if (lane == 0) {
                    tma_store_2d(&tmOut, buf, n, static_cast<int>(t.out_row + row0));
                    bulk_commit();
                }
            }
            if (t.nk > 0) {
                hand_over(TEMPTY(acc), tempty0 + 8u * acc);
                ++count;
            }
        }
        // rows of no expert are zero
        if (args.mode == kRows) {
            const int64_t first = __ldg(args.offsets + args.experts);
            const int64_t total = (args.rows - first) * args.N;
            const int64_t step = static_cast<int64_t>(gridDim.x) * 32 * C::kEpiWarps;
            for (int64_t i = static_cast<int64_t>(blockIdx.x) * 32 * C::kEpiWarps + threadIdx.x - 64; i < total; i += step) {
                const int64_t r = i / args.N;
                mx_store1<T>(args.out, (first + r) * args.ldo + (i - r * args.N), 0.f);
            }
        }
        if (lane == 0) bulk_wait<0>();
        __syncwarp();
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    if (warp == 1) tmem_dealloc_pair(tmem_base, 512);
}

// -------------------------------------------------------------------------------------- few kernel

// Waits until the count at `at` in shared memory is over `n`; bounded as mbar_wait is.
__device__ __forceinline__ bool count_wait(uint32_t at, int n, const Fault &fault, int site) {
    const uint64_t t0 = global_timer_ns();
    for (uint32_t it = 1; it < kWaitMaxIters; ++it) {
        int v;
        asm volatile("ld.acquire.cta.shared::cta.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
        if (v > n) return true;
        if ((it & 255u) == 0u) {
            if (*reinterpret_cast<volatile int *>(fault.word) != 0) {
                fault.at(0);
                return false;
            }
            if (global_timer_ns() - t0 > kWaitTimeoutNs) break;
        }
    }
    fault.at(site);
    return false;
}

struct FewArgs {
    void *out;
    int64_t ldo;
    const float *bias;
    int M, N;                        // tokens (dense), weight rows of a matrix
    int nk, last_steps;
    int mode;                        // dense or rows
    const int32_t *offsets, *tiles;
    int experts;
    int w_tiles;                     // 128-row scale tiles of each expert's weight
    int64_t rows;
    int w_early;                     // the weight is not written by the kernel before this one
    const void *x;                   // FUSE: the tokens themselves, K values a row
    int64_t ldx;
    int K;
    const int32_t *order;            // FUSE, rows: row r is slot order[r]'s token (fan > 0) or x's row r
    int fan;
    int vec_out;                     // four neighbouring outputs are aligned to their bytes
    int *host_fault;
};

enum Fuse { kFuseNone = 0, kFusePlain = 1, kFuseRotate = 2 };

constexpr int kFewThreads = 192;
constexpr int kFewMaxStages = 5;
constexpr int kFewCols = 256;                             // TMEM columns: two CTAs an SM
template <int FUSE>
struct FewCfg {
    static constexpr int kRing = FUSE == kFuseNone ? 100 * 1024 : 80 * 1024;  // two CTAs an SM
    static constexpr int kSlots = FUSE == kFuseRotate ? 8 * kSlotBytes : 0;   // the rotations' turns
    static constexpr int kBarAt = kRing + kSlots;
    static constexpr size_t kSmem = kBarAt + 256;
    static_assert(kBarAt % 16 == 0 && 2 * (kSmem + 1024) <= 228 * 1024, "two CTAs an SM");
};

struct FewMaps {
    CUtensorMap x[4];  // boxes of 16, 32, 64, 128 tokens
};

// One CTA: 128 rows of a weight x up to 128 tokens, over its cluster rank's share of K.
//   warp 0     TMA producer   warp 1  TMEM, scale copies and MMAs   warps 2-5  drain
// FUSE: the drain's warps first make the tokens' operand themselves: eight half-warps take pairs of
// rows of a k-block (a 256-value group), quantize them, behind the rotation or not, straight into
// the swizzled stage and its scale tiles, and arrive on the stage's FULL barrier beside the TMA
// unit's bytes.  They learn that a stage is free from a count that the producer keeps of the k-blocks
// whose stage it has found empty: a slot's next task may lie two turns of the ring on (one pair of
// rows, four stages), where the parity of EMPTY can't tell the turn.  Every CTA repeats that for its
// share of K, which the weight's bytes hide while the tokens are few, and one launch and the
// operand's way through memory are saved.
// One row of 4096 bf16, rotated, against 14336: 7.0 us, 4.4 TB/s of the weight; of that the launch and
// the rotation take 2 to 3 us, and 224 CTAs fill 148 SMs unevenly.
template <int T, int FUSE>
__global__ void __launch_bounds__(kFewThreads, 2)
    few_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmSW,
               const __grid_constant__ FewMaps tmX, const __grid_constant__ CUtensorMap tmSX, const FewArgs args) {
    using C = FewCfg<FUSE>;
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {
        if (threadIdx.x == 0) Fault{&g_mx4_fault, args.host_fault}.at(197);
        return;
    }
    uint32_t splits;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
    const uint32_t rank = cluster_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Fault fault{&g_mx4_fault, args.host_fault};
    const int nb = blockIdx.x / static_cast<int>(splits);
    int e = 0, x_row, x_sf = blockIdx.y, count;
    if (args.mode == kRows) {
        pdl_wait();
        const int64_t first = __ldg(args.offsets + args.experts), total = (args.rows - first) * args.N;
        const int64_t step = static_cast<int64_t>(gridDim.x) * gridDim.y * kFewThreads;
        for (int64_t i = (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * kFewThreads + threadIdx.x; i < total; i += step) {
            const int64_t r = i / args.N;
            mx_store1<T>(args.out, (first + r) * args.ldo + (i - r * args.N), 0.f);
        }
        if (x_sf >= __ldg(args.tiles + args.experts)) return;  // no rows: the cluster's CTAs all leave
        e = find_group(args.tiles, args.experts, x_sf);
        x_row = __ldg(args.offsets + e) + (x_sf - __ldg(args.tiles + e)) * 128;
        count = min(128, __ldg(args.offsets + e + 1) - x_row);
    } else {
        x_row = x_sf * 128;
        count = min(128, args.M - x_row);
    }
    const int box = count <= 16 ? 0 : count <= 32 ? 1 : count <= 64 ? 2 : 3;
    const int nt = 16 << box;
    const int k0 = static_cast<int>(rank) * args.nk / static_cast<int>(splits);
    const int k1 = (static_cast<int>(rank) + 1) * args.nk / static_cast<int>(splits);

    const uint32_t ring = smem_u32(smem);
    const int w_bytes = 128 * kCodeRow, x_bytes = nt * kCodeRow;
    const uint32_t stage_bytes = w_bytes + x_bytes + 2 * kScaleBlock;
    const int stages = min(kFewMaxStages, static_cast<int>(C::kRing / stage_bytes));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::kBarAt);
    const uint32_t bar0 = smem_u32(bars);
    auto FULL = [&](int s) { return bar0 + 8u * s; };
    auto EMPTY = [&](int s) { return bar0 + 8u * (kFewMaxStages + s); };
    const uint32_t done = bar0 + 8u * (2 * kFewMaxStages);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * kFewMaxStages + 1);
    const uint32_t freed = smem_u32(tmem_slot + 1);  // FUSE: k-blocks whose stage is free
    const int pairs = (count + 1) / 2;  // FUSE: row pairs of a k-block

    if (threadIdx.x == 0) {
        tmem_slot[1] = 0;
        for (int s = 0; s < kFewMaxStages; ++s) {
            mbar_init(FULL(s), FUSE == kFuseNone ? 1 : 1 + pairs);
            mbar_init(EMPTY(s), 1);
        }
        mbar_init(done, 1);
        fence_mbar_init();
        prefetch_tmap(&tmW);
        prefetch_tmap(&tmSW);
        if (FUSE == kFuseNone) {
            prefetch_tmap(&tmX.x[box]);
            prefetch_tmap(&tmSX);
        }
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_slot), kFewCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        const int w_row = __shfl_sync(0xFFFFFFFFu, e, 0) * args.N + nb * 128, w_sf = __shfl_sync(0xFFFFFFFFu, e, 0) * args.w_tiles + nb;
        const int row0 = __shfl_sync(0xFFFFFFFFu, x_row, 0);
        auto load_w = [&](int st, int kb) {
            const uint32_t at = ring + st * stage_bytes;
            tma_load_2d(at, &tmW, FULL(st), kb * kCodeRow, w_row);
            tma_load_2d(at + w_bytes + x_bytes, &tmSW, FULL(st), kb * 256, w_sf);
        };
        int pre = 0;
        if (args.mode == kDense) {
            if (args.w_early)
                for (; pre < stages && k0 + pre < k1; ++pre)
                    if (elect_one()) load_w(pre, k0 + pre);
            __syncwarp();
            pdl_wait();
        }
        int stage = 0;
        uint32_t ph = 0, issued = 0;
        for (int kb = k0; kb < k1; ++kb) {
            if (!warp_wait(EMPTY(stage), ph ^ 1u, fault, 111)) break;
            if (elect_one()) {
                if (FUSE != kFuseNone) asm volatile("st.release.cta.shared::cta.b32 [%0], %1;" ::"r"(freed), "r"(issued + 1) : "memory");
                mbar_expect_tx(FULL(stage), FUSE == kFuseNone ? stage_bytes : w_bytes + kScaleBlock);
                const uint32_t at = ring + stage * stage_bytes;
                if (static_cast<int>(issued) >= pre) load_w(stage, kb);
                if (FUSE == kFuseNone) {
                    tma_load_2d(at + w_bytes, &tmX.x[box], FULL(stage), kb * kCodeRow, row0);
                    tma_load_2d(at + w_bytes + x_bytes + kScaleBlock, &tmSX, FULL(stage), kb * 256, x_sf);
                }
            }
            __syncwarp();
            ++issued;
            if (++stage == stages) { stage = 0; ph ^= 1u; }
        }
        pdl_trigger();
        const uint32_t n = static_cast<uint32_t>(stages);
        for (uint32_t s = 0; s < n && s < issued; ++s) {
            const uint32_t last = s + ((issued - 1 - s) / n) * n;
            drain_wait(EMPTY(s), (last / n) & 1u, fault);
        }
    } else if (warp == 1) {
        const uint32_t idesc[2] = {idesc_mx4(128, nt, 0), idesc_mx4(128, nt, 1)};
        const uint32_t sfa = tmem + 128, sfb = sfa + 8;
        int stage = 0;
        uint32_t ph = 0;
        for (int kb = k0; kb < k1; ++kb) {
            if (!warp_wait(FULL(stage), ph, fault, 112)) break;
            tc_fence_after();
            const uint32_t at = ring + stage * stage_bytes;
            const uint32_t sw = at + w_bytes + x_bytes, sx = sw + kScaleBlock;
            const int steps = kb + 1 == args.nk ? args.last_steps : 4;
            if (elect_one()) {
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
                    copy_scales<1>(sfa + 4 * kt, scale_desc(sw + kt * kMxTileBytes));
                    copy_scales<1>(sfb + 4 * kt, scale_desc(sx + kt * kMxTileBytes));
                }
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    if (kk < steps)
                        umma_mx4<1>(tmem, umma_sdesc_sw128(at + kk * 32, 16, 1024), umma_sdesc_sw128(at + w_bytes + kk * 32, 16, 1024),
                                    idesc[kk & 1], sfa + 4 * (kk >> 1), sfb + 4 * (kk >> 1), kb > k0 || kk > 0 ? 1u : 0u);
                }
                umma_commit(EMPTY(stage));
            }
            __syncwarp();
            if (++stage == stages) { stage = 0; ph ^= 1u; }
        }
        if (elect_one()) umma_commit(done);
        __syncwarp();
        drain_wait(done, 0, fault);
    } else if constexpr (FUSE != kFuseNone) {
        // task t: k-block k0 + t / pairs, rows 2 (t % pairs) and the next; eight slots, task by task,
        // so every stage is freed by k-blocks whose tasks come earlier
        const int slot = (warp - 2) * 2 + (lane >> 4), l = lane & 15;
        const int tasks = (k1 - k0) * pairs;
        if (args.mode == kDense) pdl_wait();  // x
        auto bring = [&](int r, int kb) {
            if (r >= count) return zero_run<T>();
            int64_t row = x_row + r;
            if (args.fan > 0) row = __ldg(args.order + row) / args.fan;
            const uint8_t *p = static_cast<const uint8_t *>(args.x) + row * args.ldx * mx_size(T);
            return load_run<T, true>(p, kb * 256 + l * 16, args.K, false);
        };
        int t = slot, rp = 0, kb = k0;
        Run<T> A = zero_run<T>(), B = zero_run<T>();
        if (t < tasks) {
            kb = k0 + t / pairs;
            rp = t % pairs;
            A = bring(2 * rp, kb);
            B = bring(2 * rp + 1, kb);
        }
        bool ok = true;
        for (int it = 0; ok && it < tasks; it += 8) {
            const bool mine = t < tasks;
            PairCodes q;
            if constexpr (FUSE == kFuseRotate) {
                const uint32_t tile = ring + C::kRing + slot * kSlotBytes;
                rotate_to_shared<T>(A, B, tile, l);
                q = quantize_pairs<T>(pairs_from_shared<T>(tile, l));
                __syncwarp();
            } else {
                q = quantize_runs<T>(A, B);
            }
            const int r = 2 * rp, local = kb - k0, stage = local % stages;
            t += 8;
            if (t < tasks) {  // the next task's loads, before this one's wait
                kb = k0 + t / pairs;
                rp = t % pairs;
                A = bring(2 * rp, kb);
                B = bring(2 * rp + 1, kb);
            }
            if (mine) ok = count_wait(freed, local, fault, 113);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (mine && ok) {
                const uint32_t at = ring + stage * stage_bytes + w_bytes, sx = at + x_bytes + kScaleBlock;
                // K-major rows of 128 bytes, 16-byte chunk c of row r at c ^ (r & 7)
                const uint32_t a0 = at + r * 128 + (((l >> 1) ^ (r & 7)) << 4) + (l & 1) * 8;
                asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(a0), "r"(q.c0.x), "r"(q.c0.y) : "memory");
                const uint32_t a1 = at + (r + 1) * 128 + (((l >> 1) ^ ((r + 1) & 7)) << 4) + (l & 1) * 8;
                asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(a1), "r"(q.c1.x), "r"(q.c1.y) : "memory");
                if ((l & 7) == 0) {
                    const uint32_t s0 = sx + (l >> 3) * kMxTileBytes + (r & 31) * 16 + (r >> 5) * 4;
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(s0), "r"(q.w0) : "memory");
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(s0 + 16), "r"(q.w1) : "memory");
                }
                fence_async_smem();
            }
            __syncwarp();
            if (mine && ok && l == 0) mbar_arrive(FULL(stage));
        }
    }
    __syncthreads();  // every load has landed and every MMA is done: the ring is free
    tc_fence_after();
    if (splits == 1) {
        // a lane is a row of the weight: for each token a warp stores 32 neighbouring outputs
        pdl_wait();  // the output may be what the kernel before still reads
        if (warp >= 2) {
            const int quarter = warp & 3, n = nb * 128 + quarter * 32 + lane;
            const uint32_t taddr = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
            const float bias = args.bias && n < args.N ? __ldg(args.bias + n) : 0.f;
            for (int c = 0; c < nt; c += 32) {
                uint32_t r[32];
                tmem_ld32(taddr + c, r);
                tmem_wait_ld(r);
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (c + j < count && n < args.N) {
                        const float v = __uint_as_float(r[j]);
                        mx_store1<T>(args.out, (x_row + c + j) * args.ldo + n, args.bias ? __fadd_rn(v, bias) : v);
                    }
            }
        }
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        if (warp == 1) tmem_dealloc(tmem, kFewCols);
        return;
    }
    // partial sums [token][128 rows] in this CTA's shared memory
    float *part = reinterpret_cast<float *>(smem);
    if (warp >= 2) {
        const int quarter = warp & 3;
        const uint32_t taddr = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
        for (int c = 0; c < nt; c += 32) {
            uint32_t r[32];
            tmem_ld32(taddr + c, r);
            tmem_wait_ld(r);
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (c + j < count) part[(c + j) * 128 + quarter * 32 + lane] = k1 > k0 ? __uint_as_float(r[j]) : 0.f;
        }
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, kFewCols);
    pdl_wait();
    // this rank's share of the rows, four at a time: all ranks' parts, in the order of the ranks
    const int share = 128 / static_cast<int>(splits), shift = 29 - __clz(share);  // log2(share / 4)
    const uint32_t mine = smem_u32(part);
    for (int i = threadIdx.x; i < (count << shift); i += kFewThreads) {
        const int t = i >> shift, row = static_cast<int>(rank) * share + 4 * (i & ((1 << shift) - 1));
        const int n = nb * 128 + row;
        if (n >= args.N) continue;
        float v[8][4];
#pragma unroll
        for (uint32_t s = 0; s < 8; ++s)
            if (s < splits)
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[s][0]), "=f"(v[s][1]), "=f"(v[s][2]), "=f"(v[s][3]) : "r"(peer_smem(mine + (t * 128 + row) * 4, s)));
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float sum = v[0][q];
#pragma unroll
            for (uint32_t s = 1; s < 8; ++s)
                if (s < splits) sum = __fadd_rn(sum, v[s][q]);
            if (args.bias && n + q < args.N) sum = __fadd_rn(sum, __ldg(args.bias + n + q));
            v[0][q] = sum;
        }
        const int64_t at = (x_row + t) * args.ldo + n;
        if (args.vec_out && n + 4 <= args.N) {
            if constexpr (T == kMxF32) *reinterpret_cast<float4 *>(static_cast<float *>(args.out) + at) = make_float4(v[0][0], v[0][1], v[0][2], v[0][3]);
            else *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(args.out) + at) = make_uint2(mx_join<T>(v[0][0], v[0][1]), mx_join<T>(v[0][2], v[0][3]));
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (n + q < args.N) mx_store1<T>(args.out, at + q, v[0][q]);
        }
    }
    cluster_sync();  // the others have read this CTA's parts
}

// One warp waits on a barrier that nothing arrives on: the products' own wait, made to give up.
__global__ void wait_probe_kernel(uint64_t limit_ns, int site, int *host_fault) {
    __shared__ __align__(8) uint64_t bar;
    const uint32_t b = smem_u32(&bar);
    if (threadIdx.x == 0) {
        mbar_init(b, 1);
        fence_mbar_init();
    }
    __syncwarp();
    warp_wait(b, 0, Fault{&g_mx4_fault, host_fault}, site, limit_ns);
}

// -------------------------------------------------------------------------------------------- host

// The host's fault word: memory of this library's that the devices write, zero while no wait has given up.
// Its mapping is asked for at every launch, so that a reset of the device only costs another registration.
alignas(4096) volatile int g_host_fault[1024];

// the devices' address of it, or null with the error recorded
int *host_fault() {
    void *host = const_cast<int *>(g_host_fault), *p = nullptr;
    if (cudaHostGetDevicePointer(&p, host, 0) == cudaSuccess) return static_cast<int *>(p);
    cudaGetLastError();
    static std::mutex one;
    const std::lock_guard<std::mutex> lock(one);
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;  // no part of a graph that may be being captured
    cudaThreadExchangeStreamCaptureMode(&mode);
    cudaHostRegister(host, sizeof(g_host_fault), cudaHostRegisterPortable | cudaHostRegisterMapped);
    cudaThreadExchangeStreamCaptureMode(&mode);
    cudaGetLastError();
    if (cudaHostGetDevicePointer(&p, host, 0) == cudaSuccess) return static_cast<int *>(p);
    launch_status("mxfp4 (the fault word's registration)");
    return nullptr;
}

// 0, or 7 with the error recorded: outputs since the fault are not complete
int earlier_fault() {
    const int site = g_host_fault[0];
    if (!site) return 0;
    set_error("mxfp4: an earlier product gave up a wait on the device (site " + std::to_string(site) +
              "); outputs since then are not complete.  xpuint8_fault_status(1) clears it");
    return 7;
}

struct Operand {
    const uint8_t *codes, *scales;
    int64_t rows, K, tiles;  // rows of codes; 128-row scale tiles
};

bool code_map(CUtensorMap *m, const Operand &o, int box_rows) {
    const int64_t bytes = (o.K + 31) / 32 * 16;
    return make_map(m, o.codes, bytes, o.rows, bytes, kCodeRow, box_rows);
}
bool scale_map(CUtensorMap *m, const Operand &o, int box_tiles) {
    const int64_t words = (o.K + 127) / 128 * 128;
    return make_map(m, o.scales, words, o.tiles, words * 4, 256, box_tiles, CU_TENSOR_MAP_DATA_TYPE_UINT32, CU_TENSOR_MAP_SWIZZLE_NONE);
}
bool out_map(CUtensorMap *m, void *out, int type, int64_t rows, int64_t cols, int64_t ldo) {
    const CUtensorMapDataType dt = type == kMxF32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : type == kMxF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                    : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return make_map(m, out, cols, rows, ldo * mx_size(type), type == kMxF32 ? 32 : 64, 32, dt, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int BN, int T>
int resident_pairs(int dev) {
    static std::atomic<int> cached[32] = {};
    if (dev >= 0 && dev < 32) {
        const int c = cached[dev].load(std::memory_order_relaxed);
        if (c > 0) return c;
    }
    auto kern = pair_kernel<BN, T>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(PairCfg<BN>::kSmemBytes)) != cudaSuccess) return -1;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(2 * num_sms());
    cfg.blockDim = dim3(PairCfg<BN>::kThreads);
    cfg.dynamicSmemBytes = PairCfg<BN>::kSmemBytes;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) return -1;
    if (dev >= 0 && dev < 32) cached[dev].store(n, std::memory_order_relaxed);
    return n;
}

struct PairMaps {
    CUtensorMap a, b, sa, sb, out;
};

template <int BN, int T>
int launch_pair(cudaStream_t s, const PairMaps &m, const PairArgs &a, int64_t tiles) {
    int dev = 0;
    cudaGetDevice(&dev);
    const int resident = resident_pairs<BN, T>(dev);
    if (resident <= 0) {
        set_error("no CTA pair of the MXFP4 product fits on the device");
        return 5;
    }
    auto kern = pair_kernel<BN, T>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(PairCfg<BN>::kSmemBytes)) != cudaSuccess)
        return launch_status("mxfp4_mm (shared memory attribute)");
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(2 * static_cast<uint32_t>(std::min<int64_t>(tiles, resident)));
    cfg.blockDim = dim3(PairCfg<BN>::kThreads);
    cfg.dynamicSmemBytes = PairCfg<BN>::kSmemBytes;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cudaLaunchKernelEx(&cfg, kern, m.a, m.b, m.sa, m.sb, m.out, a);
    return launch_status("mxfp4_mm");
}

template <int BN>
int launch_pair_type(cudaStream_t s, const PairMaps &m, const PairArgs &a, int64_t tiles, int type) {
    switch (type) {
        case kMxBf16: return launch_pair<BN, kMxBf16>(s, m, a, tiles);
        case kMxF16: return launch_pair<BN, kMxF16>(s, m, a, tiles);
        default: return launch_pair<BN, kMxF32>(s, m, a, tiles);
    }
}

// `a` complete but for the tile counts; max_m: 256-row tiles (rows: at most)
int run_pair(cudaStream_t s, PairArgs a, const Operand &A, const Operand &B, int type, int64_t out_rows, int64_t max_m) {
    if (int rc = earlier_fault()) return rc;
    if (!(a.host_fault = host_fault())) return 5;
    // 256 or 128 columns a tile, by the rounds that the pairs take.  A k-block takes 0.32 us at 256
    // columns and nearly as long at 128 (0.9 of it: an MMA's time hardly depends on its columns), and a
    // tile costs its hand-over and the end of its drain, 7.5 k-blocks' time at 256 columns and 5 at
    // 128 (measured at 8192 x 14336 and 18944 x 128 to 256, K 1024 to 16384).  So the narrow tile wins
    // where it turns one round of few tiles into one of more: 1000 x 1024 x 1024 5.8 us against 7.3,
    // 4096 x 1280 x 5120 25.5 us wide against 30 narrow.
    const int64_t matrices = a.mode == kContraction ? a.experts : 1;
    const int64_t pairs = num_sms() / 2;
    const int64_t nk = a.mode == kContraction ? std::max<int64_t>(1, A.K / BK / a.experts) : a.nk;
    auto cost = [&](int bn) {
        const int64_t tiles = max_m * matrices * ((a.N + bn - 1) / bn);
        return (tiles + pairs - 1) / pairs * (bn == 256 ? 10 * nk + 75 : 9 * nk + 50);
    };
    const int bn = cost(128) < cost(256) ? 128 : 256;
    a.num_n = (a.N + bn - 1) / bn;
    const int64_t tiles = max_m * matrices * a.num_n;
    if (tiles > 0x7FFFFFFF) {
        set_error("mxfp4_mm: too many output tiles");
        return 2;
    }
    const int es = mx_size(type);
    a.tma_out = (reinterpret_cast<uintptr_t>(a.out) & 15) == 0 && (a.ldo * es) % 16 == 0;
    PairMaps m{};
    if (!code_map(&m.a, A, 128) || !code_map(&m.b, B, bn / 2) || !scale_map(&m.sa, A, 1) || !scale_map(&m.sb, B, bn / 128)) return 2;
    if (a.tma_out && !out_map(&m.out, a.out, type, out_rows, a.N, a.ldo)) return 2;
    return bn == 256 ? launch_pair_type<256>(s, m, a, tiles, type) : launch_pair_type<128>(s, m, a, tiles, type);
}

template <int T, int FUSE>
int launch_few(cudaStream_t s, const CUtensorMap &w, const CUtensorMap &sw, const FewMaps &x, const CUtensorMap &sx, const FewArgs &a, int splits, int64_t slots) {
    auto kern = few_kernel<T, FUSE>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(FewCfg<FUSE>::kSmem)) != cudaSuccess)
        return launch_status("mxfp4_mm (shared memory attribute)");
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<uint32_t>(splits);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(static_cast<uint32_t>((a.N + 127) / 128 * splits), static_cast<uint32_t>(slots));
    cfg.blockDim = dim3(kFewThreads);
    cfg.dynamicSmemBytes = FewCfg<FUSE>::kSmem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cudaLaunchKernelEx(&cfg, kern, w, sw, x, sx, a);
    return launch_status("mxfp4_mm");
}

template <int T>
int launch_few(cudaStream_t s, const CUtensorMap &w, const CUtensorMap &sw, const FewMaps &x, const CUtensorMap &sx, const FewArgs &a, int splits, int64_t slots, int fuse) {
    switch (fuse) {
        case kFuseNone: return launch_few<T, kFuseNone>(s, w, sw, x, sx, a, splits, slots);
        case kFusePlain: return launch_few<T, kFusePlain>(s, w, sw, x, sx, a, splits, slots);
        default: return launch_few<T, kFuseRotate>(s, w, sw, x, sx, a, splits, slots);
    }
}

// X tokens (null where they are quantised in the kernel), W weight rows; slots: 128-token tiles (rows:
// at most)
int run_few(cudaStream_t s, FewArgs a, const Operand *X, const Operand &W, int type, int64_t slots, int fuse) {
    if (int rc = earlier_fault()) return rc;
    if (!(a.host_fault = host_fault())) return 5;
    if (slots > 65535) {
        set_error("mxfp4_mm: too many token tiles");
        return 2;
    }
    // the contraction is split while the CTAs do not fill the device twice and each part has two
    // k-blocks at least
    a.vec_out = a.ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
    const int64_t tiles = (a.N + 127) / 128 * slots;
    int splits = 1;
    while (splits < 8 && tiles * splits * 2 <= 2 * num_sms() && a.nk >= splits * 4) splits *= 2;
    CUtensorMap w, sw, sx{};
    FewMaps x{};
    if (!code_map(&w, W, 128) || !scale_map(&sw, W, 1)) return 2;
    if (X) {
        if (!scale_map(&sx, *X, 1)) return 2;
        // the boxes that some tile's tokens take: a dense tile's, or any where an expert's count picks it
        const auto box = [](int n) { return n <= 16 ? 0 : n <= 32 ? 1 : n <= 64 ? 2 : 3; };
        const int last = box((a.M - 1) % 128 + 1);
        for (int i = 0; i < 4; ++i)
            if ((a.mode == kRows || i == last || (i == 3 && a.M > 128)) && !code_map(&x.x[i], *X, 16 << i)) return 2;
    }
    switch (type) {
        case kMxBf16: return launch_few<kMxBf16>(s, w, sw, x, sx, a, splits, slots, fuse);
        case kMxF16: return launch_few<kMxF16>(s, w, sw, x, sx, a, splits, slots, fuse);
        default: return launch_few<kMxF32>(s, w, sw, x, sx, a, splits, slots, fuse);
    }
}

bool aligned(const void *p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
cudaStream_t as_stream(const void *s) { return static_cast<cudaStream_t>(const_cast<void *>(s)); }

int check(const char *what, int32_t type, std::initializer_list<const void *> operands, const void *out, std::initializer_list<int64_t> sizes) {
    if (type < 0 || type > 2) {
        set_error(std::string(what) + ": the element type must be 0 (bf16), 1 (fp16) or 2 (fp32)");
        return 2;
    }
    for (const void *p : operands)
        if (!p || !aligned(p, 16)) {
            set_error(std::string(what) + ": an operand is null or not 16-byte aligned");
            return 2;
        }
    if (!out || !aligned(out, mx_size(type))) {
        set_error(std::string(what) + ": the output is null or not aligned to its elements");
        return 2;
    }
    for (int64_t n : sizes)
        if (n <= 0 || n > 0x7FFFFF00ll) {
            set_error(std::string(what) + ": sizes must be positive and fit in 31 bits");
            return 2;
        }
    return 0;
}

void set_k(int64_t K, int &nk, int &last_steps) {
    nk = static_cast<int>((K + BK - 1) / BK);
    last_steps = static_cast<int>((K - static_cast<int64_t>(nk - 1) * BK + 63) / 64);
}

FewArgs few_args(void *out, int64_t ldo, int64_t M, int64_t N, int64_t K) {
    FewArgs a{};
    a.out = out;
    a.ldo = ldo;
    a.M = static_cast<int>(M);
    a.N = static_cast<int>(N);
    a.K = static_cast<int>(K);
    set_k(K, a.nk, a.last_steps);
    a.rows = M;
    a.w_tiles = static_cast<int>((N + 127) / 128);
    return a;
}

}  // namespace

int mx4_mm(cudaStream_t s, const uint8_t *a_codes, const uint8_t *a_scales, const uint8_t *b_codes, const uint8_t *b_scales,
           const float *bias, void *out, int type, int64_t ldo, int64_t M, int64_t N, int64_t K, bool b_early) {
    const Operand A{a_codes, a_scales, M, K, (M + 127) / 128}, B{b_codes, b_scales, N, K, (N + 127) / 128};
    // The few-row kernel reads a weight once for up to 64 rows with less to start than the pairs' (4096 x
    // 4096: 6.3 us at 16 rows against 8.8, 8.4 against 8.8 at 64, 11.7 against 9.1 at 128).  Beyond that
    // it wins only where a long contraction is left to fewer tiles than there are pairs, which it splits:
    // N 4096, K 14336: 12.6 us at 64 rows against 21.8, 18.2 at 256 against 22.5, 25.9 at 384 against 23.2.
    const int64_t nk = (K + BK - 1) / BK;
    if (M <= 64 || (M <= 256 && nk > 24 && (N + 127) / 128 < num_sms() / 2)) {
        FewArgs a = few_args(out, ldo, M, N, K);
        a.bias = bias;
        a.mode = kDense;
        a.w_early = b_early;
        return run_few(s, a, &A, B, type, (M + 127) / 128, kFuseNone);
    }
    PairArgs a{};
    a.out = out;
    a.ldo = ldo;
    a.bias = bias;
    a.M = static_cast<int>(M);
    a.N = static_cast<int>(N);
    a.num_m = static_cast<int>((M + 255) / 256);
    set_k(K, a.nk, a.last_steps);
    a.mode = kDense;
    a.b_early = b_early;
    return run_pair(s, a, A, B, type, M, a.num_m);
}

int mx4_token_mm(cudaStream_t s, const void *x, int64_t ldx, const uint8_t *b_codes, const uint8_t *b_scales, const float *bias, void *out,
                 int type, int64_t M, int64_t N, int64_t K, bool rotate) {
    FewArgs a = few_args(out, N, M, N, K);
    a.bias = bias;
    a.mode = kDense;
    a.w_early = 0;  // the kernel before may be the one that wrote the weight
    a.x = x;
    a.ldx = ldx;
    return run_few(s, a, nullptr, Operand{b_codes, b_scales, N, K, (N + 127) / 128}, type, 1, rotate ? kFuseRotate : kFusePlain);
}

int mx4_expert_token_mm(cudaStream_t s, const void *x, int64_t ldx, const int32_t *order, int64_t fan, const uint8_t *b_codes,
                        const uint8_t *b_scales, void *out, int type, const int32_t *offsets, const int32_t *tiles, int64_t rows,
                        int64_t max_tiles, int64_t N, int64_t K, int64_t experts, bool rotate) {
    FewArgs a = few_args(out, N, rows, N, K);
    a.mode = kRows;
    a.offsets = offsets;
    a.tiles = tiles;
    a.experts = static_cast<int>(experts);
    a.x = x;
    a.ldx = ldx;
    a.order = order;
    a.fan = static_cast<int>(fan);
    return run_few(s, a, nullptr, Operand{b_codes, b_scales, experts * N, K, experts * ((N + 127) / 128)}, type, max_tiles,
                   rotate ? kFuseRotate : kFusePlain);
}

int mx4_expert_mm(cudaStream_t s, const uint8_t *a_codes, const uint8_t *a_scales, const uint8_t *b_codes, const uint8_t *b_scales,
                  void *out, int type, int64_t ldo, const int32_t *offsets, const int32_t *tiles, int64_t rows, int64_t max_tiles,
                  int64_t N, int64_t K, int64_t experts) {
    const Operand A{a_codes, a_scales, rows, K, max_tiles};
    const Operand B{b_codes, b_scales, experts * N, K, experts * ((N + 127) / 128)};
    // by the mean rows of an expert: 64 experts of 2816 x 2048 take 50 us at 32 rows against the pairs'
    // 57, 56 against 57 at 48, 63 against 57 at 64; 8 of 5632 x 2048 13.8 against 18.2, 15.9 against
    // 18.4, 19.2 against 18.5
    if (rows <= experts * 48) {
        FewArgs a = few_args(out, ldo, rows, N, K);
        a.mode = kRows;
        a.offsets = offsets;
        a.tiles = tiles;
        a.experts = static_cast<int>(experts);
        return run_few(s, a, &A, B, type, max_tiles, kFuseNone);
    }
    PairArgs a{};
    a.out = out;
    a.ldo = ldo;
    a.M = static_cast<int>(rows);
    a.N = static_cast<int>(N);
    set_k(K, a.nk, a.last_steps);
    a.mode = kRows;
    a.offsets = offsets;
    a.tiles = tiles;
    a.experts = static_cast<int>(experts);
    a.b_tiles = static_cast<int>((N + 127) / 128);
    a.rows = rows;
    // 256-row tiles: no more than the 128-row ones
    const int64_t max_m = std::min(max_tiles, rows / 256 + std::min(experts, rows));
    return run_pair(s, a, A, B, type, rows, max_m);
}

int mx4_expert_dw(cudaStream_t s, const uint8_t *a_codes, const uint8_t *a_scales, const uint8_t *b_codes, const uint8_t *b_scales,
                  void *out, int type, const int32_t *tiles, int64_t max_tiles, int64_t M, int64_t N, int64_t experts) {
    const Operand A{a_codes, a_scales, M, max_tiles * 128, (M + 127) / 128};
    const Operand B{b_codes, b_scales, N, max_tiles * 128, (N + 127) / 128};
    PairArgs a{};
    a.out = out;
    a.ldo = N;
    a.M = static_cast<int>(M);
    a.N = static_cast<int>(N);
    a.num_m = static_cast<int>((M + 255) / 256);
    a.mode = kContraction;
    a.tiles = tiles;
    a.experts = static_cast<int>(experts);
    return run_pair(s, a, A, B, type, experts * M, a.num_m);
}

int mx4_fault_status(int reset) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_mx4_fault, sizeof(int)) != cudaSuccess) {
        set_error("could not read the MXFP4 product's fault word");
        return -1;
    }
    if (!v) v = g_host_fault[0];  // another device's
    if (reset && v) {
        const int zero = 0;
        cudaMemcpyToSymbol(g_mx4_fault, &zero, sizeof(int));
        g_host_fault[0] = 0;
    }
    return v;
}

}  // namespace xpuint8

using namespace xpuint8;

extern "C" {

int xpuint8_mxfp4_wait_probe(int64_t limit_ns, int32_t site) {
    if (site == 0) {
        set_error("mxfp4_wait_probe: the site must not be 0");
        return 2;
    }
    int *const host = host_fault();
    if (!host) return 5;
    // at least 1 us, at most the products' own limit
    const int64_t limit = std::min(std::max<int64_t>(limit_ns, 1000), static_cast<int64_t>(kWaitTimeoutNs));
    wait_probe_kernel<<<1, 32>>>(static_cast<uint64_t>(limit), site, host);
    if (const int rc = launch_status("mxfp4_wait_probe")) return rc;
    return cudaStreamSynchronize(nullptr) == cudaSuccess ? 0 : launch_status("mxfp4_wait_probe");
}

int xpuint8_mxfp4_mm_stream(const void *stream, const uint8_t *a_codes, const uint8_t *a_scales,
                            const uint8_t *b_codes, const uint8_t *b_scales, const float *bias,
                            void *out, int32_t type, int64_t ldo, int64_t M, int64_t N,
                            int64_t K) {
    if (int rc = check("mxfp4_mm", type, {a_codes, a_scales, b_codes, b_scales}, out, {M, N, K})) return rc;
    if (ldo < N || !aligned(bias, 16)) {
        set_error("mxfp4_mm: the output's row stride must be at least N and the bias 16-byte aligned");
        return 2;
    }
    return mx4_mm(as_stream(stream), a_codes, a_scales, b_codes, b_scales, bias, out, type, ldo, M, N, K, false);
}

int xpuint8_mxfp4_expert_mm_stream(const void *stream, const uint8_t *a_codes,
                                   const uint8_t *a_scales, const uint8_t *b_codes,
                                   const uint8_t *b_scales, void *out, int32_t type,
                                   const int32_t *offsets, const int32_t *tiles, int64_t rows,
                                   int64_t max_tiles, int64_t N, int64_t K, int64_t experts) {
    if (int rc = check("mxfp4_expert_mm", type, {a_codes, a_scales, b_codes, b_scales}, out, {rows, max_tiles, N, K, experts})) return rc;
    if (!offsets || !tiles || experts > kMaxExperts || experts * N > 0x7FFFFF00ll || max_tiles > 65535) {
        set_error("mxfp4_expert_mm: offsets and tiles, 1 to 1024 experts, experts x N below 2^31, at most 65535 tiles");
        return 2;
    }
    return mx4_expert_mm(as_stream(stream), a_codes, a_scales, b_codes, b_scales, out, type, N, offsets, tiles, rows, max_tiles, N, K, experts);
}

int xpuint8_mxfp4_expert_dw_stream(const void *stream, const uint8_t *a_codes,
                                   const uint8_t *a_scales, const uint8_t *b_codes,
                                   const uint8_t *b_scales, void *out, int32_t type,
                                   const int32_t *tiles, int64_t max_tiles, int64_t M, int64_t N,
                                   int64_t experts) {
    if (int rc = check("mxfp4_expert_dw", type, {a_codes, a_scales, b_codes, b_scales}, out, {max_tiles, M, N, experts})) return rc;
    if (!tiles || experts > kMaxExperts || max_tiles > 65535 || experts * M > 0x7FFFFF00ll) {
        set_error("mxfp4_expert_dw: tiles, 1 to 1024 experts, at most 65535 tiles, experts x M below 2^31");
        return 2;
    }
    return mx4_expert_dw(as_stream(stream), a_codes, a_scales, b_codes, b_scales, out, type, tiles, max_tiles, M, N, experts);
}

}  // extern "C"
