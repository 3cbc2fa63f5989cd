// The MXFP4 linears as one C call each: the quantizers and products of mxfp4.cu and gemm_mx4.cu in
// order on the caller's stream, over caller scratch.
//
//   linear         y = Q(x) Wq^T (+ bias): up to 8 tokens in one launch (quantised inside the product)
//   train          y = Q(x) Q(w)^T (+ bias), and what the gradients need later: x and w quantised along
//                  the other axis, in the same read
//   grad           dx = Q(dy) Q(w^T)^T, dw = Q(dy^T) Q(x^T)^T, each turned back where x and w were rotated
//   expert_*       the same by expert, rows in the plan's order
//
// Rotated gradients go from the product to the rotation in fp32, and are rounded once.  Rounded to their
// type before the rotation as well, dw's error against 64 bits is 1.41 times one rounding's (two
// independent ones) and a dx summed over a token's experts 1.9 times; and a group's value before the
// rotation can be 16 times the largest after it, which fp16 may not hold.
#include <cuda_runtime.h>

#include <algorithm>
#include <string>

#include "internal.h"
#include "mx4.h"
#include "xpu_kernels/convrot.h"

namespace xpuint8 {
namespace {

constexpr int64_t kMaxExperts = 1024;

bool aligned(const void *p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
cudaStream_t as_stream(const void *s) { return static_cast<cudaStream_t>(const_cast<void *>(s)); }
int size_of(int type) { return type == 2 ? 4 : 2; }

// pieces of a scratch buffer, each 256-byte aligned; with a null base only the size is taken
struct Scratch {
    uint8_t *base;
    int64_t at = 0;
    explicit Scratch(void *p) : base(static_cast<uint8_t *>(p)) {}
    uint8_t *take(int64_t bytes) {
        uint8_t *p = base ? base + at : nullptr;
        at += (bytes + 255) / 256 * 256;
        return p;
    }
};

int fail(const char *what, const char *why) {
    set_error(std::string(what) + ": " + why);
    return 2;
}

int check(const char *what, std::initializer_list<int32_t> types, std::initializer_list<int64_t> sizes, int64_t K, int32_t rotate) {
    for (int32_t t : types)
        if (t < 0 || t > 2) return fail(what, "the element type must be 0 (bf16), 1 (fp16) or 2 (fp32)");
    for (int64_t n : sizes)
        if (n <= 0 || n > 0x7FFFFF00ll) return fail(what, "sizes must be positive and fit in 31 bits");
    if (rotate && K % 256) {
        set_error("K must be divisible by the ConvRot group size (256)");
        return 3;
    }
    return 0;
}

int check_pointers(const char *what, std::initializer_list<const void *> sixteen) {
    for (const void *p : sixteen)
        if (!p || !aligned(p, 16)) return fail(what, "a required pointer is null or not 16-byte aligned");
    return 0;
}

int check_plan(const char *what, std::initializer_list<const void *> words, int64_t tokens, int64_t fan, int64_t max_tiles, int64_t N, int64_t K,
               int64_t experts) {
    for (const void *p : words)
        if (!p || !aligned(p, 4)) return fail(what, "the plan's arrays are null or not 4-byte aligned");
    if (experts > kMaxExperts || max_tiles > 65535 || experts * std::max(N, K) > 0x7FFFFF00ll || tokens * std::max<int64_t>(fan, 1) > 0x7FFFFF00ll)
        return fail(what, "at most 1024 experts and 65535 tiles, experts x rows below 2^31");
    return 0;
}

struct Codes {
    uint8_t *codes, *scales;
};
Codes take(Scratch &s, int64_t rows, int64_t K) { return {s.take(mx4_code_bytes(rows, K)), s.take(mx4_scale_bytes(rows, K))}; }
Codes take_stack(Scratch &s, int64_t n, int64_t rows, int64_t K) { return {s.take(n * mx4_code_bytes(rows, K)), s.take(n * mx4_scale_bytes(rows, K))}; }
// rows of the plan: scales in its padded tiles
Codes take_rows(Scratch &s, int64_t rows, int64_t max_tiles, int64_t K) { return {s.take(mx4_code_bytes(rows, K)), s.take(mx4_scale_bytes(max_tiles * 128, K))}; }

struct TrainSaved {
    Codes x, w;  // [K] rows along the tokens, [K] rows along N
};
TrainSaved train_saved(Scratch &s, int64_t M, int64_t N, int64_t K, int want) {
    TrainSaved t{};
    if (want & 2) t.x = take(s, K, M);
    if (want & 1) t.w = take(s, K, N);
    return t;
}
TrainSaved expert_saved(Scratch &s, int64_t max_tiles, int64_t N, int64_t K, int64_t experts, int want) {
    TrainSaved t{};
    if (want & 2) t.x = take(s, K, max_tiles * 128);
    if (want & 1) t.w = take_stack(s, experts, K, N);
    return t;
}

struct TrainWork {
    Codes x, w;
};
TrainWork train_work(Scratch &s, int64_t M, int64_t N, int64_t K) { return {take(s, M, K), take(s, N, K)}; }

struct GradWork {
    Codes rows, cols;
    float *dx, *dw;
};
GradWork grad_work(Scratch &s, int64_t M, int64_t N, int64_t K, int rotate, int want) {
    GradWork g{};
    if (want & 1) g.rows = take(s, M, N);
    if (want & 2) g.cols = take(s, N, M);
    if ((want & 1) && rotate) g.dx = reinterpret_cast<float *>(s.take(M * K * 4));
    if ((want & 2) && rotate) g.dw = reinterpret_cast<float *>(s.take(N * K * 4));
    return g;
}
// fp32 rows that are summed afterwards: 16-byte aligned, for the product's stores and the sum's loads (22544
// rows of 850: 54 and 66 us packed)
int64_t sum_pitch(int64_t K) { return (K + 3) / 4 * 4; }
GradWork expert_grad_work(Scratch &s, int64_t rows, int64_t max_tiles, int64_t N, int64_t K, int64_t experts, bool turn_dx, int rotate, int want) {
    GradWork g{};
    if (want & 1) g.rows = take_rows(s, rows, max_tiles, N);
    if (want & 2) g.cols = take(s, N, max_tiles * 128);
    if ((want & 1) && turn_dx) g.dx = reinterpret_cast<float *>(s.take(rows * sum_pitch(K) * 4));
    if ((want & 2) && rotate) g.dw = reinterpret_cast<float *>(s.take(experts * N * K * 4));
    return g;
}

int quantize_for_train(cudaStream_t s, const Mx4Both &b) {
    if (b.col_codes) return mx4_quantize_both(s, b);
    return mx4_quantize_rows(s, b.x, b.type, b.ldx, b.row_codes, b.row_scales, nullptr, b.rows * b.matrices, b.cols, b.rows, b.rotate);
}

// the tokens' rows can be loaded in whole 16-byte vectors, which the product that quantises them wants
bool whole_rows(const void *x, int type, int64_t ldx) { return aligned(x, 16) && (ldx * size_of(type)) % 16 == 0; }

}  // namespace
}  // namespace xpuint8

using namespace xpuint8;

extern "C" {

int64_t xpuint8_mxfp4_linear_workspace_bytes(int64_t M, int64_t K) {
    if (M < 0 || K <= 0) return -1;
    Scratch s(nullptr);
    take(s, M, K);
    return s.at;
}

int xpuint8_mxfp4_linear_stream(const void *stream, const void *x, int32_t type, int64_t ldx,
                                const uint8_t *w_codes, const uint8_t *w_scales, const float *bias,
                                void *out, void *workspace, int64_t M, int64_t N, int64_t K,
                                int32_t rotate) {
    const char *what = "mxfp4_linear";
    if (int rc = check(what, {type}, {M, N, K}, K, rotate)) return rc;
    if (int rc = check_pointers(what, {w_codes, w_scales})) return rc;
    if (!x || !aligned(x, size_of(type)) || !out || !aligned(out, size_of(type)) || !aligned(bias, 16) || ldx < K)
        return fail(what, "x and out aligned to their elements, the bias to 16 bytes, and ldx at least K");
    cudaStream_t s = as_stream(stream);
    if (M <= kMx4Tokens && whole_rows(x, type, ldx)) return mx4_token_mm(s, x, ldx, w_codes, w_scales, bias, out, type, M, N, K, rotate != 0);
    if (int rc = check_pointers(what, {workspace})) return rc;
    Scratch work(workspace);
    const Codes q = take(work, M, K);
    if (int rc = mx4_quantize_rows(s, x, type, ldx, q.codes, q.scales, nullptr, M, K, M, rotate != 0)) return rc;
    return mx4_mm(s, q.codes, q.scales, w_codes, w_scales, bias, out, type, N, M, N, K, true);
}

int64_t xpuint8_mxfp4_train_saved_workspace_bytes(int64_t M, int64_t N, int64_t K, int32_t want) {
    if (M < 0 || N <= 0 || K <= 0) return -1;
    Scratch s(nullptr);
    train_saved(s, M, N, K, want);
    return s.at;
}
int64_t xpuint8_mxfp4_train_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M < 0 || N <= 0 || K <= 0) return -1;
    Scratch s(nullptr);
    train_work(s, M, N, K);
    return s.at;
}

int xpuint8_mxfp4_train_stream(const void *stream, const void *x, int32_t type, int64_t ldx,
                               const void *w, int32_t w_type, int64_t ldw, const float *bias,
                               void *out, void *saved, void *workspace, int64_t M, int64_t N,
                               int64_t K, int32_t rotate, int32_t want) {
    const char *what = "mxfp4_train";
    if (int rc = check(what, {type, w_type}, {M, N, K}, K, rotate)) return rc;
    if (int rc = check_pointers(what, {workspace})) return rc;
    if (!x || !aligned(x, size_of(type)) || !w || !aligned(w, size_of(w_type)) || !out || !aligned(out, size_of(type)) ||
        !aligned(bias, 16) || ldx < K || ldw < K || (want && (!saved || !aligned(saved, 16))))
        return fail(what, "x, w and out aligned to their elements, bias and saved to 16 bytes, row strides at least K");
    cudaStream_t s = as_stream(stream);
    Scratch keep(saved), work(workspace);
    const TrainSaved t = train_saved(keep, M, N, K, want);
    const TrainWork q = train_work(work, M, N, K);
    Mx4Both b;
    b.x = w;
    b.type = w_type;
    b.ldx = ldw;
    b.rows = N;
    b.cols = K;
    b.rotate = rotate != 0;
    b.row_codes = q.w.codes;
    b.row_scales = q.w.scales;
    b.col_codes = t.w.codes;
    b.col_scales = t.w.scales;
    if (int rc = quantize_for_train(s, b)) return rc;
    b.x = x;
    b.type = type;
    b.ldx = ldx;
    b.rows = M;
    b.row_codes = q.x.codes;
    b.row_scales = q.x.scales;
    b.col_codes = t.x.codes;
    b.col_scales = t.x.scales;
    if (int rc = quantize_for_train(s, b)) return rc;
    // the weight's quantizer is done before x's begins: the product may read its codes early
    return mx4_mm(s, q.x.codes, q.x.scales, q.w.codes, q.w.scales, bias, out, type, N, M, N, K, true);
}

int64_t xpuint8_mxfp4_grad_workspace_bytes(int64_t M, int64_t N, int64_t K, int32_t /*w_type*/, int32_t rotate, int32_t want) {
    if (M < 0 || N <= 0 || K <= 0) return -1;
    Scratch s(nullptr);
    grad_work(s, M, N, K, rotate, want);
    return s.at;
}

int xpuint8_mxfp4_grad_stream(const void *stream, const void *dy, int32_t type, int64_t ld_dy,
                              const void *saved, void *dx, void *dw, int32_t w_type,
                              void *workspace, int64_t M, int64_t N, int64_t K, int32_t rotate,
                              int32_t want) {
    const char *what = "mxfp4_grad";
    if (int rc = check(what, {type, w_type}, {M, N, K}, K, rotate)) return rc;
    if (int rc = check_pointers(what, {saved, workspace})) return rc;
    const bool want_x = (want & 1) && dx, want_w = (want & 2) && dw;
    if (!dy || !aligned(dy, size_of(type)) || ld_dy < N || (dx && !want_x) || (dw && !want_w) || (!want_x && !want_w) ||
        !aligned(dx, 16) || !aligned(dw, 16))
        return fail(what, "dy aligned to its elements with a row stride of at least N, dx and dw 16-byte aligned and kept for by want");
    cudaStream_t s = as_stream(stream);
    Scratch keep(const_cast<void *>(saved)), work(workspace);
    const TrainSaved t = train_saved(keep, M, N, K, want);
    const int have = (want_x ? 1 : 0) | (want_w ? 2 : 0);
    const GradWork g = grad_work(work, M, N, K, rotate, have);
    Mx4Both b;
    b.x = dy;
    b.type = type;
    b.ldx = ld_dy;
    b.rows = M;
    b.cols = N;
    b.row_codes = g.rows.codes;
    b.row_scales = g.rows.scales;
    b.col_codes = g.cols.codes;
    b.col_scales = g.cols.scales;
    if (int rc = quantize_for_train(s, b)) return rc;
    if (want_x) {
        void *to = rotate ? static_cast<void *>(g.dx) : dx;
        if (int rc = mx4_mm(s, g.rows.codes, g.rows.scales, t.w.codes, t.w.scales, nullptr, to, rotate ? 2 : type, K, M, K, N, true)) return rc;
        if (rotate)
            if (int rc = mx4_turn(s, g.dx, K, dx, type, M, K, nullptr, nullptr, 1, true)) return rc;
    }
    if (want_w) {
        void *to = rotate ? static_cast<void *>(g.dw) : dw;
        if (int rc = mx4_mm(s, g.cols.codes, g.cols.scales, t.x.codes, t.x.scales, nullptr, to, rotate ? 2 : w_type, K, N, K, M, true)) return rc;
        if (rotate)
            if (int rc = mx4_turn(s, g.dw, K, dw, w_type, N, K, nullptr, nullptr, 1, true)) return rc;
    }
    return 0;
}

int64_t xpuint8_mxfp4_expert_linear_workspace_bytes(int64_t rows, int64_t max_tiles, int64_t K) {
    if (rows < 0 || max_tiles < 0 || K <= 0) return -1;
    Scratch s(nullptr);
    take_rows(s, rows, max_tiles, K);
    return s.at;
}

int xpuint8_mxfp4_expert_linear_stream(const void *stream, const void *x, int32_t type,
                                       int64_t ldx, const uint8_t *w_codes,
                                       const uint8_t *w_scales, void *out, void *workspace,
                                       const int32_t *order, const int32_t *positions,
                                       const int32_t *scale_rows, const int32_t *offsets,
                                       const int32_t *tiles, int64_t tokens, int64_t fan,
                                       int64_t max_tiles, int64_t N, int64_t K, int64_t experts,
                                       int32_t rotate, int32_t sorted) {
    const char *what = "mxfp4_expert_linear";
    const int64_t rows = tokens * fan;
    if (int rc = check(what, {type}, {tokens, fan, max_tiles, N, K, experts}, K, rotate)) return rc;
    if (int rc = check_plan(what, {order, positions, scale_rows, offsets, tiles}, tokens, fan, max_tiles, N, K, experts)) return rc;
    if (int rc = check_pointers(what, {w_codes, w_scales})) return rc;
    if (!x || !aligned(x, size_of(type)) || !out || !aligned(out, size_of(type)) || ldx < K)
        return fail(what, "x and out aligned to their elements, and ldx at least K");
    cudaStream_t s = as_stream(stream);
    if (rows <= kMx4ExpertRows && whole_rows(x, type, ldx))
        return mx4_expert_token_mm(s, x, ldx, order, sorted ? 0 : fan, w_codes, w_scales, out, type, offsets, tiles, rows, max_tiles, N, K, experts, rotate != 0);
    if (int rc = check_pointers(what, {workspace})) return rc;
    Scratch work(workspace);
    const Codes q = take_rows(work, rows, max_tiles, K);
    if (int rc = mx4_quantize_sorted(s, x, type, ldx, q.codes, q.scales, nullptr, sorted ? order : nullptr, positions, scale_rows,
                                     sorted ? rows : tokens, sorted ? 1 : fan, K, rotate != 0))
        return rc;
    return mx4_expert_mm(s, q.codes, q.scales, w_codes, w_scales, out, type, N, offsets, tiles, rows, max_tiles, N, K, experts);
}

int64_t xpuint8_mxfp4_expert_train_saved_workspace_bytes(int64_t max_tiles, int64_t N, int64_t K, int64_t experts, int32_t want) {
    if (max_tiles < 0 || N <= 0 || K <= 0 || experts <= 0) return -1;
    Scratch s(nullptr);
    expert_saved(s, max_tiles, N, K, experts, want);
    return s.at;
}
int64_t xpuint8_mxfp4_expert_train_workspace_bytes(int64_t rows, int64_t max_tiles, int64_t N, int64_t K, int64_t experts) {
    if (rows < 0 || max_tiles < 0 || N <= 0 || K <= 0 || experts <= 0) return -1;
    Scratch s(nullptr);
    take_rows(s, rows, max_tiles, K);
    take_stack(s, experts, N, K);
    return s.at;
}

int xpuint8_mxfp4_expert_train_stream(const void *stream, const void *x, int32_t type,
                                      int64_t ldx, const void *w, int32_t w_type, void *out,
                                      void *saved, void *workspace, const int32_t *order,
                                      const int32_t *positions, const int32_t *scale_rows,
                                      const int32_t *offsets, const int32_t *tiles,
                                      int64_t tokens, int64_t fan, int64_t max_tiles, int64_t N,
                                      int64_t K, int64_t experts, int32_t rotate, int32_t sorted,
                                      int32_t want) {
    const char *what = "mxfp4_expert_train";
    const int64_t rows = tokens * fan;
    if (int rc = check(what, {type, w_type}, {tokens, fan, max_tiles, N, K, experts}, K, rotate)) return rc;
    if (int rc = check_plan(what, {order, positions, scale_rows, offsets, tiles}, tokens, fan, max_tiles, N, K, experts)) return rc;
    if (int rc = check_pointers(what, {workspace})) return rc;
    if (!x || !aligned(x, size_of(type)) || !w || !aligned(w, size_of(w_type)) || !out || !aligned(out, size_of(type)) || ldx < K ||
        (want && (!saved || !aligned(saved, 16))))
        return fail(what, "x, w and out aligned to their elements, saved to 16 bytes, and ldx at least K");
    cudaStream_t s = as_stream(stream);
    Scratch keep(saved), work(workspace);
    const TrainSaved t = expert_saved(keep, max_tiles, N, K, experts, want);
    const Codes xq = take_rows(work, rows, max_tiles, K), wq = take_stack(work, experts, N, K);
    Mx4Both b;
    b.x = w;
    b.type = w_type;
    b.ldx = K;
    b.rows = N;
    b.cols = K;
    b.matrices = experts;
    b.rotate = rotate != 0;
    b.row_codes = wq.codes;
    b.row_scales = wq.scales;
    b.col_codes = t.w.codes;
    b.col_scales = t.w.scales;
    if (int rc = quantize_for_train(s, b)) return rc;
    if (t.x.codes) {
        Mx4Both r;
        r.x = x;
        r.type = type;
        r.ldx = ldx;
        r.rows = rows;
        r.cols = K;
        r.rotate = rotate != 0;
        r.row_codes = xq.codes;
        r.row_scales = xq.scales;
        r.col_codes = t.x.codes;
        r.col_scales = t.x.scales;
        r.offsets = offsets;
        r.tiles = tiles;
        r.order = order;
        r.experts = experts;
        r.max_tiles = max_tiles;
        r.fan = sorted ? 0 : fan;
        if (int rc = mx4_quantize_both(s, r)) return rc;
    } else if (int rc = mx4_quantize_sorted(s, x, type, ldx, xq.codes, xq.scales, nullptr, sorted ? order : nullptr, positions, scale_rows,
                                            sorted ? rows : tokens, sorted ? 1 : fan, K, rotate != 0)) {
        return rc;
    }
    return mx4_expert_mm(s, xq.codes, xq.scales, wq.codes, wq.scales, out, type, N, offsets, tiles, rows, max_tiles, N, K, experts);
}

int64_t xpuint8_mxfp4_expert_grad_workspace_bytes(int64_t rows, int64_t max_tiles, int64_t N, int64_t K, int64_t experts,
                                                  int32_t /*w_type*/, int32_t rotate, int32_t sorted, int32_t want) {
    if (rows < 0 || max_tiles < 0 || N <= 0 || K <= 0 || experts <= 0) return -1;
    Scratch s(nullptr);
    expert_grad_work(s, rows, max_tiles, N, K, experts, rotate || !sorted, rotate, want);
    return s.at;
}

int xpuint8_mxfp4_expert_grad_stream(const void *stream, const void *dy, int32_t type,
                                     int64_t ld_dy, const void *saved, void *dx, void *dw,
                                     int32_t w_type, void *workspace, const int32_t *order,
                                     const int32_t *positions, const int32_t *scale_rows,
                                     const int32_t *offsets, const int32_t *tiles, int64_t tokens,
                                     int64_t fan, int64_t max_tiles, int64_t N, int64_t K,
                                     int64_t experts, int32_t rotate, int32_t sorted,
                                     int32_t want) {
    const char *what = "mxfp4_expert_grad";
    const int64_t rows = tokens * fan;
    if (int rc = check(what, {type, w_type}, {tokens, fan, max_tiles, N, K, experts}, K, rotate)) return rc;
    if (int rc = check_plan(what, {order, positions, scale_rows, offsets, tiles}, tokens, fan, max_tiles, N, K, experts)) return rc;
    if (int rc = check_pointers(what, {saved, workspace})) return rc;
    const bool want_x = (want & 1) && dx, want_w = (want & 2) && dw;
    if (!dy || !aligned(dy, size_of(type)) || ld_dy < N || (dx && !want_x) || (dw && !want_w) || (!want_x && !want_w) ||
        !aligned(dx, 16) || !aligned(dw, 16))
        return fail(what, "dy aligned to its elements with a row stride of at least N, dx and dw 16-byte aligned and kept for by want");
    cudaStream_t s = as_stream(stream);
    Scratch keep(const_cast<void *>(saved)), work(workspace);
    const TrainSaved t = expert_saved(keep, max_tiles, N, K, experts, want);
    const bool turn_dx = rotate || !sorted;
    const int have = (want_x ? 1 : 0) | (want_w ? 2 : 0);
    const GradWork g = expert_grad_work(work, rows, max_tiles, N, K, experts, turn_dx, rotate, have);
    if (want_w) {
        Mx4Both b;
        b.x = dy;
        b.type = type;
        b.ldx = ld_dy;
        b.rows = rows;
        b.cols = N;
        b.row_codes = g.rows.codes;
        b.row_scales = g.rows.scales;
        b.col_codes = g.cols.codes;
        b.col_scales = g.cols.scales;
        b.offsets = offsets;
        b.tiles = tiles;
        b.experts = experts;
        b.max_tiles = max_tiles;
        if (int rc = mx4_quantize_both(s, b)) return rc;
    } else if (int rc = mx4_quantize_sorted(s, dy, type, ld_dy, g.rows.codes, g.rows.scales, nullptr, order, positions, scale_rows, rows, 1, N, false)) {
        return rc;
    }
    if (want_x) {
        void *to = turn_dx ? static_cast<void *>(g.dx) : dx;
        if (int rc = mx4_expert_mm(s, g.rows.codes, g.rows.scales, t.w.codes, t.w.scales, to, turn_dx ? 2 : type, turn_dx ? sum_pitch(K) : K, offsets, tiles, rows, max_tiles, K, N, experts)) return rc;
        if (turn_dx)
            if (int rc = mx4_turn(s, g.dx, sum_pitch(K), dx, type, sorted ? rows : tokens, K, sorted ? nullptr : positions, sorted ? nullptr : scale_rows, sorted ? 1 : fan, rotate != 0)) return rc;
    }
    if (want_w) {
        void *to = rotate ? static_cast<void *>(g.dw) : dw;
        if (int rc = mx4_expert_dw(s, g.cols.codes, g.cols.scales, t.x.codes, t.x.scales, to, rotate ? 2 : w_type, tiles, max_tiles, N, K, experts)) return rc;
        if (rotate)
            if (int rc = mx4_turn(s, g.dw, K, dw, w_type, experts * N, K, nullptr, nullptr, 1, true)) return rc;
    }
    return 0;
}

}  // extern "C"
