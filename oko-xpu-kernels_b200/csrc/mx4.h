// Host side of the MXFP4 kernels: enqueue on `s` and return 0, or a code with the error recorded.
// Arguments are checked by the C entries; `type` is 0 bf16, 1 fp16, 2 fp32.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace xpuint8 {

// bytes of a matrix's codes and scales
inline int64_t mx4_code_bytes(int64_t rows, int64_t K) { return rows * ((K + 31) / 32) * 16; }
inline int64_t mx4_scale_bytes(int64_t rows, int64_t K) { return (rows + 127) / 128 * ((K + 127) / 128) * 512; }

// ------------------------------------------------------------------------- quantization (mxfp4.cu)
int mx4_quantize_rows(cudaStream_t s, const void *x, int type, int64_t ldx, uint8_t *codes, uint8_t *scales, void *rotated, int64_t rows,
                      int64_t K, int64_t matrix_rows, bool rotate);
int mx4_quantize_sorted(cudaStream_t s, const void *x, int type, int64_t ldx, uint8_t *codes, uint8_t *scales, void *rotated,
                        const int32_t *order, const int32_t *positions, const int32_t *scale_rows, int64_t rows, int64_t fan,
                        int64_t K, bool rotate);
int mx4_quantize_columns(cudaStream_t s, const void *x, int type, int64_t ldx, uint8_t *codes, uint8_t *scales, int64_t rows,
                         int64_t cols, int64_t matrices, const int32_t *offsets, const int32_t *tiles, int64_t experts, int64_t max_tiles);
// one read of x [matrices][rows, cols] for codes along the columns (row_*) and along the rows (col_*);
// either may be null.  Experts (offsets): rows of the plan, from x's rows (fan 0) or its tokens.
struct Mx4Both {
    const void *x = nullptr;
    int type = 0;
    int64_t ldx = 0, rows = 0, cols = 0, matrices = 1;
    bool rotate = false;
    uint8_t *row_codes = nullptr, *row_scales = nullptr, *col_codes = nullptr, *col_scales = nullptr;
    const int32_t *offsets = nullptr, *tiles = nullptr, *order = nullptr;
    int64_t experts = 0, max_tiles = 0, fan = 0;
};
int mx4_quantize_both(cudaStream_t s, const Mx4Both &b);
// out [rows, K] = fp32 rows (or, with positions, the sums of each token's rows), rounded once to `type`: rotated
// (K a multiple of 256, the rows contiguous); else x's rows are `ldx` apart, a multiple of 4, and only
// sums are wanted
int mx4_turn(cudaStream_t s, const float *x, int64_t ldx, void *out, int type, int64_t rows, int64_t K, const int32_t *positions,
             const int32_t *scale_rows, int64_t fan, bool rotate);

// ------------------------------------------------------------------------------ products (gemm_mx4.cu)
// b_early: B is not written by the kernel just before on the stream
int mx4_mm(cudaStream_t s, const uint8_t *a_codes, const uint8_t *a_scales, const uint8_t *b_codes, const uint8_t *b_scales,
           const float *bias, void *out, int type, int64_t ldo, int64_t M, int64_t N, int64_t K, bool b_early);
int mx4_expert_mm(cudaStream_t s, const uint8_t *a_codes, const uint8_t *a_scales, const uint8_t *b_codes, const uint8_t *b_scales,
                  void *out, int type, int64_t ldo, const int32_t *offsets, const int32_t *tiles, int64_t rows, int64_t max_tiles,
                  int64_t N, int64_t K, int64_t experts);
int mx4_expert_dw(cudaStream_t s, const uint8_t *a_codes, const uint8_t *a_scales, const uint8_t *b_codes, const uint8_t *b_scales,
                  void *out, int type, const int32_t *tiles, int64_t max_tiles, int64_t M, int64_t N, int64_t experts);
// few tokens quantised inside the product: x [M, K] of the output's type, M <= kMx4Tokens
constexpr int64_t kMx4Tokens = 8;
int mx4_token_mm(cudaStream_t s, const void *x, int64_t ldx, const uint8_t *b_codes, const uint8_t *b_scales, const float *bias, void *out,
                 int type, int64_t M, int64_t N, int64_t K, bool rotate);
// the same by expert, rows <= kMx4ExpertRows: row r comes from x's row r (fan 0) or token order[r] / fan
constexpr int64_t kMx4ExpertRows = 128;
int mx4_expert_token_mm(cudaStream_t s, const void *x, int64_t ldx, const int32_t *order, int64_t fan, const uint8_t *b_codes,
                        const uint8_t *b_scales, void *out, int type, const int32_t *offsets, const int32_t *tiles, int64_t rows,
                        int64_t max_tiles, int64_t N, int64_t K, int64_t experts, bool rotate);

}  // namespace xpuint8
