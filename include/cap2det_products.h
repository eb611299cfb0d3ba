/*
 * cap2det_products.h — C-ABI of the low-precision and grouped matrix products of libcap2det_hip.so,
 * beside the convolution / fully-connected products of cap2det_hip.h.  The reference multiplies fp32
 * matrices only (slim.fully_connected, models/cap2det_model.py:79-88): these products have no counterpart
 * there.
 *
 * Conventions (those of cap2det_hip.h, and)
 *   - matrices are row-major with a row pitch `ld*` in ELEMENTS; columns are contiguous.
 *   - a type argument is one of the C2DP_* numbers below.
 *   - a pitch is at most C2DP_MAX_PITCH bytes, else C2D_ERR_UNSUPPORTED.  16-byte aligned base
 *     pointers, pitches and contraction lengths take the direct global -> LDS loads; any others are
 *     right too, through registers, and slower.
 *   - rows, n, k, cols and batch are at most C2DP_MAX_SIZE and groups at most C2DP_MAX_GROUPS, else
 *     C2D_ERR_UNSUPPORTED; so are the rare sizes below that which make 2^30 tiles or more.
 *   - sums are fp32, but for the products within a block of an 8-bit product with a bf16 result: see c2dp_fp8_matmul.
 *
 * Groups.  `offsets` is a DEVICE array of groups + 1 int32 row numbers: group e owns the rows
 * [offsets[e], offsets[e + 1]) and may be empty.  Values are clamped to [0, rows] and an offset below an
 * earlier one counts as that one, so that no array makes a product touch memory outside its operands.
 * Rows in no group are not read; in a product's result they are left as they were, or set to zero
 * when `clear_rest` is not 0.
 */
#ifndef CAP2DET_PRODUCTS_H_
#define CAP2DET_PRODUCTS_H_

#include "cap2det_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Bumped whenever an entry point below is added or a signature changes. */
#define C2DP_ABI_VERSION 100
int c2dp_version(void);

#define C2DP_F32 0
#define C2DP_BF16 1
#define C2DP_E4M3 2 /* OCP 8-bit, 3 bits of mantissa, largest value 448 */
#define C2DP_E5M2 3 /* OCP 8-bit, 2 bits of mantissa, largest value 57344 */

#define C2DP_BLOCK 128             /* elements of the contraction that share a scale */
#define C2DP_MAX_PITCH (1 << 22)   /* bytes */
#define C2DP_MAX_SIZE (1 << 30)
#define C2DP_MAX_GROUPS (1 << 16)  /* every workgroup looks through all offsets: time grows with groups^2 */

/* 8-bit values and fp32 scales of `batch` matrices x [rows][cols] (x_type C2DP_F32 or C2DP_BF16; matrix
 * i begins at x + i * x_batch elements).  Blocks are block_rows x 128, block_rows 1 or 128:
 *   s = max(max |x| of the block / F, 2^-126),  scale = s as fp32,  q = the 8-bit value nearest to x / s (s as
 * it is before it is rounded), ties to even; F is the largest value of q_type (C2DP_E4M3 / C2DP_E5M2).  A NaN stays one
 * and takes no part in the maximum; an infinity makes every value of its block a NaN.
 *   q     [batch][rows][cols]
 *   scale [batch][ceil(rows / block_rows)][ceil(cols / 128)] */
int c2dp_fp8_quantize(const void* x, int x_type, long long ldx, long long x_batch, void* q, int q_type,
                      float* scale, int batch, int rows, int cols, int block_rows, void* stream);

/* y[i][j] = act( sum over blocks c of 128 k of
 *                  a_scale[i][c] * b_scale[e][j / 128][c] * sum_{k in c} a[i][k] * b[e][j][k]
 *                + bias[e][j] ),   e the group of row i; the two scales are multiplied first, as fp32.
 *   a       [rows][k]       C2DP_E4M3 or C2DP_E5M2 (a_type), pitch lda
 *   a_scale [rows][ceil(k / 128)]
 *   b       [groups][n][k]  C2DP_E4M3, contiguous
 *   b_scale [groups][ceil(n / 128)][ceil(k / 128)]
 *   offsets NULL with groups == 1: every row belongs to the one matrix
 *   bias    [groups][n] fp32 or NULL;  relu != 0 applies max(., 0)
 *   y       [rows][n]       C2DP_F32 or C2DP_BF16 (y_type), pitch ldy
 * An fp32 y has fp32 sums throughout.  For a bf16 y the 8-bit matrix instructions add the products of 8 consecutive k
 * (from a multiple of 8) after they have cut each off, towards zero, at 2^-13 of the largest max(|a|, t) max(|b|, 2^-6)
 * of those that are not zero, t the least normal value of a_type (2^-6, 2^-14): at most 7 * 2^-13 of that for
 * each 8 k, before the scales.  Products of which none is 2^-7 of the largest or less lose nothing.  Everything behind that is fp32. */
int c2dp_fp8_matmul(const void* a, int a_type, long long lda, const float* a_scale, const void* b,
                    const float* b_scale, const int32_t* offsets, int groups, const float* bias, int relu,
                    void* y, int y_type, long long ldy, int rows, int n, int k, int clear_rest, void* stream);

/* y[i][j] = sum_k x[i][k] * w[e][j][k], e the group of row i.  x and w are both C2DP_F32 or both
 * C2DP_BF16 (x_type); y_type is x_type, or C2DP_F32 for bf16 operands.
 *   x [rows][k] pitch ldx;  w [groups][n][k] contiguous;  y [rows][n] pitch ldy */
int c2dp_grouped_matmul(const void* x, int x_type, long long ldx, const void* w, const int32_t* offsets,
                        int groups, void* y, int y_type, long long ldy, int rows, int n, int k,
                        int clear_rest, void* stream);

/* Input gradient: dx[i][k] = sum_j dy[i][j] * w[e][j][k].  Types as above (dy, w: dy_type).
 *   dy [rows][n] pitch lddy;  w [groups][n][k] contiguous;  dx [rows][k] pitch lddx */
int c2dp_grouped_matmul_dgrad(const void* dy, int dy_type, long long lddy, const void* w,
                              const int32_t* offsets, int groups, void* dx, int dx_type, long long lddx,
                              int rows, int n, int k, int clear_rest, void* stream);

/* Weight gradient: dw[e][j][k] = sum over the rows i of group e of dy[i][j] * x[i][k] (fp32; an empty group's
 * is zero), or dw += that when accumulate is not 0.  dy and x share x_type.  The rows of a group may be
 * dealt to several workgroups; their sums are joined in a fixed order (no atomics).
 *   x [rows][k] pitch ldx;  dy [rows][n] pitch lddy;  dw [groups][n][k] contiguous
 *   workspace: c2dp_grouped_matmul_wgrad_workspace_bytes(...) bytes, 16-byte aligned (may be NULL when that is
 *   0); its contents need not be set, and calls that may run at the same time need one each. */
unsigned long long c2dp_grouped_matmul_wgrad_workspace_bytes(int groups, int rows, int n, int k, int x_type);
int c2dp_grouped_matmul_wgrad(const void* x, int x_type, long long ldx, const void* dy, long long lddy,
                              const int32_t* offsets, int groups, float* dw, int rows, int n, int k,
                              int accumulate, void* workspace, unsigned long long workspace_bytes,
                              void* stream);

#ifdef __cplusplus
}
#endif
#endif /* CAP2DET_PRODUCTS_H_ */
