/*
 * bz_mx.h -- C ABI of the operators over microscaled (MX) blocks: quantising
 * rows to them, reading them back, and products of rows quantised that way
 * with a 4-bit microscaled weight.  The products of bf16 rows with such a
 * weight are bz_gemv and bz_gemm_tiled (bz_gemv.h, BZ_W_MXFP4_TILED).  No
 * counterpart in the reference, whose weights are int4 or fp8
 * (models/int4_linear.py, models/fp8_linear.py).
 *
 * A block is 32 consecutive columns of a row: elements of a narrow
 * floating-point type and one scale code c (a byte) that stands for
 * 2^(c - 127).  With a the largest magnitude of the block,
 *   c = max(floor(log2 a) - emax, -126) + 127   (a = 0: 1),
 *   element = value / 2^(c - 127) rounded to the nearest (ties to the even
 *   code), magnitudes above the type's largest to the largest.
 * A block with a NaN or an infinity gets c = 255 and reads back as NaN; its
 * elements mean nothing.
 *   BZ_MX_E2M1  4 bits, emax 2, largest 6; two to a byte, the even column in
 *               the low half;
 *   BZ_MX_E4M3  8 bits (OCP FP8 E4M3), emax 8, largest 448.
 *
 * Conventions as in bz_gemv.h: device pointers, nothing is allocated or
 * synchronised, errors are returned before any launch.
 */
#ifndef BZ_MX_H
#define BZ_MX_H

#include "bz_gemv.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum bz_mx_elem { BZ_MX_E2M1 = 0, BZ_MX_E4M3 = 1 } bz_mx_elem;

/* x types of bz_mx_quantize beside BZ_DT_BF16 and BZ_DT_F32. */
#define BZ_MX_F16 2

/* Layouts of quantised rows.
 * BZ_MX_ROWS : codes uint8 [M][K/2] (e2m1) or [M][K] (e4m3), scales uint8
 *              [M][K/32]; K % 32 == 0.  With e2m1 this is the weight format
 *              BZ_W_MXFP4.
 * BZ_MX_TILED: the operand order of the matrix cores (bz_mx_device.h), in one
 *              buffer of bz_mx_rows_bytes bytes with the rows rounded up to 16
 *              (the added rows hold zeros); K % 128 == 0.  With e2m1 it is
 *              the weight format BZ_W_MXFP4_TILED.  scales is NULL. */
typedef enum bz_mx_layout { BZ_MX_ROWS = 0, BZ_MX_TILED = 1 } bz_mx_layout;

/* Bytes of BZ_MX_TILED rows, 0 when K % 128 or a size is not positive. */
size_t bz_mx_rows_bytes(int32_t elem, int32_t M, int32_t K);

/* Quantise x [M][ldx] (bf16, fp32 or fp16; K columns, ldx >= K; any ldx and
 * any alignment of the type's own size).  codes is 16-byte aligned for
 * BZ_MX_TILED, 4-byte aligned for BZ_MX_ROWS. */
int bz_mx_quantize(const void* x, int32_t x_dtype, int64_t ldx, int32_t M, int32_t K, int32_t elem, int32_t layout,
                   void* codes, void* scales, void* stream);

/* Read BZ_MX_ROWS back: out [M][ldo] bf16 or fp32 (exact but where a bf16
 * cannot hold a value below 2^-126 or above its range).  codes 4-byte
 * aligned; any alignment of out. */
int bz_mx_dequantize(const void* codes, const void* scales, int32_t elem, int32_t M, int32_t K, void* out,
                     int32_t out_dtype, int64_t ldo, void* stream);

/* out[M][N] = q(x) @ w_eff^T (+ residual): x already quantised, BZ_MX_TILED
 * rows of `elem`; w a BZ_W_MXFP4_TILED weight of N rows; products and sums on
 * the block-scaled matrix instructions, fp32 accumulation.  residual (bf16
 * or fp32, [M][ldr], may alias out) is added when not NULL.  out is bf16 or
 * fp32 [M][ldo].
 * With 8-bit elements the instruction adds the products of eight consecutive
 * columns on a grid of 2^-13 of the largest's power of two (each product cut
 * toward zero) before its fp32 sums, so that an fp32 result of K = 10240
 * random columns is 2e-5 of its norm off and a bf16 one differs from that of
 * plain fp32 sums in 1.4 % of its elements; 4-bit products lose nothing.
 * bz_mx_gemm_workspace gives the bytes of workspace the call needs (16-byte
 * aligned, zero-filled before its first use; every call leaves its counters
 * zero; calls that share it must not overlap), 0 where K is not sliced.  cfg =
 * 0 takes the built-in launch shape, else the tile of a workgroup, 32 rows of x
 * | 64 of the weight << 8 | K slices << 16 (a part left 0 keeps the rule's
 * choice; tiles of 1, 2, 4 or 6 and 2, 4 and 4, or 8 (e2m1) or 6 (e4m3) and
 * 4).  K up to 2^22. */
size_t bz_mx_gemm_workspace(int32_t elem, int32_t M, int32_t N, int32_t K, int32_t cfg);
int bz_mx_gemm(int32_t elem, const void* xq, int32_t M, const void* w, int32_t N, int32_t K, const void* residual,
               int32_t residual_dtype, int64_t ldr, void* out, int32_t out_dtype, int64_t ldo, void* workspace,
               size_t workspace_bytes, int32_t cfg, void* stream);

/* The same product for up to 32 rows of bf16 x, quantised inside the launch:
 * x [M][ldx] bf16, 16-byte aligned rows (ldx % 8 == 0).  The result is that of
 * bz_mx_quantize and bz_mx_gemm up to the order of its fp32 sums.  Workspace
 * as for bz_mx_gemm; bz_mx_gemv_workspace is (size_t)-1 where the call is
 * refused: K above 2^22 or too long for 64 K slices, slices of more than 4096
 * workgroups' columns or whose sums reach 2^31 bytes, a forced shape that is
 * not built or whose sums do not fit LDS.  cfg = 0 takes the built-in launch
 * shape, else row blocks per workgroup (1 .. 8) | units of 128 columns per
 * wave (1 .. 6, 8) << 8 | K slices << 16 (a part left 0 keeps the rule's
 * choice). */
size_t bz_mx_gemv_workspace(int32_t elem, int32_t M, int32_t N, int32_t K, int32_t cfg);
int bz_mx_gemv(int32_t elem, const void* x, int64_t ldx, int32_t M, const void* w, int32_t N, int32_t K,
               const void* residual, int32_t residual_dtype, int64_t ldr, void* out, int32_t out_dtype, int64_t ldo,
               void* workspace, size_t workspace_bytes, int32_t cfg, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* BZ_MX_H */
