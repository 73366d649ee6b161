/* C ABI of the operators on 4-bit weights and 8-bit activations (MI355X, gfx950).
 *
 * The pieces that a decoder with weights in 4 bits is made of, and that itts_qwen_create with
 * ITTS_QWEN_W4 (itts_qwen.h) runs: a root-mean-square norm whose output is 8-bit codes with
 * group scales, products of such rows with 4-bit weights, both in one call, and the packing of
 * float weights.  No counterpart in the reference, whose weights are FP32.
 *
 * All pointers are DEVICE pointers.  Calls only enqueue kernels on `stream` (a hipStream_t; NULL
 * is the null stream) of the current device, to which the pointers and the stream belong: no
 * allocation, no copy, no synchronisation, no state kept between calls.  They may be captured
 * into a graph and may run at once from several threads and streams, as long as their outputs
 * and workspaces are apart.  Matrices are row-major with unit column stride; strides are row
 * strides in elements, at least the columns for outputs.  An output may be one of the call's inputs where
 * this says so; otherwise outputs and workspace overlap neither inputs nor each other (columns of one wider
 * matrix do not), which the calls check.  A call with no
 * rows does nothing.  Up to 2^20 columns k, 2^26 weight rows n, 2^30 rows (products: 1048560, and
 * rows * n up to 2^36; packing and unpacking: 2^33 packed bytes).
 *
 * Status codes are those of itts_gpt.h: ITTS_EINVAL for arguments that the checks refuse (nothing
 * is enqueued), ITTS_ERUNTIME for a failed launch.  itts_ops_last_error() has the message of the
 * calling thread's last failure.
 *
 * Number formats
 *   group      columns that share a scale: 32, 64 or 128.
 *   columns    of codes and weights are padded to kp, k rounded up to a multiple of 128.
 *   8 bits     int8 codes [rows][kp] and float scales [rows][kp / group]; a code stands for
 *              code * scale.  scale = max |y| of the group / 127, code = y / scale to the nearest,
 *              halves to even.  A group of zeros has scale 0; one with an infinity or NaN has scale
 *              NaN and codes 0, so that what is computed from it is NaN.  Codes of the padding are
 *              0, and so are the scales of groups that lie in it.
 *   4 bits     codes -8..7 and BF16 scales.  scale = max(max w / 7, max -w / 8) of the group,
 *              rounded to BF16; code = w / scale to the nearest, halves to even; zeros and values
 *              that are not finite as above.
 *   packed     tiles of 16 rows x 128 columns, 1024 bytes: byte 16 (16 j + r) + 8 p + i holds the
 *              codes (two's complement) of row r at columns 64 p + 8 j + i (low half) and
 *              64 p + 32 + 8 j + i (high half), r < 16, j < 4, p < 2, i < 8.  The tiles of the
 *              same 16 rows follow each other; rows are padded to a multiple of 16.  Scales:
 *              [tile row][tile][16 rows][128 / group].  Codes and scales of the padding are 0.
 */
#ifndef ITTS_OPS_H
#define ITTS_OPS_H

#include <stddef.h>
#include <stdint.h>

#include "itts_gpt.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of float matrices. */
#define ITTS_T_F32 0
#define ITTS_T_BF16 1
#define ITTS_T_F16 2

/* flags of the products */
#define ITTS_Q4_SWIGLU 1u /* columns 2i and 2i + 1 become silu(column 2i) * column 2i + 1: n / 2 columns come out */

const char* itts_ops_last_error(void);

/* h = x + residual, rounded to the element type `dtype` (h = x without a residual);
 * y = h * weight / sqrt(mean(h^2) + eps) as 8-bit codes with scales.
 * x, residual, h_out, values: [rows][cols] of `dtype`; weight [cols] of weight_dtype, which is
 * `dtype` or F32.  residual, h_out and values may be NULL; h_out (which receives h) may be x or
 * residual themselves.  values receives what the codes stand for (code * scale in FP32), rounded to `dtype`.
 * q: [rows][kp], 16-byte aligned; scales: [rows][kp / group].
 * The mean, the norm and the choice of the codes are formed in 64 bits: codes and scales are those
 * of the formula, whatever the order of the sums. */
int itts_rmsnorm_q8(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, const void* weight,
                    int32_t weight_dtype, int32_t dtype, int64_t rows, int64_t cols, float eps, int32_t group, void* h_out,
                    int64_t h_stride, void* values, int64_t values_stride, int8_t* q, float* scales, void* stream);

/* The same without the norm: y = x. */
int itts_q8_quantize(const void* x, int64_t x_stride, int32_t dtype, int64_t rows, int64_t cols, int32_t group, void* values,
                     int64_t values_stride, int8_t* q, float* scales, void* stream);

/* Bytes of `packed` and number of scales for an n x k matrix; 0 for sizes that are refused. */
size_t itts_q4_packed_bytes(int64_t n, int64_t k);
size_t itts_q4_scale_count(int64_t n, int64_t k, int32_t group);

/* w [n][k] of `dtype` to 4 bits.  packed: itts_q4_packed_bytes bytes, 16-byte aligned; scales:
 * itts_q4_scale_count BF16 numbers, 16-byte aligned. */
int itts_q4_pack(const void* w, int64_t w_stride, int32_t dtype, int64_t n, int64_t k, int32_t group, void* packed, void* scales,
                 void* stream);
/* What packed weights stand for, rounded to `dtype`: out [n][k]. */
int itts_q4_unpack(const void* packed, const void* scales, int64_t n, int64_t k, int32_t group, int32_t dtype, void* out,
                   int64_t out_stride, void* stream);

/* out[m][j] = sum over k of x[m][k] w[j][k], x and w being what the codes q, qscales [rows] and
 * packed, scales [n] stand for; + bias[j] (F32 [n] or NULL); SwiGLU with ITTS_Q4_SWIGLU (n even);
 * + residual[m][j] (`dtype`, or NULL); rounded to `dtype` once.  out may be residual itself.
 * The codes' products are summed exactly within a group, the groups in FP32.  A group's two scales are
 * multiplied in FP32 first: where their product leaves its range, so does what the group adds: infinite or NaN
 * above it, with fewer bits where the product is under 2e-37. */
int itts_q4_matmul(const int8_t* q, const float* qscales, int64_t rows, const void* packed, const void* scales, int64_t n, int64_t k,
                   int32_t group, const float* bias, const void* residual, int64_t residual_stride, uint32_t flags, int32_t dtype,
                   void* out, int64_t out_stride, void* stream);

/* itts_rmsnorm_q8 (without residual; norm_weight NULL: itts_q8_quantize) of x [rows][k] of x_dtype,
 * then itts_q4_matmul on the codes, with the same result.  A few rows take one launch and no
 * workspace; for others `workspace` (256-byte aligned) holds itts_q4_linear_workspace bytes. */
size_t itts_q4_linear_workspace(int64_t rows, int64_t n, int64_t k, int32_t group);
int itts_q4_linear(const void* x, int64_t x_stride, int32_t x_dtype, int64_t rows, const void* norm_weight, int32_t weight_dtype,
                   float eps, const void* packed, const void* scales, int64_t n, int64_t k, int32_t group, const float* bias,
                   const void* residual, int64_t residual_stride, uint32_t flags, int32_t dtype, void* out, int64_t out_stride,
                   void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
