/*
 * mxfp4.h — C ABI of the microscaled 4-bit (MXFP4) side of the linear path.
 *
 * Same library (mini-sglang-fork_b200/_w8a8_tp.so), conventions, status codes
 * and error channel as w8a8_tp.h: raw device pointers, `stream` a cudaStream_t
 * as void*, every call returns an int status and never throws, allocates or
 * synchronises; shapes and alignment are checked on the host before any
 * launch.  No call needs a workspace, and no call keeps device state, so calls
 * on several streams, in several threads and in several captured graphs are
 * independent.
 *
 * An MXFP4 matrix [R, K] (K % 32 == 0) is two buffers:
 *   data   [R, K / 2] bytes, two E2M1 codes per byte, the even column in the
 *          low half (sign, 2-bit exponent, 1-bit mantissa: 0, 0.5, 1, 1.5, 2,
 *          3, 4, 6);
 *   scales [ceil(R / 128), 2 ceil(K / 256), 512] bytes, one E8M0 byte (the
 *          value 2^(b - 127), 255 = NaN) per 32 columns of a row, in tiles of
 *          128 rows x 4 blocks: row r, block c of a tile at
 *          (r % 32) * 16 + (r / 32) * 4 + c.  This is the order in which the
 *          tensor core's scale copy reads them.  The bytes of blocks beyond
 *          K are zero (the quantisers write them); those of rows beyond R are
 *          not written and not used.
 * Quantisation of a block: s = 2^(floor(log2 amax) - 2), at least 2^-127;
 * code = E2M1(x / s) rounded to nearest, ties to even, saturating at 6.  A
 * block of zeros has scale byte 0; a block that holds an infinity or a NaN, or in
 * the fused forms a product beyond fp32's largest number, has scale byte 255 and
 * zero codes (E8M0 could hold such a product's scale; a dequantised one would not
 * fit fp32).
 *
 * dtype arguments: 0 = bf16, 1 = fp16, 2 = fp32 (where an entry allows it).
 *
 * No counterpart in the reference, whose linears are bf16 (M/ = python/minisgl/):
 *   _LinearTPImpl.forward M/layers/linear.py:31-32, silu_and_mul
 *   M/layers/activation.py:9-12, RMSNorm / RMSNormFused M/layers/norm.py:8-38,
 *   GatedMLP M/models/utils.py:25-50.
 */
#ifndef MXFP4_H_
#define MXFP4_H_

#include <stddef.h>
#include <stdint.h>

#include "w8a8_tp.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of the scale tiles of an [rows, K] matrix (0 for a bad shape). */
int64_t mxfp4_scale_bytes(int64_t rows, int64_t K);

/* x[M, K] bf16 or fp16 (row stride ldx elements) -> MXFP4.  K % 32 == 0,
 * ldx % 8 == 0, 16-byte aligned x, data and scales. */
int mxfp4_quant(const void* x, int64_t ldx, int dtype, uint8_t* data, uint8_t* scales, int64_t M,
                int64_t K, void* stream);

/* MXFP4 -> the values it stands for, bf16, fp16 or fp32 (contiguous [M, K]).
 * Every code times a scale of at least 2^-126 is exact in bf16 and fp32 while
 * it is finite there; fp16 rounds to nearest even. */
int mxfp4_dequant(const uint8_t* data, const uint8_t* scales, void* out, int dtype, int64_t M, int64_t K,
                  void* stream);

/* gate_up[M, 2I] bf16 or fp16 (row stride ld) -> MXFP4 of
 * y = gate / (1 + exp(-gate)) * up, [M, I].  y is not rounded before it is
 * quantised; values that land next to a rounding border are evaluated in 64
 * bits.  So are blocks with a gate below -40 or a NaN: a call takes longer the
 * more of those there are (4096 x 12288: 46 us; 57 and 159 us with 1 and 10 % of
 * the blocks).  I % 32 == 0, ld % 8 == 0. */
int mxfp4_silu_mul_quant(const void* gate_up, int64_t ld, int dtype, uint8_t* data, uint8_t* scales,
                         int64_t M, int64_t I, void* stream);

/* v = x + residual (fp32; x alone when residual is null), residual <- v in
 * place (rounded to dtype), then MXFP4 of y = v / sqrt(mean(v^2) + eps) *
 * weight, y not rounded before it is quantised: values next to a rounding border
 * are evaluated in 64 bits.  So are blocks whose largest magnitude is below 2^-92
 * of the row's root mean square, blocks of zeros in a row that is not all zeros
 * among them: a row with padded or pruned channels takes longer (4097 x 5120:
 * 30 us; 35, 59 and 77 us with 1, 10 and 50 % of the weight's blocks zero).  x,
 * residual and weight share `dtype` (bf16 or fp16).  K % 32 == 0, K <= 32768, ldx and ldr % 8 == 0,
 * 16-byte aligned pointers, eps >= 0. */
int mxfp4_rmsnorm_quant(const void* x, int64_t ldx, void* residual, int64_t ldr, const void* weight, float eps,
                        int dtype, uint8_t* data, uint8_t* scales, int64_t M, int64_t K, void* stream);

/* C[M, N] = round(A B^T + bias): A [M, K], B [N, K] MXFP4, products and sums
 * of a block scaled and accumulated in fp32 by the tensor core
 * (tcgen05.mma kind::mxf4), bias[N] (nullable) and C of type `dtype` (bf16 or
 * fp16).  Any M and N; K % 32 == 0; 16-byte aligned operands. */
int mxfp4_gemm(const uint8_t* a_data, const uint8_t* a_scales, const uint8_t* b_data, const uint8_t* b_scales,
               const void* bias, void* C, int dtype, int64_t M, int64_t N, int64_t K, void* stream);

/* gate_up GEMM with SiLU*mul and requantisation in its epilogue: B = [gate
 * (I rows); up (I rows)] MXFP4 [2I, K], bias[2I] (nullable) of type `dtype`;
 * the result is MXFP4 of y = silu(A gate^T + bias) * (A up^T + bias), [M, I],
 * from the fp32 accumulators (the bias added in fp32), y not rounded before it
 * is quantised: values next to a rounding border are evaluated more closely,
 * up to 64 bits, as in mxfp4_silu_mul_quant.  I % 128 == 0 (W8A8_ERR_UNSUPPORTED otherwise:
 * take mxfp4_gemm_silu_quant_halves). */
int mxfp4_gemm_silu_quant(const uint8_t* a_data, const uint8_t* a_scales, const uint8_t* b_data,
                          const uint8_t* b_scales, const void* bias, int dtype, uint8_t* y_data,
                          uint8_t* y_scales, int64_t M, int64_t I, int64_t K, void* stream);

/* The scale tiles of [gate; up] ([2I, K], I % 32 == 0) as those of gate [I, K]
 * and then those of up [I, K], 2 mxfp4_scale_bytes(I, K) bytes in all: where
 * I % 128 != 0 the up rows start inside a tile, from where the tensor core
 * cannot read them.  16-byte aligned pointers. */
int mxfp4_half_scales(const uint8_t* scales, uint8_t* half_scales, int64_t I, int64_t K, void* stream);

/* mxfp4_gemm_silu_quant for any I % 32 == 0, with the scales of B as
 * mxfp4_half_scales lays them out. */
int mxfp4_gemm_silu_quant_halves(const uint8_t* a_data, const uint8_t* a_scales, const uint8_t* b_data,
                                 const uint8_t* b_half_scales, const void* bias, int dtype, uint8_t* y_data,
                                 uint8_t* y_scales, int64_t M, int64_t I, int64_t K, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MXFP4_H_ */
