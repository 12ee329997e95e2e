/*
 * gpvae_lowbit.h — C ABI of libgpvae_lowbit.so: dense layers with weights in 4 bits, and checkpoints of activations
 * in 8 bits, for the encoder / decoder of a GP-prior VAE on MI355X (gfx950).
 *
 * The conventions are those of gpvae.h (plain C, DEVICE pointers owned by the caller, row-major matrices with a
 * leading dimension in elements, asynchronous stream-ordered calls that never synchronise and never allocate, return
 * value 0 or -(1-based index of the first bad argument), gpvae_lowbit_last_error() for the reason), with these
 * differences:
 *   - `dtype` is the type of the floating matrices: GPVAE_LB_F32, GPVAE_LB_BF16 or GPVAE_LB_F16 (sums are float32
 *     in every case); 1 (float64 in gpvae.h) is refused;
 *   - any element-aligned base pointer and any leading dimension >= the number of columns is accepted, and nothing
 *     outside the rows x cols elements of a matrix is read or written;
 *   - code and exponent arrays are dense, 16-byte aligned, of the sizes the *_bytes queries give.
 *
 * Both formats keep ONE power of two 2^e for a square tile of 8 x 8 values, as the byte e + 127.  e is the smallest
 * integer (>= -125 for w4, >= -126 for q8) with largest magnitude <= top * 2^e (top: 6 for w4, 127 for q8, 255 for q8
 * after a ReLU; a tile of zeros has e = 0), but at most 125 (w4), 121 (q8), 120 (q8 after a ReLU): top * 2^e stays
 * finite, and only magnitudes above it (2.55e38 for w4, 3.38e38 for q8) saturate.  A tile that holds an infinity or a NaN gets the byte 255 and
 * reads as NaN throughout.  Every value the formats can hold is exactly a bfloat16 number.
 * The products take a floating operand apart into bfloat16 pieces without rounding (three for float32, two for float16;
 * bits below 2^-133, bfloat16's smallest, are dropped), so that only the float32 sums round.
 *
 *   w4   weights W [K, N] of a dense layer y = x W + b:  codes uint32 [ceil(K/32)][Np][4], Np = N rounded up to 32:
 *        nibble i (low first) of codes[kb][n][j] is row 32 kb + 8 j + i of column n — bit 3 the sign, bits 0-2 one of
 *        0, 0.5, 1, 1.5, 2, 3, 4, 6.  exps uint8 [ceil(K/32)][Np / 8][4]: tile (rows 32 kb + 8 j ..., columns 8 t ...)
 *        at [kb][t][j].  Rows past K and columns past N hold zero codes.
 *   q8   a matrix X [M, K]: codes uint8 [ceil(M/8)][Kp][8], Kp = K rounded up to 32: byte i of codes[mb][k] is row
 *        8 mb + i of column k — two's complement, or 0 .. 255 when stored with relu != 0.  exps uint8
 *        [ceil(M/8)][Kp / 8].  Rows past M and columns past K hold zero codes.
 */
#ifndef GPVAE_LOWBIT_H
#define GPVAE_LOWBIT_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define GPVAE_LOWBIT_ABI_VERSION 1

enum { GPVAE_LB_F32 = 0, GPVAE_LB_BF16 = 2, GPVAE_LB_F16 = 3 };

int gpvae_lowbit_abi_version(void);
const char *gpvae_lowbit_last_error(void);

/* ---- w4: weights in 4 bits ------------------------------------------------------------------------------
 * gpvae_quant_w4   W [K, ldw] -> codes, exps: every value to the nearest of its tile's 15, ties to the even code.
 * gpvae_load_w4    the values W~ the codes stand for, out [K, ldo] (exact in float32 and bfloat16).
 * 1 <= K <= 2^30, 1 <= N <= 2^25 (here and in the products; M up to 2^30 in every call).  A workspace query of sizes
 * that its call refuses gives 0.                                                                            */
int64_t gpvae_w4_code_bytes(int64_t K, int64_t N);
int64_t gpvae_w4_exp_bytes(int64_t K, int64_t N);
int gpvae_quant_w4(void *stream, int dtype, int64_t K, int64_t N, const void *W, int64_t ldw, void *codes, void *exps);
int gpvae_load_w4(void *stream, int dtype, int64_t K, int64_t N, const void *codes, const void *exps, void *out,
                  int64_t ldo);

/* Y[m][n] = act(sum_k X[m][k] W~[k][n] + bias[n]); bias [N] (dtype) may be NULL; relu != 0: act = max(0, .).
 * X [M, ldx], Y [M, ldy], not overlapping.  work: gpvae_dense_w4_workspace_bytes() bytes, 16-byte aligned
 * (may be NULL when that is 0); its contents on entry do not matter.  Same inputs, same bits.               */
int64_t gpvae_dense_w4_workspace_bytes(int dtype, int64_t M, int64_t K, int64_t N);
int gpvae_dense_w4(void *stream, int dtype, int64_t M, int64_t K, int64_t N, const void *X, int64_t ldx,
                   const void *codes, const void *exps, const void *bias, int relu, void *Y, int64_t ldy, void *work);

/* The product with the transposed weights: dX[m][k] = sum_n dY[m][n] W~[k][n] where mask[m][k], 0 elsewhere (whatever
 * the sum is there, an infinity or a NaN too).  dY [M, lddy], dX [M, lddx], not overlapping.
 * act_codes: the q8 codes of the layer's input A [M, K] stored with relu != 0; mask = (code != 0), i.e. A > 0 or NaN, so
 * dX is the gradient BEFORE the previous layer's ReLU.  act_codes NULL: no mask.                            */
int64_t gpvae_dense_vjp_w4_workspace_bytes(int dtype, int64_t M, int64_t K, int64_t N);
int gpvae_dense_vjp_w4(void *stream, int dtype, int64_t M, int64_t K, int64_t N, const void *dY, int64_t lddy,
                       const void *codes, const void *exps, const void *act_codes, void *dX, int64_t lddx, void *work);

/* ---- q8: activation checkpoints in 8 bits -----------------------------------------------------------------
 * gpvae_store_q8   relu == 0: the checkpoint of X [M, ldx] (nearest, ties to even; Y must be NULL).
 *                  relu != 0: Y = max(X, 0) (NaN stays NaN) and the checkpoint of Y, codes 0 .. 255; a positive
 *                  value never becomes code 0, so (code != 0) is the ReLU's mask.  Y [M, ldy] may be NULL, or X
 *                  itself (ldy == ldx), and must not overlap X otherwise.
 * gpvae_load_q8    the values X~ the checkpoint stands for, out [M, ldo] (exact in float32; exact in bfloat16).
 * M = 0 is an empty checkpoint; K >= 1.                                                                     */
int64_t gpvae_q8_code_bytes(int64_t M, int64_t K);
int64_t gpvae_q8_exp_bytes(int64_t M, int64_t K);
int gpvae_store_q8(void *stream, int dtype, int64_t M, int64_t K, const void *X, int64_t ldx, int relu, void *Y,
                   int64_t ldy, void *codes, void *exps);
int gpvae_load_q8(void *stream, int dtype, int64_t M, int64_t K, int relu, const void *codes, const void *exps,
                  void *out, int64_t ldo);

/* Parameter gradients of a dense layer y = x W + b from the checkpoint of its input:
 *   dW[k][n] = sum_m X~[m][k] dY[m][n],   db[n] = sum_m dY[m][n]       (float32, overwritten; M = 0: zeros)
 * dW and db must not overlap dY or each other.
 * relu: how the checkpoint was stored.  dY [M, lddy] (dtype); dW [K, lddw]; db [N] may be NULL.  work as above.
 * N and (for M > 1) lddy at most 2^26, ceil(K / 128) ceil(N / 128) below 2^23. */
int64_t gpvae_dense_grads_q8_workspace_bytes(int dtype, int64_t M, int64_t K, int64_t N);
int gpvae_dense_grads_q8(void *stream, int dtype, int64_t M, int64_t K, int64_t N, int relu, const void *codes,
                         const void *exps, const void *dY, int64_t lddy, float *dW, int64_t lddw, float *db, void *work);

#ifdef __cplusplus
}
#endif
#endif /* GPVAE_LOWBIT_H */
