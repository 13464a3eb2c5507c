// gen9blas MI355X: operators of large language models on 4-bit weights and mixtures of experts (libgen9blas_llm.so).
//
// These entry points have no counterpart in the reference. They live in a library of their own, beside libgen9blas.so
// (which exports the reference's surface only), and run on its stream and device: gen9blas_init opens the device,
// gen9blas_hip_stream() gives the stream, gen9blas_flush() waits.
//
// Rules shared by every entry point
// - Operands are device memory, used in place at any element alignment. One in host memory, or one that runs past the
//   end of its allocation, is INVALID_ARG before anything runs. A result overlaps no operand.
// - A call queues its kernels on the library's stream and returns; gen9blas_flush() waits for them. The stream orders
//   itself after work on the legacy null stream and before work queued there later.
// - Return value: 0, or a negative gen9blas_status with the text in gen9blas_llm_error(). Functions returning pointers
//   return NULL on error and set gen9blas_llm_last_status(). Non-positive M, T or rows make a call a no-op.
// - Work buffers belong to the process and grow on demand (growing waits for queued work): callers serialize calls.
// - type is GEN9BLAS_H (FP16) or GEN9BLAS_S (FP32); sums are FP32, each result is rounded once.
#pragma once
#include <stddef.h>
#include <stdint.h>
#include "gen9blas.h"
#ifdef __cplusplus
extern "C" {
#endif

// The text of the last error of this library, and the status of its last call.
GEN9BLAS_API const char *gen9blas_llm_error(void);
GEN9BLAS_API int gen9blas_llm_last_status(void);

// ---- Microscaled 4-bit matrices (MX4) ----
// Rows of E2M1 values (±0, 0.5, 1, 1.5, 2, 3, 4, 6), each 32 consecutive values of a row sharing one E8M0 scale 2^(s−127),
// s = 0..254 (255: every value of the block is NaN), as in the OCP Microscaling Formats specification (MXFP4).
// `count` matrices of `rows` × K in one object (count > 1: the weights of `count` experts), in device memory that the
// object owns, in the order in which the matrix cores take them. Limits: count, rows, K ≥ 1, K ≤ 2^31 − 128, and
// count · ⌈rows/16⌉ · ⌈K/512⌉ < 2^24 (137 G values).
typedef struct gen9blas_mx4 gen9blas_mx4;
// A matrix (or `count` of them) of zeros.
GEN9BLAS_API gen9blas_mx4 *gen9blas_mx4_create(int count, int rows, int K);
// Waits for queued work, then frees the matrix. NULL is a no-op.
GEN9BLAS_API void gen9blas_mx4_free(gen9blas_mx4 *Q);
// Q = X rounded to MX4; matrix b at X + b·sX, row stride ldx (elements). The scale of a block is 2^(⌊log2 max|x|⌋ − 2)
// (at least 2^−127); x / scale goes to the nearest E2M1 value, ties to the even code, beyond 6 to ±6. A block that
// holds an infinity or NaN becomes NaN.
GEN9BLAS_API int gen9blas_mx4_quantize(int type, const void *X, int ldx, int64_t sX, gen9blas_mx4 *Q);
// Q from rows as checkpoints hold them: two codes to a byte, the even one in the low half (bit 3 of a code is the sign),
// row stride ldc bytes; and a byte s for each 32 values, row stride lds bytes. Matrix b follows at rows · ldc and
// rows · lds bytes.
GEN9BLAS_API int gen9blas_mx4_load(const uint8_t *codes, int ldc, const uint8_t *scales, int lds, gen9blas_mx4 *Q);
// X = the values of Q, in FP32 (exact but for values past 2^128, which are infinite there).
GEN9BLAS_API int gen9blas_mx4_dequantize(const gen9blas_mx4 *Q, float *X, int ldx, int64_t sX);
// C (M×N) = A (M×K, FP16 or FP32) · Wᵀ, W (N×K) a single MX4 matrix. The products are exact, but for: FP16, terms of a row
// of W more than 2^36 below its largest scale may be rounded; FP32, elements of A below 2^−110 lose the bits below 2^−133,
// products are FP32 numbers (nothing below 2^−149), and a value of W past 2^128 is infinite. C in the type of A.
GEN9BLAS_API int gen9blas_mx4_gemm(int type, int M, const void *A, int lda, const gen9blas_mx4 *W, void *C, int ldc);
// C (M×N, FP16 or FP32 as `type` says) = A · Wᵀ, both MX4 (M×K, N×K): products on the 4-bit matrix cores.
GEN9BLAS_API int gen9blas_mx4_gemm_q(int type, const gen9blas_mx4 *A, const gen9blas_mx4 *W, void *C, int ldc);

// ---- Mixture of experts ----
// score: how a logit becomes an expert's score.
enum { GEN9BLAS_SOFTMAX = 0, GEN9BLAS_SIGMOID = 1 };
// The k experts of each token and their weights, from the router's logits (T×E, row stride ldl, 1 <= E <= 1024,
// 1 <= k <= min(E, 64)).
// - choice: by score + bias (bias: E floats or NULL; softmax without a bias: by the logit, which is in the same order),
//   the largest first, the lowest index first among equal ones.
// - groups > 1 (at most 64, a divisor of E): only the experts of the top_groups best groups of E/groups consecutive
//   experts are chosen; a group counts as the sum of its two largest choices (sigmoid) or its largest one (softmax).
// - weights: the chosen experts' scores (without bias), divided by their sum if renorm, times scale.
// - A logit of −inf is an expert that is masked: never chosen. Places that are left over get id −1 and weight 0. A NaN
//   logit is not chosen either, and makes the row's weights NaN (softmax with a bias: all scores of the row are NaN, so all
//   its ids are −1). Scores whose sum is 0 renormalise to weights 0.
// ids and weights are T×k, dense.
GEN9BLAS_API int gen9blas_moe_route(int type, int T, int E, const void *logits, int ldl, const float *bias, int score,
                                    int groups, int top_groups, int k, int renorm, float scale, int *ids, float *weights);
// The products of each token's rows with its experts' weights. ids: T×S, dense; W: E = count matrices N×K (E <= 1024).
// The row of token t, place s is X + t·ldt + s·lds (lds = 0: one row for all places of a token); y(t, s) = row · W[ids(t, s)]ᵀ.
// - gate != NULL (as W): y(t, s) = silu(row · gate[ids(t, s)]ᵀ) · (row · W[ids(t, s)]ᵀ), silu(z) = z / (1 + e^−z).
// - weights == NULL: C(t, s) = y(t, s) at C + t·ldct + s·ldcs (ldcs >= N, ldct >= (S − 1)·ldcs + N).
// - weights (T×S floats, dense): C(t) = Σ_s weights(t, s) · y(t, s) at C + t·ldct, in the order of s; ldcs is not read. S = 0: zeros
//   (weights still not NULL, ids and X not read).
// An id outside 0..E−1 is an empty place: its y is 0, and its weight is not read.
GEN9BLAS_API int gen9blas_moe_gemm(int type, int T, int S, const int *ids, const void *X, int64_t ldt, int64_t lds,
                                   const gen9blas_mx4 *W, const gen9blas_mx4 *gate, const float *weights, void *C,
                                   int64_t ldct, int64_t ldcs);

#ifdef __cplusplus
}
#endif
