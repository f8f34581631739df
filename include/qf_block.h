/*
 * qf_block.h — C ABI of the MI355X (gfx950) operators for block-scaled FP8 checkpoints: e4m3 weights with one fp32
 * scale for each 128 x 128 block, W[n, k] = q[n, k] * scale[n / 128, k / 128].
 *
 *   qf_fp8_w8a16_gemm     the product at decode widths (M <= 16), bf16 activations
 *   qf_fp8_w8a8_linear    the product at any M, activations quantised per token and block of 128
 *   qf_quantize_tokens_fp8  that quantiser by itself
 *   qf_block_norm_rows    the norms before and after a block, with its gate and residual scale
 *   qf_moe_few_tokens     a whole mixture-of-experts layer for up to 16 tokens
 *
 * Pointers are device pointers, strides are in elements, the last dimension is contiguous, calls run on `stream` (a
 * hipStream_t, NULL = the null stream) without host synchronisation and may be captured in a HIP graph.  Every entry
 * point checks its arguments before any HIP call and returns a qf_status.  Results do not depend on timing: sums run in
 * a fixed order.
 *
 * Layouts of e4m3 weights (qf_layout): row-major [N, K] with row stride ldw, or the TILED image of the same bytes that
 * qf_w8a16_repack makes (1 KiB tiles of 16 channels x 64 k).  K % 64 == 0; the last block of K may be half a block and
 * the last block of N any part of one.
 */
#ifndef QF_BLOCK_H
#define QF_BLOCK_H

#include <stddef.h>
#include <stdint.h>

#include "qf_w8a16.h" /* qf_status, qf_layout, qf_dtype */

#ifdef __cplusplus
extern "C" {
#endif

#define QF_BLOCK_ABI_VERSION 1
/* Values a scale covers, along N and along K. */
#define QF_FP8_BLOCK 128
/* Largest M of qf_fp8_w8a16_gemm and T of qf_moe_few_tokens. */
#define QF_FP8_MAX_DECODE_M 16
/* Longest K of qf_fp8_w8a8_linear. */
#define QF_FP8_MAX_W8A8_K 262144
/* Longest row of qf_block_norm_rows. */
#define QF_BLOCK_NORM_MAX_N 32768
/* Most experts, and experts a token, of qf_moe_few_tokens. */
#define QF_MOE_MAX_EXPERTS 512
#define QF_MOE_MAX_TOP_K 16

typedef enum qf_gate { QF_GATE_NONE = 0, QF_GATE_CHANNEL = 1, QF_GATE_TOKEN = 2, QF_GATE_FULL = 3 } qf_gate;
typedef enum qf_act { QF_ACT_NONE = 0, QF_ACT_SIGMOID = 1 } qf_act;

/* ABI version of the loaded library (QF_BLOCK_ABI_VERSION). */
int qf_block_abi_version(void);

/* y[m, n] = sum over blocks of scale[n / 128, kb] * sum_{k in kb} x[m, k] * q[n, k] (+ bias[n]): x bf16 [M, K] (row
 * stride ldx), w e4m3, scale fp32 [ceil(N / 128), ceil(K / 128)] contiguous, bias bf16 [N] or NULL, y bf16 or fp32
 * [M, N] (row stride ldy).  1 <= M <= 16.  Products are exact, sums fp32, y is rounded once.  x and w 16-byte aligned,
 * ldx % 8 == 0, row-major ldw % 16 == 0, both at most 2^26, else QF_ERR_UNSUPPORTED.  (Where K is split, one arrival counter
 * serves several tiles of 16 channels; QF_W8A16_COUNTER_BYTES of them reach past a million channels.) */
int qf_fp8_w8a16_gemm(const uint16_t* x, int64_t ldx, const uint8_t* w, int64_t ldw, int layout, const float* scale,
                      const uint16_t* bias, void* y, int64_t ldy, int out_dtype, int M, int N, int K, void* workspace,
                      size_t workspace_bytes, void* stream);

/* Bytes of workspace of qf_fp8_w8a16_gemm: 0 where K is not split (and for sizes that are not served), else
 * QF_W8A16_COUNTER_BYTES of arrival counters, which must be zero and are left zero, and the partial sums; calls that may
 * run at the same time need distinct ones (16-byte aligned).  Host-only. */
size_t qf_fp8_w8a16_workspace_bytes(int M, int N, int K, int layout);

/* xq[m, k] = e4m3(x[m, k] / s_a[m, kb]), s_a[m, kb] = max_{k in kb} |x[m, k]| / 448 in fp32, both roundings to nearest
 * even; a block of zeros has scale 0 and values 0, a block that holds an infinity or NaN gives NaN there.  x bf16 [M, K]
 * (row stride ldx), xq e4m3 [M, K] (row stride ldq, a multiple of 8, 8-byte aligned), s_a fp32 [M, ceil(K / 128)]
 * contiguous.  K % 64 == 0. */
int qf_quantize_tokens_fp8(const uint16_t* x, int64_t ldx, int M, int K, uint8_t* xq, int64_t ldq, float* s_a,
                           void* stream);

/* Bytes of workspace of qf_fp8_w8a8_linear: the quantised activations with their scales, and the partial sums where K is
 * split.  0 for sizes that are not served.  Host-only. */
size_t qf_fp8_w8a8_workspace_bytes(int M, int N, int K);

/* y[m, n] = sum over blocks of s_a[m, kb] * scale[n / 128, kb] * sum_{k in kb} xq[m, k] * q[n, k] (+ bias[n]), with xq and
 * s_a those of qf_quantize_tokens_fp8.  The products are not exact: of 8 neighbouring k (from a multiple of 8 on) the f8
 * matrix instruction adds them aligned to the largest exponent sum e among them (of 2^e <= |xq q| < 2^(e + 2)), and drops
 * what lies below 2^(e - 13); products that are multiples of it are added whole.  Measured on normal values that is 1.5e-5
 * to 3.6e-5 of a result, about 15 bits, also with fp32 output.  The sums of the groups and blocks are fp32, y is rounded
 * once.  1 <= M < 2^28, K <= QF_FP8_MAX_W8A8_K; shapes, strides, layouts and alignment as qf_fp8_w8a16_gemm.  The workspace
 * needs no clearing and is free again when the last launch ends; calls that may run at the same time need distinct ones
 * (16-byte aligned). */
int qf_fp8_w8a8_linear(const uint16_t* x, int64_t ldx, const uint8_t* w, int64_t ldw, int layout, const float* scale,
                       const uint16_t* bias, void* y, int64_t ldy, int out_dtype, int M, int N, int K,
                       void* workspace, size_t workspace_bytes, void* stream);

/* p = x * rsqrt(mean(x^2) + eps) * (weight_offset + post_weight), or x itself where post_weight is NULL;
 * y = residual + alpha * act(gate) * p;  h = y * rsqrt(mean(y^2) + eps) * (weight_offset + pre_weight) (of y before its
 * rounding; pre_weight NULL: no factor).  x bf16 [M, N]; residual and y bf16, or fp32 with residual_f32; h bf16; weights
 * bf16 [N]; gate bf16: none, [N] (CHANNEL), one a row (TOKEN, stride ldg) or [M, N] (FULL).  y may be the residual and h
 * may be x (the same rows); no other overlap.  N % 8 == 0, N <= QF_BLOCK_NORM_MAX_N, 16-byte aligned rows. */
int qf_block_norm_rows(const uint16_t* x, int64_t ldx, const void* residual, int64_t ldr, int residual_f32,
                       const uint16_t* post_weight, const uint16_t* pre_weight, float weight_offset,
                       const uint16_t* gate, int64_t ldg, int gate_kind, int gate_act, float alpha, float eps, int M,
                       int N, void* y, int64_t ldy, uint16_t* h, int64_t ldh, void* stream);

/* Bytes of workspace of qf_moe_few_tokens; 0 for sizes that are not served.  Host-only. */
size_t qf_moe_few_workspace_bytes(int T, int E, int top_k, int H, int I);

/* One mixture-of-experts layer for T <= 16 tokens: token t takes the top_k largest of its E router logits (the lowest
 * index first among equal ones, NaN largest), weighs expert e by c = softmax(logits)[e] (divided by the sum of the
 * chosen ones with renormalize; 0 for a row of -inf only, and an expert of weight 0 is not read for that token), and
 *   y[t] = sum_e c[t, e] * W2_e a_e,   a_e = silu(Wgate_e x[t]) * (Wup_e x[t]), kept to 16 bits between the products.
 * x bf16 [T, H], logits bf16 or fp32 [T, E] (row stride ldl), y bf16 [T, H].  w13: the TILED image of [E * 2 I, H] (each
 * expert's I gate rows, then its I up rows), s13 fp32 [E, 2, ceil(I / 128), ceil(H / 128)]; w2: the image of [E * H, I],
 * s2 fp32 [E, ceil(H / 128), ceil(I / 128)].  H and I multiples of 64, top_k <= min(E, QF_MOE_MAX_TOP_K), E <=
 * QF_MOE_MAX_EXPERTS.  Workspace as for qf_fp8_w8a8_linear. */
int qf_moe_few_tokens(const uint16_t* x, int64_t ldx, const void* logits, int64_t ldl, int logits_f32, const uint8_t* w13,
                      const float* s13, const uint8_t* w2, const float* s2, uint16_t* y, int64_t ldy, int T, int E,
                      int top_k, int H, int I, int renormalize, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* QF_BLOCK_H */
