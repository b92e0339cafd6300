/* SPDX-License-Identifier: Unlicense */

/* Operations of the B200 build without a counterpart in the reference's
 * ops.h: the channels-last ("token-major") 3 x 3 convolution the models
 * run (the reference's VGG convolutions, roma.c:742-768 and 1000-1027,
 * go through ops_conv2d on channel-major maps; this build keeps feature
 * maps channels-last so that every convolution is an implicit GEMM with
 * K-major operands), and the tensor-core status of the library. */

#ifndef I_COREGISTRATION_B200_OPS_B200_H
#define I_COREGISTRATION_B200_OPS_B200_H

#include "ops.h"

#ifdef __cplusplus
extern "C" {
#endif

/* 3 x 3 convolution, stride 1, zero padding 1, of a channels-last
 * (H, W, C) float32 map into (H, W, K): weights in the PyTorch layout
 * (K, C, 3, 3), bias per output channel (may be NULL), activation after
 * the bias. With o->precision OPS_BF16 and C a multiple of 64 it runs
 * as an implicit GEMM on tcgen05 tensor cores (the input and weights
 * rounded to bfloat16, 3-D TMA boxes of the map per tap, no im2col
 * buffer); otherwise in float32. */
void ops_conv3x3_cl(struct ops *o, cl_mem in, int H, int W, int C, cl_mem w,
                    cl_mem b, int K, int act, float slope, cl_mem out);

/* Multi-head attention of a fused token-major qkv buffer (N rows of 3 Dm
 * float32: queries, keys, values; head h at columns h (Dm / heads) of
 * each) into out (N x Dm): O = softmax(scale Q K^T) V per head, the
 * transformer attention of the models (the reference computes it with
 * two ops_gemm and ops_softmax_rows, roma.c:675-694). With o->precision
 * OPS_BF16 and a head size of 64 or 128 it runs the fused tcgen05 kernel
 * (bfloat16 operands, the probabilities rounded to bfloat16, float32
 * accumulation, no score matrix); otherwise the float32 kernel of
 * ops_attention. */
void ops_attention_qkv(struct ops *o, cl_mem qkv, int N, int Dm, int heads,
                       float scale, cl_mem out);

/* Depthwise 5 x 5 convolution, zero padding 2, + bias + ReLU of a
 * channels-last (H, W, C) float32 map into (H, W, C): the first half of a
 * RoMa refiner block with its BatchNorm folded (roma_dwconv5,
 * roma_kernels.cl:256-284, on channel-major maps). Weights (C, 1, 5, 5),
 * bias C floats. With o->precision OPS_BF16 the map is rounded to
 * bfloat16 and the model's bfloat16 kernel runs (float32 arithmetic,
 * bfloat16 result), as inside roma_match. */
void roma_dwconv5_cl(struct ops *o, cl_mem in, int H, int W, int C, cl_mem wt,
                     cl_mem bias, cl_mem out);

/* One hidden block of a RoMa refiner on a channels-last (H, W, C)
 * float32 map: out = W_pw relu(dw5x5(in) + b_dw) + b_pw, the depthwise
 * 5 x 5 convolution of roma_dwconv5_cl followed by the 1 x 1 convolution
 * the reference runs after it (roma.c:970-985, 1080-1094). pw_w is
 * (C, C) output-major, pw_b C floats. With o->precision OPS_BF16 and C
 * 32, 64 or 128 the model's fused tensor-core kernel runs (the depthwise
 * result rounded to bfloat16 in shared memory, float32 accumulation,
 * bfloat16 result); otherwise the two steps run one after the other. No
 * reference counterpart. */
void roma_refiner_block_cl(struct ops *o, cl_mem in, int H, int W, int C, cl_mem dw_w,
                           cl_mem dw_b, cl_mem pw_w, cl_mem pw_b, cl_mem out);

/* Local correlation of channels-last (H, W, C) float32 maps f1 and f2 at
 * the warp flow ((2, H, W) normalized coordinates, channel-major as in
 * the models) into out, channels-last (H, W, (2r + 1)^2): roma_local_corr
 * (roma_kernels.cl:153-192) on the models' layout. With o->precision
 * OPS_BF16 the maps are rounded to bfloat16 and the model's bfloat16
 * kernel runs (float32 arithmetic), as inside roma_match. */
void roma_local_corr_cl(struct ops *o, cl_mem f1, cl_mem f2, int C, int H, int W, int r,
                        cl_mem flow, cl_mem out);

/* ops_gemm that allocates no device memory; it has no counterpart in the
 * reference. Same arguments, meaning and results as ops_gemm. With
 * o->precision OPS_BF16, ops_gemm packs the operands to bfloat16 in a
 * buffer it grows with cudaMalloc; this variant packs them into a fixed
 * device array of ops_gemm_noalloc_max_bytes() bytes (16 MiB) that is part
 * of the library. It is meant for callers that must not allocate while
 * they run: a plug-in whose host framework's caching allocator already
 * holds the device's free memory, or a pipeline that does all allocation at
 * start-up because cudaMalloc synchronises the device. A product whose
 * packed operands, 2 (M + N) K nb bytes plus alignment, exceed the array is
 * rejected with an error naming the sizes (ops_gemm still runs it). The
 * first call on each device looks up the array's address and may load
 * the library's module there, so make it before any stream capture. All
 * calls on a device share the one array: calls that overlap in time
 * (several streams, host threads or ops contexts) corrupt each other's
 * results and must be serialised by the caller. Float32 products
 * (OPS_FP32, or shapes the tensor-core path does not take) stage nothing. */
void ops_gemm_noalloc(struct ops *o, int M, int N, int K, struct opnd A,
                      struct opnd B, int transb, struct opnd C, int nb, int nb1,
                      cl_mem bias, int biasrow, cl_mem R, long roff, float alpha,
                      int act, float slope);

/* Size in bytes of ops_gemm_noalloc's scratch array. */
size_t ops_gemm_noalloc_max_bytes(void);

/* ---- 8-bit linear layers, rotary positions, group norm ----
 *
 * Element types are named per buffer, apart from o->precision: OPS_FP32
 * float, OPS_BF16 bfloat16 (offsets, leading dimensions and strides in
 * elements of that type). The entry points below check their operands
 * against the buffers' sizes, run on the ops context's device whichever
 * the calling thread's current one is, allocate nothing, and may be
 * captured into a CUDA graph; an empty call (no rows, no columns, no
 * pixels) does nothing. Outputs may not overlap inputs but where said. */

/* x sigmoid(x): an activation of the operations below only. */
#define ACT_SILU 5

/* Largest product depth of ops_gemm_i8: 2^17 - 1, so that no sum of
 * products of 8-bit integers passes 32 bits. */
#define OPS_I8_MAX_K 131071

/* Row pitch in bytes of K 8-bit integers for ops_gemm_i8: K rounded up to
 * a multiple of 16. */
int ops_i8_ld(int K);

/* Rows of X (rows x C, C at most 2^30, type xtype) to 8-bit integers with
 * one scale each:
 *   s = max |x| / 127 (float32, rounded to nearest), q = x / s
 * rounded to the nearest integer (ties to even; decided on the exact
 * quotient) within -127..127. Q holds bytes (Q.ld in bytes), S float32
 * from element soff on, one per row. A row of zeros gets s = 0 and q = 0;
 * a row that holds an infinity or NaN gets s = NaN and q = 0, so that the
 * products of that row alone are NaN. Used for tokens (a scale per token)
 * and for weights (W is out x in: a scale per output channel). No
 * reference counterpart. */
void ops_quant_i8(struct ops *o, long rows, int C, struct opnd X, int xtype, struct opnd Q,
                  cl_mem S, long soff);

/* C = act((A B^T) sa sb + bias) + R for 8-bit A (M x K, a scale sa[i] per
 * row) and B (N x K, the PyTorch Linear layout, a scale sb[j] per row):
 * the sums are exact 32-bit integers. A and B start at a multiple of 16
 * bytes and their ld is one too (ops_i8_ld; bytes beyond K are not used).
 * bias is float32 per column or NULL; R is NULL or a buffer of C's type
 * and layout from element roff on, and may be C itself. ctype is the type
 * of C and R. K is at most OPS_I8_MAX_K; K = 0 gives act(bias) + R,
 * whatever the scales hold (ops_quant_i8 writes none for rows without
 * columns). A sum times sa is rounded to float32 before sb: it cannot overflow
 * there for rows of values below 2e31. Up to 8 rows of small layers run
 * kernels that stream B once, others the tcgen05 integer tensor cores, in deep
 * products of few tiles with the depth split; a row's results are the same
 * bits by all of them. No reference counterpart (ops_gemm there is float32
 * only). */
void ops_gemm_i8(struct ops *o, int M, int N, int K, struct opnd A, cl_mem sa, struct opnd B,
                 cl_mem sb, cl_mem bias, struct opnd C, int ctype, cl_mem R, long roff, int act,
                 float slope);

/* Size in bytes of the work buffer of ops_linear_i8 (0: none needed). */
size_t ops_linear_i8_bytes(int rows, int in);

/* ops_linear over 8-bit weights: Y[rows, out] = act(X[rows, in] W^T + b)
 * + R with X (type xtype) quantised per row as by ops_quant_i8, W and sw
 * the weights' rows and scales as ops_quant_i8 left them, and the other
 * arguments as in ops_gemm_i8 (Y is C there). The same result as
 * ops_quant_i8 followed by ops_gemm_i8; few rows take one launch. work:
 * at least ops_linear_i8_bytes(rows, in) bytes of device memory at a
 * multiple of 16 bytes, NULL where that is 0; calls that may overlap in
 * time (streams, graphs) each need their own. No reference counterpart. */
void ops_linear_i8(struct ops *o, int rows, int in, int out, struct opnd X, int xtype,
                   struct opnd W, cl_mem sw, cl_mem bias, struct opnd Y, int ytype, cl_mem R,
                   long roff, int act, float slope, cl_mem work);

/* Frequencies of a rotary encoding (ops_rotary_plan fills it). */
#define OPS_ROTARY_MAX 256 /* Largest number of rotated columns. */
struct ops_rotary {
    int rot;         /* Rotated columns of each head, from its first on. */
    int axes;        /* Positions per token: 1, or 2 (row and column). */
    int interleaved; /* Pairs (2f, 2f + 1), or (f, f + rot / 2) with 0. */
    float mscale;    /* Factor on the rotated columns. */
    uint64_t step[OPS_ROTARY_MAX / 2]; /* Turns per position, in 2^-64. */
};

/* Frequency scalings: for positions beyond those a model was trained on. */
#define OPS_ROTARY_PLAIN 0
#define OPS_ROTARY_LINEAR 1 /* Every frequency over factor. */
#define OPS_ROTARY_NTK 2    /* base times factor^(n / (n - 2)). */
#define OPS_ROTARY_PARTS 3  /* Few turns over length: over factor; many: kept. */

/* The frequencies of rot columns (even; a multiple of 2 axes): with n =
 * rot / axes columns per axis, w_i = base^(-2 i / n) radians per position
 * for i < n / 2, first those of axis 0, then those of axis 1. scaling
 * changes them by factor (> 0): LINEAR divides them; NTK raises the base
 * (n > 2); PARTS (the "NTK-by-parts" rule of YaRN, Peng et al. 2023)
 * takes g w + (1 - g) w / factor with g = clamp((r - 1) / 31, 0, 1) for r =
 * length w / 2 pi turns over the trained length, and sets mscale to
 * 0.1 ln(factor) + 1 for factors above 1 (1 otherwise). Host only; no device
 * is needed. */
void ops_rotary_plan(struct ops_rotary *r, int rot, int axes, int interleaved, double base,
                     int scaling, double factor, long length);

/* Rotary positions of rows x nh heads of d columns (at most 2^30 in a row; a
 * token's heads beside each other: the queries, or queries and keys, of a qkv buffer): Y = X
 * with each pair (a, b) of a head's first r->rot columns replaced by
 * mscale (a cos t - b sin t, a sin t + b cos t), t = w_f p, and the other
 * columns as they were. p is pos0 plus the token's entry of pos (int32,
 * rows x axes, packed), or pos0 + row with pos NULL (one axis only).
 * Angles are kept as 64-bit fractions of a turn, exact to 2^-33 turns at
 * any 31-bit position. Y may be X (in place: only rotated columns are
 * read and written) or memory of its own. ops_rope is the float32 form
 * with a table. No reference counterpart. */
void ops_rotary(struct ops *o, const struct ops_rotary *r, long rows, int nh, int d,
                struct opnd X, struct opnd Y, int type, cl_mem pos, long pos0);

/* Size in bytes of the work buffer of ops_groupnorm_cl (0: none needed). */
size_t ops_groupnorm_cl_bytes(int nimg, long HW, int C, int groups);

/* Group norm with an activation over nimg (at most 65535) channels-last maps
 * (HW pixels of C channels, both at most 2^30; image i from X.off + i X.s0
 * on, pixels X.ld apart):
 * Y = act((x - mean) / sqrt(var + eps) g[c] + b[c]) with the mean and the
 * biased variance of each image's C / groups neighbouring channels over
 * all pixels, held in float32; g and b float32 (both or neither NULL). A group
 * whose squared distances from its mean add up to more than float32 holds (of
 * values beyond some 1e16) has an infinite variance: Y = act(b); one whose
 * values themselves add up to more (beyond some 1e30) is NaN.
 * Y may be X (the same offset, strides and type). work: at least
 * ops_groupnorm_cl_bytes() bytes of device memory at a multiple of 16
 * bytes, NULL where that is 0; calls that may overlap in time each need
 * their own. No reference counterpart (ops_chan_stats and
 * ops_chan_affine normalise single channels of channel-major maps). */
void ops_groupnorm_cl(struct ops *o, int nimg, long HW, int C, int groups, struct opnd X,
                      int xtype, struct opnd Y, int ytype, cl_mem g, cl_mem b, float eps,
                      int act, float slope, cl_mem work);

/* Non-zero when a bounded wait of a tensor-core kernel ran out since the
 * last call (the kernel then stopped and its results are invalid); the
 * code is cleared. */
int coreg_tc_status(void);

#ifdef __cplusplus
}
#endif

#endif /* I_COREGISTRATION_B200_OPS_B200_H */
