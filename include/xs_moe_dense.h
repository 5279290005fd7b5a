/*
 * xs_moe_dense.h -- C ABI of the dense operators around the MoE layer: projections and a gated MLP whose weights are held as
 * 4-bit integers with group scales, and the norm / gate / residual step between two blocks.
 *
 * Conventions as in xs_moe.h: plain pointers and sizes, 0 or a negative XsMoeStatus, device pointers marked _dev, contiguous
 * row-major tensors, work is enqueued on `stream` and the call returns without waiting, every call can be captured into a
 * graph.  Tensors must live on the current device; a pointer to host memory or to another device's memory is refused
 * ("device mismatch").  A workspace serves calls that do not overlap on the device: two streams, or two graphs that may run
 * at the same time, need one each.  xs_moe_workspace_init clears its status word once, xs_moe_check_flags reads it.
 * tokens == 0 is a valid call that does nothing.
 */
#ifndef XS_MOE_DENSE_H
#define XS_MOE_DENSE_H

#include "xs_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A matrix W (rows, cols) in 4 bits:  W[n][k] = (q[n][k] - z[n][k / group]) * s[n][k / group].
 *   codes  (rows, cols / 2) bytes   q in 0..15, the even column in the low nibble (the byte order of XS_MOE_FP4_MX32)
 *   scales (rows, cols / group)     bf16, any value
 *   zeros  (rows, cols / group)     bytes, the low four bits are the zero point; NULL: 8 everywhere
 * group is 32, 64 or 128; cols is a multiple of group; rows is any positive number; none is above 2^30.  codes are 16-byte aligned, scales 2-byte.
 * The reference has no quantised weights (xstar_cpp/include/dtype.h:8-12); the matrix takes the place of `weight` in its
 * linear op, x * W^T (xstar_cpp/src/ops/linear.cpp:20-31). */
typedef struct XsMoeW4 {
    const void *codes_dev;
    const void *scales_dev;
    const uint8_t *zeros_dev;
    int32_t rows;
    int32_t cols;
    int32_t group;
    int32_t reserved; /* must be zero */
} XsMoeW4;

typedef enum XsMoeActivation {
    XS_MOE_SILU = 0,     /* v / (1 + exp(-v)) */
    XS_MOE_GELU_TANH = 1 /* v / 2 * (1 + tanh(sqrt(2 / pi) * (v + 0.044715 v^3))) */
} XsMoeActivation;

/* out (tokens, rows) bf16 = x (tokens, cols) bf16 times W^T; f32 sums, one rounding at the end.  Small
 * batches (up to 8 tokens of 32768 columns, up to 16 of 8192) multiply with the exact weights; their tokens are below 2^123, so that a
 * group's sum of (q - z) x is within f32.  Larger ones go to the tensor core in f16, tokens and weight rows scaled by powers of
 * two: a weight is rounded once to 11 bits, fewer where its scale is below 2^-20 of the largest of its row, and tokens are exact
 * down to 2^-27 of their largest element (smaller elements are off by 2^-39 of it at most).
 * x is 16-byte aligned; what a call writes may not overlap what it reads.  Takes the role of gemm_launch behind linear
 * (xstar_cpp/include/ops/gemm.h:165-176). */
int xs_moe_linear_w4_workspace_bytes(const XsMoeW4 *w, int32_t tokens, size_t *bytes);
int xs_moe_linear_w4(const XsMoeW4 *w, const void *x_dev, int32_t tokens, void *out_dev, void *workspace_dev,
                     size_t workspace_bytes, void *stream);

/* h (tokens, I) bf16 = act(x Wg^T) * (x Wu^T), gate_up (2I, H) with the I gate rows first: both projections, the activation and
 * the product in one kernel, f32 until the one rounding of h.  Takes the role of gemm_silu_and_mul_launch
 * (xstar_cpp/include/ops/mlp.h:95-102).  Workspace: xs_moe_linear_w4_workspace_bytes of gate_up. */
int xs_moe_gated_w4(const XsMoeW4 *gate_up, int32_t activation, const void *x_dev, int32_t tokens, void *h_dev,
                    void *workspace_dev, size_t workspace_bytes, void *stream);

/* out (tokens, H) bf16 = (act(x Wg^T) * (x Wu^T)) Wd^T, gate_up (2I, H), down (H, I): the reference's
 * mlp(x, gate_up_weight, down_weight) (xstar_cpp/include/ops/mlp.h:51) with 4-bit weights.  The product of the first half is
 * held in f32 and rounded once, to f16, after a power of two has brought each token's largest element of it (up to 16 tokens: each
 * part of a token that is summed together) to 2^13 .. 2^14: 11 bits down to 2^-27 of that element. */
int xs_moe_mlp_w4_workspace_bytes(const XsMoeW4 *gate_up, const XsMoeW4 *down, int32_t tokens, size_t *bytes);
int xs_moe_mlp_w4(const XsMoeW4 *gate_up, const XsMoeW4 *down, int32_t activation, const void *x_dev, int32_t tokens,
                  void *out_dev, void *workspace_dev, size_t workspace_bytes, void *stream);

typedef enum XsMoeGate {
    XS_MOE_GATE_NONE = 0,
    XS_MOE_GATE_CHANNEL = 1, /* (hidden)       */
    XS_MOE_GATE_ROW = 2,     /* (rows)         */
    XS_MOE_GATE_FULL = 3     /* (rows, hidden) */
} XsMoeGate;

/* The step between two blocks, one pass:
 *     r' = residual + residual_scale * gate . N(y; post_weight)          -> residual_out (rows, hidden) bf16
 *     n  = N(r'; next_weight)                                            -> next_out (rows, hidden) bf16
 *     N(v; w) = v / sqrt(mean(v^2) + eps) * (weight_offset + w)
 * post_weight_dev NULL: y enters as it is.  gate_dev NULL with XS_MOE_GATE_NONE.  next_weight_dev and next_out_dev both NULL:
 * only r'.  y_dev NULL (then post_weight, gate and residual_out are NULL too): r' = residual, only n is written -- a block's
 * first norm.  All tensors bf16; sums of squares and r' are held in f32, n is computed from r' before its rounding.
 * residual_out may be residual or y itself, next_out may be y or residual itself (same address); other overlaps are refused.
 * hidden is at most 57344, rows 2^30.  Takes the role of rmsnorm_launch and add_launch (xstar_cpp/include/ops/rmsnorm.h:46-52,
 * xstar_cpp/include/ops/add.h:38) in the tail of the reference's block (xstar_cpp/src/ops/transformer_block.cpp:353). */
typedef struct XsMoeNormResidual {
    const void *y_dev;
    const void *residual_dev;
    const void *post_weight_dev;
    const void *gate_dev;
    const void *next_weight_dev;
    void *residual_out_dev;
    void *next_out_dev;
    int32_t gate_kind; /* XsMoeGate */
    int32_t rows;
    int32_t hidden;
    float eps;
    float residual_scale;
    float weight_offset; /* 0, or 1 for weights stored as w - 1 */
    int32_t reserved[2]; /* must be zero */
} XsMoeNormResidual;
int xs_moe_norm_residual(const XsMoeNormResidual *args, void *stream);

/* The norms of one feed-forward half block: out = x + residual_scale * gate . N(F(N(x; pre_weight)); post_weight).
 * out may be x itself (same address). */
typedef struct XsMoeBlockNorms {
    const void *pre_weight_dev;  /* (hidden) bf16 */
    const void *post_weight_dev; /* (hidden) bf16 or NULL */
    const void *gate_dev;        /* bf16 or NULL */
    int32_t gate_kind;           /* XsMoeGate */
    float eps;
    float residual_scale;
    float weight_offset;
    int32_t reserved[2]; /* must be zero */
} XsMoeBlockNorms;

/* F = the 4-bit gated MLP.  Its input, the normed rows, is rounded once, to bf16 in small batches and to f16 in larger ones, and its result
 * once, to bf16. */
int xs_moe_mlp_w4_block_workspace_bytes(const XsMoeW4 *gate_up, const XsMoeW4 *down, int32_t tokens, size_t *bytes);
int xs_moe_mlp_w4_block(const XsMoeW4 *gate_up, const XsMoeW4 *down, int32_t activation, const XsMoeBlockNorms *norms,
                        const void *x_dev, int32_t tokens, void *out_dev, void *workspace_dev, size_t workspace_bytes,
                        void *stream);

/* F = the MoE layer: xs_moe_block_forward with a norm, a gate and a scale on the branch.  With weight_offset 0 the first norm is
 * xs_moe_rmsnorm's, so the expert choices are those of xs_moe_block_forward. */
int xs_moe_normed_block_workspace_bytes(const XsMoeConfig *cfg, size_t *bytes);
int xs_moe_normed_block_forward(const XsMoeConfig *cfg, const XsMoeWeights *w, const XsMoeBlockNorms *norms, const void *x_dev,
                                void *out_dev, void *workspace_dev, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif
