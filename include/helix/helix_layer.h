/* helix_layer.h -- the operators around the scan in a recurrent layer:
 *
 *   helix_norm_*         root-mean-square norm with the residual's addition,
 *                        stored as it is or in 8 bits with scales, and its
 *                        backward pass
 *   helix_group_norm_*   norm of the groups of a token's channels (a head's, say)
 *                        with an activation or a gate, stored as it is or in 8
 *                        bits, and its backward pass
 *   helix_matmul_fp8_*   product of two 8-bit matrices with a scale for each
 *                        block of 128 along the sum
 *   helix_gated_scan_*   gated linear recurrence per channel, and its backward
 *                        pass
 *   helix_delta_rule_*   gated delta rule: a recurrence whose state is a matrix
 *                        per head, and its backward pass
 *
 * The reference has no counterpart of them. They keep helix.h's manner: they
 * enqueue kernels on the caller's stream and never allocate, synchronize or
 * wait; every check is made before the first launch, so an error leaves nothing
 * enqueued; helix_ctx_last_error() says what was wrong; scratch is the caller's
 * and needs no initial value. `stream` is a hipStream_t. A host-only context
 * makes the same checks and then returns HELIX_ERR_NO_DEVICE.
 *
 * Strides (`ld_*`, `tok_*`, `seq_*`) count elements and are not negative; the
 * last dimension of every matrix is contiguous. Outputs overlap neither inputs
 * nor each other, unless an operator says otherwise.
 *
 * 8-bit matrices. A row of n elements is n e4m3 bytes (OCP: no infinities, 448
 * the largest) and ceil(n / 128) scale bytes, one for each block of 128 elements
 * (the last may be shorter). A scale byte e stands for 2^(e - 127); 255 is a NaN.
 * Scaling by a power of two is exact, so a block loses no precision to its
 * scale, and the matrix instructions of gfx950 apply it by themselves.
 */
#ifndef HELIX_LAYER_H
#define HELIX_LAYER_H

#include "helix/helix.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Elements of a row that share a scale. */
#define HELIX_FP8_BLOCK 128

/* Largest row of helix_norm_*, and largest sum of helix_matmul_fp8_encode. */
#define HELIX_LAYER_MAX_DIM (1 << 20)

/* ------------------------------------------------------------------------- */
/* Norm                                                                      */
/* ------------------------------------------------------------------------- */

/* Per row:  h = x + residual,  rstd = 1 / sqrt(mean(h^2) + eps),
 *           out = h * rstd * weight
 * in fp32 throughout: the norm is that of the sum before it is rounded to the
 * storage type. With q, out is stored in 8 bits: a block's scale is the least
 * power of two (from 2^-126 up) at which its largest magnitude is at most 448.
 * A NaN of out is a NaN in y or q, an infinity a NaN in q; a block's NaNs do not
 * enter its scale.
 *
 * helix_quantize_fp8_encode is the same without the norm: out = x + residual. It
 * takes q, and no y, weight or rstd. */
typedef struct {
    int64_t     rows;         /* 0: nothing is done                           */
    int32_t     dim;          /* 1 .. HELIX_LAYER_MAX_DIM                     */
    int32_t     io_dtype;     /* helix_dtype of x, residual, h and y          */
    int32_t     weight_dtype; /* HELIX_F32 or io_dtype                        */
    float       eps;
    const void* x;
    const void* residual;     /* NULL: none, h = x                            */
    const void* weight;       /* dim                                          */
    void*       h;            /* x + residual, rounded once (may be x or
                                 residual, at their strides); NULL: not
                                 stored                                       */
    void*       y;            /* out; exactly one of y and q                  */
    void*       q;            /* out in e4m3                                  */
    void*       scale;        /* its scales                                   */
    float*      rstd;         /* rows; NULL: not stored                       */
    int64_t     ld_x, ld_residual, ld_h, ld_y, ld_q, ld_scale;
} helix_norm_args;

helix_status helix_norm_encode(helix_ctx* ctx, void* stream, const helix_norm_args* args);
helix_status helix_quantize_fp8_encode(helix_ctx* ctx, void* stream, const helix_norm_args* args);

/* Gradients of out (stored as y) and h, from dy and dh:
 *   n = h rstd,  t = dy weight,  dx = rstd (t - n mean(t n)) + dh
 *   dweight = sum over rows of dy n                       (fp32)
 * dx is the gradient of x and of residual alike. The rows of dweight's sum are
 * added in an order that depends on the shape alone. */
typedef struct {
    int64_t      rows;
    int32_t      dim;
    int32_t      io_dtype;     /* of dy, h, dh and dx                         */
    int32_t      weight_dtype;
    int32_t      reserved;     /* 0                                           */
    const void*  dy;
    const void*  h;            /* as helix_norm_encode stored it              */
    const void*  weight;
    const float* rstd;
    const void*  dh;           /* gradient of h; NULL: none                   */
    void*        dx;           /* may be dy or dh, at their strides           */
    float*       dweight;      /* dim; NULL: not wanted; 0 without rows       */
    void*        scratch;      /* helix_norm_backward_scratch_size() bytes,
                                  16-byte aligned; none is needed without
                                  dweight                                     */
    uint64_t     scratch_bytes;
    int64_t      ld_dy, ld_h, ld_dh, ld_dx;
} helix_norm_backward_args;

/* From rows, dim and dweight (NULL: 0); the other fields are not read. */
size_t       helix_norm_backward_scratch_size(const helix_norm_backward_args* args);
helix_status helix_norm_backward_encode(helix_ctx* ctx, void* stream, const helix_norm_backward_args* args);

/* ------------------------------------------------------------------------- */
/* Group norm                                                                */
/* ------------------------------------------------------------------------- */

/* The activation a: of the gate where there is one, else of the norm itself. */
typedef enum {
    HELIX_ACT_NONE    = 0,   /* a(u) = u                                      */
    HELIX_ACT_SILU    = 1,   /* u / (1 + exp(-u))                             */
    HELIX_ACT_SIGMOID = 2    /* 1 / (1 + exp(-u))                             */
} helix_activation;

/* Largest group of helix_group_norm_*, and largest row of it in 8 bits where
 * blocks of 128 do not line up with the groups. */
#define HELIX_GROUP_NORM_MAX_GROUP 8192
#define HELIX_GROUP_NORM_MAX_ROW   16384

/* A row's channels are `groups` groups of dim / groups neighbours. Per group:
 *   mean, rstd = 1 / sqrt(mean((x - mean)^2) + eps),  n = (x - mean) rstd
 *   z = n weight + bias
 *   out = z a(gate) with a gate, a(z) without
 * in fp32 throughout, rounded once; with q, out is stored in 8 bits as
 * helix_norm_encode stores it. Blocks line up with the groups where dim / groups
 * is a multiple of 128, or 32 or 64 and dim a multiple of 128. */
typedef struct {
    int64_t     rows;         /* 0: nothing is done                           */
    int32_t     dim;          /* 1 .. HELIX_LAYER_MAX_DIM                     */
    int32_t     groups;       /* divides dim; dim / groups is at most
                                 HELIX_GROUP_NORM_MAX_GROUP                   */
    int32_t     io_dtype;     /* helix_dtype of x, gate and y                 */
    int32_t     weight_dtype; /* HELIX_F32 or io_dtype: of weight and bias    */
    int32_t     activation;   /* helix_activation                             */
    float       eps;
    const void* x;
    const void* weight;       /* dim                                          */
    const void* bias;         /* dim; NULL: none                              */
    const void* gate;         /* NULL: none                                   */
    void*       y;            /* out (may be x or gate, at their strides);
                                 exactly one of y and q                       */
    void*       q;            /* out in e4m3                                  */
    void*       scale;        /* its scales                                   */
    float*      mean;         /* rows x groups, dense; NULL: not stored       */
    float*      rstd;         /* the same                                     */
    int64_t     ld_x, ld_gate, ld_y, ld_q, ld_scale;
} helix_group_norm_args;

helix_status helix_group_norm_encode(helix_ctx* ctx, void* stream, const helix_group_norm_args* args);

/* Gradients, from dy (of y). With dz = dy a(gate), or dy a'(z) without a gate:
 *   dgate = dy z a'(gate)
 *   t = dz weight,  dx = rstd (t - mean(t) - n mean(t n))    (means of a group)
 *   dweight = sum over rows of dz n,  dbias = sum over rows of dz  (fp32)
 * The rows of these sums are added in an order that depends on the shape alone. */
typedef struct {
    int64_t      rows;         /* 0: dweight and dbias are 0                  */
    int32_t      dim, groups;
    int32_t      io_dtype;     /* of dy, x, gate, dx and dgate                */
    int32_t      weight_dtype;
    int32_t      activation;
    int32_t      reserved;     /* 0                                           */
    const void*  dy;
    const void*  x;
    const void*  weight;
    const void*  bias;         /* NULL: none                                  */
    const void*  gate;         /* NULL: none                                  */
    const float* mean;         /* as helix_group_norm_encode stored them      */
    const float* rstd;
    void*        dx;           /* may be dy or x, at their strides            */
    void*        dgate;        /* NULL without a gate, else wanted            */
    float*       dweight;      /* dim; NULL: not wanted                       */
    float*       dbias;        /* dim; NULL: not wanted                       */
    void*        scratch;      /* helix_group_norm_backward_scratch_size()
                                  bytes, 16-byte aligned; none is needed
                                  without dweight and dbias                   */
    uint64_t     scratch_bytes;
    int64_t      ld_dy, ld_x, ld_gate, ld_dx, ld_dgate;
} helix_group_norm_backward_args;

/* From rows, dim, groups, dweight and dbias (NULL: not wanted). */
size_t       helix_group_norm_backward_scratch_size(const helix_group_norm_backward_args* args);
helix_status helix_group_norm_backward_encode(helix_ctx* ctx, void* stream, const helix_group_norm_backward_args* args);

/* ------------------------------------------------------------------------- */
/* Product of 8-bit matrices                                                 */
/* ------------------------------------------------------------------------- */

/* c[i][j] = sum over k of a[i][k] b[j][k], a and b with their scales.
 *
 * With out_dtype HELIX_F32 every product is exact and their sum is fp32's. With
 * HELIX_F16 and HELIX_BF16 the sum, in fp32 and rounded once, is of products that
 * the 8-bit matrix instruction has cut: each of eight that neighbour along k at
 * 2^-13 of the largest of the eight. That is up to 7 2^-13 of the sum of the
 * products' magnitudes; on normal operands with k = 2048 2e-5 of a result (rms),
 * where rounding to f16 leaves 2.1e-4 and to bf16 1.7e-3. It does not shrink where
 * products cancel. Whole numbers and others that the cut spares come out exact.
 *
 * a and b are 16-byte aligned and ld_a and ld_b multiples
 * of 16; k is any length, and what lies between k and ld does not matter. */
typedef struct {
    int32_t     m, n, k;       /* m or n 0: nothing is done; k at least 1     */
    int32_t     out_dtype;     /* helix_dtype of c                            */
    const void* a;             /* (m, k) e4m3                                 */
    const void* a_scale;       /* (m, ceil(k / 128))                          */
    const void* b;             /* (n, k) e4m3                                 */
    const void* b_scale;       /* (n, ceil(k / 128))                          */
    void*       c;             /* (m, n)                                      */
    void*       scratch;       /* helix_matmul_fp8_scratch_size() bytes (for
                                  parts of the sum where c is small, and for
                                  scales whose rows do not start at multiples
                                  of four bytes), 16-byte aligned             */
    uint64_t    scratch_bytes;
    int64_t     ld_a, ld_a_scale, ld_b, ld_b_scale, ld_c;
} helix_matmul_fp8_args;

/* From the arguments without their scratch; addresses count by their alignment. */
size_t       helix_matmul_fp8_scratch_size(const helix_matmul_fp8_args* args);
helix_status helix_matmul_fp8_encode(helix_ctx* ctx, void* stream, const helix_matmul_fp8_args* args);

/* ------------------------------------------------------------------------- */
/* Gated linear recurrence                                                   */
/* ------------------------------------------------------------------------- */

/* Per sequence and channel, with f_t = sigmoid(g_t) and the state in fp32:
 *   h_t = f_t h_(t-1) + (1 - f_t) v_t,   h_(-1) = h0
 * g = +inf keeps the state and takes no v (a finite v), g = -inf takes v alone.
 * An infinite v or h0 leaves its channel infinite or NaN from its token on (NaN
 * where the product of the gates since has reached zero in fp32).
 * n_tok = 1 is the step of a single token. h0, last, dh_last and dh0 are dense
 * fp32 (n_seq, n_chan); last may be h0. */
typedef struct {
    int32_t      n_seq, n_tok, n_chan;  /* n_seq or n_chan 0: nothing is
                                  done; n_tok 0: last = h0                    */
    int32_t      io_dtype;     /* of g, v and h                               */
    const void*  g;
    const void*  v;
    const float* h0;           /* NULL: zero                                  */
    void*        h;            /* may be g or v, at their strides             */
    float*       last;         /* h of the last token; NULL: not stored       */
    void*        scratch;      /* helix_gated_scan_scratch_size() bytes,
                                  16-byte aligned                             */
    uint64_t     scratch_bytes;
    int64_t      seq_g, tok_g, seq_v, tok_v, seq_h, tok_h;
} helix_gated_scan_args;

/* From n_seq, n_tok and n_chan; the other fields are not read. */
size_t       helix_gated_scan_scratch_size(const helix_gated_scan_args* args);
helix_status helix_gated_scan_encode(helix_ctx* ctx, void* stream, const helix_gated_scan_args* args);

/* Gradients, from dh (of every h) and dh_last (of last):
 *   lambda_t = dh_t + f_(t+1) lambda_(t+1),  dh_last added to the last one's
 *   dv_t = lambda_t (1 - f_t)
 *   dg_t = lambda_t (h_(t-1) - v_t) f_t (1 - f_t)
 *   dh0  = f_0 lambda_0 */
typedef struct {
    int32_t      n_seq, n_tok, n_chan;  /* n_seq or n_chan 0: nothing is
                                  done; n_tok 0: dh0 = dh_last                */
    int32_t      io_dtype;     /* of dh, g, v, h, dg and dv                   */
    const void*  dh;
    const void*  g;
    const void*  v;
    const void*  h;            /* as helix_gated_scan_encode stored it        */
    const float* h0;           /* NULL: zero                                  */
    const float* dh_last;      /* NULL: zero                                  */
    void*        dg;
    void*        dv;
    float*       dh0;          /* NULL: not stored                            */
    void*        scratch;      /* helix_gated_scan_backward_scratch_size()    */
    uint64_t     scratch_bytes;
    int64_t      seq_dh, tok_dh, seq_g, tok_g, seq_v, tok_v, seq_h, tok_h, seq_dg, tok_dg, seq_dv, tok_dv;
} helix_gated_scan_backward_args;

size_t       helix_gated_scan_backward_scratch_size(const helix_gated_scan_backward_args* args);
helix_status helix_gated_scan_backward_encode(helix_ctx* ctx, void* stream,
                                              const helix_gated_scan_backward_args* args);

/* ------------------------------------------------------------------------- */
/* Gated delta rule                                                          */
/* ------------------------------------------------------------------------- */

/* Largest n_key and n_val. */
#define HELIX_DELTA_MAX_KEY 128
#define HELIX_DELTA_MAX_VAL (1 << 16)

/* Per sequence and value head, with the state S (n_key x n_val) in fp32:
 *   S_t = e^(g_t) S_(t-1) + beta_t k_t (v_t - e^(g_t) S_(t-1)' k_t)'
 *   o_t = scale S_t' q_t,   S_(-1) = s0
 * Value head h has the queries and keys of head h / (n_head / n_qk_head). g is the
 * logarithm of the decay: 0 keeps the state, -inf forgets it; a token with g = 0
 * and beta = 0 leaves the state as it is. Keys are taken as they are: of length
 * one at most, with beta up to 2, they keep the state bounded.
 *
 * Products keep fp32 accuracy (operands in three bf16 parts, fp32 sums; of a
 * chunk's operands below 2^-110, 2^-134), whatever the storage type; o is rounded
 * to it once. Inputs may be any finite numbers, the type's largest too; what is
 * formed of them (S, S' k, S' q, what a token brings, the products of a chunk's keys
 * and queries) has to stay below bf16's largest, 3.3895e38.
 * What is not finite (g = -inf apart) stays where the formulas take it: an element
 * of v or s0 in its column of o and s, one of q in its token's o, one of k, g or
 * beta in its heads' o and s; but in a call of chunks the o of tokens before it in
 * its chunk of 64 may be NaN too. Other heads and sequences are not touched. A
 * masked token's q, k and v have to be finite, as 0 times a NaN is one.
 *
 * n_tok = 1 is the step of a single token; s may be s0. Strides are any that are
 * not negative (o's elements do not overlap); 64 tokens of q, k, v or o span
 * less than 2^31 bytes. g and beta are fp32 with dense heads; s0 and s are dense
 * (n_seq, n_head, n_key, n_val). */
typedef struct {
    int32_t      n_seq, n_tok;       /* n_seq or n_head 0: nothing is done;
                                        n_tok 0: s = s0; n_seq * n_head is
                                        below 2^31                            */
    int32_t      n_qk_head, n_head;  /* the first divides the second          */
    int32_t      n_key, n_val;
    int32_t      io_dtype;           /* of q, k, v and o                      */
    float        scale;
    const void*  q;                  /* (n_seq, n_tok, n_qk_head, n_key)      */
    const void*  k;                  /* the same                              */
    const void*  v;                  /* (n_seq, n_tok, n_head, n_val)         */
    const float* g;                  /* (n_seq, n_tok, n_head)                */
    const float* beta;               /* the same                              */
    const float* s0;                 /* NULL: zero                            */
    void*        o;                  /* as v                                  */
    float*       s;                  /* the state after the last token        */
    void*        scratch;            /* helix_delta_rule_scratch_size() bytes,
                                        16-byte aligned                       */
    uint64_t     scratch_bytes;
    int64_t      seq_q, tok_q, head_q, seq_k, tok_k, head_k, seq_v, tok_v, head_v;
    int64_t      seq_g, tok_g, seq_beta, tok_beta, seq_o, tok_o, head_o;
} helix_delta_rule_args;

/* From the sizes and io_dtype; the other fields are not read. */
size_t       helix_delta_rule_scratch_size(const helix_delta_rule_args* args);
helix_status helix_delta_rule_encode(helix_ctx* ctx, void* stream, const helix_delta_rule_args* args);

/* Gradients, from d_o (of every o) and d_s (of s). The states are formed again.
 * dq and dk of a head that value heads share are the sums over them, in fp32 and in
 * the heads' order; the heads that share one have n_head / n_qk_head * ceil(n_val /
 * 16) below 2^32 / 640. What is not finite (g = -inf apart) may reach every gradient
 * of its sequence's heads that the formulas give it a part in, at tokens before and
 * after it; one of v and s0 has none in dv and ds0, one of d_o and d_s only its
 * column of them. Other heads and sequences are not touched. */
typedef struct {
    int32_t      n_seq, n_tok;       /* n_seq or n_head 0: nothing is done;
                                        n_tok 0: ds0 = d_s                    */
    int32_t      n_qk_head, n_head;
    int32_t      n_key, n_val;
    int32_t      io_dtype;           /* of d_o, q, k, v, dq, dk and dv        */
    float        scale;
    const void*  d_o;                /* (n_seq, n_tok, n_head, n_val)         */
    const void*  q;
    const void*  k;
    const void*  v;
    const float* g;
    const float* beta;
    const float* s0;                 /* NULL: zero                            */
    const float* d_s;                /* dense (n_seq, n_head, n_key, n_val);
                                        NULL: zero                            */
    void*        dq;                 /* the outputs are dense                 */
    void*        dk;
    void*        dv;
    float*       dg;
    float*       dbeta;
    float*       ds0;                /* may be d_s                            */
    void*        scratch;            /* helix_delta_rule_backward_scratch_size()
                                        bytes, 16-byte aligned                */
    uint64_t     scratch_bytes;
    int64_t      seq_do, tok_do, head_do, seq_q, tok_q, head_q, seq_k, tok_k, head_k, seq_v, tok_v, head_v;
    int64_t      seq_g, tok_g, seq_beta, tok_beta;
} helix_delta_rule_backward_args;

/* From the sizes; the other fields are not read. */
size_t       helix_delta_rule_backward_scratch_size(const helix_delta_rule_backward_args* args);
helix_status helix_delta_rule_backward_encode(helix_ctx* ctx, void* stream, const helix_delta_rule_backward_args* args);

#ifdef __cplusplus
}
#endif

#endif /* HELIX_LAYER_H */
