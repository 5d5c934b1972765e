/* helix_layer.h -- the operators around the scan in a recurrent layer:
 *
 *   helix_norm_*         root-mean-square norm with the residual's addition,
 *                        stored as it is or in 8 bits with scales, and its
 *                        backward pass
 *   helix_matmul_fp8_*   product of two 8-bit matrices with a scale for each
 *                        block of 128 along the sum
 *   helix_gated_scan_*   gated linear recurrence per channel, and its backward
 *                        pass
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

#ifdef __cplusplus
}
#endif

#endif /* HELIX_LAYER_H */
