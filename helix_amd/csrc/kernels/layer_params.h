/* layer_params.h -- kernel arguments of the layer operators (helix_layer.h),
 * shared by the C++ runtime and the gfx950 kernels and passed by value. Plain C.
 * Strides are in elements; the runtime has checked every shape and pointer. */
#ifndef HELIX_LAYER_PARAMS_H
#define HELIX_LAYER_PARAMS_H

#include <stdint.h>

/* Elements of a row that share a scale in 8-bit storage. */
#define HELIX_BLOCK 128

typedef struct {
    const void* x;
    const void* residual;   /* may be null                                     */
    const void* weight;     /* null: no norm (quantise)                        */
    void*       h;          /* may be null                                     */
    void*       y;          /* null: 8-bit output                              */
    uint8_t*    q;
    uint8_t*    scale;
    float*      rstd;       /* may be null                                     */
    long long   ld_x, ld_residual, ld_h, ld_y, ld_q, ld_scale;
    long long   rows;
    int         dim;
    int         w_f32;      /* weight is f32 (else the storage type)           */
    float       eps;
} HelixNormParams;

typedef struct {
    const void*  dy;
    const void*  h;
    const void*  weight;
    const float* rstd;
    const void*  dh;        /* may be null                                     */
    void*        dx;
    float*       dweight;   /* may be null                                     */
    float*       part;      /* [parts][dim] sums of dweight                    */
    long long    ld_dy, ld_h, ld_dh, ld_dx;
    long long    rows;
    long long    part_rows; /* rows of each part                               */
    int          dim;
    int          w_f32;
    int          parts;
} HelixNormBwdParams;

typedef struct {
    const uint8_t* a;
    const uint8_t* a_scale;
    const uint8_t* b;
    const uint8_t* b_scale;
    void*          c;
    long long      ld_a, ld_a_scale, ld_b, ld_b_scale, ld_c;
    int            m, n, k;
    int            f16;     /* c is f16 (else bf16), in the tiled kernel       */
    /* Tiled kernel: bands of gm rows of tiles, band = gm x columns of tiles, and
     * 2^32 / d + 1 of band, gm and the last band's rows. */
    int            gm;
    unsigned       band, inv_band, inv_gm, inv_rest;
    int            stride;  /* tiles from a workgroup's one to its next          */
    int            parts, part_blocks;   /* of the sum, and blocks of each but the last */
    float*         part;    /* [parts][m][n to a multiple of 4]                */
} HelixMatmulParams;

/* Gated recurrence: tokens of a thread's run, forward and backward, chunks of a
 * group, and most tokens that one thread walks by itself. */
#define HELIX_GS_RUN 8
#define HELIX_GS_RUN_BWD 4
#define HELIX_GS_GROUP 8
#define HELIX_GS_STEPS 16

/* Scratch that the chunks of a stream (64 channels of a sequence) are joined
 * through, filled with ones; unused with one chunk. */
typedef struct {
    unsigned*           ticket;   /* one less than the next ticket             */
    unsigned long long* part;     /* [stream][chunk][64] (A, B) of a chunk     */
    unsigned*           left;     /* [stream][group][64] state after a group   */
    int                 n_chunk, n_group;
} HelixGatedScanJoin;

typedef struct {
    const void*  g;
    const void*  v;
    const float* h0;        /* may be null                                     */
    void*        h;
    float*       last;      /* may be null                                     */
    long long    seq_g, tok_g, seq_v, tok_v, seq_h, tok_h;
    int          n_seq, n_tok, n_chan;
    int          n_slab;    /* ceil(n_chan / 64)                               */
    HelixGatedScanJoin join;
} HelixGatedScanParams;

typedef struct {
    const void*  dh;
    const void*  g;
    const void*  v;
    const void*  h;
    const float* h0;        /* may be null                                     */
    const float* dh_last;   /* may be null                                     */
    void*        dg;
    void*        dv;
    float*       dh0;       /* may be null                                     */
    long long    seq_dh, tok_dh, seq_g, tok_g, seq_v, tok_v, seq_h, tok_h, seq_dg, tok_dg, seq_dv, tok_dv;
    int          n_seq, n_tok, n_chan;
    int          n_slab;    /* ceil(n_chan / 64)                               */
    HelixGatedScanJoin join;
} HelixGatedScanBwdParams;

#endif
