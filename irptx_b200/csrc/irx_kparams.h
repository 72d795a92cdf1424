/* irx_kparams.h -- kernel parameter blocks, shared by the host launcher (C) and the sm_100a
 * kernels (CUDA). Each kernel takes one of these by value; the launcher fills it from a
 * plan and the caller's device pointers. Plain C layout, no pointers into host memory. */

#ifndef IRX_KPARAMS_H
#define IRX_KPARAMS_H

#include <stdint.h>
#include <cuda.h>            /* CUtensorMap: the TMA descriptor, 64-byte aligned */
#include "irx_int.h"

/* Threads per block of the full reduction (the launcher and the kernels agree on it). */
#define IRX_RED_ALL_THREADS 256

/* Device-side error word, written by a kernel whose bounded wait ran out. */
#define IRX_KERR_TIMEOUT   1u
#define IRX_KERR_TMEM      2u
#define IRX_KERR_INDEX     4u      /* a page, sequence, position or length outside the cache */

typedef struct {
    const void *ptr;        /* UNI_ARG: the const buffer */
    uint32_t    bits;       /* UNI_LIT: f32 bits */
    int32_t     off;        /* UNI_ARG: element offset */
    uint8_t     kind, dt;   /* uni_kind_t, dt_t */
    uint8_t     pad[2];
} irx_kuni_t;

typedef struct {
    const void *in[PROG_NSTREAM];
    void       *out[4];
    irx_kuni_t  uni[PROG_NUNI];
    irx_prog_t  prog[4];
    irx_prog_t  uprog;
    int64_t     begin, end;         /* element range of this launch (a shard) */
    uint8_t     in_dt[PROG_NSTREAM], out_dt[4];
    uint8_t     nin, nout, nuni, vec_ok;
} irx_kpw_t;

/* The per-graph pointwise kernel's parameters (jit.c writes the same layout into its source). */
typedef struct {
    const void *in[PROG_NSTREAM];
    void       *out[4];
    const void *uni[PROG_NUNI];     /* UNI_ARG: the const buffer; others unused */
    int64_t     begin, end;
    int32_t     vec_ok, pad;
} irx_kpwj_t;

typedef struct {
    const void *x;
    void       *y;
    float      *partial;            /* REDUCE_ALL: one float per block (scratch) */
    unsigned   *ticket;             /* REDUCE_ALL: arrival counter (scratch), left at 0 */
    irx_kuni_t  uni[PROG_NUNI];
    irx_prog_t  pre, uprog;
    int64_t     rows, cols;         /* this launch's rows (REDUCE_ALL: 1) */
    int64_t     row0;               /* first row (shards) */
    int64_t     begin, end;         /* REDUCE_ALL: element range of this launch */
    uint8_t     op, x_dt, y_dt, has_pre, out_reg, tot_reg, nuni, accumulate;
    uint8_t     vec_ok, pad[7];
} irx_kred_t;

typedef struct {
    const void *x, *w;
    void       *y;
    irx_kuni_t  uni[PROG_NUNI];
    irx_prog_t  stat_pre[ROW_MAX_STAT], epi, uprog;
    int64_t     rows, cols, row0;
    uint8_t     stat_op[ROW_MAX_STAT], stat_reg[ROW_MAX_STAT];
    uint8_t     x_dt, w_dt, y_dt, has_w, nstat, nuni, bulk_ok, kind;
    uint32_t    eps_bits;
    uint32_t    smem_row_bytes;     /* bytes of one staged row buffer */
    unsigned   *err;                /* device error word */
    uint8_t     ecache;             /* softmax: 1 keep exp(x - max) in the staged f32 row, 0 recompute */
    uint8_t     rk;                 /* written-out forms: 1/2/4 = cols / (256 * 8), the row held in
                                     * registers; 0 the loop form */
    uint8_t     pad2[6];
} irx_krow_t;

typedef struct {
    CUtensorMap tma_a, tma_b;       /* tcgen05 path: A [M,K] and B ([K,N] or [N,K]) tiles */
    CUtensorMap tma_c;              /* wide pair path: C [M, n1] (the launch's columns), stored by TMA */
    const void *a, *b;
    void       *c;
    int64_t     m, n, k;
    int64_t     n0, n1;             /* column range of this launch (N-column shards) */
    unsigned   *err;                /* device error word */
    uint8_t     b_kmajor;
    uint8_t     no_loads;           /* failure injection (tests): the producers issue no loads */
    uint8_t     stages;             /* CTA-pair kernel: depth of the shared-memory ring */
    uint8_t     group;              /* CTA-pair kernel: 256-row tile rows walked together (L2 reuse) */
    uint8_t     pad[4];
    uint64_t    wait_ns;            /* limit of each device wait, ns (0: IRX_WAIT_NS) */
} irx_kmm_t;

typedef struct {
    CUtensorMap tma_q, tma_k, tma_v;  /* tcgen05 path: [B*H*S, D] views */
    const void *q, *k, *v;
    void       *o;
    int64_t     b, h, s, d;
    int64_t     sq, sk, dqk, dv;    /* general shape (SIMT path) */
    int64_t     bh0, bh1;           /* batch*head range of this launch */
    float       scale;
    float       divisor;            /* scale_div: the score is dot / divisor, as the graph writes it */
    unsigned   *err;
    unsigned   *sched;              /* persistent form: the next unit to hand out (zeroed per launch) */
    uint8_t     causal, k_t, scale_div, pad[5];
} irx_kat_t;

/* Decode attention: blocks whose partials the workspace holds, and its layout: 2 slots a block, each
 * rows x dp accumulators then rows (max, sum) pairs, then the tickets (a work unit each) and the
 * group counters (a slot each). */
#define IRX_DEC_MAX_CTAS 512

/* Ring depth, 16-key blocks of a warp's tile and shared memory of the two decode kernels, by padded head
 * size and query rows of a work unit (the launcher and the kernels agree on them; the share is the
 * block's part of the work). */
#define IRX_DEC_SHARE 320
#define IRX_DEC_TC_KM(dp) ((dp) == 64 ? 2 : 1)
#define IRX_DEC_TC_ST(dp, nt) ((dp) == 256 || ((dp) == 128 && (nt) == 2) ? 2 : 3)
#define IRX_DEC_ST_NW(dp) ((dp) == 256 ? 8 : 16)
#define IRX_DEC_TC_SMEM(dp, nt, km, st) (4 * (st) * 2 * 16 * (km) * (dp) * 2 + 2 * 8 * ((dp) + 4) * 4 + 4 * 8 * (nt) * 8 + \
                                         IRX_DEC_SHARE + 4 * (st) * (192 * (km) + 8))
#define IRX_DEC_ST_SMEM(dp, rows, st) (IRX_DEC_ST_NW(dp) * ((st) * 8 * (2 * (dp) + 16) * 4 + (rows) * (dp) * 4 + 8 * (rows) * 4 + \
                                       8 * (rows) + (st) * 104) + (rows) * (dp) * 4 + IRX_DEC_SHARE)

typedef struct {
    const void *q, *k, *v;
    const int32_t *table, *lens;
    void       *o;
    float      *lse;                /* NULL: not asked for */
    float      *part;
    unsigned   *ticket, *gcount;
    unsigned   *err;
    int64_t     q_stride, page_stride, head_stride, token_stride, pages;
    int32_t     batch, cols, page_size, heads, group, d;
    int32_t     h0, h1;             /* kv heads of this launch (a shard) */
    int32_t     split;              /* work units per kv head */
    int32_t     window, sinks;
    float       scale2;             /* scale * log2(e) */
    uint8_t     dt, vec, pshift, pad;   /* vec: rows can be moved 16 bytes at a time */
    uint64_t    pmul;               /* page of a position: (position * pmul) >> pshift */
} irx_kdec_t;

/* Cache append: one warp per (token, part of the token's row). */
typedef struct {
    const void *kn, *vn;
    const int32_t *seq, *pos, *table;
    void       *k, *v;
    unsigned   *err;
    int64_t     stride, page_stride, head_stride, token_stride, pages;   /* in vectors */
    int64_t     t0, t1;             /* tokens of this launch */
    int32_t     batch, cols, page_size, heads, dv;      /* dv: vectors of a head's row */
    int32_t     parts;              /* warps per token */
} irx_kapp_t;

#define IRX_APPEND_VEC 2            /* vectors of keys, and of values, a lane of a warp moves */
#define IRX_COPY_TILE 512           /* vectors a block of the page copy moves at a time */

/* Page copy: runs of `run` vectors at (i1, i2) of every (pair, layer) of both pools. */
typedef struct {
    const int32_t *pairs;
    void       *k, *v;
    unsigned   *err;
    int64_t     page_stride, layer_stride, s1, s2, pages;                 /* in vectors */
    int64_t     p0, p1;             /* pairs of this launch */
    int64_t     run, tiles;         /* tiles: blocks' worth of work per (pair, layer, pool) */
    int32_t     n1, n2, layers, pad;
} irx_kcpy_t;

/* 4-bit matrix-vector products: ring depth and shared memory by 8-column blocks of tokens. */
#define IRX_MV4_STAGES 3
#define IRX_MV4_SMEM(nt) (IRX_MV4_STAGES * (128 * 128 + (nt) * 8 * (512 + 64)) + 2 * 128 * (9 * 4 + ((nt) == 1 ? 9 * 4 : 8)) + 1024 + 64)

typedef struct {
    CUtensorMap tma_w;              /* w's bytes of this launch's rows, in boxes of 128 x 128 */
    unsigned   *err;
    const void *x;
    const uint8_t *w, *z;           /* z: NULL when every zero point is 8 */
    const void *s;
    void       *y;
    int64_t     m, n, k, x_stride, w_stride;
    int64_t     n0, n1;             /* rows of w of this launch */
    int32_t     group, groups;
    int32_t     ck;                 /* blocks of a cluster, 1 to 8: slices of k */
    uint8_t     dt, sdt, gshift, pad;
    uint64_t    gmul;               /* group of k: (k / 32 * gmul) >> gshift */
} irx_kmv4_t;

#endif /* IRX_KPARAMS_H */
