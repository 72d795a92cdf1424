/* step.c -- the host side of the operators around the cache in a model's step: rotary positions (alone and
 * on the way into a paged cache), attention over packed prompts, and the draw of the next token.
 * Descriptors into plans, and their launches, as serve.c has them for the cache's own operators.
 * Kernels: kernels/rope.cu, prompt.cu and sample.cu. */

#include <math.h>
#include "serve.h"

#define TWO_PI 6.283185307179586476925286766559

/* ---- rotary positions ---- */

int irx_rope_freqs(int rot, double base, int scaling, double factor, double original, double fast, double slow, double *freqs)
{
    int i;
    double low, high;
    irx_clear_error();
    if (!freqs) return irx_fail(E093, "frequencies with nowhere to put them");
    if (rot < 2 || rot % 2 || rot > MAX_DIM) return irx_fail(E042, "a rotated width that is odd or outside 2 to 256");
    if (!(base > 1.0) || !isfinite(base)) return irx_fail(E042, "a rotation base that is not a number above 1");
    if (scaling < IRX_ROPE_PLAIN || scaling > IRX_ROPE_BANDS) return irx_fail(E042, "a scaling of no known kind");
    if (scaling != IRX_ROPE_PLAIN && (!(factor >= 1.0) || !isfinite(factor))) return irx_fail(E042, "a context factor that is not a number of at least 1");
    if (scaling >= IRX_ROPE_YARN && (!(original > 0.0) || !isfinite(original) || !(fast > slow) || !(slow > 0.0) || !isfinite(fast)))
        return irx_fail(E042, "an original context or turns that are not above 0, or fast turns that are not above the slow");
    if (scaling == IRX_ROPE_NTK && rot > 2) base *= pow(factor, rot / (rot - 2.0));
    for (i = 0; i < rot / 2; i++) freqs[i] = pow(base, -2.0 * i / rot);
    if (scaling == IRX_ROPE_LINEAR)
        for (i = 0; i < rot / 2; i++) freqs[i] /= factor;
    if (scaling == IRX_ROPE_YARN) {
        /* the pairs that turn `fast` times and once `slow` times within the original context */
        low = floor(rot * log(original / (fast * TWO_PI)) / (2.0 * log(base)));
        high = ceil(rot * log(original / (slow * TWO_PI)) / (2.0 * log(base)));
        if (low < 0.0) low = 0.0;
        if (high > rot - 1) high = rot - 1;
        for (i = 0; i < rot / 2; i++) {
            double r = (i - low) / (high - low > 0.001 ? high - low : 0.001);
            r = r < 0.0 ? 0.0 : r > 1.0 ? 1.0 : r;
            freqs[i] = freqs[i] / factor * r + freqs[i] * (1.0 - r);
        }
    }
    if (scaling == IRX_ROPE_BANDS)
        for (i = 0; i < rot / 2; i++) {
            double r = (original * freqs[i] / TWO_PI - slow) / (fast - slow);     /* turns within the original context */
            r = r < 0.0 ? 0.0 : r > 1.0 ? 1.0 : r;
            freqs[i] = freqs[i] / factor * (1.0 - r) + freqs[i] * r;
        }
    return 0;
}

static int rope_of(irx_ropep_t *a, const irx_rope_t *r, int dim)
{
    int i;
    if (!r || !r->freqs) return irx_fail(E093, "a rotation without frequencies");
    if (dim < 1 || dim > MAX_DIM) return irx_fail(E042, "a head size outside 1 to 256");
    if (r->pairs < 1 || 2 * (int64_t)r->pairs > dim) return irx_fail(E042, "no rotated pairs, or more than the head holds");
    if (!isfinite(r->amplitude)) return irx_fail(E042, "an amplitude that is not finite");
    a->pairs = r->pairs;
    a->inter = r->interleaved != 0;
    a->amp = r->amplitude;
    for (i = 0; i < r->pairs; i++) {
        /* 2^31 positions of a frequency up to 2^10 turn fewer than 2^42 times: 2^-11 of a turn is still exact */
        if (!isfinite(r->freqs[i]) || fabs(r->freqs[i]) > 1024.0) return irx_fail(E042, "a frequency that is not a number within 1024 radians a position");
        a->freq[i] = (r->backward ? -1.0 : 1.0) * r->freqs[i] / TWO_PI;
    }
    return 0;
}

int irx_compile_rope(const irx_rope_t *r, int dtype, long long tokens, int heads, int head_dim, long long x_stride,
                     long long y_stride, irx_plan_t *plan)
{
    irx_plan_int_t *p = begin(plan, FAM_ROPE, "rope");
    irx_ropep_t *a;
    int64_t row;
    if (!p) return 1;
    a = &p->u.ro;
    if (!float_dt(dtype)) return irx_fail(E024, "a rotation whose dtype is not f32 or bf16");
    if (rope_of(a, r, head_dim)) return 1;
    if (tokens < 1 || tokens > MAX_COUNT || heads < 1) return irx_fail(E042, "a rotation of no tokens or heads");
    row = (int64_t)heads * head_dim;
    if (row > (1 << 20)) return irx_fail(E042, "a token's heads past 2^20 elements");
    if (x_stride < 0 || x_stride > MAX_STRIDE || (x_stride && x_stride < row) || y_stride < 0 || y_stride > MAX_STRIDE ||
        (y_stride && y_stride < row)) return irx_fail(E042, "tokens' rows that overlap");
    a->c.dt = (uint8_t)dtype;
    a->c.dim = head_dim;
    a->n = tokens;
    a->heads = heads;
    a->x_stride = x_stride ? x_stride : row;
    a->y_stride = y_stride ? y_stride : row;
    if ((double)tokens * a->x_stride > MAX_SPAN || (double)tokens * a->y_stride > MAX_SPAN)
        return irx_fail(E042, "a rotation larger than an address space");
    add(p, KA_IN, dtype, (tokens - 1) * a->x_stride + row);
    add(p, KA_IN, DT_I32, tokens);
    add(p, KA_OUT, dtype, (tokens - 1) * a->y_stride + row);
    return finish(p);
}

int irx_compile_rope_append(const irx_kv_cache_t *cache, const irx_rope_t *r, long long tokens, int heads, long long stride,
                            long long out_stride, irx_plan_t *plan)
{
    irx_plan_int_t *p = begin(plan, FAM_ROPE_APPEND, "rope_append");
    irx_ropep_t *a;
    int64_t qrow, krow;
    if (!p) return 1;
    a = &p->u.ro;
    if (irx_cache_of(&a->c, cache, 1) || rope_of(a, r, a->c.dim)) return 1;
    if (r->backward) return irx_fail(E042, "an append of the transposed rotation");
    if (tokens < 1 || tokens > MAX_COUNT) return irx_fail(E042, "an append of no tokens");
    if (heads < 1) return irx_fail(E042, "an append with no query heads");
    qrow = (int64_t)heads * a->c.dim;
    krow = (int64_t)a->c.heads * a->c.dim;
    if (qrow + 2 * krow > (1 << 20)) return irx_fail(E042, "a token's heads past 2^20 elements");
    if (stride < 0 || stride > MAX_STRIDE || (stride && (stride < qrow || stride < krow)) || out_stride < 0 ||
        out_stride > MAX_STRIDE || (out_stride && out_stride < qrow)) return irx_fail(E042, "tokens' rows that overlap");
    a->n = tokens;
    a->heads = heads;
    a->x_stride = stride;                                  /* 0: each of q, k and v packed */
    a->y_stride = out_stride ? out_stride : qrow;
    if ((double)tokens * (stride ? stride : qrow > krow ? qrow : krow) > MAX_SPAN || (double)tokens * a->y_stride > MAX_SPAN)
        return irx_fail(E042, "new tokens larger than an address space");
    add(p, KA_IN, a->c.dt, (tokens - 1) * (stride ? stride : qrow) + qrow);
    add(p, KA_IN, a->c.dt, (tokens - 1) * (stride ? stride : krow) + krow);
    add(p, KA_IN, a->c.dt, (tokens - 1) * (stride ? stride : krow) + krow);
    add(p, KA_IN, DT_I32, tokens);
    add(p, KA_IN, DT_I32, tokens);
    add(p, KA_IN, DT_I32, (int64_t)a->c.batch * a->c.cols);
    add(p, KA_OUT, a->c.dt, (tokens - 1) * a->y_stride + qrow);
    add(p, KA_OUT, a->c.dt, irx_cache_span(&a->c));
    add(p, KA_OUT, a->c.dt, irx_cache_span(&a->c));
    p->arg_zero[7] = p->arg_zero[8] = 1;
    return finish(p);
}

static int launch_rope(const irx_plan_int_t *p, irx_dev_t *d, unsigned s, unsigned ns, void *const *args, void *st)
{
    const irx_ropep_t *a = &p->u.ro;
    const irx_kvc_t *c = &a->c;
    const int es = esz(c->dt), vmax = 16 / es, app = p->fam == FAM_ROPE_APPEND;
    static irx_krope_t k;
    size_t mix;
    long long u0, u1;
    int64_t n, warps;
    int i, v;
    memset(&k, 0, sizeof k);
    irx_unit_range(a->n, s, ns, &u0, &u1);
    if (u0 >= u1) return 0;
    k.q = args[0];
    k.heads = a->heads; k.d = c->dim; k.pairs = a->pairs;
    k.kv_stride = k.x_stride = a->x_stride; k.y_stride = a->y_stride;
    k.t0 = u0; k.t1 = u1;
    k.amp = a->amp;
    k.inter = a->inter;
    k.err = (unsigned *)(size_t)d->err;
    for (i = 0; i < a->pairs; i++) k.freq[i] = a->freq[i];
    if (app) {
        k.kn = args[1]; k.vn = args[2];
        k.seq = (const int32_t *)args[3]; k.pos = (const int32_t *)args[4]; k.table = (const int32_t *)args[5];
        k.qo = args[6]; k.k = args[7]; k.v = args[8];
        k.kv = c->heads;
        if (!a->x_stride) {
            k.x_stride = (int64_t)a->heads * c->dim;
            k.kv_stride = (int64_t)c->heads * c->dim;
        }
        k.page_stride = c->page_stride; k.head_stride = c->head_stride; k.token_stride = c->token_stride;
        k.pages = c->pages; k.batch = c->batch; k.cols = c->cols; k.page_size = c->page_size;
    } else {
        k.pos = (const int32_t *)args[1];
        k.qo = args[2];
    }
    /* 16 bytes at a time when every row, and both halves of its rotated part, begin on 16 bytes */
    mix = (size_t)k.q | (size_t)k.kn | (size_t)k.vn | (size_t)k.qo | (size_t)k.k | (size_t)k.v |
          ((size_t)k.x_stride | (size_t)k.kv_stride | (size_t)k.y_stride | (size_t)k.page_stride | (size_t)k.head_stride |
           (size_t)k.token_stride | (size_t)k.d | (size_t)a->pairs) * (size_t)es;
    v = mix % 16 == 0 ? vmax : 1;
    k.items = k.pairs / v + (k.d - 2 * k.pairs + 2 * v - 1) / (2 * v);      /* two vectors each */
    /* A warp for each token shares the token's angles; with few tokens more warps each (down to one item a
     * lane), until the GPU has sixteen for every SM. */
    n = (int64_t)(k.heads + 2 * k.kv) * k.items;
    k.parts = (int32_t)((16ll * d->sms + (u1 - u0) - 1) / (u1 - u0));
    if (k.parts > (n + 31) / 32) k.parts = (int32_t)((n + 31) / 32);
    k.chunk = (int32_t)((n + k.parts - 1) / k.parts + 31) / 32 * 32;
    k.parts = (int32_t)((n + k.chunk - 1) / k.chunk);
    warps = (u1 - u0) * k.parts;
    if ((warps + 3) / 4 > MAX_COUNT) return irx_fail(E042, "a rotation past one launch's blocks");
    return irx_dev_launch(d, K_ROPE + (c->dt == DT_BF16 ? 0 : 3) + (v == 1 ? 2 : 32 % k.items ? 1 : 0), (unsigned)((warps + 3) / 4), 128, 0, 1, st, &k);
}

/* ---- attention over packed prompts ---- */

int irx_compile_prompt(const irx_prompt_t *m, irx_plan_t *plan)
{
    irx_plan_int_t *p = begin(plan, FAM_PROMPT, "prompt");
    irx_prm_t *a;
    int64_t qrow, krow;
    if (!p) return 1;
    a = &p->u.pr;
    if (!m) return irx_fail(E093, "a prompt of no descriptor");
    if (!float_dt(m->dtype)) return irx_fail(E024, "a prompt whose dtype is not f32 or bf16");
    if (m->tokens < 1 || m->tokens > (1 << 30)) return irx_fail(E042, "prompts' tokens outside 1 to 2^30");
    if (m->batch < 1 || m->batch > (1 << 16)) return irx_fail(E042, "sequences outside 1 to 2^16");
    if (m->head_dim < 1 || m->head_dim > MAX_DIM) return irx_fail(E042, "a head size outside 1 to 256");
    if (m->kv_heads < 1 || m->heads < 1 || m->heads % m->kv_heads) return irx_fail(E042, "query heads that are not a multiple of the key-value heads");
    if (m->window < 0 || m->sinks < 0) return irx_fail(E042, "a window or sink count below 0");
    if (m->sinks && !m->window) return irx_fail(E042, "sinks without a window");
    if (!isfinite(m->scale)) return irx_fail(E042, "a scale that is not finite");
    if (fabsf(m->scale) > MAX_SCALE) return irx_fail(E042, "a scale past 2.35e38, which f32 does not hold times log2(e)");
    qrow = (int64_t)m->heads * m->head_dim;
    krow = (int64_t)m->kv_heads * m->head_dim;
    if (m->q_stride < 0 || m->q_stride > MAX_STRIDE || (m->q_stride && m->q_stride < qrow) || m->kv_stride < 0 ||
        m->kv_stride > MAX_STRIDE || (m->kv_stride && m->kv_stride < krow)) return irx_fail(E042, "tokens' rows that overlap");
    a->dt = (uint8_t)m->dtype;
    a->tokens = m->tokens;
    a->batch = m->batch; a->heads = m->heads; a->kv_heads = m->kv_heads; a->dim = m->head_dim;
    a->q_stride = m->q_stride ? m->q_stride : qrow;
    a->kv_stride = m->kv_stride ? m->kv_stride : krow;
    a->window = m->window; a->sinks = m->sinks;
    a->lse = m->lse != 0;
    memcpy(&a->scale_bits, &m->scale, 4);
    if ((double)a->tokens * a->q_stride > MAX_SPAN || (double)a->tokens * a->kv_stride > MAX_SPAN)
        return irx_fail(E042, "a prompt larger than an address space");
    /* the units of the kernel with the smaller tiles, 64 rows each and a broken one for each sequence */
    if ((double)a->heads * a->tokens / 64 + 2.0 * a->kv_heads * a->batch > 2e9) return irx_fail(E042, "more than 2^31 - 1 tiles of work");
    add(p, KA_IN, a->dt, (a->tokens - 1) * a->q_stride + qrow);
    add(p, KA_IN, a->dt, (a->tokens - 1) * a->kv_stride + krow);
    add(p, KA_IN, a->dt, (a->tokens - 1) * a->kv_stride + krow);
    add(p, KA_IN, DT_I32, (int64_t)a->batch + 1);
    add(p, KA_OUT, a->dt, a->tokens * qrow);
    if (a->lse) add(p, KA_OUT, DT_F32, a->tokens * a->heads);
    return finish(p);
}

static int launch_prompt(const irx_plan_int_t *p, irx_dev_t *d, unsigned s, unsigned ns, void *const *args, void *st)
{
    const irx_prm_t *a = &p->u.pr;
    const int es = esz(a->dt), al = 16 / es;
    static irx_kprm_t k;
    long long u0, u1;
    int64_t grid, want;
    float scale;
    int dp, kk;
    memset(&k, 0, sizeof k);
    irx_unit_range(a->kv_heads, s, ns, &u0, &u1);
    if (u0 >= u1) return 0;
    memcpy(&scale, &a->scale_bits, 4);
    k.q = args[0]; k.k = args[1]; k.v = args[2];
    k.starts = (const int32_t *)args[3];
    k.o = args[4];
    k.lse = a->lse ? (float *)args[5] : NULL;
    k.err = (unsigned *)(size_t)d->err;
    k.tokens = a->tokens; k.q_stride = a->q_stride; k.kv_stride = a->kv_stride;
    k.batch = a->batch; k.heads = a->heads; k.kv_heads = a->kv_heads; k.group = a->heads / a->kv_heads; k.d = a->dim;
    k.h0 = (int32_t)u0; k.h1 = (int32_t)u1;
    k.window = a->window; k.sinks = a->sinks;
    k.scale2 = (float)((double)scale * 1.4426950408889634);
    k.dt = a->dt;
    k.vec = (uint8_t)(a->dim % al == 0 && a->q_stride % al == 0 && a->kv_stride % al == 0 && a_to(k.q, 16) && a_to(k.k, 16) &&
                      a_to(k.v, 16) && a_to(k.o, 16));
    dp = a->dim <= 64 ? 64 : a->dim <= 128 ? 128 : 256;
    if (a->dt == DT_BF16 && k.vec && k.group <= 128 && (int64_t)a->heads * a->dim < (1 << 24) && a->q_stride < MAX_STRIDE / 2 && a->kv_stride < MAX_STRIDE / 2) {
        const int tp = 128 / k.group, nt = dp == 256 ? 1 : 2;  /* tokens of a tile, tiles of a unit */
        const cuuint64_t es2 = 2, qd[4] = {(cuuint64_t)a->dim, (cuuint64_t)k.group, (cuuint64_t)a->kv_heads, (cuuint64_t)a->tokens};
        const cuuint64_t qs[3] = {qd[0] * es2, qd[0] * qd[1] * es2, (cuuint64_t)a->q_stride * es2};
        const cuuint64_t kd[3] = {qd[0], qd[2], qd[3]}, ks[2] = {qd[0] * es2, (cuuint64_t)a->kv_stride * es2};
        const cuuint32_t qb[4] = {64, (cuuint32_t)k.group, 1, (cuuint32_t)tp}, kb[3] = {64, 1, dp == 256 ? 64 : 128};
        if (irx_dev_tmap(&k.tma_q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, (void *)(size_t)k.q, qd, qs, qb, CU_TENSOR_MAP_SWIZZLE_128B) ||
            irx_dev_tmap(&k.tma_k, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, (void *)(size_t)k.k, kd, ks, kb, CU_TENSOR_MAP_SWIZZLE_128B) ||
            irx_dev_tmap(&k.tma_v, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, (void *)(size_t)k.v, kd, ks, kb, CU_TENSOR_MAP_SWIZZLE_128B))
            return 1;
        want = ((a->tokens + nt * tp - 1) / (nt * tp) + a->batch) * (u1 - u0);
        return irx_dev_launch(d, K_PR_TC + (dp == 64 ? 0 : dp == 128 ? 1 : 2), (unsigned)(want < d->sms ? want : d->sms), 128 * nt + 128,
                              (unsigned)(dp == 256 ? IRX_PR_WIDE_SMEM : IRX_PR_TC_SMEM(dp)), 1, st, &k);
    }
    kk = K_PR_ST + (dp == 64 ? 0 : dp == 128 ? 1 : 2);
    want = ((a->tokens * k.group + 63) / 64 + a->batch) * (u1 - u0);
    if (irx_serve_grid(d, kk, IRX_PR_ST_THREADS(dp), IRX_PR_ST_SMEM(dp), want, &grid)) return 1;
    return irx_dev_launch(d, kk, (unsigned)grid, IRX_PR_ST_THREADS(dp), IRX_PR_ST_SMEM(dp), 1, st, &k);
}

/* ---- the draw of a token ---- */

int irx_compile_sample(const irx_sample_t *m, irx_plan_t *plan)
{
    irx_plan_int_t *p = begin(plan, FAM_SAMPLE, "sample");
    irx_smp_t *a;
    if (!p) return 1;
    a = &p->u.sm;
    if (!m) return irx_fail(E093, "a draw of no descriptor");
    if (!float_dt(m->dtype)) return irx_fail(E024, "logits whose dtype is not f32 or bf16");
    if (m->rows < 1 || m->rows > MAX_COUNT / 8) return irx_fail(E042, "rows outside 1 to 2^28 - 1");
    if (m->vocab < 1 || m->vocab > (1 << 30)) return irx_fail(E042, "a vocabulary outside 1 to 2^30");
    if (m->stride < 0 || m->stride > MAX_STRIDE || (m->stride && m->stride < m->vocab)) return irx_fail(E042, "rows of logits that overlap");
    a->dt = (uint8_t)m->dtype;
    a->rows = m->rows;
    a->vocab = m->vocab;
    a->stride = m->stride ? m->stride : m->vocab;
    a->logprob = m->logprob != 0;
    if ((double)a->rows * a->stride > MAX_SPAN) return irx_fail(E042, "logits larger than an address space");
    add(p, KA_IN, a->dt, (a->rows - 1) * a->stride + a->vocab);
    add(p, KA_IN, DT_F32, a->rows);
    add(p, KA_IN, DT_I32, a->rows);
    add(p, KA_IN, DT_F32, a->rows);
    add(p, KA_IN, DT_F32, a->rows);
    add(p, KA_IN, DT_F32, a->rows);
    add(p, KA_OUT, DT_I32, a->rows);
    if (a->logprob) add(p, KA_OUT, DT_F32, a->rows);
    return finish(p);
}

static int launch_sample(const irx_plan_int_t *p, irx_dev_t *d, unsigned s, unsigned ns, void *const *args, void *st)
{
    const irx_smp_t *a = &p->u.sm;
    const int epw = a->dt == DT_BF16 ? 2 : 1;              /* elements of a word */
    static irx_ksmp_t k;
    long long u0, u1;
    int64_t nc, words, room = (d->smem_optin - IRX_SMP_FIXED - 16) / 4;
    int far, j;
    memset(&k, 0, sizeof k);
    irx_unit_range(a->rows, s, ns, &u0, &u1);
    if (u0 >= u1) return 0;
    k.x = args[0];
    k.temperature = (const float *)args[1]; k.top_k = (const int32_t *)args[2]; k.top_p = (const float *)args[3];
    k.min_p = (const float *)args[4]; k.u = (const float *)args[5];
    k.token = (int32_t *)args[6];
    k.logprob = a->logprob ? (float *)args[7] : NULL;
    k.err = (unsigned *)(size_t)d->err;
    k.r0 = u0; k.stride = a->stride; k.n = a->vocab;
    while ((1ll << k.kbits) < a->vocab) k.kbits++;
    k.kbits = 62 - k.kbits;                                 /* a row's weights sum to at most 2^62 */
    if (k.kbits > 46) k.kbits = 46;
    k.big = 6755399441055744.0;
    k.two52 = 4503599627370496.0;
    for (j = 0; j < 4; j++) k.series[j] = (j ? k.series[j - 1] : 1.0) * (0.69314718055994530942 / 128.0) / (j + 1);
    for (j = 0; j < 128; j++) k.tab[j] = ldexp(exp2(j / 128.0), k.kbits);
    /* Blocks of a cluster: as few as hold the row in their shared memory, since every block pays for the row's settings
     * and exchanges. With few rows more, down to 4096 elements each, as long as all rows' blocks run at once. Measured
     * with 2, 4 and 8 blocks: 64 rows of 128001 bf16 logits, top-k and top-p, 28, 38, 55 us; f32 (2 do not hold it) 52 with 4, 61
     * with 8; 256 rows of 151999, top-p, bf16 216, 202, 267 (the filters are on the device: the rule does not see them), f32 293
     * with 4, 318 with 8; one row of 128001 f32 17.7 with 4, 15.4 with 8. */
    for (nc = 1;; nc *= 2) {
        words = (a->vocab + epw - 1 + nc * epw * IRX_SMP_THREADS - 1) / (nc * epw * IRX_SMP_THREADS) | 1;
        if (nc == 8) break;
        if (words * IRX_SMP_THREADS > room) continue;
        if (words * epw * IRX_SMP_THREADS <= 4096 || (u1 - u0) * nc * 2 > d->sms) break;
    }
    k.words = (int32_t)words;
    far = words * IRX_SMP_THREADS > room;
    return irx_dev_launch(d, K_SMP + (a->dt == DT_BF16 ? 0 : 2) + far, (unsigned)((u1 - u0) * nc), IRX_SMP_THREADS,
                          (unsigned)(IRX_SMP_FIXED + (far ? 0 : words * IRX_SMP_THREADS * 4 + 16)), (unsigned)nc, st, &k);
}

/* ---- one entry for the launch switch, and the plans' descriptions ---- */

int irx_launch_step(const irx_plan_int_t *p, irx_dev_t *d, unsigned s, unsigned ns, void *const *args, void *st)
{
    int i;
    for (i = 0; i < p->narg; i++)
        if (!a_to(args[i], (size_t)esz(p->arg_dt[i]))) return irx_fail(E093, "a device pointer that its elements' size does not divide");
    switch (p->fam) {
    case FAM_PROMPT: return launch_prompt(p, d, s, ns, args, st);
    case FAM_SAMPLE: return launch_sample(p, d, s, ns, args, st);
    default: return launch_rope(p, d, s, ns, args, st);
    }
}

void irx_step_text(const irx_plan_int_t *p, char *buf, size_t cap)
{
    if (p->fam == FAM_PROMPT) {
        const irx_prm_t *a = &p->u.pr;
        float sc;
        memcpy(&sc, &a->scale_bits, 4);
        snprintf(buf, cap, "prompt tokens=%lld batch=%d heads=%d kv_heads=%d d=%d window=%d sinks=%d lse=%d scale=%g dtype=%s",
                 (long long)a->tokens, a->batch, a->heads, a->kv_heads, a->dim, a->window, a->sinks, a->lse, (double)sc, dname(a->dt));
    } else if (p->fam == FAM_SAMPLE) {
        const irx_smp_t *a = &p->u.sm;
        snprintf(buf, cap, "sample rows=%lld vocab=%lld logprob=%d dtype=%s", (long long)a->rows, (long long)a->vocab, a->logprob, dname(a->dt));
    } else {
        const irx_ropep_t *a = &p->u.ro;
        if (p->fam == FAM_ROPE)
            snprintf(buf, cap, "rope tokens=%lld heads=%d d=%d rot=%d pairs=%s dtype=%s", (long long)a->n, a->heads, a->c.dim,
                     2 * a->pairs, a->inter ? "interleaved" : "halves", dname(a->c.dt));
        else
            snprintf(buf, cap, "rope_append tokens=%lld heads=%d kv_heads=%d d=%d rot=%d pairs=%s page=%d pages=%lld dtype=%s",
                     (long long)a->n, a->heads, a->c.heads, a->c.dim, 2 * a->pairs, a->inter ? "interleaved" : "halves",
                     a->c.page_size, (long long)a->c.pages, dname(a->c.dt));
    }
}

/* The work that a launch cannot do without; a prompt's, of one sequence that fills it (the starts are only
 * known on the device). */
void irx_step_work(const irx_plan_int_t *p, double *bytes, double *flops)
{
    *bytes = *flops = 0;
    if (p->fam == FAM_PROMPT) {
        const irx_prm_t *a = &p->u.pr;
        const double n = (double)a->tokens, w = a->window && a->window < n ? a->window : n;
        double seen = w * (w + 1) / 2 + (n - w) * w;
        if (a->window && n > w) {
            const double sk = a->sinks < n - w ? a->sinks : n - w;
            seen += sk * (sk + 1) / 2 + (n - w - sk) * sk;
        }
        *bytes = 2 * n * (a->heads + a->kv_heads) * a->dim * esz(a->dt);
        *flops = 4 * seen * a->heads * a->dim;
    } else if (p->fam == FAM_SAMPLE) {
        const irx_smp_t *a = &p->u.sm;
        *bytes = (double)a->rows * ((double)a->vocab * esz(a->dt) + 24 + 4 * a->logprob);
        *flops = (double)a->rows * a->vocab;
    } else {
        const irx_ropep_t *a = &p->u.ro;
        const double rows = p->fam == FAM_ROPE ? a->heads : a->heads + 2 * a->c.heads;
        *bytes = 2.0 * a->n * rows * a->c.dim * esz(a->c.dt) + (p->fam == FAM_ROPE ? 4.0 : 8.0) * a->n;
        *flops = 6.0 * a->n * (p->fam == FAM_ROPE ? a->heads : a->heads + a->c.heads) * a->pairs;
    }
}
