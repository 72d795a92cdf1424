/* serve.c -- the serving operators' host side: descriptors into plans, and their launches.
 *
 * Decode attention, the paged cache's append and page copy, and 4-bit matrix-vector products are
 * not KIR graphs (a page table's indirection is not in the KIR), so each has a descriptor of its
 * own; the plan it compiles to is an ordinary one. Kernels: kernels/decode.cu, kvpages.cu and
 * matvec4.cu. */

#include "serve.h"

#define MAX_32 (1ll << 30)

/* Elements from the first to past the last of a pool. */
int64_t irx_cache_span(const irx_kvc_t *c)
{
    return (c->pages - 1) * c->page_stride + (int64_t)(c->heads - 1) * c->head_stride +
           (int64_t)(c->page_size - 1) * c->token_stride + c->dim;
}

/* The three axes over rows, by stride; each must start past the end of what lies inside it. */
static int rows_overlap(const irx_kvc_t *c)
{
    int64_t st[3] = {c->page_stride, c->head_stride, c->token_stride}, n[3] = {c->pages, c->heads, c->page_size};
    int64_t inner = c->dim;
    int i, j;
    for (i = 0; i < 3; i++)
        for (j = i + 1; j < 3; j++)
            if (st[j] < st[i]) {
                int64_t t = st[i]; st[i] = st[j]; st[j] = t;
                t = n[i]; n[i] = n[j]; n[j] = t;
            }
    for (i = 0; i < 3; i++) {
        if (n[i] == 1) continue;
        if (st[i] < inner) return 1;
        inner += (n[i] - 1) * st[i];
    }
    return 0;
}

int irx_cache_of(irx_kvc_t *o, const irx_kv_cache_t *c, int tabled)
{
    if (!c) return irx_fail(E093, "an operator over no cache descriptor");
    if (!float_dt(c->dtype)) return irx_fail(E024, "a cache whose dtype is not f32 or bf16");
    if (c->heads < 1 || c->page_size < 1 || c->pages < 1 || c->pages > MAX_COUNT)
        return irx_fail(E042, "a cache without heads, pages or page slots");
    if (c->head_dim < 1 || c->head_dim > MAX_DIM) return irx_fail(E042, "a cache head size outside 1 to 256");
    if (tabled && (c->batch < 1 || c->table_cols < 1)) return irx_fail(E042, "a cache without a page table");
    if (tabled && (int64_t)c->table_cols * c->page_size > MAX_COUNT)
        return irx_fail(E042, "a page table of more than 2^31 - 1 tokens a sequence");
    memset(o, 0, sizeof *o);
    o->dt = (uint8_t)c->dtype;
    o->heads = c->heads; o->dim = c->head_dim; o->page_size = c->page_size; o->pages = c->pages;
    o->batch = tabled ? c->batch : 1; o->cols = tabled ? c->table_cols : 1;
    o->page_stride = c->page_stride; o->head_stride = c->head_stride; o->token_stride = c->token_stride;
    if (!c->page_stride && !c->head_stride && !c->token_stride) {
        o->token_stride = c->head_dim;
        o->head_stride = (int64_t)c->page_size * c->head_dim;
        o->page_stride = o->head_stride * c->heads;
    }
    if (o->page_stride < 0 || o->head_stride < 0 || o->token_stride < 0 || o->page_stride > MAX_STRIDE ||
        o->head_stride > MAX_STRIDE || o->token_stride > MAX_STRIDE)
        return irx_fail(E042, "a cache stride below 0 or above 2^40");
    if ((double)o->pages * o->page_stride > MAX_SPAN || (double)o->heads * o->head_stride > MAX_SPAN ||
        (double)o->page_size * o->token_stride > MAX_SPAN)
        return irx_fail(E042, "a cache larger than an address space");
    if (rows_overlap(o)) return irx_fail(E041, "a cache whose strides make rows overlap");
    return 0;
}

/* ---- decode ---- */

/* The workspace serves either kernel: an unaligned bf16 launch takes the second. */
static int64_t dec_units(const irx_dec_t *a)
{
    return (int64_t)a->c.batch * a->c.heads * (a->split[0] > a->split[1] ? a->split[0] : a->split[1]);
}

static int64_t dec_part_bytes(const irx_dec_t *a)
{
    return 2ll * a->max_ctas * (a->rows[0] > a->rows[1] ? a->rows[0] : a->rows[1]) * (a->dp + 2) * 4;
}

int irx_compile_decode(const irx_kv_cache_t *cache, int heads, long long q_stride, float scale, int window, int sinks, int lse,
                       irx_plan_t *plan)
{
    irx_plan_int_t *p = begin(plan, FAM_DECODE, "decode");
    irx_dec_t *a;
    int64_t per, chunks, qrow;
    int g, i;
    if (!p) return 1;
    a = &p->u.dec;
    if (irx_cache_of(&a->c, cache, 1)) return 1;
    if (heads < 1 || heads % a->c.heads) return irx_fail(E042, "query heads that are not a multiple of the cache's heads");
    if (window < 0 || sinks < 0) return irx_fail(E042, "a window or sink count below 0");
    if (sinks && !window) return irx_fail(E042, "sinks without a window");
    if (!(scale == scale) || scale - scale != 0.0f) return irx_fail(E042, "a scale that is not finite");
    if (scale > MAX_SCALE || scale < -MAX_SCALE) return irx_fail(E042, "a scale past 2.35e38, which f32 does not hold times log2(e)");
    qrow = (int64_t)heads * a->c.dim;
    if (q_stride < 0 || q_stride > MAX_STRIDE || (q_stride && q_stride < qrow))
        return irx_fail(E042, "query rows that overlap");
    if ((double)a->c.batch * (q_stride ? q_stride : qrow) > MAX_SPAN) return irx_fail(E042, "queries larger than an address space");
    a->heads = heads;
    a->q_stride = q_stride ? q_stride : qrow;
    a->window = window;
    a->sinks = sinks;
    a->lse = lse != 0;
    memcpy(&a->scale_bits, &scale, 4);
    g = heads / a->c.heads;
    a->dp = a->c.dim <= 64 ? 64 : a->c.dim <= 128 ? 128 : 256;
    a->rows[0] = g > 8 && a->dp <= 128 ? 16 : 8;
    a->rows[1] = g > 4 ? 8 : 4;
    for (i = 0; i < 2; i++) a->split[i] = (g + a->rows[i] - 1) / a->rows[i];
    /* no more blocks than chunks of a full cache: what the workspace has to hold */
    per = ((int64_t)a->c.cols * a->c.page_size + 63) / 64;
    chunks = dec_units(a) > IRX_DEC_MAX_CTAS ? IRX_DEC_MAX_CTAS : dec_units(a) * per;
    a->max_ctas = chunks < IRX_DEC_MAX_CTAS ? (int32_t)chunks : IRX_DEC_MAX_CTAS;
    if (dec_units(a) > MAX_COUNT) return irx_fail(E042, "more than 2^31 - 1 rows of work");
    add(p, KA_IN, a->c.dt, (int64_t)(a->c.batch - 1) * a->q_stride + qrow);
    add(p, KA_IN, a->c.dt, irx_cache_span(&a->c));
    add(p, KA_IN, a->c.dt, irx_cache_span(&a->c));
    add(p, KA_IN, DT_I32, (int64_t)a->c.batch * a->c.cols);
    add(p, KA_IN, DT_I32, a->c.batch);
    add(p, KA_OUT, a->c.dt, (int64_t)a->c.batch * qrow);
    if (a->lse) add(p, KA_OUT, DT_F32, (int64_t)a->c.batch * heads);
    add(p, KA_WORK, DT_U8, dec_part_bytes(a) + 4 * (dec_units(a) + 2ll * a->max_ctas));
    return finish(p);
}

int irx_serve_grid(irx_dev_t *d, int k, int block, size_t smem, int64_t want, int64_t *g)
{
    if (!d->occ[k] && irx_dev_occupancy(d, k, block, smem, &d->occ[k])) return 1;
    *g = (int64_t)d->sms * d->occ[k];
    if (want < *g) *g = want;
    if (*g < 1) *g = 1;
    return 0;
}

static int launch_decode(const irx_plan_int_t *p, irx_dev_t *d, unsigned s, unsigned ns, void *const *args, void *st)
{
    const irx_dec_t *a = &p->u.dec;
    static irx_kdec_t k;
    const int es = esz(a->c.dt), al = 16 / es, last = p->narg - 1;
    long long u0, u1;
    int64_t grid;
    int rows, kk, st_, block = 128;
    size_t smem;
    float scale;
    memset(&k, 0, sizeof k);
    irx_unit_range(a->c.heads, s, ns, &u0, &u1);
    if (u0 >= u1) return 0;
    memcpy(&scale, &a->scale_bits, 4);
    k.q = args[0]; k.k = args[1]; k.v = args[2];
    k.table = (const int32_t *)args[3]; k.lens = (const int32_t *)args[4];
    k.o = args[5];
    k.lse = a->lse ? (float *)args[6] : NULL;
    if (!a_to(args[last], 16)) return irx_fail(E093, "a decode workspace that is not 16-byte aligned");
    k.part = (float *)args[last];
    k.ticket = (unsigned *)((char *)args[last] + dec_part_bytes(a));
    k.gcount = k.ticket + dec_units(a);
    k.err = (unsigned *)(size_t)d->err;
    k.q_stride = a->q_stride;
    k.page_stride = a->c.page_stride; k.head_stride = a->c.head_stride; k.token_stride = a->c.token_stride;
    k.pages = a->c.pages;
    k.batch = a->c.batch; k.cols = a->c.cols; k.page_size = a->c.page_size;
    k.heads = a->heads; k.group = a->heads / a->c.heads; k.d = a->c.dim;
    k.h0 = (int32_t)u0; k.h1 = (int32_t)u1;
    k.window = a->window; k.sinks = a->sinks;
    k.scale2 = (float)((double)scale * 1.4426950408889634);
    k.dt = a->c.dt;
    k.vec = (uint8_t)(a->c.dim % al == 0 && a->c.page_stride % al == 0 && a->c.head_stride % al == 0 &&
                      a->c.token_stride % al == 0 && a_to(k.k, 16) && a_to(k.v, 16) && a_to(k.q, 4) &&
                      a->q_stride * es % 4 == 0 && a_to(k.o, 16));
    {   /* division by the page size of numbers below 2^31: ceil(2^(31 + l) / d), l = ceil(log2 d) */
        const uint64_t ps = (uint64_t)a->c.page_size;
        int l = 0;
        while ((1ull << l) < ps) l++;
        k.pshift = (uint8_t)(31 + l);
        k.pmul = ((1ull << l << 31) + ps - 1) / ps;
    }
    st_ = !k.vec || a->c.dt != DT_BF16;
    rows = a->rows[st_];
    k.split = a->split[st_];
    if (!st_) {
        const int nt = rows / 8;
        kk = K_DEC_TC + (a->dp == 64 ? nt - 1 : a->dp == 128 ? 1 + nt : 4);
        smem = (size_t)IRX_DEC_TC_SMEM(a->dp, nt, IRX_DEC_TC_KM(a->dp), IRX_DEC_TC_ST(a->dp, nt));
    } else {
        kk = K_DEC_ST + (a->dp == 64 ? 0 : a->dp == 128 ? 2 : 4) + (rows == 8);
        smem = (size_t)IRX_DEC_ST_SMEM(a->dp, rows, 1);
        block = 32 * IRX_DEC_ST_NW(a->dp);
    }
    if (irx_serve_grid(d, kk, block, smem, a->max_ctas, &grid)) return 1;
    return irx_dev_launch(d, kk, (unsigned)grid, (unsigned)block, (unsigned)smem, 1, st, &k);
}

/* ---- the cache's moves ---- */

int irx_compile_kv_append(const irx_kv_cache_t *cache, long long tokens, long long stride, irx_plan_t *plan)
{
    irx_plan_int_t *p = begin(plan, FAM_KV_APPEND, "kv_append");
    irx_kv_t *a;
    int64_t row;
    if (!p) return 1;
    a = &p->u.kv;
    if (irx_cache_of(&a->c, cache, 1)) return 1;
    row = (int64_t)a->c.heads * a->c.dim;
    if (tokens < 1 || tokens > MAX_COUNT) return irx_fail(E042, "an append of no tokens");
    if (row > (1 << 20)) return irx_fail(E042, "a token's keys past 2^20 elements");
    if (stride < 0 || stride > MAX_STRIDE || (stride && stride < row)) return irx_fail(E042, "new tokens' rows that overlap");
    if ((double)tokens * (stride ? stride : row) > MAX_SPAN) return irx_fail(E042, "new tokens larger than an address space");
    a->n = tokens;
    a->stride = stride ? stride : row;
    add(p, KA_IN, a->c.dt, (tokens - 1) * a->stride + row);
    add(p, KA_IN, a->c.dt, (tokens - 1) * a->stride + row);
    add(p, KA_IN, DT_I32, tokens);
    add(p, KA_IN, DT_I32, tokens);
    add(p, KA_IN, DT_I32, (int64_t)a->c.batch * a->c.cols);
    add(p, KA_OUT, a->c.dt, irx_cache_span(&a->c));
    add(p, KA_OUT, a->c.dt, irx_cache_span(&a->c));
    p->arg_zero[5] = p->arg_zero[6] = 1;
    return finish(p);
}

int irx_compile_kv_copy(const irx_kv_cache_t *cache, long long pairs, int layers, long long layer_stride, irx_plan_t *plan)
{
    irx_plan_int_t *p = begin(plan, FAM_KV_COPY, "kv_copy");
    irx_kv_t *a;
    if (!p) return 1;
    a = &p->u.kv;
    if (irx_cache_of(&a->c, cache, 0)) return 1;
    if (pairs < 1 || pairs > MAX_COUNT) return irx_fail(E042, "a copy of no pages");
    if (layers < 1) return irx_fail(E042, "a copy in no layers");
    if (layer_stride < 0 || layer_stride > MAX_STRIDE || (layers > 1 && layer_stride && layer_stride < irx_cache_span(&a->c)))
        return irx_fail(E041, "layers whose pools overlap");
    a->n = pairs;
    a->layers = layers;
    a->layer_stride = layer_stride ? layer_stride : a->c.pages * a->c.page_stride;
    if (layers > 1 && a->layer_stride < irx_cache_span(&a->c)) return irx_fail(E041, "layers whose pools overlap");
    if ((double)layers * a->layer_stride > MAX_SPAN) return irx_fail(E042, "a cache larger than an address space");
    if ((double)pairs * layers * a->c.heads * a->c.page_size * a->c.dim > MAX_SPAN)
        return irx_fail(E042, "a copy of more elements than 64 bits count");
    add(p, KA_IN, DT_I32, 2 * pairs);
    add(p, KA_OUT, a->c.dt, (layers - 1) * a->layer_stride + irx_cache_span(&a->c));
    add(p, KA_OUT, a->c.dt, (layers - 1) * a->layer_stride + irx_cache_span(&a->c));
    p->arg_zero[1] = p->arg_zero[2] = 1;
    return finish(p);
}

/* The widest vector, 16, 4 or 2 bytes, that divides every one of the byte counts in `or_all` (their
 * bitwise or, pointers included); 0, 1 or 2: the kernel of that width. */
static int width(size_t or_all, int *bytes)
{
    *bytes = or_all % 16 == 0 ? 16 : or_all % 4 == 0 ? 4 : 2;
    return *bytes == 16 ? 0 : *bytes == 4 ? 1 : 2;
}

static int launch_append(const irx_plan_int_t *p, irx_dev_t *d, unsigned s, unsigned ns, void *const *args, void *st)
{
    const irx_kv_t *a = &p->u.kv;
    const irx_kvc_t *c = &a->c;
    const size_t es = (size_t)esz(c->dt);
    static irx_kapp_t k;
    long long u0, u1;
    int vb, w;
    int64_t warps;
    memset(&k, 0, sizeof k);
    irx_unit_range(a->n, s, ns, &u0, &u1);
    if (u0 >= u1) return 0;
    w = width((size_t)args[0] | (size_t)args[1] | (size_t)args[5] | (size_t)args[6] |
              ((size_t)a->stride | (size_t)c->page_stride | (size_t)c->head_stride | (size_t)c->token_stride | (size_t)c->dim) * es, &vb);
    vb /= (int)es;
    k.kn = args[0]; k.vn = args[1];
    k.seq = (const int32_t *)args[2]; k.pos = (const int32_t *)args[3]; k.table = (const int32_t *)args[4];
    k.k = args[5]; k.v = args[6];
    k.err = (unsigned *)(size_t)d->err;
    k.stride = a->stride / vb; k.page_stride = c->page_stride / vb; k.head_stride = c->head_stride / vb;
    k.token_stride = c->token_stride / vb;
    k.pages = c->pages;
    k.t0 = u0; k.t1 = u1;
    k.batch = c->batch; k.cols = c->cols; k.page_size = c->page_size; k.heads = c->heads;
    k.dv = c->dim / vb;
    k.parts = (c->heads * k.dv + 32 * IRX_APPEND_VEC - 1) / (32 * IRX_APPEND_VEC);
    warps = (u1 - u0) * k.parts;
    if ((warps + 3) / 4 > MAX_COUNT) return irx_fail(E042, "an append past one launch's blocks");
    return irx_dev_launch(d, K_KV_APPEND + w, (unsigned)((warps + 3) / 4), 128, 0, 1, st, &k);
}

static int launch_copy(const irx_plan_int_t *p, irx_dev_t *d, unsigned s, unsigned ns, void *const *args, void *st)
{
    const irx_kv_t *a = &p->u.kv;
    const irx_kvc_t *c = &a->c;
    const size_t es = (size_t)esz(c->dt);
    static irx_kcpy_t k;
    long long u0, u1;
    int vb, w, tok_inner;
    int64_t run, s1, s2, n1, n2, grid, want;
    memset(&k, 0, sizeof k);
    irx_unit_range(a->n, s, ns, &u0, &u1);
    if (u0 >= u1) return 0;
    /* a page as n2 x n1 runs of contiguous elements: the axes by stride, dense ones folded into the run */
    tok_inner = c->token_stride <= c->head_stride;
    run = c->dim;
    n1 = tok_inner ? c->page_size : c->heads;
    s1 = tok_inner ? c->token_stride : c->head_stride;
    n2 = tok_inner ? c->heads : c->page_size;
    s2 = tok_inner ? c->head_stride : c->token_stride;
    if (n1 == 1 || s1 == run) { run *= n1; n1 = 1; s1 = 0; }
    if (n1 == 1 && (n2 == 1 || s2 == run)) { run *= n2; n2 = 1; s2 = 0; }
    w = width((size_t)args[1] | (size_t)args[2] |
              ((size_t)run | (size_t)s1 | (size_t)s2 | (size_t)c->page_stride | (size_t)a->layer_stride) * es, &vb);
    vb /= (int)es;
    k.pairs = (const int32_t *)args[0];
    k.k = args[1]; k.v = args[2];
    k.err = (unsigned *)(size_t)d->err;
    k.page_stride = c->page_stride / vb; k.layer_stride = a->layer_stride / vb;
    k.s1 = s1 / vb; k.s2 = s2 / vb;
    k.pages = c->pages;
    k.p0 = u0; k.p1 = u1;
    k.run = run / vb;
    k.n1 = (int32_t)n1; k.n2 = (int32_t)n2; k.layers = a->layers;
    k.tiles = (k.run * n1 * n2 + IRX_COPY_TILE - 1) / IRX_COPY_TILE;
    want = (u1 - u0) * k.tiles * a->layers * 2;
    if (irx_serve_grid(d, K_KV_COPY + w, 256, 0, want, &grid)) return 1;
    return irx_dev_launch(d, K_KV_COPY + w, (unsigned)grid, 256, 0, 1, st, &k);
}

/* ---- 4-bit matrix-vector products ---- */

int irx_compile_matvec4(const irx_matvec4_t *m, irx_plan_t *plan)
{
    irx_plan_int_t *p = begin(plan, FAM_MATVEC4, "matvec4");
    irx_mv4_t *a;
    int64_t groups;
    if (!p) return 1;
    a = &p->u.mv;
    if (!m) return irx_fail(E093, "a matvec4 of no descriptor");
    if (!float_dt(m->dtype) || !float_dt(m->scale_dtype)) return irx_fail(E024, "a matvec4 whose dtypes are not f32 or bf16");
    if (m->m < 1 || m->n < 1 || m->k < 1 || m->m > MAX_COUNT || m->n > MAX_COUNT || m->k > MAX_COUNT)
        return irx_fail(E042, "a matvec4 size outside 1 to 2^31 - 1");
    if (m->group < 1) return irx_fail(E042, "a group of no weights");
    if (m->x_stride < 0 || m->x_stride > MAX_STRIDE || (m->x_stride && m->x_stride < m->k) || m->w_stride < 0 ||
        m->w_stride > MAX_STRIDE || (m->w_stride && m->w_stride < (m->k + 1) / 2))
        return irx_fail(E042, "rows of x or w that overlap");
    groups = (m->k + m->group - 1) / m->group;
    a->m = m->m; a->n = m->n; a->k = m->k;
    a->x_stride = m->x_stride ? m->x_stride : m->k;
    a->w_stride = m->w_stride ? m->w_stride : (m->k + 1) / 2;
    a->group = m->group;
    a->groups = (int32_t)groups;
    a->dt = (uint8_t)m->dtype; a->sdt = (uint8_t)m->scale_dtype;
    a->zeros = m->zeros != 0;
    if ((double)a->m * a->n > MAX_SPAN || (double)a->n * a->w_stride > MAX_SPAN || (double)a->m * a->x_stride > MAX_SPAN)
        return irx_fail(E042, "a matvec4 larger than an address space");
    add(p, KA_IN, a->dt, (a->m - 1) * a->x_stride + a->k);
    add(p, KA_IN, DT_U8, (a->n - 1) * a->w_stride + (a->k + 1) / 2);
    add(p, KA_IN, a->sdt, a->n * groups);
    if (a->zeros) add(p, KA_IN, DT_U8, a->n * groups);
    add(p, KA_OUT, a->dt, a->m * a->n);
    return finish(p);
}

/* How many slices of k, and how much shared memory. Up to two blocks an SM a block's speed is bound by its own
 * latencies, so the most slices (a cluster's blocks, 1 to 8) whose clusters all fit at once. The GPU
 * packs clusters as tightly as shared memory lets it, which leaves SMs idle when the grid does not
 * fill it, so a launch asks for as much as keeps its blocks at the fewest an SM that hold them all.
 * Measured (bf16, one token, 14336 k): 71 tiles in 4 slices at two an SM 22.0 us, in 3 26.8, in 2 34.0; 74
 * tiles, of which 71 clusters of 4 fit, in 4 31.9, in 3 (the rule's) 26.8, in 2 24.9; 14337 rows of 4096, 4
 * tokens, in 2 12.7, in 1 13.7 at one an SM, in 4 16.0. A third block an SM does not fit its shared memory. */
static int mv4_split(irx_dev_t *d, int i, unsigned need, int64_t tiles, int64_t steps, unsigned *ck, unsigned *smem)
{
    unsigned r, c, best = 0;
    *ck = 1;
    *smem = need;
    for (r = 1; r <= 2; r++) {
        /* what an SM can share out (228 KB, 1 KB of it taken by each block) over r blocks */
        unsigned room = (unsigned)(228 / r - 1) * 1024;
        if (room > (unsigned)d->smem_optin) room = (unsigned)d->smem_optin;
        if (room < need) break;
        for (c = 1; c <= 8 && c <= steps; c++) {
            short *fit = &d->mv4_fit[i][r - 1][c];
            if (!*fit) {
                int n = 1;
                if (irx_dev_max_clusters(d, K_MV4 + i, 4096 * c, 256, room, c, &n)) return 1;
                *fit = (short)(n < 32767 ? n : 32767);
            }
            if (tiles <= *fit && c > best) {
                best = c;
                *ck = c;
                *smem = room;
            }
        }
    }
    return 0;
}

static int launch_mv4(const irx_plan_int_t *p, irx_dev_t *d, unsigned s, unsigned ns, void *const *args, void *st)
{
    const irx_mv4_t *a = &p->u.mv;
    static irx_kmv4_t k;
    long long u0, u1;
    int64_t grid;
    memset(&k, 0, sizeof k);
    irx_unit_range(a->n, s, ns, &u0, &u1);
    if (u0 >= u1) return 0;
    k.x = args[0]; k.w = (const uint8_t *)args[1]; k.s = args[2];
    k.z = a->zeros ? (const uint8_t *)args[3] : NULL;
    k.y = args[a->zeros ? 4 : 3];
    k.m = a->m; k.n = a->n; k.k = a->k; k.x_stride = a->x_stride; k.w_stride = a->w_stride;
    k.n0 = u0; k.n1 = u1;
    k.group = a->group; k.groups = a->groups;
    k.dt = a->dt; k.sdt = a->sdt;
    k.err = (unsigned *)(size_t)d->err;
    /* the kernels below count rows, tokens and k in 32 bits, some of them past the end */
    if (a->m <= MAX_32 && a->n <= MAX_32 && a->k <= MAX_32 && a->n * a->groups <= MAX_COUNT && a->k % 32 == 0 &&
        a->group % 32 == 0 && a->w_stride % 16 == 0 && a_to(k.w, 16) && (a->dt == DT_F32 ||
        (a->x_stride % 8 == 0 && a_to(k.x, 16)))) {
        /* columns: one a token, three for f32 tokens; 8 or 16 of them at a time */
        const int f32 = a->dt == DT_F32, gv = a->group % 128 == 0 ? 2 : a->group % 64 == 0 ? 1 : 0;
        const int nt = a->m > (f32 ? 2 : 8) ? 2 : 1, tok = f32 ? (nt == 1 ? 2 : 5) : 8 * nt;
        const int64_t tiles = ((u1 - u0 + 127) / 128) * ((a->m + tok - 1) / tok), steps = (a->k + 255) / 256;
        unsigned ck, smem;
        if (mv4_split(d, 6 * f32 + gv * 2 + nt - 1, (unsigned)IRX_MV4_SMEM(nt), tiles, steps, &ck, &smem)) return 1;
        if (tiles * ck > MAX_COUNT) return irx_fail(E042, "a matvec4 past one launch's blocks");
        const cuuint64_t dims[2] = {(cuuint64_t)a->k / 2, (cuuint64_t)u1}, strides[1] = {(cuuint64_t)a->w_stride};
        const cuuint32_t box[2] = {128, 128};
        if (irx_dev_tmap(&k.tma_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void *)(size_t)k.w, dims, strides, box,
                         CU_TENSOR_MAP_SWIZZLE_128B)) return 1;
        k.ck = (int32_t)ck;
        {   /* division by d = group / 32 of numbers below 2^26: ceil(2^(26 + l) / d), l = ceil(log2 d) */
            const uint64_t d32 = (uint64_t)a->group / 32;
            int l = 0;
            while ((1ull << l) < d32) l++;
            k.gshift = (uint8_t)(26 + l);
            k.gmul = ((1ull << (26 + l)) + d32 - 1) / d32;
        }
        return irx_dev_launch(d, K_MV4 + 6 * f32 + gv * 2 + nt - 1, (unsigned)(tiles * ck), 256, smem, ck, st, &k);
    }
    if (irx_serve_grid(d, K_MV4_ANY, 256, 0, ((u1 - u0) * ((a->m + 3) / 4) + 7) / 8, &grid)) return 1;
    return irx_dev_launch(d, K_MV4_ANY, (unsigned)grid, 256, 0, 1, st, &k);
}

/* ---- one entry for the launch switch, and the plans' descriptions ---- */

int irx_launch_serve(const irx_plan_int_t *p, irx_dev_t *d, unsigned s, unsigned ns, void *const *args, void *st)
{
    int i;
    for (i = 0; i < p->narg; i++)
        if (!a_to(args[i], (size_t)esz(p->arg_dt[i]))) return irx_fail(E093, "a device pointer that its elements' size does not divide");
    switch (p->fam) {
    case FAM_DECODE: return launch_decode(p, d, s, ns, args, st);
    case FAM_KV_APPEND: return launch_append(p, d, s, ns, args, st);
    case FAM_KV_COPY: return launch_copy(p, d, s, ns, args, st);
    default: return launch_mv4(p, d, s, ns, args, st);
    }
}

void irx_serve_text(const irx_plan_int_t *p, char *buf, size_t cap)
{
    if (p->fam == FAM_DECODE) {
        const irx_dec_t *a = &p->u.dec;
        const int st = a->c.dt != DT_BF16 || a->c.dim % 8;
        float sc;
        memcpy(&sc, &a->scale_bits, 4);
        snprintf(buf, cap, "decode batch=%d heads=%d kv_heads=%d d=%d page=%d pages=%lld window=%d sinks=%d lse=%d scale=%g "
                 "dtype=%s kernel=irx_dec_%s_%d_%d", a->c.batch, a->heads, a->c.heads, a->c.dim, a->c.page_size,
                 (long long)a->c.pages, a->window, a->sinks, a->lse, (double)sc, dname(a->c.dt),
                 st ? "st" : "tc", a->dp, st ? a->rows[1] : a->rows[0] / 8);
    } else if (p->fam == FAM_MATVEC4) {
        const irx_mv4_t *a = &p->u.mv;
        snprintf(buf, cap, "matvec4 m=%lld n=%lld k=%lld group=%d zeros=%d dtype=%s", (long long)a->m, (long long)a->n,
                 (long long)a->k, a->group, a->zeros, dname(a->dt));
    } else {
        const irx_kv_t *a = &p->u.kv;
        if (p->fam == FAM_KV_APPEND)
            snprintf(buf, cap, "kv_append tokens=%lld heads=%d d=%d page=%d pages=%lld dtype=%s", (long long)a->n, a->c.heads,
                     a->c.dim, a->c.page_size, (long long)a->c.pages, dname(a->c.dt));
        else
            snprintf(buf, cap, "kv_copy pairs=%lld layers=%d heads=%d d=%d page=%d pages=%lld dtype=%s", (long long)a->n,
                     a->layers, a->c.heads, a->c.dim, a->c.page_size, (long long)a->c.pages, dname(a->c.dt));
    }
}

/* The work that a launch cannot do without (weights, keys and values once, whatever the kernels read again); a
 * decode's, of a full cache (the lengths are only known on the device). */
void irx_serve_work(const irx_plan_int_t *p, double *bytes, double *flops)
{
    *bytes = *flops = 0;
    if (p->fam == FAM_DECODE) {
        const irx_dec_t *a = &p->u.dec;
        const double es = esz(a->c.dt);
        double vis = (double)a->c.cols * a->c.page_size;
        if (a->window && vis > a->window) {
            const double before = vis - a->window;
            vis = a->window + (a->sinks < before ? a->sinks : before);
        }
        vis *= a->c.batch;
        *bytes = 2 * vis * a->c.heads * a->c.dim * es + 2.0 * a->c.batch * a->heads * a->c.dim * es;
        *flops = 4 * vis * a->heads * a->c.dim;
    } else if (p->fam == FAM_KV_APPEND) {
        *bytes = 4.0 * p->u.kv.n * p->u.kv.c.heads * p->u.kv.c.dim * esz(p->u.kv.c.dt) + 8.0 * p->u.kv.n;
    } else if (p->fam == FAM_KV_COPY) {
        const irx_kv_t *a = &p->u.kv;
        *bytes = 4.0 * a->n * a->layers * a->c.heads * a->c.page_size * a->c.dim * esz(a->c.dt) + 8.0 * a->n;
    } else {
        const irx_mv4_t *a = &p->u.mv;
        *bytes = (double)a->n * ((a->k + 1) / 2) + (double)a->n * a->groups * (esz(a->sdt) + a->zeros) +
                 (double)a->m * (a->n + a->k) * esz(a->dt);
        *flops = 2.0 * a->m * a->n * a->k;
    }
}
