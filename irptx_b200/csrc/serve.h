/* serve.h -- what the operators compiled from descriptors share (serve.c, step.c). */
#ifndef IRX_SERVE_H
#define IRX_SERVE_H

#include <stdio.h>
#include <string.h>
#include "irx_int.h"
#include "irx_kparams.h"
#include "launch.h"
#include "../../include/irx.h"

#define MAX_DIM 256
#define MAX_COUNT 0x7fffffffll
#define MAX_STRIDE (1ll << 40)
#define MAX_SCALE 2.35e38f                 /* of scores: times log2(e) still an f32 number */
#define MAX_SPAN 9e17                      /* elements; sums of a few stay below 2^63 */

static inline int esz(int dt) { return dt == DT_BF16 ? 2 : dt == DT_U8 ? 1 : 4; }

static inline int float_dt(int dt) { return dt == DT_BF16 || dt == DT_F32; }

static inline const char *dname(int dt) { return dt == DT_BF16 ? "bf16" : "f32"; }

static inline int a_to(const void *q, size_t n) { return ((size_t)q % n) == 0; }

static inline irx_plan_int_t *begin(irx_plan_t *plan, int fam, const char *name)
{
    irx_plan_int_t *p = (irx_plan_int_t *)plan;
    irx_clear_error();
    if (!plan) {
        irx_fail(E093, "a compile with no plan storage");
        return NULL;
    }
    memset(plan, 0, sizeof *plan);
    p->fam = (uint8_t)fam;
    snprintf(p->kname, sizeof p->kname, "%s", name);
    return p;
}

static inline void add(irx_plan_int_t *p, int kind, int dt, int64_t elems)
{
    p->arg_kind[p->narg] = (uint8_t)kind;
    p->arg_dt[p->narg] = (uint8_t)dt;
    p->arg_elems[p->narg] = elems;
    p->narg++;
}

static inline int finish(irx_plan_int_t *p) { p->magic = IRX_PLAN_MAGIC; return 0; }

/* A cache descriptor checked into its plan form; the elements from the first to past the last of its pools. */
int irx_cache_of(irx_kvc_t *o, const irx_kv_cache_t *c, int tabled);
int64_t irx_cache_span(const irx_kvc_t *c);

/* One resident wave of kernel k, at most `want` blocks. */
int irx_serve_grid(irx_dev_t *d, int k, int block, size_t smem, int64_t want, int64_t *g);

#endif
