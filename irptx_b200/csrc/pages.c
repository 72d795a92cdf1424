/* pages.c -- the host side of a paged cache: which pages each sequence owns.
 *
 * A pool of `pages` pages is shared by at most max_seqs sequences, each a row of a page table. A page
 * has a count of the sequences that hold it: a fork shares all pages, and a sequence that is about
 * to write into a shared last page first gets a page of its own (copy on write), as one (src, dst)
 * pair for a page copy. Compaction moves the live pages to the front of the pool, as a list of such
 * pairs whose destinations were all free. Nothing here touches the device: the caller uploads
 * the table and runs the pairs (irx_compile_kv_copy) on its stream before the launches that use
 * them. Not thread-safe: one owner per manager, as the scheduler that calls it.
 *
 * A caller gathers the pairs of several calls into one launch, whose copies run in no order. So until the
 * table is read, which a caller does once a step to upload it, no page is one pair's destination and in
 * another pair: a page of a pair that nobody holds any more waits instead of being free, and a copy of
 * a page that is itself still to be copied takes the first one's source. */

#include <stdlib.h>
#include <string.h>
#include "irx_int.h"
#include "../../include/irx.h"

struct irx_pages {
    int pages, page_size, cols, max_seqs, nfree, nwait, pairs, compacted;
    int *free_, *refs;              /* the free pages (a stack), and each page's holders */
    int *from;                      /* a page in a pair handed out since the table was last read: the page that
                                     * holds its contents until then (a source: itself); others: -1 */
    int *table;                     /* [max_seqs, cols], -1 where nothing is held */
    int *len;                       /* tokens of each sequence; -1: no such sequence */
};

irx_pages_t *irx_pages_new(int pages, int page_size, int max_seqs, int table_cols)
{
    irx_pages_t *m;
    int i;
    irx_clear_error();
    if (pages < 1 || page_size < 1 || max_seqs < 1 || table_cols < 1 || (long long)table_cols * page_size > 0x7fffffffll ||
        (long long)max_seqs * table_cols > 0x7fffffffll) {
        irx_fail(E042, "a page manager without pages, sequences or columns, or past 2^31 - 1 tokens a sequence");
        return NULL;
    }
    m = (irx_pages_t *)calloc(1, sizeof *m);
    if (m) {
        m->pages = m->nfree = pages;
        m->page_size = page_size;
        m->cols = table_cols;
        m->max_seqs = max_seqs;
        m->free_ = (int *)malloc(sizeof(int) * (size_t)pages);
        m->refs = (int *)calloc((size_t)pages, sizeof(int));
        m->from = (int *)malloc(sizeof(int) * (size_t)pages);
        m->table = (int *)malloc(sizeof(int) * (size_t)max_seqs * (size_t)table_cols);
        m->len = (int *)malloc(sizeof(int) * (size_t)max_seqs);
    }
    if (!m || !m->free_ || !m->refs || !m->from || !m->table || !m->len) {
        irx_pages_delete(m);
        irx_fail(E094, "host memory for a page manager");
        return NULL;
    }
    for (i = 0; i < pages; i++) m->free_[i] = pages - 1 - i;             /* page 0 is handed out first */
    for (i = 0; i < max_seqs; i++) m->len[i] = -1;
    memset(m->from, 0xff, sizeof(int) * (size_t)pages);
    memset(m->table, 0xff, sizeof(int) * (size_t)max_seqs * (size_t)table_cols);
    return m;
}

void irx_pages_delete(irx_pages_t *m)
{
    if (!m) return;
    free(m->free_);
    free(m->refs);
    free(m->from);
    free(m->table);
    free(m->len);
    free(m);
}

static int no_seq(const irx_pages_t *m, int seq)
{
    if (!m) return irx_fail(E093, "a page manager that does not exist");
    if (seq < 0 || seq >= m->max_seqs || m->len[seq] < 0) return irx_fail(E093, "a sequence that is not open");
    return 0;
}

static int held(const irx_pages_t *m, int len) { return (int)(((long long)len + m->page_size - 1) / m->page_size); }

static void put(irx_pages_t *m, int page)
{
    if (--m->refs[page]) return;
    if (m->from[page] < 0) m->free_[m->nfree++] = page;
    else m->nwait++;
}

static int take(irx_pages_t *m) { const int page = m->free_[--m->nfree]; m->refs[page] = 1; return page; }

/* The pair that fills `dst`, a page of no pair, with what `page` holds once the pairs before it have run. */
static void move(irx_pages_t *m, int page, int dst, int pair[2])
{
    const int src = m->from[page] < 0 ? page : m->from[page];
    m->from[src] = m->from[dst] = src;
    pair[0] = src;
    pair[1] = dst;
    m->pairs = 1;
}

/* The free pages by number, the lowest to be handed out first. */
static void sort_free(irx_pages_t *m)
{
    int i;
    for (m->nfree = 0, i = m->pages - 1; i >= 0; i--) if (!m->refs[i] && m->from[i] < 0) m->free_[m->nfree++] = i;
}

/* The pairs handed out so far run before whatever follows: their pages are like any others again. */
static void settle(irx_pages_t *m)
{
    int i;
    for (i = m->pages - 1; i >= 0; i--) {
        if (m->from[i] >= 0 && !m->refs[i]) m->free_[m->nfree++] = i;
        m->from[i] = -1;
    }
    if (m->compacted) sort_free(m);
    m->nwait = m->pairs = m->compacted = 0;
}

static int new_seq(irx_pages_t *m)
{
    int i;
    for (i = 0; i < m->max_seqs; i++) if (m->len[i] < 0) return i;
    irx_fail(E081, "a page manager whose sequences are all open");
    return -1;
}

int irx_pages_open(irx_pages_t *m)
{
    int s;
    irx_clear_error();
    if (!m) { irx_fail(E093, "a page manager that does not exist"); return -1; }
    if ((s = new_seq(m)) >= 0) m->len[s] = 0;
    return s;
}

int irx_pages_extend(irx_pages_t *m, int seq, int tokens, int pair[2])
{
    int have, want, need, i, *row, shared;
    irx_clear_error();
    if (pair) pair[0] = pair[1] = -1;
    if (no_seq(m, seq)) return 1;
    if (!pair || tokens < 0) return irx_fail(E093, "an extension by fewer than 0 tokens, or with nowhere to put its pair");
    if ((long long)m->len[seq] + tokens > (long long)m->cols * m->page_size)
        return irx_fail(E081, "a sequence longer than its row of the page table");
    row = m->table + (size_t)seq * (size_t)m->cols;
    have = held(m, m->len[seq]);
    want = held(m, m->len[seq] + tokens);
    /* the first new token lands in a page that another sequence holds too */
    shared = tokens > 0 && m->len[seq] % m->page_size != 0 && m->refs[row[have - 1]] > 1;
    need = want - have + shared;
    if (need > m->nfree)
        return irx_fail(E094, need > m->nfree + m->nwait ? "a cache page: all of them are held"
                                                         : "a cache page: those left are in copies handed out since the table was last read");
    if (shared) {
        const int page = row[have - 1], own = take(m);
        move(m, page, own, pair);
        put(m, page);
        row[have - 1] = own;
    }
    for (i = have; i < want; i++) row[i] = take(m);
    m->len[seq] += tokens;
    return 0;
}

int irx_pages_fork(irx_pages_t *m, int seq)
{
    int s, i, n;
    irx_clear_error();
    if (no_seq(m, seq) || (s = new_seq(m)) < 0) return -1;
    n = held(m, m->len[seq]);
    m->len[s] = m->len[seq];
    for (i = 0; i < n; i++) {
        const int page = m->table[(size_t)seq * (size_t)m->cols + (size_t)i];
        m->table[(size_t)s * (size_t)m->cols + (size_t)i] = page;
        m->refs[page]++;
    }
    return s;
}

int irx_pages_close(irx_pages_t *m, int seq)
{
    int i, n, *row;
    irx_clear_error();
    if (no_seq(m, seq)) return 1;
    row = m->table + (size_t)seq * (size_t)m->cols;
    n = held(m, m->len[seq]);
    for (i = n - 1; i >= 0; i--) {
        put(m, row[i]);
        row[i] = -1;
    }
    m->len[seq] = -1;
    return 0;
}

int irx_pages_compact(irx_pages_t *m, int *pairs, int cap)
{
    int live, lo = 0, hi, end, room, n = 0, i, *to;
    size_t j;
    irx_clear_error();
    if (!m) { irx_fail(E093, "a page manager that does not exist"); return -1; }
    live = m->pages - m->nfree - m->nwait;
    /* the live pages end up in [0, end): their number, and past the pages that wait for their copies */
    for (end = room = 0; room < live; end++) room += m->refs[end] || m->from[end] < 0;
    for (i = end; i < m->pages; i++) n += m->refs[i] > 0;
    if (n > cap || (n && !pairs)) { irx_fail(E093, "more page moves than the caller's list holds"); return -1; }
    if (!n) return 0;
    to = (int *)malloc(sizeof(int) * (size_t)m->pages);
    if (!to) { irx_fail(E094, "host memory for a compaction"); return -1; }
    for (i = 0; i < m->pages; i++) to[i] = i;
    /* live pages past the end go into the holes below it */
    for (hi = end, n = 0; hi < m->pages; hi++) {
        if (!m->refs[hi]) continue;
        while (m->refs[lo] || m->from[lo] >= 0) lo++;
        move(m, hi, lo, pairs + 2 * n);
        to[hi] = lo;
        m->refs[lo] = m->refs[hi];
        m->refs[hi] = 0;
        n++;
    }
    for (j = 0; j < (size_t)m->max_seqs * (size_t)m->cols; j++) if (m->table[j] >= 0) m->table[j] = to[m->table[j]];
    free(to);
    sort_free(m);
    m->nwait = m->pages - live - m->nfree;
    m->compacted = 1;
    return n;
}

int irx_pages_free(const irx_pages_t *m) { return m ? m->nfree : 0; }

int irx_pages_len(const irx_pages_t *m, int seq) { return m && seq >= 0 && seq < m->max_seqs ? m->len[seq] : -1; }

const int *irx_pages_table(irx_pages_t *m)
{
    if (!m) return NULL;
    if (m->pairs) settle(m);
    return m->table;
}
