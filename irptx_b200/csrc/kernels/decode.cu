// decode.cu -- attention of one new token per sequence over a paged key-value cache.
//
// For a sequence b of n tokens, its newest token's query head h sees the keys
//     j in [0, min(sinks, n - window)) and [n - window, n)      (every j < n without a window)
// of key-value head h / group:  o = sum_j softmax_j(scale * q.k_j) v_j, zeros when n = 0, and
// lse = ln sum_j exp(scale * q.k_j) (-inf when n = 0).
//
// Bound: every visible key and value row is read and takes 4 * group operations per element, so HBM
// bounds it (group operations a byte in bf16). A unit, (sequence, kv head, row block), reads its keys
// for 16 query rows at most (8 at head sizes past 128 and in f32): wider groups are several units and
// read them as often. The work is cut by keys, not by rows: the visible keys of all units are laid
// end to end in chunks of 64 or 128 keys and the chunks are dealt out evenly, a contiguous range to
// each block of one resident wave, whatever the lengths are. A block whose range covers a whole
// unit writes its output; a unit that several blocks share is joined by the last of them to
// arrive, which folds the blocks' partials in key order, so the result does not depend on which
// block that was. Past DEC_JOIN partials they are folded in groups first, by the last block of
// each group, so a single long sequence's join is not one block's work.
//
// Measured (bf16, 8 kv heads of 128 and 32 query heads): two sequences of 120 to 131 thousand tokens
// (1.0 GB) in 163 us, 6.2 TB/s; 31 of 1 to 4096 tokens (259 MB) in 49 us, 5.3 TB/s. Of those 49
// about 2 are the launch, 2.6 pass before the first keys can be asked for (lengths, then the page
// table), the keys stream for 37 at 7 TB/s, and 5 are the ends: warps meet, partials are written,
// counted and folded. One sequence of 17 tokens takes 5.5 us, those latencies alone. Sixteen sequences of 8192
// tokens: 4 rows a group 90 us (5.9 TB/s), 16 rows 102, 32 rows, read twice, 183; head size 80, whose rows
// lie in tiles of 128, 79 us (4.3 TB/s), 96 79 (5.1), 256 170 (6.3), 256 with 16 rows, read twice, 330.
#pragma once
#include "tc.cuh"
#include "kvpages.cu"

#define DEC_JOIN 16

// A place in the laid-out chunks: chunk j of the unit (kv head h0 + h, row block rb) of sequence b. A
// chunk is K positions from a multiple of K (what a thread block takes in one step): the first `cs`
// of a sequence's chunks are those that hold sinks, the others those from number wb on; keys outside
// the mask are dropped in their tile.
struct DecCur {
    int b, h, rb, j;
    int nch, n, lo, sk, cs, wb;       // of sequence b: chunks, tokens, window start, sinks before it
};

__device__ __forceinline__ int dec_len(const irx_kdec_t &p, int n)
{
    const int64_t cap = (int64_t)p.cols * p.page_size;
    return n < 0 ? 0 : (int64_t)n > cap ? (int)cap : n;
}

template <int K>
__device__ __forceinline__ int dec_blocks(int n) { return n / K + (n % K != 0); }

// Sequence c.b's numbers, from its length.
template <int K>
__device__ __forceinline__ void dec_enter(const irx_kdec_t &p, DecCur &c, int len)
{
    c.n = dec_len(p, len);
    c.lo = c.sk = c.cs = c.wb = 0;
    if (p.window > 0 && c.n > p.window) {
        c.lo = c.n - p.window;
        c.sk = min(p.sinks, c.lo);
        c.cs = dec_blocks<K>(c.sk);
        c.wb = max(c.lo / K, c.cs);
    }
    c.nch = c.cs + dec_blocks<K>(c.n) - c.wb;
}

template <int K>
__device__ __forceinline__ void dec_next(const irx_kdec_t &p, DecCur &c)
{
    if (++c.j < c.nch) return;
    c.j = 0;
    if (++c.rb < p.split) return;
    c.rb = 0;
    if (++c.h < p.h1 - p.h0) return;
    c.h = 0;
    do {
        if (++c.b >= p.batch) { c.n = 0; c.nch = 0x7fffffff; return; }        // past the end
        dec_enter<K>(p, c, p.lens[c.b]);
    } while (c.nch == 0);
}

// The first position of the cursor's chunk j, and whether a tile of `keys` positions from pos shows any
// key, or shows all of them.
template <int K>
__device__ __forceinline__ int dec_pos(const DecCur &c, int j) { return (j < c.cs ? j : j - c.cs + c.wb) * K; }
__device__ __forceinline__ bool dec_any(const DecCur &c, int pos, int keys) { return pos < c.n && (pos > c.lo - keys || pos < c.sk); }
__device__ __forceinline__ bool dec_all(const DecCur &c, int pos, int keys) { return c.n - pos >= keys && (pos >= c.lo || c.sk - pos >= keys); }
__device__ __forceinline__ bool dec_sees(const DecCur &c, int pos) { return pos < c.n && (pos >= c.lo || pos < c.sk); }

struct DecShare {
    long long c0, c1, q;              // this block's chunks; the first r blocks have q + 1, the others q
    long long wsum[16];               // a warp each
    int geff, r, b, u, j;
    int last[2];
    // the shares of units that other blocks hold too: [0] the one that began before this block, [1] the
    // one that goes on after it; pieces = 0: none
    struct { long long unit; int first, pieces, b, head0, live; } pend[2];
};

// What a unit takes on the line that is dealt out: its chunks and EXTRA more, about what its end costs
// (its warps meet, write and begin anew). Without them blocks that hold many short units finish late:
// measured at 31 sequences of 1 to 4096 tokens, the last block at 52 us, the median one at 39.
template <int EXTRA>
__device__ __forceinline__ long long dec_cost(int nch) { return nch ? nch + EXTRA : 0; }

__device__ __forceinline__ long long dec_div(long long a, long long b)         // not below 0; mostly 32 bits
{
    return ((a | b) >> 32) == 0 ? (long long)((unsigned)a / (unsigned)b) : a / b;
}

// The block's chunk range and where it starts: every block sums the chunks of all sequences (a
// segment of them per thread, then a scan), so nothing has to run before the kernel.
template <int THREADS, int K, int EXTRA>
__device__ __forceinline__ void dec_partition(const irx_kdec_t &p, int upb, DecShare &S)
{
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = THREADS / 32;
    const int seg = (p.batch + THREADS - 1) / THREADS, b0 = tid * seg, b1 = min(p.batch, b0 + seg);
    long long sum = 0;
    DecCur w;
    for (int b = b0; b < b1; b++) {
        const int raw = p.lens[b];
        dec_enter<K>(p, w, raw);
        if (raw != w.n && blockIdx.x == 0) irx_flag(p.err, IRX_KERR_INDEX);
        sum += dec_cost<EXTRA>(w.nch);
    }
    long long inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) S.wsum[warp] = inc;
    __syncthreads();
    long long total = 0, before = 0;
#pragma unroll
    for (int i = 0; i < nw; i++) {
        if (i == warp) before = total;
        total += S.wsum[i];
    }
    total *= upb;
    const int geff = (int)min((long long)gridDim.x, total), i = blockIdx.x;
    const long long q = geff ? dec_div(total, geff) : 0;
    const int r = (int)(total - q * geff);
    const long long c0 = i < geff ? i * q + min(i, r) : 0, c1 = i < geff ? c0 + q + (i < r) : 0;
    if (tid == 0) {
        S.c0 = c0; S.c1 = c1; S.q = q; S.r = r; S.geff = geff;
        S.pend[0].pieces = S.pend[1].pieces = 0;
    }
    const long long ex = (before + inc - sum) * upb;
    if (c0 < c1 && c0 >= ex && c0 < ex + sum * upb) {    // exactly one thread's segment holds c0
        long long at = c0 - ex;
        for (int b = b0; b < b1; b++) {
            dec_enter<K>(p, w, p.lens[b]);
            const long long cost = dec_cost<EXTRA>(w.nch);
            if (at < cost * upb) {
                const long long u = dec_div(at, cost);
                S.b = b; S.u = (int)u; S.j = (int)(at - u * cost);
                break;
            }
            at -= cost * upb;
        }
    }
    __syncthreads();
}

// The block's first chunk, at place c0 of the line.
template <int K, int EXTRA>
__device__ __forceinline__ long long dec_start(const irx_kdec_t &p, const DecShare &S, DecCur &c)
{
    c.b = S.b;
    c.h = S.u / p.split;
    c.rb = S.u % p.split;
    c.j = S.j;
    dec_enter<K>(p, c, p.lens[c.b]);
    if (c.j < c.nch) return S.c0;
    const long long at = S.c0 + (c.nch + EXTRA - c.j);   // the share begins in a unit's end: with the next unit then
    c.j = c.nch - 1;
    dec_next<K>(p, c);
    return at;
}

// The place of the next chunk on the line, from a chunk at place c.
template <int EXTRA>
__device__ __forceinline__ long long dec_step(const DecCur &w, long long c) { return c + (w.j + 1 < w.nch ? 1 : 1 + EXTRA); }

// The block that holds chunk c.
__device__ __forceinline__ int dec_block_of(const DecShare &S, long long c)
{
    const long long big = (long long)S.r * (S.q + 1);
    return (int)(c < big ? dec_div(c, S.q + 1) : S.r + dec_div(c - big, S.q));
}

// Partials: slot s holds `rows` x dp accumulators, then rows (max, sum) pairs. Maxima are of
// scale2 * q.k, the log2 domain.
__device__ __forceinline__ float *dec_slot(const irx_kdec_t &p, int s, int rows, int dp)
{
    return p.part + (int64_t)s * rows * (dp + 2);
}

__device__ __forceinline__ void dec_store_out(const irx_kdec_t &p, int b, int head, int d0, float4 v)
{
    const int64_t o = ((int64_t)b * p.heads + head) * p.d + d0;
    const float a[4] = {v.x, v.y, v.z, v.w};
    if (p.vec) {
        if (d0 >= p.d) return;
        if (p.dt == DT_BF16) {
            uint2 r;
            __nv_bfloat162 *hh = reinterpret_cast<__nv_bfloat162 *>(&r);
            hh[0] = __floats2bfloat162_rn(a[0], a[1]);
            hh[1] = __floats2bfloat162_rn(a[2], a[3]);
            *reinterpret_cast<uint2 *>(reinterpret_cast<__nv_bfloat16 *>(p.o) + o) = r;
        } else {
            *reinterpret_cast<float4 *>(reinterpret_cast<float *>(p.o) + o) = v;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) if (d0 + i < p.d) irx_st1(p.o, p.dt, o + i, a[i]);
}

// Fold `cnt` partials, in slots first, rest0 + step, rest0 + 2 step, ..., in that order, by the whole block.
// With `fin` the result is the unit's output, else it becomes the partial of the first slot. Every thread
// weighs the partials of its own row, so that all its loads are on their way at once and no
// barrier is needed.
template <int DP, int ROWS, int THREADS>
__device__ __forceinline__ void dec_fold(const irx_kdec_t &p, int first, int rest0, int step, int cnt, bool fin, int b,
                                         int head0, int live, float2 *sw)
{
    for (int it = threadIdx.x; it < live * (DP / 4); it += THREADS) {
        const int r = it / (DP / 4), d0 = (it % (DP / 4)) * 4;
        if (d0 >= p.d) continue;
        float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float m = -INFINITY, l = 0.0f;
        for (int k0 = 0; k0 < cnt; k0 += 8) {
            float4 v[8];
            float2 s[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                s[k] = make_float2(-INFINITY, 0.0f);
                if (k0 + k < cnt) {
                    const float *o = dec_slot(p, k0 + k ? rest0 + (k0 + k) * step : first, ROWS, DP);
                    s[k] = __ldcg(reinterpret_cast<const float2 *>(o + ROWS * DP) + r);
                    v[k] = __ldcg(reinterpret_cast<const float4 *>(o + r * DP + d0));
                }
            }
            float mn = m;
#pragma unroll
            for (int k = 0; k < 8; k++) mn = fmaxf(mn, s[k].x);
            const float base = mn == -INFINITY ? 0.0f : mn, f0 = exp2f(m - base);
            a.x *= f0; a.y *= f0; a.z *= f0; a.w *= f0;
            l *= f0;
            m = mn;
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (k0 + k < cnt) {
                    const float f = exp2f(s[k].x - base);
                    l += f * s[k].y;
                    a.x += f * v[k].x; a.y += f * v[k].y; a.z += f * v[k].z; a.w += f * v[k].w;
                }
        }
        if (fin) {
            const float inv = 1.0f / l;
            dec_store_out(p, b, head0 + r, d0, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
            if (p.lse && d0 == 0) p.lse[(int64_t)b * p.heads + head0 + r] = (m + log2f(l)) * 0.6931471805599453f;
        } else {
            __stcg(reinterpret_cast<float4 *>(dec_slot(p, first, ROWS, DP) + r * DP + d0), a);
            if (d0 == 0) sw[r] = make_float2(m, l);
        }
    }
    if (fin) return;
    __syncthreads();                                     // every thread has read the first slot's pairs
    if (threadIdx.x < live) __stcg(reinterpret_cast<float2 *>(dec_slot(p, first, ROWS, DP) + ROWS * DP) + threadIdx.x, sw[threadIdx.x]);
}

// A unit's share of this block is done. `acc(r, d0, k)` gives the block's four accumulators of row r
// from d0 (item k of this thread), `ml(r)` its (max, sum). Chunk c is the share's last one. A unit
// that is all here is written out; a part of one becomes a partial, which dec_join looks after at
// the end of the block: waiting for the arrival count here would stall the block's loads.
template <int DP, int ROWS, int THREADS, class Acc, class Ml>
__device__ __forceinline__ void dec_finish(const irx_kdec_t &p, DecShare &S, const DecCur &cur, long long c, int upb, Acc acc, Ml ml)
{
    const int tid = threadIdx.x;
    const int head0 = (p.h0 + cur.h) * p.group + cur.rb * ROWS, live = min(ROWS, p.group - cur.rb * ROWS);
    const long long ua = c - cur.j, ub = ua + cur.nch;       // the unit's chunks
    const bool alone = ua >= S.c0 && ub <= S.c1;
    const int which = ua >= S.c0 ? 1 : 0, slot = 2 * (int)blockIdx.x + which;
#pragma unroll
    for (int k = 0; k < (ROWS * DP / 4 + THREADS - 1) / THREADS; k++) {
        const int it = tid + k * THREADS, r = it / (DP / 4), d0 = (it % (DP / 4)) * 4;
        if (r >= live || d0 >= p.d) continue;
        const float4 a = acc(r, d0, k);
        const float2 s = ml(r);
        if (alone) {
            const float inv = 1.0f / s.y;
            dec_store_out(p, cur.b, head0 + r, d0, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
            if (p.lse && d0 == 0) p.lse[(int64_t)cur.b * p.heads + head0 + r] = (s.x + log2f(s.y)) * 0.6931471805599453f;
        } else {
            float *o = dec_slot(p, slot, ROWS, DP);
            __stcg(reinterpret_cast<float4 *>(o + r * DP + d0), a);
            if (d0 == 0) __stcg(reinterpret_cast<float2 *>(o + ROWS * DP) + r, s);
        }
    }
    if (!alone && tid == 0) {
        const int first = dec_block_of(S, ua);
        S.pend[which].unit = (long long)cur.b * upb + cur.h * p.split + cur.rb;
        S.pend[which].first = first;
        S.pend[which].pieces = dec_block_of(S, ub - 1) - first + 1;
        S.pend[which].b = cur.b;
        S.pend[which].head0 = head0;
        S.pend[which].live = live;
    }
}

// The end of a block: its partials arrive at their units' counters; the last block to arrive folds a
// unit's partials, and leaves the counter at zero. Up to DEC_JOIN partials fold at once; more
// fold in groups of DEC_JOIN first, each into its first slot, by the last block of the group.
template <int DP, int ROWS, int THREADS>
__device__ __forceinline__ void dec_join(const irx_kdec_t &p, DecShare &S, float2 *sw)
{
    // one arrival that publishes what the block's threads wrote before the last barrier, and shows the last
    // block to arrive what all the others published
    auto arrive = [&](unsigned *ctr, int want) {
        unsigned a;
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(a) : "l"(ctr) : "memory");
        if (a == (unsigned)want - 1) *ctr = 0;
        return a == (unsigned)want - 1 ? 1 : 0;
    };
    if (!(S.pend[0].pieces | S.pend[1].pieces)) return;  // (a barrier ended the last unit's share)
    if (threadIdx.x < 2) {
        const auto &e = S.pend[threadIdx.x];
        int last = 0;
        if (e.pieces > DEC_JOIN) {
            const int g = ((int)blockIdx.x - e.first) / DEC_JOIN;
            last = arrive(p.gcount + 2 * (e.first + g * DEC_JOIN) + (g ? 0 : 1), min(DEC_JOIN, e.pieces - g * DEC_JOIN));
        } else if (e.pieces) {
            last = arrive(p.ticket + e.unit, e.pieces);
        }
        S.last[threadIdx.x] = last;
    }
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < 2; i++) {
        const auto e = S.pend[i];
        if (!S.last[i]) continue;
        if (e.pieces > DEC_JOIN) {
            const int g = ((int)blockIdx.x - e.first) / DEC_JOIN, g0 = e.first + g * DEC_JOIN, ng = (e.pieces + DEC_JOIN - 1) / DEC_JOIN;
            dec_fold<DP, ROWS, THREADS>(p, 2 * g0 + (g ? 0 : 1), 2 * g0, 2, min(DEC_JOIN, e.pieces - g * DEC_JOIN), false, e.b, e.head0, e.live, sw);
            __syncthreads();
            if (threadIdx.x == 0) S.last[i] = arrive(p.ticket + e.unit, ng);
            __syncthreads();
            if (!S.last[i]) continue;
            dec_fold<DP, ROWS, THREADS>(p, 2 * e.first + 1, 2 * e.first, 2 * DEC_JOIN, ng, true, e.b, e.head0, e.live, sw);
        } else {
            dec_fold<DP, ROWS, THREADS>(p, 2 * e.first + 1, 2 * e.first, 2, e.pieces, true, e.b, e.head0, e.live, sw);
        }
    }
}

// Sequences with no tokens: zeros, and -inf for the log-sum.
__device__ __forceinline__ void dec_empty(const irx_kdec_t &p)
{
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
        if (p.lens[b] > 0) continue;
        const int r0 = p.h0 * p.group, nr = (p.h1 - p.h0) * p.group;
        for (int i = threadIdx.x; i < nr * p.d; i += blockDim.x)
            irx_st1(p.o, p.dt, ((int64_t)b * p.heads + r0) * p.d + i, 0.0f);
        if (p.lse)
            for (int i = threadIdx.x; i < nr; i += blockDim.x) p.lse[(int64_t)b * p.heads + r0 + i] = -INFINITY;
    }
}

// Where a warp's key rows of the tiles to come lie: for each tile of its ring, for each of the tile's keys,
// the key's page (copied from the table asynchronously, a whole ring ahead of its use, so that no load of
// keys waits for the table) and the rest of its offset, -1 where there is no such key.
// `bad`: of the tile that is in the slot now, the keys that the table puts outside the pool, a bit each (the
// matrix kernel reads it only where there are any).
template <int KEYS>
struct DecRows {
    long long off[KEYS];
    int page[KEYS];
    unsigned bad, pad;
};

// pos / page_size by a multiplication, exact below 2^31 (the launcher's constants).
__device__ __forceinline__ unsigned dec_page_of(const irx_kdec_t &p, int pos) { return (unsigned)(((uint64_t)(unsigned)pos * p.pmul) >> p.pshift); }

template <int KEYS>
__device__ __forceinline__ void dec_lookup(const irx_kdec_t &p, const DecCur &c, bool more, int pos0, DecRows<KEYS> &R)
{
    const int lane = threadIdx.x & 31;
    if (lane < KEYS) {
        const int pos = pos0 + lane;
        long long off = -1;
        if (more && dec_sees(c, pos)) {
            const unsigned pi = dec_page_of(p, pos);
            off = (long long)((unsigned)pos - pi * (unsigned)p.page_size) * p.token_stride + (long long)(p.h0 + c.h) * p.head_stride;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;"
                         :: "r"(irx_smem_u32(&R.page[lane])), "l"(p.table + ((int64_t)c.b * p.cols + pi)) : "memory");
        }
        R.off[lane] = off;
    }
}

// The element offset of the tile's key `i`: -1 when there is none, -2 (flagged) when the table's page is
// not one of the pool's. Such a key is left out of the softmax, as one outside the mask is.
template <int KEYS>
__device__ __forceinline__ long long dec_row(const irx_kdec_t &p, const DecRows<KEYS> &R, int i)
{
    const long long off = R.off[i];
    if (off < 0) return -1;
    const int page = R.page[i];
    if (page < 0 || page >= p.pages) {
        irx_flag(p.err, IRX_KERR_INDEX);
        return -2;
    }
    return off + (long long)page * p.page_stride;
}

// ---- bf16: matrix instructions ----
// The transposed products: S^T[16 keys x 8 rows] = K Q^T and O^T[16 dims x 8 rows] += V^T P^T, so that
// the few query rows sit on the instruction's narrow side (8) and keys or dims on its wide one.
// S^T's accumulators become P^T's operand by an 8x8 transpose across the warp. Each warp owns 16
// keys of a chunk (32 at head size 64, where 16 are too little work for what a tile costs) and its
// own ring of ST tiles filled by 16-byte asynchronous copies, so warps meet only where a unit ends. mma.sync runs far below tcgen05's rate, but at 8 to 16 rows
// the products take 24 to 48 instructions per 8 KB (D = 128), which HBM delivers in about 360
// cycles per SM: the tensor pipe is idle most of the time and tcgen05's 128-row tiles would be
// filled with padding.
// P enters the product as two bf16 numbers, its upper half truncated and the rest rounded, 16 bits in
// all: the tensor pipe has room for the second product, and the output is then as near the
// definition as one rounded once at the end. (The rest of a weight that is not 0 is kept above 0, so that an
// infinite value does not meet 0 there: at 2^-126, or 2^-16 of the weight where that is less, since
// a weight of 0 must add nothing under values of 2^120.)

__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

__device__ __forceinline__ uint32_t trans8(uint32_t x)
{
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// 16 bytes global -> shared, or 16 zero bytes when `bytes` is 0.
__device__ __forceinline__ void cp16(uint32_t dst, const void *src, uint32_t bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ void cp16(uint32_t dst, const void *src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(dst), "l"(src) : "memory");
}

__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }

#define DEC_TC_WARPS 4

template <int DP, int NT, int KM, int ST>
struct DecTc {
    static constexpr int THREADS = DEC_TC_WARPS * 32, ROWS = 8 * NT, KEYS = 16 * KM, K = DEC_TC_WARPS * KEYS, TILE = KEYS * DP * 2, QS = DP + 4;
    // ring, one 8-row block of two warps' accumulators, (max, sum) pairs, the share, the rings' row places
    static constexpr int RING = DEC_TC_WARPS * ST * 2 * TILE;
    static constexpr int MERGE = DEC_TC_WARPS / 2 * 8 * QS * 4;
    static constexpr int ML = DEC_TC_WARPS * ROWS * 8;
    static constexpr int PLACES = RING + MERGE + ML + IRX_DEC_SHARE;
    static constexpr int SMEM = PLACES + DEC_TC_WARPS * ST * (int)sizeof(DecRows<KEYS>);
    static_assert(SMEM == IRX_DEC_TC_SMEM(DP, NT, KM, ST), "the launcher's shared memory size");
    static_assert(sizeof(DecShare) <= IRX_DEC_SHARE, "shared memory");
};

// A tile, 16 KM keys, lies in 64-dim columns of 128 bytes a key, 16-byte pieces swizzled by row against
// bank conflicts.
// (Filling tiles by TMA, a page's 8 or 16 rows a box, measured no better: 171 against 164 us for two
// sequences of 125k tokens, 54 against 52 for 31 of 2k.)
template <int DP, int NT, int KM, int ST>
__device__ __forceinline__ void dec_tc_body(const irx_kdec_t &p)
{
    using T = DecTc<DP, NT, KM, ST>;
    constexpr int EX = DP == 64 ? 3 : DP == 128 ? 2 : 1;
    extern __shared__ __align__(128) unsigned char sm[];
    float *merge = reinterpret_cast<float *>(sm + T::RING);
    float2 *wml = reinterpret_cast<float2 *>(sm + T::RING + T::MERGE);
    DecShare &S = *reinterpret_cast<DecShare *>(sm + T::RING + T::MERGE + T::ML);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    DecRows<T::KEYS> *rows = reinterpret_cast<DecRows<T::KEYS> *>(sm + T::PLACES) + warp * ST;
    const int upb = (p.h1 - p.h0) * p.split;

    irx_pdl_enter();
    dec_partition<T::THREADS, T::K, EX>(p, upb, S);
    if (S.c0 < S.c1) {
        DecCur tl, cu;                                       // the tile whose rows are looked up next, the one in work
        const long long cfirst = dec_start<T::K, EX>(p, S, tl);
        cu = tl;
        const uint32_t ring = irx_smem_u32(sm) + warp * (ST * 2 * T::TILE);
        long long tc = cfirst;                                 // the chunk that `tl` is at
        constexpr int CPR = DP / 8, RPI = 32 / CPR, NI = T::KEYS / RPI;
        const int lrow = lane / CPR, lch = lane % CPR;
        const bool cin = lch * 8 < p.d;
        unsigned bads = 0;                                     // slots whose tile has bad keys
        auto lookup = [&](int st) {
            dec_lookup<T::KEYS>(p, tl, tc < S.c1, dec_pos<T::K>(tl, tl.j) + warp * T::KEYS, rows[st]);
            if (tc < S.c1) {
                tc = dec_step<EX>(tl, tc);
                dec_next<T::K>(p, tl);
            }
        };
        auto fetch = [&](int st) {
            const long long off = dec_row<T::KEYS>(p, rows[st], lane & (T::KEYS - 1));
            const uint32_t kd = ring + st * (2 * T::TILE);
            if (DP < 256 && __all_sync(0xffffffffu, off >= 0) && p.d == DP) {      // every row whole: offsets by way of shared memory
                if (lane < T::KEYS) rows[st].off[lane] = off;
                __syncwarp();
                const char *src = reinterpret_cast<const char *>(p.k) + lch * 16;
                const long long dv = reinterpret_cast<const char *>(p.v) - reinterpret_cast<const char *>(p.k);
#pragma unroll
                for (int i = 0; i < NI; i++) {
                    const int row = i * RPI + lrow;
                    const char *k = src + rows[st].off[row] * 2;
                    const uint32_t d = kd + (lch >> 3) * (T::KEYS * 128) + row * 128 + (((lch & 7) ^ (row & 7)) << 4);
                    cp16(d, k);
                    cp16(d + T::TILE, k + dv);
                }
                bads &= ~(1u << st);
            } else if (__any_sync(0xffffffffu, off != -1)) {
                const unsigned bad = __ballot_sync(0xffffffffu, off == -2);
                if (lane == 0) rows[st].bad = bad;
                bads = (bads & ~(1u << st)) | (bad ? 1u << st : 0);
#pragma unroll
                for (int i = 0; i < NI; i++) {
                    const int row = i * RPI + lrow;
                    const long long o = __shfl_sync(0xffffffffu, off, row);
                    const uint32_t d = kd + (lch >> 3) * (T::KEYS * 128) + row * 128 + (((lch & 7) ^ (row & 7)) << 4);
                    const int64_t e = o >= 0 && cin ? o + lch * 8 : 0;
                    const uint32_t nb = o >= 0 && cin ? 16 : 0;
                    cp16(d, reinterpret_cast<const __nv_bfloat16 *>(p.k) + e, nb);
                    cp16(d + T::TILE, reinterpret_cast<const __nv_bfloat16 *>(p.v) + e, nb);
                }
            }
            __syncwarp();
            lookup(st);
            cp_commit();
        };
        for (int s = 0; s < ST; s++) lookup(s);
        cp_commit();
        cp_wait<0>();
        __syncwarp();
        for (int s = 0; s < ST; s++) fetch(s);

        uint32_t q[DP / 16][NT][2];
        float o[DP / 16][NT][4], m[NT][2], l[NT][2];
        int st = 0;
        bool fresh = true;
        auto load_q = [&](const DecCur &w) {                 // a unit's query rows
            const __nv_bfloat16 *qg = reinterpret_cast<const __nv_bfloat16 *>(p.q) + (int64_t)w.b * p.q_stride;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const int r = w.rb * T::ROWS + nt * 8 + g;
                const __nv_bfloat16 *row = qg + (int64_t)((p.h0 + w.h) * p.group + r) * p.d;
#pragma unroll
                for (int ks = 0; ks < DP / 16; ks++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int d0 = ks * 16 + h * 8 + 2 * t;
                        q[ks][nt][h] = r < p.group && d0 < p.d ? *reinterpret_cast<const uint32_t *>(row + d0) : 0u;
                    }
            }
        };
        if (cfirst < S.c1) load_q(cu);
        for (long long c = cfirst; c < S.c1;) {
            if (fresh) {                                     // a unit starts: an empty state
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    m[nt][0] = m[nt][1] = -INFINITY;
                    l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
                    for (int i = 0; i < DP / 16; i++)
#pragma unroll
                        for (int j = 0; j < 4; j++) o[i][nt][j] = 0.0f;
                }
                fresh = false;
            }
            cp_wait<ST - 1>();
            __syncwarp();
            const int pos = dec_pos<T::K>(cu, cu.j) + warp * T::KEYS;
            if (dec_any(cu, pos, T::KEYS)) {
                const uint32_t kb = ring + st * (2 * T::TILE), vb = kb + T::TILE;
                const bool whole = dec_all(cu, pos, T::KEYS) && !(bads >> st & 1);
                const unsigned bad = bads >> st & 1 ? rows[st].bad : 0;
                // S^T: two sums per 16 keys where there are 16 only, of even and odd steps: half the chain
                float s[KM][NT][4], s2[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        s2[nt][i] = 0.0f;
#pragma unroll
                        for (int km = 0; km < KM; km++) s[km][nt][i] = 0.0f;
                    }
                {
                    const int row = (lane & 7) + ((lane >> 3) & 1) * 8, ch = lane >> 4;
#pragma unroll
                    for (int ks = 0; ks < DP / 16; ks++)
#pragma unroll
                        for (int km = 0; km < KM; km++) {
                            uint32_t a[4];
                            ldsm4(a, kb + (ks >> 2) * (T::KEYS * 128) + (km * 16 + row) * 128 + (((2 * (ks & 3) + ch) ^ (row & 7)) << 4));
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) mma_16816(KM == 1 && (ks & 1) ? s2[nt] : s[km][nt], a, q[ks][nt][0], q[ks][nt][1]);
                        }
                }
                bool in[KM][2];
#pragma unroll
                for (int km = 0; km < KM; km++)
#pragma unroll
                    for (int h = 0; h < 2; h++) in[km][h] = whole || (dec_sees(cu, pos + km * 16 + h * 8 + g) && !(bad >> (km * 16 + h * 8 + g) & 1));
                uint32_t pb[KM][NT][2], pl[KM][NT][2];       // P^T's upper and lower halves
                bool grew = false;
                float al[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        float x = -INFINITY;
#pragma unroll
                        for (int km = 0; km < KM; km++)
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                float &v = s[km][nt][i + 2 * h];
                                if (KM == 1) v += s2[nt][i + 2 * h];
                                v = in[km][h] ? v * p.scale2 : -INFINITY;
                                x = fmaxf(x, v);
                            }
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                        const float mn = fmaxf(m[nt][i], x), base = mn == -INFINITY ? 0.0f : mn;
                        al[nt][i] = exp2f(m[nt][i] - base);
                        grew = grew || mn > m[nt][i];
                        m[nt][i] = mn;
                        float sum = 0.0f;
#pragma unroll
                        for (int km = 0; km < KM; km++)
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                float &v = s[km][nt][i + 2 * h];
                                v = exp2f(v - base);
                                sum += v;
                            }
                        l[nt][i] = l[nt][i] * al[nt][i] + sum;
                    }
#pragma unroll
                    for (int km = 0; km < KM; km++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const float x = s[km][nt][2 * h], y = s[km][nt][2 * h + 1];
                            const uint32_t hi = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
                            const __nv_bfloat162 lo = __floats2bfloat162_rn(fmaxf(x - __uint_as_float(hi << 16), fminf(x * 0x1p-16f, 0x1p-126f)),
                                                                            fmaxf(y - __uint_as_float(hi & 0xffff0000u), fminf(y * 0x1p-16f, 0x1p-126f)));
                            pb[km][nt][h] = trans8(hi);
                            pl[km][nt][h] = trans8(*reinterpret_cast<const uint32_t *>(&lo));
                        }
                }
                if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                    for (int i = 0; i < DP / 16; i++)
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            o[i][nt][0] *= al[nt][0]; o[i][nt][1] *= al[nt][1];
                            o[i][nt][2] *= al[nt][0]; o[i][nt][3] *= al[nt][1];
                        }
                }
                {
                    const int row = (lane & 7) + (lane >> 4) * 8, ch = (lane >> 3) & 1;
#pragma unroll
                    for (int km = 0; km < KM; km++)
#pragma unroll
                        for (int i = 0; i < DP / 16; i++) {
                            uint32_t a[4];
                            ldsm4t(a, vb + (i >> 2) * (T::KEYS * 128) + (km * 16 + row) * 128 + (((2 * (i & 3) + ch) ^ (row & 7)) << 4));
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                mma_16816(o[i][nt], a, pb[km][nt][0], pb[km][nt][1]);
                                mma_16816(o[i][nt], a, pl[km][nt][0], pl[km][nt][1]);
                            }
                        }
                }
            }
            __syncwarp();
            fetch(st);
            if (++st == ST) st = 0;
            const long long cnext = dec_step<EX>(cu, c);
            if (cu.j + 1 == cu.nch || cnext >= S.c1) {
                // the unit's share ends: the warps' states meet in shared memory, one 8-row block at a time,
                // while the next unit's query rows are on their way
                if (cnext < S.c1) {
                    DecCur nx = cu;
                    dec_next<T::K>(p, nx);
                    load_q(nx);
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        float x = l[nt][i];
                        x += __shfl_xor_sync(0xffffffffu, x, 4);
                        x += __shfl_xor_sync(0xffffffffu, x, 8);
                        x += __shfl_xor_sync(0xffffffffu, x, 16);
                        if (g == 0) wml[warp * T::ROWS + nt * 8 + 2 * t + i] = make_float2(m[nt][i], x);
                    }
                __syncthreads();
                constexpr int PT = 8 * DP / 4 / T::THREADS;      // float4 items of an 8-row block per thread
                float4 keep[NT * PT];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float f[2];
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        float M = -INFINITY;
#pragma unroll
                        for (int w = 0; w < DEC_TC_WARPS; w++) M = fmaxf(M, wml[w * T::ROWS + nt * 8 + 2 * t + i].x);
                        f[i] = exp2f(m[nt][i] - (M == -INFINITY ? 0.0f : M));
                    }
                    if (nt) __syncthreads();
                    // the upper two warps' go to the lower two, whose sums then meet
                    float *mb = merge + (warp & 1) * (8 * T::QS);
#pragma unroll
                    for (int up = 1; up >= 0; up--) {
                        if (warp >> 1 == up) {
#pragma unroll
                            for (int i = 0; i < DP / 16; i++)
#pragma unroll
                                for (int j = 0; j < 4; j++) {
                                    float *a = mb + (2 * t + (j & 1)) * T::QS + i * 16 + g + (j >> 1) * 8;
                                    *a = up ? o[i][nt][j] * f[j & 1] : o[i][nt][j] * f[j & 1] + *a;
                                }
                        }
                        __syncthreads();
                    }
#pragma unroll
                    for (int k = 0; k < PT; k++) {
                        const int it = threadIdx.x + k * T::THREADS, r = it / (DP / 4), d0 = (it % (DP / 4)) * 4;
                        const float4 a = *reinterpret_cast<const float4 *>(merge + r * T::QS + d0);
                        const float4 v = *reinterpret_cast<const float4 *>(merge + 8 * T::QS + r * T::QS + d0);
                        keep[nt * PT + k] = make_float4(a.x + v.x, a.y + v.y, a.z + v.z, a.w + v.w);
                    }
                }
                auto ml = [&](int r) {
                    float M = -INFINITY, L = 0.0f;
#pragma unroll
                    for (int w = 0; w < DEC_TC_WARPS; w++) M = fmaxf(M, wml[w * T::ROWS + r].x);
#pragma unroll
                    for (int w = 0; w < DEC_TC_WARPS; w++) {
                        const float2 x = wml[w * T::ROWS + r];
                        L += x.y * exp2f(x.x - (M == -INFINITY ? 0.0f : M));
                    }
                    return make_float2(M, L);
                };
                dec_finish<DP, T::ROWS, T::THREADS>(p, S, cu, c, upb, [&](int, int, int k) { return keep[k]; }, ml);
                __syncthreads();                             // wml and merge are free again
                fresh = true;
            }
            dec_next<T::K>(p, cu);
            c = cnext;
        }
        cp_wait<0>();
        dec_join<DP, T::ROWS, T::THREADS>(p, S, wml);
    }
    dec_empty(p);
}

// ---- f32, and rows that cannot be moved 16 bytes at a time: FP32 units ----
// The same cut of the work with 16 warps of 8 keys (8 warps at head size 256), a tile each: the warps
// cover each other's waits (8 warps with two tiles each took 181 us against 131 for six sequences
// of 30k tokens, 4 f32 heads of 128, 737 MB: 5.6 TB/s). A warp's four lanes per key each take every fourth 16
// bytes of the key's row for all query rows (the rows sit in shared memory and are broadcast),
// then every lane owns DP/32 dims of the accumulators and reads the values' rows across. f32
// products and sums throughout; with 8 rows a unit they bound it (221 us there), and so they do at head size 64
// (179 us for the same bytes). At 512 threads a thread has 128 registers, of which some are spilled (152 to
// 352 bytes a thread, most with 8 rows at 128).

template <int DP, int ROWS, int ST>
struct DecSt {
    static constexpr int NW = IRX_DEC_ST_NW(DP), THREADS = NW * 32, K = NW * 8, KS = DP + 16;
    static constexpr int TILE = 8 * (KS + DP) * 4;
    static constexpr int RING = NW * ST * TILE;
    static constexpr int MERGE = NW * ROWS * DP * 4;
    static constexpr int Q = ROWS * DP * 4;
    static constexpr int PB = NW * ROWS * 8 * 4;
    static constexpr int ML = NW * ROWS * 8;
    static constexpr int SMEM = RING + MERGE + Q + PB + ML + IRX_DEC_SHARE + NW * ST * (int)sizeof(DecRows<8>);
    static_assert(SMEM == IRX_DEC_ST_SMEM(DP, ROWS, ST), "the launcher's shared memory size");
};

template <int DP, int ROWS, int ST>
__device__ __forceinline__ void dec_st_body(const irx_kdec_t &p)
{
    using T = DecSt<DP, ROWS, ST>;
    constexpr int EX = 1;
    extern __shared__ __align__(128) unsigned char sm[];
    float *merge = reinterpret_cast<float *>(sm + T::RING);
    float *qs = merge + T::MERGE / 4;
    float *pball = qs + T::Q / 4;
    float2 *wml = reinterpret_cast<float2 *>(pball + T::PB / 4);
    DecShare &S = *reinterpret_cast<DecShare *>(reinterpret_cast<float *>(wml) + T::ML / 4);
    DecRows<8> *rows = reinterpret_cast<DecRows<8> *>(reinterpret_cast<float *>(wml) + (T::ML + IRX_DEC_SHARE) / 4) + (threadIdx.x >> 5) * ST;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, key = lane >> 2, quarter = lane & 3;
    const int upb = (p.h1 - p.h0) * p.split;
    constexpr int VW = DP / 32 < 4 ? DP / 32 : 4, NJ = DP / 32 / VW;

    irx_pdl_enter();
    dec_partition<T::THREADS, T::K, EX>(p, upb, S);
    if (S.c0 < S.c1) {
        DecCur tl, cu;
        const long long cfirst = dec_start<T::K, EX>(p, S, tl);
        cu = tl;
        float *myring = reinterpret_cast<float *>(sm) + warp * (ST * T::TILE / 4);
        float *pb = pball + warp * (ROWS * 8);
        long long tc = cfirst;
        auto lookup = [&](int st) {
            dec_lookup<8>(p, tl, tc < S.c1, dec_pos<T::K>(tl, tl.j) + warp * 8, rows[st]);
            if (tc < S.c1) {
                tc = dec_step<EX>(tl, tc);
                dec_next<T::K>(p, tl);
            }
        };
        auto fetch = [&](int st) {
            const long long off = dec_row<8>(p, rows[st], lane & 7);
            if (__any_sync(0xffffffffu, off != -1)) {
                float *kd = myring + st * (T::TILE / 4), *vd = kd + 8 * T::KS;
                const unsigned bad = __ballot_sync(0xffffffffu, off == -2);
                if (lane == 0) rows[st].bad = bad;
                if (p.vec) {
                    constexpr int CPR = DP / 4;              // 16-byte pieces of a row
#pragma unroll
                    for (int i = 0; i < 8 * CPR / 32; i++) {
                        const int it = i * 32 + lane, row = it / CPR, ch = it % CPR;
                        const long long o = __shfl_sync(0xffffffffu, off, row);
                        const bool in = o >= 0 && ch * 4 < p.d;
                        const int64_t e = in ? o + ch * 4 : 0;
                        cp16(irx_smem_u32(kd + row * T::KS + ch * 4), reinterpret_cast<const float *>(p.k) + e, in ? 16 : 0);
                        cp16(irx_smem_u32(vd + row * DP + ch * 4), reinterpret_cast<const float *>(p.v) + e, in ? 16 : 0);
                    }
                } else {
                    for (int it = lane; it < 8 * DP; it += 32) {
                        const int row = it / DP, d = it % DP;
                        const long long o = __shfl_sync(0xffffffffu, off, row);
                        const bool in = o >= 0 && d < p.d;
                        kd[row * T::KS + d] = in ? irx_ld1(p.k, p.dt, o + d) : 0.0f;
                        vd[row * DP + d] = in ? irx_ld1(p.v, p.dt, o + d) : 0.0f;
                    }
                }
            }
            __syncwarp();
            lookup(st);
            cp_commit();
        };
        for (int s = 0; s < ST; s++) lookup(s);
        cp_commit();
        cp_wait<0>();
        __syncwarp();
        for (int s = 0; s < ST; s++) fetch(s);

        float o[ROWS][NJ * VW], m[ROWS], l[ROWS];
        int st = 0, live = 0;
        bool fresh = true;
        for (long long c = cfirst; c < S.c1;) {
            if (fresh) {
                const int hk = p.h0 + cu.h, rb = cu.rb;
                live = min(ROWS, p.group - rb * ROWS);
                for (int i = threadIdx.x; i < ROWS * DP; i += T::THREADS) {
                    const int r = i / DP, d = i % DP;
                    qs[i] = r < live && d < p.d
                          ? irx_ld1(p.q, p.dt, (int64_t)cu.b * p.q_stride + (int64_t)(hk * p.group + rb * ROWS + r) * p.d + d) : 0.0f;
                }
#pragma unroll
                for (int r = 0; r < ROWS; r++) {
                    m[r] = -INFINITY;
                    l[r] = 0.0f;
#pragma unroll
                    for (int j = 0; j < NJ * VW; j++) o[r][j] = 0.0f;
                }
                fresh = false;
                __syncthreads();
            }
            cp_wait<ST - 1>();
            __syncwarp();
            const int pos = dec_pos<T::K>(cu, cu.j) + warp * 8;
            if (dec_any(cu, pos, 8)) {
                const bool in = dec_sees(cu, pos + key) && !(rows[st].bad >> key & 1);
                const float *kt = myring + st * (T::TILE / 4), *vt = kt + 8 * T::KS;
                float s[ROWS];
#pragma unroll
                for (int r = 0; r < ROWS; r++) s[r] = 0.0f;
#pragma unroll (ROWS / 4)
                for (int i = 0; i < DP / 16; i++) {
                    const float4 k4 = *reinterpret_cast<const float4 *>(kt + key * T::KS + (4 * i + quarter) * 4);
#pragma unroll
                    for (int r = 0; r < ROWS; r++) {
                        const float4 q4 = *reinterpret_cast<const float4 *>(qs + r * DP + (4 * i + quarter) * 4);
                        s[r] = fmaf(q4.x, k4.x, s[r]);
                        s[r] = fmaf(q4.y, k4.y, s[r]);
                        s[r] = fmaf(q4.z, k4.z, s[r]);
                        s[r] = fmaf(q4.w, k4.w, s[r]);
                    }
                }
#pragma unroll
                for (int r = 0; r < ROWS; r++) {
                    float x = s[r];
                    x += __shfl_xor_sync(0xffffffffu, x, 1);
                    x += __shfl_xor_sync(0xffffffffu, x, 2);
                    x = in ? x * p.scale2 : -INFINITY;
                    float mx = x;
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    const float mn = fmaxf(m[r], mx), base = mn == -INFINITY ? 0.0f : mn;
                    const float e = exp2f(x - base);
                    if (mn > m[r]) {
                        const float al = exp2f(m[r] - base);
                        l[r] *= al;
#pragma unroll
                        for (int j = 0; j < NJ * VW; j++) o[r][j] *= al;
                        m[r] = mn;
                    }
                    l[r] += e;
                    if (quarter == 0) pb[r * 8 + key] = e;
                }
                __syncwarp();
#pragma unroll
                for (int kk = 0; kk < 8; kk += 4) {
                    float v[4][NJ * VW];
#pragma unroll
                    for (int k = 0; k < 4; k++)
#pragma unroll
                        for (int j = 0; j < NJ; j++) {
                            const float *a = vt + (kk + k) * DP + j * 128 + lane * VW;
                            if constexpr (VW == 4) {
                                const float4 x = *reinterpret_cast<const float4 *>(a);
                                v[k][j * 4] = x.x; v[k][j * 4 + 1] = x.y; v[k][j * 4 + 2] = x.z; v[k][j * 4 + 3] = x.w;
                            } else {
                                const float2 x = *reinterpret_cast<const float2 *>(a);
                                v[k][0] = x.x; v[k][1] = x.y;
                            }
                        }
#pragma unroll
                    for (int r = 0; r < ROWS; r++) {
                        const float4 e = *reinterpret_cast<const float4 *>(pb + r * 8 + kk);
#pragma unroll
                        for (int j = 0; j < NJ * VW; j++) {
                            o[r][j] = fmaf(e.x, v[0][j], o[r][j]);
                            o[r][j] = fmaf(e.y, v[1][j], o[r][j]);
                            o[r][j] = fmaf(e.z, v[2][j], o[r][j]);
                            o[r][j] = fmaf(e.w, v[3][j], o[r][j]);
                        }
                    }
                }
            }
            __syncwarp();
            fetch(st);
            if (++st == ST) st = 0;
            const long long cnext = dec_step<EX>(cu, c);
            if (cu.j + 1 == cu.nch || cnext >= S.c1) {
#pragma unroll
                for (int r = 0; r < ROWS; r++) {
                    float x = l[r];
                    x += __shfl_xor_sync(0xffffffffu, x, 4);
                    x += __shfl_xor_sync(0xffffffffu, x, 8);
                    x += __shfl_xor_sync(0xffffffffu, x, 16);
                    if (lane == 0) wml[warp * ROWS + r] = make_float2(m[r], x);
                }
                __syncthreads();
#pragma unroll
                for (int r = 0; r < ROWS; r++) {
                    float M = -INFINITY;
#pragma unroll
                    for (int w = 0; w < T::NW; w++) M = fmaxf(M, wml[w * ROWS + r].x);
                    const float f = exp2f(m[r] - (M == -INFINITY ? 0.0f : M));
#pragma unroll
                    for (int j = 0; j < NJ * VW; j++)
                        merge[(warp * ROWS + r) * DP + (j / VW) * 128 + lane * VW + j % VW] = o[r][j] * f;
                }
                __syncthreads();
                for (int it = threadIdx.x; it < ROWS * DP; it += T::THREADS) {
                    float a = 0.0f;
#pragma unroll
                    for (int w = 0; w < T::NW; w++) a += merge[w * ROWS * DP + it];
                    qs[it] = a;                                  // the query rows are done with
                }
                __syncthreads();
                auto ml = [&](int r) {
                    float M = -INFINITY, L = 0.0f;
#pragma unroll
                    for (int w = 0; w < T::NW; w++) M = fmaxf(M, wml[w * ROWS + r].x);
#pragma unroll
                    for (int w = 0; w < T::NW; w++) {
                        const float2 x = wml[w * ROWS + r];
                        L += x.y * exp2f(x.x - (M == -INFINITY ? 0.0f : M));
                    }
                    return make_float2(M, L);
                };
                auto acc = [&](int r, int d0, int) { return *reinterpret_cast<const float4 *>(qs + r * DP + d0); };
                dec_finish<DP, ROWS, T::THREADS>(p, S, cu, c, upb, acc, ml);
                __syncthreads();
                fresh = true;
            }
            dec_next<T::K>(p, cu);
            c = cnext;
        }
        cp_wait<0>();
        dec_join<DP, ROWS, T::THREADS>(p, S, wml);
    }
    dec_empty(p);
}

#define DEC_TC(DP, NT) \
    extern "C" __global__ void __launch_bounds__(DEC_TC_WARPS * 32) irx_dec_tc_##DP##_##NT(const __grid_constant__ irx_kdec_t p) \
    { dec_tc_body<DP, NT, IRX_DEC_TC_KM(DP), IRX_DEC_TC_ST(DP, NT)>(p); }
#define DEC_STK(DP, ROWS) \
    extern "C" __global__ void __launch_bounds__(IRX_DEC_ST_NW(DP) * 32) irx_dec_st_##DP##_##ROWS(const __grid_constant__ irx_kdec_t p) \
    { dec_st_body<DP, ROWS, 1>(p); }

DEC_TC(64, 1) DEC_TC(64, 2) DEC_TC(128, 1) DEC_TC(128, 2) DEC_TC(256, 1)
DEC_STK(64, 4) DEC_STK(64, 8) DEC_STK(128, 4) DEC_STK(128, 8) DEC_STK(256, 4) DEC_STK(256, 8)
