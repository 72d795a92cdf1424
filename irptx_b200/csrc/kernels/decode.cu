// decode.cu -- attention of one new token per sequence over a paged key-value cache.
//
// For a sequence b of n tokens, its newest token's query head h sees the keys
//     j in [0, min(sinks, n - window)) and [n - window, n)      (every j < n without a window)
// of key-value head h / group:  o = sum_j softmax_j(scale * q.k_j) v_j, zeros when n = 0, and
// lse = ln sum_j exp(scale * q.k_j) (-inf when n = 0).
//
// Bound: every visible key and value row is read once and takes 4 * group operations per
// element, so HBM bounds it (group operations a byte in bf16). The work is therefore cut by
// keys, not by rows: the visible keys of all (sequence, kv head, row block) units are laid end to
// end in chunks of IRX_DEC_KEYS keys and the chunks are dealt out evenly, a contiguous range to
// each block of one resident wave, whatever the lengths are. A block whose range covers a whole
// unit writes its output; a unit that several blocks share is joined by the last of them to
// arrive, which folds the blocks' partials in key order, so the result does not depend on which
// block that was. Past DEC_JOIN partials they are folded in groups first, by the last block of
// each group, so a single long sequence's join is not one block's work.
#pragma once
#include "tc.cuh"
#include "kvpages.cu"

#define DEC_JOIN 16

struct DecCur {                       // a place in the laid-out chunks: chunk j of unit u of sequence b
    int b, u, j, nch, nvis, lo, sk;   // of sequence b: chunks, visible keys, window start, sinks before it
};

__device__ __forceinline__ int dec_len(const irx_kdec_t &p, int b)
{
    const int n = p.lens[b];
    const int64_t cap = (int64_t)p.cols * p.page_size;
    return n < 0 ? 0 : (int64_t)n > cap ? (int)cap : n;
}

__device__ __forceinline__ int dec_vis(const irx_kdec_t &p, int n, int &lo, int &sk)
{
    lo = sk = 0;
    if (p.window > 0 && n > p.window) {
        lo = n - p.window;
        sk = p.sinks < lo ? p.sinks : lo;
        return sk + p.window;
    }
    return n;
}

__device__ __forceinline__ int dec_chunks(int nvis) { return (nvis + IRX_DEC_KEYS - 1) / IRX_DEC_KEYS; }

__device__ __forceinline__ void dec_enter(const irx_kdec_t &p, DecCur &c)      // sequence c.b's numbers
{
    c.nvis = dec_vis(p, dec_len(p, c.b), c.lo, c.sk);
    c.nch = dec_chunks(c.nvis);
}

__device__ __forceinline__ void dec_next(const irx_kdec_t &p, DecCur &c, int upb)
{
    if (++c.j < c.nch) return;
    c.j = 0;
    if (++c.u < upb) return;
    c.u = 0;
    do {
        if (++c.b >= p.batch) { c.nvis = c.lo = c.sk = 0; c.nch = 0x7fffffff; return; }   // past the end
        dec_enter(p, c);
    } while (c.nch == 0);
}

struct DecShare {
    long long c0, c1, total;          // this block's chunks and all chunks
    long long wsum[8];                // a warp each
    int geff, b, u, j, last;
    unsigned arrived;
};

// The block's chunk range and where it starts: every block sums the chunks of all sequences (a
// segment of them per thread, then a scan), so nothing has to run before the kernel.
template <int THREADS>
__device__ __forceinline__ void dec_partition(const irx_kdec_t &p, int upb, DecShare &S)
{
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = THREADS / 32;
    const int seg = (p.batch + THREADS - 1) / THREADS, b0 = tid * seg, b1 = min(p.batch, b0 + seg);
    long long sum = 0;
    for (int b = b0; b < b1; b++) {
        int lo, sk;
        const int raw = p.lens[b], n = dec_len(p, b);
        if (raw != n && blockIdx.x == 0) irx_flag(p.err, IRX_KERR_INDEX);
        sum += dec_chunks(dec_vis(p, n, lo, sk));
    }
    long long inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) S.wsum[warp] = inc;
    __syncthreads();
    if (tid == 0) {
        long long a = 0;
        for (int w = 0; w < nw; w++) { const long long v = S.wsum[w]; S.wsum[w] = a; a += v; }
        S.total = a * upb;
        S.geff = (int)min((long long)gridDim.x, S.total);
        S.c0 = S.c1 = 0;
        if ((int)blockIdx.x < S.geff) {
            S.c0 = blockIdx.x * S.total / S.geff;
            S.c1 = (blockIdx.x + 1) * S.total / S.geff;
        }
    }
    __syncthreads();
    if (S.c0 == S.c1) return;
    const long long ex = (S.wsum[warp] + inc - sum) * upb;
    if (S.c0 >= ex && S.c0 < ex + sum * upb) {           // exactly one thread's segment holds c0
        long long r = S.c0 - ex;
        for (int b = b0; b < b1; b++) {
            int lo, sk;
            const long long nch = dec_chunks(dec_vis(p, dec_len(p, b), lo, sk));
            if (r < nch * upb) { S.b = b; S.u = (int)(r / nch); S.j = (int)(r % nch); break; }
            r -= nch * upb;
        }
    }
    __syncthreads();
}

// The block that holds chunk c (block i starts at floor(i * total / geff)).
__device__ __forceinline__ int dec_block_of(const DecShare &S, long long c) { return (int)(((c + 1) * S.geff - 1) / S.total); }

// Byte-free part of a tile's addressing: the element offset of visible key jj of sequence b, kv head
// hk, given its page; -1 when there is none.
__device__ __forceinline__ int dec_pos(const DecCur &c, int jj) { return jj < c.sk ? jj : jj - c.sk + c.lo; }

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

// Fold `cnt` partials, slot(i) = i ? s0 + i * step + adj : s_first, in order, by the whole block. With
// `final` the result is the unit's output, else it becomes the partial of the first slot.
// `sw` holds cnt x ROWS weights and ROWS (max, sum) pairs.
template <int DP, int ROWS, int THREADS>
__device__ __forceinline__ void dec_fold(const irx_kdec_t &p, int first, int rest0, int step, int cnt, bool fin, int b,
                                         int head0, int live, float *sw)
{
    const int tid = threadIdx.x;
    float *mx = sw + cnt * ROWS;
    __syncthreads();
    for (int i = tid; i < cnt * ROWS; i += THREADS) {
        const int k = i / ROWS, r = i % ROWS;
        const int s = k ? rest0 + k * step : first;
        sw[i] = __ldcg(dec_slot(p, s, ROWS, DP) + ROWS * DP + 2 * r);
    }
    __syncthreads();
    if (tid < ROWS) {
        float m = -INFINITY, l = 0.0f;
        for (int k = 0; k < cnt; k++) m = fmaxf(m, sw[k * ROWS + tid]);
        const float base = m == -INFINITY ? 0.0f : m;
        for (int k = 0; k < cnt; k++) {
            const int s = k ? rest0 + k * step : first;
            const float f = exp2f(sw[k * ROWS + tid] - base);
            sw[k * ROWS + tid] = f;
            l += f * __ldcg(dec_slot(p, s, ROWS, DP) + ROWS * DP + 2 * tid + 1);
        }
        mx[2 * tid] = m;
        mx[2 * tid + 1] = l;
    }
    __syncthreads();
    for (int it = tid; it < ROWS * DP / 4; it += THREADS) {
        const int r = it / (DP / 4), d0 = (it % (DP / 4)) * 4;
        if (r >= live || d0 >= p.d) continue;
        float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int k0 = 0; k0 < cnt; k0 += 8) {
            float4 v[8];
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (k0 + k < cnt) {
                    const int s = k0 + k ? rest0 + (k0 + k) * step : first;
                    v[k] = __ldcg(reinterpret_cast<const float4 *>(dec_slot(p, s, ROWS, DP) + r * DP + d0));
                }
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (k0 + k < cnt) {
                    const float f = sw[(k0 + k) * ROWS + r];
                    a.x += f * v[k].x; a.y += f * v[k].y; a.z += f * v[k].z; a.w += f * v[k].w;
                }
        }
        if (fin) {
            const float l = mx[2 * r + 1];
            dec_store_out(p, b, head0 + r, d0, make_float4(a.x / l, a.y / l, a.z / l, a.w / l));
            if (p.lse && d0 == 0)
                p.lse[(int64_t)b * p.heads + head0 + r] = (mx[2 * r] + log2f(l)) * 0.6931471805599453f;
        } else {
            *reinterpret_cast<float4 *>(dec_slot(p, first, ROWS, DP) + r * DP + d0) = a;
        }
    }
    if (!fin && tid < ROWS) {
        float *ml = dec_slot(p, first, ROWS, DP) + ROWS * DP + 2 * tid;
        ml[0] = mx[2 * tid];
        ml[1] = mx[2 * tid + 1];
    }
}

// One arrival on a counter: true in every thread of the last of `want` blocks to arrive, which
// leaves the counter at zero and sees what the others wrote before they arrived.
__device__ __forceinline__ bool dec_arrive(unsigned *ctr, unsigned want, DecShare &S)
{
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        const unsigned a = atomicAdd(ctr, 1u);
        S.last = a == want - 1;
        if (S.last) *ctr = 0;
    }
    __syncthreads();
    if (!S.last) return false;
    __threadfence();
    return true;
}

// A unit's share of this block is done. `acc(r, d0, k)` gives the block's four accumulators of row r
// from d0 (item k of this thread), `ml(r)` its (max, sum). Chunk c is the share's last one.
template <int DP, int ROWS, int THREADS, class Acc, class Ml>
__device__ __forceinline__ void dec_finish(const irx_kdec_t &p, DecShare &S, const DecCur &cur, long long c, int upb,
                                           float *sw, Acc acc, Ml ml)
{
    const int tid = threadIdx.x;
    const int hk = p.h0 + cur.u / p.split, rb = cur.u % p.split;
    const int head0 = hk * p.group + rb * ROWS, live = min(ROWS, p.group - rb * ROWS);
    const long long ua = c - cur.j, ub = ua + cur.nch;       // the unit's chunks
    const bool alone = ua >= S.c0 && ub <= S.c1;
    const int slot = 2 * (int)blockIdx.x + (ua >= S.c0 ? 1 : 0);
#pragma unroll
    for (int k = 0; k < (ROWS * DP / 4 + THREADS - 1) / THREADS; k++) {
        const int it = tid + k * THREADS, r = it / (DP / 4), d0 = (it % (DP / 4)) * 4;
        if (r >= live || d0 >= p.d) continue;
        const float4 a = acc(r, d0, k);
        const float2 s = ml(r);
        if (alone) {
            dec_store_out(p, cur.b, head0 + r, d0, make_float4(a.x / s.y, a.y / s.y, a.z / s.y, a.w / s.y));
            if (p.lse && d0 == 0) p.lse[(int64_t)cur.b * p.heads + head0 + r] = (s.x + log2f(s.y)) * 0.6931471805599453f;
        } else {
            float *o = dec_slot(p, slot, ROWS, DP);
            __stcg(reinterpret_cast<float4 *>(o + r * DP + d0), a);
            if (d0 == 0) __stcg(reinterpret_cast<float2 *>(o + ROWS * DP + 2 * r), s);
        }
    }
    if (alone) return;
    const int first = dec_block_of(S, ua), pieces = dec_block_of(S, ub - 1) - first + 1;
    const int64_t unit = (int64_t)cur.b * upb + cur.u;
    if (pieces <= DEC_JOIN) {
        if (dec_arrive(p.ticket + unit, (unsigned)pieces, S))
            dec_fold<DP, ROWS, THREADS>(p, 2 * first + 1, 2 * first, 2, pieces, true, cur.b, head0, live, sw);
        return;
    }
    // partials fold in groups of DEC_JOIN, each into its first slot, and the groups' folds into the output
    const int g = ((int)blockIdx.x - first) / DEC_JOIN, ng = (pieces + DEC_JOIN - 1) / DEC_JOIN;
    const int g0 = first + g * DEC_JOIN, gn = min(DEC_JOIN, pieces - g * DEC_JOIN);
    const int gslot = 2 * g0 + (g ? 0 : 1);
    if (!dec_arrive(p.gcount + gslot, (unsigned)gn, S)) return;
    dec_fold<DP, ROWS, THREADS>(p, gslot, 2 * g0, 2, gn, false, cur.b, head0, live, sw);
    if (!dec_arrive(p.ticket + unit, (unsigned)ng, S)) return;
    dec_fold<DP, ROWS, THREADS>(p, 2 * first + 1, 2 * first, 2 * DEC_JOIN, ng, true, cur.b, head0, live, sw);
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

// The page of the key `jj` (visible index) of the cursor's sequence, or -1 (flagged) when the table
// holds no page of the pool there.
__device__ __forceinline__ int dec_page(const irx_kdec_t &p, const DecCur &c, int jj, unsigned &slot)
{
    const unsigned pos = (unsigned)dec_pos(c, jj), pi = pos / (unsigned)p.page_size;
    slot = pos - pi * (unsigned)p.page_size;
    const int page = p.table[(int64_t)c.b * p.cols + pi];
    return page < 0 ? -1 : page;
}

__device__ __forceinline__ int64_t dec_offset(const irx_kdec_t &p, int page, unsigned slot, int hk)
{
    if (page < 0 || page >= p.pages) {
        irx_flag(p.err, IRX_KERR_INDEX);
        return -1;
    }
    return (int64_t)page * p.page_stride + (int64_t)slot * p.token_stride + (int64_t)hk * p.head_stride;
}

// ---- bf16: matrix instructions ----
// The transposed products: S^T[16 keys x 8 rows] = K Q^T and O^T[16 dims x 8 rows] += V^T P^T, so that
// the few query rows sit on the instruction's narrow side (8) and keys or dims on its wide one.
// S^T's accumulators become P^T's operand by an 8x8 transpose across the warp. Each warp
// owns 16 keys of a chunk and its own ring of ST tiles filled by 16-byte asynchronous copies, so
// warps meet only where a unit ends. mma.sync runs far below tcgen05's rate, but at 8 to 16 rows
// the products take 16 to 32 instructions per 8 KB (D = 128), which HBM delivers in about 360
// cycles per SM: the tensor pipe is idle most of the time and tcgen05's 128-row tiles would be
// filled with padding.
// P is rounded to bf16 for the product (as V is bf16), the sum of exps takes the same rounded
// values so that the weights still sum to one.

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

__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }

#define DEC_TC_WARPS 4

template <int DP, int NT, int ST>
struct DecTc {
    static constexpr int THREADS = DEC_TC_WARPS * 32, ROWS = 8 * NT, TILE = 16 * DP * 2, QS = DP + 4;
    // ring, then one 8-row block of the warps' accumulators (reused for a fold's weights), then
    // (max, sum) pairs and the share
    static constexpr int RING = DEC_TC_WARPS * ST * 2 * TILE;
    static constexpr int MERGE = DEC_TC_WARPS * 8 * QS * 4;
    static constexpr int ML = DEC_TC_WARPS * ROWS * 8;
    static constexpr int SMEM = RING + MERGE + ML + IRX_DEC_SHARE;
    static_assert(SMEM == IRX_DEC_TC_SMEM(DP, NT, ST), "the launcher's shared memory size");
    static_assert((IRX_DEC_MAX_CTAS / DEC_JOIN + 2) * ROWS * 4 <= MERGE && sizeof(DecShare) <= IRX_DEC_SHARE, "shared memory");
};

template <int DP, int NT, int ST>
__device__ __forceinline__ void dec_tc_body(const irx_kdec_t &p)
{
    using T = DecTc<DP, NT, ST>;
    extern __shared__ __align__(128) unsigned char sm[];
    unsigned char *ring = sm;
    float *merge = reinterpret_cast<float *>(sm + T::RING);
    float2 *wml = reinterpret_cast<float2 *>(sm + T::RING + T::MERGE);
    DecShare &S = *reinterpret_cast<DecShare *>(sm + T::RING + T::MERGE + T::ML);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int upb = (p.h1 - p.h0) * p.split;

    irx_pdl_enter();
    dec_partition<T::THREADS>(p, upb, S);
    if (S.c0 < S.c1) {
        DecCur ld, cu;
        ld.b = S.b; ld.u = S.u; ld.j = S.j;
        dec_enter(p, ld);
        cu = ld;
        const __nv_bfloat16 *kg = reinterpret_cast<const __nv_bfloat16 *>(p.k), *vg = reinterpret_cast<const __nv_bfloat16 *>(p.v);
        const uint32_t myring = irx_smem_u32(ring) + warp * (ST * 2 * T::TILE);
        constexpr int CPR = DP / 8, RPI = 32 / CPR, NI = 16 / RPI;
        const int lrow = lane / CPR, lch = lane % CPR;
        const bool cin = lch * 8 < p.d;
        long long lc = S.c0;                                 // the chunk that `ld` is at
        int pg = -1;
        unsigned slot = 0;
        // each lane looks up one key row's page a tile ahead of its use
        auto lookup = [&]() {
            const int jj = ld.j * IRX_DEC_KEYS + warp * 16 + (lane & 15);
            pg = -2;                                         // no such key
            if (lc < S.c1 && jj < ld.nvis) pg = dec_page(p, ld, jj, slot);
        };
        auto fetch = [&](int st) {
            if (lc < S.c1) {
                const int64_t off = pg == -2 ? -1 : dec_offset(p, pg, slot, p.h0 + ld.u / p.split);
                if (__any_sync(0xffffffffu, pg != -2)) {
                    const uint32_t kd = myring + st * (2 * T::TILE), vd = kd + T::TILE;
#pragma unroll
                    for (int i = 0; i < NI; i++) {
                        const int row = i * RPI + lrow;
                        const int64_t o = __shfl_sync(0xffffffffu, off, row);
                        const uint32_t d = row * (DP * 2) + ((lch ^ (row & 7)) << 4);
                        const int64_t e = o >= 0 && cin ? o + lch * 8 : 0;
                        const uint32_t nb = o >= 0 && cin ? 16 : 0;
                        cp16(kd + d, kg + e, nb);
                        cp16(vd + d, vg + e, nb);
                    }
                }
                lc++;
                dec_next(p, ld, upb);
                lookup();
            }
            cp_commit();
        };
        lookup();
        for (int s = 0; s < ST; s++) fetch(s);

        uint32_t q[DP / 16][NT][2];
        float o[DP / 16][NT][4], m[NT][2], l[NT][2];
        int st = 0;
        bool fresh = true;
        for (long long c = S.c0; c < S.c1; c++) {
            if (fresh) {                                     // a unit starts: its query rows, an empty state
                const int hk = p.h0 + cu.u / p.split, rb = cu.u % p.split;
                const __nv_bfloat16 *qg = reinterpret_cast<const __nv_bfloat16 *>(p.q) + (int64_t)cu.b * p.q_stride;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const int r = rb * T::ROWS + nt * 8 + g;
                    const __nv_bfloat16 *row = qg + (int64_t)(hk * p.group + r) * p.d;
#pragma unroll
                    for (int ks = 0; ks < DP / 16; ks++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int d0 = ks * 16 + h * 8 + 2 * t;
                            q[ks][nt][h] = r < p.group && d0 < p.d ? *reinterpret_cast<const uint32_t *>(row + d0) : 0u;
                        }
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
            const int nv = cu.nvis - (cu.j * IRX_DEC_KEYS + warp * 16);
            if (nv > 0) {
                const uint32_t kb = myring + st * (2 * T::TILE), vb = kb + T::TILE;
                float s[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
                {
                    const int row = (lane & 7) + ((lane >> 3) & 1) * 8, ch = lane >> 4;
#pragma unroll
                    for (int ks = 0; ks < DP / 16; ks++) {
                        uint32_t a[4];
                        ldsm4(a, kb + row * (DP * 2) + (((2 * ks + ch) ^ (row & 7)) << 4));
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) mma_16816(s[nt], a, q[ks][nt][0], q[ks][nt][1]);
                    }
                }
                uint32_t pb[NT][2];
                bool grew = false;
                float al[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int key = g + (i >> 1) * 8;
                        s[nt][i] = key < nv ? s[nt][i] * p.scale2 : -INFINITY;
                    }
                    float pr[4];
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        float x = fmaxf(s[nt][i], s[nt][i + 2]);
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                        const float mn = fmaxf(m[nt][i], x), base = mn == -INFINITY ? 0.0f : mn;
                        al[nt][i] = exp2f(m[nt][i] - base);
                        grew = grew || mn > m[nt][i];
                        m[nt][i] = mn;
                        pr[i] = __bfloat162float(__float2bfloat16_rn(exp2f(s[nt][i] - base)));
                        pr[i + 2] = __bfloat162float(__float2bfloat16_rn(exp2f(s[nt][i + 2] - base)));
                        l[nt][i] = l[nt][i] * al[nt][i] + (pr[i] + pr[i + 2]);
                    }
                    const __nv_bfloat162 p0 = __floats2bfloat162_rn(pr[0], pr[1]), p1 = __floats2bfloat162_rn(pr[2], pr[3]);
                    pb[nt][0] = trans8(*reinterpret_cast<const uint32_t *>(&p0));
                    pb[nt][1] = trans8(*reinterpret_cast<const uint32_t *>(&p1));
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
                    for (int i = 0; i < DP / 16; i++) {
                        uint32_t a[4];
                        ldsm4t(a, vb + row * (DP * 2) + (((2 * i + ch) ^ (row & 7)) << 4));
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) mma_16816(o[i][nt], a, pb[nt][0], pb[nt][1]);
                    }
                }
            }
            __syncwarp();
            fetch(st);
            if (++st == ST) st = 0;
            if (cu.j + 1 == cu.nch || c + 1 == S.c1) {
                // the unit's share ends: the warps' states meet in shared memory, one 8-row block at a time
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
                    float *mb = merge + warp * (8 * T::QS);
#pragma unroll
                    for (int i = 0; i < DP / 16; i++)
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            mb[(2 * t + (j & 1)) * T::QS + i * 16 + g + (j >> 1) * 8] = o[i][nt][j] * f[j & 1];
                    __syncthreads();
#pragma unroll
                    for (int k = 0; k < PT; k++) {
                        const int it = threadIdx.x + k * T::THREADS, r = it / (DP / 4), d0 = (it % (DP / 4)) * 4;
                        float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                        for (int w = 0; w < DEC_TC_WARPS; w++) {
                            const float4 v = *reinterpret_cast<const float4 *>(merge + w * (8 * T::QS) + r * T::QS + d0);
                            a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
                        }
                        keep[nt * PT + k] = a;
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
                dec_finish<DP, T::ROWS, T::THREADS>(p, S, cu, c, upb, merge, [&](int, int, int k) { return keep[k]; }, ml);
                __syncthreads();                             // wml and merge are free again
                fresh = true;
            }
            dec_next(p, cu, upb);
        }
        cp_wait<0>();
    }
    dec_empty(p);
}

// ---- f32, and rows that cannot be moved 16 bytes at a time: FP32 units ----
// The same cut of the work with 8 warps of 8 keys. A warp's four lanes per key each take every
// fourth 16 bytes of the key's row for all query rows (the rows sit in shared memory and are
// broadcast), then every lane owns DP/32 dims of the accumulators and reads the values' rows
// across. f32 products and sums throughout.
#define DEC_ST_WARPS 8

template <int DP, int NT, int ST>
struct DecSt {
    static constexpr int THREADS = DEC_ST_WARPS * 32, ROWS = 8 * NT, KS = DP + 16;
    static constexpr int TILE = 8 * (KS + DP) * 4;
    static constexpr int RING = DEC_ST_WARPS * ST * TILE;
    static constexpr int MERGE = DEC_ST_WARPS * 8 * DP * 4;
    static constexpr int Q = ROWS * DP * 4;
    static constexpr int PB = DEC_ST_WARPS * ROWS * 8 * 4;
    static constexpr int ML = DEC_ST_WARPS * ROWS * 8;
    static constexpr int SMEM = RING + MERGE + Q + PB + ML + IRX_DEC_SHARE;
    static_assert(SMEM == IRX_DEC_ST_SMEM(DP, NT, ST), "the launcher's shared memory size");
    static_assert((IRX_DEC_MAX_CTAS / DEC_JOIN + 2) * ROWS * 4 <= MERGE, "shared memory");
};

template <int DP, int NT, int ST>
__device__ __forceinline__ void dec_st_body(const irx_kdec_t &p)
{
    using T = DecSt<DP, NT, ST>;
    extern __shared__ __align__(128) unsigned char sm[];
    float *merge = reinterpret_cast<float *>(sm + T::RING);
    float *qs = merge + T::MERGE / 4;
    float *pball = qs + T::Q / 4;
    float2 *wml = reinterpret_cast<float2 *>(pball + T::PB / 4);
    DecShare &S = *reinterpret_cast<DecShare *>(reinterpret_cast<float *>(wml) + T::ML / 4);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, key = lane >> 2, quarter = lane & 3;
    const int upb = (p.h1 - p.h0) * p.split;
    constexpr int VW = DP / 32 < 4 ? DP / 32 : 4, NJ = DP / 32 / VW;

    irx_pdl_enter();
    dec_partition<T::THREADS>(p, upb, S);
    if (S.c0 < S.c1) {
        DecCur ld, cu;
        ld.b = S.b; ld.u = S.u; ld.j = S.j;
        dec_enter(p, ld);
        cu = ld;
        float *myring = reinterpret_cast<float *>(sm) + warp * (ST * T::TILE / 4);
        float *pb = pball + warp * (T::ROWS * 8);
        long long lc = S.c0;
        int pg = -1;
        unsigned slot = 0;
        auto lookup = [&]() {
            const int jj = ld.j * IRX_DEC_KEYS + warp * 8 + (lane & 7);
            pg = -2;
            if (lc < S.c1 && jj < ld.nvis) pg = dec_page(p, ld, jj, slot);
        };
        auto fetch = [&](int st) {
            if (lc < S.c1) {
                const int64_t off = pg == -2 ? -1 : dec_offset(p, pg, slot, p.h0 + ld.u / p.split);
                if (__any_sync(0xffffffffu, pg != -2)) {
                    float *kd = myring + st * (T::TILE / 4), *vd = kd + 8 * T::KS;
                    if (p.vec) {
                        constexpr int CPR = DP / 4;              // 16-byte pieces of a row
#pragma unroll
                        for (int i = 0; i < 8 * CPR / 32; i++) {
                            const int it = i * 32 + lane, row = it / CPR, ch = it % CPR;
                            const int64_t o = __shfl_sync(0xffffffffu, off, row);
                            const bool in = o >= 0 && ch * 4 < p.d;
                            const int64_t e = in ? o + ch * 4 : 0;
                            cp16(irx_smem_u32(kd + row * T::KS + ch * 4), reinterpret_cast<const float *>(p.k) + e, in ? 16 : 0);
                            cp16(irx_smem_u32(vd + row * DP + ch * 4), reinterpret_cast<const float *>(p.v) + e, in ? 16 : 0);
                        }
                    } else {
                        for (int it = lane; it < 8 * DP; it += 32) {
                            const int row = it / DP, d = it % DP;
                            const int64_t o = __shfl_sync(0xffffffffu, off, row);
                            const bool in = o >= 0 && d < p.d;
                            kd[row * T::KS + d] = in ? irx_ld1(p.k, p.dt, o + d) : 0.0f;
                            vd[row * DP + d] = in ? irx_ld1(p.v, p.dt, o + d) : 0.0f;
                        }
                    }
                }
                lc++;
                dec_next(p, ld, upb);
                lookup();
            }
            cp_commit();
        };
        lookup();
        for (int s = 0; s < ST; s++) fetch(s);

        float o[T::ROWS][NJ * VW], m[T::ROWS], l[T::ROWS];
        int st = 0, live = 0;
        bool fresh = true;
        for (long long c = S.c0; c < S.c1; c++) {
            if (fresh) {
                const int hk = p.h0 + cu.u / p.split, rb = cu.u % p.split;
                live = min(T::ROWS, p.group - rb * T::ROWS);
                for (int i = threadIdx.x; i < T::ROWS * DP; i += T::THREADS) {
                    const int r = i / DP, d = i % DP;
                    qs[i] = r < live && d < p.d
                          ? irx_ld1(p.q, p.dt, (int64_t)cu.b * p.q_stride + (int64_t)(hk * p.group + rb * T::ROWS + r) * p.d + d) : 0.0f;
                }
#pragma unroll
                for (int r = 0; r < T::ROWS; r++) {
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
            const int nv = cu.nvis - (cu.j * IRX_DEC_KEYS + warp * 8);
            if (nv > 0) {
                const float *kt = myring + st * (T::TILE / 4), *vt = kt + 8 * T::KS;
                float s[T::ROWS];
#pragma unroll
                for (int r = 0; r < T::ROWS; r++) s[r] = 0.0f;
#pragma unroll 4
                for (int i = 0; i < DP / 16; i++) {
                    const float4 k4 = *reinterpret_cast<const float4 *>(kt + key * T::KS + (4 * i + quarter) * 4);
#pragma unroll
                    for (int r = 0; r < T::ROWS; r++) {
                        const float4 q4 = *reinterpret_cast<const float4 *>(qs + r * DP + (4 * i + quarter) * 4);
                        s[r] = fmaf(q4.x, k4.x, s[r]);
                        s[r] = fmaf(q4.y, k4.y, s[r]);
                        s[r] = fmaf(q4.z, k4.z, s[r]);
                        s[r] = fmaf(q4.w, k4.w, s[r]);
                    }
                }
#pragma unroll
                for (int r = 0; r < T::ROWS; r++) {
                    float x = s[r];
                    x += __shfl_xor_sync(0xffffffffu, x, 1);
                    x += __shfl_xor_sync(0xffffffffu, x, 2);
                    x = key < nv ? x * p.scale2 : -INFINITY;
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
                    for (int r = 0; r < T::ROWS; r++) {
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
            if (cu.j + 1 == cu.nch || c + 1 == S.c1) {
#pragma unroll
                for (int r = 0; r < T::ROWS; r++) {
                    float x = l[r];
                    x += __shfl_xor_sync(0xffffffffu, x, 4);
                    x += __shfl_xor_sync(0xffffffffu, x, 8);
                    x += __shfl_xor_sync(0xffffffffu, x, 16);
                    if (lane == 0) wml[warp * T::ROWS + r] = make_float2(m[r], x);
                }
                __syncthreads();
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    if (nt) __syncthreads();
#pragma unroll
                    for (int r8 = 0; r8 < 8; r8++) {
                        const int r = nt * 8 + r8;
                        float M = -INFINITY;
#pragma unroll
                        for (int w = 0; w < DEC_ST_WARPS; w++) M = fmaxf(M, wml[w * T::ROWS + r].x);
                        const float f = exp2f(m[r] - (M == -INFINITY ? 0.0f : M));
#pragma unroll
                        for (int j = 0; j < NJ * VW; j++)
                            merge[(warp * 8 + r8) * DP + (j / VW) * 128 + lane * VW + j % VW] = o[r][j] * f;
                    }
                    __syncthreads();
                    for (int it = threadIdx.x; it < 8 * DP; it += T::THREADS) {
                        float a = 0.0f;
#pragma unroll
                        for (int w = 0; w < DEC_ST_WARPS; w++) a += merge[w * 8 * DP + it];
                        qs[nt * 8 * DP + it] = a;                // the query rows are done with
                    }
                }
                __syncthreads();
                auto ml = [&](int r) {
                    float M = -INFINITY, L = 0.0f;
#pragma unroll
                    for (int w = 0; w < DEC_ST_WARPS; w++) M = fmaxf(M, wml[w * T::ROWS + r].x);
#pragma unroll
                    for (int w = 0; w < DEC_ST_WARPS; w++) {
                        const float2 x = wml[w * T::ROWS + r];
                        L += x.y * exp2f(x.x - (M == -INFINITY ? 0.0f : M));
                    }
                    return make_float2(M, L);
                };
                auto acc = [&](int r, int d0, int) { return *reinterpret_cast<const float4 *>(qs + r * DP + d0); };
                dec_finish<DP, T::ROWS, T::THREADS>(p, S, cu, c, upb, merge, acc, ml);
                __syncthreads();
                fresh = true;
            }
            dec_next(p, cu, upb);
        }
        cp_wait<0>();
    }
    dec_empty(p);
}

#define DEC_TC(DP, NT, ST) \
    extern "C" __global__ void __launch_bounds__(DEC_TC_WARPS * 32) irx_dec_tc_##DP##_##NT(const __grid_constant__ irx_kdec_t p) \
    { dec_tc_body<DP, NT, ST>(p); }
#define DEC_STK(DP, NT, ST) \
    extern "C" __global__ void __launch_bounds__(DEC_ST_WARPS * 32) irx_dec_st_##DP##_##NT(const __grid_constant__ irx_kdec_t p) \
    { dec_st_body<DP, NT, ST>(p); }

DEC_TC(64, 1, IRX_DEC_TC_ST(64, 1)) DEC_TC(64, 2, IRX_DEC_TC_ST(64, 2))
DEC_TC(128, 1, IRX_DEC_TC_ST(128, 1)) DEC_TC(128, 2, IRX_DEC_TC_ST(128, 2))
DEC_TC(256, 1, IRX_DEC_TC_ST(256, 1))
DEC_STK(64, 1, IRX_DEC_ST_ST(64)) DEC_STK(64, 2, IRX_DEC_ST_ST(64))
DEC_STK(128, 1, IRX_DEC_ST_ST(128)) DEC_STK(128, 2, IRX_DEC_ST_ST(128))
DEC_STK(256, 1, IRX_DEC_ST_ST(256))
