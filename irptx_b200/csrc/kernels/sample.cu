// sample.cu -- the draw of the next token: temperature, top-k, top-p, min-p and one uniform number a row.
//
// A row's weights are w_i = exp((x_i - max) / T), held as 64-bit integers, 2^kbits for a weight of 1, so
// every sum of them is exact: it does not depend on how the row is cut into blocks, warps and
// lanes, nor on the order in which histogram cells are added to. Tokens are ordered by their logit, equal ones
// by index; top-k keeps the first k of that order, top-p the shortest beginning of those whose weights
// reach p times theirs, min-p what weighs at least min_p times the first. So what is kept is every logit above a
// threshold and the first few, by index, of those equal to it. The drawn token is the first, by index,
// at which the kept weights' running sum passes u times their total.
//
// One cluster of 1 to 8 blocks a row; the row is read once, into the blocks' shared memory (rows too long for
// that are read again for each pass). A threshold is found by histograms of 2048 cells over the blocks:
// first of (max - x) in equal steps, up to where weights round to zero, then of the bits of the cell's
// range, until the cell is a single number. Every block adds up an equal slice of the cells.
#pragma once
#include "tc.cuh"

#define SMP_WARPS (IRX_SMP_THREADS / 32)
#define SMP_NEG_INF 0x007fffffu          // the key of -infinity

struct smp_shared {
    unsigned cnt[IRX_SMP_BINS], lo[IRX_SMP_BINS], hi[IRX_SMP_BINS];      // a cell's tokens and its weight, in two words
    double tab[32];                      // 2^(j / 32)
    uint64_t red[SMP_WARPS], xa[2][8];   // warps' parts; what every block of the cluster posted, two exchanges of it
    unsigned redc[SMP_WARPS], xc[2][8];
    uint64_t before, weight;             // the cell found: the weight above it, its own
    unsigned above, count, cell;
};
static_assert(sizeof(smp_shared) <= IRX_SMP_FIXED, "the launcher's size");

// Keys order as the logits do: equal numbers (both zeros) have equal keys, NaN counts as -infinity.
__device__ __forceinline__ unsigned smp_key(float x)
{
    const unsigned u = __float_as_uint(x == x ? x + 0.0f : -INFINITY);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float smp_value(unsigned key)
{
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

struct smp_row {
    double max, c, low;                  // 2^((x - max) c); below 2^low it rounds to no weight
    double one;                          // 2^kbits
    float maxf, step;                    // cells of the first histogram: (max - x) * step
    unsigned top;                        // the maximum's key
    const double *tab;
};

// The weight of a logit relative to the row's largest, in 64 bits; 0 when it is too small to count.
// 2^z = 2^(i / 32) 2^r with i = round(32 z), |r| <= 1/64: a table of 32 and the exponential series to r^5, whose
// rest is below 2^-48.
__device__ __forceinline__ double smp_exp(const smp_row &q, unsigned key)
{
    if (key == q.top) return 1.0;        // (infinity too)
    const double z = ((double)smp_value(key) - q.max) * q.c;
    if (!(z >= q.low)) return 0.0;
    const double big = 211106232532992.0;                  // 1.5 * 2^47: a sum with it is a multiple of 1/32
    const double f = z + big;
    const int i = __double2loint(f);
    const double y = (z - (f - big)) * 0.693147180559945309417;
    double e = fma(y, 1.0 / 120.0, 1.0 / 24.0);
    e = fma(e, y, 1.0 / 6.0);
    e = fma(e, y, 0.5);
    e = fma(e, y, 1.0);
    e = fma(e, y, 1.0) * q.tab[i & 31];
    return __hiloint2double(__double2hiint(e) + ((i >> 5) << 20), __double2loint(e));
}

__device__ __forceinline__ uint64_t smp_weight(const smp_row &q, double e) { return __double2ull_rn(e * q.one); }

// The cell of the first histogram, IRX_SMP_BINS for what has no weight. Never falls as keys fall.
__device__ __forceinline__ unsigned smp_cell(const smp_row &q, unsigned key)
{
    if (key == q.top) return 0;
    const float f = fminf(q.maxf - smp_value(key), 3.4028234663852886e38f) * q.step;
    return f < (float)IRX_SMP_BINS ? (unsigned)f : IRX_SMP_BINS;
}

// The largest key of [lo, hi] whose cell is at least b, when lo's is. A whole warp calls it.
__device__ __forceinline__ unsigned smp_last(const smp_row &q, unsigned lo, unsigned hi, unsigned b)
{
    while (lo < hi) {
        const unsigned step = (hi - lo) / 32 + 1;
        const uint64_t k = (uint64_t)lo + (uint64_t)step * (threadIdx.x & 31);
        const unsigned yes = __ballot_sync(0xffffffffu, k <= hi && smp_cell(q, (unsigned)k) >= b);
        lo += (__popc(yes) - 1) * step;
        hi = min((uint64_t)hi, (uint64_t)lo + step - 1);
    }
    return lo;
}

__device__ __forceinline__ uint64_t smp_warp_sum(uint64_t v)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ uint64_t smp_warp_scan(uint64_t v)          // inclusive
{
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
    }
    return v;
}

__device__ __forceinline__ unsigned smp_ld32(const void *local, unsigned rank)
{
    unsigned v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_addr(local, rank)) : "memory");
    return v;
}

__device__ __forceinline__ void smp_st32(void *local, unsigned rank, unsigned v)
{
    asm volatile("st.shared::cluster.u32 [%0], %1;" :: "r"(cluster_addr(local, rank)), "r"(v) : "memory");
}

__device__ __forceinline__ void smp_st64(void *local, unsigned rank, uint64_t v)
{
    asm volatile("st.shared::cluster.u64 [%0], %1;" :: "r"(cluster_addr(local, rank)), "l"(v) : "memory");
}

__device__ __forceinline__ void smp_cluster_sync()
{
    __syncwarp();
    cluster_sync();
}

// Every block of the cluster learns every block's (a, c); `turn` alternates, so that one exchange's values
// are not written over before all have read them.
__device__ __forceinline__ void smp_post(smp_shared &sh, unsigned rank, unsigned nc, unsigned &turn, uint64_t a, unsigned c)
{
    turn ^= 1u;
    if (threadIdx.x < nc) {
        smp_st64(&sh.xa[turn][rank], threadIdx.x, a);
        smp_st32(&sh.xc[turn][rank], threadIdx.x, c);
    }
    smp_cluster_sync();
}

// One pass over a block's elements: f(index in the block, key).
template <class T, class F>
__device__ __forceinline__ void smp_each(const T *x, int n, F f)
{
    for (int i = threadIdx.x; i < n; i += IRX_SMP_THREADS) f(i, smp_key((float)x[i]));
}

struct smp_cut { unsigned key, ties; };  // what is kept: keys above, and the first `ties` of those equal

// The cell of the histogram in which the running count (want: count) or weight reaches `target`, from cell 0 on;
// false when all of them together do not. Fills sh.cell, above, before, count, weight of every block.
__device__ __forceinline__ bool smp_find(smp_shared &sh, unsigned rank, unsigned nc, unsigned &turn, bool by_weight, uint64_t target)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int slice = IRX_SMP_BINS / nc, each = (slice + IRX_SMP_THREADS - 1) / IRX_SMP_THREADS;
    smp_cluster_sync();                                  // every block's histogram is whole
    unsigned c[4], cs = 0;
    uint64_t w[4], ws = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        c[i] = 0;
        w[i] = 0;
        const int b = threadIdx.x * each + i;
        if (i < each && b < slice) {
            const int cell = rank * slice + b;
            for (unsigned r = 0; r < nc; r++) {
                c[i] += smp_ld32(&sh.cnt[cell], r);
                if (by_weight) w[i] += (uint64_t)smp_ld32(&sh.lo[cell], r) + ((uint64_t)smp_ld32(&sh.hi[cell], r) << 32);
            }
        }
        cs += c[i];
        ws += w[i];
    }
    const uint64_t ci = smp_warp_scan(cs), wi = by_weight ? smp_warp_scan(ws) : 0;
    if (lane == 31) {
        sh.redc[warp] = (unsigned)ci;
        sh.red[warp] = wi;
    }
    __syncthreads();
    uint64_t cb = ci - cs, wb = wi - ws, ct = 0, wt = 0;
    for (int i = 0; i < SMP_WARPS; i++) {
        if (i < warp) {
            cb += sh.redc[i];
            wb += sh.red[i];
        }
        ct += sh.redc[i];
        wt += sh.red[i];
    }
    smp_post(sh, rank, nc, turn, wt, (unsigned)ct);
    uint64_t all = 0;
    for (unsigned r = 0; r < nc; r++) {
        const uint64_t rw = sh.xa[turn][r];
        const unsigned rc = sh.xc[turn][r];
        if (r < rank) {
            cb += rc;
            wb += rw;
        }
        all += by_weight ? rw : rc;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint64_t b = by_weight ? wb : cb, n = by_weight ? w[i] : c[i];
        if (b < target && target <= b + n) {             // one thread of the cluster
            for (unsigned r = 0; r < nc; r++) {
                smp_st32(&sh.cell, r, rank * slice + threadIdx.x * each + i);
                smp_st32(&sh.above, r, (unsigned)cb);
                smp_st32(&sh.count, r, c[i]);
                smp_st64(&sh.before, r, wb);
                smp_st64(&sh.weight, r, w[i]);
            }
        }
        cb += c[i];
        wb += w[i];
    }
    smp_cluster_sync();
    return target <= all;
}

// The threshold at which the running count (weights: running weight) reaches `target`, over the keys from `from` up;
// key 0 when all of them do not.
template <class T>
__device__ __forceinline__ smp_cut smp_select(smp_shared &sh, const smp_row &q, const T *x, int n, unsigned rank, unsigned nc, unsigned &turn,
                                              bool by_weight, uint64_t target, unsigned from, unsigned floor_key)
{
    unsigned lo = 0, hi = 0, shift = 0;
    uint64_t above = 0, before = 0;
    for (int level = 0;; level++) {
        __syncthreads();
        for (int b = threadIdx.x; b < IRX_SMP_BINS; b += IRX_SMP_THREADS) {
            sh.cnt[b] = 0;
            sh.lo[b] = 0;
            sh.hi[b] = 0;
        }
        __syncthreads();
        smp_each(x, n, [&](int, unsigned key) {
            if (key < from || key <= SMP_NEG_INF) return;
            unsigned cell;
            if (!level) cell = smp_cell(q, key);
            else cell = key < lo || key > hi ? IRX_SMP_BINS : (hi - key) >> shift;
            if (cell >= IRX_SMP_BINS) return;
            atomicAdd(&sh.cnt[cell], 1u);
            if (by_weight) {
                const uint64_t w = smp_weight(q, smp_exp(q, key));
                const unsigned wl = (unsigned)w, old = atomicAdd(&sh.lo[cell], wl), carry = old + wl < old;
                if ((unsigned)(w >> 32) + carry) atomicAdd(&sh.hi[cell], (unsigned)(w >> 32) + carry);
            }
        });
        if (!smp_find(sh, rank, nc, turn, by_weight, target - (by_weight ? before : above))) return {0u, 0xffffffffu};
        const unsigned cell = sh.cell, count = sh.count;
        above += sh.above;
        before += sh.before;
        if (!level) {
            hi = smp_last(q, floor_key, q.top, cell);
            lo = smp_cell(q, floor_key) > cell ? smp_last(q, floor_key, q.top, cell + 1) + 1 : floor_key;
        } else {
            const unsigned h = hi - (cell << shift);
            lo = h - lo > (1u << shift) - 1u ? h - ((1u << shift) - 1u) : lo;
            hi = h;
        }
        if (lo == hi) {                                  // a single number: how many of its tokens
            uint64_t ties = target - above;
            if (by_weight) {
                const uint64_t w = smp_weight(q, smp_exp(q, lo));
                ties = (target - before + w - 1) / w;
            }
            return {lo, (unsigned)min(ties, (uint64_t)count)};
        }
        shift = 0;
        while (((hi - lo) >> shift) >= IRX_SMP_BINS) shift++;
    }
}

// floor(f * v) for f in [0, 1), v below 2^62, exact for f of at least 2^-38.
__device__ __forceinline__ uint64_t smp_part(float f, uint64_t v, bool up)
{
    const uint64_t a = (uint64_t)((double)f * 4611686018427387904.0);           // 2^62
    const uint64_t hi = __umul64hi(a, v), lo = a * v;
    return (hi << 2 | lo >> 62) + (up && (lo << 2) != 0);
}

template <class T, bool FAR>
__device__ __forceinline__ void smp_body(const irx_ksmp_t &p)
{
    irx_pdl_enter();
    extern __shared__ __align__(16) unsigned char smp_raw[];
    smp_shared &sh = *reinterpret_cast<smp_shared *>(smp_raw);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned rank = cluster_rank(), nc, turn = 0;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(nc));
    const int64_t row = p.r0 + blockIdx.x / nc, base = (int64_t)rank * p.per;
    const int n = (int)max((int64_t)0, min(p.per, p.n - base));
    const T *src = reinterpret_cast<const T *>(p.x) + row * p.stride + base;
    T *data = reinterpret_cast<T *>(smp_raw + IRX_SMP_FIXED);
    const T *x = FAR ? src : data;

    // the row into shared memory; its largest logit, the lowest index of it, and its smallest finite one
    uint64_t best = 0;
    unsigned least = 0xffffffffu;
    auto see = [&](int i, float v) {
        const unsigned key = smp_key(v);
        const uint64_t k = (uint64_t)key << 32 | (unsigned)(0x7fffffff - (base + i));
        best = max(best, k);
        if (key > SMP_NEG_INF) least = min(least, key);
    };
    if (threadIdx.x < 32) sh.tab[threadIdx.x] = exp2((double)threadIdx.x / 32.0);
    {
        constexpr int V = 16 / sizeof(T);
        const int nv = p.vec ? n / V : 0;
        for (int i = threadIdx.x; i < nv; i += IRX_SMP_THREADS) {
            const uint4 r = *reinterpret_cast<const uint4 *>(src + (int64_t)i * V);
            if (!FAR) *reinterpret_cast<uint4 *>(data + i * V) = r;
            const T *e = reinterpret_cast<const T *>(&r);
#pragma unroll
            for (int j = 0; j < V; j++) see(i * V + j, (float)e[j]);
        }
        for (int i = nv * V + threadIdx.x; i < n; i += IRX_SMP_THREADS) {
            const T e = src[i];
            if (!FAR) data[i] = e;
            see(i, (float)e);
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    least = __reduce_min_sync(0xffffffffu, least);
    if (lane == 0) {
        sh.red[warp] = best;
        sh.redc[warp] = least;
    }
    __syncthreads();
    for (int i = 0; i < SMP_WARPS; i++) {
        best = max(best, sh.red[i]);
        least = min(least, sh.redc[i]);
    }
    smp_post(sh, rank, nc, turn, best, least);
    for (unsigned r = 0; r < nc; r++) {
        best = max(best, sh.xa[turn][r]);
        least = min(least, sh.xc[turn][r]);
    }
    smp_row q;
    q.top = (unsigned)(best >> 32);
    const float t = p.temperature[row];
    if (q.top <= SMP_NEG_INF || !(t > 0.0f)) {           // nothing to draw from, or the largest logit itself
        if (rank == 0 && threadIdx.x == 0) {
            const bool none = q.top <= SMP_NEG_INF;
            p.token[row] = none ? -1 : (int)(0x7fffffff - (unsigned)best);
            if (p.logprob) p.logprob[row] = none ? -INFINITY : 0.0f;
        }
        return;
    }
    q.tab = sh.tab;
    q.maxf = smp_value(q.top);
    q.max = (double)q.maxf;
    q.c = 1.4426950408889634074 / (double)t;
    q.low = -(double)(p.kbits + 1);
    q.one = (double)(1ull << p.kbits);
    {
        const double reach = (p.kbits + 2) / q.c, have = q.max - (double)smp_value(min(least, q.top)), r = reach < have ? reach : have;
        q.step = r > 0.0 && r < 1e300 ? (float)min(2047.9 / r, 3.0e38) : 1.0f;
    }

    smp_cut cut = {0u, 0xffffffffu};
    const int k = p.top_k[row];
    const float tp = p.top_p[row];
    const float mp = p.min_p[row], least_p = mp > 0.0f ? fminf(mp, 1.0f) : 0.0f;
    if (k > 0 && k < p.n) cut = smp_select(sh, q, x, n, rank, nc, turn, false, (uint64_t)k, 0u, min(least, q.top));
    if (tp < 1.0f) {
        // the weight of what top-k kept, of which top-p keeps its part
        uint64_t w = 0;
        unsigned eq = 0;
        smp_each(x, n, [&](int, unsigned key) {
            if (key > cut.key) w += smp_weight(q, smp_exp(q, key));
            eq += key == cut.key;
        });
        w = smp_warp_sum(w);
        eq = __reduce_add_sync(0xffffffffu, eq);
        __syncthreads();
        if (lane == 0) {
            sh.red[warp] = w;
            sh.redc[warp] = eq;
        }
        __syncthreads();
        w = 0;
        eq = 0;
        for (int i = 0; i < SMP_WARPS; i++) {
            w += sh.red[i];
            eq += sh.redc[i];
        }
        smp_post(sh, rank, nc, turn, w, eq);
        w = 0;
        eq = 0;
        for (unsigned r = 0; r < nc; r++) {
            w += sh.xa[turn][r];
            eq += sh.xc[turn][r];
        }
        if (cut.key) w += min(eq, cut.ties) * smp_weight(q, smp_exp(q, cut.key));
        uint64_t target = tp > 0.0f ? smp_part(tp, w, true) : 1;
        if (target < 1) target = 1;
        const smp_cut c2 = smp_select(sh, q, x, n, rank, nc, turn, true, target, cut.key, min(least, q.top));
        if (c2.key > cut.key) cut = c2;
        else cut.ties = min(cut.ties, c2.ties);          // (the same key, or none: the whole is reached)
    }

    // the kept weights of every warp's stretch of the row, and where u times their total falls
    const int stretch = (int)(p.per / SMP_WARPS), s0 = min(n, warp * stretch), s1 = min(n, s0 + stretch);
    const double e_cut = cut.key ? smp_exp(q, cut.key) : 0.0;
    const uint64_t w_cut = e_cut >= least_p ? smp_weight(q, e_cut) : 0;
    uint64_t w = 0;
    unsigned eq = 0;
    for (int i = s0 + lane; i < s1; i += 32) {
        const unsigned key = smp_key((float)x[i]);
        if (key > cut.key) {
            const double e = smp_exp(q, key);
            if (e >= least_p) w += smp_weight(q, e);
        }
        eq += key == cut.key;
    }
    w = smp_warp_sum(w);
    eq = __reduce_add_sync(0xffffffffu, eq);
    __syncthreads();
    if (lane == 0) {
        sh.red[warp] = w;
        sh.redc[warp] = eq;
    }
    __syncthreads();
    uint64_t wt = 0;
    unsigned et = 0;
    for (int i = 0; i < SMP_WARPS; i++) {
        wt += sh.red[i];
        et += sh.redc[i];
    }
    smp_post(sh, rank, nc, turn, wt, et);
    uint64_t total = 0, run = 0;
    unsigned ties = cut.ties, mine = 0;                  // ties: left to keep; mine: of them, this block's
    for (unsigned r = 0; r < nc; r++) {
        const unsigned have = min(ties, sh.xc[turn][r]);
        if (r == rank) {
            run = total;
            mine = ties;
        }
        total += sh.xa[turn][r] + have * w_cut;
        ties -= have;
    }
    const float u = p.u[row];
    const uint64_t at = smp_part(u > 0.0f ? fminf(u, 0.99999994f) : 0.0f, total, false);
    for (int i = 0; i < warp; i++) {
        const unsigned have = min(mine, sh.redc[i]);
        run += sh.red[i] + have * w_cut;
        mine -= have;
    }
    if (at < run || at >= run + w + (uint64_t)min(mine, eq) * w_cut) return;
    for (int i0 = s0; i0 < s1; i0 += 32) {               // one warp of the cluster
        const int i = i0 + lane;
        const unsigned key = i < s1 ? smp_key((float)x[i]) : 0u;
        double e = i < s1 && key >= cut.key ? smp_exp(q, key) : 0.0;
        const unsigned same = __ballot_sync(0xffffffffu, i < s1 && key == cut.key);
        if (e < least_p || (key == cut.key && __popc(same & ((1u << lane) - 1u)) >= mine)) e = 0.0;
        mine -= min(mine, (unsigned)__popc(same));
        const uint64_t sum = smp_warp_scan(smp_weight(q, e));
        const unsigned past = __ballot_sync(0xffffffffu, run + sum > at);
        if (past) {
            if (lane == __ffs(past) - 1) {
                p.token[row] = (int)(base + i);
                if (p.logprob) p.logprob[row] = (float)(log(e) - log((double)total / q.one));
            }
            return;
        }
        run += __shfl_sync(0xffffffffu, sum, 31);
    }
}

extern "C" __global__ void __launch_bounds__(IRX_SMP_THREADS) irx_sample_bf16(const __grid_constant__ irx_ksmp_t p) { smp_body<__nv_bfloat16, false>(p); }
extern "C" __global__ void __launch_bounds__(IRX_SMP_THREADS) irx_sample_bf16_far(const __grid_constant__ irx_ksmp_t p) { smp_body<__nv_bfloat16, true>(p); }
extern "C" __global__ void __launch_bounds__(IRX_SMP_THREADS) irx_sample_f32(const __grid_constant__ irx_ksmp_t p) { smp_body<float, false>(p); }
extern "C" __global__ void __launch_bounds__(IRX_SMP_THREADS) irx_sample_f32_far(const __grid_constant__ irx_ksmp_t p) { smp_body<float, true>(p); }
