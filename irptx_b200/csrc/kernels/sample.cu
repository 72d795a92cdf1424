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
// that are read again for each pass), where thread t holds words t * words and on: an odd number of
// them, so that a warp's reads fall into 32 banks. Tokens per cell of (max - x), 2048 equal cells up to where
// weights round to zero, or their weights, show the cell in which a filter ends. When that cell and those
// above it hold few tokens (top-k, or a peaked row), they go to the first block, which finishes alone. Otherwise the
// cell's own tokens are resolved, by the first block when they are few, else by histograms of the cell's
// range, and every thread adds up its stretch's kept weights.
//
// Bound by instructions for many rows (30 an element without filters, 67 with top-p: 128 rows of 151999 normal bf16
// logits 41 and 81 us, 138 with top-p from 0.8 to 0.95 at temperatures from 0.6 to 1.4, against 6 us for reading them) and by
// its exchanges and passes, one after another, for few (one row of 128001, top-k and top-p: 15.4 us). The sums need a
// weight once for each value, which a bf16 row has a few thousand of; here it is computed for each token.
#pragma once
#include "tc.cuh"

#define SMP_WARPS (IRX_SMP_THREADS / 32)
#define SMP_FEW 1024                     // tokens that one block finishes alone
#define SMP_CELLS (IRX_SMP_BINS / IRX_SMP_THREADS)      // cells of a thread, in a cluster of one
#define SMP_OWN (SMP_FEW / IRX_SMP_THREADS)             // few tokens: a thread's
#define SMP_STEP 4                       // words that a thread takes at a time

struct smp_shared {
    union {
        struct { unsigned cnt[IRX_SMP_BINS + 32], lo[IRX_SMP_BINS], hi[IRX_SMP_BINS]; };   // a cell's tokens, or its weight in two words
        struct { uint64_t mine[SMP_FEW], list[SMP_FEW], weight_of[SMP_FEW]; };        // few tokens: this block's, the row's, their weights
    };
    double tab[128];
    uint64_t red[3][SMP_WARPS], xa[2][8], xb[2][8], xd[2][8];      // warps' parts; what the cluster's blocks posted, two exchanges of it
    unsigned redc[SMP_WARPS], xc[2][8];
    uint64_t before, weight;             // the cell found: the weight above it, its own
    unsigned above, count, cell;         // tokens above it, its own
    unsigned few, key, ties;
    uint64_t bar;
};
static_assert(sizeof(smp_shared) <= IRX_SMP_FIXED, "the launcher's size");
static_assert(3 * IRX_SMP_THREADS * sizeof(unsigned) <= SMP_FEW * sizeof(uint64_t), "three words a thread in the list's place");

// Logits as numbers that order and weigh as defined: NaN as -infinity. For rows whose largest is infinite (then such
// logits are 0 and all others -infinity) or below -1e30 (then the largest is taken away from all: exactly, wherever a
// weight is left) a second step follows, so that a number far below the largest exists.
enum { SMP_PLAIN, SMP_INFINITE, SMP_LOW };
__device__ __forceinline__ float smp_shift(float x, int mode, float top)
{
    return mode == SMP_INFINITE ? (x == INFINITY ? 0.0f : -INFINITY) : mode == SMP_LOW ? x - top : x;
}

// Keys order as the numbers do: the magnitude's bits, counted up or down from 2^31 (bf16: 2^15), which is the key of both
// zeros. Neighbouring keys are neighbouring numbers, none is left out: "above the number of the key below" and "from this
// key on" are the same everywhere, at 0 too.
template <class T> struct smp_type;
template <> struct smp_type<float> {
    static const int N = 1;
    static const unsigned PAD = 0xff800000u;             // -infinity
    __device__ static __forceinline__ float get(unsigned w, int) { return __uint_as_float(w); }
    __device__ static __forceinline__ unsigned put(float a, float) { return __float_as_uint(a); }
    // the larger of each element; of a number and NaN, the number
    __device__ static __forceinline__ unsigned most(unsigned a, unsigned b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
    __device__ static __forceinline__ unsigned key(float x)
    {
        const unsigned u = __float_as_uint(x);
        return u & 0x80000000u ? 0u - u : u | 0x80000000u;
    }
    __device__ static __forceinline__ float value(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : 0u - k); }
};
template <> struct smp_type<__nv_bfloat16> {
    static const int N = 2;
    static const unsigned PAD = 0xff80ff80u;
    __device__ static __forceinline__ float get(unsigned w, int h) { return __uint_as_float(h ? w & 0xffff0000u : w << 16); }
    __device__ static __forceinline__ unsigned most(unsigned a, unsigned b)
    {
        const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&b));
        return *reinterpret_cast<const unsigned *>(&m);
    }
    __device__ static __forceinline__ unsigned put(float a, float b) { return __float_as_uint(a) >> 16 | (__float_as_uint(b) & 0xffff0000u); }
    __device__ static __forceinline__ unsigned key(float x)
    {
        const unsigned u = __float_as_uint(x) >> 16;
        return u & 0x8000u ? (0u - u) & 0xffffu : u | 0x8000u;
    }
    __device__ static __forceinline__ float value(unsigned k) { return __uint_as_float((k & 0x8000u ? k & 0x7fffu : (0u - k) & 0xffffu) << 16); }
};

struct smp_row {
    double c, at_max;                    // a weight is 2^(kbits + (x c - at_max) / 128)
    float maxf, floor, step;             // at the floor and below it rounds to 0; cells: (max - x) / 2 * step
    uint64_t one;                        // the largest logit's weight
    const double *tab;
};

// The weight of a logit above the floor, in the low 52 bits under those of 2^52. 2^(z / 128) = 2^(i / 128) 2^(r / 128),
// i = round(z), |r| <= 1/2: a table of 128, kbits in it, and the exponential series to r^4, whose rest is below 2^-49.
// The last sum, with 2^52, leaves the rounded integer. at_max is rounded once a row, which scales all its weights
// alike. The floor keeps i above -30000 (see T below), so that exponents are added without a check.
__device__ __forceinline__ uint64_t smp_raw(const irx_ksmp_t &p, const smp_row &q, float x)
{
    const double z = fma((double)x, q.c, -q.at_max);
    const double f = z + p.big;
    const int i = __double2loint(f);
    const double r = z - (f - p.big), t = q.tab[i & 127];
    double e = fma(r, p.series[3], p.series[2]);
    e = fma(e, r, p.series[1]);
    e = fma(e, r, p.series[0]);
    e = fma(e, r, 1.0);
    e = fma(e, __hiloint2double(__double2hiint(t) + (i & ~127) * (1 << 13), __double2loint(t)), p.two52);
    return (uint64_t)__double_as_longlong(e);
}
#define SMP_RAW 0x4330000000000000ull    // the bits of 2^52: a sum of n raw weights has n of them too many

__device__ __forceinline__ uint64_t smp_weight(const irx_ksmp_t &p, const smp_row &q, float x) { return smp_raw(p, q, fmaxf(x, q.floor)) - SMP_RAW; }

// The cell of the first histogram, `none` (at least IRX_SMP_BINS) for what has no weight. Never falls as x falls.
__device__ __forceinline__ unsigned smp_cell(const smp_row &q, float x, unsigned none = IRX_SMP_BINS)
{
    const float f = fmaf(fmaf(-0.5f, x, 0.5f * q.maxf), q.step, 8388608.0f);         // 2^23: the sum's low bits are the cell
    return x > q.floor && f < 8388608.0f + IRX_SMP_BINS ? __float_as_uint(f) - 0x4b000000u : none;
}

// A key whose number is the floor or lies below it.
template <class T>
__device__ __forceinline__ unsigned smp_least(const smp_row &q) { return smp_type<T>::key(q.floor) - (smp_type<T>::N - 1); }

// The largest key of [lo, hi] for which f holds, when it holds for lo and for no key above one for which it does not. A whole
// warp calls it.
template <class F>
__device__ __forceinline__ unsigned smp_last(unsigned lo, unsigned hi, F f)
{
    while (lo < hi) {
        const unsigned step = (hi - lo) / 32 + 1;
        const uint64_t k = (uint64_t)lo + (uint64_t)step * (threadIdx.x & 31);
        const unsigned yes = __ballot_sync(0xffffffffu, k <= hi && f((unsigned)min(k, (uint64_t)hi)));
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

__device__ __forceinline__ unsigned smp_add32(void *local, unsigned rank, unsigned v)
{
    unsigned old;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(cluster_addr(local, rank)), "r"(v) : "memory");
    return old;
}

__device__ __forceinline__ void smp_cluster_sync()
{
    __syncwarp();
    cluster_sync();
}

// Every block of the cluster learns every block's (a, c, b, d); `turn` alternates, so that one exchange's values
// are not written over before all have read them.
__device__ __forceinline__ void smp_post(smp_shared &sh, unsigned rank, unsigned nc, unsigned &turn, uint64_t a, unsigned c,
                                         uint64_t b = 0, uint64_t d = 0)
{
    turn ^= 1u;
    if (threadIdx.x < nc) {
        smp_st64(&sh.xa[turn][rank], threadIdx.x, a);
        smp_st64(&sh.xb[turn][rank], threadIdx.x, b);
        smp_st64(&sh.xd[turn][rank], threadIdx.x, d);
        smp_st32(&sh.xc[turn][rank], threadIdx.x, c);
    }
    smp_cluster_sync();
}

// A block's words, by thread: in shared memory, cleaned, or (FAR) in the row itself.
template <class T, bool FAR> struct smp_data {
    unsigned *data;                      // this thread's first word
    const T *src;                        // the row's element 0 of this thread
    int64_t left;                        // the row's elements from there on
    int words, mode;
    float top;
    __device__ __forceinline__ unsigned word(int j) const
    {
        if (!FAR) return data[j];
        float e[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int h = 0; h < smp_type<T>::N; h++)
            if (j * smp_type<T>::N + h < left) e[h] = smp_shift(fmaxf((float)src[(int64_t)j * smp_type<T>::N + h], -INFINITY), mode, top);
        return smp_type<T>::put(e[0], e[1]);
    }
    // f(number, index among this thread's elements) for each of them
    template <class F> __device__ __forceinline__ void each(F f) const
    {
#pragma unroll 4
        for (int j = 0; j < words; j++) {
            const unsigned w = word(j);
#pragma unroll
            for (int h = 0; h < smp_type<T>::N; h++) f(smp_type<T>::get(w, h), j * smp_type<T>::N + h);
        }
    }
};

// f(number, index) for the few numbers above `from` and up to `to`: looked for SMP_STEP words at a time, with one branch.
template <class T, bool FAR, class F>
__device__ __forceinline__ void smp_pick(const smp_data<T, FAR> &x, float from, float to, F f)
{
    typedef smp_type<T> ty;
    for (int j0 = 0; j0 < x.words; j0 += SMP_STEP) {
        unsigned hits = 0;
#pragma unroll
        for (int j = 0; j < SMP_STEP; j++) {
            const unsigned w = j0 + j < x.words ? x.word(j0 + j) : ty::PAD;
#pragma unroll
            for (int h = 0; h < ty::N; h++) {
                const float v = ty::get(w, h);
                if (v > from && v <= to) hits |= 1u << (j * ty::N + h);
            }
        }
        for (; hits; hits &= hits - 1) {
            const int b = __ffs(hits) - 1;
            f(ty::get(x.word(j0 + b / ty::N), b % ty::N), j0 * ty::N + b);
        }
    }
}

struct smp_cut { float above; unsigned ties; };     // what is kept: what is above, and the first `ties` of those equal

// Sums over the block of N numbers and of `c`; the warps' parts stay in red and redc. All threads get the totals.
template <int N>
__device__ __forceinline__ void smp_block_sums(smp_shared &sh, uint64_t (&w)[N], unsigned &c)
{
#pragma unroll
    for (int i = 0; i < N; i++) w[i] = smp_warp_sum(w[i]);
    c = __reduce_add_sync(0xffffffffu, c);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
        for (int i = 0; i < N; i++) sh.red[i][threadIdx.x >> 5] = w[i];
        sh.redc[threadIdx.x >> 5] = c;
    }
    __syncthreads();
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < N; i++) w[i] = smp_warp_sum(lane < SMP_WARPS ? sh.red[i][lane] : 0);
    c = __reduce_add_sync(0xffffffffu, lane < SMP_WARPS ? sh.redc[lane] : 0u);
}

__device__ __forceinline__ void smp_clear(smp_shared &sh, bool by_weight)
{
    __syncthreads();
    for (int b = threadIdx.x; b < IRX_SMP_BINS; b += IRX_SMP_THREADS) {
        if (!by_weight) sh.cnt[b] = 0;
        else sh.lo[b] = sh.hi[b] = 0;
    }
    __syncthreads();
}

__device__ __forceinline__ void smp_tally(smp_shared &sh, unsigned cell, bool by_weight, uint64_t w)
{
    if (!by_weight) {
        atomicAdd(&sh.cnt[cell], 1u);
        return;
    }
    const unsigned wl = (unsigned)w, old = atomicAdd(&sh.lo[cell], wl), up = (unsigned)(w >> 32) + (old + wl < old);
    if (up) atomicAdd(&sh.hi[cell], up);
}

// The cell of the blocks' histograms in which the running count, or weight, reaches `target`, from cell 0 on; false when
// all of them together do not. With `part`, a share of all: target = the least integer not below part / 2^62 times
// the whole weight, at least 1. SMP_GUESS: the weights are guessed from the cells' tokens, `bits` being what a cell
// takes from a weight's logarithm. Fills every block's sh.cell, above and count, before and weight.
enum { SMP_COUNT, SMP_WEIGHT, SMP_GUESS };
__device__ __forceinline__ uint64_t smp_part(uint64_t part, uint64_t v, bool up)
{
    const uint64_t hi = __umul64hi(part, v), lo = part * v;
    return (hi << 2 | lo >> 62) + (up && (lo << 2) != 0);
}

__device__ __forceinline__ bool smp_find(smp_shared &sh, unsigned rank, unsigned nc, unsigned &turn, int mode, uint64_t &target, uint64_t part, float bits = 0.0f)
{
    const bool by_weight = mode != SMP_COUNT;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int slice = IRX_SMP_BINS / nc, each = (slice + IRX_SMP_THREADS - 1) / IRX_SMP_THREADS;
    smp_cluster_sync();                                  // every block's histogram is whole
    unsigned c[SMP_CELLS], cs = 0;
    uint64_t w[SMP_CELLS], ws = 0;
#pragma unroll
    for (int i = 0; i < SMP_CELLS; i++) {
        c[i] = 0;
        w[i] = 0;
        const int b = threadIdx.x * each + i;
        if (i < each && b < slice) {
            const int cell = rank * slice + b;
            unsigned a[8], l[8], h[8];
#pragma unroll
            for (int r = 0; r < 8; r++) {
                a[r] = l[r] = h[r] = 0;
                if (r >= nc) continue;
                if (mode == SMP_WEIGHT) {
                    l[r] = smp_ld32(&sh.lo[cell], r);
                    h[r] = smp_ld32(&sh.hi[cell], r);
                } else a[r] = smp_ld32(&sh.cnt[cell], r);
            }
#pragma unroll
            for (int r = 0; r < 8; r++) {
                c[i] += a[r];
                w[i] += (uint64_t)l[r] + ((uint64_t)h[r] << 32);
            }
            if (mode == SMP_GUESS) w[i] = (uint64_t)((float)c[i] * exp2f(32.0f - bits * (float)cell));
        }
        cs += c[i];
        ws += w[i];
    }
    const unsigned ci = (unsigned)smp_warp_scan(cs);
    const uint64_t wi = by_weight ? smp_warp_scan(ws) : 0;
    if (lane == 31) {
        sh.redc[warp] = ci;
        sh.red[0][warp] = wi;
    }
    __syncthreads();
    uint64_t wt = lane < SMP_WARPS ? sh.red[0][lane] : 0;
    unsigned ct = lane < SMP_WARPS ? sh.redc[lane] : 0;
    uint64_t wb = wi - ws + smp_warp_sum(lane < warp ? wt : 0);
    unsigned cb = ci - cs + __reduce_add_sync(0xffffffffu, lane < warp ? ct : 0u);
    wt = smp_warp_sum(wt);
    ct = __reduce_add_sync(0xffffffffu, ct);
    smp_post(sh, rank, nc, turn, wt, ct);
    uint64_t all = 0, whole = 0;
    for (unsigned r = 0; r < nc; r++) {
        const uint64_t rw = sh.xa[turn][r];
        const unsigned rc = sh.xc[turn][r];
        if (r < rank) {
            cb += rc;
            wb += rw;
        }
        whole += rw;
        all += by_weight ? rw : rc;
    }
    if (part) target = max(smp_part(part, whole, true), (uint64_t)1);
#pragma unroll
    for (int i = 0; i < SMP_CELLS; i++) {
        const uint64_t b = by_weight ? wb : cb, n = by_weight ? w[i] : c[i];
        if (b < target && target <= b + n) {             // one thread of the cluster
            for (unsigned r = 0; r < nc; r++) {
                smp_st32(&sh.cell, r, rank * slice + threadIdx.x * each + i);
                smp_st32(&sh.above, r, cb);
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

// This block's few tokens (n of them in sh.mine) into block 0's list, behind those of the blocks before it. Ends with a
// cluster barrier.
__device__ __forceinline__ void smp_hand_over(smp_shared &sh, unsigned n, unsigned at)
{
    for (unsigned i = threadIdx.x; i < n; i += IRX_SMP_THREADS) smp_st64(&sh.list[at + i], 0, sh.mine[i]);
    smp_cluster_sync();
}

__device__ __forceinline__ uint64_t smp_token(float v, int64_t i) { return (uint64_t)~smp_type<float>::key(v) << 32 | (unsigned)i; }

__device__ __forceinline__ float smp_number(uint64_t token) { return smp_type<float>::value(~(unsigned)(token >> 32)); }

// The threshold among the m tokens of block 0's list, numbers with keys from lo to hi, of which `left` tokens, or that much
// weight, are to be kept: histograms of 256 cells of the range, by block 0, until a cell is one number.
template <class T>
__device__ __forceinline__ smp_cut smp_among(const irx_ksmp_t &p, smp_shared &sh, const smp_row &q, unsigned rank, unsigned nc, unsigned m,
                                             unsigned lo, unsigned hi, uint64_t left, bool by_weight)
{
    typedef smp_type<T> ty;
    if (rank == 0) {
        unsigned *low = reinterpret_cast<unsigned *>(sh.weight_of), *high = low + 256;   // a cell's sum in two words
        const int lane = threadIdx.x & 31;
        unsigned key[SMP_OWN];
        uint64_t w[SMP_OWN];
#pragma unroll
        for (int a = 0; a < SMP_OWN; a++) {
            const unsigned i = threadIdx.x + a * IRX_SMP_THREADS;
            const float v = i < m ? smp_number(sh.list[i]) : 0.0f;
            key[a] = i < m ? ty::key(v) : ~0u;
            w[a] = i < m ? by_weight ? smp_weight(p, q, v) : 1 : 0;
        }
        for (;;) {
            unsigned shift = 0;
            while (((hi - lo) >> shift) >= 256) shift++;
            for (int b = threadIdx.x; b < 512; b += IRX_SMP_THREADS) low[b] = 0;
            __syncthreads();
#pragma unroll
            for (int a = 0; a < SMP_OWN; a++)
                if (key[a] >= lo && key[a] <= hi) {
                    const unsigned cell = (hi - key[a]) >> shift, wl = (unsigned)w[a], old = atomicAdd(&low[cell], wl);
                    const unsigned up = (unsigned)(w[a] >> 32) + (old + wl < old);
                    if (up) atomicAdd(&high[cell], up);
                }
            __syncthreads();
            if (threadIdx.x < 32) {                      // 8 cells a lane
                uint64_t c[8], sum = 0;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    c[i] = (uint64_t)high[lane * 8 + i] << 32 | low[lane * 8 + i];
                    sum += c[i];
                }
                uint64_t b = smp_warp_scan(sum) - sum;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (b < left && left <= b + c[i]) {
                        sh.cell = lane * 8 + i;
                        sh.before = b;
                        sh.weight = c[i];
                    }
                    b += c[i];
                }
            }
            __syncthreads();
            left -= sh.before;
            hi -= sh.cell << shift;
            lo = hi - lo > (1u << shift) - 1u ? hi - ((1u << shift) - 1u) : lo;
            if (lo == hi) break;
        }
        if (threadIdx.x < nc) {                          // sh.weight is that of this number's tokens, all alike
            const uint64_t one = by_weight ? smp_weight(p, q, ty::value(lo)) : 1, ties = (left + one - 1) / one;
            const bool all = ties * one >= sh.weight;    // none of them is cut off: up to the number below
            smp_st32(&sh.key, threadIdx.x, all ? lo - 1 : lo);
            smp_st32(&sh.ties, threadIdx.x, all ? 0 : (unsigned)ties);
        }
    }
    if (threadIdx.x == 0) sh.few = 0;
    smp_cluster_sync();
    return {ty::value(sh.key), sh.ties};
}

// After a first histogram whose cell has been found: the exact threshold in it. The cell's tokens go to block 0 when they
// are few and all of them count (gather), else histograms of its range follow.
template <class T, bool FAR>
__device__ __forceinline__ smp_cut smp_resolve(const irx_ksmp_t &p, smp_shared &sh, const smp_row &q, const smp_data<T, FAR> &x, unsigned rank, unsigned nc,
                                               unsigned &turn, bool by_weight, uint64_t target, bool gather)
{
    typedef smp_type<T> ty;
    const unsigned least = smp_least<T>(q), top = ty::key(q.maxf), cell = sh.cell;
    unsigned hi = smp_last(least, top, [&](unsigned k) { return smp_cell(q, ty::value(k)) >= cell; });
    unsigned lo = smp_last(least, top, [&](unsigned k) { return smp_cell(q, ty::value(k)) > cell; }) + 1;
    uint64_t count = sh.count;                           // at most
    if (by_weight) {
        const uint64_t w = smp_weight(p, q, ty::value(lo));
        count = w ? sh.weight / w : ~0ull;
    }
    uint64_t left = target - (by_weight ? sh.before : sh.above);
    if (lo != hi && gather && count <= SMP_FEW) {
        smp_pick(x, ty::value(lo - 1), ty::value(hi), [&](float v, int) { sh.mine[atomicAdd(&sh.few, 1u)] = smp_token(v, 0); });
        __syncthreads();
        const unsigned n = sh.few;
        unsigned at = 0, m = 0;
        smp_post(sh, rank, nc, turn, 0, n);
        for (unsigned r = 0; r < nc; r++) {
            if (r == rank) at = m;
            m += sh.xc[turn][r];
        }
        smp_hand_over(sh, n, at);
        return smp_among<T>(p, sh, q, rank, nc, m, lo, hi, left, by_weight);
    }
    while (lo != hi) {
        unsigned shift = 0;
        while (((hi - lo) >> shift) >= IRX_SMP_BINS) shift++;
        smp_clear(sh, by_weight);
        const float from = ty::value(lo), to = ty::value(hi);
        x.each([&](float v, int) {
            if (v >= from && v <= to) smp_tally(sh, (hi - ty::key(v)) >> shift, by_weight, by_weight ? smp_weight(p, q, v) : 0);
        });
        smp_find(sh, rank, nc, turn, by_weight ? SMP_WEIGHT : SMP_COUNT, left, 0);
        left -= by_weight ? sh.before : sh.above;
        hi -= sh.cell << shift;
        count = by_weight ? sh.weight / max(smp_weight(p, q, ty::value(hi)), (uint64_t)1) : sh.count;
        lo = hi - lo > (1u << shift) - 1u ? hi - ((1u << shift) - 1u) : lo;
    }
    const uint64_t w = by_weight ? smp_weight(p, q, ty::value(lo)) : 1, ties = (left + w - 1) / w;
    // (count is exact here: a single number's tokens weigh the same)
    return ties >= count ? smp_cut{ty::value(lo - 1), 0u} : smp_cut{ty::value(lo), (unsigned)ties};
}

struct smp_settings { uint64_t k, part, least, whole; float u; };      // part: top-p in 2^-62, 0 off; least: min-p's weight

// Block 0, with all tokens that a filter may keep in its list, m of them: all filters and the draw. s.whole: the row's
// weight, when top-k is off.
__device__ __forceinline__ void smp_finish(const irx_ksmp_t &p, smp_shared &sh, const smp_row &q, unsigned m, int64_t row, const smp_settings &s)
{
    uint64_t me[SMP_OWN], w[SMP_OWN], better[SMP_OWN] = {};
    unsigned order[SMP_OWN] = {}, none = 0;
#pragma unroll
    for (int a = 0; a < SMP_OWN; a++) {
        const unsigned i = threadIdx.x + a * IRX_SMP_THREADS;
        me[a] = i < m ? sh.list[i] : ~0ull;
        w[a] = i < m ? smp_weight(p, q, smp_number(me[a])) : 0;
        if (i < m) sh.weight_of[i] = w[a];
    }
    __syncthreads();
#pragma unroll 4
    for (unsigned j = 0; j < m; j++) {                   // how many come before each, and their weight
        const uint64_t other = sh.list[j], ow = sh.weight_of[j];
#pragma unroll
        for (int a = 0; a < SMP_OWN; a++)
            if (other < me[a]) {
                order[a]++;
                better[a] += ow;
            }
    }
    uint64_t whole[1] = {s.whole};
    bool keep[SMP_OWN];
#pragma unroll
    for (int a = 0; a < SMP_OWN; a++) keep[a] = threadIdx.x + a * IRX_SMP_THREADS < m && (!s.k || order[a] < s.k);
    if (s.k && s.part) {
        whole[0] = 0;
#pragma unroll
        for (int a = 0; a < SMP_OWN; a++) whole[0] += keep[a] ? w[a] : 0;
        smp_block_sums(sh, whole, none);
    }
    const uint64_t target = s.part ? max(smp_part(s.part, whole[0], true), (uint64_t)1) : ~0ull;
    uint64_t all[1] = {0};
#pragma unroll
    for (int a = 0; a < SMP_OWN; a++) {
        keep[a] = keep[a] && better[a] < target && w[a] >= s.least;
        if (!keep[a]) w[a] = 0;
        all[0] += w[a];
    }
    smp_block_sums(sh, all, none);                     // (its barriers: all have read weight_of)
#pragma unroll
    for (int a = 0; a < SMP_OWN; a++)
        if (threadIdx.x + a * IRX_SMP_THREADS < m) sh.weight_of[threadIdx.x + a * IRX_SMP_THREADS] = w[a];
    __syncthreads();
    const uint64_t total = all[0], at = smp_part((uint64_t)((double)s.u * 4611686018427387904.0), total, false);
    uint64_t run[SMP_OWN] = {};
#pragma unroll 4
    for (unsigned j = 0; j < m; j++) {                   // the kept weight at lower indexes
        const unsigned other = (unsigned)sh.list[j];
        const uint64_t ow = sh.weight_of[j];
#pragma unroll
        for (int a = 0; a < SMP_OWN; a++)
            if (other < (unsigned)me[a]) run[a] += ow;
    }
#pragma unroll
    for (int a = 0; a < SMP_OWN; a++)
        if (run[a] <= at && at < run[a] + w[a]) {        // one thread
            p.token[row] = (int)(unsigned)me[a];
            if (p.logprob) p.logprob[row] = (float)(log((double)w[a] / (double)total));
        }
}

template <class T, bool FAR>
__device__ __forceinline__ void smp_body(const irx_ksmp_t &p)
{
    typedef smp_type<T> ty;
    cluster_arrive();                                    // (waited for before the first exchange)
    irx_pdl_enter();
    extern __shared__ __align__(16) unsigned char smp_bytes[];
    smp_shared &sh = *reinterpret_cast<smp_shared *>(smp_bytes);
    unsigned *data = reinterpret_cast<unsigned *>(smp_bytes + IRX_SMP_FIXED);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned rank = cluster_rank(), nc, turn = 0;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(nc));
    const int64_t row = p.r0 + blockIdx.x / nc, per = (int64_t)p.words * IRX_SMP_THREADS * ty::N;
    const T *line = reinterpret_cast<const T *>(p.x) + row * p.stride;
    // a row that begins inside a word: its words count from there, with one element of nothing first
    const int lead = !FAR && ((size_t)line & 3) ? 1 : 0;
    const int64_t base = (int64_t)rank * per - lead, here = max((int64_t)0, min(per, p.n - base));
    const T *src = line + base;
    if (!FAR) data += ((size_t)src & 15) / 4;            // as far past 16 bytes as in memory
    const int64_t first = base + (int64_t)threadIdx.x * p.words * ty::N;               // this thread's first element
    smp_data<T, FAR> x = {data + threadIdx.x * p.words, src + (int64_t)threadIdx.x * p.words * ty::N, p.n - first, p.words, SMP_PLAIN, 0.0f};
    const float t = p.temperature[row], tp = p.top_p[row], mp = p.min_p[row], un = p.u[row];
    const int k = p.top_k[row];

    // the row into shared memory, padded with -infinity: what lies between multiples of 16 bytes in one copy
    unsigned bytes = 0;
    if (threadIdx.x < 128) sh.tab[threadIdx.x] = p.tab[threadIdx.x];
    if (threadIdx.x == 0) sh.few = 0;
    if (!FAR) {
        const size_t a0 = (size_t)src, from = (a0 + (base < 0 ? sizeof(T) : 0) + 15) & ~(size_t)15, to = (a0 + here * sizeof(T)) & ~(size_t)15;
        bytes = to > from ? (unsigned)(to - from) : 0;
        if (threadIdx.x == 0) {
            irx_mbar_init(&sh.bar, 1);
            irx_fence_mbar_init();
            if (bytes) {
                irx_mbar_expect_tx(&sh.bar, bytes);
                irx_bulk_g2s(reinterpret_cast<unsigned char *>(data) + (from - a0), reinterpret_cast<const void *>(from), bytes, &sh.bar);
            }
        }
        T *e = reinterpret_cast<T *>(data);
        const int64_t i0 = (int64_t)(from - a0) / (int64_t)sizeof(T), i1 = i0 + bytes / sizeof(T);       // copied
        if (threadIdx.x < i0 && bytes) e[threadIdx.x] = base + threadIdx.x >= 0 ? src[threadIdx.x] : (T)-INFINITY;
        for (int64_t i = (bytes ? i1 : 0) + threadIdx.x; i < per; i += IRX_SMP_THREADS)
            e[i] = i < here && base + i >= 0 ? src[i] : (T)-INFINITY;
    }
    __syncthreads();
    if (bytes && !irx_mbar_wait(&sh.bar, 0) && lane == 0) atomicOr(p.err, IRX_KERR_TIMEOUT);
    unsigned high = ty::PAD;
#pragma unroll 4
    for (int j = 0; j < x.words; j++) {
        const unsigned w = ty::most(x.word(j), ty::PAD);
        high = ty::most(high, w);
        if (!FAR) x.data[j] = w;
    }
    float top = fmaxf(ty::get(high, 0), ty::get(high, ty::N - 1));
    const unsigned tk = __reduce_max_sync(0xffffffffu, smp_type<float>::key(top));
    if (lane == 0) sh.redc[warp] = tk;
    __syncthreads();
    unsigned best = 0;
#pragma unroll
    for (int i = 0; i < SMP_WARPS; i++) best = max(best, sh.redc[i]);
    __syncwarp();
    cluster_wait();                                      // every block of the cluster has begun: its shared memory may be written
    smp_post(sh, rank, nc, turn, 0, best);
    for (unsigned r = 0; r < nc; r++) best = max(best, sh.xc[turn][r]);
    top = smp_type<float>::value(best);
    if (top == -INFINITY || !(t > 0.0f)) {               // nothing to draw from, or the largest logit itself
        unsigned at = 0xffffffffu;
        if (top > -INFINITY) {
            x.each([&](float v, int i) { if (v == top) at = min(at, (unsigned)(first + i)); });
            at = __reduce_min_sync(0xffffffffu, at);
            __syncthreads();
            if (lane == 0) sh.redc[warp] = at;
            __syncthreads();
            for (int i = 0; i < SMP_WARPS; i++) at = min(at, sh.redc[i]);
            smp_post(sh, rank, nc, turn, 0, at);
            for (unsigned r = 0; r < nc; r++) at = min(at, sh.xc[turn][r]);
        }
        if (rank == 0 && threadIdx.x == 0) {
            p.token[row] = (int)at;
            if (p.logprob) p.logprob[row] = at == 0xffffffffu ? -INFINITY : 0.0f;
        }
        return;
    }
    x.mode = top == INFINITY ? SMP_INFINITE : top < -1e30f ? SMP_LOW : SMP_PLAIN;
    x.top = top;
    if (x.mode != SMP_PLAIN) {
        if (!FAR)
            for (int j = 0; j < x.words; j++) {
                const unsigned w = x.data[j];
                x.data[j] = ty::put(smp_shift(ty::get(w, 0), x.mode, top), smp_shift(ty::get(w, ty::N - 1), x.mode, top));
            }
        top = 0.0f;
    }
    // T is at most 1e20, so that the floor, 48 T ln 2 under the largest, is a finite number, and at least 2^-30 |max|, below
    // which numbers next to the largest weigh nothing all the same
    smp_row q;
    const double temp = fmax(fmin((double)t, 1e20), fabs((double)top) * 9.3132257461547852e-10);
    const float reach = __double2float_ru((p.kbits + 2) * 0.69314718055994531 * temp);
    q.tab = sh.tab;
    q.maxf = top;
    q.c = 184.66496523378731354 / temp;                  // 128 log2(e) / T
    q.at_max = (double)top * q.c;
    q.floor = __fsub_rd(top, reach);
    q.one = smp_weight(p, q, top);
    q.step = (float)fmin(2.0 * 2047.6 / (double)reach, 3.0e38);
    smp_settings s;
    s.k = k > 0 && k < p.n ? k : 0;
    s.part = tp >= 1.0f || tp != tp ? 0 : tp > 0.0f ? max((uint64_t)((double)tp * 4611686018427387904.0), (uint64_t)1) : 1;
    s.least = mp > 0.0f ? (uint64_t)ceil((double)fminf(mp, 1.0f) * (double)q.one) : 0;
    s.u = un > 0.0f ? fminf(un, 0.99999994f) : 0.0f;
    s.whole = 0;

    smp_cut cut = {q.floor, 0};                          // (at the floor nothing weighs)
    uint64_t kept = 0;                                   // this thread's kept weight and its tokens at the threshold, when `known`
    unsigned at_cut = 0;
    bool tallied = false, known = false;
    if (s.k || s.part) {
        smp_clear(sh, false);
        unsigned *cells = sh.cnt;                        // what has no weight goes behind them, each lane to a place of its own
        x.each([&](float v, int) { atomicAdd(cells + smp_cell(q, v, IRX_SMP_BINS + lane), 1u); });
        tallied = true;
    }
    if (s.k) {
        uint64_t target = s.k;
        if (!smp_find(sh, rank, nc, turn, SMP_COUNT, target, 0)) s.k = 0;      // fewer have any weight: all of those
        else if (sh.above + sh.count <= SMP_FEW) {
            const unsigned cell = sh.cell, below = smp_last(smp_least<T>(q), ty::key(q.maxf), [&](unsigned kk) { return smp_cell(q, ty::value(kk)) > cell; });
            smp_pick(x, ty::value(below), INFINITY, [&](float v, int i) { sh.mine[atomicAdd(&sh.few, 1u)] = smp_token(v, first + i); });
            __syncthreads();
            const unsigned n = sh.few;
            unsigned at = 0, m = 0;
            smp_post(sh, rank, nc, turn, 0, n);
            for (unsigned r = 0; r < nc; r++) {
                if (r == rank) at = m;
                m += sh.xc[turn][r];
            }
            smp_hand_over(sh, n, at);
            if (rank == 0) smp_finish(p, sh, q, m, row, s);
            return;
        } else {
            cut = smp_resolve(p, sh, q, x, rank, nc, turn, false, target, true);
            tallied = false;
        }
    }
    bool found = false;
    if (s.part && tallied) {
        // Top-p alone. The cell of its threshold is guessed from the cells' tokens; one pass then adds up the row's weight and
        // that above the cell, and gathers the tokens in it (in the next one too, when the guess is near its edge). If the
        // threshold does not lie among them, or they are too many, the weights' own histogram follows. With few tokens
        // from there up, all of them are gathered.
        uint64_t target = 0;
        smp_find(sh, rank, nc, turn, SMP_GUESS, target, s.part, (float)(2.0 * q.c / 128.0 / (double)q.step));
        const float in_cell = (float)(target - sh.before) / (float)sh.weight;
        const unsigned least = smp_least<T>(q), tk = ty::key(q.maxf), c0 = sh.cell - (in_cell < 0.2f && sh.cell), c1 = sh.cell + (in_cell > 0.8f);
        const bool few = sh.above + sh.count <= SMP_FEW / 2;
        const unsigned kb = smp_last(least, tk, [&](unsigned kk) { return smp_cell(q, ty::value(kk)) > min(c1, IRX_SMP_BINS - 1u); });
        const unsigned ko = few ? tk : smp_last(least, tk, [&](unsigned kk) { return smp_cell(q, ty::value(kk)) >= c0; });
        const float below = ty::value(kb), over = ty::value(ko);
        uint64_t sum[3] = {0, 0, 0};                     // the whole, what is over the gathered cells, what is in them
        for (int j0 = 0; j0 < x.words; j0 += SMP_STEP) {
            unsigned hits = 0;
#pragma unroll
            for (int j = 0; j < SMP_STEP; j++) {
                const unsigned word = j0 + j < x.words ? x.word(j0 + j) : ty::PAD;
#pragma unroll
                for (int h = 0; h < ty::N; h++) {
                    const float v = ty::get(word, h);
                    const uint64_t w = smp_raw(p, q, fmaxf(v, q.floor));
                    sum[0] += w;
                    sum[1] += v > over ? w : SMP_RAW;
                    if (v > below && v <= over) hits |= 1u << (j * ty::N + h);
                }
            }
            for (; hits; hits &= hits - 1) {
                const int b = __ffs(hits) - 1;
                const float v = ty::get(x.word(j0 + b / ty::N), b % ty::N);
                sum[2] += smp_weight(p, q, v);
                const unsigned at = atomicAdd(&sh.few, 1u);
                if (at < SMP_FEW) sh.mine[at] = smp_token(v, first + j0 * ty::N + b);
            }
        }
        const uint64_t read = (uint64_t)((x.words + SMP_STEP - 1) / SMP_STEP * SMP_STEP * ty::N) * SMP_RAW;
        sum[0] -= read;
        sum[1] -= read;
        const uint64_t own = sum[1];
        unsigned none = 0, at = 0, m = 0;
        smp_block_sums(sh, sum, none);
        const unsigned n = sh.few;
        smp_post(sh, rank, nc, turn, sum[0], n, sum[1], sum[2]);
        uint64_t above = 0, in = 0;
        for (unsigned r = 0; r < nc; r++) {
            if (r == rank) at = m;
            m = min(m + sh.xc[turn][r], SMP_FEW + 1u);
            s.whole += sh.xa[turn][r];
            above += sh.xb[turn][r];
            in += sh.xd[turn][r];
        }
        target = max(smp_part(s.part, s.whole, true), (uint64_t)1);
        found = m <= SMP_FEW && above < target && target <= above + in;
        if (found) {
            smp_hand_over(sh, n, at);
            if (few) {
                if (rank == 0) smp_finish(p, sh, q, m, row, s);
                return;
            }
            cut = smp_among<T>(p, sh, q, rank, nc, m, kb + 1, ko, target - above, true);
            if (!s.least) {                              // what is kept of the gathered cells, to the threads that it came from
                unsigned *lo = reinterpret_cast<unsigned *>(sh.list), *hi = lo + IRX_SMP_THREADS, *eq = hi + IRX_SMP_THREADS;
                lo[threadIdx.x] = hi[threadIdx.x] = eq[threadIdx.x] = 0;
                __syncthreads();
                for (unsigned i = threadIdx.x; i < n; i += IRX_SMP_THREADS) {
                    const float v = smp_number(sh.mine[i]);
                    const int whose = (int)((unsigned)sh.mine[i] - base) / (p.words * ty::N);
                    if (v > cut.above) {
                        const uint64_t w = smp_weight(p, q, v);
                        const unsigned wl = (unsigned)w, old = atomicAdd(&lo[whose], wl);
                        atomicAdd(&hi[whose], (unsigned)(w >> 32) + (old + wl < old));
                    } else if (cut.ties && v == cut.above) atomicAdd(&eq[whose], 1u);
                }
                __syncthreads();
                kept = own + ((uint64_t)hi[threadIdx.x] << 32 | lo[threadIdx.x]);
                at_cut = eq[threadIdx.x];
                known = true;
            }
        } else {
            __syncthreads();
            if (threadIdx.x == 0) sh.few = 0;
        }
    }
    if (s.part && !found) {
        // the weights of what top-k kept, by cell; of those at its threshold only the first
        smp_clear(sh, true);
        x.each([&](float v, int) {
            const unsigned cell = smp_cell(q, v);
            if (v > cut.above && cell < IRX_SMP_BINS) smp_tally(sh, cell, true, smp_weight(p, q, v));
        });
        if (cut.ties && rank == 0) {
            __syncthreads();
            const unsigned cell = smp_cell(q, cut.above);
            if (threadIdx.x == 0 && cell < IRX_SMP_BINS) {
                const uint64_t sum = ((uint64_t)sh.hi[cell] << 32 | sh.lo[cell]) + cut.ties * smp_weight(p, q, cut.above);
                sh.lo[cell] = (unsigned)sum;
                sh.hi[cell] = (unsigned)(sum >> 32);
            }
        }
        uint64_t target = 0;
        smp_find(sh, rank, nc, turn, SMP_WEIGHT, target, s.part);
        const smp_cut c = smp_resolve(p, sh, q, x, rank, nc, turn, true, target, !s.k);
        if (c.above > cut.above || (c.above == cut.above && c.ties < cut.ties)) cut = c;
    }
    if (s.least) {                                       // min-p as a threshold: the last number that weighs too little
        const unsigned key = smp_last(smp_least<T>(q), ty::key(q.maxf), [&](unsigned kk) { return smp_weight(p, q, ty::value(kk)) < s.least; });
        const float v = ty::value(key);
        if (v >= cut.above) cut = {v, 0};
    }

    // the kept weights of every thread's stretch of the row, and where u times their total falls. What is not kept counts as
    // at the floor, with no weight; words of which no lane of a warp keeps any are passed over.
    const uint64_t w_eq = cut.ties ? smp_weight(p, q, cut.above) : 0;
    uint64_t sums[1] = {kept};
    unsigned eq = at_cut;
    if (known) {
    } else if (cut.above == q.floor) {                   // nothing is cut: no floor but the weights' own
        x.each([&](float v, int) { sums[0] += smp_raw(p, q, fmaxf(v, q.floor)); });
        sums[0] -= (uint64_t)(x.words * ty::N) * SMP_RAW;
    } else for (int j0 = 0; j0 < x.words; j0 += SMP_STEP) {
        float v[SMP_STEP * ty::N];
        bool any = false;
#pragma unroll
        for (int j = 0; j < SMP_STEP; j++) {
            const unsigned word = j0 + j < x.words ? x.word(j0 + j) : ty::PAD;
#pragma unroll
            for (int h = 0; h < ty::N; h++) {
                v[j * ty::N + h] = ty::get(word, h);
                any |= v[j * ty::N + h] >= cut.above;
            }
        }
        if (!__any_sync(0xffffffffu, any)) continue;
        if (cut.ties)
#pragma unroll
            for (int j = 0; j < SMP_STEP * ty::N; j++) eq += v[j] == cut.above;
#pragma unroll
        for (int j = 0; j < SMP_STEP * ty::N; j++) sums[0] += smp_raw(p, q, v[j] > cut.above ? v[j] : q.floor) - SMP_RAW;
    }
    const uint64_t w_mine = sums[0];
    const unsigned eq_mine = eq;
    smp_block_sums(sh, sums, eq);
    smp_post(sh, rank, nc, turn, sums[0], eq);
    uint64_t total = 0, run = 0;
    unsigned ties = cut.ties, left = 0;                  // ties: left to keep; left: of them, for this block
    for (unsigned r = 0; r < nc; r++) {
        const unsigned have = min(ties, sh.xc[turn][r]);
        if (r == rank) {
            run = total;
            left = ties;
        }
        total += sh.xa[turn][r] + have * w_eq;
        ties -= have;
    }
    const uint64_t at = smp_part((uint64_t)((double)s.u * 4611686018427387904.0), total, false);
    if (at < run || at >= run + sums[0] + min(left, eq) * w_eq) return;      // one block goes on
    for (int i = 0; i < warp; i++) {
        const unsigned have = min(left, sh.redc[i]);
        run += sh.red[0][i] + have * w_eq;
        left -= have;
    }
    if (at < run || at >= run + sh.red[0][warp] + min(left, sh.redc[warp]) * w_eq) return;      // one warp
    const unsigned before = (unsigned)smp_warp_scan(eq_mine) - eq_mine;
    left -= min(left, before);
    const uint64_t own = w_mine + min(left, eq_mine) * w_eq, sum = smp_warp_scan(own);
    const int who = __ffs(__ballot_sync(0xffffffffu, run + sum > at)) - 1;             // the lane whose stretch it is
    run = __shfl_sync(0xffffffffu, run + sum - own, who);
    left = __shfl_sync(0xffffffffu, left, who);
    const int64_t off = (int64_t)(warp * 32 + who) * p.words;
    const smp_data<T, FAR> y = {data + off, src + off * ty::N, p.n - base - off * ty::N, p.words, x.mode, x.top};
    for (int i0 = 0; i0 < p.words * ty::N; i0 += 32) {
        const int i = i0 + lane;
        const float v = i < p.words * ty::N ? ty::get(y.word(i / ty::N), i % ty::N) : -INFINITY;
        const bool same = cut.ties && v == cut.above;
        const unsigned all = __ballot_sync(0xffffffffu, same);
        const uint64_t e = v > cut.above || (same && __popc(all & ((1u << lane) - 1u)) < left) ? smp_weight(p, q, v) : 0;
        left -= min(left, (unsigned)__popc(all));
        const uint64_t up = smp_warp_scan(e);
        const unsigned past = __ballot_sync(0xffffffffu, run + up > at);
        if (past) {
            if (lane == __ffs(past) - 1) {
                p.token[row] = (int)(base + off * ty::N + i);
                if (p.logprob) p.logprob[row] = (float)log((double)e / (double)total);
            }
            return;
        }
        run += __shfl_sync(0xffffffffu, up, 31);
    }
}

extern "C" __global__ void __launch_bounds__(IRX_SMP_THREADS) irx_sample_bf16(const __grid_constant__ irx_ksmp_t p) { smp_body<__nv_bfloat16, false>(p); }
extern "C" __global__ void __launch_bounds__(IRX_SMP_THREADS) irx_sample_bf16_far(const __grid_constant__ irx_ksmp_t p) { smp_body<__nv_bfloat16, true>(p); }
extern "C" __global__ void __launch_bounds__(IRX_SMP_THREADS) irx_sample_f32(const __grid_constant__ irx_ksmp_t p) { smp_body<float, false>(p); }
extern "C" __global__ void __launch_bounds__(IRX_SMP_THREADS) irx_sample_f32_far(const __grid_constant__ irx_ksmp_t p) { smp_body<float, true>(p); }
