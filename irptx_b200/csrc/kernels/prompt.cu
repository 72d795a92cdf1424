// prompt.cu -- causal attention over packed prompts: O = softmax(Q K^T * scale, masked) V, sequence by
// sequence, grouped heads.
//
// Sequence s is the tokens [starts[s], starts[s + 1]) of the packed rows; token i of a sequence sees
// its tokens j <= i, with a window those with j > i - window or j < sinks. The query heads that share a
// key-value head are rows of the same tiles: row r of a (sequence, key-value head) is token
// r / group, head r % group, so a short prompt fills a tile with its heads and every key tile
// read serves the whole group.
//
// A unit is one tile of rows of one (sequence, key-value head). The blocks find their units from
// `starts` alone, heaviest first: units are numbered by their tile's place in its sequence,
// from the last place down, and the blocks take them in turns; nothing on the host and no
// counter in memory is needed, and a row's result does not depend on which block takes it.
#pragma once
#include "tc.cuh"

struct pr_unit { int base, len, tile, head; };          // first row of the sequence, its tokens, tile, kv head

// Tokens of sequence s0 + lane (0 past the last one), and its first row. 0 too, and `bad`, when its starts fall, leave the
// packed rows, or an earlier start is above its own: then no two sequences share a row. highest: the largest
// start so far, INT_MIN at first. A whole warp calls it.
__device__ __forceinline__ int pr_len(const irx_kprm_t &p, int s0, int &highest, int &base, bool &bad)
{
    const int lane = threadIdx.x & 31, s = s0 + lane;
    int a = 0x80000000, b = 0;
    if (s < p.batch) {
        a = p.starts[s];
        b = p.starts[s + 1];
    }
    int m = a;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, m, o);
        if (lane >= o) m = max(m, x);
    }
    m = max(m, highest);
    highest = __shfl_sync(0xffffffffu, m, 31);
    base = a;
    bad = s < p.batch && (a < 0 || b < a || b > p.tokens || m > a);
    return s < p.batch && !bad ? b - a : 0;
}

// Tiles of a sequence of n tokens: mul rows a token, per rows a tile.
struct pr_rows {
    int mul, per;
    __device__ __forceinline__ int tiles(int n) const
    {
        if (mul == 1) return (int)(((unsigned)n + (unsigned)per - 1) / (unsigned)per);
        return (int)(((int64_t)n * mul + per - 1) / per);
    }
};

// What a warp knows of all units: the first 32 sequences (one a lane), the most tiles of one, the units.
struct pr_list {
    pr_rows rows;
    int tiles, base, len, highest, most;
    int64_t units;
};

// Tiles of sequence s0 + lane, its rows and the state for the next 32.
__device__ __forceinline__ int pr_chunk(const irx_kprm_t &p, const pr_list &l, int s0, int &highest, int &base, int &len)
{
    if (!s0) {
        highest = l.highest;
        base = l.base;
        len = l.len;
        return l.tiles;
    }
    bool bad;
    len = pr_len(p, s0, highest, base, bad);
    return l.rows.tiles(len);
}

// A whole warp calls these. pr_start: the list; block 0 reports the sequences that are skipped.
__device__ __forceinline__ pr_list pr_start(const irx_kprm_t &p, pr_rows rows)
{
    pr_list l;
    l.rows = rows;
    l.highest = 0x80000000;
    int sum = 0, most = 0, highest = 0x80000000, base, len;
    for (int s0 = 0; s0 < p.batch; s0 += 32) {
        bool bad;
        len = pr_len(p, s0, highest, base, bad);
        if (bad && blockIdx.x == 0) atomicOr(p.err, IRX_KERR_INDEX);
        const int n = rows.tiles(len);
        if (!s0) {
            l.tiles = n;
            l.base = base;
            l.len = len;
            l.highest = highest;
        }
        sum += n;
        most = max(most, n);
    }
    l.most = __reduce_max_sync(0xffffffffu, most);
    l.units = (int64_t)__reduce_add_sync(0xffffffffu, sum) * (p.h1 - p.h0);
    return l;
}

// Unit u, below l.units.
__device__ __forceinline__ pr_unit pr_find(const irx_kprm_t &p, const pr_list &l, int64_t u)
{
    const int nh = p.h1 - p.h0, lane = threadIdx.x & 31;
    int lo = 0, hi = l.most, after = 0;                  // after: tiles numbered hi and later, a head
    while (hi - lo > 1) {                                // the last t with u below the units of tiles t and later, 32 guesses at a time
        const int step = (hi - lo + 31) / 32, t = lo + (lane + 1) * step;
        int c = 0, highest, base, len;
        for (int s0 = 0; s0 < p.batch; s0 += 32) {
            const int nt = pr_chunk(p, l, s0, highest, base, len), n = min(32, p.batch - s0);
            for (int i = 0; i < n; i++) c += max(0, __shfl_sync(0xffffffffu, nt, i) - t);
        }
        const int k = __popc(__ballot_sync(0xffffffffu, t < hi && (int64_t)c * nh > u));
        if (lo + (k + 1) * step < hi) {
            hi = lo + (k + 1) * step;
            after = __shfl_sync(0xffffffffu, c, k);
        }
        lo += k * step;
    }
    const int off = (int)(u - (int64_t)after * nh);
    int skip = off / nh, highest;                        // among the sequences that have a tile number lo
    pr_unit r = {0, 0, lo, p.h0 + off % nh};
    for (int s0 = 0; s0 < p.batch; s0 += 32) {
        int base, len;
        const unsigned has = __ballot_sync(0xffffffffu, pr_chunk(p, l, s0, highest, base, len) > lo);
        const int c = __popc(has);
        if (skip < c) {
            const int at = __fns(has, 0, skip + 1);
            r.base = __shfl_sync(0xffffffffu, base, at);
            r.len = __shfl_sync(0xffffffffu, len, at);
            break;
        }
        skip -= c;
    }
    return r;
}

// This block's unit of turn i: the blocks take turns forwards and backwards, so that none has the heaviest of each.
__device__ __forceinline__ int64_t pr_turn(int i)
{
    return (int64_t)i * gridDim.x + (i & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}

// ---- FP32 units: f32 rows, and bf16 rows that the matrix instructions do not take ----
//
// 64 query rows against tiles of 64 keys, as f32 in shared memory: keys and values each in a buffer of their own, so that
// values arrive while scores are computed and the next keys during the second product; two blocks fit an SM up to 128
// columns. A thread holds R x 4 scores and R rows x DP / 16 columns of the output in registers and multiplies two numbers an
// instruction; a 16-byte read costs its four accesses of the shared memory also where lanes read the same, so at R = 4 that
// memory is busier than the FP32 units (71 and 61 %). R = 8 (128 threads) reads less (44 and 56 %) and has half the warps: 147 against 154 us
// for 2093 tokens in five prompts, 16 heads on 4 of 128; at 64 columns 87 against 86, so 4 there, and above 128, where the
// registers end. A key row's groups of four floats are permuted by the row's place in its eight, so that the 16 key
// rows read together fall into different banks.
#define PS_ROWS 64
#define PS_KEYS 64

// n rows of d numbers into 64 rows of DP, zeros behind both; f32 rows of whole 16 bytes asynchronously
template <int DP, int NT, bool SWZ>
__device__ __forceinline__ void ps_fill(float *dst, const void *src, int dt, int64_t row0, int64_t stride, int64_t off, int n, int d, bool vec)
{
    if (vec && dt == DT_F32) {
        const float *from = reinterpret_cast<const float *>(src) + row0 * stride + off;
#pragma unroll
        for (int e0 = 0; e0 < 64 * (DP / 4); e0 += NT) {
            const int e = e0 + threadIdx.x, r = e / (DP / 4), c = (e % (DP / 4)) * 4;
            const bool there = r < n && c < d;
            cp16(irx_smem_u32(dst + r * DP + (SWZ ? c ^ (r & 7) << 2 : c)), there ? from + r * stride + c : from, there ? 16 : 0);
        }
        return;
    }
    for (int e = threadIdx.x; e < 64 * DP; e += NT) {
        const int r = e / DP, c = e % DP;
        dst[r * DP + (SWZ ? c ^ (r & 7) << 2 : c)] = r < n && c < d ? irx_ld1(src, dt, (row0 + r) * stride + off + c) : 0.0f;
    }
}

template <int DP, int R>
__device__ __forceinline__ void ps_body(const irx_kprm_t &p)
{
    irx_pdl_enter();
    extern __shared__ __align__(16) float ps_smem[];
    float *sq = ps_smem, *sk = sq + 64 * DP, *sv = sk + 64 * DP, *sp = sv + 64 * DP;       // queries, keys, values, weights
    constexpr int NC = DP / 64, NT = 1024 / R;           // 4-column groups of the output a thread owns; threads
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, odd = ty & 1;      // of a warp's two fours of rows, the second has
    const pr_list list = pr_start(p, pr_rows{p.group, PS_ROWS});               // its queries and weights in other banks
    for (int turn = 0;; turn++) {
        const int64_t u = pr_turn(turn);
        if (u >= list.units) break;
        const pr_unit un = pr_find(p, list, u);
        const int64_t r0 = (int64_t)un.tile * PS_ROWS, rows = (int64_t)un.len * p.group;
        const int nr = (int)min((int64_t)PS_ROWS, rows - r0);
        const int first = (int)(r0 / p.group), skip = (int)(r0 - (int64_t)first * p.group), last = first + (skip + nr - 1) / p.group;
        const int lo = p.window ? max(0, first - p.window + 1) : 0, sinks = min(p.sinks, lo);
        const int nsink = (sinks + PS_KEYS - 1) / PS_KEYS, ntiles = nsink + (last - lo) / PS_KEYS + 1;
        auto begin = [&](int kt) { return kt < nsink ? kt * PS_KEYS : lo + (kt - nsink) * PS_KEYS; };
        auto end = [&](int kt) { return kt < nsink ? sinks : last + 1; };
        auto keys = [&](int kt) {
            ps_fill<DP, NT, true>(sk, p.k, p.dt, un.base + begin(kt), p.kv_stride, (int64_t)un.head * p.d, min(PS_KEYS, end(kt) - begin(kt)), p.d, p.vec);
            cp_commit();
        };
        __syncthreads();                                 // the unit before is done with
        if (p.vec && p.dt == DT_F32) {
#pragma unroll
            for (int e0 = 0; e0 < 64 * (DP / 4); e0 += NT) {
                const int e = e0 + threadIdx.x, r = e / (DP / 4), c = (e % (DP / 4)) * 4, t = (skip + r) / p.group;
                const bool there = r < nr && c < p.d;
                const float *from = reinterpret_cast<const float *>(p.q) + (un.base + first + t) * p.q_stride
                                    + (int64_t)(un.head * p.group + skip + r - t * p.group) * p.d + c;
                cp16(irx_smem_u32(sq + r * DP + (c ^ (r / R & 1) << 2)), there ? (const void *)from : p.q, there ? 16 : 0);
            }
        } else
            for (int e = threadIdx.x; e < 64 * DP; e += NT) {
                const int r = e / DP, c = e % DP, t = (skip + r) / p.group;
                sq[r * DP + (c ^ (r / R & 1) << 2)] = r < nr && c < p.d ? irx_ld1(p.q, p.dt, (un.base + first + t) * p.q_stride
                                                                         + (int64_t)(un.head * p.group + skip + r - t * p.group) * p.d + c) : 0.0f;
            }
        keys(0);
        int tok[R];
        float m[R], l[R];
        float2 o[R][NC * 2];
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int r = min(ty * R + i, nr - 1);
            tok[i] = first + (skip + r) / p.group;
            m[i] = -3.0e38f;
            l[i] = 0.0f;
#pragma unroll
            for (int c = 0; c < NC * 2; c++) o[i][c] = make_float2(0.0f, 0.0f);
        }
        for (int kt = 0; kt < ntiles; kt++) {
            const int kb = begin(kt), kend = end(kt), nk = min(PS_KEYS, kend - kb);
            // a tile that some row does not see in whole: masked, and what is hidden passed over
            const bool cut = kt < nsink || nk < PS_KEYS || kb + PS_KEYS - 1 > first || (p.window && kb <= last - p.window);
            cp_wait<0>();
            __syncthreads();                             // the keys are there, the values before are done with
            ps_fill<DP, NT, false>(sv, p.v, p.dt, un.base + kb, p.kv_stride, (int64_t)un.head * p.d, nk, p.d, p.vec);
            cp_commit();
            float2 s2[R][4];
#pragma unroll
            for (int i = 0; i < R; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) s2[i][j] = make_float2(0.0f, 0.0f);
#pragma unroll (R == 8 ? 2 : 4)
            for (int c = 0; c < DP; c += 4) {
                float4 a[R], b[4];
#pragma unroll
                for (int i = 0; i < R; i++)
                    a[i] = *reinterpret_cast<const float4 *>(sq + (ty * R + i) * DP + (c ^ odd << 2));
#pragma unroll
                for (int j = 0; j < 4; j++)
                    b[j] = *reinterpret_cast<const float4 *>(sk + (tx + 16 * j) * DP + (c ^ (tx & 7) << 2));
#pragma unroll
                for (int i = 0; i < R; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        s2[i][j] = __ffma2_rn(make_float2(a[i].z, a[i].w), make_float2(b[j].z, b[j].w),
                                              __ffma2_rn(make_float2(a[i].x, a[i].y), make_float2(b[j].x, b[j].y), s2[i][j]));
            }
            float s[R][4];
#pragma unroll
            for (int i = 0; i < R; i++) {
                float mx = -3.0e38f;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int key = kb + tx + 16 * j;
                    s[i][j] = (s2[i][j].x + s2[i][j].y) * p.scale2;
                    if (cut && (key >= kend || key > tok[i] || (p.window && key <= tok[i] - p.window && key >= p.sinks))) s[i][j] = -INFINITY;
                    mx = s[i][j] > mx || s[i][j] != s[i][j] ? s[i][j] : mx;      // a NaN stays
                }
#pragma unroll
                for (int x = 8; x; x >>= 1) {
                    const float y = __shfl_xor_sync(0xffffffffu, mx, x);
                    mx = y > mx || y != y ? y : mx;
                }
                const float mn = m[i] > mx || m[i] != m[i] ? m[i] : mx, r = exp2f(m[i] - mn);
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float w = exp2f(s[i][j] - mn);
                    sum += w;                            // a weight of -0: of a score of -infinity, not one that vanished
                    sp[(ty * R + i) * 64 + tx + (16 * j ^ odd << 4)] = s[i][j] == -INFINITY ? -0.0f : w;
                }
                m[i] = mn;
                l[i] = l[i] * r + sum;                   // of this lane's keys: joined at the end
#pragma unroll
                for (int c = 0; c < NC * 2; c++) o[i][c] = __fmul2_rn(o[i][c], make_float2(r, r));
            }
            cp_wait<0>();
            __syncthreads();                             // the values are there, the keys done with (a row's weights are made and read by one half warp)
            if (kt + 1 < ntiles) keys(kt + 1);
#pragma unroll 2
            for (int j0 = 0; j0 < PS_KEYS; j0 += 4) {
                float w[R][4];
#pragma unroll
                for (int i = 0; i < R; i++) {
                    const float4 x = *reinterpret_cast<const float4 *>(sp + (ty * R + i) * 64 + (j0 ^ odd << 4));
                    w[i][0] = x.x; w[i][1] = x.y; w[i][2] = x.z; w[i][3] = x.w;
                }
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int g = 0; g < NC; g++) {
                        const float4 x = *reinterpret_cast<const float4 *>(sv + (j0 + j) * DP + g * 64 + tx * 4);
#pragma unroll
                        for (int i = 0; i < R; i++) {
                            if (cut && __float_as_uint(w[i][j]) == 0x80000000u) continue;
                            o[i][g * 2] = __ffma2_rn(make_float2(w[i][j], w[i][j]), make_float2(x.x, x.y), o[i][g * 2]);
                            o[i][g * 2 + 1] = __ffma2_rn(make_float2(w[i][j], w[i][j]), make_float2(x.z, x.w), o[i][g * 2 + 1]);
                        }
                    }
            }
        }
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int r = ty * R + i;
#pragma unroll
            for (int x = 8; x; x >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
            if (r >= nr) continue;
            const int h = un.head * p.group + skip + r - (tok[i] - first) * p.group;
            const int64_t row = (int64_t)(un.base + tok[i]) * p.heads + h;
            const float inv = 1.0f / l[i];
            if (p.lse && tx == 0) p.lse[row] = (m[i] + log2f(l[i])) * 0.6931471806f;
#pragma unroll
            for (int g = 0; g < NC; g++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const int col = g * 64 + tx * 4 + c;
                    if (col < p.d) irx_st1(p.o, p.dt, row * p.d + col, (c & 1 ? o[i][g * 2 + c / 2].y : o[i][g * 2 + c / 2].x) * inv);
                }
        }
    }
}

#define PS_KERNEL(DP, B) extern "C" __global__ void __launch_bounds__(IRX_PR_ST_THREADS(DP), B) irx_prompt_st_##DP(const __grid_constant__ irx_kprm_t p) { ps_body<DP, 1024 / IRX_PR_ST_THREADS(DP)>(p); }
PS_KERNEL(64, 2)
PS_KERNEL(128, 2)
PS_KERNEL(256, 1)
