// prompt_tc.cu -- attention over packed prompts on the 5th-generation tensor cores: bf16, head sizes up to 128
// in multiples of 8, up to 128 query heads a key-value head.
//
// A unit is two 128-row tiles of one (sequence, key-value head): tp = 128 / group tokens each with all
// their heads, loaded as one box of the queries (64 columns, group, 1, tp). Keys and values come in tiles of
// 128 tokens, boxes that begin at any row; columns past the head size are filled with zeros by the
// copy. The pipeline is irx_attn_bf16's (attn.cu): scores S_t = Q_t K^T into TMEM, one thread a row for the softmax,
// P over the scores' columns, O_t += P_t V, each tile's softmax under the other tile's products. What differs:
//   * warp 8 finds the block's units from `starts` (prompt.cu) and hands them out with the loads;
//   * key tiles may begin anywhere and are masked by token: a window's edge and the sinks' tiles too;
//   * warps 10 and 11 look through the values of the tiles that a mask cuts. Rows that no query of the unit
//     sees become zeros, for another sequence's numbers or uninitialised ones may lie there and 0 * NaN is NaN.
//     Infinities and NaN in the others become zeros too, and the unit is marked: its rows add those that they
//     see at the end. Tiles seen in whole need neither.
#pragma once
#include "prompt.cu"

struct pt_info { int base, len, tok0, head, lo, nsink, n0, n1, sk, end, dirty; };

__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, int c0, int c1, int c2, int c3, uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 :: "r"(irx_smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3),
                    "r"(irx_smem_u32(bar)) : "memory");
}

// The largest of three, NaN if one of them is.
__device__ __forceinline__ float pt_max3(float a, float b, float c)
{
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// First token of key tile j, and whether some row of tokens [first, last] does not see all of it.
__device__ __forceinline__ int pt_key(const pt_info &f, int j) { return j < f.nsink ? 128 * j : f.lo + 128 * (j - f.nsink); }

__device__ __forceinline__ bool pt_cut(const irx_kprm_t &p, const pt_info &f, int j, int first, int last)
{
    const int kb = pt_key(f, j);
    return j < f.nsink || kb + 127 > first || (p.window && kb <= last - p.window);
}

// The lowest n bits, n any number.
__device__ __forceinline__ uint32_t pt_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

#define PT_HALF 16384                       // 128 rows of 64 columns

template <int DP>
__device__ __forceinline__ void pt_body(const irx_kprm_t &p)
{
    constexpr int NB = DP / 64, TILE = NB * PT_HALF;
    irx_pdl_enter();
    extern __shared__ __align__(1024) unsigned char pt_smem[];
    unsigned char *sq = pt_smem, *sk = sq + 2 * TILE, *sv = sk + 2 * TILE;
    if (irx_smem_u32(pt_smem) & 1023u) {
        if (threadIdx.x == 0) atomicOr(p.err, IRX_KERR_TIMEOUT);
        return;
    }
    uint64_t *bars = reinterpret_cast<uint64_t *>(sv + 2 * TILE);
    uint64_t *q_full = bars, *k_full = bars + 1, *k_empty = bars + 3, *v_full = bars + 5, *v_empty = bars + 7;
    uint64_t *s_full = bars + 9, *p_full = bars + 11, *pv_done = bars + 13, *done = bars + 15, *q_empty = bars + 16, *o_free = bars + 17;
    uint64_t *u_full = bars + 19, *u_empty = bars + 21, *v_ok = bars + 23;
    uint32_t *tslot = reinterpret_cast<uint32_t *>(bars + 25);
    volatile pt_info *infos = reinterpret_cast<volatile pt_info *>(bars + 26);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = p.group, tp = 128 / g;
    if (threadIdx.x < 25) {
        const int i = threadIdx.x;          // p_full, o_free: a tile's rows; u_empty: MMA, 8 softmax and 2 value warps
        irx_mbar_init(&bars[i], i == 11 || i == 12 || i == 17 || i == 18 ? 128 : i == 21 || i == 22 ? 11 : i >= 23 ? 2 : 1);
        irx_fence_mbar_init();
        if (i == 0) {
            tma_prefetch_desc(&p.tma_q);
            tma_prefetch_desc(&p.tma_k);
            tma_prefetch_desc(&p.tma_v);
        }
    }
    if (warp == 9) tmem_alloc(tslot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = *tslot;
    auto read = [&](int us) {
        pt_info f;
        f.base = infos[us].base; f.len = infos[us].len; f.tok0 = infos[us].tok0; f.head = infos[us].head;
        f.lo = infos[us].lo; f.nsink = infos[us].nsink; f.n0 = infos[us].n0; f.n1 = infos[us].n1; f.sk = infos[us].sk;
        f.end = infos[us].end; f.dirty = 0;
        return f;
    };
    if (warp >= 8) {
      at_reg_dec();
      if (warp == 8) {                                        // units and loads
        int kv = 0;
        const pr_list list = pr_start(p, pr_rows{1, 2 * tp});
        int ok = 1;
        for (int uc = 0; ok; uc++) {
            const int us = uc & 1;
            const int64_t u = pr_turn(uc);
            pt_info f = {};
            if (u < list.units) {
                const pr_unit un = pr_find(p, list, u);
                f.base = un.base; f.len = un.len; f.head = un.head;
                f.tok0 = un.tile * 2 * tp;
                const int e0 = min(f.tok0 + tp, f.len), e1 = min(f.tok0 + 2 * tp, f.len);
                f.end = e1;
                f.lo = p.window ? max(0, f.tok0 - p.window + 1) : 0;
                f.sk = min(p.sinks, f.lo);
                f.nsink = (f.sk + 127) / 128;
                f.n0 = f.nsink + (e0 - f.lo + 127) / 128;
                f.n1 = e1 > e0 ? f.nsink + (e1 - f.lo + 127) / 128 : 0;
            }
            if (lane == 0) {
                ok = at_wait(&u_empty[us], ((uc >> 1) & 1) ^ 1, p.err);
                if (ok) {
                    infos[us].base = f.base; infos[us].len = f.len; infos[us].tok0 = f.tok0; infos[us].head = f.head;
                    infos[us].lo = f.lo; infos[us].nsink = f.nsink; infos[us].n0 = f.n0; infos[us].n1 = f.n1;
                    infos[us].sk = f.sk; infos[us].end = f.end; infos[us].dirty = 0;
                    irx_mbar_arrive(&u_full[us]);
                }
                if (ok && f.n0) {
                    const int nmax = max(f.n0, f.n1), nt = f.n1 ? 2 : 1;
                    if (uc > 0) ok = at_wait(q_empty, (uc - 1) & 1, p.err);
                    if (ok) {
                        irx_mbar_expect_tx(q_full, (uint32_t)(nt * NB * tp * g * 128));
                        for (int t = 0; t < nt; t++)
                            for (int b = 0; b < NB; b++)
                                tma_load_4d(sq + t * TILE + b * PT_HALF, &p.tma_q, 64 * b, 0, f.head, f.base + f.tok0 + t * tp, q_full);
                    }
                    for (int t = 0; t <= nmax && ok; t++) {
                        if (t < nmax) {
                            const int gi = kv + t, sl = gi & 1;
                            if (!(ok = at_wait(&k_empty[sl], ((gi >> 1) & 1) ^ 1, p.err))) break;
                            irx_mbar_expect_tx(&k_full[sl], TILE);
                            for (int b = 0; b < NB; b++)
                                tma_load_3d(sk + sl * TILE + b * PT_HALF, &p.tma_k, 64 * b, f.head, f.base + pt_key(f, t), &k_full[sl]);
                        }
                        if (t >= 1) {
                            const int gi = kv + t - 1, sl = gi & 1;
                            if (!(ok = at_wait(&v_empty[sl], ((gi >> 1) & 1) ^ 1, p.err))) break;
                            irx_mbar_expect_tx(&v_full[sl], TILE);
                            for (int b = 0; b < NB; b++)
                                tma_load_3d(sv + sl * TILE + b * PT_HALF, &p.tma_v, 64 * b, f.head, f.base + pt_key(f, t - 1), &v_full[sl]);
                        }
                    }
                    kv += nmax;
                }
                if (!f.n0) ok = 0;                            // that was the end
            }
            ok = __shfl_sync(0xffffffffu, ok, 0);
        }
      } else if (warp == 9) {
        if (elect_one()) {                                    // MMA: P0 V, S0', P1 V, S1' per key tile
            const uint32_t id_qk = umma_idesc_bf16(128, 128, 0), id_pv = umma_idesc_bf16(128, DP, 1);
            const uint32_t sq_a = irx_smem_u32(sq), sk_a = irx_smem_u32(sk), sv_a = irx_smem_u32(sv);
            bool ok = true;
            int kv = 0, it0 = 0, it1 = 0, uo0 = 0, uo1 = 0;
            for (int uc = 0; ok; uc++) {
                const int us = uc & 1;
                if (!(ok = at_wait(&u_full[us], (uc >> 1) & 1, p.err))) break;
                const int n0 = infos[us].n0, n1 = infos[us].n1, nmax = max(n0, n1);
                irx_mbar_arrive(&u_empty[us]);
                if (!n0) break;
                int sleft = n0 + n1;                          // score products of this unit still to issue
                if (!(ok = at_wait(q_full, uc & 1, p.err))) break;
                for (int j = -1; j < nmax && ok; j++) {
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        const int nt = t ? n1 : n0;
                        if (!ok) break;
                        if (j >= 0 && j < nt) {               // O_t (+)= P_t V_j
                            const int gi = kv + j;
                            if (j == 0 && (t ? uo1 : uo0) > 0 && !(ok = at_wait(&o_free[t], ((t ? uo1 : uo0) - 1) & 1, p.err))) break;
                            if (!(ok = at_wait(&p_full[t], ((t ? it1 : it0) + j) & 1, p.err))) break;
                            if (!(ok = at_wait(&v_full[gi & 1], (gi >> 1) & 1, p.err))) break;
                            if (!(ok = at_wait(&v_ok[gi & 1], (gi >> 1) & 1, p.err))) break;
                            tc_fence_after();
                            const uint32_t bv = sv_a + (gi & 1) * TILE;
#pragma unroll
                            for (int kk = 0; kk < 8; kk++)
                                umma_bf16_tmem_a(tbase + 256 + t * 128, tbase + t * 128 + kk * 8,
                                                 umma_desc_sw128(bv + kk * 16 * 128, PT_HALF, 1024), id_pv, (j | kk) != 0);
                            umma_commit(&pv_done[t]);
                        }
                        if (j + 1 < nt) {                     // S_t = Q_t K_{j+1}^T
                            const int gi = kv + j + 1;
                            if (!(ok = at_wait(&k_full[gi & 1], (gi >> 1) & 1, p.err))) break;
                            tc_fence_after();
                            const uint32_t aq = sq_a + t * TILE, bk = sk_a + (gi & 1) * TILE;
#pragma unroll
                            for (int kk = 0; kk < DP / 16; kk++)
                                umma_bf16(tbase + t * 128, at_kmajor_desc(aq, kk), at_kmajor_desc(bk, kk), id_qk, kk > 0);
                            umma_commit(&s_full[t]);
                            if (--sleft == 0) umma_commit(q_empty);
                        }
                    }
                    if (!ok) break;
                    if (j >= 0) umma_commit(&v_empty[(kv + j) & 1]);
                    if (j + 1 < nmax) umma_commit(&k_empty[(kv + j + 1) & 1]);
                }
                if (!ok) break;
                it0 += n0;
                uo0++;
                if (n1) { it1 += n1; uo1++; }
                kv += nmax;
            }
            umma_commit(done);
            at_wait(done, 0, p.err);
        }
        __syncwarp();
        asm volatile("bar.sync 1, 288;" ::: "memory");         // the softmax warps are done with TMEM
        tc_fence_after();
        tmem_dealloc(tbase, 512);
      } else {                                                // warps 10 and 11: 64 rows each of every value tile
        int ok = 1, kv = 0;
        for (int uc = 0; ok; uc++) {
            const int us = uc & 1;
            ok = __all_sync(0xffffffffu, at_wait(&u_full[us], (uc >> 1) & 1, p.err));
            if (!ok) break;
            const pt_info f = read(us);
            if (!f.n0) break;
            const int nmax = max(f.n0, f.n1);
            for (int j = 0; j < nmax; j++) {
                const int gi = kv + j;
                ok = __all_sync(0xffffffffu, at_wait(&v_full[gi & 1], (gi >> 1) & 1, p.err));
                if (!ok) break;
                if (pt_cut(p, f, j, f.tok0, f.end - 1)) {
                    const int seen = (j < f.nsink ? f.sk : f.end) - pt_key(f, j);
                    uint4 *v = reinterpret_cast<uint4 *>(sv + (gi & 1) * TILE);
                    uint32_t worst = 0;                       // the largest magnitudes of either half, as integers
#pragma unroll 4
                    for (int i = 0; i < NB * 16; i++) {       // 4 rows of 8 vectors a step
                        const int row = (warp - 10) * 64 + (i & 15) * 4 + (lane >> 3);
                        uint4 *at = v + (i >> 4) * (PT_HALF / 16) + row * 8 + (lane & 7);
                        const uint4 x = *at;
                        if (row >= seen) *at = make_uint4(0u, 0u, 0u, 0u);
                        else worst = __vmaxu2(__vmaxu2(worst, __vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu)),
                                              __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
                    }
                    // an exponent of all ones: find them
                    const bool odd = __any_sync(0xffffffffu, (worst & 0xffffu) >= 0x7f80u || worst >> 16 >= 0x7f80u);
                    if (odd)
                        for (int i = 0; i < NB * 16; i++) {
                            const int row = (warp - 10) * 64 + (i & 15) * 4 + (lane >> 3);
                            uint4 *at = v + (i >> 4) * (PT_HALF / 16) + row * 8 + (lane & 7);
                            const uint4 x = *at;
                            uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (int e = 0; e < 4; e++) w[e] &= ~__vcmpeq2(w[e] & 0x7f807f80u, 0x7f807f80u);
                            *at = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    if (odd) infos[us].dirty = 1;
                    fence_proxy_async_smem();
                }
                __syncwarp();
                if (lane == 0) irx_mbar_arrive(&v_ok[gi & 1]);
            }
            kv += nmax;
            if (lane == 0) irx_mbar_arrive(&u_empty[us]);
        }
      }
    } else {                                                   // softmax: warps 0-3 tile 0, 4-7 tile 1
        at_reg_inc();
        const int t = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t tl = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tS = tbase + tl + t * 128, tO = tbase + tl + 256 + t * 128;
        const float sl2 = fabsf(p.scale2);
        uint4 *stage = reinterpret_cast<uint4 *>(sv + 2 * TILE + 1024) + warp * 256;
        const int inv_g = (65535 + g) / g, tok_stride = p.heads * p.d;        // row / g = (row * inv_g) >> 16 below 128
        const int mytok = t * tp + r / g, myhead = r % g;      // within the unit, within the group
        bool ok = true;
        int it = 0;
        for (int uc = 0; ok; uc++) {
            const int us = uc & 1;
            ok = __all_sync(0xffffffffu, at_wait(&u_full[us], (uc >> 1) & 1, p.err));
            if (!ok) break;
            const pt_info f = read(us);
            if (!f.n0) break;
            const int n = t ? f.n1 : f.n0;
            const int tok = f.tok0 + mytok;
            const int first = f.tok0 + t * tp, last = min(first + tp, f.len) - 1;
            float m = -3.0e38f, l = 0.0f;
            for (int j = 0; j < n; j++) {
                ok = __all_sync(0xffffffffu, at_wait(&s_full[t], (it + j) & 1, p.err));
                if (!ok) break;
                tc_fence_after();
                float v[128];
                tmem_ld128(tS, v);
                if (p.scale2 < 0.0f) {
#pragma unroll
                    for (int c = 0; c < 128; c++) v[c] = -v[c];
                }
                const int kb = pt_key(f, j);
                const bool edge = j >= f.nsink && p.window && kb <= last - p.window;
                if (edge || j < f.nsink || kb + 127 > first) {
                    // the columns this row sees, as bits: up to `up`, and with a window from `low` on or before `sink`
                    const int up = (j < f.nsink ? min(tok, f.sk - 1) : tok) - kb, low = edge ? tok - p.window + 1 - kb : 0, sink = p.sinks - kb;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        uint32_t see = pt_below(up + 1 - 32 * k);
                        if (edge) see &= ~pt_below(low - 32 * k) | pt_below(sink - 32 * k);
#pragma unroll
                        for (int c = 0; c < 32; c++)
                            if (!(see & (1u << c))) v[k * 32 + c] = -INFINITY;
                    }
                }
                float mk[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    mk[k] = pt_max3(v[k * 32], v[k * 32 + 1], v[k * 32 + 2]);
#pragma unroll
                    for (int c = 3; c < 31; c += 2) mk[k] = pt_max3(mk[k], v[k * 32 + c], v[k * 32 + c + 1]);
                }
                mk[0] = pt_max3(mk[0], v[31], v[63]);
                mk[1] = pt_max3(mk[1], v[95], v[127]);
                float mnew = pt_max3(m, pt_max3(mk[0], mk[1], mk[2]) * sl2, mk[3] * sl2);
                mnew = mnew < INFINITY ? mnew : NAN;          // a score that is NaN or infinite: the row is NaN
                // O and l keep a maximum up to a factor of 256 behind (attn.cu); each row decides for itself, so that
                // its bits do not depend on the others of its warp
                const bool grown = !(mnew <= m + 8.0f);
                if (j == 0) {
                    m = mnew;
                } else if (__any_sync(0xffffffffu, grown)) {
                    ok = __all_sync(0xffffffffu, at_wait(&pv_done[t], (it + j - 1) & 1, p.err));
                    if (!ok) break;
                    tc_fence_after();
                    const float alpha = grown ? at_ex2(m - mnew) : 1.0f;
                    if (grown) m = mnew;
                    l *= alpha;
#pragma unroll 1
                    for (int cc = 0; cc < DP / 32; cc++) {
                        float o[32];
                        tmem_ld32(tO + cc * 32, o);
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] *= alpha;
                        tmem_st32(tO + cc * 32, o);
                    }
                }
                uint32_t pk[64];
                l += at_softmax_row(v, sl2, m, pk);
                tmem_st64(tS, pk);
                tc_fence_before();
                irx_mbar_arrive(&p_full[t]);
            }
            if (!ok) break;
            it += n;
            if (n) {
                ok = __all_sync(0xffffffffu, at_wait(&pv_done[t], (it - 1) & 1, p.err));
                if (!ok) break;
                tc_fence_after();
                const bool mine = r < tp * g && tok < f.len;
                const bool odd = infos[us].dirty != 0;
                const float inv = m > -2.9e38f ? 1.0f / l : NAN;      // (every score -infinity, or NaN: NaN)
                const int64_t orow = (int64_t)(f.base + tok) * p.heads + f.head * g + myhead;
                if (mine && p.lse) p.lse[orow] = m < -2.9e38f ? -INFINITY : (m + log2f(l)) * 0.6931471806f;
                __nv_bfloat16 *o_at = reinterpret_cast<__nv_bfloat16 *>(p.o) + ((int64_t)(f.base + first) * p.heads + f.head * g) * p.d;
                const int rows = (last + 1 - first) * g;      // of this tile
#pragma unroll 1
                for (int cc = 0; cc < DP / 32; cc++) {
                    float o[32];
                    tmem_ld32(tO + cc * 32, o);
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] *= inv;
                    if (odd && mine) {                        // the infinities and NaN this row sees in the cut tiles
                        for (int j = 0; j < n; j++) {
                            if (!pt_cut(p, f, j, f.tok0, f.end - 1)) continue;
                            const int kb = pt_key(f, j), ke = min(kb + 128, j < f.nsink ? f.sk : tok + 1);
                            for (int key = kb; key < ke; key++) {
                                if (p.window && key <= tok - p.window && key >= p.sinks) continue;
                                const __nv_bfloat16 *vr = reinterpret_cast<const __nv_bfloat16 *>(p.v) + (int64_t)(f.base + key) * p.kv_stride +
                                                          (int64_t)f.head * p.d + cc * 32;
#pragma unroll
                                for (int e = 0; e < 32; e++) {
                                    const float x = cc * 32 + e < p.d ? __bfloat162float(vr[e]) : 0.0f;
                                    if (!(fabsf(x) < INFINITY)) o[e] += x;
                                }
                            }
                        }
                    }
                    // 64 columns at a time through the warp's 4 KB, so that a store covers four rows' 128 bytes, not 32 rows'
                    // 16 (chunks of 16 bytes, swizzled by row)
                    uint4 *st = stage + lane * 8;
#pragma unroll
                    for (int j8 = 0; j8 < 4; j8++)
                        st[((cc & 1) * 4 + j8) ^ (lane & 7)] = make_uint4(at_pack_bf16(o[j8 * 8 + 0], o[j8 * 8 + 1]), at_pack_bf16(o[j8 * 8 + 2], o[j8 * 8 + 3]),
                                                                          at_pack_bf16(o[j8 * 8 + 4], o[j8 * 8 + 5]), at_pack_bf16(o[j8 * 8 + 6], o[j8 * 8 + 7]));
                    if (!(cc & 1)) continue;
                    __syncwarp();
                    const int col = (cc >> 1) * 64 + (lane & 7) * 8;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int row = i * 4 + (lane >> 3), full = (warp & 3) * 32 + row, tk = (full * inv_g) >> 16;
                        if (full < rows && col < p.d)
                            *reinterpret_cast<uint4 *>(o_at + tk * tok_stride + (full - tk * g) * p.d + col) = stage[row * 8 + ((lane & 7) ^ (row & 7))];
                    }
                    __syncwarp();
                }
                tc_fence_before();
                irx_mbar_arrive(&o_free[t]);
            }
            __syncwarp();
            if (lane == 0) irx_mbar_arrive(&u_empty[us]);
        }
        tc_fence_before();
        asm volatile("bar.arrive 1, 288;" ::: "memory");
    }
}

extern "C" __global__ void __launch_bounds__(AT_THREADS, 1) irx_prompt_tc_64(const __grid_constant__ irx_kprm_t p) { pt_body<64>(p); }
extern "C" __global__ void __launch_bounds__(AT_THREADS, 1) irx_prompt_tc_128(const __grid_constant__ irx_kprm_t p) { pt_body<128>(p); }
