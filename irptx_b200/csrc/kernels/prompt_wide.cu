// prompt_wide.cu -- attention over packed prompts on the tensor cores, bf16, for head sizes above 128, up to 256 in
// multiples of 8: prompt_tc.cu's roles with one tile of 128 rows and key tiles of 64.
//
// The accumulator takes half of TMEM and the queries 64 KB, so a CTA holds one tile of rows; what hides a tile's softmax
// there, the other tile's products, is here the tile's own: its scores have two buffers, and those of the next step
// are computed during a step's softmax. (For head sizes up to 128 this form is the slower one: a product 64 keys
// wide takes as long as one of 128, its queries' rows being what it waits for. 16001 tokens of 128: 2.38 against 2.10 ms.)
// Before it, these head sizes took FP32 units: 2000 tokens, 8 heads of 256, 1135 us, now 42; 8000 tokens, 16 heads on 4 of 256,
// 528 us (992 TFLOP/s), of 192, computed as 256, 487.
#pragma once
#include "prompt_tc.cu"

#define PT_KBLK 8192                        // a key or value tile's block of 64 columns: 64 rows

__device__ __forceinline__ int pw_key(const pt_info &f, int j) { return j < f.nsink ? 64 * j : f.lo + 64 * (j - f.nsink); }

__device__ __forceinline__ bool pw_cut(const irx_kprm_t &p, const pt_info &f, int j)
{
    const int kb = pw_key(f, j);
    return j < f.nsink || kb + 63 > f.tok0 || (p.window && kb <= f.end - 1 - p.window);
}

extern "C" __global__ void __launch_bounds__(256, 1) irx_prompt_tc_256(const __grid_constant__ irx_kprm_t p)
{
    constexpr int DP = 256;
    constexpr int NB = DP / 64, RING = IRX_PR_WIDE_RING, QT = NB * PT_HALF, KT = NB * PT_KBLK, W = 4;      // W: the first of the last four warps
    irx_pdl_enter();
    extern __shared__ __align__(1024) unsigned char pt_smem[];
    unsigned char *sq = pt_smem, *sk = sq + QT, *sv = sk + RING * KT;
    if (irx_smem_u32(pt_smem) & 1023u) {
        if (threadIdx.x == 0) atomicOr(p.err, IRX_KERR_TIMEOUT);
        return;
    }
    uint64_t *bars = reinterpret_cast<uint64_t *>(sv + RING * KT);
    uint64_t *q_full = bars, *q_empty = bars + 1, *done = bars + 2, *u_full = bars + 3, *u_empty = bars + 5, *o_free = bars + 7;
    uint64_t *k_full = bars + 8, *k_empty = k_full + RING, *v_full = k_empty + RING, *v_empty = v_full + RING, *v_ok = v_empty + RING;
    uint64_t *s_full = v_ok + RING, *p_full = s_full + 2, *pv_done = p_full + 2;                // by buffer
    constexpr int NBAR = 8 + 5 * RING + 6;
    uint32_t *tslot = reinterpret_cast<uint32_t *>(bars + NBAR);
    volatile pt_info *infos = reinterpret_cast<volatile pt_info *>(bars + NBAR + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = p.group, tp = 128 / g;
    if (threadIdx.x < NBAR) {
        const int i = threadIdx.x, x = i - (8 + 4 * RING);    // x: from v_ok on
        // o_free, p_full: the rows; u_empty: the products' warp, the softmax warps and the two value warps
        irx_mbar_init(&bars[i], i == 7 || (x >= RING + 2 && x < RING + 4) ? 128 : i == 5 || i == 6 ? 7 : x >= 0 && x < RING ? 2 : 1);
        irx_fence_mbar_init();
        if (i == 0) {
            tma_prefetch_desc(&p.tma_q);
            tma_prefetch_desc(&p.tma_k);
            tma_prefetch_desc(&p.tma_v);
        }
    }
    if (warp == W + 1) tmem_alloc(tslot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = *tslot;
    auto read = [&](int us) {
        pt_info f;
        f.base = infos[us].base; f.len = infos[us].len; f.tok0 = infos[us].tok0; f.head = infos[us].head;
        f.lo = infos[us].lo; f.nsink = infos[us].nsink; f.n0 = infos[us].n0; f.n1 = 0; f.sk = infos[us].sk;
        f.end = infos[us].end; f.dirty = 0;
        return f;
    };
    if (warp >= W) {
      if (warp == W) {                                        // units and loads
        int kv = 0;
        const pr_list list = pr_start(p, pr_rows{1, tp});
        int ok = 1;
        for (int uc = 0; ok; uc++) {
            const int us = uc & 1;
            const int64_t u = pr_turn(uc);
            pt_info f = {};
            if (u < list.units) {
                const pr_unit un = pr_find(p, list, u);
                f.base = un.base; f.len = un.len; f.head = un.head;
                f.tok0 = un.tile * tp;
                f.end = min(f.tok0 + tp, f.len);
                f.lo = p.window ? max(0, f.tok0 - p.window + 1) : 0;
                f.sk = min(p.sinks, f.lo);
                f.nsink = (f.sk + 63) / 64;
                f.n0 = f.nsink + (f.end - f.lo + 63) / 64;
            }
            if (elect_one()) {
                ok = at_wait(&u_empty[us], ((uc >> 1) & 1) ^ 1, p.err);
                if (ok) {
                    infos[us].base = f.base; infos[us].len = f.len; infos[us].tok0 = f.tok0; infos[us].head = f.head;
                    infos[us].lo = f.lo; infos[us].nsink = f.nsink; infos[us].n0 = f.n0;
                    infos[us].sk = f.sk; infos[us].end = f.end; infos[us].dirty = 0;
                    irx_mbar_arrive(&u_full[us]);
                }
                if (ok && f.n0) {
                    const int n = f.n0;
                    if (uc > 0) ok = at_wait(q_empty, (uc - 1) & 1, p.err);
                    if (ok) {
                        irx_mbar_expect_tx(q_full, (uint32_t)(NB * tp * g * 128));
                        for (int b = 0; b < NB; b++)
                            tma_load_4d(sq + b * PT_HALF, &p.tma_q, 64 * b, 0, f.head, f.base + f.tok0, q_full);
                    }
                    for (int t = 0; t <= n && ok; t++) {   // K0, K1, V0, K2, V1, ...: in the order of their use
                        if (t < n) {
                            const int gi = kv + t, sl = gi % RING;
                            if (!(ok = at_wait(&k_empty[sl], ((gi / RING) & 1) ^ 1, p.err))) break;
                            irx_mbar_expect_tx(&k_full[sl], KT);
                            for (int b = 0; b < NB; b++)
                                tma_load_3d(sk + sl * KT + b * PT_KBLK, &p.tma_k, 64 * b, f.head, f.base + pw_key(f, t), &k_full[sl]);
                        }
                        if (t >= 1) {
                            const int gi = kv + t - 1, sl = gi % RING;
                            if (!(ok = at_wait(&v_empty[sl], ((gi / RING) & 1) ^ 1, p.err))) break;
                            irx_mbar_expect_tx(&v_full[sl], KT);
                            for (int b = 0; b < NB; b++)
                                tma_load_3d(sv + sl * KT + b * PT_KBLK, &p.tma_v, 64 * b, f.head, f.base + pw_key(f, t - 1), &v_full[sl]);
                        }
                    }
                    kv += n;
                }
                if (!f.n0) ok = 0;                            // that was the end
            }
            ok = __all_sync(0xffffffffu, ok);
            kv = __reduce_max_sync(0xffffffffu, kv);           // (the elected lane counted)
        }
      } else if (warp == W + 1) {
        if (elect_one()) {                                    // the products
            const uint32_t id_qk = umma_idesc_bf16(128, 64, 0), id_pv = umma_idesc_bf16(128, DP, 1);
            const uint32_t sq_a = irx_smem_u32(sq), sk_a = irx_smem_u32(sk), sv_a = irx_smem_u32(sv);
            bool ok = true;
            int kv = 0, uo = 0, sleft = 0;
            auto scores = [&](int gi) {                       // of key tile gi, which is the block's step gi too
                if (!(ok = at_wait(&k_full[gi % RING], (gi / RING) & 1, p.err))) return;
                tc_fence_after();
                const uint32_t bk = sk_a + (gi % RING) * KT;
#pragma unroll
                for (int kk = 0; kk < DP / 16; kk++)
                    umma_bf16(tbase + (gi & 1) * 64, umma_desc_sw128(sq_a + (kk >> 2) * PT_HALF + (kk & 3) * 32, 16, 1024),
                              umma_desc_sw128(bk + (kk >> 2) * PT_KBLK + (kk & 3) * 32, 16, 1024), id_qk, kk > 0);
                umma_commit(&s_full[gi & 1]);
                umma_commit(&k_empty[gi % RING]);
                if (--sleft == 0) umma_commit(q_empty);
            };
            for (int uc = 0; ok; uc++) {
                const int us = uc & 1;
                if (!(ok = at_wait(&u_full[us], (uc >> 1) & 1, p.err))) break;
                const int n = infos[us].n0;
                irx_mbar_arrive(&u_empty[us]);
                if (!n) break;
                sleft = n;                                    // score products of this unit still to issue
                if (!(ok = at_wait(q_full, uc & 1, p.err))) break;
                scores(kv);
                if (ok && n > 1) scores(kv + 1);
                for (int j = 0; j < n && ok; j++) {
                    const int gi = kv + j, b = gi & 1;
                    if (j == 0 && uo > 0 && !(ok = at_wait(o_free, (uo - 1) & 1, p.err))) break;
                    if (!(ok = at_wait(&p_full[b], (gi >> 1) & 1, p.err))) break;
                    if (!(ok = at_wait(&v_full[gi % RING], (gi / RING) & 1, p.err))) break;
                    if (!(ok = at_wait(&v_ok[gi % RING], (gi / RING) & 1, p.err))) break;
                    tc_fence_after();
                    const uint32_t bv = sv_a + (gi % RING) * KT;
#pragma unroll
                    for (int kk = 0; kk < 4; kk++)            // O (+)= P V
                        umma_bf16_tmem_a(tbase + 256, tbase + b * 64 + kk * 8, umma_desc_sw128(bv + kk * 16 * 128, PT_KBLK, 1024), id_pv,
                                         (j | kk) != 0);
                    umma_commit(&pv_done[b]);
                    umma_commit(&v_empty[gi % RING]);
                    if (j + 2 < n) scores(gi + 2);
                }
                uo++;
                kv += n;
            }
            umma_commit(done);
            at_wait(done, 0, p.err);
        }
        __syncwarp();
        asm volatile("bar.sync 1, %0;" :: "n"(160) : "memory");      // the softmax warps are done with TMEM
        tc_fence_after();
        tmem_dealloc(tbase, 512);
      } else {                                                // 32 rows each of every value tile
        int ok = 1, kv = 0;
        for (int uc = 0; ok; uc++) {
            const int us = uc & 1;
            ok = __all_sync(0xffffffffu, at_wait(&u_full[us], (uc >> 1) & 1, p.err));
            if (!ok) break;
            const pt_info f = read(us);
            if (!f.n0) break;
            for (int j = 0; j < f.n0; j++) {
                const int gi = kv + j;
                ok = __all_sync(0xffffffffu, at_wait(&v_full[gi % RING], (gi / RING) & 1, p.err));
                if (!ok) break;
                if (pw_cut(p, f, j)) {
                    const int seen = (j < f.nsink ? f.sk : f.end) - pw_key(f, j);
                    uint4 *v = reinterpret_cast<uint4 *>(sv + (gi % RING) * KT);
                    uint32_t worst = 0;                       // the largest magnitudes of either half, as integers
#pragma unroll 4
                    for (int i = 0; i < NB * 8; i++) {        // 4 rows of 8 vectors a step
                        const int row = (warp - W - 2) * 32 + (i & 7) * 4 + (lane >> 3);
                        uint4 *at = v + (i >> 3) * (PT_KBLK / 16) + row * 8 + (lane & 7);
                        const uint4 x = *at;
                        if (row >= seen) *at = make_uint4(0u, 0u, 0u, 0u);
                        else worst = __vmaxu2(__vmaxu2(worst, __vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu)),
                                              __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
                    }
                    // an exponent of all ones: find them
                    const bool odd = __any_sync(0xffffffffu, (worst & 0xffffu) >= 0x7f80u || worst >> 16 >= 0x7f80u);
                    if (odd)
                        for (int i = 0; i < NB * 8; i++) {
                            const int row = (warp - W - 2) * 32 + (i & 7) * 4 + (lane >> 3);
                            uint4 *at = v + (i >> 3) * (PT_KBLK / 16) + row * 8 + (lane & 7);
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
                if (lane == 0) irx_mbar_arrive(&v_ok[gi % RING]);
            }
            kv += f.n0;
            if (lane == 0) irx_mbar_arrive(&u_empty[us]);
        }
      }
    } else {                                                   // softmax: four warps a tile
        const int r = warp * 32 + lane;
        const uint32_t tS = tbase + ((uint32_t)(warp * 32) << 16), tO = tS + 256;
        const float sl2 = pt_sl2(p.scale2);
        uint4 *stage = reinterpret_cast<uint4 *>(sv + RING * KT + 1024) + warp * 256;
        const int inv_g = (65535 + g) / g, tok_stride = p.heads * p.d;        // row / g = (row * inv_g) >> 16 below 128
        const int mytok = r / g, myhead = r % g;               // within the unit, within the group
        bool ok = true;
        int it = 0;
        for (int uc = 0; ok; uc++) {
            const int us = uc & 1;
            ok = __all_sync(0xffffffffu, at_wait(&u_full[us], (uc >> 1) & 1, p.err));
            if (!ok) break;
            const pt_info f = read(us);
            if (!f.n0) break;
            const int n = f.n0, tok = f.tok0 + mytok, first = f.tok0, last = f.end - 1;
            float m = -3.0e38f, l = 0.0f;
            for (int j = 0; j < n; j++) {
                const int i = it + j, b = i & 1;
                ok = __all_sync(0xffffffffu, at_wait(&s_full[b], (i >> 1) & 1, p.err));
                if (!ok) break;
                tc_fence_after();
                const int kb = pw_key(f, j);
                const bool edge = j >= f.nsink && p.window && kb <= last - p.window;
                const int up = (j < f.nsink ? min(tok, f.sk - 1) : tok) - kb, low = edge ? tok - p.window + 1 - kb : -0x40000000;
                auto done_before = [&]() {                    // the product of the step before, which writes O
                    ok = __all_sync(0xffffffffu, at_wait(&pv_done[b ^ 1], ((i - 1) >> 1) & 1, p.err));
                    tc_fence_after();
                    return ok;
                };
                const pt_row row = {tS + b * 64, tO, up, low, p.sinks - kb, edge || j < f.nsink || kb + 63 > first, !(p.scale2 > 0.0f), j == 0, p.scale2, sl2};
                pt_step<DP, 64>(row, m, l, done_before);
                if (!ok) break;
                tc_fence_before();
                irx_mbar_arrive(&p_full[b]);
            }
            if (!ok) break;
            it += n;
            {
                ok = __all_sync(0xffffffffu, at_wait(&pv_done[(it - 1) & 1], ((it - 1) >> 1) & 1, p.err));
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
                            if (!pw_cut(p, f, j)) continue;
                            const int kb = pw_key(f, j), ke = min(kb + 64, j < f.nsink ? f.sk : tok + 1);
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
                irx_mbar_arrive(o_free);
            }
            __syncwarp();
            if (lane == 0) irx_mbar_arrive(&u_empty[us]);
        }
        tc_fence_before();
        asm volatile("bar.arrive 1, %0;" :: "n"(160) : "memory");
    }
}

